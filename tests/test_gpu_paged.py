"""The paged key/value cache: bookkeeping, append and attention against plain
forms in 64 bits, and a step of them together.

Bars of the attention, per element, from its formula: with A = sum_j w_j |v_j| / sum_j w_j
  - a score is a sum of Dh products in fp32, off by at most Dh 2^-24 sum |q k| scale,
    and fp32's log2(e), scale, maximum and exponential add under 2^-22 (1 + |s|): a
    weight is off by e^d - 1 for the sum d of these, and the sum of the weights too;
  - a probability rounded to 16 bits: half a unit, 2^-8 (bf16) or 2^-11 (f16), or as
    two terms 2^-16 and 2^-22, of A;
  - fp32 sums of the keys: (keys / 64 + 128) 2^-24 of A (tiles are summed one by one);
  - the result's own rounding, 2^-8, 2^-11 or 2^-24 of the result (f16: at least half
    of its least number, 2^-25).
"""
import numpy as np
import pytest

from janis_amd import _lib, synth
from janis_amd.engine import BF16, F16, F32, I32, HipBackend, JanisHipError
from tests.conftest import Graph, put, step

pytestmark = pytest.mark.gpu
HALF = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: 2.0 ** -24}  # half a unit, relative
NAN = np.float32(np.nan)


def rounded(a, dt):
    a = np.asarray(a, np.float32)
    if dt == BF16:
        return synth.bf16_bits_to_f32(synth.f32_to_bf16_bits(a))
    return a.astype(np.float16).astype(np.float32) if dt == F16 else a


def up(hip, a, dt):
    a = np.asarray(a, np.float32)
    if dt == BF16:
        return hip.FromBF16Bits(synth.f32_to_bf16_bits(a), *a.shape)
    return hip.FromRaw(F16, a.astype(np.float16), *a.shape) if dt == F16 else hip.FromFloats(a, *a.shape)


def ints(hip, a):
    a = np.asarray(a, np.int32)
    return hip.FromRaw(I32, a, *a.shape) if a.size else hip.empty(I32, *a.shape)


# ---- bookkeeping -------------------------------------------------------------------

def plan_ref(new, kv, page, tables, free, count, rows, n_pages):
    """jh_paged_plan one request and page after the other."""
    tables, free, R = tables.copy(), free.copy(), len(new)
    B = tables.shape[1]
    blocks = lambda n: -(-n // page)  # noqa: E731
    none = np.full(rows, -1, np.int32)
    fail = lambda st: (kv.copy(), count, np.zeros(R + 1, np.int32), none, none, st, tables, free)  # noqa: E731
    if any(k < 0 or k > B * page or k + max(0, n) > B * page for n, k in zip(new, kv)):
        return fail(1)
    if sum(max(0, n) for n in new) > rows:
        return fail(2)
    back = [int(tables[r][j]) for r in range(R) if new[r] < 0 for j in range(blocks(kv[r]))]
    want = sum(blocks(k + n) - blocks(k) for n, k in zip(new, kv) if n >= 0)
    if count < 0 or count > n_pages or want > count + len(back):
        return fail(3)
    stack = list(free[:count]) + back
    if len(stack) > n_pages or any(p < 0 or p >= n_pages for p in back + list(stack[len(stack) - want:])):
        return fail(4)
    free[count:len(stack)] = back
    top, after, starts, pos, slots = len(stack), [], [0], [], []
    for r in range(R):
        for p in range(kv[r], kv[r] + max(0, int(new[r]))):
            if p % page == 0:
                top -= 1
                tables[r][p // page] = free[top]
            pos.append(p)
            slots.append(tables[r][p // page] * page + p % page)
        after.append(0 if new[r] < 0 else kv[r] + new[r])
        starts.append(len(pos))
    pad = [-1] * (rows - len(pos))
    return np.array(after), top, np.array(starts), np.array(pos + pad), np.array(slots + pad), 0, tables, free


def plan_case(seed, R, page, rows, hi=200, done=0.1, spare=20):
    rng = np.random.default_rng(seed)
    kv = rng.integers(0, hi, R).astype(np.int32)
    kv[::3] -= kv[::3] % page  # page borders
    new = rng.integers(0, 4, R).astype(np.int32)
    new[rng.random(R) < done] = -1
    if R > 2:
        new[R // 2] = max(0, rows - int(np.maximum(new, 0).sum()) - 3 + max(0, new[R // 2]))
    blocks = -(-kv // page)
    n_pages = int(blocks.sum() + np.maximum(new, 0).sum() // page + R + spare)
    order = rng.permutation(n_pages).astype(np.int32)
    B = int((-(-(kv + np.maximum(new, 0)) // page)).max()) + 2
    tables = np.full((R, B), -7, np.int32)
    at = 0
    for r in range(R):
        tables[r, :blocks[r]] = order[at:at + blocks[r]]
        at += blocks[r]
    free = np.full(n_pages, -9, np.int32)
    free[:n_pages - at] = order[at:]
    return new, kv, tables, free, n_pages - at, n_pages


def run_plan(hip, new, kv, page, tables, free, count, rows, in_place=False):
    d = [ints(hip, x) for x in (new, kv, tables, free, [count])]
    R = len(new)
    out = [ints(hip, np.full(n, -5)) for n in (R, 1, R + 1, rows, rows, 1)]
    if in_place:
        out[0], out[1] = d[1], d[4]
    hip.PagedPlan(d[0], d[1], page, d[2], d[3], d[4], out=tuple(out))
    got = [hip.Ints(t) if t.numel else np.zeros(t.shape, np.int32) for t in out]
    return got[0], got[1][0], got[2], got[3], got[4], got[5][0], hip.Ints(d[2]), hip.Ints(d[3])


def same_plan(got, want):
    for name, g, w in zip(("kv", "count", "starts", "positions", "slots", "status", "tables", "free"), got, want):
        assert np.array_equal(g, w), (name, g, w)


@pytest.mark.parametrize("R,page,rows", [(1, 16, 1), (1, 1, 40), (3, 4, 30), (64, 16, 200), (65, 16, 1025), (700, 32, 3000),
                                         (1025, 8, 2500), (2048, 64, 9000)])
@pytest.mark.parametrize("in_place", [False, True])
def test_plan(hip, R, page, rows, in_place):
    new, kv, tables, free, count, n_pages = plan_case(R + page, R, page, max(rows, 4 * R))
    rows = max(rows, 4 * R)
    step(f"jh_paged_plan R={R} page={page} rows={rows} in_place={in_place}")
    want = plan_ref(new, kv, page, tables, free, count, rows, n_pages)
    assert want[5] == 0
    same_plan(run_plan(hip, new, kv, page, tables, free, count, rows, in_place), want)


def test_plan_everything_at_its_end(hip):
    """No requests; only finished ones; no free page left behind; a full table."""
    step("jh_paged_plan at its ends")
    z = np.zeros(0, np.int32)
    same_plan(run_plan(hip, z, z, 16, np.zeros((0, 3), np.int32), np.arange(5), 5, 7),
              plan_ref(z, z, 16, np.zeros((0, 3), np.int32), np.arange(5, dtype=np.int32), 5, 7, 5))
    new, kv = np.array([-1, -1, -2], np.int32), np.array([33, 0, 16], np.int32)
    tables = np.array([[4, 2, 0], [9, 9, 9], [1, 9, 9]], np.int32)
    free = np.array([3, -1, -1, -1, -1], np.int32)
    want = plan_ref(new, kv, 16, tables, free, 1, 2, 5)
    assert want[1] == 5 and list(want[7]) == [3, 4, 2, 0, 1]
    same_plan(run_plan(hip, new, kv, 16, tables, free, 1, 2), want)
    new, kv = np.array([31, 17], np.int32), np.array([17, 15], np.int32)  # 3 of 3 and 2 of 3 blocks: one page each
    tables = np.array([[4, 2, -1], [1, -1, -1]], np.int32)
    free = np.array([3, 0, -1, -1, -1], np.int32)
    want = plan_ref(new, kv, 16, tables, free, 2, 48, 5)
    assert want[5] == 0 and want[1] == 0 and want[3][-1] == 31
    same_plan(run_plan(hip, new, kv, 16, tables, free, 2, 48), want)


@pytest.mark.parametrize("what,status", [("kv below 0", 1), ("kv past the table", 1), ("new past the table", 1), ("rows", 2),
                                         ("pages", 3), ("count", 3), ("table", 4), ("stack", 4), ("room", 4)])
@pytest.mark.parametrize("in_place", [False, True])
def test_plan_refused_on_the_device(hip, what, status, in_place):
    """A step that cannot be done leaves everything as it was and plans no row."""
    new, kv = np.array([5, -1, 40, 1], np.int32), np.array([30, 20, 16, 7], np.int32)
    tables = np.array([[0, 1, -1, -1], [2, 3, -1, -1], [4, -1, -1, -1], [5, -1, -1, -1]], np.int32)
    free, count, rows = np.array([6, 7, 8, -1, -1, -1, -1, -1, -1, -1], np.int32), 3, 46
    assert plan_ref(new, kv, 16, tables, free, count, rows, 10)[5] == 0
    if what == "kv below 0": kv[3] = -1
    if what == "kv past the table": kv[1] = 65
    if what == "new past the table": new[0] = 35
    if what == "rows": rows = 45
    if what == "pages": count = 1
    if what == "count": count = 11
    if what == "table": tables[1, 1] = 10
    if what == "stack": free[2] = -1
    if what == "room": free[3:], count = 9, 9
    want = plan_ref(new, kv, 16, tables, free, count, rows, 10)
    assert want[5] == status
    step(f"jh_paged_plan refuses: {what}")
    same_plan(run_plan(hip, new, kv, 16, tables, free, count, rows, in_place), want)
    hip.SetChecks(True)
    try:
        with pytest.raises(JanisHipError) as e:
            run_plan(hip, new, kv, 16, tables, free, count, rows)
        assert e.value.code == _lib.JH_ERR_INVALID
    finally:
        hip.SetChecks(False)


# ---- append --------------------------------------------------------------------------

def append_ref(qkv, Hq, Hk, D, qw, kw, eps, angle, slots, n_slots):
    """{row: (q [Hq, D], k [Hk, D], v [Hk, D])} in 64 bits, before the pages' rounding."""
    T = qkv.shape[0]
    x = qkv.astype(np.float64).reshape(T, Hq + 2 * Hk, D)

    def head(x, w):
        if w is not None:
            x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
        if angle is None:
            return x
        c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
        a, b = x[..., :D // 2], x[..., D // 2:]
        return np.concatenate([a * c - b * s, a * s + b * c], -1)

    return head(x[:, :Hq], qw), head(x[:, Hq:Hq + Hk], kw), x[:, Hq + Hk:]


@pytest.mark.parametrize("T,Hq,Hk,D,page,act,cache,norm,rope", [
    (1, 32, 8, 128, 16, BF16, BF16, "both", "base"), (1, 1, 1, 64, 1, F32, F16, "both", "base"),
    (7, 5, 1, 256, 4, F32, BF16, "both", "freqs"), (33, 16, 2, 64, 32, BF16, F16, "q", "base"),
    (300, 8, 8, 128, 64, F32, F16, "none", "base"), (65, 0, 3, 128, 16, F32, BF16, "k", "none"),
    (20, 40, 4, 256, 128, BF16, F16, "both", "none"), (600, 4, 2, 64, 16, F32, BF16, "both", "scaled")])
def test_append(hip, T, Hq, Hk, D, page, act, cache, norm, rope):
    """Rows apart by more than a row, slots in any order, some of them none (-1, or
    past the pages): what no slot names stays as it was. One rounding to the
    pages' dtype beside fp32's own: the norm's sum of D squares, a root, a
    quotient, three products and a sum, (D / 2 + 10) 2^-24 of the two rotated
    features' size, and the angle's, exact in double up to 2^-30 here."""
    rng = np.random.default_rng(T * 31 + D)
    n_pages, width = -(-T // page) + 3, (Hq + 2 * Hk) * D
    qkv = rounded(3 * rng.standard_normal((T, width + 24)), act)
    ws = [rounded(rng.standard_normal(D) * 0.3 + 1, F16) if norm in ("both", n) else None for n in ("q", "k")]
    pos = rng.integers(0, 200000, T).astype(np.int32)
    slots = rng.permutation(n_pages * page)[:T].astype(np.int32)
    slots[T // 2] = -1 if T > 1 else slots[0]
    if T > 10:
        slots[3], slots[T - 1], slots[5] = n_pages * page, -1, -(2 ** 31)
    base, scale, freqs = {"base": (1e6, 1.0, None), "scaled": (1e4, 0.25, None), "none": (0.0, 1.0, None),
                          "freqs": (7.0, 1.0, (3.0 ** np.arange(D // 2).clip(0, 30)).astype(np.float32))}[rope]
    inv = 1.0 / freqs.astype(np.float64) if freqs is not None else np.float64(np.float32(base) or 1.0) ** (-2.0 * np.arange(D // 2) / D)
    angle = None if rope == "none" else pos[:, None].astype(np.float64) * scale * inv
    eps = np.float32(1e-6)
    q, k, v = append_ref(qkv[:, :width], Hq, Hk, D, *ws, np.float64(eps), angle, slots, n_pages * page)
    old = rounded(rng.standard_normal((2, n_pages, Hk, page, D)), cache)
    old_q = rounded(rng.standard_normal((T, max(Hq, 1), D)), cache)
    X = hip._view(up(hip, qkv, act), (T, width), (width + 24, 1))
    kp, vp, qo = up(hip, old[0], cache), up(hip, old[1], cache), up(hip, old_q, cache)
    F = hip.FromFloats(freqs) if freqs is not None else None
    W = [up(hip, w, F16) if w is not None else None for w in ws]
    step(f"jh_paged_qk_norm_rope_append T={T} Hq={Hq} Hk={Hk} D={D} page={page} {act} {cache} {norm} {rope}")
    got_q = hip.PagedQKNormRoPEAppend(X, Hq, Hk, *W, float(eps), base, scale, ints(hip, pos) if angle is not None else None,
                                      ints(hip, slots), kp, vp, freqs=F, q_out=qo if Hq else None)
    assert (got_q is None) == (Hq == 0)
    gk, gv, gq = hip.Floats(kp), hip.Floats(vp), hip.Floats(qo)
    want_k, want_v, want_q = old[0].astype(np.float64), old[1].astype(np.float64), old_q.astype(np.float64)
    size_k, size_q = np.zeros_like(want_k), np.zeros_like(want_q)
    both = lambda x: np.tile(np.hypot(x[..., :D // 2], x[..., D // 2:]), 2)  # noqa: E731
    for t in range(T):
        if 0 <= slots[t] < n_pages * page:
            p, r = divmod(int(slots[t]), page)
            want_k[p, :, r], want_v[p, :, r], size_k[p, :, r] = k[t], rounded(v[t], cache), both(k[t])
            if Hq:
                want_q[t], size_q[t] = q[t], both(q[t])
    assert np.array_equal(gv, want_v.astype(np.float32))
    tiny = 2.0 ** -25 if cache == F16 else 0.0
    for g, w, size in ((gk, want_k, size_k), (gq, want_q, size_q)):
        bar = (HALF[cache] * np.abs(w) * 1.01 + tiny) * (size > 0) + (D / 2 + 10) * 2.0 ** -24 * size
        assert (np.abs(g - w) <= bar).all(), np.max(np.abs(g - w) - bar)


def test_append_as_one_token(hip):
    """One row has the keys, values and queries of jh_qk_norm_rope_append, up to one
    unit of the pages' dtype (its angles are rounded to fp32: at position 50 by
    at most 2^-19, a tenth of a unit of f16)."""
    Hq, Hk, D, page, pos = 8, 2, 128, 16, 50
    rng = np.random.default_rng(5)
    qkv = up(hip, 2 * rng.standard_normal((1, (Hq + 2 * Hk) * D)), F32)
    qw, kw = (up(hip, rng.standard_normal(D), BF16) for _ in range(2))
    kc, vc = (up(hip, np.zeros((1, Hk, 64, D)), F16) for _ in range(2))
    kp, vp = (up(hip, np.zeros((4, Hk, page, D)), F16) for _ in range(2))
    step("append of one row beside jh_qk_norm_rope_append")
    q1 = hip.Floats(hip.QKNormRoPEAppend(qkv, Hq, Hk, qw, kw, 1e-6, 1e6, 1.0, pos, kc, vc))
    q2 = hip.Floats(hip.PagedQKNormRoPEAppend(qkv, Hq, Hk, qw, kw, 1e-6, 1e6, 1.0, ints(hip, [pos]), ints(hip, [pos]), kp, vp))
    k1, k2 = hip.Floats(kc)[0, :, pos], hip.Floats(kp)[3, :, pos % page]
    assert np.array_equal(hip.Floats(vc)[0, :, pos], hip.Floats(vp)[3, :, pos % page])
    for a, b in ((q1.reshape(-1), q2.reshape(-1)), (k1.reshape(-1), k2.reshape(-1))):
        assert (np.abs(a - b) <= 2.0 ** -10 * np.maximum(np.abs(a), 2.0 ** -3)).all()


# ---- attention ------------------------------------------------------------------------

class Paged:
    """Requests of (new, keys) with random queries and pages in a shuffled pool
    whose other slots and pages are NaN."""

    def __init__(self, hip, lens, Hq, Hk, D, page, dt, seed=0, spread=1.5, pad=0, extra_blocks=2, k=None, v=None):
        rng = np.random.default_rng(seed + 1000 * D + Hq)
        self.lens, self.Hq, self.Hk, self.D, self.page, self.dt, self.scale = lens, Hq, Hk, D, page, dt, D ** -0.5
        blocks = [-(-kv // page) for _, kv in lens]
        self.n_pages = sum(blocks) + 3
        order = rng.permutation(self.n_pages)
        self.tables = np.full((len(lens), max(blocks, default=0) + extra_blocks), 2 ** 30, np.int32)
        self.starts = np.concatenate([[0], np.cumsum([n for n, _ in lens])]).astype(np.int32)
        self.T = int(self.starts[-1]) + pad
        self.q = rounded(spread * rng.standard_normal((self.T, Hq, D)), dt)
        self.k = k or [rounded(spread * rng.standard_normal((Hk, kv, D)), dt) for _, kv in lens]
        self.v = v or [rounded(rng.standard_normal((Hk, kv, D)), dt) for _, kv in lens]
        at = 0
        pools = np.full((2, self.n_pages, Hk, page, D), np.nan, np.float32)
        for r, (_, kv) in enumerate(lens):
            mine = order[at:at + blocks[r]]
            self.tables[r, :blocks[r]] = mine
            at += blocks[r]
            for j, p in enumerate(mine):
                n = min(page, kv - j * page)
                pools[0, p, :, :n] = self.k[r][:, j * page:j * page + n]
                pools[1, p, :, :n] = self.v[r][:, j * page:j * page + n]
        self.pools = pools
        self.hip = hip
        self.Q, self.K, self.V = up(hip, self.q, dt), up(hip, pools[0], dt), up(hip, pools[1], dt)
        self.TAB, self.ST = ints(hip, self.tables), ints(hip, self.starts)
        self.KV = ints(hip, [kv for _, kv in lens])

    def ref(self, out_dt):
        """(expected, bar) [T, Hq, D]; rows behind the last: NaN."""
        G = self.Hq // self.Hk
        want, bar = np.full((2, self.T, self.Hq, self.D), np.nan)
        for r, (n, kv) in enumerate(self.lens):
            p_half = HALF[self.dt] ** 2 if out_dt == F32 or n * G <= 64 else HALF[self.dt]
            for i in range(n):
                seen = kv - n + i + 1
                t = self.starts[r] + i
                if seen <= 0:
                    want[t], bar[t] = 0.0, 0.0
                    continue
                for h in range(self.Hk):
                    k, v = self.k[r][h, :seen].astype(np.float64), self.v[r][h, :seen].astype(np.float64)
                    q = self.q[t, h * G:(h + 1) * G].astype(np.float64)
                    with np.errstate(all="ignore"):
                        s = q @ k.T * self.scale
                        rest = (np.abs(q) @ np.abs(k).T).max(-1) * self.scale
                        w = np.exp(s - s.max(-1, keepdims=True))
                        w /= w.sum(-1, keepdims=True)
                        o, A = w @ v, w @ np.abs(v)
                        d = self.D * 2.0 ** -24 * rest + 2.0 ** -22 * (1 + np.abs(s).max(-1))
                        rel = 2 * np.expm1(2 * d) + p_half + (seen / 64 + 128) * 2.0 ** -24
                        want[t, h * G:(h + 1) * G] = o
                        bar[t, h * G:(h + 1) * G] = A * rel[:, None] * 1.01 + HALF[out_dt] * np.abs(o) * 1.01 + (2.0 ** -25 if out_dt == F16 else 0)
        return want, bar

    def run(self, out_dt, max_new=None, **kw):
        if max_new is None:
            max_new = max([n for n, _ in self.lens], default=0)
        fill = up(self.hip, np.full((self.T, self.Hq, self.D), 7.0), out_dt)
        a = dict(q=self.Q, k=self.K, v=self.V)
        a.update(kw)
        out = self.hip.PagedAttention(a["q"], a["k"], a["v"], self.TAB, self.ST, self.KV, self.scale, maxNew=max_new, out=fill)
        got = self.hip.Floats(out)
        assert (got[self.starts[-1]:] == 7.0).all(), "rows behind the last"
        return got


def close(got, want, bar, rows):
    g, w, b = got[:rows].astype(np.float64), want[:rows], bar[:rows]
    off = np.abs(g - w) - b
    assert (off <= 0).all(), (np.unravel_index(np.argmax(off), off.shape), float(off.max()), float(np.abs(g - w).max()))


def check(hip, lens, Hq, Hk, D, page, dt, out_dts, pad=0, seed=0, spread=1.5):
    c = Paged(hip, lens, Hq, Hk, D, page, dt, seed=seed, pad=pad, spread=spread)
    for out_dt in out_dts:
        step(f"jh_paged_attention lens={str(lens)[:60]} Hq={Hq} Hk={Hk} D={D} page={page} dt={dt} out={out_dt}")
        want, bar = c.ref(out_dt)
        close(c.run(out_dt), want, bar, c.starts[-1])
    return c


# single tokens: lengths around the key tiles and pages, requests without new tokens
@pytest.mark.parametrize("lens", [[(1, 1)], [(1, 2)], [(1, 31)], [(1, 33)], [(1, 64), (1, 65)], [(1, 700)],
                                  [(1, 127), (0, 0), (1, 1), (0, 40), (1, 300)], [(1, 4099)]])
@pytest.mark.parametrize("Hq,Hk,D,page,dt", [(8, 2, 128, 16, BF16), (4, 4, 64, 64, F16), (10, 2, 128, 8, F16),
                                             (16, 1, 64, 32, BF16), (8, 1, 256, 16, BF16), (3, 1, 256, 128, F16)])
def test_attention_one_token(hip, lens, Hq, Hk, D, page, dt):
    check(hip, lens, Hq, Hk, D, page, dt, (dt, F32), pad=len(lens) % 3)


# several tokens: rows of a kv head around 16, 32 and 128, keys around 64
@pytest.mark.parametrize("lens", [[(2, 2)], [(4, 40)], [(5, 64), (3, 4)], [(9, 129)], [(33, 33)], [(32, 95), (1, 500), (64, 64)],
                                  [(130, 700), (2, 1200), (0, 9), (31, 31)], [(257, 257)]])
@pytest.mark.parametrize("Hq,Hk,D,page,dt", [(8, 2, 128, 16, BF16), (4, 4, 64, 64, F16), (6, 2, 128, 8, F16),
                                             (16, 1, 64, 128, BF16), (4, 2, 256, 32, BF16), (5, 1, 256, 16, F16)])
def test_attention_many_tokens(hip, lens, Hq, Hk, D, page, dt):
    check(hip, lens, Hq, Hk, D, page, dt, (BF16, F16, F32) if len(lens) < 3 else (dt, F32), pad=len(lens) % 3)


# 8 and 16 kv heads: the parts of split keys are joined inside the launch
@pytest.mark.parametrize("lens", [[(1, 700)], [(1, 4099), (0, 3), (1, 129), (2, 1500)], [(1, 9001)], [(3, 2000)]])
@pytest.mark.parametrize("Hq,Hk,D,page,dt", [(32, 8, 128, 16, BF16), (8, 8, 64, 64, F16), (24, 8, 128, 32, F16), (16, 16, 64, 16, BF16),
                                             (16, 8, 256, 16, BF16)])
def test_attention_joined_in_the_launch(hip, lens, Hq, Hk, D, page, dt):
    c = check(hip, lens, Hq, Hk, D, page, dt, (dt, F32), pad=1)
    assert np.array_equal(c.run(F32), c.run(F32))  # counters are left at zero, parts joined in order


def test_attention_many_requests(hip):
    """More requests than lanes of a wave, of every length."""
    rng = np.random.default_rng(3)
    for R, top in ((65, 4), (150, 1), (300, 2)):
        lens = [(int(n), int(n + k)) for n, k in zip(rng.integers(0, top + 1, R), rng.integers(0, 200, R))]
        check(hip, lens, 4, 2, 64, 16, BF16, (BF16,), pad=3)


def test_attention_rows_without_keys(hip):
    """Fewer keys than new tokens: the first tokens see nothing and are zeros."""
    for lens in ([(3, 0), (1, 0), (2, 5)], [(70, 10), (40, 0), (5, 9)]):
        c = check(hip, lens, 4, 2, 128, 16, BF16, (BF16, F32), pad=1)
        assert (c.run(BF16)[:3] == 0).all()


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("n,kv,Hk", [(1, 500, 2), (6, 500, 2), (90, 300, 2), (90, 2500, 2), (1, 700, 8), (7, 700, 8)])
def test_attention_not_finite(hip, dt, n, kv, Hk):
    """Infinities and NaN in keys and values reach the rows that see them, and
    no others of the same tile; scores of -inf weigh nothing; a row of them alone
    is NaN, as 0 / 0 is."""
    Hq, D = 2 * Hk, 128
    rng = np.random.default_rng(n + kv)
    k = [rounded(rng.standard_normal((Hk, kv, D)), dt)]
    v = [rounded(rng.standard_normal((Hk, kv, D)), dt)]
    v[0][0, kv - max(1, n // 2), 5] = np.inf
    v[0][1, kv - 1, 9] = np.nan
    v[0][1, kv // 2, 11] = -np.inf
    k[0][1, kv - 2, 3] = np.nan if n > 2 else 1.0
    c = Paged(hip, [(n, kv)], Hq, Hk, D, 16, dt, k=k, v=v)
    want, bar = c.ref(F32)
    for out_dt in (F32, dt):
        step(f"jh_paged_attention not finite n={n} kv={kv} dt={dt} out={out_dt}")
        got, (want, bar) = c.run(out_dt), c.ref(out_dt)
        assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(np.isinf(got), np.isinf(want))
        fine = np.isfinite(want)
        assert (np.abs(got - want)[fine] <= bar[fine]).all()
    # every score of kv head 0 -inf (q positive, a key feature -inf)
    c.q[:] = np.abs(c.q) + 0.1
    c.k[0][0, :, 7] = -np.inf
    c.k[0][1, 1::2, 7] = -np.inf
    c.k[0][1, kv - 2, 3] = 1.0
    v[0][0, kv - max(1, n // 2), 5] = v[0][1, kv - 1, 9] = v[0][1, kv // 2, 11] = 1.0
    d = Paged(hip, [(n, kv)], Hq, Hk, D, 16, dt, k=c.k, v=v)
    d.q[:] = rounded(c.q, dt)
    d.Q = up(hip, d.q, dt)
    got, (want, bar) = d.run(F32), d.ref(F32)
    assert np.isnan(got[:, :2]).all() and np.isfinite(got[:, 2:]).all()
    assert (np.abs(got - want)[:, 2:] <= bar[:, 2:] * 2 + 1e-6).all()


def test_attention_values_of_the_small_weights(hip):
    """f16 pages, one key that takes nearly all weight and has values of 0: the
    result is the small weights', down to 2^-20 of the largest, and keeps its
    precision."""
    Hq, Hk, D, kv = 4, 2, 128, 200
    for n in (1, 60):
        rng = np.random.default_rng(n)
        k = [rounded(0.05 * rng.standard_normal((Hk, kv, D)), F16)]
        v = [rounded(rng.standard_normal((Hk, kv, D)), F16)]
        q1 = np.ones(D)
        k[0][:, 0] = rounded(13.8 / D ** 0.5 * q1, F16)
        v[0][:, 0] = 0.0
        c = Paged(hip, [(n, kv)], Hq, Hk, D, 16, F16, k=k, v=v)
        c.q[:] = 1.0
        c.Q = up(hip, c.q, F16)
        step(f"jh_paged_attention small weights n={n}")
        for out_dt in (F16, F32):
            got, (want, bar) = c.run(out_dt), c.ref(out_dt)
            close(got, want, bar, n)


def test_attention_scales_and_sizes(hip):
    """Large and tiny scales, queries of very different sizes."""
    for dt in (BF16, F16):
        for scale in (1e-30, 1e-3, 3.0):
            c = Paged(hip, [(40, 100), (1, 90)], 4, 2, 64, 16, dt)
            c.scale = scale
            c.q *= rounded(10.0 ** np.linspace(-3, 1, c.T), dt)[:, None, None]
            c.q = rounded(c.q, dt)
            c.Q = up(hip, c.q, dt)
            step(f"jh_paged_attention scale={scale} dt={dt}")
            want, bar = c.ref(F32)
            close(c.run(F32), want, bar, c.T)


def test_attention_strides_hint_and_shared_pages(hip):
    """Queries inside wider rows, keys and values that alternate in one buffer,
    requests that share pages, and a wrong max_new: the same results."""
    Hq, Hk, D, page, dt = 8, 2, 128, 16, BF16
    c = Paged(hip, [(1, 200), (40, 100), (3, 50)], Hq, Hk, D, page, dt)
    want, bar = c.ref(dt)
    wide = np.full((c.T, Hq + 3, D), np.nan, np.float32)
    wide[:, :Hq] = c.q
    W = up(hip, wide, dt)
    Q = hip._view(W, (c.T, Hq, D), ((Hq + 3) * D, D, 1))
    both = up(hip, np.stack([c.pools[0], c.pools[1]], 1), dt)
    shape, st = c.pools[0].shape, (2 * Hk * page * D, page * D, D, 1)
    K, V = hip._view(both, shape, st), hip._view(both, shape, st, Hk * page * D)
    step("jh_paged_attention strides and hints")
    for max_new in (40, 1, 0, 5, c.T):
        close(c.run(dt, max_new=max_new, q=Q, k=K, v=V), want, bar, c.T)
    # the third request reads the first one's pages
    c.tables[2] = c.tables[0]
    c.k[2], c.v[2] = c.k[0][:, :50], c.v[0][:, :50]
    c.TAB = ints(hip, c.tables)
    want, bar = c.ref(dt)
    close(c.run(dt), want, bar, c.T)


def test_attention_bad_pages_and_lengths(hip):
    """A page outside the pool makes the rows that see it NaN, and no others; lengths
    are held to their buffers. With checks on, JH_ERR_INVALID."""
    for n, kv in ((1, 100), (60, 100)):
        c = Paged(hip, [(n, kv), (2, 64)], 4, 2, 128, 16, BF16, extra_blocks=0)
        want, bar = c.ref(BF16)
        for bad in (c.n_pages, -1, 2 ** 31 - 1):
            c.tables[0, 5] = bad  # keys 80 .. 95
            c.TAB = ints(hip, c.tables)
            step(f"jh_paged_attention bad page {bad} n={n}")
            got = c.run(BF16)
            hit = kv - n + np.arange(n) >= 80
            assert np.isnan(got[:n][hit]).all()
            close(got[:n][~hit], want[:n][~hit], bar[:n][~hit], n)
            close(got[n:], want[n:], bar[n:], 2)
        hip.SetChecks(True)
        try:
            with pytest.raises(JanisHipError, match="page"):
                c.run(BF16)
        finally:
            hip.SetChecks(False)
    c = Paged(hip, [(2, 64), (3, 20)], 4, 2, 64, 16, BF16, extra_blocks=0)
    for starts, kv in (([0, 2, 9], [64, 20]), ([0, 7, 5], [64, 20]), ([-3, 2, 5], [64, 20]), ([0, 2, 5], [2 ** 31 - 1, -5])):
        c.ST, c.KV = ints(hip, starts), ints(hip, kv)
        step(f"jh_paged_attention starts={starts} kv={kv}")
        c.hip.PagedAttention(c.Q, c.K, c.V, c.TAB, c.ST, c.KV, c.scale, maxNew=3)
        hip.Sync()
        hip.SetChecks(True)
        try:
            with pytest.raises(JanisHipError):
                c.hip.PagedAttention(c.Q, c.K, c.V, c.TAB, c.ST, c.KV, c.scale, maxNew=3)
        finally:
            hip.SetChecks(False)


def test_attention_far_page(hip):
    """Pages whose offset passes 32 bits (in elements and bytes)."""
    Hk, D, page = 1, 128, 16
    stride = (1 << 32) + 64  # elements: three pages span 16 GiB
    try:
        big = hip.empty(BF16, 2 * stride + Hk * page * D)
    except JanisHipError:
        pytest.skip("no room for the pool")
    rng = np.random.default_rng(8)
    for n in (1, 40):
        kv = 40
        k, v = (rounded(rng.standard_normal((Hk, 48, D)), BF16) for _ in range(2))
        K = hip._view(big, (3, Hk, page, D), (stride, page * D, D, 1))
        q = rounded(rng.standard_normal((n, 1, D)), BF16)
        out = {}
        pools = []
        for a in (k, v):
            pools.append(a.reshape(Hk, 3, page, D).transpose(1, 0, 2, 3))
        V = hip._view(big, (3, Hk, page, D), (stride, page * D, D, 1), Hk * page * D) if stride > 2 * Hk * page * D else None
        small = [up(hip, p, BF16) for p in pools]
        for src, dst in zip(small, (K, V)):
            # page 2 of the last only fits keys: values of page 2 lie in the first gap
            for j in range(3 if dst is K else 2):
                hip._copy(hip.Slice(src, 0, j, j + 1), hip._view(dst, (1, Hk, page, D), (stride, page * D, D, 1), j * stride))
        kvs = min(kv, 32)
        starts, lens, tab = ints(hip, [0, n]), ints(hip, [kvs]), ints(hip, [[0, 1]])
        step(f"jh_paged_attention far pages n={n}")
        K2, V2 = (hip._view(t, (2, Hk, page, D), (stride, page * D, D, 1)) for t in (K, V))
        out = hip.Floats(hip.PagedAttention(up(hip, q, BF16), K2, V2, tab, starts, lens, D ** -0.5, maxNew=n))
        near = [up(hip, p[:2], BF16) for p in pools]
        want = hip.Floats(hip.PagedAttention(up(hip, q, BF16), near[0], near[1], tab, starts, lens, D ** -0.5, maxNew=n))
        assert np.array_equal(out, want)
    hip.Sync()
    big.free()


def test_attention_rows_that_overlap(hip):
    """row_starts that go up and down: no fault, and the calls after it are right
    (the counters of the joined parts stay at zero)."""
    c = Paged(hip, [(1, 3000), (1, 900), (2, 50), (1, 4000)], 32, 8, 128, 16, BF16)
    want, bar = c.ref(BF16)
    good = c.ST
    for bad in ([0, 5, 0, 5, 0], [0, 5, 1, 5, 5], [5, 0, 5, 0, 5], [0, 1, 2, 9, 5]):
        c.ST = ints(hip, bad)
        step(f"jh_paged_attention row_starts {bad}")
        hip.PagedAttention(c.Q, c.K, c.V, c.TAB, c.ST, c.KV, c.scale, maxNew=2)
        c.ST = good
        for _ in range(2):
            close(c.run(BF16), want, bar, c.T)


def test_attention_captured_without_workspace():
    """A call whose keys would be split still captures on a context whose workspace
    was never sized (they stay whole), and replays to its result."""
    b = HipBackend(0)
    for n in (1, 50):
        c = Paged(b, [(n, 1500), (1, 40)], 8, 8, 64, 16, F16)
        out = up(b, np.zeros((c.T, 8, 64)), F32)
        step(f"jh_paged_attention captured first n={n}")
        g = Graph(b, lambda: b.PagedAttention(c.Q, c.K, c.V, c.TAB, c.ST, c.KV, c.scale, maxNew=n, out=out))
        want, bar = c.ref(F32)
        for _ in range(3):
            put(b, out, np.zeros((c.T, 8, 64), np.float32))
            g.replay()
            close(b.Floats(out), want, bar, c.T)
        g.close()
    b.Close()


def test_attention_sizes_its_workspace():
    """The first call of a context sizes the workspace for exactly its parts (a call
    that needs more than it was given says so)."""
    for lens, Hq, Hk, D in (([(9, 900)], 32, 8, 128), ([(1, 5000)], 32, 8, 128), ([(12, 3000), (1, 40)], 32, 8, 64), ([(200, 900)], 8, 2, 64),
                            ([(5, 2000)], 16, 2, 128), ([(40, 700)], 8, 8, 256), ([(64, 400)], 8, 8, 64), ([(1, 300)] * 70, 8, 8, 64)):
        b = HipBackend(0)
        check(b, lens, Hq, Hk, D, 16, BF16, (BF16,))
        b.Close()


def test_attention_graphs_share_workspace_and_counters():
    """Two captured calls of different sizes whose parts are joined in their launch, in
    turn, eager calls of other head counts between them, and again after a call that grew
    the workspace: the eager bits each time."""
    b = HipBackend(0)
    cases = [Paged(b, [(1, 3000), (1, 90)], 32, 8, 128, 16, BF16, seed=1), Paged(b, [(7, 900)] * 3, 64, 16, 64, 32, F16, seed=2)]
    other = Paged(b, [(1, 2000)], 16, 4, 128, 16, BF16, seed=3)
    big = Paged(b, [(400, 2500)] * 4, 8, 8, 128, 16, BF16, seed=4)
    outs = [up(b, np.zeros((c.T, c.Hq, c.D)), F32) for c in cases]

    def call(i):
        c = cases[i]
        b.PagedAttention(c.Q, c.K, c.V, c.TAB, c.ST, c.KV, c.scale, maxNew=max(n for n, _ in c.lens), out=outs[i])

    wants = []
    for i, c in enumerate(cases):  # (sizes the workspace)
        step(f"jh_paged_attention eager, then captured: {c.lens}")
        call(i)
        want, bar = c.ref(F32)
        wants.append(b.Floats(outs[i]))
        close(wants[i], want, bar, c.T)
    graphs = [Graph(b, lambda i=i: call(i)) for i in range(2)]
    for turn in range(4):
        if turn == 2:
            big.run(F32)
        for i, c in enumerate(cases):
            put(b, outs[i], np.zeros((c.T, c.Hq, c.D), np.float32))
            graphs[i].replay()
            assert np.array_equal(b.Floats(outs[i]), wants[i]), (turn, i)
            other.run(F32)
    for g in graphs:
        g.close()
    b.Close()


def test_attention_two_contexts_and_streams():
    """Calls of two contexts in flight together on one GPU, and one on a caller's
    stream, each with its own workspace and counters."""
    import torch

    bs = [HipBackend(0), HipBackend(0)]
    stream = torch.cuda.Stream()
    bs[1].SetStream(stream.cuda_stream)
    cs = [Paged(b, [(1, 5000), (3, 700), (1, 9)], 16, 8, 128, 16, BF16, seed=i) for i, b in enumerate(bs)]
    refs = [c.ref(BF16) for c in cs]
    outs = [up(c.hip, np.full((c.T, 16, 128), 7.0), BF16) for c in cs]
    for b in bs:
        b.Sync()
    step("jh_paged_attention on two contexts at once")
    for _ in range(20):
        for c, o in zip(cs, outs):
            c.hip.PagedAttention(c.Q, c.K, c.V, c.TAB, c.ST, c.KV, c.scale, maxNew=3, out=o)
    for c, o, (want, bar) in zip(cs, outs, refs):
        close(c.hip.Floats(o), want, bar, c.T)
    for b in bs:
        b.Close()


def test_attention_repeats_bits(hip):
    c = Paged(hip, [(1, 3000), (20, 900), (1, 50)], 8, 2, 128, 16, BF16)
    step("jh_paged_attention twice")
    a, b = c.run(F32), c.run(F32)
    assert np.array_equal(a, b)


# ---- refusals of the C entries --------------------------------------------------------------

def refused(hip, name, good, changes):
    """The entry with `good` arguments (by name, in order) and each change: its code."""
    fn, L = getattr(hip._L, name), hip._L
    for code, change in changes:
        args = dict(good, **change)
        step(f"{name} refuses {change}")
        assert set(change) <= set(good)
        assert fn(hip._ctx, *args.values()) == code, (change, L.jh_last_error(hip._ctx))
        assert name.encode() in L.jh_last_error(hip._ctx)


def test_refusals(hip):
    INVALID, UNSUPPORTED = _lib.JH_ERR_INVALID, _lib.JH_ERR_UNSUPPORTED
    t = hip.empty(F32, 1 << 16)
    p = t.ptr
    good = dict(new=p, kv=p + 64, R=2, T=4, page=16, tab=p + 1024, blocks=4, free=p + 2048, pages=8, count=p + 4096, kvo=p + 64,
                co=p + 4096, starts=p + 5000 * 4, pos=p + 6000 * 4, slots=p + 7000 * 4, status=p + 8000 * 4)
    refused(hip, "jh_paged_plan", good, [
        (INVALID, dict(page=0)), (INVALID, dict(page=24)), (INVALID, dict(page=1 << 17)), (INVALID, dict(R=-1)), (INVALID, dict(T=-1)),
        (INVALID, dict(blocks=-1)), (INVALID, dict(pages=-1)), (INVALID, dict(pages=1 << 28)), (UNSUPPORTED, dict(R=2049)),
        (UNSUPPORTED, dict(T=(1 << 30) + 1))] + [(INVALID, {k: None}) for k in
                                                 ("new", "kv", "tab", "free", "count", "kvo", "co", "starts", "pos", "slots", "status")])
    good = dict(qkv=p, dt=F32, T=2, stride=6 * 64, hq=2, hk=2, d=64, qw=p, kw=p, wdt=F32, eps=1e-6, base=1e4, scale=1.0, freqs=None,
                pos=p, slots=p, k=p, v=p, pdt=BF16, pages=2, page=16, pstride=2 * 16 * 64, qo=p)
    refused(hip, "jh_paged_qk_norm_rope_append", good, [
        (INVALID, dict(dt=F16)), (INVALID, dict(wdt=I32)), (UNSUPPORTED, dict(pdt=F32)), (INVALID, dict(pdt=I32)),
        (UNSUPPORTED, dict(d=96)), (UNSUPPORTED, dict(d=512)), (INVALID, dict(hk=0)), (INVALID, dict(hq=-1)), (INVALID, dict(T=-1)),
        (INVALID, dict(stride=6 * 64 - 8)), (INVALID, dict(stride=6 * 64 + 4)), (INVALID, dict(pstride=2 * 16 * 64 - 8)),
        (INVALID, dict(pstride=2 * 16 * 64 + 2)), (INVALID, dict(page=12)), (INVALID, dict(pages=1 << 28)), (INVALID, dict(base=-1.0)),
        (INVALID, dict(base=float("nan"))), (INVALID, dict(base=float("inf"))), (INVALID, dict(qkv=p + 4)), (INVALID, dict(qo=p + 8)),
        (INVALID, dict(k=p + 2)), (INVALID, dict(v=p + 2))] + [(INVALID, {k: None}) for k in ("qkv", "pos", "slots", "k", "v", "qo")])
    good = dict(q=p, qs=2 * 64, k=p, v=p, pdt=BF16, pages=2, page=16, pstride=2 * 16 * 64, tab=p, blocks=2, starts=p, kv=p, R=1, T=2,
                new=1, hq=2, hk=2, d=64, scale=0.1, out=p, odt=BF16)
    refused(hip, "jh_paged_attention", good, [
        (UNSUPPORTED, dict(pdt=F32)), (INVALID, dict(pdt=I32)), (INVALID, dict(odt=I32)), (INVALID, dict(pages=0)), (INVALID, dict(pages=-1)),
        (INVALID, dict(page=0)), (INVALID, dict(page=20)), (UNSUPPORTED, dict(page=4)), (INVALID, dict(hq=3)), (INVALID, dict(hq=0)),
        (INVALID, dict(hk=0)), (UNSUPPORTED, dict(d=32)), (INVALID, dict(qs=64)), (INVALID, dict(qs=2 * 64 + 4)), (INVALID, dict(pstride=64)),
        (INVALID, dict(R=-1)), (INVALID, dict(T=-1)), (INVALID, dict(new=-1)), (INVALID, dict(blocks=-1)), (UNSUPPORTED, dict(R=65537)),
        (UNSUPPORTED, dict(T=1 << 30)), (UNSUPPORTED, dict(blocks=(1 << 26) + 1)), (INVALID, dict(scale=0.0)), (INVALID, dict(scale=-1.0)),
        (INVALID, dict(scale=float("nan"))), (INVALID, dict(scale=float("inf"))), (INVALID, dict(q=p + 8)), (INVALID, dict(out=p + 4)),
        (INVALID, dict(k=p + 2))] + [(INVALID, {k: None}) for k in ("q", "k", "v", "tab", "starts", "kv", "out")])


def test_nothing_to_do(hip):
    """No rows or no requests: a success that touches nothing (null buffers among them)."""
    L, c = hip._L, hip._ctx
    assert L.jh_paged_attention(c, None, 64, None, None, BF16, 1, 16, 1024, None, 0, None, None, 1, 0, 0, 1, 1, 64, 0.1, None, BF16) == 0
    assert L.jh_paged_attention(c, None, 64, None, None, BF16, 1, 16, 1024, None, 0, None, None, 0, 3, 1, 1, 1, 64, 0.1, None, BF16) == 0
    assert L.jh_paged_qk_norm_rope_append(c, None, F32, 0, 192, 1, 1, 64, None, None, F32, 0.0, 0.0, 1.0, None, None, None, None, None,
                                          BF16, 0, 16, 1024, None) == 0


def test_values_checked(hip):
    """JH_CHECK_VALUES names the operator whose result holds a NaN, and does not look
    at the rows behind the last."""
    c = Paged(hip, [(1, 40), (2, 30)], 4, 2, 64, 16, BF16, pad=2)
    fill = up(hip, np.full((c.T, 4, 64), np.nan), BF16)
    hip.SetChecks(_lib.JH_CHECK_VALUES)
    try:
        hip.PagedAttention(c.Q, c.K, c.V, c.TAB, c.ST, c.KV, c.scale, maxNew=2, out=fill)
        c.tables[1, 0] = 2 ** 30
        with pytest.raises(JanisHipError, match="jh_paged_attention") as e:
            hip.PagedAttention(c.Q, c.K, c.V, ints(hip, c.tables), c.ST, c.KV, c.scale, maxNew=2, out=fill)
        assert e.value.code == _lib.JH_ERR_NONFINITE
    finally:
        hip.SetChecks(False)


# ---- a step of them together ------------------------------------------------------------

def test_step_captured(hip):
    """A server's steps as one captured graph -- plan, append, attention of one
    layer -- replayed over changing batches: prompts in pieces, single tokens,
    idle, finished and refused requests, eager work between the replays. Keys,
    values and results against contiguous histories in 64 bits."""
    Hq, Hk, D, page, R, T, B, n_pages, dt = 4, 2, 128, 16, 5, 64, 12, 40, F16
    rng = np.random.default_rng(11)
    b = HipBackend(0)
    width = (Hq + 2 * Hk) * D
    qkv, new = up(b, np.zeros((T, width)), F32), ints(b, np.zeros(R))
    kv, tables = ints(b, np.zeros(R)), ints(b, np.full((R, B), -1))
    free, count = ints(b, np.arange(n_pages)), ints(b, [n_pages])
    starts, pos, slots, status = ints(b, np.zeros(R + 1)), ints(b, np.zeros(T)), ints(b, np.zeros(T)), ints(b, [0])
    kp, vp = (up(b, np.full((n_pages, Hk, page, D), np.nan), dt) for _ in range(2))
    qn, kn = (up(b, np.ones(D) + 0.1 * rng.standard_normal(D), BF16) for _ in range(2))
    q, out = up(b, np.zeros((T, Hq, D)), dt), up(b, np.zeros((T, Hq, D)), F32)
    w = [b.Floats(t).astype(np.float64) for t in (qn, kn)]
    inv = 1e4 ** (-2.0 * np.arange(D // 2) / D)

    def one_step():
        b.PagedPlan(new, kv, page, tables, free, count, out=(kv, count, starts, pos, slots, status))
        b.PagedQKNormRoPEAppend(qkv, Hq, Hk, qn, kn, 1e-6, 1e4, 1.0, pos, slots, kp, vp, q_out=q)
        b.PagedAttention(q, kp, vp, tables, starts, kv, D ** -0.5, maxNew=T, out=out)

    step("paged step, eager, then captured")
    one_step()  # sizes the workspace; no new tokens: nothing changes
    b.Sync()
    g = Graph(b, one_step)
    held = [[np.zeros((0, Hk, D))] * 2 for _ in range(R)]
    steps = [[17, 0, 0, 1, 0], [1, 30, 0, 1, 2], [1, 1, 33, 20, 1], [1, 1, 1, 0, -1], [-1, 20, 1, 3, 0], [40, 1, 5, 1, 16],
             [64, 1, 0, 0, 0], [0, 0, 0, 0, 500], [1, 1, 1, 1, 1], [1, -1, 30, -1, -1], [1, 1, 1, 1, 1]]
    for i, ns in enumerate(steps):
        x = rounded(2 * rng.standard_normal((T, width)), F32)
        put(b, qkv, x)
        put(b, new, np.array(ns, np.int32))
        before = b.Ints(kv)
        put(b, out, np.full((T, Hq, D), 7.0, np.float32))
        g.replay()
        st = b.Ints(status)[0]
        total = sum(max(0, n) for n in ns)
        fits = total <= T and all(len(h[0]) + max(0, n) <= B * page for h, n in zip(held, ns))
        assert (st == 0) == fits, (i, st)
        got, ntab, nkv = b.Floats(out), b.Ints(tables), b.Ints(kv)
        if st:
            assert np.array_equal(nkv, before) and (got == 7.0).all()
            continue
        t = 0
        for r, n in enumerate(ns):
            if n < 0:
                held[r] = [np.zeros((0, Hk, D))] * 2
            first = len(held[r][0])
            m = max(0, n)
            p = np.arange(first, first + m)
            Q, Kn, Vn = append_ref(x[t:t + m], Hq, Hk, D, *w, 1e-6, p[:, None] * inv, None, None)
            held[r] = [np.concatenate([held[r][0], Kn]), np.concatenate([held[r][1], Vn])]
            assert nkv[r] == first + m
            k, v = held[r]
            for j in range(m):
                seen = first + j + 1
                for h in range(Hq):
                    s = k[:seen, h // 2] @ Q[j, h] * D ** -0.5
                    e = np.exp(s - s.max())
                    A = e @ np.abs(v[:seen, h // 2]) / e.sum()
                    want = e @ v[:seen, h // 2] / e.sum()
                    # q, k and v were rounded to f16: a score is off by 2^-11 (2 + 2^-11) sum |q k| scale
                    d = 2.0 ** -10 * np.max(np.abs(k[:seen, h // 2]) @ np.abs(Q[j, h])) * D ** -0.5 * 1.05
                    bar = A * (2 * np.expm1(d) + 2.0 ** -10)
                    assert (np.abs(got[t + j, h] - want) <= bar).all(), (i, r, j, h)
            t += m
        assert (got[t:] == 7.0).all()
        mine = [int(ntab[r, c]) for r in range(R) for c in range(-(-int(nkv[r]) // page))]
        assert len(set(mine)) == len(mine) and len(mine) + b.Ints(count)[0] == n_pages
        hip.Floats(hip.Add(up(hip, np.ones(300), F32), up(hip, np.ones(300), F32)))
    g.close()
    b.Close()


# ---- probabilities in two terms, whatever the result's type --------------------------------

def fp32_bar(c, out_dt):
    """(expected, bar): the bar of fp32 results, whose probabilities are two terms of the
    pages' dtype, and one rounding of the result to out_dt."""
    want, bar = c.ref(F32)
    return want, bar + HALF[out_dt] * np.abs(want) * 1.01 + (2.0 ** -25 if out_dt == F16 else 0)


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("lens,Hq,Hk,D", [([(70, 300)], 4, 2, 64), ([(257, 257), (3, 90)], 8, 2, 128), ([(40, 2500), (1, 70)], 8, 2, 128),
                                          ([(50, 200)], 4, 2, 256)])
def test_attention_probabilities_are_not_rounded(hip, dt, lens, Hq, Hk, D):
    """Results of 16 bits in tiles of 128 rows are as near as fp32's, rounded once, also
    where they have more bits than the pages; the hint chooses kernels of the same precision."""
    c = Paged(hip, lens, Hq, Hk, D, 16, dt, spread=0.25)
    for out_dt in (BF16, F16):
        want, bar = fp32_bar(c, out_dt)
        for max_new in (lens[0][0], 1):
            step(f"jh_paged_attention two terms {lens} D={D} dt={dt} out={out_dt} hint={max_new}")
            close(c.run(out_dt, max_new=max_new), want, bar, c.starts[-1])


# ---- the plan: pages that requests go on filling ----------------------------------------------

@pytest.mark.parametrize("bad", [-1, 7, 2 ** 30])
@pytest.mark.parametrize("in_place", [False, True])
def test_plan_page_in_use_outside(hip, bad, in_place):
    """New tokens that begin inside a page whose number is outside the pool: nothing is
    planned. Such numbers where no token goes (a request without new tokens, a last page
    that is full, earlier pages) are not looked at."""
    page, rows, n_pages = 16, 8, 7
    kv, free, count = np.array([20, 16, 40, 5], np.int32), np.array([5, 6, -1, -1, -1, -1, -1], np.int32), 2
    tables = np.array([[0, 1, -1, -1], [2, -1, -1, -1], [bad, bad, 3, -1], [4, -1, -1, -1]], np.int32)
    new = np.array([2, 1, 3, 0], np.int32)
    tables[1, 0] = tables[3, 0] = bad
    step(f"jh_paged_plan page {bad} where no token goes, in_place={in_place}")
    want = plan_ref(new, kv, page, tables, free, count, rows, n_pages)
    assert want[5] == 0 and (want[4][:6] >= 0).all()
    same_plan(run_plan(hip, new, kv, page, tables, free, count, rows, in_place), want)
    for r, at in ((0, 1), (2, 2), (3, 0)):
        t, n = tables.copy(), new.copy()
        t[r, at], n[r] = bad, 1
        none = np.full(rows, -1, np.int32)
        step(f"jh_paged_plan page {bad} in use by request {r}")
        same_plan(run_plan(hip, n, kv, page, t, free, count, rows, in_place),
                  (kv, count, np.zeros(5, np.int32), none, none, _lib.JH_PLAN_TABLE, t, free))
    hip.SetChecks(True)
    try:
        with pytest.raises(JanisHipError, match="page number"):
            run_plan(hip, n, kv, page, t, free, count, rows)
    finally:
        hip.SetChecks(False)


def test_values_checked_between_the_ends(hip):
    """Rows before the first request's belong to nobody: left as they were, and not
    looked at by JH_CHECK_VALUES, whose index counts from the result's start."""
    c = Paged(hip, [(2, 40), (3, 30)], 4, 2, 64, 16, BF16, pad=4)
    want, bar = c.ref(BF16)
    shift = 3
    Q = np.zeros_like(c.q)
    Q[shift:shift + 5] = c.q[:5]
    Q, ST = up(hip, Q, BF16), ints(hip, c.starts + shift)
    fill = up(hip, np.full((c.T, 4, 64), np.nan), BF16)
    hip.SetChecks(_lib.JH_CHECK_INDICES | _lib.JH_CHECK_VALUES)
    try:
        step("jh_paged_attention checked, rows of nobody at both ends")
        got = hip.Floats(hip.PagedAttention(Q, c.K, c.V, c.TAB, ST, c.KV, c.scale, maxNew=3, out=fill))
        assert np.isnan(got[:shift]).all() and np.isnan(got[shift + 5:]).all()
        close(got[shift:], want, bar, 5)
        hip.SetChecks(_lib.JH_CHECK_VALUES)
        c.tables[1, 0] = 2 ** 30
        with pytest.raises(JanisHipError, match=f"index {(shift + 2) * 4 * 64}"):
            hip.PagedAttention(Q, c.K, c.V, ints(hip, c.tables), ST, c.KV, c.scale, maxNew=3, out=fill)
    finally:
        hip.SetChecks(False)


def test_refusal_of_rows_past_the_grid(hip):
    """A wave per row: more rows than a grid has room for are refused before the launch."""
    t = hip.empty(F32, 1 << 12)
    p = t.ptr
    good = dict(qkv=p, dt=F32, T=0, stride=6 * 64, hq=2, hk=2, d=64, qw=p, kw=p, wdt=F32, eps=1e-6, base=1e4, scale=1.0, freqs=None,
                pos=p, slots=p, k=p, v=p, pdt=BF16, pages=2, page=16, pstride=2 * 16 * 64, qo=p)
    refused(hip, "jh_paged_qk_norm_rope_append", good, [(_lib.JH_ERR_UNSUPPORTED, dict(T=T)) for T in ((1 << 25) + 1, 1 << 31, 1 << 62)])


# ---- long walks: what a block looks up, shares out or repeats more than once --------------------

def expected(c, out_dt, tokens=None):
    """(tokens, expected, bar) as Paged.ref gives them for fp32 results, then one rounding
    to out_dt, for some tokens; keys with a score of -inf weigh nothing, and nothing of
    them enters the bar."""
    G = c.Hq // c.Hk
    owner = [(r, i) for r, (n, _) in enumerate(c.lens) for i in range(n)]
    tokens = list(range(len(owner))) if tokens is None else sorted(set(tokens))
    want, bar = np.zeros((2, len(tokens), c.Hq, c.D))
    for at, t in enumerate(tokens):
        r, i = owner[t]
        n, kv = c.lens[r]
        seen = kv - n + i + 1
        for h in range(c.Hk):
            k, v = c.k[r][h, :seen].astype(np.float64), c.v[r][h, :seen].astype(np.float64)
            q = c.q[t, h * G:(h + 1) * G].astype(np.float64)
            s = q @ k.T * c.scale
            live = np.isfinite(s).all(0)
            assert (s[:, ~live] == -np.inf).all() and live.any()
            k, v, s = k[live], v[live], s[:, live]
            rest = (np.abs(q) @ np.abs(k).T).max(-1) * c.scale
            w = np.exp(s - s.max(-1, keepdims=True))
            w /= w.sum(-1, keepdims=True)
            o, A = w @ v, w @ np.abs(v)
            d = c.D * 2.0 ** -24 * rest + 2.0 ** -22 * (1 + np.abs(s).max(-1))
            rel = 2 * np.expm1(2 * d) + HALF[c.dt] ** 2 + (seen / 64 + 128) * 2.0 ** -24
            want[at, h * G:(h + 1) * G] = o
            bar[at, h * G:(h + 1) * G] = A * rel[:, None] * 1.01
    bar += (HALF[out_dt] + 2.0 ** -24) * 1.01 * np.abs(want) + (2.0 ** -25 if out_dt == F16 else 0)
    assert np.isfinite(want).all() and np.isfinite(bar).all()
    return tokens, want, bar


def near(got, e):
    tokens, want, bar = e
    off = np.abs(got[tokens].astype(np.float64) - want) - bar
    assert (off <= 0).all(), (np.unravel_index(np.argmax(off), off.shape), float(off.max()))


def sharing(hip, R, new, kv, Hq, Hk, D, page, dt, seed=0):
    """R requests of `new` tokens over the same kv keys and pages, queries of their own."""
    c = Paged(hip, [(new, kv)], Hq, Hk, D, page, dt, seed=seed, pad=(R - 1) * new)
    c.lens, c.k, c.v = [(new, kv)] * R, c.k * R, c.v * R
    c.tables, c.starts = np.repeat(c.tables, R, 0), np.arange(R + 1, dtype=np.int32) * new
    c.TAB, c.ST, c.KV = ints(hip, c.tables), ints(hip, c.starts), ints(hip, [kv] * R)
    return c


def captured_whole(lens, Hq, Hk, D, page, dt, out_dt, seed=0):
    """The call captured on a context without a workspace, where keys are not split."""
    b = HipBackend(0)
    c = Paged(b, lens, Hq, Hk, D, page, dt, seed=seed)
    n = max(n for n, _ in lens)
    out = up(b, np.zeros((c.T, Hq, D)), out_dt)
    step(f"jh_paged_attention whole keys {str(lens)[:50]} Hq={Hq} Hk={Hk} D={D} dt={dt} out={out_dt}")
    g = Graph(b, lambda: b.PagedAttention(c.Q, c.K, c.V, c.TAB, c.ST, c.KV, c.scale, maxNew=n, out=out))
    e = expected(c, out_dt, [t for t in range(c.T) if t < 3 or t > c.T - 4 or t % 23 == 0])
    for _ in range(2):
        put(b, out, np.zeros((c.T, Hq, D), np.float32 if out_dt == F32 else np.uint16))
        g.replay()
        near(b.Floats(out), e)
    g.close()
    b.Close()


CUS = 256  # of an MI355X


@pytest.mark.parametrize("dt,D,page", [(BF16, 128, 16), (F16, 128, 32), (BF16, 64, 8), (F16, 256, 64)])
def test_attention_few_rows_look_up_pages_again(dt, D, page):
    """A part of more than 16 tiles of 32 keys for each of four waves, three times over."""
    kv = 5003
    assert kv > 2 * 16 * 4 * 32
    captured_whole([(1, kv), (3, 2100)], 4, 2, D, page, dt, dt)


@pytest.mark.parametrize("Hk,D", [(64, 64), (32, 128)])
def test_attention_split_parts_look_up_pages_again(hip, Hk, D):
    """The same in split parts that are joined inside the launch: a decode batch whose
    parts have more than 2048 keys each."""
    R, kv = 16, 17000 if Hk == 32 else 9000
    room = CUS * (4 if D == 64 else 2) // Hk  # blocks at once, per kv head; split over at most twice that
    assert R * kv / (2 * room + R) > 16 * 4 * 32
    c = sharing(hip, R, 1, kv, Hk, Hk, D, 16, BF16)
    step(f"jh_paged_attention parts of many keys Hk={Hk} D={D}")
    near(c.run(BF16), expected(c, BF16, [0, 7, 15]))


@pytest.mark.parametrize("dt,D,page,out_dt", [(BF16, 128, 16, BF16), (F16, 64, 32, F16), (F16, 128, 64, F32), (BF16, 256, 16, BF16)])
@pytest.mark.parametrize("others", [0, 8])
def test_attention_many_rows_look_up_pages_again(dt, D, page, out_dt, others):
    """More than 32 tiles of 64 keys for each group of waves: alone, where eight waves are
    two groups (one of four at a head_dim of 256), and beside so many requests that blocks
    have four."""
    kv, Hk, G = 4700, 32 if others else 2, 2
    tiles = 1 + others + (70 * G + others * 66 * G) // 128
    assert (tiles * Hk > CUS) == bool(others) and kv > (2 if others or D == 256 else 1) * 32 * 64 * (1 if others or D == 256 else 2)
    captured_whole([(70, kv)] + [(66, 67)] * others, Hk * G, Hk, D, page, dt, out_dt)


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("Hq,Hk,D,lens", [(256, 32, 128, [(130, 300)]), (256, 32, 64, [(130, 300)]), (64, 32, 128, [(70, 90)] * 4 + [(200, 400), (1, 900), (0, 5)]),
                                          (48, 16, 64, [(90, 500)] * 9 + [(1, 70)] * 3), (32, 8, 128, [(1030, 1203)]), (32, 8, 64, [(1030, 1030)])])
def test_attention_more_tiles_than_cus(hip, dt, Hq, Hk, D, lens):
    """Long runs in so many tiles that blocks have four waves: all result types."""
    rows = sum(n for n, _ in lens) * (Hq // Hk)
    assert (min(len(lens), rows) + rows // 128) * Hk > CUS
    c = Paged(hip, lens, Hq, Hk, D, 16, dt, pad=2)
    T = int(c.starts[-1])
    some = [t for t in range(T) if t < 2 or t > T - 3 or t % 41 == 0] + [int(s) for s in c.starts[:-1] if s < T] + [int(s) - 1 for s in c.starts if s > 0]
    for out_dt in (BF16, F16, F32):
        step(f"jh_paged_attention four waves Hq={Hq} Hk={Hk} D={D} lens={str(lens)[:40]} dt={dt} out={out_dt}")
        near(c.run(out_dt), expected(c, out_dt, some))


@pytest.mark.parametrize("n,kv,Hk", [(1, 500, 2), (6, 500, 2), (90, 300, 2), (90, 2500, 2), (1, 700, 8), (130, 200, 32)])
@pytest.mark.parametrize("dt", [BF16, F16])
def test_attention_scores_of_minus_infinity(hip, dt, n, kv, Hk):
    """Keys whose scores are -inf weigh nothing; the others' results keep their bar. Half
    of the keys, whole tiles of them, and a first tile without any other."""
    Hq, D = 2 * Hk, 128
    rng = np.random.default_rng(n + kv + Hk)
    k, v = (rounded(rng.standard_normal((Hk, kv, D)), dt) for _ in range(2))
    k[0, 1::2, 7] = -np.inf
    k[1, :kv - n, 7] = -np.inf
    if kv - n > 130:
        k[1, 100, 7] = 0.5
    c = Paged(hip, [(n, kv)], Hq, Hk, D, 16, dt, k=[k], v=[v])
    c.q[:] = rounded(np.abs(c.q) + 0.125, dt)
    c.Q = up(hip, c.q, dt)
    for out_dt in (dt, F32):
        step(f"jh_paged_attention scores of -inf n={n} kv={kv} Hk={Hk} dt={dt} out={out_dt}")
        near(c.run(out_dt), expected(c, out_dt))


@pytest.mark.parametrize("page,done,fresh", [(1, 30, 7000), (1, 45, 4500), (8, 30, 40000)])
@pytest.mark.parametrize("in_place", [False, True])
def test_plan_of_many_pages(hip, page, done, fresh, in_place):
    """More pages than one round of the block takes (four for each of 1024 threads) come
    back and are taken: past what came back into the stack, and not."""
    rng = np.random.default_rng(fresh)
    R = 60
    kv = (rng.integers(150, 250, R) * page + rng.integers(0, page, R)).astype(np.int32)
    new = np.ones(R, np.int32)
    new[rng.permutation(R)[:done]] = -1
    left = np.flatnonzero(new > 0)
    new[left[0]], new[left[1]] = fresh // 3, fresh - fresh // 3
    rows = int(np.maximum(new, 0).sum()) + 9
    blocks = -(-kv // page)
    back = int(blocks[new < 0].sum())
    take = int((-(-(kv + np.maximum(new, 0)) // page) - blocks)[new >= 0].sum())
    assert back > 4096 and take > 4096 and (take > back) == (fresh == 7000)
    spare = 3000
    n_pages = int(blocks.sum()) + spare
    order = rng.permutation(n_pages).astype(np.int32)
    tables = np.full((R, int((-(-(kv + np.maximum(new, 0)) // page)).max()) + 1), -7, np.int32)
    at = 0
    for r in range(R):
        tables[r, :blocks[r]] = order[at:at + blocks[r]]
        at += blocks[r]
    free = np.full(n_pages, -9, np.int32)
    free[:spare] = order[at:]
    step(f"jh_paged_plan page={page}: {back} pages back, {take} taken, {rows} rows, in_place={in_place}")
    want = plan_ref(new, kv, page, tables, free, spare, rows, n_pages)
    assert want[5] == 0
    same_plan(run_plan(hip, new, kv, page, tables, free, spare, rows, in_place), want)
    # a bad number among those of the later rounds: nothing is planned
    t = tables.copy()
    last = int(np.flatnonzero(new < 0)[-1])
    t[last, blocks[last] - 1] = n_pages
    want = plan_ref(new, kv, page, t, free, spare, rows, n_pages)
    assert want[5] == _lib.JH_PLAN_TABLE
    same_plan(run_plan(hip, new, kv, page, t, free, spare, rows, in_place), want)


@pytest.mark.parametrize("n,kv", [(1, 300), (6, 300), (90, 200)])
def test_attention_values_below_the_normal_numbers(hip, n, kv):
    """f16 values of a few of its least steps (2^-24) are used as they are, not as zeros."""
    Hq, Hk, D = 4, 2, 128
    rng = np.random.default_rng(n)
    k = [rounded(0.5 * rng.standard_normal((Hk, kv, D)), F16)]
    v = [(rng.integers(-300, 300, (Hk, kv, D)) * 2.0 ** -24).astype(np.float32)]
    assert np.array_equal(rounded(v[0], F16), v[0])
    c = Paged(hip, [(n, kv)], Hq, Hk, D, 16, F16, k=k, v=v)
    step(f"jh_paged_attention small values n={n}")
    near(c.run(F32), expected(c, F32))
