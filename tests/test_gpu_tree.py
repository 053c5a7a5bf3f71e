"""Trees of drafted tokens over the paged cache: positions and masks, attention, the
agreed path, and a step of them together, against plain forms in 64 bits.

Bars of the attention are those of tests/test_gpu_paged.py, from the same formula."""
import numpy as np
import pytest

from janis_amd import _lib, synth
from janis_amd.engine import BF16, F16, F32, I32, U32, HipBackend, JanisHipError, PagedLayers
from tests.conftest import Graph, put, step
from tests.test_gpu_paged import HALF, Paged, append_ref, ints, refused, rounded, up

pytestmark = pytest.mark.gpu


def tree(rng, n, wide=5, roots=1):
    """Parents of a tree (or `roots` of them) of n rows."""
    return [-1 if i < roots else int(rng.integers(max(0, i - wide), i)) for i in range(n)]


def masks_of(parents, words):
    """(depth, mask words) of each row, one way up after the other."""
    out = []
    for i in range(len(parents)):
        bits, at, depth = 0, i, -1
        while at >= 0:
            bits, at, depth = bits | 1 << at, parents[at], depth + 1
        out.append((depth, [bits >> 32 * w & 0xFFFFFFFF for w in range(words)]))
    return out


# ---- positions and masks ---------------------------------------------------------------

def tree_plan_ref(parents, starts, kv, T, words):
    pos, mask = np.full(T, -1, np.int64), np.zeros((T, words), np.uint32)
    for r in range(len(kv)):
        a, n = starts[r], starts[r + 1] - starts[r]
        if n > 32 * words:
            pos[a:a + n] = kv[r] - n + np.arange(n)
            continue
        own = [int(p) if -1 <= p < i else -1 for i, p in enumerate(parents[a:a + n])]
        for i, (depth, bits) in enumerate(masks_of(own, words)):
            pos[a + i], mask[a + i] = kv[r] - n + depth, bits
    return pos, mask


def run_tree_plan(hip, parents, starts, kv, T, words):
    pos, mask = ints(hip, np.full(T, 77)), hip.FromRaw(U32, np.full((T, words), 77, np.uint32), T, words)
    hip.PagedTreePlan(ints(hip, parents), ints(hip, starts), ints(hip, kv), out=(pos, mask))
    return hip.Ints(pos), hip.Ints(mask).view(np.uint32)


@pytest.mark.parametrize("words,ns", [(1, [1]), (1, [32]), (1, [33]), (1, [5, 0, 1, 31, 32, 33, 100]), (2, [64, 65, 63, 33, 2]), (3, [96, 97, 65, 64]),
                                      (4, [128, 100, 7, 200]), (16, [512, 513, 449, 1, 300, 64]), (5, [160] * 9)])
@pytest.mark.parametrize("kind", ["chain", "star", "narrow", "wide", "forest"])
def test_tree_plan(hip, words, ns, kind):
    rng = np.random.default_rng(words + len(ns))
    make = {"chain": lambda n: list(range(-1, n - 1)), "star": lambda n: [-1] + [0] * (n - 1), "narrow": lambda n: tree(rng, n, 3),
            "wide": lambda n: tree(rng, n, 200), "forest": lambda n: tree(rng, n, 40, roots=4)}[kind]
    front, pad = 3, 70
    parents = [9] * front + [p for n in ns for p in make(n)[:n]] + [-9] * pad
    starts = (front + np.concatenate([[0], np.cumsum(ns)])).astype(np.int32)
    kv = (np.array(ns) + rng.integers(0, 1000, len(ns))).astype(np.int32)
    kv[-1] = ns[-1]
    T = len(parents)
    step(f"jh_paged_tree_plan words={words} ns={ns[:6]} {kind}")
    got = run_tree_plan(hip, np.array(parents), starts, kv, T, words)
    want = tree_plan_ref(parents, starts, kv, T, words)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


def test_tree_plan_parents_that_are_none(hip):
    """A row's own number, a later one, numbers below -1 and past the request count as -1;
    with checks on they are refused. Those of runs are not looked at."""
    parents = np.array([0, 0, 2, 7, -2, 2 ** 31 - 1, -2 ** 31, 3] + [5] * 40, np.int32)
    starts, kv = np.array([0, 8, 48], np.int32), np.array([20, 50], np.int32)
    step("jh_paged_tree_plan parents that are none")
    got, want = run_tree_plan(hip, parents, starts, kv, 48, 1), tree_plan_ref(parents, starts, kv, 48, 1)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
    hip.SetChecks(True)
    try:
        with pytest.raises(JanisHipError, match="parent"):
            run_tree_plan(hip, parents, starts, kv, 48, 1)
        with pytest.raises(JanisHipError, match="row_starts"):
            run_tree_plan(hip, parents, np.array([0, 49, 48]), kv, 48, 1)
        parents[:8] = [-1, 0, 1, 0, 3, 4, -1, 6]
        got, want = run_tree_plan(hip, parents, starts, kv, 48, 1), tree_plan_ref(parents, starts, kv, 48, 1)
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
    finally:
        hip.SetChecks(False)


def test_tree_plan_many_and_no_requests(hip):
    rng = np.random.default_rng(4)
    for R, words in ((3000, 1), (700, 2), (0, 1)):
        ns = rng.integers(0, 12, R)
        parents = [p for n in ns for p in tree(rng, n)] + [-1] * 900
        starts = np.concatenate([[0], np.cumsum(ns)]).astype(np.int32)
        kv = (ns + rng.integers(0, 100, R)).astype(np.int32)
        step(f"jh_paged_tree_plan R={R}")
        got = run_tree_plan(hip, np.array(parents), starts, kv, len(parents), words)
        want = tree_plan_ref(parents, starts, kv, len(parents), words)
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
    # row_starts that leave the rows: no fault
    step("jh_paged_tree_plan row_starts outside")
    for starts in ([-5, 70, 3], [0, 2 ** 31 - 1, 4], [9, 5, 60]):
        run_tree_plan(hip, np.array(tree(rng, 40)), np.array(starts), np.array([30, 30]), 40, 2)


# ---- attention -----------------------------------------------------------------------------

class Trees(Paged):
    """Paged, with masks [T, words] of trees (or those given)."""

    def __init__(self, hip, lens, Hq, Hk, D, page, dt, words=2, masks=None, seed=0, **kw):
        super().__init__(hip, lens, Hq, Hk, D, page, dt, seed=seed, **kw)
        rng = np.random.default_rng(seed + 5)
        self.words = words
        self.mask = np.zeros((self.T, words), np.uint32)
        for r, (n, _) in enumerate(lens):
            if n <= 32 * words:
                for i, (_, bits) in enumerate(masks_of(tree(rng, n), words)):
                    self.mask[self.starts[r] + i] = bits
        if masks is not None:
            self.mask = masks(self, rng)
        self.M = hip.FromRaw(U32, self.mask, *self.mask.shape)

    def sees(self, r, i):
        """Keys that token i of request r sees."""
        n, kv = self.lens[r]
        base = kv - n
        if n > 32 * self.words:
            return np.arange(max(0, base + i + 1))
        bits = [b for b in range(n) if self.mask[self.starts[r] + i, b // 32] >> (b % 32) & 1]
        keys = np.concatenate([np.arange(max(0, base)), base + np.array(bits, np.int64)]).astype(np.int64)
        return keys[keys >= 0]

    def ref(self, out_dt, tokens=None):
        """(tokens, expected, bar): fp32 results' bar with probabilities of two terms, and
        one rounding to out_dt."""
        G = self.Hq // self.Hk
        owner = [(r, i) for r, (n, _) in enumerate(self.lens) for i in range(n)]
        tokens = list(range(len(owner))) if tokens is None else sorted(set(tokens))
        want, bar = np.zeros((2, len(tokens), self.Hq, self.D))
        for at, t in enumerate(tokens):
            keys = self.sees(*owner[t])
            if keys.size == 0:
                continue
            for h in range(self.Hk):
                k, v = self.k[owner[t][0]][h, keys].astype(np.float64), self.v[owner[t][0]][h, keys].astype(np.float64)
                q = self.q[t, h * G:(h + 1) * G].astype(np.float64)
                with np.errstate(all="ignore"):
                    s = q @ k.T * self.scale
                    rest = (np.abs(q) @ np.abs(k).T).max(-1) * self.scale
                    w = np.exp(s - s.max(-1, keepdims=True))
                    w /= w.sum(-1, keepdims=True)
                    o, A = w @ v, w @ np.abs(v)
                    d = self.D * 2.0 ** -24 * rest + 2.0 ** -22 * (1 + np.abs(s).max(-1))
                    rel = 2 * np.expm1(2 * d) + HALF[self.dt] ** 2 + (keys.size / 64 + 128) * 2.0 ** -24
                    want[at, h * G:(h + 1) * G] = o
                    bar[at, h * G:(h + 1) * G] = A * rel[:, None] * 1.01
        bar += (HALF[out_dt] + 2.0 ** -24) * 1.01 * np.abs(want) + (2.0 ** -25 if out_dt == F16 else 0)
        return tokens, want, bar

    def run(self, out_dt, max_new=None, **kw):
        if max_new is None:
            max_new = max([n for n, _ in self.lens], default=0)
        fill = up(self.hip, np.full((self.T, self.Hq, self.D), 7.0), out_dt)
        a = dict(q=self.Q, k=self.K, v=self.V, mask=self.M)
        a.update(kw)
        got = self.hip.Floats(self.hip.PagedTreeAttention(a["q"], a["k"], a["v"], self.TAB, self.ST, self.KV, a["mask"], self.scale,
                                                          maxNew=max_new, out=fill))
        assert (got[self.starts[-1]:] == 7.0).all(), "rows behind the last"
        return got


def near(got, ref):
    tokens, want, bar = ref
    g = got[tokens].astype(np.float64)
    assert np.array_equal(np.isnan(g), np.isnan(want)) and np.array_equal(np.isinf(g), np.isinf(want))
    fine = np.isfinite(want)
    off = np.where(fine, np.abs(np.where(fine, g, 0.0) - np.where(fine, want, 0.0)) - bar, -1.0)
    assert (off <= 0).all(), (np.unravel_index(np.argmax(off), off.shape), float(off.max()))


def check(hip, lens, Hq, Hk, D, page, dt, out_dts, words=2, **kw):
    c = Trees(hip, lens, Hq, Hk, D, page, dt, words=words, **kw)
    for out_dt in out_dts:
        step(f"jh_paged_tree_attention lens={str(lens)[:60]} Hq={Hq} Hk={Hk} D={D} page={page} words={words} dt={dt} out={out_dt}")
        near(c.run(out_dt), c.ref(out_dt))
    return c


# trees around the tiles of 32 and 128 rows and of 32 and 64 keys, with and without committed keys
@pytest.mark.parametrize("lens,words", [([(1, 1)], 1), ([(1, 700)], 1), ([(7, 7)], 1), ([(8, 40)], 1), ([(16, 717)], 1), ([(31, 63), (32, 95), (33, 33)], 2),
                                        ([(64, 64), (1, 129), (64, 1500)], 2), ([(5, 300), (0, 70), (63, 200), (2, 2), (17, 1234)], 2),
                                        ([(128, 500), (100, 100)], 4), ([(300, 420)], 16), ([(512, 700), (20, 20)], 16)])
@pytest.mark.parametrize("Hq,Hk,D,page,dt", [(8, 2, 128, 16, BF16), (4, 4, 64, 64, F16), (10, 2, 128, 8, F16), (16, 1, 64, 32, BF16),
                                             (4, 2, 256, 32, BF16), (5, 1, 256, 16, F16)])
def test_attention(hip, lens, words, Hq, Hk, D, page, dt):
    check(hip, lens, Hq, Hk, D, page, dt, (dt, F32), words=words, pad=len(lens) % 3)


# 8 and 16 kv heads: parts of split keys joined inside the launch, or by a second one
@pytest.mark.parametrize("lens,words", [([(2, 700)], 1), ([(8, 4099), (0, 3), (3, 129)], 1), ([(16, 9001)], 1), ([(60, 5000)], 2), ([(30, 900)] * 20, 1)])
@pytest.mark.parametrize("Hq,Hk,D,page,dt", [(32, 8, 128, 16, BF16), (8, 8, 64, 64, F16), (24, 8, 128, 32, F16), (16, 8, 256, 16, BF16)])
def test_attention_joined(hip, lens, words, Hq, Hk, D, page, dt):
    c = check(hip, lens[:6], Hq, Hk, D, page, dt, (dt, F32), words=words, pad=1)
    assert np.array_equal(c.run(F32), c.run(F32))  # counters are left at zero, parts joined in order


@pytest.mark.parametrize("Hq,Hk,D,page,dt", [(32, 8, 128, 16, BF16), (8, 8, 64, 64, F16), (24, 8, 128, 32, F16), (16, 8, 256, 16, BF16), (32, 4, 128, 16, F16)])
def test_attention_joined_batch(hip, Hq, Hk, D, page, dt):
    """A batch whose tiles are nearly all cut: parts in the workspace, joined by the second launch."""
    c = Trees(hip, [(30, 900)] * 20, Hq, Hk, D, page, dt, words=1, pad=1)
    tokens = np.random.default_rng(D).integers(0, 600, 90)
    for out_dt in (dt, F32):
        step(f"jh_paged_tree_attention 20 x 30 of 900 Hq={Hq} Hk={Hk} D={D} page={page} dt={dt} out={out_dt}")
        got = c.run(out_dt)
        near(got, c.ref(out_dt, tokens))
        assert np.array_equal(got, c.run(out_dt))


def test_attention_causal_masks_are_paged_attention(hip):
    """A chain's mask gives the results of jh_paged_attention (keys may be split elsewhere)."""
    for lens, Hq, Hk, D in (([(7, 900), (1, 60)], 32, 8, 128), ([(64, 900), (33, 40)], 8, 2, 128), ([(100, 100)], 4, 4, 64), ([(40, 300)], 4, 2, 256)):
        c = Trees(hip, lens, Hq, Hk, D, 16, BF16, words=4, masks=lambda c, rng: np.concatenate(
            [np.array([b for _, b in masks_of(list(range(-1, n - 1)), 4)], np.uint32) for n, _ in lens]))
        step(f"jh_paged_tree_attention as a chain {lens}")
        tokens, want, bar = c.ref(F32)
        got, plain = c.run(F32), Paged.run(c, F32)
        near(got, (tokens, want, bar))
        near(got, (tokens, plain[tokens].astype(np.float64), 2 * bar))


def test_attention_runs_beside_trees(hip):
    """Prompts' pieces longer than the mask's bits are causal, and their masks not looked at."""
    def junk(c, rng):
        m = rng.integers(0, 2 ** 32, c.mask.shape, dtype=np.uint32)
        for r, (n, _) in enumerate(c.lens):
            if n <= 32 * c.words:
                m[c.starts[r]:c.starts[r + 1]] = c.mask[c.starts[r]:c.starts[r + 1]]
        return m

    for lens, words in (([(33, 90), (32, 90), (200, 900), (1, 50)], 1), ([(65, 65), (64, 400), (300, 300), (0, 7)], 2)):
        for Hq, Hk, D, dt in ((8, 2, 128, BF16), (32, 8, 64, F16)):
            check(hip, lens, Hq, Hk, D, 16, dt, (dt,), words=words, masks=junk, pad=2)


def test_attention_any_mask(hip):
    """Bits at random, rows that see nothing of the new tokens, nothing at all (zeros),
    only one far bit; bits past the request's rows do not count."""
    def some(c, rng):
        m = rng.integers(0, 2 ** 32, c.mask.shape, dtype=np.uint32)
        m[::3] = 0
        m[1::7] = 0xFFFFFFFF
        m[2::5] = 0
        m[2::5, -1] = 1 << 20
        return m

    for lens, words in (([(30, 30), (5, 5), (12, 300)], 1), ([(64, 64), (60, 61), (3, 40)], 2), ([(128, 128), (90, 1200)], 4), ([(20, 5), (3, 0)], 1)):
        for Hq, Hk, D, dt in ((8, 2, 128, BF16), (8, 8, 64, F16), (4, 1, 256, BF16)):
            c = check(hip, lens, Hq, Hk, D, 16, dt, (dt, F32), words=words, masks=some, pad=1)
            got = c.run(F32)
            for r, (n, _) in enumerate(lens):
                for i in range(n):
                    if c.sees(r, i).size == 0:
                        assert (got[c.starts[r] + i] == 0).all()


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("n,kv,Hk", [(6, 500, 2), (30, 400, 8), (60, 300, 2), (64, 64, 2)])
def test_attention_not_finite(hip, dt, n, kv, Hk):
    """Infinities and NaN of a drafted token's key and value reach the rows that see it,
    and none of its siblings."""
    D = 128
    rng = np.random.default_rng(n + kv)
    k, v = (rounded(rng.standard_normal((Hk, kv, D)), dt) for _ in range(2))
    base = kv - n
    v[0, base + n // 2, 5] = np.inf
    v[1, base + 1, 9] = np.nan
    k[1, base + n // 3, 3] = np.nan
    c = Trees(hip, [(n, kv)], 2 * Hk, Hk, D, 16, dt, words=2, k=[k], v=[v])
    for out_dt in (F32, dt):
        step(f"jh_paged_tree_attention not finite n={n} kv={kv} dt={dt} out={out_dt}")
        near(c.run(out_dt), c.ref(out_dt))


def test_attention_strides_and_hints(hip):
    c = Trees(hip, [(9, 200), (40, 100), (3, 50)], 8, 2, 128, 16, BF16)
    ref = c.ref(BF16)
    wide = np.full((c.T, 11, 128), np.nan, np.float32)
    wide[:, :8] = c.q
    Q = hip._view(up(hip, wide, BF16), (c.T, 8, 128), (11 * 128, 128, 1))
    both = up(hip, np.stack([c.pools[0], c.pools[1]], 1), BF16)
    shape, st = c.pools[0].shape, (2 * 2 * 16 * 128, 16 * 128, 128, 1)
    K, V = hip._view(both, shape, st), hip._view(both, shape, st, 2 * 16 * 128)
    step("jh_paged_tree_attention strides and hints")
    for max_new in (40, 1, 0, 5, c.T):
        near(c.run(BF16, max_new=max_new, q=Q, k=K, v=V, mask=hip.FromRaw(I32, c.mask.view(np.int32), *c.mask.shape)), ref)


def test_attention_bad_pages_and_lengths(hip):
    """A page outside the pool: NaN for the rows that see a key in it or behind it."""
    for n, words in ((6, 1), (40, 2)):
        c = Trees(hip, [(n, 100), (2, 64)], 4, 2, 128, 16, BF16, words=words, extra_blocks=0)
        tokens, want, bar = c.ref(BF16)
        c.tables[0, 6] = c.n_pages  # keys 96 ..
        c.TAB = ints(hip, c.tables)
        step(f"jh_paged_tree_attention bad page n={n}")
        got = c.run(BF16)
        hit = np.array([c.sees(0, i).max() >= 96 for i in range(n)] + [False, False])
        assert hit.any() and np.isnan(got[:n + 2][hit]).all()
        some = [t for t in tokens if not hit[t]]
        near(got, (some, want[some], bar[some]))
        hip.SetChecks(True)
        try:
            with pytest.raises(JanisHipError, match="jh_paged_tree_attention: page"):
                c.run(BF16)
        finally:
            hip.SetChecks(False)
    c = Trees(hip, [(2, 64), (3, 20)], 4, 2, 64, 16, BF16, extra_blocks=0)
    for starts, kv in (([0, 2, 9], [64, 20]), ([0, 7, 5], [64, 20]), ([-3, 2, 5], [64, 20]), ([0, 2, 5], [2 ** 31 - 1, -5])):
        c.ST, c.KV = ints(hip, starts), ints(hip, kv)
        step(f"jh_paged_tree_attention starts={starts} kv={kv}")
        hip.PagedTreeAttention(c.Q, c.K, c.V, c.TAB, c.ST, c.KV, c.M, c.scale, maxNew=3)
        hip.Sync()


def test_attention_many_requests(hip):
    """More requests than a wave has lanes, most without rows or with one."""
    rng = np.random.default_rng(17)
    n = np.where(rng.random(300) < 0.5, 0, rng.integers(1, 21, 300))
    lens = [(int(x), int(x + rng.integers(0, 300) * (rng.random() < 0.8))) for x in n]
    c = Trees(hip, lens, 8, 8, 64, 16, BF16, words=1, pad=2)
    step(f"jh_paged_tree_attention R=300 rows={c.T}")
    got = c.run(F32)
    near(got, c.ref(F32, rng.integers(0, int(n.sum()), 200)))
    assert np.array_equal(got, c.run(F32))


@pytest.mark.parametrize("Hq,Hk,D,page,dt", [(8, 8, 64, 16, F16), (16, 8, 128, 16, BF16), (8, 4, 256, 32, BF16)])
def test_attention_blocks_of_many_tiles(hip, Hq, Hk, D, page, dt):
    """Blocks that walk several tiles of all kinds, over and over: the same bits each time."""
    rng = np.random.default_rng(D)
    lens = [(int(n), int(n + rng.integers(0, 600))) for n in rng.choice([1, 8, 20, 40, 64, 100], 128 if D < 256 else 64)]
    c = Trees(hip, lens, Hq, Hk, D, page, dt, words=4, pad=1)
    step(f"jh_paged_tree_attention blocks of many tiles R={len(lens)} rows={c.T} Hq={Hq} Hk={Hk} D={D}")
    got = c.run(dt)
    near(got, c.ref(dt, rng.integers(0, c.T - 1, 150)))
    out = up(hip, np.zeros((c.T, Hq, D)), dt)
    want = hip.Bytes(hip.PagedTreeAttention(c.Q, c.K, c.V, c.TAB, c.ST, c.KV, c.M, c.scale, maxNew=100, out=out))
    assert np.array_equal(hip.Floats(out)[:-1], got[:-1])
    for turn in range(60):
        hip.PagedTreeAttention(c.Q, c.K, c.V, c.TAB, c.ST, c.KV, c.M, c.scale, maxNew=100, out=out)
        assert hip.Bytes(out) == want, turn


@pytest.mark.parametrize("where", ["behind", "between", "before", "around"])
@pytest.mark.parametrize("idle", [1, 60, 252, 700, 2044])
def test_attention_idle_slots(hip, where, idle):
    """Requests without rows beside four with some change nothing: the line is the same, and its cuts."""
    active = [(16, 700), (100, 1500), (3, 3000), (40, 200)]
    c = Trees(hip, active, 16, 8, 64, 16, BF16, words=2)
    want = c.run(F32)
    near(want, c.ref(F32))
    gaps = {"behind": [0, 0, 0, 0, idle], "between": [0, idle // 3, idle // 3, idle - 2 * (idle // 3), 0], "before": [idle, 0, 0, 0, 0],
            "around": [idle // 2, 0, 1, 0, idle - idle // 2 - 1] if idle > 1 else [1, 0, 0, 0, 0]}[where]
    starts, kv, tables = [0], [], []
    for i, gap in enumerate(gaps):
        for _ in range(gap):
            starts.append(starts[-1]), kv.append(50), tables.append(np.full(c.tables.shape[1], -1, np.int32))
        if i < 4:
            starts.append(starts[-1] + active[i][0]), kv.append(active[i][1]), tables.append(c.tables[i])
    c.ST, c.KV, c.TAB = ints(hip, starts), ints(hip, kv), ints(hip, np.array(tables))
    step(f"jh_paged_tree_attention {idle} idle slots {where}")
    assert np.array_equal(c.run(F32), want)


def test_attention_more_heads_than_blocks(hip):
    """A block to a kv head, which walks all tiles: nothing is cut, no workspace."""
    lens = [(9, 100), (0, 5), (33, 200), (1, 1)]
    c = Trees(hip, lens, 600, 600, 64, 16, F16, words=2)
    step("jh_paged_tree_attention Hk=600")
    near(c.run(F16), c.ref(F16))


def test_attention_two_contexts_and_streams():
    """Two contexts at once, each with its stream and workspace, on calls whose tiles are cut."""
    import torch
    bs, stream = [HipBackend(0), HipBackend(0)], torch.cuda.Stream()
    bs[1].SetStream(stream.cuda_stream)
    cs = [Trees(b, [(30, 5000), (5, 700)], 32, 8, 128, 16, BF16, seed=i) for i, b in enumerate(bs)]
    want = [c.run(F32) for c in cs]
    outs = [up(b, np.zeros((c.T, c.Hq, c.D)), F32) for b, c in zip(bs, cs)]
    for b in bs:
        b.Sync()
    step("jh_paged_tree_attention of two contexts at once")
    for _ in range(20):
        for b, c, o in zip(bs, cs, outs):
            b.PagedTreeAttention(c.Q, c.K, c.V, c.TAB, c.ST, c.KV, c.M, c.scale, maxNew=30, out=o)
    for b, c, o, w in zip(bs, cs, outs, want):
        assert np.array_equal(b.Floats(o), w)
        near(w, c.ref(F32))
        b.Close()


def far_pool(hip, pool, far):
    """[P, Hk, page, D] bf16 bits with pages `far` elements apart: the buffer, the tensor and its pages."""
    P, Hk, page, D = pool.shape
    raw = hip.empty(BF16, (P - 1) * far + Hk * page * D)
    pages = [hip._view(raw, (Hk, page, D), (page * D, D, 1), i * far) for i in range(P)]
    for view, bits in zip(pages, pool):
        put(hip, view, bits)
    return raw, hip._view(raw, pool.shape, (far, page * D, D, 1)), pages


def test_far_pages(hip):
    """Pages that lie past 2^32 bytes: attention over them, and kept rows moved between them."""
    far = (1 << 31) + 8
    c = Trees(hip, [(12, 20)], 2, 1, 64, 8, BF16, words=1, extra_blocks=0)
    m = Step(1, [12], 8, 1, 1, 1, 64, agree=1.0, far=9)
    want = m.ref()
    assert (np.diff(want[3][want[3] >= 0]) > 1).any()
    try:
        pools = [far_pool(hip, x, far) for x in (synth.f32_to_bf16_bits(c.pools[0]), synth.f32_to_bf16_bits(c.pools[1]), *m.pools[:, 0])]
    except JanisHipError:
        pytest.skip("no room")
    step("jh_paged_tree_attention far pages")
    near(c.run(F32, k=pools[0][1], v=pools[1][1]), c.ref(F32))
    m.up(hip)
    m.lay = PagedLayers([pools[2][1]], [pools[3][1]])
    step("jh_paged_tree_commit far pages")
    m.call(hip)
    got = list(m.got(hip))
    got[7] = np.array([[[np.frombuffer(hip.Bytes(hip._c(v)), np.uint16).reshape(v.shape) for v in pool[2]]] for pool in pools[2:]])
    same(got, want)
    hip.Sync()
    m.lay = None
    for raw, *_ in pools:
        raw.free()


def test_attention_graphs(hip):
    """Captured without a workspace (keys stay whole) and with one, replayed between eager
    calls of another size: each time the eager bits, or the formula's."""
    b = HipBackend(0)
    cs = [Trees(b, [(20, 1500), (1, 40)], 8, 8, 64, 16, F16, seed=1), Trees(b, [(6, 3000), (8, 90)], 32, 8, 128, 16, BF16, seed=2)]
    outs = [up(b, np.zeros((c.T, c.Hq, c.D)), F32) for c in cs]
    call = lambda i: b.PagedTreeAttention(cs[i].Q, cs[i].K, cs[i].V, cs[i].TAB, cs[i].ST, cs[i].KV, cs[i].M, cs[i].scale,  # noqa: E731
                                          maxNew=20, out=outs[i])
    refs = [c.ref(F32) for c in cs]
    step("jh_paged_tree_attention captured first")
    graphs = [Graph(b, lambda: call(0))]
    call(1)
    graphs.append(Graph(b, lambda: call(1)))
    eager = b.Floats(outs[1])
    for turn in range(3):
        for i, c in enumerate(cs):
            put(b, outs[i], np.zeros((c.T, c.Hq, c.D), np.float32))
            graphs[i].replay()
            got = b.Floats(outs[i])
            near(got, refs[i])
            assert i == 0 or np.array_equal(got, eager)
            cs[i].run(F32)
    for g in graphs:
        g.close()
    b.Close()


# ---- the path that the model agrees with ---------------------------------------------------

class Step:
    """One step's trees, tables and pages: `ns` rows of requests with kv keys (the new
    ones among them)."""

    def __init__(self, seed, ns, page=16, words=1, layers=0, Hk=2, D=64, known=None, agree=0.8, pad=3, front=0, far=60, vocab=50):
        rng = np.random.default_rng(seed)
        self.page, self.words, self.R, self.layers, self.Hk, self.D = page, words, len(ns), layers, Hk, D
        self.ns = ns = np.array(ns, np.int32)
        self.kv = (ns + rng.integers(0, far, len(ns))).astype(np.int32)
        self.starts = (front + np.concatenate([[0], np.cumsum(ns)])).astype(np.int32)
        self.T = T = int(self.starts[-1]) + pad
        blocks = -(-self.kv // page)
        self.n_pages = int(blocks.sum()) + 4
        order = rng.permutation(self.n_pages).astype(np.int32)
        self.tables = np.full((self.R, int(blocks.max(initial=0)) + 1), -7, np.int32)
        at = 0
        for r in range(self.R):
            self.tables[r, :blocks[r]] = order[at:at + blocks[r]]
            at += blocks[r]
        self.count = self.n_pages - at
        self.free = np.full(self.n_pages, -9, np.int32)
        self.free[:self.count] = order[at:]
        self.parents, self.slots = np.full(T, -5, np.int32), np.full(T, -1, np.int32)
        self.tokens, self.chosen = rng.integers(0, vocab, T).astype(np.int32), rng.integers(0, vocab, T).astype(np.int32)
        self.known = None if known is None else np.array(known, np.int32)
        for r, n in enumerate(ns):
            a = self.starts[r]
            self.parents[a:a + n] = tree(rng, int(n), 6)
            pos = self.kv[r] - n + np.arange(n)
            self.slots[a:a + n] = self.tables[r, pos // page] * page + pos % page
            for i in range(1, n):  # the model agrees with some child of most rows
                if rng.random() < agree:
                    self.chosen[a + self.parents[a + i]] = self.tokens[a + i]
            if self.known is not None:
                k = min(max(int(self.known[r]), 1), int(n))
                if 0 < k < n and rng.random() < agree:
                    self.parents[a + k], self.chosen[a + k - 1] = k - 1, self.tokens[a + k]
        self.pools = rng.integers(0, 2 ** 15, (2, layers, self.n_pages, Hk, page, D)).astype(np.uint16)

    def ref(self):
        free, top, pools = self.free.copy(), self.count, self.pools.copy()
        after, accepted, nexts, path = [], [], [], np.full(self.T, -1, np.int64)
        for r, n in enumerate(int(x) for x in self.ns):
            a = int(self.starts[r])
            k = n if n > 32 * self.words else min(max(1 if self.known is None else int(self.known[r]), 1), n)
            mine = list(range(k))
            while mine:
                more = [i for i in range(mine[-1] + 1, n) if self.parents[a + i] == mine[-1] and self.tokens[a + i] == self.chosen[a + mine[-1]]]
                if n > 32 * self.words or not more:
                    break
                mine.append(more[0])
            path[a:a + len(mine)] = [a + i for i in mine]
            nexts.append(self.chosen[a + mine[-1]] if mine else -1)
            accepted.append(len(mine))
            new = int(self.kv[r]) - n + len(mine)
            for b in range(-(-new // self.page), -(-int(self.kv[r]) // self.page)):
                free[top] = self.tables[r, b]
                top += 1
            after.append(new)
            for j, i in enumerate(mine):
                s, d = divmod(int(self.slots[a + i]), self.page), divmod(int(self.slots[a + j]), self.page)
                pools[:, :, d[0], :, d[1]] = pools[:, :, s[0], :, s[1]]
        return np.array(after), top, np.array(accepted), path, np.array(nexts), 0, free, pools

    def up(self, b):
        z = lambda a: ints(b, a)  # noqa: E731
        self.d = dict(parents=z(self.parents), tokens=z(self.tokens), starts=z(self.starts), kv=z(self.kv), tables=z(self.tables), free=z(self.free),
                      count=z([self.count]), slots=z(self.slots), known=None if self.known is None else z(self.known), chosen=z(self.chosen))
        shape = self.pools.shape[2:]
        self.k, self.v = ([b.FromBF16Bits(p, *shape) for p in pool] for pool in self.pools)
        self.lay = PagedLayers(self.k, self.v) if self.layers else None
        self.out = [z(np.full(n, -5)) for n in (self.R, 1, self.R, self.T, self.R, 1)]

    def call(self, b, **kw):
        d = dict(self.d, **kw)
        b.PagedTreeCommit(d["parents"], d["tokens"], d["chosen"], d["starts"], d["kv"], self.words, self.page, d["tables"], d["free"], d["count"],
                          d["slots"], layers=self.lay, known=d["known"], out=tuple(self.out))

    def got(self, b):
        o = [b.Ints(t) if t.numel else np.zeros(0, np.int32) for t in self.out]
        bits = lambda t: np.frombuffer(b.Bytes(t), np.uint16).reshape(t.shape)  # noqa: E731
        pools = np.array([[bits(t) for t in ts] for ts in (self.k, self.v)]) if self.layers else self.pools
        return o[0], o[1][0], o[2], o[3], o[4], o[5][0], b.Ints(self.d["free"]), pools


def same(got, want):
    for name, g, w in zip(("kv", "count", "accepted", "path", "next", "status", "free", "pools"), got, want):
        assert np.array_equal(g, w), (name, g, w)


@pytest.mark.parametrize("ns,page,words,layers,Hk,D", [
    ([1], 16, 1, 1, 1, 64), ([12], 16, 1, 3, 8, 128), ([32, 0, 33, 7, 1, 20], 8, 1, 2, 2, 64), ([60] * 9 + [64, 65, 90], 4, 2, 1, 3, 256),
    ([40, 500, 513, 3], 32, 16, 2, 1, 128), ([5] * 70, 1, 1, 0, 1, 64), ([20] * 3, 2, 1, 65, 2, 64), ([9] * 8, 64, 1, 130, 1, 64)])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("agree", [0.0, 0.9, 1.0])
def test_commit(hip, ns, page, words, layers, Hk, D, in_place, agree):
    c = Step(len(ns) + page, ns, page, words, layers, Hk, D, agree=agree, front=2)
    c.up(hip)
    if in_place:
        c.out[0], c.out[1] = c.d["kv"], c.d["count"]
    step(f"jh_paged_tree_commit ns={ns[:6]} page={page} words={words} layers={layers} in_place={in_place} agree={agree}")
    want = c.ref()
    c.call(hip)
    same(c.got(hip), want)


@pytest.mark.parametrize("known", ["one", "some", "all", "past"])
def test_commit_known_rows(hip, known):
    """Known rows are kept whatever the model says, and their parents not looked at."""
    rng = np.random.default_rng(9)
    ns = rng.integers(0, 33, 40)
    k = {"one": np.ones(40), "some": rng.integers(0, 12, 40), "all": ns, "past": np.where(rng.random(40) < 0.5, -3, 2 ** 31 - 1)}[known]
    c = Step(3, ns, 8, 1, 1, known=k)
    c.parents[c.starts[:-1][ns > 0]] = 2 ** 31 - 1
    c.up(hip)
    step(f"jh_paged_tree_commit known={known}")
    want = c.ref()
    c.call(hip)
    same(c.got(hip), want)


def test_commit_choices_apart(hip):
    """The model's tokens as the first column of wider rows; of several children with the
    token the first; parents that are not earlier rows belong to no path."""
    c = Step(5, [20] * 12, 16, 1, 1, vocab=2, agree=1.0)
    c.parents[3::9] = 25
    c.parents[4::11] = -3
    want = c.ref()
    c.up(hip)
    wide = np.full((c.T, 5), -1, np.int32)
    wide[:, 0] = c.chosen
    step("jh_paged_tree_commit choices of two columns")
    c.call(hip, chosen=ints(hip, wide))
    same(c.got(hip), want)
    assert max(want[2]) > 3


@pytest.mark.parametrize("R,n,words", [(700, 20, 1), (2048, 9, 1), (3, 9000, 1), (40, 512, 16), (1, 1, 1)])
def test_commit_many_rows(hip, R, n, words):
    """More rows than the block looks at together; trees across that border; no request."""
    rng = np.random.default_rng(R)
    ns = np.maximum(1, rng.integers(n // 2, n + 1, R))
    if n == 9000:
        ns[1] = 30
    c = Step(R, ns, 16, words, 1 if R < 100 else 0, Hk=1, agree=0.9, far=2000)
    c.up(hip)
    step(f"jh_paged_tree_commit R={R} rows={c.T}")
    want = c.ref()
    c.call(hip)
    same(c.got(hip), want)


def test_commit_no_requests(hip):
    c = Step(1, [], pad=5)
    c.up(hip)
    step("jh_paged_tree_commit without requests")
    c.call(hip)
    got = c.got(hip)
    assert got[1] == c.count and got[5] == 0 and (got[3] == -1).all() and np.array_equal(got[6], c.free)


@pytest.mark.parametrize("what,status", [("kv below the rows", 1), ("kv past the table", 1), ("starts decrease", 2), ("starts leave", 2), ("starts below", 2),
                                         ("count below", 3), ("count past", 3), ("page outside", 4), ("page below", 4), ("no room", 4)])
@pytest.mark.parametrize("in_place", [False, True])
def test_commit_refused_on_the_device(hip, what, status, in_place):
    """Then nothing is done: lengths, stack, keys and values are as they were."""
    c = Step(11, [20, 0, 30, 5], 4, 1, 2, agree=0.6)
    want = c.ref()
    back = want[1] - c.count
    assert back > 1 and (np.diff(want[3][:20][want[3][:20] >= 0]) > 1).any()
    if what == "kv below the rows": c.kv[2] = 29
    if what == "kv past the table": c.kv[1] = c.tables.shape[1] * 4 + 1
    if what.startswith("starts"): c.kv[:] = c.tables.shape[1] * 4
    if what == "starts decrease": c.starts[1:3] = 30, 20
    if what == "starts leave": c.starts[4] = c.T + 1
    if what == "starts below": c.starts[0] = -1
    if what == "count below": c.count = -1
    if what == "count past": c.count = c.n_pages + 1
    if what == "page outside": c.tables[2, -(-int(c.kv[2]) // 4) - 1] = c.n_pages
    if what == "page below": c.tables[2, -(-int(c.kv[2]) // 4) - 1] = -1
    if what == "no room": c.count = c.n_pages - back + 1
    c.up(hip)
    if in_place:
        c.out[0], c.out[1] = c.d["kv"], c.d["count"]
    step(f"jh_paged_tree_commit refuses: {what}")
    c.call(hip)
    none = np.full(4, -1)
    same(c.got(hip), (c.kv, c.count, np.zeros(4), np.full(c.T, -1), none, status, c.free, c.pools))
    hip.SetChecks(True)
    try:
        with pytest.raises(JanisHipError, match="nothing done") as e:
            c.call(hip)
        assert e.value.code == _lib.JH_ERR_INVALID
    finally:
        hip.SetChecks(False)


@pytest.mark.parametrize("n,page,words,layers,Hk,D,known", [
    (32, 16, 1, 2, 1, 64, None), (33, 16, 1, 2, 1, 64, None), (64, 4, 2, 70, 2, 64, 3), (512, 1, 16, 1, 3, 128, 40), (511, 64, 16, 2, 2, 256, 500),
    (130, 8, 5, 0, 1, 64, 1), (0, 16, 1, 2, 1, 64, None), (700, 16, 16, 1, 1, 64, 9)])
@pytest.mark.parametrize("in_place", ["", "kv", "count"])
def test_commit_single_request(hip, n, page, words, layers, Hk, D, known, in_place):
    """A request by itself takes one launch where nothing is updated in place."""
    c = Step(n, [n], page, words, layers, Hk, D, known=None if known is None else [known], agree=0.97, front=1, far=300)
    c.up(hip)
    if in_place == "kv":
        c.out[0] = c.d["kv"]
    if in_place == "count":
        c.out[1] = c.d["count"]
    step(f"jh_paged_tree_commit n={n} page={page} words={words} layers={layers} known={known} in_place={in_place!r}")
    want = c.ref()
    c.call(hip)
    same(c.got(hip), want)


@pytest.mark.parametrize("what,status", [("kv below the rows", 1), ("starts leave", 2), ("count past", 3), ("page outside", 4), ("no room", 4)])
@pytest.mark.parametrize("in_place", [False, True])
def test_commit_single_request_refused_on_the_device(hip, what, status, in_place):
    c = Step(11, [30], 4, 1, 2, agree=0.6)
    want = c.ref()
    back = want[1] - c.count
    assert back > 1 and (np.diff(want[3][want[3] >= 0]) > 1).any()
    if what == "kv below the rows": c.kv[0] = 29
    if what == "starts leave": c.starts[1] = c.T + 1
    if what == "count past": c.count = c.n_pages + 1
    if what == "page outside": c.tables[0, -(-int(c.kv[0]) // 4) - 1] = c.n_pages
    if what == "no room": c.count = c.n_pages - back + 1
    c.up(hip)
    if in_place:
        c.out[0], c.out[1] = c.d["kv"], c.d["count"]
    step(f"jh_paged_tree_commit of one request refuses: {what}")
    c.call(hip)
    same(c.got(hip), (c.kv, c.count, np.zeros(1), np.full(c.T, -1), np.full(1, -1), status, c.free, c.pools))


@pytest.mark.parametrize("what,status", [("kv below the rows", 1), ("count below", 3), ("count past", 3)])
@pytest.mark.parametrize("n,words,front", [(600, 1, 37), (90, 2, 100), (513, 16, 5)])
@pytest.mark.parametrize("in_place", [False, True])
def test_commit_single_run_refused_on_the_device(hip, what, status, n, words, front, in_place):
    """A request of more rows than bits, behind rows that nobody has: path is -1 everywhere."""
    c = Step(n, [n], 16, words, 1, front=front, pad=70)
    if what == "kv below the rows": c.kv[0] = n - 1
    if what == "count below": c.count = -1
    if what == "count past": c.count = c.n_pages + 1
    c.up(hip)
    if in_place:
        c.out[0], c.out[1] = c.d["kv"], c.d["count"]
    step(f"jh_paged_tree_commit of one run of {n} behind {front} rows refuses: {what}")
    for _ in range(20):
        c.call(hip)
        same(c.got(hip), (c.kv, c.count, np.zeros(1), np.full(c.T, -1), np.full(1, -1), status, c.free, c.pools))


@pytest.mark.parametrize("n,words,front", [(600, 1, 37), (90, 2, 100)])
def test_commit_single_run(hip, n, words, front):
    c = Step(n, [n], 16, words, 1, front=front, pad=70)
    c.up(hip)
    step(f"jh_paged_tree_commit of one run of {n} behind {front} rows")
    c.call(hip)
    same(c.got(hip), c.ref())


def test_commit_captured_first():
    """The workspace cannot grow in a capture: the same call goes before it. Replays find
    other lengths, paths and pages."""
    b = HipBackend(0)
    c = Step(8, [20] * 40, 16, 4, 2, agree=0.9)
    c.up(b)
    step("jh_paged_tree_commit captured first")

    def refused():
        with pytest.raises(JanisHipError, match="make the same call once before"):
            c.call(b)
    Graph(b, refused).close()
    c.call(b)
    same(c.got(b), c.ref())
    graph = Graph(b, lambda: c.call(b))
    for seed in (9, 10, 11):  # other trees over the same slots
        m = Step(seed, [20] * 40, 16, 4, 2, agree=0.9)
        c.parents, c.tokens, c.chosen = m.parents, m.tokens, m.chosen
        for name in ("parents", "tokens", "chosen", "free"):
            put(b, c.d[name], getattr(c, name))
        for ts, pool in zip((c.k, c.v), c.pools):
            for t, bits in zip(ts, pool):
                put(b, t, bits)
        graph.replay()
        same(c.got(b), c.ref())
        other = Step(1, [3] * 5, 16, 1, 1)  # (another call's heads and moves in the same workspace)
        other.up(b)
        other.call(b)
        same(other.got(b), other.ref())
    graph.close()
    b.Close()


def test_commit_slots_outside(hip):
    """Rows whose slot is outside the pages are not moved, and none is written there."""
    c = Step(21, [25] * 6, 16, 1, 2, agree=1.0)
    want = list(c.ref())
    moved = [(j, int(i)) for j, i in enumerate(want[3]) if i >= 0 and i != j]
    pools = c.pools.copy()
    c.slots[moved[0][0]] = c.n_pages * 16
    c.slots[moved[1][1]] = -1
    c.slots[moved[2][1]] = -2 ** 31
    for j, i in moved[:1] + moved[3:]:
        s, d = int(c.slots[i]), int(c.slots[j])
        if 0 <= s < c.n_pages * 16 and 0 <= d < c.n_pages * 16:
            pools[:, :, d // 16, :, d % 16] = pools[:, :, s // 16, :, s % 16]
    for j, i in moved[1:3]:
        s, d = int(c.slots[i]), int(c.slots[j])
        assert not 0 <= s < c.n_pages * 16 or not 0 <= d < c.n_pages * 16
    c.up(hip)
    step("jh_paged_tree_commit slots outside")
    c.call(hip)
    want[7] = pools
    same(c.got(hip), want)


def test_commit_pages_apart(hip):
    """Layers whose keys and values alternate in one buffer, f16."""
    c = Step(31, [25] * 6, 16, 1, 2, agree=1.0)
    want = c.ref()
    c.up(hip)
    N, Hk, page, D = c.pools.shape[2:]
    both = [hip.FromRaw(F16, np.stack([c.pools[0, i], c.pools[1, i]], 1), N, 2, Hk, page, D) for i in range(2)]
    st = (2 * Hk * page * D, page * D, D, 1)
    views = [[hip._view(t, (N, Hk, page, D), st, x * Hk * page * D) for t in both] for x in (0, 1)]
    c.lay = PagedLayers(*views)
    step("jh_paged_tree_commit pages apart")
    c.call(hip)
    got = list(c.got(hip))
    raw = [np.frombuffer(hip.Bytes(t), np.uint16).reshape(N, 2, Hk, page, D) for t in both]
    got[7] = np.array([[t[:, x] for t in raw] for x in (0, 1)])
    same(got, want)


# ---- refusals ------------------------------------------------------------------------------

def test_refusals(hip):
    INVALID, UNSUPPORTED = _lib.JH_ERR_INVALID, _lib.JH_ERR_UNSUPPORTED
    import ctypes
    t = hip.empty(F32, 1 << 16)
    p = t.ptr
    good = dict(par=p, starts=p, kv=p, R=2, T=4, words=1, pos=p + 4096, mask=p + 8192)
    refused(hip, "jh_paged_tree_plan", good, [
        (INVALID, dict(words=0)), (UNSUPPORTED, dict(words=17)), (INVALID, dict(R=-1)), (INVALID, dict(T=-1)), (UNSUPPORTED, dict(R=65537)),
        (UNSUPPORTED, dict(T=(1 << 30) + 1))] + [(INVALID, {k: None}) for k in ("par", "starts", "kv", "pos", "mask")])
    good = dict(q=p, qs=2 * 64, k=p, v=p, pdt=BF16, pages=2, page=16, pstride=2 * 16 * 64, tab=p, blocks=2, starts=p, kv=p, mask=p, words=1, R=1,
                T=2, new=1, hq=2, hk=2, d=64, scale=0.1, out=p, odt=BF16)
    refused(hip, "jh_paged_tree_attention", good, [
        (INVALID, dict(words=0)), (UNSUPPORTED, dict(words=17)), (INVALID, dict(mask=None)), (UNSUPPORTED, dict(pdt=F32)), (INVALID, dict(odt=I32)),
        (INVALID, dict(pages=0)), (INVALID, dict(page=20)), (UNSUPPORTED, dict(page=4)), (INVALID, dict(hq=3)), (UNSUPPORTED, dict(d=32)),
        (INVALID, dict(qs=64)), (INVALID, dict(R=-1)), (UNSUPPORTED, dict(T=1 << 30)), (INVALID, dict(scale=0.0)), (INVALID, dict(q=p + 8)),
        (INVALID, dict(k=p + 2))] + [(INVALID, {k: None}) for k in ("q", "k", "v", "tab", "starts", "kv", "out")])
    one = lambda x: (ctypes.c_void_p * 1)(x)  # noqa: E731
    good = dict(par=p, tok=p, cho=p, cs=1, known=p, starts=p, kv=p, R=2, T=4, words=1, page=16, tab=p, blocks=2, free=p, pages=2, count=p, slots=p,
                kvo=p, co=p, acc=p, path=p, nxt=p, status=p, ks=one(p), vs=one(p), layers=1, pdt=BF16, hk=2, d=64, pstride=2 * 16 * 64)
    refused(hip, "jh_paged_tree_commit", good, [
        (INVALID, dict(words=0)), (UNSUPPORTED, dict(words=17)), (INVALID, dict(cs=0)), (INVALID, dict(R=-1)), (INVALID, dict(T=-1)),
        (UNSUPPORTED, dict(R=2049)), (UNSUPPORTED, dict(T=(1 << 30) + 1)), (INVALID, dict(page=0)), (INVALID, dict(page=24)), (INVALID, dict(pages=-1)),
        (INVALID, dict(blocks=-1)), (INVALID, dict(layers=-1)), (UNSUPPORTED, dict(layers=65537)), (UNSUPPORTED, dict(pdt=F32)), (INVALID, dict(pdt=I32)),
        (UNSUPPORTED, dict(d=96)), (INVALID, dict(hk=0)), (INVALID, dict(pstride=64)), (INVALID, dict(pstride=2 * 16 * 64 + 4)),
        (INVALID, dict(ks=one(p + 8))), (INVALID, dict(vs=one(None))), (INVALID, dict(ks=None)), (INVALID, dict(vs=None))] +
        [(INVALID, {k: None}) for k in ("par", "tok", "cho", "starts", "kv", "tab", "free", "count", "slots", "kvo", "co", "acc", "path", "nxt", "status")])


def test_nothing_to_do(hip):
    L, c = hip._L, hip._ctx
    assert L.jh_paged_tree_plan(c, None, None, None, 3, 0, 1, None, None) == 0
    assert L.jh_paged_tree_attention(c, None, 64, None, None, BF16, 1, 16, 1024, None, 0, None, None, None, 1, 1, 0, 0, 1, 1, 64, 0.1, None, BF16) == 0


def test_checks_refuse_a_capture(hip):
    """Checks read indices back, which a stream under capture cannot do."""
    c, t = Step(1, [5]), Trees(hip, [(5, 40)], 4, 2, 64, 16, BF16)
    c.up(hip)

    def calls():
        for call in (lambda: c.call(hip), lambda: run_checked_plan(), lambda: hip.PagedTreeAttention(
                t.Q, t.K, t.V, t.TAB, t.ST, t.KV, t.M, t.scale, out=out)):
            with pytest.raises(JanisHipError, match="capturing"):
                call()

    out = up(hip, np.zeros((t.T, 4, 64)), F32)
    pos, mask = ints(hip, np.zeros(c.T)), hip.FromRaw(U32, np.zeros((c.T, 1), np.uint32), c.T, 1)
    run_checked_plan = lambda: hip.PagedTreePlan(c.d["parents"], c.d["starts"], c.d["kv"], out=(pos, mask))  # noqa: E731
    hip.SetChecks(True)
    try:
        step("checked calls under capture")
        Graph(hip, calls).close()
    finally:
        hip.SetChecks(False)


# ---- a step of them together ------------------------------------------------------------

def test_step_captured():
    """A server's steps with drafts as one captured graph -- plan, tree plan, append,
    attention, logits, their likeliest tokens, commit -- of a model of two layers whose
    next token depends on all before it, replayed over changing batches. Drafts are half
    right; what is kept has to be the sequence that the model makes alone, token by
    token, in 64 bits."""
    V, Hq, Hk, D, page, R, T, B, n_pages, words, L = 61, 4, 2, 64, 8, 4, 96, 20, 64, 1, 2
    rng = np.random.default_rng(2)
    b = HipBackend(0)
    width = (Hq + 2 * Hk) * D
    # row -> q/k/v of both layers by token (a layer here reads the embedding and the result of
    # the layer before it through the host: what is tested is the cache around it)
    emb = rounded(2.5 * rng.standard_normal((L, V, width)), BF16)
    head = rounded(rng.standard_normal((V, Hq * D)), BF16).astype(np.float64)
    inv = 1e4 ** (-2.0 * np.arange(D // 2) / D)
    new, kv, tables = ints(b, np.zeros(R)), ints(b, np.zeros(R)), ints(b, np.full((R, B), -1))
    free, count = ints(b, np.arange(n_pages)), ints(b, [n_pages])
    starts, pos, slots, status = ints(b, np.zeros(R + 1)), ints(b, np.zeros(T)), ints(b, np.zeros(T)), ints(b, [0])
    parents, tokens, known = ints(b, np.zeros(T)), ints(b, np.zeros(T)), ints(b, np.ones(R))
    mask = b.FromRaw(U32, np.zeros((T, words), np.uint32), T, words)
    qkv = [b.FromBF16Bits(np.zeros((T, width), np.uint16), T, width) for _ in range(L)]
    caches = [[up(b, np.full((n_pages, Hk, page, D), np.nan), F16) for _ in range(L)] for _ in range(2)]
    layers = PagedLayers(*caches)
    q = [up(b, np.zeros((T, Hq, D)), F16) for _ in range(L)]
    out = [up(b, np.zeros((T, Hq, D)), F32) for _ in range(L)]
    logits, chosen = up(b, np.zeros((T, V)), F32), ints(b, np.zeros((T, 3)))
    ent, top = up(b, np.zeros(T), F32), up(b, np.zeros((T, 3)), F32)
    done = [ints(b, np.zeros(n)) for n in (R, T, R, 1)]  # accepted, path, next, status

    def first_half():
        b.PagedPlan(new, kv, page, tables, free, count, out=(kv, count, starts, pos, slots, status))
        b.PagedTreePlan(parents, starts, kv, out=(pos, mask))
        for i in range(L):
            b.PagedQKNormRoPEAppend(qkv[i], Hq, Hk, None, None, 1e-6, 1e4, 1.0, pos, slots, caches[0][i], caches[1][i], q_out=q[i])
            b.PagedTreeAttention(q[i], caches[0][i], caches[1][i], tables, starts, kv, mask, D ** -0.5, maxNew=T, out=out[i])

    def second_half():
        b.TokenLogProbs(logits, topK=3, out=(None, ent, chosen, top))
        b.PagedTreeCommit(parents, tokens, chosen, starts, kv, words, page, tables, free, count, slots, layers=layers, known=known,
                          out=(kv, count, *done))

    step("drafted step, eager, then captured")
    first_half(), second_half()
    b.Sync()
    graphs = [Graph(b, first_half), Graph(b, second_half)]

    def alone(seq):
        """The model's logits after seq, in 64 bits."""
        x = np.zeros(Hq * D)
        for i in range(L):
            p = np.arange(len(seq))
            Q, K, W = append_ref(emb[i][seq], Hq, Hk, D, None, None, 0.0, p[:, None] * inv, None, None)
            for h in range(Hq):
                s = K[:, h // 2] @ Q[-1, h] * D ** -0.5
                e = np.exp(s - s.max())
                x[h * D:(h + 1) * D] += (e / e.sum()) @ W[:, h // 2]
        return head @ x

    seqs = [list(rng.integers(0, V, n)) for n in (1, 9, 40, 3)]  # what is known; the last of it is not in the cache
    held = [0] * R
    total = 0
    for turn in range(9):
        ns, par, tok, kn = [], np.full(T, -1, np.int32), np.zeros(T, np.int32), []
        at = 0
        for r in range(R):
            if turn == 4 and r == 1:  # idle
                ns.append(0), kn.append(1)
                continue
            fresh = seqs[r][held[r]:]
            rows = [(i - 1, t) for i, t in enumerate(fresh)]
            if len(fresh) < 20:  # drafts: the model's own next tokens among others
                ahead, end = list(seqs[r]), len(rows) - 1
                for _ in range(3):
                    right = int(np.argmax(alone(ahead)))
                    wrong = [int(x) for x in rng.integers(0, V, 2)]
                    last = end
                    for t in (wrong[0], right, wrong[1]) if rng.random() < 0.75 else wrong:
                        rows.append((last, t))
                        if t == right and end == last:
                            end = len(rows) - 1
                    if end == last:
                        break
                    ahead.append(right)
            ns.append(len(rows)), kn.append(len(fresh))
            par[at:at + len(rows)], tok[at:at + len(rows)] = zip(*rows)
            at += len(rows)
        assert at <= T
        put(b, new, np.array(ns, np.int32)), put(b, parents, par), put(b, tokens, tok), put(b, known, np.array(kn, np.int32))
        for i in range(L):
            put(b, qkv[i], (emb[i][tok].view(np.uint32) >> 16).astype(np.uint16))
        before = b.Ints(kv)
        graphs[0].replay()
        assert b.Ints(status)[0] == 0
        x = sum(b.Floats(o).reshape(T, -1).astype(np.float64) for o in out)
        lg = (x @ head.T).astype(np.float32)
        put(b, logits, lg)
        graphs[1].replay()
        accepted, path, nxt, st = (b.Ints(t) for t in done)
        assert st[0] == 0
        at = 0
        for r in range(R):
            if not ns[r]:
                assert accepted[r] == 0 and nxt[r] == -1
                continue
            mine = path[at:at + accepted[r]]
            assert (np.diff(mine) > 0).all() and list(mine[:kn[r]] - at) == list(range(kn[r]))
            gained = [int(tok[t]) for t in mine[kn[r]:]] + [int(nxt[r])]
            for t in gained:  # (f16 queries, keys and values: near ties of the two best aside)
                z = alone(seqs[r])
                best = np.sort(z)[-2:]
                assert t == np.argmax(z) or best[1] - z[t] < 0.02 * np.abs(z).max(), (turn, r)
                seqs[r].append(t)
            total += len(gained) - 1
            held[r] = len(seqs[r]) - 1
            at += ns[r]
        nkv, ntab = b.Ints(kv), b.Ints(tables)
        assert list(nkv) == held and (nkv >= before).all()
        pages = [int(ntab[r, c]) for r in range(R) for c in range(-(-int(nkv[r]) // page))]
        left = list(b.Ints(free)[:b.Ints(count)[0]])
        assert sorted(pages + left) == list(range(n_pages))
        # the cache holds the kept tokens' keys, one after the other
        for r in range(R):
            for i in range(L):
                K = append_ref(emb[i][seqs[r][:held[r]]], Hq, Hk, D, None, None, 0.0, np.arange(held[r])[:, None] * inv, None, None)[1]
                pool = b.Floats(caches[0][i])
                mine = pool[ntab[r, :-(-held[r] // page)]].transpose(1, 0, 2, 3).reshape(Hk, -1, D)[:, :held[r]]
                assert (np.abs(mine.transpose(1, 0, 2) - K) <= 2.0 ** -10 * np.maximum(np.abs(K), 1.0) * 8).all(), (turn, r, i)
    assert total > 12  # drafts were kept
    for g in graphs:
        g.close()
    b.Close()
