"""Log probabilities of given tokens, entropy and likeliest tokens against the formula in
64 bits.

Bars, with d = scale (x - max x): a difference is rounded once and multiplied (two roundings
of d), e^d is off by 2^-22 of itself beside e^d |d| 2^-23, so that a sum of n of them, made
in fp32 by at most n / 64 + 64 additions in a row, is off by (n / 64 + 128) 2^-24 of itself
and as much again for the exponentials, whose mean |d| enters; its logarithm by as much, and by
2^-23 of itself. A log probability adds the rounding of its own d and of the result; the
entropy is a logarithm less a quotient of two such sums."""
import numpy as np
import pytest

from janis_amd import _lib
from janis_amd.engine import BF16, F32, HipBackend, JanisHipError
from tests.conftest import Graph, put, step
from tests.test_gpu_paged import ints, refused, rounded, up

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def ref(x, scale, tokens, k):
    """(logprobs, bar, entropy, bar, ids, their logprobs, bar) of rows x; NaN rows as the
    header has them."""
    x = x.astype(np.float64)
    T, V = x.shape
    bad = np.isnan(x).any(1) | (x == np.inf).any(1) | (x == -np.inf).all(1)
    with np.errstate(all="ignore"):
        d = scale * (x - x.max(1, keepdims=True))
        e = np.where(x == -np.inf, 0.0, np.exp(d))
        S = e.sum(1)
        dd = np.where(e > 0, d, 0.0)
        mean = (e * np.abs(dd)).sum(1) / S
        H = np.log(S) - (e * dd).sum(1) / S
    rel = (V / 64 + 128) * U * 2 + 4 * U * (1 + mean)
    bar_ln = rel + 2 * U * np.log(np.maximum(S, 1.0))
    bar_h = bar_ln + mean * (2 * rel + 4 * U) + 2 * U * np.abs(H)
    ln = np.log(np.where(S > 0, S, 1.0))[:, None]
    lp = lambda at: np.take_along_axis(d, at, 1) - ln  # noqa: E731
    bar_lp = lambda v: bar_ln[:, None] + 4 * U * (np.abs(v) + ln) + U  # noqa: E731
    key = np.where(np.isnan(x), -np.inf, x) + 0.0
    ids = np.argsort(-key, axis=1, kind="stable")[:, :k]
    out = []
    for at in (tokens, ids):
        if at is None:
            out.append((None, None))
            continue
        ok = (at >= 0) & (at < V)
        v = np.where(ok, lp(np.where(ok, at, 0)), np.nan)
        v[bad] = np.nan
        out.append((v, bar_lp(np.where(np.isfinite(v), v, 0.0))))
    H[bad] = np.nan
    return *out[0], H, bar_h, ids, *out[1]


def close(got, want, bar, what):
    g = got.astype(np.float64)
    assert np.array_equal(np.isnan(g), np.isnan(want)), what
    assert np.array_equal(g == -np.inf, want == -np.inf) and not (g == np.inf).any(), what
    fine = np.isfinite(want)
    off = np.abs(np.where(fine, g, 0.0) - np.where(fine, want, 0.0)) - bar
    assert (off[fine] <= 0).all(), (what, float(off[fine].max()))


def check(hip, x, dt, scale=1.0, tokens=None, k=0, entropy=True, X=None):
    X = up(hip, x, dt) if X is None else X
    t = None if tokens is None else ints(hip, tokens)
    step(f"jh_token_logprobs {x.shape} dt={dt} scale={scale} tokens={None if tokens is None else tokens.shape} k={k} entropy={entropy}")
    lp, ent, ids, top = hip.TokenLogProbs(X, t, k, scale, entropy)
    two = None if tokens is None else tokens.reshape(x.shape[0], -1)
    want = ref(x, np.float64(np.float32(scale)), two, k)
    if tokens is not None:
        close(hip.Floats(lp).reshape(two.shape), want[0], want[1], "logprobs")
    if entropy:
        close(hip.Floats(ent), want[2], want[3], "entropy")
    if k:
        assert np.array_equal(hip.Ints(ids), want[4]), "ids"
        close(hip.Floats(top), want[5], want[6], "top")
    return want


def some(rng, T, V, dt, size=3.0):
    return rounded(size * rng.standard_normal((T, V)), dt)


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("T,V,k,n", [(1, 1, 1, 1), (1, 7, 7, 2), (3, 8, 5, 1), (2, 31, 31, 3), (5, 33, 32, 1), (4, 100, 1, 64), (2, 1023, 20, 1), (7, 1025, 32, 4),
                                     (3, 4097, 8, 1), (1, 8191, 20, 1), (2, 16385, 20, 0), (1, 50021, 20, 1), (9, 32001, 0, 2), (1, 151936, 32, 1),
                                     (6, 151936, 5, 3), (1, 300007, 20, 1)])
def test_logprobs(hip, dt, T, V, k, n):
    rng = np.random.default_rng(V + T)
    check(hip, some(rng, T, V, dt), dt, tokens=rng.integers(0, V, (T, n)).astype(np.int32) if n else None, k=k)


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("T,V,k", [(300, 1003, 5), (700, 517, 32), (2500, 65, 3), (80, 40001, 20), (33, 151936, 2)])
def test_logprobs_many_rows(hip, dt, T, V, k):
    rng = np.random.default_rng(V)
    check(hip, some(rng, T, V, dt), dt, tokens=rng.integers(0, V, T).astype(np.int32), k=k)


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("V", [500, 8200, 50021, 151936])
def test_logprobs_ties(hip, dt, V):
    """Equal logits: the lower token first, also where thousands are equal."""
    rng = np.random.default_rng(V)
    x = np.zeros((8, V), np.float32)
    x[1] = -0.0
    x[1, ::3] = 0.0
    x[2] = rng.integers(0, 3, V)
    x[3] = np.arange(V) % 7
    x[4, V // 2:] = 1.0
    x[5] = -np.arange(V)  # falling
    x[6] = np.arange(V)  # rising
    x[7, rng.permutation(V)[:12]] = 2.0
    x = rounded(x, dt)
    for k in (1, 5, 32):
        check(hip, x, dt, tokens=np.full((8, 1), V - 1, np.int32), k=k)


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("T,V", [(6, 300), (6, 33000), (6, 151936), (200, 5001)])
def test_logprobs_masked_and_not_finite(hip, dt, T, V):
    """Rows of which few tokens are left, rows of -inf alone, and rows with a NaN or +inf."""
    rng = np.random.default_rng(T + V)
    x = some(rng, T, V, dt)
    keep = rng.random((T, V)) < 0.01
    keep[:, V // 2] = True
    x[~keep] = -np.inf
    x[0, :] = -np.inf
    x[0, 17] = 3.0
    x[1, :] = -np.inf
    x[2, V - 1] = np.nan
    x[3, 5] = np.inf
    x[4, :V // 2] = some(rng, 1, V // 2, dt)[0]
    tokens = np.tile(np.array([17, V // 2, 0], np.int32), (T, 1))
    for k in (0, 3, 32):
        check(hip, x, dt, tokens=tokens, k=k)
    # tokens that stand together, and those of one lane of a block
    x = np.full((3, V), -np.inf, np.float32)
    x[0, :V // 3] = some(rng, 1, V // 3, dt)[0]
    x[1, ::64] = some(rng, 1, -(-V // 64), dt)[0]
    x[2, V // 2:V // 2 + 20] = some(rng, 1, 20, dt)[0]
    check(hip, x, dt, tokens=np.full((3, 1), V // 2, np.int32), k=32)


def test_logprobs_tokens_outside(hip):
    """NaN for a token that is none; refused with checks on, -1 aside."""
    rng = np.random.default_rng(3)
    x = some(rng, 4, 900, F32)
    t = np.array([[-1, 0], [900, 899], [2 ** 31 - 1, -2 ** 31], [5, -1]], np.int32)
    check(hip, x, F32, tokens=t, k=2)
    hip.SetChecks(True)
    try:
        with pytest.raises(JanisHipError, match="token 900"):
            check(hip, x, F32, tokens=t)
        t[1:3] = -1
        check(hip, x, F32, tokens=t, k=2)
    finally:
        hip.SetChecks(False)


@pytest.mark.parametrize("scale", [1e-30, 1e-3, 0.7, 1.7, 50.0, 1e30])
def test_logprobs_scales(hip, scale):
    rng = np.random.default_rng(5)
    for dt, V in ((BF16, 3001), (F32, 20000)):
        check(hip, some(rng, 5, V, dt), dt, scale=scale, tokens=rng.integers(0, V, 5).astype(np.int32), k=4)


def test_logprobs_sizes_of_logits(hip):
    """Far from 0, peaked (a log probability near 0 keeps its digits), and as large as differences can be in fp32."""
    rng = np.random.default_rng(6)
    V = 5003
    x = some(rng, 5, V, F32)
    x[0] += 3000.0
    x[1, 77] = 40.0
    x[2] *= 1e-3
    x[3] = 1e38 * np.sign(x[3])
    x[4, 5] = 25.0
    t = np.array([[77, 5]] * 5, np.int32)
    want = check(hip, x, F32, tokens=t, k=6)
    assert -1e-6 < want[0][1, 0] < 0
    check(hip, rounded(x[[0, 1, 2, 4]], BF16), BF16, tokens=t[:4], k=6)


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("extra", [1, 3, 8, 100])
def test_logprobs_rows_apart(hip, dt, extra):
    """Rows inside wider ones (a padded vocabulary), whose rest holds NaN; any alignment of a row."""
    rng = np.random.default_rng(extra)
    for T, V in ((9, 1001), (4, 20003), (300, 70)):
        wide = np.full((T, V + extra), np.nan, np.float32)
        wide[:, :V] = some(rng, T, V, dt)
        W = up(hip, wide, dt)
        check(hip, wide[:, :V], dt, tokens=rng.integers(0, V, T).astype(np.int32), k=9, X=hip._view(W, (T, V), (V + extra, 1)))


def test_logprobs_shapes_of_the_mirror(hip):
    """Leading axes, one row without any, results that are given and results that are not wanted."""
    rng = np.random.default_rng(8)
    x = some(rng, 6, 300, F32)
    want = ref(x, 1.0, np.full((6, 1), 4), 3)
    X = up(hip, x.reshape(2, 3, 300), F32)
    lp, ent, ids, top = hip.TokenLogProbs(X, ints(hip, np.full((2, 3), 4)), 3)
    assert lp.shape == (2, 3) and ent.shape == (2, 3) and ids.shape == top.shape == (2, 3, 3)
    close(hip.Floats(lp).reshape(6, 1), want[0], want[1], "logprobs")
    assert np.array_equal(hip.Ints(ids).reshape(6, 3), want[4])
    lp, ent, ids, top = hip.TokenLogProbs(up(hip, x[0], F32), None, 3, entropy=False)
    assert lp is None and ent is None and ids.shape == (3,) and np.array_equal(hip.Ints(ids), want[4][0])
    mine = up(hip, np.zeros(6), F32)
    assert hip.TokenLogProbs(up(hip, x, F32), out=(None, mine, None, None))[1] is mine
    close(hip.Floats(mine), want[2], want[3], "entropy")
    assert hip.TokenLogProbs(up(hip, x, F32), entropy=False) == (None, None, None, None)


def test_logprobs_graphs_and_growth():
    """Captured calls of different sizes on one context, replayed in turn, also after a call
    that grew the workspace: the eager bits. A capture that the workspace is too small for
    says so."""
    b = HipBackend(0)
    rng = np.random.default_rng(9)
    xs = [some(rng, 1, 151936, F32), some(rng, 12, 50021, BF16)]
    X = [up(b, xs[0], F32), up(b, xs[1], BF16)]
    big = up(b, some(rng, 64, 151936, BF16), BF16)
    outs = [(None, up(b, np.zeros(T), F32), ints(b, np.zeros((T, 20))), up(b, np.zeros((T, 20)), F32)) for T in (1, 12)]
    call = lambda i: b.TokenLogProbs(X[i], topK=20, out=outs[i])  # noqa: E731
    read = lambda i: [b.Floats(outs[i][1]), b.Ints(outs[i][2]), b.Floats(outs[i][3])]  # noqa: E731
    step("jh_token_logprobs eager, captured, replayed")
    call(0), call(1)
    wants = [read(i) for i in range(2)]
    graphs = [Graph(b, lambda i=i: call(i)) for i in range(2)]
    for turn in range(4):
        if turn == 2:
            b.TokenLogProbs(big, topK=32)
        for i in range(2):
            for t in outs[i][1:]:
                put(b, t, np.zeros(t.shape, np.float32))
            graphs[i].replay()
            assert all(np.array_equal(g, w) for g, w in zip(read(i), wants[i])), (turn, i)
            call(1 - i)
    for g in graphs:
        g.close()
    b.Close()


def test_logprobs_captured_first():
    """Rows that are split need a workspace, which cannot grow in a capture: the call says so, and works
    after one outside."""
    b = HipBackend(0)
    x = some(np.random.default_rng(14), 3, 50021, F32)
    X = up(b, x, F32)
    out = (None, up(b, np.zeros(3), F32), ints(b, np.zeros((3, 4))), up(b, np.zeros((3, 4)), F32))
    call = lambda: b.TokenLogProbs(X, topK=4, out=out)  # noqa: E731
    step("jh_token_logprobs captured first")

    def refused_call():
        with pytest.raises(JanisHipError, match="make the same call once before") as e:
            call()
        assert e.value.code == _lib.JH_ERR_INVALID
    Graph(b, refused_call).close()
    call()
    graph = Graph(b, call)
    want = ref(x, 1.0, None, 4)
    for _ in range(3):
        put(b, out[1], np.zeros(3, np.float32)), put(b, out[2], np.zeros((3, 4), np.int32))
        graph.replay()
        close(b.Floats(out[1]), want[2], want[3], "entropy")
        assert np.array_equal(b.Ints(out[2]), want[4])
        call()
    graph.close()
    b.Close()


def test_logprobs_two_contexts_and_streams():
    import torch

    bs = [HipBackend(0), HipBackend(0)]
    stream = torch.cuda.Stream()
    bs[1].SetStream(stream.cuda_stream)
    rng = np.random.default_rng(10)
    xs = [some(rng, 5, 60001, F32), some(rng, 5, 60001, F32)]
    X = [up(b, x, F32) for b, x in zip(bs, xs)]
    outs = [b.TokenLogProbs(x, topK=9) for b, x in zip(bs, X)]
    for b in bs:
        b.Sync()
    step("jh_token_logprobs on two contexts at once")
    for _ in range(20):
        for b, x, o in zip(bs, X, outs):
            b.TokenLogProbs(x, topK=9, out=o)
    for b, x, o in zip(bs, xs, outs):
        want = ref(x, 1.0, None, 9)
        close(b.Floats(o[1]), want[2], want[3], "entropy")
        assert np.array_equal(b.Ints(o[2]), want[4])
        b.Close()


def test_logprobs_far_rows(hip):
    """Rows that lie past 2^32 bytes and elements."""
    stride = (1 << 32) - 4
    try:
        X = hip.empty(BF16, stride + 3000)
    except JanisHipError:
        pytest.skip("no room")
    rng = np.random.default_rng(11)
    x = some(rng, 2, 3000, BF16)
    for i in range(2):
        hip._copy(up(hip, x[i], BF16), hip._view(X, (3000,), (1,), i * stride))
    check(hip, x, BF16, tokens=np.array([[5], [6]], np.int32), k=4, X=hip._view(X, (2, 3000), (stride, 1)))
    hip.Sync()
    X.free()


@pytest.mark.parametrize("T", [(1 << 23) + 1, (1 << 24) - 1, 1 << 24])
def test_logprobs_most_rows(hip, T):
    """As many rows as there may be, in which 1009 rows come again and again."""
    rng = np.random.default_rng(13)
    x, t = some(rng, 1009, 5, BF16), rng.integers(0, 5, 1009).astype(np.int32)
    want = ref(x, 1.0, t[:, None], 1)
    at = np.arange(T) % 1009
    X, tokens = up(hip, x[at], BF16), ints(hip, t[at])
    step(f"jh_token_logprobs rows={T}")
    lp, ent, ids, top = hip.TokenLogProbs(X, tokens, 1)
    for got, w, bar in ((hip.Floats(lp), want[0][:, 0], want[1][:, 0]), (hip.Floats(ent), want[2], want[3]), (hip.Floats(top)[:, 0], want[5][:, 0], want[6][:, 0])):
        assert (np.abs(got - w[at]) <= bar[at]).all()
    assert np.array_equal(hip.Ints(ids)[:, 0], want[4][at, 0])
    hip.Sync()


def test_refusals(hip):
    INVALID, UNSUPPORTED = _lib.JH_ERR_INVALID, _lib.JH_ERR_UNSUPPORTED
    t = hip.empty(F32, 1 << 16)
    p = t.ptr
    good = dict(x=p, dt=F32, T=2, V=100, stride=100, scale=1.0, tok=p, n=1, k=5, lp=p, ent=p, ids=p, top=p)
    refused(hip, "jh_token_logprobs", good, [
        (INVALID, dict(dt=1)), (INVALID, dict(dt=3)), (INVALID, dict(T=-1)), (INVALID, dict(V=0)), (INVALID, dict(n=-1)), (INVALID, dict(k=-1)),
        (UNSUPPORTED, dict(T=(1 << 24) + 1)), (UNSUPPORTED, dict(V=(1 << 28) + 1, stride=1 << 29)), (UNSUPPORTED, dict(k=33)), (UNSUPPORTED, dict(n=65)),
        (INVALID, dict(V=4)), (INVALID, dict(stride=99)), (INVALID, dict(stride=(1 << 32) + 1)), (INVALID, dict(scale=0.0)), (INVALID, dict(scale=-1.0)),
        (INVALID, dict(scale=float("nan"))), (INVALID, dict(scale=float("inf"))), (INVALID, dict(x=p + 8)), (INVALID, dict(x=None)), (INVALID, dict(tok=None)),
        (INVALID, dict(lp=None)), (INVALID, dict(ids=None)), (INVALID, dict(top=None))])
    assert hip._L.jh_token_logprobs(hip._ctx, None, F32, 0, 100, 100, 1.0, None, 0, 5, None, None, None, None) == 0
    with pytest.raises(JanisHipError, match="capturing"):
        hip.SetChecks(True)
        try:
            out = up(hip, np.zeros((2, 1)), F32)
            tok = ints(hip, [[1], [2]])
            X = up(hip, np.zeros((2, 50)), F32)
            Graph(hip, lambda: hip.TokenLogProbs(X, tok, out=(out, None, None, None)))
        finally:
            hip.SetChecks(False)


def test_logprobs_on_a_stream_without_all_cus():
    """A stream that leaves a CU out does not keep blocks on the XCDs as the join in the
    launch needs it: the parts are joined by a second one, to the same bits."""
    import ctypes

    from tests.conftest import hip_runtime

    b, rt = HipBackend(0), hip_runtime()
    rng = np.random.default_rng(12)
    cases = [(some(rng, 1, 151936, F32), F32, 20), (some(rng, 40, 50021, BF16), BF16, 5), (some(rng, 9, 151936, BF16), BF16, 0)]
    Xs = [up(b, x, dt) for x, dt, _ in cases]
    read = lambda out: [b.Floats(out[1])] + ([b.Ints(out[2]), b.Floats(out[3])] if out[2] is not None else [])  # noqa: E731
    wants = [read(b.TokenLogProbs(X, topK=k)) for X, (_, _, k) in zip(Xs, cases)]
    mask = (ctypes.c_uint32 * 8)(*([0xFFFFFFFF] * 7 + [0x7FFFFFFF]))
    stream = ctypes.c_void_p()
    assert rt.hipExtStreamCreateWithCUMask(ctypes.byref(stream), 8, mask) == 0
    b.SetStream(stream.value)
    for X, (x, dt, k), want in zip(Xs, cases, wants):
        step(f"jh_token_logprobs {x.shape} joined by a second launch")
        assert all(np.array_equal(g, w) for g, w in zip(read(b.TokenLogProbs(X, topK=k)), want))
    b.SetStream(None)
    b.Close()
    assert rt.hipStreamDestroy(stream) == 0
