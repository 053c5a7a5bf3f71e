"""The Python mirror of the drafted trees and of the log probabilities without a device:
what it refuses before the library is called, and what it passes on. The library is a
stub that keeps its arguments."""
import pytest

from janis_amd import engine
from janis_amd.engine import BF16, F16, F32, I32, U32, HipBackend, JanisHipError, PagedLayers

R, T, B, P, HQ, HK, PAGE, D, W, V = 3, 10, 5, 20, 4, 2, 16, 64, 2, 100


class Calls:
    def __init__(self):
        self.made = []

    def __getattr__(self, name):
        def call(*args):
            self.made.append((name, args))
            return 0
        return call


@pytest.fixture
def b(monkeypatch):
    monkeypatch.setattr(engine, "check", lambda ctx, rc: None)
    be = HipBackend.__new__(HipBackend)
    be._L, be._ctx, be._arena, be._sweeper, be._kv_reserve = Calls(), 1, None, None, 0
    yield be
    be._ctx = None


def tensor(b, shape, dt, at=1 << 20):
    return b.Wrap(at, shape, dt)


def plan_args(b):
    t = lambda *s: tensor(b, s, I32)  # noqa: E731
    return dict(parents=t(T), rowStarts=t(R + 1), kvLens=t(R), out=(t(T), tensor(b, (T, W), U32)))


def attention_args(b):
    pages = (P, HK, PAGE, D)
    return dict(q=tensor(b, (T, HQ, D), F16), k_pages=tensor(b, pages, F16), v_pages=tensor(b, pages, F16),
                blockTables=tensor(b, (R, B), I32), rowStarts=tensor(b, (R + 1,), I32), kvLens=tensor(b, (R,), I32),
                mask=tensor(b, (T, W), U32), scale=0.125, maxNew=4, out=tensor(b, (T, HQ, D), F32))


def layers(b, n=3, pages=P, page=PAGE):
    return PagedLayers(*([tensor(b, (pages, HK, page, D), BF16, at << 20) for at in range(first, first + n)] for first in (1, 9)))


def commit_args(b):
    t = lambda *s: tensor(b, s, I32)  # noqa: E731
    return dict(parents=t(T), tokens=t(T), chosen=t(T), rowStarts=t(R + 1), kvLens=t(R), maskWords=W, pageSize=PAGE, blockTables=t(R, B),
                freePages=t(P), freeCount=t(1), slots=t(T), layers=layers(b), known=t(R), out=(t(R), t(1), t(R), t(T), t(R), t(1)))


def logprobs_args(b):
    return dict(logits=tensor(b, (T, V), BF16), tokens=tensor(b, (T, 2), I32), topK=4,
                out=(tensor(b, (T, 2), F32), tensor(b, (T,), F32), tensor(b, (T, 4), I32), tensor(b, (T, 4), F32)))


CALLS = {"PagedTreePlan": plan_args, "PagedTreeAttention": attention_args, "PagedTreeCommit": commit_args, "TokenLogProbs": logprobs_args}


def out_with(i, shape, dt=I32):
    return lambda b, a: a["out"][:i] + (None if shape is None else tensor(b, shape, dt),) + a["out"][i + 1:]


REFUSED = [
    ("PagedTreePlan", {"parents": ((T,), F32)}), ("PagedTreePlan", {"parents": ((T + 1,), I32)}), ("PagedTreePlan", {"rowStarts": ((R,), I32)}),
    ("PagedTreePlan", {"kvLens": ((R + 1,), I32)}), ("PagedTreePlan", {"kvLens": ((R,), F32)}), ("PagedTreePlan", {"out": None}),
    ("PagedTreePlan", {"maskWords": W + 1}), ("PagedTreePlan", {"out": out_with(0, (T + 1,))}), ("PagedTreePlan", {"out": out_with(0, (T,), F32)}),
    ("PagedTreePlan", {"out": out_with(1, (T + 1, W), U32)}), ("PagedTreePlan", {"out": out_with(1, (T * W,), U32)}),
    ("PagedTreePlan", {"out": out_with(1, (T, W), F32)}),
    ("PagedTreePlan", {"out": lambda b, a: (a["out"][0], b.Slice(tensor(b, (T, W + 1), U32), 1, 0, W))}),
    ("PagedTreeAttention", {"mask": ((T + 1, W), U32)}), ("PagedTreeAttention", {"mask": ((T,), U32)}), ("PagedTreeAttention", {"mask": ((T, W), F32)}),
    ("PagedTreeAttention", {"mask": lambda b, a: b.Slice(tensor(b, (T, W + 1), U32), 1, 0, W)}),
    ("PagedTreeAttention", {"q": ((T, HQ, D), BF16)}), ("PagedTreeAttention", {"q": ((T, HQ * D), F16)}),
    ("PagedTreeAttention", {"blockTables": ((R + 1, B), I32)}), ("PagedTreeAttention", {"rowStarts": ((R,), I32)}),
    ("PagedTreeAttention", {"kvLens": ((R + 1,), I32)}), ("PagedTreeAttention", {"out": ((T, HQ, D + 1), F32)}),
    ("PagedTreeAttention", {"v_pages": ((P, HK, PAGE, D), BF16)}),
    ("PagedTreeCommit", {"parents": ((T + 1,), I32)}), ("PagedTreeCommit", {"tokens": ((T - 1,), I32)}), ("PagedTreeCommit", {"tokens": ((T,), F32)}),
    ("PagedTreeCommit", {"chosen": ((T + 1,), I32)}), ("PagedTreeCommit", {"chosen": ((T,), U32)}), ("PagedTreeCommit", {"chosen": ((T, 1, 1), I32)}),
    ("PagedTreeCommit", {"chosen": ((T, 0), I32)}), ("PagedTreeCommit", {"rowStarts": ((R,), I32)}), ("PagedTreeCommit", {"kvLens": ((R + 1,), I32)}),
    ("PagedTreeCommit", {"blockTables": ((R - 1, B), I32)}), ("PagedTreeCommit", {"blockTables": ((R * B,), I32)}),
    ("PagedTreeCommit", {"freeCount": ((2,), I32)}), ("PagedTreeCommit", {"slots": ((T + 1,), I32)}), ("PagedTreeCommit", {"known": ((R + 1,), I32)}),
    ("PagedTreeCommit", {"known": ((R,), F32)}), ("PagedTreeCommit", {"freePages": ((P + 1,), I32)}), ("PagedTreeCommit", {"pageSize": PAGE * 2}),
    ("PagedTreeCommit", {"layers": lambda b, a: layers(b, pages=P - 1)}), ("PagedTreeCommit", {"out": out_with(0, (R + 1,))}),
    ("PagedTreeCommit", {"out": out_with(1, (2,))}), ("PagedTreeCommit", {"out": out_with(2, (R - 1,))}), ("PagedTreeCommit", {"out": out_with(3, (T + 1,))}),
    ("PagedTreeCommit", {"out": out_with(4, (R,), F32)}), ("PagedTreeCommit", {"out": out_with(5, (2,))}),
    ("TokenLogProbs", {"tokens": ((T, 2), F32)}), ("TokenLogProbs", {"tokens": ((T + 1, 2), I32)}), ("TokenLogProbs", {"tokens": ((T, 3), I32)}),
    ("TokenLogProbs", {"tokens": None}), ("TokenLogProbs", {"topK": 5}), ("TokenLogProbs", {"topK": 0}), ("TokenLogProbs", {"out": out_with(0, None)}),
    ("TokenLogProbs", {"out": out_with(0, (T, 2), I32)}), ("TokenLogProbs", {"out": out_with(1, (T, 2), F32)}),
    ("TokenLogProbs", {"out": out_with(2, (T, 4), F32)}), ("TokenLogProbs", {"out": out_with(2, None)}), ("TokenLogProbs", {"out": out_with(3, None)}),
    ("TokenLogProbs", {"out": lambda b, a: (b.Slice(tensor(b, (T, 3), F32), 1, 0, 2),) + a["out"][1:]}),
]


@pytest.mark.parametrize("i", range(len(REFUSED)), ids=lambda i: f"{REFUSED[i][0]}-{'-'.join(REFUSED[i][1])}-{i}")
def test_refused_before_the_library(b, i):
    op, change = REFUSED[i]
    a = CALLS[op](b)
    for k, v in change.items():
        a[k] = v(b, a) if callable(v) else tensor(b, *v) if isinstance(v, tuple) else v
    with pytest.raises(JanisHipError) as e:
        getattr(b, op)(**a)
    assert e.value.code == engine._lib.JH_ERR_INVALID and op in str(e.value)
    assert not b._L.made


def test_layers_refused(b):
    k = [tensor(b, (P, HK, PAGE, D), BF16)] * 2
    for ks, vs in (([], []), (k, k[:1]), (k, [k[0], tensor(b, (P, HK, PAGE, D), F16)]), ([k[0], tensor(b, (P, HK, 2 * PAGE, D), BF16)],) * 2,
                   ([k[0], b.Slice(tensor(b, (P, 2 * HK, PAGE, D), BF16), 1, 0, HK)],) * 2, ([tensor(b, (P, HK, PAGE * D), BF16)],) * 2):
        with pytest.raises(JanisHipError) as e:
            PagedLayers(ks, vs)
        assert e.value.code == engine._lib.JH_ERR_INVALID


def test_plan_passed_on(b):
    a = plan_args(b)
    assert b.PagedTreePlan(**a) is a["out"]
    (name, c), = b._L.made
    assert name == "jh_paged_tree_plan" and c[4:7] == (R, T, W) and c[7:] == (a["out"][0].ptr, a["out"][1].ptr)
    b._L.made.clear()
    a["out"] = (a["out"][0], tensor(b, (T, W), I32))  # the words as I32
    assert b.PagedTreePlan(**a, maskWords=W) is a["out"]


def test_attention_passed_on(b):
    """Pages that alternate in one buffer, and queries that lie apart."""
    both = tensor(b, (P, 2 * HK, PAGE, D), F16)
    a = attention_args(b)
    a["k_pages"], a["v_pages"] = b.Slice(both, 1, 0, HK), b.Slice(both, 1, HK, 2 * HK)
    a["q"] = b.Slice(tensor(b, (T, HQ + 3, D), F16), 1, 0, HQ)
    a["mask"] = tensor(b, (T, W), U32, 7 << 20)
    assert b.PagedTreeAttention(**a) is a["out"]
    (name, c), = b._L.made
    assert name == "jh_paged_tree_attention"
    assert c[2] == (HQ + 3) * D and c[4] - c[3] == HK * PAGE * D * 2 and c[5:9] == (F16, P, PAGE, 2 * HK * PAGE * D)
    assert c[10] == B and c[13:15] == (7 << 20, W) and c[15:22] == (R, T, 4, HQ, HK, D, 0.125) and c[23] == F32


def test_commit_passed_on(b):
    """Choices as a column of wider rows, lengths and the count in place, no layers."""
    a = commit_args(b)
    a["chosen"] = tensor(b, (T, 5), I32)
    a["out"] = (a["kvLens"], a["freeCount"]) + a["out"][2:]
    assert b.PagedTreeCommit(**a) is a["out"]
    (name, c), = b._L.made
    assert name == "jh_paged_tree_commit"
    assert c[4] == 5 and c[5] == a["known"].ptr and c[8:12] == (R, T, W, PAGE) and c[13] == B and c[15] == P
    assert c[18] == a["kvLens"].ptr and c[19] == a["freeCount"].ptr
    assert list(c[24]) == [1 << 20, 2 << 20, 3 << 20] and list(c[25]) == [9 << 20, 10 << 20, 11 << 20]
    assert c[26:] == (3, BF16, HK, D, HK * PAGE * D)
    b._L.made.clear()
    a = commit_args(b)
    a["layers"] = a["known"] = None
    a["chosen"] = b.Slice(tensor(b, (T, 5), I32), 1, 2, 3)
    assert b.PagedTreeCommit(**a) is a["out"]
    c = b._L.made[0][1]
    assert c[3] == (1 << 20) + 8 and c[4] == 5 and c[5] is None and c[24:27] == (None, None, 0)


def test_logprobs_passed_on(b):
    a = logprobs_args(b)
    a["logits"] = b.Slice(tensor(b, (T, V + 28), BF16), 1, 0, V)
    assert b.TokenLogProbs(**a) is a["out"]
    (name, c), = b._L.made
    assert name == "jh_token_logprobs" and c[2:7] == (BF16, T, V, V + 28, 1.0) and c[8:10] == (2, 4)
    b._L.made.clear()
    # a token to a row, rows of two axes, no entropy, no alternatives
    lp = tensor(b, (2, 5), F32)
    b.TokenLogProbs(tensor(b, (2, 5, V), F32), tensor(b, (2, 5), I32), scale=0.5, out=(lp, None, None, None))
    c = b._L.made.pop()[1]
    assert c[2:7] == (F32, 10, V, V, 0.5) and c[8:10] == (1, 0) and c[10:] == (lp.ptr, None, None, None)
    # one row
    ent = tensor(b, (1,), F32)
    b.TokenLogProbs(tensor(b, (V,), F32), out=(None, ent, None, None))
    c = b._L.made.pop()[1]
    assert c[3:6] == (1, V, V) and c[7] is None and c[10:] == (None, ent.ptr, None, None)
