"""The paged cache's Python mirror without a device: what it refuses before the library
is called, and what it passes on. The library is a stub that keeps its arguments."""
import pytest

from janis_amd import engine
from janis_amd.engine import BF16, F16, F32, I32, HipBackend, JanisHipError

R, T, B, P, HQ, HK, PAGE, D = 3, 10, 5, 20, 4, 2, 16, 64


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
    return dict(newLens=t(R), kvLens=t(R), pageSize=PAGE, blockTables=t(R, B), freePages=t(P), freeCount=t(1),
                out=(t(R), t(1), t(R + 1), t(T), t(T), t(1)))


def append_args(b):
    pages = (P, HK, PAGE, D)
    return dict(qkv=tensor(b, (T, (HQ + 2 * HK) * D), F32), n_heads=HQ, n_kv_heads=HK, q_norm=tensor(b, (D,), BF16),
                k_norm=tensor(b, (D,), BF16), eps=1e-6, base=1e6, rope_scale=1.0, positions=tensor(b, (T,), I32),
                slots=tensor(b, (T,), I32), k_pages=tensor(b, pages, BF16), v_pages=tensor(b, pages, BF16),
                freqs=tensor(b, (D // 2,), F32), q_out=tensor(b, (T, HQ, D), BF16))


def attention_args(b):
    pages = (P, HK, PAGE, D)
    return dict(q=tensor(b, (T, HQ, D), F16), k_pages=tensor(b, pages, F16), v_pages=tensor(b, pages, F16),
                blockTables=tensor(b, (R, B), I32), rowStarts=tensor(b, (R + 1,), I32), kvLens=tensor(b, (R,), I32),
                scale=0.125, maxNew=4, out=tensor(b, (T, HQ, D), F32))


CALLS = {"PagedPlan": plan_args, "PagedQKNormRoPEAppend": append_args, "PagedAttention": attention_args}


def out_with(i, shape, dt=I32):
    return lambda b, a: a["out"][:i] + (tensor(b, shape, dt),) + a["out"][i + 1:]


REFUSED = [
    ("PagedPlan", {"newLens": ((R,), F32)}), ("PagedPlan", {"newLens": ((R + 1,), I32)}), ("PagedPlan", {"kvLens": ((R - 1,), I32)}),
    ("PagedPlan", {"blockTables": ((R - 1, B), I32)}), ("PagedPlan", {"blockTables": ((R * B,), I32)}),
    ("PagedPlan", {"blockTables": ((R, B), F32)}), ("PagedPlan", {"freeCount": ((2,), I32)}), ("PagedPlan", {"freePages": ((P,), F32)}),
    ("PagedPlan", {"out": None}),
    ("PagedPlan", {"out": out_with(0, (R + 1,))}), ("PagedPlan", {"out": out_with(1, (2,))}), ("PagedPlan", {"out": out_with(2, (R,))}),
    ("PagedPlan", {"out": out_with(4, (T + 1,))}), ("PagedPlan", {"out": out_with(5, (2,))}), ("PagedPlan", {"out": out_with(5, (1,), F32)}),
    ("PagedQKNormRoPEAppend", {"qkv": ((T, (HQ + 2 * HK) * D + 1), F32)}), ("PagedQKNormRoPEAppend", {"qkv": ((T + 1, (HQ + 2 * HK) * D), F32)}),
    ("PagedQKNormRoPEAppend", {"n_kv_heads": HK + 1}), ("PagedQKNormRoPEAppend", {"slots": ((T,), F32)}),
    ("PagedQKNormRoPEAppend", {"positions": ((T - 1,), I32)}), ("PagedQKNormRoPEAppend", {"positions": ((T,), F32)}),
    ("PagedQKNormRoPEAppend", {"q_norm": ((D + 1,), BF16)}), ("PagedQKNormRoPEAppend", {"k_norm": ((D,), F32)}),
    ("PagedQKNormRoPEAppend", {"freqs": ((D,), F32)}), ("PagedQKNormRoPEAppend", {"freqs": ((D // 2,), BF16)}),
    ("PagedQKNormRoPEAppend", {"q_out": ((T, HQ, D), F32)}), ("PagedQKNormRoPEAppend", {"q_out": ((T, HQ + 1, D), BF16)}),
    ("PagedQKNormRoPEAppend", {"v_pages": ((P, HK, PAGE, D), F16)}), ("PagedQKNormRoPEAppend", {"v_pages": ((P + 1, HK, PAGE, D), BF16)}),
    ("PagedQKNormRoPEAppend", {"k_pages": ((P, HK, PAGE * D), BF16), "v_pages": ((P, HK, PAGE * D), BF16)}),
    ("PagedAttention", {"q": ((T, HQ, D), BF16)}), ("PagedAttention", {"q": ((T, HQ * D), F16)}), ("PagedAttention", {"q": ((T, HQ, D * 2), F16)}),
    ("PagedAttention", {"blockTables": ((R + 1, B), I32)}), ("PagedAttention", {"blockTables": ((R, B), F32)}),
    ("PagedAttention", {"rowStarts": ((R,), I32)}), ("PagedAttention", {"kvLens": ((R + 1,), I32)}), ("PagedAttention", {"kvLens": ((R,), F32)}),
    ("PagedAttention", {"out": ((T, HQ, D + 1), F32)}), ("PagedAttention", {"v_pages": ((P, HK, PAGE, D), BF16)}),
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


def test_insides_of_pages_must_be_dense(b):
    whole = tensor(b, (P, HK, 2 * PAGE, D), F16)
    for pages in (b.Slice(whole, 2, 0, PAGE), b.Transpose(tensor(b, (P, PAGE, HK, D), F16), 0, 2, 1, 3)):
        a = attention_args(b)
        a["k_pages"] = a["v_pages"] = pages
        with pytest.raises(JanisHipError, match="dense"):
            b.PagedAttention(**a)
    assert not b._L.made


def test_what_is_passed_on(b):
    """Pages that alternate in one buffer, queries and products that lie apart."""
    both = tensor(b, (P, 2 * HK, PAGE, D), F16)
    a = attention_args(b)
    a["k_pages"], a["v_pages"] = b.Slice(both, 1, 0, HK), b.Slice(both, 1, HK, 2 * HK)
    a["q"] = b.Slice(tensor(b, (T, HQ + 3, D), F16), 1, 0, HQ)
    assert b.PagedAttention(**a) is a["out"]
    (name, c), = b._L.made
    assert name == "jh_paged_attention"
    assert c[2] == (HQ + 3) * D and c[4] - c[3] == HK * PAGE * D * 2 and c[5:9] == (F16, P, PAGE, 2 * HK * PAGE * D)
    assert c[10] == B and c[13:20] == (R, T, 4, HQ, HK, D, 0.125) and c[21] == F32
    b._L.made.clear()
    a = append_args(b)
    a["qkv"] = b.Slice(tensor(b, (T, (HQ + 2 * HK) * D + 24), F32), 1, 0, (HQ + 2 * HK) * D)
    assert b.PagedQKNormRoPEAppend(**a) is a["q_out"]
    (name, c), = b._L.made
    assert name == "jh_paged_qk_norm_rope_append"
    assert c[2:8] == (F32, T, (HQ + 2 * HK) * D + 24, HQ, HK, D) and c[10] == BF16 and c[19:23] == (BF16, P, PAGE, HK * PAGE * D)
    b._L.made.clear()
    a = append_args(b)
    a["n_heads"], a["q_out"], a["qkv"] = 0, None, tensor(b, (T, 2 * HK * D), F32)
    assert b.PagedQKNormRoPEAppend(**a) is None and b._L.made[0][1][-1] is None
    b._L.made.clear()
    a = plan_args(b)
    assert b.PagedPlan(**a) is a["out"]
    (name, c), = b._L.made
    assert name == "jh_paged_plan" and c[3:6] == (R, T, PAGE) and c[7] == B and c[9] == P


def test_pages_that_are_dense_whatever_their_strides_say(b):
    """Strides of axes of length 1 do not matter: pages that hold [page, heads, dim] with one
    head, pages of one key, a pool of one page."""
    one_head = b.Transpose(tensor(b, (P, PAGE, 1, D), F16), 0, 2, 1, 3)
    one_page = b._view(tensor(b, (HK, PAGE, D), F16), (1, HK, PAGE, D), (0, PAGE * D, D, 1))
    for pages, hq, stride in ((one_head, HQ, PAGE * D), (one_page, HQ, HK * PAGE * D)):
        a = attention_args(b)
        a["k_pages"] = a["v_pages"] = pages
        assert b.PagedAttention(**a) is a["out"]
        assert b._L.made.pop()[1][5:9] == (F16, pages.shape[0], PAGE, stride)
    one_key = b.Transpose(tensor(b, (P, 1, HK, D), BF16), 0, 2, 1, 3)
    a = append_args(b)
    a["k_pages"], a["v_pages"] = one_key, tensor(b, (P, HK, 1, D), BF16)
    assert b.PagedQKNormRoPEAppend(**a) is a["q_out"]
    assert b._L.made.pop()[1][19:23] == (BF16, P, 1, HK * D)
    # keys and values whose pages lie apart differently are still refused
    a["v_pages"] = b.Slice(tensor(b, (P, 2 * HK, 1, D), BF16), 1, 0, HK)
    with pytest.raises(JanisHipError, match="alike"):
        b.PagedQKNormRoPEAppend(**a)
    assert not b._L.made
