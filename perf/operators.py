"""What the paged key/value cache is measured on: the calls that a program makes
which serves a batch of requests of different lengths with a quantized
Qwen3-style model.

A case is a dict of plain values with a "kind":

  plan       one step's bookkeeping: pages for the new tokens of every request
             from the stack of free ones, finished requests' pages back to it,
             and each new token's position and slot
  append     the rows of a q/k/v product: q/k norms, rotation, keys and values to
             their slots, queries out
  attention  causal attention of every request's new tokens over its pages

The lengths of the requests follow from the case alone (`_lens`), all values from
the seed. Each pass is given its plain form in torch operations of 32 bits (64
for angles), and the framework's call where `own` is true.
"""
import math
import random

import torch

own = False

EPS = 1e-6
THETA = 1e6
TORCH = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ---- the cases -------------------------------------------------------------------

def listed():
    return [
        # bookkeeping of a decode step of 64 conversations
        {"name": "plan_64", "kind": "plan", "req": 64, "rows": 64, "page": 16, "kv_lo": 100, "kv_hi": 8000, "many": 0, "mix": 1},
        # of a large server's step: many conversations, some finished, pieces of prompts among them
        {"name": "plan_700", "kind": "plan", "req": 700, "rows": 8192, "page": 16, "kv_lo": 20, "kv_hi": 8000, "many": 24, "mix": 2},
        # one conversation's next token
        {"name": "append_1", "kind": "append", "rows": 1, "pad": 0, "heads": 32, "kv": 8, "dim": 128, "page": 16, "act": "bf16", "cache": "bf16"},
        # the next tokens of a captured step's 57 conversations, in a batch padded to 64
        {"name": "append_57", "kind": "append", "rows": 57, "pad": 7, "heads": 32, "kv": 4, "dim": 128, "page": 32, "act": "f32", "cache": "f16"},
        # a prompt's piece
        {"name": "append_4001", "kind": "append", "rows": 4001, "pad": 0, "heads": 32, "kv": 8, "dim": 128, "page": 16, "act": "bf16", "cache": "bf16"},
        # one conversation at a chat's length: the least call of a decode loop
        {"name": "attention_1x700", "kind": "attention", "req": 1, "new_lo": 1, "new_hi": 1, "many": 0, "kv_lo": 700, "kv_hi": 700, "pad": 0,
         "heads": 32, "kv": 8, "dim": 128, "page": 16, "cache": "bf16", "mix": 1},
        # 64 conversations of all lengths
        {"name": "attention_64", "kind": "attention", "req": 64, "new_lo": 1, "new_hi": 1, "many": 0, "kv_lo": 100, "kv_hi": 8000, "pad": 0,
         "heads": 32, "kv": 8, "dim": 128, "page": 16, "cache": "bf16", "mix": 3},
        # one token over a book
        {"name": "attention_1x100k", "kind": "attention", "req": 1, "new_lo": 1, "new_hi": 1, "many": 0, "kv_lo": 100001, "kv_hi": 100001, "pad": 0,
         "heads": 32, "kv": 4, "dim": 128, "page": 64, "cache": "f16", "mix": 1},
        # drafted tokens of 16 conversations verified at once, a padded batch
        {"name": "attention_verify", "kind": "attention", "req": 16, "new_lo": 2, "new_hi": 7, "many": 0, "kv_lo": 500, "kv_hi": 5000, "pad": 9,
         "heads": 32, "kv": 4, "dim": 128, "page": 32, "cache": "bf16", "mix": 4},
        # a short prompt from an empty cache
        {"name": "attention_513", "kind": "attention", "req": 1, "new_lo": 513, "new_hi": 513, "many": 0, "kv_lo": 513, "kv_hi": 513, "pad": 0,
         "heads": 32, "kv": 8, "dim": 128, "page": 16, "cache": "f16", "mix": 1},
        # the next piece of a long prompt
        {"name": "attention_2000", "kind": "attention", "req": 1, "new_lo": 2000, "new_hi": 2000, "many": 0, "kv_lo": 8000, "kv_hi": 8000, "pad": 0,
         "heads": 32, "kv": 8, "dim": 128, "page": 16, "cache": "bf16", "mix": 1},
        # two pieces of prompts beside 22 conversations, heads of 64
        {"name": "attention_mixed", "kind": "attention", "req": 24, "new_lo": 1, "new_hi": 1, "many": 2, "kv_lo": 300, "kv_hi": 4000, "pad": 0,
         "heads": 16, "kv": 4, "dim": 64, "page": 16, "cache": "bf16", "mix": 5},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("plan", "append", "append", "attention", "attention", "attention", "attention"))
    heads, kv, dim = rng.choice(((32, 8, 128), (32, 4, 128), (16, 8, 128), (32, 8, 64), (16, 4, 64)))
    page, cache, mix = rng.choice((16, 16, 32, 64, 128)), rng.choice(("bf16", "f16")), rng.randint(10, 10**6)
    if kind == "plan":
        req = _log_int(rng, 1, 700)
        many = 0 if rng.random() < 0.5 else min(req, rng.randint(1, 16))
        return {"kind": kind, "req": req, "rows": req + 500 * many, "page": page, "kv_lo": rng.randint(1, 300), "kv_hi": _log_int(rng, 400, 8000),
                "many": many, "mix": mix}
    if kind == "append":
        return {"kind": kind, "rows": _log_int(rng, 1, 4000), "pad": rng.choice((0, 0, 1, 30)), "heads": heads, "kv": kv, "dim": dim, "page": page,
                "act": rng.choice(("bf16", "f32")), "cache": cache}
    shape = rng.choice(("one", "batch", "batch", "verify", "prompt", "prompt", "mixed"))
    c = {"kind": kind, "req": 1, "new_lo": 1, "new_hi": 1, "many": 0, "kv_lo": 1, "kv_hi": 1, "pad": rng.choice((0, 0, 5)), "heads": heads, "kv": kv,
         "dim": dim, "page": page, "cache": cache, "mix": mix}
    if shape == "one":
        c["kv_lo"] = c["kv_hi"] = _log_int(rng, 1, 100000)
    elif shape == "batch":
        c.update(req=_log_int(rng, 2, 64), kv_lo=rng.randint(1, 300), kv_hi=_log_int(rng, 400, 8000))
    elif shape == "verify":
        c.update(req=_log_int(rng, 1, 24), new_lo=2, new_hi=rng.randint(3, 8), kv_lo=rng.randint(10, 500), kv_hi=_log_int(rng, 600, 5000))
    elif shape == "prompt":
        new = _log_int(rng, 9, 1900)
        past = 0 if rng.random() < 0.4 else _log_int(rng, 10, 6000)
        c.update(req=rng.choice((1, 1, 2)) if new < 700 else 1, new_lo=new, new_hi=new, kv_lo=new + past, kv_hi=new + past)
    else:
        c.update(req=rng.randint(3, 24), many=rng.randint(1, 3), kv_lo=rng.randint(50, 400), kv_hi=_log_int(rng, 700, 4000))
    return c


def _lens(c):
    """Every request's (new tokens, keys): for a plan the keys before the step,
    for attention those after it, the new ones among them."""
    rng = random.Random(c["mix"])
    out = []
    for r in range(c["req"]):
        kv = _log_int(rng, c["kv_lo"], c["kv_hi"])
        if c["kind"] == "plan":
            new = -1 if c["many"] and rng.random() < 0.05 else 1  # finished, or one token more
            if r < c["many"]:
                new = rng.randint(1, c["rows"] // c["many"] - c["req"] // c["many"] - 1) if c["rows"] > c["req"] + c["many"] else 1
        else:
            new = rng.randint(c["new_lo"], c["new_hi"])
            if r < c["many"]:
                new, kv = rng.randint(200, 700), kv + 700
        out.append((new, kv if c["kind"] == "plan" else max(kv, new)))
    return out


def work(c):
    if c["kind"] == "plan":
        lens, p = _lens(c), c["page"]
        pages = sum(-(-max(0, kv + n) // p) - -(-kv // p) if n >= 0 else -(-kv // p) for n, kv in lens)
        rows = sum(max(0, n) for n, _ in lens)
        return {"bytes": 16 * len(lens) + 12 * c["rows"] + 8 * pages, "flops": rows}
    if c["kind"] == "append":
        n = c["rows"] * (c["heads"] + 2 * c["kv"]) * c["dim"]
        return {"bytes": n * ((4 if c["act"] == "f32" else 2) + 2) + 8 * c["rows"], "flops": 8 * n}
    lens = _lens(c)
    rows, keys = sum(n for n, _ in lens), sum(kv for _, kv in lens)
    seen = sum(n * (kv - n) + n * (n + 1) // 2 for n, kv in lens)
    return {"bytes": 4 * keys * c["kv"] * c["dim"] + 4 * rows * c["heads"] * c["dim"], "flops": 4 * seen * c["heads"] * c["dim"]}


# ---- inputs ----------------------------------------------------------------------

def _blocks(kv, page):
    return -(-kv // page)


def _tables(lens, page, n_pages, gen):
    """Block tables of requests of these lengths over shuffled pages (-1 past a
    request's own), and the pages that are left, as a stack."""
    order = torch.randperm(n_pages, device="cuda", generator=gen).to(torch.int32)
    blocks = torch.tensor([_blocks(kv, page) for kv in lens], device="cuda")
    first = torch.cumsum(blocks, 0) - blocks
    j = torch.arange(max(1, max(_blocks(kv, page) for kv in lens)), device="cuda")
    at = (first[:, None] + j).clamp_(max=n_pages - 1)
    table = torch.where(j < blocks[:, None], order[at], torch.full_like(at, -1, dtype=torch.int32))
    used = sum(_blocks(kv, page) for kv in lens)
    return table, order[used:], used


def _inputs(c, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(shape, dtype, scale=1.0, mean=0.0):
        return torch.randn(shape, device="cuda", generator=gen).mul_(scale).add_(mean).to(dtype)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    if c["kind"] == "plan":
        lens, page = _lens(c), c["page"]
        new, kv = [n for n, _ in lens], [k for _, k in lens]
        used = sum(_blocks(k, page) for k in kv)
        n_pages = used + sum(_blocks(max(0, n), page) + 1 for n in new) + 50
        table, left, _ = _tables(kv, page, n_pages, gen)
        blocks = max(_blocks(k + max(0, n), page) for n, k in lens)
        tables = torch.full((len(kv), blocks + 3), -1, dtype=torch.int32, device="cuda")
        tables[:, :table.shape[1]] = table
        free = torch.full((n_pages,), -1, dtype=torch.int32, device="cuda")
        free[:left.numel()] = left
        return {"new": ints(new), "kv": ints(kv), "tables": tables, "free": free, "count": ints([left.numel()])}
    D, page, cache = c["dim"], c["page"], TORCH[c["cache"]]
    if c["kind"] == "append":
        T = c["rows"] + c["pad"]
        n_pages = _blocks(c["rows"], page) + 5
        slots = torch.randperm(n_pages * page, device="cuda", generator=gen)[:T].to(torch.int32)
        pos = torch.randint(0, 100000, (T,), dtype=torch.int32, device="cuda", generator=gen)
        slots[c["rows"]:] = -1
        pos[c["rows"]:] = -1
        d = {"qkv": normal((T, (c["heads"] + 2 * c["kv"]) * D), TORCH[c["act"]], 2.0), "pos": pos, "slots": slots,
             "q_norm": normal((D,), torch.bfloat16, 0.1, 1.5), "k_norm": normal((D,), torch.bfloat16, 0.1, 1.5),
             "q_out": torch.zeros((T, c["heads"], D), dtype=cache, device="cuda")}
        for name in ("k_pages", "v_pages"):
            d[name] = normal((n_pages, c["kv"], page, D), cache)
        return d
    lens = _lens(c)
    kv = [k for _, k in lens]
    n_pages = sum(_blocks(k, page) for k in kv) + 7
    tables, _, _ = _tables(kv, page, n_pages, gen)
    starts = [0]
    for n, _ in lens:
        starts.append(starts[-1] + n)
    T = starts[-1] + c["pad"]
    return {"q": normal((T, c["heads"], D), cache, 1.5), "k_pages": normal((n_pages, c["kv"], page, D), cache, 1.5),
            "v_pages": normal((n_pages, c["kv"], page, D), cache), "tables": tables, "starts": ints(starts), "kv": ints(kv),
            "out": torch.zeros((T, c["heads"], D), dtype=cache if cache == torch.bfloat16 else torch.float16, device="cuda")}


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if case["kind"] == "plan":  # the buffers that a server keeps for its steps
        def i32(n):
            return torch.zeros((n,), dtype=torch.int32, device="cuda")
        s.update(kv_out=i32(case["req"]), count_out=i32(1), starts=i32(case["req"] + 1), pos=i32(case["rows"]), slots=i32(case["rows"]), status=i32(1))
    elif case["kind"] == "attention":
        lens = _lens(case)
        s.update(rows=sum(n for n, _ in lens), max_new=max(n for n, _ in lens), max_kv=max(kv for _, kv in lens))
    return s


# ---- the framework's calls ---------------------------------------------------------

_engine = []


def _backend():
    """The program's one backend and its stream, which torch's work goes to from then
    on: inputs are ready when the backend reads them, and what reads its results waits."""
    if not _engine:
        from janis_amd.engine import HipBackend
        b, stream = HipBackend(0), torch.cuda.Stream()
        b.SetStream(stream.cuda_stream)
        stream.wait_stream(torch.cuda.current_stream())
        torch.cuda.set_stream(stream)
        _engine.extend((b, stream, stream.cuda_stream))
    return _engine


def _ordered(call, c, s):
    """One of the calls below, in the order of the caller's stream where that is another one."""
    b, stream, handle = _backend()
    if torch._C._cuda_getCurrentRawStream(0) == handle:
        return call(b, c, s)
    caller = torch.cuda.current_stream()
    stream.wait_stream(caller)
    out = call(b, c, s)
    caller.wait_stream(stream)
    return out


def _handles(b, s):
    """The engine's handles on the state's buffers, made once as a program keeps them."""
    if "handles" not in s:
        from janis_amd.engine import BF16, F16, F32, I32
        code = {torch.bfloat16: BF16, torch.float16: F16, torch.float32: F32, torch.int32: I32}
        s["handles"] = {k: b.Wrap(t.data_ptr(), tuple(t.shape), code[t.dtype], keep=t) for k, t in s.items() if isinstance(t, torch.Tensor)}
    return s["handles"]


def _own_plan(b, c, s):
    h = _handles(b, s)
    b.PagedPlan(h["new"], h["kv"], c["page"], h["tables"], h["free"], h["count"],
                out=(h["kv_out"], h["count_out"], h["starts"], h["pos"], h["slots"], h["status"]))
    return _plan_out(s["kv_out"], s["count_out"], s["starts"], s["pos"], s["slots"], s["status"], s["tables"], s["free"])


def _own_append(b, c, s):
    h = _handles(b, s)
    b.PagedQKNormRoPEAppend(h["qkv"], c["heads"], c["kv"], h["q_norm"], h["k_norm"], EPS, THETA, 1.0, h["pos"], h["slots"], h["k_pages"],
                            h["v_pages"], q_out=h["q_out"])
    return {"q": s["q_out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _own_attention(b, c, s):
    h = _handles(b, s)
    b.PagedAttention(h["q"], h["k_pages"], h["v_pages"], h["tables"], h["starts"], h["kv"], c["dim"] ** -0.5, maxNew=s["max_new"], out=h["out"])
    return {"out": s["out"]}


# ---- the plain forms -----------------------------------------------------------------

def _plan_out(kv, count, starts, pos, slots, status, tables, free):
    return {"kv": kv, "count": count, "starts": starts, "positions": pos, "slots": slots, "status": status, "tables": tables, "free": free}


def _plain_plan(c, s):
    page, R, T = c["page"], c["req"], c["rows"]
    new, kv, tables, free, count = s["new"].long(), s["kv"].long(), s["tables"], s["free"], s["count"].long()
    N, B = free.numel(), tables.shape[1]
    done = new < 0
    n = new.clamp(min=0)
    after = torch.where(done, torch.zeros_like(kv), kv + n)
    old, want = (kv + page - 1) // page, (after + page - 1) // page
    back = torch.where(done, old, torch.zeros_like(old))
    take = torch.where(done, torch.zeros_like(old), want - old)
    j = torch.arange(B, device="cuda")
    # finished requests' pages onto the stack (the last place takes what is not one)
    to = torch.where(j < back[:, None], count + (torch.cumsum(back, 0) - back)[:, None] + j, torch.full_like(j, N).expand(R, B))
    stack = torch.cat((free, free[:1])).scatter(0, to.reshape(-1), tables.reshape(-1))[:N]
    top = count + back.sum()
    # new pages off its top
    at = (top - 1 - (torch.cumsum(take, 0) - take)[:, None] - (j - old[:, None])).clamp(0, N - 1)
    fresh = (j >= old[:, None]) & (j < want[:, None]) & ~done[:, None]
    table = torch.where(fresh, stack[at], tables)
    starts = torch.cat((torch.zeros_like(count), torch.cumsum(n, 0)))
    i = torch.arange(T, device="cuda")
    r = torch.searchsorted(starts[1:], i, right=True).clamp(max=R - 1)
    pos = kv[r] + i - starts[r]
    slot = table[r, (pos // page).clamp(0, B - 1)].long() * page + pos % page
    live = i < starts[R]
    none = torch.full_like(pos, -1)
    as32 = [x.to(torch.int32) for x in (after, top - take.sum(), starts, torch.where(live, pos, none), torch.where(live, slot, none))]
    return _plan_out(*as32, torch.zeros_like(s["status"]), table, stack)


def _plain_append(c, s):
    T, Hq, Hk, D, page = c["rows"], c["heads"], c["kv"], c["dim"], c["page"]
    x = s["qkv"][:T].float().view(T, Hq + 2 * Hk, D)

    def normed(x, w):
        return x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()

    angle = s["pos"][:T, None].double() * THETA ** (torch.arange(D // 2, device="cuda", dtype=torch.float64) * (-2.0 / D))
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]

    def turned(x):
        a, b = x[..., :D // 2], x[..., D // 2:]
        return torch.cat((a * cos - b * sin, a * sin + b * cos), -1)

    s["q_out"][:T] = turned(normed(x[:, :Hq], s["q_norm"])).to(s["q_out"].dtype)
    block, at = (s["slots"][:T] // page).long(), (s["slots"][:T] % page).long()
    s["k_pages"][block, :, at] = turned(normed(x[:, Hq:Hq + Hk], s["k_norm"])).to(s["k_pages"].dtype)
    s["v_pages"][block, :, at] = x[:, Hq + Hk:].to(s["v_pages"].dtype)
    return {"q": s["q_out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _plain_attention(c, s):
    R, Hq, Hk, D, page, n, L, T = c["req"], c["heads"], c["kv"], c["dim"], c["page"], s["max_new"], s["max_kv"], s["rows"]
    G = Hq // Hk
    pages = s["tables"][:, :_blocks(L, page)].clamp(min=0).long()

    def keys(pool):  # [R, Hk, keys, D]
        return pool[pages].float().transpose(1, 2).reshape(R, Hk, -1, D)

    starts, kv = s["starts"].long(), s["kv"].long()
    count = starts[1:] - starts[:-1]
    i = torch.arange(n, device="cuda")
    q = s["q"][(starts[:-1, None] + i).clamp(max=T - 1)].float()  # [R, n, Hq, D]
    q = q.view(R, n, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(R, Hk, G * n, D)
    sc = torch.matmul(q, keys(s["k_pages"]).transpose(2, 3).contiguous()).mul_(D ** -0.5)
    seen = torch.arange(sc.shape[-1], device="cuda") < ((kv - count)[:, None] + i + 1)[:, :, None]  # [R, n, keys]
    sc = sc.view(R, Hk, G, n, -1).masked_fill_(~seen[:, None, None], -math.inf)
    sc = sc.sub_(sc.amax(-1, keepdim=True)).exp_()
    total = sc.sum(-1, keepdim=True)
    o = torch.matmul(sc.view(R, Hk, G * n, -1), keys(s["v_pages"])).view(R, Hk, G, n, D) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(R * n, Hq, D)
    row = torch.arange(T, device="cuda")
    r = torch.searchsorted(starts[1:], row, right=True)
    s["out"][:T] = o[r * n + row - starts[r]].to(s["out"].dtype)
    return {"out": s["out"]}


def run(s):
    c = s["case"]
    if own:
        return _ordered({"plan": _own_plan, "append": _own_append, "attention": _own_attention}[c["kind"]], c, s)
    return {"plan": _plain_plan, "append": _plain_append, "attention": _plain_attention}[c["kind"]](c, s)


# ---- the definitions, in 64 bits ------------------------------------------------------

def exact(case, seed):
    c, d = case, _inputs(case, seed)
    if c["kind"] == "plan":
        return _exact_plan(c, d)
    if c["kind"] == "append":
        Hq, Hk, D, page = c["heads"], c["kv"], c["dim"], c["page"]
        q, k, v = d["q_out"].double(), d["k_pages"].double(), d["v_pages"].double()
        T = c["rows"]
        x = d["qkv"][:T].double().view(T, -1, D)
        inv = torch.tensor([THETA ** (-2.0 * i / D) for i in range(D // 2)], dtype=torch.float64, device="cuda")
        turn = torch.polar(torch.ones(T, D // 2, dtype=torch.float64, device="cuda"), d["pos"][:T, None].double() * inv)[:, None]

        def head(x, w):
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.double()
            z = torch.complex(x[..., :D // 2].contiguous(), x[..., D // 2:].contiguous()) * turn
            return torch.cat((z.real, z.imag), -1)

        q[:T] = head(x[:, :Hq], d["q_norm"])
        slots = d["slots"][:T].long()
        k.transpose(1, 2)[slots // page, slots % page] = head(x[:, Hq:Hq + Hk], d["k_norm"])
        v.transpose(1, 2)[slots // page, slots % page] = x[:, Hq + Hk:]
        return {"q": q, "k_pages": k, "v_pages": v}
    out = d["out"].double()
    Hk, G, D = c["kv"], c["heads"] // c["kv"], c["dim"]
    at = 0
    for r, (n, kv) in enumerate(_lens(c)):
        pages = d["tables"][r, :_blocks(kv, c["page"])].long()
        k = d["k_pages"][pages].transpose(0, 1).reshape(Hk, -1, D)[:, :kv].double()
        v = d["v_pages"][pages].transpose(0, 1).reshape(Hk, -1, D)[:, :kv].double()
        for h in range(Hk):
            q = d["q"][at:at + n, h * G:(h + 1) * G].double()  # [n, G, D]
            w = (q.reshape(n * G, D) @ k[h].t()).view(n, G, kv) / math.sqrt(D)
            hidden = torch.arange(kv, device="cuda")[None, :] > torch.arange(kv - n, kv, device="cuda")[:, None]
            w = torch.softmax(w.masked_fill(hidden[:, None], -math.inf), -1)
            out[at:at + n, h * G:(h + 1) * G] = (w.view(n * G, kv) @ v[h]).view(n, G, D)
        at += n
    return {"out": out}


def _exact_plan(c, d):
    """The same bookkeeping, one request and one page after the other."""
    page, T = c["page"], c["rows"]
    new, kv, tables, free = d["new"].tolist(), d["kv"].tolist(), d["tables"].tolist(), d["free"].tolist()
    top = d["count"].item()
    for r, n in enumerate(new):
        if n < 0:
            for j in range(_blocks(kv[r], page)):
                free[top] = tables[r][j]
                top += 1
    starts, pos, slots, after = [0], [], [], []
    for r, n in enumerate(new):
        for p in range(kv[r], kv[r] + max(0, n)):
            if p % page == 0:
                top -= 1
                tables[r][p // page] = free[top]
            pos.append(p)
            slots.append(tables[r][p // page] * page + p % page)
        after.append(0 if n < 0 else kv[r] + n)
        starts.append(len(pos))
    pad = [-1] * (T - len(pos))
    as32 = [torch.tensor(x, dtype=torch.int32) for x in (after, [top], starts, pos + pad, slots + pad, [0], tables, free)]
    return _plan_out(*as32)
