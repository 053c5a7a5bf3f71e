"""What drafted trees over the paged cache are measured on: the calls that a server makes
which lets a small model draft several continuations of every conversation as a tree
of tokens, and has the large model look at all of them in one step.

A case is a dict of plain values with a "kind":

  plan       one step's trees: from every drafted token's parent, its position and
             the bits of the tokens of its request that it sees
  attention  attention of the drafted tokens over the pages: all committed keys of
             their request, and the drafted ones on the way from the root to themselves
  logprobs   log probabilities of given tokens, the entropy and the likeliest tokens
             of rows of logits
  commit     the path that the large model agrees with: lengths, pages that are not
             needed after all, and the kept keys and values of all layers moved together

The requests' lengths and trees follow from the case alone (`_trees`), all values from
the seed. Each pass is given its plain form in torch operations of 32 bits, and the
framework's call where `own` is true.
"""
import math
import random

import torch

own = False

TORCH = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
LAYERS = 36


# ---- the cases -------------------------------------------------------------------

def listed():
    return [
        # one conversation's small tree: the least bookkeeping of a step
        {"name": "plan_1x12", "kind": "plan", "req": 1, "n_lo": 12, "n_hi": 12, "runs": 0, "kv_lo": 700, "kv_hi": 700, "words": 1, "pad": 0, "mix": 1},
        # a large server's step: 256 conversations' trees, three prompts' pieces among them, a padded batch
        {"name": "plan_256", "kind": "plan", "req": 256, "n_lo": 8, "n_hi": 60, "runs": 3, "kv_lo": 50, "kv_hi": 8000, "words": 2, "pad": 77, "mix": 2},
        # one conversation at a chat's length, a tree of 16
        {"name": "attention_1x16", "kind": "attention", "req": 1, "n_lo": 16, "n_hi": 16, "runs": 0, "kv_lo": 700, "kv_hi": 700, "words": 1, "pad": 0,
         "heads": 32, "kv": 8, "dim": 128, "page": 16, "cache": "bf16", "mix": 3},
        # 16 conversations with trees of 8 to 32 tokens, a padded batch
        {"name": "attention_16", "kind": "attention", "req": 16, "n_lo": 8, "n_hi": 32, "runs": 0, "kv_lo": 500, "kv_hi": 5000, "words": 1, "pad": 9,
         "heads": 32, "kv": 4, "dim": 128, "page": 32, "cache": "f16", "mix": 4},
        # one conversation over a long document, a tree of 63
        {"name": "attention_1x63_30k", "kind": "attention", "req": 1, "n_lo": 63, "n_hi": 63, "runs": 0, "kv_lo": 30001, "kv_hi": 30001, "words": 2, "pad": 0,
         "heads": 32, "kv": 8, "dim": 128, "page": 64, "cache": "bf16", "mix": 5},
        # 64 conversations of all lengths with trees of up to 60 tokens, a prompt's piece beside them
        {"name": "attention_64", "kind": "attention", "req": 64, "n_lo": 20, "n_hi": 60, "runs": 1, "kv_lo": 100, "kv_hi": 8000, "words": 2, "pad": 0,
         "heads": 32, "kv": 8, "dim": 128, "page": 16, "cache": "bf16", "mix": 6},
        # the next token of one conversation, with the 20 alternatives that a client may ask for
        {"name": "logprobs_1", "kind": "logprobs", "rows": 1, "vocab": 151936, "top": 20, "tokens": 1, "entropy": 1, "logits": "f32", "allowed": 1.0, "mix": 7},
        # a step of 64 conversations; each row's drafted tokens looked up
        {"name": "logprobs_64", "kind": "logprobs", "rows": 64, "vocab": 151936, "top": 5, "tokens": 3, "entropy": 1, "logits": "f32", "allowed": 1.0, "mix": 8},
        # rows under a grammar that leaves a few tokens of an odd vocabulary
        {"name": "logprobs_300_grammar", "kind": "logprobs", "rows": 300, "vocab": 50021, "top": 8, "tokens": 1, "entropy": 0, "logits": "bf16", "allowed": 0.002, "mix": 9},
        # a prompt's tokens scored
        {"name": "logprobs_1000", "kind": "logprobs", "rows": 1000, "vocab": 151936, "top": 1, "tokens": 1, "entropy": 1, "logits": "bf16", "allowed": 1.0, "mix": 10},
        # one conversation's step
        {"name": "commit_1x16", "kind": "commit", "req": 1, "n_lo": 16, "n_hi": 16, "runs": 0, "kv_lo": 700, "kv_hi": 700, "words": 1, "pad": 0, "kv": 8,
         "dim": 128, "page": 16, "cache": "bf16", "mix": 32},
        # 64 conversations' step with a prompt's piece among them
        {"name": "commit_64", "kind": "commit", "req": 64, "n_lo": 8, "n_hi": 32, "runs": 1, "kv_lo": 100, "kv_hi": 8000, "words": 1, "pad": 5, "kv": 8,
         "dim": 128, "page": 16, "cache": "bf16", "mix": 12},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("plan", "attention", "attention", "attention", "logprobs", "logprobs", "commit"))
    mix = rng.randint(100, 10**6)
    if kind == "logprobs":
        vocab = _log_int(rng, 1000, 151936)
        c = {"kind": kind, "rows": _log_int(rng, 1, min(4000, 1000 * 151936 // vocab)), "vocab": vocab, "top": rng.choice((0, 1, 5, 8, 20, 32)),
             "tokens": rng.choice((0, 1, 1, 4)), "entropy": rng.choice((1, 1, 0)), "logits": rng.choice(("bf16", "f32")),
             "allowed": rng.choice((1.0, 1.0, 1.0, 0.01)), "mix": mix}
        if not c["top"] and not c["tokens"]:
            c["entropy"] = 1
        return c
    heads, kv, dim = rng.choice(((32, 8, 128), (32, 4, 128), (16, 8, 128), (32, 8, 64), (16, 4, 64)))
    words = rng.choice((1, 1, 2, 2, 4))
    hi = rng.randint(4, 32 * words)
    c = {"kind": kind, "req": _log_int(rng, 1, 256 if kind == "plan" else 64), "n_lo": rng.randint(1, hi), "n_hi": hi, "runs": 0, "kv_lo": rng.randint(130, 400),
         "kv_hi": _log_int(rng, 500, 8000), "words": words, "pad": rng.choice((0, 0, 7)), "mix": mix}
    if rng.random() < 0.3 and c["req"] > 2:
        c["runs"] = rng.randint(1, 2)
    if kind == "plan":
        return c
    c.update(kv=kv, dim=dim, page=rng.choice((16, 16, 32, 64)), cache=rng.choice(("bf16", "f16")))
    if kind == "attention":
        c["heads"] = heads
        if c["req"] > 30:  # no dearer than the listed ones
            c["n_hi"] = min(c["n_hi"], 60)
            c["n_lo"] = min(c["n_lo"], 20)
        if c["req"] == 1 and rng.random() < 0.5:
            c["kv_lo"] = c["kv_hi"] = _log_int(rng, 500, 30000)
    return c


def _trees(c):
    """Every request's (parents of its new tokens, keys with the new ones). A new token's
    parent is the number of an earlier one of its request, -1 for the first; a prompt's
    piece (longer than the mask's bits) is a chain."""
    rng = random.Random(c["mix"])
    out = []
    for r in range(c["req"]):
        if r < c["runs"]:
            n = rng.randint(32 * c["words"] + 20, 32 * c["words"] + 200)
            parents = list(range(-1, n - 1))
        else:
            n = rng.randint(c["n_lo"], c["n_hi"])
            parents = [-1] + [max(0, i - 1 - int(rng.random() ** 2 * min(i, 9))) for i in range(1, n)]
        out.append((parents, max(_log_int(rng, c["kv_lo"], c["kv_hi"]), n) if n <= 32 * c["words"] else n + _log_int(rng, c["kv_lo"], c["kv_hi"])))
    return out


def _depths(parents):
    d = []
    for p in parents:
        d.append(0 if p < 0 else d[p] + 1)
    return d


def work(c):
    if c["kind"] == "logprobs":
        n = c["rows"] * c["vocab"]
        return {"bytes": n * (2 if c["logits"] == "bf16" else 4) + c["rows"] * (8 * c["tokens"] + 8 * c["top"] + 4 * c["entropy"]), "flops": 5 * n}
    trees = _trees(c)
    rows, R = sum(len(p) for p, _ in trees), c["req"]
    if c["kind"] == "plan":
        return {"bytes": 8 * R + rows * (8 + 4 * c["words"]) + c["pad"] * (4 + 4 * c["words"]), "flops": sum(sum(_depths(p)) for p, _ in trees) + rows}
    if c["kind"] == "commit":
        moved = sum(sum(i != j for j, i in enumerate(_accept(c, r, p)[1])) for r, (p, _) in enumerate(trees) if r >= c["runs"])
        return {"bytes": LAYERS * moved * 8 * c["kv"] * c["dim"] + 16 * rows + 24 * R, "flops": rows}
    keys = sum(kv for _, kv in trees)
    seen = sum(len(p) * (kv - len(p)) + sum(_depths(p)) + len(p) for p, kv in trees)
    return {"bytes": 4 * keys * c["kv"] * c["dim"] + 4 * rows * c["heads"] * c["dim"] + 4 * rows * c["words"], "flops": 4 * seen * c["heads"] * c["dim"]}


# ---- inputs ----------------------------------------------------------------------

def _blocks(kv, page):
    return -(-kv // page)


def _accept(c, r, parents):
    """The path of request r that will be agreed with (its numbers in the request): a walk
    from the first token to children at random, as long as no row that moves lands on
    one that is still to be read, so that a pass may be repeated on its state."""
    rng = random.Random(c["mix"] * 1000 + r)
    path = [0]
    while True:
        children = [i for i, p in enumerate(parents) if p == path[-1]]
        if not children or rng.random() < 0.2:
            break
        path.append(rng.choice(children))
        if any(i < len(path) and i != j for j, i in enumerate(path)):
            path.pop()
            break
    return rng, path


def _inputs(c, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(shape, dtype, scale=1.0):
        return torch.randn(shape, device="cuda", generator=gen).mul_(scale).to(dtype)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    if c["kind"] == "logprobs":
        T, V = c["rows"], c["vocab"]
        x = normal((T, V), torch.float32, 2.5)
        if c["allowed"] < 1.0:
            x.masked_fill_(torch.rand((T, V), device="cuda", generator=gen) >= c["allowed"], -math.inf)
            x[:, V // 3] = 1.0  # (no row is left without a token)
        d = {"logits": x.to(TORCH[c["logits"]])}
        if c["tokens"]:
            d["tokens"] = torch.randint(0, V, (T, c["tokens"]), dtype=torch.int32, device="cuda", generator=gen)
            if c["allowed"] < 1.0:
                d["tokens"].fill_(V // 3)
        return d
    trees = _trees(c)
    parents = [p for t, _ in trees for p in t]
    kv, starts = [k for _, k in trees], [0]
    for t, _ in trees:
        starts.append(starts[-1] + len(t))
    T = starts[-1] + c["pad"]
    shift = int(torch.randint(0, 40, (1,), device="cuda", generator=gen).item())
    if c["kind"] == "plan":  # (another seed: other lengths)
        return {"parents": ints(parents + [-5] * c["pad"]), "starts": ints(starts), "kv": ints([k + shift for k in kv])}
    D, page, cache, Hk = c["dim"], c["page"], TORCH[c["cache"]], c["kv"]
    d = {"parents": ints(parents + [-1] * c["pad"]), "starts": ints(starts), "kv": ints(kv)}
    if c["kind"] == "attention":
        blocks = [_blocks(k, page) for k in kv]
        n_pages = sum(blocks) + 7
        order = torch.randperm(n_pages, device="cuda", generator=gen).to(torch.int32).tolist()
        tables, at = [], 0
        for n in blocks:
            tables.append(order[at:at + n] + [-1] * (max(blocks) - n))
            at += n
        d.update(q=normal((T, c["heads"], D), cache, 1.5), k_pages=normal((n_pages, Hk, page, D), cache, 1.5), v_pages=normal((n_pages, Hk, page, D), cache),
                 tables=ints(tables), out=torch.zeros((T, c["heads"], D), dtype=cache, device="cuda"))
        d["mask"] = _plain_plan(c, d)["mask"]
        return d
    # commit: the pool holds the pages that new tokens lie in; a table's older entries name others
    first = [(k - len(t)) // page for t, k in trees]
    held = [_blocks(k, page) - f for k, f in zip(kv, first)]
    n_pages = sum(held) + 9
    order = torch.randperm(n_pages, device="cuda", generator=gen).to(torch.int32).tolist()
    most = max(f + h for f, h in zip(first, held))
    tables, slots, at = [], [], 0
    for (t, k), f, h in zip(trees, first, held):
        mine = order[at:at + h]
        at += h
        tables.append([0] * f + mine + [-1] * (most - f - h))
        slots += [mine[p // page - f] * page + p % page for p in range(k - len(t), k)]
    tokens = torch.randint(0, 151936, (T,), dtype=torch.int32, device="cuda", generator=gen).tolist()
    chosen = torch.randint(0, 151936, (T,), dtype=torch.int32, device="cuda", generator=gen).tolist()
    known = []
    for r, (t, _) in enumerate(trees):
        known.append(len(t) if r < c["runs"] else 1)
        if r >= c["runs"]:
            rng, path = _accept(c, r, t)
            for a, b in zip(path, path[1:]):
                chosen[starts[r] + a] = tokens[starts[r] + b]
            end = starts[r] + path[-1]
            taken = {tokens[starts[r] + i] for i, p in enumerate(t) if p == path[-1]}
            while chosen[end] in taken:
                chosen[end] = (chosen[end] + 1) % 151936
            # (a sibling with the same token: the first of them counts)
            for a, b in zip(path, path[1:]):
                for i in range(b):
                    if t[i] == a and tokens[starts[r] + i] == tokens[starts[r] + b]:
                        tokens[starts[r] + i] = (tokens[starts[r] + i] + 1) % 151936
    free = order[at:] + [-1] * at
    d.update(tokens=ints(tokens), chosen=ints(chosen), known=ints(known), tables=ints(tables), slots=ints(slots + [-1] * c["pad"]), free=ints(free),
             count=ints([n_pages - at]))
    for name in ("k_pages", "v_pages"):
        d[name] = normal((LAYERS, n_pages, Hk, page, D), cache)
    return d


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case

    def buffer(shape, dtype=torch.int32):
        return torch.zeros(shape, dtype=dtype, device="cuda")

    # the buffers that a server keeps for its steps
    if case["kind"] == "plan":
        T = s["parents"].numel()
        s.update(positions=buffer(T), mask=buffer((T, case["words"])))
    elif case["kind"] == "commit":
        R, T = case["req"], s["parents"].numel()
        s.update(kv_out=buffer(R), count_out=buffer(1), accepted=buffer(R), path=buffer(T), next=buffer(R), status=buffer(1))
    elif case["kind"] == "logprobs":
        T, f = case["rows"], torch.float32
        if case["tokens"]:
            s["logprobs"] = buffer((T, case["tokens"]), f)
        if case["entropy"]:
            s["entropy"] = buffer(T, f)
        if case["top"]:
            s.update(top_ids=buffer((T, case["top"])), top_logprobs=buffer((T, case["top"]), f))
    if case["kind"] == "attention":
        lens = [(len(p), kv) for p, kv in _trees(case)]
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
        from janis_amd.engine import BF16, F16, F32, I32, PagedLayers
        code = {torch.bfloat16: BF16, torch.float16: F16, torch.float32: F32, torch.int32: I32}
        h = {k: b.Wrap(t.data_ptr(), tuple(t.shape), code[t.dtype], keep=t) for k, t in s.items() if isinstance(t, torch.Tensor)}
        if s["case"]["kind"] == "commit":
            caches = [[b.Wrap(t.data_ptr(), tuple(t.shape), code[t.dtype], keep=t) for t in s[k]] for k in ("k_pages", "v_pages")]
            h["layers"] = PagedLayers(*caches)  # a cache to a layer
        s["handles"] = h
    return s["handles"]


def _own_plan(b, c, s):
    h = _handles(b, s)
    b.PagedTreePlan(h["parents"], h["starts"], h["kv"], out=(h["positions"], h["mask"]))
    return {"positions": s["positions"], "mask": s["mask"]}


def _own_attention(b, c, s):
    h = _handles(b, s)
    b.PagedTreeAttention(h["q"], h["k_pages"], h["v_pages"], h["tables"], h["starts"], h["kv"], h["mask"], c["dim"] ** -0.5, maxNew=s["max_new"],
                         out=h["out"])
    return {"out": s["out"]}


def _own_logprobs(b, c, s):
    h = _handles(b, s)
    b.TokenLogProbs(h["logits"], tokens=h.get("tokens"), topK=c["top"],
                    out=(h.get("logprobs"), h.get("entropy"), h.get("top_ids"), h.get("top_logprobs")))
    return {k: s[k] for k in ("logprobs", "entropy", "top_ids", "top_logprobs") if k in s}


def _own_commit(b, c, s):
    h = _handles(b, s)
    b.PagedTreeCommit(h["parents"], h["tokens"], h["chosen"], h["starts"], h["kv"], c["words"], c["page"], h["tables"], h["free"], h["count"], h["slots"],
                      layers=h["layers"], known=h["known"],
                      out=(h["kv_out"], h["count_out"], h["accepted"], h["path"], h["next"], h["status"]))
    return _commit_out(s["kv_out"], s["count_out"], s["accepted"], s["path"], s["next"], s["status"], s["free"], s["k_pages"], s["v_pages"])


# ---- the plain forms -----------------------------------------------------------------

def _rows(starts, kv, T):
    """Of each of T rows: its request (clamped), whether it has one, its number in it, and
    the request's new tokens and keys."""
    starts, kv = starts.long(), kv.long()
    t = torch.arange(T, device="cuda")
    live = t < starts[-1]
    r = torch.searchsorted(starts[1:], t, right=True).clamp(max=kv.numel() - 1)
    return t, r, live, t - starts[r], (starts[1:] - starts[:-1])[r], kv[r]


def _plain_plan(c, s):
    T, W = s["parents"].numel(), c["words"]
    t, r, live, i, n, kv = _rows(s["starts"], s["kv"], T)
    tree = live & (n <= 32 * W)
    # ancestors, twice as far with each round
    up = torch.where(tree & (s["parents"] >= 0), t - i + s["parents"].long(), torch.full_like(t, -1))
    sees = tree[:, None] & (torch.arange(32 * W, device="cuda") == i[:, None])
    far = 1
    while far < 32 * W:
        sees = sees | (sees[up.clamp(min=0)] & (up >= 0)[:, None])
        up = torch.where(up >= 0, up[up.clamp(min=0)], up)
        far *= 2
    depth = torch.where(tree, sees.sum(-1) - 1, i)
    bits = (sees.view(T, W, 32).long() << torch.arange(32, device="cuda")).sum(-1)
    bits = torch.where(bits >= 2**31, bits - 2**32, bits)
    return {"positions": torch.where(live, kv - n + depth, torch.full_like(kv, -1)).to(torch.int32), "mask": bits.to(torch.int32)}


def _plain_attention(c, s):
    R, Hq, Hk, D, page, n, L, T, W = c["req"], c["heads"], c["kv"], c["dim"], c["page"], s["max_new"], s["max_kv"], s["rows"], c["words"]
    G = Hq // Hk
    pages = s["tables"][:, :_blocks(L, page)].clamp(min=0).long()

    def keys(pool):  # [R, Hk, keys, D]
        return pool[pages].float().transpose(1, 2).reshape(R, Hk, -1, D)

    starts, kv = s["starts"].long(), s["kv"].long()
    count = starts[1:] - starts[:-1]
    i = torch.arange(n, device="cuda")
    rows = (starts[:-1, None] + i).clamp(max=T - 1)
    q = s["q"][rows].float()  # [R, n, Hq, D]
    q = q.view(R, n, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(R, Hk, G * n, D)
    sc = torch.matmul(q, keys(s["k_pages"]).transpose(2, 3).contiguous()).mul_(D ** -0.5)
    # key number among the new tokens; the committed ones come before
    j = torch.arange(sc.shape[-1], device="cuda") - (kv - count)[:, None]  # [R, keys]
    at = j.clamp(0, 32 * W - 1)
    word = s["mask"][rows].gather(2, (at // 32)[:, None].expand(R, n, -1))
    on_the_way = ((word >> (at % 32)[:, None]) & 1).bool() & (j < 32 * W)[:, None]
    run = (count > 32 * W)[:, None, None]  # a prompt's piece: causal
    seen = (j < 0)[:, None] | torch.where(run, j[:, None] <= i[:, None], on_the_way & (j < count[:, None])[:, None])
    sc = sc.view(R, Hk, G, n, -1).masked_fill_(~seen[:, None, None], -math.inf)
    sc = sc.sub_(sc.amax(-1, keepdim=True)).exp_()
    total = sc.sum(-1, keepdim=True)
    o = torch.matmul(sc.view(R, Hk, G * n, -1), keys(s["v_pages"])).view(R, Hk, G, n, D) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(R * n, Hq, D)
    row = torch.arange(T, device="cuda")
    r = torch.searchsorted(starts[1:], row, right=True)
    s["out"][:T] = o[r * n + row - starts[r]].to(s["out"].dtype)
    return {"out": s["out"]}


def _plain_logprobs(c, s):
    x = s["logits"].float()
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    total = e.sum(-1, keepdim=True)
    log_total = torch.log(total)
    out = {}
    if c["tokens"]:
        out["logprobs"] = x.gather(1, s["tokens"].long()) - m - log_total
    if c["entropy"]:
        out["entropy"] = (log_total - (e * torch.where(e > 0, x - m, torch.zeros_like(x))).sum(-1, keepdim=True) / total)[:, 0]
    if c["top"]:
        v, i = torch.sort(x, dim=-1, descending=True, stable=True)
        out["top_ids"] = i[:, :c["top"]].to(torch.int32)
        out["top_logprobs"] = v[:, :c["top"]] - m - log_total
    return out


def _commit_out(kv, count, accepted, path, next_, status, free, k, v):
    return {"kv": kv, "count": count, "accepted": accepted, "path": path, "next": next_, "status": status, "free": free, "k_pages": k, "v_pages": v}


def _plain_commit(c, s):
    T, W, R, page, N = s["parents"].numel(), c["words"], c["req"], c["page"], s["free"].numel()
    t, r, live, i, n, kv = _rows(s["starts"], s["kv"], T)
    known = torch.where(n > 32 * W, n, s["known"].long()[r])
    up = torch.where(i < known, i - 1, s["parents"].long())
    up = torch.where(live & (up >= 0), t - i + up, torch.full_like(t, -1))
    at = up.clamp(min=0)
    agrees = live & (i >= known) & (i[at] >= known - 1) & (up >= 0) & (s["tokens"] == s["chosen"][at])
    # of children with the same token the first
    first = torch.full_like(t, T).scatter_reduce(0, at, torch.where(agrees, t, torch.full_like(t, T)), "amin")
    kept = live & ((i < known) | (agrees & (first[at] == t)))
    far = 1
    while far < 32 * W:  # and all on the way to it
        kept = kept & ((up < 0) | (i < known) | kept[at])
        up = torch.where((up >= 0) & (i >= known), up[at], torch.full_like(up, -1))
        at = up.clamp(min=0)
        far *= 2
    lens, starts = s["kv"].long(), s["starts"].long()
    before = torch.cat((torch.zeros_like(t[:1]), torch.cumsum(kept, 0)))
    accepted = before[starts[1:]] - before[starts[:-1]]
    place = torch.where(kept, starts[r] + before[:-1] - before[starts[r]], torch.full_like(t, T))
    path = torch.full((T + 1,), -1, dtype=torch.int64, device="cuda").scatter(0, place, t)[:T]
    path[T - c["pad"]:] = -1
    end = path[(starts[:-1] + accepted - 1).clamp(min=0)]
    next_ = torch.where(accepted > 0, s["chosen"][end.clamp(min=0)].long(), torch.full_like(end, -1))
    after = lens - (starts[1:] - starts[:-1]) + accepted
    # pages that no kept token needs, onto the stack
    old, want = (lens + page - 1) // page, (after + page - 1) // page
    back = old - want
    j = torch.arange(s["tables"].shape[1], device="cuda")
    top = s["count"].long()
    to = torch.where((j >= want[:, None]) & (j < old[:, None]), top + (torch.cumsum(back, 0) - back)[:, None] + j - want[:, None],
                     torch.full((R, j.numel()), N, device="cuda"))
    free = torch.cat((s["free"], s["free"][:1])).scatter(0, to.reshape(-1), s["tables"].reshape(-1))[:N]
    src, dst = s["slots"][path.clamp(min=0)].long(), s["slots"].long()
    moves = (path >= 0) & (path != t)
    src, dst = torch.where(moves, src, dst.clamp(min=0)), dst.clamp(min=0)
    # (rows that do not move write what is there; those of nobody write what is in the first row's slot)
    src, dst = torch.where(live, src, dst[0]), torch.where(live, dst, dst[0])
    for name in ("k_pages", "v_pages"):
        p = s[name]
        p[:, dst // page, :, dst % page] = p[:, src // page, :, src % page]
    as32 = [x.to(torch.int32) for x in (after, top + back.sum(), accepted, path, next_)]
    return _commit_out(*as32, torch.zeros_like(s["status"]), free, s["k_pages"], s["v_pages"])


def run(s):
    c = s["case"]
    if own:
        return _ordered({"plan": _own_plan, "attention": _own_attention, "logprobs": _own_logprobs, "commit": _own_commit}[c["kind"]], c, s)
    return {"plan": _plain_plan, "attention": _plain_attention, "logprobs": _plain_logprobs, "commit": _plain_commit}[c["kind"]](c, s)


# ---- the definitions, in 64 bits ------------------------------------------------------

def exact(case, seed):
    c, d = case, _inputs(case, seed)
    if c["kind"] == "plan":
        return _exact_plan(c, d)
    if c["kind"] == "commit":
        return _exact_commit(c, d)
    if c["kind"] == "logprobs":
        out, parts = {}, []
        for row in d["logits"].split(64):  # (rows of 64: a whole call in 64 bits is large)
            parts.append(torch.log_softmax(row.double(), -1))
        if c["tokens"]:
            out["logprobs"] = torch.cat([p.gather(1, t.long()) for p, t in zip(parts, d["tokens"].split(64))])
        if c["entropy"]:
            out["entropy"] = torch.cat([torch.special.entr(p.exp()).sum(-1) for p in parts])
        if c["top"]:
            ids = []
            for row in d["logits"].split(64):
                # distinct keys: the value's order as a whole number, then the lower index
                u = row.float().add(0.0).view(torch.int32).long()
                key = torch.where(u >= 0, u, -(u & 0x7FFFFFFF)) * 2**20 - torch.arange(c["vocab"], device="cuda")
                ids.append(torch.topk(key, c["top"], dim=-1).indices)
            out["top_ids"] = torch.cat(ids).to(torch.int32)
            out["top_logprobs"] = torch.cat([p.gather(1, i) for p, i in zip(parts, ids)])
        return out
    out = d["out"].double()
    Hk, G, D = c["kv"], c["heads"] // c["kv"], c["dim"]
    at = 0
    for r, (parents, kv) in enumerate(_trees(c)):
        n = len(parents)
        pages = d["tables"][r, :_blocks(kv, c["page"])].long()
        k = d["k_pages"][pages].transpose(0, 1).reshape(Hk, -1, D)[:, :kv].double()
        v = d["v_pages"][pages].transpose(0, 1).reshape(Hk, -1, D)[:, :kv].double()
        hidden = torch.zeros((n, kv), dtype=torch.bool)
        hidden[:, kv - n:] = True
        for i, p in enumerate(parents):
            if p >= 0:
                hidden[i] = hidden[p]
            hidden[i, kv - n + i] = False
        hidden = hidden.cuda()
        for h in range(Hk):
            q = d["q"][at:at + n, h * G:(h + 1) * G].double()  # [n, G, D]
            w = (q.reshape(n * G, D) @ k[h].t()).view(n, G, kv) / math.sqrt(D)
            w = torch.softmax(w.masked_fill(hidden[:, None], -math.inf), -1)
            out[at:at + n, h * G:(h + 1) * G] = (w.view(n * G, kv) @ v[h]).view(n, G, D)
        at += n
    return {"out": out}


def _exact_plan(c, d):
    """Each token's way to the root, one after the other."""
    pos, bits, W = [], [], c["words"]
    for (parents, _), kv in zip(_trees(c), d["kv"].tolist()):
        n = len(parents)
        for i in range(n):
            if n > 32 * W:
                pos.append(kv - n + i)
                bits.append([0] * W)
                continue
            sees, at, depth = 0, i, -1
            while at >= 0:
                sees, at, depth = sees | 1 << at, parents[at], depth + 1
            pos.append(kv - n + depth)
            words = [sees >> 32 * w & 0xFFFFFFFF for w in range(W)]
            bits.append([x - 2**32 if x >= 2**31 else x for x in words])
    pos += [-1] * c["pad"]
    bits += [[0] * W] * c["pad"]
    return {"positions": torch.tensor(pos, dtype=torch.int32), "mask": torch.tensor(bits, dtype=torch.int32)}


def _exact_commit(c, d):
    """The same, one request and one token after the other."""
    page = c["page"]
    tokens, chosen, known, kv, tables, slots = (d[k].tolist() for k in ("tokens", "chosen", "known", "kv", "tables", "slots"))
    free, top = d["free"].tolist(), d["count"].item()
    k, v = d["k_pages"].double(), d["v_pages"].double()
    after, accepted, path, nexts, moves, at = [], [], [], [], [], 0
    for r, (parents, _) in enumerate(_trees(c)):
        n = len(parents)
        mine = list(range(n if n > 32 * c["words"] else known[r]))
        while True:
            want = chosen[at + mine[-1]]
            more = [i for i in range(mine[-1] + 1, n) if parents[i] == mine[-1] and tokens[at + i] == want]
            if not more:
                break
            mine.append(more[0])
        nexts.append(want)
        accepted.append(len(mine))
        path += [at + i for i in mine] + [-1] * (n - len(mine))
        moves += [(slots[at + i], slots[at + j]) for j, i in enumerate(mine) if i != j]
        new = kv[r] - n + len(mine)
        for b in range(_blocks(new, page), _blocks(kv[r], page)):
            free[top] = tables[r][b]
            top += 1
        after.append(new)
        at += n
    if moves:
        src, dst = (torch.tensor(x, device="cuda") for x in zip(*moves))
        for p in (k, v):
            p.transpose(2, 3)[:, dst // page, dst % page] = p.transpose(2, 3)[:, src // page, src % page]
    as32 = [torch.tensor(x, dtype=torch.int32) for x in (after, [top], accepted, path + [-1] * c["pad"], nexts, [0], free)]
    return _commit_out(*as32, k, v)
