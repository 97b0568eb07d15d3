"""Performance cases of the operators between the linears of a decode step over drafted tokens: what a program that
verifies drafts with p8x runs beside the products of perf/cases.py. Head counts and widths are those of the models
that bench.py and the tests use (Llama-3.1-8B, Qwen3-4B, Qwen3-14B), the rest is generic.

A case is a dict: "op" and that op's options.
  norm    h' = h + alpha act(gate) N_post(y), x = N_pre(h'): the end of one block and the start of the next
  attn    attention of each sequence's drafted tokens (a tree: every token sees its ancestors) over its cache and the
          drafts themselves; one token is plain decode
  score   the attention weight that the accepted tokens gave to every cached slot, added to the slots' scores
  append  the accepted tokens' keys and values, rounded to the cache's type, written behind each sequence's slots
  evict   a cache cut to a budget: first and latest tokens and the highest scores stay, kept slots past the
          budget move into the freed ones
"""
import math
import os
import sys

import torch

own = False
DEV = "cuda" if torch.cuda.is_available() else "cpu"
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# hidden width, query heads, key/value heads of the models (head_dim 128)
MODELS = {"llama8b": (4096, 32, 8), "qwen4b": (2560, 32, 8), "qwen14b": (5120, 40, 8)}


def listed():
    return [
        # one token of a decode step: the smallest call there is
        {"name": "norm_1", "op": "norm", "n": 1, "C": 4096, "y": "f32", "h": "f32", "x": "f32", "post": "none", "pre": "rms", "gate": "none"},
        # a long prompt of odd length with a block's output normed, gated per token and scaled
        {"name": "norm_1500", "op": "norm", "n": 1500, "C": 5120, "y": "f32", "h": "f32", "x": "bf16", "post": "rms", "pre": "rms", "gate": "sigmoid"},
        # plain decode of one sequence, activations in f32 as the linears take them
        {"name": "attn_1", "op": "attn", "seqs": 1, "tokens": 1, "len": 1001, "heads": 32, "kv": 8, "D": 128, "page": 64, "q": "f32", "cache": "f16", "layout": "head"},
        # sixteen sequences of differing lengths decoded together, short chains of drafts, small pages, five heads a group
        {"name": "attn_batch", "op": "attn", "seqs": 16, "tokens": 3, "len": 8190, "heads": 40, "kv": 8, "D": 128, "page": 16, "q": "bf16", "cache": "bf16", "layout": "slot"},
        # eight drafted tokens (as many as a product's columns) over a long context
        {"name": "attn_long", "op": "attn", "seqs": 1, "tokens": 8, "len": 131071, "heads": 32, "kv": 8, "D": 128, "page": 256, "q": "f32", "cache": "bf16", "layout": "head"},
        # full trees over several sequences: the most rows a sequence has
        {"name": "attn_tree64", "op": "attn", "seqs": 4, "tokens": 64, "len": 16383, "heads": 32, "kv": 8, "D": 128, "page": 32, "q": "f16", "cache": "f16", "layout": "slot"},
        # one accepted token of one sequence
        {"name": "score_1", "op": "score", "seqs": 1, "tokens": 1, "len": 1001, "heads": 32, "kv": 8, "D": 128, "page": 64, "q": "f32", "cache": "f16", "layout": "head"},
        # the accepted paths of several trees over long contexts
        {"name": "score_tree", "op": "score", "seqs": 4, "tokens": 16, "len": 32767, "heads": 32, "kv": 8, "D": 128, "page": 32, "q": "bf16", "cache": "bf16", "layout": "slot"},
        # the accepted path of one tree of eight
        {"name": "append_8", "op": "append", "seqs": 1, "tokens": 8, "len": 1001, "heads": 32, "kv": 8, "D": 128, "page": 64, "q": "f32", "cache": "f16", "layout": "head"},
        # a prompt chunk of odd length
        {"name": "append_1500", "op": "append", "seqs": 1, "tokens": 1500, "len": 1001, "heads": 32, "kv": 8, "D": 128, "page": 16, "q": "f32", "cache": "bf16", "layout": "slot"},
        # a cache a few slots over its budget, as after every step
        {"name": "evict_8", "op": "evict", "seqs": 1, "len": 1008, "budget": 1000, "heads": 32, "kv": 8, "D": 128, "page": 64, "cache": "f16", "layout": "head"},
        # long prompts cut to half
        {"name": "evict_half", "op": "evict", "seqs": 4, "len": 32767, "budget": 16001, "heads": 32, "kv": 8, "D": 128, "page": 32, "cache": "bf16", "layout": "slot"},
    ]


def _log(rng, lo, hi):
    """an integer spread over the logarithm of lo .. hi"""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("norm", "attn", "attn", "attn", "score", "append", "evict"))
    if op == "norm":
        c = {"op": op, "n": _log(rng, 1, 1500), "C": _log(rng, 256, 17408)}
        c["C"] = min(c["C"], 1500 * 5120 // c["n"])
        for k in ("y", "h", "x"):
            c[k] = rng.choice(("f32", "f32", "bf16", "f16"))
        c["post"], c["pre"] = rng.choice(("none", "rms", "layer")), rng.choice(("rms", "rms", "layer"))
        c["gate"] = rng.choice(("none", "linear", "sigmoid", "shared"))
        return c
    h, kv = rng.choice(((32, 8), (40, 8), (32, 8), (16, 16), (24, 3), (28, 4)))
    c = {"op": op, "heads": h, "kv": kv, "D": rng.choice((64, 128, 128, 128, 256)), "page": rng.choice((16, 32, 48, 64, 256)),
         "cache": rng.choice(("f16", "bf16")), "layout": rng.choice(("head", "slot")), "seqs": _log(rng, 1, 24)}
    slots = 100000 * 8 * 128 // (kv * c["D"] * c["seqs"])   # of a sequence, so that no case holds more than the listed ones
    if op == "evict":
        c["len"] = _log(rng, 32, max(33, slots // 2))
        c["budget"] = max(16, int(c["len"] * rng.uniform(0.3, 1.1)))
        return c
    c["q"] = rng.choice(("f32", c["cache"]))
    c["tokens"] = _log(rng, 1, 1500 // c["seqs"]) if op == "append" else _log(rng, 1, 64)
    if op != "append":
        slots = min(slots, int(3e10) // (4 * c["D"] * h * c["tokens"] * c["seqs"]))   # nor computes more
    c["len"] = _log(rng, 1, max(2, slots))
    return c


# ------------------------------------------------------------------------------------------------- inputs
def _lens(c):
    """cached slots of each sequence: the case's length, the others spread below it"""
    return [c["len"] if s == 0 else max(1, int(c["len"] * (0.1 + 0.9 * ((0.618034 * s) % 1.0)))) for s in range(c["seqs"])]


def _tokens(c):
    """tokens of each sequence"""
    return [c["tokens"] - (5 * s) % c["tokens"] for s in range(c["seqs"])]


def _trees(c, gen):
    """(ancestor masks of all tokens, accepted sets of all sequences): each token's parent is drawn from those before it
    (half of the time the one right before), a drawn token's path is accepted; 64 bits a token"""
    mask, accept = [], []
    for t in _tokens(c):
        m = []
        for j in range(t):
            r = torch.randint(0, max(1, j), (2,), generator=gen).tolist()
            parent = j - 1 if r[0] % 2 else r[1]
            m.append((m[parent] if j else 0) | 1 << j)
        mask += m
        accept.append(max(m[int(torch.randint(0, t, (1,), generator=gen))], m[t // 2], key=lambda v: bin(v).count("1")))
    signed = [v - (1 << 64) if v >> 63 else v for v in mask + accept]
    return signed[:len(mask)], signed[len(mask):]


def _cap(c):
    """slots that a sequence has room for"""
    return c["len"] + c.get("tokens", 0)


def _cache(c, s, g):
    """keys and values in pages of a shuffled pool; channels of differing size as keys have them"""
    S, kv, D, page = c["seqs"], c["kv"], c["D"], c["page"]
    per = -(-_cap(c) // page)
    n = S * per + 3
    shape = (n, kv, page, D) if c["layout"] == "head" else (n, page, kv, D)
    ch = torch.exp(0.4 * torch.randn(D, device=DEV, generator=g))
    s["k"] = torch.empty(shape, device=DEV, dtype=DT[c["cache"]])
    s["v"] = torch.empty(shape, device=DEV, dtype=DT[c["cache"]])
    for i in range(0, n, 1024):   # bounds the f32 copy
        s["k"][i:i + 1024] = torch.randn((min(1024, n - i),) + shape[1:], device=DEV, generator=g) * ch
        s["v"][i:i + 1024] = torch.randn((min(1024, n - i),) + shape[1:], device=DEV, generator=g)
    s["pages"] = torch.randperm(n, device=DEV, generator=g)[:S * per].view(S, per).int()
    s["len"] = torch.tensor(_lens(c), device=DEV, dtype=torch.int32)
    s["len_out"] = torch.zeros_like(s["len"])
    return ch


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(seed)
    gen = torch.Generator().manual_seed(seed + 1)
    s = {"case": c}

    def randn(*shape):
        return torch.randn(shape, device=DEV, generator=g)
    if c["op"] == "norm":
        n, C = c["n"], c["C"]
        ch = torch.exp(0.5 * randn(C))
        s["y"] = (randn(n, C) * ch * 0.3).to(DT[c["y"]])
        s["h"] = (randn(n, C) * ch).to(DT[c["h"]])
        s["h_out"], s["x"] = torch.zeros_like(s["h"]), torch.zeros(n, C, device=DEV, dtype=DT[c["x"]])
        for side in ("post", "pre"):
            s["w_" + side] = 1.0 + 0.2 * randn(C) if c[side] != "none" else None
            s["b_" + side] = 0.1 * randn(C) if c[side] == "layer" else None
        s["gate"] = None if c["gate"] == "none" else randn(C if c["gate"] == "shared" else n, *(() if c["gate"] == "shared" else (C,)))
        return s
    S, kv, D, H = c["seqs"], c["kv"], c["D"], c["heads"]
    ch = _cache(c, s, g)
    if c["op"] == "evict":
        # heavy hitters among many slots that got next to nothing, some of them exactly nothing
        sc = torch.exp(3.0 * randn(S, kv, _cap(c)) - 4.0)
        s["score"] = torch.where(sc < 1e-3, torch.zeros_like(sc), sc)
        s["pos"] = torch.arange(_cap(c), device=DEV, dtype=torch.int32).expand(S, kv, -1).contiguous()
        s["score_out"], s["pos_out"] = torch.zeros_like(s["score"]), torch.zeros_like(s["pos"])
        moves = min(c["budget"], max(0, _cap(c) - c["budget"]))
        s["ws"] = torch.zeros(S * kv * (8 * moves + 32768), device=DEV, dtype=torch.uint8)
        return s
    toks = _tokens(c)
    n = sum(toks)
    s["first"] = torch.tensor([sum(toks[:i]) for i in range(S + 1)], device=DEV, dtype=torch.int32)
    s["at"] = torch.cat([torch.arange(t, device=DEV, dtype=torch.int32) + l for t, l in zip(toks, _lens(c))])   # positions
    # q, k and v side by side in one buffer, as the layer's products leave them
    qkv = torch.cat([1.5 * randn(n, H * D), randn(n, kv, D).mul(ch).view(n, kv * D), randn(n, kv * D)], 1).to(DT[c["q"]])
    s["qkv"] = qkv
    s["q"], s["kn"], s["vn"] = (qkv[:, a:b].unflatten(1, (-1, D)) for a, b in ((0, H * D), (H * D, H * D + kv * D), (H * D + kv * D, (H + 2 * kv) * D)))
    if c["op"] == "append" and c["tokens"] > 64:
        s["accept"] = None   # a prompt: all of it
    else:
        mask, accept = _trees(c, gen)
        s["mask"] = torch.tensor(mask, device=DEV, dtype=torch.int64)
        s["accept"] = torch.tensor(accept, device=DEV, dtype=torch.int64)
    s["pos"] = torch.arange(_cap(c), device=DEV, dtype=torch.int32).expand(S, kv, -1).contiguous()
    if c["op"] in ("attn", "score"):
        s["out"] = torch.zeros(n, H, D, device=DEV, dtype=DT[c["q"]])
        s["lse"] = torch.zeros(n, H, device=DEV)
        s["ws"] = torch.zeros(96 << 20, device=DEV, dtype=torch.uint8)
    if c["op"] == "score":
        s["lse"] = _attention(s)[1]   # what the attention of these tokens left
        s["score"] = torch.rand(S, kv, _cap(c), device=DEV, generator=g) * 0.1
        s["score_out"] = torch.zeros_like(s["score"])
    return s


# ------------------------------------------------------------------------------------------------- plain forms
def _f32_norm(v, kind, w, b):
    if kind == "none":
        return v
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + 1e-6) * w
    return v if b is None else v + b


def _norm(s):
    c = s["case"]
    u = _f32_norm(s["y"].float(), c["post"], s["w_post"], s["b_post"])
    if s["gate"] is not None:
        u = u * (torch.sigmoid(s["gate"]) if c["gate"] == "sigmoid" else s["gate"])
    h = s["h"].float() + 0.7 * u
    s["h_out"].copy_(h)
    s["x"].copy_(_f32_norm(h, c["pre"], s["w_pre"], s["b_pre"]))
    return {"h": s["h_out"], "x": s["x"]}


def _slots(s, t):
    """[seqs, kv, slots, D] of a pool, in 32 bits"""
    t = t if s["case"]["layout"] == "head" else t.transpose(1, 2)
    t = t[s["pages"].long()].transpose(1, 2)   # [S, kv, pages, page, D]
    return t.flatten(2, 3)[:, :, :s["case"]["len"]].float()


def _padded(s):
    """(token of each sequence's place [S, T], whether there is one)"""
    first = s["first"].long()
    t = torch.arange(s["case"]["tokens"], device=DEV)
    there = t < (first[1:] - first[:-1])[:, None]
    return torch.where(there, first[:-1, None] + t, 0), there


def _scores(s):
    """(scaled scores [S, kv, G, T, slots + T] with -inf where unseen, padded tokens, which are there)"""
    c = s["case"]
    S, kv, D, T, G = c["seqs"], c["kv"], c["D"], c["tokens"], c["heads"] // c["kv"]
    tok, there = _padded(s)
    q = s["q"][tok].float().view(S, T, kv, G, D).permute(0, 2, 3, 1, 4).reshape(S, kv, G * T, D)
    kn = s["kn"][tok].to(DT[c["cache"]]).float().permute(0, 2, 1, 3)
    k = torch.cat([_slots(s, s["k"]), kn], 2)
    sc = (torch.matmul(q, k.transpose(2, 3)) * D ** -0.5).view(S, kv, G, T, -1)
    ctx = torch.arange(c["len"], device=DEV) < s["len"][:, None]
    tree = (s["mask"][tok][:, :, None] >> torch.arange(T, device=DEV)) & 1 == 1
    seen = torch.cat([ctx[:, None].expand(-1, T, -1), tree & there[:, None]], 2) & there[:, :, None]
    return sc.masked_fill(~seen[:, None, None], -math.inf), tok, there


def _attention(s):
    c = s["case"]
    S, kv, D, T, H = c["seqs"], c["kv"], c["D"], c["tokens"], c["heads"]
    sc, tok, there = _scores(s)
    m = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(m == -math.inf, 0.0, m))
    z = p.sum(-1, keepdim=True)
    v = torch.cat([_slots(s, s["v"]), s["vn"][tok].to(DT[c["cache"]]).float().permute(0, 2, 1, 3)], 2)
    o = torch.matmul((p / z.clamp_min(1e-30)).view(S, kv, -1, v.shape[2]), v).view(S, kv, H // kv, T, D)
    lse = (m + torch.log(z)).squeeze(-1)
    rows = there.flatten().argsort(descending=True, stable=True)[:s["q"].shape[0]]   # places in the tokens' order
    out = o.permute(0, 3, 1, 2, 4).reshape(S * T, H, D)[rows]
    return out, lse.permute(0, 3, 1, 2).reshape(S * T, H)[rows]


def _attn(s):
    out, lse = _attention(s)
    s["out"].copy_(out)
    s["lse"].copy_(lse)
    return {"out": s["out"], "lse": s["lse"]}


def _accepted(s):
    """(which padded tokens are accepted [S, T], their rank)"""
    _, there = _padded(s)
    if s["accept"] is not None:
        there = there & ((s["accept"][:, None] >> torch.arange(there.shape[1], device=DEV)) & 1 == 1)
    return there, there.cumsum(1) - 1


def _score(s):
    c = s["case"]
    S, kv, T = c["seqs"], c["kv"], c["tokens"]
    sc, tok, _ = _scores(s)
    take, rank = _accepted(s)
    lse = s["lse"][tok].view(S, T, kv, -1).permute(0, 2, 3, 1)[..., None]
    w = torch.where(take[:, None, None, :, None], torch.exp(sc - lse), 0.0).sum((2, 3))   # [S, kv, slots + T]
    n = c["len"]
    ctx = torch.arange(n, device=DEV) < s["len"][:, None, None]
    new = s["score_out"].clone()
    new[:, :, :n] = torch.where(ctx, 0.9 * s["score"][:, :, :n] + w[:, :, :n], new[:, :, :n])
    at = torch.where(take, s["len"][:, None] + rank, new.shape[2])[:, None].expand(-1, kv, -1).long()
    new = torch.cat([new, new[:, :, :1]], 2).scatter(2, at, w[:, :, n:])[:, :, :-1]   # the last place takes what is not accepted
    s["score_out"].copy_(new)
    return s["score_out"]


def _at(s, slot):
    """(page, place in the page) of slots [S, ...]"""
    page = s["case"]["page"]
    S = slot.shape[0]
    return s["pages"].long().gather(1, (slot // page).view(S, -1)).view(slot.shape), slot % page


def _append(s):
    c = s["case"]
    take, rank = _accepted(s)
    tok, _ = _padded(s)
    last = torch.where(take, rank, 0).argmax(1, keepdim=True)   # those not accepted write the last accepted row again
    tok = torch.where(take, tok, tok.gather(1, last))
    rank = torch.where(take, rank, rank.gather(1, last))
    slot = s["len"][:, None].long() + rank
    page, place = _at(s, slot)
    for name, new in (("k", s["kn"]), ("v", s["vn"])):
        pool = s[name].transpose(1, 2) if c["layout"] == "head" else s[name]
        pool[page, place] = new[tok].to(pool.dtype)
    s["pos"].scatter_(2, slot[:, None].expand(-1, c["kv"], -1), s["at"][tok][:, None].expand(-1, c["kv"], -1))
    s["len_out"].copy_(s["len"] + take.sum(1))
    return {"k": s["k"], "v": s["v"], "pos": s["pos"], "len": s["len_out"]}


def _protect(c):
    """(first tokens, latest tokens) that an eviction keeps"""
    return min(4, c["budget"] // 4), c["budget"] // 8


def _evict(s):
    c = s["case"]
    S, kv, L, budget = c["seqs"], c["kv"], _cap(c), c["budget"]
    sinks, recent = _protect(c)
    slot = torch.arange(L, device=DEV)
    valid = slot < s["len"][:, None, None].expand(S, kv, 1)
    end = torch.where(valid, s["pos"], -1).amax(2, keepdim=True) + 1
    kind = valid.int() + (valid & ((s["pos"] < sinks) | (s["pos"] >= end - recent))).int()
    order = s["score"].argsort(dim=2, descending=True, stable=True)
    order = order.gather(2, kind.gather(2, order).argsort(dim=2, descending=True, stable=True))
    keep = torch.zeros_like(valid).scatter(2, order[:, :, :budget], True) & valid
    s["score_out"][:, :, :budget] = torch.where(valid, s["score"], s["score_out"])[:, :, :budget]
    s["pos_out"][:, :, :budget] = torch.where(valid, s["pos"], s["pos_out"])[:, :, :budget]
    M = min(budget, max(0, L - budget))
    if M:
        hole, mover = valid & ~keep & (slot < budget), keep & (slot >= budget)
        real = torch.arange(M, device=DEV) < hole.sum(2, keepdim=True)
        idle = (budget + torch.arange(M, device=DEV)).expand(S, kv, -1)   # slots past the budget are never written: they stand for no move
        dst = torch.where(real, hole.int().argsort(dim=2, descending=True, stable=True)[:, :, :M], idle)
        src = torch.where(real, mover.int().argsort(dim=2, descending=True, stable=True)[:, :, :M], idle)
        h = torch.arange(kv, device=DEV)[:, None].expand(S, kv, M)
        (p0, o0), (p1, o1) = _at(s, src), _at(s, dst)
        for name in ("k", "v"):
            pool = s[name] if c["layout"] == "head" else s[name].transpose(1, 2)
            pool[p1, h, o1] = pool[p0, h, o0]
        for name in ("score", "pos"):
            new = s[name].gather(2, src)
            s[name + "_out"].scatter_(2, dst, torch.where(real, new, s[name + "_out"].gather(2, dst)))
    s["len_out"].copy_(s["len"].clamp_max(budget))
    return {"k": s["k"], "v": s["v"], "score": s["score_out"], "pos": s["pos_out"], "len": s["len_out"]}


PLAIN = {"norm": _norm, "attn": _attn, "score": _score, "append": _append, "evict": _evict}


# ------------------------------------------------------------------------------------------------- the framework's calls
def _operator(s):
    """The framework's operator object for the state's buffers: kept by the program, as its buffers are."""
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pingala8-llm_amd"))
    import p8x
    c = s["case"]
    dt = {"f32": p8x.F32, "f16": p8x.F16, "bf16": p8x.BF16}
    ptr = {k: v.data_ptr() for k, v in s.items() if isinstance(v, torch.Tensor)}
    if c["op"] == "norm":
        kind = {"none": p8x.NORM_NONE, "rms": p8x.NORM_RMS, "layer": p8x.NORM_LAYER}
        return p8x.NormResidual(
            c["n"], c["C"], y=ptr["y"], y_dtype=dt[c["y"]], h=ptr["h"], h_dtype=dt[c["h"]], h_out=ptr["h_out"], x=ptr["x"], x_dtype=dt[c["x"]],
            post=kind[c["post"]], w_post=ptr.get("w_post"), b_post=ptr.get("b_post"), pre=kind[c["pre"]], w_pre=ptr.get("w_pre"), b_pre=ptr.get("b_pre"),
            gate=ptr.get("gate"), gate_act=p8x.GATE_SIGMOID if c["gate"] == "sigmoid" else p8x.GATE_LINEAR,
            ld_gate=0 if c["gate"] == "shared" else c["C"], alpha=0.7, eps_post=1e-6, eps_pre=1e-6)
    st = s["k"].stride()
    cache = p8x.KvCache(
        dt[c["cache"]], c["seqs"], c["kv"], c["D"], k=ptr["k"], v=ptr["v"], page_stride=st[0], head_stride=st[1 if c["layout"] == "head" else 2],
        slot_stride=st[2 if c["layout"] == "head" else 1], page_size=c["page"], n_pages=s["k"].shape[0], pages=ptr["pages"],
        ld_pages=s["pages"].shape[1], len=ptr["len"], max_len=_cap(c))
    if c["op"] == "evict":
        sinks, recent = _protect(c)
        return p8x.KvEvict(cache, c["budget"], score=ptr["score"], score_out=ptr["score_out"], pos=ptr["pos"], pos_out=ptr["pos_out"],
                           len_out=ptr["len_out"], n_sink=sinks, n_recent=recent, workspace=ptr["ws"], workspace_bytes=s["ws"].numel())
    n, ld = s["qkv"].shape
    draft = dict(n_tokens=n, max_tokens=c["tokens"], first=ptr["first"], k=ptr["kn"], v=ptr["vn"], kv_dtype=dt[c["q"]], ld_kv=ld)
    if c["op"] == "append":
        return p8x.KvAppend(cache, accept=ptr.get("accept"), at=ptr["at"], pos=ptr["pos"], len_out=ptr["len_out"], **draft)
    draft.update(n_heads=c["heads"], q=ptr["q"], q_dtype=dt[c["q"]], ld_q=ld, mask=ptr["mask"], scale=c["D"] ** -0.5, lse=ptr["lse"])
    if c["op"] == "attn":
        return p8x.AttnTree(cache, out=ptr["out"], workspace=ptr["ws"], workspace_bytes=s["ws"].numel(), **draft)
    return p8x.KvScore(cache, accept=ptr["accept"], score=ptr["score"], score_out=ptr["score_out"], decay=0.9, **draft)


def _results(s):
    return {"norm": lambda: {"h": s["h_out"], "x": s["x"]}, "attn": lambda: {"out": s["out"], "lse": s["lse"]}, "score": lambda: s["score_out"],
            "append": lambda: {"k": s["k"], "v": s["v"], "pos": s["pos"], "len": s["len_out"]},
            "evict": lambda: {"k": s["k"], "v": s["v"], "score": s["score_out"], "pos": s["pos_out"], "len": s["len_out"]}}[s["case"]["op"]]()


def run(s):
    if not own:
        return PLAIN[s["case"]["op"]](s)
    if "call" not in s:
        s["call"] = _operator(s)
        s["result"] = _results(s)
    s["call"].run()
    return s["result"]


# ------------------------------------------------------------------------------------------------- bytes and operations
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def _popcounts(c):
    """a tree's accepted path, about: its depth grows with the logarithm of its tokens' number"""
    return [min(t, int(2 + math.log2(t))) if c["tokens"] <= 64 else t for t in _tokens(c)]


def work(case):
    c = case
    if c["op"] == "norm":
        n = c["n"] * c["C"]
        b = n * (SIZE[c["y"]] + 2 * SIZE[c["h"]] + SIZE[c["x"]]) + 4 * c["C"] * sum((0, 1, 2)[("none", "rms", "layer").index(c[k])] for k in ("post", "pre"))
        b += {"none": 0, "shared": 4 * c["C"]}.get(c["gate"], 4 * n)
        return {"bytes": b, "flops": 12.0 * n}
    S, kv, D, H = c["seqs"], c["kv"], c["D"], c["heads"]
    row = 2 * kv * D   # a slot's keys or values, in bytes
    lens = _lens(c)
    if c["op"] == "evict":
        left = [min(n, c["budget"]) for n in lens]
        # expected moves: a kept slot lies past the budget with the share of slots that do
        moved = sum(b * (n - b) / n for n, b in zip(lens, left))
        return {"bytes": sum(8 * kv * n + 8 * kv * b for n, b in zip(lens, left)) + 4 * row * moved, "flops": 4.0 * kv * sum(lens)}
    toks, acc = _tokens(c), _popcounts(c)
    if c["op"] == "append":
        return {"bytes": sum(acc) * (2 * kv * D * (SIZE[c["q"]] + 2) + 4 * kv), "flops": 2.0 * kv * D * sum(acc)}
    if c["op"] == "attn":
        b = sum(2 * row * n + t * (2 * H + 2 * kv) * D * SIZE[c["q"]] + 4 * t * H for n, t in zip(lens, toks))
        return {"bytes": b, "flops": sum(4.0 * D * H * t * (n + t) for n, t in zip(lens, toks))}
    return {"bytes": sum((row + 8 * kv) * n + a * (H + kv) * D * SIZE[c["q"]] for n, a in zip(lens, acc)),
            "flops": sum(2.0 * D * H * a * (n + a) for n, a in zip(lens, acc))}


# ------------------------------------------------------------------------------------------------- 64-bit results
def _exact_norm(s):
    c = s["case"]

    def norm(v, side):
        if c[side] == "none":
            return v
        mean = v.sum(1) / c["C"] if c[side] == "layer" else torch.zeros_like(v[:, 0])
        var = ((v - mean[:, None]) ** 2).sum(1) / c["C"]
        v = (v - mean[:, None]) / (var + 1e-6).sqrt()[:, None] * s["w_" + side].double()
        return v + s["b_" + side].double() if c[side] == "layer" else v
    g = 1.0 if s["gate"] is None else s["gate"].double()
    g = 1.0 / (1.0 + torch.exp(-g)) if c["gate"] == "sigmoid" else g
    h = s["h"].double() + 0.7 * g * norm(s["y"].double(), "post")
    return {"h": h, "x": norm(h, "pre")}


def _rows(s, name, seq, head, slots):
    """64-bit keys or values of one sequence's slots and key/value head"""
    page = s["case"]["page"]
    at = s["pages"][seq].long()[slots // page]
    t = s[name]
    return (t[at, head, slots % page] if s["case"]["layout"] == "head" else t[at, slots % page, head]).double()


def _each(s):
    """for every sequence and key/value head: (tokens' range, head, 64-bit scores [T, G, slots + T], -inf where unseen)"""
    c = s["case"]
    G, first = c["heads"] // c["kv"], s["first"].tolist()
    for i, n in enumerate(_lens(c)):
        a, b = first[i], first[i + 1]
        slots = torch.arange(n, device=DEV)
        bits = torch.tensor([[(m >> j) & 1 for j in range(b - a)] for m in s["mask"][a:b].tolist()], device=DEV, dtype=torch.bool)
        for h in range(c["kv"]):
            k = torch.cat([_rows(s, "k", i, h, slots), s["kn"][a:b, h].to(DT[c["cache"]]).double()])
            q = s["q"][a:b, h * G:(h + 1) * G].double()
            sc = (q.reshape(-1, c["D"]) @ k.t().contiguous() / math.sqrt(c["D"])).view(b - a, G, -1)
            sc[:, :, n:].masked_fill_(~bits[:, None], -math.inf)
            yield i, h, a, b, slots, sc


def _exact_attn(s):
    c = s["case"]
    G = c["heads"] // c["kv"]
    out = torch.zeros(s["q"].shape, device=DEV, dtype=torch.float64)
    lse = torch.zeros(s["q"].shape[:2], device=DEV, dtype=torch.float64)
    for i, h, a, b, slots, sc in _each(s):
        v = torch.cat([_rows(s, "v", i, h, slots), s["vn"][a:b, h].to(DT[c["cache"]]).double()])
        z = torch.logsumexp(sc, 2)
        lse[a:b, h * G:(h + 1) * G] = z
        out[a:b, h * G:(h + 1) * G] = (torch.exp(sc - z[:, :, None]).view(-1, v.shape[0]) @ v).view(b - a, G, -1)
    return {"out": out, "lse": lse}


def _exact_score(s):
    c = s["case"]
    G, new = c["heads"] // c["kv"], s["score_out"].double().clone()
    for i, h, a, b, slots, sc in _each(s):
        n = len(slots)
        took = [j for j in range(b - a) if (int(s["accept"][i]) >> j) & 1]
        w = torch.exp(sc - s["lse"][a:b, h * G:(h + 1) * G, None].double())[took].sum((0, 1))
        new[i, h, :n] = 0.9 * s["score"][i, h, :n].double() + w[:n]
        new[i, h, n:n + len(took)] = w[n:][took]
    return new


def _exact_evict(s):
    """Moves only: the caches as they are after them. Sorted on the host, one head after another."""
    c = s["case"]
    budget, (sinks, recent) = c["budget"], _protect(c)
    out = {k: s[f].cpu().clone() for k, f in (("k", "k"), ("v", "v"), ("score", "score_out"), ("pos", "pos_out"))}
    score, pos, pages = s["score"].cpu(), s["pos"].cpu(), s["pages"].cpu().long()
    for i, n in enumerate(_lens(c)):
        for h in range(c["kv"]):
            p = pos[i, h, :n]
            safe = (p < sinks) | (p >= int(p.max()) + 1 - recent)
            rank = torch.where(safe, math.inf, score[i, h, :n].double())
            kept = torch.sort(-rank, stable=True).indices[:budget]
            is_kept = torch.zeros(n, dtype=torch.bool)
            is_kept[kept] = True
            src = torch.nonzero(is_kept[budget:]).flatten() + budget
            dst = torch.nonzero(~is_kept[:budget]).flatten()
            to = torch.arange(min(n, budget))
            to[dst] = src
            out["score"][i, h, :len(to)], out["pos"][i, h, :len(to)] = score[i, h, to], p[to]
            for name in ("k", "v"):
                t = out[name] if c["layout"] == "head" else out[name].transpose(1, 2)
                t[pages[i][dst // c["page"]], h, dst % c["page"]] = t[pages[i][src // c["page"]], h, src % c["page"]]
    return {**out, "len": s["len"].cpu().clamp_max(budget)}


def _exact_append(s):
    c = s["case"]
    out = {k: s[k].cpu().clone() for k in ("k", "v", "pos")}
    first, pages, at = s["first"].tolist(), s["pages"].cpu().long(), s["at"].cpu()
    kn, vn = s["kn"].cpu(), s["vn"].cpu()
    ends = []
    for i, n in enumerate(_lens(c)):
        toks = [j for j in range(first[i + 1] - first[i]) if s["accept"] is None or (int(s["accept"][i]) >> j) & 1]
        for r, j in enumerate(toks):
            page, place = int(pages[i, (n + r) // c["page"]]), (n + r) % c["page"]
            for name, new in (("k", kn), ("v", vn)):
                (out[name][page, :, place] if c["layout"] == "head" else out[name][page, place])[:] = new[first[i] + j].to(out[name].dtype)
            out["pos"][i, :, n + r] = at[first[i] + j]
        ends.append(n + len(toks))
    return {**out, "len": torch.tensor(ends, dtype=torch.int32)}


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "attn": _exact_attn, "score": _exact_score, "append": _exact_append, "evict": _exact_evict}[case["op"]](s)
