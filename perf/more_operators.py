"""Performance cases of what a prompt and a drafted token need between the linears of a model with rotary positions: the
rotation of queries and keys, the keys' way into the cache with it, and the attention of a prompt's tokens over that cache.
Head counts and widths are those of the models that bench.py and the tests use (Llama-3.1-8B, Qwen3-4B, Qwen3-14B), the
rest is generic.

A case is a dict: "op" and that op's options.
  rope    queries and keys of a layer's products, each head normed where the model does, rotated by their positions
  append  the same, with the keys written behind each sequence's cached slots in the cache's type, the values beside them
  attn    causal attention of each sequence's newest tokens, which are its last cached slots, over its cache
"""
import math
import os
import sys

import torch

own = False
DEV = "cuda" if torch.cuda.is_available() else "cpu"
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
BASE, EPS = 500000.0, 1e-6
# how angles are scaled for contexts beyond those of training: kind, factor, trained length, two bounds
SCALING = {"none": dict(kind="none", factor=1.0, original=8192, low=1.0, high=4.0), "linear": dict(kind="linear", factor=4.0, original=8192, low=1.0, high=4.0),
           "bands": dict(kind="bands", factor=8.0, original=8192, low=1.0, high=4.0), "yarn": dict(kind="yarn", factor=4.0, original=32768, low=1.0, high=32.0)}


def listed():
    return [
        # one token of a decode step: the smallest call there is
        {"name": "rope_1", "op": "rope", "n": 1, "heads": 32, "kv": 8, "D": 128, "rot": 128, "layout": "half", "in": "f32", "out": "f32", "norm": False, "scaling": "bands", "far": 1001},
        # drafted tokens of a few sequences, neighbouring elements as pairs, half of each head
        {"name": "rope_drafts", "op": "rope", "n": 64, "heads": 16, "kv": 16, "D": 128, "rot": 64, "layout": "pairs", "in": "f32", "out": "f16", "norm": False, "scaling": "linear", "far": 100000},
        # a prompt of odd length with normed heads, far into a scaled context
        {"name": "rope_1500", "op": "rope", "n": 1500, "heads": 40, "kv": 8, "D": 128, "rot": 128, "layout": "half", "in": "f32", "out": "bf16", "norm": True, "scaling": "yarn", "far": 120000},
        # the newest tokens of sequences decoded together
        {"name": "append_24", "op": "append", "seqs": 24, "tokens": 1, "len": 4095, "heads": 32, "kv": 8, "D": 128, "page": 64, "in": "f32", "cache": "f16", "layout": "head", "rot": 128, "rope": "half", "norm": True, "scaling": "none"},
        # a prompt chunk of odd length behind a cached one
        {"name": "append_1500", "op": "append", "seqs": 1, "tokens": 1500, "len": 1001, "heads": 32, "kv": 8, "D": 128, "page": 16, "in": "bf16", "cache": "bf16", "layout": "slot", "rot": 128, "rope": "half", "norm": False, "scaling": "bands"},
        # one token over a short cache
        {"name": "attn_1", "op": "attn", "seqs": 1, "tokens": 1, "len": 1001, "heads": 32, "kv": 8, "D": 128, "page": 64, "q": "f16", "cache": "f16", "layout": "head"},
        # a question as the first turn, queries as the products leave them
        {"name": "attn_19", "op": "attn", "seqs": 1, "tokens": 19, "len": 0, "heads": 32, "kv": 8, "D": 128, "page": 16, "q": "f32", "cache": "f16", "layout": "head"},
        # a prompt of the benchmark's length
        {"name": "attn_512", "op": "attn", "seqs": 1, "tokens": 512, "len": 0, "heads": 32, "kv": 8, "D": 128, "page": 64, "q": "bf16", "cache": "bf16", "layout": "head"},
        # sequences of differing lengths with chunks of differing sizes, small pages, five heads a group
        {"name": "attn_batch", "op": "attn", "seqs": 16, "tokens": 301, "len": 4099, "heads": 40, "kv": 8, "D": 128, "page": 16, "q": "bf16", "cache": "bf16", "layout": "slot"},
        # a chunk of a long document, f32 accuracy
        {"name": "attn_chunk_f32", "op": "attn", "seqs": 1, "tokens": 999, "len": 15001, "heads": 32, "kv": 8, "D": 128, "page": 64, "q": "f32", "cache": "f16", "layout": "head"},
        # wide heads
        {"name": "attn_wide", "op": "attn", "seqs": 2, "tokens": 2049, "len": 8190, "heads": 16, "kv": 16, "D": 256, "page": 48, "q": "bf16", "cache": "bf16", "layout": "slot"},
        # a long prompt at once
        {"name": "attn_8190", "op": "attn", "seqs": 1, "tokens": 8190, "len": 0, "heads": 32, "kv": 8, "D": 128, "page": 256, "q": "f16", "cache": "f16", "layout": "head"},
    ]


def _log(rng, lo, hi):
    """an integer spread over the logarithm of lo .. hi"""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("rope", "append", "attn", "attn", "attn"))
    h, kv = rng.choice(((32, 8), (40, 8), (32, 8), (16, 16), (24, 3), (28, 4)))
    c = {"op": op, "heads": h, "kv": kv, "D": rng.choice((64, 128, 128, 128, 256))}
    if op != "attn":
        c["rot"] = rng.choice((c["D"], c["D"], c["D"] // 2, 8 * rng.randint(1, c["D"] // 8)))
        c["norm"], c["scaling"] = rng.random() < 0.4, rng.choice(tuple(SCALING))
        c["in"] = rng.choice(("f32", "f32", "bf16", "f16"))
    if op == "rope":
        c["n"], c["layout"], c["far"] = _log(rng, 1, 4096), rng.choice(("half", "half", "pairs")), _log(rng, 1, 1000000)
        c["out"] = rng.choice(("f32", "bf16", "f16"))
        return c
    c.update(page=rng.choice((16, 32, 48, 64, 256)), cache=rng.choice(("f16", "bf16")), layout=rng.choice(("head", "slot")), seqs=_log(rng, 1, 24))
    c["tokens"] = _log(rng, 1, 8190 // c["seqs"])
    slots = 100000 * 8 * 128 // (kv * c["D"] * c["seqs"])   # of a sequence, so that no case holds more than the memory of a long context
    if op == "append":
        c["rope"] = rng.choice(("half", "half", "pairs"))
        if c["in"] != "f32":
            c["in"] = c["cache"]
    else:
        c["q"] = rng.choice(("f32", c["cache"], c["cache"]))
        if c["q"] == "f32":
            c["tokens"] = min(c["tokens"], 2048)
        # nor computes more than the largest
        most = 5.4e11 / (4 * c["D"] * h * c["tokens"] * c["seqs"]) - c["tokens"] / 2
        while most < 0:
            c["tokens"] //= 2
            most = 5.4e11 / (4 * c["D"] * h * c["tokens"] * c["seqs"]) - c["tokens"] / 2
        slots = min(slots, int(most))
    c["len"] = _log(rng, 1, max(2, slots)) - 1
    return c


# ------------------------------------------------------------------------------------------------- inputs
def _lens(c):
    """slots of each sequence before its new tokens: the case's length, the others spread below it"""
    return [c["len"] if s == 0 else int(c["len"] * (0.1 + 0.9 * ((0.618034 * s) % 1.0))) for s in range(c["seqs"])]


def _tokens(c):
    """new tokens of each sequence"""
    return [c["tokens"] if s == 0 else max(1, int(c["tokens"] * (0.1 + 0.9 * ((0.754878 * s) % 1.0)))) for s in range(c["seqs"])]


def _cap(c):
    """slots that a sequence has room for"""
    return c["len"] + c["tokens"]


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


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = {"case": c}
    kv, D, H = c["kv"], c["D"], c["heads"]

    def randn(*shape):
        return torch.randn(shape, device=DEV, generator=g)
    if c["op"] == "rope":
        n = c["n"]
        # q, k and v side by side in one buffer, as the layer's products leave them
        s["qkv"] = torch.cat([1.5 * randn(n, H * D), randn(n, 2 * kv * D)], 1).to(DT[c["in"]])
        s["at"] = torch.arange(n, device=DEV, dtype=torch.int32) + c["far"]
        s["q_out"], s["k_out"] = (torch.zeros(n, h, D, device=DEV, dtype=DT[c["out"]]) for h in (H, kv))
    else:
        _cache(c, s, g)
        toks = _tokens(c)
        n = sum(toks)
        s["first"] = torch.tensor([sum(toks[:i]) for i in range(len(toks) + 1)], device=DEV, dtype=torch.int32)
        if c["op"] == "append":
            s["qkv"] = torch.cat([1.5 * randn(n, H * D), randn(n, 2 * kv * D)], 1).to(DT[c["in"]])
            s["len"] = torch.tensor(_lens(c), device=DEV, dtype=torch.int32)
            s["at"] = torch.cat([torch.arange(t, device=DEV, dtype=torch.int32) + l for t, l in zip(toks, _lens(c))])
            s["pos"] = torch.arange(_cap(c), device=DEV, dtype=torch.int32).expand(c["seqs"], kv, -1).contiguous()
            s["len_out"] = torch.zeros_like(s["len"])
            s["q_out"] = torch.zeros(n, H, D, device=DEV, dtype=DT[c["cache"]])
        else:
            s["q"] = (1.5 * randn(n, H, D)).to(DT[c["q"]])
            s["len"] = torch.tensor([a + b for a, b in zip(_lens(c), toks)], device=DEV, dtype=torch.int32)
            s["out"] = torch.zeros(n, H, D, device=DEV, dtype=DT[c["q"]])
            s["lse"] = torch.zeros(n, H, device=DEV)
            s["ws"] = torch.zeros(192 << 20, device=DEV, dtype=torch.uint8)
    if "qkv" in s:
        s["xq"], s["xk"], s["xv"] = (s["qkv"][:, a:b].unflatten(1, (-1, D)) for a, b in ((0, H * D), (H * D, H * D + kv * D), (H * D + kv * D, (H + 2 * kv) * D)))
        s["w_q"], s["w_k"] = (1.0 + 0.2 * randn(D) if c["norm"] else None for _ in range(2))
    return s


# ------------------------------------------------------------------------------------------------- plain forms
def _angles(c):
    """(angle of one position for each pair, factor of the rotated elements), 64 bits"""
    r, sc = c["rot"], SCALING[c["scaling"]]
    i = torch.arange(r // 2, device=DEV, dtype=torch.float64)
    th = BASE ** (-2.0 * i / r)
    f = sc["factor"]
    if sc["kind"] == "linear":
        th = th / f
    elif sc["kind"] == "bands":   # slow pairs divided, fast ones kept, those between interpolated
        turns = sc["original"] * th / (2 * math.pi)
        keep = ((turns - sc["low"]) / (sc["high"] - sc["low"])).clamp(0, 1)
        th = keep * th + (1 - keep) * th / f
    elif sc["kind"] == "yarn":
        def pair(turns):
            return r * math.log(sc["original"] / (turns * 2 * math.pi)) / (2 * math.log(BASE))
        lo, hi = max(0, math.floor(pair(sc["high"]))), min(r - 1, math.ceil(pair(sc["low"])))
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return th / f * ramp + th * (1 - ramp), 0.1 * math.log(f) + 1
    return th, 1.0


def _turn(c, layout, x, at, w):
    """heads normed and rotated, in 32 bits"""
    x = x.float()
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    th, amp = _angles(c)
    t = at.double()[:, None] * th
    co, si = (amp * torch.cos(t)).float()[:, None], (amp * torch.sin(t)).float()[:, None]
    r = c["rot"]
    a, b = (x[..., :r // 2], x[..., r // 2:r]) if layout == "half" else (x[..., 0:r:2], x[..., 1:r:2])
    ya, yb = a * co - b * si, b * co + a * si
    y = torch.cat([ya, yb], -1) if layout == "half" else torch.stack([ya, yb], -1).flatten(-2)
    return torch.cat([y, x[..., r:]], -1)


def _rope(s):
    c = s["case"]
    s["q_out"].copy_(_turn(c, c["layout"], s["xq"], s["at"], s["w_q"]))
    s["k_out"].copy_(_turn(c, c["layout"], s["xk"], s["at"], s["w_k"]))
    return {"q": s["q_out"], "k": s["k_out"]}


def _slot_of_tokens(s):
    """(sequence, slot) of each new token of an append"""
    n = s["qkv"].shape[0]
    first = s["first"].long()
    seq = torch.bucketize(torch.arange(n, device=DEV), first[1:], right=True)
    return seq, s["len"].long()[seq] + torch.arange(n, device=DEV) - first[seq]


def _append(s):
    c = s["case"]
    s["q_out"].copy_(_turn(c, c["rope"], s["xq"], s["at"], s["w_q"]))
    seq, slot = _slot_of_tokens(s)
    page, place = s["pages"].long()[seq, slot // c["page"]], slot % c["page"]
    for name, new in (("k", _turn(c, c["rope"], s["xk"], s["at"], s["w_k"])), ("v", s["xv"])):
        pool = s[name].transpose(1, 2) if c["layout"] == "head" else s[name]
        pool[page, place] = new.to(pool.dtype)
    s["pos"].transpose(1, 2)[seq, slot] = s["at"][:, None].expand(-1, c["kv"])
    s["len_out"].copy_(s["len"] + s["first"][1:] - s["first"][:-1])
    return {"q": s["q_out"], "k": s["k"], "v": s["v"], "pos": s["pos"], "len": s["len_out"]}


def _slots(s, t, seq, n):
    """[kv, n, D] of a sequence, in 32 bits"""
    c = s["case"]
    t = t[s["pages"][seq, :-(-n // c["page"])].long()]
    t = t.transpose(0, 1) if c["layout"] == "head" else t.permute(2, 0, 1, 3)
    return t.flatten(1, 2)[:, :n].float()


def _attn(s):
    c = s["case"]
    kv, D, G = c["kv"], c["D"], c["heads"] // c["kv"]
    a = 0
    for i, (old, nt) in enumerate(zip(_lens(c), _tokens(c))):
        n = old + nt
        k, v = _slots(s, s["k"], i, n), _slots(s, s["v"], i, n)
        step = max(1, (1 << 30) // (c["heads"] * n))   # tokens at a time
        for b in range(0, nt, step):
            m = min(step, nt - b)
            q = s["q"][a + b:a + b + m].float().view(m, kv, G, D).permute(1, 2, 0, 3).reshape(kv, G * m, D)
            x = (torch.matmul(q, k.transpose(1, 2)) * D ** -0.5).view(kv, G, m, n)
            hidden = torch.arange(n, device=DEV) > (old + b + torch.arange(m, device=DEV))[:, None]
            x = x.masked_fill(hidden, -math.inf)
            top = x.amax(-1, keepdim=True)
            p = torch.exp(x - top)
            z = p.sum(-1, keepdim=True)
            o = torch.matmul((p / z).view(kv, G * m, n), v).view(kv, G, m, D)
            s["out"][a + b:a + b + m] = o.permute(2, 0, 1, 3).reshape(m, kv * G, D).to(s["out"].dtype)
            s["lse"][a + b:a + b + m] = (top + torch.log(z)).squeeze(-1).permute(2, 0, 1).reshape(m, kv * G)
        a += nt
    return {"out": s["out"], "lse": s["lse"]}


PLAIN = {"rope": _rope, "append": _append, "attn": _attn}


# ------------------------------------------------------------------------------------------------- the framework's calls
def _operator(s):
    """The framework's operator object for the state's buffers: kept by the program, as its buffers are."""
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pingala8-llm_amd"))
    import numpy as np
    import p8x
    c = s["case"]
    dt = {"f32": p8x.F32, "f16": p8x.F16, "bf16": p8x.BF16}
    ptr = {k: v.data_ptr() for k, v in s.items() if isinstance(v, torch.Tensor)}
    kv, D, H = c["kv"], c["D"], c["heads"]
    if c["op"] != "attn":
        sc = SCALING[c["scaling"]]
        kind = {"none": p8x.ROPE_PLAIN, "linear": p8x.ROPE_LINEAR, "bands": p8x.ROPE_BANDS, "yarn": p8x.ROPE_YARN}[sc["kind"]]
        freq, amplitude = p8x.rope_frequencies(c["rot"], BASE, kind, factor=sc["factor"], original=sc["original"], low=sc["low"], high=sc["high"])
        s["freq"] = torch.from_numpy(np.asarray(freq).view(np.int64)).to(DEV)
        layout = c["layout"] if c["op"] == "rope" else c["rope"]
        rot = p8x.Rotation(c["rot"], s["freq"].data_ptr(), layout=p8x.ROPE_HALF if layout == "half" else p8x.ROPE_PAIRS, amplitude=amplitude,
                           w_q=ptr.get("w_q"), w_k=ptr.get("w_k"), eps=EPS)
        ld = s["qkv"].shape[1]
        heads = dict(n_heads=H, q=ptr["xq"], q_dtype=dt[c["in"]], ld_q=ld, q_out=ptr["q_out"])
        if c["op"] == "rope":
            return p8x.Rope(rot, c["n"], D, ptr["at"], q_out_dtype=dt[c["out"]], n_kv=kv, k=ptr["xk"], k_dtype=dt[c["in"]], ld_k=ld, k_out=ptr["k_out"],
                            k_out_dtype=dt[c["out"]], **heads)
    st = s["k"].stride()
    cache = p8x.KvCache(
        dt[c["cache"]], c["seqs"], kv, D, k=ptr["k"], v=ptr["v"], page_stride=st[0], head_stride=st[1 if c["layout"] == "head" else 2],
        slot_stride=st[2 if c["layout"] == "head" else 1], page_size=c["page"], n_pages=s["k"].shape[0], pages=ptr["pages"],
        ld_pages=s["pages"].shape[1], len=ptr["len"], max_len=_cap(c))
    if c["op"] == "append":
        return p8x.KvAppendRope(cache, rot, at=ptr["at"], pos=ptr["pos"], len_out=ptr["len_out"], n_tokens=s["qkv"].shape[0], max_tokens=c["tokens"],
                                first=ptr["first"], k=ptr["xk"], v=ptr["xv"], kv_dtype=dt[c["in"]], ld_kv=ld, q_out_dtype=dt[c["cache"]], **heads)
    return p8x.AttnPrompt(cache, ptr["out"], out_dtype=dt[c["q"]], lse=ptr["lse"], workspace=ptr["ws"], workspace_bytes=s["ws"].numel(),
                          n_tokens=s["q"].shape[0], max_tokens=c["tokens"], first=ptr["first"], n_heads=H, q=ptr["q"], q_dtype=dt[c["q"]], scale=D ** -0.5)


def _results(s):
    return {"rope": lambda: {"q": s["q_out"], "k": s["k_out"]}, "attn": lambda: {"out": s["out"], "lse": s["lse"]},
            "append": lambda: {"q": s["q_out"], "k": s["k"], "v": s["v"], "pos": s["pos"], "len": s["len_out"]}}[s["case"]["op"]]()


def run(s):
    if not own:
        return PLAIN[s["case"]["op"]](s)
    if "call" not in s:
        s["call"] = _operator(s)
        s["result"] = _results(s)
    s["call"].run()
    return s["result"]


# ------------------------------------------------------------------------------------------------- bytes and operations
def work(case):
    c = case
    kv, D, H = c["kv"], c["D"], c["heads"]
    if c["op"] == "rope":
        n = c["n"] * (H + kv) * D
        return {"bytes": n * (SIZE[c["in"]] + SIZE[c["out"]]) + 4 * c["n"], "flops": (7.0 if c["norm"] else 3.0) * n}
    toks, lens = _tokens(c), _lens(c)
    if c["op"] == "append":
        n = sum(toks)
        return {"bytes": n * (D * ((H + 2 * kv) * (SIZE[c["in"]] + 2)) + 4 * kv + 4), "flops": (7.0 if c["norm"] else 3.0) * n * (H + kv) * D}
    b = sum(4 * kv * D * (l + t) + 2 * t * H * D * SIZE[c["q"]] + 4 * t * H for l, t in zip(lens, toks))
    return {"bytes": b, "flops": sum(4.0 * D * H * (t * l + t * (t + 1) / 2) for l, t in zip(lens, toks))}


# ------------------------------------------------------------------------------------------------- 64-bit results
def _exact_turn(c, layout, x, at, w):
    """by complex numbers: each pair times amplitude e^(i position theta)"""
    x = x.double()
    if w is not None:
        x = x / ((x ** 2).sum(-1, keepdim=True) / c["D"] + EPS).sqrt() * w.double()
    r, sc = c["rot"], SCALING[c["scaling"]]
    theta, amp = [], 1.0
    for i in range(r // 2):
        th = math.exp(-2 * i / r * math.log(BASE))
        if sc["kind"] == "linear":
            th /= sc["factor"]
        elif sc["kind"] == "bands":
            wave = 2 * math.pi / th
            if wave > sc["original"] / sc["low"]:
                th /= sc["factor"]
            elif wave > sc["original"] / sc["high"]:
                a = (sc["original"] / wave - sc["low"]) / (sc["high"] - sc["low"])
                th = (1 - a) * th / sc["factor"] + a * th
        elif sc["kind"] == "yarn":
            amp = 1 + math.log(sc["factor"]) / 10
            ends = [r / 2 * math.log(sc["original"] / (b * 2 * math.pi)) / math.log(BASE) for b in (sc["high"], sc["low"])]
            lo, hi = max(math.floor(ends[0]), 0), min(math.ceil(ends[1]), r - 1)
            a = min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001)))
            th = a * th / sc["factor"] + (1 - a) * th
        theta.append(th)
    turn = torch.polar(torch.full((), amp, device=DEV, dtype=torch.float64), at.double()[:, None] * torch.tensor(theta, device=DEV, dtype=torch.float64))[:, None]
    y = x.clone()
    i = torch.arange(r // 2, device=DEV)
    ia, ib = (i, i + r // 2) if layout == "half" else (2 * i, 2 * i + 1)
    z = torch.complex(x[..., ia], x[..., ib]) * turn
    y[..., ia], y[..., ib] = z.real, z.imag
    return y


def _exact_rope(s):
    c = s["case"]
    return {"q": _exact_turn(c, c["layout"], s["xq"], s["at"], s["w_q"]), "k": _exact_turn(c, c["layout"], s["xk"], s["at"], s["w_k"])}


def _exact_append(s):
    c = s["case"]
    k, v, pos = s["k"].double(), s["v"].double(), s["pos"].clone()
    kn, vn = _exact_turn(c, c["rope"], s["xk"], s["at"], s["w_k"]), s["xv"].double()
    first, lens = s["first"].tolist(), _lens(c)
    for i, old in enumerate(lens):
        for t in range(first[i], first[i + 1]):
            slot = old + t - first[i]
            page, place = int(s["pages"][i, slot // c["page"]]), slot % c["page"]
            for pool, new in ((k, kn), (v, vn)):
                (pool[page, :, place] if c["layout"] == "head" else pool[page, place])[:] = new[t]
            pos[i, :, slot] = s["at"][t]
    return {"q": _exact_turn(c, c["rope"], s["xq"], s["at"], s["w_q"]), "k": k, "v": v, "pos": pos,
            "len": torch.tensor([l + t for l, t in zip(lens, _tokens(c))], dtype=torch.int32)}


def _exact_attn(s):
    """one head after another, each token's softmax over the slots up to its own"""
    c = s["case"]
    G, page = c["heads"] // c["kv"], c["page"]
    out = torch.zeros(s["q"].shape, device=DEV, dtype=torch.float64)
    lse = torch.zeros(s["q"].shape[:2], device=DEV, dtype=torch.float64)
    first = s["first"].tolist()
    for i, n in enumerate(s["len"].tolist()):
        a, b = first[i], first[i + 1]
        slot = torch.arange(n, device=DEV)
        at = s["pages"][i].long()[slot // page]
        for h in range(c["kv"]):
            k, v = ((t[at, h, slot % page] if c["layout"] == "head" else t[at, slot % page, h]).double() for t in (s["k"], s["v"]))
            kt = k.t().contiguous()
            for g in range(h * G, h * G + G):
                for x0 in range(a, b, 4096):
                    x1 = min(b, x0 + 4096)
                    x = s["q"][x0:x1, g].double() @ kt / math.sqrt(c["D"])
                    own_slot = n - (b - a) + torch.arange(x0 - a, x1 - a, device=DEV)
                    x = torch.where(slot <= own_slot[:, None], x, -math.inf)
                    z = torch.logsumexp(x, 1)
                    lse[x0:x1, g] = z
                    out[x0:x1, g] = torch.exp(x - z[:, None]) @ v
    return {"out": out, "lse": lse}


def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "append": _exact_append, "attn": _exact_attn}[case["op"]](s)
