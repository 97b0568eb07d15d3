"""Greedy decoding with drafted tokens on a cache of bounded size: the calls between the linears as a decode step uses them.

A transformer with random Pingala-8 weights (each layer: norm -> q, k, v, with --rope-base rotated by their positions -> attention of
the drafted tokens -> o -> norm -> gate, up, silu -> down; norms before and after each block) decodes one sequence. Every step runs a small
tree of tokens -- the last one and guesses of what follows, looked up from earlier occurrences -- through all layers at
once (p8x_norm_residual, p8x_mul_mat_vec, p8x_rope, p8x_attn_tree), keeps the path that the model itself would have taken, adds what it
attended to to the slots' scores (p8x_kv_score), stores its keys and values (p8x_kv_append) and cuts the cache to its budget
(p8x_kv_evict: the first positions, the last ones and the highest scores stay).

    python -m p8x.tree_decode [--layers 4] [--tokens 96] [--budget 64] [--drafts 8] [--rope-base 10000]

prints tokens, steps and milliseconds a step (calls enqueued one by one; the host chooses between steps).
"""
import argparse
import time

import numpy as np

import p8x

MAX_COLUMNS = 8   # of p8x_mul_mat_vec: tokens of a step


class Model:
    """random weights: hidden and ffn multiples of 256, vocabulary a multiple of 32; rope_base 0: positions are not rotated in"""

    def __init__(self, layers=4, hidden=512, heads=4, kv=2, head_dim=128, ffn=1024, vocab=512, seed=0, rope_base=0.0):
        self.hidden, self.heads, self.kv, self.D, self.ffn, self.vocab = hidden, heads, kv, head_dim, ffn, vocab
        rng = np.random.default_rng(seed)
        self.embedding = rng.standard_normal((vocab, hidden)).astype(np.float32)

        def linears(K, **rows):   # of one input
            shapes = [(r, K) for r in rows.values()]
            slots = [p8x.synth_random(int(rng.integers(1, 1 << 31)), r, K) for r, _ in shapes]
            p8x.share_input(slots, shapes)
            return {name: p8x.Tensor(slot, r, K) for name, slot, (r, _) in zip(rows, slots, shapes)}
        qd, kvd = heads * head_dim, kv * head_dim
        self.layers = [{**linears(hidden, q=qd, k=kvd, v=kvd), **linears(qd, o=hidden), **linears(hidden, gate=ffn, up=ffn), **linears(ffn, down=hidden)}
                       for _ in range(layers)]
        self.head = linears(hidden, head=vocab)["head"]
        self.one = p8x.DeviceBuffer.from_numpy(np.ones(hidden, np.float32))
        self.rotation = None
        if rope_base:
            freq, amplitude = p8x.rope_frequencies(head_dim, rope_base)
            self.rotation = p8x.Rotation(head_dim, p8x.DeviceBuffer.from_numpy(freq), amplitude=amplitude)
        # a norm that puts the products of random weights to the size that the next step expects
        self.half = p8x.DeviceBuffer.from_numpy(np.full(hidden, 0.5, np.float32))


class Decoder:
    """One sequence: forward(tokens, parents) -> logits of every token, then keep(path) of the same tokens."""

    def __init__(self, model, budget, n_sink=4, n_recent=16, page=64, decay=0.98):
        m = self.model = model
        if budget < n_sink + n_recent:
            raise ValueError("budget below n_sink + n_recent")
        self.budget, self.length, self.position = budget, 0, 0
        n, dev = MAX_COLUMNS, p8x.DeviceBuffer
        max_len = self.max_len = budget + n
        pages = -(-max_len // page)
        self.table = dev.from_numpy(np.random.default_rng(0).permutation(pages).astype(np.int32))   # in no order
        self.first, self.mask, self.at, self.accept = dev(8), dev(8 * n), dev(4 * n), dev(8)
        self.h, self.x, self.y = dev(4 * n * m.hidden), dev(4 * n * m.hidden), dev(4 * n * m.hidden)
        self.ld = (m.heads + 2 * m.kv) * m.D
        self.act, self.ff, self.logits = dev(4 * n * m.heads * m.D), dev(4 * n * m.ffn), dev(4 * n * m.vocab)
        self.layers = []
        for i in range(len(m.layers)):
            k, v = dev(2 * pages * page * m.kv * m.D), dev(2 * pages * page * m.kv * m.D)
            length, score, pos = dev(4), dev(4 * m.kv * max_len), dev(4 * m.kv * max_len)
            length.fill(0)
            cache = p8x.KvCache(p8x.F16, 1, m.kv, m.D, k, v, page_stride=page * m.kv * m.D, head_stride=page * m.D, slot_stride=m.D, page_size=page,
                                n_pages=pages, len=length, max_len=max_len, pages=self.table, ld_pages=pages)
            qkv, lse = dev(4 * n * self.ld), dev(4 * n * m.heads)
            self.layers.append(dict(cache=cache, qkv=qkv, lse=lse, score=score, pos=pos, len=length,
                                    evict=p8x.KvEvict(cache, budget, score, length, pos=pos, n_sink=n_sink, n_recent=n_recent)))
        self.decay = decay
        self.calls = {}   # of a number of tokens

    def _norm(self, n, y=None):
        """the residual plus a normed block output, and the next block's input"""
        m = self.model
        return p8x.NormResidual(n, m.hidden, self.h, y=y, h_out=None if y is None else self.h, x=self.x, post=p8x.NORM_NONE if y is None else p8x.NORM_RMS,
                                w_post=None if y is None else m.half, w_pre=m.one)

    def _plan(self, n):
        m, out = self.model, []
        for L in self.layers:
            at = L["qkv"].addr
            d = dict(n_tokens=n, max_tokens=n, first=self.first, q=at, k=at + 4 * m.heads * m.D, v=at + 4 * (m.heads + m.kv) * m.D, ld_q=self.ld,
                     ld_kv=self.ld, mask=self.mask, n_heads=m.heads, scale=m.D ** -0.5)
            rope = None if m.rotation is None else p8x.Rope(m.rotation, n, m.D, self.at, n_heads=m.heads, q=at, ld_q=self.ld, n_kv=m.kv,
                                                            k=d["k"], ld_k=self.ld)   # in place
            out.append(dict(rope=rope, attn=p8x.AttnTree(L["cache"], self.act, lse=L["lse"], **d),
                            score=p8x.KvScore(L["cache"], L["lse"], L["score"], accept=self.accept, decay=self.decay, **d),
                            append=p8x.KvAppend(L["cache"], accept=self.accept, at=self.at, pos=L["pos"], len_out=L["len"], **d)))
        return dict(layers=out, start=self._norm(n), add=self._norm(n, self.y))

    def forward(self, tokens, parents, stream=None):
        """tokens[0] follows the cache; parents[i] < i is the token that token i follows (-1: the cache)"""
        m, n = self.model, len(tokens)
        if not 0 < n <= MAX_COLUMNS:
            raise ValueError(f"1 .. {MAX_COLUMNS} tokens a step")
        self.n, self.depth, masks = n, [], []
        for i, p in enumerate(parents):
            masks.append((masks[p] if p >= 0 else 0) | 1 << i)
            self.depth.append(self.depth[p] + 1 if p >= 0 else self.position)
        for buf, a in ((self.h, m.embedding[list(tokens)]), (self.first, np.array([0, n], np.int32)), (self.mask, np.array(masks, np.uint64)),
                       (self.at, np.array(self.depth, np.int32))):
            p8x.hip_check(p8x.hip().hipMemcpy(buf.addr, a.ctypes.data, a.nbytes, p8x.H2D), "copy")
        if n not in self.calls:
            self.calls[n] = self._plan(n)
        c = self.calls[n]
        c["start"].run(stream)
        for L, call, w in zip(self.layers, c["layers"], m.layers):
            at = L["qkv"].addr
            for name, off in (("q", 0), ("k", m.heads * m.D), ("v", (m.heads + m.kv) * m.D)):
                w[name].mul_mat_vec_dev(self.x, at + 4 * off, n, ldy=self.ld, stream=stream)
            if call["rope"]:
                call["rope"].run(stream)
            call["attn"].run(stream)
            w["o"].mul_mat_vec_dev(self.act, self.y, n, stream=stream)
            c["add"].run(stream)
            for i in range(n):
                p8x.mul_mat_vec_glu_dev(w["gate"], w["up"], self.x.addr + 4 * i * m.hidden, self.ff.addr + 4 * i * m.ffn, stream=stream)
            w["down"].mul_mat_vec_dev(self.ff, self.y, n, stream=stream)
            c["add"].run(stream)
        m.head.mul_mat_vec_dev(self.x, self.logits, n, stream=stream)
        if stream:
            stream.sync()
        p8x.synchronize()
        return self.logits.to_numpy(np.float32, (MAX_COLUMNS, m.vocab))[:n]

    def keep(self, path, stream=None):
        """the tokens of the last forward() that are decoded now: cached, and the cache cut to its budget"""
        bits = np.array([sum(1 << i for i in path)], np.uint64)
        p8x.hip_check(p8x.hip().hipMemcpy(self.accept.addr, bits.ctypes.data, 8, p8x.H2D), "copy")
        for L, call in zip(self.layers, self.calls[self.n]["layers"]):
            call["score"].run(stream)
            call["append"].run(stream)
            L["evict"].run(stream)
        if stream:
            stream.sync()
        self.position += len(path)
        self.length = min(self.budget, self.length + len(path))

    def prompt(self, tokens):
        """logits after the last of tokens"""
        for i in range(0, len(tokens), MAX_COLUMNS):
            part = tokens[i:i + MAX_COLUMNS]
            out = self.forward(part, range(-1, len(part) - 1))
            self.keep(range(len(part)))
        return out[-1]


def guess(known, limit):
    """a tree of guesses: the last token and what followed its (and its predecessor's) earlier occurrences"""
    tokens, parents = [known[-1]], [-1]
    for i in range(len(known) - 2, -1, -1):
        if known[i] != known[-1]:
            continue
        at = 0
        for t in known[i + 1:i + limit]:
            same = [j for j in range(len(tokens)) if parents[j] == at and tokens[j] == t]
            if not same:
                if len(tokens) == limit:
                    return tokens, parents
                tokens.append(t)
                parents.append(at)
                same = [len(tokens) - 1]
            at = same[0]
    return tokens, parents


def generate(decoder, prompt, count, drafts=MAX_COLUMNS, propose=guess):
    """(tokens, steps): `count` greedy tokens after the prompt, with trees of at most `drafts` tokens"""
    out, steps = [int(np.argmax(decoder.prompt(prompt)))], 0
    while len(out) < count:
        tokens, parents = propose(list(prompt) + out, drafts)
        best = np.argmax(decoder.forward(tokens, parents), axis=1)
        path, steps = [0], steps + 1
        while True:   # the child that is the model's own next token
            out.append(int(best[path[-1]]))
            follow = [j for j in range(len(tokens)) if parents[j] == path[-1] and tokens[j] == out[-1]]
            if not follow:
                break
            path.append(follow[0])
        decoder.keep(path)
    return out[:count], steps


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    for name, value in dict(layers=4, hidden=512, heads=4, kv=2, head_dim=128, ffn=1024, vocab=512, tokens=96, budget=64, drafts=8, seed=0).items():
        ap.add_argument("--" + name.replace("_", "-"), type=int, default=value)
    ap.add_argument("--rope-base", type=float, default=0.0)
    a = ap.parse_args()
    model = Model(a.layers, a.hidden, a.heads, a.kv, a.head_dim, a.ffn, a.vocab, a.seed, a.rope_base)
    prompt = np.random.default_rng(a.seed).integers(0, a.vocab, 20).tolist()
    for drafts in (1, a.drafts):
        d = Decoder(model, a.budget)
        t = time.perf_counter()
        out, steps = generate(d, prompt, a.tokens, drafts)
        ms = (time.perf_counter() - t) * 1e3
        print(f"{drafts} tokens a step at most: {len(out)} tokens in {steps} steps, {ms / steps:.2f} ms a step (prompt included), "
              f"cache {d.length} of {d.position} positions", flush=True)


if __name__ == "__main__":
    main()
