"""Tokens that are in the cache already, and their causal attention in 64 bits with bounds of its error, for the GPU tests of
p8x_attn_prompt.

Bounds. With A = sum_j w_j |v_j| of an output element (w the softmax weights):
  scores: head_dim products summed in f32 are off by at most (D + 8) 2^-24 sum_e |q_e k_e| scale, the parts of f32 queries by
    2^-21 of the same sum (two of 11 bits, sign apart; three of 8 bits are closer), and scaling, subtracting and the exponential by
    2^-22 |s| + 2^-21: an error of that size, relative, of each weight and once more of their sum;
  weights: rounded to u of themselves, 2^-11 (fp16) or 2^-8 (bf16) for 16-bit queries, 2^-22 or 2^-24 as sums of parts for f32
    ones; on an fp16 cache also to 2^-17 (2^-22) of the largest of 64 slots, which adds up to no more than that times 64 max|v|
    over all slots, as the largest weights of the tiles add up to 1 at most;
  sums: n terms in f32, (n + 64) 2^-24 A, numerator and denominator;
  the result: half a step of its type."""
import numpy as np

import p8x
from kvcase import BF16, F16, F32, Case, from_bits, half_ulp


class Prompt(Case):
    """lens: slots in use, the new tokens among them; toks: new tokens of each sequence, the last of their slots"""

    def __init__(self, lens, toks, out=None, **o):
        o.setdefault("fused", False)
        super().__init__(lens, toks, **o)
        self.out_t = self.qt if out is None else out

    def causal(self):
        """(out, lse, bound of out, bound of lse) [n][H][D], [n][H]"""
        out, tol = np.zeros((self.n, self.H, self.D)), np.zeros((self.n, self.H, self.D))
        lse, ltol = np.full((self.n, self.H), -np.inf), np.zeros((self.n, self.H))
        f32 = self.qt == F32
        uw = {(F16, False): 2.0 ** -11, (BF16, False): 2.0 ** -8, (F16, True): 2.0 ** -22, (BF16, True): 2.0 ** -24}[self.cache, f32]
        floor = 0.0 if self.cache == BF16 else 2.0 ** -22 if f32 else 2.0 ** -17
        for s in range(self.S):
            n, nt = self.lens[s], self.toks[s]
            there = np.array([self.there(s, j) for j in range(n)], bool)
            for h in range(self.kv):
                k, v = (from_bits(np.array([self.row(p, s, j)[h] if there[j] else np.zeros(self.D, np.uint16) for j in range(n)], np.uint16).reshape(n, self.D), self.cache)
                        for p in (self.kb, self.vb))
                if not n or not nt:
                    continue
                toks = slice(self.first[s], self.first[s] + nt)
                # [nt][slots] whether a token sees a slot
                see = there & (np.arange(n) <= (n - nt + np.arange(nt))[:, None])
                some = see.any(1)
                for head in range(h * self.G, (h + 1) * self.G):
                    q = from_bits(self.qb[toks, head], self.qt)
                    x = np.where(see, self.scale * (q @ k.T), -np.inf)
                    m = np.where(some, x.max(1), 0.0)
                    z = m + np.log(np.maximum(np.exp(x - m[:, None]).sum(1), 1e-300))
                    w = np.exp(x - z[:, None]) * some[:, None]
                    lse[toks, head] = np.where(some, z, -np.inf)
                    out[toks, head] = w @ v
                    a = w @ np.abs(v)
                    qk = abs(self.scale) * np.where(see, np.abs(q) @ np.abs(k).T, 0.0).max(1)
                    big = np.where(see, np.abs(x), 0.0).max(1)
                    es = ((self.D + 8) * 2.0 ** -24 + (2.0 ** -21 if f32 else 0)) * qk + 2.0 ** -22 * big + 2.0 ** -21
                    sums = (see.sum(1) + 64) * 2.0 ** -24
                    err = a * (uw + 2 * es + 2 * sums)[:, None] * 1.01 + floor * 64 * np.abs(v).max()
                    tol[toks, head] = err + half_ulp(self.out_t) * (np.abs(out[toks, head]) + err) + (2.0 ** -25 if self.out_t == F16 else 0)
                    ltol[toks, head] = es + sums + 2.0 ** -22 * (1 + np.abs(z))
        return out, lse, tol, ltol

    def run(self, workspace=None, lse=True, stream=None, call=None):
        """(out bits, lse): rows of no sequence hold 7s before"""
        if call is None:
            call = self.make(workspace, lse)
        call.run(stream)
        p8x.synchronize()
        return self.results(lse)

    def make(self, workspace=None, lse=True):
        npdt = self.npdt = np.float32 if self.out_t == F32 else np.uint16
        self.od = self.dev(np.full((self.n, self.H, self.D), 0x7E7E if npdt == np.uint16 else 7.0, npdt))
        self.ld_ = self.dev(np.full((self.n, self.H), 7.0, np.float32)) if lse else None
        kw = {} if workspace is None else dict(workspace=workspace) if workspace else dict(workspace=0, workspace_bytes=0)
        d = dict(n_tokens=self.n, max_tokens=self.tk, first=self.dev(self.first), n_heads=self.H, q=self.dev(self.qb), q_dtype=self.qt, scale=self.scale)
        return p8x.AttnPrompt(self.make_cache(), self.od, out_dtype=self.out_t, lse=self.ld_, **kw, **d)

    def results(self, lse=True):
        return self.od.to_numpy(self.npdt, (self.n, self.H, self.D)).copy(), self.ld_.to_numpy(np.float32, (self.n, self.H)).copy() if lse else None

    def check(self, out, lse):
        used = int(self.first[-1])
        ref, rl, tol, ltol = self.causal()
        got = from_bits(out, self.out_t)
        bad = ~(np.abs(got - ref) <= tol)[:used]
        assert not bad.any(), (np.argwhere(bad)[:4], np.nanmax((np.abs(got - ref) / np.maximum(tol, 1e-300))[:used]), np.nanmax(np.abs(got - ref)[:used]))
        if lse is not None:
            with np.errstate(invalid="ignore"):   # -inf - -inf
                same = (lse == rl) | (np.abs(lse - rl) <= ltol)
            assert same[:used].all(), (np.argwhere(~same[:used])[:4], lse[:used][~same[:used]][:4], rl[:used][~same[:used]][:4])
        assert (out[used:] == (7.0 if self.out_t == F32 else 0x7E7E)).all()   # rows of no sequence
        if lse is not None:
            assert (lse[used:] == 7.0).all()
