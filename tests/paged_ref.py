"""Inputs and 64-bit results for the paged-cache operators' tests (numpy and torch on the CPU)."""
import math

import numpy as np
import torch

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
U = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}      # half a step, relative
TINY = {"f16": 2.0 ** -25, "bf16": 2.0 ** -134, "f32": 2.0 ** -150}   # half a subnormal step


class Batch:
    """Sequences of lens = [(new tokens, keys in all)], their pages scattered over a cache whose other
    slots hold `stale` (NaN by default: what a row does not see must have no effect)."""

    def __init__(self, seed, lens, nh, nkv, hd, page, t, cols=None, spare=3, stale=float("nan"), tail=0, unused=-1,
                 page_pad=0, v_scale=1.0, q_scale=2.0):
        rng = np.random.default_rng(seed)
        self.lens, self.nh, self.nkv, self.hd, self.page, self.t = lens, nh, nkv, hd, page, t
        self.B, self.G = len(lens), nh // nkv
        need = [-(-max(tot, 0) // page) for _, tot in lens]
        self.cols = cols or max(need + [1])
        self.n_pages = sum(need) + spare
        ids = rng.permutation(self.n_pages)
        self.table = np.full((self.B, self.cols), unused, np.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :min(n, self.cols)] = ids[at:at + n][:self.cols]
            at += n
        self.new = [n for n, _ in lens]
        self.seq_start = np.concatenate([[0], np.cumsum(self.new)]).astype(np.int32)
        self.kv_len = np.array([tot for _, tot in lens], np.int32)
        self.T = int(self.seq_start[-1])
        self.tokens = self.T + tail          # rows behind the last sequence
        shape = (self.n_pages, nkv, page, hd)
        self.kc = torch.full(shape, stale, dtype=DT[t])
        self.vc = torch.full(shape, stale, dtype=DT[t])
        self.K, self.V = [], []              # what the sequences hold, [keys][nkv][hd] of the cache's type
        for b in range(self.B):
            n = max(int(self.kv_len[b]), 0)
            self.K.append(torch.from_numpy(rng.standard_normal((n, nkv, hd)).astype(np.float32)).to(DT[t]))
            self.V.append(torch.from_numpy((rng.standard_normal((n, nkv, hd)) * v_scale).astype(np.float32)).to(DT[t]))
        self.q = torch.from_numpy((rng.standard_normal((self.tokens, nh, hd)) * q_scale).astype(np.float32)).to(DT[t])
        self.page_pad = page_pad
        self.write()

    def write(self):
        """Put K and V into the pages."""
        for b in range(self.B):
            for c in range(self.cols):
                pg = int(self.table[b, c])
                if 0 <= pg < self.n_pages:
                    k0 = c * self.page
                    k1 = min(k0 + self.page, self.K[b].shape[0])
                    if k1 > k0:
                        self.kc[pg, :, :k1 - k0] = self.K[b][k0:k1].transpose(0, 1)
                        self.vc[pg, :, :k1 - k0] = self.V[b][k0:k1].transpose(0, 1)

    def device(self, gpu):
        """The batch on the GPU: a PagedKV handle and its tensors."""
        def cache(x):
            if not self.page_pad:
                return x.cuda()
            flat = torch.full((self.n_pages, x[0].numel() + self.page_pad), float("nan"), dtype=x.dtype, device="cuda")
            view = flat.as_strided(x.shape, (flat.shape[1],) + x.stride()[1:])
            view.copy_(x)
            return view
        self.dkc, self.dvc = cache(self.kc), cache(self.vc)
        self.dtable = torch.from_numpy(self.table).cuda()
        self.dss = torch.from_numpy(self.seq_start).cuda()
        self.dlen = torch.from_numpy(self.kv_len).cuda()
        self.kv = gpu.PagedKV(self.dkc, self.dvc, self.dtable, self.dss, self.dlen)
        return self.kv

    def visible(self, b, i, window=0, prefix=None):
        """Key indexes that row i of sequence b sees."""
        total = int(self.kv_len[b])
        p = total - self.new[b] + i
        hi = max(p + 1, 0 if prefix is None else int(prefix[b]))
        hi = min(hi, total, self.cols * self.page)
        lo = max(0, p - window + 1) if window else 0
        j = np.arange(lo, max(lo, hi))
        ok = (self.table[b, j // self.page] >= 0) & (self.table[b, j // self.page] < self.n_pages) if len(j) else j > 0
        return j[ok]

    def attn(self, scale, window=0, prefix=None):
        """out [T][nh][hd], lse [T][nh] in 64 bits, and how far fp32 accumulation with probabilities
        rounded to the cache's type may be off (out, lse), from the counts of the roundings."""
        out = np.zeros((self.T, self.nh, self.hd))
        lse = np.full((self.T, self.nh), -math.inf)
        dout, dlse = np.zeros_like(out), np.zeros_like(lse)
        for b in range(self.B):
            Kb, Vb = self.K[b].double().numpy(), self.V[b].double().numpy()
            for i in range(self.new[b]):
                r = int(self.seq_start[b]) + i
                j = self.visible(b, i, window, prefix)
                if not len(j):
                    continue
                for g in range(self.nkv):
                    hs = slice(g * self.G, (g + 1) * self.G)
                    q = self.q[r, hs].double().numpy()
                    s = q @ Kb[j, g].T * scale                                   # [G][keys]
                    m = s.max(-1, keepdims=True)
                    e = np.exp(s - m)
                    z = e.sum(-1, keepdims=True)
                    out[r, hs] = (e / z) @ Vb[j, g]
                    lse[r, hs] = (m + np.log(z))[:, 0]
                    # scores: hd products summed in fp32, times scale, as a power of two's exponent
                    mag = (np.abs(q) @ np.abs(Kb[j, g]).T).max(-1, keepdims=True) * scale
                    es = 2.0 ** -24 * ((self.hd + 4) * mag + 4 * np.abs(s).max(-1, keepdims=True) + 8)
                    n = len(j)
                    A = (e / z) @ np.abs(Vb[j, g])
                    # probabilities: half a step each, below the type's normal range half a subnormal step
                    sub = TINY[self.t] * np.abs(Vb[j, g]).sum(0) / z
                    dout[r, hs] = A * (U[self.t] + 2 * es + 2.0 ** -24 * (2 * n + 24)) * 1.01 + sub
                    dlse[r, hs] = (es + 2.0 ** -24 * (n + 16 + 4 * np.abs(lse[r, hs])[:, None]))[:, 0]
        return out, lse, dout, dlse


def rounding(x, t):
    """Half a step of type t at x."""
    return np.maximum(np.abs(x) * U[t], TINY[t])


def rope_tables(rows, rot, seed=None):
    half = rot // 2
    if seed is None:
        ang = np.arange(rows)[:, None] * 10000.0 ** (-np.arange(half) / half)
    else:
        ang = np.random.default_rng(seed).uniform(-4, 4, (rows, half))
    return torch.from_numpy(np.cos(ang).astype(np.float32)), torch.from_numpy(np.sin(ang).astype(np.float32))


def rotate(x, cos, sin, pos, pairs):
    """x [T][heads][hd] in 64 bits rotated to pos [T], and the bound of fp32's errors in it."""
    c, s = cos.double().numpy()[pos][:, None], sin.double().numpy()[pos][:, None]
    rot = 2 * c.shape[-1]
    y, d = x.copy(), np.zeros_like(x)
    i, j = (slice(0, rot, 2), slice(1, rot, 2)) if pairs else (slice(0, rot // 2), slice(rot // 2, rot))
    a, b = x[..., i], x[..., j]
    y[..., i], y[..., j] = a * c - b * s, b * c + a * s
    d[..., i] = d[..., j] = 2.0 ** -23 * (np.abs(a) + np.abs(b)) * np.maximum(np.abs(c), np.abs(s))
    return y, d
