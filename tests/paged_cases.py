"""Paged caches, batches and their 64-bit reference results for the
paged-cache operator tests."""
import math
import random

import numpy as np
import torch

BF16 = torch.bfloat16
NAN_BITS = 0x7FC0  # what rows that no position covers hold


def bf16(x):
    return torch.as_tensor(x, dtype=torch.float32).to(BF16)


def quantize(x, bits):
    """x [..., dim] float32 -> codes, scale, bias (bf16) by the affine rule (group 64), in float32 as the cache does."""
    g = x.float().unflatten(-1, (-1, 64))
    lo, hi = g.amin(-1), g.amax(-1)
    s = torch.from_numpy((hi - lo).numpy() / np.float32((1 << bits) - 1)).to(BF16)
    s = torch.where(s == 0, torch.ones_like(s), s)
    b = lo.to(BF16)
    q = torch.from_numpy(np.rint((g - b.float()[..., None]).numpy() / s.float()[..., None].numpy()))
    return q.clamp(0, (1 << bits) - 1).flatten(-2).to(torch.uint8), s, b


def pack(q, bits):
    return q.clone() if bits == 8 else q[..., 0::2] | (q[..., 1::2] << 4)


def unpack(p, bits):
    return p if bits == 8 else torch.stack((p & 15, p >> 4), -1).flatten(-2)


def values(p, s, b, bits):
    """The values of packed codes in 64 bits."""
    g = unpack(p, bits).double().unflatten(-1, (-1, 64))
    return (g * s.double()[..., None] + b.double()[..., None]).flatten(-2)


class Cache:
    """A pool of pages on the host and the device, and a batch over it.  lens: (new, rows including them) per
    sequence.  Rows at and past a sequence's rows, and pages of nobody, hold NaN (or the largest codes and NaN scales).
    gap: rows between pages; pad: packed token rows past the batch's; spare: table entries past a sequence's pages."""

    def __init__(self, seed, lens, kv_heads, dim, bits, page, gap=0, pad=0, spare=2, k_std=1.0):
        gen = torch.Generator().manual_seed(seed)
        self.lens, self.hk, self.dim, self.bits, self.page = lens, kv_heads, dim, bits, page
        blocks = [-(-max(n, 0) // page) for _, n in lens]
        self.pages = sum(blocks) + 2
        order = list(range(self.pages))
        random.Random(seed).shuffle(order)
        self.stride = kv_heads * page + gap
        width = max(blocks, default=0) + spare
        self.table = torch.full((len(lens), width), -1, dtype=torch.int32)
        for i, n in enumerate(blocks):
            self.table[i, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
        self.start = [0]
        for n, _ in lens:
            self.start.append(self.start[-1] + n)
        self.tokens = self.start[-1] + pad
        self.rows = {}  # (k or v): per sequence, 64-bit [rows][hk][dim]
        shape = (self.pages * self.stride, dim)
        self.pool = {}
        for n in "kv":
            if bits == 16:
                full = torch.full(shape, NAN_BITS, dtype=torch.int16).view(BF16)
                self.pool[n] = full
            else:
                self.pool[n] = torch.full((shape[0], dim * bits // 8), 255, dtype=torch.uint8)
                for w in "sb":
                    self.pool[n + w] = torch.full((shape[0], dim // 64), NAN_BITS, dtype=torch.int16).view(BF16)
            self.rows[n] = []
            for i, (_, m) in enumerate(lens):
                x = (torch.randn((max(m, 0), kv_heads, dim), generator=gen) * (k_std if n == "k" else 1.0)).to(BF16)
                at = self.at(i, torch.arange(max(m, 0)))
                if bits == 16:
                    self.pool[n][at] = x
                    self.rows[n].append(x.double())
                else:
                    q, s, b = quantize(x.float(), bits)
                    self.pool[n][at], self.pool[n + "s"][at], self.pool[n + "b"][at] = pack(q, bits), s, b
                    self.rows[n].append(values(pack(q, bits), s, b, bits))
        self.gen = gen

    def at(self, seq, pos):
        """Pool rows [len(pos)][hk] of positions of one sequence."""
        page = self.table[seq][pos // self.page].long()
        return page[:, None] * self.stride + torch.arange(self.hk) * self.page + (pos % self.page)[:, None]

    def device(self, lmx, zero_stride=False):
        """(kv, batch) descriptors over device copies (kept alive on self)."""
        self.dev = {n: t.cuda() for n, t in self.pool.items()}
        d = {n: t.data_ptr() for n, t in self.dev.items()}
        stride = 0 if zero_stride else self.stride
        if self.bits == 16:
            kv = lmx.PagedKvDesc(self.pages, self.page, self.hk, self.dim, 16, stride, d["k"], d["v"])
        else:
            kv = lmx.PagedKvDesc(self.pages, self.page, self.hk, self.dim, self.bits, stride, None, None, d["k"], d["v"],
                                 d["ks"], d["kb"], d["vs"], d["vb"])
        self.index = [torch.tensor(self.start, dtype=torch.int32).cuda(),
                      torch.tensor([n for _, n in self.lens], dtype=torch.int32).cuda(), self.table.cuda()]
        batch = lmx.PagedBatch(len(self.lens), self.tokens, max([n for n, _ in self.lens], default=0),
                               self.index[0].data_ptr(), self.index[1].data_ptr(), self.index[2].data_ptr(),
                               self.table.shape[1])
        return kv, batch


def attention(cache, q, scale, window):
    """64-bit out [tokens][heads][dim], lse [tokens][heads], and per output the sums that its error scales with:
    A = sum_j p_j |v_j| (elementwise) and Q = max_j scale sum_d |q_d k_jd| (per row)."""
    n, heads, dim = q.shape
    g = heads // cache.hk
    out = torch.zeros(n, heads, dim, dtype=torch.float64)
    A, Q = torch.zeros_like(out), torch.zeros(n, heads, dtype=torch.float64)
    lse = torch.full((n, heads), -math.inf, dtype=torch.float64)
    for i, (new, rows) in enumerate(cache.lens):
        k, v = cache.rows["k"][i], cache.rows["v"][i]
        for t in range(new):
            pos = rows - new + t
            lo = max(0, pos - window + 1) if window else 0
            if pos < 0:
                continue
            at = cache.start[i] + t
            x = q[at].double().view(cache.hk, g, dim)
            z = torch.einsum("hgd,jhd->hgj", x, k[lo:pos + 1]) * scale
            Q[at] = (torch.einsum("hgd,jhd->hgj", x.abs(), k[lo:pos + 1].abs()) * scale).amax(-1).flatten()
            p = torch.softmax(z, -1)
            lse[at] = torch.logsumexp(z, -1).flatten()
            out[at] = torch.einsum("hgj,jhd->hgd", p, v[lo:pos + 1]).reshape(heads, dim)
            A[at] = torch.einsum("hgj,jhd->hgd", p, v[lo:pos + 1].abs()).reshape(heads, dim)
    return out, lse, A, Q


def device_error(lmx):
    import ctypes as C
    code = C.c_uint(0)
    lmx.call("lmx_device_error", C.byref(code), 1)
    return code.value
