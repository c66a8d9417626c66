"""64-bit references of the 4-bit paged cache's operators, from their definitions."""
from __future__ import annotations

import math

import torch

CODES = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def rope(x, pos, cos, sin, w, eps):
    """(fp64 result, what bounds its fp32 error: |y_i| + |y_(i + D/2)|) of rows x (T, H, D)."""
    y = x.double()
    if w is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    a, b = y.chunk(2, -1)
    p = pos.long().clamp(0, cos.shape[0] - 1)
    c, s = cos.double()[p][:, None], sin.double()[p][:, None]
    out = torch.cat([a * c - b * s, b * c + a * s], -1)
    out = torch.where((pos < 0)[:, None, None], 0.0, torch.where((pos >= cos.shape[0])[:, None, None], math.nan, out))
    return out, (a.abs() + b.abs()).repeat(1, 1, 2)


def quantise(x):
    """(codes, scale bytes) of values x (..., D): every code's distance in 64 bits."""
    b = x.double().unflatten(-1, (-1, 32))
    fine = torch.isfinite(b).all(-1)
    b = torch.where(fine[..., None], b, 0.0)
    top = b.abs().amax(-1)
    e = torch.full_like(top, -125)
    for k in range(-125, 125):                              # the smallest 2^e with top < 7 * 2^e, at most 2^125
        e = torch.where(top >= 7 * 2.0 ** k, float(k + 1), e)
    y = b.abs() / torch.exp2(e)[..., None]
    d = (y[..., None] - CODES.to(x.device)).abs()
    near = d.amin(-1, keepdim=True)
    tie = d == near
    even = torch.tensor([0, 2, 4, 6, 1, 3, 5, 7], device=x.device)        # the even code of a tie
    c = even[tie[..., even].int().argmax(-1)]
    c = c + 8 * torch.signbit(x.unflatten(-1, (-1, 32))).long()
    c = torch.where(fine[..., None], c, 0).flatten(-2)
    return (c[..., 0::2] + 16 * c[..., 1::2]).byte(), torch.where(fine, e + 127, 255.0).byte()


def values(c, s):
    c = torch.stack([c & 15, c >> 4], -1).flatten(-2).long()
    x = CODES.to(c.device)[c & 7] * (1 - 2 * (c >> 3))
    f = torch.where(s == 255, math.nan, torch.exp2(s.double() - 127))
    return (x.unflatten(-1, (-1, 32)) * f[..., None]).flatten(-2)


def rows_at(codes, scales, slots):
    """fp64 values (T, HKV, D) at slots of cache tensors."""
    page = codes.shape[2]
    p, o = slots.long() // page, slots.long() % page
    return values(codes[p, :, o], scales[p, :, o])


def attn(q, k, v, n, scale, weight=2.0 ** -16):
    """One sequence: q (R, HQ, D) the newest tokens of k, v (n, HKV, D) fp64.  Returns the fp64 output
    and the fp32 kernel's error bound beside the output's own rounding: sums of D exact products (each
    sum off by D 2^-24 of its terms' sizes, as a score and once more in the maximum), weights rounded
    to `weight` of themselves (two bf16 terms 2^-16; fp16, for more than 64 rows of a KV head, 2^-11), exponentials and sums over n keys ((n + 64) 2^-24); and what fp32 does not hold:
    a weight, or its second term, under 2^-126 counts as 0, so that each key may be off by 2^-125 |v|; fp16
    weights are kept times 2^7, those under 2^-21 of the largest to half of 2^-24 / 2^7: 2^-32 |v|."""
    R, HQ, D = q.shape
    HKV = k.shape[1]
    G = HQ // HKV
    out = torch.zeros(R, HQ, D, dtype=torch.float64, device=q.device)
    err = torch.zeros_like(out)
    for j in range(R):
        m = n - R + j + 1
        if m <= 0:
            continue
        x = q[j].double().view(HKV, G, D)
        kk, vv = k[:m].transpose(0, 1), v[:m].transpose(0, 1)
        w = torch.softmax((x[:, :, None] * kk[:, None]).sum(-1) * scale, -1)
        size = (x.abs()[:, :, None] * kk.abs()[:, None]).sum(-1).amax(-1) * abs(scale)
        out[j] = torch.matmul(w, vv).reshape(HQ, D)
        a = torch.matmul(w, vv.abs()).reshape(HQ, D)
        err[j] = a * (2 * size.reshape(HQ, 1) * (D + 4) * 2.0 ** -24 + weight + (m + 64) * 2.0 ** -24)
        err[j] += (2.0 ** -32 if weight > 2.0 ** -16 else 2.0 ** -125) * vv.abs().sum(1).repeat_interleave(G, 0)
    return out, err


def held(table, lens, page):
    """slots of every token of every sequence"""
    out = []
    for row, n in zip(table.tolist(), lens):
        ids = torch.tensor(row[:-(-n // page)], dtype=torch.long)
        t = torch.arange(n)
        out.append(ids[t // page] * page + t % page if n else t)
    return out


class Pool:
    """The page pool on the host, request by request."""

    def __init__(self, lens, table, free, nfree, page):
        self.lens, self.table, self.page = list(lens), [list(r) for r in table], page
        self.free, self.nfree, self.status = list(free), nfree, 0

    def pages(self, n):
        return -(-n // self.page)

    def extend(self, add, total):
        width = len(self.table[0])
        need = [self.pages(n + a) - self.pages(n) if a >= 0 else 0 for n, a in zip(self.lens, add)]
        bad = 0
        if any(a < 0 or n + a > width * self.page or n < 0 for n, a in zip(self.lens, add)):
            bad |= 1
        ok = [a if not (a < 0 or n + a > width * self.page or n < 0) else 0 for n, a in zip(self.lens, add)]
        need = [self.pages(n + a) - self.pages(n) for n, a in zip(self.lens, ok)]
        bad |= 2 * (sum(need) > self.nfree) | 4 * (sum(ok) > total)
        if bad:
            self.status |= bad
            return [-1] * total, [-1] * total, [0] * (len(add) + 1)
        slots, pos, cu = [], [], [0]
        for i, a in enumerate(add):
            for p in range(self.lens[i], self.lens[i] + a):
                if p % self.page == 0:
                    self.nfree -= 1
                    self.table[i][p // self.page] = self.free[self.nfree]
                slots.append(self.table[i][p // self.page] * self.page + p % self.page)
                pos.append(p)
            self.lens[i] += a
            cu.append(len(slots))
        pad = [-1] * (total - len(slots))
        return slots + pad, pos + pad, cu

    def truncate(self, keep):
        gone = []
        lens = list(self.lens)
        for i, k in enumerate(keep):
            n = self.lens[i] if k < 0 else min(k, self.lens[i])
            gone += [(i, c) for c in range(self.pages(n), self.pages(self.lens[i]))]
            lens[i] = n
        if self.nfree + len(gone) > len(self.free):
            self.status |= 2
            return
        for r, (i, c) in enumerate(gone):
            self.free[self.nfree + len(gone) - 1 - r] = self.table[i][c]
            self.table[i][c] = -1
        self.nfree += len(gone)
        self.lens = lens
