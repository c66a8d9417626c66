"""64-bit references of the 8-bit paged cache's operators, from their definitions."""
from __future__ import annotations

import math

import torch


def _e4m3():
    c = torch.arange(256)
    e, m = c // 8 % 16, (c % 8).double()
    x = torch.where(e == 0, m / 8 * 2.0 ** -6, (1 + m / 8) * torch.exp2(e.double() - 7))
    return torch.where(c % 128 == 127, math.nan, x * (1 - 2 * (c // 128)))


CODES = _e4m3()                                             # the value of each code; 126 is the largest, 448
MIDDLES = (CODES[:126] + CODES[1:127]) / 2


def codes_of(y):
    """Codes nearest to y (fp64, at most 448 in size), ties to the even one; NaN: 0x7f."""
    a = y.abs().nan_to_num(0.0).contiguous()
    c = torch.searchsorted(MIDDLES, a)                      # (middles below a)
    tie = (c < 126) & (MIDDLES[c.clamp(max=125)] == a)
    c = torch.where(tie & (c % 2 == 1), c + 1, c) + 128 * torch.signbit(y).long()
    return torch.where(torch.isnan(y), 127, c).byte()


def exponent(top):
    """The smallest e with top <= 448 * 2^e, -117 <= e <= 120."""
    e = -117
    while e < 120 and top > 448 * 2.0 ** e:
        e += 1
    return e


def write(c, s, kb, x, row, n, page):
    """The newest rows x (R, HKV, D) of a sequence of n tokens, put into cache tensors on the host (codes c, scales s,
    bounds kb or None)."""
    x = x.double()
    R, HKV, D = x.shape
    first = n - R
    for blk in range(max(first, 0) // page, -(-n // page)):
        pid = int(row[blk])
        if not 0 <= pid < c.shape[0]:
            continue
        p0, p1 = max(first, 0, blk * page), min(n, (blk + 1) * page)
        had = p0 - blk * page
        for h in range(HKV):
            y = x[p0 - first:p1 - first, h]
            fine = torch.isfinite(y).all(-1)
            e = exponent(float(y[fine].abs().max()) if fine.any() else 0.0)
            drop = 0
            if had:
                was = int(s[pid, h]) - 127
                e = max(e, was)
                drop = e - was
            if drop:
                old = CODES[c[pid, h, :had].long()]
                new = codes_of(old * 2.0 ** -drop)
                c[pid, h, :had] = torch.where(torch.isnan(old), c[pid, h, :had], new)
            new = codes_of(torch.where(fine[:, None], y, math.nan) * 2.0 ** -e)
            c[pid, h, had:p1 - blk * page] = new
            s[pid, h] = e + 127
            if kb is not None:
                v = CODES[new.long()][fine]
                for i, z in enumerate((v, -v)):
                    up = torch.ceil(z.amax(0) / 4).long() if len(z) else torch.full((D,), -112)
                    old = torch.ceil(kb[pid, h, i].double() * 2.0 ** -drop).long() if had else torch.full((D,), -112)
                    kb[pid, h, i] = torch.maximum(up, old).to(torch.int8)


def rows_at(codes, scales, slots):
    """fp64 values (T, HKV, D) at slots of cache tensors."""
    page = codes.shape[2]
    p, o = slots.long() // page, slots.long() % page
    return CODES.to(codes.device)[codes[p, :, o].long()] * torch.exp2(scales[p].double() - 127)[..., None]


def select(q, s, kb, row, n, page, k, first, last):
    """The chosen blocks (R, HKV, k) of the newest tokens q (R, HQ, D) of a sequence of n tokens, in whole numbers of
    Python's."""
    R, HQ, D = q.shape
    HKV = kb.shape[1]
    out = torch.full((R, HKV, k), -1, dtype=torch.int32)
    for j in range(R):
        pos = n - R + j
        seen = pos // page + 1 if pos >= 0 else 0
        if seen <= k:
            out[j, :, :seen] = torch.arange(seen, dtype=torch.int32)
            continue
        ids = row[:seen].long()
        ok = (ids >= 0) & (ids < kb.shape[0])
        b = kb[ids.clamp(0, kb.shape[0] - 1)].long()
        e = s[ids.clamp(0, kb.shape[0] - 1)].long() - 127
        for h in range(HKV):
            x = q[j, h * (HQ // HKV):(h + 1) * (HQ // HKV)].double()
            x = torch.where(torch.isfinite(x), x, 0.0)
            u = -120
            while float(x.abs().max()) > 127 * 2.0 ** u:
                u += 1
            x = torch.round(x * 2.0 ** -u).long()
            score = (x.clamp(min=0)[None] * b[:, h, 0][:, None] + (-x).clamp(min=0)[None] * b[:, h, 1][:, None]).sum(-1).amax(-1)
            keys = []
            for i in range(seen):
                if i < first or i >= seen - last:
                    keys.append((0, 0, i))
                elif ok[i]:
                    v = int(score[i]) * 2.0 ** min(int(e[i, h]), 100)          # (exact: 24 bits times a power of two)
                    keys.append((1, -v, i))
                else:
                    keys.append((2, 0, i))
            out[j, h] = torch.tensor(sorted(i for _, _, i in sorted(keys)[:k]), dtype=torch.int32)
    return out


def attn(q, k, v, n, scale, weight=2.0 ** -16, blocks=None, page=0):
    """One sequence: q (R, HQ, D) the newest tokens of k, v (n, HKV, D) fp64, blocks (R, HKV, m) or None for all keys.
    Returns the fp64 output and the fp32 kernel's error bound beside the output's own rounding: sums of D exact
    products (each sum off by D 2^-24 of its terms' sizes, as a score and once more in the maximum), weights rounded
    to `weight` of themselves (two bf16 terms 2^-16; fp16 2^-11), exponentials and sums over n keys ((n + 64) 2^-24);
    and what fp32 does not hold: a weight, or its second term, under 2^-126 counts as 0, so that each key may be off
    by 2^-125 |v|; fp16 weights are kept times 2^7, those under 2^-21 of the largest to half of 2^-24 / 2^7: 2^-32
    |v|."""
    R, HQ, D = q.shape
    HKV = k.shape[1]
    G = HQ // HKV
    out = torch.zeros(R, HQ, D, dtype=torch.float64, device=q.device)
    err = torch.zeros_like(out)
    for j in range(R):
        m = n - R + j + 1
        if m <= 0:
            continue
        for h in range(HKV):
            if blocks is None:
                at = torch.arange(m, device=q.device)
            else:
                at = (blocks[j, h].long()[:, None] * page + torch.arange(page, device=q.device)).flatten()
                at = at[(at >= 0) & (at < m)]
                if not len(at):
                    continue
            x, kk, vv = q[j, h * G:(h + 1) * G].double(), k[at, h], v[at, h]
            w = torch.softmax((x @ kk.t()) * scale, -1)
            size = (x.abs() @ kk.abs().t()).amax(-1) * abs(scale)
            out[j, h * G:(h + 1) * G] = w @ vv
            err[j, h * G:(h + 1) * G] = ((w @ vv.abs()) * (2 * size[:, None] * (D + 4) * 2.0 ** -24 + weight + (len(at) + 64) * 2.0 ** -24)
                                         + (2.0 ** -32 if weight > 2.0 ** -16 else 2.0 ** -125) * vv.abs().sum(0))
    return out, err
