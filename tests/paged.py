"""Paged caches for the tests, their tables in no order and every place that no position has
poisoned, and the operators over them in 64 bits."""
import math

import torch

E4M3 = torch.float8_e4m3fn
NAN = float("nan")


def fused(rows, width, gen, spare=0):
    """bf16 rows of `width` values inside wider ones, `spare` values apart."""
    x = torch.randn(rows, width + spare, generator=gen, device="cuda").bfloat16()
    return x[:, :width] if spare else x


class Cache:
    """lengths, new: Python lists. `poison`: what lies in rows that no position has."""

    def __init__(self, seed, lengths, new, kv_heads, width, page, cache="bf16", spare_pages=3, spare_columns=2, poison=NAN,
                 rows_behind=0, spread=1.0):
        self.gen = gen = torch.Generator("cuda").manual_seed(seed)
        self.lengths, self.new, self.kv, self.width, self.page, self.kind = lengths, new, kv_heads, width, page, cache
        need = [-(-max(0, n) // page) for n in lengths]
        self.most, self.pages = max(need) + spare_columns, sum(need) + spare_pages
        order = torch.randperm(self.pages, generator=gen, device="cuda", dtype=torch.int32)
        self.tables = torch.full((len(lengths), self.most), -1, device="cuda", dtype=torch.int32)
        at = 0
        for s, n in enumerate(need):
            self.tables[s, :n] = order[at:at + n]
            at += n
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        self.starts, self.rows = starts, starts[-1] + rows_behind
        shape = (self.pages, kv_heads, page, width)
        if cache == "bf16":
            self.keys = torch.full(shape, poison, device="cuda", dtype=torch.bfloat16)
            self.values = torch.full(shape, poison, device="cuda", dtype=torch.bfloat16)
            self.key_scales = self.value_scales = None
        else:  # 0x7f is NaN
            code = 0x7f if math.isnan(poison) else 0x7e
            self.keys = torch.full(shape, code, device="cuda", dtype=torch.uint8)
            self.values = torch.full(shape, code, device="cuda", dtype=torch.uint8)
            self.key_scales = torch.full(shape[:3], poison, device="cuda")
            self.value_scales = torch.full(shape[:3], poison, device="cuda")
        self.dense = []  # per sequence: keys, values [kv][length][width] as the cache holds them, in 64 bits
        for s, n in enumerate(lengths):
            n = max(0, n)
            k = spread * torch.randn(n, kv_heads, width, generator=gen, device="cuda")
            v = torch.randn(n, kv_heads, width, generator=gen, device="cuda")
            self.dense.append([self.put(s, 0, which, x) for which, x in (("keys", k), ("values", v))])

    def place(self, s, first, n):
        j = torch.arange(first, first + n, device="cuda")
        return self.tables[s, j // self.page].long(), j % self.page

    def put(self, s, first, which, x):
        """Writes rows x [n][kv][width] at positions from `first` on; what they are there, in 64 bits."""
        page, slot = self.place(s, first, x.shape[0])
        if self.kind == "bf16":
            b = x.bfloat16()
            getattr(self, which)[page, :, slot] = b
            return b.double().transpose(0, 1).contiguous()
        scale = torch.where(x.abs().amax(-1) > 0, x.abs().amax(-1) / 448.0, 1.0)
        code = (x / scale.unsqueeze(-1)).to(E4M3)
        getattr(self, which)[page, :, slot] = code.view(torch.uint8)
        getattr(self, which[:-1] + "_scales")[page, :, slot] = scale
        return (code.double() * scale.unsqueeze(-1).double()).transpose(0, 1).contiguous()

    def device(self, values):
        return torch.tensor(values, device="cuda", dtype=torch.int32)


def attend(c, q, heads, window=0, scale=None, no_page=()):
    """(out, bound on the error) [rows][heads][width] in 64 bits; no_page: (sequence, column) without a page.

    The bound, from the formula o = sum p v / sum p with A = sum p |v| / sum p: the weights p are rounded to
    bf16, at most 2^-8 of each, and so is the result, 2^-8 of it; scores are fp32 sums of `width` exact products,
    at most width 2^-24 of the sum of their magnitudes M, and three roundings more of the score and of its
    distance to the largest, so p is within M scale (width + 4) 2^-24, and 2^-21 for the exponential itself; that counts twice,
    once in sum p; sums of n terms in fp32 n 2^-24 of A each."""
    group = heads // c.kv
    scale = c.width ** -0.5 if scale is None else scale
    out = torch.zeros(c.rows, heads, c.width, device="cuda", dtype=torch.float64)
    tol = torch.zeros_like(out)
    for s, length in enumerate(c.lengths):
        length, n = max(0, length), c.new[s]
        if n == 0 or length == 0:
            continue
        p = torch.arange(c.lengths[s] - n, c.lengths[s], device="cuda").unsqueeze(1)
        j = torch.arange(length, device="cuda").unsqueeze(0)
        seen = j <= p
        if window:
            seen = seen & (j > p - window)
        for where, column in no_page:
            if where == s:
                seen = seen & (j // c.page != column)
        for h in range(heads):
            rows = q[c.starts[s]:c.starts[s + 1], h * c.width:(h + 1) * c.width].double()
            k, v = c.dense[s][0][h // group], c.dense[s][1][h // group]
            score = (rows @ k.t()) * scale
            score = torch.where(seen, score, -math.inf)
            top = score.amax(1, keepdim=True)
            w = torch.where(seen, (score - torch.where(top > -math.inf, top, 0.0)).exp(), 0.0)
            total = w.sum(1, keepdim=True)
            w = torch.where(total > 0, w / total, torch.where(total == 0, 0.0, total))
            v = torch.where(seen.any(0).unsqueeze(1), v, 0.0)
            dirty = ~v.isfinite()
            o = w @ torch.where(dirty, 0.0, v)
            if bool(dirty.any()):  # a value that is not finite counts where it is seen, and only there
                for at in dirty.any(1).nonzero().reshape(-1).tolist():
                    o = o + torch.where(seen[:, at:at + 1] & dirty[at], w[:, at:at + 1] * v[at], 0.0)
            a = w @ torch.where(dirty, 0.0, v).abs()
            m = (rows.abs() @ torch.where(k.isfinite(), k, 0.0).abs().t() * seen).amax(1, keepdim=True) * abs(scale)
            e = m * (c.width + 4) * 2.0 ** -24 + 2.0 ** -21
            out[c.starts[s]:c.starts[s + 1], h] = o
            tol[c.starts[s]:c.starts[s + 1], h] = a * (2.0 ** -8 + 2 * e + 2 * length * 2.0 ** -24) + o.abs() * 2.0 ** -8
    return out, tol * 1.02 + 2.0 ** -133  # products of the roundings; the least bf16 step
