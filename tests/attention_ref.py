"""Plain restatements in 64 bits of the attention operators, and the cases their tests share."""
import math

import numpy as np
import torch


def blocks(table, head, cached, new, free, block, T):
    """block_tables, one request and one token at a time."""
    table, W, q, kv, pos, slot, starts = table.copy(), table.shape[1], 0, [], [], [], [0]
    head = max(head, 0)
    for r in range(len(cached)):
        c, n = max(int(cached[r]), 0), max(int(new[r]), 0)
        n = min(n, T - q)
        held, need = min(-(-c // block), W), min(-(-(c + n) // block), W)
        for p in range(held, need):
            table[r, p] = free[head] if head < len(free) else -1
            head += 1
        for i in range(n):
            page = (c + i) // block
            b = table[r, page] if page < W else -1
            pos.append(c + i)
            slot.append(b * block + (c + i) % block if b >= 0 else -1)
        q += n
        kv.append(c + n)
        starts.append(q)
    pos += [0] * (T - q)
    slot += [-1] * (T - q)
    return table, np.array([head]), np.array(starts), np.array(kv), np.array(pos, dtype=int), np.array(slot, dtype=int)


def turn(x, positions, freqs, amplitude, interleaved, transpose=False):
    """(rotation of x [T, H, D] in float64, the sum of the magnitudes that go into each value)."""
    x = x.double()
    n = freqs.numel()
    angle = positions.double()[:, None, None] * freqs.double()
    c, s = torch.cos(angle) * amplitude, torch.sin(angle) * amplitude * (-1 if transpose else 1)
    i = torch.arange(n)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
    y, size = x.clone(), x.abs().clone()
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    size[..., a] = size[..., b] = (x[..., a].abs() + x[..., b].abs()) * amplitude
    return y, size


def attend(q, keys, values, starts, kv_lens, scale, window=0, gate=None, absent=()):
    """(o, bound) of paged attention in float64: q [T, Hq, D], keys and values per request [L, Hkv, D].
    absent: (request, position) pairs on missing pages.

    bound: bf16 rounding of the result (2^-8), of the softmax's weights and of their sum (2^-8 each, of
    sum p |v|), and the f32 dot products and exponents (D + 8 roundings of 2^-24 of scale sum |q k|, twice:
    the weight and the sum)."""
    T, Hq, D = q.shape
    o, bound = torch.zeros(T, Hq, D, dtype=torch.float64), torch.full((T, Hq, D), 1e-30, dtype=torch.float64)
    q = q.double()
    for r in range(len(kv_lens)):
        t0, t1 = int(starts[r]), int(starts[r + 1])
        K, V = keys[r].double(), values[r].double()
        L, Hkv = K.shape[0], K.shape[1]
        pos = torch.arange(int(kv_lens[r]) - (t1 - t0), int(kv_lens[r]))[:, None]
        j = torch.arange(L)
        seen = j <= pos
        if window:
            seen &= j > pos - window
        for rr, p in absent:
            if rr == r:
                seen[:, p] = False
        for h in range(Hq):
            k, v = K[:, h // (Hq // Hkv)], V[:, h // (Hq // Hkv)]
            for i in range(t1 - t0):
                m = seen[i]
                if not m.any():
                    continue
                x = q[t0 + i, h]
                s = (k[m] @ x) * scale
                size = float((k[m].abs() @ x.abs()).max()) * abs(scale)
                p = torch.softmax(s, 0)
                o[t0 + i, h] = p @ v[m]
                weight = 2 ** -7 + 2 * (D + 8) * 2 ** -24 * size
                bound[t0 + i, h] += 2 ** -8 * o[t0 + i, h].abs() + weight * (p @ v[m].abs())
    if gate is not None:
        g = 1 / (1 + torch.exp(-gate.double()))
        o, bound = o * g, bound * g * (1 + 2 ** -8)
    return o, bound


class Cache:
    """Requests' keys and values scattered over pages in no order; every other row NaN."""

    def __init__(self, lens, Hkv, D, block, seed, spare=5, width=None, scale=1.0):
        g = torch.Generator().manual_seed(seed)
        counts = [-(-n // block) for n in lens]
        n = sum(counts) + spare
        order = torch.randperm(n, generator=g).tolist()
        self.W = width or max([1] + counts)
        self.table = np.full((len(lens), self.W), -1, dtype=np.int32)
        self.k, self.v = (torch.full((n, Hkv, block, D), math.nan, dtype=torch.bfloat16) for _ in range(2))
        self.keys, self.values, at = [], [], 0
        for r, L in enumerate(lens):
            self.table[r, :counts[r]] = order[at:at + counts[r]]
            at += counts[r]
            for cache, mine, f in ((self.k, self.keys, scale), (self.v, self.values, 1.0)):
                x = (torch.randn(L, Hkv, D, generator=g) * f).to(torch.bfloat16)
                mine.append(x)
                for p in range(counts[r]):
                    rows = x[p * block:(p + 1) * block].transpose(0, 1)
                    cache[int(self.table[r, p]), :, :rows.shape[1]] = rows
