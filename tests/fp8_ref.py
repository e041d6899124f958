"""Plain restatements in 64 bits of the operators over a cache held in 8 bits, on the CPU."""
import math

import numpy as np
import torch

# the value of every E4M3 code (127 and 255: NaN)
VALUES = torch.tensor([(-1) ** (c >> 7) * ((8 + (c & 7)) * 2.0 ** ((c >> 3 & 15) - 10) if c >> 3 & 15 else (c & 7) * 2.0 ** -9)
                       if c & 127 != 127 else math.nan for c in range(256)], dtype=torch.float64)
MAGNITUDES = VALUES[:127].numpy()


def decode(codes, scales):
    """Codes [..., n, D] with scale bytes [...] as float64."""
    f = torch.where(scales == 255, math.nan, 2.0 ** (scales.double() - 127))
    return VALUES[codes.long()] * f[..., None, None]


def encode(y):
    """Codes nearest to y (float64), ties to the even one; not finite: 127.  |y| is at most 448 where finite."""
    a = y.abs().numpy()
    fine = np.isfinite(a)
    a = np.where(fine, a, 0.0)
    hi = np.searchsorted(MAGNITUDES, a).clip(max=126)  # the first code at or above
    lo = (hi - 1).clip(min=0)
    down, up = a - MAGNITUDES[lo], MAGNITUDES[hi] - a
    code = np.where((down < up) | ((down == up) & (lo % 2 == 0)), lo, hi)
    code = np.where(fine, code + 128 * np.signbit(y.numpy()), 127)
    return torch.from_numpy(code.astype(np.uint8))


def exponent(top):
    """The smallest t >= -127 with 448 * 2^t >= top."""
    if top == 0:
        return -127
    m, e = math.frexp(top)
    return max(-127, e - 9 if m <= 0.875 else e - 8)


def store(codes, scales, slots, y):
    """rope_cache_fp8's write of y [T, H, D] float64 (and the largest finite |y| of each page and head that it reached)."""
    codes, scales, tops = codes.clone(), scales.clone(), {}
    P, H, block, D = codes.shape
    rows = {}
    for i, s in enumerate(slots):
        if 0 <= s < P * block:
            rows.setdefault(s // block, []).append((i, s % block))
    for page, at in rows.items():
        i, off = [a for a, _ in at], [b for _, b in at]
        for h in range(H):
            x = y[i, h]
            fine = torch.isfinite(x)
            top = float(x[fine].abs().max()) if fine.any() else 0.0
            t, old = exponent(top), int(scales[page, h]) - 127
            if 0 not in off:
                t = max(t, old)
                if t > old:
                    codes[page, h] = encode(VALUES[codes[page, h].long()] * 2.0 ** (old - t))
            scales[page, h] = t + 127
            codes[page, h, off] = encode(x * 2.0 ** -t)
            tops[page, h] = top
    return codes, scales, tops


def same(a, b):
    """Codes alike, or both NaN."""
    return (a == b) | ((a & 127 == 127) & (b & 127 == 127))


class Cache:
    """Requests' keys and values scattered over pages in no order: `keys`, `values` [L, Hkv, D] float64 as their codes and
    scales say; every other row NaN, every other page's scales too."""

    def __init__(self, lens, Hkv, D, block, seed, spare=5, width=None, spread=0.7):
        g = torch.Generator().manual_seed(seed)
        counts = [-(-n // block) for n in lens]
        n = sum(counts) + spare
        order = torch.randperm(n, generator=g).tolist()
        self.W = width or max([1] + counts)
        self.table = np.full((len(lens), self.W), -1, dtype=np.int32)
        self.k, self.v = (torch.full((n, Hkv, block, D), 127, dtype=torch.uint8) for _ in range(2))
        self.ks, self.vs = (torch.full((n, Hkv), 255, dtype=torch.uint8) for _ in range(2))
        at = 0
        for r, L in enumerate(lens):
            self.table[r, :counts[r]] = order[at:at + counts[r]]
            at += counts[r]
            for cache, scales in ((self.k, self.ks), (self.v, self.vs)):
                for p in range(counts[r]):
                    page, m = int(self.table[r, p]), min(block, L - p * block)
                    x = torch.randn(Hkv, m, D, generator=g) * torch.exp(spread * torch.randn(Hkv, 1, 1, generator=g))
                    for h in range(Hkv):
                        t = exponent(float(x[h].abs().max()))
                        scales[page, h] = t + 127
                        cache[page, h, :m] = (x[h] * 2.0 ** -t).to(torch.float8_e4m3fn).view(torch.uint8)
        self.lens, self.block = list(lens), block

    def _wide(self, cache, scales):
        out = []
        for r, L in enumerate(self.lens):
            pages = torch.from_numpy(self.table[r, :-(-L // self.block)]).long()
            x = decode(cache[pages], scales[pages]).transpose(1, 2).reshape(-1, cache.shape[1], cache.shape[3])
            out.append(x[:L])
        return out

    @property
    def keys(self):
        return self._wide(self.k, self.ks)

    @property
    def values(self):
        return self._wide(self.v, self.vs)

    @property
    def scales(self):
        """The scale of each value row: [L, Hkv] per request (1 where it is NaN)."""
        return [self._wide(torch.full_like(self.v, 0x38), torch.where(self.vs == 255, 127, self.vs))[r][..., 0]
                for r in range(len(self.lens))]


def attend(q, keys, values, starts, kv_lens, scale, window=0, gate=None, few=False, scales=None):
    """(o, bound) of paged attention in float64, a key head's rows at a time, on q's device; q [T, Hq, D].

    bound: the result's rounding to bf16 (2^-8); of sum p |v|: the weights' rounding (two E4M3 parts: 2^-4 of 2^-4, so 2^-8;
    few: two bf16 parts, 2^-16) and as much for the sum that divides, f32 dot products and exponents (D + 8 roundings of 2^-24 of scale sum |q k|), the queries' two parts (2^-22 of the largest of 128 values, times
    the sum of |k| there), both twice: in the weight and in the sum; exp2 (2^-22 twice); f32 sums over L keys, at worst 16
    at a time in a line (L / 16 + 64 roundings of 2^-24, in the sum as well).

    Not few: E4M3's steps end at 2^-9.  The weights of 32 keys go in relative to their largest, which lies above 2^7, each
    times its value's scale over the largest scale of the 32 (scales that differ by more than 2^8: relative to the largest
    product of weight and scale); what the first part leaves is at most 2^3 and goes in times 2^5, so its own steps end at
    2^-14 and leave 2^-15: 2^-22 of the largest weight, on the codes of all 32 keys at the largest scale.  scales: those of
    the values, [L, Hkv] per request (none: 1 for all)."""
    T, Hq, D = q.shape
    o = torch.zeros(T, Hq, D, dtype=torch.float64, device=q.device)
    bound = torch.full_like(o, 1e-30)
    for r, kv in enumerate(kv_lens):
        t0, t1 = int(starts[r]), int(starts[r + 1])
        if t0 == t1 or not kv:
            continue
        K, V = keys[r].to(q.device), values[r].to(q.device)
        L, Hkv = K.shape[0], K.shape[1]
        g, j = Hq // Hkv, torch.arange(L, device=q.device)
        for a in range(t0, t1, max(1, 2048 // g)):
            b = min(t1, a + max(1, 2048 // g))
            pos = (int(kv) - t1 + torch.arange(a, b, device=q.device))[:, None, None]
            seen = (j <= pos) & ((j > pos - window) if window else True)
            for h in range(Hkv):
                k, v = K[:, h].contiguous(), V[:, h].contiguous()
                x = q[a:b, h * g:(h + 1) * g].double().reshape(-1, D)
                s = (x @ k.T.contiguous()).view(b - a, g, L) * scale
                pad = torch.nn.functional.pad(x.abs(), (0, -D % 128)).view(x.shape[0], -1, 128).amax(-1)
                pad = pad.repeat_interleave(128, 1)[:, :D]
                kt = k.abs().T.contiguous()
                size = (2 * (D + 8) * 2 ** -24 * (x.abs() @ kt) + 2 * 2 ** -22 * (pad @ kt)).view(b - a, g, L) * abs(scale)
                size = size.masked_fill(~seen, 0).nan_to_num(0.0).amax(-1, keepdim=True)
                p = torch.softmax(s.masked_fill(~seen, -math.inf), -1)
                p = torch.where(seen.any(-1, keepdim=True), p, 0.0)
                pv = torch.where(seen.any(-1, keepdim=True).expand(b - a, g, 1).reshape(-1, 1), masked(p.view(-1, L), v, seen, g), 0.0)
                o[a:b, h * g:(h + 1) * g] = pv.view(b - a, g, D)
                parts = 2 ** -16 if few else 2 ** -8
                weight = 2 * parts + size + 2 ** -21 + 2 * (L / 16 + 64) * 2 ** -24
                size_v = v.abs().nan_to_num(0.0)
                bound[a:b, h * g:(h + 1) * g] += weight * (p.view(-1, L) @ size_v).view(b - a, g, D)
                if not few:
                    f = scales[r][:, h].to(q.device) if scales else torch.ones(L, dtype=torch.float64, device=q.device)
                    grouped = lambda x, dim: torch.nn.functional.pad(x, (0, 0) * (x.dim() - 1 - dim) + (0, -L % 32)).unflatten(dim, (-1, 32))  # noqa: E731
                    pf, most = grouped((p.view(-1, L) * f).nan_to_num(0.0), 1).amax(-1), grouped(p.view(-1, L).nan_to_num(0.0), 1).amax(-1)
                    fs = grouped(f, 0)
                    top = fs.amax(-1)
                    near = top <= 2.0 ** 8 * torch.where(fs > 0, fs, math.inf).amin(-1)
                    codes = grouped(size_v / f[:, None], 0).sum(1)
                    bound[a:b, h * g:(h + 1) * g] += 2 ** -22 * (torch.where(near, most * top, pf) @ codes).view(b - a, g, D)
    bound += 2 ** -8 * o.abs().nan_to_num(0.0)
    if gate is not None:
        f = 1 / (1 + torch.exp(-gate.double()))
        o, bound = o * f, bound * f * (1 + 2 ** -8)
    return o, bound


def masked(p, v, seen, g):
    """p @ v where values of keys that a row does not see add nothing, whatever they are."""
    y = p.nan_to_num(0.0) @ v.nan_to_num(0.0)
    bad = torch.isnan(v)
    if bad.any():
        hit = (seen.expand(-1, g, -1).reshape(p.shape).double() @ bad.double()) > 0
        y = torch.where(hit, math.nan, y)
    return torch.where(torch.isnan(p).any(-1, keepdim=True), math.nan, y)
