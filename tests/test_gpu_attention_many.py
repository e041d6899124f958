"""Paged attention of many requests, many tiles and many parts of one tile: the ways of sharing the work that few requests
do not reach."""
import math

import attention_ref as ref
import numpy as np
import pytest
import torch

import qmm as Q


def attend(q, keys, values, starts, kv_lens, scale, window=0, gate=None):
    """(o, bound) of attention_ref.attend, a key head's rows at a time (on the tensors' own device)."""
    T, Hq, D = q.shape
    o = torch.zeros(T, Hq, D, dtype=torch.float64, device=q.device)
    bound = torch.full_like(o, 1e-30)
    for r, kv in enumerate(kv_lens):
        t0, t1 = int(starts[r]), int(starts[r + 1])
        if t0 == t1 or not kv:
            continue
        K, V = keys[r].to(q.device).double(), values[r].to(q.device).double()
        L, Hkv = K.shape[0], K.shape[1]
        g, j = Hq // Hkv, torch.arange(L, device=q.device)
        for a in range(t0, t1, max(1, 4096 // g)):
            b = min(t1, a + max(1, 4096 // g))
            pos = (int(kv) - t1 + torch.arange(a, b, device=q.device))[:, None, None]
            seen = (j <= pos) & ((j > pos - window) if window else True)
            for h in range(Hkv):
                k, v = K[:, h].contiguous(), V[:, h].contiguous()
                x = q[a:b, h * g:(h + 1) * g].double()
                s = (x.reshape(-1, D) @ k.T.contiguous()).view(b - a, g, L) * scale
                size = (x.abs().reshape(-1, D) @ k.abs().T.contiguous()).view(b - a, g, L) * abs(scale)
                size = size.masked_fill(~seen, 0).amax(-1, keepdim=True)
                p = torch.softmax(s.masked_fill(~seen, -math.inf), -1).nan_to_num(0.0).view(-1, L)
                o[a:b, h * g:(h + 1) * g] = (p @ v).view(b - a, g, D)
                weight = 2 ** -7 + 2 * (D + 8) * 2 ** -24 * size
                bound[a:b, h * g:(h + 1) * g] += weight * (p @ v.abs()).view(b - a, g, D)
    bound += 2 ** -8 * o.abs()
    if gate is not None:
        s = 1 / (1 + torch.exp(-gate.double()))
        o, bound = o * s, bound * s * (1 + 2 ** -8)
    return o, bound


@pytest.mark.parametrize("window", [0, 9])
def test_the_restatement_by_heads_is_the_one_by_rows(window):
    new, kv, g = [3, 0, 20, 1], [2, 7, 33, 40], torch.Generator().manual_seed(1)
    c = ref.Cache(kv, 2, 16, 8, seed=2)
    q, gate = (torch.randn(sum(new) + 2, 6, 16, generator=g) for _ in range(2))
    starts = [0] + np.cumsum(new).tolist()
    for a, b in zip(attend(q, c.keys, c.values, starts, kv, 0.3, window, gate),
                    ref.attend(q, c.keys, c.values, starts, kv, 0.3, window, gate)):
        assert torch.allclose(a, b, rtol=1e-12, atol=1e-14)


def ints(v):
    return Q.Array.from_numpy(np.asarray(v, dtype=np.int32), Q.INT32)


def dev(t):
    return Q.Array.from_torch(t.cuda().contiguous())


def check(Hq, Hkv, D, block, new, kv, seed, scale=None, window=0, gated=False, before=0, after=0):
    T, g = before + sum(new) + after, torch.Generator().manual_seed(seed)
    c = ref.Cache(kv, Hkv, D, block, seed=seed)
    q = (2 * torch.randn(T, Hq, D, generator=g)).to(torch.bfloat16).cuda()
    gate = torch.randn(T, Hq, D, generator=g).to(torch.bfloat16).cuda() if gated else None
    starts = (before + np.cumsum([0] + list(new))).tolist()
    scale = D ** -0.5 if scale is None else scale
    out = torch.full(q.shape, math.nan, dtype=torch.bfloat16, device="cuda")
    Q.paged_attention(dev(q), dev(c.k), dev(c.v), ints(c.table), ints(starts), ints(kv), scale=scale, window=window,
                      gate=dev(gate) if gated else None, out=Q.Array.from_torch(out))
    torch.cuda.synchronize()
    want, bound = attend(q, c.keys, c.values, starts, kv, scale, window, gate)
    assert not torch.isnan(out).any()
    assert ((out.double() - want).abs() <= bound).all()
    return out


def lens(R, seed, cached, new, idle=0.0, chunk=None):
    rng = np.random.default_rng(seed)
    n = rng.integers(1, new + 1, R) * (rng.random(R) >= idle)
    c = rng.integers(0, cached + 1, R)
    if chunk is not None:
        n[chunk[0]] = chunk[1]
    return n.tolist(), (c + n).tolist()


MANY = [  # Hq, Hkv, D, block, lens(...)
    (32, 8, 128, 16, dict(R=65, seed=1, cached=2000, new=1)),
    (12, 2, 256, 16, dict(R=65, seed=2, cached=300, new=3, idle=0.4, chunk=(64, 90))),
    (4, 4, 64, 24, dict(R=256, seed=3, cached=200, new=1, idle=0.2)),
    (4, 4, 64, 24, dict(R=300, seed=4, cached=200, new=4, idle=0.3, chunk=(257, 70))),
    (6, 1, 128, 7, dict(R=300, seed=5, cached=400, new=1, idle=0.5)),
    (2, 1, 64, 16, dict(R=1000, seed=6, cached=150, new=2, idle=0.6, chunk=(999, 140))),
    (8, 1, 256, 16, dict(R=1000, seed=7, cached=60, new=1)),
    (1, 1, 32, 16, dict(R=4096, seed=8, cached=40, new=1, idle=0.7)),
    (4, 1, 64, 16, dict(R=4096, seed=9, cached=30, new=1, idle=0.9, chunk=(4000, 300))),
    (4, 1, 256, 16, dict(R=4096, seed=10, cached=20, new=2, chunk=(100, 300))),
]


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,Hkv,D,block,kw", MANY)
@pytest.mark.parametrize("window", [0, 33])
def test_many_requests(Hq, Hkv, D, block, kw, window):
    check(Hq, Hkv, D, block, *lens(**kw), seed=kw["seed"], window=window, gated=window > 0)


TILES = [  # Hq, Hkv, D, new, kv: tiles per head
    (64, 1, 64, [1] * 57 + [2] * 3, [100] * 60),              # 126, of 32 rows, of no more than 64 requests
    (64, 1, 64, [1] * 300, list(range(1, 301))),              # 600, of 32 rows
    (64, 2, 64, [1] * 60 + [200, 400], [50] * 60 + [210, 700]),  # 76 of 256 rows beside 60 of up to 32
    (64, 1, 64, [300], [500]),                                # 75
    (64, 1, 64, [1040], [1040]),                              # 260
    (64, 1, 32, [3] * 70 + [600, 1], [40] * 71 + [3]),        # 70 requests of 192 rows and one of 150 tiles
    (64, 1, 128, [5] * 299 + [1], [9] * 300),                 # 599 of 256 rows
]


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,Hkv,D,new,kv", TILES)
def test_many_tiles(Hq, Hkv, D, new, kv):
    check(Hq, Hkv, D, 16, new, [max(a, b) for a, b in zip(new, kv)], seed=len(new))


PARTS = [  # Hq, Hkv, D, new, kv: one key head, so that every workgroup has a part of the one tile
    (6, 1, 256, [1], [40000]), (8, 1, 128, [1], [40001]), (1, 1, 64, [1], [140000]), (6, 1, 256, [3], [40003]),
    (4, 1, 128, [8], [50000]), (2, 1, 256, [40], [33000]), (1, 1, 128, [200], [40000]), (8, 1, 64, [6], [60000]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,Hkv,D,new,kv", PARTS)
@pytest.mark.parametrize("gated", [False, True])
def test_many_parts_of_a_tile(Hq, Hkv, D, new, kv, gated):
    check(Hq, Hkv, D, 16, new, kv, seed=D, gated=gated)


@pytest.mark.gpu
@pytest.mark.parametrize("new,kv", [([1], [700]), ([3, 1], [300, 40]), ([150, 2], [400, 9])])
def test_a_scale_of_zero_weighs_all_keys_alike(new, kv):
    for scale in (0.0, -0.0):
        check(8, 2, 128, 16, new, kv, seed=11, scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("new,kv", [([1], [700]), ([2, 0, 1], [300, 5, 40]), ([150, 2], [400, 9])])
def test_rows_before_the_first_request_are_zero(new, kv):
    out = check(6, 2, 64, 16, new, kv, seed=12, before=5, after=3)
    assert (out[:5] == 0).all() and (out[-3:] == 0).all() and (out[5:-3] != 0).any()
