"""Paged attention over a cache held in 8 bits, against a plain restatement in 64 bits (fp8_ref.py)."""
import math

import fp8_ref as ref
import numpy as np
import pytest
import torch

import qmm as Q

pytestmark = pytest.mark.gpu


def ints(v):
    return Q.Array.from_numpy(np.asarray(v, dtype=np.int32), Q.INT32)


def dev(t):
    return Q.Array.from_torch(t.cuda().contiguous())


def host(a):
    return torch.from_numpy(a.numpy().view(np.int16)).view(torch.bfloat16)


def starts_of(new):
    return [0] + np.cumsum(new).tolist()


def attention(c, q, starts, kv, **kw):
    kw.setdefault("scale", q.shape[-1] ** -0.5)
    gate = kw.pop("gate", None)
    return host(Q.paged_attention_fp8(dev(q), dev(c.k), dev(c.v), dev(c.ks), dev(c.vs), ints(c.table), ints(starts), ints(kv),
                                      gate=dev(gate) if gate is not None else None, **kw))


def close(got, want, bound):
    return ((got.double() - want.cpu()).abs() <= bound.cpu()).all()


ATTEND = [
    # Hq, Hkv, D, block, (cached, new) of each request, window
    (6, 1, 256, 16, [(0, 1)], 0),
    (24, 4, 256, 16, [(1998, 1)], 0),
    (24, 4, 256, 64, [(5000, 3), (17, 1), (0, 2)], 0),
    (8, 2, 128, 16, [(c * 37, 1) for c in range(40)], 0),
    (8, 8, 64, 24, [(100, 1), (900, 5), (0, 70)], 0),
    (16, 2, 64, 7, [(300, 4), (63, 1), (64, 1), (65, 1), (0, 1)], 40),
    (12, 4, 96, 1, [(90, 2), (5, 30)], 0),
    (10, 2, 80, 33, [(1000, 3), (200, 2)], 100),
    (3, 1, 208, 16, [(70, 40), (300, 1)], 0),
    (2, 1, 16, 16, [(40, 9), (0, 200)], 0),
    (24, 4, 256, 16, [(100, 300), (0, 77)], 0),
    (8, 1, 256, 32, [(700, 333)], 129),
    (32, 8, 128, 32, [(0, 500)], 0),
    (16, 16, 64, 24, [(0, 700), (90, 200), (400, 1), (3, 0), (0, 13)], 100),
    (4, 4, 48, 5, [(33, 300)], 0),
]


@pytest.mark.parametrize("Hq,Hkv,D,block,lens,window", ATTEND)
@pytest.mark.parametrize("gated", [False, True])
def test_attention(Hq, Hkv, D, block, lens, window, gated):
    new, kv = [n for _, n in lens], [c + n for c, n in lens]
    T, g = sum(new), torch.Generator().manual_seed(D + sum(a * 31 + b for a, b in lens))
    c = ref.Cache(kv, Hkv, D, block, seed=D)
    q = (2 * torch.randn(T, Hq, D, generator=g)).to(torch.bfloat16)
    gate = torch.randn(T, Hq, 2 * D, generator=g).to(torch.bfloat16) if gated else None
    want, bound = ref.attend(q.cuda(), c.keys, c.values, starts_of(new), kv, D ** -0.5, window,
                             gate[..., D:].cuda() if gated else None, scales=c.scales)
    got = attention(c, q, starts_of(new), kv, window=window, gate=gate)
    assert torch.isfinite(got).all()
    assert close(got, want, bound)
    assert torch.equal(got, attention(c, q, starts_of(new), kv, window=window, gate=gate))  # the same bits again


def test_rows_that_see_nothing():
    """Rows before the first key, requests without keys, rows of no request."""
    D, new, kv = 64, [5, 3, 70, 2], [2, 0, 40, 9]
    c = ref.Cache(kv, 2, D, 16, seed=1)
    q = torch.randn(sum(new) + 9, 8, D, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    want, bound = ref.attend(q.cuda(), c.keys, c.values, starts_of(new), kv, 0.125, scales=c.scales)
    got = attention(c, q, starts_of(new), kv)
    assert close(got, want, bound)
    for rows in (slice(0, 3), slice(5, 8), slice(8, 38), slice(80, 89)):
        assert (got[rows] == 0).all()
    assert (attention(c, q, [0] * 5, kv) == 0).all()


def test_without_requests_or_rows():
    c = ref.Cache([20], 2, 64, 16, seed=1)
    q = torch.randn(3, 4, 64).to(torch.bfloat16)
    cache = [dev(t) for t in (c.k, c.v, c.ks, c.vs)]
    assert (host(Q.paged_attention_fp8(dev(q), *cache, ints(np.zeros((0, 2))), ints([0]), ints([]), scale=1.0)) == 0).all()
    assert Q.paged_attention_fp8(dev(q[:0]), *cache, ints(c.table), ints([0, 0]), ints([20]), scale=1.0).shape == (0, 4, 64)
    assert (host(Q.paged_attention_fp8(dev(q), *cache, ints(np.zeros((1, 0))), ints([0, 3]), ints([3]), scale=1.0)) == 0).all()


@pytest.mark.parametrize("new", [1, 3, 90])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_missing_pages(new, D):
    """Page ids that are none: their keys are not seen, whether the table says -1 or anything else."""
    block, L = 16, 400
    c = ref.Cache([L, 30], 2, D, block, seed=3)
    q = torch.randn(new + 1, 6, D, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16)
    keys, values = c.keys, c.values
    gone = [0, 3, 9, 10, 24]
    c.table[0, gone] = [-1, c.k.shape[0], 2 ** 31 - 1, -2 ** 31, -1]
    absent = torch.zeros(L, dtype=torch.bool)
    for p in gone:
        absent[p * block:(p + 1) * block] = True
    # (the same without those keys, each row's own keys counted: rows lie past them all, but on the last page)
    want = torch.zeros(new + 1, 6, D, dtype=torch.float64)
    bound = torch.zeros_like(want)
    for i in range(new):
        see = (~absent) & (torch.arange(L) <= L - new + i)
        n = int(see.sum())
        w, b = ref.attend(q[i:i + 1], [keys[0][see]], [values[0][see]], [0, 1], [n], D ** -0.5)
        want[i], bound[i] = w[0], b[0]
    w, b = ref.attend(q[new:], [keys[1]], [values[1]], [0, 1], [30], D ** -0.5)
    want[new], bound[new] = w[0], b[0]
    assert close(attention(c, q, [0, new, new + 1], [L, 30]), want, bound)


def test_past_the_tables_width():
    D = 64
    c = ref.Cache([64], 2, D, 16, seed=3)
    q = torch.randn(10, 4, D, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16)
    for kv in (70, 2 ** 31 - 1):
        want, bound = ref.attend(q, c.keys, c.values, [0, 10], [kv], 0.125, scales=c.scales)
        assert close(attention(c, q, [0, 10], [kv]), want, bound)


@pytest.mark.parametrize("new,L", [(1, 1000), (3, 300), (200, 500), (90, 1900)])
@pytest.mark.parametrize("kind", ["sharp", "equal", "rising", "falling", "low"])
def test_extreme_scores(new, L, kind):
    """One key carries a row; all keys alike; maxima that move with every key; scores far below zero."""
    D, Hq, Hkv = 128, 8, 2
    c = ref.Cache([L], Hkv, D, 16, seed=6)
    g = torch.Generator().manual_seed(7)
    q = torch.randn(new, Hq, D, generator=g).to(torch.bfloat16)
    scale = D ** -0.5
    if kind == "sharp":
        scale = 8.0
    else:
        q = q.abs() + 0.5
        x = torch.randn(L, Hkv, D, generator=g) * 0.01
        j = torch.arange(L)[:, None, None].float()
        x += dict(equal=0 * j, rising=j / 10, falling=-j / 10, low=0 * j - 50)[kind]
        slots = [int(c.table[0, i // 16]) * 16 + i % 16 for i in range(L)]
        c.k, c.ks, _ = ref.store(c.k, c.ks, slots, x.double())
    want, bound = ref.attend(q.cuda(), c.keys, c.values, [0, new], [L], scale, scales=c.scales)
    got = attention(c, q, [0, new], [L], scale=scale)
    assert torch.isfinite(got).all() and close(got, want, bound)


@pytest.mark.parametrize("new", [1, 4, 80])
@pytest.mark.parametrize("scale", [-0.3, 0.0])
def test_other_scales(new, scale):
    c = ref.Cache([200], 1, 64, 16, seed=8)
    q = torch.rand(new, 2, 64, generator=torch.Generator().manual_seed(9)).to(torch.bfloat16) + 0.5
    want, bound = ref.attend(q, c.keys, c.values, [0, new], [200], scale, scales=c.scales)
    assert close(attention(c, q, [0, new], [200], scale=scale), want, bound)


@pytest.mark.parametrize("new,window", [(1, 0), (3, 0), (90, 0), (5, 40), (150, 70)])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_values_that_are_nan(new, window, D):
    """NaN codes reach the rows that see their keys, in their columns, and no other; a scale that is NaN the rows that see a
    key of its page, in all columns."""
    L = 400
    c = ref.Cache([L], 2, D, 16, seed=20)
    for j, h, d in ((L - 1, 0, 3), (L - 2, 1, 0), (L - 60, 0, 9), (L - 75, 1, 47), (7, 0, 5)):
        c.v[int(c.table[0, j // 16]), h, j % 16, d] = 255 if d % 2 else 127
    q = torch.randn(new, 4, D, generator=torch.Generator().manual_seed(21)).to(torch.bfloat16)
    for page in (None, 23, 20):
        if page:
            c.vs[int(c.table[0, page]), 1] = 255
        want, bound = ref.attend(q.cuda(), c.keys, c.values, [0, new], [L], D ** -0.5, window, scales=c.scales)
        got = attention(c, q, [0, new], [L], window=window).double()
        want, bound = want.cpu(), bound.cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        fine = torch.isfinite(want)
        assert ((got - want).abs() <= bound)[fine].all() and not fine.all() and fine.any()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 40, 100])
def test_keys_that_are_nan_and_not_seen(D, new):
    """NaN keys (codes or a page's scale) after a row's position do not reach it, the others are NaN."""
    L = 300
    c = ref.Cache([L], 1, D, 16, seed=22)
    q = torch.randn(new, 2, D, generator=torch.Generator().manual_seed(23)).to(torch.bfloat16)
    want, bound = ref.attend(q.cuda(), c.keys, c.values, [0, new], [L], D ** -0.5, scales=c.scales)
    c.k[int(c.table[0, (L - 30) // 16]), :, (L - 30) % 16] = 127
    got = attention(c, q, [0, new], [L])
    sees = max(0, new - 30)
    assert torch.isnan(got[sees:]).all() and close(got[:sees], want[:sees], bound[:sees])
    c.k[int(c.table[0, (L - 30) // 16]), :, (L - 30) % 16] = 0
    c.ks[int(c.table[0, 18])] = 255  # positions 288 and on
    got = attention(c, q, [0, new], [L])
    sees = max(0, new - 12)
    want, bound = ref.attend(q.cuda(), c.keys, c.values, [0, new], [L], D ** -0.5, scales=c.scales)
    assert torch.isnan(got[sees:]).all() and close(got[:sees], want[:sees], bound[:sees])


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("new,others", [(3, 0), (60, 0), (100, 0)])
def test_queries_that_are_not_finite(D, new, others):
    """Such a row is NaN, the others are what they are without it."""
    c = ref.Cache([500], 1, D, 16, seed=24)
    q = torch.randn(new, 4, D, generator=torch.Generator().manual_seed(25)).to(torch.bfloat16)
    plain = attention(c, q, [0, new], [500])
    for x in (math.nan, math.inf, -math.inf):
        q[1, 2, 7] = x
        got = attention(c, q, [0, new], [500])
        assert torch.isnan(got[1, 2]).all()
        got[1, 2] = plain[1, 2]
        assert torch.equal(got, plain)


@pytest.mark.parametrize("new", [1, 90])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_queries_and_scales_of_all_sizes(new, D):
    """Queries whose values differ by 2^20, pages whose scales differ by 2^40 (values) and 2^10 (keys)."""
    L, block = 300, 16
    c = ref.Cache([L], 2, D, block, seed=26, spread=0.2)
    g = torch.Generator().manual_seed(27)
    pages = torch.from_numpy(c.table[0]).long()
    c.vs[pages] = torch.randint(90, 130, (len(pages), 2), generator=g, dtype=torch.uint8)
    c.ks[pages] = torch.randint(112, 122, (len(pages), 2), generator=g, dtype=torch.uint8)
    q = torch.randn(new, 4, D, generator=g) * 2.0 ** -torch.randint(0, 21, (D,), generator=g)
    q = q.to(torch.bfloat16)
    want, bound = ref.attend(q.cuda(), c.keys, c.values, [0, new], [L], D ** -0.5, scales=c.scales)
    assert close(attention(c, q, [0, new], [L]), want, bound)


@pytest.mark.parametrize("new", [1, 90])
@pytest.mark.parametrize("D,block", [(64, 16), (128, 8), (256, 16), (64, 5), (128, 7), (256, 12)])
def test_value_scales_far_apart(new, D, block):
    """Pages of values from 2^-67 to 2^62, some of all zeros at the smallest scale there is: what they take of a row's weight
    is what the scores say.  (No sum passes 2^62 * 448 * 60 keys of a tile, far from f32's end.)"""
    L = 300
    c = ref.Cache([L], 2, D, block, seed=28, spread=0.2)
    g = torch.Generator().manual_seed(29)
    pages = torch.from_numpy(c.table[0]).long()
    c.vs[pages] = torch.randint(60, 190, (len(pages), 2), generator=g, dtype=torch.uint8)
    c.v[pages[::3]], c.vs[pages[::3]] = 0, 0
    q = torch.randn(new, 4, D, generator=g).to(torch.bfloat16)
    want, bound = ref.attend(q.cuda(), c.keys, c.values, [0, new], [L], D ** -0.5, scales=c.scales)
    assert close(attention(c, q, [0, new], [L]), want, bound)
    # nothing but zeros and one page: its share
    c.v[pages], c.vs[pages] = 0, 0
    c.v[pages[4]], c.vs[pages[4]] = 0x38, 127  # 1
    want, bound = ref.attend(q.cuda(), c.keys, c.values, [0, new], [L], D ** -0.5, scales=c.scales)
    assert close(attention(c, q, [0, new], [L]), want, bound)


@pytest.mark.parametrize("Hq,D,new", [(4, 256, 1), (10, 256, 3), (8, 128, 1), (8, 128, 4), (6, 64, 1), (7, 64, 4), (3, 80, 2)])
@pytest.mark.parametrize("L", [40, 700, 5000])
def test_weights_of_few_rows(Hq, D, new, L):
    """Values that nearly cancel, so that the result's own rounding hides nothing: few rows' weights lose 2^-16."""
    c = ref.Cache([L], 1, D, 16, seed=L, spread=0.0)
    x = torch.randn(D, generator=torch.Generator().manual_seed(L + D)).to(torch.bfloat16)
    q = x.expand(new, Hq, D).contiguous()
    for page in c.table[0]:  # the same value of either sign, by turns
        c.v[int(page), :, 0::2] = 0x38
        c.v[int(page), :, 1::2] = 0xB8
        c.vs[int(page)] = 127
    want, bound = ref.attend(q.cuda(), c.keys, c.values, [0, new], [L], D ** -0.5, few=True)
    assert close(attention(c, q, [0, new], [L]), want, bound)


@pytest.mark.parametrize("new", [1, 3, 90])
def test_past_32_bit_offsets(new):
    """Pages at both ends of a cache of 2^32 bytes and more."""
    Hkv, D, block = 4, 256, 16
    NB = 2 ** 32 // (Hkv * D * block) + 40
    k, v = (torch.empty(NB, Hkv, block, D, dtype=torch.uint8, device="cuda") for _ in range(2))
    ks, vs = (torch.full((NB, Hkv), 255, dtype=torch.uint8, device="cuda") for _ in range(2))
    c = ref.Cache([300], Hkv, D, block, seed=10)
    pages = [p if p % 2 else NB - 1 - p for p in range(c.table.shape[1])]
    for i, p in enumerate(pages):
        for big, small in ((k, c.k), (v, c.v), (ks, c.ks), (vs, c.vs)):
            big[p] = small[int(c.table[0, i])].cuda()
    q = torch.randn(new, 8, D, generator=torch.Generator().manual_seed(11)).to(torch.bfloat16)
    want, bound = ref.attend(q, c.keys, c.values, [0, new], [300], 1 / 16, scales=c.scales)
    got = host(Q.paged_attention_fp8(dev(q), *[Q.Array.from_torch(t) for t in (k, v, ks, vs)], ints([pages]), ints([0, new]),
                                     ints([300]), scale=1 / 16))
    assert close(got, want, bound)


def test_many_requests():
    """More requests than a wave has lanes, more tiles than a workgroup has threads; contexts cut in many parts."""
    g = torch.Generator().manual_seed(30)
    for R, most, D, Hq, Hkv in ((300, 200, 64, 4, 2), (70, 90, 128, 8, 2), (2, 40000, 128, 4, 1)):
        kv = torch.randint(0, most, (R,), generator=g).tolist()
        kv[0] = most
        new = [min(k, 1 + (r % 50 == 7) * 40) for r, k in enumerate(kv)]
        c = ref.Cache(kv, Hkv, D, 16, seed=31)
        q = torch.randn(sum(new), Hq, D, generator=g).to(torch.bfloat16)
        want, bound = ref.attend(q.cuda(), c.keys, c.values, starts_of(new), kv, D ** -0.5, scales=c.scales)
        assert close(attention(c, q, starts_of(new), kv), want, bound), R


def test_two_streams_at_once_and_in_place():
    """Long contexts, whose parts meet in the stream's workspace; results over the queries and over the gate."""
    D = 128
    c = ref.Cache([9000, 3000], 2, D, 16, seed=12)
    g = torch.Generator().manual_seed(13)
    q, gate = (torch.randn(2, 8, D, generator=g).to(torch.bfloat16) for _ in range(2))
    want, bound = ref.attend(q.cuda(), c.keys, c.values, [0, 1, 2], [9000, 3000], D ** -0.5, gate=gate.cuda(), scales=c.scales)
    cache = [dev(t) for t in (c.k, c.v, c.ks, c.vs)]
    rest = [ints(c.table), ints([0, 1, 2]), ints([9000, 3000])]
    a, w = dev(q), dev(gate)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    wrapped = [Q.Stream(s.cuda_stream) for s in streams]
    outs = [[Q.paged_attention_fp8(a, *cache, *rest, gate=w, scale=D ** -0.5, stream=s) for s in wrapped] for _ in range(10)]
    for s in wrapped:
        s.sync()
    first = host(outs[0][0])
    assert close(first, want, bound) and all(torch.equal(host(o), first) for pair in outs for o in pair)
    for out in (0, 1):
        a, w = dev(q), dev(gate)
        over = Q.paged_attention_fp8(a, *cache, *rest, gate=w, scale=D ** -0.5, out=(a, w)[out])
        assert torch.equal(host(over), first)
