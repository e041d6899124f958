"""Writes into a cache held in 8 bits, and reading it back, against plain restatements in 64 bits (fp8_ref.py)."""
import math
from ctypes import byref

import attention_ref
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
    n = a.numpy()
    return torch.from_numpy(n.view(np.int16)).view(torch.bfloat16) if a.dtype == Q.BFLOAT16 else torch.from_numpy(n)


def some_cache(P, H, block, D, seed):
    """Codes and scales of values of all sizes."""
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (P, H, block, D), generator=g, dtype=torch.uint8)
    return codes, torch.randint(110, 124, (P, H), generator=g, dtype=torch.uint8)


class Written:
    """The caches before and after a call."""

    def __init__(self, q, k, v, slots, positions, freqs, P, block, seed=1, cache=None, **kw):
        H, D = k.shape[1], k.shape[2]
        self.k, self.ks = cache[:2] if cache else some_cache(P, H, block, D, seed)
        self.v, self.vs = cache[2:] if cache else some_cache(P, H, block, D, seed + 1)
        on = [t.clone().cuda() for t in (self.k, self.v, self.ks, self.vs)]
        norms = {n: dev(kw.pop(n)) for n in ("q_norm", "k_norm") if kw.get(n) is not None}
        kw.pop("q_norm", None), kw.pop("k_norm", None)
        self.q = host(Q.rope_cache_fp8(dev(q), dev(k), dev(v), *[Q.Array.from_torch(t) for t in on], ints(positions), ints(slots),
                                       dev(freqs), **norms, **kw))
        torch.cuda.synchronize()
        self.k1, self.v1, self.ks1, self.vs1 = [t.cpu() for t in on]


def runs(lens, block, P, seed, gaps=False):
    """Slots and positions of requests' new tokens ((cached, new) each), pages in no order; gaps: rows without a slot between."""
    order, slots, pos, at = np.random.default_rng(seed).permutation(P).tolist(), [], [], 0
    for c, n in lens:
        first, last = c // block, (c + n - 1) // block
        pages = order[at:at + last - first + 1]
        at += len(pages)
        assert at <= P
        slots += [pages[p // block - first] * block + p % block for p in range(c, c + n)]
        pos += list(range(c, c + n))
        if gaps:
            slots += [-1, P * block, -7]
            pos += [0, 5, 9]
    return slots, pos


WRITES = [
    # (cached, new) of each request, Hq, Hkv, D, Dq, rotated, block
    ([(0, 1)], 6, 2, 256, 512, 64, 16),
    ([(7, 1)], 1, 1, 16, 16, 16, 1),
    ([(5, 40)], 4, 2, 256, 256, 256, 16),
    ([(c, 1 + c % 3) for c in range(0, 66, 2)], 8, 2, 128, 136, 64, 16),
    ([(30, 300), (0, 5), (64, 64)], 3, 3, 64, 64, 32, 64),
    ([(3, 700)], 2, 1, 256, 256, 32, 300),   # pages longer than a workgroup's turns
    ([(11, 90)], 5, 5, 96, 96, 48, 7),
    ([(0, 33), (33, 2)], 12, 4, 80, 160, 12, 24),
    ([(100, 17)], 4, 2, 208, 208, 0, 32),
    ([(0, 260)], 2, 2, 32, 64, 20, 1),
]


@pytest.mark.parametrize("lens,Hq,Hkv,D,Dq,rot,block", WRITES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("norm", [None, torch.bfloat16, torch.float32])
def test_write(lens, Hq, Hkv, D, Dq, rot, block, interleaved, dtype, norm):
    """Values are written as they are: their codes and scales bit for bit.  Keys, of their norm and rotation in 64 bits, to a
    code's rounding (2^-4 of the value; where subnormal half a step, 2^-10 of the scale) and the f32 arithmetic before it (24
    roundings of 2^-24 and D / 4 of the norm's sum, of what goes into a value); a page's scale exactly, but where such an error
    of its largest value passes a border.  Queries are rope_cache's, bit for bit."""
    g = torch.Generator().manual_seed(D + rot + len(lens))
    P = sum((c + n - 1) // block - c // block + 1 for c, n in lens) + 3
    slots, pos = runs(lens, block, P, seed=D, gaps=len(lens) > 1)
    T = len(slots)
    q, k, v = (torch.randn(T, h, d, generator=g).to(dtype) for h, d in ((Hq, Dq), (Hkv, D), (Hkv, D)))
    k = k * torch.exp(torch.randn(Hkv, D, generator=g)).to(dtype)
    freqs = torch.from_numpy(Q.rope_frequencies(rot, 1e5)[0]) if rot else torch.zeros(0)
    w = {n: (1 + 0.2 * torch.randn(D, generator=g)).to(norm) for n in ("q_norm", "k_norm")} if norm else {}
    out = Written(q, k, v, slots, pos, freqs, P, block, amplitude=1.1, interleaved=interleaved, **w)

    codes, scales, _ = ref.store(out.v, out.vs, slots, v.double())
    assert torch.equal(out.vs1, scales) and ref.same(out.v1, codes).all()

    y, eps = k.double(), (24 + D / 4) * 2 ** -24
    if norm:
        y = y * (y.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w["k_norm"].double()
    y, size = attention_ref.turn(y, torch.tensor(pos), freqs, float(np.float32(1.1)), interleaved)
    codes, scales, tops = ref.store(out.k, out.ks, slots, y)
    for (page, h), top in tops.items():
        if out.ks1[page, h] != scales[page, h]:
            near = {ref.exponent(top * (1 - 2 * D * eps)), ref.exponent(top * (1 + 2 * D * eps))}
            assert len(near) > 1 and int(out.ks1[page, h]) - 127 in near
    got, old = ref.decode(out.k1, out.ks1), ref.decode(out.k, out.ks)
    begun = set()
    for i, s in enumerate(slots):
        if 0 <= s < P * block:
            page, off = divmod(s, block)
            begun.add(page)
            t = 2.0 ** (out.ks1[page].double() - 127)[:, None]
            assert ((got[page, :, off] - y[i]).abs() <= 2 ** -4 * y[i].abs() + 2 ** -10 * t + 1.1 * eps * size[i]).all()
    rest = [p for p in range(P) if p not in begun]
    assert torch.equal(out.k1[rest], out.k[rest]) and torch.equal(out.ks1[rest], out.ks[rest])
    same_scale = out.ks1 == scales
    mine = torch.zeros(P * block, dtype=torch.bool)
    mine[[s for s in slots if 0 <= s < P * block]] = True
    others = ~mine.view(P, block)
    assert ref.same(out.k1, codes)[(same_scale[:, :, None] & others[:, None]).expand(-1, -1, block)].all()  # older rows, moved to the page's scale
    assert old.shape == got.shape

    as_before = Q.rope_cache(dev(q), dev(k), dev(v), *[dev(torch.zeros(P, Hkv, block, D, dtype=torch.bfloat16)) for _ in range(2)],
                             ints(pos), ints(slots), dev(freqs), amplitude=1.1, interleaved=interleaved,
                             **{n: dev(x) for n, x in w.items()})
    assert torch.equal(out.q, host(as_before))


@pytest.mark.parametrize("lens,Hq,Hkv,D,Dq,rot,block", [
    # tokens enough, and pages long enough, for the wide workgroups
    ([(30, 500), (0, 70), (100, 64)], 4, 2, 256, 512, 64, 40),
    ([(5, 600)], 2, 2, 128, 128, 128, 66),
    ([(90, 520), (0, 1)], 3, 3, 64, 64, 64, 160),
    ([(c, 1 + c % 3) for c in range(0, 620, 2)], 2, 2, 256, 256, 256, 36),
    ([(17, 540)], 1, 1, 32, 40, 16, 130),
    ([(0, 1100)], 1, 3, 208, 208, 0, 1000),
])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("norm", [None, torch.float32])
def test_write_to_long_pages(lens, Hq, Hkv, D, Dq, rot, block, interleaved, dtype, norm):
    test_write(lens, Hq, Hkv, D, Dq, rot, block, interleaved, dtype, norm)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rot", [64, 20])
def test_keys_are_the_codes_of_the_rotation(rot, interleaved):
    """Keys of `rope`, whose f32 results are those that are quantised: codes and scales bit for bit."""
    T, H, D, block, P = 75, 2, 128, 16, 9
    g = torch.Generator().manual_seed(rot)
    k = torch.randn(T, H, D, generator=g)
    slots, pos = runs([(5, T)], block, P, seed=2)
    freqs = torch.from_numpy(Q.rope_frequencies(rot, 1e4)[0])
    y = host(Q.rope(dev(k), ints(pos), dev(freqs), interleaved=interleaved))
    out = Written(k, k, k, slots, pos, freqs, P, block, interleaved=interleaved)
    codes, scales, _ = ref.store(out.k, out.ks, slots, y.double())
    assert torch.equal(out.ks1, scales) and ref.same(out.k1, codes).all()


def write_v(cache, slots, v):
    """One call's values (and the same as keys, unturned) into `cache` = (codes, scales)."""
    k = cache[0].clone(), cache[1].clone()
    q = torch.zeros(len(slots), 1, v.shape[2], dtype=v.dtype)
    out = Written(q, v, v, slots, [0] * len(slots), torch.zeros(0), cache[0].shape[0], cache[0].shape[2], cache=(*k, *cache))
    assert ref.same(out.k1, out.v1).all() and torch.equal(out.ks1, out.vs1)
    return out.v1, out.vs1


@pytest.mark.parametrize("D,block", [(256, 16), (64, 5), (128, 48)])
def test_a_page_over_many_calls(D, block):
    """Tokens one at a time and a few, of sizes that rise and fall: every call against the restatement, whose older codes
    follow the scale."""
    g = torch.Generator().manual_seed(block)
    got = want = some_cache(3, 2, block, D, seed=3)
    at = 0
    while at < 2 * block:
        n = int(torch.randint(1, 4, (1,), generator=g))
        n = min(n, 2 * block - at)
        v = torch.randn(n, 2, D, generator=g) * 2.0 ** float(torch.randint(-6, 7, (1,), generator=g))
        slots = [[2, 0][(at + i) // block] * block + (at + i) % block for i in range(n)]
        got = write_v(got, slots, v)
        want = ref.store(*want, slots, v.double())[:2]
        assert torch.equal(got[1], want[1]) and ref.same(got[0], want[0]).all(), at
        at += n


def test_growth_of_every_code_by_every_amount():
    """A page that holds every code, and a row that makes its scale grow by 1 to 30 and by the most there is."""
    D, block = 256, 16
    for by in [*range(1, 31), 200, 247]:
        codes = torch.arange(256, dtype=torch.uint8).repeat(block).view(1, 1, block, D)
        scales = torch.zeros(1, 1, dtype=torch.uint8)
        v = torch.zeros(1, 1, D)
        v[0, 0, 0] = min(448.0 * 2.0 ** (by - 127), 3.3e38)
        got = write_v((codes, scales), [3], v)
        want = ref.store(codes, scales, [3], v.double())
        assert int(got[1]) == int(want[1]) == by and ref.same(got[0], want[0]).all(), by


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_extreme_values(dtype):
    """Zeros, the smallest and largest there are, borders of the scale, infinities and NaN (which become NaN, and do not
    count for the scale)."""
    D = 32
    rows = [torch.zeros(D), torch.full((D,), 1e-45 if dtype == torch.float32 else 1e-40), torch.full((D,), 3.38e38),
            torch.linspace(-448, 448, D), torch.linspace(-449, 449, D), torch.tensor([math.inf, -math.inf, math.nan, 5.0] * 8),
            torch.full((D,), math.nan), torch.tensor([2.0 ** -e for e in range(D)]), torch.tensor([-0.0, 1.0] * 16),
            torch.tensor([3e-39, 1e-38] * 16), torch.tensor([1.75, 1.7501] * 16) * 2.0 ** -130, torch.full((D,), 448 * 2.0 ** -127)]
    v = torch.stack(rows)[:, None].to(dtype)
    for block in (1, 4):
        n = len(rows)
        cache = some_cache(n, 1, block, D, seed=5)
        cache[1][1] = 255  # a scale that is NaN: another call's page starts anew
        slots = [i * block for i in range(n)]
        got = write_v(cache, slots, v)
        want = ref.store(*cache, slots, v.double())
        assert torch.equal(got[1], want[1]), (got[1].T, want[1].T)
        for i, s in enumerate(slots):
            assert ref.same(got[0][i, 0, 0], want[0][i, 0, 0]).all(), i


def test_rows_without_a_slot_and_pages_that_are_none():
    D, P, block = 64, 4, 16
    cache = some_cache(P, 2, block, D, seed=6)
    v = torch.randn(5, 2, D)
    got = write_v(cache, [-1, P * block, 2 ** 31 - 1, -2 ** 31, -16], v)
    assert torch.equal(got[0], cache[0]) and torch.equal(got[1], cache[1])
    got = write_v(cache, [-1, 17, 18, -1, 40], v)
    want = ref.store(*cache, [-1, 17, 18, -1, 40], v.double())
    assert torch.equal(got[1], want[1]) and ref.same(got[0], want[0]).all()
    e = torch.zeros(0, 2, D)
    assert write_v(cache, [], e)[0].equal(cache[0])


def test_a_scale_that_is_nan_stays_until_its_page_starts_anew():
    D, block = 64, 16
    codes, scales = some_cache(2, 1, block, D, seed=7)
    scales[:] = 255
    v = torch.randn(1, 1, D)
    got = write_v((codes, scales), [5], v)
    assert (got[1] == 255).all()
    got = write_v(got, [0], v)
    assert got[1][0, 0] != 255 and got[1][1, 0] == 255


# ---------------------------------------------------------------- reading back


@pytest.mark.parametrize("D,H,block", [(256, 2, 16), (64, 3, 5), (16, 1, 1), (80, 40, 24), (208, 5, 7), (128, 300, 2)])
@pytest.mark.parametrize("dtype", [Q.BFLOAT16, Q.FLOAT32])
@pytest.mark.parametrize("T", [1, 70])
def test_read(D, H, block, dtype, T):
    """Every value: the code times its scale, exact in f32, rounded once in bf16 (only what underflows is)."""
    P = 9
    g = torch.Generator().manual_seed(D)
    caches = [torch.randint(0, 256, (P, H, block, D), generator=g, dtype=torch.uint8) for _ in range(2)]
    scales = [torch.randint(0, 250, (P, H), generator=g, dtype=torch.uint8) for _ in range(2)]
    scales[0][2] = 255
    slots = torch.randint(0, P * block, (T,), generator=g).tolist()
    if T > 3:
        slots[1], slots[2], slots[3], slots[9] = -1, P * block, -2 ** 31, 2 ** 31 - 1
    got = Q.cache_read_fp8(*[dev(t) for t in caches + scales], ints(slots), dtype=dtype)
    for a, codes, s in zip(got, caches, scales):
        a = host(a)
        wide = ref.decode(codes, s)
        want = torch.stack([wide[i // block, :, i % block] if 0 <= i < P * block else torch.zeros(H, D, dtype=torch.float64) for i in slots])
        want = want.float().to(a.dtype)
        assert a.shape == (T, H, D) and torch.equal(torch.isnan(a), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(a), torch.nan_to_num(want))


@pytest.mark.parametrize("dtype", [Q.BFLOAT16, Q.FLOAT32])
def test_read_every_code_at_every_scale(dtype):
    codes = torch.arange(256, dtype=torch.uint8).view(1, 1, 1, 256).repeat(256, 1, 1, 1)
    scales = torch.arange(256, dtype=torch.uint8).view(256, 1)
    k, v = Q.cache_read_fp8(dev(codes), dev(codes), dev(scales), dev(scales), ints(range(256)), dtype=dtype)
    k, v = host(k), host(v)
    want = ref.decode(codes, scales)[:, :, 0].float().to(k.dtype)
    for got in (k, v):
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(got, 0), torch.nan_to_num(want, 0))


def test_read_one_side_and_in_place():
    codes, scales = some_cache(4, 2, 8, 64, seed=8)
    slots = [3, 9, 31]
    want = ref.decode(codes, scales)[[0, 1, 3], :, [3, 1, 7]].float().to(torch.bfloat16)
    null = Q.qmm_array(None)
    c, s, i = dev(codes), dev(scales), ints(slots)
    stream = Q.Stream()
    for side in (0, 1):
        out = Q.Array()
        a = [byref(out.h), None] if side == 0 else [None, byref(out.h)]
        h = [c.h, null, s.h, null] if side == 0 else [null, c.h, null, s.h]
        assert Q.lib.qmm_cache_read_fp8(*a, *h, i.h, Q.BFLOAT16, stream.h) == 0
        assert torch.equal(torch.nan_to_num(host(out)), torch.nan_to_num(want))
    k, v = (Q.Array.from_torch(torch.zeros(3, 2, 64, device="cuda")) for _ in range(2))
    at = k.ptr, v.ptr
    Q.cache_read_fp8(c, c, s, s, i, dtype=Q.FLOAT32, k_out=k, v_out=v)
    assert (k.ptr, v.ptr) == at and torch.equal(torch.nan_to_num(host(k)), torch.nan_to_num(want.float()))
    assert Q.cache_read_fp8(c, c, s, s, ints([]))[0].shape == (0, 2, 64)


def test_past_32_bit_offsets():
    """Pages at both ends of a cache of over 2^32 bytes: written, and read back."""
    H, D, block = 4, 256, 16
    P = 2 ** 32 // (H * D * block) + 40
    codes = [torch.empty(P, H, block, D, dtype=torch.uint8, device="cuda") for _ in range(2)]
    scales = [torch.full((P, H), 100, dtype=torch.uint8, device="cuda") for _ in range(2)]
    cache = [Q.Array.from_torch(t) for t in codes + scales]
    x = torch.randn(2 * block, H, D, generator=torch.Generator().manual_seed(9)).to(torch.bfloat16)
    slots = [*range((P - 1) * block, P * block), *range(block)]
    Q.rope_cache_fp8(dev(x), dev(x), dev(-x), *cache, ints(range(2 * block)), ints(slots), dev(torch.zeros(0)))
    k, v = Q.cache_read_fp8(*cache, ints(slots), dtype=Q.FLOAT32)
    small = torch.zeros(2, H, block, D, dtype=torch.uint8), torch.zeros(2, H, dtype=torch.uint8)
    c, s, _ = ref.store(*small, list(range(2 * block)), x.double())
    want = ref.decode(c, s).transpose(1, 2).reshape(-1, H, D).float()
    assert torch.equal(host(k), want) and torch.equal(host(v), -want)


def test_two_streams_and_a_graph():
    """Writes into one layer's cache and another's at once; a captured write and read, replayed with other inputs."""
    D, H, P, block, T = 128, 2, 40, 16, 200
    g = torch.Generator().manual_seed(10)
    xs = [torch.randn(T, H, D, generator=g).to(torch.bfloat16) for _ in range(6)]
    slots, pos = runs([(3, T)], block, P, seed=11)
    start = some_cache(P, H, block, D, seed=12)
    want = [ref.store(*start, slots, x.double())[:2] for x in xs]
    f, i, p = dev(torch.zeros(0)), ints(slots), ints(pos)
    torch.cuda.synchronize()
    for pair in range(3):
        held = []
        for x, s in zip(xs[2 * pair:], (torch.cuda.Stream(), torch.cuda.Stream())):
            on = [t.clone().cuda() for t in (start[0], start[0], start[1], start[1])]
            a = dev(x)
            torch.cuda.synchronize()
            Q.rope_cache_fp8(a, a, a, *[Q.Array.from_torch(t) for t in on], p, i, f, stream=Q.Stream(s.cuda_stream))
            held.append((on, a, s))
        torch.cuda.synchronize()
        for (on, _, _), w in zip(held, want[2 * pair:]):
            assert torch.equal(on[2].cpu(), w[1]) and ref.same(on[0].cpu(), w[0]).all() and ref.same(on[1].cpu(), w[0]).all()
    x = torch.zeros(T, H, D, dtype=torch.bfloat16, device="cuda")
    on = [t.clone().cuda() for t in (start[0], start[0], start[1], start[1])]
    a, cache = Q.Array.from_torch(x), [Q.Array.from_torch(t) for t in on]
    qo, k, v = (Q.Array.from_torch(torch.empty(T, H, D, dtype=torch.bfloat16, device="cuda")) for _ in range(3))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        st = Q.Stream.torch_current()
        Q.rope_cache_fp8(a, a, a, *cache, p, i, f, q_out=qo, stream=st)
        Q.cache_read_fp8(*cache, i, k_out=k, v_out=v, stream=st)
    for y, w in zip(xs, want):
        for t, s in zip(on, (start[0], start[0], start[1], start[1])):
            t.copy_(s)
        x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(on[2].cpu(), w[1]) and ref.same(on[0].cpu(), w[0]).all()
        rows = ref.decode(*w)[[s // block for s in slots], :, [s % block for s in slots]].to(torch.bfloat16)
        assert torch.equal(torch.nan_to_num(host(k)), torch.nan_to_num(rows))


@pytest.mark.parametrize("D,rot", [(128, 128), (256, 64)])
def test_a_captured_write_to_long_pages(D, rot):
    """The wide workgroups, captured first (their LDS passes what a kernel has unasked where all of a head turns): every replay
    the eager call's codes and scales, from the same cache, with other work between."""
    H, P, block, T = 2, 12, 80, 600
    g = torch.Generator().manual_seed(13)
    slots, pos = runs([(30, T)], block, P, seed=14)
    xs = [torch.randn(T, H, D, generator=g).to(torch.bfloat16) for _ in range(3)]
    start = some_cache(P, H, block, D, seed=15)
    f, i, p = dev(torch.from_numpy(Q.rope_frequencies(rot, 1e5)[0])), ints(slots), ints(pos)
    x = torch.zeros(T, H, D, dtype=torch.bfloat16, device="cuda")
    on, eager = ([t.clone().cuda() for t in (start[0], start[0], start[1], start[1])] for _ in range(2))
    a, qo, q1 = Q.Array.from_torch(x), *(dev(torch.zeros(T, H, D, dtype=torch.bfloat16)) for _ in range(2))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        Q.rope_cache_fp8(a, a, a, *[Q.Array.from_torch(t) for t in on], p, i, f, q_out=qo, stream=Q.Stream.torch_current())
    for y in xs:
        for to in (on, eager):
            for t, s in zip(to, (start[0], start[0], start[1], start[1])):
                t.copy_(s)
        x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        Q.rope_cache_fp8(a, a, a, *[Q.Array.from_torch(t) for t in eager], p, i, f, q_out=q1, stream=Q.Stream.torch_current())
        torch.cuda.synchronize()
        assert all(torch.equal(s, t) for s, t in zip(on, eager)) and torch.equal(host(qo), host(q1))
        codes, scales, _ = ref.store(start[0], start[1], slots, y.double())
        assert torch.equal(on[3].cpu(), scales) and ref.same(on[1].cpu(), codes).all()
