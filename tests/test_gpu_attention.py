"""Block tables, rotary positions, cache writes and paged attention on the GPU, against plain
restatements in 64 bits (attention_ref.py)."""
import math

import attention_ref as ref
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
    """A library array's contents as a torch tensor."""
    n = a.numpy()
    return torch.from_numpy(n.view(np.int16)).view(torch.bfloat16) if a.dtype == Q.BFLOAT16 else torch.from_numpy(n)


# ---------------------------------------------------------------- block tables

BLOCKS = [
    # R, W, block, most cached, most new, rows beyond the tokens, free pages short by
    (1, 1, 16, 0, 1, 0, 0),
    (1, 40, 1, 9, 20, 3, 0),
    (5, 8, 16, 60, 40, 0, 0),
    (64, 70, 16, 1000, 1, 0, 0),
    (300, 90, 7, 300, 200, 11, 0),
    (1030, 9, 24, 100, 60, 0, 0),
    (33, 20, 16, 200, 100, 0, 9),    # the list of free pages runs out
    (17, 5, 16, 200, 90, 0, 0),      # lengths past the table's width
    (9, 30, 16, 100, 300, -700, 0),  # more tokens than rows
    (4096, 3, 64, 100, 3, 5, 0),
]


@pytest.mark.parametrize("R,W,block,most,fresh,extra,short", BLOCKS)
@pytest.mark.parametrize("in_place", [False, True])
def test_block_tables(R, W, block, most, fresh, extra, short, in_place):
    rng = np.random.default_rng(R * 1000 + W)
    cached, new = rng.integers(0, most + 1, R), rng.integers(0, fresh + 1, R)
    if R > 4:
        cached[1], new[1], new[2], new[R - 1] = 0, 0, -5, 0
        cached[3] = -2
    T = max(0, int(np.maximum(new, 0).sum()) + extra)
    table = np.full((R, W), -1, dtype=np.int32)
    held = np.minimum(-(-np.maximum(cached, 0) // block), W)
    pages = rng.permutation(int(held.sum()) + R * (2 + fresh // block) + 10)
    at = 0
    for r in range(R):
        table[r, :held[r]] = pages[at:at + held[r]]
        at += held[r]
    free = pages[at:].astype(np.int32)
    need = ref.blocks(table, 2, cached, new, free, block, T)[1][0]
    if short:
        free = free[:need - short]
    want = ref.blocks(table, 2, cached, new, free, block, T)
    a = dict(table=ints(table), head=ints([2]), cached=ints(cached), new=ints(new), free=ints(free))
    own = dict(table_out=a["table"], head_out=a["head"], kv_lens=a["cached"]) if in_place else {}
    got = Q.block_tables(a["table"], a["head"], a["cached"], a["new"], a["free"], block, T, **own)
    for name, g, w in zip(("table", "head", "q_starts", "kv_lens", "positions", "slots"), got, want):
        assert np.array_equal(g.numpy(), w), name
    if not in_place:
        assert np.array_equal(a["table"].numpy(), table) and np.array_equal(a["cached"].numpy(), cached)


def test_block_tables_of_nothing():
    got = Q.block_tables(ints(np.zeros((0, 4))), ints([5]), ints([]), ints([]), ints([1, 2]), 16, 3)
    table, head, starts, kv, pos, slots = [g.numpy() for g in got]
    assert table.shape == (0, 4) and head.tolist() == [5] and starts.tolist() == [0] and kv.size == 0
    assert pos.tolist() == [0, 0, 0] and slots.tolist() == [-1, -1, -1]


def test_block_tables_near_the_largest_lengths():
    top = 2 ** 31 - 1
    got = Q.block_tables(ints([[3, 4]]), ints([0]), ints([top - 2]), ints([5]), ints([7]), 2 ** 30, 5)
    table, head, starts, kv, pos, slots = [g.numpy() for g in got]
    assert table.tolist() == [[3, 4]] and head.tolist() == [0] and starts.tolist() == [0, 5]
    assert kv.tolist() == [top] and pos.tolist() == [top - 2, top - 1, top, top, top]
    assert (slots == -1).all()  # page 4's slots pass an int32


# ---------------------------------------------------------------- rotary positions

HEADS = [(1, 1, 8, 8), (3, 2, 64, 64), (5, 3, 64, 20), (2, 24, 256, 64), (7, 5, 256, 256), (4, 2, 80, 80),
         (4, 3, 96, 48), (2, 9, 136, 34), (3, 1, 192, 2), (1025, 3, 128, 128), (2, 2, 128, 0)]


def positions_of(T, g):
    p = torch.randint(0, 262144, (T,), generator=g, dtype=torch.int32)
    p[0] = 0
    if T > 2:
        p[1], p[2] = 2 ** 31 - 1, -77
    return p


@pytest.mark.parametrize("T,H,D,rot", HEADS)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rope(T, H, D, rot, interleaved, dtype):
    g = torch.Generator().manual_seed(T * 7 + D)
    x, p = torch.randn(T, H, D, generator=g).to(dtype), positions_of(T, g)
    freqs = torch.from_numpy(Q.rope_frequencies(rot, 1e6)[0] if rot else np.zeros(0, dtype=np.float32))
    for transpose in (False, True):
        want, size = ref.turn(x, p, freqs, 1.25, interleaved, transpose)
        got = host(Q.rope(dev(x), ints(p), dev(freqs), amplitude=1.25, interleaved=interleaved, transpose=transpose))
        # f32: the angle (2^-26 turns), cos and sin (2 ulp), four roundings; then the result's own in bf16
        bound = size * 2 ** -21 + (want.abs() * 2 ** -8 if dtype == torch.bfloat16 else 0)
        assert ((got.double() - want).abs() <= bound).all()
        assert torch.equal(got[..., rot:], x[..., rot:])
    xd = dev(x)
    into = Q.rope(xd, ints(p), dev(freqs), amplitude=1.25, interleaved=interleaved, transpose=True, out=xd)
    assert into is xd and torch.equal(host(xd), got)  # in place, the same bits


def test_rope_of_leading_dimensions_and_none():
    x = torch.randn(2, 3, 4, 16)
    p, f = torch.arange(6, dtype=torch.int32), torch.tensor([1.0, 0.5])
    y = host(Q.rope(dev(x), ints(p), dev(f)))
    flat = host(Q.rope(dev(x.view(6, 4, 16)), ints(p), dev(f)))
    assert y.shape == x.shape and torch.equal(y.view(6, 4, 16), flat)
    assert Q.rope(dev(torch.zeros(0, 4, 16)), ints([]), dev(f)).shape == (0, 4, 16)


def test_rope_transpose_is_the_gradient():
    """<R x, y> = <x, R^T y>, and differences of <R x, y> along each coordinate of one head."""
    g = torch.Generator().manual_seed(5)
    x, y = torch.randn(3, 2, 32, generator=g), torch.randn(3, 2, 32, generator=g)
    p, f = ints([3, 1000, 77777]), dev(torch.from_numpy(Q.rope_frequencies(24, 1e4)[0]))
    fwd = lambda v: host(Q.rope(dev(v), p, f, amplitude=1.5)).double()  # noqa: E731
    grad = host(Q.rope(dev(y), p, f, amplitude=1.5, transpose=True)).double()
    total = float((fwd(x) * y).sum())
    assert abs(total - float((grad * x).sum())) < 1e-4
    for d in range(32):
        e = torch.zeros_like(x)
        e[1, 1, d] = 1.0  # (linear: a difference of 1 has no truncation error)
        assert abs(float((fwd(x + e) * y).sum()) - total - float(grad[1, 1, d])) < 1e-4


# ---------------------------------------------------------------- norms, rotation and the cache's rows

WRITES = [  # T, Hq, Hkv, D, Dq, rot, block
    (1, 24, 4, 256, 512, 64, 16), (3, 24, 4, 256, 512, 64, 16), (5, 1, 1, 8, 8, 8, 1), (40, 6, 3, 80, 88, 80, 7),
    (17, 16, 16, 64, 64, 32, 24), (1100, 4, 2, 128, 128, 128, 64), (9, 12, 2, 96, 192, 36, 16),
]


@pytest.mark.parametrize("T,Hq,Hkv,D,Dq,rot,block", WRITES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("norm", [None, torch.bfloat16, torch.float32])
def test_rope_cache(T, Hq, Hkv, D, Dq, rot, block, interleaved, dtype, norm):
    g = torch.Generator().manual_seed(T + D)
    q, k, v = (torch.randn(T, h, d, generator=g).to(dtype) for h, d in ((Hq, Dq), (Hkv, D), (Hkv, D)))
    if T > 2:
        k[2] = 0  # the norm of nothing
    freqs, p = torch.from_numpy(Q.rope_frequencies(rot, 1e7)[0]), positions_of(T, g)
    NB = -(-T // block) + 2
    slots = torch.randperm(NB * block, generator=g)[:T].int()
    if T > 4:
        slots[1], slots[3], slots[4] = -1, NB * block, 2 ** 31 - 1  # rows that are not written
    kc, vc = (torch.randn(NB, Hkv, block, D, generator=g).to(torch.bfloat16) for _ in range(2))
    w = [None, None] if norm is None else [(1 + 0.2 * torch.randn(D, generator=g)).to(norm) for _ in range(2)]
    want = []
    for x, wt in ((q[..., :D], w[0]), (k, w[1])):
        x = x.double()
        if wt is not None:
            x = x / (x.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * wt.double()
        y, size = ref.turn(x, p, freqs, 1.0, interleaved)
        # as in test_rope, and the norm: a sum of 256 squares in a tree, a root, a quotient, two products
        want.append((y, y.abs() * 2 ** -8 + size * (2 ** -21 + 2 ** -19)))
    a = [dev(x) for x in (q, k, v, kc, vc)]
    got = host(Q.rope_cache(*a, ints(p), ints(slots), dev(freqs), interleaved=interleaved,
                            q_norm=dev(w[0]) if w[0] is not None else None,
                            k_norm=dev(w[1]) if w[1] is not None else None))
    assert ((got.double() - want[0][0]).abs() <= want[0][1]).all()
    rows = lambda c: c.transpose(1, 2).reshape(NB * block, Hkv, D)  # noqa: E731
    k_rows, v_rows = rows(host(a[3])), rows(host(a[4]))
    ok = (slots >= 0) & (slots < NB * block)
    at = slots[ok].long()
    assert ((k_rows[at].double() - want[1][0][ok]).abs() <= want[1][1][ok]).all()
    assert torch.equal(v_rows[at], v[ok].to(torch.bfloat16))
    others = torch.ones(NB * block, dtype=torch.bool)
    others[at] = False
    assert torch.equal(k_rows[others], rows(kc)[others]) and torch.equal(v_rows[others], rows(vc)[others])


# ---------------------------------------------------------------- attention

ATTEND = [  # Hq, Hkv, D, block, [(cached, new)], window
    (1, 1, 8, 16, [(0, 1)], 0),
    (24, 4, 256, 16, [(1998, 1)], 0),
    (24, 4, 256, 16, [(700, 3), (0, 3), (31, 3)], 0),
    (24, 4, 256, 16, [(300, 100)], 0),
    (24, 4, 256, 64, [(63, 1), (64, 1), (0, 65)], 0),
    (32, 8, 128, 16, [(0, 1), (1, 1), (15, 1), (16, 1), (500, 1), (4000, 1)], 0),
    (32, 8, 128, 7, [(100, 1), (3, 70), (0, 0), (40, 0), (259, 2)], 0),
    (16, 16, 64, 24, [(0, 130), (77, 1), (5, 33)], 0),
    (16, 16, 64, 24, [(0, 130), (777, 1), (500, 33)], 50),
    (8, 1, 256, 1, [(200, 4), (0, 20)], 0),
    (40, 8, 80, 32, [(90, 12), (1000, 1)], 0),
    (12, 12, 96, 16, [(64, 64), (0, 31)], 100),
    (6, 2, 136, 16, [(130, 5), (64, 64)], 0),
    (4, 4, 192, 128, [(300, 40)], 0),
    (28, 4, 128, 16, [(513, 9), (0, 300)], 0),
    (64, 1, 64, 16, [(100, 3), (33, 1)], 0),
    (2, 2, 32, 16, [(2500, 1), (100, 70)], 1),
    (5, 1, 72, 3, [(11, 6)] * 40, 4),
    (2, 2, 56, 16, [(0, 130)], 0),
    (3, 1, 120, 16, [(64, 64)], 1),
    (4, 2, 64, 16, [(100, 60), (9, 3)], 2 ** 31 - 1),
]


def attention(c, q, starts, kv, **kw):
    """Q.paged_attention of a Cache."""
    kw.setdefault("scale", q.shape[-1] ** -0.5)
    gate = kw.pop("gate", None)
    return host(Q.paged_attention(dev(q), dev(c.k), dev(c.v), ints(c.table), ints(starts), ints(kv),
                                  gate=dev(gate) if gate is not None else None, **kw))


def starts_of(new):
    return [0] + np.cumsum(new).tolist()


@pytest.mark.parametrize("Hq,Hkv,D,block,lens,window", ATTEND)
@pytest.mark.parametrize("gated", [False, True])
def test_attention(Hq, Hkv, D, block, lens, window, gated):
    new, kv = [n for _, n in lens], [c + n for c, n in lens]
    T, g = sum(new), torch.Generator().manual_seed(D + T_seed(lens))
    c = ref.Cache(kv, Hkv, D, block, seed=D)
    q = (2 * torch.randn(T, Hq, D, generator=g)).to(torch.bfloat16)
    gate = torch.randn(T, Hq, 2 * D, generator=g).to(torch.bfloat16) if gated else None
    want, bound = ref.attend(q, c.keys, c.values, starts_of(new), kv, D ** -0.5, window,
                             gate[..., D:] if gated else None)
    got = attention(c, q, starts_of(new), kv, window=window, gate=gate)
    assert torch.isfinite(got).all()
    assert ((got.double() - want).abs() <= bound).all()
    assert torch.equal(got, attention(c, q, starts_of(new), kv, window=window, gate=gate))  # the same bits again


def T_seed(lens):
    return sum(a * 31 + b for a, b in lens)


def test_attention_rows_that_see_nothing():
    """Rows before the first key, requests without keys, rows of no request."""
    D, new, kv = 64, [5, 3, 70, 2], [2, 0, 40, 9]
    c = ref.Cache(kv, 2, D, 16, seed=1)
    g = torch.Generator().manual_seed(2)
    q = torch.randn(sum(new) + 9, 8, D, generator=g).to(torch.bfloat16)
    want, bound = ref.attend(q, c.keys, c.values, starts_of(new), kv, 0.125)
    got = attention(c, q, starts_of(new), kv)
    assert ((got.double() - want).abs() <= bound).all()
    for rows in (slice(0, 3), slice(5, 8), slice(8, 38), slice(80, 89)):
        assert (got[rows] == 0).all()
    assert (attention(c, q, [0] * 5, kv) == 0).all()


def test_attention_without_requests_or_rows():
    c = ref.Cache([20], 2, 64, 16, seed=1)
    q = torch.randn(3, 4, 64).to(torch.bfloat16)
    none = Q.paged_attention(dev(q), dev(c.k), dev(c.v), ints(np.zeros((0, 2))), ints([0]), ints([]), scale=1.0)
    assert (host(none) == 0).all()
    assert Q.paged_attention(dev(q[:0]), dev(c.k), dev(c.v), ints(c.table), ints([0, 0]), ints([20]),
                             scale=1.0).shape == (0, 4, 64)
    no_width = Q.paged_attention(dev(q), dev(c.k), dev(c.v), ints(np.zeros((1, 0))), ints([0, 3]), ints([3]), scale=1.0)
    assert (host(no_width) == 0).all()


@pytest.mark.parametrize("new", [1, 3, 90])
def test_attention_on_missing_pages(new):
    """Page ids that are none: their keys are not seen, whether the table says -1 or anything else."""
    D, block, L = 128, 16, 400
    c = ref.Cache([L, 30], 2, D, block, seed=3)
    absent = [(0, p) for page in (0, 3, 9, 10, 24) for p in range(page * block, (page + 1) * block)]
    c.table[0, [0, 3, 9, 10, 24]] = [-1, c.k.shape[0], 2 ** 31 - 1, -2 ** 31, -1]
    q = torch.randn(new + 1, 6, D, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16)
    want, bound = ref.attend(q, c.keys, c.values, [0, new, new + 1], [L, 30], D ** -0.5, absent=absent)
    got = attention(c, q, [0, new, new + 1], [L, 30])
    assert ((got.double() - want).abs() <= bound).all()


def test_attention_past_the_tables_width():
    """A length beyond what the table can hold: the keys that are there are seen."""
    D, block = 64, 16
    c = ref.Cache([64], 2, D, block, seed=3)
    q = torch.randn(10, 4, D, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16)
    want, bound = ref.attend(q, c.keys, c.values, [0, 10], [70], 0.125)
    got = attention(c, q, [0, 10], [70])
    assert ((got.double() - want).abs() <= bound).all()
    far = attention(c, q, [0, 10], [2 ** 31 - 1])
    want, bound = ref.attend(q, c.keys, c.values, [0, 10], [2 ** 31 - 1], 0.125)
    assert ((far.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("new,L", [(1, 1000), (3, 300), (200, 500), (90, 1900)])
@pytest.mark.parametrize("kind", ["sharp", "equal", "rising", "falling", "low"])
def test_attention_of_extreme_scores(new, L, kind):
    """One key carries a row; all keys alike; maxima that move with every key; scores far below zero."""
    D, Hq, Hkv = 128, 8, 2
    c = ref.Cache([L], Hkv, D, 16, seed=6)
    g = torch.Generator().manual_seed(7)
    q = torch.randn(new, Hq, D, generator=g).to(torch.bfloat16)
    scale = D ** -0.5
    if kind == "sharp":
        scale = 8.0
    else:
        K = torch.randn(L, Hkv, D, generator=g) * 0.01
        q = q.abs() + 0.5
        j = torch.arange(L)[:, None, None].float()
        K += dict(equal=0 * j, rising=j / 10, falling=-j / 10, low=0 * j - 50)[kind]
        c.keys[0] = K.to(torch.bfloat16)
        for p in range(-(-L // 16)):
            rows = c.keys[0][p * 16:(p + 1) * 16].transpose(0, 1)
            c.k[int(c.table[0, p]), :, :rows.shape[1]] = rows
    want, bound = ref.attend(q, c.keys, c.values, [0, new], [L], scale)
    got = attention(c, q, [0, new], [L], scale=scale)
    assert torch.isfinite(got).all() and ((got.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("new", [1, 4, 80])
def test_attention_with_a_negative_scale_and_infinite_keys(new):
    """A key whose scores are -inf has no weight; all of them: nothing is seen of the row."""
    D, L = 64, 200
    c = ref.Cache([L], 1, D, 16, seed=8)
    q = torch.rand(new, 2, D, generator=torch.Generator().manual_seed(9)).to(torch.bfloat16) + 0.5
    want, bound = ref.attend(q, c.keys, c.values, [0, new], [L], -0.3)
    assert ((attention(c, q, [0, new], [L], scale=-0.3).double() - want).abs() <= bound).all()
    dead = [0, 17, 63, 64, 100]
    for j in dead:
        c.k[int(c.table[0, j // 16]), :, j % 16] = -math.inf
    want, bound = ref.attend(q, c.keys, c.values, [0, new], [L], 0.1, absent=[(0, j) for j in dead])
    got = attention(c, q, [0, new], [L], scale=0.1)
    assert ((got.double() - want).abs() <= bound).all()
    c.k[:] = -math.inf
    assert (attention(c, q, [0, new], [L], scale=0.1) == 0).all()


@pytest.mark.parametrize("new,window", [(1, 0), (3, 0), (90, 0), (5, 40), (150, 70)])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_attention_of_values_that_are_not_finite(new, window, D):
    """They reach the rows that see their keys, in their columns, and no other."""
    L = 400
    c = ref.Cache([L], 2, D, 16, seed=20)
    bad = [(L - 1, 0, 3, math.inf), (L - 2, 1, 0, math.nan), (L - 60, 0, 9, -math.inf), (L - 75, 1, 63, math.inf),
           (L - 76, 1, 63, -math.inf), (7, 0, 5, math.nan)]
    for j, h, d, x in bad:
        c.values[0][j, h, d] = x
        c.v[int(c.table[0, j // 16]), h, j % 16, d] = x
    q = torch.randn(new, 4, D, generator=torch.Generator().manual_seed(21)).to(torch.bfloat16)
    want, bound = ref.attend(q, c.keys, c.values, [0, new], [L], D ** -0.5, window)
    got = attention(c, q, [0, new], [L], window=window).double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got[~fine & ~torch.isnan(want)],
                                                                            want[~fine & ~torch.isnan(want)])
    assert ((got - want).abs() <= bound)[fine].all() and not fine.all()


def test_attention_of_keys_that_are_not_finite_and_not_seen():
    """NaN keys after a row's position, or before its window, do not reach it."""
    D, L, new, window = 64, 300, 100, 50
    c = ref.Cache([L], 1, D, 16, seed=22)
    for j in (L - 1, L - 2, L - 30):
        c.k[int(c.table[0, j // 16]), :, j % 16] = math.nan
    c.k[int(c.table[0, 0]), :, 0] = math.nan
    q = torch.randn(new, 2, D, generator=torch.Generator().manual_seed(23)).to(torch.bfloat16)
    want, bound = ref.attend(q, c.keys, c.values, [0, new], [L], 0.125, window)
    got = attention(c, q, [0, new], [L], window=window).double()
    sees = slice(0, new - 30)
    assert ((got - want).abs() <= bound)[sees].all()
    assert torch.isnan(got[new - 30:]).all()


@pytest.mark.parametrize("new", [1, 3, 90])
def test_attention_of_a_cache_past_32_bit_offsets(new):
    """Pages at both ends of a cache of 2^31 values and more."""
    Hkv, D, block = 4, 256, 16
    NB = 2 ** 31 // (Hkv * D * block) + 40
    k, v = (torch.empty(NB, Hkv, block, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    c = ref.Cache([300], Hkv, D, block, seed=10)
    pages = [p if p % 2 else NB - 1 - p for p in range(c.table.shape[1])]
    for i, p in enumerate(pages):
        k[p], v[p] = c.k[int(c.table[0, i])].cuda(), c.v[int(c.table[0, i])].cuda()
    q = torch.randn(new, 8, D, generator=torch.Generator().manual_seed(11)).to(torch.bfloat16)
    want, bound = ref.attend(q, c.keys, c.values, [0, new], [300], 1 / 16)
    got = host(Q.paged_attention(dev(q), Q.Array.from_torch(k), Q.Array.from_torch(v), ints([pages]), ints([0, new]),
                                 ints([300]), scale=1 / 16))
    assert ((got.double() - want).abs() <= bound).all()
    # and the write of the last page's rows
    x = torch.randn(block, Hkv, D, generator=torch.Generator().manual_seed(12)).to(torch.bfloat16)
    f = dev(torch.zeros(0, dtype=torch.float32))
    Q.rope_cache(dev(x), dev(x), dev(-x), Q.Array.from_torch(k), Q.Array.from_torch(v), ints(range(block)),
                 ints(range((NB - 1) * block, NB * block)), f)
    torch.cuda.synchronize()
    assert torch.equal(k[NB - 1].cpu(), x.transpose(0, 1)) and torch.equal(v[NB - 1].cpu(), -x.transpose(0, 1))


def test_attention_split_contexts_on_two_streams():
    """Long contexts, whose parts meet in the stream's workspace, on two streams at once."""
    D = 128
    c = ref.Cache([9000, 3000], 2, D, 16, seed=12)
    q = torch.randn(2, 8, D, generator=torch.Generator().manual_seed(13)).to(torch.bfloat16)
    want, bound = ref.attend(q, c.keys, c.values, [0, 1, 2], [9000, 3000], D ** -0.5)
    a = [dev(q), dev(c.k), dev(c.v), ints(c.table), ints([0, 1, 2]), ints([9000, 3000])]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    wrapped = [Q.Stream(s.cuda_stream) for s in streams]
    outs = [[Q.paged_attention(*a, scale=D ** -0.5, stream=s) for s in wrapped] for _ in range(10)]
    for s in wrapped:
        s.sync()
    first = host(outs[0][0])
    assert ((first.double() - want).abs() <= bound).all()
    assert all(torch.equal(host(o), first) for pair in outs for o in pair)


def test_a_captured_step_follows_the_lengths_on_the_gpu():
    """Tables, writes and attention of a decode step in one graph, replayed as the sequences grow
    (the lengths, the table and the head of the free list in place): every step equal to eager."""
    Hq, Hkv, D, block, R, W, steps = 8, 2, 128, 16, 3, 40, 20
    cached = [5, 30, 310]
    g = torch.Generator().manual_seed(14)
    NB = R * W
    start = ref.Cache(cached, Hkv, D, block, seed=15, spare=60, width=W)
    used = set(start.table[start.table >= 0].tolist())
    free = [p for p in range(start.k.shape[0]) if p not in used]
    freqs = torch.from_numpy(Q.rope_frequencies(64, 1e6)[0])
    x = [torch.randn(steps, R, h, D, generator=g).to(torch.bfloat16).cuda() for h in (Hq, Hkv, Hkv)]
    assert NB >= start.k.shape[0]

    def fresh():
        t = dict(table=torch.from_numpy(start.table.copy()), head=torch.tensor([0], dtype=torch.int32),
                 lens=torch.tensor(cached, dtype=torch.int32), new=torch.ones(R, dtype=torch.int32),
                 free=torch.tensor(free, dtype=torch.int32))
        t = {k: v.cuda() for k, v in t.items()}
        t.update(k=start.k.cuda(), v=start.v.cuda(), f=freqs.cuda(), starts=torch.zeros(R + 1, dtype=torch.int32).cuda(),
                 pos=torch.zeros(R, dtype=torch.int32).cuda(), slots=torch.zeros(R, dtype=torch.int32).cuda())
        t.update({n: torch.zeros(R, h, D, dtype=torch.bfloat16).cuda() for n, h in
                  (("xq", Hq), ("xk", Hkv), ("xv", Hkv), ("qr", Hq), ("o", Hq))})
        a = {k: Q.Array.from_torch(v, Q.INT32 if v.dtype == torch.int32 else None) for k, v in t.items()}
        return t, a

    def step(a, st):
        Q.block_tables(a["table"], a["head"], a["lens"], a["new"], a["free"], block, R, table_out=a["table"],
                       head_out=a["head"], kv_lens=a["lens"], q_starts=a["starts"], positions=a["pos"],
                       slots=a["slots"], stream=st)
        Q.rope_cache(a["xq"], a["xk"], a["xv"], a["k"], a["v"], a["pos"], a["slots"], a["f"], q_out=a["qr"], stream=st)
        Q.paged_attention(a["qr"], a["k"], a["v"], a["table"], a["starts"], a["lens"], scale=D ** -0.5, out=a["o"],
                          stream=st)

    def feed(t, i):
        for n, v in zip(("xq", "xk", "xv"), x):
            t[n].copy_(v[i])

    t, a = fresh()
    eager = []
    for i in range(steps):
        feed(t, i)
        step(a, Q.Stream.torch_current())
        eager.append(t["o"].clone())
    torch.cuda.synchronize()
    assert t["lens"].tolist() == [c + steps for c in cached]
    assert int(t["head"]) == sum(-(-(c + steps) // block) - -(-c // block) for c in cached)

    t, a = fresh()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # a first call outside the graph: the stream's workspace
        warm_t, warm = fresh()
        step(warm, Q.Stream.torch_current())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(a, Q.Stream.torch_current())
    for i in range(steps):
        feed(t, i)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(t["o"], eager[i]), i
