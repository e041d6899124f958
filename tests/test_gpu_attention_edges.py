"""Attention operators at the ends of their ranges: windows without limit, rows past a tile's end, very many tokens."""
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
    n = a.numpy()
    return torch.from_numpy(n.view(np.int16)).view(torch.bfloat16) if a.dtype == Q.BFLOAT16 else torch.from_numpy(n)


def attention(c, q, starts, kv, **kw):
    return host(Q.paged_attention(dev(q), dev(c.k), dev(c.v), ints(c.table), ints(starts), ints(kv), **kw))


@pytest.mark.parametrize("new,kv", [([8], [3]), ([100], [20]), ([6, 300, 1], [2, 40, 500])])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 90, 2 ** 30])
def test_the_largest_windows_of_rows_before_the_first_key(new, kv, window):
    """A window past every key hides none, whatever the rows' positions (some are below 0); bound: as every attention
    test."""
    D = 64
    c = ref.Cache(kv, 2, D, 16, seed=41)
    q = torch.randn(sum(new), 4, D, generator=torch.Generator().manual_seed(42)).to(torch.bfloat16)
    starts = [0] + np.cumsum(new).tolist()
    want, bound = ref.attend(q, c.keys, c.values, starts, kv, 0.125)
    got = attention(c, q, starts, kv, scale=0.125, window=window)
    assert ((got.double() - want).abs() <= bound).all() and (want != 0).any()


@pytest.mark.parametrize("D", [64, 128, 256])
def test_rows_past_a_tiles_end_have_no_part_in_it(D):
    """A tile's rows beyond its request are filled up with its first row's queries.  However far that row's scores reach
    (its own reference covers them), the other rows' results stay the same bits: nothing is run a second time for rows
    that are none."""
    new, L = 40, 540
    c = ref.Cache([L], 1, D, 16, seed=43)
    c.k[..., 5] = 0
    for j, x in ((3, 0.5), (40, 1.0)):  # (400 x / 8 in powers of 2: 36, that row's reference, and 72, less than 2^60 past it)
        c.k[int(c.table[0, j // 16]), 0, j % 16, 5] = x
    q = torch.randn(new, 1, D, generator=torch.Generator().manual_seed(44)).to(torch.bfloat16)
    q[:, 0, 5] = 0
    got = []
    for far in (4.0, 400.0):
        q[0] = 0
        q[0, 0, 5] = far
        got.append(attention(c, q, [0, new], [L], scale=0.125))
    assert torch.isfinite(got[1]).all() and torch.equal(got[0][1:], got[1][1:])


def test_rotation_of_very_many_tokens():
    """More tokens than one launch takes (2^32 lanes): the same bits as the tokens' own calls, in the rows of the cache
    as well."""
    T, D = 2 ** 24 + 77, 8
    g = torch.Generator(device="cuda").manual_seed(45)
    x = torch.randn(T, 1, D, generator=g, device="cuda").to(torch.bfloat16)
    p = torch.randint(0, 262144, (T,), generator=g, device="cuda", dtype=torch.int32)
    f = dev(torch.tensor([1.0, 0.25, 0.125, 0.01]))

    def turned(a, b, norm):
        k, v = (torch.zeros(1, 1, b - a, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        q, y = torch.empty(b - a, 1, D, dtype=torch.bfloat16, device="cuda"), torch.empty(b - a, 1, D, dtype=torch.bfloat16, device="cuda")
        A = Q.Array.from_torch
        Q.rope(A(x[a:b]), A(p[a:b], Q.INT32), f, out=A(y))
        slots = torch.arange(b - a, dtype=torch.int32, device="cuda")
        Q.rope_cache(A(x[a:b]), A(x[a:b]), A(x[a:b]), A(k), A(v), A(p[a:b], Q.INT32), A(slots, Q.INT32), f, q_out=A(q),
                     q_norm=norm)
        torch.cuda.synchronize()
        return y, q, k[0, 0], v[0, 0]

    norm = dev(torch.linspace(0.5, 2, D))
    whole = turned(0, T, norm)
    for a, b in ((0, 100), (2 ** 23 - 50, 2 ** 23 + 50), (2 ** 24 - 64, 2 ** 24 + 64 - 51), (T - 100, T)):
        for w, part in zip(whole, turned(a, b, norm)):
            assert torch.equal(w[a:b], part)
