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
