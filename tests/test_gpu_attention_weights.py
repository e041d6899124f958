"""How exact the softmax's weights of few rows are, and that their two parts leave values that are not finite alone."""
import math

import attention_ref as ref
import numpy as np
import pytest
import torch
from test_gpu_attention_many import attend, dev, ints

import qmm as Q

pytestmark = pytest.mark.gpu


def into_nan(c, q, starts, kv, scale):
    out = torch.full(q.shape, math.nan, dtype=torch.bfloat16, device="cuda")
    Q.paged_attention(dev(q), dev(c.k), dev(c.v), ints(c.table), ints(starts), ints(kv), scale=scale, out=Q.Array.from_torch(out))
    torch.cuda.synchronize()
    return out


def rewrite(c, r):
    """The pages of request r from its keys and values."""
    block = c.k.shape[2]
    for cache, mine in ((c.k, c.keys[r]), (c.v, c.values[r])):
        for p in range(-(-mine.shape[0] // block)):
            rows = mine[p * block:(p + 1) * block].transpose(0, 1)
            cache[int(c.table[r, p]), :, :rows.shape[1]] = rows


@pytest.mark.parametrize("Hq,D,new", [(4, 256, 1), (10, 256, 3), (8, 128, 1), (8, 128, 4), (6, 64, 1), (7, 64, 4), (3, 80, 2)])
@pytest.mark.parametrize("L", [40, 700, 5000])
def test_weights_of_few_rows_are_not_rounded_to_bf16(Hq, D, new, L):
    """One key's values cancel those of all the others, so that the result is small beside what it is made of and its own
    rounding hides nothing.

    Bound, of sum p |v| unless said: the result's rounding (2^-8 of itself), the two parts of a weight (2^-17), its
    exponent's error (D + 8 roundings of 2^-24 of scale sum |q k|, in the weight and in the sum) and exp2 (2^-22 twice), and
    sums of L products in f32, at worst 16 at a time in a line (L / 16 + 64 roundings of 2^-24, in the sum as well)."""
    g = torch.Generator().manual_seed(L + D)
    c = ref.Cache([L], 1, D, 16, seed=L)
    x = torch.randn(D, generator=g).to(torch.bfloat16)
    K, V = c.keys[0], c.values[0]
    V[L - new:] = 0  # (what only some of the rows see adds nothing to their sums)
    p = torch.softmax(K[:L - new, 0].double() @ x.double() * D ** -0.5, 0)
    V[3, 0] = 0
    V[3, 0] = (-(p @ V[:L - new, 0].double()) / p[3]).to(torch.bfloat16)
    rewrite(c, 0)
    q = x.expand(new, Hq, D).contiguous()
    want, _ = attend(q, c.keys, c.values, [0, new], [L], D ** -0.5)
    total, _ = attend(q, c.keys, [V.abs()], [0, new], [L], D ** -0.5)
    size = float((K[:, 0].abs().double() @ x.abs().double()).max()) * D ** -0.5
    weight = 2 ** -17 + 2 * (D + 8) * 2 ** -24 * size + 2 ** -21 + 2 * (L / 16 + 64) * 2 ** -24
    got = into_nan(c, q, [0, new], [L], D ** -0.5).cpu().double()
    assert ((got - want).abs() <= 2 ** -8 * want.abs() + weight * total).all()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 3])
def test_values_that_are_not_finite_far_from_the_masks_edges(D, new):
    """A weight of 1 has no second part (0 inf is NaN), others one below 0 (inf - inf): each key on its own gives its
    value's infinity in its column, two of both signs NaN, and the other columns what they are without them."""
    L = 3000
    c = ref.Cache([L], 2, D, 16, seed=51)
    for j, h, d, v in ((1500, 0, 3, math.inf), (1501, 0, 4, -math.inf), (900, 1, 7, math.inf), (1700, 1, 7, -math.inf),
                       (400, 1, 0, math.nan), (2100, 0, D - 1, math.inf), (64, 0, D - 1, math.inf)):
        c.values[0][j, h, d] = v
    c.keys[0][1500] *= 8  # (scores far apart: some weights next to none, some the row's own reference)
    rewrite(c, 0)
    q = torch.randn(new, 6, D, generator=torch.Generator().manual_seed(52)).to(torch.bfloat16)
    want, bound = ref.attend(q, c.keys, c.values, [0, new], [L], D ** -0.5)
    got = into_nan(c, q, [0, new], [L], D ** -0.5).cpu().double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got[torch.isinf(want)], want[torch.isinf(want)])
    assert ((got - want).abs() <= bound)[fine].all() and (~fine).any()


def test_finite_sums_past_f32_stay_infinite():
    """Values near the largest there are: a sum past f32 is infinite, not taken for a value held back."""
    L, D = 600, 64
    c = ref.Cache([L], 1, D, 16, seed=53)
    c.keys[0][:] = 0
    c.values[0][:, 0, 0] = 3e38
    rewrite(c, 0)
    q = torch.ones(1, 2, D, dtype=torch.bfloat16)
    got = into_nan(c, q, [0, 1], [L], 1.0)
    assert (got[..., 0] == math.inf).all() and torch.isfinite(got[..., 1:]).all()


@pytest.mark.parametrize("D", [64, 256])
def test_a_query_that_is_not_a_number_is_its_own_rows_only(D):
    """NaN queries (rows that nobody reads, in a step of a fixed size) give NaN, whatever the values, and the tile's other
    rows what they are without them."""
    L = 2000
    c = ref.Cache([L], 1, D, 16, seed=54)
    c.values[0][700, 0, 2] = math.inf
    rewrite(c, 0)
    q = torch.randn(3, 4, D, generator=torch.Generator().manual_seed(55)).to(torch.bfloat16)
    plain = into_nan(c, q, [0, 3], [L], D ** -0.5).cpu()
    q[1, 2] = math.nan
    got = into_nan(c, q, [0, 3], [L], D ** -0.5).cpu()
    assert torch.isnan(got[1, 2]).all()
    got[1, 2] = plain[1, 2]
    assert torch.equal(got, plain)
