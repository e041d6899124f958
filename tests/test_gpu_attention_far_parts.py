"""Contexts that several workgroups share, where the scores of some parts lie so far below the others' that f32 has no weight
for them: what is NaN or infinite among their values still reaches the rows that see it, as within one part."""
import math

import attention_ref
import fp8_ref
import pytest
import torch
from test_gpu_attention import attention
from test_gpu_attention_weights import rewrite
from test_gpu_fp8_attention import attention as attention_fp8

pytestmark = pytest.mark.gpu

L, HALF = 5000, 2500


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 3, 300])
def test_codes_that_are_nan_in_a_part_of_no_weight(D, new):
    """Scores of -256 and 256; NaN by a code and by a page's scale among the first, in heads 0 and 1."""
    c = fp8_ref.Cache([L], 3, D, 16, seed=D)
    for j in range(0, L, 16):
        page = int(c.table[0, j // 16])
        c.ks[page], c.k[page] = 127, 0xC8 if j + 16 <= HALF else 0x48  # -4, 4
    c.v[int(c.table[0, 6]), 0, 3, 5] = 127
    c.vs[int(c.table[0, 40]), 1] = 255
    q = torch.ones(new, 6, D, dtype=torch.bfloat16)
    want, bound = fp8_ref.attend(q.cuda(), c.keys, c.values, [0, new], [L], 64 / D, scales=c.scales)
    got, want, bound = attention_fp8(c, q, [0, new], [L], scale=64 / D).double(), want.cpu(), bound.cpu()
    assert torch.isnan(want[:, :2, 5]).all() and torch.isnan(want[:, 2:4]).all() and torch.isfinite(want[:, 4:]).all()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert ((got - want).abs() <= bound)[torch.isfinite(want)].all()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 3, 300])
def test_values_that_are_not_finite_in_a_part_of_no_weight(D, new):
    """The same over a bfloat16 cache: NaN, and an infinity, which is at least not lost."""
    c = attention_ref.Cache([L], 2, D, 16, seed=D)
    c.keys[0][:HALF], c.keys[0][HALF:] = -4, 4
    c.values[0][99, 0, 5], c.values[0][700, 1, 9] = math.nan, math.inf
    rewrite(c, 0)
    q = torch.ones(new, 4, D, dtype=torch.bfloat16)
    got = attention(c, q, [0, new], [L], scale=64 / D)
    assert torch.isnan(got[:, :2, 5]).all() and not torch.isfinite(got[:, 2:, 9]).any()
    c.values[0][99, 0, 5], c.values[0][700, 1, 9] = 0, 0
    want, bound = attention_ref.attend(q, c.keys, c.values, [0, new], [L], 64 / D)
    fine = torch.ones_like(got, dtype=torch.bool)
    fine[:, :2, 5], fine[:, 2:, 9] = False, False
    assert ((got.double() - want).abs() <= bound)[fine].all()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 3, 300])
def test_large_values_in_a_part_of_no_weight(D, new):
    """Finite values there add nothing, however large: 1e33 beside 1e-11."""
    c = attention_ref.Cache([L], 2, D, 16, seed=D)
    c.keys[0][:HALF], c.keys[0][HALF:] = -4, 4
    c.values[0][:HALF] = 1e33
    c.values[0][HALF:] *= 1e-11
    rewrite(c, 0)
    q = torch.ones(new, 4, D, dtype=torch.bfloat16)
    want, bound = attention_ref.attend(q, c.keys, c.values, [0, new], [L], 64 / D)
    assert ((attention(c, q, [0, new], [L], scale=64 / D).double() - want).abs() <= bound).all()
