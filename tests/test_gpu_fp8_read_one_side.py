"""One side of a cache held in 8 bits read back."""
import fp8_ref as ref
import pytest
import torch
from test_gpu_fp8_cache import dev, host, ints, some_cache

import qmm as Q

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [Q.BFLOAT16, Q.FLOAT32])
@pytest.mark.parametrize("given", [False, True])
def test_a_side_without_a_cache_is_not_read(dtype, given):
    codes, scales = some_cache(4, 2, 8, 64, seed=9)
    c, s, slots = dev(codes), dev(scales), [3, -1, 31]
    want = ref.decode(codes, scales)[[0, 0, 3], :, [3, 0, 7]].float()
    want[1] = 0
    want = want.to(torch.bfloat16) if dtype == Q.BFLOAT16 else want
    for side in (0, 1):
        out = dev(torch.zeros_like(want)) if given else None
        args = (c, None, s, None) if side == 0 else (None, c, None, s)
        got = Q.cache_read_fp8(*args, ints(slots), dtype=dtype, **{("k_out", "v_out")[side]: out})
        assert got[1 - side] is None and (not given or got[side] is out)
        assert torch.equal(torch.nan_to_num(host(got[side])), torch.nan_to_num(want))
