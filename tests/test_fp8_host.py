"""A cache held in 8 bits without a GPU: what its operators refuse, and the restatement that their tests go by."""
import math
import re
from ctypes import byref
from pathlib import Path

import fp8_ref as ref
import pytest
import torch
from test_attention_host import arr, ints, refuses
from test_attention_results_host import apart

import qmm as Q

R, W, T, Hq, Hkv, D, NB, BS = 3, 5, 4, 6, 2, 64, 9, 16
CACHE, SCALES, U8 = (NB, Hkv, BS, D), (NB, Hkv), Q.UINT8


@pytest.fixture(autouse=True)
def _clean_latch():
    Q.lib.qmm_reset_faults_for_test()
    yield
    Q.lib.qmm_reset_faults_for_test()


def cache():
    return dict(k_cache=apart(0, CACHE, U8), v_cache=apart(1, CACHE, U8), k_scales=apart(2, SCALES, U8),
                v_scales=apart(3, SCALES, U8))


def layer():
    return dict(cache(), q=apart(4, (T, Hq, D)), k=apart(5, (T, Hkv, D)), v=apart(6, (T, Hkv, D)),
                positions=apart(7, (T,), Q.INT32), slots=apart(8, (T,), Q.INT32), freqs=apart(9, (16,), Q.FLOAT32))


def attention():
    return dict(cache(), q=apart(4, (T, Hq, D)), table=apart(5, (R, W), Q.INT32), q_starts=apart(6, (R + 1,), Q.INT32),
                kv_lens=apart(7, (R,), Q.INT32), scale=0.125)


OF_CACHES = [
    (dict(k_cache=apart(0, CACHE)), "k_cache must be a uint8 array"),
    (dict(v_cache=apart(1, CACHE[1:], U8)), "v_cache must be a uint8"),
    (dict(v_cache=apart(1, (NB, Hkv, BS + 1, D), U8)), "shapes differ"),
    (dict(k_cache=arr(CACHE, U8, ptr=0x10008)), "k_cache must be 16-byte aligned"),
    (dict(k_cache=apart(0, (NB, Hkv, 0, D), U8), v_cache=apart(1, (NB, Hkv, 0, D), U8)), "needs heads and a block size"),
    (dict(k_cache=apart(0, (NB, Hkv, BS, 72), U8), v_cache=apart(1, (NB, Hkv, BS, 72), U8)), "multiple of 16 from 16 to 256, got 72"),
    (dict(k_cache=apart(0, (NB, Hkv, BS, 272), U8), v_cache=apart(1, (NB, Hkv, BS, 272), U8)), "got 272"),
    (dict(k_cache=arr((1 << 21, Hkv, 1 << 10, D), U8)), "over 2^32 - 1 keys"),
    (dict(k_scales=apart(2, (NB, Hkv), Q.FLOAT32)), "k_scales must be a uint8 array [9, 2]"),
    (dict(v_scales=apart(3, (NB + 1, Hkv), U8)), "v_scales must be a uint8 array [9, 2]"),
    (dict(v_scales=Q.Array()), "missing v_scales"),
    (dict(k_cache=Q.Array()), "missing k_cache"),
]


@pytest.mark.parametrize("change,needle", OF_CACHES + [
    (dict(q=apart(4, (T, Hq, D), Q.FLOAT32)), "all be bfloat16 or all float32"),
    (dict(q=apart(4, (T, Hq, D - 8))), "q must be [T, Hq, 64 or more"),
    (dict(q=apart(4, ((1 << 30) + 1, Hq, D))), "more than 2^30 rows"),
    (dict(k=apart(5, (T, Hkv + 1, D))), "k and v must be [4, 2, 64]"),
    (dict(v=Q.Array()), "missing input"),
    (dict(slots=ints(T - 1)), "slots must be an array of shape [4]"),
    (dict(q_norm=arr((D - 8,))), "q_norm must be [64]"),
    (dict(freqs=arr((33,), Q.FLOAT32)), "33 frequencies rotate more"),
    (dict(k_cache=apart(1, CACHE, U8)), "caches and their scales lie over one another"),
    (dict(v_scales=apart(2, SCALES, U8)), "caches and their scales lie over one another"),
    (dict(k_scales=arr(SCALES, U8, ptr=0x10000 + 64)), "caches and their scales lie over one another"),
    (dict(slots=apart(2, (T,), Q.INT32)), "caches and their scales lie over an input"),
    (dict(k=apart(1, (T, Hkv, D))), "caches and their scales lie over an input"),
    (dict(q_out=apart(0, (T, Hq, D))), "q_out lies over an input"),
    (dict(q_out=apart(2, (T, Hq, D))), "q_out lies over an input"),
])
def test_rope_cache_fp8_refuses(change, needle):
    refuses(Q.rope_cache_fp8, layer(), change, needle)


@pytest.mark.parametrize("change,needle", OF_CACHES + [
    (dict(q=apart(4, (T, Hq, D), Q.FLOAT32)), "q must be a bfloat16 array [T, Hq, 64]"),
    (dict(q=apart(4, (T, 5, D))), "5 query heads do not share 2 key heads"),
    (dict(table=ints(R, 2 ** 31 - 1)), "too many keys of all tiles"),
    (dict(q=apart(4, (1 << 27, Hq, D))), "too many rows per key head"),
    (dict(kv_lens=ints(R + 1)), "kv_lens must be an array of shape [3]"),
    (dict(table=ints(4097, W), q_starts=ints(4098), kv_lens=ints(4097)), "at most 4096"),
    (dict(gate=arr((T, Hq, D - 8))), "gate must be"),
    (dict(window=-1), "window must not be negative"),
    (dict(scale=math.nan), "scale must be finite"),
    (dict(out=apart(2, (T, Hq, D))), "the result lies over an input"),
    (dict(out=apart(3, (T, Hq, D))), "the result lies over an input"),
])
def test_paged_attention_fp8_refuses(change, needle):
    refuses(Q.paged_attention_fp8, attention(), change, needle)


@pytest.mark.parametrize("change,needle", OF_CACHES + [
    (dict(slots=arr((T,), Q.UINT32)), "slots must be int32"),
    (dict(slots=Q.Array()), "missing slots"),
    (dict(dtype=Q.FLOAT16), "dtype must be bfloat16 or float32"),
    (dict(k_out=apart(0, (T, Hkv, D))), "k_out lies over an input"),
    (dict(v_out=apart(3, (T, Hkv, D))), "v_out lies over an input"),
    (dict(k_out=apart(7, (T, Hkv, D)), v_out=apart(7, (T, Hkv, D))), "v_out lies over k_out"),
])
def test_cache_read_fp8_refuses(change, needle):
    refuses(Q.cache_read_fp8, dict(cache(), slots=apart(4, (T,), Q.INT32)), change, needle)


def test_a_handle_as_a_result_of_another_shape_is_kept():
    a = dict(cache(), slots=apart(4, (T,), Q.INT32))
    for of in ("k_cache", "v_scales", "slots"):
        with pytest.raises(Q.QmmError, match="another shape"):
            Q.cache_read_fp8(**a, v_out=a[of])
        assert a[of].ptr
    a = attention()
    with pytest.raises(Q.QmmError, match="another shape"):
        Q.paged_attention_fp8(**a, out=a["k_scales"])


def test_null_results_are_refused():
    null, stream = Q.qmm_array(None), Q.qmm_stream(None)
    assert Q.lib.qmm_paged_attention_fp8(None, *[null] * 9, 1.0, 0, stream) != 0
    assert Q.lib.qmm_rope_cache_fp8(None, *[null] * 10, 1.0, False, null, null, 1e-6, stream) != 0
    assert Q.lib.qmm_cache_read_fp8(None, None, *[null] * 5, Q.BFLOAT16, stream) != 0
    res = Q.qmm_array(None)
    assert Q.lib.qmm_cache_read_fp8(byref(res), None, *[null] * 5, Q.BFLOAT16, stream) != 0 and not res.ctx


def test_no_vector_register_of_the_kernels_is_spilled():
    """As the kernels over a bfloat16 cache."""
    lib = Path(Q.lib._name).read_bytes()
    found = {}
    for m in re.finditer(rb"\.symbol[\xa0-\xda](.{1,400}?)\.kd.{0,400}?\.vgpr_spill_count(.)", lib, re.S):
        name = m.group(1).decode("latin-1")
        if "attn_rows8_kernel" in name or "attn_chunk8_kernel" in name or "cache_write" in name or "cache_read" in name:
            found[name] = m.group(2)[0]
    assert sum("attn_rows8_kernel" in n for n in found) == 12 and sum("cache_" in n for n in found) >= 8
    assert not {n: c for n, c in found.items() if c}


# ---------------------------------------------------------------- the restatement


def test_codes_are_torchs():
    codes = torch.arange(256, dtype=torch.uint8)
    want = codes.view(torch.float8_e4m3fn).double()
    assert torch.equal(torch.nan_to_num(ref.VALUES, 1e9), torch.nan_to_num(want, 1e9))
    x = torch.cat([torch.randn(5000, generator=torch.Generator().manual_seed(1)) * s for s in (1e-3, 0.1, 1, 50, 110)])
    x = x.clamp(-448, 448)
    assert torch.equal(ref.encode(x.double()), x.to(torch.float8_e4m3fn).view(torch.uint8))
    half = torch.tensor([2.0 ** -10, 3 * 2.0 ** -10, 17.0, 19.0, 432.0, 448.0])  # ties
    assert torch.equal(ref.encode(half.double()), half.to(torch.float8_e4m3fn).view(torch.uint8))


@pytest.mark.parametrize("top,t", [(448.0, 0), (448.1, 1), (3.5, -7), (3.51, -6), (1e-45, -127), (0.0, -127),
                                   (448 * 2.0 ** -127, -127), (3.3e38, 120)])
def test_exponents(top, t):
    assert ref.exponent(top) == t


def test_a_pages_scale_grows_and_starts_anew():
    codes, scales = torch.zeros(2, 1, 4, 16, dtype=torch.uint8), torch.full((2, 1), 100, dtype=torch.uint8)
    y = torch.zeros(3, 1, 16, dtype=torch.float64)
    y[:, 0, 0] = torch.tensor([448.0, 1.0, 449.0])
    c, s, _ = ref.store(codes, scales, [4, 5], y[:2])
    assert s[1, 0] == 127 and ref.decode(c, s)[1, 0, :2, 0].tolist() == [448.0, 1.0]
    c, s, _ = ref.store(c, s, [6], y[2:])
    assert s[1, 0] == 128 and ref.decode(c, s)[1, 0, :3, 0].tolist() == [448.0, 1.0, 448.0]  # (449 rounded)
    c, s, _ = ref.store(c, s, [4], y[1:2])
    assert s[1, 0] == 127 - 8 and ref.decode(c, s)[1, 0, 0, 0] == 1.0 and s[0, 0] == 100
