"""Attention operators without a GPU: what they refuse, and the rotation's frequencies."""
import math
import re
from ctypes import byref, c_int, c_void_p
from pathlib import Path

import numpy as np
import pytest

import qmm as Q

FAKE = 0x10000  # a never-dereferenced device address: validation fails before any launch


def arr(shape, dtype=Q.BFLOAT16, ptr=FAKE):
    sh = (c_int * max(len(shape), 1))(*shape)
    return Q.Array(Q.lib.qmm_array_new_device(c_void_p(ptr), sh, len(shape), dtype))


def ints(*shape):
    return arr(shape, Q.INT32)


@pytest.fixture(autouse=True)
def _clean_latch():
    Q.lib.qmm_reset_faults_for_test()
    yield
    Q.lib.qmm_reset_faults_for_test()


def refuses(call, args, change, needle):
    args = dict(args, **change)
    with pytest.raises(Q.QmmError) as e:
        call(**args)
    assert needle in str(e.value), str(e.value)
    assert not Q.lib.qmm_error_pending()


R, W, T, Hq, Hkv, D, NB, BS = 3, 5, 4, 6, 2, 64, 9, 16


@pytest.mark.parametrize("change,needle", [
    (dict(table=ints(R * W)), "table must be an array of shape [any, any]"),
    (dict(table=arr((R, W), Q.UINT32)), "table must be int32"),
    (dict(head=ints(2)), "head must be an array of shape [1]"),
    (dict(cached_lens=ints(R + 1)), "cached_lens must be an array of shape [3]"),
    (dict(new_lens=arr((R,), Q.FLOAT32)), "new_lens must be int32"),
    (dict(free_blocks=ints(4, 4)), "free_blocks must be"),
    (dict(free_blocks=Q.Array()), "missing free_blocks"),
    (dict(block_size=0), "block_size must be positive"),
    (dict(n_tokens=-1), "n_tokens must not be negative"),
    (dict(table=ints(4097, 1), cached_lens=ints(4097), new_lens=ints(4097)), "at most 4096"),
])
def test_block_tables_refuses(change, needle):
    good = dict(table=ints(R, W), head=ints(1), cached_lens=ints(R), new_lens=ints(R), free_blocks=ints(7),
                block_size=BS, n_tokens=T)
    refuses(Q.block_tables, good, change, needle)


@pytest.mark.parametrize("change,needle", [
    (dict(x=arr((T, Hq, D), Q.FLOAT16)), "bfloat16 or float32"),
    (dict(x=arr((T, D))), "[..., T, H, D]"),
    (dict(x=arr((T, Hq, 60))), "multiple of 8 from 8 to 256, got 60"),
    (dict(x=arr((T, Hq, 264))), "got 264"),
    (dict(x=arr((T, Hq, 16))), "rotate more than the head's 16"),
    (dict(x=arr((T, Hq, D), ptr=FAKE + 2)), "16-byte aligned"),
    (dict(positions=ints(T + 1)), "positions must be an array of shape [4]"),
    (dict(positions=arr((T,), Q.UINT32)), "positions must be int32"),
    (dict(freqs=arr((4,))), "freqs must be a 1D float32"),
    (dict(freqs=Q.Array()), "missing freqs"),
    (dict(x=Q.Array()), "missing x"),
])
def test_rope_refuses(change, needle):
    refuses(Q.rope, dict(x=arr((T, Hq, D)), positions=ints(T), freqs=arr((16,), Q.FLOAT32)), change, needle)


CACHE = (NB, Hkv, BS, D)


@pytest.mark.parametrize("change,needle", [
    (dict(k_cache=arr(CACHE, Q.FLOAT32)), "k_cache must be a bfloat16"),
    (dict(v_cache=arr(CACHE[1:])), "v_cache must be a bfloat16"),
    (dict(v_cache=arr((NB, Hkv, BS + 1, D))), "shapes differ"),
    (dict(k_cache=arr(CACHE, ptr=FAKE + 8)), "k_cache must be 16-byte aligned"),
    (dict(k_cache=arr((NB, Hkv, 0, D)), v_cache=arr((NB, Hkv, 0, D))), "needs heads and a block size"),
    (dict(q=arr((T, Hq, D), Q.FLOAT32)), "all be bfloat16 or all float32"),
    (dict(q=arr((T, Hq, D - 8))), "q must be [T, Hq, 64 or more"),
    (dict(q=arr((T, Hq, D + 4))), "a multiple of 8"),
    (dict(k=arr((T, Hkv + 1, D))), "k and v must be [4, 2, 64]"),
    (dict(v=arr((T + 1, Hkv, D))), "k and v must be [4, 2, 64]"),
    (dict(v=Q.Array()), "missing input"),
    (dict(k_cache=arr((1 << 21, Hkv, 1 << 10, D))), "over 2^32 - 1 keys"),
    (dict(slots=ints(T - 1)), "slots must be an array of shape [4]"),
    (dict(q_norm=arr((D - 8,))), "q_norm must be [64]"),
    (dict(k_norm=arr((D,), Q.UINT8)), "k_norm must be [64]"),
    (dict(freqs=arr((33,), Q.FLOAT32)), "33 frequencies rotate more"),
])
def test_rope_cache_refuses(change, needle):
    good = dict(q=arr((T, Hq, D)), k=arr((T, Hkv, D)), v=arr((T, Hkv, D)), k_cache=arr(CACHE), v_cache=arr(CACHE),
                positions=ints(T), slots=ints(T), freqs=arr((16,), Q.FLOAT32))
    refuses(Q.rope_cache, good, change, needle)


def test_rope_cache_refuses_to_overwrite_a_wider_q():
    q = arr((T, Hq, 2 * D))
    with pytest.raises(Q.QmmError, match="own array only at q's layout"):
        Q.rope_cache(q, arr((T, Hkv, D)), arr((T, Hkv, D)), arr(CACHE), arr(CACHE), ints(T), ints(T),
                     arr((16,), Q.FLOAT32), q_out=arr((T, Hq, D)))


@pytest.mark.parametrize("change,needle", [
    (dict(q=arr((T, Hq, D), Q.FLOAT32)), "q must be a bfloat16 array [T, Hq, 64]"),
    (dict(q=arr((T, Hq, D + 8))), "q must be a bfloat16 array [T, Hq, 64]"),
    (dict(q=arr((T, 5, D))), "5 query heads do not share 2 key heads"),
    (dict(q=arr((T, Hq, D), ptr=FAKE + 4)), "q must be 16-byte aligned"),
    (dict(q=Q.Array()), "missing q"),
    (dict(k_cache=Q.Array()), "missing k_cache"),
    (dict(v_cache=arr((NB + 1, Hkv, BS, D))), "shapes differ"),
    (dict(k_cache=arr((NB, Hkv, BS, 12)), v_cache=arr((NB, Hkv, BS, 12))), "got 12"),
    (dict(table=ints(R)), "table must be"),
    (dict(v_cache=arr((1 << 20, 1 << 7, 1 << 5, D))), "over 2^32 - 1 keys"),
    (dict(table=ints(R, 2 ** 31 - 1)), "too many keys of all tiles"),
    (dict(q=arr((1 << 27, Hq, D))), "too many rows per key head"),
    (dict(q_starts=ints(R)), "q_starts must be an array of shape [4]"),
    (dict(kv_lens=ints(R + 1)), "kv_lens must be an array of shape [3]"),
    (dict(kv_lens=arr((R,), Q.UINT32)), "kv_lens must be int32"),
    (dict(table=ints(4097, W), q_starts=ints(4098), kv_lens=ints(4097)), "at most 4096"),
    (dict(gate=arr((T, Hq, D - 8))), "gate must be"),
    (dict(gate=arr((T, Hq, D), Q.FLOAT32)), "gate must be"),
    (dict(window=-1), "window must not be negative"),
    (dict(scale=math.inf), "scale must be finite"),
    (dict(scale=math.nan), "scale must be finite"),
])
def test_paged_attention_refuses(change, needle):
    good = dict(q=arr((T, Hq, D)), k_cache=arr(CACHE), v_cache=arr(CACHE), table=ints(R, W), q_starts=ints(R + 1),
                kv_lens=ints(R), scale=0.125)
    refuses(Q.paged_attention, good, change, needle)


def test_null_results_are_refused():
    null = Q.qmm_array(None)
    assert Q.lib.qmm_rope(None, null, null, null, 1.0, False, False, Q.qmm_stream(None)) != 0
    assert Q.lib.qmm_paged_attention(None, *[null] * 7, 1.0, 0, Q.qmm_stream(None)) != 0
    res = Q.qmm_array(None)
    assert Q.lib.qmm_rope_cache(byref(res), *[null] * 8, 1.0, False, null, null, 1e-6, Q.qmm_stream(None)) != 0
    assert not res.ctx


def test_no_vector_register_of_the_attention_kernels_is_spilled():
    """hipcc has put spills before the point where a divergent region's lanes come back (the lanes that were out
    then reload what they never stored), so these kernels are kept to their registers."""
    lib = Path(Q.lib._name).read_bytes()
    found = {}
    for m in re.finditer(rb"\.symbol[\xa0-\xda](.{1,400}?)\.kd.{0,400}?\.vgpr_spill_count(.)", lib, re.S):
        name = m.group(1).decode("latin-1")
        if "attn_" in name:
            found[name] = m.group(2)[0]
    assert sum("attn_rows_kernel" in n for n in found) == 12 and sum("attn_chunk_kernel" in n for n in found) == 6
    assert not {n: c for n, c in found.items() if c}


# ---------------------------------------------------------------- frequencies


def test_frequencies():
    f, amp = Q.rope_frequencies(64, 1e7)
    assert amp == 1 and f.dtype == np.float32
    assert np.array_equal(f, np.array([1e7 ** (-2 * i / 64) for i in range(32)], dtype=np.float32))
    f, amp = Q.rope_frequencies(64, 1e7, "linear", factor=8)
    assert amp == 1 and np.allclose(f, [1e7 ** (-2 * i / 64) / 8 for i in range(32)], rtol=2 ** -23)


def test_changed_base_reaches_the_factor_at_the_last_pair():
    """base * factor^(d / (d - 2)): pair 0 turns as before, the last one `factor` times slower."""
    plain, (f, _) = Q.rope_frequencies(32, 1e4)[0], Q.rope_frequencies(32, 1e4, "base", factor=4)
    assert f[0] == 1 and abs(plain[-1] / f[-1] - 4) < 1e-5


@pytest.mark.parametrize("kind", ["ramp", "bands"])
def test_ramped_frequencies_keep_the_fast_and_divide_the_slow(kind):
    L, slow, fast = 4096.0, 1.0, 32.0
    plain, (f, amp) = Q.rope_frequencies(128, 1e4)[0], Q.rope_frequencies(128, 1e4, kind, factor=4, original_len=L,
                                                                         slow=slow, fast=fast)
    turns, ratio = L * plain / (2 * math.pi), plain / f
    assert (np.diff(ratio) >= -1e-5).all()
    # (the ramp over pairs ends on whole ones, at most one beyond each bound)
    step = plain[0] / plain[1]
    assert np.allclose(ratio[turns > fast * step], 1) and np.allclose(ratio[turns < slow / step], 4)
    assert amp == pytest.approx(0.1 * math.log(4) + 1 if kind == "ramp" else 1)
    if kind == "bands":
        u = np.clip((turns - slow) / (fast - slow), 0, 1)
        assert np.allclose(f, plain / 4 * (1 - u) + plain * u, rtol=1e-5)


@pytest.mark.parametrize("args,kw,needle", [
    ((3, 1e4), {}, "even size"), ((0, 1e4), {}, "even size"), ((8, 1.0), {}, "base must be over 1"),
    ((8, 1e4, "linear"), dict(factor=0.5), "at least 1"), ((2, 1e4, "base"), dict(factor=2), "one pair"),
    ((8, 1e4, "ramp"), dict(factor=2), "original_len"),
    ((8, 1e4, "bands"), dict(factor=2, original_len=64, slow=4, fast=4), "fast > slow"),
])
def test_frequencies_refuse(args, kw, needle):
    with pytest.raises(Q.QmmError, match=needle):
        Q.rope_frequencies(*args, **kw)
