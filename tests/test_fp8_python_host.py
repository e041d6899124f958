"""The Python side of a cache held in 8 bits without a GPU."""
import re
import sys
from pathlib import Path

import pytest
import torch
from test_attention_results_host import apart

import qmm as Q

sys.path.insert(0, str(Path(Q.__file__).parent))


def test_rows_of_a_bfloat16_layer_are_not_read_back():
    """Its cache has no scales: refused by what it is, before anything is made."""
    from attention_layer import AttentionLayer

    layer = AttentionLayer.__new__(AttentionLayer)
    layer.eight, layer.Hkv, layer.D, layer.caches = False, 2, 64, ()
    with pytest.raises(ValueError, match="cache='e4m3'"):
        layer.read(torch.zeros(3, dtype=torch.int32), None)


def test_cache_read_fp8_of_one_side_needs_that_side():
    """A side without a cache is not read (the C call's NULL result); one that a result is asked of must be there."""
    cache, scales = apart(0, (9, 2, 16, 64), Q.UINT8), apart(1, (9, 2), Q.UINT8)
    slots, out = apart(2, (4,), Q.INT32), apart(3, (4, 2, 64))
    for args, kw, needle in (((None, None, None, None, slots), {}, "null result pointers"),
                             ((None, cache, None, scales, slots), dict(k_out=out), "missing k_cache"),
                             ((cache, None, scales, None, slots), dict(v_out=out), "missing v_cache"),
                             ((cache, None, None, None, slots), {}, "missing k_scales"),
                             ((None, cache, None, None, slots), {}, "missing v_scales"),
                             ((None, cache, None, scales, slots), dict(v_out=scales), "another shape")):
        Q.lib.qmm_reset_faults_for_test()
        with pytest.raises(Q.QmmError, match=needle):
            Q.cache_read_fp8(*args, **kw)
    Q.lib.qmm_reset_faults_for_test()


def test_the_chunk_kernels_are_among_those_looked_at_for_spills():
    """Six of them, as over a bfloat16 cache: none drops out of the search for spilled vector registers."""
    found = {}
    for m in re.finditer(rb"\.symbol[\xa0-\xda](.{1,400}?)\.kd.{0,400}?\.vgpr_spill_count(.)", Path(Q.lib._name).read_bytes(), re.S):
        found[m.group(1).decode("latin-1")] = m.group(2)[0]
    chunk = {n: c for n, c in found.items() if "attn_chunk8_kernel" in n}
    assert len(chunk) == 6 and not any(chunk.values())
