"""Results that would replace or overwrite an input: refused before anything is allocated, freed or written."""
from ctypes import byref

import pytest
from test_attention_host import BS, CACHE, D, FAKE, Hkv, Hq, R, T, W, arr, ints

import qmm as Q


@pytest.fixture(autouse=True)
def _clean_latch():
    Q.lib.qmm_reset_faults_for_test()
    yield
    Q.lib.qmm_reset_faults_for_test()


def apart(n, shape, dtype=Q.BFLOAT16):
    """The n-th array of a set that do not overlap."""
    return arr(shape, dtype, ptr=FAKE + (n << 24))


def tables():
    return dict(table=apart(0, (R, W), Q.INT32), head=apart(1, (1,), Q.INT32), cached_lens=apart(2, (R,), Q.INT32),
                new_lens=apart(3, (R,), Q.INT32), free_blocks=apart(4, (7,), Q.INT32), block_size=BS, n_tokens=R)


@pytest.mark.parametrize("out,of,needle", [
    ("q_starts", "cached_lens", "q_starts is the handle of an input of another shape"),
    ("head_out", "cached_lens", "head_out is the handle of an input of another shape"),
    ("slots", "table", "slots is the handle of an input of another shape"),
    ("positions", "new_lens", "positions lies over an input"),
    ("slots", "cached_lens", "slots lies over an input"),
])
def test_block_tables_keeps_its_inputs(out, of, needle):
    a = tables()
    with pytest.raises(Q.QmmError, match=needle):
        Q.block_tables(**a, **{out: a[of]})
    assert a[of].ptr and a[of].shape  # (the handle still holds its array)


def test_block_tables_results_apart():
    a = tables()
    both = apart(9, (R,), Q.INT32)
    with pytest.raises(Q.QmmError, match="slots lies over positions"):
        Q.block_tables(**a, positions=both, slots=both)
    with pytest.raises(Q.QmmError, match="slots lies over positions"):
        Q.block_tables(**a, positions=both, slots=arr((R,), Q.INT32, ptr=both.ptr + 4))
    none = Q.qmm_array(None)
    others = [Q.qmm_array(None) for _ in range(4)]
    ins = [a[k].h for k in ("table", "head", "cached_lens", "new_lens", "free_blocks")]
    assert Q.lib.qmm_block_tables(*[byref(x) for x in others], byref(none), byref(none), *ins, BS, R, Q.qmm_stream(None))
    assert not none.ctx and not any(x.ctx for x in others)


@pytest.mark.parametrize("of,needle", [("positions", "another shape"), ("freqs", "another shape"), ("near", "lies over an input")])
def test_rope_keeps_its_inputs(of, needle):
    a = dict(x=apart(0, (T, Hq, D)), positions=apart(1, (T,), Q.INT32), freqs=apart(2, (16,), Q.FLOAT32))
    out = arr((T, Hq, D), ptr=a["x"].ptr + 256) if of == "near" else a[of]
    with pytest.raises(Q.QmmError, match=needle):
        Q.rope(**a, out=out)


def layer(**change):
    a = dict(q=apart(0, (T, Hq, D)), k=apart(1, (T, Hkv, D)), v=apart(2, (T, Hkv, D)), k_cache=apart(3, CACHE),
             v_cache=apart(4, CACHE), positions=apart(5, (T,), Q.INT32), slots=apart(6, (T,), Q.INT32),
             freqs=apart(7, (16,), Q.FLOAT32))
    return dict(a, **change)


@pytest.mark.parametrize("q", [apart(0, (T, Hq, 2 * D)), apart(0, (T, Hq, D), Q.FLOAT32)])
def test_rope_cache_does_not_replace_q(q):
    """q's own handle as q_out where q_out's layout is another: q would be freed before it is read."""
    a = layer(q=q, **({} if q.dtype == Q.BFLOAT16 else {n: apart(i, (T, Hkv, D), Q.FLOAT32) for i, n in ((1, "k"), (2, "v"))}))
    with pytest.raises(Q.QmmError, match="own array only at q's layout"):
        Q.rope_cache(**a, q_out=a["q"])
    assert a["q"].ptr and a["q"].shape == q.shape


def test_rope_cache_keeps_its_inputs():
    a = layer(k=apart(1, (T, Hq, D)), v=apart(2, (T, Hq, D)), k_cache=apart(3, (9, Hq, BS, D)), v_cache=apart(4, (9, Hq, BS, D)))
    for of in ("k", "v"):  # (as many key heads as query heads: the shapes are alike)
        with pytest.raises(Q.QmmError, match="q_out lies over an input"):
            Q.rope_cache(**a, q_out=a[of])
    for of in ("k_cache", "slots"):
        with pytest.raises(Q.QmmError, match="another shape"):
            Q.rope_cache(**a, q_out=a[of])


def test_paged_attention_keeps_its_inputs():
    a = dict(q=apart(0, (T, Hq, D)), k_cache=apart(1, CACHE), v_cache=apart(2, CACHE), table=apart(3, (R, W), Q.INT32),
             q_starts=apart(4, (R + 1,), Q.INT32), kv_lens=apart(5, (R,), Q.INT32), scale=0.125)
    for of in ("k_cache", "table", "kv_lens"):
        with pytest.raises(Q.QmmError, match="another shape"):
            Q.paged_attention(**a, out=a[of])
    wide = apart(6, (T, Hq, 2 * D))
    with pytest.raises(Q.QmmError, match="another shape"):
        Q.paged_attention(**a, gate=wide, out=wide)
    with pytest.raises(Q.QmmError, match="lies over an input"):
        Q.paged_attention(**a, gate=wide, out=arr((T, Hq, D), ptr=wide.ptr))
    with pytest.raises(Q.QmmError, match="lies over an input"):
        Q.paged_attention(**a, out=arr((T, Hq, D), ptr=a["q"].ptr + 16))
