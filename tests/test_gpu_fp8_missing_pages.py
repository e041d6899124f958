"""Pages that are missing inside a context over a cache held in 8 bits, and the page that their keys' addresses fall on."""
import math

import fp8_ref as ref
import pytest
import torch
from test_gpu_fp8_attention import attention, close

pytestmark = pytest.mark.gpu


def with_holes(L, Hkv, D, block, seed, gone):
    """A cache of one request whose table has no page at the places `gone`, and no use for page 0; which keys there are."""
    c = ref.Cache([L], Hkv, D, block, seed=seed)
    if 0 in c.table[0]:
        spare = next(p for p in range(c.k.shape[0]) if p not in c.table[0])
        for t in (c.k, c.v, c.ks, c.vs):
            t[spare], t[0] = t[0].clone(), t[spare].clone()
        c.table[0][c.table[0] == 0] = spare
    there = torch.ones(L, dtype=torch.bool)
    for p in gone:
        there[p * block:(p + 1) * block] = False
    return c, there


def attend(c, there, q, L, window):
    """(o, bound) of fp8_ref.attend for one request's rows of q, the keys in `there` only: its bound for many rows, term by term."""
    n, Hq, D = q.shape
    K, V, f = (x[0].clone() for x in (c.keys, c.values, c.scales))
    K[~there], V[~there], f[~there] = 0, 0, 0
    g, j = Hq // K.shape[1], torch.arange(L)
    pos = (L - n + torch.arange(n))[:, None]
    seen = (j <= pos) & there & ((j > pos - window) if window else True)
    o, bound = torch.zeros(n, Hq, D, dtype=torch.float64), torch.zeros(n, Hq, D, dtype=torch.float64)
    for h in range(Hq):
        k, v, fh, x = K[:, h // g], V[:, h // g], f[:, h // g], q[:, h].double()
        p = torch.softmax((x @ k.T * D ** -0.5).masked_fill(~seen, -math.inf), -1).nan_to_num(0.0)  # (a row that sees nothing: 0)
        o[:, h] = p @ v
        most = torch.nn.functional.pad(x.abs(), (0, -D % 128)).view(n, -1, 128).amax(-1).repeat_interleave(128, 1)[:, :D]
        size = (2 * (D + 8) * 2 ** -24 * (x.abs() @ k.abs().T) + 2 * 2 ** -22 * (most @ k.abs().T)) * D ** -0.5
        weight = 2 * 2 ** -8 + size.masked_fill(~seen, 0).amax(-1, keepdim=True) + 2 ** -21 + 2 * (L / 16 + 64) * 2 ** -24
        # (two E4M3 parts: 2^-22 of 32 keys' largest weight at their largest scale, on all their codes)
        by32 = lambda t: torch.nn.functional.pad(t, (0, -L % 32)).unflatten(-1, (-1, 32))  # noqa: E731
        codes = (v.abs() / torch.where(fh > 0, fh, 1.0)[:, None]).T
        bound[:, h] = (weight * (p @ v.abs()) + 2 ** -8 * o[:, h].abs() + 1e-30
                       + 2 ** -22 * (by32(p).amax(-1) * by32(fh).amax(-1)) @ by32(codes).sum(-1).T)
    return o, bound


def check(c, there, gone, new, L, window, seed):
    c_table = c.table.copy()
    q = torch.randn(new, 4, c.k.shape[3], generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16)
    want, bound = attend(c, there, q, L, window)
    c.table[0, gone] = [(-1, c.k.shape[0], 2 ** 31 - 1, -2 ** 31)[i % 4] for i in range(len(gone))]
    got = attention(c, q, [0, new], [L], window=window)
    c.table = c_table
    assert torch.isfinite(got).all() and close(got, want, bound)


@pytest.mark.parametrize("new,window", [(1, 0), (3, 70), (90, 0), (150, 70), (90, 200)])
@pytest.mark.parametrize("D,block", [(64, 16), (128, 16), (128, 4), (256, 16), (64, 7), (96, 24), (208, 12)])
def test_the_first_pages_scales_are_nan(D, block, new, window):
    """Pages missing in the middle, at the start and, with a window, all those before its first key: page 0, which is no
    request's, holds NaN codes at scales of 255 (memory never written); no key that there is lies on it."""
    L = 400
    n = -(-L // block)
    before = (L - new - window + 1) // block if window else 1  # (pages that no row sees a key of)
    gone = sorted({*range(before), *range(n // 2, n // 2 + max(2, 40 // block)), n - 3})
    c, there = with_holes(L, 2, D, block, 40 + D, gone)
    assert (c.vs[0] == 255).all() and 0 not in c.table[0]
    check(c, there, gone, new, L, window, 41)


@pytest.mark.parametrize("new,window", [(3, 0), (90, 0), (150, 70)])
@pytest.mark.parametrize("D,block", [(64, 4), (128, 12), (256, 4), (256, 7), (256, 12), (208, 1), (256, 5), (256, 24)])
@pytest.mark.parametrize("first,others", [(121, (121,)), (119, (119, 125)), (120, (120, 112, 124)), (130, (115, 120)),
                                          (100, (115, 120)), (255, (119, 125)), (118, (118, 140))])
def test_eights_that_begin_with_missing_keys(D, block, new, window, first, others):
    """Every third page or so missing: the keys of a page that is there follow, among eight that go into the products together,
    keys of a page that is not, whose scale seems to be that of page 0: the same, larger, smaller, or NaN."""
    L = 400
    n = -(-L // block)
    gone = [p for p in range(n - 1) if p % 3 != 1] if block < 24 else [p for p in range(n - 1) if p % 2]
    c, there = with_holes(L, 2, D, block, 50 + D, gone)
    for i, p in enumerate(p for p in range(n) if p not in gone):
        c.vs[int(c.table[0, p])] = others[i % len(others)]
    c.vs[0] = first
    check(c, there, gone, new, L, window, 51)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("larger", [125, 127, 140])
def test_an_eight_after_missing_keys_beside_larger_scales(D, larger):
    """Pages of 12: none, one with page 0's scale, one with a larger: keys 12 to 15 keep their own, as 16 to 23 do."""
    c, there = with_holes(36, 2, D, 12, 60, [0])
    c.vs[int(c.table[0, 1])], c.vs[int(c.table[0, 2])], c.vs[0] = 119, larger, 119
    check(c, there, [0], 30, 36, 0, 61)
