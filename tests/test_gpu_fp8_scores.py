"""Scores over a cache held in 8 bits whose products differ far in size: as the f32 sums of the products that they are."""
import fp8_ref as ref
import pytest
import torch
from test_gpu_fp8_attention import attention, close

pytestmark = pytest.mark.gpu


def large_channels(L, D, kind, seed):
    """Keys with one value in 32 (or in eight, of signs that cancel) far above the others, as channels of trained keys are."""
    c = ref.Cache([L], 2, D, 16, seed=seed, spread=0.0)
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(L, 2, D, generator=g) * 8
    q = torch.randn(D, generator=g)
    at = dict(one=[5], each=list(range(3, D, 32)), cancel=list(range(0, D, 8)))[kind]
    x[..., at] = 448.0
    q[at] = 8.0
    if kind == "cancel":
        q[at[1::2]] = -8.0
    slots = [int(c.table[0, i // 16]) * 16 + i % 16 for i in range(L)]
    c.k, c.ks, _ = ref.store(c.k, c.ks, slots, x.double())
    return c, q


@pytest.mark.parametrize("new", [1, 4])
@pytest.mark.parametrize("D", [16, 64, 96, 128, 208, 256])
@pytest.mark.parametrize("kind", ["one", "each", "cancel"])
def test_products_of_all_sizes(kind, D, new):
    L = 500
    c, q = large_channels(L, D, kind, D)
    q = (q * (1 + 0.1 * torch.rand(new, 4, 1, generator=torch.Generator().manual_seed(new)))).to(torch.bfloat16)
    want, bound = ref.attend(q.cuda(), c.keys, c.values, [0, new], [L], D ** -0.5, few=True)
    assert close(attention(c, q, [0, new], [L]), want, bound)


@pytest.mark.parametrize("new", [40, 150])
@pytest.mark.parametrize("D", [16, 64, 96, 128, 208, 256])
@pytest.mark.parametrize("kind", ["one", "each", "cancel"])
def test_products_of_all_sizes_for_many_rows(kind, D, new):
    L = 500
    c, q = large_channels(L, D, kind, D)
    q = (q * (1 + 0.1 * torch.rand(new, 4, 1, generator=torch.Generator().manual_seed(new)))).to(torch.bfloat16)
    want, bound = ref.attend(q.cuda(), c.keys, c.values, [0, new], [L], D ** -0.5, scales=c.scales)
    assert close(attention(c, q, [0, new], [L]), want, bound)
