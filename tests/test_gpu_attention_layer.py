"""The attention layer made of the library's calls against the same layer in 64 bits."""
import sys
from pathlib import Path

import pytest
import torch

import qmm as Q

sys.path.insert(0, str(Path(Q.__file__).parent))
pytestmark = pytest.mark.gpu


def plain(layer, x, lens):
    """y [T, K] in float64 on the CPU of requests of `lens` tokens each, from the quantized weights' own values."""
    def wide(w, s):
        a = Q.dequantize(Q.Array.from_torch(w, Q.UINT32), Q.Array.from_torch(s, Q.UINT8), layer.mode, dtype=Q.FLOAT32,
                         stream=Q.Stream.torch_current())
        return torch.from_numpy(a.numpy(Q.Stream.torch_current())).double()

    Hq, Hkv, D, n = layer.Hq, layer.Hkv, layer.D, layer.freqs.numel()
    p = x.cpu().double() @ wide(layer.w, layer.s).T
    q, k, v = p.split([2 * Hq * D, Hkv * D, Hkv * D], 1)
    q, k, v = q.view(-1, Hq, 2 * D), k.view(-1, Hkv, D), v.view(-1, Hkv, D)
    q, gate = q[..., :D], q[..., D:]
    pos = torch.cat([torch.arange(L) for L in lens]).double()
    angle = pos[:, None, None] * layer.freqs.cpu().double()

    def turned(t, w):
        t = t * (t.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w.cpu().double()
        a, b = t[..., :n], t[..., n:2 * n]
        return torch.cat([a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos(), t[..., 2 * n:]], -1)

    q, k = turned(q, layer.q_norm), turned(k, layer.k_norm)
    o, t0 = torch.zeros_like(q), 0
    for L in lens:
        rows = slice(t0, t0 + L)
        mask = torch.ones(L, L).tril().bool()
        for h in range(Hq):
            j = h // (Hq // Hkv)
            w = (q[rows, h] @ k[rows, j].T * D ** -0.5).masked_fill(~mask, -torch.inf).softmax(-1)
            o[rows, h] = w @ v[rows, j]
        t0 += L
    return (o * gate.sigmoid()).flatten(1) @ wide(layer.wo, layer.so).T


@pytest.mark.parametrize("mode", ["nvfp4", "mxfp8"])
def test_layer_prefill_chunks_and_decode(mode):
    """Prompts in two chunks of uneven parts, then two decoded tokens each: every token against all at once.

    Tolerance (of the norm of y): q, k, v, the turned q and k, the weights, o and y are each rounded to bf16, a relative
    2^-9 at most each; a score (normed heads: of the size of 1, 4 at most here) moves by 4 such roundings of itself and
    its weight with it.  6 roundings on the way of the values and 4 * 4 of the scores, added up: 22 * 2^-9 = 0.043."""
    from attention_layer import AttentionLayer, Pages

    K, block, first, second = 512, 16, (37, 1, 300), (5, 64, 33)
    lens = [a + b + 2 for a, b in zip(first, second)]
    width = -(-max(lens) // block)
    layer = AttentionLayer(K, 6, 2, 64, 32, 3 * width, block, mode=mode, seed=3)
    pages = Pages(3, 3 * width, block, width)
    x = torch.randn(sum(lens), K, generator=torch.Generator().manual_seed(5)).to(torch.bfloat16).cuda()
    want = plain(layer, x, lens)
    per, got, at = list(x.split(lens)), [[] for _ in lens], [0] * 3
    s = Q.Stream.torch_current()
    for new in (first, second, (1, 1, 1), (1, 1, 1)):
        pages.new.copy_(torch.tensor(new, dtype=torch.int32))
        part = torch.cat([per[r][at[r]:at[r] + n] for r, n in enumerate(new)])
        y = layer(part, pages.step(sum(new), s), s).cpu().double()
        for r, n in enumerate(new):
            got[r].append(y[:n])
            y, at[r] = y[n:], at[r] + n
    got = torch.cat([torch.cat(g) for g in got])
    assert pages.lens.tolist() == lens
    worst = ((got - want).norm(dim=1) / want.norm(dim=1)).max()
    assert worst < 22 * 2 ** -9, float(worst)


def test_the_example_runs(capsys):
    import attention_layer

    attention_layer.main(prompts=(40, 3), tokens=4, K=512)
    assert "decode step" in capsys.readouterr().out
