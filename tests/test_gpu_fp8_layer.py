"""The attention layer over a cache held in 8 bits: its calls together, step after step and as a captured step."""
import sys
from pathlib import Path

import fp8_ref as ref
import pytest
import torch

import qmm as Q

sys.path.insert(0, str(Path(Q.__file__).parent))
pytestmark = pytest.mark.gpu

A = Q.Array.from_torch


def projections(layer, x, step, s):
    """The layer's gated q, its turned q, and k, v as the projections leave them; y from o likewise."""
    T, D = x.shape[0], layer.D

    def empty(*shape):
        return torch.empty(shape, dtype=torch.bfloat16, device="cuda")

    q, k, v, turned = empty(T, layer.Hq, 2 * D), empty(T, layer.Hkv, D), empty(T, layer.Hkv, D), empty(T, layer.Hq, D)
    Q.quantized_matmul_group(A(x), layer.ws, layer.ss, layer.mode, outs=[A(t.view(T, -1)) for t in (q, k, v)], stream=s)
    spare = [torch.zeros(layer.k_cache.shape, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    Q.rope_cache(A(q), A(k), A(v), A(spare[0]), A(spare[1]), step["positions"], step["slots"], A(layer.freqs),
                 amplitude=layer.amplitude, q_norm=layer.norms[0], k_norm=layer.norms[1], q_out=A(turned), stream=s)
    return q, turned, k, v


def keys_of(layer, k, positions):
    """k after norm and rotation, in float64."""
    n = layer.freqs.numel()
    t = k.cpu().double()
    t = t * (t.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * layer.k_norm.cpu().double()
    angle = positions.cpu().double()[:, None, None] * layer.freqs.cpu().double()
    a, b = t[..., :n], t[..., n:2 * n]
    return torch.cat([a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos(), t[..., 2 * n:]], -1)


def wide(layer, w, s):
    a = Q.dequantize(A(w, Q.UINT32), A(s, Q.UINT8), layer.mode, dtype=Q.FLOAT32, stream=Q.Stream.torch_current())
    return torch.from_numpy(a.numpy(Q.Stream.torch_current())).double()


@pytest.mark.parametrize("Hq,Hkv,D,rot,block", [(6, 2, 64, 32, 16), (8, 1, 128, 128, 24), (12, 2, 256, 64, 7)])
def test_steps(Hq, Hkv, D, rot, block):
    """Prompts in two chunks of uneven parts, then decoded tokens; after every step

    - the rows it wrote, read back, against the float64 keys and values: half a step of E4M3 (2^-4 of a value, or half of
      2^-9 of its page's scale), and 2^-12 of the row's largest for the float32 rotation and norm;
    - a row that it did not write: as it was, or where its page's scale grew off by half of 2^-9 of the new one;
    - y against attention in float64 over the codes as they are, through the output projection: attend's bound through |w|,
      and 2^-8 of y and of sum |o w| for the projection (its product of bfloat16 o and exact weights sums in float32, K * 2^-24
      below that)."""
    from attention_layer import AttentionLayer, Pages

    K, steps = 512, ((37, 1, 300), (5, 64, 33), (1, 1, 1), (2, 0, 1), (1, 1, 1))
    lens = [sum(n) for n in zip(*steps)]
    width = -(-max(lens) // block)
    layer = AttentionLayer(K, Hq, Hkv, D, rot, 3 * width, block, mode="mxfp8", seed=3, cache="e4m3")
    pages = Pages(3, 3 * width, block, width)
    x = torch.randn(sum(lens), K, generator=torch.Generator().manual_seed(5)).to(torch.bfloat16).cuda()
    wo = wide(layer, layer.wo, layer.so)
    s, at, known = Q.Stream.torch_current(), 0, {}
    for new in steps:
        n = sum(new)
        pages.new.copy_(torch.tensor(new, dtype=torch.int32))
        part, at = x[at:at + n], at + n
        step = pages.step(n, s)
        q, turned, k, v = projections(layer, part, step, s)
        before = layer.read(torch.arange(3 * width * block, dtype=torch.int32, device="cuda"), s)
        y = layer(part, step, s).cpu().double()
        every = torch.arange(3 * width * block, dtype=torch.int32, device="cuda")
        slots = pages.slots.cpu().long()
        exact = keys_of(layer, k, pages.positions), v.cpu().double()
        for i, (codes, scales) in enumerate(((layer.k_cache, layer.k_scales), (layer.v_cache, layer.v_scales))):
            codes, scales = codes.cpu(), scales.cpu()
            rows = ref.decode(codes, scales).transpose(1, 2).reshape(-1, Hkv, D)  # by slot
            got = layer.read(every, s)[i].cpu().double()
            assert torch.equal(got, rows)
            f = (2.0 ** (scales.double() - 127)).repeat_interleave(block, 0)[:, :, None]  # of each slot and head
            want = exact[i]
            off = (got[slots] - want).abs()
            assert (off <= torch.maximum(2 ** -4 * want.abs(), 2 ** -10 * f[slots]) +
                    2 ** -12 * want.abs().amax(-1, keepdim=True)).all()
            old = torch.tensor(sorted(set(known) - set(slots.tolist())), dtype=torch.long)
            assert ((got[old] - before[i].cpu().double()[old]).abs() <= 2 ** -10 * f[old]).all()
        known.update(dict.fromkeys(slots.tolist()))
        table = pages.table.cpu().long()
        kv = pages.lens.tolist()
        read = []
        for r, L in enumerate(kv):
            j = torch.arange(L)
            read.append(layer.read((table[r, j // block] * block + j % block).int().cuda(), s))
        scales = [layer.v_scales.cpu()[table[r, torch.arange(L) // block]].double().sub(127).exp2() for r, L in enumerate(kv)]
        o, bound = ref.attend(turned.cpu(), [a.cpu().double() for a, _ in read], [b.cpu().double() for _, b in read],
                              pages.starts.tolist(), kv, D ** -0.5, gate=q[..., D:].cpu(), scales=scales)
        want = o.flatten(1) @ wo.T
        room = bound.flatten(1) @ wo.abs().T + 2 ** -8 * (want.abs() + o.flatten(1).abs() @ wo.abs().T)
        assert ((y - want).abs() <= room).all(), float(((y - want).abs() / room).max())
    assert pages.lens.tolist() == lens


def test_a_captured_step_follows_the_lengths():
    """Every replay bit for bit the eager step's, from the same state, with other work between; pages are begun and grow."""
    from attention_layer import AttentionLayer, Pages

    K, R, block, prompts, tokens = 256, 3, 8, (13, 1, 130), 12
    width = -(-(max(prompts) + tokens) // block)

    def fresh():
        layer = AttentionLayer(K, 6, 2, 128, 64, R * width, block, seed=7, cache="e4m3")
        torch.manual_seed(11)
        pages = Pages(R, R * width, block, width)
        return layer, pages

    xs = torch.randn(tokens, R, K, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    xs *= torch.linspace(0.2, 3, tokens, device="cuda")[:, None, None]
    first = torch.randn(sum(prompts), K, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        s = Q.Stream.torch_current()
        sides = []
        for _ in range(2):
            layer, pages = fresh()
            pages.new.copy_(torch.tensor(prompts, dtype=torch.int32))
            layer(first, pages.step(sum(prompts), s), s)
            pages.new.fill_(1)
            sides.append((layer, pages))
        (eager, p0), (captured, p1) = sides
        x = xs[0].clone()
        assert torch.equal(eager(x, p0.step(R, s), s), captured(x, p1.step(R, s), s))
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            y = captured(x, p1.step(R, s), s)
        for i in range(1, tokens):
            x.copy_(xs[i])
            graph.replay()
            want = eager(xs[i], p0.step(R, s), s)
            stream.synchronize()
            assert torch.equal(y, want), i
            assert torch.equal(p0.lens, p1.lens)
            for name in ("k_cache", "v_cache", "k_scales", "v_scales"):
                assert torch.equal(getattr(eager, name), getattr(captured, name)), (i, name)


def test_the_example_runs(capsys):
    import attention_layer

    attention_layer.main(prompts=(40, 3), tokens=4, K=512, cache="e4m3")
    assert "[44, 7] tokens each" in capsys.readouterr().out
    with pytest.raises(ValueError, match="cache must be"):
        attention_layer.AttentionLayer(512, 2, 1, 64, 32, 1, 16, cache="int8")
