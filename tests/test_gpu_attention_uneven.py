"""Paged attention where the tokens of a step lie unevenly over the requests: some have none, another several."""
import math

import attention_ref as ref
import numpy as np
import pytest
import torch

import qmm as Q

pytestmark = pytest.mark.gpu


def ints(v):
    return Q.Array.from_numpy(np.asarray(v, dtype=np.int32), Q.INT32)


def dev(t):
    return Q.Array.from_torch(t.cuda().contiguous())


def into_nan(c, q, starts, kv, **kw):
    """paged_attention of a Cache into an array of NaN: what is left unwritten shows."""
    out = torch.full(q.shape, math.nan, dtype=torch.bfloat16, device="cuda")
    Q.paged_attention(dev(q), dev(c.k), dev(c.v), ints(c.table), ints(starts), ints(kv), out=Q.Array.from_torch(out), **kw)
    torch.cuda.synchronize()
    return out.cpu()


UNEVEN = [  # Hq, Hkv, D, block, [(cached, new)]: no more tokens than requests
    (24, 4, 256, 16, [(1000, 2), (5, 0)]),
    (24, 4, 256, 16, [(297, 3), (0, 0), (40, 0), (9, 1)]),
    (24, 4, 256, 16, [(8996, 4)] + [(0, 0)] * 3),
    (24, 4, 256, 16, [(300, 0)] * 60 + [(8990, 10)] + [(17, 0)] * 3),
    (32, 8, 128, 16, [(700, 4)] + [(30, 0)] * 7),
    (32, 8, 128, 16, [(9000, 0), (8998, 2)]),
    (16, 16, 64, 24, [(20, 0), (0, 0), (9000, 3), (300, 1)]),
    (16, 16, 64, 16, [(0, 0)] * 3 + [(280, 64)] + [(33, 0)] * 60),
    (6, 1, 80, 16, [(300, 4), (300, 0), (300, 0), (9000, 0)]),
]


@pytest.mark.parametrize("Hq,Hkv,D,block,lens", UNEVEN)
@pytest.mark.parametrize("gated", [False, True])
def test_idle_requests_beside_one_of_several_tokens(Hq, Hkv, D, block, lens, gated):
    """Every row is written, whatever request its token is of (bound: as every attention test)."""
    new, kv = [n for _, n in lens], [c + n for c, n in lens]
    T, g = sum(new), torch.Generator().manual_seed(D + len(lens))
    c = ref.Cache(kv, Hkv, D, block, seed=D)
    q = (2 * torch.randn(T, Hq, D, generator=g)).to(torch.bfloat16)
    gate = torch.randn(T, Hq, D, generator=g).to(torch.bfloat16) if gated else None
    starts = [0] + np.cumsum(new).tolist()
    want, bound = ref.attend(q, c.keys, c.values, starts, kv, D ** -0.5, 0, gate)
    got = into_nan(c, q, starts, kv, scale=D ** -0.5, gate=dev(gate) if gated else None)
    assert not torch.isnan(got).any()
    assert ((got.double() - want).abs() <= bound).all()


def test_a_captured_step_whose_tokens_move_between_requests():
    """One graph of R rows for R requests: one token each, then all of one request, then some of a few."""
    Hq, Hkv, D, block, R = 24, 4, 256, 16, 6
    lens = [2000, 310, 77, 4000, 600, 16]
    c = ref.Cache(lens, Hkv, D, block, seed=31)
    q = (2 * torch.randn(R, Hq, D, generator=torch.Generator().manual_seed(32))).to(torch.bfloat16)
    starts, out = torch.zeros(R + 1, dtype=torch.int32, device="cuda"), torch.empty(R, Hq, D, dtype=torch.bfloat16, device="cuda")
    a = [dev(q), dev(c.k), dev(c.v), ints(c.table), Q.Array.from_torch(starts, Q.INT32), ints(lens)]
    o, side = Q.Array.from_torch(out), torch.cuda.Stream()
    steps = [[1] * 6, [6, 0, 0, 0, 0, 0], [0, 3, 0, 2, 1, 0], [0, 0, 0, 5, 0, 0], [1] * 6]

    def put(new):
        starts.copy_(torch.tensor([0] + np.cumsum(new).tolist(), dtype=torch.int32))
        out.fill_(math.nan)
        torch.cuda.synchronize()

    put(steps[0])
    Q.paged_attention(*a, scale=1 / 16, out=o, stream=Q.Stream(side.cuda_stream))  # (the stream's workspace)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        Q.paged_attention(*a, scale=1 / 16, out=o, stream=Q.Stream.torch_current())
    for new in steps:
        put(new)
        graph.replay()
        torch.cuda.synchronize()
        got = out.cpu()
        want, bound = ref.attend(q, c.keys, c.values, starts.tolist(), lens, 1 / 16)
        assert not torch.isnan(got).any(), new
        assert ((got.double() - want).abs() <= bound).all(), new


@pytest.mark.parametrize("Hq,Hkv,D,lens", [
    (24, 4, 256, [(3000, 1), (5, 2)]), (8, 2, 128, [(300, 200), (900, 1), (0, 0), (17, 40)]), (4, 4, 72, [(0, 300)]),
])
def test_the_result_in_place_of_q_or_of_the_gate(Hq, Hkv, D, lens):
    """The same bits as in an array of its own, whole tiles and joined ones, both kernels."""
    new, kv = [n for _, n in lens], [c + n for c, n in lens]
    T, g = sum(new) + 2, torch.Generator().manual_seed(D)
    c = ref.Cache(kv, Hkv, D, 16, seed=D)
    q, gate = (torch.randn(T, Hq, D, generator=g).to(torch.bfloat16) for _ in range(2))
    starts = [0] + np.cumsum(new).tolist()
    apart = into_nan(c, q, starts, kv, scale=0.1, gate=dev(gate))
    for which in (0, 1):
        a = [t.cuda() for t in (q, gate)]
        h = [Q.Array.from_torch(t) for t in a]
        Q.paged_attention(h[0], dev(c.k), dev(c.v), ints(c.table), ints(starts), ints(kv), scale=0.1, gate=h[1], out=h[which])
        torch.cuda.synchronize()
        assert torch.equal(a[which].cpu(), apart) and torch.equal(a[1 - which].cpu(), (q, gate)[1 - which])
