"""A paged key/value cache held in 8 bits: plain forms, inputs and cases of its operators.

A case is a dict with an "op":

  write   head norms and rotation of q and k, k and v quantised into their cache rows
  read    cache rows back as [T, Hkv, D]
  attend  attention of each request's new tokens over its pages

Cache pages are [pages, Hkv, block, D] E4M3 codes with a scale 2^t for each page and head, held as t + 127 in 8 bits.
A request's page list is a row of the block table.  Requests' lengths are drawn from the case ("lens"), what the tensors
hold from the seed.
"""
import math
import random
import sys
from pathlib import Path

import torch

own = False


def listed():
    return [
        # one decoded token of a layer whose q projection carries the gate beside each head
        dict(name="write decode t1", op="write", R=1, nmin=1, nmax=1, ctx=8192, Hq=24, Hkv=4, D=256, Dq=512, rot=64,
             norm=True, pairs=False, dtype="bfloat16", block=16, lens=1),
        # the step of sequences decoded together, drafts of two among them; an odd page size, all of the head rotated,
        # pairs side by side, float32
        dict(name="write decode r64 f32", op="write", R=64, nmin=1, nmax=3, ctx=8192, Hq=28, Hkv=4, D=96, Dq=96, rot=96,
             norm=False, pairs=True, dtype="float32", block=24, lens=2),
        # a prompt's chunk behind an earlier one that ended inside a page
        dict(name="write chunk t2048", op="write", R=1, nmin=2048, nmax=2048, ctx=16000, Hq=24, Hkv=4, D=256, Dq=512, rot=64,
             norm=True, pairs=False, dtype="bfloat16", block=16, lens=3),
        # a short context read back exactly, to turn its keys to other positions
        dict(name="read t333 f32", op="read", R=1, nmin=333, nmax=333, Hkv=8, D=128, block=24, dtype="float32", lens=4),
        # a step's prefixes read back for a consumer of bfloat16
        dict(name="read r9 of 32768", op="read", R=9, nmin=100, nmax=32768, Hkv=4, D=256, block=64, dtype="bfloat16", lens=5),
        # one token over a short context: latency
        dict(name="attend decode 2k", op="attend", R=1, qmin=1, qmax=1, kmin=1999, kmax=1999, Hq=24, Hkv=4, D=256,
             block=16, window=0, gate=True, lens=6),
        # one token over the longest context of the models served
        dict(name="attend decode 262144", op="attend", R=1, qmin=1, qmax=1, kmin=262144, kmax=262144, Hq=24, Hkv=4,
             D=256, block=64, window=0, gate=True, lens=7),
        # sequences of all lengths decoded together
        dict(name="attend batch decode r64", op="attend", R=64, qmin=1, qmax=1, kmin=1, kmax=8192, Hq=32, Hkv=8, D=128,
             block=16, window=0, gate=False, lens=8),
        # drafts of two being verified in eight sequences
        dict(name="attend verify r8", op="attend", R=8, qmin=3, qmax=3, kmin=100, kmax=32768, Hq=24, Hkv=4, D=256,
             block=16, window=0, gate=True, lens=9),
        # a chunk of a long prompt: most of its attention time
        dict(name="attend chunk 2048 of 32768", op="attend", R=1, qmin=2048, qmax=2048, kmin=32768, kmax=32768, Hq=24,
             Hkv=4, D=256, block=16, window=0, gate=True, lens=10),
        # a prompt from its start
        dict(name="attend prompt 4000", op="attend", R=1, qmin=4000, qmax=4000, kmin=4000, kmax=4000, Hq=32, Hkv=8, D=128,
             block=32, window=0, gate=False, lens=11),
        # ragged chunks of prompts with a sliding window, a head of its own for every query, pages of an odd size
        dict(name="attend prompts r7 window", op="attend", R=7, qmin=1, qmax=2048, kmin=0, kmax=4000, Hq=16, Hkv=16,
             D=64, block=24, window=1000, gate=False, lens=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("write", "write", "read", "attend", "attend", "attend"))
    block = rng.choice((16, 16, 32, 64, 24, 128, 7))
    Hq, Hkv, D = rng.choice(((24, 4, 256), (24, 4, 256), (32, 8, 128), (64, 8, 128), (28, 4, 128), (16, 16, 64),
                             (8, 1, 256), (12, 12, 96), (40, 8, 80), (20, 4, 208)))
    dtype = rng.choice(("bfloat16", "float32"))
    lens = rng.randrange(1 << 20)
    if op == "write":
        R, n = rng.choice(((1, _log(rng, 1, 2048)), (_log(rng, 1, 256), rng.randint(1, 3)), (rng.randint(2, 9), _log(rng, 4, 200))))
        while R * n * Hq * D > 2048 * 24 * 256:
            R, n = (R, n // 2) if n > 1 else (R // 2, n)
        return dict(op=op, R=R, nmin=rng.choice((1, n)), nmax=n, ctx=_log(rng, 16, 200000), Hq=Hq, Hkv=Hkv, D=D,
                    Dq=D * rng.choice((1, 2)), rot=rng.choice((D, D // 2)), norm=rng.random() < 0.5,
                    pairs=rng.random() < 0.5, dtype=dtype, block=block, lens=lens)
    if op == "read":
        R = rng.choice((1, 1, 3, 20))
        n = _log(rng, 1, 40000 // R)
        return dict(op=op, R=R, nmin=rng.choice((1, n)), nmax=n, Hkv=Hkv, D=D, block=block, dtype=dtype, lens=lens)
    kind = rng.choice(("decode", "decode", "verify", "chunk", "chunk"))
    window = rng.choice((0, 0, _log(rng, 16, 8192)))
    case = dict(op=op, Hq=Hq, Hkv=Hkv, D=D, block=block, window=window, gate=rng.random() < 0.5, lens=lens)
    if kind == "chunk":
        R, qmax = rng.choice((1, 1, 2, 5, 9)), _log(rng, 16, 2048)
        case.update(R=R, qmin=rng.choice((1, qmax)), qmax=qmax, kmin=0, kmax=_log(rng, 16, 30720))
    else:
        R, q = _log(rng, 1, 128), 1 if kind == "decode" else rng.randint(2, 8)
        case.update(R=R, qmin=q, qmax=q, kmin=1, kmax=_log(rng, 64, 262144))
    # no more than the largest listed case: scores and gathered keys of the plain form, and the work itself
    while case["R"] * (case["kmax"] + case["qmax"]) * max(Hq * case["qmax"], 16 * Hkv * D) > 1.6e9:
        case["kmax" if case["kmax"] > 64 else "R"] //= 2
    case["kmin"] = min(case["kmin"], case["kmax"])
    return case


# ---------------------------------------------------------------- inputs


def _lens(case):
    """(cached tokens, new tokens) of each request; read: (0, its tokens)."""
    rng = random.Random(case["lens"])
    R = case["R"]
    if case["op"] == "attend":
        new = [case["qmax"] if r == 0 else rng.randint(case["qmin"], case["qmax"]) for r in range(R)]
        kmin, kmax = case["kmin"], case["kmax"]
        # contexts (the new tokens among them) spread over their logarithm, the longest always there
        kv = [kmax if r == 0 else _log(rng, kmin + 1, kmax + 1) - 1 for r in range(R)]
        return [max(0, k - n) for k, n in zip(kv, new)], new
    new = [case["nmax"] if r == 0 else _log(rng, case["nmin"], case["nmax"]) for r in range(R)]
    return [0 if case["op"] == "read" or rng.random() < 0.1 else _log(rng, 1, case["ctx"]) for r in range(R)], new


class _Rand:
    """Tensors from one seed, in the order they are asked for."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(int(seed))

    def normal(self, *shape, dtype=torch.bfloat16, scale=1.0):
        return (torch.randn(shape, generator=self.g, device="cuda") * scale).to(dtype)

    def order(self, n):
        return torch.randperm(n, generator=self.g, device="cuda").int()

    def cache(self, pages, Hkv, block, D):
        """Codes and scales of values whose size varies from head to head and page to page."""
        x = self.normal(pages, Hkv, block, D, dtype=torch.float32)
        x *= torch.exp(0.4 * self.normal(pages, Hkv, 1, 1, dtype=torch.float32))
        t = _exponent(x.abs().amax((2, 3)))
        codes = (x * _pow2(-t)[:, :, None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
        return codes, (t + 127).to(torch.uint8)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _starts(new):
    return _ints([0] + [sum(new[:i + 1]) for i in range(len(new))])


class State:
    """A case's inputs, result buffers and (once made) the library's handles."""

    def __init__(self, case):
        self.case, self.t, self.out, self.h = case, {}, {}, None


def _slots(r, cached, new, block, pages_of):
    """Cache slots of the requests' new tokens, pages in no order; how many pages there are."""
    held = [pages_of(c, n) for c, n in zip(cached, new)]  # (first page that counts, how many)
    total = 2 * sum(k for _, k in held) + 3
    order, slots, at = r.order(total), [], 0
    for (first, k), c, n in zip(held, cached, new):
        pos = torch.arange(c, c + n, device="cuda")
        slots.append(order[at:at + k][pos // block - first] * block + (pos % block).int())
        at += k
    return torch.cat(slots), total


def prepare(case, seed):
    s, r, op = State(case), _Rand(seed), case["op"]
    t = s.t
    cached, new = _lens(case)
    Hkv, D, bs, T = case["Hkv"], case["D"], case["block"], sum(new)
    s.n = T
    if op in ("write", "read"):
        pages_of = lambda c, n: (c // bs, (c + n - 1) // bs - c // bs + 1)  # noqa: E731
        t["slots"], pages = _slots(r, cached, new, bs, pages_of)
        for n in ("k", "v"):
            t[n + "_cache"], t[n + "_scales"] = r.cache(pages, Hkv, bs, D)
        dt = getattr(torch, case["dtype"])
        if op == "read":
            s.out.update(k=torch.empty(T, Hkv, D, dtype=dt, device="cuda"), v=torch.empty(T, Hkv, D, dtype=dt, device="cuda"))
            return s
        Hq = case["Hq"]
        t["q"] = r.normal(T, Hq, case["Dq"], dtype=dt)
        # keys have a few large channels
        t["k"] = (r.normal(T, Hkv, D, dtype=torch.float32) * torch.exp(0.5 * r.normal(Hkv, D, dtype=torch.float32))).to(dt)
        t["v"] = r.normal(T, Hkv, D, dtype=dt)
        t["positions"] = torch.cat([torch.arange(c, c + n, device="cuda") for c, n in zip(cached, new)]).int()
        t["freqs"] = torch.tensor([1e7 ** (-2 * i / case["rot"]) for i in range(case["rot"] // 2)], dtype=torch.float32,
                                  device="cuda")
        if case["norm"]:
            t["q_norm"], t["k_norm"] = r.normal(D, scale=0.1) + 1, r.normal(D, scale=0.1) + 1
        s.out["q"] = torch.empty(T, Hq, D, dtype=torch.bfloat16, device="cuda")
        return s
    Hq, R = case["Hq"], case["R"]
    kv = [c + n for c, n in zip(cached, new)]
    s.qmax, s.kmax = max(new), max(kv)
    pages = [-(-k // bs) for k in kv]
    W = max(pages)
    order = r.order(sum(pages) + 7)
    t["table"] = torch.full((R, W), -1, dtype=torch.int32, device="cuda")
    t["table"][torch.arange(W, device="cuda") < _ints(pages)[:, None]] = order[:sum(pages)]
    t["starts"], t["kv"] = _starts(new), _ints(kv)
    # scores of deviation 2 and more: a few keys carry most of a row
    t["q"] = r.normal(T, Hq, D, scale=2.0)
    for n in ("k", "v"):
        t[n + "_cache"], t[n + "_scales"] = r.cache(sum(pages) + 7, Hkv, bs, D)
    if case["gate"]:
        t["gate"] = r.normal(T, Hq, 2 * D)
    s.out["o"] = torch.empty(T, Hq, D, dtype=torch.bfloat16, device="cuda")
    return s


# ---------------------------------------------------------------- the library's calls


def _call(s):
    if s.h is None:  # a program makes its handles once
        sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "mlx-runner_amd"))
        import qmm as Q

        s.lib, s.stream = Q, Q.Stream.torch_current()
        s.h = {k: Q.Array.from_torch(v, Q.INT32 if v.dtype == torch.int32 else None) for k, v in s.t.items()}
        s.o = {k: Q.Array.from_torch(v) for k, v in s.out.items()}
    c, h, o, Q = s.case, s.h, s.o, s.lib
    cache = h["k_cache"], h["v_cache"], h["k_scales"], h["v_scales"]
    if c["op"] == "write":
        Q.rope_cache_fp8(h["q"], h["k"], h["v"], *cache, h["positions"], h["slots"], h["freqs"], interleaved=c["pairs"],
                         q_norm=h.get("q_norm"), k_norm=h.get("k_norm"), q_out=o["q"], stream=s.stream)
        return _written(s, s.out["q"])
    if c["op"] == "read":
        Q.cache_read_fp8(*cache, h["slots"], dtype=getattr(Q, c["dtype"].upper()), k_out=o["k"], v_out=o["v"], stream=s.stream)
        return s.out
    Q.paged_attention_fp8(h["q"], *cache, h["table"], h["starts"], h["kv"], gate=h.get("gate"), scale=c["D"] ** -0.5,
                          window=c["window"], out=o["o"], stream=s.stream)
    return s.out["o"]


def _written(s, q):
    """The caches as the values that their codes and scales stand for."""
    t = s.t
    return {"q": q, **{n + "_cache": t[n + "_cache"].view(torch.float8_e4m3fn) for n in ("k", "v")},
            **{n + "_scales": t[n + "_scales"].view(torch.float8_e8m0fnu) for n in ("k", "v")}}


# ---------------------------------------------------------------- plain forms


def _pow2(t):
    """2^t, exactly, from its bits."""
    return ((t.long() + 1023) << 52).view(torch.float64).float()


def _exponent(amax):
    """The smallest t, at least -127, with 448 * 2^t >= amax."""
    m, e = torch.frexp(amax)
    t = torch.where(m <= 0.875, e - 9, e - 8)
    return torch.where(amax > 0, t, -127).clamp(-127, 127)


def _values(codes, scales):
    """Codes [..., n, D] with scales [...]."""
    return codes.view(torch.float8_e4m3fn).float() * _pow2(scales.int() - 127)[..., None, None]


def _turn(x, positions, freqs, pairs):
    """The rotation of x [T, H, D] float32; angles in 64 bits (32 leave 0.008 rad at position 2^17)."""
    angle = (positions.double()[:, None] * freqs.double())[:, None, :]
    c, sn = angle.cos().float(), angle.sin().float()
    n = freqs.numel()
    if pairs:
        a, b = x[..., 0:2 * n:2], x[..., 1:2 * n:2]
        return torch.cat((torch.stack((a * c - b * sn, a * sn + b * c), -1).flatten(-2), x[..., 2 * n:]), -1)
    a, b = x[..., :n], x[..., n:2 * n]
    return torch.cat((a * c - b * sn, a * sn + b * c, x[..., 2 * n:]), -1)


def _normed(x, w):
    return x if w is None else x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.float()


def _store(cache, scales, slots, x):
    """x [T, Hkv, D] float32 into the rows `slots`.  A page whose first row is among them starts anew, with the scale that
    its new rows need; another page's scale only grows, and its older rows follow."""
    P, Hkv, bs, D = cache.shape
    page, off = slots.long().div(bs, rounding_mode="floor"), slots.long() % bs
    at = page[:, None].expand(-1, Hkv)
    top = torch.zeros(P, Hkv, device=x.device).scatter_reduce_(0, at, x.abs().amax(-1), "amax")
    begun = torch.zeros(P, dtype=torch.int32, device=x.device).scatter_reduce_(0, page, (off == 0).int(), "amax").bool()
    written = torch.zeros(P, dtype=torch.bool, device=x.device).index_fill_(0, page, True)
    old, need = scales.int() - 127, _exponent(top)
    t = torch.where(written[:, None], torch.where(begun[:, None], need, torch.maximum(old, need)), old)
    grown = _pow2(torch.where(begun[:, None], 0, old - t))[:, :, None, None]
    cache.copy_((cache.view(torch.float8_e4m3fn).float() * grown).to(torch.float8_e4m3fn).view(torch.uint8))
    cache[page, :, off] = (x * _pow2(-t)[page][..., None]).to(torch.float8_e4m3fn).view(torch.uint8)
    scales.copy_(t + 127)


def _write(s):
    t, c = s.t, s.case
    q = _turn(_normed(t["q"][..., :c["D"]].float(), t.get("q_norm")), t["positions"], t["freqs"], c["pairs"])
    k = _turn(_normed(t["k"].float(), t.get("k_norm")), t["positions"], t["freqs"], c["pairs"])
    _store(t["k_cache"], t["k_scales"], t["slots"], k)
    _store(t["v_cache"], t["v_scales"], t["slots"], t["v"].float())
    return _written(s, q.to(torch.bfloat16))


def _read(s):
    t, bs, out = s.t, s.case["block"], {}
    page, off = t["slots"].long().div(bs, rounding_mode="floor"), t["slots"].long() % bs
    for n in ("k", "v"):
        x = t[n + "_cache"][page, :, off].view(torch.float8_e4m3fn).float()
        out[n] = (x * _pow2(t[n + "_scales"].int() - 127)[page][..., None]).to(getattr(torch, s.case["dtype"]))
    return out


def _gathered(cache, scales, table):
    """[R, Hkv, pages * block, D] float32 of the requests' pages."""
    at = table.long().clamp(min=0)
    x = _values(cache[at], scales[at]).transpose(1, 2)
    return x.reshape(x.shape[0], x.shape[1], -1, x.shape[-1])


def _attend(s):
    t, c = s.t, s.case
    R, Hq, Hkv, D = c["R"], c["Hq"], c["Hkv"], c["D"]
    starts, kv = t["starts"].long(), t["kv"].long()
    n, dev = starts[1:] - starts[:-1], starts.device
    k, v = (_gathered(t[x + "_cache"], t[x + "_scales"], t["table"]) for x in ("k", "v"))
    i = torch.arange(s.qmax, device=dev)
    q = t["q"][(starts[:-1, None] + i).clamp(max=s.n - 1)].float() * D ** -0.5  # [R, qmax, Hq, D]
    q = q.view(R, s.qmax, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4).reshape(R, Hkv, -1, D)
    j = torch.arange(k.shape[2], device=dev)
    pos = (kv - n)[:, None] + i
    seen = j <= pos[..., None]
    if c["window"]:
        seen &= j > pos[..., None] - c["window"]
    score = torch.matmul(q, k.transpose(2, 3)).view(R, Hkv, Hq // Hkv, s.qmax, -1)
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = score.sum(-1, keepdim=True)
    o = torch.matmul(score.view(R, Hkv, -1, score.shape[-1]), v).view(R, Hkv, Hq // Hkv, s.qmax, D)
    o = (o / torch.where(total == 0, 1.0, total)).permute(0, 3, 1, 2, 4).reshape(R, s.qmax, Hq, D)
    o = o[i < n[:, None]]  # the requests' rows in order: [T, Hq, D]
    if "gate" in t:
        o = o * torch.sigmoid(t["gate"][..., D:].float())
    return o.to(torch.bfloat16)


PLAIN = {"write": _write, "read": _read, "attend": _attend}


def run(s):
    return _call(s) if own else PLAIN[s.case["op"]](s)


# ---------------------------------------------------------------- what a pass cannot do without


def work(case):
    op = case["op"]
    cached, new = _lens(case)
    Hkv, D, bs, T = case["Hkv"], case["D"], case["block"], sum(new)
    size = 4 if case.get("dtype") == "float32" else 2
    if op == "write":
        Hq = case["Hq"]
        pages = sum((c + n - 1) // bs - c // bs + 1 for c, n in zip(cached, new))
        # q, k, v in, q and the codes out; positions and slots in, scales in and out
        return {"bytes": T * D * (Hq * (size + 2) + 2 * Hkv * (size + 1)) + 8 * T + 4 * pages * Hkv,
                "flops": T * (Hq + Hkv) * (3 * case["rot"] + (4 * D if case["norm"] else 0)) + 4 * T * Hkv * D}
    if op == "read":
        return {"bytes": 2 * T * Hkv * D * (1 + size) + 4 * T + 2 * Hkv * sum(-(-n // bs) for n in new), "flops": 2 * T * Hkv * D}
    Hq, w = case["Hq"], case["window"]
    keys = pairs = 0
    for c, n in zip(cached, new):
        keys += min(c + n, w + n - 1) if w else c + n
        # query i of the chunk sees min(c + i + 1, w) keys
        full = max(0, min(n, w - c)) if w else n
        pairs += full * c + full * (full + 1) // 2 + (n - full) * w
    return {"bytes": 2 * keys * Hkv * D + 2 * T * Hq * D * (3 if case["gate"] else 2) + (4 + 2 * Hkv) * keys // bs,
            "flops": 4 * pairs * Hq * D}


# ---------------------------------------------------------------- in 64 bits


def _decoded(codes):
    """E4M3 codes to float64, from their bits."""
    sign, e, m = codes.long() >> 7, codes.long() >> 3 & 15, codes.long() & 7
    x = torch.where(e > 0, (8 + m) * 2.0 ** (e.double() - 10), m * 2.0 ** -9)
    return torch.where((codes & 127) == 127, math.nan, torch.where(sign > 0, -x, x))


def _turn64(x, positions, freqs, pairs):
    """x [T, H, D] as complex numbers times e^(i angle)."""
    n = freqs.numel()
    angle = positions.double()[:, None] * freqs.double()
    z = torch.polar(torch.ones_like(angle), angle)[:, None, :]
    y = x.double().clone()
    if pairs:
        y[..., :2 * n] = torch.view_as_real(torch.view_as_complex(y[..., :2 * n].reshape(*y.shape[:-1], n, 2)) * z).flatten(-2)
        return y
    w = torch.complex(y[..., :n], y[..., n:2 * n]) * z
    y[..., :n], y[..., n:2 * n] = w.real, w.imag
    return y


def _attend64(s):
    t, c = s.t, s.case
    cached, new = _lens(c)
    Hq, Hkv, D, bs = c["Hq"], c["Hkv"], c["D"], c["block"]
    out, at = torch.zeros(s.n, Hq, D, dtype=torch.float64, device="cuda"), 0
    for r, (have, n) in enumerate(zip(cached, new)):
        L = have + n
        pages = t["table"][r, :-(-L // bs)].long()
        pos = torch.arange(have, L, device="cuda")[:, None]
        j = torch.arange(L, device="cuda")
        hidden = j > pos
        if c["window"]:
            hidden = hidden | (j <= pos - c["window"])
        for h in range(Hkv):
            k, v = ((_decoded(t[x + "_cache"][pages, h]) * 2.0 ** (t[x + "_scales"][pages, h].double() - 127)[:, None, None])
                    .reshape(-1, D)[:L] for x in ("k", "v"))
            for g in range(h * Hq // Hkv, (h + 1) * Hq // Hkv):
                score = t["q"][at:at + n, g].double() @ k.t() / math.sqrt(D)
                out[at:at + n, g] = torch.softmax(score.masked_fill(hidden, -math.inf), -1) @ v
        at += n
    if "gate" in t:
        out = out / (1 + torch.exp(-t["gate"][..., D:].double()))
    return out


def _store64(codes, scales, slots, x):
    """The caches' codes before their rounding: page by page."""
    P, Hkv, bs, D = codes.shape
    y, rows = _decoded(codes), {}
    for i, slot in enumerate(slots.tolist()):
        rows.setdefault(slot // bs, []).append((i, slot % bs))
    for page, at in rows.items():
        i, off = torch.tensor([a for a, _ in at], device="cuda"), torch.tensor([b for _, b in at], device="cuda")
        top = x[i].abs().amax((0, 2))
        t = torch.ceil(torch.log2(top / 448)).clamp(-127, 127)
        t = torch.where(448 * 2.0 ** (t - 1) >= top, t - 1, torch.where(448 * 2.0 ** t < top, t + 1, t))  # (the logarithm is rounded)
        if all(b != 0 for _, b in at):
            old = scales[page].double() - 127
            t = torch.maximum(t, old)
            y[page] *= 2.0 ** (old - t)[:, None, None]
        y[page][:, off] = (x[i] / 2.0 ** t[:, None]).transpose(0, 1)
    return y


def exact(case, seed):
    s = prepare(case, seed)
    t, op, bs = s.t, case["op"], case["block"]
    if op == "attend":
        return _attend64(s)
    if op == "read":
        page, off = t["slots"].long() // bs, t["slots"].long() % bs
        return {n: _decoded(t[n + "_cache"])[page, :, off] * 2.0 ** (t[n + "_scales"][page].double() - 127)[..., None]
                for n in ("k", "v")}
    x = {}
    for n in ("q", "k"):
        x[n] = t[n][..., :case["D"]].double()
        if case["norm"]:
            x[n] = x[n] / (x[n].pow(2).sum(-1, keepdim=True) / case["D"] + 1e-6).sqrt() * t[n + "_norm"].double()
        x[n] = _turn64(x[n], t["positions"], t["freqs"], case["pairs"])
    return {"q": x["q"], "k_cache": _store64(t["k_cache"], t["k_scales"], t["slots"], x["k"]),
            "v_cache": _store64(t["v_cache"], t["v_scales"], t["slots"], t["v"].double()), "k_scales": None, "v_scales": None}
