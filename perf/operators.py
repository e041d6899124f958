"""Attention over a paged key/value cache, operator by operator: plain forms, inputs and cases.

A case is a dict with an "op":

  blocks  block tables, slots and positions of the step's tokens, from the requests' lengths
  rope    rotary positions of [T, H, D]
  write   head norms and rotation of q and k, k and v written to their cache rows
  attend  attention of each request's new tokens over its pages

Requests' lengths are drawn from the case ("lens"), what the tensors hold from the seed.
Cache pages are [pages, Hkv, block, D]; a request's page list is a row of the block table.
"""
import math
import random
import sys
from pathlib import Path

import torch

own = False


def listed():
    return [
        # the step of 64 sequences decoded together: one token each, now and then a new page
        dict(name="blocks decode r64", op="blocks", R=64, chunks=0, top=1, ctx=8192, block=16, lens=1),
        # a full step of a server: prompts' chunks beside hundreds of decoded sequences
        dict(name="blocks mixed r512", op="blocks", R=512, chunks=12, top=2048, ctx=32768, block=16, lens=2),
        # a draft head's few rows in float32, all of the head rotated, pairs side by side
        dict(name="rope f32 t37", op="rope", T=37, H=8, D=64, rot=64, dtype="float32", pairs=True, top=262144, amp=1.25),
        # the queries of a prompt's chunks, a quarter of each head rotated
        dict(name="rope bf16 t4096", op="rope", T=4096, H=24, D=256, rot=64, dtype="bfloat16", pairs=False, top=32768,
             amp=1.0),
        # one decoded token of a layer whose q projection carries the gate beside each head
        dict(name="write decode t1", op="write", T=1, Hq=24, Hkv=4, D=256, Dq=512, rot=64, norm=True, pairs=False,
             block=16, pages=2048, top=32768),
        # a prompt's chunk of the same layer
        dict(name="write chunk t2048", op="write", T=2048, Hq=24, Hkv=4, D=256, Dq=512, rot=64, norm=True, pairs=False,
             block=16, pages=2048, top=32768),
        # one token over a short context: latency
        dict(name="attend decode 2k", op="attend", R=1, qmin=1, qmax=1, kmin=1999, kmax=1999, Hq=24, Hkv=4, D=256,
             block=16, window=0, gate=True, lens=3),
        # one token over the longest context of the models served
        dict(name="attend decode 262144", op="attend", R=1, qmin=1, qmax=1, kmin=262144, kmax=262144, Hq=24, Hkv=4,
             D=256, block=64, window=0, gate=True, lens=4),
        # sequences of all lengths decoded together
        dict(name="attend batch decode r64", op="attend", R=64, qmin=1, qmax=1, kmin=1, kmax=8192, Hq=32, Hkv=8, D=128,
             block=16, window=0, gate=False, lens=5),
        # drafts of two being verified in eight sequences
        dict(name="attend verify r8", op="attend", R=8, qmin=3, qmax=3, kmin=100, kmax=32768, Hq=24, Hkv=4, D=256,
             block=16, window=0, gate=True, lens=6),
        # a chunk of a long prompt: most of its attention time
        dict(name="attend chunk 2048 of 32768", op="attend", R=1, qmin=2048, qmax=2048, kmin=32768, kmax=32768, Hq=24,
             Hkv=4, D=256, block=16, window=0, gate=True, lens=7),
        # ragged chunks of prompts with a sliding window, a head of its own for every query, pages of an odd size
        dict(name="attend prompts r7 window", op="attend", R=7, qmin=1, qmax=2048, kmin=0, kmax=4000, Hq=16, Hkv=16,
             D=64, block=24, window=1000, gate=False, lens=8),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("blocks", "rope", "write", "attend", "attend", "attend"))
    block = rng.choice((16, 16, 32, 64, 24, 128))
    Hq, Hkv, D = rng.choice(((24, 4, 256), (24, 4, 256), (32, 8, 128), (64, 8, 128), (28, 4, 128), (16, 16, 64),
                             (8, 1, 256), (12, 12, 96), (40, 8, 80)))
    if op == "blocks":
        R = _log(rng, 1, 512)
        return dict(op=op, R=R, chunks=min(R, rng.choice((0, 1, 4, 12))), top=_log(rng, 1, 2048), ctx=_log(rng, 16, 32768),
                    block=block, lens=rng.randrange(1 << 20))
    if op == "rope":
        T = _log(rng, 1, 4096)
        while T * Hq * D > 4096 * 24 * 256:
            T //= 2
        return dict(op=op, T=T, H=Hq, D=D, rot=rng.choice((D, D // 2, D // 4)), dtype=rng.choice(("bfloat16", "float32")),
                    pairs=rng.random() < 0.5, top=_log(rng, 4096, 262144), amp=rng.choice((1.0, 1.25)))
    if op == "write":
        T = _log(rng, 1, 2048)
        while T * Hq * D > 2048 * 24 * 256:
            T //= 2
        return dict(op=op, T=T, Hq=Hq, Hkv=Hkv, D=D, Dq=D * rng.choice((1, 2)), rot=rng.choice((D, D // 4)),
                    norm=rng.random() < 0.5, pairs=rng.random() < 0.5, block=block, pages=4096 // block * 8,
                    top=_log(rng, 4096, 262144))
    kind = rng.choice(("decode", "decode", "verify", "chunk", "chunk"))
    window = rng.choice((0, 0, _log(rng, 16, 8192)))
    case = dict(op=op, Hq=Hq, Hkv=Hkv, D=D, block=block, window=window, gate=rng.random() < 0.5,
                lens=rng.randrange(1 << 20))
    if kind == "chunk":
        R, qmax = rng.choice((1, 1, 2, 5, 9)), _log(rng, 16, 2048)
        case.update(R=R, qmin=rng.choice((1, qmax)), qmax=qmax, kmin=0, kmax=_log(rng, 16, 30720))
    else:
        R, q = _log(rng, 1, 128), 1 if kind == "decode" else rng.randint(2, 8)
        case.update(R=R, qmin=q, qmax=q, kmin=1, kmax=_log(rng, 64, 262144))
    # no more than the largest listed case: scores and gathered keys of the plain form, and the work itself
    while case["R"] * (case["kmax"] + case["qmax"]) * max(Hq * case["qmax"], 16 * Hkv * D) > 2e9:
        case["kmax" if case["kmax"] > 64 else "R"] //= 2
    case["kmin"] = min(case["kmin"], case["kmax"])
    return case


# ---------------------------------------------------------------- inputs


def _lens(case):
    """(cached tokens, new tokens) of each request."""
    rng = random.Random(case["lens"])
    R = case["R"]
    if case["op"] == "blocks":
        new = [_log(rng, 1, case["top"]) if r < case["chunks"] else 1 for r in range(R)]
        cached = [0 if r < case["chunks"] and r % 2 else _log(rng, 1, case["ctx"]) for r in range(R)]
        order = list(range(R))
        rng.shuffle(order)
        return [cached[r] for r in order], [new[r] for r in order]
    new = [case["qmax"] if r == 0 else rng.randint(case["qmin"], case["qmax"]) for r in range(R)]
    kmin, kmax = case["kmin"], case["kmax"]
    # contexts (the new tokens among them) spread over their logarithm, the longest always there
    kv = [kmax if r == 0 else _log(rng, kmin + 1, kmax + 1) - 1 for r in range(R)]
    return [max(0, k - n) for k, n in zip(kv, new)], new


class _Rand:
    """Tensors from one seed, in the order they are asked for."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(int(seed))

    def normal(self, *shape, dtype=torch.bfloat16, scale=1.0):
        return (torch.randn(shape, generator=self.g, device="cuda") * scale).to(dtype)

    def below(self, n, *shape):
        return torch.randint(0, n, shape, generator=self.g, device="cuda", dtype=torch.int32)

    def order(self, n):
        return torch.randperm(n, generator=self.g, device="cuda").int()


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _starts(new):
    return _ints([0] + [sum(new[:i + 1]) for i in range(len(new))])


def _freqs(rot):
    return torch.tensor([1e7 ** (-2 * i / rot) for i in range(rot // 2)], dtype=torch.float32, device="cuda")


class State:
    """A case's inputs, result buffers and (once made) the library's handles."""

    def __init__(self, case):
        self.case, self.t, self.out, self.h = case, {}, {}, None


def prepare(case, seed):
    s, r, op = State(case), _Rand(seed), case["op"]
    t = s.t
    if op == "blocks":
        cached, new = _lens(case)
        bs, R = case["block"], case["R"]
        W = -(-(case["ctx"] + case["top"]) // bs)
        held = [-(-c // bs) for c in cached]
        pages = r.order(sum(held) + R * (2 + case["top"] // bs))
        t["table"] = torch.full((R, W), -1, dtype=torch.int32, device="cuda")
        t["cached"], t["new"] = _ints(cached), _ints(new)
        mine = torch.arange(W, device="cuda") < _ints(held)[:, None]
        t["table"][mine] = pages[:sum(held)]
        t["free"], t["head"] = pages[sum(held):].clone(), _ints([3])
        s.n = sum(new)
        return s
    if op == "rope":
        dt = getattr(torch, case["dtype"])
        t["x"] = r.normal(case["T"], case["H"], case["D"], dtype=dt)
        t["positions"], t["freqs"] = r.below(case["top"], case["T"]), _freqs(case["rot"])
        s.out["x"] = torch.empty_like(t["x"])
        return s
    if op == "write":
        T, Hq, Hkv, D, bs = (case[k] for k in ("T", "Hq", "Hkv", "D", "block"))
        t["q"], t["k"], t["v"] = r.normal(T, Hq, case["Dq"]), r.normal(T, Hkv, D), r.normal(T, Hkv, D)
        for n in ("k_cache", "v_cache"):
            t[n] = r.normal(case["pages"], Hkv, bs, D)
        # whole pages in no order, as a request that has grown holds them
        at = r.below(case["top"] - T if case["top"] > T else 1, 1) + torch.arange(T, device="cuda", dtype=torch.int32)
        pages = r.order(case["pages"])
        t["positions"], t["slots"] = at, pages[(at - at[0]) // bs] * bs + (at - at[0]) % bs
        t["freqs"] = _freqs(case["rot"])
        if case["norm"]:
            t["q_norm"], t["k_norm"] = r.normal(D, scale=0.1) + 1, r.normal(D, scale=0.1) + 1
        s.out["q"] = torch.empty(T, Hq, D, dtype=torch.bfloat16, device="cuda")
        return s
    cached, new = _lens(case)
    Hq, Hkv, D, bs, R, T = case["Hq"], case["Hkv"], case["D"], case["block"], case["R"], sum(new)
    kv = [c + n for c, n in zip(cached, new)]
    s.n, s.qmax, s.kmax = T, max(new), max(kv)
    pages = [-(-k // bs) for k in kv]
    W = max(pages)
    order = r.order(sum(pages) + 7)
    t["table"] = torch.full((R, W), -1, dtype=torch.int32, device="cuda")
    t["table"][torch.arange(W, device="cuda") < _ints(pages)[:, None]] = order[:sum(pages)]
    t["starts"], t["kv"] = _starts(new), _ints(kv)
    # scores of deviation 2: a few keys carry most of a row
    t["q"] = r.normal(T, Hq, D, scale=2.0)
    t["k_cache"], t["v_cache"] = (r.normal(sum(pages) + 7, Hkv, bs, D) for _ in range(2))
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
        if s.case["op"] == "blocks":
            R, T = s.case["R"], s.n
            for name, n in (("head", 1), ("starts", R + 1), ("kv", R), ("positions", T), ("slots", T)):
                s.out[name] = torch.empty(n, dtype=torch.int32, device="cuda")
                s.o[name] = Q.Array.from_torch(s.out[name], Q.INT32)
    c, h, o, Q = s.case, s.h, s.o, s.lib
    if c["op"] == "blocks":
        Q.block_tables(h["table"], h["head"], h["cached"], h["new"], h["free"], c["block"], s.n, table_out=h["table"],
                       head_out=o["head"], q_starts=o["starts"], kv_lens=o["kv"], positions=o["positions"],
                       slots=o["slots"], stream=s.stream)
        return dict(s.out, table=s.t["table"])
    if c["op"] == "rope":
        Q.rope(h["x"], h["positions"], h["freqs"], amplitude=c["amp"], interleaved=c["pairs"], out=o["x"], stream=s.stream)
        return s.out["x"]
    if c["op"] == "write":
        Q.rope_cache(h["q"], h["k"], h["v"], h["k_cache"], h["v_cache"], h["positions"], h["slots"], h["freqs"],
                     interleaved=c["pairs"], q_norm=h.get("q_norm"), k_norm=h.get("k_norm"), q_out=o["q"],
                     stream=s.stream)
        return {"q": s.out["q"], "k_cache": s.t["k_cache"], "v_cache": s.t["v_cache"]}
    Q.paged_attention(h["q"], h["k_cache"], h["v_cache"], h["table"], h["starts"], h["kv"], gate=h.get("gate"),
                      scale=c["D"] ** -0.5, window=c["window"], out=o["o"], stream=s.stream)
    return s.out["o"]


# ---------------------------------------------------------------- plain forms


def _blocks(s):
    t, bs, T = s.t, s.case["block"], s.n
    table, R, W = t["table"], s.case["R"], t["table"].shape[1]
    cached, new, free = t["cached"].long(), t["new"].long(), t["free"].long()
    starts = torch.cat((torch.zeros_like(new[:1]), new.cumsum(0))).clamp(max=T)
    kv = cached + starts[1:] - starts[:-1]
    held, need = ((n + bs - 1).div(bs, rounding_mode="floor").clamp(max=W) for n in (cached, kv))
    first = t["head"].long() + (need - held).cumsum(0) - (need - held)
    page = torch.arange(W, device=table.device)
    take = first[:, None] + page - held[:, None]
    fresh = torch.where(take < free.numel(), free[take.clamp(0, free.numel() - 1)], -1)
    grown = torch.where((page >= held[:, None]) & (page < need[:, None]), fresh, table.long())
    tok = torch.arange(T, device=table.device)
    req = torch.searchsorted(starts[1:], tok, right=True)
    live, req = req < R, req.clamp(max=R - 1)
    pos = cached[req] + tok - starts[req]
    block = grown[req, pos.div(bs, rounding_mode="floor").clamp(max=W - 1)]
    ok = live & (block >= 0) & (pos < W * bs)
    table.copy_(grown)
    return {"head": (t["head"].long() + (need - held).sum()).int(), "starts": starts.int(), "kv": kv.int(),
            "positions": torch.where(live, pos, 0).int(), "slots": torch.where(ok, block * bs + pos % bs, -1).int(),
            "table": table}


def _turn(x, positions, freqs, amp, pairs):
    """The rotation of x [T, H, D] float32; angles in 64 bits (32 leave 0.008 rad at position 2^17)."""
    angle = (positions.double()[:, None] * freqs.double())[:, None, :]
    c, sn = angle.cos().float() * amp, angle.sin().float() * amp
    n = freqs.numel()
    if pairs:
        a, b = x[..., 0:2 * n:2], x[..., 1:2 * n:2]
        return torch.cat((torch.stack((a * c - b * sn, a * sn + b * c), -1).flatten(-2), x[..., 2 * n:]), -1)
    a, b = x[..., :n], x[..., n:2 * n]
    return torch.cat((a * c - b * sn, a * sn + b * c, x[..., 2 * n:]), -1)


def _rope(s):
    t, c = s.t, s.case
    return _turn(t["x"].float(), t["positions"], t["freqs"], c["amp"], c["pairs"]).to(t["x"].dtype)


def _normed(x, w):
    return x if w is None else x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.float()


def _write(s):
    t, c = s.t, s.case
    q = _normed(t["q"][..., :c["D"]].float(), t.get("q_norm"))
    k = _normed(t["k"].float(), t.get("k_norm"))
    q, k = (_turn(x, t["positions"], t["freqs"], 1.0, c["pairs"]).to(torch.bfloat16) for x in (q, k))
    page, off = t["slots"].long().div(c["block"], rounding_mode="floor"), t["slots"].long() % c["block"]
    t["k_cache"][page, :, off] = k
    t["v_cache"][page, :, off] = t["v"]
    return {"q": q, "k_cache": t["k_cache"], "v_cache": t["v_cache"]}


def _gathered(cache, table):
    """[R, Hkv, pages * block, D] float32 of the requests' pages."""
    x = cache[table.long().clamp(min=0)].transpose(1, 2)
    return x.reshape(x.shape[0], x.shape[1], -1, x.shape[-1]).float()


def _attend(s):
    t, c = s.t, s.case
    R, Hq, Hkv, D = c["R"], c["Hq"], c["Hkv"], c["D"]
    starts, kv = t["starts"].long(), t["kv"].long()
    n, dev = starts[1:] - starts[:-1], starts.device
    k, v = _gathered(t["k_cache"], t["table"]), _gathered(t["v_cache"], t["table"])
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


PLAIN = {"blocks": _blocks, "rope": _rope, "write": _write, "attend": _attend}


def run(s):
    return _call(s) if own else PLAIN[s.case["op"]](s)


# ---------------------------------------------------------------- what a pass cannot do without


def work(case):
    op = case["op"]
    if op == "blocks":
        cached, new = _lens(case)
        bs = case["block"]
        pages = sum(-(-(c + n) // bs) - -(-c // bs) for c, n in zip(cached, new))
        # lengths in and out, the new pages' ids in and out, positions and slots; a page id per token's slot
        return {"bytes": 16 * case["R"] + 8 * pages + 8 * sum(new) + 4 * case["R"], "flops": 2 * sum(new)}
    if op == "rope":
        n = case["T"] * case["H"] * case["D"]
        return {"bytes": 2 * n * (4 if case["dtype"] == "float32" else 2) + 4 * case["T"],
                "flops": 3 * case["T"] * case["H"] * case["rot"]}
    if op == "write":
        T, Hq, Hkv, D = (case[k] for k in ("T", "Hq", "Hkv", "D"))
        return {"bytes": 2 * T * D * (2 * Hq + 4 * Hkv) + 8 * T,
                "flops": T * (Hq + Hkv) * (3 * case["rot"] + (4 * D if case["norm"] else 0))}
    cached, new = _lens(case)
    Hq, Hkv, D, w = case["Hq"], case["Hkv"], case["D"], case["window"]
    keys = pairs = 0
    for c, n in zip(cached, new):
        keys += min(c + n, w + n - 1) if w else c + n
        # query i of the chunk sees min(c + i + 1, w) keys
        full = max(0, min(n, w - c)) if w else n
        pairs += full * c + full * (full + 1) // 2 + (n - full) * w
    bytes_ = 2 * (2 * keys * Hkv * D + sum(new) * Hq * D * (3 if case["gate"] else 2)) + 4 * keys // case["block"]
    return {"bytes": bytes_, "flops": 4 * pairs * Hq * D}


# ---------------------------------------------------------------- in 64 bits


def _turn64(x, positions, freqs, amp, pairs):
    """x [T, H, D] as complex numbers times amp * e^(i angle)."""
    n = freqs.numel()
    angle = positions.double()[:, None] * freqs.double()
    z = torch.polar(torch.full_like(angle, amp), angle)[:, None, :]
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
            k, v = (t[name][pages, h].reshape(-1, D)[:L].double() for name in ("k_cache", "v_cache"))
            for g in range(h * Hq // Hkv, (h + 1) * Hq // Hkv):
                score = t["q"][at:at + n, g].double() @ k.t() / math.sqrt(D)
                out[at:at + n, g] = torch.softmax(score.masked_fill(hidden, -math.inf), -1) @ v
        at += n
    if "gate" in t:
        out = out / (1 + torch.exp(-t["gate"][..., D:].double()))
    return out


def exact(case, seed):
    s = prepare(case, seed)
    t, op = s.t, case["op"]
    if op == "blocks":
        return None
    if op == "rope":
        return _turn64(t["x"], t["positions"], t["freqs"], case["amp"], case["pairs"])
    if op == "attend":
        return _attend64(s)
    out, D, bs = {}, case["D"], case["block"]
    for name in ("q", "k"):
        x = t[name][..., :D].double()
        if case["norm"]:
            x = x / (x.pow(2).sum(-1, keepdim=True) / D + 1e-6).sqrt() * t[name + "_norm"].double()
        out[name] = _turn64(x, t["positions"], t["freqs"], 1.0, case["pairs"])
    caches = {"k_cache": out.pop("k"), "v_cache": t["v"].double()}
    for name, rows in caches.items():
        cache = t[name].double().transpose(1, 2).reshape(-1, case["Hkv"], D)
        cache[t["slots"].long()] = rows
        out[name] = cache.view(-1, bs, case["Hkv"], D).transpose(1, 2)
    return out
