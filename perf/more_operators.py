"""Selective state space scans with their short causal convolution, beam search with the states that follow the beams, and dropout
from a counter-based generator: their passes as cases that can be timed, and their plain forms.

  conv     causal_conv: whole sequences (y and the inputs that the next call needs) and, where `train`, all gradients
  scan     selective_scan: whole sequences (y and the state behind the last token) and, where `train`, all gradients
  token    causal_conv_step and selective_scan_step of one token: both states updated where they lie (the scan has an x of its own, so that how
           the convolution's output was rounded stays out of its state)
  beam     beam_select over beams and vocabulary and, where there are layers, reorder_states of their scan and convolution states
  dropout  dropout, added to a residual or alone, and, where `train`, its gradients

With `own` false, run() computes them with elementary torch operations in 32 bits (scores of beams in 64); with `own` true it calls
m2_b200.  d_model and vocabulary are those of perf/cases.py (768 and 1536, 30528 tokens).
"""
import math

import numpy as np
import torch

own = False
DEVICE = "cuda"
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
END = 2                                                                       # the id that ends a text


def listed():
    return [
        # a prompt of any length in front of the scan: the layer's smallest launch
        dict(name="conv-prompt-1x1999", what="conv", train=False, dtype="bf16", batch=1, length=1999, dim=1536, width=4, ragged=False),
        # one training step: forward and all gradients, bound by memory
        dict(name="conv-train-16x2048", what="conv", train=True, dtype="bf16", batch=16, length=2048, dim=1536, width=4, ragged=False),
        # a prompt enters the cache of one conversation: y for the next layer, the state for the tokens to come
        dict(name="scan-prompt-1x1999", what="scan", train=False, dtype="bf16", batch=1, length=1999, dim=1536, state=16, groups=1, gate=True, ragged=False),
        # the longest documents that the encoder takes, one at a time: a long axis and few channels
        dict(name="scan-long-1x32768", what="scan", train=False, dtype="bf16", batch=1, length=32768, dim=768, state=16, groups=1, gate=True, ragged=False),
        # one training step's mixer at d_model 1536: forward and all gradients
        dict(name="scan-train-16x2048", what="scan", train=True, dtype="bf16", batch=16, length=2048, dim=1536, state=16, groups=1, gate=True, ragged=False),
        # float32 mode, padded texts of any length, initial states, b and c of groups of channels: fine-tuning on few texts
        dict(name="scan-train-f32-4x509", what="scan", train=True, dtype="f32", batch=4, length=509, dim=768, state=16, groups=4, gate=False, ragged=True),
        # the next token of one conversation, and of a full server
        dict(name="token-1", what="token", dtype="bf16", batch=1, dim=1536, width=4, state=16, groups=1, gate=True),
        dict(name="token-256", what="token", dtype="bf16", batch=256, dim=1536, width=4, state=16, groups=1, gate=True),
        # one step of one text's search over four beams, with the states of 12 layers
        dict(name="beam-1x4", what="beam", dtype="bf16", batch=1, beams=4, keep=4, vocab=30528, ended=False, layers=12, dim=768, state=16, width=4),
        # the same for a batch of texts, eight beams each, some of them ended
        dict(name="beam-32x8", what="beam", dtype="f32", batch=32, beams=8, keep=8, vocab=30528, ended=True, layers=12, dim=768, state=16, width=4),
        # a block's output on its way to the residual stream, fine-tuning on few short texts
        dict(name="dropout-8x128", what="dropout", train=False, dtype="f32", batch=8, length=128, dim=768, p=0.1, residual=True),
        # the same in a training step: forward and gradients
        dict(name="dropout-train-16x2048", what="dropout", train=True, dtype="bf16", batch=16, length=2048, dim=1536, p=0.1, residual=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    what = rng.choice(["conv", "conv", "scan", "scan", "scan", "token", "beam", "beam", "dropout", "dropout"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    dim = rng.choice([768, 768, 1536, 1536, _log_int(rng, 16, 2048)])
    if what == "conv":
        length = _log_int(rng, 1, 8192)
        return dict(what=what, train=rng.random() < 0.5, dtype=dtype, batch=_log_int(rng, 1, max(1, min(256, (1 << 25) // (length * dim)))), length=length,
                    dim=dim, width=rng.choice([2, 3, 4, 4, 5, 8]), ragged=rng.random() < 0.4)
    if what == "scan":
        train, state = rng.random() < 0.5, rng.choice([16, 16, 16, 8, 11, 32, 64])
        most = (1 << 29 if train and dtype == "bf16" else 1 << 28) // (dim * state)
        length = _log_int(rng, 1, min(most, 8192 if train else 32768))
        groups = rng.choice([1, 1, 2, 4]) if dim % 4 == 0 else 1
        return dict(what=what, train=train, dtype=dtype, batch=_log_int(rng, 1, min(128, most // length)), length=length, dim=dim, state=state, groups=groups,
                    gate=rng.random() < 0.7, ragged=rng.random() < 0.4)
    if what == "token":
        return dict(what=what, dtype=dtype, batch=_log_int(rng, 1, 256), dim=dim, width=rng.choice([2, 3, 4, 4, 8]), state=rng.choice([16, 16, 8, 11, 32, 64]),
                    groups=rng.choice([1, 1, 2, 4]) if dim % 4 == 0 else 1, gate=rng.random() < 0.7)
    if what == "beam":
        beams, layers = rng.choice([1, 2, 4, 4, 5, 8, 16, 32]), rng.choice([0, 1, 12])
        vocab = rng.choice([30528, 30528, _log_int(rng, 300, 131072)])
        batch = _log_int(rng, 1, max(1, min(64, 256 // beams, (1 << 24) // (beams * vocab))))
        return dict(what=what, dtype=dtype, batch=batch, beams=beams, keep=beams if layers else min(32, beams * rng.choice([1, 2])), vocab=vocab,
                    ended=rng.random() < 0.5, layers=layers, dim=768, state=16, width=4)
    tokens = _log_int(rng, 1, min(1 << 17, (1 << 25) // dim))
    length = _log_int(rng, 1, tokens)
    return dict(what=what, train=rng.random() < 0.5, dtype=dtype, batch=max(1, tokens // length), length=length, dim=dim, p=rng.choice([0.0, 0.1, 0.1, 0.25, 0.5]),
                residual=rng.random() < 0.6)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)

    def randn(*shape, dtype=torch.float32, mean=0.0, std=1.0, grad=False):
        return (torch.randn(shape, device=DEVICE, generator=g) * std + mean).to(dtype).requires_grad_(grad)

    def rand(*shape):
        return torch.rand(shape, device=DEVICE, generator=g)

    s, dtype = dict(case), TYPES[case["dtype"]]
    train = case.get("train", False)
    B, L, D = case["batch"], case.get("length", 1), case["dim"]
    s["lengths"] = torch.randint(0, L + 1, (B,), device=DEVICE, generator=g) if case.get("ragged") else None
    if case["what"] in ("conv", "token"):
        W = case["width"]
        s["w"], s["bias"] = randn(D, W, std=W ** -0.5, grad=train), randn(D, std=0.1, grad=train)
        s["u"] = randn(B, L, D + D // 4, dtype=dtype)[..., :D].requires_grad_(train)    # a part of one projection's output
        s["carried"] = randn(B, W - 1, D, dtype=dtype, grad=train) if case.get("ragged") or case["what"] == "token" else None
        if train:
            s["d_y"], s["d_carried"] = randn(B, L, D, dtype=dtype), randn(B, W - 1, D, dtype=dtype) if case["ragged"] else None
        if case["what"] == "token":
            s["u"] = s["u"][:, 0]
    if case["what"] in ("scan", "token"):
        N, G, R = case["state"], case["groups"], max(1, D // 16)
        s["delta"] = randn(B, L, D, dtype=dtype, std=0.5).requires_grad_(train)
        steps = torch.exp(rand(D) * math.log(100.0) + math.log(0.001))                  # step sizes of 0.001 to 0.1
        s["delta_bias"] = (steps + torch.log(-torch.expm1(-steps))).requires_grad_(train)
        s["a"] = (-torch.arange(1, N + 1, device=DEVICE) * torch.exp(randn(D, N, std=0.05))).requires_grad_(train)
        wide = randn(B, L, R + 2 * G * N, dtype=dtype)                                  # one projection's output: what delta is made of, b, c
        s["b"], s["c"] = (t.unflatten(-1, (G, N)).requires_grad_(train) for t in (wide[..., R:R + G * N], wide[..., R + G * N:]))
        s["skip"] = randn(D, mean=1.0, std=0.1, grad=train)
        s["z"] = randn(B, L, D + D // 4, dtype=dtype)[..., D // 4:].requires_grad_(train) if case["gate"] else None
        s["h"] = randn(B, D, N, std=0.5, grad=train) if case.get("ragged") or case["what"] == "token" else None
        s["x"] = randn(B, L, D, dtype=dtype).requires_grad_(train)
        if train:
            s["d_y"], s["d_h"] = randn(B, L, D, dtype=dtype), randn(B, D, N) if case["ragged"] else None
        if case["what"] == "token":
            for name in ("x", "delta", "b", "c") + (("z",) if case["gate"] else ()):
                s[name] = s[name][:, 0]
    if case["what"] == "beam":
        K, V = case["beams"], case["vocab"]
        x = randn(B, K, V) * (rand(B, K, 1) * 2 + 1)
        x[..., V - V // 100:] = -math.inf                                               # ids behind the vocabulary's last token
        s["logits"] = x.to(dtype)
        s["scores"] = -torch.cumsum(rand(B, K) * 2, 1) - 20
        s["finished"] = rand(B, K) < 0.2 if case["ended"] else None
        s["states"] = [t for _ in range(case["layers"]) for t in (randn(B * K, D, case["state"]), randn(B * K, case["width"] - 1, D, dtype=dtype))]
    if case["what"] == "dropout":
        s["x"] = randn(B, L, D, dtype=dtype, grad=train)
        s["r"] = randn(B, L, D, dtype=dtype, grad=train) if case["residual"] else None
        s["seed"] = torch.randint(0, 1 << 62, (2,), device=DEVICE, generator=g)
        if train:
            s["d_y"] = randn(B, L, D, dtype=dtype)
    return s


def run(s):
    return globals()[f"_{s['what']}_{'own' if own else 'plain'}"](s)


def _given(s, *names):
    return [s[n] for n in names if s[n] is not None]


# ---- what a user calls ---------------------------------------------------------------------------------------------------------------
def _conv_own(s):
    import m2_b200
    y, carried = m2_b200.causal_conv(s["u"], s["w"], s["bias"], activation="silu", initial_state=s["carried"], lengths=s["lengths"], return_state=True)
    if not s["train"]:
        return [y, carried]
    outs, ups = ([y, carried], [s["d_y"], s["d_carried"]]) if s["ragged"] else ([y], [s["d_y"]])
    return [y.detach(), carried.detach(), *torch.autograd.grad(outs, _given(s, "u", "w", "bias", "carried"), ups)]


def _scan_own(s):
    import m2_b200
    y, h = m2_b200.selective_scan(s["x"], s["delta"], s["a"], s["b"], s["c"], skip=s["skip"], gate=s["z"], delta_bias=s["delta_bias"], softplus=True,
                                  initial_state=s["h"], lengths=s["lengths"], return_state=True)
    if not s["train"]:
        return [y, h]
    outs, ups = ([y, h], [s["d_y"], s["d_h"]]) if s["ragged"] else ([y], [s["d_y"]])
    return [y.detach(), h.detach(), *torch.autograd.grad(outs, _given(s, "x", "delta", "a", "b", "c", "skip", "delta_bias", "z", "h"), ups)]


def _token_own(s):
    import m2_b200
    v = m2_b200.causal_conv_step(s["u"], s["carried"], s["w"], s["bias"], activation="silu")
    y = m2_b200.selective_scan_step(s["x"], s["delta"], s["a"], s["b"], s["c"], s["h"], skip=s["skip"], gate=s["z"], delta_bias=s["delta_bias"],
                                    softplus=True)
    return [v, y, s["carried"], s["h"]]


def _beam_own(s):
    import m2_b200
    best = m2_b200.beam_select(s["logits"], s["scores"], keep=s["keep"], finished=s["finished"], end_id=END)
    if s["layers"]:
        m2_b200.reorder_states(s["states"], best.beam)
    return [*best, *s["states"]]


def _dropout_own(s):
    import m2_b200
    y = m2_b200.dropout(s["x"], s["p"], s["seed"], residual=s["r"])
    if not s["train"]:
        return [y]
    return [y.detach(), *torch.autograd.grad([y], _given(s, "x", "r"), [s["d_y"]])]


# ---- plain forms ---------------------------------------------------------------------------------------------------------------------
def _wide(t):
    return t.detach().float() if t is not None else None


def _live(s, L):
    """(B, L, 1): whether a token lies in its text."""
    return torch.arange(L, device=DEVICE)[:, None] < s["lengths"][:, None, None] if s["lengths"] is not None else torch.ones((1, L, 1), dtype=torch.bool, device=DEVICE)


def _conv_plain(s):
    u, w, bias = _wide(s["u"]), _wide(s["w"]), _wide(s["bias"])
    (B, L, D), W, dtype = u.shape, s["width"], s["u"].dtype
    before = _wide(s["carried"]) if s["carried"] is not None else u.new_zeros((B, W - 1, D))
    live = _live(s, L)
    x = torch.cat([before, torch.where(live, u, 0.0)], 1)
    v = bias + sum(x[:, i:i + L] * w[:, i] for i in range(W))
    sig = 1 / (1 + torch.exp(-v))
    n = s["lengths"] if s["lengths"] is not None else torch.full((B,), L, device=DEVICE)
    last = n[:, None] + torch.arange(W - 1, device=DEVICE)                               # of x: the last W - 1 inputs of each text
    rows = torch.arange(B, device=DEVICE)[:, None]
    outs = [torch.where(live, v * sig, 0.0).to(dtype), x[rows, last].to(dtype)]
    if not s["train"]:
        return outs
    dv = torch.where(live, s["d_y"].float() * sig * (1 + v * (1 - sig)), 0.0)
    dx = torch.zeros_like(x)
    for i in range(W):
        dx[:, i:i + L] += dv * w[:, i]
    if s["d_carried"] is not None:
        dx[rows, last] += s["d_carried"].float()
    outs += [torch.where(live, dx[:, W - 1:], 0.0).to(dtype), torch.stack([(dv * x[:, i:i + L]).sum((0, 1)) for i in range(W)], 1), dv.sum((0, 1))]
    return outs + ([dx[:, :W - 1].to(dtype)] if s["carried"] is not None else [])


def _recurrence(a, b):
    """h_t = a_t h_{t-1} + b_t along dimension 1, in place of b: steps of one, two, four tokens and so on."""
    a, n = a.clone(), 1
    while n < b.shape[1]:
        b[:, n:] += a[:, n:] * b[:, :-n]
        if 2 * n < b.shape[1]:
            a[:, n:] = a[:, n:] * a[:, :-n]
        n *= 2
    return b


def _scan_plain(s):
    x, a, b, c, z = (_wide(s[n]) for n in ("x", "a", "b", "c", "z"))
    (B, L, D), (G, N), dtype = x.shape, b.shape[2:], s["x"].dtype
    live = _live(s, L)
    pre = _wide(s["delta"]) + _wide(s["delta_bias"])
    dt = torch.where(live, pre.clamp(min=0) + torch.log1p(torch.exp(-pre.abs())), 0.0)
    x = torch.where(live, x, 0.0)
    b, c = (torch.where(live[..., None], t, 0.0)[:, :, :, None] for t in (b, c))           # (B, L, G, 1, N)

    def per_group(t):                                                                    # (B, L, D, ...) as (B, L, G, D / G, ...)
        return t.unflatten(2, (G, D // G))

    decay = torch.exp(dt[..., None] * a)
    h = ((per_group(dt * x)[..., None] * b).flatten(2, 3))
    if s["h"] is not None:
        h[:, 0] += decay[:, 0] * s["h"].detach()
    h = _recurrence(decay, h)
    y = (per_group(h) * c).sum(-1).flatten(2) + _wide(s["skip"]) * x
    sig = 1 / (1 + torch.exp(-z)) if z is not None else None
    gated = y * z * sig if z is not None else y
    outs = [torch.where(live, gated, 0.0).to(dtype), h[:, -1].clone()]
    if not s["train"]:
        return outs
    dout = torch.where(live, s["d_y"].float(), 0.0)
    dy = dout * z * sig if z is not None else dout
    g = (per_group(dy)[..., None] * c).flatten(2, 3)
    if s["d_h"] is not None:
        g[:, -1] += s["d_h"]
    after = torch.cat([decay[:, 1:], torch.ones_like(decay[:, :1])], 1)
    g = _recurrence(after.flip(1), g.flip(1)).flip(1)
    del after
    d_b = (per_group(g) * per_group(dt * x)[..., None]).sum(3)
    d_c = (per_group(h) * per_group(dy)[..., None]).sum(3)
    gb = (per_group(g) * b).sum(-1).flatten(2)
    g *= decay                                                                           # now the gradient of the state in front of a token
    d_h0 = g[:, 0].clone()
    g[:, 1:] *= h[:, :-1]
    g[:, 0] *= s["h"].detach() if s["h"] is not None else 0.0
    d_dt = (g * a).sum(-1) + gb * x
    d_pre = torch.where(live, d_dt / (1 + torch.exp(-pre)), 0.0)
    d_x = torch.where(live, gb * dt + _wide(s["skip"]) * dy, 0.0)
    outs += [d_x.to(dtype), d_pre.to(dtype), (g * dt[..., None]).sum((0, 1)), d_b.to(dtype), d_c.to(dtype), (dy * x).sum((0, 1)), d_pre.sum((0, 1))]
    if z is not None:
        outs.append(torch.where(live, dout * y * sig * (1 + z * (1 - sig)), 0.0).to(dtype))
    return outs + ([d_h0] if s["h"] is not None else [])


def _token_plain(s):
    dtype = s["u"].dtype
    line = torch.cat([s["carried"], s["u"][:, None]], 1)
    v = (line.float() * _wide(s["w"]).t()).sum(1) + _wide(s["bias"])
    v = v / (1 + torch.exp(-v))
    s["carried"].copy_(line[:, 1:])
    x, b, c, z = (_wide(s[n]) for n in ("x", "b", "c", "z"))
    pre = s["delta"].float() + s["delta_bias"]
    dt = pre.clamp(min=0) + torch.log1p(torch.exp(-pre.abs()))
    G = b.shape[1]
    h = s["h"].mul_(torch.exp(dt[..., None] * s["a"]))
    h += ((dt * x).unflatten(1, (G, -1))[..., None] * b[:, :, None]).flatten(1, 2)
    y = (h.unflatten(1, (G, -1)) * c[:, :, None]).sum(-1).flatten(1) + s["skip"] * x
    y = y * z / (1 + torch.exp(-z)) if z is not None else y
    return [v.to(dtype), y.to(dtype), s["carried"], h]


def _beam_plain(s):
    """A beam's tokens go by their logits, equal ones by ascending id; the beams' lists by the scores, equal ones by ascending beam."""
    x, M = s["logits"], s["keep"]
    B, K, V = x.shape
    some = min(M, V)
    ids = x.sort(dim=-1, descending=True, stable=True).indices[..., :some]
    top = x.gather(-1, ids).double()
    m = x.max(-1, keepdim=True).values.double()
    score = s["scores"].double()[..., None] + (top - m - torch.log(torch.exp(x.double() - m).sum(-1, keepdim=True)))
    if s["finished"] is not None:
        ended = s["finished"][..., None]
        only = torch.arange(some, device=DEVICE) == 0
        score = torch.where(ended, torch.where(only, s["scores"].double()[..., None], -math.inf), score)
        ids = torch.where(ended, END, ids)
    best, at = score.flatten(1).sort(dim=-1, descending=True, stable=True)
    best, at = best[:, :M], at[:, :M]
    beam, token = at // some, ids.flatten(1).gather(1, at)
    none = best == -math.inf                                                             # fewer candidates than wanted
    beam, token = torch.where(none, 0, beam), torch.where(none, END, token)
    done = token == END
    if s["finished"] is not None:
        done |= s["finished"].gather(1, beam)
    if s["layers"]:
        rows = (torch.arange(B, device=DEVICE)[:, None] * K + beam).flatten()
        for t in s["states"]:
            t.copy_(t[rows])
    return [best.float(), beam, token, done, *s["states"]]


def _kept(seed, n, p):
    """Philox 4x32-10 (Salmon, Moraes, Dror, Shaw 2011): a key of 64 bits from seed[0], counters of 128 bits from (number of the group of eight
    elements, seed[1]); every word gives 16 bits to two elements, the low ones first.  An element is kept if they are not below p 2^16."""
    low = (1 << 32) - 1
    j = torch.arange(-(-n // 8), device=DEVICE)
    x0, x1, x2, x3 = j & low, j >> 32, seed[1] & low, (seed[1] >> 32) & low
    k0, k1 = seed[0] & low, (seed[0] >> 32) & low
    for _ in range(10):
        a, b = x0 * 0xD2511F53, x2 * 0xCD9E8D57
        x0, x1, x2, x3 = ((b >> 32) & low) ^ x1 ^ k0, b & low, ((a >> 32) & low) ^ x3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    words = torch.stack([w.expand(j.shape) for w in (x0, x1, x2, x3)], 1)
    return torch.stack([words & 0xffff, words >> 16], -1).flatten()[:n] >= round(p * 65536)


def _dropout_plain(s):
    x, dtype = _wide(s["x"]), s["x"].dtype
    kept = _kept(s["seed"], x.numel(), s["p"]).view(x.shape)
    scale = 65536 / (65536 - round(s["p"] * 65536))
    y = torch.where(kept, x * scale, 0.0)
    outs = [(y + _wide(s["r"]) if s["r"] is not None else y).to(dtype)]
    if not s["train"]:
        return outs
    outs.append(torch.where(kept, s["d_y"].float() * scale, 0.0).to(dtype))
    return outs + ([s["d_y"].clone()] if s["r"] is not None else [])


# ---- definitions in 64 bits ----------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return globals()[f"_{case['what']}_exact"](s)


def _conv_exact(s):
    """Text by text; gradients by differentiating the definition."""
    W, train = s["width"], s["train"]
    B, L, D = s["u"].shape
    w, bias = (s[n].detach().double().requires_grad_(train) for n in ("w", "bias"))
    parts = []
    for i in range(B):
        n = int(s["lengths"][i]) if s["lengths"] is not None else L
        u = s["u"][i].detach().double().requires_grad_(train)
        before = (s["carried"][i].detach().double() if s["carried"] is not None else torch.zeros((W - 1, D), dtype=torch.float64, device=DEVICE)).requires_grad_(train)
        with torch.enable_grad():
            x = torch.cat([before, u[:n]])
            v = torch.nn.functional.silu((x.unfold(0, W, 1) * w).sum(-1) + bias) if n else u[:0]
            y = torch.cat([v, torch.zeros((L - n, D), dtype=torch.float64, device=DEVICE)])
            carried = x[n:]
            part = [y, carried]
            if train:
                total = (y * s["d_y"][i].double()).sum() + ((carried * s["d_carried"][i].double()).sum() if s["d_carried"] is not None else 0.0)
                part += torch.autograd.grad(total, [u, w, bias, before], allow_unused=True, materialize_grads=True)
        parts.append([t.detach() for t in part])
    cols = [torch.stack(t) for t in zip(*parts)]
    if not train:
        return cols
    return cols[:3] + [cols[3].sum(0), cols[4].sum(0)] + ([cols[5]] if s["carried"] is not None else [])


def _scan_exact(s):
    """Token by token, forwards and back."""
    x, a, skip = s["x"].double(), s["a"].double(), s["skip"].double()
    (B, L, D), (G, N) = x.shape, s["b"].shape[2:]
    group = torch.arange(D, device=DEVICE) // (D // G)
    n = s["lengths"] if s["lengths"] is not None else torch.full((B,), L, device=DEVICE)
    h = s["h"].double() if s["h"] is not None else torch.zeros((B, D, N), dtype=torch.float64, device=DEVICE)
    y, states = torch.zeros_like(x), [h] if s["train"] else None

    def at(t):
        inside = (t < n)[:, None]
        pre = s["delta"][:, t].double() + s["delta_bias"].double()
        step = torch.where(inside, torch.nn.functional.softplus(pre), 0.0)
        b, c = (torch.where(inside[..., None], s[k][:, t].double(), 0.0)[:, group] for k in "bc")
        return inside, pre, step, torch.exp(step[..., None] * a), torch.where(inside, x[:, t], 0.0), b, c

    for t in range(L):
        inside, _, step, decay, u, b, c = at(t)
        h = torch.addcmul(decay * h, (step * u)[..., None], b)
        y[:, t] = torch.einsum("bdn,bdn->bd", h, c) + skip * u
        if s["train"]:
            states.append(h)
    z = s["z"].double() if s["z"] is not None else None
    live = torch.arange(L, device=DEVICE)[None, :, None] < n[:, None, None]
    outs = [torch.where(live, y * torch.nn.functional.silu(z) if z is not None else y, 0.0), h]
    if not s["train"]:
        return outs
    d_y = torch.where(live, s["d_y"].double(), 0.0)
    up = d_y * torch.nn.functional.silu(z) if z is not None else d_y
    g = s["d_h"].double() if s["d_h"] is not None else torch.zeros_like(h)
    d_x, d_delta, d_a, d_skip = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(a), torch.zeros_like(skip)
    d_b, d_c = (torch.zeros(s["b"].shape, dtype=torch.float64, device=DEVICE) for _ in "bc")
    for t in reversed(range(L)):
        inside, pre, step, decay, u, b, c = at(t)
        h = states.pop()
        e = up[:, t]
        g = torch.addcmul(g, e[..., None], c)
        d_c[:, t] = (h * e[..., None]).view(B, G, -1, N).sum(2)
        d_b[:, t] = (g * (step * u)[..., None]).view(B, G, -1, N).sum(2)
        gb = torch.einsum("bdn,bdn->bd", g, b)
        g = g * decay
        w = g * states[-1]
        d_a += (w * step[..., None]).sum(0)
        d_x[:, t] = torch.where(inside, gb * step + skip * e, 0.0)
        d_skip += (e * u).sum(0)
        d_delta[:, t] = torch.where(inside, ((w * a).sum(-1) + gb * u) * torch.sigmoid(pre), 0.0)
    outs += [d_x, d_delta, d_a, d_b, d_c, d_skip, d_delta.sum((0, 1))]
    if z is not None:
        sig = torch.sigmoid(z)
        outs.append(d_y * y * (sig + z * sig * (1 - sig)))
    return outs + ([g] if s["h"] is not None else [])


def _token_exact(s):
    line = torch.cat([s["carried"].double(), s["u"].double()[:, None]], 1)
    v = torch.nn.functional.silu(torch.einsum("bwd,dw->bd", line, s["w"].double()) + s["bias"].double())
    x = s["x"].double()
    group = torch.arange(s["dim"], device=DEVICE) // (s["dim"] // s["groups"])
    step = torch.nn.functional.softplus(s["delta"].double() + s["delta_bias"].double())
    h = torch.exp(step[..., None] * s["a"].double()) * s["h"].double() + (step * x)[..., None] * s["b"].double()[:, group]
    y = torch.einsum("bdn,bdn->bd", h, s["c"].double()[:, group]) + s["skip"].double() * x
    return [v, y * torch.nn.functional.silu(s["z"].double()) if s["z"] is not None else y, line[:, 1:], h]


def _beam_exact(s):
    lp = torch.log_softmax(s["logits"].double(), -1) + s["scores"].double()[..., None]
    B, K, V = lp.shape
    if s["finished"] is not None:
        lp[s["finished"]] = -math.inf
        at = s["finished"].nonzero()
        lp[at[:, 0], at[:, 1], END] = s["scores"].double()[at[:, 0], at[:, 1]]
    best = torch.topk(lp.flatten(1), s["keep"]).values
    return [best] + [None] * (3 + len(s["states"]))


def _dropout_exact(s):
    """The generator on the host, with numbers of 64 bits."""
    seed, call = (np.uint64(int(v)) for v in s["seed"].cpu())
    n, low, half = s["x"].numel(), np.uint64((1 << 32) - 1), np.uint64(32)
    c = [np.arange((n + 7) // 8, dtype=np.uint64) & low, np.arange((n + 7) // 8, dtype=np.uint64) >> half, call & low, call >> half]
    key = [int(seed & low), int(seed >> half)]
    for _ in range(10):
        p, q = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(q >> half) ^ c[1] ^ np.uint64(key[0]), q & low, (p >> half) ^ c[3] ^ np.uint64(key[1]), p & low]
        key = [(key[0] + 0x9E3779B9) % (1 << 32), (key[1] + 0xBB67AE85) % (1 << 32)]
    words = np.stack(np.broadcast_arrays(*c), 1).astype("<u4")
    border = round(s["p"] * 65536)
    factor = torch.from_numpy((words.view("<u2").reshape(-1)[:n] >= border) * (65536 / (65536 - border))).to(DEVICE).view(s["x"].shape)
    outs = [s["x"].double() * factor + (s["r"].double() if s["r"] is not None else 0.0)]
    if not s["train"]:
        return outs
    return outs + [s["d_y"].double() * factor] + ([s["d_y"].double()] if s["r"] is not None else [])


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------------------
def work(case):
    size, train = TYPES[case["dtype"]].itemsize, case.get("train", False)
    B, D = case["batch"], case["dim"]
    n = B * case.get("length", 1) * D
    if case["what"] == "conv":                                    # gradients: x and dy in, dx out
        small = 4 * D * (case["width"] + 1) + B * (case["width"] - 1) * D * size * (2 if case["ragged"] else 1)
        return {"bytes": n * size * (4 if train else 2) + small * (2 if train else 1), "flops": n * (2 * case["width"] + 4) * (4 if train else 1)}
    if case["what"] in ("scan", "token"):
        N, G, wide = case["state"], case["groups"], 4 if case["gate"] else 3
        rows, tables, state = n * wide * size + 2 * n // D * G * N * size, 4 * D * (N + 2), 4 * B * D * N
        if case["what"] == "token":
            carried = 2 * B * (case["width"] - 1) * D * size
            return {"bytes": rows + tables + 2 * state + carried + 2 * n * size + 4 * D * (case["width"] + 1), "flops": n * (8 * N + 2 * case["width"] + 20)}
        byte, flops = rows + tables + state * (2 if case["ragged"] else 1), n * (8 * N + 12)
        if train:                                                # what went in and the gradient of y in, all the gradients out
            byte += n * (wide - 1) * size + 2 * n // D * G * N * size + n * size + tables + (2 * state if case["ragged"] else 0)
            flops += n * (22 * N + 40)
        return {"bytes": byte, "flops": flops}
    if case["what"] == "beam":
        rows = B * case["beams"]
        byte = rows * (case["vocab"] * size + 5) + B * case["keep"] * 21
        return {"bytes": byte + 2 * case["layers"] * rows * D * (4 * case["state"] + (case["width"] - 1) * size), "flops": 6 * rows * case["vocab"]}
    tensors = 3 if case["residual"] else 2
    return {"bytes": n * size * (tensors + (2 if train else 0)) + 16, "flops": n * (16 if train else 8)}
