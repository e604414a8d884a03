"""Linear attention with a decay for each head, norms around a block with its gate and residual scale, and the log
probabilities of given tokens: their passes as cases that can be timed, and their plain forms.

  scan   linear_attention: prompts (o and the state behind the last token) and, where `train`, all its gradients
  step   linear_attention_step: one token for each sequence, the state updated where it lies
  norm   gated_residual_norm: the new residual stream and the next block's input and, where `train`, all gradients
  score  token_logprobs: log probability of the given token, entropy, best alternatives and, where `train`, the logits' gradient

With `own` false, run() computes them with elementary torch operations in 32 bits; with `own` true it calls m2_b200.
d_model and vocabulary are those of perf/cases.py (768 and 1536 in heads of 64 and 128, 30528 tokens).
"""
import math

import torch

own = False
DEVICE = "cuda"
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-5
IGNORE = -100
CHUNK = 64


def listed():
    return [
        # a prompt of any length enters the cache of one conversation: o for the next layer, the state for the tokens to come
        dict(name="scan-prompt-1x1999", what="scan", train=False, dtype="bf16", batch=1, length=1999, heads=12, kv_heads=12, dk=64, dv=64, ragged=False),
        # the longest documents that the encoder takes, one at a time: few heads, a long axis
        dict(name="scan-long-1x32768", what="scan", train=False, dtype="bf16", batch=1, length=32768, heads=12, kv_heads=12, dk=64, dv=64, ragged=False),
        # one training step's mixer at d_model 1536: forward and all gradients
        dict(name="scan-train-16x2048", what="scan", train=True, dtype="bf16", batch=16, length=2048, heads=12, kv_heads=12, dk=128, dv=128, ragged=False),
        # float32 mode, padded texts of any length, an initial state, shared key heads: fine-tuning on few texts
        dict(name="scan-train-f32-4x509", what="scan", train=True, dtype="f32", batch=4, length=509, heads=12, kv_heads=4, dk=64, dv=64, ragged=True),
        # the next token of one conversation, and of a full server
        dict(name="step-1", what="step", dtype="bf16", batch=1, heads=12, kv_heads=12, dk=64, dv=64),
        dict(name="step-256", what="step", dtype="bf16", batch=256, heads=12, kv_heads=12, dk=128, dv=128),
        # around a block while one token is decoded
        dict(name="norm-1-token", what="norm", train=False, dtype="bf16", stream="bf16", batch=1, length=1, dim=768, gate="channel", scale="number", rms=True),
        # the same for a batch of documents at d_model 1536, float32 stream, gated token by token
        dict(name="norm-64x2048", what="norm", train=False, dtype="bf16", stream="f32", batch=64, length=2048, dim=1536, gate="token", scale="number", rms=False),
        # a training step at the pretraining length: forward and all gradients, gate and scale learned
        dict(name="norm-train-256x128", what="norm", train=True, dtype="bf16", stream="f32", batch=256, length=128, dim=768, gate="sequence", scale="channel", rms=False),
        # the token just sampled, with the alternatives that an interface shows
        dict(name="score-1", what="score", train=False, dtype="bf16", rows=1, vocab=30528, top=20, ignored=False),
        # perplexity of documents, padding among the rows
        dict(name="score-4096", what="score", train=False, dtype="f32", rows=4096, vocab=30528, top=5, ignored=True),
        # the loss of a masked-LM batch with an entropy term, and its gradient
        dict(name="score-train-8192", what="score", train=True, dtype="bf16", rows=8192, vocab=30528, top=0, ignored=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    what = rng.choice(["scan", "scan", "scan", "step", "norm", "norm", "score", "score"])
    if what == "scan":
        train, dtype = rng.random() < 0.5, rng.choice(["bf16", "bf16", "f32"])
        dk, dv = rng.choice([(64, 64), (64, 64), (128, 128), (128, 128), (64, 128), (32, 32), (96, 96), (80, 40)])
        heads = rng.choice([1, 4, 6, 12, 24])
        shared = rng.choice([1, 1, 1, 2, 3]) if heads % 6 == 0 else 1
        length = _log_int(rng, 1, 4096 if train or dtype == "f32" else 32768)
        most = max(1, min(256, (1 << 20 if train or dtype == "f32" else 1 << 22) // (length * heads) * 64 // max(dk, dv)))
        return dict(what=what, train=train, dtype=dtype, batch=_log_int(rng, 1, most), length=length, heads=heads, kv_heads=heads // shared, dk=dk,
                    dv=dv, ragged=rng.random() < 0.4)
    if what == "step":
        dk, dv = rng.choice([(64, 64), (128, 128), (64, 128), (96, 96)])
        heads = rng.choice([4, 12, 24])
        return dict(what=what, dtype=rng.choice(["bf16", "f32"]), batch=_log_int(rng, 1, 256), heads=heads, kv_heads=heads // rng.choice([1, 1, 2, 4]),
                    dk=dk, dv=dv)
    if what == "norm":
        train, dim = rng.random() < 0.5, rng.choice([768, 768, 1536, 1536, _log_int(rng, 16, 4096)])
        tokens = _log_int(rng, 1, min(1 << 17, (1 << 25 if train else 1 << 27) // dim))
        length = _log_int(rng, 1, tokens)
        return dict(what=what, train=train, dtype=rng.choice(["bf16", "bf16", "f32"]), stream=rng.choice(["bf16", "f32"]), batch=max(1, tokens // length),
                    length=length, dim=dim, gate=rng.choice(["none", "channel", "sequence", "token"]), scale=rng.choice(["number", "channel"]),
                    rms=rng.random() < 0.5)
    train, vocab = rng.random() < 0.5, rng.choice([30528, _log_int(rng, 300, 131072)])
    return dict(what=what, train=train, dtype=rng.choice(["bf16", "bf16", "f32"]), rows=_log_int(rng, 1, min(16384, (1 << 27) // vocab)), vocab=vocab,
                top=rng.choice([0, 1, 5, 20]), ignored=rng.random() < 0.4)


def _decays(heads):
    """1 - 2^-5 for the first head to 1 - 2^-12 for the last one: memories of 32 to 4096 tokens."""
    e = torch.linspace(5.0, 12.0, heads, dtype=torch.float64) if heads > 1 else torch.tensor([7.0], dtype=torch.float64)
    return torch.log1p(-torch.exp2(-e)).float().to(DEVICE)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)

    def randn(*shape, dtype=torch.float32, mean=0.0, std=1.0, grad=False):
        return (torch.randn(shape, device=DEVICE, generator=g) * std + mean).to(dtype).requires_grad_(grad)

    s, dtype = dict(case), TYPES[case["dtype"]]
    if case["what"] in ("scan", "step"):
        B, L, H, K, dk, dv = case["batch"], case.get("length", 1), case["heads"], case["kv_heads"], case["dk"], case["dv"]
        wide = randn(B, L, H * dk + K * (dk + dv), dtype=dtype)               # one projection's output, in which q, k and v lie side by side
        cut = (H * dk, (H + K) * dk)
        q, k, v = wide[..., :cut[0]], wide[..., cut[0]:cut[1]], wide[..., cut[1]:]
        q, k, v = q.unflatten(-1, (H, dk)), k.unflatten(-1, (K, dk)), v.unflatten(-1, (K, dv))
        s["log_decay"] = _decays(H)
        s["lengths"] = None
        if case["what"] == "step":
            s["q"], s["k"], s["v"] = q[:, 0], k[:, 0], v[:, 0]
            s["state"] = randn(B, H, dk, dv, std=4.0)
            return s
        train = case["train"]
        s["q"], s["k"], s["v"] = (t.requires_grad_(train) for t in (q, k, v))
        s["initial"] = randn(B, H, dk, dv, grad=train) if case["ragged"] else None
        if case["ragged"]:
            s["lengths"] = torch.randint(0, L + 1, (B,), device=DEVICE, generator=g)
        if train:
            s["d_out"], s["d_state"] = randn(B, L, H, dv, dtype=dtype), randn(B, H, dk, dv) if case["ragged"] else None
    elif case["what"] == "norm":
        B, L, D, stream = case["batch"], case["length"], case["dim"], TYPES[case["stream"]]
        train = case["train"]
        s["x"], s["y"] = randn(B, L, D, dtype=stream, std=2.0, grad=train), randn(B, L, D, dtype=dtype, mean=0.1, grad=train)
        shape = {"none": None, "channel": (D,), "sequence": (B, 1, D), "token": (B, L, D)}[case["gate"]]
        s["g"] = randn(*shape, dtype=torch.float32 if case["gate"] == "channel" else dtype, mean=0.5, std=0.5, grad=train) if shape else None
        s["a"] = 0.9 if case["scale"] == "number" else randn(D, mean=0.9, std=0.1, grad=train)
        s["w1"], s["w2"] = randn(D, mean=1.0, std=0.2, grad=train), randn(D, mean=1.0, std=0.2, grad=train)
        s["b1"], s["b2"] = (None, None) if case["rms"] else (randn(D, std=0.1, grad=train), randn(D, std=0.1, grad=train))
        if train:
            s["d_r"], s["d_h"] = randn(B, L, D, dtype=stream), randn(B, L, D, dtype=dtype)
    else:
        N, V = case["rows"], case["vocab"]
        x = torch.randn((N, V), device=DEVICE, generator=g) * (torch.rand((N, 1), device=DEVICE, generator=g) * 4 + 0.5)
        x[:, V - V // 100:] = -math.inf                                       # ids behind the vocabulary's last token
        s["x"] = x.to(dtype).requires_grad_(case["train"])
        s["t"] = torch.randint(0, V - V // 100, (N,), device=DEVICE, generator=g)
        if case["ignored"]:
            s["t"] = torch.where(torch.rand(N, device=DEVICE, generator=g) < 0.2, IGNORE, s["t"])
        if case["train"]:
            s["d_lp"], s["d_h"] = randn(N, mean=-1.0, std=0.1), randn(N, std=0.1)
            s["d_top"] = randn(N, case["top"], std=0.1) if case["top"] else None
    return s


def _with(*pairs):
    return [t for use, t in pairs if use is not None]


def run(s):
    what = s["what"]
    if what == "scan":
        return _scan_own(s) if own else _scan_plain(s)
    if what == "step":
        return _step_own(s) if own else _step_plain(s)
    if what == "norm":
        return _norm_own(s) if own else _norm_plain(s)
    return _score_own(s) if own else _score_plain(s)


# ---- what a user calls ---------------------------------------------------------------------------------------------------------------
def _scan_own(s):
    import m2_b200
    o, state = m2_b200.linear_attention(s["q"], s["k"], s["v"], s["log_decay"], initial_state=s["initial"], lengths=s["lengths"], return_state=True)
    if not s["train"]:
        return [o, state]
    leaves = [s["q"], s["k"], s["v"]] + _with((s["initial"], s["initial"]))
    outs, ups = [o] + _with((s["d_state"], state)), [s["d_out"]] + _with((s["d_state"], s["d_state"]))
    return [o.detach(), state.detach(), *torch.autograd.grad(outs, leaves, ups)]


def _step_own(s):
    import m2_b200
    return [m2_b200.linear_attention_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"]), s["state"]]


def _norm_own(s):
    import m2_b200
    r, h = m2_b200.gated_residual_norm(s["x"], s["y"], gate=s["g"], residual_scale=s["a"], after_weight=s["w1"], after_bias=s["b1"],
                                       before_weight=s["w2"], before_bias=s["b2"], eps=EPS, rms=s["rms"])
    if not s["train"]:
        return [r, h]
    return [r.detach(), h.detach(), *torch.autograd.grad([r, h], _norm_leaves(s), [s["d_r"], s["d_h"]])]


def _norm_leaves(s):
    learned = s["a"] if isinstance(s["a"], torch.Tensor) else None
    return [s["x"], s["y"], s["w1"], s["w2"]] + _with((s["b1"], s["b1"]), (s["b2"], s["b2"]), (s["g"], s["g"]), (learned, learned))


def _score_own(s):
    import m2_b200
    r = m2_b200.token_logprobs(s["x"], s["t"], top=s["top"], ignore_index=IGNORE)
    outs = [r.logprob, r.entropy] + ([r.top_logprob, r.top_id] if s["top"] else [])
    if not s["train"]:
        return outs
    ups = [s["d_lp"], s["d_h"]] + _with((s["d_top"], s["d_top"]))
    return [t.detach() for t in outs] + list(torch.autograd.grad(outs[:len(ups)], [s["x"]], ups))


# ---- plain forms ---------------------------------------------------------------------------------------------------------------------
def _chunked(q, k, v, ld, s0=None):
    """o_i = sum_{j <= i} exp(ld (i - j)) (q_i . k_j) v_j + exp(ld (i + 1)) q_i s0 for float32 (B, H, L, d): products inside chunks, and with
    the state in front of each chunk, which is a product of a triangle of decays with the chunks' own sums."""
    B, H, L, _ = q.shape
    n = -(-L // CHUNK)
    q, k, v = (torch.nn.functional.pad(t, (0, 0, 0, n * CHUNK - L)).unflatten(2, (n, CHUNK)) for t in (q, k, v))
    ld = ld.double()
    i = torch.arange(CHUNK, device=q.device)
    gap = i[:, None] - i[None]
    inside = torch.where(gap >= 0, torch.exp(ld[:, None, None] * gap.clamp(min=0)), 0.0).float()[:, None]          # (H, 1, C, C)
    to_end = torch.exp(ld[:, None] * (CHUNK - 1 - i)).float()[:, None, :, None]
    from_start = torch.exp(ld[:, None] * (i + 1)).float()[:, None, :, None]
    own_sums = (k * to_end).transpose(-1, -2) @ v                                                                  # (B, H, n, dk, dv)
    m = torch.arange(n, device=q.device)
    ago = m[:, None] - 1 - m[None]
    carry = torch.where(ago >= 0, torch.exp(ld[:, None, None] * CHUNK * ago.clamp(min=0)), 0.0).float()
    front = (carry @ own_sums.flatten(-2)).unflatten(-1, own_sums.shape[-2:])
    if s0 is not None:
        front = front + torch.exp(ld[:, None] * CHUNK * m).float()[:, :, None, None] * s0[:, :, None]
    o = ((q @ k.transpose(-1, -2)) * inside) @ v + (q @ front) * from_start
    return o.flatten(2, 3)[:, :, :L]


def _heads_first(t, like=None):
    """(B, L, h, d) as float32 (B, H, L, d), shared heads repeated."""
    t = t.detach().float().transpose(1, 2)
    return t if like is None else t.repeat_interleave(like // t.shape[1], 1)


def _scan_plain(s):
    B, L, H, dk = s["q"].shape
    K, scale, dtype, ld = s["k"].shape[2], dk ** -0.5, s["q"].dtype, s["log_decay"]
    q, k, v = _heads_first(s["q"]), _heads_first(s["k"], H), _heads_first(s["v"], H)
    s0 = s["initial"].detach() if s["initial"] is not None else None
    i = torch.arange(L, device=q.device)
    n = s["lengths"] if s["lengths"] is not None else torch.full((B,), L, device=q.device)
    live = (i < n[:, None])[:, None, :, None]
    q, k, v = (torch.where(live, t, 0.0) for t in (q, k, v))
    rest = (n[:, None] - 1 - i)[:, None]                                                                           # (B, 1, L): steps to the last one
    to_last = torch.where(rest >= 0, torch.exp(ld.double()[:, None] * rest.clamp(min=0)), 0.0).float()[..., None]
    through = torch.exp(ld.double() * n[:, None]).float()[..., None, None]
    o = torch.where(live, _chunked(q, k, v, ld, s0) * scale, 0.0)
    state = (k * to_last).transpose(-1, -2) @ v
    state = state + through * s0 if s0 is not None else state
    outs = [o.transpose(1, 2).to(dtype), state]
    if not s["train"]:
        return outs
    do = torch.where(live, _heads_first(s["d_out"]), 0.0) * scale
    ds = s["d_state"]
    dq = torch.where(live, _chunked(do, v, k, ld, s0.transpose(-1, -2) if s0 is not None else None), 0.0)
    back_q, back_k, back_v, back_o = (t.flip(2) for t in (q, k, v, do))
    dks, dvs = _chunked(back_v, back_o, back_q, ld).flip(2), _chunked(back_k, back_q, back_o, ld).flip(2)
    if ds is not None:
        dks, dvs = dks + (v * to_last) @ ds.transpose(-1, -2), dvs + (k * to_last) @ ds
    dks, dvs = (torch.where(live, t, 0.0).unflatten(1, (K, H // K)).sum(2) for t in (dks, dvs))
    outs += [t.transpose(1, 2).to(dtype) for t in (dq, dks, dvs)]
    if s0 is not None:
        from_first = torch.exp(ld.double()[:, None] * (i + 1)).float()[..., None]
        outs.append((q * from_first).transpose(-1, -2) @ do + through * ds)
    return outs


def _step_plain(s):
    H = s["q"].shape[1]
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    k, v = (t.repeat_interleave(H // t.shape[1], 1) for t in (k, v))
    s["state"].mul_(torch.exp(s["log_decay"])[:, None, None]).add_(k[..., None] * v[..., None, :])
    o = (q[..., None, :] @ s["state"])[..., 0, :] * q.shape[-1] ** -0.5
    return [o.to(s["q"].dtype), s["state"]]


def _normed(x, rms):
    """x without its mean (LayerNorm) over its deviation, and one over that."""
    if not rms:
        x = x - x.mean(-1, keepdim=True)
    inv = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    return x * inv, inv


def _normed_grad(d, hat, inv, rms):
    d = d - hat * (d * hat).mean(-1, keepdim=True) - (0.0 if rms else d.mean(-1, keepdim=True))
    return d * inv


def _norm_plain(s):
    x, y = s["x"].detach().float(), s["y"].detach().float()
    a = s["a"].detach() if isinstance(s["a"], torch.Tensor) else s["a"]
    g = s["g"].detach().float() if s["g"] is not None else 1.0
    w1, w2 = s["w1"].detach(), s["w2"].detach()
    hat1, inv1 = _normed(y, s["rms"])
    n = hat1 * w1 + (s["b1"].detach() if s["b1"] is not None else 0.0)
    r = a * x + g * n
    hat2, inv2 = _normed(r, s["rms"])
    h = hat2 * w2 + (s["b2"].detach() if s["b2"] is not None else 0.0)
    outs = [r.to(s["x"].dtype), h.to(s["y"].dtype)]
    if not s["train"]:
        return outs
    dh = s["d_h"].float()
    u = s["d_r"].float() + _normed_grad(dh * w2, hat2, inv2, s["rms"])
    dn = u * g
    outs += [(a * u).to(s["x"].dtype), _normed_grad(dn * w1, hat1, inv1, s["rms"]).to(s["y"].dtype), (dn * hat1).sum((0, 1)), (dh * hat2).sum((0, 1))]
    if s["b1"] is not None:
        outs += [dn.sum((0, 1)), dh.sum((0, 1))]
    if s["g"] is not None:
        outs.append((u * n).sum_to_size(s["g"].shape).to(s["g"].dtype))
    if isinstance(s["a"], torch.Tensor):
        outs.append((u * x).sum((0, 1)))
    return outs


def _score_plain(s):
    x, t, k = s["x"].detach().float(), s["t"], s["top"]
    used = t != IGNORE
    m = x.max(-1, keepdim=True).values
    z = torch.exp(x - m).sum(-1, keepdim=True)
    lp = x - m - torch.log(z)
    p = torch.exp(lp)
    entropy = -torch.where(p > 0, p * lp, 0.0).sum(-1)
    at = torch.where(used, t, 0)[:, None]
    outs = [torch.where(used, lp.gather(1, at)[:, 0], 0.0), torch.where(used, entropy, 0.0)]
    if k:
        ids = x.sort(dim=-1, descending=True, stable=True).indices[:, :k]
        outs += [torch.where(used[:, None], lp.gather(1, ids), 0.0), torch.where(used[:, None], ids, -1)]
    if not s["train"]:
        return outs
    d_top = s["d_top"] if k else x.new_zeros((x.shape[0], 0))
    d = -p * (s["d_lp"][:, None] + d_top.sum(-1, keepdim=True)) - torch.where(p > 0, s["d_h"][:, None] * p * (lp + entropy[:, None]), 0.0)
    d.scatter_add_(1, at, s["d_lp"][:, None])
    if k:
        d.scatter_add_(1, ids, d_top)
    return outs + [torch.where(used[:, None], d, 0.0).to(s["x"].dtype)]


# ---- definitions in 64 bits ----------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"scan": _scan_exact, "step": _step_exact, "norm": _norm_exact, "score": _score_exact}[case["what"]](s)


def _scan_exact(s):
    """Row by row of the L x L matrix of weights, for a block of rows of one text at a time."""
    B, L, H, dk = s["q"].shape
    K, dv, ld = s["k"].shape[2], s["v"].shape[3], s["log_decay"].double()[:, None, None]
    o = torch.zeros((B, L, H, dv), dtype=torch.float64, device=DEVICE)
    state = torch.zeros((B, H, dk, dv), dtype=torch.float64, device=DEVICE)
    dq, dk_, dv_, d0 = (torch.zeros(t, dtype=torch.float64, device=DEVICE) for t in ((B, L, H, dk), (B, L, K, dk), (B, L, K, dv), (B, H, dk, dv)))
    rows = max(1, min(512, (1 << 28) // (H * L)))
    for b in range(B):
        n = int(s["lengths"][b]) if s["lengths"] is not None else L
        q = s["q"][b, :n].double().movedim(1, 0) * dk ** -0.5
        k, v = (s[x][b, :n].double().movedim(1, 0).repeat_interleave(H // K, 0) for x in "kv")
        s0 = s["initial"][b].double() if s["initial"] is not None else torch.zeros((H, dk, dv), dtype=torch.float64, device=DEVICE)
        j = torch.arange(n, device=DEVICE, dtype=torch.float64)
        left = torch.exp(ld * (n - 1 - j)[:, None])                                     # (H, n, 1)
        state[b] = (k * left).mT @ v + torch.exp(ld * n) * s0
        gk, gv, g0 = torch.zeros_like(k), torch.zeros_like(v), torch.zeros_like(s0)
        for at in range(0, n, rows):
            here = slice(at, min(n, at + rows))
            seen = slice(0, here.stop)
            gap = j[here, None] - j[None, seen]
            w = torch.exp(ld * gap).masked_fill_(gap < 0, 0.0)
            past = torch.exp(ld * (j[here, None] + 1))
            a = (q[:, here] @ k[:, seen].mT) * w
            o[b, here] = (a @ v[:, seen] + (q[:, here] * past) @ s0).movedim(0, 1)
            if s["train"]:
                u = s["d_out"][b, here].double().movedim(1, 0)
                c = (u @ v[:, seen].mT) * w
                dq[b, here] = (c @ k[:, seen] + (u * past) @ s0.mT).movedim(0, 1) * dk ** -0.5
                gk[:, seen] += c.mT @ q[:, here]
                gv[:, seen] += a.mT @ u
                g0 += (q[:, here] * past).mT @ u
        if s["train"]:
            if s["d_state"] is not None:
                ds = s["d_state"][b].double()
                gk, gv, g0 = gk + (v * left) @ ds.mT, gv + (k * left) @ ds, g0 + torch.exp(ld * n) * ds
            dk_[b, :n], dv_[b, :n] = (t.unflatten(0, (K, H // K)).sum(1).movedim(0, 1) for t in (gk, gv))
            d0[b] = g0
    return [o, state] + ([dq, dk_, dv_] + ([d0] if s["initial"] is not None else []) if s["train"] else [])


def _step_exact(s):
    H, K = s["q"].shape[1], s["k"].shape[1]
    head = torch.arange(H, device=DEVICE) // (H // K)
    k, v = s["k"].double()[:, head], s["v"].double()[:, head]
    new = torch.exp(s["log_decay"].double())[None, :, None, None] * s["state"].double() + torch.einsum("bhi,bhj->bhij", k, v)
    return [torch.einsum("bhi,bhij->bhj", s["q"].double(), new) / math.sqrt(s["q"].shape[-1]), new]


def _norm_exact(s):
    """Gradients by differentiating the definition."""
    leaves = [t.detach().double().requires_grad_(s["train"]) for t in _norm_leaves(s)]
    x, y, w1, w2 = leaves[:4]
    rest = leaves[4:]
    b1, b2 = (rest.pop(0), rest.pop(0)) if s["b1"] is not None else (None, None)
    g = rest.pop(0) if s["g"] is not None else torch.ones((), dtype=torch.float64, device=DEVICE)
    a = rest.pop(0) if rest else s["a"]

    def norm(t, w, b):
        if s["rms"]:
            return t / (t.square().mean(-1, keepdim=True) + EPS).sqrt() * w
        c = t - t.mean(-1, keepdim=True)
        return c / (c.square().mean(-1, keepdim=True) + EPS).sqrt() * w + b

    with torch.set_grad_enabled(s["train"]):
        r = a * x + g * norm(y, w1, b1)
        h = norm(r, w2, b2)
        if not s["train"]:
            return [r, h]
        return [r.detach(), h.detach(), *torch.autograd.grad([r, h], leaves, [s["d_r"].double(), s["d_h"].double()])]


def _score_exact(s):
    """The ids are whole numbers and have no value of their own here."""
    N, V = s["x"].shape
    k, step = s["top"], max(1, (1 << 27) // V)
    found = []
    for at in range(0, N, step):
        here = slice(at, at + step)
        x, t = s["x"][here].detach().double(), s["t"][here]
        used = (t != IGNORE).double()
        z = torch.logsumexp(x, -1)
        lp = x - z[:, None]
        p = lp.exp()
        plp = (p * lp).nan_to_num_(0.0)
        H = -plp.sum(-1)
        t = t.clamp(min=0)
        part = [lp[torch.arange(len(t), device=DEVICE), t] * used, H * used]
        if k:
            best = torch.topk(lp, k, -1).values
            part.append(best * used[:, None])
        if s["train"]:
            lost = s["d_lp"][here].double() + (s["d_top"][here].double().sum(-1) if k else 0.0)
            d = -(p * lost[:, None]) - s["d_h"][here].double()[:, None] * (plp + p * H[:, None])
            hot = torch.zeros_like(d)
            hot[torch.arange(len(t), device=DEVICE), t] = s["d_lp"][here].double()
            if k:
                ids = s["x"][here].detach().float().sort(dim=-1, descending=True, stable=True).indices[:, :k]
                hot.scatter_add_(1, ids, s["d_top"][here].double())
            part.append((d + hot) * used[:, None])
        found.append(part)
    outs = [torch.cat(p) for p in zip(*found)]
    return outs[:2] + ([outs[2], None] if k else []) + outs[2 + bool(k):]


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------------------
def work(case):
    size = TYPES[case["dtype"]].itemsize
    if case["what"] in ("scan", "step"):
        B, L, H, K, dk, dv = case["batch"], case.get("length", 1), case["heads"], case["kv_heads"], case["dk"], case["dv"]
        rows = B * L * (H * dk + K * (dk + dv) + H * dv) * size
        state = B * H * dk * dv
        if case["what"] == "step":
            return {"bytes": rows + 8 * state, "flops": 5 * state}
        c = min(CHUNK, L)
        scan = B * L * H * ((c + 1) * (dk + dv) + (4 if L > CHUNK or case["ragged"] else 2) * dk * dv)
        byte = rows + 4 * state * (2 if case["ragged"] else 1)
        if case["train"]:                                       # q, k, v and the gradient of o in, three gradients out; three such scans
            byte += rows + B * L * (H * dk + K * (dk + dv)) * size + (8 * state if case["ragged"] else 0)
            scan *= 4
        return {"bytes": byte, "flops": scan}
    if case["what"] == "norm":
        B, L, D, stream = case["batch"], case["length"], case["dim"], TYPES[case["stream"]].itemsize
        n = B * L * D
        gate = {"none": 0, "channel": 4 * D, "sequence": B * D * size, "token": n * size}[case["gate"]]
        byte = 2 * n * (stream + size) + gate + 16 * D
        if case["train"]:
            byte += 3 * n * (stream + size) + 2 * gate + 16 * D
        return {"bytes": byte, "flops": n * (50 if case["train"] else 15)}
    n = case["rows"] * case["vocab"]
    return {"bytes": n * size * (3 if case["train"] else 1) + case["rows"] * (16 + 12 * case["top"]), "flops": n * (14 if case["train"] else 6)}
