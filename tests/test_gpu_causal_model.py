"""linear_attention, gated_residual_norm and token_logprobs together, as a causal model uses them: two layers of a mixer and a GLU
MLP in sandwich norms, scored at the end -- one training step against float64, and a prompt that is continued token by token.

Bounds: both sides compute the same function; the float32 side passes through fewer than 2^9 roundings in a row on the way to any
value (two layers of sums over at most 256 terms, two norms each), each within 2^-24 of the largest magnitude at hand, and the norms
keep magnitudes near one: 2^-15 of a tensor's largest value, gradients 2^-13 (twice the depth, and sums over 2 x 37 tokens)."""
import pytest
import torch
import torch.nn.functional as F

import m2_b200
from m2_b200 import ops

pytestmark = pytest.mark.gpu
D, H, K, DH, INNER, V, LAYERS = 64, 4, 2, 16, 128, 211, 2
EPS = 1e-5


def make_weights(seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rnd(*s, scale=None):
        return (torch.randn(s, device="cuda", generator=g) * (scale or s[-1] ** -0.5)).requires_grad_()

    def ones():
        return (1 + 0.1 * torch.randn(D, device="cuda", generator=g)).requires_grad_()

    layers = [dict(qkv=rnd(H * DH + 2 * K * DH, D), o=rnd(D, H * DH), up=rnd(2 * INNER, D), down=rnd(D, INNER), gate=rnd(D, D),
                   n0=ones(), n1=ones(), n2=ones(), n3=ones(), a=ones()) for _ in range(LAYERS)]
    return dict(embed=rnd(V, D, scale=1.0), layers=layers, last=ones(), first=ones())


def leaves(w):
    return [w["embed"], w["first"], w["last"]] + [t for y in w["layers"] for t in y.values()]


LD = torch.linspace(-0.5, -0.01, H)


def mixer(h, y, lengths, states, fresh):
    q, k, v = F.linear(h, y["qkv"]).split([H * DH, K * DH, K * DH], -1)
    q, k, v = q.unflatten(-1, (H, DH)), k.unflatten(-1, (K, DH)), v.unflatten(-1, (K, DH))
    o, s = m2_b200.linear_attention(q, k, v, LD.cuda(), initial_state=states, lengths=lengths, return_state=True)
    fresh.append(s)
    return F.linear(o.flatten(-2), y["o"])


def mlp(h, y):
    a, b = F.linear(h, y["up"]).chunk(2, -1)
    return F.linear(F.gelu(a) * b, y["down"])


def forward(w, ids, lengths=None, states=None):
    """Logits and the layers' states."""
    x = w["embed"][ids]
    _, h = m2_b200.gated_residual_norm(x, x, before_weight=w["first"], eps=EPS, rms=True, residual_scale=0.0)
    fresh = []
    for i, y in enumerate(w["layers"]):
        out = mixer(h, y, lengths, states[i] if states else None, fresh)
        x, h = m2_b200.gated_residual_norm(x, out, gate=torch.sigmoid(F.linear(h, y["gate"])), residual_scale=y["a"], after_weight=y["n0"],
                                           before_weight=y["n1"], eps=EPS, rms=True)
        x, h = m2_b200.gated_residual_norm(x, mlp(h, y), after_weight=y["n2"], before_weight=y["n3"], eps=EPS, rms=True)
    _, h = m2_b200.gated_residual_norm(x, h, before_weight=w["last"], eps=EPS, rms=True)
    return F.linear(h, w["embed"] * 0.2), fresh


def reference(w, ids, lengths):
    def rms(t, weight):
        return t / (t.square().mean(-1, keepdim=True) + EPS).sqrt() * weight

    B, L = ids.shape
    x = w["embed"][ids]
    h = rms(x, w["first"])
    live = torch.arange(L, device="cuda") < lengths[:, None]
    gap = torch.arange(L, device="cuda")[:, None] - torch.arange(L, device="cuda")
    decay = torch.where(gap >= 0, torch.exp(LD.double().cuda()[:, None, None] * gap.clamp(min=0)), 0.0)
    for y in w["layers"]:
        q, k, v = F.linear(h, y["qkv"]).split([H * DH, K * DH, K * DH], -1)
        q = q.unflatten(-1, (H, DH)).transpose(1, 2)
        k, v = (t.unflatten(-1, (K, DH)).transpose(1, 2).repeat_interleave(H // K, 1) for t in (k, v))
        o = ((q @ k.mT) * DH ** -0.5 * decay) @ v
        o = torch.where(live[:, None, :, None], o, 0.0).transpose(1, 2).flatten(-2)
        x, h0 = y["a"] * x + torch.sigmoid(F.linear(h, y["gate"])) * rms(F.linear(o, y["o"]), y["n0"]), h
        h = rms(x, y["n1"])
        x = x + rms(mlp(h, y), y["n2"])
        h = rms(x, y["n3"])
    return F.linear(rms(x + h, w["last"]), w["embed"] * 0.2)


def test_training_step_of_a_padded_batch():
    w = make_weights()
    ids = torch.randint(0, V, (2, 37), device="cuda")
    lengths = torch.tensor([37, 23], device="cuda")
    targets = torch.where(torch.arange(37, device="cuda") < lengths[:, None], ids.roll(-1, 1), -100)
    logits, _ = forward(w, ids, lengths)
    out = m2_b200.token_logprobs(logits, targets, top=3)
    loss = -(out.logprob + 0.01 * out.entropy).sum() / lengths.sum()
    grads = torch.autograd.grad(loss, leaves(w))
    wide = dict(embed=w["embed"].detach().double().requires_grad_(), first=w["first"].detach().double().requires_grad_(),
                last=w["last"].detach().double().requires_grad_(),
                layers=[{n: t.detach().double().requires_grad_() for n, t in y.items()} for y in w["layers"]])
    ref = reference(wide, ids, lengths)
    used = targets != -100
    assert (logits.double() - ref)[used].abs().max() <= 2.0 ** -15 * ref.abs().max()
    lp = torch.log_softmax(ref, -1)
    got = lp.gather(-1, targets.clamp(min=0)[..., None])[..., 0]
    loss64 = -(torch.where(used, got - 0.01 * (lp.exp() * lp).sum(-1), 0.0)).sum() / lengths.sum()
    assert abs(loss.double() - loss64) <= 2.0 ** -15 * abs(loss64)
    for a, b in zip(grads, torch.autograd.grad(loss64, leaves(wide))):
        assert (a.double() - b).abs().max() <= 2.0 ** -13 * b.abs().max()
    assert (out.top_id[used] == ref.topk(3, -1).indices[used]).float().mean() > 0.99 and (out.top_id[~used] == -1).all()


def test_a_prompt_continued_token_by_token():
    """The state behind a prompt and the single-token steps give what the whole text gives, in one graph a token."""
    w = make_weights(1)
    ids = torch.randint(0, V, (3, 30), device="cuda")
    with torch.no_grad():
        whole, _ = forward(w, ids)
        _, states = forward(w, ids[:, :20])

        def step(token):
            x = w["embed"][token]
            _, h = m2_b200.gated_residual_norm(x, x, before_weight=w["first"], eps=EPS, rms=True, residual_scale=0.0)
            for y, s in zip(w["layers"], states):
                q, k, v = ops.linear_fwd(h[:, None], y["qkv"].detach(), None)[:, 0].split([H * DH, K * DH, K * DH], -1)
                o = m2_b200.linear_attention_step(q.unflatten(-1, (H, DH)), k.unflatten(-1, (K, DH)), v.unflatten(-1, (K, DH)), ld, s)
                x, h = m2_b200.gated_residual_norm(x, F.linear(o.flatten(-2), y["o"]), gate=torch.sigmoid(F.linear(h, y["gate"])), residual_scale=y["a"],
                                                   after_weight=y["n0"], before_weight=y["n1"], eps=EPS, rms=True)
                x, h = m2_b200.gated_residual_norm(x, mlp(h, y), after_weight=y["n2"], before_weight=y["n3"], eps=EPS, rms=True)
            _, h = m2_b200.gated_residual_norm(x, h, before_weight=w["last"], eps=EPS, rms=True)
            return m2_b200.token_logprobs(F.linear(h, w["embed"] * 0.2), target, top=5)

        ld = LD.cuda()
        token, target = ids[:, 20].clone(), ids[:, 21].clone()
        saved = [s.clone() for s in states]
        step(token)                                            # once outside, so that nothing is laid out while capturing
        for s, t in zip(states, saved):
            s.copy_(t)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(token)
        for s, t in zip(states, saved):
            s.copy_(t)
        for t in range(20, 29):
            token.copy_(ids[:, t])
            target.copy_(ids[:, t + 1])
            graph.replay()
            ref = torch.log_softmax(whole[:, t].double(), -1)
            got = ref.gather(-1, target[:, None])[:, 0]
            assert (out.logprob.double() - got).abs().max() <= 2.0 ** -14 * ref.abs().max()
            assert (out.top_logprob.double() - ref.topk(5, -1).values).abs().max() <= 2.0 ** -14 * ref.abs().max()


def test_calls_on_several_streams_at_once():
    """Nothing is shared between calls: the same bits on four streams side by side."""
    q, k, v = (torch.randn(2, 900, 4, 64, device="cuda").bfloat16().requires_grad_() for _ in range(3))
    x, y = torch.randn(64, 40, 768, device="cuda", requires_grad=True), torch.randn(64, 40, 768, device="cuda").bfloat16().requires_grad_()
    gate, w = torch.randn(64, 1, 768, device="cuda", requires_grad=True), torch.randn(768, device="cuda", requires_grad=True)
    logits, target = torch.randn(200, 30528, device="cuda").bfloat16().requires_grad_(), torch.randint(0, 30528, (200,), device="cuda")
    ld = LD.cuda()
    state = torch.randn(2, 4, 64, 64, device="cuda")

    def run():
        o, s = m2_b200.linear_attention(q, k, v, ld, return_state=True)
        outs = [o, s, *torch.autograd.grad([o, s], [q, k, v], [torch.ones_like(o), torch.ones_like(s)])]
        r, h = m2_b200.gated_residual_norm(x, y, gate=gate, after_weight=w, before_weight=w, eps=EPS)
        outs += [r, h, *torch.autograd.grad([r, h], [x, y, gate, w], [torch.ones_like(r), torch.ones_like(h)])]
        t = m2_b200.token_logprobs(logits, target, top=20)
        outs += [*t, *torch.autograd.grad(t.logprob.sum() + t.entropy.sum(), [logits])]
        own = state.clone()
        with torch.no_grad():
            outs += [m2_b200.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, own), own]
        return [t.detach() for t in outs]

    ref = run()
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for stream in streams:
            with torch.cuda.stream(stream):
                got.append(run())
        torch.cuda.synchronize()
        for outs in got:
            assert all(torch.equal(a, b) for a, b in zip(outs, ref))
