"""causal_conv, selective_scan, dropout, beam_select and reorder_states together with gated_residual_norm and token_logprobs, as a causal model uses them: two
layers of a scan mixer with its short convolution in pre-norm, dropped out on the way to the residual stream -- one training step against float64, the same
step captured, a prompt continued token by token, and a beam search whose states follow the beams.

Bounds: both sides compute the same function; the float32 side passes through fewer than 2^9 roundings in a row on the way to any value (two layers of sums over at most
128 terms, a scan of 37 tokens whose decays carry 2^-22 each, two norms), each within 2^-23 of the largest magnitude at hand, and the norms keep magnitudes near
one: 2^-14 of a tensor's largest value, gradients 2^-12 (twice the depth, and sums over 2 x 37 tokens)."""
import gc

import pytest
import torch
import torch.nn.functional as F

import m2_b200
from tests.test_gpu_operators_promises import launched
from tests.test_gpu_random_drop import kept

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def seeded():
    torch.manual_seed(0)


D, E, N, R, W, V, LAYERS, G = 64, 96, 16, 8, 4, 211, 2, 2
EPS, P, SEED = 1e-5, 0.2, 41


def make_weights(seed=0, grad=True):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rnd(*s, scale=None, mean=0.0):
        return (torch.randn(s, device="cuda", generator=g) * (scale or s[-1] ** -0.5) + mean).requires_grad_(grad)

    layers = [dict(into=rnd(2 * E, D), conv=rnd(E, W), conv_bias=rnd(E, scale=0.1), low=rnd(R + 2 * G * N, E), step=rnd(E, R), bias=rnd(E, scale=0.5, mean=-3.0),
                   log_a=rnd(E, N, scale=0.3), skip=rnd(E, scale=0.1, mean=1.0), out=rnd(D, E), norm=rnd(D, scale=0.1, mean=1.0)) for _ in range(LAYERS)]
    return dict(embed=rnd(V, D, scale=1.0), layers=layers, first=rnd(D, scale=0.1, mean=1.0))


def leaves(w):
    return [w["embed"], w["first"]] + [t for y in w["layers"] for t in y.values()]


def projections(h, y):
    u, z = F.linear(h, y["into"]).split([E, E], -1)
    return u, z


def inner(x, y):
    low, b, c = F.linear(x, y["low"]).split([R, G * N, G * N], -1)
    return F.linear(low, y["step"]), b.unflatten(-1, (G, N)), c.unflatten(-1, (G, N))


def forward(w, ids, lengths=None, states=None, drop=None):
    """Logits and the layers' states."""
    x = w["embed"][ids]
    _, h = m2_b200.gated_residual_norm(x, x, before_weight=w["first"], eps=EPS, rms=True, residual_scale=0.0)
    fresh = []
    for i, y in enumerate(w["layers"]):
        u, z = projections(h, y)
        before, state = states[i] if states else (None, None)
        v, before = m2_b200.causal_conv(u, y["conv"], y["conv_bias"], activation="silu", initial_state=before, lengths=lengths, return_state=True)
        delta, b, c = inner(v, y)
        o, state = m2_b200.selective_scan(v, delta, -torch.exp(y["log_a"]), b, c, skip=y["skip"], gate=z, delta_bias=y["bias"], softplus=True, initial_state=state,
                                          lengths=lengths, return_state=True)
        fresh.append((before, state))
        out = F.linear(o, y["out"])
        if drop is not None:
            x = m2_b200.dropout(out, P, drop[i], residual=x)
            _, h = m2_b200.gated_residual_norm(x, x, before_weight=y["norm"], eps=EPS, rms=True, residual_scale=0.0)
        else:
            x, h = m2_b200.gated_residual_norm(x, out, before_weight=y["norm"], eps=EPS, rms=True)
    return F.linear(h, w["embed"] * 0.2), fresh


def reference(w, ids, lengths, calls=None):
    def rms(t, weight):
        return t / (t.square().mean(-1, keepdim=True) + EPS).sqrt() * weight

    B, L = ids.shape
    x = w["embed"][ids]
    h = rms(x, w["first"])
    live = (torch.arange(L, device="cuda") < lengths[:, None])[..., None]
    group = torch.arange(E, device="cuda") // (E // G)
    for i, y in enumerate(w["layers"]):
        u, z = projections(h, y)
        v = F.pad(torch.where(live, u, 0.0), (0, 0, W - 1, 0)).unfold(1, W, 1)
        v = torch.where(live, F.silu((v * y["conv"]).sum(-1) + y["conv_bias"]), 0.0)
        delta, b, c = inner(v, y)
        s, a = torch.where(live, F.softplus(delta + y["bias"]), 0.0), -torch.exp(y["log_a"])
        state, outs = torch.zeros(B, E, N, dtype=x.dtype, device="cuda"), []
        for t in range(L):
            state = torch.exp(s[:, t, :, None] * a) * state + (s[:, t] * v[:, t])[..., None] * b[:, t][:, group]
            outs.append((state * c[:, t][:, group]).sum(-1))
        o = torch.where(live, (torch.stack(outs, 1) + y["skip"] * v) * F.silu(z), 0.0)
        out = F.linear(o, y["out"])
        if calls is not None:
            t = round(P * 65536)
            out = torch.where(kept(out.numel(), P, SEED, calls[i]).view(out.shape), out * 65536 / (65536 - t), 0.0)
        x = x + out
        h = rms(x, y["norm"])
    return F.linear(h, w["embed"] * 0.2)


def wide(w):
    up = {k: w[k].detach().double().requires_grad_() for k in ("embed", "first")}
    return dict(up, layers=[{n: t.detach().double().requires_grad_() for n, t in y.items()} for y in w["layers"]])


def loss_of(logits, ids, lengths):
    targets = torch.where(torch.arange(ids.shape[1], device="cuda") < lengths[:, None], ids.roll(-1, 1), -100)
    return -m2_b200.token_logprobs(logits, targets).logprob.sum() / lengths.sum()


def reference_loss(logits, ids, lengths):
    used = torch.arange(ids.shape[1], device="cuda") < lengths[:, None]
    lp = torch.log_softmax(logits, -1).gather(-1, ids.roll(-1, 1)[..., None])[..., 0]
    return -torch.where(used, lp, 0.0).sum() / lengths.sum()


def test_training_step_of_a_padded_batch_eager_and_captured():
    w = make_weights()
    ids, lengths = torch.randint(0, V, (2, 37), device="cuda"), torch.tensor([37, 23], device="cuda")
    drop = [torch.tensor([SEED, i], device="cuda") for i in range(LAYERS)]
    used = torch.arange(37, device="cuda") < lengths[:, None]

    def check(loss, grads, calls):
        w64 = wide(w)
        ref = reference(w64, ids, lengths, calls)
        loss64 = reference_loss(ref, ids, lengths)
        assert abs(loss.double() - loss64) <= 2.0 ** -14 * abs(loss64)
        for a, b in zip(grads, torch.autograd.grad(loss64, leaves(w64))):
            assert (a.double() - b).abs().max() <= 2.0 ** -12 * b.abs().max()
        return ref

    logits = forward(w, ids, lengths, drop=drop)[0]
    loss = loss_of(logits, ids, lengths)
    grads = torch.autograd.grad(loss, leaves(w))
    ref = check(loss, grads, [0, 1])
    assert (logits.double() - ref)[used].abs().max() <= 2.0 ** -14 * ref.abs().max()
    del logits, loss, grads, ref                             # nothing eager of these leaves may live while their gradients are captured
    gc.collect()

    # the same step in a graph: other elements are dropped in every replay
    def step():
        loss = loss_of(forward(w, ids, lengths, drop=drop)[0], ids, lengths)
        grads = torch.autograd.grad(loss, leaves(w))
        for s in drop:
            s[1] += LAYERS
        return loss.detach(), grads

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, grads = step()
    for turn in (2, 3):
        ids.copy_(torch.randint(0, V, (2, 37), device="cuda"))
        lengths.copy_(torch.tensor([5, 37], device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        check(loss, grads, [turn * 2 - 2, turn * 2 - 1])


def token(w, ids, states):
    """Logits of one token for every row, the states changed in place."""
    x = w["embed"][ids]
    _, h = m2_b200.gated_residual_norm(x, x, before_weight=w["first"], eps=EPS, rms=True, residual_scale=0.0)
    for y, (before, state) in zip(w["layers"], states):
        u, z = projections(h, y)
        v = m2_b200.causal_conv_step(u, before, y["conv"], y["conv_bias"], activation="silu")
        delta, b, c = inner(v, y)
        o = m2_b200.selective_scan_step(v, delta, -torch.exp(y["log_a"]), b, c, state, skip=y["skip"], gate=z, delta_bias=y["bias"], softplus=True)
        x, h = m2_b200.gated_residual_norm(x, F.linear(o, y["out"]), before_weight=y["norm"], eps=EPS, rms=True)
    return F.linear(h, w["embed"] * 0.2)


def test_a_prompt_continued_token_by_token():
    w = make_weights(1, grad=False)
    ids = torch.randint(0, V, (3, 30), device="cuda")
    whole, _ = forward(w, ids)
    _, states = forward(w, ids[:, :20])
    for t in range(20, 30):
        got = token(w, ids[:, t], states)
        assert (got - whole[:, t]).abs().max() <= 2.0 ** -13 * whole.abs().max()


def test_a_beam_search_in_a_graph():
    """Every step in one captured graph; scores are those of the texts found, by the whole model, and the best of all (beam, token) pairs are taken."""
    B, K, STEPS, END = 2, 4, 6, 7
    w = make_weights(2, grad=False)
    prompt = torch.randint(0, V, (B, 9), device="cuda")
    _, states = forward(w, prompt[:, :-1])
    states = [tuple(t.repeat_interleave(K, 0).contiguous() for t in s) for s in states]
    flat = [t for s in states for t in s]
    ids = prompt[:, -1:].expand(B, K).clone()
    scores = torch.full((B, K), -float("inf"), device="cuda")
    scores[:, 0] = 0
    finished = torch.zeros(B, K, dtype=torch.bool, device="cuda")
    texts = torch.zeros(B, K, STEPS, dtype=torch.long, device="cuda")
    at = torch.zeros((), dtype=torch.long, device="cuda")

    def step():
        logits = token(w, ids.flatten(), states).unflatten(0, (B, K))
        best = m2_b200.beam_select(logits, scores, finished=finished, end_id=END)
        m2_b200.reorder_states(flat + [texts.view(B * K, STEPS)], best.beam)
        texts.scatter_(2, at.expand(B, K, 1), best.token[..., None])
        scores.copy_(best.score)
        finished.copy_(best.finished)
        ids.copy_(best.token)
        at.add_(1)

    kept_values = [t.clone() for t in (*flat, ids, scores, finished, texts, at)]
    step()
    for t, v in zip((*flat, ids, scores, finished, texts, at), kept_values):
        t.copy_(v)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for t, v in zip((*flat, ids, scores, finished, texts, at), kept_values):
        t.copy_(v)
    beams = [[(0.0, [])] for _ in range(B)]                   # the same search over whole texts
    for _ in range(STEPS):
        graph.replay()
        for i in range(B):
            found = []
            for s, text in beams[i]:
                if END in text:
                    found.append((s, text + [END]))
                    continue
                line = torch.cat([prompt[i], torch.tensor(text, dtype=torch.long, device="cuda")])
                lp = torch.log_softmax(forward(w, line[None])[0][0, -1].double(), -1)
                top = lp.topk(K + 1)
                found += [(s + v, text + [j]) for v, j in zip(top.values.tolist(), top.indices.tolist())]
            found.sort(key=lambda f: -f[0])
            assert found[K - 1][0] - found[K][0] > 1e-3 or found[K][1][:-1] == found[K - 1][1][:-1], "a tie: another seed is wanted"
            beams[i] = found[:K]
        torch.cuda.synchronize()
        for i in range(B):
            n = int(at)
            mine = sorted(zip(texts[i, :, :n].tolist(), scores[i].tolist()))
            want = sorted((text, s) for s, text in beams[i])
            assert [m[0] for m in mine] == [q[0] for q in want]
            assert max(abs(m[1] - q[1]) for m, q in zip(mine, want)) <= 2.0 ** -10


def test_calls_on_several_streams_at_once():
    """Nothing is shared between calls: the same bits on four streams side by side."""
    x, delta, z = (torch.randn(1, 900, 96, device="cuda").bfloat16().requires_grad_() for _ in range(3))
    b, c = (torch.randn(1, 900, 16, device="cuda").bfloat16().requires_grad_() for _ in range(2))
    a, cw = -torch.rand(96, 16, device="cuda"), torch.randn(96, 4, device="cuda", requires_grad=True)
    logits, scores = torch.randn(2, 4, 30528, device="cuda"), torch.zeros(2, 4, device="cuda")
    state = torch.randn(8, 500, device="cuda")

    def run():
        v = m2_b200.causal_conv(x, cw, activation="silu")
        y, s = m2_b200.selective_scan(v, delta, a, b, c, gate=z, softplus=True, return_state=True)
        d = m2_b200.dropout(y, 0.3, 5, residual=x)
        outs = [v, y, s, d, *torch.autograd.grad([d, s], [x, delta, z, b, c, cw], [torch.ones_like(d), torch.ones_like(s)])]
        best = m2_b200.beam_select(logits, scores, end_id=3)
        own = state.clone()
        m2_b200.reorder_states(own, best.beam)
        return [t.detach() for t in (*outs, *best, own)]

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
            assert all(torch.equal(p, q) for p, q in zip(outs, ref))


def test_every_kernel_is_counted():
    found = []
    for B, L, E_, N_, dtype in ((2, 40, 64, 16, torch.bfloat16), (1, 900, 64, 16, torch.bfloat16), (1, 900, 40, 50, torch.float32), (2, 0, 64, 16, torch.float32)):
        x = torch.randn(B, L, E_, device="cuda").to(dtype).requires_grad_()
        b = torch.randn(B, L, N_, device="cuda").to(dtype)
        a, w = -torch.rand(E_, N_, device="cuda"), torch.randn(E_, 4, device="cuda", requires_grad=True)
        found.append(launched(lambda: m2_b200.selective_scan(x.detach(), x.detach(), a, b, b, softplus=True)))
        found.append(launched(lambda: m2_b200.causal_conv(x.detach(), w.detach())))
        up = torch.ones_like(x)
        found.append(launched(lambda: torch.autograd.grad(m2_b200.selective_scan(x, x.detach(), a, b, b, softplus=True), [x], up)))
        found.append(launched(lambda: torch.autograd.grad(m2_b200.causal_conv(x, w), [x, w], up)))
        found.append(launched(lambda: torch.autograd.grad(m2_b200.dropout(x, 0.5, 1), [x], up)))
    logits, scores = torch.randn(2, 4, 9000, device="cuda"), torch.zeros(2, 4, device="cuda")
    beam = torch.zeros(2, 4, dtype=torch.long, device="cuda")
    found.append(launched(lambda: m2_b200.beam_select(logits, scores)))
    for states in ([], [torch.zeros(8, 4, device="cuda")], [torch.zeros(8, 4, device="cuda"), torch.zeros(8, 3, device="cuda"), torch.zeros(8, 3, dtype=torch.uint8, device="cuda")],
                   [torch.zeros(8, 4, device="cuda") for _ in range(200)]):
        found.append(launched(lambda: m2_b200.reorder_states(states, beam)))
    assert all(p == q for p, q in found), found
    assert found[0] == (1, 1) and found[5] == (3, 3)


def test_a_tensor_of_another_stream():
    """A call on a side stream that waits for the producer's: what it returns may be used behind it."""
    x = torch.randn(2, 600, 96, device="cuda")
    w, side = torch.randn(96, 4, device="cuda"), torch.cuda.Stream()
    ref = m2_b200.causal_conv(x * 2, w)
    y = x * 2
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = m2_b200.causal_conv(y, w)
        y.record_stream(side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, ref)
