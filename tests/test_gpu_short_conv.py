"""causal_conv and causal_conv_step against their definition in 64 bits.

Bounds: a value is a sum of W products and a bias, in float32, an error of at most (W + 1) 2^-24 of the sum M of their absolute values; silu multiplies by a sigmoid with
2^-22 + |v| 2^-23 (the exp) + 2 2^-23 (the quotient), below 2^-19 for |v| < 16, and passes v's own error on by a slope below 1.1.  Sums of gradients add 2^-24 a term.
An output is rounded once to its type."""
import pytest
import torch
import torch.nn.functional as F

import m2_b200
from tests.test_gpu_linear_attention import U16, U32, within

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def seeded():
    torch.manual_seed(0)


SHAPES = [(1, 1, 1, 1), (1, 1, 8, 4), (2, 33, 64, 4), (3, 70, 100, 3), (2, 40, 24, 2), (2, 129, 130, 4), (2, 300, 768, 4), (1, 700, 33, 8), (2, 65, 64, 5), (2, 9, 96, 7), (2, 50, 16, 1),
          (1, 2, 32, 8), (1, 3000, 40, 4)]
EPS = 2.0 ** -18


def definition(x, w, bias, state, lengths, silu):
    """y and the last W - 1 inputs, in 64 bits, differentiable."""
    B, L, D = x.shape
    W = w.shape[1]
    ys, states = [], []
    for i in range(B):
        n = int(lengths[i].clamp(0, L)) if lengths is not None else L
        line = torch.cat([state[i] if state is not None else x.new_zeros((W - 1, D)), x[i, :n]])
        v = (line.unfold(0, W, 1) * w).sum(-1) + (bias if bias is not None else 0.0) if n else x[i, :0]
        ys.append(torch.cat([F.silu(v) if silu else v, x.new_zeros((L - n, D))]))
        states.append(line[n:])
    return torch.stack(ys), torch.stack(states)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("silu,ragged", [(True, False), (False, True), (True, True)])
def test_whole_sequences_and_gradients(shape, silu, ragged, dtype):
    B, L, D, W = shape
    g = torch.Generator(device="cuda").manual_seed(L)

    def rnd(*s):
        return torch.randn(s, device="cuda", generator=g)

    t = [rnd(B, L, D).to(dtype), rnd(D, W) * W ** -0.5, rnd(D) if silu else None, rnd(B, W - 1, D).to(dtype) if ragged else None]
    lengths = torch.randint(0, L + 1, (B,), device="cuda", generator=g) if ragged else None
    leaves = [v.clone().requires_grad_() if v is not None else None for v in t]
    x, w, bias, state = leaves
    y, last = m2_b200.causal_conv(x, w, bias, activation="silu" if silu else None, initial_state=state, lengths=lengths, return_state=True)
    with torch.no_grad():
        y2 = m2_b200.causal_conv(*t[:3], activation="silu" if silu else None, initial_state=t[3], lengths=lengths)
    assert torch.equal(y, y2)
    d_y, d_last = rnd(B, L, D).to(dtype), rnd(B, W - 1, D).to(dtype)
    given = [v for v in leaves if v is not None]
    grads = torch.autograd.grad([y, last], given, [d_y, d_last])
    wide = [v.double().requires_grad_() if v is not None else None for v in t]
    ref = definition(*wide, lengths, silu)
    refs = torch.autograd.grad(ref, [v for v in wide if v is not None], [d_y.double(), d_last.double()], allow_unused=True, materialize_grads=True)
    size = [v.double().abs().requires_grad_() if v is not None else None for v in t]
    M = definition(*size, lengths, False)
    Ms = torch.autograd.grad(M, [v for v in size if v is not None], [d_y.double().abs(), d_last.double().abs()], allow_unused=True, materialize_grads=True)
    kind = U16 if dtype == torch.bfloat16 else U32
    one = EPS + (W + 4) * U32 * (1 + M[0].max())             # silu'' < 0.5: a gradient also sees the error of v
    within(y, ref[0], kind * ref[0].abs() + one * M[0], "y")
    assert torch.equal(last.double(), ref[1])
    for p, r, m, v in zip(grads, refs, Ms, given):
        assert p.dtype == v.dtype
        k = kind if v.dtype == dtype and v.dim() == 3 else U32
        within(p, r, k * r.abs() + 1.2 * (2 * one + (B * L if v.dim() < 3 else W) * U32) * m, str(tuple(v.shape)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,D,W", [(1, 1, 1), (1, 8, 4), (3, 100, 3), (2, 65, 8), (300, 64, 4), (4, 30, 2)])
def test_single_tokens(B, D, W, dtype):
    """Token by token: y as the whole sequence has it, the state as it leaves it."""
    L = 11
    g = torch.Generator(device="cuda").manual_seed(D)
    x, w, bias = torch.randn(B, L, D, device="cuda", generator=g).to(dtype), torch.randn(D, W, device="cuda", generator=g) * W ** -0.5, torch.randn(D, device="cuda", generator=g)
    wide = torch.zeros(B, (W - 1) * D + 3, dtype=dtype, device="cuda")
    state = wide[:, 1:1 + (W - 1) * D].unflatten(1, (W - 1, D)) if W > 1 else torch.zeros(B, 0, D, dtype=dtype, device="cuda")
    first = torch.randn(B, W - 1, D, device="cuda", generator=g).to(dtype)
    state.copy_(first)
    ref, last = definition(x.double(), w.double(), bias.double(), first.double(), None, True)
    M = definition(x.double().abs(), w.double().abs(), bias.double().abs(), first.double().abs(), None, False)[0]
    for i in range(L):
        y = m2_b200.causal_conv_step(x[:, i], state, w, bias, activation="silu")
        within(y, ref[:, i], (U16 if dtype == torch.bfloat16 else U32) * ref[:, i].abs() + (EPS + (W + 4) * U32) * M[:, i], f"token {i}")
    assert torch.equal(state.double(), last) and not wide[:, 0].any() and not wide[:, 1 + (W - 1) * D:].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D,W", [(64, 4), (65, 3), (40, 8), (768, 4)])
def test_strides_and_alignment(D, W, dtype):
    B, L = 2, 70
    x, w = torch.randn(B, L, D, device="cuda").to(dtype), torch.randn(D, W, device="cuda")
    before, g = torch.randn(B, W - 1, D, device="cuda").to(dtype), torch.randn(B, L, D, device="cuda").to(dtype)
    lengths = torch.tensor([70, 3], device="cuda")

    def run(x, g):
        x, v, b = x.detach().requires_grad_(), w.clone().requires_grad_(), before.clone().requires_grad_()
        y, s = m2_b200.causal_conv(x, v, activation="silu", initial_state=b, lengths=lengths, return_state=True)
        return [y, s, *torch.autograd.grad([y, s], [x, v, b], [g, torch.ones_like(s)])]

    ref = run(x, g)
    for off in (0, 1, 4, 8):
        wide = torch.zeros(B, L, D + off + 8, dtype=dtype, device="cuda")
        wide[..., off:off + D] = x
        other = torch.zeros_like(wide)
        other[..., off:off + D] = g
        got = run(wide[..., off:off + D], other[..., off:off + D])
        assert all(torch.equal(p, q) for p, q in zip(got, ref))
    got = run(x.transpose(1, 2).contiguous().transpose(1, 2), g.transpose(0, 1).contiguous().transpose(0, 1))
    assert all(torch.equal(p, q) for p, q in zip(got, ref))
    # what lies behind a text is not read, and nothing of it is returned
    bad, up = x.clone(), g.clone()
    bad[1, 3:] = up[1, 3:] = float("nan")
    assert all(torch.equal(p, q) for p, q in zip(run(bad, up), ref))
    assert not ref[0][1, 3:].any() and not ref[2][1, 3:].any()


def test_a_state_is_handed_on():
    x, w, b = (torch.randn(2, 50, 24, device="cuda", requires_grad=True), torch.randn(24, 4, device="cuda", requires_grad=True), torch.randn(24, device="cuda"))
    whole = m2_b200.causal_conv(x, w, b, activation="silu")
    y, s, state = [], None, None
    for at, to in ((0, 1), (1, 3), (3, 3), (3, 20), (20, 50)):
        v, state = m2_b200.causal_conv(x[:, at:to], w, b, activation="silu", initial_state=state, return_state=True)
        y.append(v)
    parts = torch.cat(y, 1)
    assert torch.equal(parts, whole)
    for p, q in zip(torch.autograd.grad(parts.sum(), [x, w]), torch.autograd.grad(whole.sum(), [x, w])):
        assert (p - q).abs().max() <= 200 * U32 * q.abs().max()


def test_nan_reaches_the_next_tokens_of_its_channel_alone():
    x, w = torch.randn(1, 40, 16, device="cuda"), torch.randn(16, 4, device="cuda")
    y = m2_b200.causal_conv(x, w)
    for value in (float("nan"), float("inf")):
        bad = x.clone()
        bad[0, 10, 3] = value
        z = m2_b200.causal_conv(bad, w)
        hit = torch.zeros_like(y, dtype=torch.bool)
        hit[0, 10:14, 3] = True
        assert torch.equal(z[~hit], y[~hit]) and not torch.isfinite(z[hit]).any()


def test_empty_batches_and_sequences():
    w = torch.randn(6, 3, device="cuda", requires_grad=True)
    for B, L in ((0, 4), (2, 0), (0, 0)):
        x, s = torch.randn(B, L, 6, device="cuda", requires_grad=True), torch.randn(B, 2, 6, device="cuda", requires_grad=True)
        y, t = m2_b200.causal_conv(x, w, initial_state=s, return_state=True)
        assert y.shape == (B, L, 6) and torch.equal(t, s)
        d = torch.autograd.grad([y, t], [x, w, s], [torch.ones_like(y), torch.ones_like(t)])
        assert not d[0].any() and not d[1].any() and torch.equal(d[2], torch.ones_like(s))


def test_twice_the_same_bits_and_gradients_of_some():
    x, w, b = torch.randn(3, 500, 64, device="cuda").bfloat16().requires_grad_(), torch.randn(64, 4, device="cuda", requires_grad=True), torch.randn(64, device="cuda", requires_grad=True)
    up = torch.randn(3, 500, 64, device="cuda").bfloat16()
    runs = [torch.autograd.grad(m2_b200.causal_conv(x, w, b, activation="silu"), [x, w, b], up) for _ in range(2)]
    assert all(torch.equal(p, q) for p, q in zip(*runs))
    for i, keep in enumerate(((x, w.detach(), b.detach()), (x.detach(), w, b.detach()), (x.detach(), w.detach(), b))):
        (d,) = torch.autograd.grad(m2_b200.causal_conv(*keep, activation="silu"), [(x, w, b)[i]], up)
        assert torch.equal(d, runs[0][i])


def test_offsets_beyond_2_31_elements():
    FAR, L, D = 2 ** 31 + 64, 30, 64
    x, w = torch.randn(2, L, D, device="cuda").bfloat16(), torch.randn(D, 4, device="cuda")
    far = torch.empty(FAR + L * D, dtype=torch.bfloat16, device="cuda").as_strided((2, L, D), (FAR, D, 1))
    far.copy_(x)
    p, q = far.detach().requires_grad_(), x.clone().requires_grad_()
    y, z = m2_b200.causal_conv(p, w), m2_b200.causal_conv(q, w)
    assert torch.equal(y, z) and torch.equal(torch.autograd.grad(y, [p], z)[0], torch.autograd.grad(z, [q], z.detach())[0])
