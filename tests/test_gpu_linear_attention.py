"""linear_attention and linear_attention_step on the GPU against the definition in float64, token by token.

Bounds, element by element.  Let M be what the operator gives for |q|, |k|, |v| (and |state|): every product that enters an output
enters M with its absolute value.  float32: an output is a nest of sums of at most dk, 64 and 2 L / 64 terms with a handful of
roundings around them, so it is off by less than (dk + 64 + L / 32 + 16) 2^-24 M.  bf16: every product passes one more rounding of
half a step, 2^-8 (of its weight, or of the state that q meets), and the output one: 2^-8 (M + |o|), sums as in float32 but up to
twice as far off where tensor cores cut instead of rounding."""
import pytest
import torch

import m2_b200

pytestmark = pytest.mark.gpu
U32, U16 = 2.0 ** -24, 2.0 ** -8


def definition(q, k, v, ld, scale, s0, lengths):
    """float64; differentiable."""
    B, L, H, dk = q.shape
    K, dv = v.shape[2:]
    s = s0 if s0 is not None else q.new_zeros(B, H, dk, dv)
    k, v = k.repeat_interleave(H // K, 2), v.repeat_interleave(H // K, 2)
    out = []
    for t in range(L):
        on = (torch.full((B,), L, device=q.device) if lengths is None else lengths) > t
        on = on[:, None, None]
        new = torch.exp(ld)[None, :, None, None] * s + torch.where(on, k[:, t], 0)[..., None] * torch.where(on, v[:, t], 0)[..., None, :]
        s = torch.where(on[..., None], new, s)
        out.append(torch.where(on, scale * (torch.where(on, q[:, t], 0)[..., None] * s).sum(-2), 0))
    return (torch.stack(out, 1) if out else q.new_zeros(B, 0, H, dv)), s


def make(B, L, H, K, dk, dv, dtype, seed=0, strong=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    wide = torch.randn(B, L, H * dk + K * (dk + dv) + 3, device="cuda", generator=g).to(dtype)
    q, k, v = wide[..., :H * dk], wide[..., H * dk:(H + K) * dk], wide[..., (H + K) * dk:(H + K) * dk + K * dv]
    q, k, v = q.unflatten(-1, (H, dk)), k.unflatten(-1, (K, dk)), v.unflatten(-1, (K, dv))
    low = -3.0 if strong else -0.1
    ld = torch.linspace(low, -2.0 ** -12, H, device="cuda") if H > 1 else torch.tensor([low], device="cuda")
    return q, k, v, ld, torch.randn(B, H, dk, dv, device="cuda", generator=g)


def slack(dtype, L, d, M, ref):
    n = (d + 64 + L / 32 + 16) * U32
    return (U16 * (M + ref.abs()) + 2 * n * M) if dtype == torch.bfloat16 else (n * M + U32 * ref.abs())


def within(got, ref, bound, what):
    off = (got.double() - ref).abs()
    assert torch.isfinite(got).all(), what
    assert (off <= bound + 1e-30).all(), f"{what}: {(off / (bound + 1e-30)).max().item():.2f} of the bound at {off.argmax().item()}"


SHAPES = [
    # B, L, H, K, dk, dv
    (1, 1, 1, 1, 1, 1),
    (2, 1, 4, 2, 64, 64),
    (1, 2, 2, 2, 64, 64),
    (2, 63, 2, 1, 64, 64),
    (1, 64, 3, 3, 64, 128),
    (2, 65, 4, 4, 128, 64),
    (1, 129, 2, 2, 128, 128),
    (3, 200, 6, 2, 32, 16),
    (1, 130, 2, 1, 80, 40),
    (2, 77, 3, 3, 7, 5),
    (1, 100, 2, 2, 96, 104),
    (1, 700, 2, 2, 64, 64),
    (1, 1111, 1, 1, 72, 128),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("state", [False, True])
def test_forward_and_gradients(shape, dtype, state):
    B, L, H, K, dk, dv = shape
    q, k, v, ld, s0 = make(*shape, dtype, seed=L + dk, strong=L % 2 == 1)
    s0 = s0 if state else None
    lengths = torch.tensor([max(0, L - 17 * i * (i + 1)) for i in range(B)], device="cuda", dtype=torch.int32) if state else None
    scale = 0.37
    leaves = [t.detach().requires_grad_() for t in (q, k, v)] + ([s0.requires_grad_()] if state else [])
    o, s = m2_b200.linear_attention(*leaves[:3], ld, scale=scale, initial_state=s0, lengths=lengths, return_state=True)
    g = torch.Generator(device="cuda").manual_seed(5)
    do, ds = torch.randn(o.shape, device="cuda", generator=g).to(dtype), torch.randn(s.shape, device="cuda", generator=g)
    grads = torch.autograd.grad([o, s], leaves, [do, ds] if state else [do, torch.zeros_like(ds)])
    wide = [t.detach().double().requires_grad_() for t in leaves]
    ro, rs = definition(*wide[:3], ld.double(), scale, wide[3] if state else None, lengths)
    rg = torch.autograd.grad([ro, rs], wide, [do.double(), ds.double() * state])
    big = [t.detach().double().abs().requires_grad_() for t in leaves]
    mo, ms = definition(*big[:3], ld.double(), scale, big[3] if state else None, lengths)
    mg = torch.autograd.grad([mo, ms], big, [do.double().abs(), ds.double().abs() * state])
    within(o, ro, slack(dtype, L, dk, mo, ro), "o")
    within(s, rs, (64 + L / 32 + 16) * 2 * U32 * ms, "state")
    for name, got, ref, M, d in zip(("dq", "dk", "dv"), grads, rg, mg, (dv, dv, dk)):
        within(got, ref, slack(dtype, L, d + H // K, M, ref), name)
    if state:
        within(grads[3], rg[3], (64 + L / 32 + 16) * 2 * U32 * mg[3], "d initial_state")
        for b in range(B):
            n = int(lengths[b])
            assert not o[b, n:].any() and not any(t[b, n:].any() for t in grads[:3])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_long_axis_in_segments_equals_the_same_in_pieces(dtype):
    """One long text (its axis is cut over many blocks) against the text in pieces, each from the state of the last."""
    q, k, v, ld, s0 = make(1, 5000, 2, 1, 64, 64, dtype, seed=3)
    o, s = m2_b200.linear_attention(q, k, v, ld, initial_state=s0, return_state=True)
    parts, state = [], s0
    for at in range(0, 5000, 190):
        p, state = m2_b200.linear_attention(q[:, at:at + 190], k[:, at:at + 190], v[:, at:at + 190], ld, initial_state=state, return_state=True)
        parts.append(p)
    M, ms = m2_b200.linear_attention(q.abs().float(), k.abs().float(), v.abs().float(), ld, initial_state=s0.abs(), return_state=True)
    ref = torch.cat(parts, 1).double()
    within(o, ref, 2 * slack(dtype, 5000, 64, M.double() * 1.01, ref), "o")
    within(s, state.double(), 2 * (64 + 5000 / 32 + 16) * 2 * U32 * ms.double() * 1.01, "state")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dk,dv", [(64, 64), (64, 128), (40, 72)])
def test_texts_that_end_in_any_segment(dk, dv, dtype):
    """Texts of very different lengths whose axis is cut: they end in front of, on and behind the cuts, and gradients run back from there."""
    L, H, K = 650, 2, 1
    lengths = torch.tensor([0, 1, 127, 128, 129, 400, 512, 650], device="cuda")
    q, k, v, ld, s0 = make(len(lengths), L, H, K, dk, dv, dtype, seed=11)
    leaves = [t.detach().requires_grad_() for t in (q, k, v, s0)]
    o, s = m2_b200.linear_attention(*leaves[:3], ld, initial_state=leaves[3], lengths=lengths, return_state=True)
    do, ds = torch.randn_like(o), torch.randn_like(s)
    grads = torch.autograd.grad([o, s], leaves, [do, ds])
    runs = []
    for sign in (lambda t: t, torch.abs):                   # the definition, and of the absolute values
        wide = [sign(t.detach().double()).requires_grad_() for t in leaves]
        out = definition(*wide[:3], ld.double(), dk ** -0.5, wide[3], lengths)
        runs.append([*out, *torch.autograd.grad(out, wide, [sign(do.double()), sign(ds.double())])])
    ref, big = runs
    for name, got, r, M, d in zip(("o", "state", "dq", "dk", "dv", "d initial"), [o, s, *grads], ref, big, (dk, 0, dv, dv + 2, dk + 2, 0)):
        within(got, r, slack(dtype if d else torch.float32, L, d + 80, M, r), name)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_values_behind_a_text_are_not_read(dtype):
    q, k, v, ld, s0 = make(3, 150, 2, 2, 64, 64, dtype)
    n = torch.tensor([0, 97, 150], device="cuda")
    clean = m2_b200.linear_attention(q, k, v, ld, initial_state=s0, lengths=n, return_state=True)
    q, k, v = (t.clone() for t in (q, k, v))
    for t in (q, k, v):
        for b in range(3):
            t[b, int(n[b]):] = float("nan") if b else float("inf")
    leaves = [t.requires_grad_() for t in (q, k, v)]
    o, s = m2_b200.linear_attention(*leaves, ld, initial_state=s0, lengths=n, return_state=True)
    assert torch.equal(o, clean[0]) and torch.equal(s, clean[1])
    assert torch.equal(s[0], s0[0]) and not o[0].any()
    do = torch.ones_like(o)
    do[0], do[1, 97:] = float("nan"), float("nan")
    for g in torch.autograd.grad(o, leaves, do):
        assert torch.isfinite(g).all() and not g[0].any() and not g[1, 97:].any()


def test_lengths_outside_the_tensor_are_cut():
    q, k, v, ld, _ = make(2, 40, 2, 2, 16, 16, torch.float32)
    a = m2_b200.linear_attention(q, k, v, ld, lengths=torch.tensor([-3, 99], device="cuda"))
    b = m2_b200.linear_attention(q, k, v, ld, lengths=torch.tensor([0, 40], device="cuda"))
    assert torch.equal(a, b)


def test_no_memory_and_full_memory():
    """log_decay of -inf: each token sees itself alone; 0: plain sums."""
    q, k, v, _, _ = make(1, 90, 2, 2, 32, 32, torch.float32)
    ld = torch.tensor([-float("inf"), 0.0], device="cuda")
    o, s = m2_b200.linear_attention(q, k, v, ld, scale=1.0, return_state=True)
    alone = (q[:, :, 0].double() * k[:, :, 0].double()).sum(-1, keepdim=True) * v[:, :, 0].double()
    assert (o[:, :, 0].double() - alone).abs().max() < 1e-4
    assert (s[:, 0].double() - k[:, -1, 0].double()[..., None] * v[:, -1, 0].double()[:, None]).abs().max() < 1e-5
    ro, rs = definition(q.double(), k.double(), v.double(), ld.double(), 1.0, None, None)
    assert (o[:, :, 1].double() - ro[:, :, 1]).abs().max() < 1e-3 and (s[:, 1].double() - rs[:, 1]).abs().max() < 1e-4


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", ["heads first", "odd offset", "channels apart"])
def test_layouts(dtype, layout):
    q, k, v, ld, _ = (t.contiguous() for t in make(2, 70, 4, 2, 64, 64, dtype))
    ref = m2_b200.linear_attention(q, k, v, ld)
    if layout == "heads first":
        q, k, v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v))
    elif layout == "odd offset":
        q, k, v = (torch.cat([t.reshape(-1)[:1], t.reshape(-1)])[1:].view(t.shape) for t in (q, k, v))
    else:
        q, k, v = (t.transpose(2, 3).contiguous().transpose(2, 3) for t in (q, k, v))
    assert torch.equal(m2_b200.linear_attention(q, k, v, ld), ref)


def test_gradient_against_differences():
    """o is linear in each of q, k and v: a difference of any width is the derivative, up to the rounding of both sums."""
    q, k, v, ld, s0 = make(2, 150, 4, 2, 48, 64, torch.float32)
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v, s0)]

    def f(q, k, v, s0):
        return m2_b200.linear_attention(q, k, v, ld, initial_state=s0, return_state=True)

    outs = f(*leaves)
    w = [torch.randn_like(t) for t in outs]
    grads = torch.autograd.grad(outs, leaves, w)
    for i, leaf in enumerate(leaves):
        d = torch.randn_like(leaf)
        with torch.no_grad():
            hi, lo = (f(*[t + sign * d if j == i else t for j, t in enumerate(leaves)]) for sign in (1, -1))
        diff = sum(((a.double() - b.double()) * c.double()).sum() for a, b, c in zip(hi, lo, w)) / 2
        ours = (grads[i].double() * d.double()).sum()
        size = sum((a.double().abs() * c.double().abs()).sum() for a, c in zip(hi, w))
        assert abs(diff - ours) <= 300 * U32 * size


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 1), (3, 4, 2, 64, 64), (2, 3, 3, 128, 128), (2, 2, 1, 96, 40), (5, 2, 2, 7, 70), (256, 12, 12, 64, 64)])
def test_steps_equal_the_definition_and_the_sequence(shape, dtype):
    B, H, K, dk, dv = shape
    L = 5
    q, k, v, ld, s0 = make(B, L, H, K, dk, dv, dtype, seed=9)
    state = s0.clone()
    outs = [m2_b200.linear_attention_step(q[:, t], k[:, t], v[:, t], ld, state) for t in range(L)]
    ro, rs = definition(q.double(), k.double(), v.double(), ld.double(), dk ** -0.5, s0.double(), None)
    mo, ms = definition(q.double().abs(), k.double().abs(), v.double().abs(), ld.double(), dk ** -0.5, s0.double().abs(), None)
    o = torch.stack(outs, 1)
    within(o, ro, (U16 if dtype == torch.bfloat16 else U32) * ro.abs() + (dk + 4 * L + 8) * U32 * mo, "o")
    within(state, rs, (4 * L + 4) * U32 * ms, "state")
    po, ps = m2_b200.linear_attention(q, k, v, ld, initial_state=s0, return_state=True)
    within(po, ro, slack(dtype, L, dk, mo, ro), "o of the sequence")
    within(ps, rs, (64 + 16) * 2 * U32 * ms, "state of the sequence")


def test_step_in_a_larger_cache():
    """The state is a slice of a cache: nothing beside it changes."""
    q, k, v, ld, s0 = make(2, 1, 4, 4, 16, 12, torch.bfloat16)
    cache = torch.randn(3, 6, 16, 12, device="cuda")
    before = cache.clone()
    ref = before[:2, 1:5].clone()
    o = m2_b200.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, cache[:2, 1:5])
    o2 = m2_b200.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, ref)
    assert torch.equal(o, o2) and torch.equal(cache[:2, 1:5], ref)
    mask = torch.ones_like(cache, dtype=torch.bool)
    mask[:2, 1:5] = False
    assert torch.equal(cache[mask], before[mask])


def test_refusals_on_the_device():
    q, k, v, ld, s0 = make(2, 4, 4, 4, 16, 16, torch.float32)
    with pytest.raises(RuntimeError, match="constant"):
        m2_b200.linear_attention(q, k, v, ld.clone().requires_grad_())
    for scale in (0.0, float("nan"), float("inf"), 1e-45):
        with pytest.raises(ValueError, match="scale"):
            m2_b200.linear_attention(q, k, v, ld, scale=scale)
        with pytest.raises(ValueError, match="scale"):
            m2_b200.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, s0, scale=scale)
    with pytest.raises(ValueError, match="initial_state"):
        m2_b200.linear_attention(q, k, v, ld, initial_state=s0.bfloat16())
    with pytest.raises(ValueError, match="lengths"):
        m2_b200.linear_attention(q, k, v, ld, lengths=torch.tensor([1.0, 2.0], device="cuda"))
    with pytest.raises(ValueError, match="lengths"):
        m2_b200.linear_attention(q, k, v, ld, lengths=torch.tensor([1, 2]))
    with pytest.raises(RuntimeError, match="up to 128|1 to 128"):
        m2_b200.linear_attention(torch.zeros(1, 2, 1, 129, device="cuda"), torch.zeros(1, 2, 1, 129, device="cuda"), torch.zeros(1, 2, 1, 8, device="cuda"), ld[:1])
    step = (q[:, 0], k[:, 0], v[:, 0], ld)
    with pytest.raises(ValueError, match="in place"):
        m2_b200.linear_attention_step(*step, s0[:1].expand(2, 4, 16, 16))
    with pytest.raises(ValueError, match="in place"):
        m2_b200.linear_attention_step(*step, s0.transpose(2, 3))
    with pytest.raises(RuntimeError, match="no gradient"):
        m2_b200.linear_attention_step(q[:, 0].clone().requires_grad_(), *step[1:], s0)


def test_a_changed_state_is_seen_by_autograd():
    q, k, v, ld, s0 = make(1, 6, 2, 2, 16, 16, torch.float32)
    q = q.detach().clone().requires_grad_()
    o = m2_b200.linear_attention(q, k, v, ld, initial_state=s0)
    m2_b200.linear_attention_step(q[:, 0].detach(), k[:, 0], v[:, 0], ld, s0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        o.sum().backward()


def test_empty():
    q, k, v, ld, s0 = make(2, 0, 2, 2, 16, 16, torch.float32)
    s0.requires_grad_()
    o, s = m2_b200.linear_attention(q, k, v, ld, initial_state=s0, return_state=True)
    assert o.shape == (2, 0, 2, 16) and torch.equal(s, s0)
    (g,) = torch.autograd.grad(s, [s0], torch.full_like(s, 2.0))
    assert torch.equal(g, torch.full_like(g, 2.0))
    q, k, v, ld, s0 = make(0, 5, 2, 2, 16, 16, torch.float32)
    assert m2_b200.linear_attention(q, k, v, ld).shape == (0, 5, 2, 16)
    assert m2_b200.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, s0).shape == (0, 2, 16)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_same_bits_twice_on_another_stream_and_in_a_graph(dtype):
    q, k, v, ld, s0 = make(1, 900, 4, 2, 64, 64, dtype)
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v, s0)]

    def run():
        o, s = m2_b200.linear_attention(*leaves[:3], ld, initial_state=leaves[3], return_state=True)
        return [o.detach(), s.detach(), *torch.autograd.grad([o, s], leaves, [torch.ones_like(o), torch.ones_like(s)])]

    ref = run()
    assert all(torch.equal(a, b) for a, b in zip(ref, run()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(ref, other))
    torch.cuda.synchronize()
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a = run()
    with torch.cuda.graph(second):
        b = run()
    with torch.no_grad():
        for t in leaves:
            t.mul_(0.5)
    graph.replay()
    second.replay()
    graph.replay()
    new = run()
    assert all(torch.equal(x, y) and torch.equal(x, z) for x, y, z in zip(new, a, b))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_state_in_and_out_in_the_same_memory(dtype):
    """A caller of the C interface continues a text in place, the axis cut over many blocks."""
    import ctypes as C
    from m2_b200 import _lib, linear_attn as la
    q, k, v, ld, s0 = (t.contiguous() for t in make(2, 3000, 3, 3, 64, 64, dtype))
    ref = m2_b200.linear_attention(q, k, v, ld, initial_state=s0, return_state=True)
    for _ in range(5):
        state, o = s0.clone(), torch.empty_like(v)
        a = la._args(q, k, v, ld, 64 ** -0.5, state, None, o, state)
        work = la._workspace(a, q.device, 0)
        assert work is not None
        m2_b200.ops._launch("m2_linear_attention_fwd", q, _lib.lib().m2_linear_attention_fwd, C.byref(a))
        assert torch.equal(o, ref[0]) and torch.equal(state, ref[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_more_sequences_than_a_grid_axis(dtype):
    q, k, v, ld, s0 = make(70001, 3, 1, 1, 4, 4, dtype)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o, s = m2_b200.linear_attention(*leaves, ld, initial_state=s0, return_state=True)
    grads = torch.autograd.grad(o, leaves, torch.ones_like(o))
    tail = [t.detach()[-5:].clone().requires_grad_() for t in leaves]
    ro, rs = m2_b200.linear_attention(*tail, ld, initial_state=s0[-5:], return_state=True)
    assert torch.equal(o[-5:], ro) and torch.equal(s[-5:], rs)
    for a, b in zip(grads, torch.autograd.grad(ro, tail, torch.ones_like(ro))):
        assert torch.equal(a[-5:], b)
    state, few = s0.clone(), s0[-5:].clone()
    with torch.no_grad():
        o = m2_b200.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, state)
        ro = m2_b200.linear_attention_step(q[-5:, 0], k[-5:, 0], v[-5:, 0], ld, few)
    assert torch.equal(o[-5:], ro) and torch.equal(state[-5:], few)
