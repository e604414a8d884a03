"""What the documentation of linear_attention, gated_residual_norm and token_logprobs says beside their formulas."""
import gc

import pytest
import torch

import m2_b200
from m2_b200 import ops
from tests.test_gpu_linear_attention import U16, U32, definition, make, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,L,H,dk,dv", [(2, 200, 3, 64, 64), (1, 1500, 2, 64, 64), (2, 300, 2, 128, 128), (1, 1500, 2, 40, 72), (1, 900, 1, 128, 64)])
def test_o_does_not_depend_on_whether_the_state_is_returned(B, L, H, dk, dv, dtype):
    q, k, v = (torch.randn(B, L, H, d, device="cuda").to(dtype) for d in (dk, dk, dv))
    ld = torch.linspace(-0.1, -2.0 ** -10, H, device="cuda")
    alone = m2_b200.linear_attention(q, k, v, ld)
    o, _ = m2_b200.linear_attention(q, k, v, ld, return_state=True)
    assert torch.equal(alone, o)


def kernel_ms(fn, runs=12):
    """The shortest device time of the launches that fn() makes."""
    ops.PROFILE = ops.LaunchProfile()
    try:
        for _ in range(runs):
            fn()
        torch.cuda.synchronize()
        (events,) = ops.PROFILE.events.values()
        return min(s.elapsed_time(e) for s, e in events)
    finally:
        ops.PROFILE = None


def test_ignored_rows_are_not_read_by_the_gradient():
    """1 GB is written whatever the targets are, and as much is read where all rows are used: without the reading it takes about half as long."""
    x = torch.randn(16384, 30528, device="cuda", dtype=torch.bfloat16).requires_grad_()
    took = []
    for target in (5, -100):
        out = m2_b200.token_logprobs(x, torch.full((16384,), target, device="cuda"))
        took.append(kernel_ms(lambda: torch.autograd.grad(out.logprob, [x], torch.ones_like(out.logprob), retain_graph=True)))
    assert took[1] < 0.75 * took[0]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [1, 7, 517, 4097, 20000])
def test_gradient_of_ignored_rows_is_zero_up_to_its_ends(V, dtype):
    """What the kernel leaves out would hold the bits of the memory's last user."""
    x = torch.randn(7, V, device="cuda").to(dtype).requires_grad_()
    t = torch.tensor([-100, 0, -100, V - 1, -100, -100, 0], device="cuda")
    out = m2_b200.token_logprobs(x, t)
    rubbish = torch.full_like(x, float("nan"))
    del rubbish
    (d,) = torch.autograd.grad(out.logprob.sum() + out.entropy.sum(), [x])
    assert not d[t == -100].any() and torch.isfinite(d).all()
    p = torch.softmax(x.detach().double(), -1)
    for row in (1, 3, 6):                                   # beside ignored rows: the gradient of its own
        H = -(p[row] * p[row].log()).sum()
        ref = -p[row] - p[row] * (p[row].log() + H)
        ref[t[row]] += 1
        assert (d[row].double() - ref).abs().max() <= torch.finfo(dtype).eps / 2 * ref.abs().max() + (V / 256 + 128) * 2.0 ** -24 * 40


def launched(fn):
    """What ops.LAUNCHES counts of a call, and the kernels of a graph that holds the call."""
    from cuda.bindings import runtime
    fn()
    torch.cuda.synchronize()
    graph, before = torch.cuda.CUDAGraph(keep_graph=True), ops.LAUNCHES
    with torch.cuda.graph(graph):
        fn()
    counted = ops.LAUNCHES - before
    count = runtime.cudaGraphGetNodes(graph.raw_cuda_graph(), 0)[2]
    nodes = runtime.cudaGraphGetNodes(graph.raw_cuda_graph(), count)[1]
    kind = runtime.cudaGraphNodeType.cudaGraphNodeTypeKernel
    return counted, sum(runtime.cudaGraphNodeGetType(n)[1] == kind for n in nodes)


def test_every_kernel_is_counted():
    ld = torch.linspace(-0.1, -0.01, 4, device="cuda")
    found = []
    for L, K, dk, dv, dtype in ((64, 4, 64, 64, torch.bfloat16), (2000, 4, 64, 64, torch.bfloat16), (2000, 2, 64, 128, torch.bfloat16), (64, 2, 64, 128, torch.bfloat16),
                                (2000, 2, 32, 32, torch.float32), (0, 4, 64, 64, torch.bfloat16)):
        q, k, v = (torch.randn(1, L, h, d, device="cuda").to(dtype) for h, d in ((4, dk), (K, dk), (K, dv)))
        found.append(launched(lambda: m2_b200.linear_attention(q, k, v, ld)))
        q, k, v = (t.requires_grad_() for t in (q, k, v))

        def gradients():                                    # one graph: the forward pass and, behind it, its gradients
            o = m2_b200.linear_attention(q, k, v, ld)
            torch.autograd.grad(o, [q, k, v], up)

        up = torch.ones(1, L, 4, dv, dtype=dtype, device="cuda")
        found.append(launched(gradients))
    q, state = torch.randn(2, 4, 64, device="cuda"), torch.zeros(2, 4, 64, 64, device="cuda")
    found.append(launched(lambda: m2_b200.linear_attention_step(q, q, q, ld, state)))
    found.append(launched(lambda: m2_b200.linear_attention_step(q[:0], q[:0], q[:0], ld, state[:0])))
    x, w = torch.randn(3, 50, 256, device="cuda", requires_grad=True), torch.ones(256, device="cuda", requires_grad=True)
    gate, up = torch.ones(3, 1, 256, device="cuda", requires_grad=True), torch.ones(3, 50, 256, device="cuda")
    for wanted in ([x], [x, w], [x, gate]):
        fixed = [t if any(t is v for v in wanted) else t.detach() for t in (w, gate)]
        found.append(launched(lambda: torch.autograd.grad(m2_b200.gated_residual_norm(x, x.detach(), gate=fixed[1], after_weight=fixed[0])[0], wanted, up)))
    t, up = torch.zeros(3, 50, dtype=torch.long, device="cuda"), torch.ones(3, 50, device="cuda")
    found.append(launched(lambda: m2_b200.token_logprobs(x.detach(), t, top=3)))
    found.append(launched(lambda: torch.autograd.grad(m2_b200.token_logprobs(x, t)[0], [x], up)))
    assert all(a == b for a, b in found), found
    assert found[0] == (1, 1) and found[2] == (3, 3) and found[5][0] > 9, found


@pytest.mark.parametrize("step", [8, 1])
def test_rows_may_overlap(step):
    """Windows of one tensor, read in place: a row's neighbour begins before it ends."""
    base = torch.randn(2000, device="cuda")
    rows, w = base.unfold(0, 768, step), torch.randn(768, device="cuda")
    apart = rows.contiguous()
    t = torch.arange(len(rows), device="cuda") % 768
    got, ref = (m2_b200.token_logprobs(x, t, top=3) for x in (rows, apart))
    assert torch.equal(got.top_id, ref.top_id)
    for a, b in zip(got[:3], ref[:3]):                      # where a row begins decides which thread adds which values
        assert torch.equal(a, b) if step == 8 else (a - b).abs().max() <= (768 / 256 + 64) * 2.0 ** -24 + 16 * 2.0 ** -24 * (b.abs().max() + 40)
    for gate, after in ((None, w), (rows, w), (rows, None)):
        got = m2_b200.gated_residual_norm(rows, rows, gate=gate, after_weight=after, before_weight=w, eps=1e-5)
        ref = m2_b200.gated_residual_norm(apart, apart, gate=gate if gate is None else apart, after_weight=after, before_weight=w, eps=1e-5)
        for a, b in zip(got, ref):
            assert torch.equal(a, b) if step == 8 else ((a - b).abs() <= 256 * 2.0 ** -24 * b.abs().amax(-1, keepdim=True)).all()
    x = base.clone().requires_grad_()                       # the gradient of a value is the sum over the rows that hold it
    (d,) = torch.autograd.grad(m2_b200.token_logprobs(x.unfold(0, 768, step), t).logprob.sum(), [x])
    y = base.double().requires_grad_()
    (e,) = torch.autograd.grad(torch.log_softmax(y.unfold(0, 768, step), -1).gather(-1, t[:, None]).sum(), [y])
    assert (d.double() - e).abs().max() <= (768 / 256 + 128 + len(rows)) * 2.0 ** -24 * len(rows)


def peak(fn):
    """Bytes that fn() holds beyond what was held before, at most, and what it returns."""
    gc.collect()
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out = fn()
    return torch.cuda.max_memory_allocated() - before, out


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_logits_of_a_batch_are_read_in_place(dtype):
    V = 4096
    x = torch.randn(5, 33, V, device="cuda").to(dtype)
    t = torch.randint(0, V, (5, 32), device="cuda")
    t[2, 3:] = -100
    swapped = torch.randn(32, 5, V, device="cuda").to(dtype).transpose(0, 1)
    layouts = [x[:, :-1], x[:, 1:], swapped, x[:1, :-1].expand(5, 32, V), x.as_strided((5, 32, V), (V, 8, 1)), x[:, None, :-1].expand(5, 1, 32, V),
               x[:, None, :-1, :V // 2 * 2]]
    for y in layouts:
        u = t.view(y.shape[:-1])
        apart = y.contiguous()
        used, got = peak(lambda: m2_b200.token_logprobs(y, u, top=4))
        ref = m2_b200.token_logprobs(apart, u, top=4)
        assert used < apart.numel() * apart.element_size() / 4
        assert all(torch.equal(a, b) for a, b in zip(got, ref))
        y, apart = y.detach().requires_grad_(), apart.requires_grad_()
        ups = [torch.randn_like(a) for a in ref[:3]]
        outs = m2_b200.token_logprobs(y, u, top=4)
        used, (d,) = peak(lambda: torch.autograd.grad(outs[:3], [y], ups))
        (e,) = torch.autograd.grad(m2_b200.token_logprobs(apart, u, top=4)[:3], [apart], ups)
        assert torch.equal(d, e) and used < 1.25 * apart.numel() * apart.element_size()


def test_logits_that_have_to_be_copied_are_copied_once():
    x = torch.randn(3, 2, 8, 2, 2048, device="cuda").transpose(1, 3).requires_grad_()      # (3, 2, 8, 2, V): no two strides
    t = torch.randint(0, 2048, x.shape[:-1], device="cuda")
    out, ref = m2_b200.token_logprobs(x, t, top=2), m2_b200.token_logprobs(x.detach().contiguous(), t, top=2)
    assert all(torch.equal(a, b) for a, b in zip(out, ref))
    used, (d,) = peak(lambda: torch.autograd.grad(out.logprob, [x], torch.ones_like(out.logprob)))
    assert used < 1.5 * x.numel() * 4
    apart = x.detach().contiguous().requires_grad_()
    (e,) = torch.autograd.grad(m2_b200.token_logprobs(apart, t).logprob, [apart], torch.ones_like(out.logprob))
    assert torch.equal(d, e)
    columns = torch.randn(2048, 6, device="cuda").t()
    assert torch.equal(m2_b200.token_logprobs(columns, t[0, 0, :6, 0]).logprob, m2_b200.token_logprobs(columns.contiguous(), t[0, 0, :6, 0]).logprob)


def test_groups_of_rows_far_apart():
    far = 2 ** 31 + 64
    big = torch.empty(far + 3 * 512, dtype=torch.bfloat16, device="cuda")
    y = big.as_strided((2, 3, 512), (far, 512, 1))
    near = torch.randn(2, 3, 512, device="cuda").bfloat16()
    y.copy_(near)
    t = torch.randint(0, 512, (2, 3), device="cuda")
    assert all(torch.equal(a, b) for a, b in zip(m2_b200.token_logprobs(y, t, top=2), m2_b200.token_logprobs(near, t, top=2)))


def test_rows_of_norms_that_have_to_be_copied_are_copied_once():
    x, y, gate = (torch.randn(8, 513, 1024, device="cuda")[:, :-1].requires_grad_() for _ in range(3))
    w, size = torch.randn(1024, device="cuda"), 8 * 512 * 1024 * 4
    up = [torch.randn(8, 512, 1024, device="cuda") for _ in range(2)]
    outs = m2_b200.gated_residual_norm(x, y, gate=gate, after_weight=w, before_weight=w, eps=1e-5)
    used, grads = peak(lambda: torch.autograd.grad(outs, [x, y, gate], up))
    assert used < 4.5 * size                                # three gradients and the blocks' column sums; three copies more are 6.5
    apart = [t.detach().contiguous().requires_grad_() for t in (x, y, gate)]
    refs = m2_b200.gated_residual_norm(apart[0], apart[1], gate=apart[2], after_weight=w, before_weight=w, eps=1e-5)
    assert all(torch.equal(a, b) for a, b in zip(outs, refs))
    assert all(torch.equal(a, b) for a, b in zip(grads, torch.autograd.grad(refs, apart, up)))
    # broadcast over the batch: copied, and the gradient summed
    row = torch.randn(1, 512, 1024, device="cuda", requires_grad=True)
    (d,) = torch.autograd.grad(m2_b200.gated_residual_norm(row.expand(8, 512, 1024), apart[1].detach(), residual_scale=2.0)[0], [row], up[0])
    assert (d - 2 * up[0].sum(0, keepdim=True)).abs().max() <= 8 * 2.0 ** -24 * 2 * up[0].abs().sum(0).max()


@pytest.mark.parametrize("D", [31, 96, 257, 600, 768, 1000, 1280, 1536, 1792, 2056, 4096, 8000])
def test_rows_of_equal_values_are_normalised_to_zero(D):
    """A sum of D values of 8 bits is exact in float32, so their mean is too; at the default eps a mean that is off by a step of
    float32 makes a value of about 0.1 of nothing."""
    c = torch.cat([torch.arange(128, 256, device="cuda") / 128, torch.arange(-255, -127, device="cuda") * 3.0])[:, None]
    c = c.bfloat16().float()
    y = c.expand(-1, D).contiguous()
    w, b = torch.rand(D, device="cuda") + 0.5, torch.randn(D, device="cuda")
    for x in (y, y.bfloat16()):
        r, h = m2_b200.gated_residual_norm(x, torch.zeros_like(x), before_weight=w, before_bias=b)
        assert torch.equal(r, x) and torch.equal(h, b.to(x.dtype).expand_as(h))
        r, h = m2_b200.gated_residual_norm(torch.zeros_like(x), x, after_weight=w, after_bias=b, before_weight=w)
        assert torch.equal(r, b.to(x.dtype).expand_as(r))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("L", [150, 2000])
def test_an_infinity_stays_in_its_channels_and_behind_its_token(L, dtype):
    q, k, v = (torch.randn(1, L, 2, 64, device="cuda").to(dtype) for _ in range(3))
    ld = torch.tensor([-0.01, -0.02], device="cuda")
    o, s = m2_b200.linear_attention(q, k, v, ld, return_state=True)
    bad = k.clone()
    bad[0, 100, 0, 3] = float("inf")
    p, t = m2_b200.linear_attention(q, bad, v, ld, return_state=True)
    assert torch.equal(p[:, :, 1], o[:, :, 1]) and torch.equal(p[:, :100], o[:, :100]) and not torch.isfinite(p[0, 100:, 0]).any()
    assert not torch.isfinite(t[0, 0, 3]).any() and torch.equal(t[0, 1], s[0, 1])
    assert torch.equal(t[0, 0, :3], s[0, 0, :3]) and torch.equal(t[0, 0, 4:], s[0, 0, 4:])
    bad = v.clone()
    bad[0, 100, 0, 3] = float("inf")
    p, t = m2_b200.linear_attention(q, k, bad, ld, return_state=True)
    assert torch.equal(p[:, :, 1], o[:, :, 1]) and torch.equal(p[:, :37], o[:, :37]) and not torch.isfinite(p[0, 100:, 0, 3]).any()
    assert torch.equal(p[..., :3], o[..., :3]) and torch.equal(p[..., 4:], o[..., 4:])
    assert not torch.isfinite(t[0, 0, :, 3]).any() and torch.equal(t[..., :3], s[..., :3]) and torch.equal(t[..., 4:], s[..., 4:])


def test_lengths_are_whole_numbers():
    q, ld = torch.zeros(2, 3, 2, 8, device="cuda"), torch.zeros(2, device="cuda")
    for dtype in (torch.complex64, torch.float32, torch.bool):
        with pytest.raises(ValueError, match="lengths"):
            m2_b200.linear_attention(q, q, q, ld, lengths=torch.ones(2, device="cuda").to(dtype))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [700, 1500, 5000, 30528])
def test_alternatives_of_rows_of_nan(V, dtype):
    """NaN goes before all, by ascending id, however many there are."""
    x = torch.randn(4, V, device="cuda").to(dtype)
    x[0] = float("nan")
    x[1, ::2] = float("nan")
    x[2, 1::2] = float("nan")
    x[3, 0] = float("nan")
    out = m2_b200.token_logprobs(x, torch.zeros(4, dtype=torch.long, device="cuda"), top=32)
    ids = torch.arange(32, device="cuda")
    assert torch.equal(out.top_id[0], ids) and torch.equal(out.top_id[1], 2 * ids) and torch.equal(out.top_id[2], 2 * ids + 1)
    rest = x[3, 1:].float().sort(descending=True, stable=True).indices[:31] + 1
    assert out.top_id[3, 0] == 0 and torch.equal(out.top_id[3, 1:], rest)
    assert torch.isnan(out.top_logprob).all() and torch.isnan(out.logprob).all()


@pytest.mark.parametrize("state", [False, True])
@pytest.mark.parametrize("shape", [(3, 1, 4, 2, 64, 64), (2, 50, 4, 2, 64, 64), (2, 300, 4, 4, 64, 64), (1, 1100, 2, 1, 64, 64), (2, 200, 2, 2, 128, 128), (1, 700, 2, 2, 128, 64),
                                   (1, 130, 2, 1, 80, 40)])
def test_bfloat16_scans_round_to_bfloat16_once(shape, state):
    """Operands of the tensor cores have two parts of 8 bits, the first cut and the second rounded: what is left out is below 2^-7 times
    half a step, 2^-15 of the operand.  A product has up to two such operands (a weight's or the state's, and in gradients a key's in the
    state): 2^-14 of M, what the operator gives for the absolute values; sums as in float32 but up to twice as far off; the output's half
    step once."""
    B, L, H, K, dk, dv = shape
    q, k, v, ld, s0 = make(*shape, torch.bfloat16, seed=L)
    leaves = [t.detach().requires_grad_() for t in ((q, k, v, s0) if state else (q, k, v))]
    o, s = m2_b200.linear_attention(*leaves[:3], ld, initial_state=leaves[3] if state else None, return_state=True)
    g = torch.Generator(device="cuda").manual_seed(7)
    do, ds = torch.randn(o.shape, device="cuda", generator=g).bfloat16(), torch.randn(s.shape, device="cuda", generator=g) * state
    grads = torch.autograd.grad([o, s], leaves, [do, ds])
    runs = []
    for sign in (lambda t: t, torch.abs):
        wide = [sign(t.detach().double()).requires_grad_() for t in leaves]
        out = definition(*wide[:3], ld.double(), dk ** -0.5, wide[3] if state else None, None)
        runs.append([out[0], *torch.autograd.grad(out, wide, [sign(do.double()), sign(ds.double())])[:3]])
    for name, got, ref, M, d in zip(("o", "dq", "dk", "dv"), [o, *grads[:3]], *runs, (dk, dv, dv, dk)):
        within(got, ref, U16 * ref.abs() + (2.0 ** -14 + 2 * (d + 64 + L / 32 + 16 + H // K) * U32) * M, name)
