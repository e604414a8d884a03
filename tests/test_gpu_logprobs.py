"""token_logprobs on the GPU against float64.

Bounds: a logit's distance to the maximum and the log of the sum are each rounded once or twice, the sum of V positive terms runs
through at most V / 256 + 40 additions in a row and an exponential is within 2^-22 of its value: log probabilities and entropies are
within (V / 256 + 64) 2^-24 + 8 2^-24 (|value| + |largest distance used|) of the definition; a gradient has in addition its type's
half step."""
import pytest
import torch

import m2_b200
from m2_b200 import ops

pytestmark = pytest.mark.gpu
INF = float("inf")
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def definition(x, t, top, ignore=-100):
    x = x.double()
    used = t != ignore
    lp = torch.log_softmax(x, -1)
    none = (x == -INF).all(-1)
    lp = torch.where(none[..., None], -INF, lp)
    p = lp.exp()
    H = -torch.where(p > 0, p * lp.clamp(min=-1e300), 0.0).sum(-1)
    H = torch.where(torch.isnan(lp).any(-1), torch.nan, H)
    got = lp.gather(-1, torch.where(used, t, 0)[..., None])[..., 0]
    ids = x.sort(dim=-1, descending=True, stable=True).indices[..., :top]
    best = lp.gather(-1, ids)
    return (torch.where(used, got, 0.0), torch.where(used, H, 0.0), torch.where(used[..., None], best, 0.0), torch.where(used[..., None], ids, -1))


def gradient(x, t, ids, g_lp, g_h, g_top, ignore=-100):
    x = x.double()
    used = (t != ignore)[..., None]
    lp = torch.log_softmax(x, -1)
    p = lp.exp()
    H = -torch.where(p > 0, p * lp, 0.0).sum(-1, keepdim=True)
    d = -p * (g_lp[..., None] + g_top.sum(-1, keepdim=True)) - torch.where(p > 0, g_h[..., None] * p * (lp + H), 0.0)
    d = d.scatter_add(-1, torch.where(used, t[..., None], 0), g_lp[..., None].double())
    d = d.scatter_add(-1, ids.clamp(min=0), g_top.double())
    return torch.where(used & ~(x == -INF).all(-1, keepdim=True), d, 0.0)


def close(got, ref, V, what):
    assert got.dtype == torch.float32
    fine = torch.isfinite(ref)
    assert torch.equal(torch.isnan(got), torch.isnan(ref)) and torch.equal(got[~fine & ~torch.isnan(ref)].double(), ref[~fine & ~torch.isnan(ref)]), what
    off = (got[fine].double() - ref[fine]).abs()
    bound = (V / 256 + 64) * 2.0 ** -24 + 8 * 2.0 ** -24 * (ref[fine].abs() + 40)
    assert (off <= bound).all(), f"{what}: {(off / bound).max().item():.2f} of the bound"


def logits(N, V, dtype, seed=0, spread=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(N, V, device="cuda", generator=g) * spread).to(dtype), torch.randint(0, V, (N,), device="cuda", generator=g)


def check(x, t, top):
    out = m2_b200.token_logprobs(x, t, top=top)
    ref = definition(x, t, top)
    V = x.shape[-1]
    for name, a, b in zip(("logprob", "entropy", "top_logprob"), out[:3], ref[:3]):
        close(a, b, V, name)
    assert torch.equal(out.top_id, ref[3])
    return out


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,V,top", [(1, 1, 1), (3, 2, 2), (1, 7, 7), (5, 33, 32), (2, 63, 20), (7, 1000, 5), (300, 501, 3), (1, 30528, 20), (2, 30522, 32),
                                     (3, 30528, 0), (1, 131072, 20), (400, 8191, 1), (1, 262147, 32), (2, 5, 0)])
def test_values(N, V, top, dtype):
    x, t = logits(N, V, dtype, seed=V)
    check(x, t, top)
    check(x, t.int(), top)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,V,top", [(1, 1, 1), (3, 2, 2), (5, 33, 32), (7, 1000, 5), (2, 30528, 20), (300, 501, 0), (1, 70001, 3)])
def test_gradients(N, V, top, dtype):
    x, t = logits(N, V, dtype, seed=V + 1)
    x.requires_grad_()
    out = m2_b200.token_logprobs(x, t, top=top)
    g_lp, g_h, g_top = torch.randn(N, device="cuda"), torch.randn(N, device="cuda"), torch.randn(N, top, device="cuda")
    (d,) = torch.autograd.grad(out[:3], [x], [g_lp, g_h, g_top])
    ref = gradient(x.detach(), t, out.top_id, g_lp, g_h, g_top)
    size = g_lp.abs() + g_top.abs().sum(-1) + g_h.abs() * 32
    bound = U[dtype] * ref.abs() + (V / 256 + 128) * 2.0 ** -24 * size.double()[:, None]
    assert ((d.double() - ref).abs() <= bound).all()
    for pick, g in ((0, g_lp), (1, g_h)):                                   # one of the outputs alone
        (d,) = torch.autograd.grad(m2_b200.token_logprobs(x, t, top=top)[pick], [x], g)
        none = torch.zeros_like(g_lp)
        ref = gradient(x.detach(), t, out.top_id, g_lp if pick == 0 else none, g_h if pick else none, torch.zeros_like(g_top))
        assert ((d.double() - ref).abs() <= U[dtype] * ref.abs() + (V / 256 + 128) * 2.0 ** -24 * size.double()[:, None]).all()


def test_gradient_against_differences():
    x, t = logits(4, 300, torch.float32)
    x.requires_grad_()
    w = [torch.randn(4, device="cuda"), torch.randn(4, device="cuda"), torch.randn(4, 5, device="cuda")]
    (g,) = torch.autograd.grad(m2_b200.token_logprobs(x, t, top=5)[:3], [x], w)
    d, e = torch.randn_like(x), 2.0 ** -8
    with torch.no_grad():
        f = [sum((o.double() * c.double()).sum() for o, c in zip(m2_b200.token_logprobs(x + s * e * d, t, top=5)[:3], w)) for s in (1, -1)]
    assert abs((f[0] - f[1]) / (2 * e) - (g.double() * d.double()).sum()) <= 2e-3 * g.double().norm() * d.double().norm()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_equal_logits_go_by_id(dtype):
    for V in (40, 3000, 30528):
        x = torch.zeros(3, V, dtype=dtype, device="cuda")
        x[1] = -0.0
        x[1, ::2] = 0.0
        x[2, ::3] = 1.0
        check(x, torch.tensor([0, 1, V - 1], device="cuda"), 20)
        x = torch.randint(-4, 3, (6, V), device="cuda").to(dtype)
        check(x, torch.arange(6, device="cuda"), 32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [50, 30528])
def test_masked_infinite_and_nan_logits(dtype, V):
    x, t = logits(9, V, dtype)
    t[:] = 7
    lowest = torch.finfo(dtype).min
    x[0, :] = -INF                       # nothing left
    x[1, :] = -INF
    x[1, 7] = 2.0                        # one token left
    x[2, :] = lowest                     # masked with the type's lowest value: all equal
    x[3, ::2] = lowest
    x[4, ::2] = -INF
    x[5, 11] = float("nan")
    x[6, 12] = INF
    x[7, 12] = x[7, 13] = torch.finfo(dtype).max
    x[8, :] = -INF
    x[8, [3, 9]] = 1.0                   # fewer tokens than alternatives
    out = check(x, t, 10)
    assert out.top_id[5, 0] == 11 and out.top_id[6, 0] == 12 and out.logprob[0] == -INF and out.entropy[0] == 0 and out.logprob[1] == 0
    fine = [0, 1, 2, 3, 4, 8]
    x = x[fine].clone().requires_grad_()
    out = m2_b200.token_logprobs(x, t[fine], top=10)
    g = [torch.ones_like(v) for v in out[:3]]
    (d,) = torch.autograd.grad(out[:3], [x], g)
    assert torch.isfinite(d).all() and not d[0].any()
    ref = gradient(x.detach(), t[fine], out.top_id, *g)
    assert ((d.double() - ref).abs() <= U[dtype] * ref.abs() + 300 * 2.0 ** -24 * 50)[[1, 2, 3, 4, 5]].all()


def test_ignored_rows_are_not_read():
    x, t = logits(6, 999, torch.bfloat16)
    t[[1, 4]] = -100
    x[1], x[4] = float("nan"), INF
    x.requires_grad_()
    out = m2_b200.token_logprobs(x, t, top=3)
    assert not out.logprob[[1, 4]].any() and not out.entropy[[1, 4]].any() and not out.top_logprob[[1, 4]].any() and (out.top_id[[1, 4]] == -1).all()
    (d,) = torch.autograd.grad(out[:3], [x], [torch.ones_like(v) for v in out[:3]])
    assert torch.isfinite(d).all() and not d[[1, 4]].any() and d[0].any()
    t[:] = 5
    out = m2_b200.token_logprobs(x.detach(), t, ignore_index=5)
    assert not out.logprob.any()


def test_targets_outside_the_vocabulary():
    assert ops.device_status() == 0
    x, t = logits(3, 50, torch.float32)
    t[0], t[2] = 50, -1
    x.requires_grad_()
    out = m2_b200.token_logprobs(x, t, top=2)
    assert torch.isnan(out.logprob[[0, 2]]).all() and torch.isfinite(out.logprob[1]) and torch.isfinite(out.entropy).all()
    assert ops.device_status() == ops.DEV_BAD_INDEX
    (d,) = torch.autograd.grad(out.logprob[1] + out.entropy.sum(), [x])
    assert torch.isfinite(d).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layouts(dtype):
    x, t = logits(6, 517, dtype)
    ref = m2_b200.token_logprobs(x, t, top=4)
    apart = torch.cat([x, x], -1)[:, :517]
    odd = torch.cat([x.reshape(-1)[:1], x.reshape(-1)])[1:].view(6, 517)
    columns = x.t().contiguous().t()
    for y in (apart, odd, columns, x.view(2, 3, 517)):
        out = m2_b200.token_logprobs(y, t.view(y.shape[:-1]), top=4)
        for name, a, b in zip(ref._fields, out, ref):
            assert a.shape[:y.dim() - 1] == y.shape[:-1]
            if name == "top_id":
                assert torch.equal(a.view(b.shape), b)
            else:
                close(a.view(b.shape), b.double(), 2 * 517, name)
        z = y.detach().requires_grad_()
        (d,) = torch.autograd.grad(m2_b200.token_logprobs(z, t.view(y.shape[:-1])).logprob.sum(), [z])
        assert d.shape == y.shape
    one = m2_b200.token_logprobs(x[0], t[0], top=4)
    assert one.logprob.shape == () and torch.equal(one.top_id, ref.top_id[0])
    row = x[:1].expand(6, 517)
    assert torch.equal(m2_b200.token_logprobs(row, t[:1].expand(6)).logprob, ref.logprob[:1].expand(6))


def test_refusals_on_the_device():
    x, t = logits(2, 40, torch.float32)
    for top in (-1, 33, 41):
        with pytest.raises(ValueError):
            m2_b200.token_logprobs(x, t, top=top)
    with pytest.raises(ValueError):
        m2_b200.token_logprobs(x[:, :0], t)


def test_empty():
    x, t = logits(0, 40, torch.float32)
    x.requires_grad_()
    out = m2_b200.token_logprobs(x, t, top=3)
    assert out.top_id.shape == (0, 3)
    (d,) = torch.autograd.grad(out.logprob.sum(), [x])
    assert d.shape == (0, 40)


def test_same_bits_twice_on_another_stream_and_in_a_graph():
    x, t = logits(5, 30528, torch.bfloat16)
    x.requires_grad_()

    def run():
        out = m2_b200.token_logprobs(x, t, top=20)
        return [*(v.detach() for v in out), *torch.autograd.grad(out[:3], [x], [torch.ones_like(v) for v in out[:3]])]

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
        x.mul_(0.5)
    graph.replay()
    second.replay()
    graph.replay()
    assert all(torch.equal(p, q) and torch.equal(p, r) for p, q, r in zip(run(), a, b))
