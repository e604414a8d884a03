"""gated_residual_norm on the GPU against the definition in float64 and its derivatives.

Bounds.  With u the output type's half step (bf16 2^-8, float32 2^-24): |got - ref| <= u |ref| + 128 2^-24 m, m the largest
magnitude in the output's row: statistics are sums of at most 8 + 5 + 32 roundings in a row, and a handful of products follow.
Column sums: the sum of the absolute values of their terms times (rows + 128) 2^-24, and what the terms bring along: all but those of
N_before's parameters are c u with u the gradient of r and c the derivative of r by the parameter.  u is itself a difference of
values as large as the row's largest, so u_j is off by up to 128 2^-24 max |u| however small it is, and so is c_j (a normalised value, say) by 128 2^-24 max |c|: the sum
by |c_j| max |u| + max |c| |u_j| times 128 2^-24.  The same holds for N_before's weight with dh in u's place, which is exact, and r's
normalised values in c's."""
import pytest
import torch

import m2_b200

pytestmark = pytest.mark.gpu
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
NAMES = ("x", "y", "gate", "scale", "w1", "b1", "w2", "b2")


def definition(x, y, gate, scale, w1, b1, w2, b2, eps, rms):
    def norm(t, w, b):
        if w is None:
            return t
        c = t if rms else t - t.mean(-1, keepdim=True)
        n = c / (c.square().mean(-1, keepdim=True) + eps).sqrt() * w
        return n if b is None else n + b

    n = norm(y, w1, b1)
    r = scale * x + (n if gate is None else gate * n)
    return r, (norm(r, w2, b2) if w2 is not None else None)


def make(B, L, D, xt, yt, gate, scale, after, before, bias, seed=0, gate_type=None):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rnd(*shape, mean=0.0, dtype=torch.float32):
        return (torch.randn(shape, device="cuda", generator=g) + mean).to(dtype)

    shape = {"none": None, "channel": (D,), "sequence": (B, 1, D), "token": (B, L, D)}[gate]
    return dict(x=rnd(B, L, D, mean=0.5, dtype=xt) * 2, y=rnd(B, L, D, mean=-1.0, dtype=yt), gate=rnd(*shape, dtype=gate_type or yt) if shape else None,
                scale=rnd(D, mean=1.0) if scale == "channel" else 0.7, w1=rnd(D, mean=1.0) if after else None, b1=rnd(D) if after and bias else None,
                w2=rnd(D, mean=1.0) if before else None, b2=rnd(D) if before and bias else None)


def call(t, eps, rms):
    return m2_b200.gated_residual_norm(t["x"], t["y"], gate=t["gate"], residual_scale=t["scale"], after_weight=t["w1"], after_bias=t["b1"],
                                       before_weight=t["w2"], before_bias=t["b2"], eps=eps, rms=rms)


def near(got, ref, what):
    m = ref.abs().amax(-1, keepdim=True)
    off = (got.double() - ref).abs()
    bound = U[got.dtype] * ref.abs() + 128 * 2.0 ** -24 * m + 1e-30
    assert (off <= bound).all(), f"{what}: {(off / bound).max().item():.2f} of the bound"


CASES = [
    # B, L, D, x, y, gate, scale, after, before, bias, rms
    (1, 1, 1, "f", "f", "token", "channel", True, True, True, False),
    (1, 1, 768, "b", "b", "channel", "number", True, True, False, True),
    (2, 3, 8, "f", "b", "sequence", "channel", True, True, True, False),
    (3, 5, 257, "f", "b", "token", "number", True, True, True, False),
    (2, 130, 768, "f", "b", "sequence", "channel", True, True, True, False),
    (40, 3, 768, "b", "b", "sequence", "number", True, True, False, True),
    (700, 4, 64, "f", "f", "sequence", "channel", True, True, True, False),
    (3000, 5, 16, "f", "b", "sequence", "channel", True, True, True, False),
    (20000, 2, 8, "f", "b", "sequence", "number", True, True, False, True),
    (1, 3000, 40, "f", "b", "sequence", "channel", True, True, True, False),
    (2, 9, 1536, "b", "f", "token", "channel", False, True, True, True),
    (2, 9, 1536, "f", "b", "none", "number", True, False, True, False),
    (4, 50, 96, "b", "b", "none", "number", False, True, True, False),
    (1, 7, 2056, "f", "b", "channel", "channel", True, True, True, False),
    (1, 5, 4096, "f", "b", "token", "channel", True, True, False, True),
    (1, 3, 8192, "b", "b", "channel", "number", True, True, True, False),
    (2, 4, 8191, "f", "f", "token", "channel", True, True, True, False),
    (1, 2500, 31, "b", "f", "token", "channel", True, True, True, True),
    (3, 4, 16, "f", "b", "none", "channel", False, False, False, False),
    (2, 30, 256, "f", "f", "sequence", "channel", True, True, True, False),
    (3, 5, 512, "b", "b", "token", "number", True, True, True, False),
    (1, 9, 1024, "f", "b", "sequence", "number", True, True, False, True),
    (2, 5, 1280, "b", "f", "token", "channel", True, False, True, False),
    (2, 3, 1792, "f", "f", "channel", "channel", False, True, True, False),
    (2, 4, 2048, "f", "f", "token", "channel", True, True, True, False),
    (2, 3, 2560, "f", "b", "sequence", "channel", True, True, True, False),
]


@pytest.mark.parametrize("case", CASES)
def test_forward_and_gradients(case):
    B, L, D, xt, yt, gate, scale, after, before, bias, rms = case
    kind = {"f": torch.float32, "b": torch.bfloat16}
    t = make(B, L, D, kind[xt], kind[yt], gate, scale, after, before, bias, seed=D, gate_type=torch.float32 if D % 2 or D % 512 == 0 else None)
    eps = 1e-5
    names = [n for n in NAMES if isinstance(t[n], torch.Tensor)]
    for n in names:
        t[n].requires_grad_()
    r, h = call(t, eps, rms)
    with torch.no_grad():
        r2, h2 = call(t, eps, rms)
    assert torch.equal(r, r2) and (h is None or torch.equal(h, h2))
    # parameters for each row, so that the terms of their sums are seen
    wide = {n: (t[n].detach().double() if isinstance(t[n], torch.Tensor) else t[n]) for n in NAMES}
    for n in names:
        if n not in ("x", "y"):
            wide[n] = wide[n].expand(B, L, D).contiguous()
        wide[n].requires_grad_()
    rr, rh = definition(*(wide[n] for n in NAMES), eps, rms)
    near(r, rr, "r")
    if before:
        near(h, rh, "h")
    else:
        assert h is None
    dr = torch.randn(r.shape, device="cuda").to(r.dtype)
    outs, ups = [r], [dr]
    routs, rups = [rr], [dr.double()]
    if before:
        dh = torch.randn(h.shape, device="cuda").to(h.dtype)
        outs, ups, routs, rups = outs + [h], ups + [dh], routs + [rh], rups + [dh.double()]
    got = torch.autograd.grad(outs, [t[n] for n in names], ups)
    ref = torch.autograd.grad(routs, [wide[n] for n in names], rups, retain_graph=True)
    (u,) = torch.autograd.grad(routs, [rr], rups, retain_graph=True)
    by = torch.autograd.grad(rr, [wide[n] for n in names], torch.ones_like(rr), allow_unused=True)
    most = lambda v: v.abs().amax(-1, keepdim=True)  # noqa: E731
    hat = definition(rr.detach(), 0 * rr.detach(), None, 1.0, None, None, torch.ones_like(rr), None, eps, rms)[1]
    for n, a, b, c in zip(names, got, ref, by):
        if b.shape == a.shape:
            # where D is 1 or 2 the derivative of a LayerNorm is a difference that leaves only its rounding: measure by the incoming gradient
            m = torch.maximum(b.abs().amax(-1, keepdim=True), 8 * (dr.double().abs() + (dh.double().abs() if before else 0)).amax(-1, keepdim=True))
            bound = U[a.dtype] * b.abs() + 128 * 2.0 ** -24 * m
        else:
            dims = (1,) if t[n].dim() == 3 else (0, 1)
            size = b.abs().sum(dims) + (1e-3 if D <= 2 else 0)
            own = (c.abs() * most(u) + most(c) * u.abs()).sum(dims) if c is not None else (most(hat) * dh.double().abs()).sum(dims)
            b = b.sum(dims)
            a = a.reshape(b.shape)
            bound = U[a.dtype] * b.abs() + 2.0 ** -24 * ((B * L + 128) * size + 128 * own)
        off = (a.double() - b).abs()
        assert (off <= bound + 1e-30).all(), f"d {n}: {(off / (bound + 1e-30)).max().item():.2f} of the bound"


def test_only_one_of_the_outputs_is_used():
    t = make(2, 6, 64, torch.float32, torch.bfloat16, "token", "channel", True, True, True)
    wide = {n: v.double().requires_grad_() if isinstance(v, torch.Tensor) else v for n, v in t.items()}
    for n in NAMES:
        t[n].requires_grad_()
    for pick in (0, 1):
        out, ref = call(t, 1e-5, False)[pick], definition(*(wide[n] for n in NAMES), 1e-5, False)[pick]
        w = torch.randn_like(out)
        got = torch.autograd.grad(out, [t["x"], t["y"]], w)
        for a, b in zip(got, torch.autograd.grad(ref, [wide["x"], wide["y"]], w.double())):
            near(a, b, f"output {pick}")
    (gw,) = torch.autograd.grad(call(t, 1e-5, False)[0], [t["w2"]], torch.ones(2, 6, 64, device="cuda"), allow_unused=True)
    assert gw is None or not gw.any()


@pytest.mark.parametrize("layout", ["rows apart", "odd offset", "columns apart", "expanded"])
def test_layouts(layout):
    t = make(4, 6, 64, torch.float32, torch.bfloat16, "token", "number", True, True, True)
    if layout == "expanded":
        t["x"], t["y"] = (v[:1, :1].expand(4, 6, 64) for v in (t["x"], t["y"]))
    ref = call({n: v.contiguous() if isinstance(v, torch.Tensor) else v for n, v in t.items()}, 1e-5, False)
    for n in ("x", "y", "gate"):
        if layout == "rows apart":
            t[n] = torch.cat([t[n], t[n]], -1)[..., :64]
        elif layout == "odd offset":
            t[n] = torch.cat([t[n].reshape(-1)[:1], t[n].reshape(-1)])[1:].view(4, 6, 64)
        elif layout == "columns apart":
            t[n] = t[n].transpose(1, 2).contiguous().transpose(1, 2)
    got = call(t, 1e-5, False)
    assert torch.equal(ref[0], got[0]) and torch.equal(ref[1], got[1])


def test_gradient_against_differences():
    """Central differences along random directions, in steps of 2^-7: their own error is of the order of 2^-14 and the rounding's."""
    t = make(2, 5, 96, torch.float32, torch.float32, "sequence", "channel", True, True, True)
    for n in NAMES:
        t[n] = t[n].clone().requires_grad_()
    w = [torch.randn(2, 5, 96, device="cuda") for _ in range(2)]
    grads = torch.autograd.grad(list(call(t, 1e-3, False)), [t[n] for n in NAMES], w)
    e = 2.0 ** -7
    for n, g in zip(NAMES, grads):
        d = torch.randn_like(t[n])
        with torch.no_grad():
            f = [sum((o.double() * c.double()).sum() for o, c in zip(call(dict(t, **{n: t[n] + s * e * d}), 1e-3, False), w)) for s in (1, -1)]
        diff, ours = (f[0] - f[1]) / (2 * e), (g.double() * d.double()).sum()
        assert abs(diff - ours) <= 2e-3 * (g.double().norm() * d.double().norm()), n


def test_constant_rows_and_types_of_parameters():
    x = torch.zeros(3, 32, device="cuda")
    w = torch.ones(32, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    r, h = m2_b200.gated_residual_norm(x, x + 3, after_weight=w, before_weight=w)
    assert not r.any() and not h.any()
    r, h = m2_b200.gated_residual_norm(x, x, after_weight=w, before_weight=w, rms=True)
    assert not r.any() and not h.any()
    (g,) = torch.autograd.grad(h.sum(), [w])
    assert g.dtype == torch.bfloat16 and torch.isfinite(g).all()


def test_refusals_on_the_device():
    x = torch.zeros(2, 3, 16, device="cuda")
    for kw in (dict(gate=x[:, :2]), dict(gate=torch.zeros(2, 16, device="cuda")), dict(after_bias=x[0, 0]), dict(before_weight=x[0]), dict(eps=-1.0),
               dict(residual_scale=torch.ones(3, device="cuda")), dict(after_weight=torch.ones(16))):
        with pytest.raises(ValueError):
            m2_b200.gated_residual_norm(x, x, **kw)
    with pytest.raises(TypeError):
        m2_b200.gated_residual_norm(x.half(), x.half())
    with pytest.raises(RuntimeError, match="up to 8192"):
        m2_b200.gated_residual_norm(torch.zeros(1, 8193, device="cuda"), torch.zeros(1, 8193, device="cuda"))


def test_empty():
    x = torch.zeros(2, 0, 16, device="cuda", requires_grad=True)
    w = torch.ones(16, device="cuda", requires_grad=True)
    r, h = m2_b200.gated_residual_norm(x, x, before_weight=w)
    assert r.shape == h.shape == x.shape
    gx, gw = torch.autograd.grad([r, h], [x, w], [torch.zeros_like(r), torch.zeros_like(h)])
    assert gx.shape == x.shape and not gw.any()


def test_same_bits_twice_on_another_stream_and_in_a_graph():
    t = make(5, 100, 768, torch.float32, torch.bfloat16, "sequence", "channel", True, True, True)
    for n in NAMES:
        t[n] = t[n].clone().requires_grad_()

    def run():
        r, h = call(t, 1e-5, False)
        return [r.detach(), h.detach(), *torch.autograd.grad([r, h], [t[n] for n in NAMES], [torch.ones_like(r), torch.ones_like(h)])]

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
        for n in NAMES:
            t[n].mul_(0.5)
    graph.replay()
    second.replay()
    graph.replay()
    assert all(torch.equal(x, y) and torch.equal(x, z) for x, y, z in zip(run(), a, b))
