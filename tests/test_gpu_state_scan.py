"""selective_scan and selective_scan_step against their definition in 64 bits, token by token.

Bounds.  Every value is a sum of products, so its error is counted against M, the same sum of absolute values.  A decay exp(s a) carries 2^-22 (the exp)
and half a step of its exponent; over an age of T = sum |s a| that is 2^-22 for each of up to L tokens, and T times the relative error of s a, which is
below 2^-19 (softplus of |v| < 10: an exp of v with 2^-22 + 2 |v| 2^-24, a quotient, a polynomial).  T exp(-T) and exp(-T) are below 1.22 exp(-T / 2), so M takes half
of every exponent.  Sums add one 2^-24 for each of their terms; an output is rounded once to its type."""
import pytest
import torch

import m2_b200
from m2_b200 import ops
from tests.test_gpu_linear_attention import U16, U32, within

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def seeded():
    torch.manual_seed(0)


SHAPES = [  # B, L, D, N, G: one of each; odd sizes; groups whose channels fill no tile; 8 and 16 states a lane; a long axis with few channels (cut into segments)
    (1, 1, 1, 1, 1), (2, 33, 64, 16, 1), (3, 70, 100, 11, 4), (2, 64, 24, 8, 3), (2, 129, 130, 16, 2), (2, 100, 40, 20, 1), (2, 77, 66, 33, 2), (1, 40, 8, 64, 1),
    (1, 700, 72, 16, 1), (2, 515, 136, 5, 2), (1, 530, 20, 30, 1), (1, 300, 20, 50, 1)]


def make(B, L, D, N, G, dtype, seed=0, gate=True, plain=False):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rnd(*s, std=1.0, mean=0.0):
        return torch.randn(s, device="cuda", generator=g) * std + mean

    t = dict(x=rnd(B, L, D).to(dtype), delta=rnd(B, L, D, std=0.5).to(dtype), a=-torch.exp(rnd(D, N)), b=rnd(B, L, G, N).to(dtype), c=rnd(B, L, G, N).to(dtype))
    if plain:
        t["delta"] = (rnd(B, L, D).abs() * 0.1).to(dtype)
        return t
    t.update(skip=rnd(D), delta_bias=rnd(D, mean=-3.0), initial_state=rnd(B, D, N))
    if gate:
        t["gate"] = rnd(B, L, D).to(dtype)
    return t


def definition(t, softplus, lengths, d_y=None, d_state=None, size=False):
    """y and the state and, with d_y, all gradients; size: of absolute values, with half the decays' exponents, and what the sums of a tile may lose."""
    f = (lambda v: v.double().abs()) if size else (lambda v: v.double())
    x, a = f(t["x"]), f(t["a"])
    (B, L, D), N, G = x.shape, a.shape[1], t["b"].shape[2]
    n = lengths if lengths is not None else torch.full((B,), L, device=x.device)
    live = (torch.arange(L, device=x.device) < n[:, None])[..., None]
    v = t["delta"].double() + (t["delta_bias"].double() if "delta_bias" in t else 0.0)
    s = torch.where(live, torch.nn.functional.softplus(v) if softplus else v, 0.0)
    slope = torch.sigmoid(v) if softplus else torch.ones_like(v)
    decay = torch.exp(s[..., None] * t["a"].double() * (0.5 if size else 1.0))
    s = s.abs() if size else s
    grp = torch.arange(D, device=x.device) // (D // G)
    b, c = f(t["b"])[:, :, grp], f(t["c"])[:, :, grp]
    z = t["gate"].double() if "gate" in t else None
    sig = torch.sigmoid(z) if z is not None else None
    silu = f(z * sig) if z is not None else torch.ones_like(x)
    skip = f(t["skip"]) if "skip" in t else torch.zeros(D, dtype=torch.float64, device=x.device)
    h = f(t["initial_state"]) if "initial_state" in t else torch.zeros((B, D, N), dtype=torch.float64, device=x.device)
    before, hs = [], []
    x = torch.where(live, x, 0.0)
    for i in range(L):
        before.append(h)
        h = decay[:, i] * h + (s[:, i] * x[:, i])[..., None] * torch.where(live[:, i, :, None], b[:, i], 0.0)
        hs.append(h)
    out = dict(state=h)
    hs, before = (torch.stack(q, 1) if L else x.new_zeros((B, 0, D, N)) for q in (hs, before))
    raw = (hs * c).sum(-1) + skip * x
    out["y"] = torch.where(live, raw * silu, 0.0)
    if d_y is None:
        return out
    d_y = torch.where(live, f(d_y), 0.0)
    e = d_y * silu
    g = f(d_state) if d_state is not None else torch.zeros_like(h)
    gs, ws = [], []
    for i in reversed(range(L)):
        g = g + e[:, i, :, None] * c[:, i]
        gs.append(g)
        g = g * decay[:, i]
        ws.append(g * before[:, i])
    gs, ws = (torch.stack(q[::-1], 1) if L else hs for q in (gs, ws))
    gb = (gs * b).sum(-1)
    lost = 0.0
    if size:                             # sums along a tile: |a| v e and |a| g b s x of its 32 tokens
        r = ((hs * c * e[..., None] + gs * b * (s * x)[..., None]) * a).sum(-1)
        r = torch.nn.functional.pad(r, (0, 0, 0, -L % 32)).unflatten(1, (-1, 32)).sum(2, keepdim=True).expand(-1, -1, 32, -1).flatten(1, 2)[:, :L]
        lost = 32 * r
    d_s = (ws * a).sum(-1) + gb * x
    d_v = torch.where(live, d_s * slope, 0.0)
    out.update(x=torch.where(live, gb * s + skip * e, 0.0), delta=d_v, a=(ws * s[..., None]).sum((0, 1)), skip=(e * x).sum((0, 1)), delta_bias=d_v.sum((0, 1)),
               initial_state=g, lost=torch.where(live, lost * slope, 0.0) if size else None)
    out["b"] = (gs * (s * x)[..., None]).unflatten(2, (G, D // G)).sum(3)
    out["c"] = (hs * e[..., None]).unflatten(2, (G, D // G)).sum(3)
    if z is not None:
        # silu' = sig + z sig (1 - sig) is 0 near z = -1.28 by cancellation: its error is counted against the sum of its two terms' sizes, as every sum's is
        out["gate"] = d_y * raw * sig * (1 + (z.abs() if size else z) * (1 - sig))
    return out


def eps(L, N):
    return 2.0 ** -18 + L * (2.0 ** -22 + 2 * U32) + (N + 40) * U32


def rounding(dtype):
    return U16 if dtype == torch.bfloat16 else U32


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("how", ["all", "ragged", "plain"])
def test_whole_sequences_and_gradients(shape, dtype, how):
    B, L, D, N, G = shape
    t = make(*shape, dtype, seed=L, gate=how != "ragged", plain=how == "plain")
    softplus = how != "plain"
    lengths = torch.randint(0, L + 1, (B,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(L)) if how == "ragged" else None
    leaves = {k: v.clone().requires_grad_() for k, v in t.items()}
    y, state = m2_b200.selective_scan(**leaves, softplus=softplus, lengths=lengths, return_state=True)
    with torch.no_grad():
        y2, state2 = m2_b200.selective_scan(**t, softplus=softplus, lengths=lengths, return_state=True)
    assert torch.equal(y, y2) and torch.equal(state, state2)
    g = torch.Generator(device="cuda").manual_seed(7)
    d_y, d_state = torch.randn(y.shape, device="cuda", generator=g).to(dtype), torch.randn(state.shape, device="cuda", generator=g)
    grads = dict(zip(leaves, torch.autograd.grad([y, state], list(leaves.values()), [d_y, d_state])))
    ref, M = (definition(t, softplus, lengths, d_y, d_state, size) for size in (False, True))
    one = eps(L, N)
    within(y, ref["y"], rounding(dtype) * ref["y"].abs() + 2 * one * M["y"], "y")
    within(state, ref["state"], U32 * ref["state"].abs() + one * M["state"], "state")
    for k in leaves:
        assert grads[k].dtype == leaves[k].dtype and grads[k].shape == leaves[k].shape
        kind = rounding(dtype) if k in ("x", "delta", "b", "c", "gate") else U32
        terms = {"b": D // G, "c": D // G, "a": B * L, "skip": B * L, "delta_bias": B * L}.get(k, 0)
        extra = {"delta": U32 * M["lost"], "delta_bias": U32 * M["lost"].sum((0, 1))}.get(k, 0.0)
        within(grads[k], ref[k], kind * ref[k].abs() + (3 * one + terms * U32) * M[k] + extra, k)


def test_the_definition_is_differentiated_rightly():
    """The formulas above against torch's derivative of the loop, in 64 bits."""
    t = {k: v.double() for k, v in make(2, 9, 6, 5, 2, torch.float32).items()}
    leaves = {k: v.clone().requires_grad_() for k, v in t.items()}
    out = definition(leaves, True, torch.tensor([9, 4], device="cuda"))
    d_y, d_state = torch.randn_like(out["y"]), torch.randn_like(out["state"])
    auto = torch.autograd.grad([out["y"], out["state"]], list(leaves.values()), [d_y, d_state])
    with torch.no_grad():
        ref = definition(t, True, torch.tensor([9, 4], device="cuda"), d_y, d_state)
    for k, v in zip(leaves, auto):
        assert (v - ref[k]).abs().max() <= 1e-12 * ref[k].abs().max().clamp(min=1)


def test_gradients_against_differences():
    """Along random directions: differences of the definition in 64 bits, steps of 1e-4 (error below 1e-6 of the sum of sizes)."""
    t = make(2, 50, 20, 16, 2, torch.float32, seed=5)
    leaves = {k: v.clone().requires_grad_() for k, v in t.items()}
    y = m2_b200.selective_scan(**leaves, softplus=True)
    w = torch.randn_like(y)
    grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), w)))
    for k in t:
        way = torch.randn_like(t[k]).double()
        vals = []
        for step in (1e-4, -1e-4):
            u = {n: v.double() for n, v in t.items()}
            u[k] = u[k] + step * way
            vals.append((definition(u, True, None)["y"] * w.double()).sum())
        diff, got = (vals[0] - vals[1]) / 2e-4, (grads[k].double() * way).sum()
        assert abs(diff - got) <= 1e-4 * (grads[k].double() * way).norm() + 1e-5


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,D,N,G", [(1, 1, 1, 1), (3, 100, 16, 4), (2, 65, 11, 1), (5, 24, 64, 3), (2, 768, 16, 1), (2, 6, 6, 2)])
def test_single_tokens(B, D, N, G, dtype):
    t = make(B, 1, D, N, G, dtype, seed=D)
    state = t.pop("initial_state")
    ref = definition({**t, "initial_state": state}, True, None)
    M = definition({**t, "initial_state": state}, True, None, size=True)
    one = {k: v[:, 0] if k in ("x", "delta", "b", "c", "gate") else v for k, v in t.items()}
    wide = torch.zeros(B, D * N + 3, device="cuda")          # states a distance apart, not on 16 bytes
    far = wide[:, 1:1 + D * N].unflatten(1, (D, N))
    for own in (state.clone(), far):
        own.copy_(state)
        version = own._version
        y = m2_b200.selective_scan_step(state=own, softplus=True, **one)
        assert own._version > version
        within(y, ref["y"][:, 0], rounding(dtype) * ref["y"][:, 0].abs() + 2 * eps(1, N) * M["y"][:, 0], "y")
        within(own, ref["state"], U32 * ref["state"].abs() + eps(1, N) * M["state"], "state")
    assert not wide[:, 0].any() and not wide[:, 1 + D * N:].any()


def test_b_and_c_of_one_group_may_have_no_group_dimension():
    t = make(2, 20, 12, 8, 1, torch.float32)
    flat = {**t, "b": t["b"][:, :, 0], "c": t["c"][:, :, 0]}
    p, q = (m2_b200.selective_scan(**u) for u in (t, flat))    # steps are negative here and states overflow: bits are compared
    assert torch.equal(p.view(torch.int32), q.view(torch.int32))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 65, 192])
def test_strides_and_alignment(D, dtype):
    """Slices of projections, rows off 16 bytes, channels apart, expanded rows: the same bits as packed tensors."""
    B, L, N = 2, 45, 16
    t = make(B, L, D, N, 1, dtype, seed=3)
    lengths = torch.tensor([45, 17], device="cuda")
    g = torch.randn(B, L, D, device="cuda").to(dtype)

    def run(t, g):
        leaves = {k: v.detach().requires_grad_() for k, v in t.items()}
        y, s = m2_b200.selective_scan(**leaves, softplus=True, lengths=lengths, return_state=True)
        return [y, s, *torch.autograd.grad(y, list(leaves.values()), g)]

    ref = run(t, g)
    for off in (0, 1, 3, 8):
        wide = torch.zeros(B, L, 3 * D + 2 * N + off, dtype=dtype, device="cuda")
        cut = [off, off + D, off + 2 * D, off + 3 * D, off + 3 * D + N]
        views = dict(x=wide[..., cut[0]:cut[1]], delta=wide[..., cut[1]:cut[2]], gate=wide[..., cut[2]:cut[3]],
                     b=wide[..., cut[3]:cut[4]].unsqueeze(2), c=wide[..., cut[4]:].unsqueeze(2))
        for k, v in views.items():
            v.copy_(t[k])
        assert all(torch.equal(p, q) for p, q in zip(run({**t, **views}, g), ref))
    apart = {k: torch.stack([t[k], torch.zeros_like(t[k])], -1)[..., 0] for k in ("x", "delta", "gate", "b", "c")}
    assert all(torch.equal(p, q) for p, q in zip(run({**t, **apart}, torch.stack([g, g], -1)[..., 0]), ref))
    turned = {k: t[k].transpose(0, 1).contiguous().transpose(0, 1) for k in ("x", "delta", "gate", "b", "c")}
    assert all(torch.equal(p, q) for p, q in zip(run({**t, **turned}, g.transpose(0, 1).contiguous().transpose(0, 1)), ref))
    row = t["x"][:1, :1].contiguous()
    same = {**t, "x": row.expand(B, L, D)}
    copied = {**t, "x": row.expand(B, L, D).contiguous()}
    assert torch.equal(m2_b200.selective_scan(**same, softplus=True), m2_b200.selective_scan(**copied, softplus=True))


def test_what_lies_behind_a_text_is_not_read():
    B, L, D, N = 3, 100, 64, 16
    t = make(B, L, D, N, 1, torch.float32)
    lengths = torch.tensor([0, 31, 100], device="cuda")
    g = torch.randn(B, L, D, device="cuda")
    dead = torch.arange(L, device="cuda") >= lengths[:, None]

    def run(t, g):
        leaves = {k: v.detach().requires_grad_() for k, v in t.items()}
        y, s = m2_b200.selective_scan(**leaves, softplus=True, lengths=lengths, return_state=True)
        return [y, s, *torch.autograd.grad([y, s], list(leaves.values()), [g, torch.ones_like(s)])]

    ref = run(t, g)
    bad = {k: v.clone() for k, v in t.items()}
    for k in ("x", "delta", "gate", "b", "c"):
        bad[k][dead] = float("nan")
    up = g.clone()
    up[dead] = float("nan")
    got = run(bad, up)
    assert all(torch.equal(p, q) for p, q in zip(got, ref)) and not ref[0][dead].any()
    for i in (2, 3, 5, 6, 10):                                # x, delta, b, c, gate
        assert not ref[i][dead].any()
    assert torch.equal(ref[1][0], t["initial_state"][0])
    # lengths out of range are cut
    out = m2_b200.selective_scan(**t, softplus=True, lengths=torch.tensor([-5, 31, 10 ** 9], device="cuda"))
    assert torch.equal(out, ref[0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("L", [60, 700])
def test_nan_and_infinity_stay_in_their_channel_and_behind_their_token(L, dtype):
    t = make(1, L, 70, 16, 1, dtype)
    y, s = m2_b200.selective_scan(**t, softplus=True, return_state=True)
    for what, value in (("x", float("inf")), ("x", float("nan")), ("delta", float("nan"))):
        bad = {k: v.clone() for k, v in t.items()}
        bad[what][0, 37, 5] = value
        p, q = m2_b200.selective_scan(**bad, softplus=True, return_state=True)
        others = [i for i in range(70) if i != 5]
        assert torch.equal(p[..., others], y[..., others]) and torch.equal(p[:, :37], y[:, :37]) and torch.equal(q[:, others], s[:, others])
        assert not torch.isfinite(p[0, 37, 5]) and not torch.isfinite(q[0, 5]).all()


def test_states_that_do_not_fade_and_fade_at_once():
    """a = 0 sums; a = -1e30 forgets: h is the token's own."""
    t = make(2, 90, 32, 4, 1, torch.float32, plain=True)
    t["a"] = torch.tensor([0.0, -1e30, 0.0, -1e30], device="cuda").expand(32, 4).contiguous()
    t["delta"] = t["delta"] + 0.01
    _, s = m2_b200.selective_scan(**t, return_state=True)
    fed = (t["delta"] * t["x"]).double()[..., None] * t["b"].double()
    sums = fed.sum(1)
    assert (s[..., 0::2] - sums[..., 0::2]).abs().max() <= 90 * U32 * fed.abs().sum(1).max()
    assert torch.equal(s[..., 1::2], ((t["delta"] * t["x"])[..., None] * t["b"])[:, -1][..., 1::2])


@pytest.mark.parametrize("L", [100, 700])
def test_an_empty_state_that_would_grow_stays_empty(L):
    """Factors of e^20 a token: what is never fed is zero, not infinity times zero, forwards and back."""
    t = make(1, L, 64, 4, 1, torch.float32, plain=True)
    t["a"] = torch.tensor([20.0, -1.0, 20.0, -1.0], device="cuda").expand(64, 4).contiguous()
    t["delta"] = torch.ones_like(t["delta"])
    t["b"][..., ::2] = 0
    t["c"][..., ::2] = 0
    leaves = {k: v.clone().requires_grad_() for k, v in t.items()}
    y, s = m2_b200.selective_scan(**leaves, return_state=True)
    fading = {**t, "a": t["a"][:, 1::2].contiguous(), "b": t["b"][..., 1::2], "c": t["c"][..., 1::2]}
    p, q = m2_b200.selective_scan(**fading, return_state=True)
    assert not s[..., ::2].any() and (s[..., 1::2] - q).abs().max() <= 2 * eps(L, 4) * 40 and (y - p).abs().max() <= 2 * eps(L, 4) * 100
    d = torch.autograd.grad(y, [leaves["x"], leaves["delta"]], torch.ones_like(y))
    assert all(torch.isfinite(v).all() for v in d)


def test_a_state_is_handed_on():
    """Two halves with the state between them are the whole, forwards and in the gradients, within the bounds of both."""
    B, L, D, N = 2, 128, 64, 16
    t = make(B, L, D, N, 1, torch.float32)
    leaves = {k: v.clone().requires_grad_() for k, v in t.items()}
    y, s = m2_b200.selective_scan(**leaves, softplus=True, return_state=True)
    seq = ("x", "delta", "b", "c", "gate")
    first = m2_b200.selective_scan(**{k: v[:, :70] if k in seq else v for k, v in leaves.items()}, softplus=True, return_state=True)
    second = m2_b200.selective_scan(**{k: v[:, 70:] if k in seq else v for k, v in leaves.items() if k != "initial_state"}, initial_state=first[1], softplus=True,
                                    return_state=True)
    halves = torch.cat([first[0], second[0]], 1)
    M = definition(t, True, None, torch.ones_like(y), torch.ones_like(s), size=True)
    within(halves, y.double(), 4 * eps(L, N) * M["y"], "y")
    for (k, p), q in zip(zip(leaves, torch.autograd.grad([y, s], list(leaves.values()), [torch.ones_like(y), torch.ones_like(s)])),
                         torch.autograd.grad([halves, second[1]], list(leaves.values()), [torch.ones_like(y), torch.ones_like(s)])):
        within(p, q.double(), (8 * eps(L, N) + (D + B * L) * U32) * M[k] + (U32 * M["lost"] if k == "delta" else U32 * M["lost"].sum((0, 1)) if k == "delta_bias" else 0.0), k)


def test_empty_batches_and_sequences():
    for B, L in ((0, 5), (2, 0), (0, 0)):
        t = make(B, L, 10, 3, 1, torch.float32)
        leaves = {k: v.clone().requires_grad_() for k, v in t.items()}
        y, s = m2_b200.selective_scan(**leaves, softplus=True, return_state=True)
        assert y.shape == (B, L, 10) and torch.equal(s, t["initial_state"])
        grads = torch.autograd.grad([y, s], list(leaves.values()), [torch.ones_like(y), torch.ones_like(s)])
        for k, v in zip(leaves, grads):
            assert v.shape == t[k].shape and torch.equal(v, torch.ones_like(v) if k == "initial_state" else torch.zeros_like(v))
    t = make(0, 1, 10, 3, 1, torch.float32)
    state = t.pop("initial_state")
    assert m2_b200.selective_scan_step(state=state, **{k: v[:, 0] if k in ("x", "delta", "b", "c", "gate") else v for k, v in t.items()}).shape == (0, 10)


def test_twice_the_same_bits_and_gradients_of_some():
    t = make(2, 400, 96, 16, 2, torch.bfloat16)
    leaves = {k: v.clone().requires_grad_() for k, v in t.items()}
    g = torch.randn(2, 400, 96, device="cuda").bfloat16()

    def run(leaves, wanted):
        return torch.autograd.grad(m2_b200.selective_scan(**leaves, softplus=True), [leaves[k] for k in wanted], g)

    ref = dict(zip(leaves, run(leaves, leaves)))
    assert all(torch.equal(p, q) for p, q in zip(ref.values(), run(leaves, leaves)))
    for wanted in (["x"], ["a", "skip"], ["b"], ["initial_state"], ["gate", "delta_bias"]):
        some = {k: v if k in wanted else v.detach() for k, v in leaves.items()}
        assert all(torch.equal(ref[k], v) for k, v in zip(wanted, run(some, wanted)))
    y, s = m2_b200.selective_scan(**leaves, softplus=True, return_state=True)       # the state alone
    (p,) = torch.autograd.grad(s, [leaves["initial_state"]], torch.ones_like(s))
    want = definition(t, True, None, torch.zeros_like(t["x"]), torch.ones_like(s))["initial_state"]
    assert (p - want).abs().max() <= 3 * eps(400, 16)


def test_offsets_beyond_2_31_elements():
    FAR, L, D, N = 2 ** 31 + 64, 70, 64, 16
    t = make(2, L, D, N, 1, torch.bfloat16)
    big = torch.empty(FAR + L * D, dtype=torch.bfloat16, device="cuda")
    far = big.as_strided((2, L, D), (FAR, D, 1))
    ref = m2_b200.selective_scan(**t, softplus=True)
    for k in ("x", "delta", "gate"):
        far.copy_(t[k])
        assert torch.equal(m2_b200.selective_scan(**{**t, k: far}, softplus=True), ref)
    leaves = {k: v.clone().requires_grad_() for k, v in t.items()}
    far.copy_(t["x"])
    up = torch.randn_like(ref)
    q = torch.autograd.grad(m2_b200.selective_scan(**leaves, softplus=True), [leaves["x"]], up)[0]
    own = far.detach().requires_grad_()
    assert torch.equal(torch.autograd.grad(m2_b200.selective_scan(**{**leaves, "x": own}, softplus=True), [own], up)[0], q)
    assert ops.device_status() == 0
