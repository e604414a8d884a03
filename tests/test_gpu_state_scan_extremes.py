"""selective_scan and selective_scan_step at the ends of their range, against the definition in 64 bits: states that forget at once or hardly at all, states that
grow, tokens that outweigh all others, and what a NaN or an infinity may reach.

Bounds, where steps are given (softplus off) and float32.  The errors are counted against M, the same sums of absolute values with half of every decay's exponent.
A decay exp(s a) carries the exp's 2^-22 and two roundings of its exponent, T 2^-23 of it for T = |s a|, and T exp(-T) <= 0.74 exp(-T / 2).  With T >= 1 a token,
the ages k of a sum contribute k (2^-22 + 2^-23) exp(-k T / 2) of it at most, below 2^-21 in all.  Sums of n terms are off by n 2^-24 of M: N states, two products and
the recurrences' own two roundings a token (below 8 with the same weights)."""
import pytest
import torch

import m2_b200
from tests.test_gpu_linear_attention import U32, within
from tests.test_gpu_state_scan import definition, make

pytestmark = pytest.mark.gpu
LOWEST, NONE = torch.finfo(torch.float32).min, -float("inf")


@pytest.fixture(autouse=True)
def seeded():
    with torch.random.fork_rng():                              # other files' random numbers are those they would have alone
        torch.manual_seed(0)
        yield


def strong(N):
    return (N + 16) * U32 + 2.0 ** -21


@pytest.mark.parametrize("value", [-1e30, LOWEST, NONE])
@pytest.mark.parametrize("L,N", [(33, 4), (60, 20), (64, 50), (700, 16)])
def test_states_that_forget_at_once(L, N, value):
    """exp(s a) is 0 for every step above zero, and 1 for a step of 0: behind a text nothing fades, whatever a is."""
    B, D = 2, 40
    t = make(B, L, D, N, 1, torch.float32, plain=True)
    t["a"][:, ::2] = value
    t["delta"] = t["delta"] + 0.01
    t["initial_state"] = torch.randn(B, D, N, device="cuda")
    t["gate"] = torch.randn(B, L, D, device="cuda")
    lengths = torch.tensor([L, L - 30], device="cuda")
    leaves = {k: v.clone().requires_grad_() for k, v in t.items()}
    y, s = m2_b200.selective_scan(**leaves, lengths=lengths, return_state=True)
    up, d_s = torch.randn_like(y), torch.randn_like(s)
    grads = dict(zip(leaves, torch.autograd.grad([y, s], list(leaves.values()), [up, d_s])))
    finite = {**t, "a": t["a"].clamp(min=-1e30)}                # the same function of steps that are 0 or 0.01 at least
    ref, M = (definition(finite, False, lengths, up, d_s, size) for size in (False, True))
    one = strong(N) + L * 2.0 ** -21                           # every other state fades as it likes
    within(y, ref["y"], U32 * ref["y"].abs() + 2 * one * M["y"], "y")
    within(s, ref["state"], U32 * ref["state"].abs() + one * M["state"], "state")
    last = torch.stack([(t["delta"] * t["x"])[i, n - 1, :, None] * t["b"][i, n - 1] for i, n in enumerate(lengths.tolist())])
    assert torch.equal(s[..., ::2], last[..., ::2])
    for k in ("x", "a", "b", "c", "gate", "initial_state"):
        terms = {"b": D, "c": D, "a": B * L}.get(k, 0)
        within(grads[k], ref[k], U32 * ref[k].abs() + (3 * one + terms * U32) * M[k], k)
    assert not grads["a"][:, ::2].any() and not grads["initial_state"][..., ::2].any()


@pytest.mark.parametrize("N", [4, 6])
@pytest.mark.parametrize("value", [LOWEST, NONE, -LOWEST])
def test_a_step_of_zero_changes_no_state(N, value):
    B, D = 2, 10
    t = make(B, 1, D, N, 1, torch.float32, plain=True)
    t["a"][:, ::2] = value
    t["delta"].zero_()
    state = torch.randn(B, D, N, device="cuda")
    own = state.clone()
    m2_b200.selective_scan_step(state=own, **{k: v[:, 0] if k in ("x", "delta", "b", "c") else v for k, v in t.items()})
    assert torch.equal(own, state)
    _, s = m2_b200.selective_scan(**t, initial_state=state, return_state=True)
    assert torch.equal(s, state)


FADING = [(-1e2, 5.0), (-16.0, 5.0), (-1e4, 1.0), (-1e30, 0.1), (LOWEST, 0.1)]


@pytest.mark.parametrize("a,step", FADING)
@pytest.mark.parametrize("L,N", [(64, 4), (45, 4), (600, 4), (64, 20), (70, 40)])
def test_steps_of_states_that_fade_fast(L, N, a, step):
    """The gradient of a step is sum_n a g exp(s a) h + x sum_n g b.  Where a state forgets, the first part is next to nothing and the second is left, whatever a is."""
    B, D = 2, 24
    t = make(B, L, D, N, 1, torch.float32, plain=True)
    t["a"] = torch.full((D, N), a, device="cuda") * (0.5 + torch.rand(D, N, device="cuda") * 0.5)
    t["delta"] = step * (1 + torch.rand(B, L, D, device="cuda"))
    leaves = {k: v.clone().requires_grad_() for k, v in t.items()}
    y, s = m2_b200.selective_scan(**leaves, return_state=True)
    up, d_s = torch.randn_like(y), torch.randn_like(s)
    grads = dict(zip(leaves, torch.autograd.grad([y, s], list(leaves.values()), [up, d_s])))
    ref, M = (definition(t, False, None, up, d_s, size) for size in (False, True))
    for k in ("delta", "x", "a"):
        within(grads[k], ref[k], U32 * ref[k].abs() + (3 * strong(N) + (B * L * U32 if k == "a" else 0.0)) * M[k], k)


@pytest.mark.parametrize("what", ["dy", "x", "both"])
@pytest.mark.parametrize("L,N", [(64, 4), (600, 4), (64, 20), (70, 40)])
def test_a_token_that_outweighs_the_others_leaves_their_gradients_alone(L, N, what):
    """One gradient of y, or one x, a million times the others': tokens behind the first, and in front of the second, do not depend on it."""
    B, D = 2, 24
    t = make(B, L, D, N, 1, torch.float32, plain=True)
    t["a"] = -1 - torch.rand(D, N, device="cuda")
    t["delta"] = 1 + torch.rand(B, L, D, device="cuda")
    up, d_s = torch.randn(B, L, D, device="cuda"), torch.randn(B, D, N, device="cuda")
    for at in (5, 18, 27, 43):
        if what != "x":
            up[:, at, ::3] *= 1e6
        if what != "dy":
            t["x"][:, at, ::3] *= 1e6
    leaves = {k: v.clone().requires_grad_() for k, v in t.items()}
    y, s = m2_b200.selective_scan(**leaves, return_state=True)
    grads = dict(zip(leaves, torch.autograd.grad([y, s], list(leaves.values()), [up, d_s])))
    ref, M = (definition(t, False, None, up, d_s, size) for size in (False, True))
    for k in ("delta", "x", "a"):
        within(grads[k], ref[k], U32 * ref[k].abs() + (3 * strong(N) + (B * L * U32 if k == "a" else 0.0)) * M[k], k)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("L,N", [(60, 16), (700, 16), (100, 20), (60, 40)])
def test_what_is_not_finite_reaches_no_gradient_that_does_not_depend_on_it(L, N, dtype):
    """A gradient of y at one token: gradients of its channel up to this token.  An x: gradients of its channel behind it (and its own).  Bits of all others stay."""
    D, T, CH = 70, 37, 5
    t = make(1, L, D, N, 1, dtype)

    def run(t, up):
        leaves = {k: v.clone().requires_grad_() for k, v in t.items()}
        y, s = m2_b200.selective_scan(**leaves, softplus=True, return_state=True)
        return dict(zip(leaves, torch.autograd.grad([y, s], list(leaves.values()), [up, torch.ones_like(s)])))

    up = torch.randn(1, L, D, device="cuda").to(dtype)
    ref = run(t, up)
    others = [i for i in range(D) if i != CH]
    for value in (float("nan"), float("inf")):
        bad = up.clone()
        bad[0, T, CH] = value
        got = run(t, bad)
        for k in ("x", "delta", "gate"):
            assert torch.equal(got[k][..., others], ref[k][..., others]) and torch.equal(got[k][:, T + 1:], ref[k][:, T + 1:]), k
        assert torch.equal(got["gate"][:, :T], ref["gate"][:, :T]) and torch.equal(got["b"][:, T + 1:], ref["b"][:, T + 1:])
        assert torch.equal(got["c"][:, :T], ref["c"][:, :T]) and torch.equal(got["c"][:, T + 1:], ref["c"][:, T + 1:])
        assert not torch.isfinite(got["x"][0, T, CH]) and not torch.isfinite(got["delta"][0, T, CH])
        bad = {k: v.clone() for k, v in t.items()}
        bad["x"][0, T, CH] = value
        got = run(bad, up)
        for k in ("x", "delta", "gate"):
            assert torch.equal(got[k][..., others], ref[k][..., others]) and torch.equal(got[k][:, :T], ref[k][:, :T]), k
        assert torch.equal(got["x"][:, T + 1:], ref["x"][:, T + 1:])
        assert torch.equal(got["b"][:, :T], ref["b"][:, :T]) and torch.equal(got["b"][:, T + 1:], ref["b"][:, T + 1:])
        assert torch.equal(got["c"][:, :T], ref["c"][:, :T])


@pytest.mark.parametrize("L,N", [(100, 4), (700, 4), (100, 20), (60, 40)])
def test_gradients_beside_an_empty_state_that_would_grow(L, N):
    """Factors of e^20 a token on states that are neither fed nor read: all gradients are those of the fading states alone, and theirs are zero."""
    D = 64
    t = make(1, L, D, N, 1, torch.float32, plain=True)
    t["a"] = -1 - torch.rand(D, N, device="cuda")
    t["a"][:, ::2] = 20.0
    t["delta"] = torch.ones_like(t["delta"])
    t["b"][..., ::2] = 0
    t["c"][..., ::2] = 0
    leaves = {k: v.clone().requires_grad_() for k, v in t.items()}
    y = m2_b200.selective_scan(**leaves)
    up = torch.randn_like(y)
    grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), up)))
    fading = {**t, "a": t["a"][:, 1::2], "b": t["b"][..., 1::2], "c": t["c"][..., 1::2]}
    ref, M = (definition(fading, False, None, up, None, size) for size in (False, True))
    for k, v in grads.items():
        if k in ("a", "b", "c"):
            assert not v[..., ::2].any(), k
            v = v[..., 1::2]
        terms = {"b": D, "c": D, "a": L}.get(k, 0)
        within(v, ref[k], U32 * ref[k].abs() + (3 * strong(N) + terms * U32) * M[k], k)


@pytest.mark.parametrize("L,N", [(64, 4), (700, 16), (64, 20), (100, 40)])
@pytest.mark.parametrize("rate,start", [(1.0, 1e-30), (-1.0, 1e30)])
def test_factors_beyond_float32_between_states_within_it(L, N, rate, start):
    """exp(a times the steps of a tile, or of a segment) is e^128 or e^-128, beyond float32; the state of 1e-30 (1e30) in front and that behind are not.
    Errors: 2^-22 for each of the 64 decays of a step that is not 0, and 128 times what the exponents are off by: two roundings, and one for each of the 64 sums on the way
    to the sum of the steps (all steps are equal, so these may all go one way)."""
    B, D = 2, 24
    t = make(B, L, D, N, 1, torch.float32, plain=True)
    t["a"] = torch.full((D, N), 20.0 * rate, device="cuda")
    t["delta"] = torch.zeros(B, L, D, device="cuda")
    first, tokens, step = (64, 64, 0.1) if L > 100 else (32, 20, 0.32)
    t["delta"][:, first:first + tokens] = step
    t["x"].zero_()
    t["initial_state"] = start * (1 + torch.rand(B, D, N, device="cuda"))
    leaves = {k: v.clone().requires_grad_() for k, v in t.items()}
    y, s = m2_b200.selective_scan(**leaves, return_state=True)
    d_s = start * torch.randn(B, D, N, device="cuda").sign()
    (g,) = torch.autograd.grad(s, [leaves["initial_state"]], d_s)
    total = (t["delta"].double()[..., None] * t["a"].double()).sum(1)
    one = 64 * 2.0 ** -22 + 128 * (2 + 64) * U32 + 64 * U32
    within(s, t["initial_state"].double() * torch.exp(total), one * (t["initial_state"].double() * torch.exp(total)).abs(), "state")
    within(g, d_s.double() * torch.exp(total), one * (d_s.double() * torch.exp(total)).abs(), "gradient")


def test_more_blocks_than_places_for_what_they_put_aside():
    """With more than 16 states blocks beyond 4096 take one sequence after another: each sequence's gradients are those of a smaller batch."""
    B, L, D, N, G = 1100, 40, 16, 20, 4                        # 4400 blocks; 2200 in each half
    t = make(B, L, D, N, G, torch.float32)
    lengths = torch.randint(0, L + 1, (B,), device="cuda")
    up, d_s = torch.randn(B, L, D, device="cuda"), torch.randn(B, D, N, device="cuda")

    def run(part):
        leaves = {k: (v if k in ("a", "skip", "delta_bias") else v[part]).clone().requires_grad_() for k, v in t.items()}
        y, s = m2_b200.selective_scan(**leaves, softplus=True, lengths=lengths[part], return_state=True)
        return dict(zip(leaves, torch.autograd.grad([y, s], list(leaves.values()), [up[part], d_s[part]])))

    whole, halves = run(slice(None)), [run(slice(0, B // 2)), run(slice(B // 2, B))]
    M = definition(t, True, lengths, up, d_s, size=True)
    for k, v in whole.items():
        if k in ("a", "skip", "delta_bias"):
            within(v, sum(h[k].double() for h in halves), 32 * U32 * M[k], k)      # the same parts, in eights of other neighbours
        else:
            assert torch.equal(v, torch.cat([h[k] for h in halves])), k


@pytest.mark.parametrize("B,L,D,N,G", [(2, 512, 64, 16, 1), (1, 2048, 64, 16, 1), (2, 512, 64, 20, 1), (2, 512, 64, 40, 2)])
def test_roundings_in_training_add_up_as_independent_ones_do(B, L, D, N, G):
    """Steps of 0.001 to 0.1 and a of -1 to -N, as models begin with.  A value is a nest of sums of 32 tokens of a tile, at three roundings each, of the tiles that a state
    lives through, of N states or D channels and of a handful around them: k below 3 32 + 2 N + D + 16 roundings and exps in a row that matter, each 2^-24 in size (the exps'
    2^-22 at most, and 2^-24 in the mean).  Independent ones add up to k^(1/2) 2^-24 of the sum of sizes, in the 2-norm; a bias, or a difference of large terms, does not."""
    g = torch.Generator(device="cuda").manual_seed(L + N)

    def rnd(*s, std=1.0, mean=0.0):
        return torch.randn(s, device="cuda", generator=g) * std + mean

    steps = torch.exp(torch.rand(D, device="cuda", generator=g) * 4.6 - 6.9)
    t = dict(x=rnd(B, L, D), delta=rnd(B, L, D, std=0.5), a=-torch.arange(1, N + 1, device="cuda") * torch.exp(rnd(D, N, std=0.05)), b=rnd(B, L, G, N), c=rnd(B, L, G, N),
             skip=rnd(D, mean=1.0, std=0.1), delta_bias=steps + torch.log(-torch.expm1(-steps)), gate=rnd(B, L, D), initial_state=rnd(B, D, N, std=0.5))
    leaves = {k: v.clone().requires_grad_() for k, v in t.items()}
    y, s = m2_b200.selective_scan(**leaves, softplus=True, return_state=True)
    up, d_s = torch.randn(B, L, D, device="cuda", generator=g), torch.randn(B, D, N, device="cuda", generator=g)
    got = dict(zip(leaves, torch.autograd.grad([y, s], list(leaves.values()), [up, d_s])), y=y.detach(), state=s.detach())
    ref, M = (definition(t, True, None, up, d_s, size) for size in (False, True))
    most = (3 * 32 + 2 * N + D + 16) ** 0.5 * U32
    found = {k: ((v.double() - ref[k]).norm() / (most * M[k].norm())).item() for k, v in got.items()}
    assert max(found.values()) <= 1, found
