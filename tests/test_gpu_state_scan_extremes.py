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
    torch.manual_seed(0)


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
