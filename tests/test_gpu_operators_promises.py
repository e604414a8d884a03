"""What the documentation of linear_attention, gated_residual_norm and token_logprobs says beside their formulas."""
import pytest
import torch

import m2_b200
from m2_b200 import ops

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
