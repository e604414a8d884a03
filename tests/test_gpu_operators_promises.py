"""What the documentation of linear_attention, gated_residual_norm and token_logprobs says beside their formulas."""
import pytest
import torch

import m2_b200

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,L,H,dk,dv", [(2, 200, 3, 64, 64), (1, 1500, 2, 64, 64), (2, 300, 2, 128, 128), (1, 1500, 2, 40, 72), (1, 900, 1, 128, 64)])
def test_o_does_not_depend_on_whether_the_state_is_returned(B, L, H, dk, dv, dtype):
    q, k, v = (torch.randn(B, L, H, d, device="cuda").to(dtype) for d in (dk, dk, dv))
    ld = torch.linspace(-0.1, -2.0 ** -10, H, device="cuda")
    alone = m2_b200.linear_attention(q, k, v, ld)
    o, _ = m2_b200.linear_attention(q, k, v, ld, return_state=True)
    assert torch.equal(alone, o)
