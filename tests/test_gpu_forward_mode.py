"""Forward-mode derivatives are refused by every function of causal models: none may return a value without its tangent."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

import m2_b200

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def seeded():
    with torch.random.fork_rng():                              # other files' random numbers are those they would have alone
        torch.manual_seed(0)
        yield


def calls():
    x, w = torch.randn(2, 5, 8, device="cuda"), torch.randn(8, 4, device="cuda")
    a, b = -torch.rand(8, 4, device="cuda"), torch.randn(2, 5, 4, device="cuda")
    state = torch.randn(2, 8, 4, device="cuda")
    carried = torch.randn(2, 3, 8, device="cuda")
    logits, scores = torch.randn(2, 3, 50, device="cuda"), torch.zeros(2, 3, device="cuda")
    q = torch.randn(2, 5, 2, 8, device="cuda")
    decay, s = -torch.rand(2, device="cuda"), torch.randn(2, 2, 8, 8, device="cuda")
    targets = torch.zeros(2, 3, dtype=torch.long, device="cuda")
    rows = torch.randn(6, 4, device="cuda")
    beam = torch.zeros(2, 3, dtype=torch.long, device="cuda")
    return [
        (m2_b200.causal_conv, dict(x=x, weight=w, bias=w[:, 0].contiguous(), initial_state=carried), {}),
        (m2_b200.causal_conv_step, dict(x=x[:, 0].contiguous(), state=carried, weight=w, bias=w[:, 0].contiguous()), {}),
        (m2_b200.selective_scan, dict(x=x, delta=x.clone(), a=a, b=b, c=b.clone(), skip=w[:, 0].contiguous(), gate=x.clone(), delta_bias=w[:, 1].contiguous(), initial_state=state), {}),
        (m2_b200.selective_scan_step, dict(x=x[:, 0].contiguous(), delta=x[:, 1].contiguous(), a=a, b=b[:, 0].contiguous(), c=b[:, 1].contiguous(), state=state), {}),
        (m2_b200.beam_select, dict(logits=logits, scores=scores), {}),
        (lambda state: m2_b200.reorder_states([state], beam), dict(state=rows), {}),
        (m2_b200.dropout, dict(x=x, residual=x.clone()), dict(p=0.5, seed=3)),
        (m2_b200.linear_attention, dict(q=q, k=q.clone(), v=q.clone(), log_decay=decay, initial_state=s), {}),
        (m2_b200.linear_attention_step, dict(q=q[:, 0].contiguous(), k=q[:, 1].contiguous(), v=q[:, 2].contiguous(), log_decay=decay, state=s), {}),
        (m2_b200.gated_residual_norm, dict(x=x, y=x.clone(), before_weight=w[:, 0].contiguous()), {}),
        (m2_b200.token_logprobs, dict(logits=logits), dict(targets=targets)),
    ]


@pytest.mark.parametrize("i", range(11))
def test_a_tangent_is_refused(i):
    fn, tensors, rest = calls()[i]
    fn(**tensors, **rest)                                      # without a tangent it runs, outside and inside of a level
    with fwAD.dual_level():
        fn(**tensors, **rest)
        for name, t in tensors.items():
            kept = {k: v.clone() for k, v in tensors.items()}
            dual = {**kept, name: fwAD.make_dual(t.clone(), torch.ones_like(t))}
            for context in (torch.enable_grad(), torch.no_grad()):
                with context, pytest.raises(RuntimeError, match="forward"):
                    fn(**dual, **rest)
