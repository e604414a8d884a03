"""Offsets beyond 2^31 elements: results there are those of the same values near by, bit for bit."""
import pytest
import torch

import m2_b200

pytestmark = pytest.mark.gpu
FAR = 2 ** 31 + 64


def test_linear_attention_reads_far_sequences():
    big = torch.empty(FAR + 70 * 64, dtype=torch.bfloat16, device="cuda")
    near = torch.randn(3, 2, 70, 1, 64, device="cuda").bfloat16()
    far = big.as_strided((2, 70, 1, 64), (FAR, 64, 64, 1))
    ld = torch.tensor([-0.05], device="cuda")
    for i in range(3):                                     # q, k and v by turns
        far.copy_(near[i])
        args = [far if i == j else near[j] for j in range(3)]
        a, b = (m2_b200.linear_attention(*t, ld, return_state=True) for t in (args, near))
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    far.copy_(near[0])
    leaf = far.detach().requires_grad_()
    (g,) = torch.autograd.grad(m2_b200.linear_attention(leaf, near[1], near[2], ld), [leaf], near[1])
    leaf = near[0].clone().requires_grad_()
    (h,) = torch.autograd.grad(m2_b200.linear_attention(leaf, near[1], near[2], ld), [leaf], near[1])
    assert torch.equal(g, h)


def test_step_updates_far_states():
    big = torch.empty(FAR + 64 * 64, dtype=torch.float32, device="cuda")
    far = big.as_strided((2, 1, 64, 64), (FAR, 64 * 64, 64, 1))
    near = torch.randn(2, 1, 64, 64, device="cuda")
    far.copy_(near)
    q = torch.randn(2, 1, 64, device="cuda")
    ld = torch.tensor([-0.05], device="cuda")
    assert torch.equal(m2_b200.linear_attention_step(q, q, q, ld, far), m2_b200.linear_attention_step(q, q, q, ld, near))
    assert torch.equal(far, near)


@pytest.mark.parametrize("n", [768, 600])
def test_norms_read_far_rows(n):
    big = torch.empty(FAR + n, dtype=torch.bfloat16, device="cuda")
    far = big.as_strided((2, n), (FAR, 1))
    near, w = torch.randn(2, n, device="cuda").bfloat16(), torch.randn(n, device="cuda")
    far.copy_(near)
    outs = []
    for t in (far, near):
        leaf = t.detach().requires_grad_()
        r, h = m2_b200.gated_residual_norm(leaf, leaf, gate=leaf, after_weight=w, before_weight=w)
        outs.append([r, h, *torch.autograd.grad([r, h], [leaf], [near, near])])
    assert all(torch.equal(a, b) for a, b in zip(*outs))


def test_token_logprobs_of_far_rows():
    N, V = 70001, 32768
    x = torch.zeros(N, V, dtype=torch.bfloat16, device="cuda")
    x[-3:] = torch.randn(3, V, device="cuda") * 3
    t = torch.arange(N, device="cuda") % V
    x.requires_grad_()
    out = m2_b200.token_logprobs(x, t, top=4)
    (d,) = torch.autograd.grad(out.logprob.sum() + out.entropy.sum(), [x])
    few = x.detach()[-3:].clone().requires_grad_()
    ref = m2_b200.token_logprobs(few, t[-3:], top=4)
    (e,) = torch.autograd.grad(ref.logprob.sum() + ref.entropy.sum(), [few])
    assert torch.equal(out.top_id[-3:], ref.top_id)
    for a, b in ((out.logprob[-3:], ref.logprob), (out.entropy[-3:], ref.entropy), (d[-3:].float(), e.float())):
        # few rows are shared by more blocks: other sums, within (V / 128 + 64) roundings of float32 and one of bf16
        assert (a - b).abs().max() <= (V / 128 + 64) * 2.0 ** -24 * 32 + 2.0 ** -8 * b.abs().max()
    assert (out.logprob[:5] + torch.log(torch.tensor(float(V)))).abs().max() < 1e-5
