"""What linear_attention, linear_attention_step, gated_residual_norm and token_logprobs refuse, on the host: no GPU is touched."""
import ctypes as C

import pytest
import torch

import m2_b200
from m2_b200 import _lib


def qkv(B=2, L=5, H=4, K=2, dk=8, dv=6, dtype=torch.float32):
    return (torch.zeros(B, L, H, dk, dtype=dtype), torch.zeros(B, L, K, dk, dtype=dtype), torch.zeros(B, L, K, dv, dtype=dtype), torch.zeros(H))


def test_linear_attention_refuses_what_does_not_belong_together():
    q, k, v, ld = qkv()
    with pytest.raises(RuntimeError, match="CUDA"):
        m2_b200.linear_attention(q, k, v, ld)
    with pytest.raises(ValueError, match="dimensions"):
        m2_b200.linear_attention(q[0], k, v, ld)
    with pytest.raises(ValueError, match="belong together"):
        m2_b200.linear_attention(q, k[:, :4], v, ld)
    with pytest.raises(ValueError, match="belong together"):
        m2_b200.linear_attention(q[:, :, :3], k, v, ld[:3])
    with pytest.raises(ValueError, match="belong together"):
        m2_b200.linear_attention(q, k, v[:, :, :1], ld)
    with pytest.raises(ValueError, match="belong together"):
        m2_b200.linear_attention(q[..., :0], k[..., :0], v, ld)
    with pytest.raises(TypeError, match="float32"):
        m2_b200.linear_attention(q.half(), k.half(), v.half(), ld)
    with pytest.raises(TypeError, match="float32"):
        m2_b200.linear_attention(q, k.bfloat16(), v, ld)
    with pytest.raises(ValueError, match="log_decay"):
        m2_b200.linear_attention(q, k, v, ld[:2])


def test_step_refuses_what_does_not_belong_together():
    q, k, v, ld = qkv()
    with pytest.raises(RuntimeError, match="CUDA"):
        m2_b200.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, torch.zeros(2, 4, 8, 6))
    with pytest.raises(ValueError, match="dimensions"):
        m2_b200.linear_attention_step(q, k, v, ld, torch.zeros(2, 4, 8, 6))


def test_gated_residual_norm_refuses():
    x = torch.zeros(2, 3, 16)
    with pytest.raises(RuntimeError, match="CUDA"):
        m2_b200.gated_residual_norm(x, x)
    with pytest.raises(ValueError, match="one shape"):
        m2_b200.gated_residual_norm(x, x[:1])


def test_token_logprobs_refuses():
    x, t = torch.zeros(3, 7), torch.zeros(3, dtype=torch.long)
    with pytest.raises(RuntimeError, match="CUDA"):
        m2_b200.token_logprobs(x, t)
    with pytest.raises(ValueError, match="one target"):
        m2_b200.token_logprobs(x, t[:2])
    with pytest.raises(TypeError, match="logits"):
        m2_b200.token_logprobs(x.double(), t)
    with pytest.raises(TypeError, match="targets"):
        m2_b200.token_logprobs(x, t.float())


def refused(fn, *args):
    rc = fn(*(C.byref(a) if isinstance(a, C.Structure) else a for a in args), None)
    return rc, _lib.lib().m2_last_error().decode()


def test_c_entries_refuse_before_any_launch():
    lib = _lib.lib()
    for fn, n in ((lib.m2_linear_attention_fwd, 1), (lib.m2_linear_attention_bwd, 2), (lib.m2_linear_attention_step, 1), (lib.m2_residual_norm_fwd, 1),
                  (lib.m2_residual_norm_bwd, 2), (lib.m2_token_logprobs_fwd, 1), (lib.m2_token_logprobs_bwd, 1)):
        rc, msg = refused(fn, *[None] * n)
        assert rc == 1 and "NULL" in msg
    a = _lib.LinearAttentionArgs(batch=1, seq_len=4, heads=4, kv_heads=3, dk=8, dv=8, scale=1.0)
    assert refused(lib.m2_linear_attention_fwd, a)[0] == 1
    a.kv_heads = 4
    assert refused(lib.m2_linear_attention_fwd, a) == (1, "m2_linear_attention_fwd: q, k, v or log_decay is NULL")
    a.dk = 129
    assert refused(lib.m2_linear_attention_fwd, a)[0] == 2
    a.dk, a.dtype = 8, 2
    assert refused(lib.m2_linear_attention_fwd, a)[0] == 2
    a.dtype, a.scale = 0, 0.0
    assert refused(lib.m2_linear_attention_fwd, a)[0] == 1
    a.scale, a.batch = float("inf"), 1
    assert refused(lib.m2_linear_attention_fwd, a)[0] == 1
    s = _lib.LinearAttentionStepArgs(batch=1, heads=4, kv_heads=4, dk=8, dv=8, scale=1.0)
    assert refused(lib.m2_linear_attention_step, s)[0] == 1
    s.batch = 5000000
    assert refused(lib.m2_linear_attention_step, s)[0] == 2
    n = _lib.ResidualNormArgs(rows=4, seq_len=3, n=8, ldx=8, ldy=8)
    assert refused(lib.m2_residual_norm_fwd, n)[0] == 1
    n.seq_len, n.n = 4, 8193
    assert refused(lib.m2_residual_norm_fwd, n)[0] == 2
    n.n = 8
    assert refused(lib.m2_residual_norm_fwd, n) == (1, "m2_residual_norm_fwd: x, y or the gate is NULL")
    t = _lib.TokenLogprobsArgs(rows=2, vocab=8, top=9, ld=8)
    assert refused(lib.m2_token_logprobs_fwd, t)[0] == 1
    t.top = 33
    t.vocab = t.ld = 64
    assert refused(lib.m2_token_logprobs_fwd, t)[0] == 1
    t.top, t.dtype = 0, 2
    assert refused(lib.m2_token_logprobs_fwd, t)[0] == 2
    t.dtype = 0
    assert refused(lib.m2_token_logprobs_fwd, t) == (1, "m2_token_logprobs_fwd: logits or targets are NULL")
    # no rows: nothing to do, and nothing to check
    for fn, args in ((lib.m2_token_logprobs_fwd, _lib.TokenLogprobsArgs(vocab=8)), (lib.m2_residual_norm_fwd, _lib.ResidualNormArgs(seq_len=1, n=8)),
                     (lib.m2_linear_attention_fwd, _lib.LinearAttentionArgs(heads=1, kv_heads=1, dk=8, dv=8, scale=1.0))):
        assert refused(fn, args)[0] == 0


def test_workspaces():
    lib = _lib.lib()
    assert lib.m2_linear_attention_workspace(1, 64, 4, 4, 64, 64, 1, 0) == 0                 # a short text needs none
    assert lib.m2_linear_attention_workspace(2, 10, 4, 2, 8, 6, 1, 1) == 2 * 10 * 4 * 14 * 4  # gradients of shared heads
    assert lib.m2_linear_attention_workspace(0, 64, 4, 4, 64, 64, 1, 0) == 0
    assert lib.m2_residual_norm_workspace(0, 1, 8, 0) == 0
    assert lib.m2_residual_norm_workspace(1, 1, 8, 0) == 6 * 8 * 4
