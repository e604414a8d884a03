"""Workspaces of linear_attention and gated_residual_norm, rows of token_logprobs, types of decays, on the host: no GPU is touched."""
import ctypes as C

import pytest
import torch

import m2_b200
from m2_b200 import _lib, linear_attn, ops

SOMEWHERE = 1 << 20                      # nothing is read: the calls are refused before any launch


def refused(fn, *args):
    return fn(*(C.byref(a) for a in args), None), _lib.lib().m2_last_error().decode()


def test_a_workspace_that_is_too_small_is_refused():
    lib = _lib.lib()
    a = _lib.LinearAttentionArgs(batch=1, seq_len=4000, heads=2, kv_heads=1, dk=64, dv=64, dtype=1, scale=1.0)
    a.q = a.k = a.v = a.log_decay = a.o = a.workspace = SOMEWHERE
    g = _lib.LinearAttentionGrads(d_o=SOMEWHERE, d_q=SOMEWHERE, d_k=SOMEWHERE, d_v=SOMEWHERE)
    for fn, more, backward in ((lib.m2_linear_attention_fwd, (), 0), (lib.m2_linear_attention_bwd, (g,), 1)):
        need = lib.m2_linear_attention_workspace(1, 4000, 2, 1, 64, 64, 1, backward)
        assert need > 0
        for a.workspace_bytes in (0, need - 4):
            rc, msg = refused(fn, a, *more)
            assert rc == 1 and str(need) in msg
    a.workspace, a.workspace_bytes = None, need
    assert refused(lib.m2_linear_attention_bwd, a, g)[0] == 1
    n = _lib.ResidualNormArgs(rows=40, seq_len=10, n=64, ldx=64, ldy=64, gate_kind=2, ldg=64, norm_after=1)
    n.x = n.y = n.gate = n.stats = SOMEWHERE
    need = lib.m2_residual_norm_workspace(40, 10, 64, 2)
    for size in (0, need - 4):
        rc, msg = refused(lib.m2_residual_norm_bwd, n, _lib.ResidualNormGrads(workspace=SOMEWHERE, workspace_bytes=size))
        assert rc == 1 and str(need) in msg


def test_the_size_is_asked_for_on_the_tensors_device(monkeypatch):
    """GPUs of different sizes: the larger one's plan has more segments than the smaller one's workspace has room for."""
    now = [0]
    asked = []

    class On:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, now[0] = now[0], self.index

        def __exit__(self, *_):
            now[0] = self.before

    class Fake:
        @staticmethod
        def m2_linear_attention_workspace(*args):
            asked.append(now[0])
            return 4 * (100 + now[0])

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: now[0], raising=False)
    monkeypatch.setattr(torch.cuda, "device", On)
    monkeypatch.setattr(_lib, "lib", lambda: Fake)
    empty = torch.empty
    monkeypatch.setattr(torch, "empty", lambda n, dtype, device: empty(n, dtype=dtype))
    for index in (0, 1):
        a = _lib.LinearAttentionArgs()
        w = linear_attn._workspace(a, torch.device("cuda", index), 0)
        assert w.numel() == 100 + index and a.workspace == w.data_ptr() and a.workspace_bytes == 4 * (100 + index)
    assert asked == [0, 1] and now == [0]
    assert ops._on_device(1, lambda x: (x, now[0]), 5) == (5, 1)


def test_groups_of_rows_that_make_no_sense_are_refused():
    for group, ld_group in ((-1, 8), (1, -8), (1 << 28, 8)):
        t = _lib.TokenLogprobsArgs(rows=2, vocab=8, ld=8, group=group, ld_group=ld_group, logits=SOMEWHERE, targets=SOMEWHERE)
        rc, msg = refused(_lib.lib().m2_token_logprobs_fwd, t)
        assert rc == 1 and "groups" in msg


def test_a_long_axis_is_cut_into_as_many_pieces_as_run_at_once():
    """148 multiprocessors, a B200's, which are also assumed where there is no GPU."""
    lib = _lib.lib()

    def pieces(dk, dv, dtype, backward):
        size = lib.m2_linear_attention_workspace(1, 1 << 16, 2, 2, dk, dv, dtype, backward)
        return size // (4 * (3 if backward else 1) * 2 * dk * dv)

    for dk, dv, dtype, an_sm in ((64, 64, 1, 3), (128, 64, 1, 2), (96, 64, 0, 2), (97, 64, 0, 1), (128, 64, 0, 1), (64, 64, 0, 2)):
        assert pieces(dk, dv, dtype, 0) <= an_sm * 148 // 2 < 1.1 * pieces(dk, dv, dtype, 0)
        tiles = 2 * ((dk + 63) // 64) + 1                  # of the three gradients
        assert pieces(dk, dv, dtype, 1) <= an_sm * 148 // (2 * tiles) < 1.1 * pieces(dk, dv, dtype, 1)


def test_complex_decays_are_refused():
    q, ld = torch.zeros(1, 2, 3, 8), torch.zeros(3, dtype=torch.complex64)
    with pytest.raises(TypeError, match="log_decay"):
        m2_b200.linear_attention(q, q, q, ld)
    with pytest.raises(TypeError, match="log_decay"):
        m2_b200.linear_attention_step(q[:, 0], q[:, 0], q[:, 0], ld, torch.zeros(1, 3, 8, 8))
