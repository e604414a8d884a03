"""Workspaces of causal_conv and selective_scan, on the host: no GPU is touched."""
import torch

from m2_b200 import _lib, state_scan


def test_the_size_is_asked_for_on_the_tensors_device(monkeypatch):
    """GPUs of different sizes: the larger one's plan has more segments than the smaller one's workspace has room for."""
    now, asked = [0], []

    class On:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, now[0] = now[0], self.index

        def __exit__(self, *_):
            now[0] = self.before

    class Fake:
        @staticmethod
        def m2_selective_scan_workspace(*args):
            asked.append(now[0])
            return 4 * (100 + now[0])

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: now[0], raising=False)
    monkeypatch.setattr(torch.cuda, "device", On)
    monkeypatch.setattr(_lib, "lib", lambda: Fake)
    empty = torch.empty
    monkeypatch.setattr(torch, "empty", lambda n, dtype, device: empty(n, dtype=dtype))
    for index in (0, 1):
        a = _lib.SelectiveScanArgs()
        w = state_scan._workspace(a, torch.device("cuda", index), 0)
        assert w.numel() == 100 + index and a.workspace == w.data_ptr() and a.workspace_bytes == 4 * (100 + index)
    assert asked == [0, 1] and now == [0]


def test_a_long_axis_is_cut_into_as_many_pieces_as_run_at_once():
    """148 multiprocessors, a B200's, which are also assumed where there is no GPU: 4 blocks an SM of 64 channels forwards, 3 back, 2 with more than 16 states
    (of 32 channels with more than 32)."""
    lib = _lib.lib()

    def pieces(batch, dim, states, groups, backward):
        size = lib.m2_selective_scan_workspace(batch, 1 << 15, dim, states, groups, backward) // 4
        np = 16 if states <= 16 else 32 if states <= 32 else 64
        if backward:                     # without the parts of the gradients: of b and c for each tile, of the parameters for each segment
            tiles = -(-dim // groups // (32 if np == 64 else 64))
            size -= 2 * tiles * batch * (1 << 15) * groups * np
            return size / (batch * dim * (np + 1 + np + 2) + (batch * groups * tiles * 14336 if np > 16 else 0))
        return size / (batch * dim * (np + 1))

    for batch, dim, states, groups, blocks, an_sm in ((1, 768, 16, 1, 12, 4), (2, 768, 11, 2, 24, 4), (1, 768, 20, 1, 12, 2), (1, 768, 50, 1, 24, 2), (3, 100, 16, 1, 6, 4)):
        n = pieces(batch, dim, states, groups, 0)
        assert n == int(n) and n * blocks <= an_sm * 148 < 1.3 * n * blocks
        n = pieces(batch, dim, states, groups, 1)
        assert n == int(n) and n * blocks <= min(an_sm, 3) * 148 < 1.3 * n * blocks
    assert pieces(20, 768, 16, 1, 0) == 0                       # 240 blocks: not cut
    assert lib.m2_selective_scan_saves(2, 100, 30, 5, 1) == 4 * 2 * 4 * 30 * 16 and lib.m2_selective_scan_saves(2, 0, 30, 5, 1) == 0
    assert lib.m2_causal_conv_workspace(1, 100, 8, 4) == 4 * 7 * 5 * 8 and lib.m2_causal_conv_workspace(0, 5, 8, 4) == 0
