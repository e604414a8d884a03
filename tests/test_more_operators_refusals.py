"""What causal_conv, selective_scan, beam_select, reorder_states and dropout refuse, on the host: no GPU is touched."""
import ctypes as C

import pytest
import torch

import m2_b200
from m2_b200 import _lib, beams

SOMEWHERE = 1 << 20                      # nothing is read: the calls are refused before any launch


def refused(fn, *args):
    return fn(*(C.byref(a) if isinstance(a, C.Structure) else a for a in args), None), _lib.lib().m2_last_error().decode()


def test_causal_conv_refuses():
    x, w = torch.zeros(2, 5, 6), torch.zeros(6, 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        m2_b200.causal_conv(x, w)
    with pytest.raises(RuntimeError, match="CUDA"):
        m2_b200.causal_conv_step(x[:, 0], torch.zeros(2, 3, 6), w)
    for args in ((x[0], w), (x, w[:5]), (x, w[0]), (x, torch.zeros(6, 9)), (x, torch.zeros(6, 0)), (x[..., :0], w[:0])):
        with pytest.raises(ValueError):
            m2_b200.causal_conv(*args)
    with pytest.raises(TypeError):
        m2_b200.causal_conv(x.half(), w)
    with pytest.raises(ValueError, match="activation"):
        m2_b200.causal_conv(x, w, activation="gelu")


def scan_args(B=2, L=5, D=12, N=4, G=3):
    return dict(x=torch.zeros(B, L, D), delta=torch.zeros(B, L, D), a=torch.zeros(D, N), b=torch.zeros(B, L, G, N), c=torch.zeros(B, L, G, N))


def test_selective_scan_refuses():
    t = scan_args()
    with pytest.raises(RuntimeError, match="CUDA"):
        m2_b200.selective_scan(**t)
    with pytest.raises(RuntimeError, match="CUDA"):
        m2_b200.selective_scan_step(**{k: v[:, 0] if v.dim() > 2 else v for k, v in t.items()}, state=torch.zeros(2, 12, 4))
    for wrong in (dict(delta=torch.zeros(2, 5, 11)), dict(gate=torch.zeros(2, 4, 12)), dict(a=torch.zeros(11, 4)), dict(a=torch.zeros(12, 65)), dict(a=torch.zeros(12, 0)),
                  dict(a=torch.zeros(12)), dict(b=torch.zeros(2, 5, 3, 5)), dict(b=torch.zeros(2, 4, 3, 4), c=torch.zeros(2, 4, 3, 4)),
                  dict(b=torch.zeros(2, 5, 5, 4), c=torch.zeros(2, 5, 5, 4)), dict(c=torch.zeros(2, 5, 4)), dict(x=torch.zeros(5, 12))):
        with pytest.raises(ValueError):
            m2_b200.selective_scan(**{**t, **wrong})
    for wrong in (dict(x=t["x"].bfloat16()), dict(b=t["b"].half()), dict(gate=t["x"].double())):
        with pytest.raises(TypeError):
            m2_b200.selective_scan(**{**t, **wrong})


def test_beams_and_dropout_refuse():
    x, s = torch.zeros(2, 3, 7), torch.zeros(2, 3)
    with pytest.raises(RuntimeError, match="CUDA"):
        m2_b200.beam_select(x, s)
    with pytest.raises(ValueError):
        m2_b200.beam_select(x, s[:1])
    with pytest.raises(ValueError):
        m2_b200.beam_select(x[0], s[0])
    with pytest.raises(TypeError):
        m2_b200.beam_select(x.double(), s)
    with pytest.raises(TypeError):
        m2_b200.beam_select(x, s.long())
    beam = torch.zeros(2, 3, dtype=torch.long)
    with pytest.raises(RuntimeError, match="CUDA"):
        m2_b200.reorder_states([torch.zeros(6, 4)], beam)
    for wrong in (beam[0], beam.int(), torch.zeros(2, 33, dtype=torch.long), beam[:, :0]):
        with pytest.raises(ValueError):
            m2_b200.reorder_states([torch.zeros(6, 4)], wrong)
    with pytest.raises(RuntimeError, match="CUDA"):
        m2_b200.dropout(x, 0.1, 0)
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError):
            m2_b200.dropout(x, p, 0)
    with pytest.raises(TypeError):
        m2_b200.dropout(x.half(), 0.1, 0)


def test_states_that_share_memory_are_found():
    assert beams._apart([(0, 16, 16), (64, 16, 16)], 4) and not beams._apart([(0, 16, 16), (48, 16, 16)], 4)
    assert not beams._apart([(0, 16, 16), (0, 16, 16)], 4)
    assert beams._apart([(0, 16, 64), (16, 16, 64), (48, 16, 64), (32, 16, 64)], 4)                 # rows side by side
    assert not beams._apart([(0, 16, 64), (8, 16, 64)], 4) and not beams._apart([(0, 16, 64), (56, 16, 64)], 4)
    assert not beams._apart([(0, 16, 64), (32, 16, 32)], 4)
    assert beams._apart([(0, 0, 0), (0, 16, 16)], 4)


def test_c_entries_refuse_before_any_launch():
    lib = _lib.lib()
    for fn, n in ((lib.m2_causal_conv_fwd, 1), (lib.m2_causal_conv_bwd, 2), (lib.m2_causal_conv_step, 1), (lib.m2_selective_scan_fwd, 1), (lib.m2_selective_scan_bwd, 2),
                  (lib.m2_selective_scan_step, 1), (lib.m2_beam_select, 1), (lib.m2_reorder_states, 1), (lib.m2_dropout, 1)):
        rc, msg = refused(fn, *[None] * n)
        assert rc == 1 and "NULL" in msg
    c = _lib.CausalConvArgs(batch=2, seq_len=9, dim=8, taps=4)
    assert refused(lib.m2_causal_conv_fwd, c) == (1, "m2_causal_conv_fwd: x or weight is NULL")
    c.taps = 9
    assert refused(lib.m2_causal_conv_fwd, c)[0] == 2
    c.taps, c.dtype = 4, 2
    assert refused(lib.m2_causal_conv_fwd, c)[0] == 2
    c.dtype, c.x, c.weight = 0, SOMEWHERE, SOMEWHERE
    g = _lib.CausalConvGrads(d_y=SOMEWHERE, d_x=SOMEWHERE, workspace=SOMEWHERE)
    need = lib.m2_causal_conv_workspace(2, 9, 8, 4)
    for g.workspace_bytes in (0, need - 4):
        rc, msg = refused(lib.m2_causal_conv_bwd, c, g)
        assert rc == 1 and str(need) in msg
    c.x = SOMEWHERE + 1
    assert refused(lib.m2_causal_conv_fwd, c)[0] not in (0, 4)
    s = _lib.SelectiveScanArgs(batch=1, seq_len=4000, dim=8, states=4, groups=3)
    assert refused(lib.m2_selective_scan_fwd, s)[0] == 1
    s.groups = 2
    assert refused(lib.m2_selective_scan_fwd, s)[1].endswith("a, b or c is NULL")
    s.states = 65
    assert refused(lib.m2_selective_scan_fwd, s)[0] == 2
    s.states, s.dtype = 4, 2
    assert refused(lib.m2_selective_scan_fwd, s)[0] == 2
    s.dtype = 1
    s.x = s.delta = s.b = s.c = s.a = s.y = s.workspace = s.saves = SOMEWHERE
    need, keep = lib.m2_selective_scan_workspace(1, 4000, 8, 4, 2, 0), lib.m2_selective_scan_saves(1, 4000, 8, 4, 2)
    assert need > 0 and keep == 125 * 8 * 16 * 4
    for s.workspace_bytes, s.saves_bytes, size in ((need - 4, keep, need), (need, keep - 4, keep)):
        rc, msg = refused(lib.m2_selective_scan_fwd, s)
        assert rc == 1 and str(size) in msg
    o = _lib.SelectiveScanGrads(d_y=SOMEWHERE, d_x=SOMEWHERE, d_delta=SOMEWHERE, d_b=SOMEWHERE, d_c=SOMEWHERE)
    need = lib.m2_selective_scan_workspace(1, 4000, 8, 4, 2, 1)
    for s.workspace_bytes, s.saves_bytes, size in ((need - 4, keep, need), (need, 0, keep)):
        rc, msg = refused(lib.m2_selective_scan_bwd, s, o)
        assert rc == 1 and str(size) in msg
    o.d_gate = SOMEWHERE                                        # a gradient of no gate
    assert refused(lib.m2_selective_scan_bwd, s, o)[0] == 1
    st = _lib.SelectiveScanStepArgs(batch=2, dim=8, states=4, groups=1)
    assert refused(lib.m2_selective_scan_step, st)[0] == 1
    st.x = st.delta = st.a = st.b = st.c = st.state = st.y = SOMEWHERE
    st.s_b = 31
    assert "overlap" in refused(lib.m2_selective_scan_step, st)[1]
    cs = _lib.CausalConvStepArgs(batch=2, dim=8, taps=4, x=SOMEWHERE, weight=SOMEWHERE, state=SOMEWHERE, y=SOMEWHERE, s_b=23)
    assert "overlap" in refused(lib.m2_causal_conv_step, cs)[1]
    b = _lib.BeamSelectArgs(batch=1, beams=33, vocab=9, keep=1)
    assert refused(lib.m2_beam_select, b)[0] == 1
    b.beams, b.keep = 3, 33
    assert refused(lib.m2_beam_select, b)[0] == 1
    b.keep, b.finished, b.end_id = 3, SOMEWHERE, -1
    assert "end_id" in refused(lib.m2_beam_select, b)[1]
    b.finished = None
    b.logits = b.scores = b.score = b.beam = b.token = b.workspace = SOMEWHERE
    need = lib.m2_beam_select_workspace(1, 3, 9, 3)
    b.workspace_bytes = need - 1
    rc, msg = refused(lib.m2_beam_select, b)
    assert rc == 1 and str(need) in msg
    rows = (_lib.BeamState * 1)(_lib.BeamState(SOMEWHERE, 64, 60))
    r = _lib.ReorderStatesArgs(batch=1, beams=2, count=1, beam=SOMEWHERE, states=rows)
    assert refused(lib.m2_reorder_states, r)[0] == 1
    d = _lib.DropoutArgs(n=8, threshold=65537)
    assert refused(lib.m2_dropout, d)[0] == 1
    d.threshold = 100
    assert refused(lib.m2_dropout, d) == (1, "m2_dropout: x or y is NULL")
    # nothing to do, and nothing to check
    for fn, a in ((lib.m2_causal_conv_fwd, _lib.CausalConvArgs(dim=8, taps=4)), (lib.m2_selective_scan_fwd, _lib.SelectiveScanArgs(dim=8, states=4, groups=1)),
                  (lib.m2_beam_select, _lib.BeamSelectArgs(beams=1, keep=1, vocab=5)), (lib.m2_reorder_states, _lib.ReorderStatesArgs(batch=3, beams=2)), (lib.m2_dropout, _lib.DropoutArgs())):
        assert refused(fn, a)[0] == 0
