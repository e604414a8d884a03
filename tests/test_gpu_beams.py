"""beam_select and reorder_states against their definition in 64 bits.

Ids are equal, as the order of 64-bit scores is: logits here are sums of a few random numbers, whose scores lie further apart than the kernel's log of the sum of
exponentials can be off, (V / 128 + 64) 2^-24 + 2^-22; a test says so before it compares.  A score is rounded to float32 once."""
import itertools

import pytest
import torch

import m2_b200
from m2_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def seeded():
    torch.manual_seed(0)


NONE = -float("inf")


def definition(logits, scores, keep, finished=None, end_id=None):
    """By lists: (score, beam, token) of every text, best first, and the smallest gap between neighbours in the order."""
    B, K, V = logits.shape
    lp = torch.log_softmax(logits.double(), -1) + scores.double()[..., None]
    lp = torch.where(torch.isneginf(logits.double()).all(-1, keepdim=True), NONE, lp)
    out, gap = [], float("inf")
    for i in range(B):
        rows = []
        for k in range(K):
            if finished is not None and finished[i, k]:
                rows.append((scores[i, k].double().item(), k, end_id))
            else:
                ids = logits[i, k].float().sort(descending=True, stable=True).indices[:keep].tolist()
                rows += [(lp[i, k, j].item(), k, j) for j in ids]
        rows = [r for r in rows if r[0] != NONE]
        order = sorted(range(len(rows)), key=lambda n: (rows[n][0] == rows[n][0], -rows[n][0], n))
        best = [rows[n] for n in order[:keep]]
        some = [rows[n] for n in order[:keep + 1]]
        gap = min([gap] + [p[0] - q[0] for p, q in itertools.pairwise(some) if p[1] != q[1]])
        out.append(best + [(NONE, 0, end_id if end_id is not None else 0)] * (keep - len(best)))
    return out, gap


def check(logits, scores, keep=None, finished=None, end_id=None, apart=True):
    keep_n = keep or logits.shape[1]
    ref, gap = definition(logits, scores, keep_n, finished, end_id)
    got = m2_b200.beam_select(logits, scores, keep=keep, finished=finished, end_id=end_id)
    assert got.score.shape == got.beam.shape == got.token.shape == (logits.shape[0], keep_n)
    lost = (logits.shape[-1] / 128 + 64) * 2.0 ** -24 + 2.0 ** -22
    assert gap > lost or not apart, f"a gap of {gap}: other inputs are wanted"
    for i, rows in enumerate(ref):
        assert got.beam[i].tolist() == [r[1] for r in rows] and got.token[i].tolist() == [r[2] for r in rows]
        want = torch.tensor([r[0] for r in rows], dtype=torch.float64)
        have = got.score[i].double().cpu()
        finite = torch.isfinite(want)
        assert torch.equal(torch.nan_to_num(want[~finite]), torch.nan_to_num(have[~finite]))
        assert ((have - want)[finite].abs() <= lost + 2.0 ** -24 * want[finite].abs()).all()
        if end_id is not None:
            ended = [r[2] == end_id or (finished is not None and bool(finished[i, r[1]])) for r in rows]
            assert got.finished[i].tolist() == ended
    if end_id is None:
        assert got.finished is None
    return got


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,K,V,keep", [(1, 1, 1, 1), (1, 1, 40, 32), (2, 3, 5, None), (3, 4, 1000, None), (1, 4, 30528, None), (2, 8, 4097, 16), (1, 32, 700, 32), (5, 5, 9000, 10),
                                        (1, 2, 131072, 4), (40, 8, 600, None), (2, 32, 33, None)])
def test_selection(B, K, V, keep, dtype):
    g = torch.Generator(device="cuda").manual_seed(B * V + K)
    logits = (torch.randn(B, K, V, device="cuda", generator=g) * 3).to(dtype)
    scores = -torch.rand(B, K, device="cuda", generator=g) * 5
    check(logits, scores, keep)
    end = V // 2
    finished = torch.rand(B, K, device="cuda", generator=g) < 0.4
    check(logits, scores, keep, finished, end)
    check(logits, scores, keep, None, end)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masks_ties_and_first_steps(dtype):
    B, K, V = 2, 4, 5000
    logits = torch.randn(B, K, V, device="cuda").to(dtype)
    logits[:, 1:] = logits[:, :1]                             # a first step: all beams alike
    scores = torch.tensor([[0.0, NONE, NONE, NONE], [-1.0, -1.0, -1.0, -1.0]], device="cuda")
    got = check(logits, scores, apart=False)
    assert (got.beam[0] == 0).all() and got.beam[1].tolist() == [0, 1, 2, 3]
    for lowest in (-1e9, -3.4e38):                            # masked by large numbers instead
        got = check(logits, torch.tensor([[0.0, lowest, lowest, lowest]] * 2, device="cuda"), apart=False)
        assert (got.beam == 0).all()
    tied = torch.zeros(1, 2, 3000, device="cuda", dtype=dtype)  # all equal: ascending ids, ascending beams
    got = check(tied, torch.zeros(1, 2, device="cuda"), 5, apart=False)
    assert got.token.tolist() == [[0, 1, 2, 3, 4]] and got.beam.tolist() == [[0] * 5]
    masked = torch.full((1, 2, 3000), NONE, device="cuda", dtype=dtype)
    masked[0, 1, 77] = 1.0                                    # one token is left, and fewer than wanted
    got = check(masked, torch.zeros(1, 2, device="cuda"), 4)
    assert got.token.tolist() == [[77, 0, 0, 0]] and got.beam.tolist() == [[1, 0, 0, 0]] and got.score[0, 0] == 0
    got = check(torch.full_like(masked, NONE), torch.zeros(1, 2, device="cuda"), 2, end_id=9)
    assert got.token.tolist() == [[9, 9]] and torch.isneginf(got.score).all()
    low = torch.full((1, 2, 3000), torch.finfo(dtype).min, device="cuda", dtype=dtype)
    low[0, 0, 5] = 2.0                                        # masked by the type's lowest value
    got = check(low, torch.zeros(1, 2, device="cuda"), 3, apart=False)
    assert got.token.tolist() == [[5, 0, 1]] and got.beam.tolist() == [[0, 1, 1]]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [700, 30528])
def test_nan_and_infinity_come_first(V, dtype):
    for value in (float("nan"), float("inf")):
        logits, scores = torch.randn(1, 3, V, device="cuda").to(dtype), torch.zeros(1, 3, device="cuda")
        logits[0, 1, 500] = value
        got = m2_b200.beam_select(logits, scores)
        assert got.beam.tolist() == [[1, 1, 1]] and got.token[0, 0] == 500 and torch.isnan(got.score).all()
    scores = torch.tensor([[0.0, float("nan"), 1.0]], device="cuda")
    got = m2_b200.beam_select(torch.randn(1, 3, V, device="cuda").to(dtype), scores, keep=1)
    assert got.beam.tolist() == [[1]] and torch.isnan(got.score).all()


def test_ended_beams():
    logits, scores = torch.randn(2, 3, 400, device="cuda"), torch.tensor([[-1.0, -2.0, -50.0], [0.5, -0.5, NONE]], device="cuda")
    logits[0, 0] = float("nan")                               # not read
    finished = torch.tensor([[True, False, False], [True, True, True]], device="cuda")
    got = check(torch.where(finished[..., None], torch.zeros_like(logits), logits), scores, 5, finished, 7)
    again = m2_b200.beam_select(logits, scores, keep=5, finished=finished, end_id=7)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    assert again.token[1].tolist() == [7] * 5 and again.beam[1].tolist() == [0, 1, 0, 0, 0] and again.finished[1].all()


def test_strides():
    logits = torch.randn(3, 4, 2001, device="cuda")
    scores = torch.randn(3, 4, device="cuda")
    ref = m2_b200.beam_select(logits, scores)
    padded = torch.zeros(3, 4, 2050, device="cuda")
    padded[..., 3:2004] = logits
    layouts = [padded[..., 3:2004], logits.transpose(0, 1).contiguous().transpose(0, 1), logits.transpose(1, 2).contiguous().transpose(1, 2)]
    for x in layouts:
        got = m2_b200.beam_select(x, scores.t().contiguous().t())
        assert torch.equal(got.beam, ref.beam) and torch.equal(got.token, ref.token) and (got.score - ref.score).abs().max() <= 80 * 2.0 ** -24 * 10
    alike = logits[:, :1].expand(3, 4, 2001)
    assert torch.equal(m2_b200.beam_select(alike, scores).token, m2_b200.beam_select(alike.contiguous(), scores).token)
    assert torch.equal(m2_b200.beam_select(logits, scores.double()).beam, ref.beam)
    big = torch.empty(2 ** 31 + 9000, dtype=torch.bfloat16, device="cuda")
    far = big.as_strided((2, 2, 2000), (2 ** 31 + 64, 2048, 1))
    far.copy_(logits[:2, :2, :2000])
    near = far.contiguous()
    assert all(torch.equal(a, b) for a, b in zip(m2_b200.beam_select(far, scores[:2, :2])[:3], m2_b200.beam_select(near, scores[:2, :2])[:3]))
    empty = m2_b200.beam_select(logits[:0], scores[:0], end_id=1)
    assert [tuple(t.shape) for t in empty] == [(0, 4)] * 4


@pytest.mark.parametrize("B,K", [(1, 1), (3, 2), (2, 4), (5, 5), (2, 8), (1, 13), (2, 32), (70, 3)])
def test_states_follow_their_beams(B, K):
    g = torch.Generator(device="cuda").manual_seed(B * K)
    states = [torch.randn(B * K, 70, 16, device="cuda"), torch.randn(B * K, 3, 70, device="cuda").bfloat16(), torch.randn(B * K, 5, device="cuda").half(),
              torch.randint(0, 99, (B * K,), device="cuda"), torch.randint(0, 99, (B * K, 7), device="cuda", dtype=torch.uint8), torch.randn(B * K, 0, 4, device="cuda"),
              torch.randn(B * K, 3, 1000, device="cuda")[:, 1], torch.randn(B * K, 1001, device="cuda")[:, 1:], torch.randn(B * K, 2, 33, device="cuda", dtype=torch.float64)]
    outside = [states[6]._base, states[7]._base]
    kept = [t.clone() for t in outside]
    for beam in (torch.randint(0, K, (B, K), device="cuda", generator=g), torch.arange(K, device="cuda").expand(B, K), torch.arange(K, device="cuda").flip(0).expand(B, K),
                 torch.full((B, K), K - 1, device="cuda"), torch.stack([torch.randperm(K, device="cuda") for _ in range(B)])):
        rows = (torch.arange(B, device="cuda")[:, None] * K + beam).flatten()
        want = [s[rows] for s in states]
        versions = [s._version for s in states]
        m2_b200.reorder_states(states, beam)
        assert all(torch.equal(a, b) for a, b in zip(states, want)) and all(s._version > v for s, v in zip(states, versions))
    assert torch.equal(outside[0][:, [0, 2]], kept[0][:, [0, 2]]) and torch.equal(outside[1][:, 0], kept[1][:, 0])
    assert ops.device_status() == 0


def test_layers_of_one_cache_and_many_states():
    cache = torch.randn(6, 12, 64, device="cuda")             # rows of twelve layers, side by side
    many = [torch.randn(6, 8, device="cuda") for _ in range(250)]
    beam = torch.tensor([[2, 2, 0], [1, 0, 1]], device="cuda")
    rows = torch.tensor([2, 2, 0, 4, 3, 4], device="cuda")
    want, wants = cache[rows], [t[rows] for t in many]
    m2_b200.reorder_states([cache[:, i] for i in range(12)] + many, beam)
    assert torch.equal(cache, want) and all(torch.equal(a, b) for a, b in zip(many, wants))
    single = torch.randn(6, 9, device="cuda")
    want = single[rows]
    m2_b200.reorder_states(single, beam)
    assert torch.equal(single, want)


def test_a_beam_that_is_none_is_clamped_and_reported():
    state = torch.arange(8.0, device="cuda")[:, None].repeat(1, 64)
    m2_b200.reorder_states([state], torch.tensor([[0, -3, 9, 2], [3, 3, 1 << 40, 0]], device="cuda"))
    assert state[:, 0].tolist() == [0, 0, 3, 2, 7, 7, 7, 4]
    assert ops.device_status() == 16 and ops.device_status() == 0


def test_states_far_apart():
    far = torch.empty(3 * (2 ** 30 + 64), dtype=torch.float32, device="cuda").view(3, -1)[:, :70]
    far.copy_(torch.randn(3, 70, device="cuda"))
    want = far[[2, 0, 0]]
    m2_b200.reorder_states([far], torch.tensor([[2, 0, 0]], device="cuda"))
    assert torch.equal(far, want)


def test_refusals_on_the_device():
    s = torch.randn(4, 6, device="cuda")
    beam = torch.zeros(2, 2, dtype=torch.long, device="cuda")
    for bad in ([s, s], [s, s[:, 1:]], [s.t().contiguous().t()], [torch.randn(1, 6, device="cuda").expand(4, 6)], [s, s.view(2, 12)[:, :6].repeat(2, 1)[:3]]):
        with pytest.raises(ValueError):
            m2_b200.reorder_states(bad, beam)
    with pytest.raises(RuntimeError, match="gradient"):
        m2_b200.reorder_states([s.clone().requires_grad_()], beam)
    logits, scores = torch.randn(2, 3, 50, device="cuda"), torch.zeros(2, 3, device="cuda")
    with pytest.raises(RuntimeError, match="gradient"):
        m2_b200.beam_select(logits.clone().requires_grad_(), scores)
    for wrong in (dict(keep=0), dict(keep=33), dict(end_id=-1), dict(finished=scores > 0), dict(finished=scores, end_id=1)):
        with pytest.raises(ValueError):
            m2_b200.beam_select(logits, scores, **wrong)
