"""Long sums whose roundings all go one way: softmax denominators of peaked and of rising rows, and parameters' gradients over long and over many sequences."""
import pytest
import torch

import m2_b200

pytestmark = pytest.mark.gpu
U32 = 2.0 ** -24


@pytest.fixture(autouse=True)
def seeded():
    with torch.random.fork_rng():                              # other files' random numbers are those they would have alone
        torch.manual_seed(0)
        yield


def score_errors(logits, keep=2):
    B, K, V = logits.shape
    got = m2_b200.beam_select(logits, torch.zeros(B, K, device="cuda"), keep=keep)
    lp = torch.log_softmax(logits.double(), -1)
    ref = lp[torch.arange(B, device="cuda")[:, None], got.beam, got.token]
    return (got.score.double() - ref).abs(), ref


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,K", [(1, 4), (40, 8)])              # a row is shared by blocks, and is not
@pytest.mark.parametrize("V", [30528, 131072])
def test_scores_of_peaked_and_rising_rows(B, K, V, dtype):
    """Every exponential is within 2 2^-24 of its own size (its argument's rounding is added back), sums of a piece's up to 8 take 3 more, and what follows is in 64
    bits: 5 2^-24 of the sum, below 2^-21, whatever the number of logits; the score itself is rounded once."""
    at = torch.arange(B * K, device="cuda").view(B, K, 1) * 3001 % V
    rows = []
    for high, low in ((0.0, -18.1), (2.2, -9.3), (1.7, -8.9), (30.3, 19.1), (0.1, 0.0)):
        x = torch.full((B, K, V), low, device="cuda")
        rows.append(x.scatter_(2, at, high))
    rows.append((torch.arange(V, device="cuda") * 2.0 ** -20).expand(B, K, V).contiguous())
    rows.append((torch.arange(V, device="cuda") * 2.0 ** -10).expand(B, K, V).contiguous())
    rows.append((torch.arange(V, device="cuda") * -2.0 ** -14).expand(B, K, V).contiguous())
    rows.append(torch.randn(B, K, V, device="cuda", generator=torch.Generator(device="cuda").manual_seed(V)) * 4)
    worst = []
    for x in rows:
        off, ref = score_errors(x.to(dtype))
        worst.append(((off - U32 * ref.abs()) / 2.0 ** -21).max().item())
    assert max(worst) <= 1, worst


# 1 + 2^-12 + 2^-14, four thousand times one by one in float32, is off by 0.75, three eighths of a step of the sum each time
ODD = 1 + 2.0 ** -12 + 2.0 ** -14


@pytest.mark.parametrize("B,L,D", [(56, 8192, 2048), (65536, 16, 8), (2, 8192, 64)])   # a thread for each long sequence; many short ones; cut
def test_taps_gradients_over_long_and_many_sequences(B, L, D):
    """A thread adds at most 256 tokens in float32 (256 2^-24 of the sum, were all roundings to go one way), the threads' sums are added in 64 bits."""
    x = torch.ones(1, 1, D, device="cuda").expand(B, L, D)
    w, bias = torch.zeros(D, 4, device="cuda", requires_grad=True), torch.zeros(D, device="cuda", requires_grad=True)
    y = m2_b200.causal_conv(x, w, bias)
    d_w, d_b = torch.autograd.grad(y, [w, bias], torch.full((1, 1, D), ODD, device="cuda").expand(B, L, D))
    for i in range(4):
        n = B * (L - (3 - i))
        assert (d_w[:, i].double() - n * ODD).abs().max() <= 257 * U32 * n * ODD
    assert (d_b.double() - B * L * ODD).abs().max() <= 257 * U32 * B * L * ODD


@pytest.mark.parametrize("B,L,D,N", [(32768, 2, 8, 4), (8192, 40, 8, 20)])
def test_parameters_gradients_of_scans_over_many_sequences(B, L, D, N):
    """The sums of the sequences are added in 64 bits; within one there are L terms."""
    x = torch.ones(1, 1, 1, device="cuda").expand(B, L, D)
    b = torch.ones(1, 1, 1, device="cuda").expand(B, L, N)
    a, skip, bias = torch.zeros(D, N, device="cuda", requires_grad=True), torch.zeros(D, device="cuda", requires_grad=True), torch.zeros(D, device="cuda", requires_grad=True)
    initial = torch.ones(1, 1, 1, device="cuda").expand(B, D, N)
    y = m2_b200.selective_scan(x, x, a, b, b, skip=skip, delta_bias=bias, initial_state=initial)
    grads = torch.autograd.grad(y, [a, skip, bias], torch.full((1, 1, 1), ODD, device="cuda").expand(B, L, D))
    t = torch.arange(1, L + 1, dtype=torch.float64)
    # steps 1 and no fading: h_t = 1 + t, dy_t / da = sum_{s <= t} h_{s-1} = sum_{s <= t} s, dy_t / dstep_s = 1 a state for s <= t
    want = [B * ODD * (t * (t + 1) / 2).sum().item(), B * L * ODD, B * ODD * N * t.sum().item()]
    for got, ref in zip(grads, want):
        assert (got.double() - ref).abs().max() <= (2 * L + N + 8) * U32 * ref


def test_gradients_along_a_long_axis_are_handed_on_by_tiles():
    """The gradient of the initial state through 16384 tokens that hardly fade, in two segments, all terms of one sign: every tile of 32 tokens of a segment rounds what it
    carries by its decays' 2^-22 and two roundings more, and its own terms by 40 of each; token by token the same decay's rounding, up to 2^-25, would come 8192 times."""
    L, G, N = 16384, 200, 16
    delta = torch.ones(1, 1, G, device="cuda").expand(1, L, G)
    a = -(torch.arange(1, N + 1, device="cuda") * 2.0 ** -15 * 1.1).expand(G, N).contiguous()
    b, c = torch.zeros(1, 1, G, N, device="cuda").expand(1, L, G, N), torch.ones(1, 1, G, N, device="cuda").expand(1, L, G, N)
    initial = torch.zeros(1, G, N, device="cuda", requires_grad=True)
    y = m2_b200.selective_scan(delta, delta, a, b, c, initial_state=initial)
    (got,) = torch.autograd.grad(y, [initial], torch.ones_like(y))
    ages = torch.arange(1, L + 1, dtype=torch.float64, device="cuda")
    terms = torch.exp(a.double()[0, :, None] * ages)
    ref, age = terms.sum(1), (terms * (ages % (L // 2))).sum(1) / terms.sum(1)          # of the terms within their segments
    off = ((got[0].double() - ref).abs() / ref).amax(0)
    bound = age / 32 * (2.0 ** -22 + 2 * U32) + 40 * U32
    assert (off <= bound).all(), (off / bound).tolist()
