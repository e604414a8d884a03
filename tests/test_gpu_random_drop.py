"""dropout: which elements are kept is decided by Philox 4x32-10, written here once more with Python's integers; kept values are one product and one sum in float32."""
import gc

import pytest
import torch

import m2_b200

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def seeded():
    torch.manual_seed(0)


U32, U16 = 2.0 ** -24, 2.0 ** -8


def philox(counter, key):
    """The published generator for one block (counter: four words, key: two)."""
    c, k, low = list(counter), list(key), (1 << 32) - 1
    for _ in range(10):
        p, q = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(q >> 32) ^ c[1] ^ k[0], q & low, (p >> 32) ^ c[3] ^ k[1], p & low]
        k = [(k[0] + 0x9E3779B9) & low, (k[1] + 0xBB67AE85) & low]
    return c


def kept(n, p, seed, call=0):
    low, out = (1 << 32) - 1, []
    for j in range((n + 7) // 8):
        for w in philox([j & low, j >> 32, call & low, call >> 32], [seed & low, seed >> 32]):
            out += [w & 0xffff, w >> 16]
    return torch.tensor(out[:n], device="cuda") >= round(p * 65536)


def test_the_generator_gives_its_published_numbers():
    assert philox([0] * 4, [0] * 2) == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]
    assert philox([0xffffffff] * 4, [0xffffffff] * 2) == [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (9,), (3, 5), (2, 33, 24), (5000,), (1, 4099)])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 0.999, 1.0])
def test_values_and_gradients(shape, dtype, p):
    x, r = (torch.randn(shape, device="cuda").to(dtype).requires_grad_() for _ in range(2))
    seed, call = 0x123456789abcdef0, 0xfedcba987654321
    for s, res in ((seed, None), (seed, r), (torch.tensor([seed, call], device="cuda"), r), ((1 << 64) - 1, None), (-1, None)):
        number = (call if isinstance(s, torch.Tensor) else 0)
        mask = kept(x.numel(), p, seed if isinstance(s, torch.Tensor) else s & ((1 << 64) - 1), number).view(shape)
        t = round(p * 65536)
        scale = 65536 / (65536 - t) if t < 65536 else 0.0
        y = m2_b200.dropout(x, p, s, residual=res)
        ref = torch.where(mask, x.double() * scale, 0.0)
        size = ref.abs() * 3 * U32                              # the scale, the product and the sum
        if res is not None:
            ref = ref + r.double()
        assert y.dtype == dtype and ((y.double() - ref).abs() <= (U16 if dtype == torch.bfloat16 else U32) * ref.abs() + size).all()
        up = torch.randn_like(y)
        d = torch.autograd.grad(y, [x] + ([r] if res is not None else []), up)
        ref = torch.where(mask, up.double() * scale, 0.0)
        assert ((d[0].double() - ref).abs() <= ((U16 if dtype == torch.bfloat16 else U32) + 3 * U32) * ref.abs()).all() and (d[0][~mask] == 0).all()
        if res is not None:
            assert torch.equal(d[1], up)


def test_what_is_dropped_is_zero_whatever_it_was():
    x = torch.full((1000,), float("nan"), device="cuda")
    y = m2_b200.dropout(x, 0.5, 3)
    mask = kept(1000, 0.5, 3)
    assert torch.isnan(y[mask]).all() and not y[~mask].any()
    assert not m2_b200.dropout(torch.full((100,), float("inf"), device="cuda"), 1.0, 3).any()


def test_one_mask_for_every_type_stride_and_split():
    x = torch.ones(6, 50, 40, device="cuda")
    base = m2_b200.dropout(x, 0.3, 11) != 0
    assert torch.equal(m2_b200.dropout(x.bfloat16(), 0.3, 11) != 0, base)
    assert torch.equal(m2_b200.dropout(x.transpose(0, 2).contiguous().transpose(0, 2), 0.3, 11) != 0, base)
    assert torch.equal(m2_b200.dropout(torch.ones(7, 50, 40, device="cuda")[1:], 0.3, 11) != 0, base)
    odd = torch.ones(6 * 50 * 40 + 1, device="cuda")[1:].view(6, 50, 40)       # off 16 bytes
    assert torch.equal(m2_b200.dropout(odd, 0.3, 11) != 0, base) and torch.equal(m2_b200.dropout(odd.bfloat16(), 0.3, 11) != 0, base)
    other = m2_b200.dropout(x, 0.3, 12) != 0
    both = (other & base).float().mean()
    assert abs(both - 0.49) < 5 * (0.49 * 0.51 / x.numel()) ** 0.5              # five deviations of as many independent draws


def test_the_share_that_is_kept():
    n = 1 << 24
    for p in (0.1, 0.5):
        share = (m2_b200.dropout(torch.ones(n, device="cuda"), p, 5) != 0).double().mean()
        q = 1 - round(p * 65536) / 65536
        assert abs(share - q) < 6 * (q * (1 - q) / n) ** 0.5


def test_far_elements():
    n = 2 ** 31 + 4096
    x = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    x[-1000:] = 1
    y = m2_b200.dropout(x, 0.5, 77)
    start = (n - 1000) // 8
    low, bits = (1 << 32) - 1, []
    for j in range(start, (n + 7) // 8):
        for w in philox([j & low, j >> 32, 0, 0], [77, 0]):
            bits += [w & 0xffff, w >> 16]
    mask = torch.tensor(bits[n - 1000 - start * 8:][:1000], device="cuda") >= 32768
    assert torch.equal(y[-1000:] != 0, mask)


def test_a_captured_step_drops_other_elements_in_every_replay():
    gc.collect()
    x = torch.ones(4096, device="cuda", requires_grad=True)
    seed = torch.tensor([9, 0], device="cuda")
    d = torch.zeros(4096, device="cuda")

    def step():
        y = m2_b200.dropout(x, 0.25, seed)
        d.copy_(torch.autograd.grad(y.sum(), [x])[0])
        seed[1] += 1
        return y.detach()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step()
    for call in (1, 2, 3):
        graph.replay()
        mask = kept(4096, 0.25, 9, call)
        assert torch.equal(y != 0, mask) and torch.equal(d != 0, mask)
    # a seed that changes between the two passes is found out
    y = m2_b200.dropout(x, 0.25, seed)
    seed[1] += 1
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y.sum(), [x])


def test_empty():
    x = torch.zeros(0, 5, device="cuda", requires_grad=True)
    y = m2_b200.dropout(x, 0.5, 1)
    assert y.shape == (0, 5) and torch.autograd.grad(y.sum(), [x])[0].shape == (0, 5)
