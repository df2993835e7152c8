"""How exact the vocabulary loss is for float32 tensors: relative 2-norms of its outputs against 64 bits, with a limit that
products left out and sums left to the tensor cores' truncating adder do not keep.

LIMIT = 2^-19: a run of 32 truncating additions loses half a last bit, 2^-24 of the sum, in each on average, 32 * 2^-24 where all of
them carry the whole sum; the products that are left out (2^-24 on average), exponentials and logits that are off by some 2^-21 in a part of the
slope only, and the rounding of the runs' sums (U each) are small beside that, since no output's sum is at its full size in every step."""
import pytest
import torch

LIMIT = 2.0 ** -19


def distance(got, want):
    return float((got.double() - want).norm() / want.norm())


# ------------------------------------------------------------------------------ the limit itself, on the CPU
def cut(v, bits):
    """Towards zero to so many significant bits."""
    mantissa, exponent = torch.frexp(v)
    return torch.ldexp((mantissa * 2.0 ** bits).trunc(), exponent - bits)


def planes(v):
    """The three bf16 planes of float32 values, in float64."""
    hi = cut(v.double(), 8)
    mid = cut(v.double() - hi, 8)
    return hi, mid, v.double() - hi - mid


ALL = ((0, 0), (0, 1), (1, 0), (1, 1), (0, 2), (2, 0))


def emulated(a, b, products=ALL, run=32):
    """a @ b as the kernel forms it: 16 terms a step, hi x hi and the smaller products in a 24-bit sum each that is cut after
    every step, the sums of `run` steps added in float32."""
    pa, pb = planes(a), planes(b)
    total = torch.zeros(len(a), b.shape[1])
    for first in range(0, a.shape[1], 16 * run):
        sums = [torch.zeros(len(a), b.shape[1], dtype=torch.float64) for _ in range(2)]
        for k in range(first, min(first + 16 * run, a.shape[1]), 16):
            for i, j in products:
                which = 0 if i + j == 0 else 1
                sums[which] = cut(sums[which] + pa[i][:, k:k + 16] @ pb[j][k:k + 16], 24)
        total = total + (sums[0].float() + sums[1].float())
    return total


def slope_and_weight(words=10007):
    """s of some rows and weights, as they meet in d_hidden."""
    g = torch.Generator().manual_seed(0)
    s = torch.softmax(torch.randn(12, words, generator=g) * 2, 1)
    s[torch.arange(12), torch.randint(0, words // 3, (12,), generator=g)] -= 1
    return s, torch.randn(words, 10, generator=g)


def test_planes_are_the_number():
    v = torch.randn(1000, generator=torch.Generator().manual_seed(1)) * 10.0 ** torch.linspace(-20, 20, 1000)
    assert torch.equal(sum(planes(v)), v.double())
    assert all(torch.equal(p.to(torch.bfloat16).double(), p) for p in planes(v))


def test_limit_tells_the_kernels_arithmetic_from_less():
    s, w = slope_and_weight()
    want = s.double() @ w.double()
    assert distance(emulated(s, w), want) < LIMIT
    # the three smallest products left out, all but hi x hi, and sums that stay in the truncating adder
    assert distance(emulated(s, w, ALL[:3]), want) > LIMIT
    assert distance(emulated(s, w, ALL[:1]), want) > LIMIT
    assert distance(emulated(s, w, run=1 << 20), want) > LIMIT


@pytest.mark.parametrize("depth", [515, 2048])
def test_limit_tells_products_of_logits(depth):
    g = torch.Generator().manual_seed(2)
    h, w = torch.randn(12, depth, generator=g), torch.randn(depth, 10, generator=g)
    want = h.double() @ w.double()
    assert distance(emulated(h, w), want) < LIMIT
    assert distance(emulated(h, w, ALL[:3]), want) > LIMIT


# ------------------------------------------------------------------------------ the kernels
@pytest.mark.gpu
@pytest.mark.parametrize("rows,width,vocab", [(64, 48, 10007), (777, 515, 10007), (4500, 48, 900), (2048, 1024, 4000), (40, 2048, 700)])
def test_float32_outputs_are_exact_to_the_limit(built_library, rows, width, vocab):
    import deepity_b200 as dp
    g = torch.Generator(device="cuda").manual_seed(rows)
    hidden, bias = torch.randn(rows, width, generator=g, device="cuda"), torch.randn(vocab, generator=g, device="cuda")
    weight = torch.randn(vocab, width, generator=g, device="cuda") * (2.0 / width ** 0.5)
    targets = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    grad = torch.linspace(0.5, 2.0, rows, device="cuda") / rows
    logits = hidden.double() @ weight.double().T + bias.double()
    s = torch.softmax(logits, 1)
    s[torch.arange(rows, device="cuda"), targets] -= 1
    s *= grad.double()[:, None]
    loss, lse = dp.vocab_cross_entropy(hidden, weight, targets, bias)
    got = dp.vocab_cross_entropy_backward(grad, hidden, weight, targets, lse, bias)
    assert distance(lse, torch.logsumexp(logits, 1)) < LIMIT
    assert distance(got.hidden, s @ weight.double()) < LIMIT
    assert distance(got.weight, s.T @ hidden.double()) < LIMIT
    assert distance(got.bias, s.sum(0)) < LIMIT


@pytest.mark.gpu
@pytest.mark.parametrize("rows,width", [(5, 1000), (40, 515), (300, 2048)])
def test_float32_logits_are_exact_to_the_limit(built_library, rows, width):
    """With every other word out the logarithm of the sum is the one logit left."""
    import deepity_b200 as dp
    g = torch.Generator(device="cuda").manual_seed(width)
    hidden, weight = (torch.randn(n, width, generator=g, device="cuda") for n in (rows, 500))
    targets = torch.zeros(rows, device="cuda", dtype=torch.int64)
    found = []
    for word in (0, 77, 300, 499):
        bias = torch.full((500,), -float("inf"), device="cuda")
        bias[word] = 0.0
        found.append(dp.vocab_cross_entropy(hidden, weight, targets, bias)[1])
    want = hidden.double() @ weight[[0, 77, 300, 499]].double().T
    assert distance(torch.stack(found, 1), want) < LIMIT
