"""f32 heads are multiplied as sums of three bf16 numbers, six products of nine. Here every result is ONE product of two f32
numbers (all others are zeros), so that each of the six shows: the smallest are up to 2^-16 or 2^-17 of the whole, and a bound of
2^-21 tells when one is missing, which the sum of many products' absolute values would hide."""
import pytest
import torch

import hiptensor_b200 as ht

IGNORE = -100
PAIRS = [(0, 2), (1, 1), (2, 0), (0, 1), (1, 0), (0, 0)]
# A bf16 number of 8 bits next to x in [1, 2) is off by at most half a step, 2^-8; what is left, below 2^-8, has steps of 2^-16, so
# its bf16 number is off by at most 2^-17; the third part is exact. What is left out, (1, 2), (2, 1) and (2, 2): 2^-8 * 2^-17,
# twice, and 2^-34. Added up in the tensor cores, small products first: truncated where the last and largest comes in, 2^-23, and
# the smaller ones' truncations, 2^-8 of that, twice; one rounding of the sum of the chunks and one of the result, 2^-24 each.
LEFT_OUT = 2.0 ** -24 + 2.0 ** -34
BOUND = LEFT_OUT + 2.0 ** -23 * (1 + 2.0 ** -7) + 2 * 2.0 ** -24


def numbers(*shape, seed, device):
    """+-[1, 2), all mantissas."""
    g = torch.Generator(device=device).manual_seed(seed)
    x = 1 + torch.rand(shape, generator=g, device=device)
    return torch.where(torch.rand(shape, generator=g, device=device) < 0.5, x, -x)


def parts(x):
    out = []
    for _ in range(3):
        out.append(x.bfloat16().float())
        x = x - out[-1]
    return out


@pytest.mark.parametrize("missing", [None] + PAIRS)
def test_the_bound_tells_a_missing_product(missing):
    a, b = numbers(300, seed=1, device="cpu"), numbers(300, seed=2, device="cpu")
    x, y = parts(a), parts(b)
    got = sum(x[i].double() * y[j].double() for i, j in PAIRS if (i, j) != missing)
    exact = a.double() * b.double()
    off = float(((got - exact) / exact).abs().max())
    assert off <= LEFT_OUT if missing is None else off > 4 * BOUND


def desc(h, x):
    return h.tensor_descriptor(x.shape, x.stride(), ht.R_32F)


def space(h, plan, gradient):
    n = h.cross_entropy_workspace_size(plan, gradient)
    return torch.full((n,), 0xFF, device="cuda", dtype=torch.uint8), n


@pytest.mark.gpu
@pytest.mark.parametrize("t", [3, 9, 40, 200, 300])
@pytest.mark.parametrize("v,d", [(2, 24), (300, 200), (700, 1100)])
def test_a_logit_of_one_product(t, v, d):
    """The class in the middle has logits of 32 to 128 and all others 0: the loss of another class is the logit."""
    h = ht.Handle()
    w = numbers(d, seed=3, device="cuda")
    at = torch.arange(t, device="cuda") * 37 % d
    H, W = torch.zeros(t, d, device="cuda"), torch.zeros(v, d, device="cuda")
    W[v // 2] = w
    x = numbers(t, seed=4, device="cuda").abs() * w[at].sign()
    H[torch.arange(t, device="cuda"), at] = x
    y = torch.full((t,), (v // 2 + 1) % v, device="cuda")
    loss, lse = torch.empty(t, device="cuda"), torch.empty(t, device="cuda")
    plan = h.cross_entropy_plan(desc(h, H), (0, 2), desc(h, W), (1, 2), IGNORE)
    h.cross_entropy(plan, 32.0, H, W, y, loss, lse, *space(h, plan, False))
    want = 32 * x.double() * w[at].double()
    # the other classes add at most v e^-32; alpha is exact; the loss is rounded once more
    bound = (BOUND + 2.0 ** -24) * want + v * 1.3e-14
    for got in (loss, lse):
        assert bool(((got.double() - want).abs() <= bound).all()), float(((got.double() - want).abs() / bound).max())


@pytest.mark.gpu
@pytest.mark.parametrize("t", [3, 9, 40, 200, 300])
@pytest.mark.parametrize("v,d", [(300, 24), (777, 200), (1031, 1100)])
def test_gradients_of_one_product(t, v, d):
    """An lse far above every logit leaves the target's entry, -gradLoss, alone in each row of P; every token has a class of its own."""
    h = ht.Handle()
    H, W, g = numbers(t, d, seed=5, device="cuda"), numbers(v, d, seed=6, device="cuda"), numbers(t, seed=7, device="cuda")
    y = torch.arange(t, device="cuda") * 11 % v  # (no v is a multiple of 11)
    assert len(set(y.tolist())) == t
    lse = torch.full((t,), 1e4, device="cuda")
    dH, dW = torch.empty_like(H), torch.empty_like(W)
    plan = h.cross_entropy_plan(desc(h, H), (0, 2), desc(h, W), (1, 2), IGNORE)
    h.cross_entropy_gradient(plan, 1.0, H, W, y, lse, g, dH, dW, *space(h, plan, True))
    for got, other in ((dH, W[y]), (dW[y], H)):
        want = -g.double()[:, None] * other.double()
        off = ((got.double() - want) / want).abs()
        assert bool((off <= BOUND).all()), float(off.max() / BOUND)
    dW[y] = 0
    assert not bool(dW.any())
