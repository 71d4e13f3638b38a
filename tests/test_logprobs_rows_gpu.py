"""token_logprobs on the GPU row by row: every row against a bound of its own, formed of the terms that are rounded for that row, so that a row
of large or lowest values says nothing about the others."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24      # half a step of fp32, relative


def check_rows(got, z, tokens, top, steps):
    """got of z [M, V] against float64, on the GPU too.  With u = 2^-24, d = max - logit, p the probabilities, D and D2 the sums of p d and
    p d^2, and to first order:
      an exponential     the difference u d, the product with log2 e 1.25 u d, the exponential of 2 itself 2 u:  (2.25 d + 2) u
      its way to the sum where sums are joined under a larger maximum, another factor of that kind (its d's add up to d), a product and an
                         addition: 4 u a step; a tree of up to 16 values 4 u, a compensated sum over tiles 2 u.  `steps`: as often as a
                         thread's maximum rises, 8 that make threads to a row, 8 more where it is in pieces:
                         log sum off by  (2.25 D + 8 + 4 steps) u =: S
      a log probability  S, the difference u d, the logarithm 2 u |log sum|, the result u |log p|
      the entropy        S, 2 u |log sum|, the result u; and of the quotient sum p d its terms (2.25 d + 2.25 for the factor, 1 for its product),
                         their way (as above) and the sum it is divided by:  (2.25 D2 + 3.25 D + D (8 + 4 steps) + D S / u + 2 D) u
    Masked logits (p = 0) add nothing to D and D2."""
    x = z.double()
    lp = torch.log_softmax(x, 1)
    p = lp.exp()
    most = x.amax(1)
    d = torch.where(p > 0, most[:, None] - x, torch.zeros_like(x))
    D, D2 = (p * d).sum(1), (p * d * d).sum(1)
    entropy = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(1)
    log_sum = torch.logsumexp(x - most[:, None], 1)
    S = 2.25 * D + 8 + 4 * steps

    def close(a, b, tol):
        a = a.double()
        assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.isinf(), b.isinf())
        ok = torch.isfinite(b)
        over = torch.where(ok, (a - b).abs() - tol * U, torch.full_like(b, -1.0))
        assert (over <= 0).all(), (over.argmax().item(), float((a - b)[ok].abs().max()), float(over.max()))

    def log_probability(a, at, expected):
        gap = most[:, None] - x.gather(1, at)
        close(a, expected, S[:, None] + gap + 2 * log_sum.abs()[:, None] + expected.abs())

    pad = (tokens < 0) | (tokens >= z.shape[1])
    at = tokens.clamp(0, z.shape[1] - 1)[:, None]
    given = lp.gather(1, at)
    log_probability(torch.where(pad, given[:, 0], got.logprobs.double())[:, None], at, given)
    assert (got.logprobs[pad] == 0).all() and (got.ranks[pad] == 0).all()
    if top:
        order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top]
        assert torch.equal(got.top_ids, order)
        log_probability(got.top_logprobs, order, lp.gather(1, order))
    close(got.entropy, entropy, S + 2 * log_sum.abs() + entropy + 2.25 * D2 + D * (3.25 + 8 + 4 * steps + S + 2))


def scores(z, tokens, top):
    from tyloquant_amd import runtime as R
    return R.token_logprobs(z, tokens, top)


def first(got, n):
    return type(got)(*(part[:n] for part in got))


def logits(seed, M, V, dtype):
    g = torch.Generator(device="cuda").manual_seed(seed)
    z = torch.randn(M, V, generator=g, device="cuda")
    return (z * z.abs() * 0.75 + 1.5).to(dtype), torch.randint(0, V, (M,), generator=g, device="cuda")


def few_values(seed, V, gap):
    """a row of two values, the larger at some 1500 places, so that every thread of a block has met one in its first tile"""
    g = torch.Generator(device="cuda").manual_seed(seed)
    z = torch.full((V,), -gap, device="cuda")
    z[torch.randperm(V, generator=g, device="cuda")[:1024]] = 0.0
    z[:2048:4] = 0.0
    return z


@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_rows_of_few_values(dtype):
    """long rows of equal values, a block each and in pieces: what one addition loses every other may lose too"""
    V, M = 151936, 1025
    rows = torch.stack([few_values(i, V, gap) for i, gap in enumerate((0.0, 0.3, 1.0, 2.7, 4.0, 5.3, 7.7, 9.1, 11.0, 12.5))]).to(dtype)
    n = len(rows)
    tokens = torch.arange(n, device="cuda") * 4             # of the larger value
    check_rows(scores(rows, tokens, 3), rows, tokens, 3, 1 + 16)
    many = scores(rows.repeat(-(-M // n), 1)[:M], tokens.repeat(-(-M // n))[:M], 3)
    for part in many:                                       # rows of a kind alike
        assert all((part[k::n] == part[k]).all() for k in range(n))
    check_rows(first(many, n), rows, tokens, 3, 8)


@pytest.mark.parametrize("M,V", [(1030, 151936), (1030, 50001), (6, 151936), (40, 32000)])
@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
def test_random_rows(dtype, M, V):
    """peaked rows as a head leaves them; of many rows the first forty by their bounds"""
    z, tokens = logits(V, M, V, dtype)
    got, n = scores(z, tokens, 5), min(M, 40)
    check_rows(first(got, n), z[:n], tokens[:n], 5, -(-V // 2048) + 16)


@pytest.mark.parametrize("V", [100, 9000, 70000])
@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("copies", [1, 110])
def test_masked_rows_and_ties(V, dtype, copies):
    """rows masked but for a few or one, all equal, ties, the lowest value as a mask, ascending and descending: each by its own bound"""
    z, tokens = logits(3, 10, V, dtype)
    z[0, : V - 3] = -math.inf
    z[1, :] = -math.inf
    z[1, V - 1] = 2.0
    z[2, 5:] = -math.inf
    z[3, :] = 1.25
    z[4] = (torch.arange(V, device="cuda") % 7).to(dtype)
    z[5, V // 2:] = torch.finfo(dtype).min
    z[6, : V // 3] = -math.inf
    z[7] = torch.arange(V, device="cuda").flip(0).to(dtype)
    z[8] = torch.arange(V, device="cuda").to(dtype)
    z[9, ::2] = 0.0
    z[9, 1::2] = -0.0
    tokens[0] = tokens[1] = V - 1
    tokens[2] = 7       # a masked one
    tokens[4], tokens[5] = V, -1
    z, tokens = z.repeat(copies, 1), tokens.repeat(copies)
    check_rows(scores(z, tokens, 20), z, tokens, 20, -(-V // 2048) + 16)


@pytest.mark.parametrize("copies", [1, 180])
def test_rows_far_from_zero(copies):
    """an offset that all logits of a row share is no part of its bound; rows so wide that few exponentials are left"""
    g = torch.Generator(device="cuda").manual_seed(5)
    z = torch.randn(6, 30000, generator=g, device="cuda")
    tokens = torch.randint(0, 30000, (6,), generator=g, device="cuda")
    z[0] *= 1000
    z[1] += 1.0e6
    z[2] -= 3.0e4
    z[3] *= 1e-6
    z[4] = z[4] * 40 - 500
    z[5, 11] = 90.0
    z, tokens = z.repeat(copies, 1), tokens.repeat(copies)
    check_rows(scores(z, tokens, 5), z, tokens, 5, 15 + 16)


def test_rows_of_equal_logits():
    """log softmax and entropy of V equal logits are log V: sums of ones are exact, what is left is one logarithm, off by one step at most
    (2^-23 relative)"""
    wrong = []
    for V in [*range(2, 200, 7), *range(1000, 160000, 2111)]:
        z = torch.zeros(1, V, device="cuda")
        got = scores(z, torch.zeros(1, dtype=torch.int64, device="cuda"), 1)
        for value, want in ((got.logprobs, -math.log(V)), (got.entropy, math.log(V)), (got.top_logprobs, -math.log(V))):
            if abs(float(value) - want) > 2 * U * math.log(V):
                wrong.append((V, float(value) - want))
    assert not wrong, wrong
