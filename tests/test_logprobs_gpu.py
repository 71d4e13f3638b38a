"""token_logprobs on the GPU against log-softmax in float64: every type, lengths, masks that leave a row little or nothing, ties, padding."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def oracle(z, tokens, top):
    """in float64, on the CPU; ids by a stable sort: of equal logits the lower token first.  Ranks go by the differences to the largest logit as
    fp32 has them."""
    z = z.detach().cpu().float().reshape(-1, z.shape[-1])
    below = z - torch.where(z.isnan(), -math.inf, z).amax(1, keepdim=True)
    z = z.double()
    tokens = tokens.cpu().reshape(-1)
    lp = torch.log_softmax(z, 1)
    p = lp.exp()
    entropy = -torch.where(p > 0, p * lp, torch.where(lp.isnan(), lp, torch.zeros_like(p))).sum(1)
    pad = (tokens < 0) | (tokens >= z.shape[1])
    at = tokens.clamp(0, z.shape[1] - 1)[:, None]
    given = z.gather(1, at)
    logprob = torch.where(pad, torch.zeros(1, dtype=torch.float64), lp.gather(1, at)[:, 0])
    rank = torch.where(pad, 0, 1 + (below > below.gather(1, at)).sum(1))
    order = torch.sort(torch.where(z.isnan(), -math.inf, z), dim=1, descending=True, stable=True).indices
    last = torch.sort(z.isnan().gather(1, order).int(), dim=1, stable=True).indices      # NaN behind -infinity too
    order = order.gather(1, last)[:, :top]
    return logprob, rank, entropy, order, lp.gather(1, order)


def check(z, tokens, top):
    """fp32: the exponentials and their sum are off by a few 2^-24 (rounded product 2^-24 of an argument up to 88, corrected to first order;
    exponential 2^-23; 32 + 8 sums a thread and wave), 2^-20 in all; the logarithm and the two differences round at the size of their terms."""
    from tyloquant_amd import runtime as R
    got = R.token_logprobs(z, tokens, top)
    logprob, rank, entropy, order, best = oracle(z, tokens, top)
    lead = tuple(z.shape[:-1])
    assert tuple(got.logprobs.shape) == tuple(got.ranks.shape) == tuple(got.entropy.shape) == lead and tuple(got.top_ids.shape) == lead + (top,)
    assert got.ranks.dtype == got.top_ids.dtype == torch.int64 and got.logprobs.dtype == got.entropy.dtype == got.top_logprobs.dtype == FP32
    finite = z.double()[torch.isfinite(z)]
    size = float(finite.abs().max()) if finite.numel() else 1.0
    tol = 2.0 ** -20 + 4 * 2.0 ** -24 * size

    def close(a, b, scale=1.0):
        a, b = a.cpu().double().reshape(b.shape), b
        assert torch.equal(a.isnan(), b.isnan())
        assert torch.equal(a.isinf(), b.isinf())
        ok = torch.isfinite(b)
        assert ((a - b)[ok].abs() <= tol * scale + 4 * 2.0 ** -24 * b[ok].abs()).all(), float((a - b)[ok].abs().max())

    close(got.logprobs, logprob)
    close(got.entropy, entropy, 1.0 + 2 * math.log(z.shape[-1] + 1))      # its terms are weighted by up to that many nats
    close(got.top_logprobs, best)
    finite_rows = ~entropy.isnan()
    assert torch.equal(got.ranks.cpu().reshape(-1)[finite_rows], rank[finite_rows])
    assert torch.equal(got.top_ids.cpu().reshape(order.shape), order)
    return got


def logits(seed, M, V, dtype, peaked=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    z = torch.randn(M, V, generator=g, device="cuda")
    if peaked:
        z = z * z.abs() * 0.75 + 1.5
    return z.to(dtype), torch.randint(0, V, (M,), generator=g, device="cuda")


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("M,V,top", [(1, 1, 1), (1, 2, 0), (3, 63, 20), (2, 64, 64), (5, 1000, 64), (7, 8192, 5), (1, 8193, 20), (1, 151936, 20), (4, 40001, 7),
                                     (33, 32000, 1), (300, 16384, 5), (1025, 9000, 3), (1, 400000, 64)])
def test_sizes(dtype, M, V, top):
    check(*logits(M + V, M, V, dtype), top)


@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_layouts(dtype):
    z, tokens = logits(1, 12, 5000, dtype)
    want = check(z[:, 8:4000], tokens % 3992, 5)
    check(z[:, 1:4000], tokens % 3999, 5)
    check(z[::2], tokens[::2], 9)
    check(z.reshape(3, 4, 5000), tokens.reshape(3, 4), 3)
    check(z[:1].expand(12, 5000), tokens, 4)
    check(logits(2, 5000, 6, dtype)[0].t(), tokens[:6], 4)
    check(z[0], tokens[0], 5)
    assert tuple(check(z[:0], tokens[:0], 5).top_ids.shape) == (0, 5)
    again = check(z[:, 8:4000].contiguous(), tokens % 3992, 5)
    assert all(torch.equal(a, b) for a, b in zip(want, again))


@pytest.mark.parametrize("V", [100, 9000, 70000])
@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_masks_and_ties(V, dtype):
    """rows masked but for a few, one or none; all equal; long runs of ties; the type's lowest value as a mask"""
    z, tokens = logits(3, 10, V, dtype)
    z[0, :] = -math.inf
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
    tokens[1] = V - 1
    tokens[2] = 7       # a masked one
    check(z, tokens, 20)
    check(z, tokens, 1)


def test_padding_infinities_and_nan():
    z, tokens = logits(4, 8, 20000, FP32)
    tokens[0], tokens[1], tokens[2] = -100, 20000, -1
    z[3, 77] = math.inf
    z[4, 19999] = math.nan
    z[5, :] = math.nan
    z[6, 3] = math.nan
    z[6, 4:] = -math.inf
    check(z, tokens, 10)


def test_wide_rows_of_one_size():
    """spread so wide that all but a few exponentials are zero, and logits far from zero"""
    z, tokens = logits(5, 6, 30000, FP32, peaked=False)
    z[0] *= 1000
    z[1] += 1.0e6
    z[2] -= 3.0e4
    z[3] *= 1e-6
    z[4] = z[4] * 40 - 500
    z[5, 11] = 90.0
    check(z, tokens, 5)


@pytest.mark.parametrize("V", [3000, 40000])
@pytest.mark.parametrize("M", [5, 1200])
def test_ranks_beside_close_neighbours(M, V):
    """logits above the token's that the difference to the largest tells from it or not: none, a few, more than a block keeps; far below the largest"""
    z, tokens = logits(8, M, V, FP32)
    many = {0: 0, 1: 3, 2: 63, 3: 64, 4: 500}
    for row, n in many.items():
        g = torch.Generator(device="cuda").manual_seed(row)
        z[row, 7] = 0.1
        at = torch.randperm(V - 8, generator=g, device="cuda")[:n] + 8
        z[row, at] = 0.1 + torch.rand(n, generator=g, device="cuda") * 3e-6
        z[row, V - 1] = 14.0 if row % 2 else 80.5
        tokens[row] = 7
    check(z, tokens, 3)


def test_graph_and_streams():
    from tyloquant_amd import runtime as R
    z, tokens = logits(6, 3, 50000, FP32)
    many, more = logits(7, 1100, 4000, BF16)
    work = lambda: [*R.token_logprobs(z, tokens, 20), *R.token_logprobs(many, more, 5)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = work()
        graphs.append((g, out))
    for k in range(3):
        z.copy_(logits(10 + k, 3, 50000, FP32)[0])
        many.copy_(logits(20 + k, 1100, 4000, BF16)[0])
        want = work()
        for g, out in graphs:
            for o in out:
                o.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))
    with torch.cuda.stream(side):
        got = work()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
