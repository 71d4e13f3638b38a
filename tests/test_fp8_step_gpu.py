"""The FP8 operators together, as a program runs them: a decode step through a layer of experts, the head and the scores of its tokens, and a
prefill chunk through the grouped products; every stage against float64 of what went into it, and the whole in a graph."""
import pytest
import torch

import mx8_ref as P
from mx8_ref import BF16, FP32
from test_logprobs_gpu import oracle
from test_mx8_gpu import check_pairs, tensor
from test_mx_layer_gpu import Layer, check_route, router

pytestmark = pytest.mark.gpu
E, K, H, I, V = 8, 3, 384, 256, 1000


class Step:
    def __init__(self):
        self.layer = Layer("MXFP8", E, H, I)
        self.head, self.hw = tensor(77, V, H)

    def few(self, x, logits, tokens):
        """up to 16 tokens: the whole layer in one call"""
        from tyloquant_amd import runtime as R
        from tyloquant_amd import runtime_moe as RM
        from tyloquant_amd import runtime_mx8 as R8
        y, ids, weights = RM.mx_moe_ffn_forward(self.layer.gate_up, self.layer.down, x, logits, K, normalize=True)
        h = (x.float() + y).to(BF16)
        z = R8.mx8_scaled_matmul(self.head, h, out_dtype=FP32)
        return [y, ids, weights, h, z, *R.token_logprobs(z, tokens, 5)]

    def many(self, x, logits, tokens):
        """a prefill chunk: products grouped by expert"""
        from tyloquant_amd import runtime as R
        from tyloquant_amd import runtime_moe as RM
        from tyloquant_amd import runtime_mx8 as R8
        ids, weights = RM.moe_topk(logits, K, normalize=True)
        route = RM.build_moe_route_plan(ids, E)
        hidden = R8.mx8_moe_glu(self.layer.gate_up, R8.mx8_quantize(x), route)
        pairs = R8.mx8_moe_matmul(self.layer.down, hidden.reshape(-1, I), route, routed=True, out_dtype=FP32)
        y = RM.moe_weighted_reduce(pairs, weights)
        h = (x.float() + y).to(BF16)
        z = R8.mx8_scaled_matmul(self.head, h, out_dtype=FP32)
        return [y, ids, weights, h, z, *R.token_logprobs(z, tokens, 5), hidden, pairs]


def inputs(seed, T):
    return P.make_x(seed, T, H, BF16), router(seed + 1, T, E), torch.randint(0, V, (T,), device="cuda", generator=torch.Generator("cuda").manual_seed(seed))


def check_scores(z, tokens, scores):
    lp, rank, entropy, order, best = oracle(z, tokens, 5)
    size = float(z.abs().max())
    for got, want in ((scores[0], lp), (scores[2], entropy), (scores[4], best)):
        assert ((got.cpu().double() - want).abs() <= (2.0 ** -20 + 2.0 ** -22 * size) * 16).all()
    assert torch.equal(scores[1].cpu(), rank) and torch.equal(scores[3].cpu(), order)


@pytest.mark.parametrize("T", [1, 7, 16])
def test_decode_step(T):
    s = Step()
    x, logits, tokens = inputs(T, T)
    y, ids, weights, h, z, *scores = s.few(x, logits, tokens)
    check_route(ids, weights, logits, K, "softmax", True)
    s.layer.check(y, x, ids, weights)
    P.check(z, P.rounded(h), s.hw)
    check_scores(z, tokens, scores)


@pytest.mark.parametrize("T", [9, 40, 333])
def test_prefill_chunk(T):
    s = Step()
    x, logits, tokens = inputs(T, T)
    y, ids, weights, h, z, *rest = s.many(x, logits, tokens)
    scores, hidden, pairs = rest[:5], rest[5], rest[6]
    check_pairs(hidden, P.rounded(x), s.layer.gu, ids, 2 * I, E, False, True)
    check_pairs(pairs, P.rounded(hidden.reshape(-1, I)), s.layer.dn, ids, H, E, True, False)
    P.check(z, P.rounded(h), s.hw)
    check_scores(z, tokens, scores)


def test_both_ways_agree():
    """quantised activations cost what they cost: an element of E4M3 is off by up to 2^-4, a product of some hundred of them by far less"""
    s = Step()
    x, logits, tokens = inputs(5, 12)
    few, many = s.few(x, logits, tokens), s.many(x, logits, tokens)
    assert torch.equal(few[1], many[1])
    assert (few[0] - many[0]).norm() <= 2.0 ** -4 * few[0].norm()


def test_a_step_in_a_graph():
    s = Step()
    x, logits, tokens = inputs(3, 10)
    work = lambda: s.few(x, logits, tokens) + s.many(x, logits, tokens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for n in range(4):
        for a, b in zip((x, logits, tokens), inputs(20 + n, 10)):
            a.copy_(b)
        want = work()
        for o in out:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
