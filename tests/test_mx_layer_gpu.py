"""A whole layer of routed experts for a few tokens on the GPU against float64: formats, token counts, routers, shared experts, experts that
hold NaN, graphs."""
import math

import pytest
import torch

import mx8_ref as P
from mx8_ref import BF16, FP16, FP32

pytestmark = pytest.mark.gpu


def fp4_weight(seed, rows, K):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randint(0, 256, (rows, K // 2), generator=g, device="cuda", dtype=torch.uint8),
            torch.randint(117, 123, (rows, K // 32), generator=g, device="cuda", dtype=torch.uint8))


def fp4_values(v, s):
    t = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=v.device)
    t = torch.cat((t, -t))
    return torch.stack((t[(v & 15).long()], t[(v >> 4).long()]), -1).flatten(1) * P.powers(s).repeat_interleave(32, 1)


def tensor(fmt, seed, rows, K, out=None):
    from tyloquant_amd.runtime_mx import MxWeight
    v, s = P.make_weight(seed, rows, K) if fmt == "MXFP8" else fp4_weight(seed, rows, K)
    return MxWeight.from_tensors(fmt, v, s, out=out), (P.weight if fmt == "MXFP8" else fp4_values)(v, s)


class Layer:
    def __init__(self, fmt, E, H, I, S=0, seed=1):
        self.E, self.H, self.I, self.S = E, H, I, S
        self.gate_up, self.gu = tensor(fmt, seed, E * 2 * I, H, 2 * I)
        self.down, self.dn = tensor(fmt, seed + 1, E * H, I, H)
        self.shared = None
        if S:
            (a, self.sgu), (b, self.sdn) = tensor(fmt, seed + 2, 2 * S, H), tensor(fmt, seed + 3, H, S)
            self.shared = a, b

    def one(self, x, gu, dn, gelu):
        """float64 of one expert, and a bound of what fp32 sums and the activation cost: a product of K terms is off by at most K 2^-24 of its
        magnitudes (each sum rounds once), the hidden row by its three parts (2^-24), the activation by 2^-20"""
        h = P.gate(x @ gu.T, gelu)
        mag = (x.abs() @ gu.abs().T) * (x.shape[-1] * 2.0 ** -24)
        (g, u), (dg, du) = (x @ gu.T).chunk(2, -1), mag.chunk(2, -1)
        dh = 1.13 * dg * u.abs() + (P.gate(torch.cat((g.abs(), torch.ones_like(u)), -1), gelu).abs() + 1.13 * dg) * du + 2.0 ** -20 * h.abs()
        return h @ dn.T, (dh + h.abs() * (dn.shape[-1] + 1) * 2.0 ** -24) @ dn.abs().T

    def check(self, out, x, ids, weights, gate=None, gelu=False):
        x, half = x.double(), P.HALF[out.dtype]
        want, tol = torch.zeros(x.shape[0], self.H, dtype=torch.float64, device="cuda"), torch.zeros(x.shape[0], self.H, dtype=torch.float64, device="cuda")
        for e in ids.unique().tolist():
            t, r = torch.nonzero(ids == e, as_tuple=True)
            y, d = self.one(x[t], self.gu[e * 2 * self.I:(e + 1) * 2 * self.I], self.dn[e * self.H:(e + 1) * self.H], gelu)
            p = weights[t, r].double()[:, None]
            want[t] += p * y
            tol[t] += p.abs() * d + 2.0 ** -22 * (p * y).abs()
        if self.S:
            y, d = self.one(x, self.sgu, self.sdn, gelu)
            p = torch.ones(x.shape[0], 1, dtype=torch.float64, device="cuda") if gate is None else torch.sigmoid(gate.double())[:, None]
            want += p * y
            tol += p * d + 2.0 ** -22 * (p * y).abs()
        got = out.double()
        assert torch.equal(got.isnan(), want.isnan())
        ok = ~want.isnan()
        over = ((got - want).abs() - half * want.abs() - tol - 1e-30)[ok]
        assert over.numel() == 0 or over.max() <= 0, float(over.max())
        if out.dtype == FP32 and ok.all():   # errors do not line up: far below their bound
            assert (got - want).norm() <= 4e-6 * want.norm(), float((got - want).norm() / want.norm())


def router(seed, T, E):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(T, E, generator=g, device="cuda")


def check_route(ids, weights, logits, k, mode, normalize, bias=None, scale=1.0):
    from tyloquant_amd import runtime_moe as RM
    wi, ww = RM.moe_topk(logits, k, use_sigmoid=mode == "sigmoid", use_sqrt_softplus=mode == "sqrt_softplus", normalize=normalize,
                         delayed_softmax=mode == "delayed", bias=bias, scale=scale)
    assert torch.equal(ids, wi)
    assert ((weights - ww).abs() <= 2.0 ** -21 * ww.abs()).all()      # the same formula; the softmax's sum in another order


CASES = [("MXFP8", 8, 128, 128, 0), ("MXFP8", 16, 256, 384, 0), ("MXFP8", 5, 1152, 128, 128), ("MXFP4", 8, 32, 32, 0), ("MXFP4", 7, 288, 96, 0),
         ("MXFP4", 12, 2880, 160, 64), ("MXFP4", 300, 256, 32, 32), ("MXFP8", 70, 384, 256, 256), ("MXFP8", 3, 4096, 256, 0), ("MXFP4", 4, 4096, 1024, 0)]


@pytest.mark.parametrize("fmt,E,H,I,S", CASES)
def test_layer(fmt, E, H, I, S):
    from tyloquant_amd import runtime_moe as RM
    layer = Layer(fmt, E, H, I, S)
    for T, k, dtype, out, normalize in ((1, 1, BF16, FP32, False), (1, min(E, 8), FP16, BF16, True), (2, 2, BF16, FP32, True), (5, 3, FP16, FP32, False),
                                        (6, min(E, 4), BF16, FP16, True), (8, 2, FP16, FP32, True), (9, 3, FP16, FP32, True), (16, min(E, 16), BF16, FP32, True),
                                        (16, 1, FP16, FP32, False)):
        x, logits = P.make_x(T, T, H, dtype), router(T + k, T, E)
        y, ids, weights = RM.mx_moe_ffn_forward(layer.gate_up, layer.down, x, logits, k, normalize=normalize, shared=layer.shared, out_dtype=out)
        assert y.dtype == out and tuple(y.shape) == (T, H)
        check_route(ids, weights, logits, k, "softmax", normalize)
        layer.check(y, x, ids, weights)


@pytest.mark.parametrize("fmt", ["MXFP8", "MXFP4"])
@pytest.mark.parametrize("H", [4224, 8192, 8320, 16512])
def test_long_rows(fmt, H):
    """rows whose activations no longer stay in registers among them"""
    from tyloquant_amd import runtime_moe as RM
    layer = Layer(fmt, 4, H, 128)
    for T, dtype in ((1, BF16), (3, FP16), (12, FP16), (16, BF16)):
        x, logits = P.make_x(T, T, H, dtype), router(T, T, 4)
        y, ids, weights = RM.mx_moe_ffn_forward(layer.gate_up, layer.down, x, logits, 2)
        layer.check(y, x, ids, weights)


@pytest.mark.parametrize("mode", ["softmax", "sigmoid", "sqrt_softplus", "delayed"])
@pytest.mark.parametrize("E,k", [(6, 3), (64, 8), (257, 16), (1024, 5)])
def test_routers(mode, E, k):
    from tyloquant_amd import runtime_moe as RM
    layer = Layer("MXFP4", E, 64, 32, 32)
    x, logits = P.make_x(3, 7, 64, BF16), router(9, 7, E)
    logits[1] = 0.5                       # all alike: the lowest experts
    logits[2, ::2] = logits[2, 1]         # ties
    logits[3, 1:] = -math.inf             # one alone
    logits[4, E // 2] = math.nan          # the last of all
    bias = router(10, 1, E)[0] * 0.1
    gate = router(11, 7, 1)[:, 0]
    for normalize in (False,) if mode == "delayed" else (False, True):
        for b in (None, bias):
            if mode in ("sqrt_softplus", "delayed"):
                logits[3, 1:] = -30.0
            args = dict(use_sigmoid=mode == "sigmoid", use_sqrt_softplus=mode == "sqrt_softplus", delayed_softmax=mode == "delayed", normalize=normalize)
            y, ids, weights = RM.mx_moe_ffn_forward(layer.gate_up, layer.down, x, logits, k, router_bias=b, router_scale=2.5, shared=layer.shared,
                                                    shared_gate=gate, activation=1, **args)
            check_route(ids, weights, logits, k, mode, normalize, b, 2.5)
            layer.check(y, x, ids, weights, gate, gelu=True)


@pytest.mark.parametrize("fmt", ["MXFP8", "MXFP4"])
def test_nan_and_infinity_stay_where_they_are(fmt):
    """an expert whose weights hold NaN touches the tokens that take it and no others; a token's own infinity no other token"""
    from tyloquant_amd import runtime_moe as RM
    layer = Layer(fmt, 6, 256, 128)
    layer.gate_up.scales.view(6, -1)[2].fill_(255)
    layer.down.scales.view(6, -1)[4, 1] = 255
    torch.cuda.synchronize()
    values = P.weight if fmt == "MXFP8" else fp4_values
    layer.gu, layer.dn = values(layer.gate_up.values, layer.gate_up.scales), values(layer.down.values, layer.down.scales)
    for T in (4, 5, 11):
        x, logits = P.make_x(T, T, 256, BF16), router(T, T, 6)
        logits[0, 2] = 9.0
        logits[1, 4] = 9.0
        logits[2, 2] = logits[2, 4] = -9.0
        logits[3, 2] = logits[3, 4] = -9.0
        x[3, 17] = math.nan
        y, ids, weights = RM.mx_moe_ffn_forward(layer.gate_up, layer.down, x, logits, 2)
        assert y[0].isnan().all() and y[3].isnan().all() and not y[2].isnan().any() and y[1].isnan().any()
        layer.check(y, x, ids, weights)


def test_layouts():
    from tyloquant_amd import runtime_moe as RM
    layer = Layer("MXFP8", 8, 256, 128)
    wide = P.make_x(1, 9, 512, BF16)
    logits = router(2, 9, 8)
    for x in (wide[:, :256], wide[:, 3:259], P.make_x(3, 256, 9, BF16).t(), wide[:1, :256].expand(9, 256)):
        y, ids, weights = RM.mx_moe_ffn_forward(layer.gate_up, layer.down, x, logits, 3)
        layer.check(y, x, ids, weights)
    y, ids, weights = RM.mx_moe_ffn_forward(layer.gate_up, layer.down, wide[:, :256], logits.half(), 3)
    layer.check(y, wide[:, :256], ids, weights)
    assert RM.mx_moe_ffn_forward(layer.gate_up, layer.down, wide[:0, :256], logits[:0], 3)[0].shape == (0, 256)


@pytest.mark.parametrize("fmt", ["MXFP8", "MXFP4"])
def test_few_compute_units(fmt, cu_count):
    """blocks that go through many row-blocks, of several experts and the shared one; results in one piece, some or as many as there can be"""
    from tyloquant_amd import runtime_moe as RM
    layer = Layer(fmt, 6, 384, 256, 128)
    for T in (1, 6, 16):
        x, logits = P.make_x(4, T, 384, BF16), router(5, T, 6)
        for n in (1, 3, 7, 13, 100, 1000):
            cu_count(n)
            y, ids, weights = RM.mx_moe_ffn_forward(layer.gate_up, layer.down, x, logits, 3, shared=layer.shared)
            layer.check(y, x, ids, weights)
            again = RM.mx_moe_ffn_forward(layer.gate_up, layer.down, x, logits, 3, shared=layer.shared)
            assert all(torch.equal(a, b) for a, b in zip((y, ids, weights), again))


def test_graph_replays_and_streams():
    from tyloquant_amd import runtime_moe as RM
    layers = [Layer("MXFP8", 8, 256, 256, 128), Layer("MXFP4", 8, 256, 256)]
    xs, zs = [P.make_x(T, T, 256, BF16) for T in (1, 5, 16)], [router(T, T, 8) for T in (1, 5, 16)]

    def work():
        return [o for l in layers for x, z in zip(xs, zs) for o in RM.mx_moe_ffn_forward(l.gate_up, l.down, x, z, 3, shared=l.shared)]

    side, graphs = torch.cuda.Stream(), []
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = work()
        graphs.append((g, out))
    for n in range(3):
        for x, z in zip(xs, zs):
            x.copy_(P.make_x(50 + n, *x.shape, BF16))
            z.copy_(router(60 + n, *z.shape))
        want = work()
        for g, out in graphs:
            for o in out:
                o.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))
    other, got = torch.cuda.Stream(), []
    for s in (side, other):
        s.wait_stream(torch.cuda.current_stream())
    for s in (side, other):
        with torch.cuda.stream(s):
            got.append([work() for _ in range(3)][-1])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for both in got for a, b in zip(both, want))
