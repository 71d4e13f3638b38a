"""Calls of the FP8 products and of the layer of experts that their descriptions allow and the other tests do not make."""
import math

import numpy as np
import pytest
import torch

import mx8_ref as P
from mx8_ref import BF16, FP16, FP32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("M", [4, 16])
def test_rows_quantised_by_the_product_itself(dtype, M):
    """every finite 16-bit pattern, in order and shuffled, against the unit matrix: what the product's own blocks quantise is what the quantiser
    makes of it.  Results below fp32's normal values may be flushed."""
    from tyloquant_amd import runtime_mx8 as R8
    from tyloquant_amd.runtime_mx import MxWeight
    K = 4096
    w = MxWeight.from_tensors("MXFP8", (torch.eye(K, device="cuda") * 0x38).to(torch.uint8), torch.full((K // 128, K // 128), 127, dtype=torch.uint8, device="cuda"))
    bits = np.arange(65536, dtype=np.uint32).astype(np.uint16)
    for order in (bits, np.random.default_rng(5).permutation(bits)):
        x = torch.from_numpy(order.view(np.int16).copy()).view(dtype)
        x = torch.where(torch.isfinite(x), x, torch.zeros((), dtype=dtype)).reshape(-1, K).cuda()
        for rows in x.split(M):
            want = R8.mx8_quantize(rows).dequantize()
            got = R8.mx8_scaled_matmul(w, rows, out_dtype=FP32)
            small = want.abs() < 2.0 ** -126
            assert torch.equal(torch.where(small, 0.0, got), torch.where(small, 0.0, want))
            assert (got[small].abs() <= want[small].abs()).all()
            assert torch.equal(got, R8.mx8_scaled_matmul(w, R8.mx8_quantize(rows), out_dtype=FP32))


@pytest.mark.parametrize("E", [5, 64, 300])
def test_routers_without_a_choice(E):
    """logits that are masked throughout, NaN, or infinite: the selection is moe_topk's, token by token, and no token touches another"""
    from tyloquant_amd import runtime_moe as RM
    from test_mx_layer_gpu import Layer, router
    layer = Layer("MXFP8", E, 128, 128)
    x, z = P.make_x(1, 8, 128, BF16), router(2, 8, E)
    z[0] = -math.inf
    z[1] = math.nan
    z[2, 3] = math.inf
    z[3, 1], z[3, 4] = math.inf, math.nan
    z[4] = torch.finfo(FP32).min
    z[5, 2] = -math.inf
    for mode in ({}, dict(use_sigmoid=True), dict(use_sqrt_softplus=True), dict(delayed_softmax=True)):
        y, ids, weights = RM.mx_moe_ffn_forward(layer.gate_up, layer.down, x, z, 3, **mode)
        wi, ww = RM.moe_topk(z, 3, **mode)
        assert torch.equal(ids, wi) and torch.equal(weights.isnan(), ww.isnan())
        real = ~ww.isnan()
        assert ((weights - ww)[real & torch.isfinite(ww)].abs() <= 2.0 ** -21 * ww[real & torch.isfinite(ww)].abs()).all()
        calm = torch.isfinite(ww).all(1)
        assert calm[4:].all() and torch.isfinite(y[calm]).all()
        layer.check(y[calm], x[calm], ids[calm], weights[calm])


def test_bf16_results_that_go_to_a_neighbour():
    """What the cut-off products cost a bf16 result: a rounding to the neighbour, of one in some hundred.  An error of 2^-16 of the results' size, in
    the mean 0.8 of it, crosses a border with the chance of its share of a step.  Normal results: 0.8 2^-k of them at most lie in the octave from
    2^-k of their size, whose steps are 2^(-k - 7): 0.8 2^7 0.8 2^-16 = 0.00125 an octave, nine octaves until a step is as small as the error,
    0.0016 of the results below those and 0.0005 above their size: 0.0134."""
    from tyloquant_amd import runtime_mx8 as R8
    from tyloquant_amd.runtime_mx import MxWeight
    codes, scales = P.make_weight(3, 2048, 4096, spread=0)
    w, wd = MxWeight.from_tensors("MXFP8", codes, scales), P.weight(codes, scales)
    for M in (3, 16, 30, 300):
        x = torch.randn(M, 4096, generator=torch.Generator("cuda").manual_seed(M), device="cuda").to(BF16)
        got, want = R8.mx8_scaled_matmul(w, x), (P.rounded(x) @ wd.T).to(BF16)
        off = got != want
        assert off.float().mean() <= 0.0134, float(off.float().mean())
        step = (got.view(torch.int16).int() - want.view(torch.int16).int()).abs()[off & (want.abs() > want.float().std() / 16)]
        assert step.numel() == 0 or step.max() == 1
