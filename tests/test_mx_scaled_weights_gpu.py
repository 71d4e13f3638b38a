"""Weights of products of microscaled operands over a program's life: scales rewritten in place, inference tensors."""
import numpy as np
import pytest
import torch

import mx_scaled_ref as P
from test_mx_scaled_gpu import hidden, quantized

pytestmark = pytest.mark.gpu


def want(x, v, s, act="MXFP6"):
    xq, w = quantized(x, act), P.values(P.unpack(v), s, "MXFP4")
    return xq @ w.T, P.sum_bound(xq, w)


def test_scales_rewritten_in_place_are_seen():
    """By eager calls at once, and by a captured product after one: mx_matmul and dequantize read the bytes as they lie."""
    from tyloquant_amd import runtime_mx as RX
    rng = np.random.default_rng(61)
    v, s, _ = P.weight(rng, 80, 352)
    scales = torch.from_numpy(s).cuda()
    w = RX.MxWeight.from_tensors("MXFP4", torch.from_numpy(v).cuda(), scales)
    x = hidden(rng, 9, 352).to(torch.bfloat16)
    xd = x.cuda()
    P.check(RX.mx_scaled_matmul(w, xd), *want(x, v, s), "float32")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = RX.mx_scaled_matmul(w, xd)
    for k in range(3):
        s = rng.integers(118, 126, s.shape, dtype=np.uint8)
        scales.copy_(torch.from_numpy(s))
        P.check(RX.mx_scaled_matmul(w, xd), *want(x, v, s), "float32")
        graph.replay()
        torch.cuda.synchronize()
        P.check(held, *want(x, v, s), "float32")
    scales += 1
    with pytest.raises(RuntimeError, match="before a graph is captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            RX.mx_scaled_matmul(w, xd)
    P.check(RX.mx_scaled_glu(w, xd, out_dtype=torch.float16), P.glu(want(x, v, s + 1)[0]), P.glu_bound(*want(x, v, s + 1)), "float16")


def test_inference_tensors():
    """They have no count of writes: laid out once, and again where the caller says so."""
    from tyloquant_amd import runtime_mx as RX
    rng = np.random.default_rng(62)
    v, s, _ = P.weight(rng, 48, 288)
    x = hidden(rng, 3, 288).to(torch.float16)
    with torch.inference_mode():
        scales = torch.from_numpy(s).cuda().clone()
        w = RX.MxWeight.from_tensors("MXFP4", torch.from_numpy(v).cuda(), scales)
        for _ in range(2):
            P.check(RX.mx_scaled_matmul(w, x.cuda()), *want(x, v, s), "float32")
        s = s + 1
        scales.copy_(torch.from_numpy(s))
        w.laid_scales(again=True)
        P.check(RX.mx_scaled_matmul(w, x.cuda()), *want(x, v, s), "float32")
