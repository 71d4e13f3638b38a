"""Every kernel that the rules of the products of microscaled operands can choose, named by the plan that each case has to take: tiles of
one tensor, whole and with K in pieces, plain and gated.  Fewer compute units than the card's let small tensors take the tiles of large
ones; the kernels are the same."""
import ctypes as C

import numpy as np
import pytest
import torch

import mx_scaled_ref as P
from test_mx_scaled_gpu import hidden, make_weight, quantized

pytestmark = pytest.mark.gpu
KIND = {"MXFP4": 4, "MXFP6": 6}

TILES = [  # activations, compute units, rows, out, K, plan (5 + the tile's index), pieces of K; out divided by two is odd in most
    ("MXFP4", 1, 150, 330, 1056, 5, 1), ("MXFP4", 16, 37, 134, 2336, 5, 5), ("MXFP4", 256, 64, 300, 4096, 5, 16),
    ("MXFP4", 5, 222, 390, 1056, 6, 1), ("MXFP4", 12, 75, 134, 5504, 6, 4),
    ("MXFP4", 2, 196, 330, 1056, 7, 1), ("MXFP4", 256, 601, 4100, 2080, 7, 1), ("MXFP4", 12, 100, 330, 6240, 7, 4),
    ("MXFP4", 4, 222, 390, 3680, 8, 1), ("MXFP4", 1, 601, 390, 1440, 8, 1),
    ("MXFP4", 1, 222, 391, 1440, 9, 1), ("MXFP4", 1, 222, 390, 1440, 9, 1), ("MXFP4", 1, 460, 1030, 2080, 9, 1), ("MXFP4", 2, 196, 1186, 5504, 9, 2),
    ("MXFP6", 3, 150, 330, 1056, 10, 1), ("MXFP6", 12, 37, 134, 1440, 10, 6), ("MXFP6", 256, 64, 300, 4096, 10, 16),
    ("MXFP6", 2, 222, 330, 1056, 11, 1), ("MXFP6", 1, 222, 331, 1056, 11, 1), ("MXFP6", 12, 222, 390, 2080, 11, 3),
    ("MXFP6", 1, 150, 330, 1440, 12, 1), ("MXFP6", 1, 530, 602, 2080, 12, 1), ("MXFP6", 3, 150, 390, 2880, 12, 3)]


@pytest.mark.parametrize("act,cus,rows,out,K,plan,pieces", TILES)
def test_tiles(act, cus, rows, out, K, plan, pieces, cu_count):
    from tyloquant_amd import _lib as L
    from tyloquant_amd import runtime_mx as RX
    cu_count(cus)
    got = C.c_int()
    assert (L.lib().mfq_hip_mx_scaled_plan(KIND[act], out, K, rows, 0, C.byref(got)), got.value) == (plan, pieces)
    rng = np.random.default_rng(rows + out + K)
    w, wv = make_weight(rng, out, K)
    for dtype, results in ((torch.bfloat16, (torch.float32, torch.float16)), (torch.float16, (torch.bfloat16,))):
        x = hidden(rng, rows, K).to(dtype)
        xq = quantized(x, act)
        want, err = xq @ wv.T, P.sum_bound(xq, wv)
        for given in (x.cuda(), RX.mx_quantize(x.cuda(), act)):
            for result in results:
                P.check(RX.mx_scaled_matmul(w, given, act=act, out_dtype=result), want, err, str(result)[6:], 1e-6)
                if out % 2 == 0 and result != torch.float32:
                    for gelu in (False, True):
                        h = RX.mx_scaled_glu(w, given, act=act, activation=int(gelu), out_dtype=result)
                        P.check(h, P.glu(want, gelu), P.glu_bound(want, err, gelu), str(result)[6:])
