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


FEW = [  # rows that do not fit the LDS: activations, rows, out, K, plan plain, plan gated
    ("MXFP4", 5, 130, 17440, 3, 3), ("MXFP4", 16, 96, 17440, 3, 3), ("MXFP4", 20, 130, 8224, 2, 4), ("MXFP4", 31, 98, 12288, 4, 4), ("MXFP4", 32, 64, 17440, 4, 4),
    ("MXFP6", 13, 98, 12288, 3, 3), ("MXFP6", 9, 130, 17440, 3, 3), ("MXFP6", 20, 130, 5632, 2, 4), ("MXFP6", 17, 98, 8224, 4, 4), ("MXFP6", 32, 64, 12288, 4, 4)]


@pytest.mark.parametrize("act,rows,out,K,plan,gated", FEW)
def test_few_rows_past_the_lds(act, rows, out, K, plan, gated):
    """One and two tiles of 16 rows on the stream kernel, plain and gated (and gated alone, where gate and up leave less room)."""
    from tyloquant_amd import _lib as L
    from tyloquant_amd import runtime_mx as RX
    assert [L.lib().mfq_hip_mx_scaled_plan(KIND[act], out, K, rows, g, None) for g in (0, 1)] == [plan, gated]
    rng = np.random.default_rng(rows + out + K)
    w, wv = make_weight(rng, out, K)
    x = hidden(rng, rows, K).to(torch.bfloat16)
    xq = quantized(x, act)
    want, err = xq @ wv.T, P.sum_bound(xq, wv)
    for given in (x.cuda(), RX.mx_quantize(x.cuda(), act)):
        P.check(RX.mx_scaled_matmul(w, given, act=act), want, err, "float32", 1e-6)
        for result, gelu in ((torch.bfloat16, False), (torch.float16, True)):
            h = RX.mx_scaled_glu(w, given, act=act, activation=int(gelu), out_dtype=result)
            P.check(h, P.glu(want, gelu), P.glu_bound(want, err, gelu), str(result)[6:])


EXPERTS = [  # tokens, routes, experts, out, K, plans: MXFP4 plain and gated, MXFP6 plain and gated, with rows that come quantised
    (12, 2, 8, 50, 17440, (3, 3, 3, 3)),                                                  # few pairs, rows past the LDS
    (37, 3, 16, 34, 15136, (1, 3, 3, 3)), (10, 1, 70, 48, 12288, (1, 1, 3, 3)),
    (40, 4, 8, 144, 2880, (5, 5, 10, 10)), (90, 4, 8, 330, 2080, (5, 5, 10, 10)),          # tiles whose stages come round several times
    (330, 4, 8, 330, 1440, (8, 8, 11, 11)), (180, 2, 2, 198, 2880, (8, 8, 11, 11)), (700, 2, 7, 130, 3104, (8, 8, 11, 11))]


@pytest.mark.parametrize("act", list(KIND))
@pytest.mark.parametrize("T,R,E,out,K,plans", EXPERTS)
def test_routed_experts(act, T, R, E, out, K, plans):
    """A pool that holds all experts but one, in an order of its own, ids that are none among the routes; rows of the experts that it has
    not stay as they are."""
    from tyloquant_amd import _lib as L
    from tyloquant_amd import runtime_moe as RM
    from tyloquant_amd import runtime_mx as RX
    assert tuple(L.lib().mfq_hip_mx_moe_plan(k, K, T * R, E, 1, g, 1) for k in (4, 6) for g in (0, 1)) == plans
    rng = np.random.default_rng(T + R + E + out + K)
    held = rng.permutation(E)[: E - 1]
    w, wv = make_weight(rng, len(held) * out, K, out=out)
    slot = np.full(E, -1, np.int32)
    slot[held] = np.arange(len(held))
    ids = rng.integers(0, E, (T, R)).astype(np.int32)
    ids[rng.random((T, R)) < 0.1] = -1
    ids[T // 2, 0] = E + 3
    flat = ids.reshape(-1)
    none = (flat < 0) | (flat >= E)
    route = RM.build_moe_route_plan(torch.from_numpy(ids).cuda(), E)
    slots = torch.from_numpy(slot).cuda()
    for routed in (False, True):
        x = hidden(rng, T * R if routed else T, K).to(torch.float16 if routed else torch.bfloat16)
        xq = quantized(x, act)
        want, err, theirs = np.zeros((T * R, out)), np.zeros((T * R, out)), none.copy()
        for e in held:
            p = np.flatnonzero(flat == e)
            theirs[p] = True
            we, xe = wv[slot[e] * out: slot[e] * out + out], xq[p if routed else p // R]
            want[p], err[p] = xe @ we.T, P.sum_bound(xe, we)
        for given in (x.cuda(), RX.mx_quantize(x.cuda(), act)):
            y = torch.full((T, R, out), 7.5, device="cuda")
            RX.mx_moe_into(w, given, route, y, act=act, routed=routed, slot=slots)
            P.check(y, np.where(theirs[:, None], want, 7.5).reshape(T, R, out), err.reshape(T, R, out), "float32")
            for gelu in (False, True):
                h = torch.full((T, R, out // 2), 7.5, device="cuda", dtype=torch.bfloat16)
                RX.mx_moe_into(w, given, route, h, act=act, routed=routed, glu=True, activation=int(gelu), slot=slots)
                P.check(h, np.where(theirs[:, None], P.glu(want, gelu), 7.5).reshape(T, R, -1), P.glu_bound(want, err, gelu).reshape(T, R, -1), "bfloat16")


@pytest.mark.parametrize("act", list(KIND))
@pytest.mark.parametrize("rows", [1, 16, 20, 40, 200])
def test_scales_at_both_ends(act, rows):
    """Weights with scales 254 and 0 against activations small and large enough for the sums to be ordinary numbers: a product of codes and
    both scales passes no type on its way that its result does not."""
    from tyloquant_amd import runtime_mx as RX
    rng = np.random.default_rng(rows)
    out, K = 80, 416
    v = rng.integers(0, 256, (out, K // 2), dtype=np.uint8)
    for byte, size in ((254, 2.0 ** -112), (253, 2.0 ** -120), (0, 2.0 ** 120), (1, 2.0 ** 110)):
        s = rng.integers(200, 208, (out, K // 32), dtype=np.uint8) if byte > 128 else rng.integers(2, 10, (out, K // 32), dtype=np.uint8)
        s[::3] = byte
        s[1, 4] = byte
        w = RX.MxWeight.from_tensors("MXFP4", torch.from_numpy(v).cuda(), torch.from_numpy(s).cuda())
        wv = P.values(P.unpack(v), s, "MXFP4")
        x = (hidden(rng, rows, K) * size).to(torch.float32)
        xq = quantized(x, act)
        P.check(RX.mx_scaled_matmul(w, x.cuda(), act=act), xq @ wv.T, P.sum_bound(xq, wv), "float32")
