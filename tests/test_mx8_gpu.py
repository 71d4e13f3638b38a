"""FP8 products by blocks of 128 on the GPU against 64-bit sums over the same codes: quantisation byte by byte, every kernel behind
mx8_scaled_matmul / mx8_scaled_glu / mx8_moe_matmul / mx8_moe_glu, their borders, graphs and streams."""
import ctypes as C

import numpy as np
import pytest
import torch

import mx8_ref as P
from mx8_ref import BF16, FP16, FP32

pytestmark = pytest.mark.gpu


def tensor(seed, rows, K, out=None):
    from tyloquant_amd.runtime_mx import MxWeight
    v, s = P.make_weight(seed, rows, K)
    return MxWeight.from_tensors("MXFP8", v, s, out=out), P.weight(v, s)


# ---- quantisation ---------------------------------------------------------------------------------------------------
def same_rows(q, x):
    """the bytes of a quantisation against the oracle's; float64 values"""
    codes, scales = P.quantize(x.reshape(-1, x.shape[-1]))
    M, blocks = scales.shape
    got = q.scales.permute(1, 0, 2).reshape(M, -1)[:, :blocks].cpu().numpy()
    assert np.array_equal(got, scales)
    assert np.array_equal(q.values.cpu().numpy() & 127, codes & 127)
    zero = (codes & 127) == 0        # of which the sign says nothing
    assert np.array_equal(q.values.cpu().numpy()[~zero], codes[~zero])
    return P.values(torch.from_numpy(codes)) * P.powers(torch.from_numpy(scales)).repeat_interleave(128, 1)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_every_16_bit_pattern(dtype):
    """All patterns of the type in blocks of neighbours and shuffled, with infinities and NaN and without"""
    from tyloquant_amd import runtime_mx8 as R8
    bits = np.arange(65536, dtype=np.uint32).astype(np.uint16)
    for order in (bits, np.random.default_rng(3).permutation(bits)):
        x = torch.from_numpy(order.view(np.int16).copy()).view(dtype)
        for rows in (x, x[torch.isfinite(x)]):
            rows = rows[: rows.numel() // 640 * 640].reshape(-1, 640)
            q = R8.mx8_quantize(rows.cuda())
            want = same_rows(q, rows)
            got = q.dequantize().cpu().double()
            assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want.float().double())) and torch.equal(got.isnan(), want.isnan())


def test_borders_of_scales_and_elements():
    from tyloquant_amd import runtime_mx8 as R8
    rows = []
    for top in (448.0, 448.0 * (1 + 2.0 ** -23), 447.0, 240.0, 2.0 ** -118, 2.0 ** -119, 2.0 ** -126, 2.0 ** -140, 0.0, 3.0e38):
        v = torch.zeros(128, dtype=torch.float64)
        v[0] = top
        v[1:65] = torch.linspace(0, 1, 64, dtype=torch.float64) * top
        v[65:] = -top * torch.exp2(-torch.arange(63, dtype=torch.float64) / 3)
        rows.append(v)
    # ties: midpoints of neighbouring elements, and just beside them
    grid = torch.tensor(P.magnitudes(), dtype=torch.float64)
    mid = (grid[1:] + grid[:-1]) / 2
    for f in (1.0, 1 - 2.0 ** -20, 1 + 2.0 ** -20):
        rows.append(torch.cat((torch.tensor([448.0], dtype=torch.float64), mid * f, torch.zeros(1, dtype=torch.float64))))
    x = torch.stack(rows).float()
    q = R8.mx8_quantize(x.cuda())
    want = same_rows(q, x)
    assert torch.equal(q.dequantize().cpu().double(), want.float().double())


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("rows,K", [(1, 128), (3, 640), (17, 1152), (130, 4096), (2, 20480)])
def test_quantize_rows_in_any_layout(dtype, rows, K):
    from tyloquant_amd import runtime_mx8 as R8
    wide = P.make_x(5, rows, K + 256, dtype)
    for x in (wide[:, :K], wide[:, 64:64 + K], wide[:, 1:1 + K], wide[:, :K].contiguous(), P.make_x(6, K, rows, dtype).t(), wide[:1, :K].expand(rows, K)):
        q = R8.mx8_quantize(x)
        want = same_rows(q, x)
        for out in (FP32, BF16, FP16):
            assert torch.equal(q.dequantize(out).cpu(), want.to(FP32).to(out))
    q = R8.mx8_quantize(wide[:, :K].reshape(1, rows, K))
    assert tuple(q.dequantize().shape) == (1, rows, K)
    assert tuple(R8.mx8_quantize(wide[:0, :K]).dequantize().shape) == (0, K)


# ---- one tensor -----------------------------------------------------------------------------------------------------
SIZES = [(1, 128, 1), (16, 256, 2), (130, 384, 3), (200, 640, 5), (4096, 4096, 1), (1000, 1152, 16), (260, 4096, 13), (300, 5120, 17), (72, 2560, 32),
         (96, 12288, 2), (40, 20480, 9), (40, 10240, 31), (64, 10368, 20), (50, 20608, 3), (256, 2560, 33), (300, 1024, 129), (640, 512, 300), (1100, 1152, 777),
         (2048, 896, 2100), (6400, 384, 4096), (100, 6400, 70)]


@pytest.mark.parametrize("out,K,M", SIZES)
def test_linear(out, K, M):
    from tyloquant_amd import runtime_mx8 as R8
    w, wd = tensor(out + K, out, K)
    for dtype, result in ((BF16, BF16), (FP16, FP32), (FP32, FP16)):
        x = P.make_x(M, M, K, dtype)
        xd = P.rounded(x)
        P.check(R8.mx8_scaled_matmul(w, x, out_dtype=result), xd, wd)
        if out % 2 == 0 and result != FP32:
            P.check(R8.mx8_scaled_glu(w, x, out_dtype=result), xd, wd, glu=True)
    P.check(R8.mx8_scaled_matmul(w, R8.mx8_quantize(x), out_dtype=FP32), xd, wd)
    if out % 2 == 0:
        P.check(R8.mx8_scaled_glu(w, R8.mx8_quantize(x), activation=1, out_dtype=FP16), xd, wd, glu=True, gelu=True)


FORCED = [(11776, 1536, 601), (9216, 2048, 777), (15360, 1024, 777), (4096, 256, 1100)]


def test_sizes_reach_every_kernel():
    from tyloquant_amd import _lib as L
    splits = C.c_int()
    kinds = {L.lib().mfq_hip_mx8_scaled_plan(out, K, M, C.byref(splits)) for out, K, M in SIZES + FORCED}
    assert kinds == {0, 1, 2, 3, 4, 5, 6}
    assert {L.lib().mfq_hip_mx8_moe_plan(K, T * R, E, T > 8) for T, R, E, _, K in EXPERTS} == {0, 1, 3, 4, 5}



@pytest.mark.parametrize("out,K,M", FORCED)
def test_larger_tiles(out, K, M):
    from tyloquant_amd import runtime_mx8 as R8
    w, wd = tensor(out, out, K)
    x = P.make_x(M, M, K, BF16)
    xd = P.rounded(x)
    P.check(R8.mx8_scaled_matmul(w, x), xd, wd)
    P.check(R8.mx8_scaled_glu(w, x), xd, wd, glu=True)
    w, wd = tensor(out + 1, out - 70, K)      # up rows that begin inside a block of scales
    P.check(R8.mx8_scaled_glu(w, x), xd, wd, glu=True)
    P.check(R8.mx8_scaled_matmul(w, x, out_dtype=FP32), xd, wd)


@pytest.mark.parametrize("M", [1, 7, 40, 300])
def test_layouts_of_activations(M):
    from tyloquant_amd import runtime_mx8 as R8
    w, wd = tensor(1, 144, 640)
    wide = P.make_x(2, M, 1280, BF16)
    for x in (wide[:, :640], wide[:, 320:960], wide[:, 3:643], P.make_x(4, 640, M, BF16).t(), wide[:1, :640].expand(M, 640)):
        P.check(R8.mx8_scaled_matmul(w, x), P.rounded(x), wd)
    y = R8.mx8_scaled_matmul(w, wide[:, :640].reshape(1, M, 640))
    assert tuple(y.shape) == (1, M, 144) and torch.equal(y[0], R8.mx8_scaled_matmul(w, wide[:, :640]))
    assert tuple(R8.mx8_scaled_matmul(w, wide[:0, :640]).shape) == (0, 144)


@pytest.mark.parametrize("M", [1, 20, 100])
def test_infinities_and_nan(M):
    """a row of activations with one gives NaN in its own results alone, a neuron of weights with a NaN or the NaN scale in its own"""
    from tyloquant_amd.runtime_mx import MxWeight
    from tyloquant_amd import runtime_mx8 as R8
    v, s = P.make_weight(7, 300, 512)
    v[5, 100] = 0x7F
    v[250, 3] = 0xFF
    s[1, 2] = 255
    w, wd = MxWeight.from_tensors("MXFP8", v, s), P.weight(v, s)
    x = P.make_x(8, M, 512, BF16)
    x[M // 2, 200] = float("inf")
    x[M - 1, 511] = float("nan")
    P.check(R8.mx8_scaled_matmul(w, x, out_dtype=FP32), P.rounded(x), wd)
    y = R8.mx8_scaled_matmul(w, torch.zeros_like(x), out_dtype=FP32)
    assert torch.equal(y.isnan().any(0), wd.isnan().any(1)) and (torch.nan_to_num(y) == 0).all()


def test_extreme_scales():
    """scales of weights at both ends, and of activations"""
    from tyloquant_amd.runtime_mx import MxWeight
    from tyloquant_amd import runtime_mx8 as R8
    v, s = P.make_weight(9, 256, 256)
    for ws, xs in ((0, 2.0 ** 100), (254, 2.0 ** -118), (1, 2.0 ** 120), (200, 2.0 ** -60)):
        s.fill_(ws)
        w = MxWeight.from_tensors("MXFP8", v, s)
        for M in (3, 64):
            x = (P.make_x(10, M, 256, FP32).double() * xs).float()
            P.check(R8.mx8_scaled_matmul(w, x, out_dtype=FP32), P.rounded(x), P.weight(v, s))


def test_pool_expert_and_rows_left_alone():
    """one expert of a pool; a call writes its own results and nothing beside them"""
    from tyloquant_amd import _lib as L
    from tyloquant_amd import runtime_mx8 as R8
    w, wd = tensor(11, 3 * 256, 384, out=256)
    lib = L.lib()
    for M in (2, 30, 150):
        x = P.make_x(M, M, 384, BF16)
        for e in range(3):
            P.check(R8.mx8_scaled_matmul(w, x, expert=e), P.rounded(x), wd[e * 256:(e + 1) * 256])
        y = torch.full((M + 2, 300), 7.0, dtype=BF16, device="cuda")
        need = lib.mfq_hip_mx8_scaled_gemm_workspace_bytes(256, 384, M, 0)
        ws = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
        L.check(lib.mfq_hip_mx8_scaled_gemm_rows(w.values.data_ptr(), w.scales.data_ptr(), w.rows, 384, 256, 256, x.data_ptr(), L.X_BF16, 384, None, M, 0, 0,
                                                 y[1].data_ptr(), L.X_BF16, 300, ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream))
        assert torch.equal(y[1:M + 1, :256], R8.mx8_scaled_matmul(w, x, expert=1))
        y[1:M + 1, :256] = 7.0
        assert (y == 7.0).all()


def test_short_workspace_takes_fewer_pieces():
    from tyloquant_amd import _lib as L
    lib, splits = L.lib(), C.c_int()
    out, K, M = 128, 4096, 64
    assert lib.mfq_hip_mx8_scaled_plan(out, K, M, C.byref(splits)) >= 3 and splits.value > 1
    w, wd = tensor(12, out, K)
    x = P.make_x(1, M, K, BF16)
    xd = P.rounded(x)
    need = lib.mfq_hip_mx8_scaled_gemm_workspace_bytes(out, K, M, 0)
    from tyloquant_amd import runtime_mx8 as R8
    q = R8.mx8_quantize(x)
    part = lib.mfq_hip_mx8_scaled_gemm_workspace_bytes(out, K, M, 1)
    for room in (part, part // 2, part // splits.value, 0):
        ws = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
        y = torch.empty(M, out, device="cuda")
        L.check(lib.mfq_hip_mx8_scaled_gemm_rows(w.values.data_ptr(), w.scales.data_ptr(), out, K, 0, out, q.values.data_ptr(), 0, 0, q.scales.data_ptr(), M, 0, 0,
                                                 y.data_ptr(), L.X_F32, out, ws.data_ptr(), room, torch.cuda.current_stream().cuda_stream))
        P.check(y, xd, wd)


# ---- routed experts -------------------------------------------------------------------------------------------------
def routes(seed, T, R, E, dropped=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    score = torch.randn(T, E, generator=g, device="cuda") + torch.randn(E, generator=g, device="cuda")
    ids = score.topk(R, 1).indices.to(torch.int32)
    gone = torch.rand(T, R, generator=g, device="cuda") < dropped
    bad = torch.tensor([-1, E, -7, E + 100], dtype=torch.int32, device="cuda")[torch.arange(T * R, device="cuda").reshape(T, R) % 4]
    return torch.where(gone, bad, ids)


def check_pairs(got, xd, wd, ids, out, E, routed, glu, holds=None):
    """got [T, R, ..]: every pair against its expert, zeros where there is none"""
    T, R = ids.shape
    flat, got = ids.reshape(-1).long(), got.reshape(T * R, -1)
    none = (flat < 0) | (flat >= E)
    assert (got[none] == 0).all()
    for e in range(E):
        pairs = torch.nonzero(flat == e)[:, 0]
        if len(pairs):
            place = e if holds is None else holds[e]
            if place < 0:
                continue
            P.check(got[pairs], xd[pairs if routed else pairs // R], wd[place * out:(place + 1) * out], glu)


EXPERTS = [(1, 8, 16, 256, 256), (5, 2, 4, 128, 640), (8, 1, 3, 384, 128), (9, 2, 8, 256, 384), (61, 4, 12, 128, 512), (200, 2, 5, 256, 1024), (700, 8, 16, 384, 256),
           (2100, 2, 4, 256, 128), (40, 2, 70, 128, 256), (100, 2, 8, 128, 20608), (12, 2, 8, 128, 4608), (150, 2, 3, 128, 2176)]


@pytest.mark.parametrize("T,R,E,out,K", EXPERTS)
def test_experts(T, R, E, out, K):
    from tyloquant_amd import runtime_moe as RM
    from tyloquant_amd import runtime_mx8 as R8
    w, wd = tensor(T + E, E * out, K, out=out)
    for dropped in (0.0, 0.2):
        ids = routes(T, T, R, E, dropped)
        route = RM.build_moe_route_plan(ids, E)
        x = P.make_x(T, T, K, BF16)
        xd = P.rounded(x)
        check_pairs(R8.mx8_moe_matmul(w, x, route, out_dtype=FP32), xd, wd, ids, out, E, False, False)
        check_pairs(R8.mx8_moe_glu(w, R8.mx8_quantize(x), route), xd, wd, ids, out, E, False, True)
        x = P.make_x(T + 1, T * R, K, FP16)
        check_pairs(R8.mx8_moe_matmul(w, x, route, routed=True, out_dtype=BF16), P.rounded(x), wd, ids, out, E, True, False)
    everyone = torch.zeros_like(ids)      # all pairs to one expert, the same one twice in a token
    x = P.make_x(T, T, K, BF16)
    check_pairs(R8.mx8_moe_glu(w, x, RM.build_moe_route_plan(everyone, E), out_dtype=FP16), P.rounded(x), wd, everyone, out, E, False, True)
    nobody = torch.full_like(ids, -1)
    assert (R8.mx8_moe_matmul(w, x, RM.build_moe_route_plan(nobody, E)) == 0).all()


@pytest.mark.parametrize("T", [3, 50, 600])
def test_experts_of_another_pool_are_left_alone(T):
    from tyloquant_amd import runtime_moe as RM
    from tyloquant_amd import runtime_mx8 as R8
    E, out, K = 6, 128, 256
    w, wd = tensor(3, 3 * out, K, out=out)
    holds = [-1, 2, 0, -1, 1, -1]
    slot = torch.tensor(holds, dtype=torch.int32, device="cuda")
    ids = routes(T, T, 2, E, 0.1)
    route = RM.build_moe_route_plan(ids, E)
    x = P.make_x(T, T, K, BF16)
    out_rows = torch.full((T, 2, out), 5.0, device="cuda")
    R8.mx8_moe_into(w, x, route, out_rows, slot=slot)
    check_pairs(out_rows, P.rounded(x), wd, ids, out, E, False, False, holds)
    others = torch.isin(ids, torch.tensor([0, 3, 5], device="cuda"))
    assert (out_rows[others] == 5.0).all()


# ---- as programs use them -------------------------------------------------------------------------------------------
def test_graph_replays_and_streams():
    """captured calls of few rows, tiles, a split and experts, replayed among eager work; the same on a stream of its own; two at once"""
    from tyloquant_amd import runtime_moe as RM
    from tyloquant_amd import runtime_mx8 as R8
    w, _ = tensor(21, 512, 1024)
    pool, _ = tensor(22, 8 * 256, 1024, out=256)
    xs = [P.make_x(M, M, 1024, BF16) for M in (1, 24, 70, 600)]
    ids = routes(23, 600, 2, 8, 0.1)

    def work():
        route = RM.build_moe_route_plan(ids, 8)
        return [R8.mx8_scaled_matmul(w, x) for x in xs] + [R8.mx8_scaled_glu(w, x) for x in xs] + [R8.mx8_moe_glu(pool, xs[3], route)]

    side, graphs, outs = torch.cuda.Stream(), [], []
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(work())
        graphs.append(g)
    for k in range(3):
        for x in xs:
            x.copy_(P.make_x(100 + k, x.shape[0], 1024, BF16))
        want = work()
        for g, got in zip(graphs, outs):
            for o in got:
                o.fill_(3.0)
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want))
    other = torch.cuda.Stream()
    for s in (side, other):
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for s in (side, other):
        with torch.cuda.stream(s):
            got.append([work() for _ in range(3)][-1])
    torch.cuda.synchronize()
    for both in got:
        assert all(torch.equal(a, b) for a, b in zip(both, want))


def test_results_do_not_change_from_call_to_call():
    from tyloquant_amd import runtime_mx8 as R8
    w, _ = tensor(31, 384, 4096)
    for M in (3, 30, 100):
        x = P.make_x(M, M, 4096, BF16)
        first = R8.mx8_scaled_matmul(w, x)
        assert all(torch.equal(first, R8.mx8_scaled_matmul(w, x)) for _ in range(5))
        assert torch.equal(first, R8.mx8_scaled_matmul(w, R8.mx8_quantize(x)))
