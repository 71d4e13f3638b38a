"""Products of microscaled operands on the GPU against 64-bit sums over the same codes: quantisation bit by bit, every kernel behind
mx_scaled_matmul / mx_scaled_glu / mx_moe_matmul / mx_moe_glu, their borders, refusals of the host layer, graphs and streams."""
import numpy as np
import pytest
import torch

import mx_scaled_ref as P

pytestmark = pytest.mark.gpu
ACTS = ("MXFP4", "MXFP6")
L2 = 1e-6    # 2-norm: roundings of fp32 sums do not line up


def hidden(rng, rows, K, scale=1.0):
    x = rng.standard_normal((rows, K)) * scale
    x[:, rng.permutation(K)[: max(1, K // 1000)]] *= 20
    return torch.from_numpy(x)


def make_weight(rng, rows, K, out=None):
    from tyloquant_amd.runtime_mx import MxWeight
    v, s, w = P.weight(rng, rows, K)
    return MxWeight.from_tensors("MXFP4", torch.from_numpy(v).cuda(), torch.from_numpy(s).cuda(), out=out), w


def quantized(x, act):
    """fp64 values of the rows after quantisation, from the oracle"""
    codes, scales = P.quantize(x.double().cpu().numpy(), act)
    return P.values(codes, scales, act)


# ---- quantisation ---------------------------------------------------------------------------------------------------
def same_rows(q, x, act):
    M, K = q.rows, q.neuron_len
    codes, scales = P.quantize(x.double().cpu().numpy().reshape(M, K), act)
    got = P.plain_scales(q.scales.cpu().numpy(), M, K)
    assert np.array_equal(got[:, : K // 32], scales) and not got[:, K // 32:].any()
    assert np.array_equal(q.values.cpu().numpy(), P.pack(codes, act))
    return P.values(codes, scales, act)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_every_16_bit_pattern(act, dtype):
    """All patterns of the type in blocks of neighbours (one binade each) and shuffled (blocks of all magnitudes, infinities and NaN in
    some), and without those two."""
    from tyloquant_amd import runtime_mx as RX
    bits = np.arange(65536, dtype=np.uint32).astype(np.uint16)
    rng = np.random.default_rng(3)
    for order in (bits, rng.permutation(bits)):
        x = torch.from_numpy(order.view(np.int16).copy()).view(dtype)
        for rows in (x, x[torch.isfinite(x)]):
            rows = rows[: rows.numel() // 256 * 256].reshape(-1, 256)
            q = RX.mx_quantize(rows.cuda(), act)
            want = same_rows(q, rows, act)
            P.check(q.dequantize(), want, np.zeros_like(want), "float32")
            if dtype == torch.float16:      # the values fit the type they came from, but for fp16's last subnormal steps
                got = q.dequantize(torch.float16).cpu()
                assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(torch.from_numpy(want).float().half()))


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("rows,K", [(1, 32), (1, 4096), (3, 96), (5, 1440), (17, 288), (300, 2880), (64, 17408)])
def test_quantize_sizes_types_and_strides(act, rows, K):
    from tyloquant_amd import runtime_mx as RX
    rng = np.random.default_rng(rows + K)
    x = hidden(rng, rows, K + 24)
    x[0, 3] = 0.0
    x[-1, 24:56] = 0.0                          # a block of zeros
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        t = x.to(dtype).cuda()
        for part in (t[:, :K].contiguous(), t[:, :K], t[:, 8: K + 8], t[:, 5: K + 5], t[:, 24: K + 24]):
            q = RX.mx_quantize(part, act)
            want = same_rows(q, part, act)
            for out in (torch.float32, torch.bfloat16, torch.float16):
                assert torch.equal(q.dequantize(out).cpu(), torch.from_numpy(want).float().to(out))
    shaped = RX.mx_quantize(t[:, :K].reshape(1, rows, K), act)
    assert shaped.shape == (1, rows, K) and shaped.dequantize().shape == (1, rows, K)
    assert RX.mx_quantize(t[:0, :K], act).dequantize().shape == (0, K)


@pytest.mark.parametrize("act", ACTS)
def test_quantize_fp32_extremes(act):
    """Magnitudes from fp32's subnormals to its largest, exact halves between codes, signed zeros."""
    from tyloquant_amd import runtime_mx as RX
    rng = np.random.default_rng(5)
    grid = P.GRID[act]
    mid = (grid[1:] + grid[:-1]) / 2
    near = np.concatenate([grid, mid, np.nextafter(mid.astype(np.float32), np.float32(0)), np.nextafter(mid.astype(np.float32), np.float32(1e9)), -mid, -grid])
    near = np.resize(near, (len(near) // 31 + 1) * 31).reshape(-1, 31)
    near = np.concatenate([np.full((len(near), 1), grid[-1]), near], 1)              # the largest element fixes the scale
    blocks = [near * 2.0 ** e for e in (-140, -126, -100, 0, 90, 118)]
    blocks.append(np.exp2(rng.uniform(-149, 127.9, (500, 32))) * rng.choice([-1, 1], (500, 32)))
    blocks.append(np.zeros((2, 32)) * np.array([[1], [-1]]))
    with np.errstate(over="ignore"):
        x = np.concatenate(blocks).astype(np.float32)
    x[4, 7], x[9, 0], x[11, 31] = np.inf, -np.inf, np.nan
    x = torch.from_numpy(x)
    q = RX.mx_quantize(x.cuda(), act)
    want = same_rows(q, x, act)
    P.check(q.dequantize(), want, np.zeros_like(want), "float32")


# ---- one tensor ---------------------------------------------------------------------------------------------------
SHAPES = [  # rows, out, K: streamed with the rows in LDS, through the ring, two tiles; tiles of three sizes; pieces of K; ragged everything
    (1, 16, 32), (1, 48, 96), (1, 4096, 4096), (2, 100, 1440), (5, 257, 512), (7, 64, 17408), (13, 1000, 2880), (16, 33, 12288), (3, 4096, 288),
    (16, 512, 256), (17, 96, 544), (31, 130, 4096), (32, 2048, 1440), (33, 128, 288), (64, 300, 4096), (65, 129, 1440), (100, 4096, 2048),
    (129, 1000, 2880), (200, 256, 96), (300, 2048, 4096), (257, 17408, 512), (601, 4096, 544), (1024, 9000, 1024), (2049, 4112, 352)]


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("rows,out,K", SHAPES)
def test_scaled_matmul(act, rows, out, K):
    from tyloquant_amd import runtime_mx as RX
    rng = np.random.default_rng(rows * 7 + out + K)
    w, wv = make_weight(rng, out, K)
    for dtype, result in ((torch.bfloat16, torch.float32), (torch.float16, torch.bfloat16), (torch.float32, torch.float16)):
        x = hidden(rng, rows, K).to(dtype)
        xq = quantized(x, act)
        want = xq @ wv.T
        err = P.sum_bound(xq, wv)
        y = RX.mx_scaled_matmul(w, x.cuda(), act=act, out_dtype=result)
        assert y.dtype == result and y.shape == (rows, out)
        P.check(y, want, err, str(result)[6:], L2)
        again = RX.mx_scaled_matmul(w, RX.mx_quantize(x.cuda(), act), out_dtype=result)
        P.check(again, want, err, str(result)[6:], L2)
        if out % 2 == 0 and result != torch.float32:
            for gelu in (False, True):
                h = RX.mx_scaled_glu(w, x.cuda(), act=act, activation=int(gelu), out_dtype=result)
                assert h.shape == (rows, out // 2)
                P.check(h, P.glu(want, gelu), P.glu_bound(want, err, gelu), str(result)[6:])


@pytest.mark.parametrize("act", ACTS)
def test_scaled_matmul_strided_rows_experts_and_shapes(act):
    from tyloquant_amd import runtime_mx as RX
    rng = np.random.default_rng(11)
    w, wv = make_weight(rng, 3 * 80, 352, out=80)
    for rows in (1, 4, 40, 300):
        wide = hidden(rng, rows, 352 + 40).to(torch.bfloat16).cuda()
        for part in (wide[:, :352], wide[:, 3: 355], wide[:, 40:]):
            xq = quantized(part, act)
            for e in (0, 2):
                we = wv[e * 80: e * 80 + 80]
                P.check(RX.mx_scaled_matmul(w, part, act=act, expert=e), xq @ we.T, P.sum_bound(xq, we), "float32")
    x3 = wide[:, :352].reshape(3, 100, 352)
    y3 = RX.mx_scaled_matmul(w, x3, act=act, expert=1)
    assert y3.shape == (3, 100, 80) and torch.equal(y3.reshape(300, 80), RX.mx_scaled_matmul(w, wide[:, :352], act=act, expert=1))
    assert RX.mx_scaled_matmul(w, wide[:0, :352], act=act).shape == (0, 80)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("rows", [1, 16, 20, 40, 150, 600])
def test_nan_and_extreme_scales(act, rows):
    """Scale byte 255 of a weight block makes its neuron NaN, an infinity or a NaN in a row of activations that row; scales 0 and 254
    and K that ends inside a macro; nothing else is touched."""
    from tyloquant_amd import runtime_mx as RX
    from tyloquant_amd.runtime_mx import MxWeight
    rng = np.random.default_rng(rows)
    v, s, _ = P.weight(rng, 272, 416)
    s[3, 0], s[100, 12], s[271, 5] = 255, 255, 255
    s[7, 2], s[8, 12] = 0, 200
    w = MxWeight.from_tensors("MXFP4", torch.from_numpy(v).cuda(), torch.from_numpy(s).cuda())
    wv = P.values(P.unpack(v), s, "MXFP4")
    x = hidden(rng, rows, 416).to(torch.bfloat16)
    if rows > 2:
        x[1, 5], x[rows - 1, 415] = float("inf"), float("nan")
    xq = quantized(x, act)
    with np.errstate(invalid="ignore"):
        want, err = xq @ wv.T, P.sum_bound(xq, wv)
    assert np.isnan(want).any() and not np.isnan(want).all()
    P.check(RX.mx_scaled_matmul(w, x.cuda(), act=act), want, np.nan_to_num(err), "float32")


# ---- routed experts -------------------------------------------------------------------------------------------------
def routes(rng, T, R, E, kind):
    if kind == "one":                                   # all on one expert, whose group is the whole batch
        ids = np.full((T, R), E - 1)
    else:
        p = np.exp(rng.standard_normal(E))
        ids = np.stack([rng.choice(E, R, replace=False, p=p / p.sum()) for _ in range(T)])
    if kind == "dropped":
        ids[rng.random((T, R)) < 0.2] = -1
        ids[0, 0] = E + 5
    return ids.astype(np.int32)


MOE = [  # tokens, routes, experts, out, K, how routed
    (1, 8, 64, 96, 288, "any"), (1, 1, 3, 16, 32, "any"), (5, 4, 8, 130, 1440, "dropped"), (8, 8, 16, 64, 512, "one"), (9, 2, 4, 48, 96, "dropped"),
    (9, 1, 200, 64, 352, "any"), (30, 4, 32, 300, 544, "dropped"), (61, 8, 64, 256, 512, "dropped"), (40, 4, 8, 144, 2880, "any"), (100, 1, 4, 128, 256, "one"),
    (200, 4, 16, 500, 288, "any"), (300, 2, 130, 64, 1440, "dropped"), (700, 8, 32, 272, 512, "dropped"), (513, 4, 8, 512, 352, "any"), (400, 2, 70, 96, 64, "one")]


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("T,R,E,out,K,how", MOE)
def test_moe_matmul(act, T, R, E, out, K, how):
    from tyloquant_amd import runtime_moe as RM
    from tyloquant_amd import runtime_mx as RX
    rng = np.random.default_rng(T + R + E + out + K)
    w, wv = make_weight(rng, E * out, K, out=out)
    wv = wv.reshape(E, out, K)
    ids = routes(rng, T, R, E, how)
    route = RM.build_moe_route_plan(torch.from_numpy(ids).cuda(), E)
    assert (route.ids_dst is None) == (T <= 8)
    for routed in (False, True):
        x = hidden(rng, T * R if routed else T, K).to(torch.bfloat16 if routed else torch.float16)
        xq = quantized(x, act)
        want, err = np.zeros((T * R, out)), np.zeros((T * R, out))
        for e in range(E):
            p = np.flatnonzero(ids.reshape(-1) == e)
            xe = xq[p if routed else p // R]
            want[p], err[p] = xe @ wv[e].T, P.sum_bound(xe, wv[e])
        for result in (torch.float32, torch.bfloat16):
            y = RX.mx_moe_matmul(w, x.cuda(), route, act=act, routed=routed, out_dtype=result)
            assert y.shape == (T, R, out)
            P.check(y, want.reshape(T, R, out), err.reshape(T, R, out), str(result)[6:])
            assert not y.reshape(T * R, out)[torch.from_numpy((ids.reshape(-1) < 0) | (ids.reshape(-1) >= E))].any()
        q = RX.mx_quantize(x.cuda(), act)
        P.check(RX.mx_moe_matmul(w, q, route, routed=routed), want.reshape(T, R, out), err.reshape(T, R, out), "float32")
        for gelu in (False, True):
            h = RX.mx_moe_glu(w, x.cuda(), route, act=act, routed=routed, activation=int(gelu), out_dtype=torch.float16)
            P.check(h, P.glu(want, gelu).reshape(T, R, -1), P.glu_bound(want, err, gelu).reshape(T, R, -1), "float16")
