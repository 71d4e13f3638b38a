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
    (1, 16, 32), (1, 48, 96), (1, 4096, 4096), (2, 100, 1440), (6, 300, 8192), (8, 40, 8224), (9, 64, 4096), (16, 1030, 4096), (15, 48, 4384), (5, 257, 512), (7, 64, 17408), (13, 1000, 2880), (16, 33, 12288), (3, 4096, 288),
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
    (9, 1, 200, 64, 352, "any"), (20, 3, 16, 48, 4096, "dropped"), (20, 3, 16, 48, 4128, "any"), (30, 4, 32, 300, 544, "dropped"), (61, 8, 64, 256, 512, "dropped"), (40, 4, 8, 144, 2880, "any"), (100, 1, 4, 128, 256, "one"),
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


def test_moe_slots_leave_other_cohorts_alone():
    """A pool that holds some of the experts, in an order of its own: rows of the others' pairs stay, rows of no expert become zeros."""
    from tyloquant_amd import runtime_moe as RM
    from tyloquant_amd import runtime_mx as RX
    rng = np.random.default_rng(21)
    E, out, K, held = 9, 80, 352, [7, 2, 4]
    w, wv = make_weight(rng, len(held) * out, K, out=out)
    slot = np.full(E, -1, np.int32)
    slot[held] = np.arange(len(held))
    for T, R in ((3, 4), (50, 2), (300, 3)):
        ids = rng.integers(-1, E, (T, R)).astype(np.int32)
        route = RM.build_moe_route_plan(torch.from_numpy(ids).cuda(), E)
        x = hidden(rng, T, K).to(torch.bfloat16)
        xq = quantized(x, "MXFP6")
        y = torch.full((T, R, out), 7.5, device="cuda")
        RX.mx_moe_into(w, x.cuda(), route, y, act="MXFP6", slot=torch.from_numpy(slot).cuda())
        want, err = np.full((T * R, out), 7.5), np.zeros((T * R, out))
        flat = ids.reshape(-1)
        want[flat < 0] = 0
        for e in held:
            p = np.flatnonzero(flat == e)
            we = wv[slot[e] * out: slot[e] * out + out]
            want[p], err[p] = xq[p // R] @ we.T, P.sum_bound(xq[p // R], we)
        P.check(y, want.reshape(T, R, out), err.reshape(T, R, out), "float32")


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("T,R", [(1300, 3), (30000, 2)])
def test_hundreds_of_experts_in_tiles(act, T, R):
    """More experts than the block that writes the table of tiles has threads, part of them in this pool, some without rows."""
    from tyloquant_amd import runtime_moe as RM
    from tyloquant_amd import runtime_mx as RX
    rng = np.random.default_rng(T + R)
    E, out, K = 300, 40, 64
    held = np.sort(rng.permutation(E)[:280])
    w, wv = make_weight(rng, len(held) * out, K, out=out)
    slot = np.full(E, -1, np.int32)
    slot[held] = np.arange(len(held))
    ids = np.minimum(rng.integers(-1, E, (T, R)), E - 9).astype(np.int32)      # eight experts get nothing, the one before many
    route = RM.build_moe_route_plan(torch.from_numpy(ids).cuda(), E)
    x = hidden(rng, T, K).to(torch.bfloat16)
    xq = quantized(x, act)
    want, err, flat = np.full((T * R, out), -2.5), np.zeros((T * R, out)), ids.reshape(-1)
    want[flat < 0] = 0
    for e in held:
        p = np.flatnonzero(flat == e)
        we = wv[slot[e] * out: slot[e] * out + out]
        want[p], err[p] = xq[p // R] @ we.T, P.sum_bound(xq[p // R], we)
    for rows in (x.cuda(), RX.mx_quantize(x.cuda(), act)):
        y = torch.full((T, R, out), -2.5, device="cuda")
        RX.mx_moe_into(w, rows, route, y, act=act, slot=torch.from_numpy(slot).cuda())
        P.check(y, want.reshape(T, R, out), err.reshape(T, R, out), "float32")


def mixed_moe(rng, E, out, K):
    """a NINTM tensor of two MXFP4 cohorts and a NINT4 one between them"""
    import synth
    from oracle import mfq_oracle as O
    from tyloquant_amd import formats as F
    from tyloquant_amd import runtime_moe as RM
    order = rng.permutation(E)
    parts = [np.sort(order[: E // 2]), np.sort(order[E // 2: E - 2]), np.sort(order[E - 2:])]
    pools, dense = [], np.zeros((E, out, K))
    for ids, fmt in zip(parts, ("MXFP4", "NINT4", "MXFP4")):
        if fmt == "MXFP4":
            v, s, d = P.weight(rng, len(ids) * out, K)
            blob = F.write_mx("MXFP4", len(ids) * out, K, v, s)
        else:
            t = synth.nint_random(rng, len(ids) * out, K, 4, 24, 6)
            blob, d = O.pack_nint(t), O.dequantize_nint(t).astype(np.float64)
        pools.append((ids.astype(np.int32), fmt, blob))
        dense[ids] = d.reshape(len(ids), out, K)
    return RM.NintMoeWeight.from_blob(F.nintm_blob(E, out, K, pools)), dense, parts


@pytest.mark.parametrize("T", [4, 40, 200])
@pytest.mark.parametrize("act", ACTS)
def test_mixed_tensor_takes_the_quantised_path_where_it_can(act, T):
    """NintMoeWeight.forward(act=...): MXFP4 cohorts as mx_moe_matmul, the NINT cohort as before; without act as before."""
    from tyloquant_amd import runtime_moe as RM
    rng = np.random.default_rng(T)
    E, out, K, R = 12, 96, 384, 3
    w, dense, parts = mixed_moe(rng, E, out, K)
    ids = rng.integers(0, E, (T, R)).astype(np.int32)
    route = RM.build_moe_route_plan(torch.from_numpy(ids).cuda(), E)
    x = hidden(rng, T, K).to(torch.bfloat16)
    got = w.forward(x.cuda(), route, act=act).double().cpu().numpy().reshape(T * R, out)
    plain = w.forward(x.cuda(), route).double().cpu().numpy().reshape(T * R, out)
    xq, x64, flat = quantized(x, act), x.double().numpy(), ids.reshape(-1)
    for e in range(E):
        p = np.flatnonzero(flat == e)
        if not len(p):
            continue
        exact = x64[p // R] @ dense[e].T
        if e in parts[1]:
            assert np.array_equal(got[p], plain[p])
        else:
            want = xq[p // R] @ dense[e].T
            assert (np.abs(got[p] - want) <= P.sum_bound(xq[p // R], dense[e])).all()
        assert np.linalg.norm(plain[p] - exact) <= 1e-3 * np.linalg.norm(exact)


@pytest.mark.parametrize("T", [1, 20, 150])
@pytest.mark.parametrize("act", ACTS)
def test_feed_forward_block_of_quantised_experts(act, T):
    """nint_moe_ffn_forward(act=...): router, gate/up with its GLU, down and the weighted sum as they run together; against 64 bits
    with the hidden rows rounded and quantised where the block does."""
    from tyloquant_amd import formats as F
    from tyloquant_amd import runtime_moe as RM
    rng = np.random.default_rng(T + 1)
    E, H, W, R = 10, 352, 160, 4
    ids = rng.permutation(E)
    tensors, dense = [], []
    for out, K in ((2 * W, H), (H, W)):
        pools, d = [], np.zeros((E, out, K))
        for part in (np.sort(ids[:6]), np.sort(ids[6:])):
            v, s, dv = P.weight(rng, len(part) * out, K)
            pools.append((part.astype(np.int32), "MXFP4", F.write_mx("MXFP4", len(part) * out, K, v, s)))
            d[part] = dv.reshape(len(part), out, K)
        tensors.append(RM.NintMoeWeight.from_blob(F.nintm_blob(E, out, K, pools)))
        dense.append(d)
    x = hidden(rng, T, H).to(torch.bfloat16)
    logits = torch.from_numpy(rng.standard_normal((T, E)).astype(np.float32))
    out, chosen, weights = RM.nint_moe_ffn_forward(*tensors, x.cuda(), logits.cuda(), R, normalize=True, act=act)
    chosen, weights = chosen.cpu().numpy(), weights.double().cpu().numpy()
    route = RM.build_moe_route_plan(torch.from_numpy(chosen).cuda(), E)
    hid = tensors[0].forward_glu(x.cuda(), route, act=act).cpu()          # fp16, as the block makes it
    xq = quantized(x, act)
    want_h, err_h, want, err = np.zeros((T, R, W)), np.zeros((T, R, W)), np.zeros((T, H)), np.zeros((T, H))
    for t in range(T):
        for r in range(R):
            e = chosen[t, r]
            y, b = xq[t: t + 1] @ dense[0][e].T, P.sum_bound(xq[t: t + 1], dense[0][e])
            want_h[t, r], err_h[t, r] = P.glu(y)[0], P.glu_bound(y, b)[0]
            hq = quantized(hid[t, r: r + 1], act)
            want[t] += weights[t, r] * (hq @ dense[1][e].T)[0]
            err[t] += abs(weights[t, r]) * P.sum_bound(hq, dense[1][e])[0]
    P.check(hid, want_h, err_h, "float16")
    # the weighted sum: R products and sums in fp32, each off by half a step of a partial sum
    err += (R + 1) * 2.0 ** -23 * (np.abs(want) + err)
    P.check(out, want, err + 1e-6 * np.abs(want).max(), "float32")


# ---- graphs, streams, borders ------------------------------------------------------------------------------------------
def test_captured_calls_replay():
    """Linear (fused, few rows, tiles with K split, gated), pairs and routed experts in one graph, replayed between eager work, against
    eager calls; a first use of a weight under capture is refused."""
    from tyloquant_amd import runtime_moe as RM
    from tyloquant_amd import runtime_mx as RX
    rng = np.random.default_rng(31)
    w, _ = make_weight(rng, 512, 2048)
    pool, _ = make_weight(rng, 8 * 128, 288, out=128)
    x = [torch.randn(m, 2048, device="cuda", dtype=torch.bfloat16) for m in (1, 9, 40)]
    xe = [torch.randn(t, 288, device="cuda", dtype=torch.bfloat16) for t in (2, 100)]
    routes_ = [RM.build_moe_route_plan(torch.from_numpy(routes(rng, t, 2, 8, "dropped")).cuda(), 8) for t in (2, 100)]

    def step():
        y = [RX.mx_scaled_matmul(w, v, act="MXFP6") for v in x] + [RX.mx_scaled_glu(w, x[2], act="MXFP4")]
        y += [RX.mx_moe_matmul(pool, v, r, act="MXFP4") for v, r in zip(xe, routes_)]
        return y + [RX.mx_quantize(x[1], "MXFP6").dequantize(torch.bfloat16)]

    eager = step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(4):
        for v in x + xe:
            v.copy_(torch.randn(v.shape, device="cuda"))
        eager = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, held)), k
    fresh, _ = make_weight(rng, 64, 256)
    with pytest.raises(RuntimeError, match="laid_scales"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            RX.mx_scaled_matmul(fresh, torch.zeros(1, 256, device="cuda", dtype=torch.bfloat16))
    assert RX.mx_scaled_matmul(fresh, torch.zeros(1, 256, device="cuda", dtype=torch.bfloat16)).shape == (1, 64)


def test_two_streams_and_repeated_calls_agree():
    """The same weight from two streams at once (each call has scratch of its own) gives the bits of one call alone."""
    from tyloquant_amd import runtime_mx as RX
    rng = np.random.default_rng(33)
    w, _ = make_weight(rng, 1024, 1440)
    xs = [torch.randn(m, 1440, device="cuda", dtype=torch.float16) for m in (1, 12, 70, 500)]
    alone = [RX.mx_scaled_matmul(w, x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for k in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append([RX.mx_scaled_matmul(w, x) for x in xs])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for ys in got for a, b in zip(ys, alone))


@pytest.mark.parametrize("rows", [1, 3, 16, 32, 50, 130])
def test_nothing_behind_the_results_is_written(rows):
    """The C call with a row stride above the results and rows behind the last; a workspace with no room for pieces of K."""
    from tyloquant_amd import _lib as L
    from tyloquant_amd.runtime import _stream
    rng = np.random.default_rng(rows)
    out, K, ldy = 102, 1440, 109
    w, wv = make_weight(rng, out, K)
    x = hidden(rng, rows, K).to(torch.bfloat16)
    xd, xq = x.cuda(), quantized(x, "MXFP4")
    want, err = xq @ wv.T, P.sum_bound(xq, wv)
    lib = L.lib()
    need = lib.mfq_hip_mx_scaled_gemm_workspace_bytes(4, out, K, rows, 0)
    least = 0 if need == 0 else -(-rows * 6 * 128 // 256) * 256 + -(-rows // 32) * 6 * 256
    for room in {need, least}:
        for dtype, code in ((torch.float32, L.X_F32), (torch.bfloat16, L.X_BF16)):
            y = torch.full((rows + 2, ldy), -3.0, dtype=dtype, device="cuda")
            ws = torch.empty(max(room, 16), dtype=torch.uint8, device="cuda")
            L.check(lib.mfq_hip_mx_scaled_gemm_rows(w.values.data_ptr(), w.laid_scales().data_ptr(), out, K, 0, out, 4, xd.data_ptr(), L.X_BF16, K, None,
                                                    rows, 0, 0, y.data_ptr(), code, ldy, ws.data_ptr(), room, _stream()))
            P.check(y[:rows, :out], want, err, str(dtype)[6:])
            assert (y[rows:] == -3).all() and (y[:, out:] == -3).all()
    if need:
        rc = lib.mfq_hip_mx_scaled_gemm_rows(w.values.data_ptr(), w.laid_scales().data_ptr(), out, K, 0, out, 4, xd.data_ptr(), L.X_BF16, K, None,
                                             rows, 0, 0, y.data_ptr(), code, ldy, ws.data_ptr(), least - 1, _stream())
        assert rc == L.ERR_WORKSPACE


def test_long_rows():
    """K past what the LDS holds of activations, for one row, a few and two tiles; offsets of a tensor of many rows."""
    from tyloquant_amd import runtime_mx as RX
    rng = np.random.default_rng(41)
    for out, K, ms in ((20, 70016, (1, 3, 20)), (70000, 64, (1, 5, 40))):
        w, wv = make_weight(rng, out, K)
        for m in ms:
            x = hidden(rng, m, K).to(torch.bfloat16)
            for act in ACTS:
                xq = quantized(x, act)
                P.check(RX.mx_scaled_matmul(w, x.cuda(), act=act), xq @ wv.T, P.sum_bound(xq, wv), "float32", L2)


def test_cpp_runtime_linear():
    """mfq_rt_linear_forward_scaled on a loaded MXFP4 blob: the bits of the Python layer; its refusals."""
    import ctypes as C
    from pathlib import Path
    from tyloquant_amd import _lib as L
    from tyloquant_amd import formats as F
    from tyloquant_amd import runtime as R
    from tyloquant_amd import runtime_mx as RX
    rt = C.CDLL(str(Path(R.__file__).resolve().parent / "lib" / "libmfq_runtime.so"))
    rt.mfq_rt_last_error.restype = C.c_char_p
    rt.mfq_rt_load_quant_linear.argtypes = [C.c_char_p, C.c_char_p, C.c_size_t, C.POINTER(C.c_void_p)]
    rt.mfq_rt_free_quant_linear.argtypes = [C.c_void_p]
    rt.mfq_rt_linear_forward_scaled.argtypes = [C.c_void_p, C.c_int, C.c_void_p, C.c_int, C.c_int64, C.c_int, C.c_int, C.c_int, C.c_void_p, C.c_int,
                                                C.c_void_p]
    rng = np.random.default_rng(51)
    v, s, _ = P.weight(rng, 160, 1440)
    blob = F.write_mx("MXFP4", 160, 1440, v, s)
    lin = R.load_quant_linear("MXFP4", blob).weight
    h = C.c_void_p()
    assert rt.mfq_rt_load_quant_linear(b"MXFP4", blob, len(blob), C.byref(h)) == 0
    for m in (200, 1, 9):
        x = hidden(rng, m, 1440).to(torch.float16).cuda()
        for glu, act in ((0, 4), (1, 6)):
            y = torch.empty((m, 80 if glu else 160), dtype=torch.bfloat16, device="cuda")
            assert rt.mfq_rt_linear_forward_scaled(h, act, x.data_ptr(), L.X_F16, 1440, m, glu, 0, y.data_ptr(), L.X_BF16, None) == 0
            torch.cuda.synchronize()
            call = RX.mx_scaled_glu if glu else RX.mx_scaled_matmul
            assert torch.equal(y, call(lin, x, act="MXFP4" if act == 4 else "MXFP6", out_dtype=torch.bfloat16))
    assert rt.mfq_rt_linear_forward_scaled(h, 8, x.data_ptr(), L.X_F16, 1440, 9, 0, 0, y.data_ptr(), L.X_BF16, None) != 0
    assert b"kind 8" in rt.mfq_rt_last_error()
    rt.mfq_rt_free_quant_linear(h)


def test_cpp_runtime_capture():
    """A first product under capture is refused and leaves the handle good; a captured one replays after calls that need more room."""
    import ctypes as C
    from pathlib import Path
    from tyloquant_amd import _lib as L
    from tyloquant_amd import formats as F
    from tyloquant_amd import runtime as R
    from tyloquant_amd import runtime_mx as RX
    rt = C.CDLL(str(Path(R.__file__).resolve().parent / "lib" / "libmfq_runtime.so"))
    rt.mfq_rt_last_error.restype = C.c_char_p
    rt.mfq_rt_load_quant_linear.argtypes = [C.c_char_p, C.c_char_p, C.c_size_t, C.POINTER(C.c_void_p)]
    rt.mfq_rt_free_quant_linear.argtypes = [C.c_void_p]
    rt.mfq_rt_linear_forward_scaled.argtypes = [C.c_void_p, C.c_int, C.c_void_p, C.c_int, C.c_int64, C.c_int, C.c_int, C.c_int, C.c_void_p, C.c_int,
                                                C.c_void_p]
    rng = np.random.default_rng(53)
    v, s, _ = P.weight(rng, 512, 2080)
    blob = F.write_mx("MXFP4", 512, 2080, v, s)
    lin = R.load_quant_linear("MXFP4", blob).weight
    h = C.c_void_p()
    assert rt.mfq_rt_load_quant_linear(b"MXFP4", blob, len(blob), C.byref(h)) == 0
    x = [hidden(rng, m, 2080).to(torch.bfloat16).cuda() for m in (9, 40, 700)]
    y = [torch.empty((len(t), 512), device="cuda") for t in x]

    def call(i):
        return rt.mfq_rt_linear_forward_scaled(h, 6, x[i].data_ptr(), L.X_BF16, 2080, len(x[i]), 0, 0, y[i].data_ptr(), L.X_F32,
                                               torch.cuda.current_stream().cuda_stream)
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        assert call(0) != 0
        y[2].zero_()
    assert b"before a graph is captured" in rt.mfq_rt_last_error()
    assert call(0) == 0
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert call(0) == 0
    for k in range(3):
        assert call(1) == 0 and call(2) == 0
        x[0].copy_(hidden(rng, 9, 2080))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, RX.mx_scaled_matmul(lin, b)) for a, b in zip(y, x)), k
    del graph
    rt.mfq_rt_free_quant_linear(h)


def test_refusals_of_the_host_layer():
    from tyloquant_amd import runtime_moe as RM
    from tyloquant_amd import runtime_mx as RX
    from tyloquant_amd.runtime_mx import MxRows, MxWeight
    rng = np.random.default_rng(43)
    w, _ = make_weight(rng, 64, 256, out=32)
    x = torch.zeros(3, 256, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="MXFP4 or MXFP6"):
        RX.mx_quantize(x, "MXFP8")
    with pytest.raises(ValueError, match="divisible by 32"):
        RX.mx_quantize(x[:, :40])
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        RX.mx_quantize(x.double())
    with pytest.raises(ValueError, match="current GPU"):
        RX.mx_quantize(x.cpu())
    with pytest.raises(ValueError, match="width 128 != neuron length 256"):
        RX.mx_scaled_matmul(w, x[:, :128])
    with pytest.raises(ValueError, match="width 128 != neuron length 256"):
        RX.mx_scaled_matmul(w, RX.mx_quantize(x[:, :128]))
    with pytest.raises(ValueError, match="MXFP4 or MXFP6"):
        RX.mx_scaled_matmul(w, x, act="MXFP8")
    with pytest.raises(TypeError, match="results are"):
        RX.mx_scaled_matmul(w, x, out_dtype=torch.float64)
    with pytest.raises(ValueError, match="16-bit type"):
        RX.mx_scaled_glu(w, x, out_dtype=torch.float32)
    with pytest.raises(IndexError):
        RX.mx_scaled_matmul(w, x, expert=2)
    route = RM.build_moe_route_plan(torch.zeros(3, 2, dtype=torch.int32, device="cuda"), 2)
    with pytest.raises(ValueError, match="3 rows for 3 tokens of 2 routes"):
        RX.mx_moe_matmul(w, x, route, routed=True)
    with pytest.raises(ValueError, match="2 experts, a route plan for 3"):
        RX.mx_moe_matmul(w, x, RM.build_moe_route_plan(route.ids, 3))
    with pytest.raises(ValueError, match="uint8"):
        MxRows("MXFP4", torch.zeros(3, 128, device="cuda"), torch.zeros(256, device="cuda"), (3, 256))
    with pytest.raises(ValueError, match="must be contiguous uint8"):
        MxRows("MXFP6", torch.zeros(3, 128, device="cuda", dtype=torch.uint8), torch.zeros(256, device="cuda", dtype=torch.uint8), (3, 256))
    with pytest.raises(ValueError, match="current GPU, got cpu"):
        RX.mx_moe_into(w, x, route, torch.empty(3, 2, 32, device="cuda"), slot=torch.zeros(2, dtype=torch.int32))
    moe, _, _ = mixed_moe(rng, 8, 64, 96)
    for call in (moe.forward, moe.forward_glu):
        with pytest.raises(ValueError, match="MXFP4 or MXFP6"):
            call(torch.zeros(3, 96, device="cuda"), RM.build_moe_route_plan(route.ids, 8), act="MXFP8")
    v8, s8 = torch.zeros(128, 128, device="cuda", dtype=torch.uint8), torch.zeros(1, 1, device="cuda", dtype=torch.uint8)
    with pytest.raises(ValueError, match="use mx_matmul"):
        RX.mx_scaled_matmul(MxWeight.from_tensors("MXFP8", v8, s8), x[:, :128])
    with pytest.raises(ValueError, match="values .* and scales"):
        MxWeight.from_tensors("MXFP4", v8, s8)
