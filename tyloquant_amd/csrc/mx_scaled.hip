// Products of microscaled operands (mx_scaled.hpp): MXFP4 weights, read in place, against activations quantised to MXFP4 or MXFP6; one
// tensor, or the tensors of routed experts.
#include "mx_scaled.hpp"

namespace mfq {
namespace {

enum MxsMode { kLinear = 0, kPairs = 1, kMapped = 2 };

// ---- tiles of routed experts --------------------------------------------------------------------------------------------------
// Rows of expert e, pairs bounds[e] .. bounds[e + 1] of the route map, are cut into tiles of `rows`.  Every wave finds its tile from the
// bounds themselves, 64 experts at a time.
__device__ __forceinline__ int mxs_tiles_of(const MxsArgs &a, int e, int rows) {
    if (e >= a.E || (a.slot && a.slot[e] < 0)) return 0;
    return (a.bounds[e + 1] - a.bounds[e] + rows - 1) / rows;
}
__device__ __forceinline__ int mxs_total_tiles(const MxsArgs &a, int rows, int lane) {
    int n = 0;
    for (int e = lane; e < a.E; e += 64) n += mxs_tiles_of(a, e, rows);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
    return __builtin_amdgcn_readfirstlane(n);
}
// the expert that tile t belongs to and the number of its first tile; t is below the total
__device__ __forceinline__ void mxs_find_tile(const MxsArgs &a, int rows, int lane, int t, int &expert, int &first) {
    int before = 0;
    expert = 0; first = 0;
    for (int c = 0; c < a.E; c += 64) {
        const int n = mxs_tiles_of(a, c + lane, rows);
        int upto = n;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int other = __shfl_up(upto, o, 64);
            if (lane >= o) upto += other;
        }
        const unsigned long long over = __ballot(before + upto > t);
        if (over) {
            const int l = __ffsll(over) - 1;
            expert = c + l;
            first = before + __builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(n, l);
            return;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
    }
}
// Pairs whose expert id is none get rows of zeros: each block looks at its share of the pairs.
__device__ __forceinline__ void mxs_zero_rows(const MxsArgs &a, int block, int blocks, int tid, int nt) {
    const int cols = a.glu ? a.nrows / 2 : a.nrows, words = cols * (a.y_dtype == MFQ_X_F32 ? 2 : 1);  // of two bytes
    for (int p = block; p < a.pairs; p += blocks) {
        const int e = a.ids[p];
        if (e >= 0 && e < a.E) continue;
        uint16_t *row = static_cast<uint16_t *>(a.y) + static_cast<int64_t>(p) * a.ldy * (a.y_dtype == MFQ_X_F32 ? 2 : 1);
        for (int i = tid; i < words; i += nt) row[i] = 0;
    }
}

// ---- few rows, long K -------------------------------------------------------------------------------------------------------------
// A block owns NB row-blocks of 16 neurons (with GLU one of gate rows and that of their up rows) and up to 16 * MT rows of activations; its
// waves take the macros of K in turn, each through a ring of two stages of its own in LDS (no barrier in the loop), activations and weights
// alike, and their sums meet in LDS.  For rows of activations that do not fit the LDS beside the weights' ring (flow kernel, below).
template <int AK, int MT, int NB>
struct StreamShape {
    static constexpr int W = NB * 2048, WS = 256, X = MT * 16 * mx_macro_bytes(AK), XS = 256;
    static constexpr int STAGE = W + WS + X + XS;
    static constexpr int REQ = 2 * NB + 1 + MT * (AK == 4 ? 2 : 3) + 1;  // requests of a stage
};

template <int AK, int MT, int NB, int MODE>
__global__ __launch_bounds__(512) void mxs_stream_kernel(MxsArgs a) {
    using S = StreamShape<AK, MT, NB>;
    constexpr int D = 2;
    static_assert(NB <= 2 && MT <= 2, "a stage's scales are one request of four bytes a lane");
    extern __shared__ __attribute__((aligned(128))) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, nwaves = blockDim.x >> 6;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15, g = lane >> 4;
    const int nblk = a.K / 32, nmac = (nblk + 7) / 8;
    constexpr int XMAC = mx_macro_bytes(AK);
    const int64_t wrow = a.K / 2, xrow = static_cast<int64_t>(nmac) * XMAC;
    const int width = a.glu ? a.nrows / 2 : a.nrows;  // results of a row

    int expert = 0, m0 = 0, rows = a.M, first = 0;
    if constexpr (MODE == kMapped) {
        if (blockIdx.x == 0) mxs_zero_rows(a, blockIdx.y, gridDim.y, tid, blockDim.x);
        if (static_cast<int>(blockIdx.y) >= mxs_total_tiles(a, 16 * MT, lane)) return;
        int t0;
        mxs_find_tile(a, 16 * MT, lane, blockIdx.y, expert, t0);
        first = a.bounds[expert] + (static_cast<int>(blockIdx.y) - t0) * 16 * MT;
        rows = min(16 * MT, a.bounds[expert + 1] - first);
    } else {
        m0 = static_cast<int>(blockIdx.y) * 16 * MT;
        rows = min(16 * MT, a.M - m0);
    }
    if constexpr (MODE != kLinear) {
        if (a.slot) expert = a.slot[expert];
        if (expert < 0) return;
        expert = __builtin_amdgcn_readfirstlane(expert);
    }
    // row of the activations, and of y, that row m of the block is
    auto pair_of = [&](int m) { return MODE == kMapped ? a.ids_dst[first + m] : m0 + m; };
    auto src_of = [&](int m) {
        const int p = pair_of(m);
        return MODE == kLinear || a.routed ? p : p / a.R;
    };
    // neuron of row i of row-block b: with GLU the second row-block holds the up rows of the first one's gate rows
    const int n0 = static_cast<int>(blockIdx.x) * 16 * (a.glu ? NB / 2 : NB);
    auto neuron = [&](int b, int i) {
        if (NB == 2 && a.glu) return b * width + min(n0 + i, width - 1);
        return min(n0 + b * 16 + i, a.nrows - 1);
    };

    const uint8_t *wbase = a.wv + static_cast<int64_t>(expert) * a.nrows * wrow;
    const __amdgpu_buffer_rsrc_t win = wave_window(wbase, static_cast<uint32_t>(a.nrows * wrow));
    const __amdgpu_buffer_rsrc_t swin = wave_window(a.ws, 0xffffff00u);  // offsets of 32 bits from the first row: the host sees to it
    uint32_t wv[2 * NB];
    const int piece = lane & 7;
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i) {
        const int row = 8 * (i & 1) + (lane >> 3);
        wv[i] = static_cast<uint32_t>(neuron(i >> 1, row) * wrow) + 16u * (piece ^ mx_key(row));
    }
    const uint32_t wsv = mx_scale_at(a.row0 + expert * a.nrows + neuron(NB == 2 ? lane >> 5 : 0, (lane >> 1) & 15), nmac) + 4u * (lane & 1);
    // rows of a mapped tile lie anywhere: the window is all of them (under 2 GB, the host sees to it); else the block's own
    const int64_t base = MODE == kLinear ? m0 : 0;
    const int span = MODE == kLinear ? rows : a.M;
    const __amdgpu_buffer_rsrc_t xwin = wave_window(a.xv + base * xrow, static_cast<uint32_t>(span * xrow));
    const __amdgpu_buffer_rsrc_t xswin = wave_window(a.xs, 0xffffff00u);
    uint32_t xv[MT * 2], xv2[MT], xsv = 0;
    {
#pragma unroll
        for (int i = 0; i < MT * 2; ++i) {
            const int row = 8 * i + (lane >> 3);
            xv[i] = static_cast<uint32_t>((src_of(min(row, rows - 1)) - base) * xrow) + 16u * (piece ^ mx_key(row & 15));
        }
        if constexpr (AK == 6) {
#pragma unroll
            for (int t = 0; t < MT; ++t)
                xv2[t] = static_cast<uint32_t>((src_of(min(16 * t + (lane >> 2), rows - 1)) - base) * xrow) + 128u + 16u * row_order_quarter(lane >> 2, lane & 3);
        }
        xsv = mx_scale_at(src_of(min(MT == 2 ? lane >> 1 : (lane >> 1) & 15, rows - 1)), nmac) + 4u * (lane & 1);
    }

    uint8_t *ring = lds + wave * (D * S::STAGE);

    // Pieces of weights behind the last block of a row: the last one again.  The activations there are zeros.
    auto issue = [&](int stage, int mac) {
        uint8_t *to = ring + stage * S::STAGE;
        const int last = nblk - 1 - 8 * mac;  // of the macro's pieces
        const int xat = mac * XMAC;
#pragma unroll
        for (int i = 0; i < 2 * NB; ++i) {
            uint32_t off = wv[i];
            if (last < 7) off -= 16u * max(0, (piece ^ mx_key(8 * (i & 1) + (lane >> 3))) - last);
            copy16<2>(win, to + i * 1024, off, mac * 128);
        }
        if (NB == 2 || lane < 32) copy4(swin, to + S::W, wsv, mac * 256);
        {
            uint8_t *xto = to + S::W + S::WS;
#pragma unroll
            for (int i = 0; i < 2 * MT; ++i) copy16<0>(xwin, xto + i * 1024, xv[i], xat);
            if constexpr (AK == 6) {
#pragma unroll
                for (int t = 0; t < MT; ++t) copy16<0>(xwin, xto + (2 * MT + t) * 1024, xv2[t], xat);
            }
            if (MT == 2 || lane < 32) copy4(xswin, xto + S::X, xsv, mac * 256);
        }
    };

    const int mine = (nmac - wave + nwaves - 1) / nwaves;  // macros wave, wave + nwaves, ...
#pragma unroll
    for (int i = 0; i < D; ++i)
        if (i < mine) issue(i, wave + i * nwaves);

    float4_t acc[NB][MT];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[b][t] = float4_t{0.f, 0.f, 0.f, 0.f};
    const int key = mx_key(r);
    int stage = 0;
    for (int i = 0; i < mine; ++i) {
        // younger stages in flight: those of the next D - 1 macros
        const int left = mine - 1 - i;
        if (left >= 1) wait_vmcnt<S::REQ>();
        else wait_vmcnt<0>();
        const uint8_t *at = ring + stage * S::STAGE;
        u32x4_t w[2][NB];
        u32x4_t x[2][MT], tail[MT] = {};
        uint32_t sw[NB], sx[MT];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            sw[b] = *reinterpret_cast<const uint16_t *>(at + S::W + b * 128 + r * 8 + 2 * g);
#pragma unroll
            for (int s = 0; s < 2; ++s) w[s][b] = *reinterpret_cast<const u32x4_t *>(at + b * 2048 + r * 128 + (((2 * g + s) ^ key) << 4));
        }
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const uint8_t *x0 = at + S::W + S::WS;
            sx[t] = *reinterpret_cast<const uint16_t *>(x0 + S::X + t * 128 + r * 8 + 2 * g);
#pragma unroll
            for (int s = 0; s < 2; ++s) x[s][t] = *reinterpret_cast<const u32x4_t *>(x0 + t * 2048 + r * 128 + (((2 * g + s) ^ key) << 4));
            if constexpr (AK == 6) tail[t] = *reinterpret_cast<const u32x4_t *>(x0 + (2 * MT + t) * 1024 + row_order_lane(lane));
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the stage is free for the next copies
        if (i + D < mine) issue(stage, wave + (i + D) * nwaves);
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                acc[b][t] = mx_scale_mfma<AK, 0>(w[0][b], x[0][t], tail[t].x, tail[t].y, acc[b][t], sw[b], sx[t]);
                acc[b][t] = mx_scale_mfma<AK, 1>(w[1][b], x[1][t], tail[t].z, tail[t].w, acc[b][t], sw[b], sx[t]);
            }
        stage = stage + 1 == D ? 0 : stage + 1;
    }

    // sums over the waves; all copies have landed
    __syncthreads();
    float4_t *red = reinterpret_cast<float4_t *>(lds);
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int t = 0; t < MT; ++t) red[(wave * NB * MT + b * MT + t) * 64 + lane] = acc[b][t];
    __syncthreads();
    const int items = (NB == 2 && a.glu ? 1 : NB) * MT * 64;
    for (int i = tid; i < items; i += blockDim.x) {
        float4_t v = red[i];
        for (int k = 1; k < nwaves; ++k) {
            const float4_t o = red[k * NB * MT * 64 + i];
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] += o[j];
        }
        if (NB == 2 && a.glu) {
            float4_t u = red[MT * 64 + i];
            for (int k = 1; k < nwaves; ++k) {
                const float4_t o = red[(k * NB + 1) * MT * 64 + i];
#pragma unroll
                for (int j = 0; j < 4; ++j) u[j] += o[j];
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = glu_value(v[j], u[j], a.gelu);
        }
        const int b = i / (MT * 64), m = (i / 64) % MT * 16 + (i & 15), n = n0 + b * 16 + ((i >> 4) & 3) * 4;
        if (m >= rows) continue;
        const int64_t out = pair_of(m) * a.ldy + n;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (n + j < width) store_rounded(a.y, out + j, v[j], a.y_dtype);
    }
}

// ---- few rows ---------------------------------------------------------------------------------------------------------------------
// The activations of a tile of up to 16 * MT rows lie in LDS for the whole of K.  A block takes a range of row-blocks of 16 neurons (with GLU
// those of the gate rows, each with that of its up rows), macro after macro, as one stream that its waves share evenly; a wave keeps a ring of
// D stages of weights ahead, across the ends of row-blocks.  Sums of a row-block that lies in several waves' shares meet in LDS, in the order
// of the waves.  Bound by the weights' way from memory.  61 tokens of 8 routes over 64 experts of 4096 x 2048, MXFP4 (295 MB): 57 us with
// quantised rows, 61 quantising them, where a block for every 16 neurons, its waves on different macros (stream kernel), took 167; 12288 x 4096
// at 16 rows 10.9 us in a graph, 12.2 there.
// SMALL: rows that the block itself quantises where they come as bf16, fp16 or fp32; only as many as there are are kept (small_rows).
template <int AK, int MT, int NB>
struct FlowShape {
    static constexpr int W = NB * 2048, STAGE = W + 256, REQ = 2 * NB + 1;
    static constexpr int XM = MT * 16 * mx_macro_bytes(AK) + 256;  // a macro of activations and its scales
    static constexpr int small_macro(int rows) { return (rows * (mx_macro_bytes(AK) + 8) + 15) & ~15; }
};
__host__ __device__ __forceinline__ constexpr int rows_kept(int rows) { return rows > 8 ? 16 : rows > 4 ? 8 : rows > 2 ? 4 : rows; }

template <int AK, int MT, int NB, int D, int MODE, bool SMALL>
__global__ __launch_bounds__(512) void mxs_flow_kernel(MxsArgs a, int chunks) {
    using S = FlowShape<AK, MT, NB>;
    static_assert(NB <= 2 && MT <= 2 && (!SMALL || MT == 1), "a stage's scales are one request of four bytes a lane");
    static_assert(D == 3, "the waits of the loop");
    extern __shared__ __attribute__((aligned(128))) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, nwaves = blockDim.x >> 6;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15, g = lane >> 4;
    const int nblk = a.K / 32, nmac = (nblk + 7) / 8;
    constexpr int XMAC = mx_macro_bytes(AK);
    const int64_t wrow = a.K / 2, xrow = static_cast<int64_t>(nmac) * XMAC;
    const int width = NB == 2 ? a.nrows / 2 : a.nrows;  // results of a row

    const int tile = static_cast<int>(blockIdx.x) / chunks, chunk = static_cast<int>(blockIdx.x) - tile * chunks;
    int expert = 0, m0 = 0, first = 0, rows;
    if constexpr (MODE == kPairs) {
        expert = a.ids[tile];
        if (expert < 0 || expert >= a.E) {
            if (chunk == 0) mxs_zero_rows(a, tile, a.pairs, tid, blockDim.x);
            return;
        }
        if (a.slot) expert = a.slot[expert];
        if (expert < 0) return;
        expert = __builtin_amdgcn_readfirstlane(expert);
        rows = 1;
    } else if constexpr (MODE == kMapped) {
        mxs_zero_rows(a, blockIdx.x, gridDim.x, tid, blockDim.x);
        if (tile >= mxs_total_tiles(a, 16 * MT, lane)) return;
        int t0;
        mxs_find_tile(a, 16 * MT, lane, tile, expert, t0);
        first = a.bounds[expert] + (tile - t0) * 16 * MT;
        rows = min(16 * MT, a.bounds[expert + 1] - first);
        if (a.slot) expert = a.slot[expert];
        expert = __builtin_amdgcn_readfirstlane(expert);
    } else {
        m0 = tile * 16 * MT;
        rows = min(16 * MT, a.M - m0);
    }
    auto pair_of = [&](int m) { return MODE == kPairs ? tile : MODE == kMapped ? a.ids_dst[first + m] : m0 + m; };
    auto src_of = [&](int m) {
        const int p = pair_of(m);
        return MODE == kLinear || a.routed ? p : p / a.R;
    };
    // the block's row-blocks, and this wave's share of their macros
    const int rbs = (width + 15) / 16;
    const int rb0 = static_cast<int>(static_cast<int64_t>(rbs) * chunk / chunks), rb1 = static_cast<int>(static_cast<int64_t>(rbs) * (chunk + 1) / chunks);
    const int total = (rb1 - rb0) * nmac, item0 = static_cast<int>(static_cast<int64_t>(total) * wave / nwaves);
    const int items = static_cast<int>(static_cast<int64_t>(total) * (wave + 1) / nwaves) - item0;

    uint8_t *xres = lds + nwaves * (D * S::STAGE);
    const int kept = SMALL ? rows_kept(rows) : 16 * MT;  // rows of activations in LDS, a power of two
    const int xm = SMALL ? S::small_macro(kept) : S::XM, xtail = kept * 128, xsat = kept * XMAC;  // of a macro; where FP6's second part and the scales begin
    if constexpr (!SMALL) {
        // macro after macro as the copies of the kernel above leave them
        const int64_t base = MODE == kLinear ? m0 : 0;
        const int span = MODE == kLinear ? rows : a.M;
        const __amdgpu_buffer_rsrc_t xwin = wave_window(a.xv + base * xrow, static_cast<uint32_t>(span * xrow));
        const __amdgpu_buffer_rsrc_t xswin = wave_window(a.xs, 0xffffff00u);
        uint32_t xv[2 * MT], xv2[MT];
#pragma unroll
        for (int i = 0; i < 2 * MT; ++i) {
            const int row = 8 * i + (lane >> 3);
            xv[i] = static_cast<uint32_t>((src_of(min(row, rows - 1)) - base) * xrow) + 16u * ((lane & 7) ^ mx_key(row & 15));
        }
#pragma unroll
        for (int t = 0; t < MT; ++t)
            xv2[t] = static_cast<uint32_t>((src_of(min(16 * t + (lane >> 2), rows - 1)) - base) * xrow) + 128u + 16u * row_order_quarter(lane >> 2, lane & 3);
        const uint32_t xsv = mx_scale_at(src_of(min(MT == 2 ? lane >> 1 : (lane >> 1) & 15, rows - 1)), nmac) + 4u * (lane & 1);
        for (int mac = wave; mac < nmac; mac += nwaves) {
            uint8_t *to = xres + mac * xm;
            const int xat = mac * XMAC;
#pragma unroll
            for (int i = 0; i < 2 * MT; ++i) copy16<0>(xwin, to + i * 1024, xv[i], xat);
            if constexpr (AK == 6) {
#pragma unroll
                for (int t = 0; t < MT; ++t) copy16<0>(xwin, to + (2 * MT + t) * 1024, xv2[t], xat);
            }
            if (MT == 2 || lane < 32) copy4(xswin, to + xsat, xsv, mac * 256);
        }
    }

    const __amdgpu_buffer_rsrc_t win = wave_window(a.wv + static_cast<int64_t>(expert) * a.nrows * wrow, static_cast<uint32_t>(a.nrows * wrow));
    const __amdgpu_buffer_rsrc_t swin = wave_window(a.ws, 0xffffff00u);  // offsets of 32 bits from the first row: the host sees to it
    uint8_t *ring = lds + wave * (D * S::STAGE);
    const int piece = lane & 7;
    const uint32_t off0 = static_cast<uint32_t>((lane >> 3) * wrow) + 16u * (piece ^ mx_key(lane >> 3));
    const uint32_t off1 = static_cast<uint32_t>((8 + (lane >> 3)) * wrow) + 16u * (piece ^ mx_key(8 + (lane >> 3)));
    // the next copies: stage, row-block, macro
    int to_stage = 0, to_rb = rb0 + item0 / nmac, to_mac = item0 - item0 / nmac * nmac;
    uint32_t wsv = 0;
    auto scales_of = [&](int rb) {
        const int b = NB == 2 ? lane >> 5 : 0;
        return mx_scale_at(a.row0 + expert * a.nrows + b * width + min(rb * 16 + ((lane >> 1) & 15), width - 1), nmac) + 4u * (lane & 1);
    };
    wsv = scales_of(to_rb);
    auto issue = [&] {
        uint8_t *to = ring + to_stage * S::STAGE;
        const int last = nblk - 1 - 8 * to_mac, valid = width - to_rb * 16;
#pragma unroll
        for (int i = 0; i < 2 * NB; ++i) {
            const int row = 8 * (i & 1) + (lane >> 3);
            uint32_t off = i & 1 ? off1 : off0;
            // neurons behind the last one, and pieces of weights behind the last block of a row: the last ones again
            if (valid < 16) off -= static_cast<uint32_t>(max(0, row - (valid - 1)) * wrow);
            if (last < 7) off -= 16u * max(0, (piece ^ mx_key(row)) - last);
            copy16<2>(win, to + i * 1024, off, static_cast<int>(static_cast<uint32_t>((to_rb * 16 + (i >> 1) * width) * wrow) + to_mac * 128u));
        }
        if (NB == 2 || lane < 32) copy4(swin, to + S::W, wsv, to_mac * 256);
        to_stage = to_stage + 1 == D ? 0 : to_stage + 1;
        if (++to_mac == nmac) {
            to_mac = 0;
            wsv = scales_of(++to_rb);
        }
    };
    if constexpr (!SMALL)
        for (int i = 0; i < D; ++i)
            if (i < items) issue();
    if constexpr (SMALL) {
        // A thread a block of 32 columns: quantised here, or copied.  Before the first weights are asked for, behind which these reads would come
        // (4096 x 4096 in a graph, one row 5.7 -> 5.2 us, four 6.2 -> 5.6, sixteen 8.1 -> 7.8).
        const int per_row = nmac * 8;
        for (int u = tid; u < rows * per_row; u += blockDim.x) {
            const int m = u / per_row, block = u - m * per_row, p = block & 7;
            const int64_t src = src_of(m);
            u32x6_t q = {};
            uint32_t byte = 0;
            if (a.xraw) {
                if (block < nblk) {
                    const int64_t from = src * a.ldx + 32 * block;
                    if (a.x_dtype == MFQ_X_F32) a.x_wide ? mx_quantize_block<AK, MFQ_X_F32, true>(a.xraw, from, q, byte) : mx_quantize_block<AK, MFQ_X_F32, false>(a.xraw, from, q, byte);
                    else if (a.x_dtype == MFQ_X_F16) a.x_wide ? mx_quantize_block<AK, MFQ_X_F16, true>(a.xraw, from, q, byte) : mx_quantize_block<AK, MFQ_X_F16, false>(a.xraw, from, q, byte);
                    else a.x_wide ? mx_quantize_block<AK, MFQ_X_BF16, true>(a.xraw, from, q, byte) : mx_quantize_block<AK, MFQ_X_BF16, false>(a.xraw, from, q, byte);
                }
            } else {
                const uint8_t *row = a.xv + src * xrow + (block >> 3) * XMAC;
                const u32x4_t v = *reinterpret_cast<const u32x4_t *>(row + p * 16);
                q[0] = v.x; q[1] = v.y; q[2] = v.z; q[3] = v.w;
                if constexpr (AK == 6) {
                    const u32x2_t t = *reinterpret_cast<const u32x2_t *>(row + 128 + p * 8);
                    q[4] = t.x; q[5] = t.y;
                }
                byte = a.xs[mx_scale_at(src, nmac) + (block >> 3) * 256 + p];
            }
            uint8_t *to = xres + (block >> 3) * xm;
            *reinterpret_cast<u32x4_t *>(to + m * 128 + ((p ^ mx_key(m)) << 4)) = u32x4_t{q[0], q[1], q[2], q[3]};
            if constexpr (AK == 6) *reinterpret_cast<u32x2_t *>(to + xtail + m * 64 + row_order_quarter(m, p >> 1) * 16 + (p & 1) * 8) = u32x2_t{q[4], q[5]};
            to[xsat + m * 8 + p] = static_cast<uint8_t>(byte);
        }
        for (int i = 0; i < D; ++i)
            if (i < items) issue();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    } else {
        // what is older than the weights' first stages
        if (items >= D) wait_vmcnt<D * S::REQ>();
        else wait_vmcnt<0>();
    }
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");

    int64_t out_row[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) out_row[t] = t * 16 + r < rows ? static_cast<int64_t>(pair_of(t * 16 + r)) * a.ldy : -1;
    const bool f32 = a.y_dtype == MFQ_X_F32;
    const bool wide = a.ldy % 4 == 0 && reinterpret_cast<uintptr_t>(a.y) % 16 == 0;
    float4_t acc[NB][MT];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[b][t] = float4_t{0.f, 0.f, 0.f, 0.f};
    // results of row-block rb, from v (and u: gate and up)
    auto put = [&](int rb, const float4_t (&sum)[NB][MT]) {
        const int n = rb * 16 + 4 * g;
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            float4_t v = sum[0][t];
            if constexpr (NB == 2) {
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = glu_value(v[j], sum[1][t][j], a.gelu);
            }
            if (out_row[t] < 0 || n >= width) continue;
            if (wide && n + 4 <= width) {
                if (f32) *reinterpret_cast<float4_t *>(static_cast<float *>(a.y) + out_row[t] + n) = v;
                else *reinterpret_cast<u32x2_t *>(static_cast<uint16_t *>(a.y) + out_row[t] + n) =
                    u32x2_t{mx_pack16(v[0], v[1], a.y_dtype), mx_pack16(v[2], v[3], a.y_dtype)};
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (n + j < width) store_rounded(a.y, out_row[t] + n + j, v[j], a.y_dtype);
            }
        }
    };
    const int m_ = r & (kept - 1), key = mx_key(m_), xrow16 = SMALL ? m_ : r;
    const int wkey = mx_key(r);
    int stage = 0, rb = rb0 + item0 / nmac, mac = item0 - item0 / nmac * nmac;
    bool whole = mac == 0;  // of the current row-block from its first macro on
    float4_t head[NB][MT];  // the sums of a row-block that another wave has begun
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int t = 0; t < MT; ++t) head[b][t] = float4_t{0.f, 0.f, 0.f, 0.f};
    for (int i = 0; i < items; ++i) {
        // younger than this stage: those of the next D - 1 items, and the stores of results, which only make the wait longer
        const int left = items - 1 - i;
        if (left >= D - 1) wait_vmcnt<(D - 1) * S::REQ>();
        else if (left == 1) wait_vmcnt<S::REQ>();
        else wait_vmcnt<0>();
        const uint8_t *at = ring + stage * S::STAGE, *xat = xres + mac * xm;
        u32x4_t w[2][NB], x[2][MT], tail[MT] = {};
        uint32_t sw[NB], sx[MT];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            sw[b] = *reinterpret_cast<const uint16_t *>(at + S::W + b * 128 + r * 8 + 2 * g);
#pragma unroll
            for (int s = 0; s < 2; ++s) w[s][b] = *reinterpret_cast<const u32x4_t *>(at + b * 2048 + r * 128 + (((2 * g + s) ^ wkey) << 4));
        }
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            sx[t] = *reinterpret_cast<const uint16_t *>(xat + xsat + t * 128 + xrow16 * 8 + 2 * g);
#pragma unroll
            for (int s = 0; s < 2; ++s) x[s][t] = *reinterpret_cast<const u32x4_t *>(xat + t * 2048 + xrow16 * 128 + (((2 * g + s) ^ key) << 4));
            if constexpr (AK == 6)
                tail[t] = *reinterpret_cast<const u32x4_t *>(xat + xtail + t * 1024 + (SMALL ? m_ * 64 + row_order_quarter(m_, g) * 16 : row_order_lane(lane)));
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the stage is free for the next copies
        if (i + D < items) issue();
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                acc[b][t] = mx_scale_mfma<AK, 0>(w[0][b], x[0][t], tail[t].x, tail[t].y, acc[b][t], sw[b], sx[t]);
                acc[b][t] = mx_scale_mfma<AK, 1>(w[1][b], x[1][t], tail[t].z, tail[t].w, acc[b][t], sw[b], sx[t]);
            }
        stage = stage + 1 == D ? 0 : stage + 1;
        if (++mac < nmac) continue;
        if (whole) put(rb, acc);
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                if (!whole) head[b][t] = acc[b][t];
                acc[b][t] = float4_t{0.f, 0.f, 0.f, 0.f};
            }
        mac = 0;
        ++rb;
        whole = true;
    }
    if (total % nwaves == 0 && total / nwaves % nmac == 0) return;  // every row-block lies in one wave's share
    // Row-blocks of several shares: each wave leaves what it has of the one it came into (head) and of the one it stopped in.  A share within one
    // row-block, begun and not ended by it, is a head as well.
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int t = 0; t < MT; ++t)
            if (!whole) head[b][t] = acc[b][t];
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    float4_t *left = reinterpret_cast<float4_t *>(ring);
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            left[(b * MT + t) * 64 + lane] = head[b][t];
            left[(NB * MT + b * MT + t) * 64 + lane] = acc[b][t];
        }
    static_assert(2 * NB * MT * 1024 <= D * S::STAGE, "sums in the wave's ring");
    __syncthreads();
    auto wave_of = [&](int item) { return static_cast<int>((static_cast<int64_t>(item + 1) * nwaves - 1) / total); };
    for (int k = wave; k < rb1 - rb0; k += nwaves) {
        const int w0 = wave_of(k * nmac), w1 = wave_of(k * nmac + nmac - 1);
        if (w0 == w1) continue;
        float4_t sum[NB][MT];
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                sum[b][t] = reinterpret_cast<const float4_t *>(lds + w0 * (D * S::STAGE))[(NB * MT + b * MT + t) * 64 + lane];
                for (int o = w0 + 1; o <= w1; ++o) {
                    const float4_t v = reinterpret_cast<const float4_t *>(lds + o * (D * S::STAGE))[(b * MT + t) * 64 + lane];
#pragma unroll
                    for (int j = 0; j < 4; ++j) sum[b][t][j] += v[j];
                }
            }
        put(rb0 + k, sum);
    }
}

// ---- many rows: tiles -----------------------------------------------------------------------------------------------------------
// A block of WN * WM waves owns BN neurons x BM rows, a wave BN / WN x BM / WM of them in squares of 32.  K goes macro by macro through a
// ring of R stages in LDS.  Lane (r, h) multiplies block 4 h + s of the macro in step s of four, so its four scales are one word.  While
// the squares of a step are multiplied the fragments of the next are read; before the last step the macro has been read, its stage
// takes the macro R further on: one barrier a macro.  The 16-byte pieces of a line are turned by (row / 2) & 7 (FP6's second part: by
// (row / 4) & 3), with which the four passes of a read meet every bank once.
// What bounds it is the way of the operands from L2 to LDS and into L2: 16384 x 10240 at 4096 rows takes 372 us on the 256 x 256 tile, 286 us
// without its copies, 297 without its products, 180 with copies of the same two macros again and again (all in L2); the clock falls to
// 1.8 GHz meanwhile.  Tried and no faster: activations through registers half a macro out of step, copies and LDS reads between the
// squares one by one, lines asked for two to five macros ahead (a compute unit's requests are answered in their order).
// Lines of 64 bytes, half a macro a stage and twice as many stages, were slower (17408 x 5120 at 8192 rows: 635 us where whole lines in two
// stages of 16 x 16 squares had taken 475): a request fetches lines of 128 bytes.
template <int AK, int BN, int BM, int R>
struct TileShape {
    static constexpr int W = BN * 128, X = BM * 128, X2 = AK == 6 ? BM * 64 : 0, WS = BN * 8, XS = BM * 8;
    static constexpr int STAGE = W + X + X2 + WS + XS;
    static constexpr int LDS = R * STAGE + BM * 4;  // and the rows of y
};
// Partial results of a split over K: rows of two halves, each a whole number of 16 bytes, so that the up rows' sums of a gated product begin on
// such a boundary as well as the gate rows'.
__host__ __device__ __forceinline__ constexpr int part_half(int nrows) { return ((nrows + 1) / 2 + 3) / 4 * 4; }
constexpr int64_t part_bytes(int M, int nrows) { return static_cast<int64_t>(M) * part_half(nrows) * 8; }
constexpr int kTilePitch = 64 * 4 + 16, kTileOut = 32 * kTilePitch;  // 64 results of 32 rows on their way out

template <int AK, int BN, int BM, int WN, int WM, int R, int MODE>
__global__ __launch_bounds__(WN *WM * 64) __attribute__((amdgpu_waves_per_eu(BN * BM / (WN * WM) > 8192 ? 1 : 2))) void mxs_tile_kernel(MxsArgs a) {
    using S = TileShape<AK, BN, BM, R>;
    constexpr int NW = WN * WM, TN = BN / 32 / WN, TM = BM / 32 / WM;
    // requests of a wave for a stage; every wave issues as many, some twice
    constexpr int CW = BN / 8, CX = BM / 8, CT = AK == 6 ? BM / 16 : 0, DW = BN / 32, DX = BM / 32;
    constexpr int PW = (CW + NW - 1) / NW, PX = (CX + NW - 1) / NW, PT = (CT + NW - 1) / NW, QW = (DW + NW - 1) / NW, QX = (DX + NW - 1) / NW;
    constexpr int PER = PW + PX + PT + QW + QX, XMAC = mx_macro_bytes(AK);
    static_assert(TN % 2 == 0 && R >= 2, "gate and up in one wave");
    extern __shared__ __attribute__((aligned(128))) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wn = wave % WN, wm = wave / WN;
    const int r = lane & 31, h = lane >> 5;
    const int nblk = a.K / 32, nmac = (nblk + 7) / 8;
    const int64_t wrow = a.K / 2, xrow = static_cast<int64_t>(nmac) * XMAC;
    const int width = a.glu ? a.nrows / 2 : a.nrows, step = a.glu ? BN / 2 : BN;  // results of a row; of a tile
    const int tiles_n = (width + step - 1) / step;

    int tn = 0, tm = 0, expert = 0, first = 0, rows, m0 = 0;
    if constexpr (MODE == kMapped) {
        mxs_zero_rows(a, blockIdx.x, gridDim.x, tid, NW * 64);
        const int total = __builtin_amdgcn_readfirstlane(a.table[0].x) * tiles_n, per = (total + 7) / 8;
        const int t = (blockIdx.x & 7) * per + (blockIdx.x >> 3);  // an XCD takes neighbouring tiles
        if (t >= total || static_cast<int>(blockIdx.x >> 3) >= per) return;
        const i32x4v_t at = a.table[1 + t / tiles_n];
        expert = __builtin_amdgcn_readfirstlane(at.x);
        const int pairs = __builtin_amdgcn_readfirstlane(at.w), count = (pairs + BM - 1) / BM;
        const int in = t - __builtin_amdgcn_readfirstlane(at.y) * tiles_n;  // of the expert's tiles, those of the same neurons side by side
        tn = in / count;
        const int i = in % count * BM;
        first = __builtin_amdgcn_readfirstlane(at.z) + i;
        rows = min(BM, pairs - i);
    } else {
        if (!tile_of_block(tiles_n, (a.M + BM - 1) / BM, tn, tm)) return;
        m0 = tm * BM;
        rows = min(BM, a.M - m0);
    }
    const int n0 = tn * step;
    auto pair_of = [&](int m) { return MODE == kMapped ? a.ids_dst[first + m] : m0 + m; };
    auto src_of = [&](int m) {
        const int p = pair_of(m);
        return MODE == kLinear || a.routed ? p : p / a.R;
    };
    // neuron of row l of the tile: with GLU the second half of a wave's squares holds the up rows of the first half's gate rows
    auto neuron = [&](int l) {
        if (!a.glu) return min(n0 + l, a.nrows - 1);
        const int j = l >> 5, w_ = j / TN, t = j % TN;
        const int n = min(n0 + (w_ * (TN / 2) + t % (TN / 2)) * 32 + (l & 31), width - 1);
        return t < TN / 2 ? n : width + n;
    };
    int *row_of = reinterpret_cast<int *>(lds + R * S::STAGE);
    for (int m = tid; m < BM; m += NW * 64) row_of[m] = m < rows ? pair_of(m) : -1;

    const __amdgpu_buffer_rsrc_t win = wave_window(a.wv + static_cast<int64_t>(expert) * a.nrows * wrow, static_cast<uint32_t>(a.nrows * wrow));
    const __amdgpu_buffer_rsrc_t swin = wave_window(a.ws, 0xffffff00u);  // offsets of 32 bits from the first row: the host sees to it
    const int64_t base = MODE == kLinear ? m0 : 0;
    const int span = MODE == kLinear ? rows : a.M;
    const __amdgpu_buffer_rsrc_t xwin = wave_window(a.xv + base * xrow, static_cast<uint32_t>(span * xrow));
    const __amdgpu_buffer_rsrc_t xswin = wave_window(a.xs, 0xffffff00u);
    uint32_t wv[PW], xv[PX], xv2[PT > 0 ? PT : 1], wsv[QW], xsv[QX];
    const int wp = (lane & 7) ^ ((lane >> 4) & 3), wq = wp ^ 4;  // piece of the line that lane's copy takes, in the lower and upper half of 16 rows
#pragma unroll
    for (int p = 0; p < PW; ++p) {
        const int q = min(wave + NW * p, CW - 1);
        wv[p] = static_cast<uint32_t>(neuron(q * 8 + (lane >> 3)) * wrow) + 16u * (q & 1 ? wq : wp);
    }
#pragma unroll
    for (int p = 0; p < PX; ++p) {
        const int q = min(wave + NW * p, CX - 1);
        xv[p] = static_cast<uint32_t>((src_of(min(q * 8 + (lane >> 3), rows - 1)) - base) * xrow) + 16u * (q & 1 ? wq : wp);
    }
#pragma unroll
    for (int p = 0; p < PT; ++p)
        xv2[p] = static_cast<uint32_t>((src_of(min(min(wave + NW * p, CT - 1) * 16 + (lane >> 2), rows - 1)) - base) * xrow) + 128u +
                 16u * ((lane & 3) ^ ((lane >> 4) & 3));
#pragma unroll
    for (int p = 0; p < QW; ++p) wsv[p] = mx_scale_at(a.row0 + neuron(min(wave + NW * p, DW - 1) * 32 + (lane >> 1)) + expert * a.nrows, nmac) + 4u * (lane & 1);
#pragma unroll
    for (int p = 0; p < QX; ++p) xsv[p] = mx_scale_at(src_of(min(min(wave + NW * p, DX - 1) * 32 + (lane >> 1), rows - 1)), nmac) + 4u * (lane & 1);

    // Macros behind the last one: the last one again, into a stage that nobody reads.  Pieces of weights behind the last block of a row:
    // the last one again; the activations there are zeros.
    const int per_split = (nmac + a.splits - 1) / a.splits;
    const int st0 = static_cast<int>(blockIdx.y) * per_split, st1 = min(nmac, st0 + per_split);
    auto issue = [&](uint32_t buffer, int want) {
        const int st = min(want, st1 - 1);
        uint8_t *to = lds + buffer;
        const int last = nblk - 1 - 8 * st, xat = st * XMAC;
        const uint32_t back = last < 7 ? 16u * max(0, wp - last) : 0u, back2 = last < 7 ? 16u * max(0, wq - last) : 0u;
#pragma unroll
        for (int p = 0; p < PW; ++p) {
            const int q = min(wave + NW * p, CW - 1);
            copy16<0>(win, to + q * 1024, wv[p] - (q & 1 ? back2 : back), st * 128);
        }
#pragma unroll
        for (int p = 0; p < PX; ++p) copy16<0>(xwin, to + S::W + min(wave + NW * p, CX - 1) * 1024, xv[p], xat);
#pragma unroll
        for (int p = 0; p < PT; ++p) copy16<0>(xwin, to + S::W + S::X + min(wave + NW * p, CT - 1) * 1024, xv2[p], xat);
#pragma unroll
        for (int p = 0; p < QW; ++p) copy4(swin, to + S::W + S::X + S::X2 + min(wave + NW * p, DW - 1) * 256, wsv[p], st * 256);
#pragma unroll
        for (int p = 0; p < QX; ++p) copy4(xswin, to + S::W + S::X + S::X2 + S::WS + min(wave + NW * p, DX - 1) * 256, xsv[p], st * 256);
    };

    float16_t acc[TM][TN];
#pragma unroll
    for (int m = 0; m < TM; ++m)
#pragma unroll
        for (int n = 0; n < TN; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[m][n][i] = 0.f;

    // fragments of a step: those of the current one and the next
    u32x4_t w0[TN], w1[TN], x0[TM], x1[TM], tail[TM] = {}, tail2[TM] = {}, tail_next[TM];
    uint32_t sw[TN], sx[TM], sw_next[TN], sx_next[TM];
    const uint32_t key = (r >> 1) & 7, line = r * 128, line2 = r * 64, key2 = (r >> 2) & 3, ps = r * 8 + 4 * h;
    auto read_codes = [&](uint32_t buffer, int s, u32x4_t (&w)[TN], u32x4_t (&x)[TM]) {
        const uint32_t at = buffer + line + (((4 * h + s) ^ key) << 4);
#pragma unroll
        for (int n = 0; n < TN; ++n) w[n] = *reinterpret_cast<const u32x4_t *>(lds + at + (wn * TN + n) * 4096);
#pragma unroll
        for (int m = 0; m < TM; ++m) x[m] = *reinterpret_cast<const u32x4_t *>(lds + at + S::W + (wm * TM + m) * 4096);
    };
    auto read_tail = [&](uint32_t buffer, int half, u32x4_t (&t)[TM]) {
        if constexpr (AK == 6) {
            const uint32_t at = buffer + S::W + S::X + line2 + (((2 * h + half) ^ key2) << 4);
#pragma unroll
            for (int m = 0; m < TM; ++m) t[m] = *reinterpret_cast<const u32x4_t *>(lds + at + (wm * TM + m) * 2048);
        }
    };
    auto read_scales = [&](uint32_t buffer) {
        const uint32_t at = buffer + S::W + S::X + S::X2 + ps;
#pragma unroll
        for (int n = 0; n < TN; ++n) sw_next[n] = *reinterpret_cast<const uint32_t *>(lds + at + (wn * TN + n) * 256);
#pragma unroll
        for (int m = 0; m < TM; ++m) sx_next[m] = *reinterpret_cast<const uint32_t *>(lds + at + S::WS + (wm * TM + m) * 256);
    };
    auto take = [&] {
#pragma unroll
        for (int n = 0; n < TN; ++n) sw[n] = sw_next[n];
#pragma unroll
        for (int m = 0; m < TM; ++m) {
            sx[m] = sx_next[m];
            if constexpr (AK == 6) tail[m] = tail_next[m];
        }
    };
    auto multiply = [&](auto SS, const u32x4_t (&w)[TN], const u32x4_t (&x)[TM], const u32x4_t (&t)[TM]) {
        constexpr int s = SS.value;
#pragma unroll
        for (int m = 0; m < TM; ++m)
#pragma unroll
            for (int n = 0; n < TN; ++n)
                acc[m][n] = mx_scale_mfma32<AK, s>(w[n], x[m], s % 2 ? t[m].z : t[m].x, s % 2 ? t[m].w : t[m].y, acc[m][n], sw[n], sx[m]);
    };

#pragma unroll
    for (int i = 0; i < R; ++i) issue(i * S::STAGE, st0 + i);
    wait_vmcnt<(R - 1) * PER>();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    uint32_t cur = 0;
    read_codes(cur, 0, w0, x0);
    read_scales(cur);
    read_tail(cur, 0, tail_next);
    take();
    for (int st = st0; st < st1; ++st) {
        read_codes(cur, 1, w1, x1);
        multiply(std::integral_constant<int, 0>{}, w0, x0, tail);
        read_codes(cur, 2, w0, x0);
        read_tail(cur, 1, tail2);
        multiply(std::integral_constant<int, 1>{}, w1, x1, tail);
        read_codes(cur, 3, w1, x1);
        multiply(std::integral_constant<int, 2>{}, w0, x0, tail2);
        // the next macro has landed, and every wave has read this one
        wait_vmcnt<(R - 2) * PER>();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        issue(cur, st + R);
        cur = cur + S::STAGE == R * S::STAGE ? 0u : cur + S::STAGE;
        read_codes(cur, 0, w0, x0);
        read_scales(cur);
        read_tail(cur, 0, tail_next);
        multiply(std::integral_constant<int, 3>{}, w1, x1, tail2);
        take();
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");  // late copies must not land in reused LDS
    __syncthreads();

    // Results leave through LDS so that the lanes of a store lie side by side in a row: two squares at a time, 32 rows of 64.
    // The stores are nontemporal: results are not read here again, and kept in L2 they push out the operands that other tiles still read
    // (8192 rows of FP4 by 17408 x 5120, bf16 out: 470 -> 445 us; 2048 rows of FP6 by 24576 x 4096, gated, fp16 out: 187 -> 177).
    uint8_t *area = lds + wave * kTileOut;
    const bool partial = a.splits > 1, f32 = partial || a.y_dtype == MFQ_X_F32;
    const int half = part_half(a.nrows);  // of partial results: where the up rows' begin
    uint8_t *y = reinterpret_cast<uint8_t *>(partial ? a.part + static_cast<int64_t>(blockIdx.y) * a.M * (2 * half) : a.y);
    const int64_t ldy = partial ? 2 * half : a.ldy;
    const bool wide = ldy % (f32 ? 4 : 8) == 0 && reinterpret_cast<uintptr_t>(y) % 16 == 0;
    // columns n .. n + 64 of the 32 rows from mt on, from the two squares p and q; none from `end` on
    auto put = [&](const float16_t &p, const float16_t &q, int mt, int n, int end) __attribute__((always_inline)) {
        if (f32) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                *reinterpret_cast<float4_t *>(area + r * kTilePitch + (8 * j + 4 * h) * 4) = float4_t{p[4 * j], p[4 * j + 1], p[4 * j + 2], p[4 * j + 3]};
                *reinterpret_cast<float4_t *>(area + r * kTilePitch + (32 + 8 * j + 4 * h) * 4) = float4_t{q[4 * j], q[4 * j + 1], q[4 * j + 2], q[4 * j + 3]};
            }
            wave_sync();
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int row = k * 4 + (lane >> 4), c = n + (lane & 15) * 4, to_row = row_of[mt + row];
                const float4_t v = *reinterpret_cast<const float4_t *>(area + row * kTilePitch + (lane & 15) * 16);
                if (to_row < 0 || c >= end) continue;
                float *o = reinterpret_cast<float *>(y) + static_cast<int64_t>(to_row) * ldy + c;
                if (wide && c + 4 <= end) {
                    __builtin_nontemporal_store(v, reinterpret_cast<float4_t *>(o));
                } else {
#pragma unroll
                    for (int t = 0; t < 4; ++t)
                        if (c + t < end) o[t] = v[t];
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                *reinterpret_cast<u32x2_t *>(area + r * kTilePitch + (8 * j + 4 * h) * 2) =
                    u32x2_t{mx_pack16(p[4 * j], p[4 * j + 1], a.y_dtype), mx_pack16(p[4 * j + 2], p[4 * j + 3], a.y_dtype)};
                *reinterpret_cast<u32x2_t *>(area + r * kTilePitch + (32 + 8 * j + 4 * h) * 2) =
                    u32x2_t{mx_pack16(q[4 * j], q[4 * j + 1], a.y_dtype), mx_pack16(q[4 * j + 2], q[4 * j + 3], a.y_dtype)};
            }
            wave_sync();
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int row = k * 8 + (lane >> 3), c = n + (lane & 7) * 8, to_row = row_of[mt + row];
                const u32x4_t v = *reinterpret_cast<const u32x4_t *>(area + row * kTilePitch + (lane & 7) * 16);
                if (to_row < 0 || c >= end) continue;
                uint16_t *o = reinterpret_cast<uint16_t *>(y) + static_cast<int64_t>(to_row) * ldy + c;
                if (wide && c + 8 <= end) {
                    __builtin_nontemporal_store(v, reinterpret_cast<u32x4_t *>(o));
                } else {
#pragma unroll
                    for (int t = 0; t < 8; ++t)
                        if (c + t < end) o[t] = static_cast<uint16_t>(v[t >> 1] >> (16 * (t & 1)));
                }
            }
        }
        wave_sync();
    };
    static_for<TM>([&](auto MI) __attribute__((always_inline)) {
        constexpr int m = MI.value;
        const int mt = (wm * TM + m) * 32;
        if (mt >= rows) return;
        static_for<TN / 2>([&](auto BI) __attribute__((always_inline)) {
            constexpr int b = BI.value;
            if (!a.glu) {
                put(acc[m][2 * b], acc[m][2 * b + 1], mt, n0 + (wn * TN + 2 * b) * 32, width);
            } else if constexpr (TN == 2) {  // 32 columns: one square, twice
                const int at = n0 + wn * 32, end = min(at + 32, width);
                if (partial) {
                    put(acc[m][0], acc[m][0], mt, at, end);
                    put(acc[m][1], acc[m][1], mt, half + at, half + end);
                } else {
                    float16_t v;
#pragma unroll
                    for (int i = 0; i < 16; ++i) v[i] = glu_value(acc[m][0][i], acc[m][1][i], a.gelu);
                    put(v, v, mt, at, end);
                }
            } else if constexpr (b < TN / 4) {
                const int at = n0 + (wn * (TN / 2) + 2 * b) * 32;
                if (partial) {
                    put(acc[m][2 * b], acc[m][2 * b + 1], mt, at, width);
                    put(acc[m][TN / 2 + 2 * b], acc[m][TN / 2 + 2 * b + 1], mt, half + at, half + width);
                } else {
                    float16_t u, v;
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        u[i] = glu_value(acc[m][2 * b][i], acc[m][TN / 2 + 2 * b][i], a.gelu);
                        v[i] = glu_value(acc[m][2 * b + 1][i], acc[m][TN / 2 + 2 * b + 1][i], a.gelu);
                    }
                    put(u, v, mt, at, width);
                }
            }
        });
    });
}

// the pieces of a split over K, added in their order
__global__ __launch_bounds__(256) void mxs_join_kernel(MxsArgs a) {
    const int width = a.glu ? a.nrows / 2 : a.nrows, half = part_half(a.nrows);
    const int64_t all = static_cast<int64_t>(a.M) * (2 * half);
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < static_cast<int64_t>(a.M) * width; i += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t m = i / width;
        const int n = static_cast<int>(i - m * width);
        const float *p = a.part + m * (2 * half) + n;
        float v = 0.f, u = 0.f;
        for (int s = 0; s < a.splits; ++s) v += p[s * all];
        if (a.glu) {
            for (int s = 0; s < a.splits; ++s) u += p[s * all + half];
            v = glu_value(v, u, a.gelu);
        }
        store_rounded(a.y, m * a.ldy + n, v, a.y_dtype);
    }
}

// ---- launches -------------------------------------------------------------------------------------------------------------------
// Rows that every block of the flow kernel quantises itself, which saves a launch: up to four, and up to sixteen while they hold no more than
// so many values.  4096 x 4096 at 8 rows 6.5 us in a graph, 8.1 with the quantiser's launch, at 16 rows 7.8 and 8.2, 12288 x 4096 at 16 rows 10.9
// and 11.1; 4096 x 8192 at 16 rows, beyond it, 12.8 and 10.4.  One call after the other from Python: 9.2 and 13.8.
constexpr int kSmallRows = 4, kSmallValues = 1 << 16;
constexpr bool small_rows(int64_t M, int K) { return M <= kSmallRows || (M <= 16 && M * K <= kSmallValues); }

template <int AK, int MT, int NB, int MODE>
int launch_stream_nb(const MxsArgs &a, int tiles, hipStream_t st) {
    using S = StreamShape<AK, MT, NB>;
    const int nmac = mx_macros(a.K);
    int nwaves = nmac < 8 ? nmac : 8;
    while (nwaves > 1 && nwaves * static_cast<size_t>(2) * S::STAGE > kMaxDynamicLds) --nwaves;
    const size_t lds = nwaves * static_cast<size_t>(2) * S::STAGE;
    static_assert(NB * MT * 1024 <= 2 * S::STAGE, "sums in the ring");
    const int width = a.glu ? a.nrows / 2 : a.nrows, per = 16 * (a.glu ? NB / 2 : NB);
    auto kern = mxs_stream_kernel<AK, MT, NB, MODE>;
    if (int rc = allow_dynamic_lds(reinterpret_cast<const void *>(kern), lds, "mx_scaled")) return rc;
    hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(ceil_div(width, per)), static_cast<unsigned>(tiles)), dim3(64 * nwaves), lds, st, a);
    return check_launch("mx_scaled (stream)");
}
template <int AK, int MT, int MODE>
int launch_stream(const MxsArgs &a, int tiles, hipStream_t st) {
    return a.glu ? launch_stream_nb<AK, MT, 2, MODE>(a, tiles, st) : launch_stream_nb<AK, MT, 1, MODE>(a, tiles, st);
}

// Waves of a block of the flow kernel: as many as fit the LDS beside `x` bytes of activations, eight at most; 0: K is too long for it.
int flow_waves(size_t ring, size_t x, size_t *lds) {
    for (int n = 8; n >= 2; --n) {
        *lds = n * ring + x;
        if (*lds <= kMaxDynamicLds) return n;
    }
    return 0;
}
constexpr int kFlowStages = 3;
template <int AK, int MT, int NB>
size_t flow_x_bytes(int K, int small_rows) {
    using S = FlowShape<AK, MT, NB>;
    return static_cast<size_t>(mx_macros(K)) * (small_rows ? S::small_macro(rows_kept(small_rows)) : S::XM);
}
template <int AK, int MT, int NB, int MODE, bool SMALL>
int launch_flow_nb(const MxsArgs &a, int tiles, int busy, hipStream_t st) {
    constexpr int D = kFlowStages;
    using S = FlowShape<AK, MT, NB>;
    size_t lds;
    const int nwaves = flow_waves(static_cast<size_t>(D) * S::STAGE, flow_x_bytes<AK, MT, NB>(a.K, SMALL ? MODE == kPairs ? 1 : MODE == kMapped ? 16 : a.M : 0), &lds);
    if (!nwaves) return MFQ_ERR_UNSUPPORTED;
    const int width = a.glu ? a.nrows / 2 : a.nrows, rbs = static_cast<int>(ceil_div(width, 16));
    // blocks of a tile: two for each compute unit where the LDS has room for two
    const int want = device_cu_count() * (2 * lds <= kMaxDynamicLds ? 2 : 1);
    int chunks = static_cast<int>(ceil_div(want, busy > 0 ? busy : 1));
    if (chunks > rbs) chunks = rbs;
    chunks = static_cast<int>(ceil_div(rbs, ceil_div(rbs, chunks)));  // as many row-blocks in each
    auto kern = mxs_flow_kernel<AK, MT, NB, D, MODE, SMALL>;
    if (int rc = allow_dynamic_lds(reinterpret_cast<const void *>(kern), lds, "mx_scaled")) return rc;
    MFQ_REQUIRE(static_cast<int64_t>(tiles) * chunks < (1ll << 31), MFQ_ERR_UNSUPPORTED, "mx_scaled: %d tiles", tiles);
    hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(tiles * chunks)), dim3(64 * nwaves), lds, st, a, chunks);
    return check_launch("mx_scaled (flow)");
}
// tiles: at most; busy: about as many have rows
template <int AK, int MT, int MODE, bool SMALL = false>
int launch_flow(const MxsArgs &a, int tiles, int busy, hipStream_t st) {
    return a.glu ? launch_flow_nb<AK, MT, 2, MODE, SMALL>(a, tiles, busy, st) : launch_flow_nb<AK, MT, 1, MODE, SMALL>(a, tiles, busy, st);
}

int tile_rows_mapped(int kind) { return kind == 1 ? 64 : 128; }
// tiles of a call with a route map: at most
int64_t tiles_mapped(int64_t pairs, int E, int rows) { return ceil_div(pairs, rows) + (E < pairs ? E : pairs); }

template <int AK, int BN, int BM, int WN, int WM, int R, int MODE>
int launch_tile(const MxsArgs &a, hipStream_t st) {
    using S = TileShape<AK, BN, BM, R>;
    const int width = a.glu ? a.nrows / 2 : a.nrows;
    const int64_t tiles_n = ceil_div(width, a.glu ? BN / 2 : BN);
    const int64_t tiles_m = MODE == kMapped ? tiles_mapped(a.pairs, a.E, BM) : ceil_div(a.M, BM);
    const int64_t blocks = (tiles_n * tiles_m + 7) / 8 * 8;
    MFQ_REQUIRE(blocks < (1ll << 31), MFQ_ERR_UNSUPPORTED, "mx_scaled: %lld tiles", static_cast<long long>(blocks));
    static_assert(WN * WM * kTileOut <= R * S::STAGE && S::LDS <= static_cast<int>(kMaxDynamicLds), "results leave through the ring");
    const size_t lds = S::LDS;
    auto kern = mxs_tile_kernel<AK, BN, BM, WN, WM, R, MODE>;
    if (int rc = allow_dynamic_lds(reinterpret_cast<const void *>(kern), lds, "mx_scaled")) return rc;
    hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(MODE == kLinear ? a.splits : 1)), dim3(WN * WM * 64), lds, st, a);
    return check_launch("mx_scaled (tile)");
}

int launch_join(const MxsArgs &a, hipStream_t st) {
    if (a.splits <= 1) return MFQ_OK;
    const int64_t n = static_cast<int64_t>(a.M) * (a.glu ? a.nrows / 2 : a.nrows);
    const int64_t blocks = ceil_div(n, 256);
    hipLaunchKernelGGL(mxs_join_kernel, dim3(static_cast<unsigned>(blocks < 8192 ? blocks : 8192)), dim3(256), 0, st, a);
    return check_launch("mx_scaled (join)");
}

// Kernel of a call: the flow kernel on rows that its blocks quantise (0), on one or two tiles of 16 rows (1, 2; the stream kernel where K is too long), or a
// tile of the list (3 + its index) with K in `splits` pieces.
struct MxsPlan { int kind, splits; };
constexpr int kPlanTile = 3;
// Tiles and what a launch of them takes, us: f + max(macros * l, rounds * (macros * c + e)), rounds = blocks a compute unit: l is a macro's
// way from memory with the compute unit to itself, c its share with `per_cu` blocks on it, e the end of a block.  Fitted to 12288 x 4096 and
// 4096 x 12288 at 40 to 4096 rows, MXFP4 / MXFP6: 12288 x 4096 at 40 rows 13.2, 11.6, 15.2, 19.3, 28.2 us in the order of the list (MXFP4),
// at 601 rows 31.0, 31.2, 26.6, 25.9, 34.0, at 2048 rows 82.9, 88.6, 71.4, 73.2, 72.8; MXFP6 at 128 rows 13.9 (128 x 64), 24.8, 30.1, at 2048
// 102.8, 82.0, 103.4, at 4096 279, 206, 182.
struct MxsTile { int act, n, m, per_cu; double f, l, c, e; };
constexpr MxsTile kMxsTile[] = {
    {4, 128, 64, 3, 5.5, 0.48, 0.36, 0.5}, {4, 64, 128, 2, 6.0, 0.36, 0.40, 0.5}, {4, 128, 128, 2, 6.2, 0.56, 0.62, 1.0},
    {4, 256, 128, 1, 7.3, 0.75, 1.12, 2.6}, {4, 256, 256, 1, 9.6, 1.16, 1.9, 5.0},
    {6, 128, 64, 1, 5.3, 0.47, 0.65, 0.5}, {6, 256, 128, 1, 7.2, 0.95, 1.35, 3.0}, {6, 256, 192, 1, 8.0, 1.23, 1.95, 4.0}};
constexpr int kMxsTiles = sizeof(kMxsTile) / sizeof(kMxsTile[0]), kMaxSplits = 16;

double tile_us(const MxsTile &t, int nrows, int nmac, int M, int splits, int cus) {
    const double blocks = static_cast<double>(ceil_div(nrows, t.n)) * ceil_div(M, t.m) * splits, q = blocks / cus;
    const double whole = static_cast<double>(static_cast<int64_t>(q) + (q > static_cast<int64_t>(q) ? 1 : 0));
    const double rounds = t.per_cu == 1 ? whole : (q + whole) / 2;
    const double macs = static_cast<double>(ceil_div(nmac, splits));
    double us = macs * t.l > rounds * (macs * t.c + t.e) ? macs * t.l : rounds * (macs * t.c + t.e);
    // the pieces are written, read by a second launch and written as the result
    if (splits > 1) us += 3.0 + static_cast<double>(M) * nrows * 4 * (2 * splits + 1) / 4.5e6;
    return t.f + us;
}

// whether the flow kernel holds M rows of K columns that it quantises, gate and up side by side
bool small_fits(int act, int K, int M) {
    size_t lds;
    return act == 4 ? flow_waves(kFlowStages * FlowShape<4, 1, 2>::STAGE, flow_x_bytes<4, 1, 2>(K, M), &lds) > 0
                    : flow_waves(kFlowStages * FlowShape<6, 1, 2>::STAGE, flow_x_bytes<6, 1, 2>(K, M), &lds) > 0;
}

// whether it holds MT tiles of 16 quantised rows; else the stream kernel serves them
template <int AK, int MT>
bool flow_fits(int K, bool glu) {
    size_t lds;
    return (glu ? flow_waves(kFlowStages * FlowShape<AK, MT, 2>::STAGE, flow_x_bytes<AK, MT, 2>(K, 0), &lds)
                : flow_waves(kFlowStages * FlowShape<AK, MT, 1>::STAGE, flow_x_bytes<AK, MT, 1>(K, 0), &lds)) > 0;
}
bool flow_fits(int act, int tiles, int K, bool glu) {
    if (act == 4) return tiles == 1 ? flow_fits<4, 1>(K, glu) : flow_fits<4, 2>(K, glu);
    return tiles == 1 ? flow_fits<6, 1>(K, glu) : flow_fits<6, 2>(K, glu);
}

MxsPlan plan_linear(int act, int nrows, int K, int M) {
    const int nmac = mx_macros(K);
    if (small_rows(M, K) && small_fits(act, K, M)) return {0, 1};
    if (M <= 16) return {1, 1};
    if (M <= 32) return {2, 1};
    static const int forced = tune_env("MFQ_MXS_TILE", 0), forced_split = tune_env("MFQ_MXS_SPLIT", 0);
    // what the knobs ask for where the call can have it: a tile of its kind, pieces of which none is empty
    const bool tile = forced > 0 && forced <= kMxsTiles && kMxsTile[forced - 1].act == act;
    const auto whole = [&](int s) { return s <= nmac && (s - 1) * ceil_div(nmac, s) < nmac; };
    const bool pieces = forced_split > 0 && forced_split <= kMaxSplits && whole(forced_split);
    const int cus = device_cu_count();
    MxsPlan best = {-1, 1};
    double least = 0.0;
    for (int t = 0; t < kMxsTiles; ++t) {
        if (kMxsTile[t].act != act || (tile && forced != t + 1)) continue;
        for (int s = 1; s <= kMaxSplits && s <= nmac; ++s) {
            if (!whole(s) || (pieces && s != forced_split)) continue;
            const double us = tile_us(kMxsTile[t], nrows, nmac, M, s, cus);
            if (best.kind < 0 || us < least) {
                best = {kPlanTile + t, s};
                least = us;
            }
        }
    }
    return best;
}

size_t quantized_bytes(int act, int K, int64_t M) {
    const auto up = [](int64_t n) { return (n + 255) & ~static_cast<int64_t>(255); };
    return static_cast<size_t>(up(M * mx_row_bytes(act, K)) + up(mx_scale_bytes(M, K)));
}

template <int AK>
int run_linear(const MxsArgs &a, const MxsPlan &p, hipStream_t st) {
    switch (p.kind) {
        case 0:
            return launch_flow<AK, 1, kLinear, true>(a, 1, 1, st);
        case 1:
            if (int rc = launch_flow<AK, 1, kLinear>(a, 1, 1, st); rc != MFQ_ERR_UNSUPPORTED) return rc;
            return launch_stream<AK, 1, kLinear>(a, 1, st);
        case 2:
            if (int rc = launch_flow<AK, 2, kLinear>(a, 1, 1, st); rc != MFQ_ERR_UNSUPPORTED) return rc;
            return launch_stream<AK, 2, kLinear>(a, 1, st);
        default: break;
    }
    if constexpr (AK == 4) {
        switch (p.kind - kPlanTile) {
            case 0: return launch_tile<4, 128, 64, 2, 2, 2, kLinear>(a, st);
            case 1: return launch_tile<4, 64, 128, 1, 4, 3, kLinear>(a, st);
            case 2: return launch_tile<4, 128, 128, 2, 2, 2, kLinear>(a, st);
            case 3: return launch_tile<4, 256, 128, 4, 2, 3, kLinear>(a, st);
            default: return launch_tile<4, 256, 256, 2, 4, 2, kLinear>(a, st);
        }
    } else {
        switch (p.kind - kPlanTile) {
            case 5: return launch_tile<6, 128, 64, 2, 2, 3, kLinear>(a, st);
            case 6: return launch_tile<6, 256, 128, 4, 2, 2, kLinear>(a, st);
            default: return launch_tile<6, 256, 192, 4, 2, 2, kLinear>(a, st);
        }
    }
}

// Kernel of a call with a route map, from the pairs an expert has on average: 0 waves that stream row-blocks against 16 rows (flow kernel), 1
// and 2 tiles of 128 x 64 and 256 x 128.  128 experts of 2048 x 2048, gated, MXFP4, 8 routes: at 256 tokens (16 pairs an expert) 81, 64
// and 75 us, at 2048 tokens 314, 126 and 140; 32 experts of 2880 x 1440, MXFP6, 4 routes: at 1501 tokens (188 pairs) 146, 80 and 65 us.
int plan_mapped(int64_t pairs, int E) {
    static const int forced = tune_env("MFQ_MXS_EXPERTS", 0);
    if (forced > 0 && forced <= 3) return forced - 1;
    const int64_t mean = ceil_div(pairs, E);
    return mean <= 10 ? 0 : mean < 160 ? 1 : 2;
}

// whether the blocks of a call with a route map quantise their rows themselves
bool mapped_small(int act, int K, int64_t pairs, int E) { return plan_mapped(pairs, E) == 0 && small_rows(16, K) && small_fits(act, K, 16); }

template <int AK>
int run_experts(const MxsArgs &a, hipStream_t st) {
    if (!a.ids_dst) {
        if (int rc = launch_flow<AK, 1, kPairs, true>(a, a.pairs, a.pairs, st); rc != MFQ_ERR_UNSUPPORTED) return rc;
        return fail(MFQ_ERR_UNSUPPORTED, "mx_moe_matmul: %d columns without a route map", a.K);
    }
    const auto most = [&](int rows) { return static_cast<int>(tiles_mapped(a.pairs, a.E, rows)); };
    switch (plan_mapped(a.pairs, a.E)) {
        case 0:
            if (a.xraw) return launch_flow<AK, 1, kMapped, true>(a, most(16), a.E < a.pairs ? a.E : a.pairs, st);
            if (int rc = launch_flow<AK, 1, kMapped>(a, most(16), a.E < a.pairs ? a.E : a.pairs, st); rc != MFQ_ERR_UNSUPPORTED) return rc;
            return launch_stream<AK, 1, kMapped>(a, most(16), st);
        case 1: return launch_tile<AK, 128, 64, 2, 2, 2, kMapped>(a, st);
        default: return launch_tile<AK, 256, 128, 4, 2, AK == 4 ? 3 : 2, kMapped>(a, st);
    }
}

constexpr int kMaxCols = 1 << 24;  // with which the 256 quantised rows of a tile lie within 32 bits

// Checks shared by both entry points; fills what they have in common.
int check_common(MxsArgs &a, const char *who, const void *values, const void *scales, int64_t rows, int cols, int act, const void *x, int x_dtype, int64_t ldx,
                 const void *x_scales, int64_t x_rows, int glu, int activation, const void *y, int y_dtype, int64_t ldy) {
    MFQ_REQUIRE(values && scales && x && y, MFQ_ERR_INVALID, "%s: null argument", who);
    MFQ_REQUIRE(act == 4 || act == 6, MFQ_ERR_INVALID, "%s: activations of kind %d (4 = MXFP4, 6 = MXFP6)", who, act);
    MFQ_REQUIRE(x_scales || (x_dtype >= MFQ_X_BF16 && x_dtype <= MFQ_X_F32), MFQ_ERR_INVALID, "%s: x_dtype=%d", who, x_dtype);
    MFQ_REQUIRE(y_dtype >= MFQ_X_BF16 && y_dtype <= MFQ_X_F32, MFQ_ERR_INVALID, "%s: y_dtype=%d", who, y_dtype);
    MFQ_REQUIRE(rows > 0 && cols > 0 && cols % 32 == 0, MFQ_ERR_INVALID, "%s: [%lld, %d], columns must be divisible by 32", who, static_cast<long long>(rows), cols);
    MFQ_REQUIRE(reinterpret_cast<uintptr_t>(values) % 16 == 0 && reinterpret_cast<uintptr_t>(scales) % 8 == 0, MFQ_ERR_INVALID,
                "%s: values must be 16-byte aligned, scales 8-byte aligned", who);
    if (x_scales) {
        MFQ_REQUIRE(reinterpret_cast<uintptr_t>(x) % 16 == 0 && reinterpret_cast<uintptr_t>(x_scales) % 8 == 0, MFQ_ERR_INVALID,
                    "%s: quantised activations must be 16-byte aligned, their scales 8-byte aligned", who);
    } else {
        MFQ_REQUIRE(x_rows == 1 || ldx >= cols, MFQ_ERR_INVALID, "%s: ldx=%lld < %d", who, static_cast<long long>(ldx), cols);
        MFQ_REQUIRE(reinterpret_cast<uintptr_t>(x) % (x_dtype == MFQ_X_F32 ? 4 : 2) == 0, MFQ_ERR_INVALID, "%s: unaligned x", who);
    }
    MFQ_REQUIRE(!glu || (y_dtype != MFQ_X_F32 && (activation == MFQ_GLU_SILU || activation == MFQ_GLU_GELU)), MFQ_ERR_INVALID,
                "%s: a gated product takes a 16-bit type and activation 0 or 1, not y_dtype=%d activation=%d", who, y_dtype, activation);
    MFQ_REQUIRE(reinterpret_cast<uintptr_t>(y) % (y_dtype == MFQ_X_F32 ? 4 : 2) == 0, MFQ_ERR_INVALID, "%s: unaligned y", who);
    MFQ_REQUIRE(cols <= kMaxCols, MFQ_ERR_UNSUPPORTED, "%s: %d columns", who, cols);
    MFQ_REQUIRE(mx_scale_bytes(rows, cols) < (1ll << 32) - 512 && mx_scale_bytes(x_rows, cols) < (1ll << 32) - 512, MFQ_ERR_UNSUPPORTED,
                "%s: %lld rows of weights, %lld of activations, %d columns", who, static_cast<long long>(rows), static_cast<long long>(x_rows), cols);
    a.wv = static_cast<const uint8_t *>(values);
    a.ws = static_cast<const uint8_t *>(scales);
    a.y = const_cast<void *>(y);
    a.ldy = ldy;
    a.K = cols;
    a.y_dtype = y_dtype;
    a.glu = glu != 0;
    a.gelu = activation == MFQ_GLU_GELU;
    a.splits = 1;
    return MFQ_OK;
}

// whether a block may read the activations themselves: 16-byte pieces
bool pieces(const void *x, int x_dtype, int64_t ldx, int64_t rows) {
    return reinterpret_cast<uintptr_t>(x) % 16 == 0 && (rows == 1 || ldx % (x_dtype == MFQ_X_F32 ? 4 : 8) == 0);
}

}  // namespace
}  // namespace mfq

using namespace mfq;

extern "C" size_t mfq_hip_mx_scaled_gemm_workspace_bytes(int act, int nrows, int cols, int M, int x_quantized) {
    if ((act != 4 && act != 6) || nrows <= 0 || cols <= 0 || cols % 32 != 0 || M <= 0) return 0;
    const MxsPlan p = plan_linear(act, nrows, cols, M);
    size_t n = x_quantized || p.kind == 0 ? 0 : quantized_bytes(act, cols, M);
    if (p.splits > 1) n += static_cast<size_t>(p.splits) * part_bytes(M, nrows);
    return n;
}

extern "C" int mfq_hip_mx_scaled_plan(int act, int nrows, int cols, int M, int glu, int *splits) {
    if ((act != 4 && act != 6) || nrows <= 0 || cols <= 0 || cols % 32 != 0 || cols > kMaxCols || M <= 0) return -1;
    const MxsPlan p = plan_linear(act, nrows, cols, M);
    if (splits) *splits = p.splits;
    if (p.kind >= kPlanTile) return 5 + p.kind - kPlanTile;
    return p.kind > 0 && !flow_fits(act, p.kind, cols, glu != 0) ? 2 + p.kind : p.kind;
}

extern "C" int mfq_hip_mx_scaled_gemm_rows(const void *values, const void *scales, int rows, int cols, int row0, int nrows, int act, const void *x,
                                           int x_dtype, int64_t ldx, const void *x_scales, int M, int glu, int activation, void *y, int y_dtype,
                                           int64_t ldy, void *workspace, size_t workspace_bytes, mfq_stream_t stream) {
    MxsArgs a = {};
    if (int rc = check_common(a, "mx_scaled_gemm_rows", values, scales, rows, cols, act, x, x_dtype, ldx, x_scales, M, glu, activation, y, y_dtype, ldy)) return rc;
    MFQ_REQUIRE(M > 0, MFQ_ERR_INVALID, "mx_scaled_gemm_rows: M=%d", M);
    MFQ_REQUIRE(row0 >= 0 && nrows > 0 && static_cast<int64_t>(row0) + nrows <= rows, MFQ_ERR_INVALID, "mx_scaled_gemm_rows: rows %d + %d of %d", row0, nrows, rows);
    MFQ_REQUIRE(!glu || nrows % 2 == 0, MFQ_ERR_INVALID, "mx_scaled_gemm_rows: gate and up in %d rows", nrows);
    MFQ_REQUIRE(M == 1 || ldy >= (glu ? nrows / 2 : nrows), MFQ_ERR_INVALID, "mx_scaled_gemm_rows: ldy=%lld < %d", static_cast<long long>(ldy), glu ? nrows / 2 : nrows);
    MFQ_REQUIRE(static_cast<int64_t>(nrows) * (cols / 2) < (1ll << 31), MFQ_ERR_UNSUPPORTED, "mx_scaled_gemm_rows: %d x %d weights", nrows, cols);
    const hipStream_t st = as_stream(stream);
    a.wv += static_cast<int64_t>(row0) * (cols / 2);
    a.row0 = row0;
    a.nrows = nrows;
    a.M = M;
    a.R = 1;
    MxsPlan p = plan_linear(act, nrows, cols, M);
    uint8_t *ws = static_cast<uint8_t *>(workspace);
    size_t used = 0;
    if (x_scales) {
        a.xv = static_cast<const uint8_t *>(x);
        a.xs = static_cast<const uint8_t *>(x_scales);
    } else if (p.kind == 0) {
        a.xraw = x;
        a.x_wide = pieces(x, x_dtype, ldx, M);
        a.x_dtype = x_dtype;
        a.ldx = ldx;
    } else {
        used = quantized_bytes(act, cols, M);
        MFQ_REQUIRE(ws && workspace_bytes >= used, MFQ_ERR_WORKSPACE, "mx_scaled_gemm_rows: workspace %zu < %zu", workspace_bytes, used);
        MFQ_REQUIRE(reinterpret_cast<uintptr_t>(ws) % 16 == 0, MFQ_ERR_WORKSPACE, "mx_scaled_gemm_rows: unaligned workspace");
        uint8_t *xs = ws + ((static_cast<int64_t>(M) * mx_row_bytes(act, cols) + 255) & ~static_cast<int64_t>(255));
        if (int rc = mx_quantize_launch(act, x, x_dtype, ldx, M, cols, ws, xs, st)) return rc;
        a.xv = ws;
        a.xs = xs;
    }
    if (p.splits > 1) {
        // a short workspace: K in as many pieces as it has room for
        const size_t left = workspace_bytes > used && ws ? workspace_bytes - used : 0, each = part_bytes(M, nrows);
        const int nmac = mx_macros(cols);
        if (left / each < static_cast<size_t>(p.splits)) p.splits = static_cast<int>(left / each);
        while (p.splits > 1 && (p.splits - 1) * ceil_div(nmac, p.splits) >= nmac) --p.splits;
        if (p.splits < 2 || reinterpret_cast<uintptr_t>(ws) % 16 != 0) p.splits = 1;
        a.splits = p.splits;
        a.part = reinterpret_cast<float *>(ws + used);
    }
    if (int rc = act == 4 ? run_linear<4>(a, p, st) : run_linear<6>(a, p, st)) return rc;
    return launch_join(a, st);
}

namespace {
size_t table_bytes(int64_t pairs, int E) {
    const int kind = plan_mapped(pairs, E);
    return kind < 1 ? 0 : static_cast<size_t>(tiles_mapped(pairs, E, tile_rows_mapped(kind)) + 1) * 16;
}
}  // namespace

extern "C" size_t mfq_hip_mx_moe_workspace_bytes(int act, int cols, int x_rows, int n_pairs, int E, int mapped, int x_quantized) {
    if ((act != 4 && act != 6) || cols <= 0 || cols % 32 != 0 || x_rows <= 0 || n_pairs <= 0 || E <= 0 || !mapped) return 0;
    return (x_quantized || mapped_small(act, cols, n_pairs, E) ? 0 : quantized_bytes(act, cols, x_rows)) + table_bytes(n_pairs, E);
}

extern "C" int mfq_hip_mx_moe_plan(int act, int cols, int n_pairs, int E, int mapped, int glu, int x_quantized) {
    if ((act != 4 && act != 6) || cols <= 0 || cols % 32 != 0 || cols > kMaxCols || n_pairs <= 0 || E <= 0) return -1;
    if (!mapped) return 0;
    const int kind = plan_mapped(n_pairs, E);
    if (kind > 0) return 5 + (act == 4 ? kind == 1 ? 0 : 3 : kind == 1 ? 5 : 6);
    if (!x_quantized && mapped_small(act, cols, n_pairs, E)) return 0;
    return flow_fits(act, 1, cols, glu != 0) ? 1 : 3;
}

extern "C" int mfq_hip_mx_moe_matmul(const void *values, const void *scales, int rows, int cols, int out_per_expert, const int32_t *expert_slot, int E, int act,
                                     const void *x, int x_dtype, int64_t ldx, const void *x_scales, int routed_input, const int32_t *ids, int T, int R,
                                     const int32_t *ids_dst, const int32_t *expert_bounds, int glu, int activation, void *y, int y_dtype, int64_t ldy,
                                     void *workspace, size_t workspace_bytes, mfq_stream_t stream) {
    MxsArgs a = {};
    MFQ_REQUIRE(T > 0 && R > 0 && E > 0 && static_cast<int64_t>(T) * R < (1ll << 31), MFQ_ERR_INVALID, "mx_moe_matmul: %d tokens, %d routes, %d experts", T, R, E);
    const int x_rows = routed_input ? T * R : T;
    if (int rc = check_common(a, "mx_moe_matmul", values, scales, rows, cols, act, x, x_dtype, ldx, x_scales, x_rows, glu, activation, y, y_dtype, ldy)) return rc;
    MFQ_REQUIRE(ids && !ids_dst == !expert_bounds, MFQ_ERR_INVALID, "mx_moe_matmul: ids, and both ids_dst and expert_bounds or neither");
    MFQ_REQUIRE(out_per_expert > 0 && rows % out_per_expert == 0 && (expert_slot || rows / out_per_expert >= E), MFQ_ERR_INVALID,
                "mx_moe_matmul: %d rows are not %d experts of %d", rows, E, out_per_expert);
    MFQ_REQUIRE(!glu || out_per_expert % 2 == 0, MFQ_ERR_INVALID, "mx_moe_matmul: gate and up in %d rows", out_per_expert);
    MFQ_REQUIRE(T * R == 1 || ldy >= (glu ? out_per_expert / 2 : out_per_expert), MFQ_ERR_INVALID, "mx_moe_matmul: ldy=%lld", static_cast<long long>(ldy));
    MFQ_REQUIRE(static_cast<int64_t>(out_per_expert) * (cols / 2) < (1ll << 31) && x_rows * mx_row_bytes(act, cols) < (1ll << 31),
                MFQ_ERR_UNSUPPORTED, "mx_moe_matmul: an expert of %d x %d, %d rows of activations", out_per_expert, cols, x_rows);
    if (!ids_dst) {
        MFQ_REQUIRE(T * R <= 65535, MFQ_ERR_UNSUPPORTED, "mx_moe_matmul: %d pairs without a route map", T * R);
    } else {
        MFQ_REQUIRE(ceil_div(T * R, 16) + E <= 65535 || plan_mapped(static_cast<int64_t>(T) * R, E) > 0, MFQ_ERR_UNSUPPORTED, "mx_moe_matmul: %d experts, %d pairs", E, T * R);
    }
    const hipStream_t st = as_stream(stream);
    a.nrows = out_per_expert;
    a.M = x_rows;
    a.E = E;
    a.R = R;
    a.pairs = T * R;
    a.routed = routed_input != 0;
    a.ids = ids;
    a.ids_dst = ids_dst;
    a.bounds = expert_bounds;
    a.slot = expert_slot;
    if (x_scales) {
        a.xv = static_cast<const uint8_t *>(x);
        a.xs = static_cast<const uint8_t *>(x_scales);
    } else if (!ids_dst || mapped_small(act, cols, a.pairs, E)) {
        a.xraw = x;
        a.x_wide = pieces(x, x_dtype, ldx, x_rows);
        a.x_dtype = x_dtype;
        a.ldx = ldx;
    }
    if (ids_dst) {
        const bool quantise = !x_scales && !a.xraw;
        const size_t rows_bytes = quantise ? quantized_bytes(act, cols, x_rows) : 0, tab = table_bytes(a.pairs, E), need = rows_bytes + tab;
        MFQ_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), MFQ_ERR_WORKSPACE, "mx_moe_matmul: workspace %zu < %zu", workspace_bytes, need);
        MFQ_REQUIRE(need == 0 || reinterpret_cast<uintptr_t>(workspace) % 16 == 0, MFQ_ERR_WORKSPACE, "mx_moe_matmul: unaligned workspace");
        uint8_t *ws = static_cast<uint8_t *>(workspace);
        const MxTileTable table = {expert_bounds, expert_slot, E, tile_rows_mapped(plan_mapped(a.pairs, E)), tab ? reinterpret_cast<i32x4v_t *>(ws + rows_bytes) : nullptr};
        a.table = table.out;
        uint8_t *xs = ws;
        if (quantise) {
            xs = ws + ((static_cast<int64_t>(x_rows) * mx_row_bytes(act, cols) + 255) & ~static_cast<int64_t>(255));
            a.xv = ws;
            a.xs = xs;
        }
        if (quantise || tab)
            if (int rc = mx_quantize_launch(act, x, x_scales ? MFQ_X_BF16 : x_dtype, ldx, quantise ? x_rows : 0, cols, ws, xs, st, &table)) return rc;
    }
    return act == 4 ? run_experts<4>(a, st) : run_experts<6>(a, st);
}
