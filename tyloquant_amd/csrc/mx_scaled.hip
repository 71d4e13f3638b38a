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
// the expert that tile t belongs to, the number of its first tile and how many it has; t is below the total
__device__ __forceinline__ void mxs_find_tile(const MxsArgs &a, int rows, int lane, int t, int &expert, int &first, int &count) {
    int before = 0;
    expert = 0; first = 0; count = 0;
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
            count = __builtin_amdgcn_readlane(n, l);
            first = before + __builtin_amdgcn_readlane(upto, l) - count;
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

// ---- few rows: the weights are streamed ----------------------------------------------------------------------------------------
// A block owns NB row-blocks of 16 neurons and up to 16 * MT rows of activations; its waves take the macros of K in turn, each
// through a ring of D stages of its own in LDS (no barrier in the loop), and their sums meet in LDS.  RES: the activations of the
// block lie in LDS, quantised by the block itself where they come as bf16 or fp16; else they go through the ring with the weights.
template <int AK, int MT, int NB, int D, bool RES>
struct StreamShape {
    static constexpr int W = NB * 2048, WS = 256, X = RES ? 0 : MT * 16 * mx_macro_bytes(AK), XS = RES ? 0 : 256;
    static constexpr int STAGE = W + WS + X + XS;
    static constexpr int REQ = 2 * NB + 1 + (RES ? 0 : MT * (AK == 4 ? 2 : 3) + 1);  // requests of a stage
};

template <int AK, int MT, int NB, int D, bool RES, int MODE>
__global__ __launch_bounds__(512) void mxs_stream_kernel(MxsArgs a) {
    using S = StreamShape<AK, MT, NB, D, RES>;
    static_assert(NB <= 2 && MT <= 2 && (D == 2 || D == 3), "a stage's scales are one request of four bytes a lane");
    extern __shared__ __attribute__((aligned(128))) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, nwaves = blockDim.x >> 6;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15, g = lane >> 4;
    const int nblk = a.K / 32, nmac = (nblk + 7) / 8;
    constexpr int XMAC = mx_macro_bytes(AK);
    const int64_t wrow = a.K / 2, xrow = static_cast<int64_t>(nmac) * XMAC;
    const int width = a.glu ? a.nrows / 2 : a.nrows;  // results of a row

    int expert = 0, m0 = 0, rows = a.M, first = 0;
    if constexpr (MODE == kPairs) {
        expert = a.ids[blockIdx.y];
        if (expert < 0 || expert >= a.E) {
            if (blockIdx.x == 0) mxs_zero_rows(a, blockIdx.y, a.pairs, tid, blockDim.x);
            return;
        }
        rows = 1;
    } else if constexpr (MODE == kMapped) {
        if (blockIdx.x == 0) mxs_zero_rows(a, blockIdx.y, gridDim.y, tid, blockDim.x);
        if (static_cast<int>(blockIdx.y) >= mxs_total_tiles(a, 16 * MT, lane)) return;
        int t0, count;
        mxs_find_tile(a, 16 * MT, lane, blockIdx.y, expert, t0, count);
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
    auto pair_of = [&](int m) { return MODE == kPairs ? static_cast<int>(blockIdx.y) : MODE == kMapped ? a.ids_dst[first + m] : m0 + m; };
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
    const uint8_t *sbase = a.ws + static_cast<int64_t>(expert) * a.nrows * a.sstride;
    const __amdgpu_buffer_rsrc_t win = wave_window(wbase, static_cast<uint32_t>(a.nrows * wrow));
    const __amdgpu_buffer_rsrc_t swin = wave_window(sbase, static_cast<uint32_t>(a.nrows) * a.sstride);
    uint32_t wv[2 * NB];
    const int piece = lane & 7;
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i) {
        const int row = 8 * (i & 1) + (lane >> 3);
        wv[i] = static_cast<uint32_t>(neuron(i >> 1, row) * wrow) + 16u * (piece ^ mx_key(row));
    }
    const uint32_t wsv = static_cast<uint32_t>(neuron(NB == 2 ? lane >> 5 : 0, (lane >> 1) & 15)) * a.sstride + 4u * (lane & 1);
    // rows of a mapped tile lie anywhere: the window is all of them (under 4 GB, the host sees to it); else the block's own
    const int64_t base = MODE == kLinear ? m0 : 0;
    const int span = RES ? 0 : MODE == kLinear ? rows : a.M;
    const __amdgpu_buffer_rsrc_t xwin = wave_window(a.xv + base * xrow, static_cast<uint32_t>(span * xrow));
    const __amdgpu_buffer_rsrc_t xswin = wave_window(a.xs + base * a.sstride, static_cast<uint32_t>(span) * a.sstride);
    uint32_t xv[MT * 2], xv2[MT], xsv = 0;
    if constexpr (!RES) {
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
        xsv = static_cast<uint32_t>(src_of(min(MT == 2 ? lane >> 1 : (lane >> 1) & 15, rows - 1)) - base) * a.sstride + 4u * (lane & 1);
    }

    uint8_t *ring = lds + wave * (D * S::STAGE);
    uint8_t *xres = lds + nwaves * (D * S::STAGE);  // RES: rows of whole macros, then their scales
    const int xres_row = nmac * XMAC;
    uint8_t *xres_s = xres + rows * xres_row;

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
        if (NB == 2 || lane < 32) copy4(swin, to + S::W, wsv, mac * 8);
        if constexpr (!RES) {
            uint8_t *xto = to + S::W + S::WS;
#pragma unroll
            for (int i = 0; i < 2 * MT; ++i) copy16<0>(xwin, xto + i * 1024, xv[i], xat);
            if constexpr (AK == 6) {
#pragma unroll
                for (int t = 0; t < MT; ++t) copy16<0>(xwin, xto + (2 * MT + t) * 1024, xv2[t], xat);
            }
            if (MT == 2 || lane < 32) copy4(xswin, xto + S::X, xsv, mac * 8);
        }
    };

    const int mine = (nmac - wave + nwaves - 1) / nwaves;  // macros wave, wave + nwaves, ...
#pragma unroll
    for (int i = 0; i < D; ++i)
        if (i < mine) issue(i, wave + i * nwaves);

    if constexpr (RES) {
        // the block's rows: quantised here, zeros up to whole macros, or copied
        if (a.xraw) {
            const int per_row = nmac * 32;
            for (int u = tid; u < rows * per_row; u += blockDim.x) {
                const int m = u / per_row, p = u - m * per_row;
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = 0.f;
                if (p < a.K / 8) {
                    const int64_t from = src_of(m) * a.ldx + 8 * p;
                    if (a.x_dtype == MFQ_X_F32) a.x_wide ? mx_load8<MFQ_X_F32, true>(a.xraw, from, v) : mx_load8<MFQ_X_F32, false>(a.xraw, from, v);
                    else if (a.x_dtype == MFQ_X_F16) a.x_wide ? mx_load8<MFQ_X_F16, true>(a.xraw, from, v) : mx_load8<MFQ_X_F16, false>(a.xraw, from, v);
                    else a.x_wide ? mx_load8<MFQ_X_BF16, true>(a.xraw, from, v) : mx_load8<MFQ_X_BF16, false>(a.xraw, from, v);
                }
                const uint32_t byte = mx_scale_byte(v);
                const MxStore o = mx_place<AK>(mx_codes<AK>(v, byte), p);
                if constexpr (AK == 4) *reinterpret_cast<uint32_t *>(xres + m * xres_row + o.at) = o.q.x;
                else if (o.any) *reinterpret_cast<u32x2_t *>(xres + m * xres_row + o.at) = o.q;
                if ((p & 3) == 0) xres_s[m * (nmac * 8) + (p >> 2)] = static_cast<uint8_t>(byte);
            }
        } else {
            const int per_row = xres_row / 16;
            for (int u = tid; u < rows * per_row; u += blockDim.x) {
                const int m = u / per_row, p = u - m * per_row;
                reinterpret_cast<u32x4_t *>(xres + m * xres_row)[p] = reinterpret_cast<const u32x4_t *>(a.xv + src_of(m) * xrow)[p];
            }
            for (int u = tid; u < rows * nmac; u += blockDim.x) {
                const int m = u / nmac, p = u - m * nmac;
                reinterpret_cast<u32x2_t *>(xres_s)[u] = reinterpret_cast<const u32x2_t *>(a.xs + static_cast<int64_t>(src_of(m)) * a.sstride)[p];
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    }

    float4_t acc[NB][MT];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[b][t] = float4_t{0.f, 0.f, 0.f, 0.f};
    const int key = mx_key(r);
    int stage = 0;
    for (int i = 0; i < mine; ++i) {
        const int mac = wave + i * nwaves;
        // younger stages in flight: those of the next D - 1 macros
        const int left = mine - 1 - i;
        if (D == 3 && left >= 2) wait_vmcnt<(D - 1) * S::REQ>();
        else if (left >= 1) wait_vmcnt<S::REQ>();
        else wait_vmcnt<0>();
        const uint8_t *at = ring + stage * S::STAGE;
        u32x4_t w[2][NB];
        MxFrag x[2][MT];
        uint32_t sw[NB], sx[MT];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            sw[b] = *reinterpret_cast<const uint16_t *>(at + S::W + b * 128 + r * 8 + 2 * g);
#pragma unroll
            for (int s = 0; s < 2; ++s) w[s][b] = *reinterpret_cast<const u32x4_t *>(at + b * 2048 + r * 128 + (((2 * g + s) ^ key) << 4));
        }
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            // RES: rows one after the other, read as they lie; else as the copies have left them
            const int m = min(t * 16 + r, rows - 1);
            const uint8_t *row = RES ? xres + m * xres_row + mac * XMAC : at + S::W + S::WS + t * 2048 + r * 128;
            sx[t] = *reinterpret_cast<const uint16_t *>((RES ? xres_s + m * (nmac * 8) + mac * 8 : at + S::W + S::WS + S::X + t * 128 + r * 8) + 2 * g);
#pragma unroll
            for (int s = 0; s < 2; ++s) x[s][t].x = *reinterpret_cast<const u32x4_t *>(row + ((RES ? 2 * g + s : (2 * g + s) ^ key) << 4));
            if constexpr (AK == 6) {
                const u32x4_t tail = *reinterpret_cast<const u32x4_t *>(RES ? row + 128 + g * 16 : at + S::W + S::WS + (2 * MT + t) * 1024 + row_order_lane(lane));
                x[0][t].y = u32x2_t{tail.x, tail.y};
                x[1][t].y = u32x2_t{tail.z, tail.w};
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the stage is free for the next copies
        if (i + D < mine) issue(stage, wave + (i + D) * nwaves);
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                acc[b][t] = mx_scale_mfma<AK, 0>(w[0][b], x[0][t], acc[b][t], sw[b], sx[t]);
                acc[b][t] = mx_scale_mfma<AK, 1>(w[1][b], x[1][t], acc[b][t], sw[b], sx[t]);
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

// ---- many rows: tiles -----------------------------------------------------------------------------------------------------------
// A block of WN * WM waves owns BN neurons x BM rows, a wave BN / WN x BM / WM of them.  The block copies a macro of both operands
// into one of two stages while it multiplies the other.
template <int AK, int BN, int BM>
struct TileShape {
    static constexpr int W = BN * 128, X = BM * mx_macro_bytes(AK), WS = BN * 8, XS = BM * 8;
    static constexpr int STAGE = W + X + WS + XS;
};

template <int AK, int BN, int BM, int WN, int WM, int MODE>
__global__ __launch_bounds__(WN *WM * 64) void mxs_tile_kernel(MxsArgs a) {
    using S = TileShape<AK, BN, BM>;
    constexpr int NW = WN * WM, TN = BN / 16 / WN, TM = BM / 16 / WM;
    constexpr int PW = (BN / 8 + NW - 1) / NW, PX = (BM / 8 + NW - 1) / NW;  // requests of a wave: rows of weights, of activations
    constexpr int QW = (BN / 32 + NW - 1) / NW, QX = (BM / 32 + NW - 1) / NW, PT = (BM / 16 + NW - 1) / NW;  // of scales, of FP6's second parts
    static_assert(TN % 2 == 0 && BN % 32 == 0 && BM % 32 == 0, "gate and up in one wave; whole requests");
    extern __shared__ __attribute__((aligned(128))) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wn = wave % WN, wm = wave / WN;
    const int r = lane & 15, g = lane >> 4, key = mx_key(r);
    const int nblk = a.K / 32, nmac = (nblk + 7) / 8;
    constexpr int XMAC = mx_macro_bytes(AK);
    const int64_t wrow = a.K / 2, xrow = static_cast<int64_t>(nmac) * XMAC;
    const int width = a.glu ? a.nrows / 2 : a.nrows, step = a.glu ? BN / 2 : BN;  // results of a row; of a tile
    const int tiles_n = (width + step - 1) / step;

    int tn = 0, tm = 0, expert = 0, first = 0, rows, m0 = 0;
    if constexpr (MODE == kMapped) {
        mxs_zero_rows(a, blockIdx.x, gridDim.x, tid, NW * 64);
        const int total = mxs_total_tiles(a, BM, lane) * tiles_n, per = (total + 7) / 8;
        const int t = (blockIdx.x & 7) * per + (blockIdx.x >> 3);  // an XCD takes neighbouring tiles
        if (t >= total || static_cast<int>(blockIdx.x >> 3) >= per) return;
        int t0, count;
        mxs_find_tile(a, BM, lane, t / tiles_n, expert, t0, count);
        const int in = t - t0 * tiles_n;  // of the expert's tiles, those of the same neurons side by side
        tn = in / count;
        first = a.bounds[expert] + in % count * BM;
        rows = min(BM, a.bounds[expert + 1] - first);
        if (a.slot) expert = a.slot[expert];
        expert = __builtin_amdgcn_readfirstlane(expert);
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
    // neuron of row l of the tile: with GLU the second half of a wave's row-blocks holds the up rows of the first half's gate rows
    auto neuron = [&](int l) {
        if (!a.glu) return min(n0 + l, a.nrows - 1);
        const int j = l >> 4, w_ = j / TN, t = j % TN;
        const int n = min(n0 + (w_ * (TN / 2) + t % (TN / 2)) * 16 + (l & 15), width - 1);
        return t < TN / 2 ? n : width + n;
    };

    const __amdgpu_buffer_rsrc_t win = wave_window(a.wv + static_cast<int64_t>(expert) * a.nrows * wrow, static_cast<uint32_t>(a.nrows * wrow));
    const __amdgpu_buffer_rsrc_t swin = wave_window(a.ws + static_cast<int64_t>(expert) * a.nrows * a.sstride, static_cast<uint32_t>(a.nrows) * a.sstride);
    const int64_t base = MODE == kLinear ? m0 : 0;
    const int span = MODE == kLinear ? rows : a.M;
    const __amdgpu_buffer_rsrc_t xwin = wave_window(a.xv + base * xrow, static_cast<uint32_t>(span * xrow));
    const __amdgpu_buffer_rsrc_t xswin = wave_window(a.xs + base * a.sstride, static_cast<uint32_t>(span) * a.sstride);
    const int piece = lane & 7;
    uint32_t wv[PW], xv[PX], xv2[PT], wsv[QW], xsv[QX];
#pragma unroll
    for (int p = 0; p < PW; ++p) {
        const int l = min(8 * (wave + NW * p), BN - 8) + (lane >> 3);
        wv[p] = static_cast<uint32_t>(neuron(l) * wrow) + 16u * (piece ^ mx_key(l & 15));
    }
#pragma unroll
    for (int p = 0; p < PX; ++p) {
        const int l = min(8 * (wave + NW * p), BM - 8) + (lane >> 3);
        xv[p] = static_cast<uint32_t>((src_of(min(l, rows - 1)) - base) * xrow) + 16u * (piece ^ mx_key(l & 15));
    }
    if constexpr (AK == 6) {
#pragma unroll
        for (int p = 0; p < PT; ++p) {
            const int l = min(16 * (wave + NW * p), BM - 16) + (lane >> 2);
            xv2[p] = static_cast<uint32_t>((src_of(min(l, rows - 1)) - base) * xrow) + 128u + 16u * row_order_quarter(l & 15, lane & 3);
        }
    }
#pragma unroll
    for (int p = 0; p < QW; ++p) wsv[p] = static_cast<uint32_t>(neuron(min(32 * (wave + NW * p), BN - 32) + (lane >> 1))) * a.sstride + 4u * (lane & 1);
#pragma unroll
    for (int p = 0; p < QX; ++p)
        xsv[p] = static_cast<uint32_t>(src_of(min(min(32 * (wave + NW * p), BM - 32) + (lane >> 1), rows - 1)) - base) * a.sstride + 4u * (lane & 1);

    // Pieces of weights behind the last block of a row: the last one again.  The activations there are zeros.
    auto issue = [&](int stage, int mac) {
        uint8_t *to = lds + stage * S::STAGE;
        const int last = nblk - 1 - 8 * mac;
        const int xat = mac * XMAC;
#pragma unroll
        for (int p = 0; p < PW; ++p) {
            const int q = wave + NW * p;
            if ((BN / 8) % NW != 0 && q >= BN / 8) continue;
            uint32_t off = wv[p];
            if (last < 7) off -= 16u * max(0, (piece ^ mx_key((8 * q + (lane >> 3)) & 15)) - last);
            copy16<0>(win, to + q * 1024, off, mac * 128);
        }
#pragma unroll
        for (int p = 0; p < PX; ++p) {
            const int q = wave + NW * p;
            if ((BM / 8) % NW != 0 && q >= BM / 8) continue;
            copy16<0>(xwin, to + S::W + q * 1024, xv[p], xat);
        }
        if constexpr (AK == 6) {
#pragma unroll
            for (int p = 0; p < PT; ++p) {
                const int q = wave + NW * p;
                if ((BM / 16) % NW != 0 && q >= BM / 16) continue;
                copy16<0>(xwin, to + S::W + BM * 128 + q * 1024, xv2[p], xat);
            }
        }
#pragma unroll
        for (int p = 0; p < QW; ++p) {
            const int q = wave + NW * p;
            if ((BN / 32) % NW != 0 && q >= BN / 32) continue;
            copy4(swin, to + S::W + S::X + q * 256, wsv[p], mac * 8);
        }
#pragma unroll
        for (int p = 0; p < QX; ++p) {
            const int q = wave + NW * p;
            if ((BM / 32) % NW != 0 && q >= BM / 32) continue;
            copy4(xswin, to + S::W + S::X + S::WS + q * 256, xsv[p], mac * 8);
        }
    };

    float4_t acc[TM][TN];
#pragma unroll
    for (int m = 0; m < TM; ++m)
#pragma unroll
        for (int n = 0; n < TN; ++n) acc[m][n] = float4_t{0.f, 0.f, 0.f, 0.f};

    auto multiply = [&](int stage) {
        const uint8_t *at = lds + stage * S::STAGE;
        const uint8_t *wat = at + wn * TN * 2048 + r * 128, *xat = at + S::W + wm * TM * 2048 + r * 128;
        uint32_t sw[TN], sx[TM];
        u32x4_t tail[TM];
#pragma unroll
        for (int n = 0; n < TN; ++n) sw[n] = *reinterpret_cast<const uint16_t *>(at + S::W + S::X + (wn * TN + n) * 128 + r * 8 + 2 * g);
#pragma unroll
        for (int m = 0; m < TM; ++m) {
            sx[m] = *reinterpret_cast<const uint16_t *>(at + S::W + S::X + S::WS + (wm * TM + m) * 128 + r * 8 + 2 * g);
            if constexpr (AK == 6) tail[m] = *reinterpret_cast<const u32x4_t *>(at + S::W + BM * 128 + (wm * TM + m) * 1024 + row_order_lane(lane));
        }
        static_for<2>([&](auto SS) {
            constexpr int s = SS.value;
            const int pc = ((2 * g + s) ^ key) << 4;
            u32x4_t w[TN];
            MxFrag x[TM];
#pragma unroll
            for (int n = 0; n < TN; ++n) w[n] = *reinterpret_cast<const u32x4_t *>(wat + n * 2048 + pc);
#pragma unroll
            for (int m = 0; m < TM; ++m) {
                x[m].x = *reinterpret_cast<const u32x4_t *>(xat + m * 2048 + pc);
                if constexpr (AK == 6) x[m].y = s == 0 ? u32x2_t{tail[m].x, tail[m].y} : u32x2_t{tail[m].z, tail[m].w};
            }
#pragma unroll
            for (int m = 0; m < TM; ++m)
#pragma unroll
                for (int n = 0; n < TN; ++n) acc[m][n] = mx_scale_mfma<AK, s>(w[n], x[m], acc[m][n], sw[n], sx[m]);
        });
    };

    const int per_split = (nmac + a.splits - 1) / a.splits;
    const int mac0 = static_cast<int>(blockIdx.y) * per_split, mac1 = min(nmac, mac0 + per_split);
    issue(0, mac0);
    int stage = 0;
    for (int mac = mac0; mac < mac1; ++mac) {
        // the copies of this stage have landed, and every wave has read the other one
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (mac + 1 < mac1) issue(stage ^ 1, mac + 1);
        multiply(stage);
        stage ^= 1;
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __syncthreads();

    // results leave through LDS so that the lanes of a store lie side by side in a row
    uint8_t *area = lds + wave * kRowsOut;
    const bool partial = a.splits > 1;
#pragma unroll
    for (int m = 0; m < TM; ++m) {
        const int mt = (wm * TM + m) * 16;
        auto dst = [&](int i) { return mt + i < rows ? pair_of(mt + i) : -1; };
        auto put = [&](auto NG, const float4_t *v, int col, int end, bool f32, float *y, int64_t ldy) {
            constexpr int G = NG.value;
            const bool wide = ldy % (f32 ? 4 : 8) == 0 && reinterpret_cast<uintptr_t>(y) % 16 == 0;
            if (f32) {
                float4_t o[G];
#pragma unroll
                for (int i = 0; i < G; ++i) o[i] = v[i];
                store_rows<G>(area, o, lane, col, end, y, ldy, wide, dst);
            } else {
                u32x2_t o[G];
#pragma unroll
                for (int i = 0; i < G; ++i) o[i] = u32x2_t{mx_pack16(v[i][0], v[i][1], a.y_dtype), mx_pack16(v[i][2], v[i][3], a.y_dtype)};
                store_rows16<G>(area, o, lane, col, end, reinterpret_cast<uint16_t *>(y), ldy, wide, dst);
            }
        };
        constexpr int G = TN < 4 ? TN : 4, H = TN / 2 < 4 ? TN / 2 : 4;
        if (partial) {
            float *part = a.part + static_cast<int64_t>(blockIdx.y) * a.M * a.nrows;
            if (a.glu) {
#pragma unroll
                for (int b = 0; b < TN; b += H) {
                    const int half = b >= TN / 2, at = n0 + (wn * (TN / 2) + b % (TN / 2)) * 16;
                    put(std::integral_constant<int, H>{}, &acc[m][b], half * width + at, half * width + max(at, width), true, part, a.nrows);
                }
            } else {
#pragma unroll
                for (int b = 0; b < TN; b += G) put(std::integral_constant<int, G>{}, &acc[m][b], n0 + (wn * TN + b) * 16, a.nrows, true, part, a.nrows);
            }
        } else if (a.glu) {
#pragma unroll
            for (int b = 0; b < TN / 2; b += H) {
                float4_t v[H];
#pragma unroll
                for (int i = 0; i < H; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[i][j] = glu_value(acc[m][b + i][j], acc[m][TN / 2 + b + i][j], a.gelu);
                put(std::integral_constant<int, H>{}, v, n0 + (wn * (TN / 2) + b) * 16, width, a.y_dtype == MFQ_X_F32, static_cast<float *>(a.y), a.ldy);
            }
        } else {
#pragma unroll
            for (int b = 0; b < TN; b += G)
                put(std::integral_constant<int, G>{}, &acc[m][b], n0 + (wn * TN + b) * 16, width, a.y_dtype == MFQ_X_F32, static_cast<float *>(a.y), a.ldy);
        }
    }
}

// the pieces of a split over K, added in their order
__global__ __launch_bounds__(256) void mxs_join_kernel(MxsArgs a) {
    const int width = a.glu ? a.nrows / 2 : a.nrows;
    const int64_t all = static_cast<int64_t>(a.M) * a.nrows;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < static_cast<int64_t>(a.M) * width; i += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t m = i / width;
        const int n = static_cast<int>(i - m * width);
        const float *p = a.part + m * a.nrows + n;
        float v = 0.f, u = 0.f;
        for (int s = 0; s < a.splits; ++s) v += p[s * all];
        if (a.glu) {
            for (int s = 0; s < a.splits; ++s) u += p[s * all + width];
            v = glu_value(v, u, a.gelu);
        }
        store_rounded(a.y, m * a.ldy + n, v, a.y_dtype);
    }
}

// ---- launches -------------------------------------------------------------------------------------------------------------------
constexpr int kResBytes = 32 * 1024;   // activations a block keeps in LDS
constexpr int kFuseValues = 20480;     // values up to which a block quantises its activations itself

template <int AK, int MT, int NB, int D, bool RES, int MODE>
int launch_stream(const MxsArgs &a, int tiles, hipStream_t st) {
    using S = StreamShape<AK, MT, NB, D, RES>;
    const int nmac = (a.K / 32 + 7) / 8, rows = MODE == kLinear ? (a.M < 16 * MT ? a.M : 16 * MT) : MODE == kPairs ? 1 : 16 * MT;
    const size_t res = RES ? static_cast<size_t>(rows) * nmac * (mx_macro_bytes(AK) + 8) : 0;
    int nwaves = nmac < 8 ? nmac : 8;
    while (nwaves > 1 && nwaves * static_cast<size_t>(D) * S::STAGE + res > kMaxDynamicLds) --nwaves;
    size_t lds = nwaves * static_cast<size_t>(D) * S::STAGE + res;
    const size_t red = static_cast<size_t>(nwaves) * NB * MT * 1024;
    if (lds < red) lds = red;
    const int width = a.glu ? a.nrows / 2 : a.nrows, per = 16 * (a.glu ? NB / 2 : NB);
    auto kern = mxs_stream_kernel<AK, MT, NB, D, RES, MODE>;
    if (int rc = allow_dynamic_lds(reinterpret_cast<const void *>(kern), lds, "mx_scaled")) return rc;
    hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(ceil_div(width, per)), static_cast<unsigned>(tiles)), dim3(64 * nwaves), lds, st, a);
    return check_launch("mx_scaled (stream)");
}

template <int AK, int MT, bool RES, int MODE>
int launch_stream_nb(const MxsArgs &a, int tiles, hipStream_t st) {
    if (a.glu) return launch_stream<AK, MT, 2, 2, RES, MODE>(a, tiles, st);
    return launch_stream<AK, MT, 1, 2, RES, MODE>(a, tiles, st);
}

template <int AK, int BN, int BM, int WN, int WM, int MODE>
int launch_tile(const MxsArgs &a, hipStream_t st) {
    using S = TileShape<AK, BN, BM>;
    const int width = a.glu ? a.nrows / 2 : a.nrows;
    const int64_t tiles_n = ceil_div(width, a.glu ? BN / 2 : BN);
    const int64_t tiles_m = MODE == kMapped ? ceil_div(a.pairs, BM) + (a.E < a.pairs ? a.E : a.pairs) : ceil_div(a.M, BM);
    const int64_t blocks = (tiles_n * tiles_m + 7) / 8 * 8;
    MFQ_REQUIRE(blocks < (1ll << 31), MFQ_ERR_UNSUPPORTED, "mx_scaled: %lld tiles", static_cast<long long>(blocks));
    size_t lds = 2 * S::STAGE;
    if (lds < WN * WM * static_cast<size_t>(kRowsOut)) lds = WN * WM * static_cast<size_t>(kRowsOut);
    auto kern = mxs_tile_kernel<AK, BN, BM, WN, WM, MODE>;
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

// Kernel of a call: rows up to which the weights are streamed, tile and pieces of K above.
struct MxsPlan { int kind, splits; };  // kind: 0 streamed, activations in LDS; 1, 2 streamed, one or two tiles; 3 .. 5 tiles
constexpr int kPlanTile = 3;
constexpr int kTileN[3] = {128, 256, 256}, kTileM[3] = {64, 128, 256};

MxsPlan plan_linear(int act, int nrows, int K, int M, bool glu) {
    const int nmac = (K / 32 + 7) / 8;
    if (M <= 16 && static_cast<int64_t>(M) * nmac * mx_macro_bytes(act) <= kResBytes) return {0, 1};
    if (M <= 16) return {1, 1};
    if (M <= 32) return {2, 1};
    const int cus = device_cu_count();
    const int shapes = act == 4 ? 3 : 2;
    int best = 0;
    for (int s = 0; s < shapes; ++s)
        if (ceil_div(nrows, kTileN[s]) * ceil_div(M, kTileM[s]) >= cus || s == 0) best = s;
    const int64_t tiles = ceil_div(nrows, kTileN[best]) * ceil_div(M, kTileM[best]);
    int splits = 1;
    while (splits < 8 && tiles * splits * 2 <= cus && nmac / (splits * 2) >= 2) splits *= 2;
    // no piece may be empty
    while (splits > 1 && (splits - 1) * ceil_div(nmac, splits) >= nmac) --splits;
    return {kPlanTile + best, splits};
}

size_t quantized_bytes(int act, int K, int64_t M) {
    const auto up = [](int64_t n) { return (n + 255) & ~static_cast<int64_t>(255); };
    return static_cast<size_t>(up(M * mx_row_bytes(act, K)) + up(M * mx_scale_stride(K)));
}

template <int AK>
int run_linear(const MxsArgs &a, const MxsPlan &p, hipStream_t st) {
    switch (p.kind) {
        case 0: return launch_stream_nb<AK, 1, true, kLinear>(a, 1, st);
        case 1: return launch_stream_nb<AK, 1, false, kLinear>(a, 1, st);
        case 2: return launch_stream_nb<AK, 2, false, kLinear>(a, 1, st);
        case 3: return launch_tile<AK, 128, 64, 2, 2, kLinear>(a, st);
        case 4: return launch_tile<AK, 256, 128, 4, 2, kLinear>(a, st);
        default:
            if constexpr (AK == 4) return launch_tile<AK, 256, 256, 2, 4, kLinear>(a, st);
            else return fail(MFQ_ERR_UNSUPPORTED, "mx_scaled: no such tile");
    }
}

// smallest tile of rows that holds the pairs an expert has on average, half as many again
int plan_mapped(int64_t pairs, int E) {
    const int64_t mean = ceil_div(pairs, E);
    return mean <= 10 ? 0 : mean <= 24 ? 1 : mean <= 64 ? 2 : 3;
}

template <int AK>
int run_experts(const MxsArgs &a, hipStream_t st) {
    if (!a.ids_dst) return launch_stream_nb<AK, 1, true, kPairs>(a, a.pairs, st);
    const auto most = [&](int rows) { return static_cast<int>(ceil_div(a.pairs, rows) + (a.E < a.pairs ? a.E : a.pairs)); };
    switch (plan_mapped(a.pairs, a.E)) {
        case 0: return launch_stream_nb<AK, 1, false, kMapped>(a, most(16), st);
        case 1: return launch_stream_nb<AK, 2, false, kMapped>(a, most(32), st);
        case 2: return launch_tile<AK, 128, 64, 2, 2, kMapped>(a, st);
        default: return launch_tile<AK, 256, 128, 4, 2, kMapped>(a, st);
    }
}

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
    a.wv = static_cast<const uint8_t *>(values);
    a.ws = static_cast<const uint8_t *>(scales);
    a.y = const_cast<void *>(y);
    a.ldy = ldy;
    a.K = cols;
    a.sstride = mx_scale_stride(cols);
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
    const MxsPlan p = plan_linear(act, nrows, cols, M, false);
    size_t n = x_quantized || (p.kind == 0 && static_cast<int64_t>(M) * cols <= kFuseValues) ? 0 : quantized_bytes(act, cols, M);
    if (p.splits > 1) n += static_cast<size_t>(p.splits) * M * nrows * 4;
    return n;
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
    MFQ_REQUIRE(static_cast<int64_t>(nrows) * (cols / 2) < (1ll << 32) - 256, MFQ_ERR_UNSUPPORTED, "mx_scaled_gemm_rows: %d x %d weights", nrows, cols);
    const hipStream_t st = as_stream(stream);
    a.wv += static_cast<int64_t>(row0) * (cols / 2);
    a.ws += static_cast<int64_t>(row0) * a.sstride;
    a.nrows = nrows;
    a.M = M;
    a.R = 1;
    MxsPlan p = plan_linear(act, nrows, cols, M, glu != 0);
    uint8_t *ws = static_cast<uint8_t *>(workspace);
    size_t used = 0;
    if (x_scales) {
        a.xv = static_cast<const uint8_t *>(x);
        a.xs = static_cast<const uint8_t *>(x_scales);
    } else if (p.kind == 0 && static_cast<int64_t>(M) * cols <= kFuseValues) {
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
        const size_t left = workspace_bytes > used && ws ? workspace_bytes - used : 0, each = static_cast<size_t>(M) * nrows * 4;
        const int nmac = (cols / 32 + 7) / 8;
        if (left / each < static_cast<size_t>(p.splits)) p.splits = static_cast<int>(left / each);
        while (p.splits > 1 && (p.splits - 1) * ceil_div(nmac, p.splits) >= nmac) --p.splits;
        if (p.splits < 2 || reinterpret_cast<uintptr_t>(ws) % 16 != 0) p.splits = 1;
        a.splits = p.splits;
        a.part = reinterpret_cast<float *>(ws + used);
    }
    if (int rc = act == 4 ? run_linear<4>(a, p, st) : run_linear<6>(a, p, st)) return rc;
    return launch_join(a, st);
}

extern "C" size_t mfq_hip_mx_moe_workspace_bytes(int act, int cols, int x_rows, int mapped, int x_quantized) {
    if ((act != 4 && act != 6) || cols <= 0 || cols % 32 != 0 || x_rows <= 0 || !mapped || x_quantized) return 0;
    return quantized_bytes(act, cols, x_rows);
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
    MFQ_REQUIRE(static_cast<int64_t>(out_per_expert) * (cols / 2) < (1ll << 32) - 256 && x_rows * mx_row_bytes(act, cols) < (1ll << 32) - 256,
                MFQ_ERR_UNSUPPORTED, "mx_moe_matmul: an expert of %d x %d, %d rows of activations", out_per_expert, cols, x_rows);
    const int nmac = (cols / 32 + 7) / 8;
    if (!ids_dst) {
        MFQ_REQUIRE(T * R <= 65535, MFQ_ERR_UNSUPPORTED, "mx_moe_matmul: %d pairs without a route map", T * R);
        MFQ_REQUIRE(nmac * mx_macro_bytes(act) <= 64 * 1024, MFQ_ERR_UNSUPPORTED, "mx_moe_matmul: %d columns without a route map", cols);
    } else {
        MFQ_REQUIRE(ceil_div(T * R, 16) + E <= 65535 || plan_mapped(static_cast<int64_t>(T) * R, E) > 1, MFQ_ERR_UNSUPPORTED, "mx_moe_matmul: %d experts, %d pairs", E, T * R);
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
    } else if (!ids_dst) {
        a.xraw = x;
        a.x_wide = pieces(x, x_dtype, ldx, x_rows);
        a.x_dtype = x_dtype;
        a.ldx = ldx;
    } else {
        const size_t need = quantized_bytes(act, cols, x_rows);
        MFQ_REQUIRE(workspace && workspace_bytes >= need, MFQ_ERR_WORKSPACE, "mx_moe_matmul: workspace %zu < %zu", workspace_bytes, need);
        MFQ_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, MFQ_ERR_WORKSPACE, "mx_moe_matmul: unaligned workspace");
        uint8_t *ws = static_cast<uint8_t *>(workspace);
        uint8_t *xs = ws + ((static_cast<int64_t>(x_rows) * mx_row_bytes(act, cols) + 255) & ~static_cast<int64_t>(255));
        if (int rc = mx_quantize_launch(act, x, x_dtype, ldx, x_rows, cols, ws, xs, st)) return rc;
        a.xv = ws;
        a.xs = xs;
    }
    return act == 4 ? run_experts<4>(a, st) : run_experts<6>(a, st);
}
