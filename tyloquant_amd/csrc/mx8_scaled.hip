// Products of MXFP8 weights, read in place, with activations quantised to E4M3 by blocks of 128 columns (mx8.hpp); one tensor, or the
// tensors of routed experts.
#include "mx8.hpp"

namespace mfq {
namespace {

template <int SEL>
__device__ __forceinline__ float4_t mx8_mfma(i32x8_t w, i32x8_t x, float4_t c, uint32_t sw, uint32_t sx) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, c, 0, 0, 0, static_cast<int>(sw), SEL, static_cast<int>(sx));
}
__device__ __forceinline__ float16_t mx8_mfma32(i32x8_t w, i32x8_t x, float16_t c, uint32_t sw, uint32_t sx) {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w, x, c, 0, 0, 0, static_cast<int>(sw), 0, static_cast<int>(sx));
}

// ---- few rows ---------------------------------------------------------------------------------------------------------------------
// A block owns a range of row-blocks of 16 neurons (with GLU those of the gate rows, each with that of its up rows) and up to 16 * MT rows
// of activations.  Its waves take the blocks of 128 columns in turn; a wave's activations are operands in its registers from the
// first row-block to the last, quantised there where they come as bf16, fp16 or fp32.  The weights go through a ring of D stages of the wave's
// own in LDS, lines of 128 bytes copied there directly, across the ends of row-blocks.  The waves' sums of a row-block meet in LDS, behind
// one barrier that no copy waits at, and are added in the order of the waves.  Bound by the weights' way from memory.
template <int MT, int NB>
struct FewShape {
    static constexpr int STAGE = NB * 2048, D = MT * NB == 4 ? 2 : 3, REQ = 2 * NB;  // sums and stages of 32 gated rows share the LDS
    static constexpr int RED = MT * NB * 1024;  // sums of a wave
    // beside the kernel's own 16 * MT words
    static size_t lds(int nwaves, int nkb, int blocks) { return static_cast<size_t>(nwaves) * (D * STAGE + 2 * RED) + static_cast<size_t>(NB) * blocks * nkb; }
    static constexpr size_t MOST = kMaxDynamicLds - 16 * MT * 4;
};

// A lane's 32 columns of a block of 128, whose other three lanes are 16, 32 and 48 further: as they lie, and quantised.  16-bit values are compared
// and converted in pairs as they are: less than half the instructions, and those of a wave's few rows come from memory with the launch.
template <int XD>
struct LaneColumns {
    static constexpr int PIECES = XD == MFQ_X_F32 ? 8 : 4;  // of 16 bytes
    u32x4_t v[PIECES];
};
template <int XD>
__device__ __forceinline__ void load_lane(const void *x, int64_t from, bool wide, LaneColumns<XD> &c) {
    if (wide) {
#pragma unroll
        for (int i = 0; i < c.PIECES; ++i) c.v[i] = reinterpret_cast<const u32x4_t *>(static_cast<const uint8_t *>(x) + from * (XD == MFQ_X_F32 ? 4 : 2))[i];
    } else {
#pragma unroll
        for (int i = 0; i < c.PIECES; ++i)
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                if constexpr (XD == MFQ_X_F32) {
                    c.v[i][t] = static_cast<const uint32_t *>(x)[from + 4 * i + t];
                } else {
                    const uint16_t *p = static_cast<const uint16_t *>(x) + from + 8 * i + 2 * t;
                    c.v[i][t] = p[0] | (static_cast<uint32_t>(p[1]) << 16);
                }
            }
    }
}
template <int XD>
__device__ __forceinline__ void quantize_lane(const LaneColumns<XD> &x, u32x4_t &lo, u32x4_t &hi, uint32_t &byte) {
    typedef short short2_t __attribute__((ext_vector_type(2)));
    const auto &v = x.v;
    uint32_t most = 0;
    if constexpr (XD == MFQ_X_F32) {
#pragma unroll
        for (int i = 0; i < 32; ++i) most = max(most, v[i >> 2][i & 3] & 0x7fffffffu);
    } else {
        u16x2_t pair = {0, 0};
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const uint32_t two = v[i >> 2][i & 3] & 0x7fff7fffu;
            pair = __builtin_elementwise_max(pair, __builtin_bit_cast(u16x2_t, two));
        }
        const uint32_t m = max(pair.x, pair.y);
        // of fp16 as an fp32 has it, infinities and NaN with theirs
        most = XD == MFQ_X_BF16 ? m << 16 : m >= 0x7c00u ? 0x7f800000u : __float_as_uint(f16_to_f32(static_cast<uint16_t>(m)));
    }
    most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), 16, 64)));
    most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), 32, 64)));
    byte = mx8_scale_of(most);
    const float scale = __uint_as_float(byte << 23);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        uint32_t q;
        if constexpr (XD == MFQ_X_F32) {
            q = mx8_codes(__uint_as_float(v[i][0]), __uint_as_float(v[i][1]), __uint_as_float(v[i][2]), __uint_as_float(v[i][3]), scale);
        } else {
            const uint32_t a = v[i >> 1][2 * (i & 1)], b = v[i >> 1][2 * (i & 1) + 1];
            short2_t c = {0, 0};
            if constexpr (XD == MFQ_X_F16) {
                c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(c, __builtin_bit_cast(half2_t, a), scale, false);
                c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(c, __builtin_bit_cast(half2_t, b), scale, true);
            } else {
                c = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(c, __builtin_bit_cast(bf16x2_t, a), scale, false);
                c = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(c, __builtin_bit_cast(bf16x2_t, b), scale, true);
            }
            q = __builtin_bit_cast(uint32_t, c);
        }
        (i < 4 ? lo : hi)[i & 3] = byte == 255u ? 0u : q;
    }
}

__device__ __forceinline__ void pin(i32x8_t &v) { asm volatile("" : "+v"(v)); }

template <int MT, int NB, int NM>
__global__ __launch_bounds__(512, MT * NM <= 8 ? 4 : 2) void mx8_few_kernel(MxsArgs a, int mode, int chunks, int scale_rows) {
    using S = FewShape<MT, NB>;
    constexpr int D = S::D;
    static_assert(D == 2 || D == 3, "the waits of the loop");
    extern __shared__ __attribute__((aligned(128))) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, nwaves = blockDim.x >> 6;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15, g = lane >> 4;
    const int nkb = a.K / kMx8Block, width = NB == 2 ? a.nrows / 2 : a.nrows;  // results of a row
    const int tile = static_cast<int>(blockIdx.x) / chunks, chunk = static_cast<int>(blockIdx.x) - tile * chunks;

    int expert = 0, m0 = 0, first = 0, rows;
    if (mode == kPairs) {
        expert = a.ids[tile];
        if (expert < 0 || expert >= a.E) {
            if (chunk == 0) mxs_zero_rows(a, tile, a.pairs, tid, blockDim.x);
            return;
        }
        if (a.slot) expert = a.slot[expert];
        if (expert < 0) return;
        rows = 1;
    } else if (mode == kMapped) {
        mxs_zero_rows(a, blockIdx.x, gridDim.x, tid, blockDim.x);
        if (tile >= mxs_total_tiles(a, 16 * MT, lane)) return;
        int t0;
        mxs_find_tile(a, 16 * MT, lane, tile, expert, t0);
        first = a.bounds[expert] + (tile - t0) * 16 * MT;
        rows = min(16 * MT, a.bounds[expert + 1] - first);
        if (a.slot) expert = a.slot[expert];
    } else {
        m0 = tile * 16 * MT;
        rows = min(16 * MT, a.M - m0);
    }
    expert = __builtin_amdgcn_readfirstlane(expert);
    auto pair_of = [&](int m) { return mode == kPairs ? tile : mode == kMapped ? a.ids_dst[first + m] : m0 + m; };

    const int rbs = (width + 15) / 16;
    // the first blocks of a tile have a row-block more than the last: those that come second to a compute unit
    const int each = rbs / chunks, more = rbs - each * chunks;
    const int rb0 = chunk * each + min(chunk, more), rb1 = rb0 + each + (chunk < more ? 1 : 0);
    const int mine = (nkb - wave + nwaves - 1) / nwaves;  // blocks wave, wave + nwaves, ... of K
    const int total = (rb1 - rb0) * mine;

    // the weights' ring
    const int64_t half = static_cast<int64_t>(width) * a.K;  // from a gate row to its up row
    const uint8_t *wbase = a.wv + (static_cast<int64_t>(expert) * a.nrows + rb0 * 16) * a.K;
    const int64_t span = static_cast<int64_t>(min(rb1 * 16, width) - rb0 * 16) * a.K;
    const __amdgpu_buffer_rsrc_t win = wave_window(wbase, static_cast<uint32_t>(span)), win_up = wave_window(wbase + half, static_cast<uint32_t>(span));
    uint8_t *ring = lds + wave * (D * S::STAGE);
    const int piece = lane & 7;
    const uint32_t off0 = static_cast<uint32_t>((lane >> 3) * a.K) + 16u * (piece ^ mx_key(lane >> 3));
    const uint32_t off1 = static_cast<uint32_t>((8 + (lane >> 3)) * a.K) + 16u * (piece ^ mx_key(8 + (lane >> 3)));
    int to_stage = 0, to_rb = rb0, to_m = 0;
    auto issue = [&] {
        uint8_t *to = ring + to_stage * S::STAGE;
        const int valid = width - to_rb * 16;
        const int at = static_cast<int>(static_cast<uint32_t>((to_rb - rb0) * 16) * static_cast<uint32_t>(a.K) + static_cast<uint32_t>((wave + to_m * nwaves) * kMx8Block));
#pragma unroll
        for (int i = 0; i < 2 * NB; ++i) {
            uint32_t off = i & 1 ? off1 : off0;
            // neurons behind the last one: the last one again
            if (valid < 16) off -= static_cast<uint32_t>(max(0, 8 * (i & 1) + (lane >> 3) - (valid - 1)) * a.K);
            copy16<2>(i < 2 ? win : win_up, to + i * 1024, off, at);
        }
        to_stage = to_stage + 1 == D ? 0 : to_stage + 1;
        if (++to_m == mine) {
            to_m = 0;
            ++to_rb;
        }
    };

    // The first weights are asked for, then what else a wave needs before it can use them, then the next weights: behind all of a wave's
    // weights the activations would come late, in front of them the weights.
    if (total > 0) issue();
    // scales of the weights: those of the rows' blocks of 128, all of K; a byte a thread does for all but long shares
    uint8_t *scales = lds + nwaves * (D * S::STAGE + 2 * S::RED);
    const int row_base = a.row0 + expert * a.nrows;
    int scale_count[NB];
    const uint8_t *scale_from[NB];
    uint32_t scale_first[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const int f = (row_base + b * width + rb0 * 16) >> 7, l = (row_base + b * width + min(rb1 * 16, width) - 1) >> 7;
        scale_count[b] = (l - f + 1) * nkb;
        scale_from[b] = a.ws + static_cast<int64_t>(f) * nkb;
        scale_first[b] = scale_from[b][min(tid, scale_count[b] - 1)];
    }

    // the activations, as operands: the reads of two or four blocks of K are in flight together
    i32x8_t x[NM][MT];
    uint32_t sx[(NM + 3) / 4][MT];
#pragma unroll
    for (int m = 0; m < (NM + 3) / 4; ++m)
#pragma unroll
        for (int t = 0; t < MT; ++t) sx[m][t] = 0u;
    int64_t src[MT];
    bool live[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        live[t] = 16 * t + r < rows;
        const int p = pair_of(min(16 * t + r, rows - 1));
        src[t] = mode == kLinear || a.routed ? p : p / a.R;
    }
    const auto keep = [&](int m, int t, u32x4_t lo, u32x4_t hi, uint32_t byte) __attribute__((always_inline)) {
        const bool use = live[t] && m < mine;
        const u32x4_t none = {0u, 0u, 0u, 0u};
        x[m][t] = mx8_operand(use ? lo : none, use ? hi : none);
        sx[m >> 2][t] |= (use ? byte : 0u) << (8 * (m & 3));
    };
    const auto block_of = [&](int m) { return min(wave + m * nwaves, nkb - 1); };
    const auto quantize = [&](auto XD) __attribute__((always_inline)) {
        constexpr int TYPE = XD.value, GROUP = TYPE == MFQ_X_F32 || NM > 4 ? 2 : 4;
        static_for<MT * NM / GROUP>([&](auto Q) __attribute__((always_inline)) {
            constexpr int t = Q.value / (NM / GROUP), m0 = Q.value % (NM / GROUP) * GROUP;
            LaneColumns<TYPE> c[GROUP];
#pragma unroll
            for (int m = 0; m < GROUP; ++m) load_lane<TYPE>(a.xraw, src[t] * a.ldx + block_of(m0 + m) * kMx8Block + 32 * g, a.x_wide, c[m]);
#pragma unroll
            for (int m = 0; m < GROUP; ++m) {
                u32x4_t lo, hi;
                uint32_t byte;
                quantize_lane<TYPE>(c[m], lo, hi, byte);
                keep(m0 + m, t, lo, hi, byte);
            }
            // operands now, not where they are used: what they are made of takes twice the registers
#pragma unroll
            for (int m = 0; m < GROUP; ++m) pin(x[m0 + m][t]);
        });
    };
    static_assert(NM % 4 == 0, "whole groups");
    if (a.xraw) {
        if constexpr (MT == 1) {  // more rows come quantised
            if (a.x_dtype == MFQ_X_BF16) quantize(std::integral_constant<int, MFQ_X_BF16>{});
            else if (a.x_dtype == MFQ_X_F16) quantize(std::integral_constant<int, MFQ_X_F16>{});
            else quantize(std::integral_constant<int, MFQ_X_F32>{});
        }
    } else {
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int m = 0; m < NM; ++m) {
                const u32x4_t *q = reinterpret_cast<const u32x4_t *>(a.xv + src[t] * a.K + block_of(m) * kMx8Block + 32 * g);
                keep(m, t, q[0], q[1], a.xs[mx8_scale_at(a.M, src[t], block_of(m))]);
            }
    }
#pragma unroll
    for (int i = 1; i < D; ++i)
        if (i < total) issue();
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        if (tid < scale_count[b]) scales[b * scale_rows * nkb + tid] = static_cast<uint8_t>(scale_first[b]);
        for (int i = tid + blockDim.x; i < scale_count[b]; i += blockDim.x) scales[b * scale_rows * nkb + i] = scale_from[b][i];
    }

    const int results = MT * 256;  // of a row-block; result o: row o / 16, neuron o % 16
    __shared__ int row_of[16 * MT];
    if (tid < 16 * MT) row_of[tid] = tid < rows ? pair_of(tid) : 0;
    __syncthreads();  // these, and the scales
    uint8_t *red = lds + nwaves * (D * S::STAGE);
    int stage = 0, i = 0;
    for (int rb = rb0; rb < rb1; ++rb) {
        float4_t acc[NB][MT];
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[b][t] = float4_t{0.f, 0.f, 0.f, 0.f};
        const uint8_t *srow[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int n = row_base + b * width;
            srow[b] = scales + (b * scale_rows + ((n + min(rb * 16 + r, width - 1)) >> 7) - ((n + rb0 * 16) >> 7)) * nkb + wave;
        }
        static_for<NM>([&](auto MI) __attribute__((always_inline)) {
            constexpr int m = MI.value;
            if (m >= mine) return;
            // younger than this stage: those of the next D - 1, and stores of results, which only make the wait longer
            const int left = total - 1 - i;
            if (left >= D - 1) wait_vmcnt<(D - 1) * S::REQ>();
            else if (left == 1) wait_vmcnt<S::REQ>();
            else wait_vmcnt<0>();
            const uint8_t *at = ring + stage * S::STAGE;
            u32x4_t w[NB][2];
            uint32_t sw[NB];
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                sw[b] = srow[b][m * nwaves];
#pragma unroll
                for (int s = 0; s < 2; ++s) w[b][s] = *reinterpret_cast<const u32x4_t *>(at + b * 2048 + r * 128 + (((2 * g + s) ^ mx_key(r)) << 4));
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the stage is free for the next copies
            if (i + D < total) issue();
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int t = 0; t < MT; ++t) acc[b][t] = mx8_mfma<m & 3>(mx8_operand(w[b][0], w[b][1]), x[m][t], acc[b][t], sw[b], sx[m >> 2][t]);
            stage = stage + 1 == D ? 0 : stage + 1;
            ++i;
        });
        uint8_t *slot = red + (rb & 1) * nwaves * S::RED;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int t = 0; t < MT; ++t) *reinterpret_cast<float4_t *>(slot + wave * S::RED + ((b * MT + t) * 64 + lane) * 16) = acc[b][t];
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();  // the slot's next sums come behind the next one
        asm volatile("" ::: "memory");
        for (int o = tid; o < results; o += blockDim.x) {
            const int m = o >> 4, n = o & 15, t = m >> 4;
            if (m >= rows || rb * 16 + n >= width) continue;
            const float *p = reinterpret_cast<const float *>(slot) + t * 256 + ((n >> 2) * 16 + (m & 15)) * 4 + (n & 3);
            float v = 0.f;
            for (int k = 0; k < nwaves; ++k) v += p[k * (S::RED / 4)];
            if constexpr (NB == 2) {
                float u = 0.f;
                for (int k = 0; k < nwaves; ++k) u += p[k * (S::RED / 4) + MT * 256];
                v = glu_value(v, u, a.gelu);
            }
            store_rounded(a.y, row_of[m] * a.ldy + rb * 16 + n, v, a.y_dtype);
        }
    }
}

// ---- many rows: tiles -----------------------------------------------------------------------------------------------------------
// A block of WN * WM waves owns BN neurons x BM rows, a wave BN / WN x BM / WM of them in squares of 32.  K goes by blocks of 128 through a
// ring of R stages in LDS, a line of 128 bytes a row, whose 16-byte pieces are turned by (row / 2) & 7: the four passes of a read meet every
// bank once.  Lane (r, h) multiplies pieces 4 h, 4 h + 1 and then 4 h + 2, 4 h + 3 of both operands.  While the squares of one half are
// multiplied the fragments of the other are read: one barrier a stage.  Scales: a word holds a row's next four blocks; the activations' words
// come with every stage, the weights' lie in LDS for all of K.
// A loop of nothing but 32 x 32 x 64 products of random codes reaches 3.4 PFLOP/s with one wave a SIMD and 3.8 with two (4.9 on zeros: the rest
// is the clock), which is why the largest tile has eight waves and not four of twice the squares (17408 x 5120 at 8192 rows 630 -> 585 us).
// What is left there: a stage's way from L2, one stage ahead of its use, and 5 us of start and end of each of 9 tiles a compute unit.
__host__ __device__ __forceinline__ constexpr int tile_scale_rows(int BN) { return 2 * (BN / 256 + 2); }  // blocks of 128 rows that gate and up rows touch
template <int BN, int BM, int R>
struct Tile8Shape {
    static constexpr int W = BN * 128, X = BM * 128, STAGE = W + X;
    static constexpr int XS = R * STAGE, ROWS = XS + 2 * BM * 4, WS = ROWS + BM * 4;  // where the words, the rows of y and the weights' scales begin
    static constexpr size_t lds(int nkb) { return WS + static_cast<size_t>(tile_scale_rows(BN)) * ((nkb + 3) / 4 * 4) + 16; }  // and a word that is read behind the last
};

template <int BN, int BM, int WN, int WM, int R, int MODE>
__global__ __launch_bounds__(WN *WM * 64) __attribute__((amdgpu_waves_per_eu(BN * BM / (WN * WM) > 8192 ? 1 : 2))) void mx8_tile_kernel(MxsArgs a) {
    using S = Tile8Shape<BN, BM, R>;
    constexpr int NW = WN * WM, TN = BN / 32 / WN, TM = BM / 32 / WM;
    // requests of a wave for a stage; every wave issues as many, some twice
    constexpr int CW = BN / 8, CX = BM / 8, PW = (CW + NW - 1) / NW, PX = (CX + NW - 1) / NW, PER = PW + PX + 1;
    static_assert(TN % 2 == 0 && R >= 2 && BM / 64 <= NW, "gate and up in one wave, words of scales by a wave for 64 rows");
    extern __shared__ __attribute__((aligned(128))) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wn = wave % WN, wm = wave / WN;
    const int r = lane & 31, h = lane >> 5;
    const int nkb = a.K / kMx8Block, words = (nkb + 3) / 4;
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
    // neuron of row l of the tile, as its distance from n0: with GLU the second half of a wave's squares holds the up rows of the first half's
    // gate rows
    auto neuron = [&](int l) {
        if (!a.glu) return min(l, a.nrows - 1 - n0);
        const int j = l >> 5, w_ = j / TN, t = j % TN;
        const int n = min((w_ * (TN / 2) + t % (TN / 2)) * 32 + (l & 31), width - 1 - n0);
        return t < TN / 2 ? n : width + n;
    };
    int *row_of = reinterpret_cast<int *>(lds + S::ROWS);
    for (int m = tid; m < BM; m += NW * 64) row_of[m] = m < rows ? pair_of(m) : -1;

    // the weights' scales of the gate (or all) rows' blocks, and of the up rows'
    uint8_t *wscale = lds + S::WS;
    const int row_base = a.row0 + expert * a.nrows + n0, up_rows = tile_scale_rows(BN) / 2;
    const int block0 = row_base >> 7, block1 = (row_base + width) >> 7;
    for (int b = 0; b < (a.glu ? 2 : 1); ++b) {
        const int from = b ? block1 : block0, to = (row_base + b * width + min(step, width - n0) - 1) >> 7;
        for (int i = tid; i < (to - from + 1) * nkb; i += NW * 64) {
            const int j = i / nkb;
            wscale[(b * up_rows + j) * words * 4 + i - j * nkb] = a.ws[static_cast<int64_t>(from) * nkb + i];
        }
    }
    // where the lane's words of a square's weights lie
    uint32_t wsv[TN];
#pragma unroll
    for (int n = 0; n < TN; ++n) {
        const int at = neuron((wn * TN + n) * 32 + r), up = a.glu && n >= TN / 2;
        wsv[n] = S::WS + static_cast<uint32_t>((up ? up_rows : 0) + ((row_base + at) >> 7) - (up ? block1 : block0)) * static_cast<uint32_t>(words) * 4u;
    }

    const __amdgpu_buffer_rsrc_t win = wave_window(a.wv + (static_cast<int64_t>(expert) * a.nrows + n0) * a.K, 0xffffff00u);  // offsets under 2^32: the host sees to it
    const int64_t base = MODE == kLinear ? m0 : 0;
    const int64_t span = MODE == kLinear ? rows : a.M;
    const __amdgpu_buffer_rsrc_t xwin = wave_window(a.xv + base * a.K, static_cast<uint32_t>(span * a.K));
    const __amdgpu_buffer_rsrc_t xswin = wave_window(a.xs, 0xffffff00u);
    uint32_t wv[PW], xv[PX];
    const int wp = (lane & 7) ^ ((lane >> 4) & 3), wq = wp ^ 4;  // piece of the line that lane's copy takes, in the lower and upper half of 16 rows
#pragma unroll
    for (int p = 0; p < PW; ++p) {
        const int q = min(wave + NW * p, CW - 1);
        wv[p] = static_cast<uint32_t>(neuron(q * 8 + (lane >> 3))) * static_cast<uint32_t>(a.K) + 16u * (q & 1 ? wq : wp);
    }
#pragma unroll
    for (int p = 0; p < PX; ++p) {
        const int q = min(wave + NW * p, CX - 1);
        xv[p] = static_cast<uint32_t>(src_of(min(q * 8 + (lane >> 3), rows - 1)) - base) * static_cast<uint32_t>(a.K) + 16u * (q & 1 ? wq : wp);
    }
    const uint32_t xsv = static_cast<uint32_t>(src_of(min(wave % (BM / 64) * 64 + lane, rows - 1))) * 4u;

    // Stages behind the last one: the last one again, where nobody reads it.
    const int per_split = (nkb + a.splits - 1) / a.splits;
    const int st0 = static_cast<int>(blockIdx.y) * per_split, st1 = min(nkb, st0 + per_split);
    // the words that stage st's scales are bytes of: with every stage, though they serve four, and in every wave, though a few would do, so that
    // the loop has no branch, behind which the compiler would sink the products
    auto copy_scales = [&](int st) __attribute__((always_inline)) {
        copy4(xswin, lds + S::XS + ((st >> 2) & 1) * (BM * 4) + wave % (BM / 64) * 256, xsv + static_cast<uint32_t>(st >> 2) * static_cast<uint32_t>(a.M) * 4u, 0);
    };
    auto copy_codes = [&](uint32_t buffer, int st, auto P) __attribute__((always_inline)) {
        constexpr int p = P.value;
        if constexpr (p == PW + PX) copy_scales(st);
        else if constexpr (p < PW) copy16<0>(win, lds + buffer + min(wave + NW * p, CW - 1) * 1024, wv[p], st * kMx8Block);
        else copy16<0>(xwin, lds + buffer + S::W + min(wave + NW * (p - PW), CX - 1) * 1024, xv[p - PW], st * kMx8Block);
    };

    float16_t acc[TM][TN];
#pragma unroll
    for (int m = 0; m < TM; ++m)
#pragma unroll
        for (int n = 0; n < TN; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[m][n][i] = 0.f;

    u32x4_t w0[TN][2], w1[TN][2], x0[TM][2], x1[TM][2];
    uint32_t sw[TN], sx[TM];
    const uint32_t key = (r >> 1) & 7, line = r * 128;
    // read q of half a stage's fragments
    constexpr int READS = 2 * (TN + TM), SQUARES = TM * TN;
    auto read_codes = [&](uint32_t buffer, int half, u32x4_t (&w)[TN][2], u32x4_t (&x)[TM][2], auto Q) __attribute__((always_inline)) {
        constexpr int f = Q.value / 2, s = Q.value % 2;
        const uint32_t at = buffer + line + (((4 * h + 2 * half + s) ^ key) << 4);
        if constexpr (f < TN) w[f][s] = *reinterpret_cast<const u32x4_t *>(lds + at + (wn * TN + f) * 4096);
        else x[f - TN][s] = *reinterpret_cast<const u32x4_t *>(lds + at + S::W + (wm * TM + f - TN) * 4096);
    };
    // the words of stage st's scales, and its scales in their lowest bytes
    uint32_t ww[TN], wx[TM];
    auto read_scales = [&](int st) __attribute__((always_inline)) {
        const uint32_t at = S::XS + ((st >> 2) & 1) * (BM * 4) + r * 4;
#pragma unroll
        for (int n = 0; n < TN; ++n) ww[n] = *reinterpret_cast<const uint32_t *>(lds + wsv[n] + (st >> 2) * 4);
#pragma unroll
        for (int m = 0; m < TM; ++m) wx[m] = *reinterpret_cast<const uint32_t *>(lds + at + (wm * TM + m) * 128);
    };
    auto take_scales = [&](int st) __attribute__((always_inline)) {
#pragma unroll
        for (int n = 0; n < TN; ++n) sw[n] = ww[n] >> (8 * (st & 3));
#pragma unroll
        for (int m = 0; m < TM; ++m) sx[m] = wx[m] >> (8 * (st & 3));
    };
    auto multiply = [&](const u32x4_t (&w)[TN][2], const u32x4_t (&x)[TM][2], auto Q) __attribute__((always_inline)) {
        constexpr int m = Q.value / TN, n = Q.value % TN;
        acc[m][n] = mx8_mfma32(mx8_operand(w[n][0], w[n][1]), mx8_operand(x[m][0], x[m][1]), acc[m][n], sw[n], sx[m]);
    };
    static_for<R>([&](auto I) __attribute__((always_inline)) {
        static_for<PER>([&](auto P) __attribute__((always_inline)) { copy_codes(I.value * S::STAGE, min(st0 + static_cast<int>(I.value), st1 - 1), P); });
    });
    wait_vmcnt<(R - 1) * PER>();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    uint32_t cur = 0;
    static_for<READS>([&](auto Q) __attribute__((always_inline)) { read_codes(cur, 0, w0, x0, Q); });
    read_scales(st0);
    take_scales(st0);
    // The squares of half a stage one by one, and between them what can go on meanwhile: reads of the other half's fragments, and with the second
    // half, whose stage every wave has read by then, the copies of the stage R further on.  Left to itself the compiler puts all squares behind
    // the barrier, and nothing is multiplied while fragments are read.
    for (int st = st0; st < st1; ++st) {
        static_for<SQUARES>([&](auto Q) __attribute__((always_inline)) {
            multiply(w0, x0, Q);
            static_for<READS>([&](auto P) __attribute__((always_inline)) {
                if constexpr (P.value >= READS * Q.value / SQUARES && P.value < READS * (Q.value + 1) / SQUARES) read_codes(cur, 1, w1, x1, P);
            });
            __builtin_amdgcn_sched_barrier(0);
        });
        // the next stage has landed, and every wave has read this one
        wait_vmcnt<(R - 2) * PER>();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        const uint32_t next = cur + S::STAGE == R * S::STAGE ? 0u : cur + S::STAGE;
        const int ahead = min(st + R, st1 - 1), after = min(st + 1, st1 - 1);
        read_scales(after);
        static_for<SQUARES>([&](auto Q) __attribute__((always_inline)) {
            multiply(w1, x1, Q);
            static_for<PER>([&](auto P) __attribute__((always_inline)) {
                if constexpr (P.value >= PER * Q.value / SQUARES && P.value < PER * (Q.value + 1) / SQUARES) copy_codes(cur, ahead, P);
            });
            static_for<READS>([&](auto P) __attribute__((always_inline)) {
                if constexpr (P.value >= READS * Q.value / SQUARES && P.value < READS * (Q.value + 1) / SQUARES) read_codes(next, 0, w0, x0, P);
            });
            __builtin_amdgcn_sched_barrier(0);
        });
        cur = next;
        take_scales(after);
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");  // late copies must not land in reused LDS
    __syncthreads();
    mxs_tile_results<TM, TN>(a, acc, lds + wave * kTileOut, row_of, n0, wn, wm, rows, width, lane);
}

// ---- launches -------------------------------------------------------------------------------------------------------------------
constexpr int kFewWaves = 8;
constexpr int kMostOperands = 20;  // registers hold so many blocks of 128 columns of 16 rows

// Whether a wave's share of K fits its registers.  Of 32 rows those of 4096 columns: longer ones are faster in tiles, with K in pieces
// (4096 x 12288 at 17 rows 27 us, in a tile 22; 12288 x 4096 17 and 19).
bool few_fits(int K, int tiles) { return ceil_div(K / kMx8Block, kFewWaves) <= (tiles == 1 ? kMostOperands : 4); }

template <int MT, int NB, int NM>
int launch_few_nm(const MxsArgs &a, int mode, int tiles, int busy, hipStream_t st) {
    using S = FewShape<MT, NB>;
    const int nkb = a.K / kMx8Block, nwaves = nkb < kFewWaves ? nkb : kFewWaves;
    const int width = a.glu ? a.nrows / 2 : a.nrows, rbs = static_cast<int>(ceil_div(width, 16));
    // blocks of a tile: two for each compute unit where the LDS has room for two
    const int want = device_cu_count() * (2 * S::lds(nwaves, nkb, 8) <= S::MOST - 64 * MT ? 2 : 1);
    int chunks = static_cast<int>(ceil_div(want, busy > 0 ? busy : 1));
    if (chunks > rbs) chunks = rbs;
    const auto scale_rows = [&] { return static_cast<int>((ceil_div(rbs, chunks) * 16 + 127) / 128 + 1); };
    while (chunks < rbs && S::lds(nwaves, nkb, scale_rows()) > S::MOST) chunks = chunks * 2 < rbs ? chunks * 2 : rbs;  // the scales of fewer rows
    MFQ_REQUIRE(ceil_div(rbs, chunks) * 16 * a.K < (1ll << 31), MFQ_ERR_UNSUPPORTED, "mx8_scaled: %d x %d weights", a.nrows, a.K);
    const size_t lds = S::lds(nwaves, nkb, scale_rows());
    MFQ_REQUIRE(lds <= S::MOST && grid_fits(static_cast<int64_t>(tiles) * chunks, 64 * nwaves), MFQ_ERR_UNSUPPORTED, "mx8_scaled: %d tiles of %d columns", tiles, a.K);
    auto kern = mx8_few_kernel<MT, NB, NM>;
    if (int rc = allow_dynamic_lds(reinterpret_cast<const void *>(kern), lds, "mx8_scaled")) return rc;
    hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(tiles * chunks)), dim3(64 * nwaves), lds, st, a, mode, chunks, scale_rows());
    return check_launch("mx8_scaled (few)");
}
template <int MT, int NB>
int launch_few_nb(const MxsArgs &a, int mode, int tiles, int busy, hipStream_t st) {
    const int64_t n = ceil_div(a.K / kMx8Block, kFewWaves);
    if (n <= 4) return launch_few_nm<MT, NB, 4>(a, mode, tiles, busy, st);
    if constexpr (MT == 1) {
        if (n <= 8) return launch_few_nm<1, NB, 8>(a, mode, tiles, busy, st);
        if (n <= 12) return launch_few_nm<1, NB, 12>(a, mode, tiles, busy, st);
        if (n <= kMostOperands) return launch_few_nm<1, NB, kMostOperands>(a, mode, tiles, busy, st);
    }
    return fail(MFQ_ERR_UNSUPPORTED, "mx8_scaled: %d columns", a.K);
}
// tiles: at most; busy: about as many have rows
template <int MT>
int launch_few(const MxsArgs &a, int mode, int tiles, int busy, hipStream_t st) {
    return a.glu ? launch_few_nb<MT, 2>(a, mode, tiles, busy, st) : launch_few_nb<MT, 1>(a, mode, tiles, busy, st);
}

// blocks of a launch of tiles of n x m
int64_t tile_blocks(const MxsArgs &a, int n, int m, bool mapped) {
    const int width = a.glu ? a.nrows / 2 : a.nrows;
    const int64_t tiles_m = mapped ? tiles_mapped(a.pairs, a.E, m) : ceil_div(a.M, m);
    return (ceil_div(width, a.glu ? n / 2 : n) * tiles_m + 7) / 8 * 8;
}
// the callers have seen to it that the grid fits (check_tiles)
template <int BN, int BM, int WN, int WM, int R, int MODE>
int launch_tile(const MxsArgs &a, hipStream_t st) {
    using S = Tile8Shape<BN, BM, R>;
    const int64_t blocks = tile_blocks(a, BN, BM, MODE == kMapped);
    static_assert(WN * WM * kTileOut <= R * S::STAGE, "results leave through the ring");
    const size_t lds = S::lds(a.K / kMx8Block);
    MFQ_REQUIRE(lds <= kMaxDynamicLds, MFQ_ERR_UNSUPPORTED, "mx8_scaled: %d columns", a.K);
    auto kern = mx8_tile_kernel<BN, BM, WN, WM, R, MODE>;
    if (int rc = allow_dynamic_lds(reinterpret_cast<const void *>(kern), lds, "mx8_scaled")) return rc;
    hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(MODE == kLinear ? a.splits : 1)), dim3(WN * WM * 64), lds, st, a);
    return check_launch("mx8_scaled (tile)");
}

// Kernel of a call: the few-rows kernel on rows that its blocks quantise (0) or on one or two tiles of 16 quantised rows (1, 2), or a tile of the
// list (3 + its index) with K in `splits` pieces.
struct Mx8Plan { int kind, splits; };
constexpr int kPlanTile = 3;
// Tiles and what a launch of them takes, us: f + max(blocks of K * l, rounds * (blocks of K * c + e)), rounds = blocks a compute unit: l is the
// way of a block of K from memory with the compute unit to itself, c its share with `per_cu` blocks on it, e the end of a block.
// Fitted to 12288 x 4096 and 4096 x 12288 at 40 to 8192 rows: 12288 x 4096 at 256 rows 23.7, 26.4, 27.4, 43.5 us in the order of the list, at 2048
// rows 130, 101, 97.5, 98.2, at 8192 rows 498, 397, 376, 330; 4096 x 12288 at 8192 rows 499, 372, 346, 314 (2.6 PFLOP/s).
struct Mx8Tile { int n, m, threads, per_cu; double f, l, c, e; };
constexpr Mx8Tile kMx8Tile[] = {{128, 64, 256, 3, 2.0, 0.53, 0.325, 0.2}, {128, 128, 256, 2, 4.0, 0.62, 0.47, 1.5}, {256, 128, 512, 1, 4.0, 0.61, 0.867, 3.9},
                                {256, 256, 512, 1, 2.0, 1.05, 1.5, 5.0}};
constexpr int kMx8Tiles = sizeof(kMx8Tile) / sizeof(kMx8Tile[0]), kMaxSplits = 16;

// before anything of a call is launched
int check_tiles(const MxsArgs &a, int index, bool mapped) {
    const Mx8Tile &t = kMx8Tile[index];
    const int64_t blocks = tile_blocks(a, t.n, t.m, mapped);
    MFQ_REQUIRE(grid_fits(blocks, t.threads), MFQ_ERR_UNSUPPORTED, "mx8_scaled: %lld tiles", static_cast<long long>(blocks));
    return MFQ_OK;
}

double tile_us(const Mx8Tile &t, int nrows, int nkb, int M, int splits, int cus) {
    const double blocks = static_cast<double>(ceil_div(nrows, t.n)) * ceil_div(M, t.m) * splits, q = blocks / cus;
    const double whole = static_cast<double>(static_cast<int64_t>(q) + (q > static_cast<int64_t>(q) ? 1 : 0));
    const double rounds = t.per_cu == 1 ? whole : (q + whole) / 2;
    const double kbs = static_cast<double>(ceil_div(nkb, splits));
    double us = kbs * t.l > rounds * (kbs * t.c + t.e) ? kbs * t.l : rounds * (kbs * t.c + t.e);
    // the pieces are written, read by a second launch and written as the result
    if (splits > 1) us += 3.0 + static_cast<double>(M) * nrows * 4 * (2 * splits + 1) / 4.5e6;
    return t.f + us;
}

// Rows that every block of the few-rows kernel quantises itself, which saves a launch: while the blocks' reads of them are little beside the weights.
// In a graph, by the blocks and with the quantiser's launch: 12288 x 4096 at 4 rows 13.5 and 14.6 us, at 8 15.5 and 15.9, at 12 17.0 and 16.8, at 16
// 18.2 and 17.4; 4096 x 4096 at 4 rows 8.4 and 9.8, at 16 10.5 and 11.3; 6144 x 2048 at 4 rows 9.7 and 10.1, at 16 13.4 and 12.8.  So
// from 12 rows on the two differ by 5 % either way, and one call after the other the launch costs 4 us of the host's.
constexpr int kSmallValues = 1 << 16;
bool small_rows(int64_t M, int K) { return M <= 16 && (M <= 4 || M * K <= kSmallValues); }

Mx8Plan plan_linear(int nrows, int K, int M) {
    const int nkb = K / kMx8Block;
    if (M <= 16 && few_fits(K, 1)) return {small_rows(M, K) ? 0 : 1, 1};
    if (M <= 32 && few_fits(K, 2)) return {2, 1};
    static const int forced = tune_env("MFQ_MX8_TILE", 0), forced_split = tune_env("MFQ_MX8_SPLIT", 0);
    const auto whole = [&](int s) { return s <= nkb && (s - 1) * ceil_div(nkb, s) < nkb; };
    const bool tile = forced > 0 && forced <= kMx8Tiles, pieces = forced_split > 0 && forced_split <= kMaxSplits && whole(forced_split);
    const int cus = device_cu_count();
    Mx8Plan best = {-1, 1};
    double least = 0.0;
    for (int t = 0; t < kMx8Tiles; ++t) {
        if (tile && forced != t + 1) continue;
        for (int s = 1; s <= kMaxSplits && s <= nkb; ++s) {
            if (!whole(s) || (pieces && s != forced_split)) continue;
            const double us = tile_us(kMx8Tile[t], nrows, nkb, M, s, cus);
            if (best.kind < 0 || us < least) {
                best = {kPlanTile + t, s};
                least = us;
            }
        }
    }
    return best;
}

int64_t up256(int64_t n) { return (n + 255) & ~static_cast<int64_t>(255); }
size_t quantized_bytes(int K, int64_t M) { return static_cast<size_t>(up256(M * K) + up256(mx8_scale_bytes(M, K))); }

int run_linear_tile(const MxsArgs &a, int index, hipStream_t st) {
    switch (index) {
        case 0: return launch_tile<128, 64, 2, 2, 2, kLinear>(a, st);
        case 1: return launch_tile<128, 128, 2, 2, 2, kLinear>(a, st);
        case 2: return launch_tile<256, 128, 4, 2, 3, kLinear>(a, st);
        default: return launch_tile<256, 256, 2, 4, 2, kLinear>(a, st);
    }
}

// Kernel of a call with a route map, from the pairs an expert has on average: 0 the few-rows kernel, tiles of 16 pairs; 1 + i tile i
// of kMx8Tile.  64 experts of 4096 x 4096, gated, 8 routes: at 16 tokens (2 pairs an expert) 124 us, in tiles of 128 x 64 150 and of 256 x 128 158, at 61
// (8) 243, 201 and 211, at 800 (100) -, 306 and 278; 128 experts of 2048 x 1024 at 61 tokens (4) 48, 46 and 54, at 1500 (94) -, 90 and 97.
// Two tiles of 128 x 128 fit a compute unit, so that one's start and end go beside the other's squares, which counts where K is short: 128 experts
// of 2048 x 768 at 4096 tokens 201 us in tiles of 256 x 128, 185 in these, 1024 columns at 2048 144 and 139, 8 experts of 4096 x 2048 gated
// 128 and 124; 64 of 4096 x 4096 at 2048 432 and 480.  Columns between 2048 and 4096 were not measured, nor cards of other numbers of compute units.
// An expert's last tile is half empty on average, and empty rows are multiplied like others: of tiles of 128 rows a third with 128 pairs an expert, a
// fifth with 256.
int plan_mapped(int64_t pairs, int E, int K) {
    static const int forced = tune_env("MFQ_MX8_EXPERTS", 0);
    if (forced > 0 && forced <= 4 && (forced > 1 || few_fits(K, 1))) return forced - 1;
    const int64_t mean = ceil_div(pairs, E);
    if (mean <= 4 && few_fits(K, 1)) return 0;
    return mean < 96 ? 1 : K <= 2048 ? 2 : 3;
}
int mapped_rows(int plan) { return plan == 0 ? 16 : plan == 1 ? 64 : 128; }

constexpr int kMaxCols = 1 << 17;  // whose scales fit the LDS beside a tile

int check_common(MxsArgs &a, const char *who, const void *values, const void *scales, int64_t rows, int cols, const void *x, int x_dtype, int64_t ldx,
                 const void *x_scales, int64_t x_rows, int glu, int activation, const void *y, int y_dtype) {
    MFQ_REQUIRE(values && scales && x && y, MFQ_ERR_INVALID, "%s: null argument", who);
    MFQ_REQUIRE(x_scales || (x_dtype >= MFQ_X_BF16 && x_dtype <= MFQ_X_F32), MFQ_ERR_INVALID, "%s: x_dtype=%d", who, x_dtype);
    MFQ_REQUIRE(y_dtype >= MFQ_X_BF16 && y_dtype <= MFQ_X_F32, MFQ_ERR_INVALID, "%s: y_dtype=%d", who, y_dtype);
    MFQ_REQUIRE(rows > 0 && cols > 0 && cols % kMx8Block == 0, MFQ_ERR_INVALID, "%s: [%lld, %d], columns must be divisible by 128", who, static_cast<long long>(rows), cols);
    MFQ_REQUIRE(reinterpret_cast<uintptr_t>(values) % 16 == 0, MFQ_ERR_INVALID, "%s: values must be 16-byte aligned", who);
    if (x_scales) {
        MFQ_REQUIRE(reinterpret_cast<uintptr_t>(x) % 16 == 0 && reinterpret_cast<uintptr_t>(x_scales) % 4 == 0, MFQ_ERR_INVALID,
                    "%s: quantised activations must be 16-byte aligned, their scales 4-byte aligned", who);
    } else {
        MFQ_REQUIRE(x_rows == 1 || ldx >= cols, MFQ_ERR_INVALID, "%s: ldx=%lld < %d", who, static_cast<long long>(ldx), cols);
        MFQ_REQUIRE(reinterpret_cast<uintptr_t>(x) % (x_dtype == MFQ_X_F32 ? 4 : 2) == 0, MFQ_ERR_INVALID, "%s: unaligned x", who);
    }
    MFQ_REQUIRE(!glu || (y_dtype != MFQ_X_F32 && (activation == MFQ_GLU_SILU || activation == MFQ_GLU_GELU)), MFQ_ERR_INVALID,
                "%s: a gated product takes a 16-bit type and activation 0 or 1, not y_dtype=%d activation=%d", who, y_dtype, activation);
    MFQ_REQUIRE(reinterpret_cast<uintptr_t>(y) % (y_dtype == MFQ_X_F32 ? 4 : 2) == 0, MFQ_ERR_INVALID, "%s: unaligned y", who);
    MFQ_REQUIRE(cols <= kMaxCols && mx8_scale_bytes(x_rows, cols) < (1ll << 32) - 512, MFQ_ERR_UNSUPPORTED, "%s: %lld rows of %d columns", who,
                static_cast<long long>(x_rows), cols);
    a.wv = static_cast<const uint8_t *>(values);
    a.ws = static_cast<const uint8_t *>(scales);
    a.y = const_cast<void *>(y);
    a.K = cols;
    a.y_dtype = y_dtype;
    a.glu = glu != 0;
    a.gelu = activation == MFQ_GLU_GELU;
    a.splits = 1;
    return MFQ_OK;
}
void take_raw(MxsArgs &a, const void *x, int x_dtype, int64_t ldx, int64_t rows) {
    a.xraw = x;
    a.x_wide = reinterpret_cast<uintptr_t>(x) % 16 == 0 && (rows == 1 || ldx % (x_dtype == MFQ_X_F32 ? 4 : 8) == 0);  // in pieces of 16 bytes
    a.x_dtype = x_dtype;
    a.ldx = ldx;
}

}  // namespace
}  // namespace mfq

using namespace mfq;

extern "C" size_t mfq_hip_mx8_scaled_gemm_workspace_bytes(int nrows, int cols, int M, int x_quantized) {
    if (nrows <= 0 || cols <= 0 || cols % kMx8Block != 0 || M <= 0) return 0;
    const Mx8Plan p = plan_linear(nrows, cols, M);
    size_t n = x_quantized || p.kind == 0 ? 0 : quantized_bytes(cols, M);
    if (p.splits > 1) n += static_cast<size_t>(p.splits) * part_bytes(M, nrows);
    return n;
}

extern "C" int mfq_hip_mx8_scaled_plan(int nrows, int cols, int M, int *splits) {
    if (nrows <= 0 || cols <= 0 || cols % kMx8Block != 0 || cols > kMaxCols || M <= 0) return -1;
    const Mx8Plan p = plan_linear(nrows, cols, M);
    if (splits) *splits = p.splits;
    return p.kind;
}

extern "C" int mfq_hip_mx8_scaled_gemm_rows(const void *values, const void *scales, int rows, int cols, int row0, int nrows, const void *x, int x_dtype,
                                            int64_t ldx, const void *x_scales, int M, int glu, int activation, void *y, int y_dtype, int64_t ldy,
                                            void *workspace, size_t workspace_bytes, mfq_stream_t stream) {
    MxsArgs a = {};
    MFQ_REQUIRE(M > 0, MFQ_ERR_INVALID, "mx8_scaled_gemm_rows: M=%d", M);
    if (int rc = check_common(a, "mx8_scaled_gemm_rows", values, scales, rows, cols, x, x_dtype, ldx, x_scales, M, glu, activation, y, y_dtype)) return rc;
    MFQ_REQUIRE(row0 >= 0 && row0 % kMx8Block == 0 && nrows > 0 && static_cast<int64_t>(row0) + nrows <= rows, MFQ_ERR_INVALID,
                "mx8_scaled_gemm_rows: rows %d + %d of %d (from a multiple of 128)", row0, nrows, rows);
    MFQ_REQUIRE(!glu || nrows % 2 == 0, MFQ_ERR_INVALID, "mx8_scaled_gemm_rows: gate and up in %d rows", nrows);
    MFQ_REQUIRE(M == 1 || ldy >= (glu ? nrows / 2 : nrows), MFQ_ERR_INVALID, "mx8_scaled_gemm_rows: ldy=%lld < %d", static_cast<long long>(ldy), glu ? nrows / 2 : nrows);
    MFQ_REQUIRE(!glu || static_cast<int64_t>(nrows / 2 + 256) * cols < (1ll << 32) - 512, MFQ_ERR_UNSUPPORTED, "mx8_scaled_gemm_rows: gated, %d x %d weights", nrows, cols);
    const hipStream_t st = as_stream(stream);
    a.wv += static_cast<int64_t>(row0) * cols;
    a.row0 = row0;
    a.nrows = nrows;
    a.M = M;
    a.R = 1;
    a.ldy = ldy;
    Mx8Plan p = plan_linear(nrows, cols, M);
    if (p.kind >= kPlanTile)
        if (int rc = check_tiles(a, p.kind - kPlanTile, false)) return rc;
    uint8_t *ws = static_cast<uint8_t *>(workspace);
    size_t used = 0;
    if (x_scales) {
        a.xv = static_cast<const uint8_t *>(x);
        a.xs = static_cast<const uint8_t *>(x_scales);
    } else if (p.kind == 0) {
        take_raw(a, x, x_dtype, ldx, M);
    } else {
        used = quantized_bytes(cols, M);
        MFQ_REQUIRE(ws && workspace_bytes >= used, MFQ_ERR_WORKSPACE, "mx8_scaled_gemm_rows: workspace %zu < %zu", workspace_bytes, used);
        MFQ_REQUIRE(reinterpret_cast<uintptr_t>(ws) % 16 == 0, MFQ_ERR_WORKSPACE, "mx8_scaled_gemm_rows: unaligned workspace");
        uint8_t *xs = ws + up256(static_cast<int64_t>(M) * cols);
        if (int rc = mx8_quantize_launch(x, x_dtype, ldx, M, cols, ws, xs, st)) return rc;
        a.xv = ws;
        a.xs = xs;
    }
    if (p.kind < 2) return launch_few<1>(a, kLinear, 1, 1, st);
    if (p.kind == 2) return launch_few<2>(a, kLinear, 1, 1, st);
    if (p.splits > 1) {
        // a short workspace: K in as many pieces as it has room for
        const size_t left = workspace_bytes > used && ws ? workspace_bytes - used : 0, each = part_bytes(M, nrows);
        const int nkb = cols / kMx8Block;
        if (left / each < static_cast<size_t>(p.splits)) p.splits = static_cast<int>(left / each);
        while (p.splits > 1 && (p.splits - 1) * ceil_div(nkb, p.splits) >= nkb) --p.splits;
        if (p.splits < 2 || reinterpret_cast<uintptr_t>(ws) % 16 != 0) p.splits = 1;
        a.splits = p.splits;
        a.part = reinterpret_cast<float *>(ws + used);
    }
    if (int rc = run_linear_tile(a, p.kind - kPlanTile, st)) return rc;
    return mxs_join_launch(a, st);
}

namespace {
// quantised rows, and the table of the experts' tiles
size_t moe_need(int cols, int64_t x_rows, int64_t pairs, int E, bool x_quantized, size_t *table) {
    const int plan = plan_mapped(pairs, E, cols);
    *table = plan == 0 ? 0 : static_cast<size_t>(tiles_mapped(pairs, E, mapped_rows(plan)) + 1) * 16;
    return (x_quantized || (plan == 0 && small_rows(16, cols)) ? 0 : quantized_bytes(cols, x_rows)) + *table;
}
}  // namespace

extern "C" size_t mfq_hip_mx8_moe_workspace_bytes(int cols, int x_rows, int n_pairs, int E, int mapped, int x_quantized) {
    if (cols <= 0 || cols % kMx8Block != 0 || x_rows <= 0 || n_pairs <= 0 || E <= 0 || !mapped) return 0;
    size_t table;
    return moe_need(cols, x_rows, n_pairs, E, x_quantized != 0, &table);
}

extern "C" int mfq_hip_mx8_moe_plan(int cols, int n_pairs, int E, int mapped) {
    if (cols <= 0 || cols % kMx8Block != 0 || cols > kMaxCols || n_pairs <= 0 || E <= 0) return -1;
    if (!mapped) return few_fits(cols, 1) ? 0 : -1;
    const int plan = plan_mapped(n_pairs, E, cols);
    return plan == 0 ? small_rows(16, cols) ? 0 : 1 : kPlanTile + plan - 1;
}

extern "C" int mfq_hip_mx8_moe_matmul(const void *values, const void *scales, int rows, int cols, int out_per_expert, const int32_t *expert_slot, int E,
                                      const void *x, int x_dtype, int64_t ldx, const void *x_scales, int routed_input, const int32_t *ids, int T, int R,
                                      const int32_t *ids_dst, const int32_t *expert_bounds, int glu, int activation, void *y, int y_dtype, int64_t ldy,
                                      void *workspace, size_t workspace_bytes, mfq_stream_t stream) {
    MxsArgs a = {};
    MFQ_REQUIRE(T > 0 && R > 0 && E > 0 && static_cast<int64_t>(T) * R < (1ll << 31), MFQ_ERR_INVALID, "mx8_moe_matmul: %d tokens, %d routes, %d experts", T, R, E);
    const int x_rows = routed_input ? T * R : T;
    if (int rc = check_common(a, "mx8_moe_matmul", values, scales, rows, cols, x, x_dtype, ldx, x_scales, x_rows, glu, activation, y, y_dtype)) return rc;
    MFQ_REQUIRE(ids && !ids_dst == !expert_bounds, MFQ_ERR_INVALID, "mx8_moe_matmul: ids, and both ids_dst and expert_bounds or neither");
    MFQ_REQUIRE(out_per_expert > 0 && rows % out_per_expert == 0 && (expert_slot || rows / out_per_expert >= E), MFQ_ERR_INVALID,
                "mx8_moe_matmul: %d rows are not %d experts of %d", rows, E, out_per_expert);
    MFQ_REQUIRE(rows == out_per_expert || out_per_expert % kMx8Block == 0, MFQ_ERR_INVALID, "mx8_moe_matmul: experts of %d rows, not of whole blocks of 128", out_per_expert);
    MFQ_REQUIRE(!glu || out_per_expert % 2 == 0, MFQ_ERR_INVALID, "mx8_moe_matmul: gate and up in %d rows", out_per_expert);
    MFQ_REQUIRE(T * R == 1 || ldy >= (glu ? out_per_expert / 2 : out_per_expert), MFQ_ERR_INVALID, "mx8_moe_matmul: ldy=%lld", static_cast<long long>(ldy));
    MFQ_REQUIRE(static_cast<int64_t>(out_per_expert) * cols < (1ll << 31) && static_cast<int64_t>(x_rows) * cols < (1ll << 32) - 512, MFQ_ERR_UNSUPPORTED,
                "mx8_moe_matmul: an expert of %d x %d, %d rows of activations", out_per_expert, cols, x_rows);
    const hipStream_t st = as_stream(stream);
    a.nrows = out_per_expert;
    a.M = x_rows;
    a.E = E;
    a.R = R;
    a.ldy = ldy;
    a.pairs = T * R;
    a.routed = routed_input != 0;
    a.ids = ids;
    a.ids_dst = ids_dst;
    a.bounds = expert_bounds;
    a.slot = expert_slot;
    if (x_scales) {
        a.xv = static_cast<const uint8_t *>(x);
        a.xs = static_cast<const uint8_t *>(x_scales);
    }
    if (!ids_dst) {
        MFQ_REQUIRE(few_fits(cols, 1), MFQ_ERR_UNSUPPORTED, "mx8_moe_matmul: %d columns without a route map", cols);
        if (!x_scales) take_raw(a, x, x_dtype, ldx, x_rows);
        return launch_few<1>(a, kPairs, a.pairs, a.pairs, st);
    }
    size_t table;
    const size_t need = moe_need(cols, x_rows, a.pairs, E, x_scales != nullptr, &table);
    MFQ_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), MFQ_ERR_WORKSPACE, "mx8_moe_matmul: workspace %zu < %zu", workspace_bytes, need);
    MFQ_REQUIRE(need == 0 || reinterpret_cast<uintptr_t>(workspace) % 16 == 0, MFQ_ERR_WORKSPACE, "mx8_moe_matmul: unaligned workspace");
    const int plan = plan_mapped(a.pairs, E, cols);
    if (plan > 0)
        if (int rc = check_tiles(a, plan - 1, true)) return rc;
    uint8_t *ws = static_cast<uint8_t *>(workspace);
    const size_t rows_bytes = need - table;
    const MxTileTable tab = {expert_bounds, expert_slot, E, mapped_rows(plan), table ? reinterpret_cast<i32x4v_t *>(ws + rows_bytes) : nullptr};
    a.table = tab.out;
    if (rows_bytes) {
        a.xv = ws;
        a.xs = ws + up256(static_cast<int64_t>(x_rows) * cols);
    } else if (!x_scales) {
        take_raw(a, x, x_dtype, ldx, x_rows);
    }
    if (rows_bytes || table)
        if (int rc = mx8_quantize_launch(x, x_scales ? MFQ_X_BF16 : x_dtype, ldx, rows_bytes ? x_rows : 0, cols, ws, ws + (rows_bytes ? up256(static_cast<int64_t>(x_rows) * cols) : 0), st, &tab)) return rc;
    if (plan == 0) return launch_few<1>(a, kMapped, static_cast<int>(tiles_mapped(a.pairs, E, 16)), E < a.pairs ? E : a.pairs, st);
    if (plan == 1) return launch_tile<128, 64, 2, 2, 2, kMapped>(a, st);
    return plan == 2 ? launch_tile<128, 128, 2, 2, 2, kMapped>(a, st) : launch_tile<256, 128, 4, 2, 3, kMapped>(a, st);
}
