// Products of two microscaled operands: MXFP4 weights (E2M1 nibbles) against activations quantised to MXFP4 or to MXFP6
// (E2M3), a power of two (E8M0) for every 32 columns of a row of either operand.
//   y[m, n] = sum over blocks b of 32 columns  2^(sw[n, b] - 127) * 2^(sx[m, b] - 127) * sum_k w[n, k] * x[m, k]
// v_mfma_scale_f32_16x16x128_f8f6f4 multiplies 16 rows by 16 rows over 128 columns of codes as they lie in memory and
// applies the eight scale bytes of each row pair itself, so nothing is converted on the way, and its sums are held in fp32.
// (With an FP8 operand it is half as fast, and adds products in groups of eight aligned to the largest, of which it keeps 14 bits:
// measured 5e-6 to 2e-5, 2-norm, from the same sums in 64 bits.  FP4 and FP6 gave exact sums where they fit 24 bits.)
//
// Lanes of that instruction, lane l = (r, g), r = l & 15, g = l >> 4: an operand holds columns 32 g .. 32 g + 31 of row r, four
// registers of FP4 or six of FP6; its scale register holds in the byte that the instruction names the scale of block g of row r; the
// result of lane l is row 4 g + i of the first operand by row r of the second.  A sum does not care which column sits in which slot as
// long as both operands agree: the kernels take 256 columns ("a macro": 8 blocks) for two instructions, the first over blocks
// 0, 2, 4, 6 and the second over blocks 1, 3, 5, 7, so that lane g's two scale bytes are neighbours, one 16-bit read.
//
// Quantised activations are rows of whole macros, zeros behind the last column: 128 bytes of FP4 codes in their order (low nibble =
// even column), or of FP6 the first 16 bytes of each of the eight blocks' 24 and then their last 8 (a block's codes are 192 bits,
// the first code lowest): both parts of a macro are then read from LDS 16 bytes at a time.
//
// Both operands pass through LDS, copied there directly and row by row: a request moves 8 lines of 128 bytes, eight lanes a line
// (lanes of a load in different rows occupy a compute unit's address path four times as long).  The 16-byte pieces of a line
// are turned by a key of the row, mx_key, with which each of the four passes in which the hardware serves a 16-byte read meets
// every bank once; those of FP6's second part lie as in row_order_quarter.
#pragma once
#include "common.hpp"
#include "gemv_common.hpp"
#include "tile_gemm.hpp"
#include "tune.hpp"

namespace mfq {

typedef int i32x8_t __attribute__((ext_vector_type(8)));

constexpr int kMxMacro = 256;  // columns of a macro

// Scales of both operands lie by blocks of 32 rows, and in those by macros: eight bytes a row, 256 a block of rows.  A copy of a tile's
// scales then moves whole lines, where rows one after the other (a line of 128 bytes fetched for every eight) cost as many requests as
// the codes.  Zeros behind the last column.
__host__ __device__ __forceinline__ constexpr int mx_macros(int K) { return K / kMxMacro + (K % kMxMacro != 0); }  // of any K: K + 255 may not fit
__host__ __device__ __forceinline__ constexpr uint32_t mx_scale_at(int64_t row, int nmac) {  // of the row's first macro; the next are 256 further each
    return static_cast<uint32_t>(row >> 5) * static_cast<uint32_t>(nmac) * 256u + static_cast<uint32_t>(row & 31) * 8u;
}
__host__ __device__ __forceinline__ constexpr int64_t mx_scale_bytes(int64_t rows, int K) { return (rows + 31) / 32 * mx_macros(K) * 256; }
// bytes of a macro of quantised activations, and of a row
__host__ __device__ __forceinline__ constexpr int mx_macro_bytes(int kind) { return kind == 4 ? 128 : 192; }
__host__ __device__ __forceinline__ constexpr int64_t mx_row_bytes(int kind, int K) { return static_cast<int64_t>(mx_macros(K)) * mx_macro_bytes(kind); }

// by which the pieces of a line are turned, from its row (0 .. 15): with rows p = 2, 3, 4, 5 (in pairs) in the upper half and 0, 1, 6, 7
// in the lower, for each of which the hardware reads another lane group's piece in the same pass
__device__ __forceinline__ int mx_key(int row) {
    const int p = (row >> 1) & 7;
    return (p & 1) | ((p >> 2) << 1) | ((((p >> 1) ^ (p >> 2)) & 1) << 2);
}

// x: four registers of activations, FP4 codes or the first of FP6; y, z: the rest of those
template <int AK, int SEL>
__device__ __forceinline__ float4_t mx_scale_mfma(u32x4_t w, u32x4_t x, uint32_t y, uint32_t z, float4_t c, uint32_t sw, uint32_t sx) {
    const i32x8_t a = {static_cast<int>(w.x), static_cast<int>(w.y), static_cast<int>(w.z), static_cast<int>(w.w), 0, 0, 0, 0};
    if constexpr (AK == 4) {
        const i32x8_t b = {static_cast<int>(x.x), static_cast<int>(x.y), static_cast<int>(x.z), static_cast<int>(x.w), 0, 0, 0, 0};
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 4, 4, SEL, static_cast<int>(sw), SEL, static_cast<int>(sx));
    } else {
        const i32x8_t b = {static_cast<int>(x.x), static_cast<int>(x.y), static_cast<int>(x.z), static_cast<int>(x.w),
                           static_cast<int>(y), static_cast<int>(z), 0, 0};
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 4, 2, SEL, static_cast<int>(sw), SEL, static_cast<int>(sx));
    }
}

// Copies of a wave straight into LDS, 16 or 4 bytes a lane, lane after lane from `lds` on.  POLICY: as in load_unit_win.
template <int POLICY>
__device__ __forceinline__ void copy16(__amdgpu_buffer_rsrc_t win, uint8_t *lds, uint32_t at, int base) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(win, (lds_void_t)lds, 16, at, base, 0, POLICY);
}
__device__ __forceinline__ void copy4(__amdgpu_buffer_rsrc_t win, uint8_t *lds, uint32_t at, int base) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(win, (lds_void_t)lds, 4, at, base, 0, 0);
}

// ---- the 32 x 32 form, for tiles ------------------------------------------------------------------------------------------------
// v_mfma_scale_f32_32x32x64_f8f6f4: lane l = (r, h), r = l & 31, h = l >> 5, holds columns 32 h .. 32 h + 31 of row r; results 8 j + 4 h + i of
// the first operand by row r of the second in register 4 j + i.  In a loop of nothing else it reaches 6.9 PFLOP/s on random codes
// where the 16 x 16 form reaches 5.0 (one wave a SIMD) to 5.7 (four), 9.8 against 7.3 on zeros: the rest is the clock under load.
template <int AK, int SEL>
__device__ __forceinline__ float16_t mx_scale_mfma32(u32x4_t w, u32x4_t x, uint32_t y, uint32_t z, float16_t c, uint32_t sw, uint32_t sx) {
    const i32x8_t a = {static_cast<int>(w.x), static_cast<int>(w.y), static_cast<int>(w.z), static_cast<int>(w.w), 0, 0, 0, 0};
    if constexpr (AK == 4) {
        const i32x8_t b = {static_cast<int>(x.x), static_cast<int>(x.y), static_cast<int>(x.z), static_cast<int>(x.w), 0, 0, 0, 0};
        return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 4, 4, SEL, static_cast<int>(sw), SEL, static_cast<int>(sx));
    } else {
        const i32x8_t b = {static_cast<int>(x.x), static_cast<int>(x.y), static_cast<int>(x.z), static_cast<int>(x.w),
                           static_cast<int>(y), static_cast<int>(z), 0, 0};
        return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 4, 2, SEL, static_cast<int>(sw), SEL, static_cast<int>(sx));
    }
}

// ---- quantisation of a block of 32 values ---------------------------------------------------------------------------------------
// Scale 2^(e - 2), e the exponent of the block's largest magnitude (both element types reach into the binade of 4), not below
// 2^-127; elements to nearest, ties to even, those beyond the largest element (6, or 7.5) to it.  A block that holds an infinity
// or a NaN takes the NaN scale 255 and codes of zero.
template <int PERM>
__device__ __forceinline__ uint32_t quad_perm(uint32_t v) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), PERM, 0xF, 0xF, true));
}
typedef __bf16 bf16x32_t __attribute__((ext_vector_type(32)));
typedef _Float16 half32_t __attribute__((ext_vector_type(32)));
typedef uint32_t u32x16_t __attribute__((ext_vector_type(16)));
typedef uint32_t u32x6_t __attribute__((ext_vector_type(6)));
typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));

// the scale byte of a block from the bits of its largest magnitude as an fp32
__device__ __forceinline__ uint32_t mx_scale_of(uint32_t most) {
    const int e = static_cast<int>(most >> 23);  // of a subnormal 0: its scale is 2^-127 in any case
    return e == 255 ? 255u : static_cast<uint32_t>(max(e - 2, 0));
}
// The 32 values from x[from] on; VEC: they lie on a 16-byte boundary.  q: 16 bytes of E2M1 or 24 of E2M3.  The conversions divide by the
// power of two in the exponent field of their scale, of which 0 is 2^-127, round to nearest even and saturate.
template <int AK, int XD, bool VEC>
__device__ __forceinline__ void mx_quantize_block(const void *x, int64_t from, u32x6_t &q, uint32_t &byte) {
    q = u32x6_t{};
    if constexpr (XD == MFQ_X_F32) {
        const float *p = static_cast<const float *>(x) + from;
        float16_t v[2];  // even and odd columns: the order of the conversion to E2M3
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float4_t f;
            if constexpr (VEC) f = reinterpret_cast<const float4_t *>(p)[i];
            else f = float4_t{p[4 * i], p[4 * i + 1], p[4 * i + 2], p[4 * i + 3]};
#pragma unroll
            for (int t = 0; t < 4; ++t) v[t & 1][2 * i + (t >> 1)] = f[t];
        }
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < 32; ++i) most = max(most, __float_as_uint(v[i & 1][i >> 1]) & 0x7fffffffu);
        byte = mx_scale_of(most);
        const float scale = __uint_as_float(byte << 23);
        if constexpr (AK == 6) {
            q = __builtin_bit_cast(u32x6_t, __builtin_amdgcn_cvt_scalef32_2xpk16_fp6_f32(v[0], v[1], scale));
        } else {
            static_for<4>([&](auto D) {
                constexpr int d = D.value;
                static_for<4>([&](auto T) {
                    constexpr int t = T.value;
                    q[d] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q[d], v[0][4 * d + t], v[1][4 * d + t], scale, t);
                });
            });
        }
    } else {
        const uint16_t *p = static_cast<const uint16_t *>(x) + from;
        u32x16_t v;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (VEC) {
                const u32x4_t f = reinterpret_cast<const u32x4_t *>(p)[i];
#pragma unroll
                for (int t = 0; t < 4; ++t) v[4 * i + t] = f[t];
            } else {
#pragma unroll
                for (int t = 0; t < 4; ++t) v[4 * i + t] = p[8 * i + 2 * t] | (static_cast<uint32_t>(p[8 * i + 2 * t + 1]) << 16);
            }
        }
        u16x2_t most = {0, 0};
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const uint32_t pair = v[i] & 0x7fff7fffu;
            most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2_t, pair));
        }
        const uint32_t m = max(most.x, most.y);
        // of fp16 the exponent as an fp32 has it, infinities and NaN with theirs
        byte = mx_scale_of(XD == MFQ_X_BF16 ? m << 16 : m >= 0x7c00u ? 0x7f800000u : __float_as_uint(f16_to_f32(static_cast<uint16_t>(m))));
        const float scale = __uint_as_float(byte << 23);
        if constexpr (AK == 6) {
            if constexpr (XD == MFQ_X_F16) q = __builtin_bit_cast(u32x6_t, __builtin_amdgcn_cvt_scalef32_pk32_fp6_f16(__builtin_bit_cast(half32_t, v), scale));
            else q = __builtin_bit_cast(u32x6_t, __builtin_amdgcn_cvt_scalef32_pk32_fp6_bf16(__builtin_bit_cast(bf16x32_t, v), scale));
        } else {
            static_for<4>([&](auto D) {
                constexpr int d = D.value;
                static_for<4>([&](auto T) {
                    constexpr int t = T.value;
                    const uint32_t pair = v[4 * d + t];  // by itself: a bit cast of the element reads the vector's first
                    if constexpr (XD == MFQ_X_F16) q[d] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(q[d], __builtin_bit_cast(half2_t, pair), scale, t);
                    else q[d] = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q[d], __builtin_bit_cast(bf16x2_t, pair), scale, t);
                });
            });
        }
    }
    if (byte == 255u) q = u32x6_t{};
}

// two values rounded to a 16-bit type
__device__ __forceinline__ uint32_t mx_pack16(float lo, float hi, int dtype) {
    if (dtype == MFQ_X_F16) return static_cast<uint32_t>(f32_to_f16_rne(lo)) | (static_cast<uint32_t>(f32_to_f16_rne(hi)) << 16);
    const bf16x2_t v = {static_cast<__bf16>(lo), static_cast<__bf16>(hi)};
    return __builtin_bit_cast(uint32_t, v);
}

// ---- tiles of routed experts ------------------------------------------------------------------------------------------------------
// The pairs bounds[e] .. bounds[e + 1] of expert e are cut into tiles of bm rows.  The table has an entry for each tile, those of an expert side
// by side: place of the expert in the pool, its first tile, its first pair, its number of pairs; in front of them one with their total.
typedef int i32x4v_t __attribute__((ext_vector_type(4)));
struct MxTileTable {
    const int32_t *bounds, *slot;
    int E, bm;
    i32x4v_t *out;
};
// by one block of 256 threads
__device__ __forceinline__ void mx_write_table(const MxTileTable &t, int tid) {
    __shared__ int upto[256];
    int before = 0;
    for (int c = 0; c < t.E; c += 256) {
        const int e = c + tid;
        int place = -1, first = 0, pairs = 0;
        if (e < t.E) {
            place = t.slot ? t.slot[e] : e;
            first = t.bounds[e];
            pairs = place < 0 ? 0 : t.bounds[e + 1] - first;
        }
        const int n = (pairs + t.bm - 1) / t.bm;
        upto[tid] = n;
        __syncthreads();
        for (int o = 1; o < 256; o <<= 1) {
            const int v = tid >= o ? upto[tid - o] : 0;
            __syncthreads();
            upto[tid] += v;
            __syncthreads();
        }
        const int t0 = before + upto[tid] - n;
        for (int i = 0; i < n; ++i) t.out[1 + t0 + i] = i32x4v_t{place, t0, first, pairs};
        before += upto[255];
        __syncthreads();
    }
    if (tid == 0) t.out[0] = i32x4v_t{before, 0, 0, 0};
}

// ---- launches -----------------------------------------------------------------------------------------------------------------
// Quantised rows in memory: values [M, mx_row_bytes], scales of mx_scale_bytes (rows behind the last are left as they are).
// table (optional): written by one more block of the launch; M may be 0 then.
int mx_quantize_launch(int kind, const void *x, int x_dtype, int64_t ldx, int M, int K, uint8_t *values, uint8_t *scales, hipStream_t st,
                       const MxTileTable *table = nullptr);

struct MxsArgs {
    const uint8_t *wv, *ws;  // weights: values from row row0 of the pool on, scales of the whole pool
    const uint8_t *xv, *xs;  // quantised activations
    void *y;
    const int32_t *ids, *ids_dst, *bounds, *slot;  // grouped calls: expert of a pair, pairs by expert, their bounds, place of an expert in the pool
    const i32x4v_t *table;   // and their tiles (mx_write_table)
    const void *xraw;        // activations before quantisation, for the kernel that does it itself
    int64_t ldy, ldx;
    int K, row0, nrows;      // nrows: neurons of the tensor or of an expert
    int M, E, R, pairs, routed;
    int y_dtype, glu, gelu, x_dtype, x_wide;  // glu: gate rows first, nrows / 2 results; x_wide: xraw lies in pieces of 16 bytes
    int splits;
    float *part;             // partial results of a split over K [splits][M][2 part_half(nrows)]
};

}  // namespace mfq
