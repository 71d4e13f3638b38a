// Rows of activations to microscaled codes and back (formats and layout: mx_scaled.hpp).  Bound by memory: 2 or 4 bytes read and 17/32 or
// 25/32 of a byte written a value.
#include "mx_scaled.hpp"

namespace mfq {
namespace {

constexpr int kUnits = 4;  // pieces of eight values a thread of the dequantizer takes, 256 pieces apart: their loads are in flight together

// A thread takes a block of 32 values, whose conversion to E2M3 the hardware does in one instruction and to E2M1 in sixteen, from the
// activations' own type; its codes are 16 bytes (and 8 more of E2M3) next to its neighbour's.  Its loads are 64 or 128 bytes from its
// neighbour's, which takes the address path four or eight times as long as side by side and still is the lesser evil: with a quad of
// threads a block and E2M3 rounded in integers, 2048 x 12288 bf16 to MXFP6 took 23.0 us, against 12.1; fp32 read side by side and turned
// in LDS is no faster (16383 x 4096 to MXFP4: 76 us either way, 4 TB/s).
template <int AK, int XD, bool VEC>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const void *__restrict__ x, int64_t ldx, int M, int K, uint8_t *__restrict__ values,
                                                          uint8_t *__restrict__ scales, MxTileTable table) {
    if (table.out && blockIdx.x == gridDim.x - 1) {
        mx_write_table(table, threadIdx.x);
        return;
    }
    const int nmac = mx_macros(K), per_row = nmac * 8;  // blocks behind the last column are zeros
    const int64_t u = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    const int64_t row = static_cast<int64_t>(M) * per_row < (1ll << 31) ? static_cast<int64_t>(static_cast<uint32_t>(u) / static_cast<uint32_t>(per_row)) : u / per_row;
    if (row >= M) return;
    const int block = static_cast<int>(u - row * per_row);
    const int64_t from = row * ldx + block * 32;
    uint32_t byte = 0;
    u32x6_t q = {};
    if (block < K / 32) mx_quantize_block<AK, XD, VEC>(x, from, q, byte);
    uint8_t *to = values + row * mx_row_bytes(AK, K) + (block >> 3) * mx_macro_bytes(AK);
    *reinterpret_cast<u32x4_t *>(to + (block & 7) * 16) = u32x4_t{q[0], q[1], q[2], q[3]};
    if constexpr (AK == 6) *reinterpret_cast<u32x2_t *>(to + 128 + (block & 7) * 8) = u32x2_t{q[4], q[5]};
    scales[mx_scale_at(row, nmac) + (block >> 3) * 256 + (block & 7)] = static_cast<uint8_t>(byte);
}

// a thread per eight values
template <int AK>
__global__ __launch_bounds__(256) void mx_rows_dequant_kernel(const uint8_t *__restrict__ values, const uint8_t *__restrict__ scales, int M, int K,
                                                              void *__restrict__ out, int out_dtype, int64_t ldo, bool wide) {
    const int per_row = K / 8, nmac = mx_macros(K);
    const int64_t units = static_cast<int64_t>(M) * per_row, xrow = mx_row_bytes(AK, K);
    const int64_t u0 = static_cast<int64_t>(blockIdx.x) * (256 * kUnits) + threadIdx.x;
    u32x2_t q[kUnits];
    uint32_t byte[kUnits];
    int64_t row[kUnits];
    int piece[kUnits];
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
        const int64_t u = min(u0 + 256 * i, units - 1);
        row[i] = units < (1ll << 31) ? static_cast<int64_t>(static_cast<uint32_t>(u) / static_cast<uint32_t>(per_row)) : u / per_row;
        piece[i] = static_cast<int>(u - row[i] * per_row);
        const uint8_t *from = values + row[i] * xrow;
        const uint32_t mac = static_cast<uint32_t>(piece[i]) >> 5, in = piece[i] & 31, j = piece[i] & 3;
        if constexpr (AK == 4) {
            q[i].x = *reinterpret_cast<const uint32_t *>(from + mac * 128u + in * 4u);
        } else {
            // 48 bits from bit 48 j of the block's 192, which lanes 0 to 2 read 8 bytes of
            q[i] = *reinterpret_cast<const u32x2_t *>(from + mac * 192u + (j < 2 ? (in >> 2) * 16u + j * 8u : 128u + (in >> 2) * 8u));
            const uint32_t px = quad_perm<0x90>(q[i].x), py = quad_perm<0x90>(q[i].y);  // of the lane before (lane 3 has read what lane 2 has)
            if (j == 1) q[i] = u32x2_t{(py >> 16) | (q[i].x << 16), q[i].x >> 16};
            else if (j == 2) q[i] = u32x2_t{py, q[i].x};
            else if (j == 3) q[i] = u32x2_t{(px >> 16) | (py << 16), py >> 16};
        }
        byte[i] = scales[mx_scale_at(row[i], nmac) + mac * 256u + (in >> 2)];
    }
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
        if (u0 + 256 * i >= units) continue;
        float v[8];
        if constexpr (AK == 4) {
            const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[i].x, 1.f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[i].x, 1.f, 1);
            const auto c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[i].x, 1.f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[i].x, 1.f, 3);
            v[0] = a[0]; v[1] = a[1]; v[2] = b[0]; v[3] = b[1]; v[4] = c[0]; v[5] = c[1]; v[6] = d[0]; v[7] = d[1];
        } else {
            const uint64_t all = static_cast<uint64_t>(q[i].y) << 32 | q[i].x;
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                // the five magnitude bits, moved to bits 7 .. 11 of an fp16, are the same number scaled by 2^-14
                const uint32_t c = static_cast<uint32_t>(all >> (6 * t)) & 63u;
                v[t] = f16_to_f32(static_cast<uint16_t>((c & 31u) << 7 | (c & 32u) << 10)) * 16384.f;
            }
        }
        // E8M0: 0 is 2^-127, an fp32 subnormal, 255 a NaN
        const float s = byte[i] == 255u ? __uint_as_float(0x7fffffffu) : byte[i] == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(byte[i] << 23);
#pragma unroll
        for (int t = 0; t < 8; ++t) v[t] *= s;
        const int64_t at = row[i] * ldo + piece[i] * 8;
        if (!wide) {
#pragma unroll
            for (int t = 0; t < 8; ++t) store_rounded(out, at + t, v[t], out_dtype);
        } else if (out_dtype == MFQ_X_F32) {
            float *o = static_cast<float *>(out) + at;
            *reinterpret_cast<float4_t *>(o) = float4_t{v[0], v[1], v[2], v[3]};
            *reinterpret_cast<float4_t *>(o + 4) = float4_t{v[4], v[5], v[6], v[7]};
        } else {
            u32x4_t o;
#pragma unroll
            for (int t = 0; t < 4; ++t) o[t] = mx_pack16(v[2 * t], v[2 * t + 1], out_dtype);
            // nontemporal: 2048 x 12288 MXFP6 to bf16 in 14.7 us, 16.7 without; in fp32, where a store covers half a line, it costs (64 -> 105)
            __builtin_nontemporal_store(o, reinterpret_cast<u32x4_t *>(static_cast<uint16_t *>(out) + at));
        }
    }
}

// scales of an MXFP4 payload, rows of K / 32 bytes one after the other, to where the products read them
__global__ __launch_bounds__(256) void mx_lay_scales_kernel(const uint8_t *__restrict__ scales, int64_t rows, int blocks, int nmac, uint8_t *__restrict__ out) {
    const int64_t n = (rows + 31) / 32 * nmac * 32;  // of eight bytes
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t rb = i / (nmac * 32);
        const int in = static_cast<int>(i - rb * (nmac * 32)), mac = in >> 5;
        const int64_t row = rb * 32 + (in & 31);
        uint64_t v = 0;
        if (row < rows)
            for (int b = 0; b < 8; ++b)
                if (mac * 8 + b < blocks) v |= static_cast<uint64_t>(scales[row * blocks + mac * 8 + b]) << (8 * b);
        reinterpret_cast<uint64_t *>(out)[i] = v;
    }
}

template <int AK, int XD>
void launch_quantize(const void *x, int64_t ldx, int M, int K, uint8_t *values, uint8_t *scales, hipStream_t st, const MxTileTable &table) {
    const dim3 grid(static_cast<unsigned>(ceil_div(static_cast<int64_t>(M) * (mx_macros(K) * 8), 256) + (table.out ? 1 : 0)));
    const int64_t per16 = XD == MFQ_X_F32 ? 4 : 8;
    if (reinterpret_cast<uintptr_t>(x) % 16 == 0 && (M == 1 || ldx % per16 == 0))
        hipLaunchKernelGGL((mx_quantize_kernel<AK, XD, true>), grid, dim3(256), 0, st, x, ldx, M, K, values, scales, table);
    else
        hipLaunchKernelGGL((mx_quantize_kernel<AK, XD, false>), grid, dim3(256), 0, st, x, ldx, M, K, values, scales, table);
}

}  // namespace

int mx_quantize_launch(int kind, const void *x, int x_dtype, int64_t ldx, int M, int K, uint8_t *values, uint8_t *scales, hipStream_t st, const MxTileTable *table) {
    const MxTileTable t = table ? *table : MxTileTable{};
    if (kind == 4) {
        if (x_dtype == MFQ_X_F32) launch_quantize<4, MFQ_X_F32>(x, ldx, M, K, values, scales, st, t);
        else if (x_dtype == MFQ_X_F16) launch_quantize<4, MFQ_X_F16>(x, ldx, M, K, values, scales, st, t);
        else launch_quantize<4, MFQ_X_BF16>(x, ldx, M, K, values, scales, st, t);
    } else {
        if (x_dtype == MFQ_X_F32) launch_quantize<6, MFQ_X_F32>(x, ldx, M, K, values, scales, st, t);
        else if (x_dtype == MFQ_X_F16) launch_quantize<6, MFQ_X_F16>(x, ldx, M, K, values, scales, st, t);
        else launch_quantize<6, MFQ_X_BF16>(x, ldx, M, K, values, scales, st, t);
    }
    return check_launch("mx_quantize_rows");
}

}  // namespace mfq

using namespace mfq;

extern "C" int mfq_hip_mx_quantized_row_bytes(int kind, int cols) {
    return (kind == 4 || kind == 6) && cols > 0 && cols % 32 == 0 ? static_cast<int>(mx_row_bytes(kind, cols)) : 0;
}

extern "C" int64_t mfq_hip_mx_scale_bytes(int64_t rows, int cols) { return rows > 0 && cols > 0 && cols % 32 == 0 ? mx_scale_bytes(rows, cols) : 0; }

extern "C" int mfq_hip_mx_quantize_rows(int kind, const void *x, int x_dtype, int64_t ldx, int M, int cols, void *values, void *scales,
                                        mfq_stream_t stream) {
    MFQ_REQUIRE(x && values && scales, MFQ_ERR_INVALID, "mx_quantize_rows: null argument");
    MFQ_REQUIRE(kind == 4 || kind == 6, MFQ_ERR_INVALID, "mx_quantize_rows: kind=%d", kind);
    MFQ_REQUIRE(x_dtype >= MFQ_X_BF16 && x_dtype <= MFQ_X_F32, MFQ_ERR_INVALID, "mx_quantize_rows: x_dtype=%d", x_dtype);
    MFQ_REQUIRE(M > 0 && cols > 0 && cols % 32 == 0, MFQ_ERR_INVALID, "mx_quantize_rows: [%d, %d], columns must be divisible by 32", M, cols);
    MFQ_REQUIRE(M == 1 || ldx >= cols, MFQ_ERR_INVALID, "mx_quantize_rows: ldx=%lld < %d", static_cast<long long>(ldx), cols);
    MFQ_REQUIRE(reinterpret_cast<uintptr_t>(x) % (x_dtype == MFQ_X_F32 ? 4 : 2) == 0 && reinterpret_cast<uintptr_t>(values) % 16 == 0 &&
                reinterpret_cast<uintptr_t>(scales) % 8 == 0, MFQ_ERR_INVALID, "mx_quantize_rows: values must be 16-byte aligned, scales 8-byte aligned");
    MFQ_REQUIRE(mx_scale_bytes(M, cols) < (1ll << 32), MFQ_ERR_UNSUPPORTED, "mx_quantize_rows: %d x %d values", M, cols);
    return mx_quantize_launch(kind, x, x_dtype, ldx, M, cols, static_cast<uint8_t *>(values), static_cast<uint8_t *>(scales), as_stream(stream));
}

extern "C" int mfq_hip_mx_dequant_quantized(int kind, const void *values, const void *scales, int M, int cols, int out_dtype, void *out,
                                            int64_t ldo, mfq_stream_t stream) {
    MFQ_REQUIRE(out && values && scales, MFQ_ERR_INVALID, "mx_dequant_quantized: null argument");
    MFQ_REQUIRE(kind == 4 || kind == 6, MFQ_ERR_INVALID, "mx_dequant_quantized: kind=%d", kind);
    MFQ_REQUIRE(out_dtype >= MFQ_X_BF16 && out_dtype <= MFQ_X_F32, MFQ_ERR_INVALID, "mx_dequant_quantized: out_dtype=%d", out_dtype);
    MFQ_REQUIRE(M > 0 && cols > 0 && cols % 32 == 0, MFQ_ERR_INVALID, "mx_dequant_quantized: [%d, %d], columns must be divisible by 32", M, cols);
    MFQ_REQUIRE(M == 1 || ldo >= cols, MFQ_ERR_INVALID, "mx_dequant_quantized: ldo=%lld < %d", static_cast<long long>(ldo), cols);
    MFQ_REQUIRE(reinterpret_cast<uintptr_t>(values) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % (out_dtype == MFQ_X_F32 ? 4 : 2) == 0, MFQ_ERR_INVALID,
                "mx_dequant_quantized: values must be 16-byte aligned");
    MFQ_REQUIRE(mx_scale_bytes(M, cols) < (1ll << 32), MFQ_ERR_UNSUPPORTED, "mx_dequant_quantized: %d x %d values", M, cols);
    const int64_t units = static_cast<int64_t>(M) * (cols / 8);
    const dim3 grid(static_cast<unsigned>(ceil_div(units, 256 * kUnits)));
    const bool wide = reinterpret_cast<uintptr_t>(out) % 16 == 0 && (M == 1 || ldo % (out_dtype == MFQ_X_F32 ? 4 : 8) == 0);
    auto kern = kind == 4 ? mx_rows_dequant_kernel<4> : mx_rows_dequant_kernel<6>;
    hipLaunchKernelGGL(kern, grid, dim3(256), 0, as_stream(stream), static_cast<const uint8_t *>(values), static_cast<const uint8_t *>(scales), M, cols,
                       out, out_dtype, ldo, wide);
    return check_launch("mx_dequant_quantized");
}

extern "C" int mfq_hip_mx_lay_scales(const void *scales, int64_t rows, int cols, void *out, mfq_stream_t stream) {
    MFQ_REQUIRE(scales && out && reinterpret_cast<uintptr_t>(out) % 8 == 0, MFQ_ERR_INVALID, "mx_lay_scales: null argument, or out not 8-byte aligned");
    MFQ_REQUIRE(rows > 0 && cols > 0 && cols % 32 == 0, MFQ_ERR_INVALID, "mx_lay_scales: [%lld, %d], columns must be divisible by 32",
                static_cast<long long>(rows), cols);
    const int64_t n = ceil_div(mx_scale_bytes(rows, cols) / 8, 256);
    hipLaunchKernelGGL(mx_lay_scales_kernel, dim3(static_cast<unsigned>(n < 65536 ? n : 65536)), dim3(256), 0, as_stream(stream),
                       static_cast<const uint8_t *>(scales), rows, cols / 32, mx_macros(cols), static_cast<uint8_t *>(out));
    return check_launch("mx_lay_scales");
}
