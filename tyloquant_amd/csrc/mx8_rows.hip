// Rows of activations to E4M3 with a scale for every 128 columns and back (mx8.hpp).  Bound by memory: 2 or 4 bytes read and 129/128
// written a value.
#include "mx8.hpp"

namespace mfq {
namespace {

constexpr int kUnits = 4;  // pieces of eight values a thread takes, 256 pieces apart: their loads are in flight together

// the eight values from x[from] on as fp32
template <int XD, bool VEC>
__device__ __forceinline__ void load_eight(const void *x, int64_t from, float (&v)[8]) {
    if constexpr (XD == MFQ_X_F32) {
        const float *p = static_cast<const float *>(x) + from;
        if constexpr (VEC) {
            const float4_t a = reinterpret_cast<const float4_t *>(p)[0], b = reinterpret_cast<const float4_t *>(p)[1];
#pragma unroll
            for (int t = 0; t < 4; ++t) v[t] = a[t], v[4 + t] = b[t];
        } else {
#pragma unroll
            for (int t = 0; t < 8; ++t) v[t] = p[t];
        }
    } else {
        const uint16_t *p = static_cast<const uint16_t *>(x) + from;
        if constexpr (VEC) {
            const u32x4_t a = *reinterpret_cast<const u32x4_t *>(p);
#pragma unroll
            for (int t = 0; t < 8; ++t) v[t] = x_to_f32<XD == MFQ_X_F16>(static_cast<uint16_t>(a[t >> 1] >> (16 * (t & 1))));
        } else {
#pragma unroll
            for (int t = 0; t < 8; ++t) v[t] = x_to_f32<XD == MFQ_X_F16>(p[t]);
        }
    }
}
// the largest of the 16 lanes of a row of the wave
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
    const auto other = [](uint32_t u, auto C) { return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(u), C.value, 0xF, 0xF, true)); };
    v = max(v, other(v, std::integral_constant<int, 0xB1>{}));   // lane ^ 1
    v = max(v, other(v, std::integral_constant<int, 0x4E>{}));   // lane ^ 2
    v = max(v, other(v, std::integral_constant<int, 0x141>{}));  // 7 - lane, of eight
    return max(v, other(v, std::integral_constant<int, 0x140>{}));  // 15 - lane
}

// Eight values a thread, a block of 128 in 16 neighbours: loads and stores of a wave lie side by side.
template <int XD, bool VEC>
__global__ __launch_bounds__(256) void mx8_quantize_kernel(const void *__restrict__ x, int64_t ldx, int M, int K, uint8_t *__restrict__ values,
                                                           uint8_t *__restrict__ scales, MxTileTable table) {
    if (table.out && blockIdx.x == gridDim.x - 1) {
        mx_write_table(table, threadIdx.x);
        return;
    }
    const int per_row = K / 8;
    const int64_t units = static_cast<int64_t>(M) * per_row, u0 = static_cast<int64_t>(blockIdx.x) * (256 * kUnits) + threadIdx.x;
    float v[kUnits][8];
    int64_t row[kUnits];
    int piece[kUnits];
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
        const int64_t u = min(u0 + 256 * i, units - 1);
        row[i] = units < (1ll << 31) ? static_cast<int64_t>(static_cast<uint32_t>(u) / static_cast<uint32_t>(per_row)) : u / per_row;
        piece[i] = static_cast<int>(u - row[i] * per_row);
        load_eight<XD, VEC>(x, row[i] * ldx + piece[i] * 8, v[i]);
    }
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
        uint32_t most = 0;
#pragma unroll
        for (int t = 0; t < 8; ++t) most = max(most, __float_as_uint(v[i][t]) & 0x7fffffffu);
        const uint32_t byte = mx8_scale_of(row_max(most));
        const float scale = __uint_as_float(byte << 23);
        u32x2_t q = {mx8_codes(v[i][0], v[i][1], v[i][2], v[i][3], scale), mx8_codes(v[i][4], v[i][5], v[i][6], v[i][7], scale)};
        if (byte == 255u) q = u32x2_t{0u, 0u};
        if (u0 + 256 * i >= units) continue;  // whole blocks of 16 lanes: the units of a row are
        *reinterpret_cast<u32x2_t *>(values + row[i] * K + piece[i] * 8) = q;
        if ((piece[i] & 15) == 0) scales[mx8_scale_at(M, row[i], piece[i] >> 4)] = static_cast<uint8_t>(byte);
    }
}

__global__ __launch_bounds__(256) void mx8_dequant_kernel(const uint8_t *__restrict__ values, const uint8_t *__restrict__ scales, int M, int K,
                                                          void *__restrict__ out, int out_dtype, int64_t ldo, bool wide) {
    const int per_row = K / 8;
    const int64_t units = static_cast<int64_t>(M) * per_row, u0 = static_cast<int64_t>(blockIdx.x) * (256 * kUnits) + threadIdx.x;
    u32x2_t q[kUnits];
    uint32_t byte[kUnits];
    int64_t row[kUnits];
    int piece[kUnits];
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
        const int64_t u = min(u0 + 256 * i, units - 1);
        row[i] = units < (1ll << 31) ? static_cast<int64_t>(static_cast<uint32_t>(u) / static_cast<uint32_t>(per_row)) : u / per_row;
        piece[i] = static_cast<int>(u - row[i] * per_row);
        q[i] = *reinterpret_cast<const u32x2_t *>(values + row[i] * K + piece[i] * 8);
        byte[i] = scales[mx8_scale_at(M, row[i], piece[i] >> 4)];
    }
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
        if (u0 + 256 * i >= units) continue;
        // E8M0: 0 is 2^-127, an fp32 subnormal, 255 a NaN
        const float s = byte[i] == 255u ? __uint_as_float(0x7fffffffu) : byte[i] == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(byte[i] << 23);
        float v[8];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(q[i][t], 1.f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(q[i][t], 1.f, true);
            v[4 * t] = a[0] * s; v[4 * t + 1] = a[1] * s; v[4 * t + 2] = b[0] * s; v[4 * t + 3] = b[1] * s;
        }
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
            __builtin_nontemporal_store(o, reinterpret_cast<u32x4_t *>(static_cast<uint16_t *>(out) + at));
        }
    }
}

template <int XD>
void launch_quantize(const void *x, int64_t ldx, int M, int K, uint8_t *values, uint8_t *scales, hipStream_t st, const MxTileTable &table) {
    const dim3 grid(static_cast<unsigned>(ceil_div(static_cast<int64_t>(M) * (K / 8), 256 * kUnits) + (table.out ? 1 : 0)));
    if (reinterpret_cast<uintptr_t>(x) % 16 == 0 && (M == 1 || ldx % (XD == MFQ_X_F32 ? 4 : 8) == 0))
        hipLaunchKernelGGL((mx8_quantize_kernel<XD, true>), grid, dim3(256), 0, st, x, ldx, M, K, values, scales, table);
    else
        hipLaunchKernelGGL((mx8_quantize_kernel<XD, false>), grid, dim3(256), 0, st, x, ldx, M, K, values, scales, table);
}

// blocks of 256 threads, and one more with a table
int check_values(const char *who, int M, int cols) {
    MFQ_REQUIRE(grid_fits(ceil_div(static_cast<int64_t>(M) * (cols / 8), 256 * kUnits) + 1, 256), MFQ_ERR_UNSUPPORTED, "%s: %d x %d values", who, M, cols);
    return MFQ_OK;
}
int check_shape(const char *who, int M, int cols) {
    MFQ_REQUIRE(M > 0 && cols > 0 && cols % kMx8Block == 0, MFQ_ERR_INVALID, "%s: [%d, %d], columns must be divisible by 128", who, M, cols);
    return check_values(who, M, cols);
}

}  // namespace

int mx8_quantize_launch(const void *x, int x_dtype, int64_t ldx, int M, int K, uint8_t *values, uint8_t *scales, hipStream_t st, const MxTileTable *table) {
    if (int rc = check_values("mx8_quantize_rows", M, K)) return rc;
    const MxTileTable t = table ? *table : MxTileTable{};
    if (x_dtype == MFQ_X_F32) launch_quantize<MFQ_X_F32>(x, ldx, M, K, values, scales, st, t);
    else if (x_dtype == MFQ_X_F16) launch_quantize<MFQ_X_F16>(x, ldx, M, K, values, scales, st, t);
    else launch_quantize<MFQ_X_BF16>(x, ldx, M, K, values, scales, st, t);
    return check_launch("mx8_quantize_rows");
}

}  // namespace mfq

using namespace mfq;

extern "C" int64_t mfq_hip_mx8_scale_bytes(int64_t rows, int cols) { return rows > 0 && cols > 0 && cols % kMx8Block == 0 ? mx8_scale_bytes(rows, cols) : 0; }

extern "C" int mfq_hip_mx8_quantize_rows(const void *x, int x_dtype, int64_t ldx, int M, int cols, void *values, void *scales, mfq_stream_t stream) {
    MFQ_REQUIRE(x && values && scales, MFQ_ERR_INVALID, "mx8_quantize_rows: null argument");
    MFQ_REQUIRE(x_dtype >= MFQ_X_BF16 && x_dtype <= MFQ_X_F32, MFQ_ERR_INVALID, "mx8_quantize_rows: x_dtype=%d", x_dtype);
    if (int rc = check_shape("mx8_quantize_rows", M, cols)) return rc;
    MFQ_REQUIRE(M == 1 || ldx >= cols, MFQ_ERR_INVALID, "mx8_quantize_rows: ldx=%lld < %d", static_cast<long long>(ldx), cols);
    MFQ_REQUIRE(reinterpret_cast<uintptr_t>(x) % (x_dtype == MFQ_X_F32 ? 4 : 2) == 0 && reinterpret_cast<uintptr_t>(values) % 16 == 0, MFQ_ERR_INVALID,
                "mx8_quantize_rows: values must be 16-byte aligned");
    return mx8_quantize_launch(x, x_dtype, ldx, M, cols, static_cast<uint8_t *>(values), static_cast<uint8_t *>(scales), as_stream(stream));
}

extern "C" int mfq_hip_mx8_dequant_quantized(const void *values, const void *scales, int M, int cols, int out_dtype, void *out, int64_t ldo, mfq_stream_t stream) {
    MFQ_REQUIRE(out && values && scales, MFQ_ERR_INVALID, "mx8_dequant_quantized: null argument");
    MFQ_REQUIRE(out_dtype >= MFQ_X_BF16 && out_dtype <= MFQ_X_F32, MFQ_ERR_INVALID, "mx8_dequant_quantized: out_dtype=%d", out_dtype);
    if (int rc = check_shape("mx8_dequant_quantized", M, cols)) return rc;
    MFQ_REQUIRE(M == 1 || ldo >= cols, MFQ_ERR_INVALID, "mx8_dequant_quantized: ldo=%lld < %d", static_cast<long long>(ldo), cols);
    const int size = out_dtype == MFQ_X_F32 ? 4 : 2;
    MFQ_REQUIRE(reinterpret_cast<uintptr_t>(values) % 8 == 0 && reinterpret_cast<uintptr_t>(out) % size == 0, MFQ_ERR_INVALID,
                "mx8_dequant_quantized: values must be 8-byte aligned");
    const bool wide = reinterpret_cast<uintptr_t>(out) % 16 == 0 && (M == 1 || ldo * size % 16 == 0);
    const dim3 grid(static_cast<unsigned>(ceil_div(static_cast<int64_t>(M) * (cols / 8), 256 * kUnits)));
    hipLaunchKernelGGL(mx8_dequant_kernel, grid, dim3(256), 0, as_stream(stream), static_cast<const uint8_t *>(values), static_cast<const uint8_t *>(scales), M,
                       cols, out, out_dtype, ldo, wide);
    return check_launch("mx8_dequant_quantized");
}
