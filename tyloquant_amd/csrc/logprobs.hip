// Scores of an answer from rows of logits z[0 .. V): of a given token its log probability and rank, the entropy of the row, and the
// most probable tokens with theirs.
//   m = max z, s = sum e^(z - m), t = sum (z - m) e^(z - m):   log p_i = (z_i - m) - log s,   entropy = log s - t / s
// One pass over the logits.  A thread keeps m, s and t of what it has seen, rescaled once for every 32 values (a tile of its block is 8192 of
// them); threads, waves, blocks and the pieces of a row are joined by the same rule.  A piece of -infinity alone has s = 0; a row of
// nothing else, or with +infinity or a NaN in it, gives NaN as its softmax does.
//
// The most probable: each wave keeps its best so far as whole numbers that order logits, of equal ones the lower token first, and looks at
// single values of a tile only where the tile's largest reaches the last of them, which is rare after the first tiles.  The first bar is
// the top-th largest of the 64 lanes' maxima in the first tile.  The numbers decide, not the waves: results do not depend on
// the order in which waves run.
//
// Bound by memory where there are many rows, by its two launches where there is one.  One block a row where there are rows enough; a
// row of fewer is cut into pieces of whole tiles, joined by a second launch.
#include <math.h>

#include "common.hpp"
#include "gemv_common.hpp"

namespace mfq {
namespace {

constexpr int kMaxTop = 64;                   // as many as a wave has lanes
constexpr int kVpt = 32, kTile = 256 * kVpt;  // values of a thread and of a block that are in flight together

struct LogprobArgs {
    const void *logits;
    int64_t ldl;
    int V, top, parts, per;    // parts of a row, of `per` tiles each
    const int64_t *tokens;
    float *logprob, *entropy, *top_logprobs;
    int64_t *rank, *top_ids;
    float4_t *sums;            // [rows][parts]: m, s, t and, as an int, how many logits are above the given one
    uint64_t *keys;            // [rows][parts][top]
};

// Whole numbers in the order of the logits: -0 and +0 alike, NaN below all others; 0 is no logit at all.
__device__ __forceinline__ uint32_t order_of(float v) {
    const uint32_t b = __float_as_uint(v + 0.f);
    return v != v ? 1u : b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ uint64_t key_of(float v, uint32_t i) { return static_cast<uint64_t>(order_of(v)) << 32 | (0xffffffffu - i); }
__device__ __forceinline__ int token_of(uint64_t key) { return static_cast<int>(0xffffffffu - static_cast<uint32_t>(key)); }
__device__ __forceinline__ float logit_of(uint64_t key) {
    const uint32_t o = static_cast<uint32_t>(key >> 32);
    return o == 1u ? __uint_as_float(0x7fffffffu) : __uint_as_float(o ^ (o >> 31 ? 0x80000000u : 0xffffffffu));
}

// e^z of z <= 0, which becomes at least -200 (where e^z is zero): the base-2 exponential of the rounded product, and what that has
// lost, to first order.  A NaN stays one.
__device__ __forceinline__ float exp_below(float &z) {
    constexpr float kL = 1.44269502162933349609375f, kRest = 1.92596299e-8f, kLn2 = 0.693147180559945309f;
    z = z < -200.f ? -200.f : z;
    const float p = z * kL, lost = fmaf(z, kRest, fmaf(z, kL, -p)), e = __builtin_amdgcn_exp2f(p);
    return fmaf(e * lost, kLn2, e);
}

struct Sums {
    float m, s, t;
    int above;
};
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.f : m; }
__device__ __forceinline__ Sums join(const Sums &a, const Sums &b) {
    Sums r;
    r.m = fmaxf(a.m, b.m);
    float da = a.m - base_of(r.m), db = b.m - base_of(r.m);
    const float ea = exp_below(da), eb = exp_below(db);
    r.s = ea * a.s + eb * b.s;
    r.t = ea * fmaf(da, a.s, a.t) + eb * fmaf(db, b.s, b.t);
    r.above = a.above + b.above;
    return r;
}
__device__ __forceinline__ Sums join_wave(Sums a) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) a = join(a, Sums{__shfl_xor(a.m, o, 64), __shfl_xor(a.s, o, 64), __shfl_xor(a.t, o, 64), __shfl_xor(a.above, o, 64)});
    return a;
}

// The largest `top` of the n <= 128 numbers in buf to its front, in order, by one wave; no two are equal but zeros, which go.  Returns
// how many there are then.
__device__ __forceinline__ int keep_best(uint64_t *buf, int n, int top, int lane) {
    wave_sync();
    const uint64_t a = lane < n ? buf[lane] : 0, b = lane + 64 < n ? buf[lane + 64] : 0;
    int ra = 0, rb = 0;
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
        const uint64_t o = buf[i];
        ra += o > a;
        rb += o > b;
    }
    const bool ka = a && ra < top, kb = b && rb < top;
    wave_sync();
    if (ka) buf[ra] = a;
    if (kb) buf[rb] = b;
    wave_sync();
    return __popcll(__ballot(ka)) + __popcll(__ballot(kb));
}

template <int DT>
__device__ __forceinline__ float logit_at(const void *p, int64_t i) {
    if constexpr (DT == MFQ_X_F32) return static_cast<const float *>(p)[i];
    else return x_to_f32<DT == MFQ_X_F16>(static_cast<const uint16_t *>(p)[i]);
}

// what is written of a whole row; `given`: the token's logit
__device__ __forceinline__ void put_scores(const LogprobArgs &a, int64_t row, const Sums &s, bool any, float given) {
    const float log_s = logf(s.s);
    a.entropy[row] = log_s - s.t / s.s;
    a.logprob[row] = any ? (given - s.m) - log_s : 0.f;
    a.rank[row] = any ? s.above + 1 : 0;
}
__device__ __forceinline__ void put_best(const LogprobArgs &a, int64_t row, const Sums &s, int i, uint64_t key) {
    a.top_ids[row * a.top + i] = token_of(key);
    a.top_logprobs[row * a.top + i] = (logit_of(key) - s.m) - logf(s.s);
}

template <int DT, bool VEC>
__global__ __launch_bounds__(256) void logprobs_kernel(LogprobArgs a) {
    constexpr int W = VEC ? (DT == MFQ_X_F32 ? 4 : 8) : 1, N = kVpt / W;  // values of a load, loads of a tile
    __shared__ uint64_t s_buf[4][128];
    __shared__ Sums s_sums[4];
    __shared__ int s_count[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row = blockIdx.x / a.parts;
    const int part = static_cast<int>(blockIdx.x - row * a.parts);
    const void *z = static_cast<const uint8_t *>(a.logits) + row * a.ldl * (DT == MFQ_X_F32 ? 4 : 2);
    const int64_t token = a.tokens[row];
    const bool any = token >= 0 && token < a.V;
    const float given = any ? logit_at<DT>(z, token) : INFINITY;

    Sums my = {-INFINITY, 0.f, 0.f, 0};
    uint64_t bar = 0;     // of the wave: smaller numbers are not among its best
    float bar_value = -INFINITY;
    int count = 0;        // of the wave's buffer
    uint64_t *buf = s_buf[wave];
    const int64_t first = static_cast<int64_t>(part) * a.per * kTile, end = min(first + static_cast<int64_t>(a.per) * kTile, static_cast<int64_t>(a.V));
    for (int64_t at = first; at < end; at += kTile) {
        float v[kVpt];
        const bool whole = at + kTile <= end;
        // value i * W + w of the thread is that of token at + (i * 256 + tid) * W + w
        if (whole) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int64_t k = at + (i * 256 + tid) * W;
                if constexpr (!VEC) {
                    v[i] = logit_at<DT>(z, k);
                } else if constexpr (DT == MFQ_X_F32) {
                    const float4_t f = __builtin_nontemporal_load(reinterpret_cast<const float4_t *>(static_cast<const float *>(z) + k));
#pragma unroll
                    for (int w = 0; w < 4; ++w) v[4 * i + w] = f[w];
                } else {
                    const u32x4_t f = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t *>(static_cast<const uint16_t *>(z) + k));
#pragma unroll
                    for (int w = 0; w < 8; ++w) v[8 * i + w] = x_to_f32<DT == MFQ_X_F16>(static_cast<uint16_t>(f[w >> 1] >> (16 * (w & 1))));
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < kVpt; ++i) {
                const int64_t k = at + ((i / W) * 256 + tid) * W + i % W;
                v[i] = k < end ? logit_at<DT>(z, k) : -INFINITY;
            }
        }
        float most = v[0];
#pragma unroll
        for (int i = 1; i < kVpt; ++i) most = fmaxf(most, v[i]);
        {
            const float m = fmaxf(my.m, most), base = base_of(m);
            float d = my.m - base;
            const float c = exp_below(d);
            my.t = c * fmaf(d, my.s, my.t);
            my.s *= c;
            my.m = m;
#pragma unroll
            for (int i = 0; i < kVpt; ++i) {
                float y = v[i] - base;
                const float e = exp_below(y);
                my.s += e;
                my.t = fmaf(y, e, my.t);
                my.above += v[i] > given;
            }
        }
        if (a.top == 0) continue;
        const auto index = [&](int i) { return static_cast<uint32_t>(at + ((i / W) * 256 + tid) * W + i % W); };
        const auto number = [&](int i) { return whole || index(i) < end ? key_of(v[i], index(i)) : 0; };
        if (at == first) {
            uint64_t mine = 0;
#pragma unroll
            for (int i = 0; i < kVpt; ++i) {
                const uint64_t k = number(i);
                mine = k > mine ? k : mine;
            }
            buf[lane] = mine;
            if (keep_best(buf, 64, a.top, lane) == a.top) {
                bar = buf[a.top - 1];
                bar_value = logit_of(bar);
            }
            wave_sync();
        }
        // a NaN is no reason to look, and is found where one is needed: while the bar is as low
        if (!__ballot(!(most < bar_value))) continue;
#pragma unroll
        for (int i = 0; i < kVpt; ++i) {
            const bool reach = !(v[i] < bar_value);
            if (!__ballot(reach)) continue;
            const uint64_t k = reach ? number(i) : 0;
            const bool take = k && k >= bar;
            const uint64_t takers = __ballot(take);
            if (!takers) continue;
            if (take) buf[count + __popcll(takers & ((1ull << lane) - 1))] = k;
            count += __popcll(takers);
            if (count > 64) {
                count = keep_best(buf, count, a.top, lane);
                if (count == a.top) {
                    bar = buf[a.top - 1];
                    bar_value = logit_of(bar);
                }
                wave_sync();
            }
        }
    }
    if (a.top) {
        count = keep_best(buf, count, a.top, lane);
        if (lane == 0) s_count[wave] = count;
    }
    my = join_wave(my);
    if (lane == 0) s_sums[wave] = my;
    __syncthreads();
    const Sums all = join(join(s_sums[0], s_sums[1]), join(s_sums[2], s_sums[3]));
    if (tid == 0) {
        if (a.parts == 1) put_scores(a, row, all, any, given);
        else a.sums[blockIdx.x] = float4_t{all.m, all.s, all.t, __int_as_float(all.above)};
    }
    // the waves' lists to one; a part shorter than `top` leaves zeros behind its own
    const int w = tid >> 6, i = tid & 63;
    const int kept = a.top ? s_count[0] + s_count[1] + s_count[2] + s_count[3] : 0;
    if (i < a.top && i < s_count[w]) {
        const uint64_t k = s_buf[w][i];
        int r = i;
        for (int o = 0; o < 4; ++o)
            if (o != w)
                for (int j = 0; j < s_count[o]; ++j) r += s_buf[o][j] > k;
        if (r < a.top) {
            if (a.parts == 1) put_best(a, row, all, r, k);
            else a.keys[static_cast<int64_t>(blockIdx.x) * a.top + r] = k;
        }
    }
    if (a.parts > 1 && tid >= kept && tid < a.top) a.keys[static_cast<int64_t>(blockIdx.x) * a.top + tid] = 0;
}

// the parts of a row, a block each
template <int DT>
__global__ __launch_bounds__(256) void logprobs_join_kernel(LogprobArgs a) {
    extern __shared__ uint64_t s_key[];
    __shared__ Sums s_all;
    const int tid = threadIdx.x, lane = tid & 63;
    const int64_t row = blockIdx.x;
    const int n = a.parts * a.top;
    for (int i = tid; i < n; i += 256) s_key[i] = a.keys[row * n + i];
    if (tid < 64) {
        Sums my = {-INFINITY, 0.f, 0.f, 0};
        for (int p = lane; p < a.parts; p += 64) {
            const float4_t v = a.sums[row * a.parts + p];
            my = join(my, Sums{v.x, v.y, v.z, __float_as_int(v.w)});
        }
        my = join_wave(my);
        if (lane == 0) s_all = my;
    }
    __syncthreads();
    const Sums all = s_all;
    if (tid == 0) {
        const int64_t token = a.tokens[row];
        const bool any = token >= 0 && token < a.V;
        const void *z = static_cast<const uint8_t *>(a.logits) + row * a.ldl * (DT == MFQ_X_F32 ? 4 : 2);
        put_scores(a, row, all, any, any ? logit_at<DT>(z, token) : 0.f);
    }
    for (int i = tid; i < n; i += 256) {
        const uint64_t k = s_key[i];
        if (!k) continue;
        int r = 0;
        for (int j = 0; j < n && r < a.top; ++j) r += s_key[j] > k;
        if (r < a.top) put_best(a, row, all, r, k);
    }
}

// Pieces of a row: enough blocks of 256 threads for four a compute unit, of whole tiles, none empty; their lists fit the joining block's LDS.
constexpr int kMaxLists = 4096;
int parts_of(int M, int V, int top, int *per) {
    const int64_t tiles = ceil_div(V, kTile), room = kMaxLists / (top > 0 ? top : 1);
    int64_t want = ceil_div(static_cast<int64_t>(4) * device_cu_count(), M);
    if (want > room) want = room;
    *per = static_cast<int>(ceil_div(tiles, want < tiles ? want : tiles));
    return static_cast<int>(ceil_div(tiles, *per));
}
size_t workspace_of(int M, int parts, int top) { return parts == 1 ? 0 : static_cast<size_t>(M) * parts * (sizeof(float4_t) + static_cast<size_t>(top) * 8); }

template <int DT>
int launch(const LogprobArgs &a, int M, bool wide, hipStream_t st) {
    const dim3 grid(static_cast<unsigned>(static_cast<int64_t>(M) * a.parts));
    if (wide) hipLaunchKernelGGL((logprobs_kernel<DT, true>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((logprobs_kernel<DT, false>), grid, dim3(256), 0, st, a);
    if (int rc = check_launch("token_logprobs")) return rc;
    if (a.parts == 1) return MFQ_OK;
    const size_t lds = static_cast<size_t>(a.parts) * a.top * 8;
    hipLaunchKernelGGL((logprobs_join_kernel<DT>), dim3(static_cast<unsigned>(M)), dim3(256), lds, st, a);
    return check_launch("token_logprobs (join)");
}

}  // namespace
}  // namespace mfq

using namespace mfq;

extern "C" size_t mfq_hip_token_logprobs_workspace_bytes(int M, int V, int top) {
    if (M < 1 || V < 1 || top < 0 || top > kMaxTop || top > V) return 0;
    int per;
    return workspace_of(M, parts_of(M, V, top, &per), top);
}

extern "C" int mfq_hip_token_logprobs(const void *logits, int dtype, int64_t ldl, int M, int V, const int64_t *tokens, int top, float *logprob, int64_t *rank,
                                      float *entropy, int64_t *top_ids, float *top_logprobs, void *workspace, size_t workspace_bytes, mfq_stream_t stream) {
    MFQ_REQUIRE(logits && tokens && logprob && rank && entropy, MFQ_ERR_INVALID, "token_logprobs: null argument");
    MFQ_REQUIRE(dtype >= MFQ_X_BF16 && dtype <= MFQ_X_F32, MFQ_ERR_INVALID, "token_logprobs: dtype=%d", dtype);
    MFQ_REQUIRE(M >= 1 && V >= 1 && (M == 1 || ldl >= V), MFQ_ERR_INVALID, "token_logprobs: [%d, %d] logits, ldl=%lld", M, V, static_cast<long long>(ldl));
    MFQ_REQUIRE(top >= 0 && top <= kMaxTop && top <= V, MFQ_ERR_INVALID, "token_logprobs: %d alternatives of %d tokens (at most %d)", top, V, kMaxTop);
    MFQ_REQUIRE(top == 0 || (top_ids && top_logprobs), MFQ_ERR_INVALID, "token_logprobs: null top_ids or top_logprobs");
    const int size = dtype == MFQ_X_F32 ? 4 : 2;
    MFQ_REQUIRE(reinterpret_cast<uintptr_t>(logits) % size == 0, MFQ_ERR_INVALID, "token_logprobs: unaligned logits");
    LogprobArgs a = {logits, ldl, V, top, 1, 0, tokens, logprob, entropy, top_logprobs, rank, top_ids, nullptr, nullptr};
    a.parts = parts_of(M, V, top, &a.per);
    MFQ_REQUIRE(static_cast<int64_t>(M) * a.parts < (1ll << 31), MFQ_ERR_UNSUPPORTED, "token_logprobs: %d rows", M);
    if (a.parts > 1) {
        const size_t need = workspace_of(M, a.parts, top);
        MFQ_REQUIRE(workspace && workspace_bytes >= need, MFQ_ERR_WORKSPACE, "token_logprobs: workspace %zu < %zu", workspace_bytes, need);
        MFQ_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, MFQ_ERR_WORKSPACE, "token_logprobs: unaligned workspace");
        a.sums = static_cast<float4_t *>(workspace);
        a.keys = reinterpret_cast<uint64_t *>(a.sums + static_cast<size_t>(M) * a.parts);
    }
    const bool wide = reinterpret_cast<uintptr_t>(logits) % 16 == 0 && (M == 1 || ldl * size % 16 == 0);
    const hipStream_t st = as_stream(stream);
    if (dtype == MFQ_X_F32) return launch<MFQ_X_F32>(a, M, wide, st);
    return dtype == MFQ_X_F16 ? launch<MFQ_X_F16>(a, M, wide, st) : launch<MFQ_X_BF16>(a, M, wide, st);
}
