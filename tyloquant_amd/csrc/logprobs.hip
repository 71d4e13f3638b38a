// Scores of an answer from rows of logits z[0 .. V): of a given token its log probability and rank, the entropy of the row, and the
// most probable tokens with theirs.
//   m = max z, p_i = (z_i - m) log2 e, s = sum 2^p_i, t = sum p_i 2^p_i:   log softmax_i = (z_i - m) - log s,   entropy = log s - ln 2 t / s
// One pass over the logits.  A thread keeps m, s and t of what it has seen, rescaled once for every 8 or 16 values (a tile of its block is 2048
// or 4096 of them), which are added by a tree and then to the rest by a compensated sum; threads, waves, blocks and the pieces of a row
// are joined by the same rule.  A piece of -infinity alone has s = 0; a row of nothing else, or with +infinity or a NaN in it, gives NaN
// as its softmax does.
//
// The most probable: each wave keeps its best so far as whole numbers that order logits, of equal ones the lower token first, and looks at
// single values of a tile only where the tile's largest reaches the last of them, which is rare after the first tiles of logits that differ.
// The first bar is the top-th largest of the 64 lanes' maxima in the first tile.  The numbers decide, not the waves: results do not
// depend on the order in which waves run.  Where a mask leaves fewer than `top` tokens in a wave's first tiles the bar is the mask's own value, which
// every tile reaches: each of its values is read again then, and so it is in long runs of equal logits at the bar.  2048 rows of 151936,
// 5 alternatives: 787 us with 50 tokens left, 214 unmasked, 192 either way without alternatives.
//
// A token's rank counts the tokens of larger z - m in fp32, the difference that log probabilities are formed of: logits so close together
// that it does not tell them apart are as probable as one another and have one rank, as equal ones have (the alternatives are in the order of
// the logits, so number i of them has rank i at most, from 1 on).  m is known at the end of the row only, so what is counted on the way is
// logits above the given one, and the few that lie within 2^-17 above it are kept: of those the equal ones are taken off again.  Rows
// whose m is more than 64 above the given logit (where fp32 differences are farther apart), or with more of such neighbours than are kept,
// are read once more.
//
// Bound by memory where there are many rows, by its two launches where there is one.  One block a row where there are rows enough; a
// row of fewer is cut into pieces of whole tiles, joined by a second launch.
#include <math.h>

#include "common.hpp"
#include "gemv_common.hpp"

namespace mfq {
namespace {

constexpr int kMaxTop = 64;                  // as many as a wave has lanes
constexpr float kNear = 0x1p-17f, kNearRange = 64.f;
constexpr int kNeighbours = 63;              // of a part of a row

struct LogprobArgs {
    const void *logits;
    int64_t ldl;
    int V, top, parts, per;    // parts of a row, of `per` tiles each
    const int64_t *tokens;
    float *logprob, *entropy, *top_logprobs;
    int64_t *rank, *top_ids;
    float4_t *sums;            // [rows][parts]: m, s, t and, as an int, how many logits are above the given one
    float *near;               // [rows][parts][1 + kNeighbours]: how many are close above it, as an int, and those
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

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.693147180559945309417f;
struct Sums {
    float m, s, t;
    int above;
};
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.f : m; }
__device__ __forceinline__ float exponent(float z, float base) { return (z - base) * kLog2e; }
// p 2^p has no value where p is -infinity: there 2^p is 0, as it is at -300
__device__ __forceinline__ float bounded(float p) { return fmaxf(p, -300.f); }
__device__ __forceinline__ Sums join(const Sums &a, const Sums &b) {
    Sums r;
    r.m = fmaxf(a.m, b.m);
    const float base = base_of(r.m), da = bounded(exponent(a.m, base)), db = bounded(exponent(b.m, base));
    // a piece of nothing (m = -infinity) has s = t = 0
    const float ea = __builtin_amdgcn_exp2f(da), eb = __builtin_amdgcn_exp2f(db);
    r.s = ea * a.s + eb * b.s;
    r.t = ea * fmaf(da, a.s, a.t) + eb * fmaf(db, b.s, b.t);
    r.above = a.above + b.above;
    return r;
}
__device__ __forceinline__ Sums join_wave(Sums a) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) a = join(a, Sums{__shfl_xor(a.m, o, 64), __shfl_xor(a.s, o, 64), __shfl_xor(a.t, o, 64), 0});
    return a;  // above: of the wave already
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

// log s of s = 2^k f, f from sqrt(1/2) to sqrt(2): logf(s) and ln 2 log2 s are both off by up to a step and a half of log2 s (1.6e-6 of rows that are
// flat over 100000 tokens), log f by a few 1e-8
__device__ __forceinline__ float log_of(float s) {
    int k;
    float f = frexpf(s, &k);
    if (f < 0.70710678f) {
        f *= 2.f;
        --k;
    }
    return fmaf(static_cast<float>(k), kLn2, logf(f));
}
__device__ __forceinline__ float log_probability(const Sums &s, float z) { return (z - s.m) - log_of(s.s); }
// what is written of a whole row but its token's rank; `given`: the token's logit
__device__ __forceinline__ void put_scores(const LogprobArgs &a, int64_t row, const Sums &s, bool any, float given) {
    a.entropy[row] = log_of(s.s) - s.t / s.s * kLn2;
    a.logprob[row] = any ? log_probability(s, given) : 0.f;
}
// how many of the n logits kept in `near` are as probable as the given one; whether that is all it takes
__device__ __forceinline__ int as_probable(const float *near, int n, float m, float given) {
    int same = 0;
    for (int i = 0; i < min(n, kNeighbours); ++i) same += near[i] - m == given - m;
    return same;
}
__device__ __forceinline__ bool neighbours_do(int n, float m, float given) { return n <= kNeighbours && m - given <= kNearRange; }
// the rank from the row itself, by a block of 256 threads
template <int DT>
__device__ __forceinline__ void rank_again(const LogprobArgs &a, int64_t row, const void *z, float m, float given, int *shared, int tid) {
    int n = 0;
    for (int64_t k = tid; k < a.V; k += 256 * 16) {  // sixteen reads in flight
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = logit_at<DT>(z, min(k + 256 * i, static_cast<int64_t>(a.V - 1)));
#pragma unroll
        for (int i = 0; i < 16; ++i) n += k + 256 * i < a.V && v[i] - m > given - m;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
    if ((tid & 63) == 0) shared[tid >> 6] = n;
    __syncthreads();
    if (tid == 0) a.rank[row] = 1 + shared[0] + shared[1] + shared[2] + shared[3];
}
__device__ __forceinline__ void put_best(const LogprobArgs &a, int64_t row, const Sums &s, int i, uint64_t key) {
    a.top_ids[row * a.top + i] = token_of(key);
    a.top_logprobs[row * a.top + i] = log_probability(s, logit_of(key));
}

// VPT values of a thread are in flight together: 256 of them are a tile.
template <int DT, bool VEC, int VPT>
__global__ __launch_bounds__(256, 4) void logprobs_kernel(LogprobArgs a) {
    constexpr int W = VEC ? (DT == MFQ_X_F32 ? 4 : 8) : 1, N = VPT / W, TILE = 256 * VPT;  // values of a load, loads of a tile
    constexpr int LEVELS = __builtin_ctz(VPT);
    static_assert(VPT == 1 << LEVELS, "a tree of all levels");
    __shared__ uint64_t s_buf[4][128];
    __shared__ Sums s_sums[4];
    __shared__ int s_count[4];
    __shared__ float s_near[kNeighbours];
    __shared__ int s_near_count;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row = blockIdx.x / a.parts;
    const int part = static_cast<int>(blockIdx.x - row * a.parts);
    const void *z = static_cast<const uint8_t *>(a.logits) + row * a.ldl * (DT == MFQ_X_F32 ? 4 : 2);
    const int64_t token = a.tokens[row];
    const bool any = token >= 0 && token < a.V;
    const float given = any ? logit_at<DT>(z, token) : INFINITY, close = given + kNear;
    if (tid == 0) s_near_count = 0;
    __syncthreads();

    Sums my = {-INFINITY, 0.f, 0.f, 0};
    float s_more = 0.f, t_more = 0.f;  // what rounding has added to my.s and my.t so far
    uint64_t bar = 0;     // of the wave: smaller numbers are not among its best
    float bar_value = -INFINITY;
    int count = 0;        // of the wave's buffer
    uint64_t *buf = s_buf[wave];
    const int64_t first = static_cast<int64_t>(part) * a.per * TILE, end = min(first + static_cast<int64_t>(a.per) * TILE, static_cast<int64_t>(a.V));
    for (int64_t at = first; at < end; at += TILE) {
        float v[VPT];
        const bool whole = at + TILE <= end;
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
            for (int i = 0; i < VPT; ++i) {
                const int64_t k = at + ((i / W) * 256 + tid) * W + i % W;
                v[i] = k < end ? logit_at<DT>(z, k) : -INFINITY;
            }
        }
        // The values that `which` names, one of each lane at a time: they are read again, since registers have no index.
        const auto index = [&](int i) { return static_cast<uint32_t>(at + ((i / W) * 256 + tid) * W + i % W); };
        const auto for_values = [&](auto which, auto look) __attribute__((always_inline)) {
            uint32_t left = 0;
#pragma unroll
            for (int i = 0; i < VPT; ++i) left |= (which(v[i]) ? 1u : 0u) << i;
            while (__ballot(left != 0u)) {
                const uint32_t k = index(left ? __ffs(left) - 1 : 0);
                const bool real = left && k < end;
                look(real ? logit_at<DT>(z, k) : -INFINITY, k, real);
                left &= left - 1;
            }
        };
        float most = v[0];
#pragma unroll
        for (int i = 1; i < VPT; ++i) most = fmaxf(most, v[i]);
        {
            const float m = fmaxf(my.m, most), base = base_of(m), d = bounded(exponent(my.m, base)), c = __builtin_amdgcn_exp2f(d);
            my.t = c * fmaf(d, my.s, my.t);
            t_more = c * fmaf(d, s_more, t_more);
            my.s *= c;
            s_more *= c;
            my.m = m;
            unsigned long long near = 0;
            // The tile's sums by a tree: of 2^k values in [k]; then to those of the row, with what rounding adds kept.  Added one by one, the 594 values
            // that a thread has of a row of 151936 cost up to 9e-6 of their sum where many are equal, in all threads alike, and 5e-6 in random rows
            // (now 2e-7, in the same time).
            float ts[LEVELS + 1], tt[LEVELS + 1];
#pragma unroll
            for (int i = 0; i < VPT; ++i) {
                const float p = exponent(v[i], base);
                float e = __builtin_amdgcn_exp2f(p), pe = i & 1 ? fmaf(bounded(p), e, tt[0]) : bounded(p) * e;
#pragma unroll
                for (int k = 0; k < LEVELS; ++k)
                    if ((~i & ((2 << k) - 1)) == 0) {  // numbers that end in k + 1 ones close 2^k and 2^k values
                        e += ts[k];
                        if (k > 0) pe += tt[k];
                    }
                ts[__builtin_ctz(~i)] = e;
                tt[__builtin_ctz(~i)] = pe;
                // of the wave, in scalar registers
                const unsigned long long over = __ballot(v[i] > given), beyond = __ballot(v[i] > close);
                my.above += __popcll(over);
                near |= over ^ beyond;
            }
            const auto add = [](float &sum, float &more, float v) {
                const float less = v - more, next = sum + less;
                more = (next - sum) - less;
                sum = next;
            };
            add(my.s, s_more, ts[LEVELS]);
            add(my.t, t_more, tt[LEVELS]);
            if (near) {
                for_values([&](float value) { return value > given && !(value > close); }, [&](float value, uint32_t, bool real) {
                    if (!real) return;
                    const int at_near = atomicAdd(&s_near_count, 1);
                    if (at_near < kNeighbours) s_near[at_near] = value;
                });
            }
        }
        if (a.top == 0) continue;
        if (at == first) {
            uint32_t where = index(0);  // the lowest of the largest; what pads a tile lies behind all others
#pragma unroll
            for (int i = VPT - 1; i > 0; --i) where = v[i] == most ? index(i) : where;
            where = v[0] == most ? index(0) : where;
            buf[lane] = where < end ? key_of(most, where) : 0;
            if (keep_best(buf, 64, a.top, lane) == a.top) {
                bar = buf[a.top - 1];
                bar_value = logit_of(bar);
            }
            wave_sync();
        }
        // a NaN is no reason to look, and is found where one is needed: while the bar is as low
        if (!__ballot(!(most < bar_value))) continue;
        for_values([&](float value) { return !(value < bar_value); }, [&](float value, uint32_t where, bool real) {
            const uint64_t k = real ? key_of(value, where) : 0;
            const bool take = k && k >= bar;
            const uint64_t takers = __ballot(take);
            if (!takers) return;
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
        });
    }
    if (a.top) {
        count = keep_best(buf, count, a.top, lane);
        if (lane == 0) s_count[wave] = count;
    }
    my.s -= s_more;
    my.t -= t_more;
    my = join_wave(my);
    if (lane == 0) s_sums[wave] = my;
    __syncthreads();
    const Sums all = join(join(s_sums[0], s_sums[1]), join(s_sums[2], s_sums[3]));
    if (a.parts > 1) {
        if (tid == 0) a.sums[blockIdx.x] = float4_t{all.m, all.s, all.t, __int_as_float(all.above)};
        if (tid <= kNeighbours)
            a.near[static_cast<int64_t>(blockIdx.x) * (1 + kNeighbours) + tid] = tid == 0 ? __int_as_float(s_near_count) : tid <= s_near_count ? s_near[tid - 1] : 0.f;
    } else if (tid == 0) {
        put_scores(a, row, all, any, given);
        a.rank[row] = any ? 1 + all.above - as_probable(s_near, s_near_count, all.m, given) : 0;
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
    if (a.parts > 1) {
        if (tid >= kept && tid < a.top) a.keys[static_cast<int64_t>(blockIdx.x) * a.top + tid] = 0;
    } else if (any && !neighbours_do(s_near_count, all.m, given)) {
        __syncthreads();  // after the rank that is replaced
        rank_again<DT>(a, row, z, all.m, given, s_count, tid);
    }
}

// The parts of a row, a block each.  Their lists of keys are in order: with number `step` of each list `step` of its keys are as large, so the
// ceil(top / step)-th largest of those is a bar that `top` keys reach, and few more.
template <int DT>
__global__ __launch_bounds__(256) void logprobs_join_kernel(LogprobArgs a) {
    extern __shared__ uint64_t s_key[];  // the lists' keys, and those that reach the bar
    __shared__ Sums s_sums[4];
    __shared__ int s_total[3];           // neighbours as probable, parts with too many of them, keys that reach the bar
    __shared__ uint64_t s_bar;
    __shared__ int s_count[4];
    const int tid = threadIdx.x, lane = tid & 63;
    const int64_t row = blockIdx.x;
    const int n = a.parts * a.top;
    const int64_t token = a.tokens[row];
    const bool any = token >= 0 && token < a.V;
    const void *z = static_cast<const uint8_t *>(a.logits) + row * a.ldl * (DT == MFQ_X_F32 ? 4 : 2);
    const float given = any ? logit_at<DT>(z, token) : 0.f;
    for (int i = tid; i < n; i += 256) s_key[i] = a.keys[row * n + i];
    if (tid < 3) s_total[tid] = 0;
    if (tid == 0) s_bar = 0;
    Sums my = {-INFINITY, 0.f, 0.f, 0};
    for (int p = tid; p < a.parts; p += 256) {
        const float4_t v = a.sums[row * a.parts + p];
        my = join(my, Sums{v.x, v.y, v.z, __float_as_int(v.w)});
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) my.above += __shfl_xor(my.above, o, 64);
    my = join_wave(my);
    if (lane == 0) s_sums[tid >> 6] = my;
    __syncthreads();
    const Sums all = join(join(s_sums[0], s_sums[1]), join(s_sums[2], s_sums[3]));
    for (int p = tid; p < a.parts; p += 256) {
        const float *near = a.near + (row * a.parts + p) * (1 + kNeighbours);
        const int have = __float_as_int(near[0]);
        if (have) {
            atomicAdd(&s_total[0], as_probable(near + 1, have, all.m, given));
            if (have > kNeighbours) atomicAdd(&s_total[1], 1);
        }
    }
    if (a.top) {
        const int step = (a.top + a.parts - 1) / a.parts, want = (a.top + step - 1) / step;
        for (int p = tid; p < a.parts; p += 256) {
            const uint64_t mine = s_key[p * a.top + step - 1];
            int above = 0;
#pragma unroll 8
            for (int q = 0; q < a.parts; ++q) above += s_key[q * a.top + step - 1] > mine;
            if (mine && above == want - 1) s_bar = mine;  // no two keys are equal
        }
    }
    __syncthreads();
    uint64_t *taken = s_key + n;
    const uint64_t bar = s_bar;
    for (int i = tid; i < n; i += 256)
        if (s_key[i] && s_key[i] >= bar) taken[atomicAdd(&s_total[2], 1)] = s_key[i];
    __syncthreads();
    if (tid == 0) {
        put_scores(a, row, all, any, given);
        a.rank[row] = any ? 1 + all.above - s_total[0] : 0;
    }
    const int reach = s_total[2];
    for (int i = tid; i < reach; i += 256) {
        const uint64_t k = taken[i];
        int r = 0;
#pragma unroll 8
        for (int j = 0; j < reach; ++j) r += taken[j] > k;
        if (r < a.top) put_best(a, row, all, r, k);
    }
    if (any && !neighbours_do(s_total[1] ? kNeighbours + 1 : 0, all.m, given)) {
        __syncthreads();
        rank_again<DT>(a, row, z, all.m, given, s_count, tid);
    }
}

// Pieces of a row: enough blocks of 256 threads for four a compute unit, of whole tiles, none empty; their lists fit the joining block's LDS.
// Smaller tiles where rows are few enough for each block to have one of them.
constexpr int kMaxLists = 4096, kVpt = 16;
struct LogprobPlan { int vpt, parts, per; };
LogprobPlan plan_of(int M, int V, int top) {
    const int64_t room = kMaxLists / (top > 0 ? top : 1);
    int64_t want = ceil_div(static_cast<int64_t>(4) * device_cu_count(), M);
    if (want > room) want = room;
    const int vpt = ceil_div(V, 256 * 8) <= want ? 8 : kVpt;
    const int64_t tiles = ceil_div(V, 256 * vpt), per = ceil_div(tiles, want < tiles ? want : tiles);
    return {vpt, static_cast<int>(ceil_div(tiles, per)), static_cast<int>(per)};
}
// of a part: sums, neighbours, keys
size_t workspace_of(int M, int parts, int top) {
    return parts == 1 ? 0 : static_cast<size_t>(M) * parts * (sizeof(float4_t) + (1 + kNeighbours) * 4 + static_cast<size_t>(top) * 8);
}

template <int DT>
int launch(const LogprobArgs &a, int M, int vpt, bool wide, hipStream_t st) {
    const dim3 grid(static_cast<unsigned>(static_cast<int64_t>(M) * a.parts));
    auto kern = vpt == 8 ? (wide ? logprobs_kernel<DT, true, 8> : logprobs_kernel<DT, false, 8>) : (wide ? logprobs_kernel<DT, true, kVpt> : logprobs_kernel<DT, false, kVpt>);
    hipLaunchKernelGGL(kern, grid, dim3(256), 0, st, a);
    if (int rc = check_launch("token_logprobs")) return rc;
    if (a.parts == 1) return MFQ_OK;
    const size_t lds = static_cast<size_t>(a.parts) * a.top * 16;
    if (int rc = allow_dynamic_lds(reinterpret_cast<const void *>(logprobs_join_kernel<DT>), lds, "token_logprobs")) return rc;
    hipLaunchKernelGGL((logprobs_join_kernel<DT>), dim3(static_cast<unsigned>(M)), dim3(256), lds, st, a);
    return check_launch("token_logprobs (join)");
}

}  // namespace
}  // namespace mfq

using namespace mfq;

extern "C" size_t mfq_hip_token_logprobs_workspace_bytes(int M, int V, int top) {
    if (M < 1 || V < 1 || top < 0 || top > kMaxTop || top > V) return 0;
    return workspace_of(M, plan_of(M, V, top).parts, top);
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
    const LogprobPlan p = plan_of(M, V, top);
    LogprobArgs a = {logits, ldl, V, top, p.parts, p.per, tokens, logprob, entropy, top_logprobs, rank, top_ids, nullptr, nullptr, nullptr};
    MFQ_REQUIRE(grid_fits(static_cast<int64_t>(M) * a.parts, 256), MFQ_ERR_UNSUPPORTED, "token_logprobs: %d rows", M);
    if (a.parts > 1) {
        const size_t need = workspace_of(M, a.parts, top);
        MFQ_REQUIRE(workspace && workspace_bytes >= need, MFQ_ERR_WORKSPACE, "token_logprobs: workspace %zu < %zu", workspace_bytes, need);
        MFQ_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, MFQ_ERR_WORKSPACE, "token_logprobs: unaligned workspace");
        a.sums = static_cast<float4_t *>(workspace);
        a.near = reinterpret_cast<float *>(a.sums + static_cast<size_t>(M) * a.parts);
        a.keys = reinterpret_cast<uint64_t *>(a.near + static_cast<size_t>(M) * a.parts * (1 + kNeighbours));
    }
    const bool wide = reinterpret_cast<uintptr_t>(logits) % 16 == 0 && (M == 1 || ldl * size % 16 == 0);
    const hipStream_t st = as_stream(stream);
    if (dtype == MFQ_X_F32) return launch<MFQ_X_F32>(a, M, p.vpt, wide, st);
    return dtype == MFQ_X_F16 ? launch<MFQ_X_F16>(a, M, p.vpt, wide, st) : launch<MFQ_X_BF16>(a, M, p.vpt, wide, st);
}
