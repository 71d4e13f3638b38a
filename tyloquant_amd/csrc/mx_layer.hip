// A whole layer of routed experts for up to 16 tokens, from the router's logits to the layer's output, in two launches:
//   e_1 .. e_k, p_1 .. p_k = top k of the router (mfq_hip_moe_topk's rules)
//   h_j = act(G_{e_j} x) * (U_{e_j} x),   y = sum_j p_j D_{e_j} h_j  (+ gate * D_s h_s of an expert that all tokens take)
// MXFP8 or MXFP4 tensors, activations as they come.  Every expert that some token takes is read once, for all of its tokens: bound by the
// weights' way from memory.
//
// The weights' codes are converted to bf16 with their scales, exactly (but for the smallest codes of scales 2^-127 and 2^-126, which bf16's
// subnormals cut: 1e-6 of a result), and v_mfma_f32_16x16x32_bf16 multiplies them with up to 16 columns of
// activations.  Values that bf16 does not hold go as sums of such: fp16 as two parts, the hidden rows, which are fp32, as three, each part the
// rounding of what the ones before leave.  Parts of few tokens are columns beside one another (one column a part and token); else they
// are multiplied one after the other into the same sums.  So products are exact to 2^-24 and sums are fp32: nothing is rounded to 16 bits
// but the result, where a 16-bit one is asked for.
//
// First launch: every block finds the selection for itself (a wave a token, some 100 instructions a choice), which costs less than a launch of
// its own would; blocks then share the row-blocks of all experts hit evenly.  Waves split K, their weights come through a ring in LDS (as in
// mx8_scaled.hip), their activations stay in registers.  Second launch: waves share the columns of all
// experts, and an expert's sums are weighted and added, for the tokens that take it and no others, where a wave leaves it.
// Columns of an operand that are no token's hold another's values, not zeros: their sums are not looked at.
#include "moe_topk.hpp"
#include "mx_cvt.hpp"
#include "mx_scaled.hpp"

namespace mfq {
namespace {

constexpr int kMaxTokens = 16, kMaxRoutes = 16, kMaxExperts = 1024, kMaxPairs = kMaxTokens * kMaxRoutes;

// What the first launch leaves of the selection for the second: the experts hit in ascending order, and of each who takes it, with which
// weight and by which of a token's routes.
struct LayerTable {
    int count, pad[3];
    int expert[kMaxPairs];
    uint32_t tokens[kMaxPairs];
    float weight[kMaxPairs][kMaxTokens];
    uint8_t rank[kMaxPairs][kMaxTokens];
};

struct LayerArgs {
    mfq_mx_layer w;
    const void *x;
    int64_t ldx;
    int x_f16, x_wide, T, k, mode, normalize, gelu;
    const float *logits, *bias, *shared_gate;
    float norm_floor, scale;
    int32_t *ids;
    float *weights;
    void *y;
    int y_dtype;
    int64_t ldy;
    uint16_t *hidden;         // three parts of [T * k][inter], bf16
    uint16_t *shared_hidden;  // three parts of [T][shared_inter]
    LayerTable *table;
    int pieces;               // of the columns of all experts, in the second launch
    float *partial;           // [groups of 64 results][pieces][T][64]
    int32_t *arrived;         // [groups]: pieces that are there
};

// Bytes of a row, lines of 128 bytes of it; columns of a line, and operands of 32 columns that they make.
template <int KIND>
struct LineOf {
    static constexpr int COLS = KIND == 8 ? 128 : 256, FR = COLS / 32;
    __host__ __device__ static constexpr int64_t bytes(int K) { return KIND == 8 ? K : K / 2; }
    __host__ __device__ static constexpr int lines(int K) { return (K + COLS - 1) / COLS; }
};

// ---- the selection ----------------------------------------------------------------------------------------------------------------
// largest of the wave, the same in every lane
__device__ __forceinline__ int wave_max_int(int v) {
    v = max(v, __builtin_amdgcn_update_dpp(v, v, 0xB1, 0xF, 0xF, false));   // lane ^ 1
    v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x4E, 0xF, 0xF, false));   // lane ^ 2
    v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x141, 0xF, 0xF, false));  // the other four of eight
    v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x140, 0xF, 0xF, false));  // the other eight of a row of 16
    v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x142, 0xA, 0xF, false));  // the row before, in rows 1 and 3
    v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x143, 0xC, 0xF, false));  // rows 0 and 1, in rows 2 and 3
    return __builtin_amdgcn_readlane(v, 63);
}

// The experts of one token and their weights, by one wave; up to 64 * PER experts, expert lane + 64 i in element i.
template <int PER>
__device__ __forceinline__ void select_experts(const LayerArgs &a, int t, int lane, int *ids, float *weights) {
    const float *row = a.logits + static_cast<int64_t>(t) * a.w.experts;
    float raw[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int e = lane + 64 * i;
        const float v = e < a.w.experts ? row[e] : -INFINITY;
        raw[i] = v != v ? -FLT_MAX : v;
    }
    float most = 0.f, sum = 1.f;
    if (a.mode == MFQ_TOPK_SOFTMAX) {
        most = raw[0];
#pragma unroll
        for (int i = 1; i < PER; ++i) most = fmaxf(most, raw[i]);
        most = wave_max(most);
        float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < PER; ++i) part[i & 3] += lane + 64 * i < a.w.experts ? expf(raw[i] - most) : 0.f;
        sum = (wave_sum(part[0]) + wave_sum(part[1])) + (wave_sum(part[2]) + wave_sum(part[3]));
    }
    int key[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int e = lane + 64 * i;
        key[i] = e < a.w.experts ? topk_key(topk_weight(raw[i], a.mode, most, sum) + (a.bias ? a.bias[e] : 0.f)) : INT_MIN;
    }
    float mine = 0.f;
    for (int rank = 0; rank < a.k; ++rank) {
        int best = key[0];
#pragma unroll
        for (int i = 1; i < PER; ++i) best = max(best, key[i]);
        best = wave_max_int(best);
        int expert = -1;      // the lowest of those with that score
        float value = 0.f;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const unsigned long long those = __ballot(key[i] == best);
            if (expert < 0 && those) {
                const int l = __ffsll(those) - 1;
                expert = l + 64 * i;
                value = __uint_as_float(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(__float_as_uint(raw[i])), l)));
                if (lane == l) key[i] = INT_MIN;
            }
        }
        if (lane == rank) {
            ids[rank] = expert;
            mine = topk_weight(value, a.mode, most, sum);
        }
    }
    mine = topk_finish(lane < a.k ? mine : 0.f, a.k, lane, a.mode, a.normalize, a.norm_floor) * a.scale;
    if (lane < a.k) weights[lane] = mine;
}

// Experts that some token takes, in ascending order, and who takes them.
struct Selection {
    int ids[kMaxPairs];           // [token][k]
    float weights[kMaxPairs];
    uint32_t place[kMaxExperts];  // tokens of an expert as bits, then its number in the list
    int expert[kMaxPairs];
    uint32_t tokens[kMaxPairs];   // of the list's experts
    uint8_t rank[kMaxPairs][kMaxTokens];  // which of a token's routes leads to it
    int count;
};
// by a whole block, which has filled ids; place is cleared
__device__ __forceinline__ void list_experts(Selection &s, int E, int T, int k, int tid, int nt) {
    for (int p = tid; p < T * k; p += nt) atomicOr(&s.place[s.ids[p]], 1u << (p / k));
    __syncthreads();
    if (tid < 64) {
        int n = 0;
        for (int c = 0; c < E; c += 64) {
            const uint32_t m = c + tid < E ? s.place[c + tid] : 0u;
            const unsigned long long any = __ballot(m != 0u);
            if (m) {
                const int at = n + __popcll(any & ((1ull << tid) - 1));
                s.expert[at] = c + tid;
                s.tokens[at] = m;
                s.place[c + tid] = static_cast<uint32_t>(at);
            }
            n += __popcll(any);
        }
        if (tid == 0) s.count = n;
    }
    __syncthreads();
    for (int p = tid; p < T * k; p += nt) s.rank[s.place[s.ids[p]]][p / k] = static_cast<uint8_t>(p % k);
    __syncthreads();
}

// ---- gate and up ------------------------------------------------------------------------------------------------------------------
constexpr int kUpWaves = 8;
template <int KIND>
struct UpShape {
    static constexpr int D = 3, CODES = 2 * 2048, STAGE = CODES + 256, REQ = 5, RED = 2 * 1024;
    static constexpr size_t lds(int nwaves) { return static_cast<size_t>(nwaves) * (D * STAGE + 2 * RED); }
};

// eight columns of a token's activations from `col` on as bf16: part 0 their rounding, part 1 what it leaves of fp16
__device__ __forceinline__ u32x4_t activations(const LayerArgs &a, int t, int part, int col) {
    const uint16_t *p = static_cast<const uint16_t *>(a.x) + t * a.ldx + col;
    u32x4_t v;
    if (a.x_wide) {
        v = *reinterpret_cast<const u32x4_t *>(p);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = p[2 * i] | (static_cast<uint32_t>(p[2 * i + 1]) << 16);
    }
    if (!a.x_f16) return v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float f[2] = {f16_to_f32(static_cast<uint16_t>(v[i])), f16_to_f32(static_cast<uint16_t>(v[i] >> 16))};
        if (part) {
#pragma unroll
            for (int j = 0; j < 2; ++j) f[j] = fabsf(f[j]) < INFINITY ? f[j] - bf16_to_f32(f32_to_bf16_rne(f[j])) : 0.f;
        }
        v[i] = mx_pack16(f[0], f[1], MFQ_X_BF16);
    }
    return v;
}

__device__ __forceinline__ void pin(u32x4_t &v) { asm volatile("" : "+v"(v)); }

// NL: lines of K a wave has at most, whose activations stay in registers (0: any number, read again for every row-block); SETS of 16 columns.
template <int KIND, int NL, int SETS>
__global__ __launch_bounds__(512) void mx_layer_up_kernel(LayerArgs a) {
    using S = UpShape<KIND>;
    using Line = LineOf<KIND>;
    constexpr int D = S::D, FR = Line::FR;
    static_assert(D == 3, "the waits of the loop");
    extern __shared__ __attribute__((aligned(128))) uint8_t lds[];
    __shared__ Selection sel;
    const int tid = threadIdx.x, lane = tid & 63, nt = blockDim.x, nwaves = nt >> 6;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15, g = lane >> 4;
    const int H = a.w.hidden, I = a.w.inter, T = a.T;
    const int nlines = Line::lines(H);
    const int64_t row_bytes = Line::bytes(H);

    // this lane's columns of activations
    const int mine = (nlines - wave + nwaves - 1) / nwaves;  // lines wave, wave + nwaves, ...
    const int parts = a.x_f16 ? 2 : 1;
    // token and part of column r of each set; the first of both where it has none
    int token[SETS], part[SETS];
#pragma unroll
    for (int s = 0; s < SETS; ++s) {
        const int p = SETS == 1 ? r / T : s, c = SETS == 1 ? r - p * T : r;
        const bool is = p < parts && c < T;
        token[s] = is ? c : 0;
        part[s] = is ? p : 0;
    }
    auto operand = [&](int s, int line, int f) __attribute__((always_inline)) {
        const int col = line * Line::COLS + g * (Line::COLS / 4) + 8 * f;
        const u32x4_t v = activations(a, token[s], part[s], min(col, H - 8));
        return KIND == 8 || col < H ? v : u32x4_t{0u, 0u, 0u, 0u};
    };
    u32x4_t x[NL > 0 ? NL : 1][SETS][FR];
    if constexpr (NL > 0) {
        // a line's reads together, and its operands before the next line's
        static_for<NL>([&](auto MI) __attribute__((always_inline)) {
            constexpr int m = MI.value;
#pragma unroll
            for (int s = 0; s < SETS; ++s)
#pragma unroll
                for (int f = 0; f < FR; ++f) x[m][s][f] = operand(s, min(wave + m * nwaves, nlines - 1), f);
            if (a.x_f16) {
#pragma unroll
                for (int s = 0; s < SETS; ++s)
#pragma unroll
                    for (int f = 0; f < FR; ++f) pin(x[m][s][f]);
            }
        });
    }

    for (int e = tid; e < a.w.experts; e += nt) sel.place[e] = 0u;
    for (int t = wave; t < T; t += nwaves) {
        if (a.w.experts <= 256) select_experts<4>(a, t, lane, sel.ids + t * a.k, sel.weights + t * a.k);
        else select_experts<16>(a, t, lane, sel.ids + t * a.k, sel.weights + t * a.k);
    }
    __syncthreads();
    if (blockIdx.x == 0)
        for (int p = tid; p < T * a.k; p += nt) {
            a.ids[p] = sel.ids[p];
            a.weights[p] = sel.weights[p];
        }
    list_experts(sel, a.w.experts, T, a.k, tid, nt);
    const int count = __builtin_amdgcn_readfirstlane(sel.count);
    if (blockIdx.x == gridDim.x - 1) {
        for (int i = tid; i < (H + 63) / 64; i += nt) a.arrived[i] = 0;
        if (tid == 0) a.table->count = count;
        for (int l = tid; l < count; l += nt) {
            a.table->expert[l] = sel.expert[l];
            a.table->tokens[l] = sel.tokens[l];
        }
        for (int p = tid; p < count * kMaxTokens; p += nt) {
            const int l = p / kMaxTokens, t = p % kMaxTokens;
            const bool takes = t < T && (sel.tokens[l] >> t & 1u);
            const int rank = takes ? sel.rank[l][t] : 0;
            a.table->weight[l][t] = takes ? sel.weights[t * a.k + rank] : 0.f;
            a.table->rank[l][t] = static_cast<uint8_t>(rank);
        }
    }

    // this block's row-blocks of 16 gate rows with their up rows, of all experts one after the other, the shared one last
    const int rbs = I / 16, all = count * rbs + a.w.shared_inter / 16;
    const int i0 = static_cast<int>(static_cast<int64_t>(all) * blockIdx.x / gridDim.x), i1 = static_cast<int>(static_cast<int64_t>(all) * (blockIdx.x + 1) / gridDim.x);
    const int total = (i1 - i0) * mine;

    uint8_t *ring = lds + wave * (D * S::STAGE);
    const int piece = lane & 7;
    // the next copies: stage, item's expert in the list, row-block, line
    int to_stage = 0, to_l = min(i0 / rbs, count), to_rb = i0 - to_l * rbs, to_m = 0;
    __amdgpu_buffer_rsrc_t win, swin;
    uint32_t up_off = 0, sbase = 0;  // from a gate row to its up row; MXFP8: byte of the expert's first scale, MXFP4: its first row
    int to_width = 0;
    auto enter = [&] {  // the tensor of expert to_l
        const bool shared = to_l == count;
        to_width = shared ? a.w.shared_inter : I;
        const int64_t e = shared ? 0 : __builtin_amdgcn_readfirstlane(sel.expert[min(to_l, kMaxPairs - 1)]);
        const uint8_t *v = static_cast<const uint8_t *>(shared ? a.w.shared_gate_up : a.w.gate_up) + e * 2 * I * row_bytes;
        const uint8_t *sc = static_cast<const uint8_t *>(shared ? a.w.shared_gate_up_scales : a.w.gate_up_scales);
        win = wave_window(v, static_cast<uint32_t>(2 * to_width * row_bytes));
        up_off = static_cast<uint32_t>(to_width * row_bytes);
        if constexpr (KIND == 8) {
            // the word that holds a block's byte is read whole: from the 4-byte boundary at or in front of the first scale
            const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(sc) & 3);
            swin = wave_window(sc - off, 0xffffff00u);
            sbase = off + static_cast<uint32_t>(e * 2 * I / 128) * nlines;  // gate and up rows are whole blocks
        } else {
            swin = wave_window(sc, 0xffffff00u);  // offsets of 32 bits from the first row: the host sees to it
            sbase = static_cast<uint32_t>(e * 2 * I);
        }
    };
    // MXFP8: of row-block rb, half b and line `line` of an expert, the byte of its scale
    auto scale_byte = [&](uint32_t base, int rb, int b, int line, int width) {
        return base + static_cast<uint32_t>((b * width + rb * 16) >> 7) * static_cast<uint32_t>(nlines) + static_cast<uint32_t>(line);
    };
    const int nblk = H / 32;  // pieces of 16 bytes of an MXFP4 row
    auto issue = [&] {
        uint8_t *to = ring + to_stage * S::STAGE;
        const int line = wave + to_m * nwaves;
        const int last = KIND == 8 ? 7 : nblk - 1 - 8 * line;  // of the line's pieces; behind it the last one again, where activations are zeros
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = 8 * (i & 1) + (lane >> 3);
            const uint32_t p = static_cast<uint32_t>(min(piece ^ mx_key(row), last));
            copy16<2>(win, to + i * 1024, static_cast<uint32_t>(row * row_bytes) + 16u * p,
                      static_cast<int>(static_cast<uint32_t>(to_rb * 16 * row_bytes) + (i >> 1) * up_off + static_cast<uint32_t>(line) * 128u));
        }
        if constexpr (KIND == 8) {
            if (lane < 2) copy4(swin, to + S::CODES, scale_byte(sbase, to_rb, lane, line, to_width) & ~3u, 0);
        } else {
            copy4(swin, to + S::CODES, mx_scale_at(sbase + (lane >> 5) * to_width + to_rb * 16 + ((lane >> 1) & 15), nlines) + 4u * (lane & 1), line * 256);
        }
        to_stage = to_stage + 1 == D ? 0 : to_stage + 1;
        if (++to_m == mine) {
            to_m = 0;
            if (++to_rb * 16 == to_width) {
                to_rb = 0;
                ++to_l;
                if (to_l < count || (to_l == count && a.w.shared_inter)) enter();
            }
        }
    };
    if (i0 < i1) enter();
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    uint32_t base = 0;  // of the item that is multiplied: sbase of its expert
#pragma unroll
    for (int i = 0; i < D; ++i)
        if (i < total) issue();

    uint8_t *red = lds + nwaves * (D * S::STAGE);
    int stage = 0, i = 0, l = min(i0 / rbs, count), rb = i0 - l * rbs, entered = -1;
    for (int item = i0; item < i1; ++item) {
        const bool shared = l == count;
        const int width = shared ? a.w.shared_inter : I;
        if constexpr (KIND == 8) {
            if (entered != l) {  // as `enter` has it
                const int64_t e = shared ? 0 : __builtin_amdgcn_readfirstlane(sel.expert[min(l, kMaxPairs - 1)]);
                const uintptr_t sc = reinterpret_cast<uintptr_t>(shared ? a.w.shared_gate_up_scales : a.w.gate_up_scales);
                base = static_cast<uint32_t>(sc & 3) + static_cast<uint32_t>(e * 2 * I / 128) * nlines;
                entered = l;
            }
        }
        float4_t acc[2] = {float4_t{0.f, 0.f, 0.f, 0.f}, float4_t{0.f, 0.f, 0.f, 0.f}};
        auto multiply = [&](int line, const u32x4_t (&xs)[SETS][FR]) __attribute__((always_inline)) {
            const uint8_t *at = ring + stage * S::STAGE;
            u32x4_t w[2][2];
            uint32_t raw[2];
#pragma unroll
            for (int b = 0; b < 2; ++b) {
#pragma unroll
                for (int h = 0; h < 2; ++h) w[b][h] = *reinterpret_cast<const u32x4_t *>(at + b * 2048 + r * 128 + (((2 * g + h) ^ mx_key(r)) << 4));
                if constexpr (KIND == 8) raw[b] = *reinterpret_cast<const uint32_t *>(at + S::CODES + 4 * b);
                else raw[b] = *reinterpret_cast<const uint16_t *>(at + S::CODES + b * 128 + r * 8 + 2 * g);
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the stage is free for the next copies
            if (i + D < total) issue();
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                if constexpr (KIND == 8) raw[b] = raw[b] >> (8 * (scale_byte(base, rb, b, line, width) & 3)) & 255u;
#pragma unroll
                for (int f = 0; f < FR; ++f) {
                    u32x4_t v;
                    if constexpr (KIND == 8) v = mx_cvt_fp8<0>(w[b][f >> 1][2 * (f & 1)], w[b][f >> 1][2 * (f & 1) + 1], __uint_as_float(raw[b] << 23));
                    else v = mx_cvt_fp4<0>(w[b][f >> 2][f & 3], __uint_as_float((raw[b] >> (8 * (f >> 2)) & 255u) << 23));
#pragma unroll
                    for (int s = 0; s < SETS; ++s) acc[b] = mx_mfma<0>(xs[s][f], v, acc[b]);
                }
            }
            stage = stage + 1 == D ? 0 : stage + 1;
            ++i;
        };
        auto landed = [&] {
            // younger than this stage: those of the next two, and stores of results, which only make the wait longer
            const int left = total - 1 - i;
            if (left >= D - 1) wait_vmcnt<(D - 1) * S::REQ>();
            else if (left == 1) wait_vmcnt<S::REQ>();
            else wait_vmcnt<0>();
        };
        if constexpr (NL > 0) {
            static_for<NL>([&](auto MI) __attribute__((always_inline)) {
                constexpr int m = MI.value;
                if (m >= mine) return;
                landed();
                multiply(wave + m * nwaves, x[m]);
            });
        } else {
            for (int m = 0; m < mine; ++m) {
#pragma unroll
                for (int s = 0; s < SETS; ++s)
#pragma unroll
                    for (int f = 0; f < FR; ++f) x[0][s][f] = operand(s, wave + m * nwaves, f);
                landed();
                multiply(wave + m * nwaves, x[0]);
            }
        }
        uint8_t *slot = red + (item & 1) * nwaves * S::RED;
#pragma unroll
        for (int b = 0; b < 2; ++b) *reinterpret_cast<float4_t *>(slot + wave * S::RED + b * 1024 + lane * 16) = acc[b];
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();  // the slot's next sums come behind the next one
        asm volatile("" ::: "memory");
        for (int o = tid; o < T * 16; o += nt) {
            const int t = o >> 4, n = o & 15;
            if (!shared && !(sel.tokens[l] >> t & 1u)) continue;
            float v[2] = {0.f, 0.f};
            for (int p = 0; p < (SETS == 1 ? parts : 1); ++p) {
                const int c = p * T + t;
                const float *at = reinterpret_cast<const float *>(slot) + ((c >> 2) * 16 + n) * 4 + (c & 3);
                for (int w = 0; w < nwaves; ++w) {
                    v[0] += at[w * (S::RED / 4)];
                    v[1] += at[w * (S::RED / 4) + 256];
                }
            }
            float h = glu_value(v[0], v[1], a.gelu);
            const int64_t row = shared ? t : t * a.k + sel.rank[l][t], rows = shared ? T : T * a.k;
            uint16_t *to = (shared ? a.shared_hidden : a.hidden) + row * width + rb * 16 + n;
#pragma unroll
            for (int p = 0; p < 3; ++p) {
                const uint16_t q = f32_to_bf16_rne(h);
                to[p * rows * width] = q;
                h = fabsf(h) < INFINITY ? h - bf16_to_f32(q) : 0.f;
            }
        }
        if (++rb * 16 == width) {
            rb = 0;
            ++l;
        }
    }
}

// ---- down and the weighted sum -------------------------------------------------------------------------------------------------------
// A block owns 64 results of every token, and of the columns of all experts one after the other (the shared one last) a piece, which its waves
// share in units of 128: an operand of hidden rows then serves four of weights, where reading it for each took more of a compute unit's
// address path than the weights (16 results a block: 67 MB of MXFP8 in 20 us, 116 MB for 16 tokens in 66).  The pieces of a result are added
// in their order by the block that comes last to them.
//
// The three parts of an expert's hidden rows are columns beside one another where it has five tokens or fewer, which at 16 tokens is most of
// them: a third of the reads and of the products (16 tokens of 64 experts, 8 each: 129 -> 98 us).  MANY: some may have more (T > 5), and then
// a set of columns for each part.
constexpr int kDownWaves = 8, kDownRows = 64, kMaxPieces = 16;
template <int KIND, bool MANY>
__global__ __launch_bounds__(kDownWaves * 64) void mx_layer_down_kernel(LayerArgs a) {
    constexpr int PIECES = KIND == 8 ? 2 : 1;  // of 16 bytes of a lane's 32 columns of a row
    __shared__ float s_weight[kMaxPairs][kMaxTokens];
    __shared__ int s_expert[kMaxPairs];
    __shared__ uint32_t s_tokens[kMaxPairs];
    __shared__ uint32_t s_rank[kMaxPairs][kMaxTokens / 4];
    __shared__ int s_listed, s_last;
    __shared__ float4_t red[kDownWaves][4][64];
    const int tid = threadIdx.x, lane = tid & 63, nt = kDownWaves * 64;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15, g = lane >> 4;
    const int H = a.w.hidden, I = a.w.inter, T = a.T, k = a.k;
    const int group = static_cast<int>(blockIdx.x) / a.pieces, piece = static_cast<int>(blockIdx.x) - group * a.pieces;
    {   // the table, as far as it can reach: entries behind the last are not looked at
        const int most = min(T * k, a.w.experts);
        if (tid == 0) s_listed = a.table->count;
        if (tid < most) {
            s_expert[tid] = a.table->expert[tid];
            s_tokens[tid] = a.table->tokens[tid];
        }
        for (int p = tid; p < most * (kMaxTokens / 4); p += nt) s_rank[0][p] = reinterpret_cast<const uint32_t *>(a.table->rank)[p];
        for (int p = tid; p < most * kMaxTokens; p += nt) s_weight[0][p] = a.table->weight[0][p];
    }
    __syncthreads();
    const int count = __builtin_amdgcn_readfirstlane(s_listed);

    int row[4];  // behind the last one: the last one again
#pragma unroll
    for (int b = 0; b < 4; ++b) row[b] = min(group * kDownRows + 16 * b + r, H - 1);
    const int units = (I + 127) / 128, shared_units = (a.w.shared_inter + 127) / 128;
    const int all = count * units + shared_units;
    const int lo = static_cast<int>(static_cast<int64_t>(all) * piece / a.pieces), hi = static_cast<int>(static_cast<int64_t>(all) * (piece + 1) / a.pieces);
    // The waves take neighbouring runs of units, so that the block reads its rows from memory in whole lengths: 98 -> 95 us there, and 47 -> 45 for five
    // tokens of MXFP4.  Runs half as long have sums weighted twice as often: 97, and one token of MXFP8 20.6 us for 19.2.
    const int run = max(1, min(KIND == 4 ? 8 : 4, (hi - lo + kDownWaves - 1) / kDownWaves));

    float4_t sum[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) sum[b] = float4_t{0.f, 0.f, 0.f, 0.f};
    int at = lo + wave * run, end = min(at + run, hi);
    while (at < hi) {
        const int l = min(at / units, count);
        const bool shared = l == count;
        const int first = at - l * units, n = min(end - at, (shared ? shared_units : units) - first);
        const int K = shared ? a.w.shared_inter : I;
        const int64_t e = shared ? 0 : __builtin_amdgcn_readfirstlane(s_expert[min(l, kMaxPairs - 1)]);
        const uint32_t takers = shared ? (1u << T) - 1u : __builtin_amdgcn_readfirstlane(static_cast<int>(s_tokens[min(l, kMaxPairs - 1)]));
        const uint8_t *values = static_cast<const uint8_t *>(shared ? a.w.shared_down : a.w.down) + e * H * LineOf<KIND>::bytes(K);
        const uint8_t *scales = static_cast<const uint8_t *>(shared ? a.w.shared_down_scales : a.w.down_scales);
        const uint8_t *wrow[4], *srow[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            wrow[b] = values + row[b] * LineOf<KIND>::bytes(K);
            // MXFP8: of the 64 rows, which lie within a block of 128; MXFP4: each row's
            srow[b] = KIND == 8 ? scales + ((e * H + row[0]) >> 7) * (shared ? shared_units : units) : scales + mx_scale_at(e * H + row[b], mx_macros(K)) + g;
        }
        const int last = K / 32 - 1;  // of an MXFP4 row's pieces, blocks of 32 columns
        const int someone = __ffs(takers) - 1, ntakers = __popc(takers);
        const uint16_t *hidden = shared ? a.shared_hidden : a.hidden;
        const int64_t rows = shared ? T : T * k;
        float4_t acc[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) acc[b] = float4_t{0.f, 0.f, 0.f, 0.f};
        const auto multiply = [&](auto Sets) __attribute__((always_inline)) {
            constexpr int SETS = Sets.value, U = (SETS == 1 ? 2 : 1) * (KIND == 4 ? 2 : 1);  // units in flight
            // the lane's column of hidden rows in each set; that of the expert's first token where it is none
            const uint16_t *h[SETS];
#pragma unroll
            for (int s = 0; s < SETS; ++s) {
                int t = someone, p = 0;
                if constexpr (SETS == 1) {
                    const int q = r / ntakers;
                    if (q < 3) {
                        uint32_t left = takers;
                        for (int i = r - q * ntakers; i > 0; --i) left &= left - 1;
                        t = __ffs(left) - 1;
                        p = q;
                    }
                } else if (r < T && (takers >> r & 1u)) {
                    t = r;
                    p = s;
                }
                const int64_t at_row = shared ? t : t * k + (s_rank[min(l, kMaxPairs - 1)][t >> 2] >> (8 * (t & 3)) & 255u);
                h[s] = hidden + (p * rows + at_row) * K;
            }
            for (int j0 = 0; j0 < n; j0 += U) {
                u32x4_t w[U][4][PIECES], x[U][SETS][4];
                uint32_t raw[U][4];
#pragma unroll
                for (int j = 0; j < U; ++j) {
                    const int u = first + min(j0 + j, n - 1);
                    const int block = min(4 * u + g, last);
                    // MXFP8: a read of the four lanes of a row is 64 bytes side by side, so a lane's 32 columns are 16 of either half of the unit
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
#pragma unroll
                        for (int q = 0; q < PIECES; ++q)
                            w[j][b][q] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t *>(wrow[b] + (KIND == 8 ? 128 * u + 64 * q + 16 * g : 16 * block)));
                        if (KIND == 4 || b == 0) raw[j][b] = KIND == 8 ? srow[0][u] : srow[b][static_cast<int64_t>(u >> 1) * 256 + (u & 1) * 4];
                    }
#pragma unroll
                    for (int s = 0; s < SETS; ++s)
#pragma unroll
                        for (int f = 0; f < 4; ++f)
                            x[j][s][f] = *reinterpret_cast<const u32x4_t *>(h[s] + (KIND == 8 ? 128 * u + 64 * (f >> 1) + 16 * g + 8 * (f & 1) : 32 * block + 8 * f));
                }
                asm volatile("" ::: "memory");  // all asked for before the first is used
#pragma unroll
                for (int j = 0; j < U; ++j) {
                    if (j0 + j >= n) break;
                    const bool none = KIND == 4 && 4 * (first + j0 + j) + g > last;  // columns behind the last
#pragma unroll
                    for (int s = 0; s < SETS; ++s)
#pragma unroll
                        for (int f = 0; f < 4; ++f) x[j][s][f] = none ? u32x4_t{0u, 0u, 0u, 0u} : x[j][s][f];
#pragma unroll
                    for (int b = 0; b < 4; ++b)
#pragma unroll
                        for (int f = 0; f < 4; ++f) {
                            u32x4_t v;
                            if constexpr (KIND == 8) v = mx_cvt_fp8<0>(w[j][b][f >> 1][2 * (f & 1)], w[j][b][f >> 1][2 * (f & 1) + 1], __uint_as_float(raw[j][0] << 23));
                            else v = mx_cvt_fp4<0>(w[j][b][0][f], __uint_as_float(raw[j][b] << 23));
#pragma unroll
                            for (int s = 0; s < SETS; ++s) acc[b] = mx_mfma<0>(x[j][s][f], v, acc[b]);
                        }
                }
            }
        };
        // Sums of a token are in its own column 4 g + i, or, side by side, in one a part: those go by way of the wave's place in LDS.
        float4_t got[4];
        if (!MANY || 3 * ntakers <= 16) {
            multiply(std::integral_constant<int, 1>{});
#pragma unroll
            for (int b = 0; b < 4; ++b) red[wave][b][lane] = acc[b];
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            const float *at_col = reinterpret_cast<const float *>(red[wave]) + 4 * r;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int nth = __popc(takers & ((1u << (4 * g + i)) - 1u));  // of the tokens in front; no more than five
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    float v = 0.f;
#pragma unroll
                    for (int p = 0; p < 3; ++p) {
                        const int c = p * ntakers + nth;
                        v += at_col[b * 256 + (c >> 2) * 64 + (c & 3)];
                    }
                    got[b][i] = v;
                }
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        } else if constexpr (MANY) {
            multiply(std::integral_constant<int, 3>{});
#pragma unroll
            for (int b = 0; b < 4; ++b) got[b] = acc[b];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int t = 4 * g + i;
            const bool takes = t < T && (takers >> t & 1u);
            float p = 1.f;
            if (!shared) p = s_weight[l][t];
            else if (a.shared_gate && takes) p = 1.f / (1.f + expf(-a.shared_gate[t]));
#pragma unroll
            for (int b = 0; b < 4; ++b) sum[b][i] = takes ? fmaf(p, got[b][i], sum[b][i]) : sum[b][i];
        }
        at += n;
        if (at == end) {
            at += (kDownWaves - 1) * run;
            end = min(at + run, hi);
        }
    }
#pragma unroll
    for (int b = 0; b < 4; ++b) red[wave][b][lane] = sum[b];
    __syncthreads();
    // what this block has of result o: token o / 64, row o % 64
    const auto own = [&](int o) {
        const int t = o >> 6, n = o & 63;
        const float *at = reinterpret_cast<const float *>(red) + (n >> 4) * 256 + ((t >> 2) * 16 + (n & 15)) * 4 + (t & 3);
        float v = 0.f;
        for (int w = 0; w < kDownWaves; ++w) v += at[w * 1024];
        return v;
    };
    const int live = min(kDownRows, H - group * kDownRows);
    if (a.pieces == 1) {
        for (int o = tid; o < T * 64; o += nt)
            if ((o & 63) < live) store_rounded(a.y, (o >> 6) * a.ldy + group * kDownRows + (o & 63), own(o), a.y_dtype);
        return;
    }
    // Blocks on other dies see these through memory: stores and loads of device scope, which pass by the caches that a die has to itself, and the
    // counter raised when the stores have arrived.  Fences of that scope would write those caches back and empty them: 50 us here.
    float *part = a.partial + static_cast<int64_t>(group) * a.pieces * (T * 64);
    for (int o = tid; o < T * 64; o += nt) __hip_atomic_store(part + piece * (T * 64) + o, own(o), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tid == 0) s_last = __hip_atomic_fetch_add(a.arrived + group, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == a.pieces - 1;
    __syncthreads();
    if (!s_last) return;
    asm volatile("" ::: "memory");
    for (int o = tid; o < T * 64; o += nt) {
        if ((o & 63) >= live) continue;
        float v[kMaxPieces], y = 0.f;
#pragma unroll
        for (int s = 0; s < kMaxPieces; ++s) v[s] = __hip_atomic_load(part + min(s, a.pieces - 1) * (T * 64) + o, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        for (int s = 0; s < kMaxPieces; ++s) y += s < a.pieces ? v[s] : 0.f;
        store_rounded(a.y, (o >> 6) * a.ldy + group * kDownRows + (o & 63), y, a.y_dtype);
    }
}

// ---- launches -------------------------------------------------------------------------------------------------------------------
template <int KIND, int NL, int SETS>
int launch_up(const LayerArgs &a, hipStream_t st) {
    using S = UpShape<KIND>;
    const int nlines = LineOf<KIND>::lines(a.w.hidden), nwaves = nlines < kUpWaves ? nlines : kUpWaves;
    const size_t lds = S::lds(nwaves);
    auto kern = mx_layer_up_kernel<KIND, NL, SETS>;
    static_assert(S::lds(kUpWaves) + sizeof(Selection) <= kMaxDynamicLds, "ring, sums and the selection");
    if (int rc = allow_dynamic_lds(reinterpret_cast<const void *>(kern), lds, "mx_moe_layer")) return rc;
    hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(device_cu_count())), dim3(64 * nwaves), lds, st, a);
    return check_launch("mx_moe_layer (gate and up)");
}
// up to 32 operands of activations stay in registers
template <int KIND, int SETS>
int launch_up_sets(const LayerArgs &a, hipStream_t st) {
    constexpr int MOST = 32 / (LineOf<KIND>::FR * SETS);
    const int64_t n = ceil_div(LineOf<KIND>::lines(a.w.hidden), kUpWaves);
    if constexpr (MOST >= 4)
        if (n <= MOST / 4) return launch_up<KIND, MOST / 4, SETS>(a, st);
    if (n <= MOST / 2) return launch_up<KIND, MOST / 2, SETS>(a, st);
    if (n <= MOST) return launch_up<KIND, MOST, SETS>(a, st);
    return launch_up<KIND, 0, SETS>(a, st);
}
template <int KIND>
int run_layer(const LayerArgs &a, hipStream_t st) {
    if (int rc = a.x_f16 && 2 * a.T > 16 ? launch_up_sets<KIND, 2>(a, st) : launch_up_sets<KIND, 1>(a, st)) return rc;
    const dim3 grid(static_cast<unsigned>(ceil_div(a.w.hidden, kDownRows) * a.pieces));
    if (3 * a.T > 16) hipLaunchKernelGGL((mx_layer_down_kernel<KIND, true>), grid, dim3(kDownWaves * 64), 0, st, a);
    else hipLaunchKernelGGL((mx_layer_down_kernel<KIND, false>), grid, dim3(kDownWaves * 64), 0, st, a);
    return check_launch("mx_moe_layer (down)");
}

int64_t up256(int64_t n) { return (n + 255) & ~static_cast<int64_t>(255); }
int64_t hidden_bytes(int64_t rows, int width) { return up256(3 * rows * width * 2); }
// pieces of the columns: as many as make a block for each compute unit
int pieces_of(int hidden) {
    const int64_t groups = ceil_div(hidden, kDownRows), n = device_cu_count() / groups;
    return static_cast<int>(n < 1 ? 1 : n > kMaxPieces ? kMaxPieces : n);
}
// the workspace: hidden rows, the shared expert's, the table, partial results and their counters
struct LayerSpace {
    int64_t shared_hidden, table, partial, arrived, bytes;
};
LayerSpace space_of(const mfq_mx_layer &w, int T, int k, int pieces) {
    LayerSpace s;
    const int64_t groups = ceil_div(w.hidden, kDownRows);
    s.shared_hidden = hidden_bytes(static_cast<int64_t>(T) * k, w.inter);
    s.table = s.shared_hidden + hidden_bytes(T, w.shared_inter);
    s.partial = s.table + up256(sizeof(LayerTable));
    s.arrived = s.partial + (pieces > 1 ? groups * pieces * T * 64 * 4 : 0);
    s.bytes = s.arrived + up256(groups * 4);
    return s;
}

}  // namespace
}  // namespace mfq

using namespace mfq;

extern "C" size_t mfq_hip_mx_moe_layer_workspace_bytes(const mfq_mx_layer *layer, int T, int k) {
    if (!layer || T < 1 || T > kMaxTokens || k < 1 || k > kMaxRoutes || layer->hidden < 1 || layer->inter < 1 || layer->shared_inter < 0) return 0;
    return static_cast<size_t>(space_of(*layer, T, k, pieces_of(layer->hidden)).bytes);
}

extern "C" int mfq_hip_mx_moe_layer(const mfq_mx_layer *layer, const void *x, int x_dtype, int64_t ldx, int T, const float *logits, const float *bias, int k, int mode,
                                    int normalize, float norm_floor, float scale, int activation, const float *shared_gate, int32_t *ids, float *weights, void *y,
                                    int y_dtype, int64_t ldy, void *workspace, size_t workspace_bytes, mfq_stream_t stream) {
    MFQ_REQUIRE(layer && x && logits && ids && weights && y, MFQ_ERR_INVALID, "mx_moe_layer: null argument");
    const mfq_mx_layer &w = *layer;
    MFQ_REQUIRE(w.kind == 4 || w.kind == 8, MFQ_ERR_INVALID, "mx_moe_layer: kind=%d (4 = MXFP4, 8 = MXFP8)", w.kind);
    MFQ_REQUIRE(w.gate_up && w.gate_up_scales && w.down && w.down_scales, MFQ_ERR_INVALID, "mx_moe_layer: null tensor");
    const int block = w.kind == 8 ? 128 : 32;
    MFQ_REQUIRE(w.experts > 0 && w.hidden > 0 && w.inter > 0 && w.shared_inter >= 0 && w.hidden % block == 0 && w.inter % block == 0 && w.shared_inter % block == 0,
                MFQ_ERR_INVALID, "mx_moe_layer: %d experts, widths %d, %d and %d must be divisible by %d", w.experts, w.hidden, w.inter, w.shared_inter, block);
    MFQ_REQUIRE(!w.shared_inter || (w.shared_gate_up && w.shared_gate_up_scales && w.shared_down && w.shared_down_scales), MFQ_ERR_INVALID,
                "mx_moe_layer: null tensor of the shared expert");
    MFQ_REQUIRE(w.experts <= kMaxExperts, MFQ_ERR_UNSUPPORTED, "mx_moe_layer: %d experts (at most %d)", w.experts, kMaxExperts);
    MFQ_REQUIRE(x_dtype == MFQ_X_BF16 || x_dtype == MFQ_X_F16, MFQ_ERR_INVALID, "mx_moe_layer: x_dtype=%d", x_dtype);
    MFQ_REQUIRE(y_dtype >= MFQ_X_BF16 && y_dtype <= MFQ_X_F32, MFQ_ERR_INVALID, "mx_moe_layer: y_dtype=%d", y_dtype);
    MFQ_REQUIRE(T >= 1 && T <= kMaxTokens, MFQ_ERR_UNSUPPORTED, "mx_moe_layer: %d tokens (1 to %d)", T, kMaxTokens);
    MFQ_REQUIRE(k >= 1 && k <= kMaxRoutes && k <= w.experts, MFQ_ERR_INVALID, "top_k must be in [1, min(16, experts)]");
    MFQ_REQUIRE(mode >= 0 && mode <= 3, MFQ_ERR_INVALID, "mx_moe_layer: unknown mode %d", mode);
    MFQ_REQUIRE(!(normalize && mode == MFQ_TOPK_DELAYED_SOFTMAX), MFQ_ERR_INVALID, "selected-weight normalization and delayed softmax are mutually exclusive");
    MFQ_REQUIRE(activation == MFQ_GLU_SILU || activation == MFQ_GLU_GELU, MFQ_ERR_INVALID, "mx_moe_layer: activation=%d", activation);
    MFQ_REQUIRE(T == 1 || (ldx >= w.hidden && ldy >= w.hidden), MFQ_ERR_INVALID, "mx_moe_layer: ldx=%lld or ldy=%lld < %d", static_cast<long long>(ldx),
                static_cast<long long>(ldy), w.hidden);
    const uintptr_t values = reinterpret_cast<uintptr_t>(w.gate_up) | reinterpret_cast<uintptr_t>(w.down) | reinterpret_cast<uintptr_t>(w.shared_gate_up) |
                             reinterpret_cast<uintptr_t>(w.shared_down);
    const uintptr_t scales = reinterpret_cast<uintptr_t>(w.gate_up_scales) | reinterpret_cast<uintptr_t>(w.down_scales) |
                             reinterpret_cast<uintptr_t>(w.shared_gate_up_scales) | reinterpret_cast<uintptr_t>(w.shared_down_scales);
    MFQ_REQUIRE(values % 16 == 0 && (w.kind == 8 || scales % 8 == 0) && reinterpret_cast<uintptr_t>(x) % 2 == 0 &&
                reinterpret_cast<uintptr_t>(y) % (y_dtype == MFQ_X_F32 ? 4 : 2) == 0, MFQ_ERR_INVALID, "mx_moe_layer: values must be 16-byte aligned, laid scales 8-byte aligned");
    const auto fits = [&](int64_t rows, int K) {
        return rows * K < (1ll << 32) && (w.kind == 8 ? (rows + 127) / 128 * (K / 128) : mx_scale_bytes(rows, K)) * 1ll < (1ll << 32) - 512;
    };
    const auto pool_fits = [&](int64_t rows, int K) { return (w.kind == 8 ? (rows + 127) / 128 * (K / 128) : mx_scale_bytes(rows, K)) < (1ll << 32) - 512; };
    MFQ_REQUIRE(fits(2ll * w.inter, w.hidden) && fits(2ll * w.shared_inter, w.hidden) && pool_fits(2ll * w.inter * w.experts, w.hidden) &&
                pool_fits(static_cast<int64_t>(w.hidden) * w.experts, w.inter), MFQ_ERR_UNSUPPORTED, "mx_moe_layer: %d experts of %d x %d", w.experts, w.inter, w.hidden);
    const size_t need = mfq_hip_mx_moe_layer_workspace_bytes(layer, T, k);
    MFQ_REQUIRE(workspace && workspace_bytes >= need, MFQ_ERR_WORKSPACE, "mx_moe_layer: workspace %zu < %zu", workspace_bytes, need);
    MFQ_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, MFQ_ERR_WORKSPACE, "mx_moe_layer: unaligned workspace");
    LayerArgs a = {};
    a.w = w;
    a.x = x;
    a.ldx = ldx;
    a.x_f16 = x_dtype == MFQ_X_F16;
    a.x_wide = reinterpret_cast<uintptr_t>(x) % 16 == 0 && (T == 1 || ldx % 8 == 0);
    a.T = T;
    a.k = k;
    a.mode = mode;
    a.normalize = normalize;
    a.gelu = activation == MFQ_GLU_GELU;
    a.logits = logits;
    a.bias = bias;
    a.shared_gate = shared_gate;
    a.norm_floor = norm_floor;
    a.scale = scale;
    a.ids = ids;
    a.weights = weights;
    a.y = y;
    a.y_dtype = y_dtype;
    a.ldy = ldy;
    a.pieces = pieces_of(w.hidden);
    const LayerSpace space = space_of(w, T, k, a.pieces);
    uint8_t *ws = static_cast<uint8_t *>(workspace);
    a.hidden = reinterpret_cast<uint16_t *>(ws);
    a.shared_hidden = reinterpret_cast<uint16_t *>(ws + space.shared_hidden);
    a.table = reinterpret_cast<LayerTable *>(ws + space.table);
    a.partial = reinterpret_cast<float *>(ws + space.partial);
    a.arrived = reinterpret_cast<int32_t *>(ws + space.arrived);
    return w.kind == 8 ? run_layer<8>(a, as_stream(stream)) : run_layer<4>(a, as_stream(stream));
}
