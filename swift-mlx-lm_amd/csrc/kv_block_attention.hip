// Attention over the 8-bit block KV cache.
//
// A query row of a KV head's group sees tokens low..position of its sequence; with per-block scales ks, vs and codes k, v
//   x_t = scale log2(e) ks (q . k_t),   w_t = 2^x_t / sum 2^x,   out = sum w_t vs v_t,   lse = ln 2 log2(sum 2^x_t).
// One pass over the cache with a running maximum.  What the 8-bit blocks change:
//  - Codes become f16 exactly (an int8 moved into the mantissa of 1024, minus its offset), and so do query rows, each
//    multiplied by the power of two that brings its largest element to [2^14, 2^15); products are exact, sums fp32.
//  - The values' scale joins the exponent: p_t = 2^(x_t + log2 vs - m) with m a maximum of x + log2 vs, so sum p_t v_t is
//    in units of 2^m whatever block a token is in, a weight is rounded to f16 relative to what it contributes, and
//    l = sum p_t / vs is gathered per block.  The maximum moves only when a score passes it by 2^8 (weights then reach
//    2^14 in f16), so accumulators are hardly ever rescaled.
//  - The score tile S^T = K Q^T leaves lane (n, c) = (lane % 16, lane / 16) with tokens 4c .. 4c + 3 of each sixteen for
//    query row n, which is the operand layout of out^T = V^T P^T given the order in which the cache stores values:
//    weights never leave their registers.
#include "kv_block.h"

namespace mi355q {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

struct AttentionArgs {
    KvBlockArgs kv;
    const void* q;
    void* out;
    float* lse;               // may be null
    uint32_t q_stride, out_stride, heads, group, window, q_dtype, out_dtype;
    float scale_log2;         // scale * log2(e)
    // partial results (parts > 1) of row slot ((sequence * kv_heads + head) * tiles + tile) * parts + part, 16 RT rows each
    uint32_t tiles, parts, part_blocks;
    float* part_out;          // [slot row][HD], in units of 2^m
    float2* part_ml;          // [slot row] (m, l)
    // weights wanted: scores in units of log2, [sequence * kv_heads + head][score_rows][score_stride], and each row's
    // log2 of the sum
    float* scores;
    float* lse2;
    uint32_t score_rows, score_stride;
};

constexpr float kLowest = -3.402823466e38f;
constexpr float kRaise = 8.0f, kHeadroom = 6.0f;      // log2: how far scores may pass m, and p = 2^6 at the maximum

// ---- the rows of a call ------------------------------------------------------------------------------------------------
// Row r of a KV head's rows: query token r / group, head r % group of the group.  Blocks [first, last) that rows
// [r0, r1) of a sequence see.
struct RowRange {
    int32_t low, high;        // positions of the first and the last row
    int32_t first, last;
};
__device__ __forceinline__ RowRange row_range(const AttentionArgs& a, const KvSequence& s, uint32_t r0, uint32_t r1) {
    RowRange g;
    g.low = s.first() + (int32_t)(r0 / a.group);
    g.high = s.first() + (int32_t)((r1 - 1) / a.group);
    const int64_t from = a.window ? max((int64_t)g.low - a.window + 1, (int64_t)0) : 0;
    g.first = (int32_t)(from / kKvTokens);
    g.last = g.high < 0 ? g.first : max(g.first, g.high / (int32_t)kKvTokens + 1);
    return g;
}
__device__ __forceinline__ uint32_t part_count(const AttentionArgs& a, const RowRange& g) {
    const uint32_t blocks = (uint32_t)(g.last - g.first);
    return blocks <= a.part_blocks ? 1u : (blocks + a.part_blocks - 1) / a.part_blocks;
}
// the lowest position that row r's window reaches (any number below the first token without one)
__device__ __forceinline__ int32_t row_low(const AttentionArgs& a, int32_t position) {
    return a.window && (int64_t)position >= (int64_t)a.window ? position - (int32_t)a.window + 1 : 0;
}

// ---- operands ----------------------------------------------------------------------------------------------------------
// Eight codes (already biased to c + 128) as f16: 0x64 in front of a byte is 1024 + byte.
__device__ __forceinline__ half8 codes_f16(uint32_t w0, uint32_t w1) {
    const half2v bias = {(_Float16)1152.0f, (_Float16)1152.0f};
    union { half2v h[4]; half8 v; } out;
    out.h[0] = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, w0, 0x04010400u)) - bias;
    out.h[1] = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, w0, 0x04030402u)) - bias;
    out.h[2] = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, w1, 0x04010400u)) - bias;
    out.h[3] = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, w1, 0x04030402u)) - bias;
    return out.v;
}
__device__ __forceinline__ u32x4 biased(u32x4 w) { return w ^ 0x80808080u; }

// Elements [d0, d0 + 16) of a query row as fp32 (zeros for a row that is not there).
__device__ __forceinline__ void load_query16(const AttentionArgs& a, bool there, size_t at, float (&x)[16]) {
    if (!there) {
#pragma unroll
        for (int e = 0; e < 16; e++) x[e] = 0.0f;
        return;
    }
    const uint16_t* const p = (const uint16_t*)a.q + at;
    uint32_t w[8];
    if (((uintptr_t)p & 15) == 0) {
        const u32x4 lo = *(const u32x4*)p, hi = *(const u32x4*)(p + 8);
        w[0] = lo.x; w[1] = lo.y; w[2] = lo.z; w[3] = lo.w; w[4] = hi.x; w[5] = hi.y; w[6] = hi.z; w[7] = hi.w;
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) w[e] = (uint32_t)p[2 * e] | ((uint32_t)p[2 * e + 1] << 16);
    }
#pragma unroll
    for (int e = 0; e < 16; e++) {
        const uint16_t h = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
        x[e] = a.q_dtype == MI355Q_BF16 ? bf16_to_f32(h) : f16_to_f32(h);
    }
}

// The power of two that brings a largest magnitude `top` to [2^14, 2^15), and its inverse.  Zero and the smallest numbers
// take 2^126; infinities and NaN 1 (they stay what they are).
__device__ __forceinline__ void row_power(float top, float& up, float& down) {
    const uint32_t e = __float_as_uint(top) >> 23;
    uint32_t f = 268u - e;
    f = f > 253u ? 253u : f;
    f = e == 255u ? 127u : f;
    up = __uint_as_float(f << 23);
    down = __uint_as_float((254u - f) << 23);
}

__device__ __forceinline__ float max_across(float v, uint32_t) {      // over lane groups of sixteen: lanes l, l^16, l^32, l^48
    v = fmaxf(v, lane_xor<16>(v));
    return fmaxf(v, lane_xor<32>(v));
}
__device__ __forceinline__ float sum_across(float v) {
    v += lane_xor<16>(v);
    return v + lane_xor<32>(v);
}

template <int D>
__device__ __forceinline__ void store4(void* p, size_t at, const floatx4& v, float f) {
    const float x[4] = {v.x * f, v.y * f, v.z * f, v.w * f};
    uint32_t w[2];
#pragma unroll
    for (int e = 0; e < 2; e++) {
        const uint16_t lo = D == MI355Q_BF16 ? f32_to_bf16_rne(x[2 * e]) : f32_to_f16_rne(x[2 * e]);
        const uint16_t hi = D == MI355Q_BF16 ? f32_to_bf16_rne(x[2 * e + 1]) : f32_to_f16_rne(x[2 * e + 1]);
        w[e] = (uint32_t)lo | ((uint32_t)hi << 16);
    }
    uint16_t* const q = (uint16_t*)p + at;
    if (((uintptr_t)q & 7) == 0) {
        *(uint2*)q = make_uint2(w[0], w[1]);
    } else {
        q[0] = (uint16_t)w[0]; q[1] = (uint16_t)(w[0] >> 16); q[2] = (uint16_t)w[1]; q[3] = (uint16_t)(w[1] >> 16);
    }
}
__device__ __forceinline__ void store_row4(const AttentionArgs& a, size_t at, const floatx4& v, float f) {
    if (a.out_dtype == MI355Q_BF16) store4<MI355Q_BF16>(a.out, at, v, f);
    else store4<MI355Q_F16>(a.out, at, v, f);
}

// ---- few rows: decode steps and short verifications --------------------------------------------------------------------
// A workgroup takes one KV head, 16 RT rows and one part of the visible blocks; its four wavefronts take blocks in turn,
// each with accumulators of its own, which are added at the end.  HBM-bound.
template <int HD, int RT>
__global__ __launch_bounds__(256, 2) void kv_block_attention_rows_kernel(AttentionArgs a) {
    constexpr int S = HD / 64, DT = HD / 16;
    __shared__ __align__(16) float lds_out[2][16 * RT * HD];
    __shared__ float2 lds_ml[4][16 * RT];
    const uint32_t lane = threadIdx.x & 63, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t n = lane & 15, c = lane >> 4;
    const uint32_t head = blockIdx.x % a.kv.kv_heads, part = blockIdx.x / a.kv.kv_heads, tile = blockIdx.y, b = blockIdx.z;
    const KvSequence s = kv_sequence(a.kv, b);
    const uint32_t rows = (uint32_t)s.rows * a.group, r0 = tile * 16 * RT;
    if (r0 >= rows) return;
    const uint32_t r1 = min(r0 + 16 * RT, rows);
    const RowRange g = row_range(a, s, r0, r1);
    const uint32_t parts = part_count(a, g);
    if (part >= parts) return;

    half8 q[RT][S][2];
    float factor[RT], m[RT], l[RT];
    int32_t position[RT], low[RT];
    floatx4 o[RT][DT];
#pragma unroll
    for (int t = 0; t < RT; t++) {
        const uint32_t r = r0 + t * 16 + n;
        const bool there = r < r1;
        const uint32_t token = r / a.group, h = head * a.group + r % a.group;
        position[t] = s.first() + (int32_t)token;
        low[t] = row_low(a, position[t]);
        float x[S][16], top = 0.0f;
#pragma unroll
        for (int i = 0; i < S; i++) {
            load_query16(a, there, (size_t)(s.row0 + (int32_t)token) * a.q_stride + (size_t)h * HD + i * 64 + c * 16, x[i]);
#pragma unroll
            for (int e = 0; e < 16; e++) top = fmaxf(top, fabsf(x[i][e]));
        }
        float up, down;
        row_power(max_across(top, lane), up, down);
        factor[t] = a.scale_log2 * down;
#pragma unroll
        for (int i = 0; i < S; i++)
#pragma unroll
            for (int e = 0; e < 16; e++) q[t][i][e >> 3][e & 7] = (_Float16)(x[i][e] * up);
        m[t] = kLowest;
        l[t] = 0.0f;
#pragma unroll
        for (int d = 0; d < DT; d++) o[t][d] = floatx4{0, 0, 0, 0};
    }

    const int32_t end = min(g.first + (int32_t)((part + 1) * a.part_blocks), g.last);
    for (int32_t j = g.first + (int32_t)(part * a.part_blocks + wave); j < end; j += 4) {
        const int32_t block = kv_block_id(a.kv, s.table, j);
        const int32_t base = j * (int32_t)kKvTokens;
        if (block < 0) {
            if (a.scores) {
#pragma unroll
                for (int t = 0; t < RT; t++)
                    if (r0 + t * 16 + n < r1)
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            *(floatx4*)(a.scores + ((size_t)(b * a.kv.kv_heads + head) * a.score_rows + r0 + t * 16 + n) * a.score_stride +
                                        base + k * 16 + c * 4) = floatx4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            }
            continue;
        }
        const u32x4* const kp = (const u32x4*)kv_codes<HD>(a.kv, block, head, 0) + lane;
        const u32x4* const vp = (const u32x4*)kv_codes<HD>(a.kv, block, head, 1) + lane;
        u32x4 kw[4][S], vw[DT];
#pragma unroll
        for (int k = 0; k < 4; k++)
#pragma unroll
            for (int i = 0; i < S; i++) kw[k][i] = kp[(k * S + i) * 64];
#pragma unroll
        for (int d = 0; d < DT; d++) vw[d] = vp[d * 64];
        const float ks = *kv_scale(a.kv, block, head, 0), vs = *kv_scale(a.kv, block, head, 1);
        const float vlog = vs > 0.0f ? log2f(vs) : 0.0f, vinv = vs > 0.0f ? exp2f(-vlog) : 1.0f;
        floatx4 x[RT][4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
#pragma unroll
            for (int t = 0; t < RT; t++) x[t][k] = floatx4{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < S; i++) {
                const u32x4 w = biased(kw[k][i]);
                const half8 lo = codes_f16(w.x, w.y), hi = codes_f16(w.z, w.w);
#pragma unroll
                for (int t = 0; t < RT; t++) {
                    x[t][k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, q[t][i][0], x[t][k], 0, 0, 0);
                    x[t][k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, q[t][i][1], x[t][k], 0, 0, 0);
                }
            }
        }
        // every row sees the whole block?
        const bool whole = base + 63 <= g.low && (!a.window || base >= row_low(a, g.high));
        half8 p[RT][2];
#pragma unroll
        for (int t = 0; t < RT; t++) {
            const float f = factor[t] * ks;
            float top = kLowest;
#pragma unroll
            for (int k = 0; k < 4; k++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    float v = x[t][k][i] * f;
                    if (!whole) {
                        const int32_t at = base + k * 16 + (int32_t)c * 4 + i;
                        v = at >= low[t] && at <= position[t] ? v : -INFINITY;
                    }
                    x[t][k][i] = v;
                    top = fmaxf(top, v);
                }
            if (a.scores && r0 + t * 16 + n < r1) {
                float* const at = a.scores + ((size_t)(b * a.kv.kv_heads + head) * a.score_rows + r0 + t * 16 + n) * a.score_stride + base + c * 4;
#pragma unroll
                for (int k = 0; k < 4; k++) *(floatx4*)(at + k * 16) = x[t][k];
            }
            top += vlog - kHeadroom;
            if (__ballot(top > m[t] + kRaise)) {
                const float raised = fmaxf(m[t], max_across(top, lane));
                const float shrink = exp2f(m[t] - raised);
                l[t] *= shrink;
#pragma unroll
                for (int d = 0; d < DT; d++) o[t][d] *= shrink;
                m[t] = raised;
            }
            const float shift = vlog - m[t];
            float sum = 0.0f;
#pragma unroll
            for (int k = 0; k < 4; k++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float w = __builtin_amdgcn_exp2f(x[t][k][i] + shift);
                    sum += w;
                    p[t][k >> 1][(k & 1) * 4 + i] = (_Float16)w;
                }
            l[t] += sum * vinv;
        }
#pragma unroll
        for (int d = 0; d < DT; d++) {
            const u32x4 w = biased(vw[d]);
            const half8 lo = codes_f16(w.x, w.y), hi = codes_f16(w.z, w.w);
#pragma unroll
            for (int t = 0; t < RT; t++) {
                o[t][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, p[t][0], o[t][d], 0, 0, 0);
                o[t][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, p[t][1], o[t][d], 0, 0, 0);
            }
        }
    }

    // the four wavefronts' results: to a common maximum, then added pairwise through LDS in a fixed order
#pragma unroll
    for (int t = 0; t < RT; t++) {
        l[t] = sum_across(l[t]);
        if (c == 0) lds_ml[wave][t * 16 + n] = make_float2(m[t], l[t]);
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < RT; t++) {
        float top = kLowest;
#pragma unroll
        for (int w = 0; w < 4; w++) top = fmaxf(top, lds_ml[w][t * 16 + n].x);
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; w++) sum += lds_ml[w][t * 16 + n].y * exp2f(lds_ml[w][t * 16 + n].x - top);
        const float f = exp2f(m[t] - top);
        m[t] = top;
        l[t] = sum;
#pragma unroll
        for (int d = 0; d < DT; d++) o[t][d] *= f;
    }
#pragma unroll
    for (int half = 2; half >= 1; half >>= 1) {
        if (wave >= (uint32_t)half && wave < (uint32_t)(2 * half)) {
#pragma unroll
            for (int t = 0; t < RT; t++)
#pragma unroll
                for (int d = 0; d < DT; d++) *(floatx4*)&lds_out[wave - half][((t * DT + d) * 64 + lane) * 4] = o[t][d];
        }
        __syncthreads();
        if (wave < (uint32_t)half) {
#pragma unroll
            for (int t = 0; t < RT; t++)
#pragma unroll
                for (int d = 0; d < DT; d++) o[t][d] += *(const floatx4*)&lds_out[wave][((t * DT + d) * 64 + lane) * 4];
        }
        __syncthreads();
    }
    if (wave) return;
#pragma unroll
    for (int t = 0; t < RT; t++) {
        const uint32_t r = r0 + t * 16 + n;
        if (r >= r1) continue;
        if (parts > 1) {
            const size_t slot = ((((size_t)b * a.kv.kv_heads + head) * a.tiles + tile) * a.parts + part) * (16 * RT) + t * 16 + n;
#pragma unroll
            for (int d = 0; d < DT; d++) *(floatx4*)(a.part_out + slot * HD + d * 16 + c * 4) = o[t][d];
            if (c == 0) a.part_ml[slot] = make_float2(m[t], l[t]);
            continue;
        }
        const uint32_t token = r / a.group, h = head * a.group + r % a.group;
        const size_t row = (size_t)(s.row0 + (int32_t)token);
        const float f = l[t] == 0.0f ? 0.0f : 1.0f / l[t];
#pragma unroll
        for (int d = 0; d < DT; d++) store_row4(a, row * a.out_stride + (size_t)h * HD + d * 16 + c * 4, o[t][d], f);
        if (c == 0) {
            const float lse2 = l[t] == 0.0f ? -INFINITY : m[t] + log2f(l[t]);
            if (a.lse) a.lse[row * a.heads + h] = lse2 * 0.6931471805599453f;
            if (a.scores) a.lse2[((size_t)b * a.kv.kv_heads + head) * a.score_rows + r] = lse2;
        }
    }
}

// Joins the parts of a row: one wavefront per row.
template <int HD>
__global__ __launch_bounds__(64) void kv_block_attention_join_kernel(AttentionArgs a, uint32_t tile_rows) {
    constexpr int E = HD / 64;
    const uint32_t lane = threadIdx.x, head = blockIdx.y, b = blockIdx.z, r = blockIdx.x;
    const KvSequence s = kv_sequence(a.kv, b);
    const uint32_t rows = (uint32_t)s.rows * a.group;
    if (r >= rows) return;
    const uint32_t tile = r / tile_rows, r0 = tile * tile_rows;
    const uint32_t parts = part_count(a, row_range(a, s, r0, min(r0 + tile_rows, rows)));
    if (parts == 1) return;
    const size_t slot = (((size_t)b * a.kv.kv_heads + head) * a.tiles + tile) * a.parts * tile_rows + (r - r0);
    float top = kLowest;
    for (uint32_t p = 0; p < parts; p++) top = fmaxf(top, a.part_ml[slot + (size_t)p * tile_rows].x);
    float l = 0.0f, o[E];
#pragma unroll
    for (int e = 0; e < E; e++) o[e] = 0.0f;
    for (uint32_t p = 0; p < parts; p++) {
        const size_t at = slot + (size_t)p * tile_rows;
        const float2 ml = a.part_ml[at];
        const float f = exp2f(ml.x - top);
        l += ml.y * f;
#pragma unroll
        for (int e = 0; e < E; e++) o[e] += a.part_out[at * HD + e * 64 + lane] * f;
    }
    const uint32_t token = r / a.group, h = head * a.group + r % a.group;
    const size_t row = (size_t)(s.row0 + (int32_t)token);
    const float f = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int e = 0; e < E; e++) {
        const size_t at = row * a.out_stride + (size_t)h * HD + e * 64 + lane;
        if (a.out_dtype == MI355Q_BF16) ((uint16_t*)a.out)[at] = f32_to_bf16_rne(o[e] * f);
        else ((uint16_t*)a.out)[at] = f32_to_f16_rne(o[e] * f);
    }
    if (lane == 0) {
        const float lse2 = l == 0.0f ? -INFINITY : top + log2f(l);
        if (a.lse) a.lse[row * a.heads + h] = lse2 * 0.6931471805599453f;
        if (a.scores) a.lse2[((size_t)b * a.kv.kv_heads + head) * a.score_rows + r] = lse2;
    }
}

// Weight sums from the stored scores: a thread per token, over the rows of its KV head that see it.
__global__ __launch_bounds__(256) void kv_block_weights_kernel(AttentionArgs a) {
    const uint32_t head = blockIdx.y, b = blockIdx.z;
    const KvSequence s = kv_sequence(a.kv, b);
    const int32_t t = (int32_t)(blockIdx.x * 256 + threadIdx.x);
    if (t >= s.length || s.rows <= 0) return;
    const int32_t block = kv_block_id(a.kv, s.table, t / (int32_t)kKvTokens);
    if (block < 0) return;
    const uint32_t rows = (uint32_t)s.rows * a.group;
    const size_t slot = ((size_t)b * a.kv.kv_heads + head) * a.score_rows;
    float sum = 0.0f;
    for (uint32_t r = 0; r < rows; r++) {
        const int32_t position = s.first() + (int32_t)(r / a.group);
        if (t > position || t < row_low(a, position)) continue;
        sum += exp2f(a.scores[(slot + r) * a.score_stride + t] - a.lse2[slot + r]);
    }
    kv_sums(a.kv, block, head)[t % (int32_t)kKvTokens] += sum;
}

namespace {

struct Buffers {
    char* at;
    size_t used;
    template <typename T>
    T* take(size_t count) {
        T* const p = (T*)(at ? at + used : nullptr);
        used += (count * sizeof(T) + 255) & ~(size_t)255;
        return p;
    }
};

template <int HD, int RT>
mi355q_status launch_rows(mi355q_context* ctx, hipStream_t s, AttentionArgs a, bool weights) {
    const uint32_t rows = a.kv.max_rows * a.group;
    a.tiles = (rows + 16 * RT - 1) / (16 * RT);
    uint64_t blocks = (a.kv.max_length + kKvTokens - 1) / kKvTokens;
    if (a.window) {
        const uint64_t reach = ((uint64_t)a.window + 16 * RT / a.group + 1 + kKvTokens - 2) / kKvTokens + 1;
        if (reach < blocks) blocks = reach;
    }
    const uint64_t groups = (uint64_t)a.kv.kv_heads * a.tiles * a.kv.sequences;
    uint64_t parts = (1536 + groups - 1) / groups;
    if (parts > (blocks + 3) / 4) parts = (blocks + 3) / 4;
    if (parts > 64) parts = 64;
    a.part_blocks = (uint32_t)(((blocks + parts - 1) / parts + 3) / 4 * 4);
    a.parts = (uint32_t)((blocks + a.part_blocks - 1) / a.part_blocks);
    a.score_rows = rows;
    a.score_stride = (uint32_t)((a.kv.max_length + kKvTokens - 1) / kKvTokens * kKvTokens);
    for (int pass = 0; pass < 2; pass++) {
        Buffers buf{pass ? (char*)ctx->workspace : nullptr, 0};
        if (a.parts > 1) {
            a.part_out = buf.take<float>(groups * a.parts * 16 * RT * HD);
            a.part_ml = buf.take<float2>(groups * a.parts * 16 * RT);
        }
        if (weights) {
            a.scores = buf.take<float>((size_t)a.kv.sequences * a.kv.kv_heads * rows * a.score_stride);
            a.lse2 = buf.take<float>((size_t)a.kv.sequences * a.kv.kv_heads * rows);
        }
        if (!pass && buf.used)
            if (mi355q_status st = ensure_workspace(ctx, buf.used)) return st;
    }
    kv_block_attention_rows_kernel<HD, RT><<<dim3(a.kv.kv_heads * a.parts, a.tiles, a.kv.sequences), 256, 0, s>>>(a);
    MI355Q_HIP(hipGetLastError());
    if (a.parts > 1) {
        kv_block_attention_join_kernel<HD><<<dim3(rows, a.kv.kv_heads, a.kv.sequences), 64, 0, s>>>(a, 16 * RT);
        MI355Q_HIP(hipGetLastError());
    }
    if (weights) {
        kv_block_weights_kernel<<<dim3((a.kv.max_length + 255) / 256, a.kv.kv_heads, a.kv.sequences), 256, 0, s>>>(a);
        MI355Q_HIP(hipGetLastError());
    }
    return MI355Q_OK;
}

}  // namespace
}  // namespace mi355q

using namespace mi355q;

extern "C" mi355q_status mi355q_kv_block_attention(mi355q_context* ctx, void* stream, const mi355q_kv_block_cache* cache,
                                                   const mi355q_kv_sequences* sequences, const void* q_dev,
                                                   mi355q_dtype q_dtype, uint32_t q_row_stride, uint32_t head_count,
                                                   float scale, uint32_t window, void* out_dev, mi355q_dtype out_dtype,
                                                   uint32_t out_row_stride, float* lse_dev, int accumulate_weights) {
    AttentionArgs a{};
    if (mi355q_status st = kv_block_prepare(ctx, cache, sequences, true, &a.kv)) return st;
    if (!q_dev || !out_dev) return fail(MI355Q_ERR_INVALID_ARGUMENT, "null queries or output");
    if ((q_dtype != MI355Q_F16 && q_dtype != MI355Q_BF16) || (out_dtype != MI355Q_F16 && out_dtype != MI355Q_BF16))
        return fail(MI355Q_ERR_INVALID_ARGUMENT, "attention takes and gives f16 or bf16 rows (got types %d and %d)", (int)q_dtype, (int)out_dtype);
    if (!head_count || head_count % a.kv.kv_heads)
        return fail(MI355Q_ERR_SHAPE, "%u query heads do not share %u KV heads evenly", head_count, a.kv.kv_heads);
    if (head_count > 32767) return fail(MI355Q_ERR_SHAPE, "%u query heads: at most 32767", head_count);
    const uint64_t width = (uint64_t)head_count * cache->head_dimension;
    if (q_row_stride == 0) q_row_stride = (uint32_t)width;
    if (out_row_stride == 0) out_row_stride = (uint32_t)width;
    if (q_row_stride < width || out_row_stride < width)
        return fail(MI355Q_ERR_SHAPE, "row strides %u and %u: shorter than heads x head dimension = %llu", q_row_stride, out_row_stride, (unsigned long long)width);
    if (!(scale > 0.0f) || scale > 1e30f) return fail(MI355Q_ERR_INVALID_ARGUMENT, "the scale must be a positive number (got %g)", (double)scale);
    if ((uintptr_t)q_dev % 2 || (uintptr_t)out_dev % 2 || (uintptr_t)lse_dev % 4) return fail(MI355Q_ERR_INVALID_ARGUMENT, "misaligned pointer");
    if (accumulate_weights && !a.kv.sums) return fail(MI355Q_ERR_INVALID_ARGUMENT, "the cache has no weight sums to add to");
    MI355Q_HIP(hipSetDevice(ctx->device));
    ScratchGuard guard(ctx, (hipStream_t)stream);
    if (guard.status) return guard.status;
    a.q = q_dev; a.out = out_dev; a.lse = lse_dev;
    a.q_stride = q_row_stride; a.out_stride = out_row_stride;
    a.heads = head_count; a.group = head_count / a.kv.kv_heads; a.window = window;
    a.q_dtype = (uint32_t)q_dtype; a.out_dtype = (uint32_t)out_dtype; a.scale_log2 = scale * 1.4426950408889634f;
    return kv_with_head_dimension(cache->head_dimension, [&](auto hd) -> mi355q_status {
        constexpr int HD = decltype(hd)::value;
        return launch_rows<HD, 1>(ctx, (hipStream_t)stream, a, accumulate_weights != 0);
    });
}
