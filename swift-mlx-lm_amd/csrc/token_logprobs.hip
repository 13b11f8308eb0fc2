// Log probability of a given token, entropy and the likeliest alternatives of rows of logits: one pass over the logits.
//
// With z = x - m and m the largest logit seen, a lane carries l = sum e^z and t = sum e^z z, which move to a larger
// maximum m' by e^(m - m') and t' = e^(m - m') (t + (m - m') l).  Then log softmax(x)_i = x_i - m - log l and the entropy
// is log l - t / l.  HBM-bound: a logit is read once; about ten vector instructions each, one of them an exponential.
//
// Alternatives: logits are ordered by 64-bit keys (ordered value, ~index), all distinct, so equal logits need no rule of
// their own.  A wavefront keeps a threshold that at least top_count of the logits it has seen reach; keys above it are
// collected in LDS and cut back to the top_count largest when the room runs out and at the end.  The first threshold is
// the top_count-th largest of the 64 lanes' maxima, so that of the first 1024 logits a few dozen are collected and of
// later ones only those that still belong to the largest.
#include "device_utils.h"

namespace mi355q {

constexpr uint32_t kTopMost = 32;                    // alternatives a row
constexpr uint32_t kTopRoom = 256;                   // keys a wavefront collects
constexpr uint32_t kLogprobLane = 16;                // logits of a lane per step
constexpr uint32_t kLogprobStep = 256 * kLogprobLane;
constexpr float kMasked = -INFINITY, kLargest = 3.402823466e38f;

struct LogprobArgs {
    const void* logits;
    const int32_t* tokens;
    float* logprob;
    float* entropy;
    int32_t* top_ids;
    float* top_logprobs;
    uint32_t rows, vocabulary, row_stride, top, slices, slice_length;
    // partial results of a slice: (m, l, t, unused), then `top` keys, largest first (0: none)
    float4* parts;
    unsigned long long* part_keys;
};

__device__ __forceinline__ unsigned long long logit_key(float v, uint32_t index) {
    const uint32_t u = __float_as_uint(v + 0.0f);   // -0 ranks like 0
    return ((unsigned long long)((u & 0x80000000u) ? ~u : u | 0x80000000u) << 32) | (uint32_t)~index;
}
__device__ __forceinline__ float key_logit(unsigned long long key) {
    const uint32_t u = (uint32_t)(key >> 32);
    return __uint_as_float((u & 0x80000000u) ? u ^ 0x80000000u : ~u);
}
constexpr unsigned long long kMaskedKey = ((unsigned long long)0x007FFFFFu << 32) | 0xFFFFFFFFu;   // no -inf is above it

// orders a wavefront's own accesses to its part of LDS
__device__ __forceinline__ void wave_lds_order() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

struct TopKeys {
    unsigned long long* room;                        // kTopRoom keys of LDS, this wavefront's
    unsigned long long threshold;
    uint32_t count, top, lane;

    // Cuts the collection back to its `top` largest keys, in order: every lane counts the keys above its own.
    __device__ void cut() {
        wave_lds_order();
        unsigned long long own[kTopRoom / 64];
        uint32_t rank[kTopRoom / 64];
#pragma unroll
        for (uint32_t i = 0; i < kTopRoom / 64; i++) {
            own[i] = i * 64 + lane < count ? room[i * 64 + lane] : 0;
            rank[i] = 0;
        }
        for (uint32_t k = 0; k < count; k++) {
            const unsigned long long other = room[k];
#pragma unroll
            for (uint32_t i = 0; i < kTopRoom / 64; i++) rank[i] += other > own[i] ? 1u : 0u;
        }
        wave_lds_order();
#pragma unroll
        for (uint32_t i = 0; i < kTopRoom / 64; i++)
            if (i * 64 + lane < count && rank[i] < top) room[rank[i]] = own[i];
        wave_lds_order();
        if (count >= top) {
            count = top;
            const unsigned long long last = room[top - 1];
            threshold = last > threshold ? last : threshold;
        }
    }
    // one key of each lane (0: none)
    __device__ void push(unsigned long long key) {
        uint64_t mask = __ballot(key > threshold);
        if (!mask) return;
        if (count + 64 > kTopRoom) {
            cut();
            mask = __ballot(key > threshold);
        }
        if (key > threshold) room[count + (uint32_t)__popcll(mask & ((1ull << lane) - 1))] = key;
        count += (uint32_t)__popcll(mask);
    }
};

struct LogSum {
    float m, l, t;
    __device__ void join(float om, float ol, float ot) {
        const float top = fmaxf(m, om), safe = fmaxf(top, -kLargest);
        const float d0 = fmaxf(m - safe, -1e4f), d1 = fmaxf(om - safe, -1e4f);
        const float f0 = __expf(d0), f1 = __expf(d1);
        t = f0 * (t + d0 * l) + f1 * (ot + d1 * ol);
        l = f0 * l + f1 * ol;
        m = top;
    }
};

// The row's results from its sums and its largest keys (`keys`: `top` of them, 0: none), by one wavefront.
template <int D>
__device__ void write_row(const LogprobArgs& a, uint32_t row, const LogSum& s, const unsigned long long* keys, uint32_t lane) {
    const bool some = s.l > 0.0f;
    const float log_l = some ? logf(s.l) : 0.0f;
    if (lane == 0 && a.logprob) {
        const int32_t token = a.tokens[row];
        float v = kMasked;
        if (some && (uint32_t)token < a.vocabulary) {
            const float x = load_act<D>(a.logits, (size_t)row * a.row_stride + (uint32_t)token);
            v = x != x ? kMasked : fminf(x, kLargest) - s.m - log_l;
        }
        a.logprob[row] = v;
    }
    if (lane == 0 && a.entropy) a.entropy[row] = some ? log_l - s.t / s.l : 0.0f;
    if (lane < a.top) {
        const unsigned long long key = keys[lane];
        a.top_ids[(size_t)row * a.top + lane] = key ? (int32_t)~(uint32_t)key : -1;
        a.top_logprobs[(size_t)row * a.top + lane] = key ? key_logit(key) - s.m - log_l : kMasked;
    }
}

// One workgroup per slice of a row; its wavefronts take steps of 1024 logits in turn.
template <int D>
__global__ __launch_bounds__(256) void token_logprobs_kernel(LogprobArgs a) {
    __shared__ unsigned long long room[4][kTopRoom];
    __shared__ float maxima[4][64];
    __shared__ LogSum sums[4];
    __shared__ uint32_t counts[4];
    constexpr uint32_t VE = D == MI355Q_F32 ? 4 : 8;             // logits of a 16-byte load
    const uint32_t row = blockIdx.x / a.slices, slice = blockIdx.x - row * a.slices;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t size = D == MI355Q_F32 ? 4 : 2;
    const size_t row_at = (size_t)row * a.row_stride;
    // steps start at 16-byte boundaries: `lead` elements in front of the row are skipped in its first one
    const uint32_t lead = (uint32_t)(((uintptr_t)a.logits + row_at * size) % 16) / size;
    const uint32_t begin = slice * a.slice_length, end = min(begin + a.slice_length, a.vocabulary + lead);
    TopKeys keys{room[wave], kMaskedKey, 0, a.top, lane};
    LogSum s{kMasked, 0.0f, 0.0f};
    bool first = true;
    for (uint32_t at = begin + wave * (64 * kLogprobLane); at < end; at += kLogprobStep) {
        float x[kLogprobLane];
        if (at >= lead && at + 64 * kLogprobLane <= a.vocabulary + lead) {
#pragma unroll
            for (uint32_t i = 0; i < kLogprobLane / VE; i++) {
                const size_t p = row_at + (at - lead) + i * (64 * VE) + lane * VE;
                if constexpr (D == MI355Q_F32) {
                    const float4 w = *(const float4*)((const float*)a.logits + p);
                    x[4 * i] = w.x; x[4 * i + 1] = w.y; x[4 * i + 2] = w.z; x[4 * i + 3] = w.w;
                } else {
                    const uint4 w = *(const uint4*)((const uint16_t*)a.logits + p);
                    const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const uint16_t h = (uint16_t)(ws[e >> 1] >> (16 * (e & 1)));
                        x[8 * i + e] = D == MI355Q_BF16 ? bf16_to_f32(h) : f16_to_f32(h);
                    }
                }
            }
        } else {
#pragma unroll
            for (uint32_t i = 0; i < kLogprobLane; i++) {
                const uint32_t p = at + i / VE * (64 * VE) + lane * VE + i % VE;
                x[i] = p >= lead && p < a.vocabulary + lead ? load_act<D>(a.logits, row_at + (p - lead)) : kMasked;
            }
        }
        // a NaN is dropped by every maximum: by this one, by the clamp of z below (e^z = 0) and by `x > kMasked` of the keys
        float top = kMasked;
#pragma unroll
        for (uint32_t i = 0; i < kLogprobLane; i++) top = fmaxf(top, x[i]);
        if (__ballot(top == INFINITY)) {
#pragma unroll
            for (uint32_t i = 0; i < kLogprobLane; i++) x[i] = x[i] == INFINITY ? kLargest : x[i];
            top = fminf(top, kLargest);
        }
        const float m = fmaxf(s.m, top), safe = fmaxf(m, -kLargest);
        float l = 0.0f, t = 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < kLogprobLane; i++) {
            const float z = fmaxf(x[i] - safe, -1e4f), e = __expf(z);
            l += e;
            t += e * z;
        }
        const float d = fmaxf(s.m - safe, -1e4f), f = __expf(d);
        s.t = f * (s.t + d * s.l) + t;
        s.l = f * s.l + l;
        s.m = m;
        if (a.top) {
            if (first) {                             // the top-th largest of the lanes' maxima
                maxima[wave][lane] = top;
                wave_lds_order();
                uint32_t above = 0;
                for (uint32_t k = 0; k < 64; k++) {
                    const float other = maxima[wave][k];
                    above += other > top || (other == top && k < lane) ? 1u : 0u;
                }
                const uint64_t last = __ballot(above == a.top - 1);
                const float limit = __shfl(top, (int)__builtin_ctzll(last));
                const unsigned long long key = logit_key(limit, 0xFFFFFFFFu);
                keys.threshold = key > kMaskedKey ? key : kMaskedKey;
                first = false;
            }
            const float limit = key_logit(keys.threshold);
            if (__ballot(top >= limit && top > kMasked)) {
#pragma unroll
                for (uint32_t i = 0; i < kLogprobLane; i++)
                    keys.push(x[i] > kMasked ? logit_key(x[i], at - lead + i / VE * (64 * VE) + lane * VE + i % VE) : 0);
            }
        }
    }
    if (a.top) keys.cut();
    // lanes, then wavefronts
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        const float om = __shfl_xor(s.m, o), ol = __shfl_xor(s.l, o), ot = __shfl_xor(s.t, o);
        s.join(om, ol, ot);
    }
    if (lane == 0) {
        sums[wave] = s;
        counts[wave] = keys.count;
    }
    __syncthreads();
    if (wave) return;
    for (uint32_t w = 1; w < 4; w++) s.join(sums[w].m, sums[w].l, sums[w].t);
    if (a.top) {
        for (uint32_t w = 1; w < 4; w++) keys.push(lane < counts[w] ? room[w][lane] : 0);
        keys.cut();
        if (lane >= keys.count && lane < a.top) room[0][lane] = 0;
        wave_lds_order();
    }
    if (a.slices == 1) {
        write_row<D>(a, row, s, room[0], lane);
        return;
    }
    if (lane == 0) a.parts[blockIdx.x] = make_float4(s.m, s.l, s.t, 0.0f);
    if (lane < a.top) a.part_keys[(size_t)blockIdx.x * a.top + lane] = room[0][lane];
}

// One wavefront per row joins its slices.
template <int D>
__global__ __launch_bounds__(64) void token_logprobs_join_kernel(LogprobArgs a) {
    __shared__ unsigned long long room[kTopRoom];
    const uint32_t row = blockIdx.x, lane = threadIdx.x;
    LogSum s{kMasked, 0.0f, 0.0f};
    for (uint32_t i = lane; i < a.slices; i += 64) {
        const float4 p = a.parts[(size_t)row * a.slices + i];
        s.join(p.x, p.y, p.z);
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        const float om = __shfl_xor(s.m, o), ol = __shfl_xor(s.l, o), ot = __shfl_xor(s.t, o);
        s.join(om, ol, ot);
    }
    if (a.top) {
        TopKeys keys{room, kMaskedKey, 0, a.top, lane};
        const size_t base = (size_t)row * a.slices * a.top;
        const uint32_t all = a.slices * a.top;
        for (uint32_t i = 0; i < all; i += 64) keys.push(i + lane < all ? a.part_keys[base + i + lane] : 0);
        keys.cut();
        if (lane >= keys.count && lane < a.top) room[lane] = 0;
        wave_lds_order();
    }
    write_row<D>(a, row, s, room, lane);
}

namespace {

// Slices of a row: whole steps, few enough that a slice is worth its own partial result, and enough workgroups that
// every CU has several.
void logprob_slices(LogprobArgs* a) {
    const uint32_t span = a->vocabulary + 8, steps = (span + kLogprobStep - 1) / kLogprobStep;
    uint64_t slices = (2048 + a->rows - 1) / a->rows;
    if (slices > steps) slices = steps;
    if (slices > 64) slices = 64;
    const uint32_t each = (uint32_t)((steps + slices - 1) / slices);
    a->slice_length = each * kLogprobStep;
    a->slices = (steps + each - 1) / each;
}

template <int D>
mi355q_status launch_logprobs(hipStream_t s, const LogprobArgs& a) {
    token_logprobs_kernel<D><<<dim3(a.rows * a.slices), 256, 0, s>>>(a);
    MI355Q_HIP(hipGetLastError());
    if (a.slices > 1) {
        token_logprobs_join_kernel<D><<<dim3(a.rows), 64, 0, s>>>(a);
        MI355Q_HIP(hipGetLastError());
    }
    return MI355Q_OK;
}

}  // namespace
}  // namespace mi355q

using namespace mi355q;

extern "C" mi355q_status mi355q_token_logprobs(mi355q_context* ctx, void* stream, const void* logits_dev, mi355q_dtype dtype,
                                               uint32_t row_count, uint32_t vocabulary_size, uint32_t row_stride,
                                               const int32_t* token_ids_dev, float* logprob_dev, float* entropy_dev,
                                               uint32_t top_count, int32_t* top_ids_dev, float* top_logprobs_dev) {
    if (!ctx) return fail(MI355Q_ERR_NULL_HANDLE, "context is null");
    if (!logits_dev) return fail(MI355Q_ERR_INVALID_ARGUMENT, "null logits");
    if (dtype != MI355Q_F16 && dtype != MI355Q_BF16 && dtype != MI355Q_F32)
        return fail(MI355Q_ERR_INVALID_ARGUMENT, "unknown element type %d", (int)dtype);
    if (!row_count || !vocabulary_size) return fail(MI355Q_ERR_SHAPE, "no rows or an empty vocabulary");
    if (row_count > (1u << 24) || vocabulary_size > (1u << 30))
        return fail(MI355Q_ERR_SHAPE, "%u rows of %u logits: at most 2^24 rows and 2^30 logits a row", row_count, vocabulary_size);
    if (row_stride == 0) row_stride = vocabulary_size;
    if (row_stride < vocabulary_size) return fail(MI355Q_ERR_SHAPE, "row stride %u is shorter than the vocabulary of %u", row_stride, vocabulary_size);
    if (top_count > kTopMost) return fail(MI355Q_ERR_SHAPE, "%u alternatives a row: at most %u", top_count, kTopMost);
    if (!token_ids_dev != !logprob_dev) return fail(MI355Q_ERR_INVALID_ARGUMENT, "token ids and their log probabilities go together");
    if (top_count && (!top_ids_dev || !top_logprobs_dev)) return fail(MI355Q_ERR_INVALID_ARGUMENT, "null buffers for the alternatives");
    if (!logprob_dev && !entropy_dev && !top_count) return fail(MI355Q_ERR_INVALID_ARGUMENT, "nothing is asked for");
    if ((uintptr_t)logits_dev % (dtype == MI355Q_F32 ? 4 : 2) || (uintptr_t)token_ids_dev % 4 || (uintptr_t)logprob_dev % 4 ||
        (uintptr_t)entropy_dev % 4 || (uintptr_t)top_ids_dev % 4 || (uintptr_t)top_logprobs_dev % 4)
        return fail(MI355Q_ERR_INVALID_ARGUMENT, "misaligned pointer");
    MI355Q_HIP(hipSetDevice(ctx->device));
    ScratchGuard guard(ctx, (hipStream_t)stream);
    if (guard.status) return guard.status;
    LogprobArgs a{logits_dev, token_ids_dev, logprob_dev, entropy_dev, top_ids_dev, top_logprobs_dev,
                  row_count, vocabulary_size, row_stride, top_count, 1, 0, nullptr, nullptr};
    logprob_slices(&a);
    if (a.slices > 1) {
        const size_t parts = (size_t)a.rows * a.slices;
        if (mi355q_status st = ensure_workspace(ctx, parts * (sizeof(float4) + a.top * 8))) return st;
        a.parts = (float4*)ctx->workspace;
        a.part_keys = (unsigned long long*)(a.parts + parts);
    }
    if (dtype == MI355Q_F32) return launch_logprobs<MI355Q_F32>((hipStream_t)stream, a);
    if (dtype == MI355Q_BF16) return launch_logprobs<MI355Q_BF16>((hipStream_t)stream, a);
    return launch_logprobs<MI355Q_F16>((hipStream_t)stream, a);
}
