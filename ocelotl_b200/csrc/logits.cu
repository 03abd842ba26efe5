// logits.cu -- penalties, biases and the allowed-token mask on logits, with the greedy pick.
//
// For row r and token t, with c the times t stands in the generated part of the
// row's history and "seen" that it stands anywhere in it, in this order:
//     seen:         l = l > 0 ? l / repetition : l * repetition
//     c > 0:        l = (l - frequency * c) - presence
//     biased:       l = l + (sum of the row's biases on t, in list order)
//     not allowed:  l = -inf
// each step rounded to f32 on its own (no contraction), so the result is the
// formula's to the bit.
//
// A CTA owns a run of a row's logits: it starts its logit loads, counts the row's
// history into a shared-memory table of its own run (integer atomics: the order does
// not show), adds up the biases that fall into the run, then applies everything to
// the registers and stores.  Nothing of the size of the vocabulary is kept between
// calls.  Bound: one read and one write of the logits; the history is read again by
// every run of its row, from L2.
//
// The greedy pick is argmax.cu's: one 64-bit key per run, the last run of a row
// writes the id.
#include "device.cuh"
#include "internal.cuh"

namespace ocl {

namespace {

constexpr int kThreads = 256;
constexpr uint32_t kPrompt = 0x80000000u;  // table word: seen in the prompt | times generated

struct RuleArgs {
    const float* logits;
    int64_t in_stride, vocab;
    LogitRules r;
    float* out;
    int64_t out_stride;
    int32_t* ids;
    unsigned long long* slots;
    unsigned int* counters;
    unsigned int* err;
};

// PER logits a thread, in groups of 4 that are 16-byte aligned in `logits`
// whatever the row's own alignment: the run of CTA b starts at b * chunk - shift.
template <int PER>
__global__ void __launch_bounds__(kThreads) logit_rules_kernel(const RuleArgs p) {
    constexpr int kChunk = kThreads * PER, G = PER / 4;
    __shared__ __align__(16) uint32_t table[kChunk];
    __shared__ __align__(16) float bias[kChunk];
    __shared__ unsigned long long warp_best[kThreads / 32];
    grid_wait();
    const int64_t row = blockIdx.y;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const float* x = p.logits + row * p.in_stride;
    const int shift = (int)((reinterpret_cast<uintptr_t>(x) >> 2) & 3);
    const int64_t c0 = (int64_t)blockIdx.x * kChunk - shift;

    float v[G][4];
#pragma unroll
    for (int j = 0; j < G; ++j) {
        const int64_t i = c0 + (j * kThreads + tid) * 4;
        if (i >= 0 && i + 4 <= p.vocab) {
            const float4 q = __ldcs(reinterpret_cast<const float4*>(x + i));
            v[j][0] = q.x; v[j][1] = q.y; v[j][2] = q.z; v[j][3] = q.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[j][e] = i + e >= 0 && i + e < p.vocab ? x[i + e] : 0.f;
        }
    }

    const bool counted = p.r.history != nullptr, biased = p.r.bias_ids != nullptr;
    if (counted || biased) {
        for (int i = tid; i < kChunk / 4; i += kThreads) {
            if (counted) reinterpret_cast<uint4*>(table)[i] = make_uint4(0, 0, 0, 0);
            // NaN with this payload: no bias on the token (a bias of 0 is one)
            if (biased) reinterpret_cast<uint4*>(bias)[i] = make_uint4(~0u, ~0u, ~0u, ~0u);
        }
        __syncthreads();
    }
    if (counted) {
        const int32_t* h = p.r.history + row * p.r.history_stride;
        int64_t n = p.r.history_lens[row];
        n = n < 0 ? 0 : n > p.r.history_max ? p.r.history_max : n;
        const int64_t prompt = p.r.prompt_lens ? p.r.prompt_lens[row] : 0;
        for (int64_t i = tid; i < n; i += kThreads) {
            const int64_t t = h[i];
            if (t >= p.vocab && blockIdx.x == 0) atomicAdd(p.err, 1u);
            const int64_t at = t - c0;
            if (t >= 0 && t < p.vocab && at >= 0 && at < kChunk) {
                if (i < prompt) atomicOr(table + at, kPrompt);
                else atomicAdd(table + at, 1u);
            }
        }
    }
    if (biased && warp == kThreads / 32 - 1) {  // one warp, so that biases of one token add up in list order
        const int32_t* ids = p.r.bias_ids + row * p.r.bias_stride;
        const float* values = p.r.bias_values + row * p.r.bias_stride;
        for (int64_t b = 0; b < p.r.bias_count; b += 32) {
            const int64_t t = b + lane < p.r.bias_count ? ids[b + lane] : -1;
            if (t >= p.vocab && blockIdx.x == 0) atomicAdd(p.err, 1u);
            const bool here = t >= 0 && t < p.vocab && t >= c0 && t < c0 + kChunk;
            if (!__any_sync(0xffffffffu, here)) continue;
            const float value = here ? values[b + lane] : 0.f;
            const int at = here ? (int)(t - c0) : -1 - lane;
            const uint32_t same = __match_any_sync(0xffffffffu, at);
            const bool leads = here && __ffs(same) - 1 == lane;
            float sum = 0.f;
            bool any = false;
            if (leads && __float_as_uint(bias[at]) != ~0u) sum = bias[at], any = true;
            for (int k = 0; k < 32; ++k) {
                const float f = __shfl_sync(0xffffffffu, value, k);
                if ((same >> k) & 1) sum = any ? __fadd_rn(sum, f) : f, any = true;
            }
            if (leads) bias[at] = isnan(sum) ? __uint_as_float(0x7fc00000u) : sum;
            __syncwarp();
        }
    }
    if (counted || biased) __syncthreads();

    const float rep = counted && p.r.repetition ? p.r.repetition[row] : 1.f;
    const float freq = counted && p.r.frequency ? p.r.frequency[row] : 0.f;
    const float pres = counted && p.r.presence ? p.r.presence[row] : 0.f;
    const bool use_rep = counted && p.r.repetition, use_made = counted && (p.r.frequency || p.r.presence);
    const uint32_t* allowed = p.r.allowed ? p.r.allowed + row * p.r.allowed_stride : nullptr;
    float* y = p.out ? p.out + row * p.out_stride : nullptr;
    const bool vec_out = y && ((reinterpret_cast<uintptr_t>(y) >> 2) & 3) == (uintptr_t)shift;
    unsigned long long best = 0;  // below every key of a number
#pragma unroll
    for (int j = 0; j < G; ++j) {
        const int at = (j * kThreads + tid) * 4;
        const int64_t i = c0 + at;
        if (i + 4 <= 0 || i >= p.vocab) continue;
        uint32_t seen[4] = {};
        float add[4];
        if (counted) *reinterpret_cast<uint4*>(seen) = *reinterpret_cast<const uint4*>(table + at);
        if (biased) *reinterpret_cast<float4*>(add) = *reinterpret_cast<const float4*>(bias + at);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (i + e < 0 || i + e >= p.vocab) continue;
            float l = v[j][e];
            if (seen[e]) {
                if (use_rep) l = l > 0.f ? __fdiv_rn(l, rep) : __fmul_rn(l, rep);
                const uint32_t c = seen[e] & ~kPrompt;
                if (c && use_made) l = __fsub_rn(__fsub_rn(l, __fmul_rn(freq, (float)c)), pres);
            }
            if (biased && __float_as_uint(add[e]) != ~0u) l = __fadd_rn(l, add[e]);
            if (allowed && !((allowed[(i + e) >> 5] >> ((i + e) & 31)) & 1)) l = -INFINITY;
            v[j][e] = l;
            if (p.ids) {
                if (!isnan(l)) {
                    const unsigned long long k = greedy_key(l, (uint32_t)(i + e));
                    best = k > best ? k : best;
                } else if (i + e == 0) {
                    best = ~0ull;  // a NaN at token 0 is the pick, and the largest key says so
                }
            }
        }
        if (vec_out && i >= 0 && i + 4 <= p.vocab) {
            *reinterpret_cast<float4*>(y + i) = make_float4(v[j][0], v[j][1], v[j][2], v[j][3]);
        } else if (y) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (i + e >= 0 && i + e < p.vocab) y[i + e] = v[j][e];
        }
    }
    if (!p.ids) return;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const unsigned long long k = __shfl_xor_sync(0xffffffffu, best, o);
        best = k > best ? k : best;
    }
    if (lane == 0) warp_best[warp] = best;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < kThreads / 32; ++w) best = warp_best[w] > best ? warp_best[w] : best;
        if (best) atomicMax(p.slots + row, best);
        __threadfence();
        if (atomicAdd(p.counters + row, 1u) == gridDim.x - 1) {
            __threadfence();
            const unsigned long long k = atomicExch(p.slots + row, 0ull);  // read and reset
            p.ids[row] = k == 0 || k == ~0ull ? 0 : (int32_t)(0xFFFFFFFFu - (uint32_t)(k & 0xFFFFFFFFull));
            p.counters[row] = 0;
        }
    }
}

template <int PER>
cudaError_t launch_per(const RuleArgs& a, int64_t rows, bool pdl, cudaStream_t s) {
    constexpr int64_t chunk = kThreads * PER;
    const dim3 grid((unsigned)((a.vocab + 3 + chunk - 1) / chunk), (unsigned)rows);
    return launch_kernel(logit_rules_kernel<PER>, grid, kThreads, 0, pdl, s, a);
}

}  // namespace

cudaError_t launch_logit_rules(const float* logits, int64_t in_stride, int64_t rows, int64_t vocab,
                               const LogitRules& rules, float* out, int64_t out_stride, int32_t* ids,
                               unsigned long long* slots, unsigned int* counters, unsigned int* err, int sms, bool pdl,
                               cudaStream_t s) {
    const RuleArgs a{logits, in_stride, vocab, rules, out, out_stride, ids, slots, counters, err};
    (void)sms;
    return launch_per<16>(a, rows, pdl, s);
}

}  // namespace ocl
