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
// A CTA owns a run of a row's logits: it starts its logit and history loads, marks
// the history's tokens that fall into the run in a shared-memory table (integer
// atomics: their order does not show), adds up the biases that do, then applies
// everything to the registers and stores.  Nothing of the size of the vocabulary is
// kept between calls.  Bound: one read and one write of the logits; the history is
// read again by every run of its row, from L2, with eight loads of a thread in flight.
//
// The greedy pick is argmax.cu's: one 64-bit key per run, the last run of a row
// writes the id.
#include <cstdlib>
#include "device.cuh"
#include "internal.cuh"

namespace ocl {

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
// a table word: seen in the prompt | has a bias | times generated
constexpr uint32_t kPrompt = 0x80000000u, kBiased = 0x40000000u, kTimes = 0x3fffffffu;

struct RuleArgs {
    const float* logits;
    int64_t in_stride;
    int vocab;
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
    constexpr int kChunk = kThreads * PER, G = PER / 4, H = 8;
    __shared__ __align__(16) uint32_t table[kChunk];
    __shared__ float bias[kChunk];  // only where the table says kBiased
    __shared__ unsigned long long warp_best[kWarps];
    grid_wait();
    const int64_t row = blockIdx.y;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const float* x = p.logits + row * p.in_stride;
    const int shift = (int)((reinterpret_cast<uintptr_t>(x) >> 2) & 3);
    const int64_t c0 = (int64_t)blockIdx.x * kChunk - shift;  // below 2^31 + a chunk

    const bool counted = p.r.history != nullptr, biased = p.r.bias_ids != nullptr;
    const int32_t* h = counted ? p.r.history + row * p.r.history_stride : nullptr;
    int n = 0, prompt = 0;
    int32_t seen[H];
    if (counted) {
        n = min(p.r.history_lens[row], (int)p.r.history_max);
        prompt = p.r.prompt_lens ? p.r.prompt_lens[row] : 0;
#pragma unroll
        for (int j = 0; j < H; ++j) seen[j] = j * kThreads + tid < n ? __ldg(h + j * kThreads + tid) : -1;
    }
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

    if (counted || biased) {
#pragma unroll
        for (int j = 0; j < G; ++j) reinterpret_cast<uint4*>(table)[j * kThreads + tid] = make_uint4(0, 0, 0, 0);
        __syncthreads();
        for (int b = 0; b < n; b += H * kThreads) {
#pragma unroll
            for (int j = 0; j < H; ++j) {
                const int i = b + j * kThreads + tid, t = seen[j];
                const int64_t at = t - c0;
                if (t >= p.vocab && blockIdx.x == 0) atomicAdd(p.err, 1u);
                if (t >= 0 && t < p.vocab && at >= 0 && at < kChunk) {
                    if (i < prompt) atomicOr(table + at, kPrompt);
                    else atomicAdd(table + at, 1u);
                }
                const int next = i + H * kThreads;
                seen[j] = next < n ? __ldg(h + next) : -1;
            }
        }
        if (biased && warp == kWarps - 1) {  // one warp, so that biases of one token add up in list order
            const int32_t* ids = p.r.bias_ids + row * p.r.bias_stride;
            const float* values = p.r.bias_values + row * p.r.bias_stride;
            const int count = (int)p.r.bias_count;
            int next = lane < count ? ids[lane] : -1;
            for (int b = 0; b < count; b += 32) {
                const int t = next;
                next = b + 32 + lane < count ? ids[b + 32 + lane] : -1;
                if (t >= p.vocab && blockIdx.x == 0) atomicAdd(p.err, 1u);
                const bool here = t >= 0 && t < p.vocab && t >= c0 && t < c0 + kChunk;
                if (!__any_sync(0xffffffffu, here)) continue;
                const float value = here ? values[b + lane] : 0.f;
                const int at = here ? (int)(t - c0) : -1 - lane;
                const uint32_t same = __match_any_sync(0xffffffffu, at);
                if (here && (same & ((1u << lane) - 1)) == 0) {  // the first of its token in these 32
                    const bool old = table[at] & kBiased;
                    float sum = old ? __fadd_rn(bias[at], value) : value;
                    for (uint32_t rest = same & ~(1u << lane); rest; rest &= rest - 1)
                        sum = __fadd_rn(sum, values[b + __ffs(rest) - 1]);
                    bias[at] = sum;
                    if (!old) atomicOr(table + at, kBiased);
                }
                __syncwarp();
            }
        }
        __syncthreads();
    }

    const float rep = counted && p.r.repetition ? p.r.repetition[row] : 1.f;
    const float freq = counted && p.r.frequency ? p.r.frequency[row] : 0.f;
    const float pres = counted && p.r.presence ? p.r.presence[row] : 0.f;
    const bool use_rep = counted && p.r.repetition, use_made = counted && (p.r.frequency || p.r.presence);
    const uint32_t* allowed = p.r.allowed ? p.r.allowed + row * p.r.allowed_stride : nullptr;
    float* y = p.out ? p.out + row * p.out_stride : nullptr;
    const bool vec_out = y && ((reinterpret_cast<uintptr_t>(y) >> 2) & 3) == (uintptr_t)shift;
    float top = -INFINITY;  // this thread's pick: the first of its largest numbers
    int top_at = -1;
    bool nan_first = false;
#pragma unroll
    for (int j = 0; j < G; ++j) {
        const int at = (j * kThreads + tid) * 4;
        const int64_t i = c0 + at;
        if (i + 4 <= 0 || i >= p.vocab) continue;
        if (counted || biased) {
            uint32_t w[4];
            *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(table + at);
            if (w[0] | w[1] | w[2] | w[3]) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float l = v[j][e];
                    if ((w[e] & ~kBiased) && use_rep) l = l > 0.f ? __fdiv_rn(l, rep) : __fmul_rn(l, rep);
                    const uint32_t c = w[e] & kTimes;
                    if (c && use_made) l = __fsub_rn(__fsub_rn(l, __fmul_rn(freq, (float)c)), pres);
                    if (w[e] & kBiased) l = __fadd_rn(l, bias[at + e]);
                    v[j][e] = l;
                }
            }
        }
        if (allowed) {  // the 4 bits from token i on, which may lie in two words
            const int64_t f = i < 0 ? 0 : i, g = i + 3 < p.vocab ? i + 3 : p.vocab - 1;
            const uint32_t lo = allowed[f >> 5], hi = allowed[g >> 5];
            const uint32_t bits = i < 0 ? lo << (int)-i : __funnelshift_r(lo, hi, (uint32_t)i & 31);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (!((bits >> e) & 1)) v[j][e] = -INFINITY;
        }
        if (p.ids) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (i + e < 0 || i + e >= p.vocab) continue;
                const float l = v[j][e];
                if (l > top || (top_at < 0 && l == top)) top = l, top_at = (int)(i + e);
                if (i + e == 0) nan_first = isnan(l);
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
    // 0: no number here; a NaN at token 0 is the pick, and the largest key says so
    unsigned long long best = nan_first ? ~0ull : top_at < 0 ? 0ull : greedy_key(top, (uint32_t)top_at);
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const unsigned long long k = __shfl_xor_sync(0xffffffffu, best, o);
        best = k > best ? k : best;
    }
    if (lane == 0) warp_best[warp] = best;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < kWarps; ++w) best = warp_best[w] > best ? warp_best[w] : best;
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
    const RuleArgs a{logits, in_stride, (int)vocab, rules, out, out_stride, ids, slots, counters, err};
    (void)sms;
    switch (getenv("PER") ? atoi(getenv("PER")) : 16) {
        case 4: return launch_per<4>(a, rows, pdl, s);
        case 8: return launch_per<8>(a, rows, pdl, s);
    }
    return launch_per<16>(a, rows, pdl, s);
}

}  // namespace ocl
