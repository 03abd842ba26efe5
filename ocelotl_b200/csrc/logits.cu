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
// read again by every run of its row, from L2, with up to four loads of a thread in flight.
//
// The greedy pick is argmax.cu's: one 64-bit key per run, the last run of a row
// writes the id.
//
// Measured in a graph: 190 rows of 151936 (histories up to 8000, 40 biases, masks, pick) 72 us
// = 3.2 TB/s of logits, of which the history's second and later reads take 15, the pick 8 and
// biases and masks 7; one row of 128256 4.1 us.
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

// The key of one run joins its row's; the last run writes the id.
__device__ __forceinline__ void pick_row(const RuleArgs& p, int64_t row, unsigned long long key) {
    if (key) atomicMax(p.slots + row, key);
    __threadfence();
    if (atomicAdd(p.counters + row, 1u) == gridDim.x - 1) {
        __threadfence();
        const unsigned long long k = atomicExch(p.slots + row, 0ull);  // read and reset
        p.ids[row] = k == 0 || k == ~0ull ? 0 : (int32_t)(0xFFFFFFFFu - (uint32_t)(k & 0xFFFFFFFFull));
        p.counters[row] = 0;
    }
}

// PER logits a thread, in groups of 4 that are 16-byte aligned in `logits`
// whatever the row's own alignment: the run of CTA b starts at b * chunk - shift.
// Logits of the run outside the row are NaN, which no rule changes and no pick takes.
template <int PER>
__global__ void __launch_bounds__(kThreads, 5) logit_rules_kernel(const RuleArgs p) {
    constexpr int kChunk = kThreads * PER, G = PER / 4, H = 4;
    extern __shared__ __align__(16) uint32_t table[];
    float* bias = reinterpret_cast<float*>(table + kChunk);  // only where the table says kBiased
    __shared__ unsigned long long warp_best[kWarps];
    grid_wait();
    const int64_t row = blockIdx.y;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const float* x = p.logits + row * p.in_stride;
    const int shift = (int)((reinterpret_cast<uintptr_t>(x) >> 2) & 3);
    const int c0 = (int)blockIdx.x * kChunk - shift;
    const int lo = max(c0, 0), skip = lo - c0;                     // the run's first token of the row, and its place
    const uint32_t len = (uint32_t)max(min(c0 + kChunk, p.vocab) - lo, 0);  // its tokens of the row: none in a last run behind it

    const bool counted = p.r.history != nullptr, biased = p.r.bias_ids != nullptr;
    const int32_t* h = counted ? p.r.history + row * p.r.history_stride : nullptr;
    const int room = counted ? (int)p.r.history_max : 0, count = biased ? (int)p.r.bias_count : 0;
    // What a length rules out is loaded all the same and dropped afterwards: a run waits
    // for memory once.
    int32_t seen[H];
#pragma unroll
    for (int j = 0; j < H; ++j) seen[j] = j * kThreads + tid < room ? __ldg(h + j * kThreads + tid) : -1;
    const int n = counted ? min(p.r.history_lens[row], room) : 0;
    const int prompt = counted && p.r.prompt_lens ? p.r.prompt_lens[row] : 0;
    const bool use_rep = counted && p.r.repetition, use_made = counted && (p.r.frequency || p.r.presence);
    const float rep = use_rep ? p.r.repetition[row] : 1.f;
    const float freq = use_made && p.r.frequency ? p.r.frequency[row] : 0.f;
    const float pres = use_made && p.r.presence ? p.r.presence[row] : 0.f;
    const bool adds = biased && warp == kWarps - 1;  // one warp, so that biases of one token add up in list order
    const int32_t* bias_ids = biased ? p.r.bias_ids + row * p.r.bias_stride : nullptr;
    const float* bias_values = biased ? p.r.bias_values + row * p.r.bias_stride : nullptr;
    int next_id = adds && lane < count ? bias_ids[lane] : -1;
    float next_value = adds && lane < count ? bias_values[lane] : 0.f;
    const uint32_t* allowed = p.r.allowed ? p.r.allowed + row * p.r.allowed_stride : nullptr;

    const float nan = __uint_as_float(0x7fc00000u);
    float v[G][4];
    uint32_t word[G], over[G];  // the mask word of a group's first token, and the next one where the group runs into it
#pragma unroll
    for (int j = 0; j < G; ++j) {
        const int i = c0 + (j * kThreads + tid) * 4;
        word[j] = over[j] = 0xffffffffu;
        if (i >= 0 && i + 4 <= p.vocab) {
            const float4 q = __ldcs(reinterpret_cast<const float4*>(x + i));
            v[j][0] = q.x; v[j][1] = q.y; v[j][2] = q.z; v[j][3] = q.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[j][e] = i + e >= 0 && i + e < p.vocab ? x[i + e] : nan;
        }
        if (allowed && i < p.vocab) {
            if (i >= 0) word[j] = __ldg(allowed + (i >> 5));
            if ((i & 31) > 28 && (i | 31) + 1 < p.vocab) over[j] = __ldg(allowed + (i >> 5) + 1);
        }
    }

    if (counted || biased) {
#pragma unroll
        for (int j = 0; j < G; ++j) reinterpret_cast<uint4*>(table)[j * kThreads + tid] = make_uint4(0, 0, 0, 0);
        __syncthreads();
        for (int b = 0; b < n; b += H * kThreads) {
#pragma unroll
            for (int j = 0; j < H; ++j) {
                if (b + j * kThreads >= n) break;
                const int i = b + j * kThreads + tid, t = seen[j], next = i + H * kThreads;
                seen[j] = next < n ? __ldg(h + next) : -1;
                const uint32_t at = (uint32_t)t - (uint32_t)lo;
                if (at < len && i < n) {
                    if (i < prompt) atomicOr(table + skip + at, kPrompt);
                    else atomicAdd(table + skip + at, 1u);
                }
                if (blockIdx.x == 0 && t >= p.vocab && i < n) atomicAdd(p.err, 1u);
            }
        }
        for (int b = 0; adds && b < count; b += 32) {
            const int t = next_id;
            const float value = next_value;
            next_id = b + 32 + lane < count ? bias_ids[b + 32 + lane] : -1;
            next_value = b + 32 + lane < count ? bias_values[b + 32 + lane] : 0.f;
            if (t >= p.vocab && blockIdx.x == 0) atomicAdd(p.err, 1u);
            const bool here = (uint32_t)t - (uint32_t)lo < len;
            if (!__any_sync(0xffffffffu, here)) continue;
            const int at = here ? t - c0 : -1 - lane;
            const uint32_t same = __match_any_sync(0xffffffffu, at);
            if (here && (same & ((1u << lane) - 1)) == 0) {  // the first of its token in these 32
                const bool old = table[at] & kBiased;
                float sum = old ? __fadd_rn(bias[at], value) : value;
                for (uint32_t rest = same & ~(1u << lane); rest; rest &= rest - 1)
                    sum = __fadd_rn(sum, bias_values[b + __ffs(rest) - 1]);
                bias[at] = sum;
                if (!old) atomicOr(table + at, kBiased);
            }
            __syncwarp();
        }
        __syncthreads();
    }

    float* y = p.out ? p.out + row * p.out_stride : nullptr;
    const bool vec_out = y && ((reinterpret_cast<uintptr_t>(y) >> 2) & 3) == (uintptr_t)shift;
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < G; ++j) {
        const int at = (j * kThreads + tid) * 4, i = c0 + at;
        const bool edge = i < 0 || i + 4 > p.vocab;
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
        if (allowed) {
            const uint32_t bits = __funnelshift_r(word[j], over[j], i & 31);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (!(bits & (1u << e))) v[j][e] = -INFINITY;
        }
        if (edge) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (i + e < 0 || i + e >= p.vocab) v[j][e] = nan;
        }
        top = fmaxf(top, fmaxf(fmaxf(v[j][0], v[j][1]), fmaxf(v[j][2], v[j][3])));
        if (vec_out && !edge) {
            *reinterpret_cast<float4*>(y + i) = make_float4(v[j][0], v[j][1], v[j][2], v[j][3]);
        } else if (y) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (i + e >= 0 && i + e < p.vocab) y[i + e] = v[j][e];
        }
    }
    if (!p.ids) return;
    // ---- the warp's largest number and the first token that has it, then the run's
    const uint32_t mine = (uint32_t)(greedy_key(top, 0) >> 32), most = __reduce_max_sync(0xffffffffu, mine);
    uint32_t at = 0xffffffffu;  // stays where there is no number
    if (mine == most) {
#pragma unroll
        for (int j = G - 1; j >= 0; --j)
#pragma unroll
            for (int e = 3; e >= 0; --e)
                if (v[j][e] == top) at = (uint32_t)((j * kThreads + tid) * 4 + e);
    }
    at = __reduce_min_sync(0xffffffffu, at);
    if (lane == 0) warp_best[warp] = at == 0xffffffffu ? 0ull : (unsigned long long)most << 32 | (0xffffffffu - (uint32_t)(c0 + (int)at));
    // a NaN at token 0 is the pick of its row, and the largest key says so
    const bool nan_first = blockIdx.x == 0 && tid == 0 &&
                           isnan(shift == 0 ? v[0][0] : shift == 1 ? v[0][1] : shift == 2 ? v[0][2] : v[0][3]);
    __syncthreads();
    if (tid == 0) {
        unsigned long long best = nan_first ? ~0ull : 0ull;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) best = warp_best[w] > best ? warp_best[w] : best;
        pick_row(p, row, best);
    }
}

template <int PER>
cudaError_t launch_per(const RuleArgs& a, int64_t rows, bool pdl, cudaStream_t s) {
    constexpr int64_t chunk = kThreads * PER;
    static_assert(chunk * 8 <= 48 * 1024, "no opt-in for more shared memory");
    const dim3 grid((unsigned)((a.vocab + 3 + chunk - 1) / chunk), (unsigned)rows);
    const size_t smem = (size_t)(chunk * 4) * (a.r.bias_ids ? 2 : a.r.history ? 1 : 0);  // the table, and the biases
    return launch_kernel(logit_rules_kernel<PER>, grid, kThreads, smem, pdl, s, a);
}

}  // namespace

cudaError_t launch_logit_rules(const float* logits, int64_t in_stride, int64_t rows, int64_t vocab,
                               const LogitRules& rules, float* out, int64_t out_stride, int32_t* ids,
                               unsigned long long* slots, unsigned int* counters, unsigned int* err, int sms, bool pdl,
                               cudaStream_t s) {
    const RuleArgs a{logits, in_stride, (int)vocab, rules, out, out_stride, ids, slots, counters, err};
    // Few logits: short runs, so that every SM has some.  Many: long ones, whose fixed
    // work (tables, history, pick) is shared by more logits.  Measured at 128256 logits and 600
    // tokens of history, 4 / 8 / 16 a thread: 1 row 4.0 / 4.8 / 5.4 us, 4 rows 5.0 / 5.0 / 5.6,
    // 8 rows 6.8 / 5.7 / 6.0, 32 rows 16.7 / 12.6 / 11.1.
    auto ctas = [&](int per) { return rows * ((vocab + kThreads * per - 1) / (kThreads * per)); };
    if (2 * ctas(4) <= 5 * sms) return launch_per<4>(a, rows, pdl, s);
    if (2 * ctas(8) <= 7 * sms) return launch_per<8>(a, rows, pdl, s);
    return launch_per<16>(a, rows, pdl, s);
}

}  // namespace ocl
