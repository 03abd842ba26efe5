// rope.cu -- norms of q and k per head, position rotation and the cache write in one pass.
//
// Row r of qkv (the fused projection's output) is n_heads q heads, n_kv k heads
// and n_kv v heads of head_dim floats.  For each q and k head x:
//     y = x * rsqrt(mean(x^2) + eps) * w            (no norm when w is null)
//     (y_a, y_b) of pair i < rot/2 turned by t = position * freq_i, where the pair is
//     (i, i + rot/2), or (2i, 2i + 1) when interleaved; the rest passes through.
// q goes out in f32 (the attention's input), k and v into their page, rounded to
// nearest even.
//
// The angle: freq_i is held in revolutions as a 64-bit fixed-point fraction, so
// position * step wraps modulo one revolution exactly.  The step is off by its rounding
// (2^-65 revolutions) and its evaluation in 64-bit mantissas (a few 2^-64 of it), times the
// position: 2^-45 revolutions at 131072.  The phase is then rounded to f32, by at most
// 2^-26 revolutions (9.4e-8 rad), which is the error of the angle that is used at any
// 31-bit position; an f32 product loses 2^-24 of the whole angle instead (0.008 rad at
// position 131072).
//
// One warp per head, one or more CTAs per row (the host splits the heads of few
// rows over CTAs); the row's cos and sin are computed once per CTA.
//
// Bound: the floats in and out and the cache's bytes, HBM where rows are many; few rows are
// the launch and three dependent loads (position, table, head).  Measured in a graph (32 + 8
// heads of 128): 8190 rows 62 us = 5.9 TB/s, one row 1.7 us.
#include "device.cuh"
#include "internal.cuh"

namespace ocl {

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;

struct RopeArgs {
    const float* qkv;
    int64_t qkv_stride;
    int n_heads, n_kv, groups;  // groups: CTAs per row
    KvCache kv;
    KvRows at;
    Divisor page_size;
    const float *q_norm, *k_norm;
    float eps;
    RopeTable rope;
    float* q_out;
    unsigned int* err;
};

template <int V>
__device__ __forceinline__ void load_vec(float (&d)[V], const float* p) {
    if constexpr (V == 4) {
        const float4 t = *reinterpret_cast<const float4*>(p);
        d[0] = t.x; d[1] = t.y; d[2] = t.z; d[3] = t.w;
    } else if constexpr (V == 2) {
        const float2 t = *reinterpret_cast<const float2*>(p);
        d[0] = t.x; d[1] = t.y;
    } else {
        d[0] = *p;
    }
}
template <int V>
__device__ __forceinline__ void store_vec(float* p, const float (&d)[V]) {
    if constexpr (V == 4) *reinterpret_cast<float4*>(p) = make_float4(d[0], d[1], d[2], d[3]);
    else if constexpr (V == 2) *reinterpret_cast<float2*>(p) = make_float2(d[0], d[1]);
    else *p = d[0];
}
template <int V, class T>
__device__ __forceinline__ void store_vec(T* p, const float (&d)[V]) {
    if constexpr (V == 4) *reinterpret_cast<uint2*>(p) = make_uint2(pack16(d[0], d[1], T()), pack16(d[2], d[3], T()));
    else if constexpr (V == 2) *reinterpret_cast<uint32_t*>(p) = pack16(d[0], d[1], T());
    else *p = T(d[0]);
}

// A lane holds V pairs of its head: V elements at `a` and V at `b`.
template <int D, int V, class T>
__global__ void __launch_bounds__(kThreads) qk_norm_rope_kernel(const RopeArgs p) {
    static_assert(D / 2 <= 32 * V, "one lane step covers a head");
    __shared__ float2 turn[D / 2];
    grid_wait();
    const int64_t row = blockIdx.x / p.groups;
    const int group = blockIdx.x % p.groups, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int half = p.rope.rot / 2, i0 = lane * V;  // i0: the lane's first pair
    const bool active = i0 < D / 2;                  // other lanes only take part in the reductions
    const int qk = p.n_heads + p.n_kv, heads = qk + p.n_kv, step = p.groups * kWarps;
    // first elements of the lane's two runs in a q or k head, and in a v head (as they lie)
    const bool turned = i0 < half, halves = turned && !p.rope.interleaved;
    const int a_qk = halves ? i0 : 2 * i0, b_qk = halves ? i0 + half : 2 * i0 + V;
    const float* src = p.qkv + row * p.qkv_stride;
    float x[V] = {}, y[V] = {};
    auto load = [&](int h) {
        if (!active || h >= heads) return;
        load_vec<V>(x, src + (int64_t)h * D + (h < qk ? a_qk : 2 * i0));
        load_vec<V>(y, src + (int64_t)h * D + (h < qk ? b_qk : 2 * i0 + V));
    };
    int h = group * kWarps + warp;
    load(h);  // on its way while the row's place and angles are worked out

    const int pos = p.at.positions[row];
    if ((int)threadIdx.x < half) {
        const unsigned long long phase = (unsigned long long)(long long)pos * p.rope.steps[threadIdx.x];
        float s, c;
        sincospif((float)(long long)phase * 0x1p-63f, &s, &c);  // phase as a signed fraction of a revolution
        turn[threadIdx.x] = make_float2(c, s);
    }
    int64_t slot = -1;  // the row's place in the cache: -1 when nothing is to be cached
    if (pos >= 0) {
        const int64_t seq = sequence_of(p.at, row);
        int page = -1, in_page = 0;
        const bool ok = seq >= 0 && place_of(p.at.table + seq * p.at.table_stride, p.at.max_pages, p.kv.n_pages, p.page_size, pos, page, in_page);
        if (ok) slot = page * p.kv.page_stride + in_page * p.kv.token_stride;
        else if (threadIdx.x == 0 && group == 0) atomicAdd(p.err, 1u);
    }
    __syncthreads();
    float2 t[V];  // the lane's turns, the same for every head
#pragma unroll
    for (int e = 0; e < V; ++e) t[e] = turned ? turn[i0 + e] : make_float2(1.f, 0.f);

    for (; h < heads; h += step) {
        const bool is_q = h < p.n_heads, is_v = h >= qk;
        const int a = is_v ? 2 * i0 : a_qk, b = is_v ? 2 * i0 + V : b_qk;
        float u[V], v[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            u[e] = pos >= 0 ? x[e] : 0.f;  // a padding row is zeros
            v[e] = pos >= 0 ? y[e] : 0.f;
        }
        load(h + step);
        const float* w = is_v || pos < 0 ? nullptr : is_q ? p.q_norm : p.k_norm;
        if (w) {
            float sum = 0.f;
#pragma unroll
            for (int e = 0; e < V; ++e) sum += u[e] * u[e] + v[e] * v[e];
#pragma unroll
            for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            const float inv = rsqrtf(sum * (1.0f / D) + p.eps);
            if (active) {
                float wa[V], wb[V];
                load_vec<V>(wa, w + a);
                load_vec<V>(wb, w + b);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    u[e] *= inv * wa[e];
                    v[e] *= inv * wb[e];
                }
            }
        }
        if (turned && !is_v) {
            if (halves) {
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float f = u[e], g = v[e];
                    u[e] = f * t[e].x - g * t[e].y;
                    v[e] = g * t[e].x + f * t[e].y;
                }
            } else {
                float z[2 * V];
#pragma unroll
                for (int e = 0; e < V; ++e) z[e] = u[e], z[V + e] = v[e];
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float f = z[2 * e], g = z[2 * e + 1];
                    z[2 * e] = f * t[e].x - g * t[e].y;
                    z[2 * e + 1] = g * t[e].x + f * t[e].y;
                }
#pragma unroll
                for (int e = 0; e < V; ++e) u[e] = z[e], v[e] = z[V + e];
            }
        }
        if (!active) continue;
        if (is_q) {
            float* dst = p.q_out + (row * p.n_heads + h) * D;
            store_vec<V>(dst + a, u);
            store_vec<V>(dst + b, v);
        } else if (slot >= 0) {
            T* dst = static_cast<T*>(is_v ? p.kv.v : p.kv.k) + slot + (int64_t)(h - (is_v ? qk : p.n_heads)) * p.kv.head_stride;
            store_vec<V>(dst + a, u);
            store_vec<V>(dst + b, v);
        }
    }
}

template <int D, int V>
cudaError_t launch_dim(const RopeArgs& a, int64_t rows, bool pdl, cudaStream_t s) {
    const dim3 grid((unsigned)(rows * a.groups));
    return a.kv.type == kKvBf16 ? launch_kernel(qk_norm_rope_kernel<D, V, __nv_bfloat16>, grid, kThreads, 0, pdl, s, a)
                                : launch_kernel(qk_norm_rope_kernel<D, V, __half>, grid, kThreads, 0, pdl, s, a);
}

}  // namespace

cudaError_t launch_qk_norm_rope(const float* qkv, int64_t qkv_stride, int64_t rows, int64_t n_heads, const KvCache& kv,
                                const KvRows& at, const float* q_norm, const float* k_norm, float eps,
                                const RopeTable& rope, float* q_out, unsigned int* err, int sms, bool pdl,
                                cudaStream_t s) {
    RopeArgs a{qkv, qkv_stride, (int)n_heads, (int)kv.n_kv, 1, kv, at, divisor_of((uint32_t)kv.page_size), q_norm, k_norm, eps, rope, q_out, err};
    const int64_t most = (n_heads + 2 * kv.n_kv + kWarps - 1) / kWarps;  // CTAs a row can use
    const int64_t want = (sms + rows - 1) / rows;
    a.groups = (int)(want < most ? want : most);
    if (rows * a.groups > 0x7fffffff) return cudaErrorInvalidValue;
    switch (kv.head_dim) {
        case 64: return launch_dim<64, 1>(a, rows, pdl, s);
        case 96: return launch_dim<96, 2>(a, rows, pdl, s);
        case 128: return launch_dim<128, 2>(a, rows, pdl, s);
        case 256: return launch_dim<256, 4>(a, rows, pdl, s);
    }
    return cudaErrorInvalidValue;
}

}  // namespace ocl
