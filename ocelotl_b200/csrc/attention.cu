// attention.cu -- attention of new tokens over the paged key/value cache.
//
// Row r holds token p = positions[r] of its sequence and sees tokens 0..p; query
// head h reads k/v head h / G:
//     s_j = scale * q . k_j,   o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  m = max_j s_j
// in one pass over the cache with a running m, sum and o.
//
// Bound: the cache is read once, 4 * head_dim bytes a token and k/v head, against
// 4 * G * head_dim flops: HBM.  At f32 quality the flops do not fit the FMA units
// beside that stream (G = 8: 52 TFLOP/s at 6.5 TB/s, plus the conversions), so they
// run on the tensor cores: mma.sync m16n8k16 with the up to 8 query heads of a k/v
// head as rows.  Half of the 16 rows would be empty; they carry the rest of the
// precision instead.  A f32 factor (q, and the weights p_j) is cut into 16-bit
// pieces that add up to it -- rows 0-7 the leading piece, rows 8-15 the next one,
// for bf16 a third in a second MMA -- so every product is exact and the sum has f32
// quality although q and p are never rounded to 16 bits:
//     bf16: 3 pieces of 8 bits = 24 bits;   f16: 2 pieces of 11 bits = 22 bits
// (q scaled by a power of two per head, p by 2^14, so that f16's range is enough).
// The tensor core truncates when it adds; chains are kept short (two chains over
// head_dim, one 16-token step for p.v) and joined with rounding f32 adds.
//
// Work split: the tiles (64 tokens of one row and k/v head) of all rows, in order,
// are cut into equal runs, one per resident CTA, from the positions in device
// memory -- so one captured launch stays balanced while the lengths grow.  Each of
// the 4 warps streams its own 16 tokens of a tile through a private ring of stages
// and needs no barrier inside a run.  Where 16 tokens always lie in one page (page
// sizes that are multiples of 16), one tensor-map copy (cp.async.bulk.tensor, its
// swizzle doing the bank spreading) brings the keys and one the values; other page
// sizes gather rows with cp.async.  A row whose tiles lie in
// several CTAs is joined by the last of them to arrive, in CTA order: the result
// does not depend on which one it is.  Nothing waits on another CTA.
#include <cuda.h>

#include "device.cuh"
#include "internal.cuh"

namespace ocl {

namespace {

constexpr int kWarps = kTileWarps, kThreads = 32 * kWarps;
constexpr int kHeads = 8;  // query heads of one k/v head worked on together

constexpr int stages(int d) { return d <= 96 ? 4 : 3; }
constexpr int ctas_per_sm(int d) { return d == 64 ? 3 : d == 256 ? 1 : 2; }
constexpr int max_ctas_per_sm = 3;
// 16 tokens of k or v are kept as parts of 64 elements (32 for head_dim 96): a part is
// 16 rows of 128 (64) bytes, its 16-byte chunks exclusive-or'ed with the row as the
// copy engine's 128-byte (64-byte) swizzle does.
constexpr int part_elems(int d) { return d % 64 == 0 ? 64 : 32; }
constexpr int part_bytes(int d) { return kWarpTok * part_elems(d) * 2; }
constexpr int half_bytes(int d) { return kWarpTok * d * 2; }  // k (or v) of a stage
constexpr int merge_cols(int d) { return d < 128 ? d : 128; }
constexpr bool q_in_smem(int d) { return d > 128; }
constexpr int q_bytes(int d) { return q_in_smem(d) ? d / 16 * 32 * 24 : 0; }
constexpr int slot_floats(int d) { return kHeads * d + 2 * kHeads; }

struct Shared {  // behind the ring, the merge buffer and the q fragments
    uint64_t full[kWarps][4];
    long long scan[kWarps], first_at;
    int first_row, last_in;
    uint32_t valid[kWarps][4];
    float m[kWarps][kHeads], l[kWarps][kHeads];
};
constexpr int ring_bytes(int d) { return kWarps * stages(d) * 2 * half_bytes(d); }
constexpr int merge_bytes(int d) { return kWarps * kHeads * merge_cols(d) * 4; }
constexpr int smem_bytes(int d) { return ring_bytes(d) + merge_bytes(d) + q_bytes(d) + (int)sizeof(Shared); }
static_assert(smem_bytes(256) <= 227 * 1024 && 2 * (smem_bytes(128) + 1024) <= 228 * 1024 &&
              2 * (smem_bytes(96) + 1024) <= 228 * 1024 && 3 * (smem_bytes(64) + 1024) <= 228 * 1024, "CTAs per SM");

struct AttnArgs {
    const float* q;
    int64_t q_stride;
    int rows, n_heads, n_kv, group, head_groups;
    KvCache kv;
    KvRows at;
    Divisor page_size;
    int cap;      // tokens a row of the block table can hold
    float scale;  // in units of log2
    float* out;
    float* part;
    unsigned int* counters;
    unsigned int* err;
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {  // bytes < 16: the rest is zero
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldmatrix4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
// c = a . b, and c += a . b
#define OCL_MMA(NAME, TYPE)                                                                                            \
    __device__ __forceinline__ void mma0(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,             \
                                         uint32_t b0, uint32_t b1, TYPE) {                                              \
        asm("mma.sync.aligned.m16n8k16.row.col.f32." NAME "." NAME                                             \
                     ".f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"                                   \
                     : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])                                                   \
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));                                 \
    }                                                                                                                   \
    __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, \
                                        uint32_t b1, TYPE) {                                                            \
        asm("mma.sync.aligned.m16n8k16.row.col.f32." NAME "." NAME                                             \
                     ".f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"                                       \
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])                                                   \
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));                                           \
    }
OCL_MMA("bf16", __nv_bfloat16)
OCL_MMA("f16", __half)
#undef OCL_MMA

__device__ __forceinline__ void mbar_init(uint64_t* bar) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void mbar_expect(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
                 : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return ok != 0;
}
// Wait for at most ~1 s of SM clocks; false if it gave up.
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity) {
    if (mbar_test(bar, parity)) return true;
    const long long t0 = clock64();
    while (!mbar_test(bar, parity))
        if (clock64() - t0 > 2000000000LL) return false;
    return true;
}
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int in_page, int head, int page, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %2, %4, %5}], "
        "[%6];" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(in_page), "r"(head), "r"(page), "r"(smem_u32(bar))
        : "memory");
}

template <class T> constexpr int kPieces = 3;
template <> constexpr int kPieces<__half> = 2;
template <class T> constexpr float kShift = 0.f;  // p is scaled by 2^kShift
template <> constexpr float kShift<__half> = 14.f;

__device__ __forceinline__ float ex2(float x) {  // 2 units, 0 below 2^-126
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two floats as N packed pairs of 16-bit pieces, leading piece first.
template <int N, class T>
__device__ __forceinline__ void cut(uint32_t (&w)[N], float a, float b) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        w[i] = pack16(a, b, T());
        const float2 t = unpack16(w[i], T());
        a -= t.x;
        b -= t.y;
    }
}

// Byte offset, within the k (or v) half of a stage, of 16-byte chunk `c` of row `r`:
// 8 rows of one chunk column (an ldmatrix) fall into different banks.
template <int D>
__device__ __forceinline__ int chunk_at(int c, int r) {
    constexpr int CP = part_elems(D) / 8;
    const int x = CP == 8 ? r & 7 : (r >> 1) & 3;
    return c / CP * part_bytes(D) + r * CP * 16 + ((c % CP) ^ x) * 16;
}

// PACK (bf16, at most 4 heads): rows 0-3 leading pieces, 4-7 third, 8-11 second, so that
// one MMA does what takes two with 8 heads; lanes 16-31 then hold the third pieces' part
// of o.  TILED: 16 tokens lie in one page, which the tensor maps describe as (part element,
// slot, part, k/v head, page).
template <int D, class T, bool TILED, bool PACK>
__global__ void __launch_bounds__(kThreads, ctas_per_sm(D))
    attention_kernel(const AttnArgs p, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
    constexpr int S = stages(D), KS = D / 16, NT = D / 8, C = D / 8, N = kPieces<T>;
    constexpr int kHalf = half_bytes(D), kStage = 2 * kHalf, kPart = part_bytes(D), CP2 = part_elems(D) / 16;
    constexpr int MC = merge_cols(D), kRows = PACK ? 4 : kHeads;
    extern __shared__ __align__(1024) unsigned char smem[];
    float* merge_o = reinterpret_cast<float*>(smem + ring_bytes(D));
    uint32_t* q_frag = reinterpret_cast<uint32_t*>(smem + ring_bytes(D) + merge_bytes(D));
    Shared& sh = *reinterpret_cast<Shared*>(smem + ring_bytes(D) + merge_bytes(D) + q_bytes(D));

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c4 = lane & 3;
    const int items = p.n_kv * p.head_groups;
    if (TILED && lane < S) {
        mbar_init(&sh.full[warp][lane]);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    grid_wait();

    // ---- this CTA's run of tiles
    const int per = (p.rows + kThreads - 1) / kThreads;
    const int r0 = min(tid * per, p.rows), r1 = min(r0 + per, p.rows);
    long long mine = 0;
    for (int r = r0; r < r1; ++r) mine += tiles_of(row_tokens(p.at, p.cap, r));
    long long upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long t = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += t;
    }
    if (lane == 31) sh.scan[warp] = upto;
    __syncthreads();
    long long total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) upto += sh.scan[w];
        total += sh.scan[w];
    }
    total *= items;
    const long long P = total < (long long)gridDim.x ? total : (long long)gridDim.x;
    const long long cta = blockIdx.x;
    const long long begin = cta < P ? run_begin(total, P, cta) : total, end = cta < P ? run_begin(total, P, cta + 1) : total;
    {
        const long long b = (upto - mine) * items, e = upto * items;
        if (begin < end && begin >= b && begin < e) {
            long long at = b;
            int r = r0;
            for (;; ++r) {
                const long long n = (long long)tiles_of(row_tokens(p.at, p.cap, r)) * items;
                if (begin < at + n) break;
                at += n;
            }
            sh.first_row = r;
            sh.first_at = begin - at;
        }
    }
    __syncthreads();

    // rows without tokens are zeros; rows whose place is out of range are counted
    for (int r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const int tokens = row_tokens(p.at, p.cap, r), pos = p.at.positions[r];
        if (tid == 0 && pos >= 0 && pos >= tokens) atomicAdd(p.err, 1u);
        if (tokens == 0)
            for (int i = tid; i < p.n_heads * D; i += kThreads) p.out[(int64_t)r * p.n_heads * D + i] = 0.f;
    }
    if (begin >= end) return;

    Cursor ld, cc;  // the tile to load next, the tile to compute next
    ld.row = sh.first_row;
    ld.tokens = row_tokens(p.at, p.cap, ld.row);
    ld.tiles = tiles_of(ld.tokens);
    ld.item = (int)(sh.first_at / ld.tiles);
    ld.tile = (int)(sh.first_at % ld.tiles);
    cc = ld;
    const int count = (int)(end - begin);
    int to_load = count;

    unsigned char* ring = smem + warp * S * kStage;
    const T* kbase = static_cast<const T*>(p.kv.k);
    const T* vbase = static_cast<const T*>(p.kv.v);

    // Page of this lane's token (TILED: of the warp's 16 tokens; else lanes 0-15 have one
    // each) of the tile at `ld`, looked up one tile ahead of its loads.  -1: past the
    // row's tokens, or no such page.
    const int32_t* pages = p.at.table + sequence_of(p.at, ld.row) * p.at.table_stride;
    int page = -1, in_page = 0;
    bool looked = false;
    uint32_t filled = 0;  // TILED: byte s is the number of tokens on their way to stage s
    bool failed = false;  // a bounded wait gave up: nothing more is loaded or computed
    auto look_up = [&]() {  // only starts the table's load: what it names is checked when it is used
        page = -1;
        looked = false;
        if (to_load <= 0) return;
        const int tok = ld.tile * kTileTok + warp * kWarpTok + (TILED ? 0 : lane & 15);
        if (tok < ld.tokens) {
            looked = true;
            const uint32_t nth = quotient((uint32_t)tok, p.page_size);
            in_page = (int)((uint32_t)tok - nth * p.page_size.d);
            page = pages[nth];
        }
    };
    auto load = [&](int stage) {
        if (to_load > 0) {
            const int head = p.head_groups == 1 ? ld.item : ld.item / p.head_groups;
            if (looked && (page < 0 || page >= p.kv.n_pages)) {
                page = -1;
                if (ld.item == 0 && lane < (TILED ? 1 : 16))
                    atomicAdd(p.err, TILED ? (unsigned)min(kWarpTok, ld.tokens - (ld.tile * kTileTok + warp * kWarpTok)) : 1u);
            }
            if constexpr (TILED) {
                if (page >= 0) {
                    filled |= (uint32_t)min(kWarpTok, ld.tokens - (ld.tile * kTileTok + warp * kWarpTok)) << (8 * stage);
                    if (lane == 0) {
                        const uint32_t dst = smem_u32(ring + stage * kStage);
                        uint64_t* bar = &sh.full[warp][stage];
                        mbar_expect(bar, kStage);
                        tma_load(dst, &kmap, in_page, head, page, bar);
                        tma_load(dst + kHalf, &vmap, in_page, head, page, bar);
                    }
                }
            } else {
                const int64_t off = page < 0 ? -1
                                             : (int64_t)page * p.kv.page_stride + (int64_t)in_page * p.kv.token_stride +
                                                   (int64_t)head * p.kv.head_stride;
                const uint32_t have = __ballot_sync(0xffffffffu, page >= 0) & 0xffffu;
                if (lane == 0) sh.valid[warp][stage] = have;
                if (have) {
                    const uint32_t dst = smem_u32(ring + stage * kStage);
#pragma unroll
                    for (int i = 0; i < kWarpTok * C / 32; ++i) {
                        const int idx = i * 32 + lane, r = idx / C, ch = idx % C;
                        const int64_t ro = __shfl_sync(0xffffffffu, off, r);
                        const uint32_t at = (uint32_t)chunk_at<D>(ch, r);
                        const int64_t el = ro < 0 ? 0 : ro + ch * 8;
                        cp_async16(dst + at, kbase + el, ro < 0 ? 0 : 16);
                        cp_async16(dst + kHalf + at, vbase + el, ro < 0 ? 0 : 16);
                    }
                }
            }
            --to_load;
            if (++ld.tile == ld.tiles && to_load > 0) {
                next_item(p.at, p.rows, p.cap, items, ld);
                pages = p.at.table + sequence_of(p.at, ld.row) * p.at.table_stride;
            }
            look_up();
        }
        if constexpr (!TILED) cp_commit();
    };
    // lane constants of the operand reads: chunk 2k + hi of this lane's row, per k within a part
    int k_at[CP2], v_at[CP2];
#pragma unroll
    for (int k = 0; k < CP2; ++k) {
        k_at[k] = chunk_at<D>(2 * k + ((lane >> 3) & 1), (lane & 7) + ((lane >> 4) << 3));
        v_at[k] = chunk_at<D>(2 * k + (lane >> 4), lane & 15) + kHalf;
    }

    look_up();
#pragma unroll
    for (int s = 0; s < (TILED ? S : S - 1); ++s) load(s);

    // A fragments of q: [k][0..3] = rows g, g + 8 at (k = 2c, 2c+1), then at (2c+8, 2c+9).  The
    // third pieces of two k steps share one fragment, in rows 0-7 and 8-15: each step's MMA
    // reads its own half of the result.
    constexpr bool THIRD = N == 3 && !PACK;
    constexpr int QW = THIRD ? 6 : 4;  // words per k
    uint32_t qa[q_in_smem(D) ? 1 : KS / 2][2 * QW];
    int stage = 0;
    uint32_t phase = 0;  // bit s: parity of stage s's next completed copy
    long long done = 0;  // tiles of the run behind cc
    while (done < count) {
        // ---- one item: query heads h0..h0+nh of a row, tiles [cc.tile, cc.tile + n)
        const int n = (int)min((long long)(cc.tiles - cc.tile), (long long)count - done);
        const int kvh = cc.item / p.head_groups, hg = cc.item % p.head_groups;
        const int h0 = kvh * p.group + hg * kHeads, nh = min(kHeads, p.group - hg * kHeads);
        float scale = p.scale;
        {
            const int hq = PACK ? g & 3 : g;
            const float* qr = p.q + (int64_t)cc.row * p.q_stride + (int64_t)(h0 + (hq < nh ? hq : 0)) * D + c4 * 2;
            float2 x[KS][2];
            float top = 0.f;
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    x[k][j] = hq < nh ? *reinterpret_cast<const float2*>(qr + k * 16 + j * 8) : make_float2(0.f, 0.f);
                    top = fmaxf(top, fmaxf(fabsf(x[k][j].x), fabsf(x[k][j].y)));
                }
            if constexpr (N == 2) {
                // f16 pieces: bring the head's largest |q| into [2^7, 2^8)
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const int e = max(-100, min(100, 134 - (int)((__float_as_uint(top) >> 23) & 255)));
                const float up = __uint_as_float((uint32_t)(127 + e) << 23);
                scale *= __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
                for (int k = 0; k < KS; ++k)
#pragma unroll
                    for (int j = 0; j < 2; ++j) x[k][j].x *= up, x[k][j].y *= up;
            }
#pragma unroll
            for (int k = 0; k < KS; k += 2) {
                uint32_t f[2 * QW];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    uint32_t w[2][N];
                    cut<N, T>(w[0], x[k + i][0].x, x[k + i][0].y);
                    cut<N, T>(w[1], x[k + i][1].x, x[k + i][1].y);
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        f[4 * i + 2 * j] = PACK && g >= 4 ? w[j][N - 1] : w[j][0];
                        f[4 * i + 2 * j + 1] = PACK && g >= 4 ? 0u : w[j][1];
                        if constexpr (THIRD) f[8 + 2 * j + i] = w[j][2];
                    }
                }
#pragma unroll
                for (int i = 0; i < 2 * QW; ++i) {
                    if constexpr (!q_in_smem(D)) qa[k / 2][i] = f[i];
                    else if (k / 2 % kWarps == warp) q_frag[(k / 2 * 2 * QW + i) * 32 + lane] = f[i];
                }
            }
        }
        __syncthreads();  // q_frag is written; the previous item's merge buffers are read

        float o[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t) o[t][0] = o[t][1] = 0.f;
        float m = -INFINITY, l = 0.f;  // running maximum (scaled, less kShift) and this lane's part of the sum

        for (int t = 0; t < n; ++t) {
            const int cur = stage;
            stage = stage + 1 == S ? 0 : stage + 1;
            const uint32_t base = smem_u32(ring + cur * kStage);
            uint32_t have;  // bit per token
            if constexpr (TILED) {
                if (failed) continue;
                have = (1u << ((filled >> (8 * cur)) & 255)) - 1;
                if (have) {
                    if (!__all_sync(0xffffffffu, mbar_wait(&sh.full[warp][cur], (phase >> cur) & 1))) {
                        if (lane == 0) atomicAdd(p.err + 1, 1u);
                        failed = true;
                        continue;
                    }
                    phase ^= 1u << cur;
                    filled &= ~(255u << (8 * cur));
                }
            } else {
                cp_wait<S - 2>();
                __syncwarp();
                load(cur == 0 ? S - 1 : cur - 1);  // the stage that the previous tile freed
                have = sh.valid[warp][cur];
            }
            if (have == 0) {
                if constexpr (TILED) load(cur);
                continue;
            }
            if (TILED && have != 0xffffu) {
                // slots behind the last token may hold anything, also NaN: their values are zeroed
                for (int i = lane; i < kWarpTok * C; i += 32)
                    if (!((have >> (i / C)) & 1))
                        *reinterpret_cast<uint4*>(ring + cur * kStage + kHalf + chunk_at<D>(i % C, i / C)) = make_uint4(0, 0, 0, 0);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
            }

            // ---- s = q . k for 16 tokens: two 8-token MMA columns
            float acc[2][2][4], low[2][2][4];
#pragma unroll
            for (int k = 0; k < KS; k += 2) {
                uint32_t a[2 * QW];
                if constexpr (q_in_smem(D)) {
#pragma unroll
                    for (int i = 0; i < 2 * QW; ++i) a[i] = q_frag[(k * QW + i) * 32 + lane];
                } else {
#pragma unroll
                    for (int i = 0; i < 2 * QW; ++i) a[i] = qa[k / 2][i];
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    uint32_t b[4];
                    ldmatrix4(b, base + (k + i) / CP2 * kPart + k_at[(k + i) % CP2]);
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        if (k == 0) mma0(acc[j][i], a[4 * i], a[4 * i + 1], a[4 * i + 2], a[4 * i + 3], b[2 * j], b[2 * j + 1], T());
                        else mma(acc[j][i], a[4 * i], a[4 * i + 1], a[4 * i + 2], a[4 * i + 3], b[2 * j], b[2 * j + 1], T());
                        if constexpr (THIRD) {
                            if (k == 0) mma0(low[j][i], a[8], a[9], a[10], a[11], b[2 * j], b[2 * j + 1], T());
                            else mma(low[j][i], a[8], a[9], a[10], a[11], b[2 * j], b[2 * j + 1], T());
                        }
                    }
                }
            }
            float s[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int j = i >> 1, e = i & 1;
                s[i] = acc[j][0][e + 2] + acc[j][1][e + 2];
                if constexpr (THIRD) s[i] += low[j][0][e] + low[j][1][e + 2];
                s[i] += acc[j][0][e] + acc[j][1][e];
                if constexpr (PACK) s[i] += __shfl_xor_sync(0xffffffffu, s[i], 16);
            }
            if (have != 0xffffu) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (!((have >> (8 * (i >> 1) + 2 * c4 + (i & 1))) & 1)) s[i] = -INFINITY;
            }
            float top = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const float m_new = fmaxf(m, top * scale - kShift<T>);
            const float ref = m_new == -INFINITY ? 0.f : m_new;
            const float alpha = ex2(m - ref);
            m = m_new;
            float w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = ex2(fmaf(s[i], scale, -ref));
            l = l * alpha + ((w[0] + w[1]) + (w[2] + w[3]));

            // ---- o = o * alpha + p . v
            uint32_t pa[2][N];
            cut<N, T>(pa[0], w[0], w[1]);
            cut<N, T>(pa[1], w[2], w[3]);
            if constexpr (PACK) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    pa[j][0] = g >= 4 ? pa[j][2] : pa[j][0];
                    pa[j][1] = g >= 4 ? 0u : pa[j][1];
                }
            }
#pragma unroll
            for (int c = 0; c < NT; c += 2) {
                uint32_t b[4];
                ldmatrix4_t(b, base + c / 2 / CP2 * kPart + v_at[c / 2 % CP2]);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float d[4];
                    if constexpr (THIRD) {
                        mma0(d, pa[0][2], 0u, pa[1][2], 0u, b[2 * j], b[2 * j + 1], T());
                        mma(d, pa[0][0], pa[0][1], pa[1][0], pa[1][1], b[2 * j], b[2 * j + 1], T());
                    } else {
                        mma0(d, pa[0][0], pa[0][1], pa[1][0], pa[1][1], b[2 * j], b[2 * j + 1], T());
                    }
                    o[c + j][0] = fmaf(o[c + j][0], alpha, d[0] + d[2]);
                    o[c + j][1] = fmaf(o[c + j][1], alpha, d[1] + d[3]);
                }
            }
            if constexpr (TILED) {
                __syncwarp();  // every lane has read the stage
                load(cur);
            }
        }

        // ---- join the four warps
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        if (c4 == 0) sh.m[warp][g] = m, sh.l[warp][g] = l;
        const long long item_begin = begin + done - cc.tile, item_end = item_begin + cc.tiles;
        const long long c0 = run_of(total, P, item_begin), c1 = run_of(total, P, item_end - 1);
        const bool whole = c0 == c1;
        float* slot = p.part + (2 * cta + (cta == c0 ? 1 : 0)) * slot_floats(D);
#pragma unroll
        for (int col0 = 0; col0 < D; col0 += MC) {
            if (col0) __syncthreads();  // the previous columns are read
#pragma unroll
            for (int t = 0; t < MC / 8; ++t)
                *reinterpret_cast<float2*>(merge_o + (warp * kHeads + g) * MC + ((t * 8 + c4 * 2) ^ ((g & 3) << 3))) =
                    make_float2(o[col0 / 8 + t][0], o[col0 / 8 + t][1]);
            __syncthreads();
#pragma unroll
            for (int i = 0; i < (kRows * MC / 4 + kThreads - 1) / kThreads; ++i) {
                const int idx = i * kThreads + tid, h = idx / (MC / 4), col = idx % (MC / 4) * 4;
                if (idx >= kRows * MC / 4) break;
                float top = -INFINITY;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sh.m[w][h]);
                const float ref = top == -INFINITY ? 0.f : top;
                float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
                float sum = 0.f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    const float f = ex2(sh.m[w][h] - ref);
                    float4 x = *reinterpret_cast<const float4*>(merge_o + (w * kHeads + h) * MC + (col ^ ((h & 3) << 3)));
                    if constexpr (PACK) {  // h + 4 has the same swizzle
                        const float4 z = *reinterpret_cast<const float4*>(merge_o + (w * kHeads + h + 4) * MC + (col ^ ((h & 3) << 3)));
                        x.x += z.x; x.y += z.y; x.z += z.z; x.w += z.w;
                    }
                    sum += sh.l[w][h] * f;
                    a.x += x.x * f; a.y += x.y * f; a.z += x.z * f; a.w += x.w * f;
                }
                if (h >= nh) continue;
                if (whole) {
                    const float inv = sum == 0.f ? 0.f : 1.0f / sum;
                    *reinterpret_cast<float4*>(p.out + ((int64_t)cc.row * p.n_heads + h0 + h) * D + col0 + col) =
                        make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv);
                } else {
                    __stcg(reinterpret_cast<float4*>(slot + h * D + col0 + col), a);
                    if (col0 + col == 0) {
                        __stcg(slot + kHeads * D + h, top);
                        __stcg(slot + kHeads * D + kHeads + h, sum);
                    }
                }
            }
        }
        if (!whole) {
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                sh.last_in = atomicAdd(p.counters + c0, 1u) == (unsigned)(c1 - c0);
                if (sh.last_in) p.counters[c0] = 0;
                __threadfence();
            }
            __syncthreads();
            if (sh.last_in) {
                // ---- this CTA is the last one of the item: join all, in CTA order
                const int parts = (int)(c1 - c0) + 1;
                const float* first = p.part + (2 * c0 + 1) * slot_floats(D);
                const float* rest = p.part + 2 * c0 * slot_floats(D);
                auto part_of = [&](int i) { return i == 0 ? first : rest + (int64_t)2 * i * slot_floats(D); };
                for (int h = warp; h < nh; h += kWarps) {
                    float top = -INFINITY;
                    for (int i = lane; i < parts; i += 32) top = fmaxf(top, __ldcg(part_of(i) + kHeads * D + h));
#pragma unroll
                    for (int s = 16; s; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
                    const float ref = top == -INFINITY ? 0.f : top;
                    float sum = 0.f;
                    for (int i = lane; i < parts; i += 32)
                        sum += __ldcg(part_of(i) + kHeads * D + kHeads + h) * ex2(__ldcg(part_of(i) + kHeads * D + h) - ref);
#pragma unroll
                    for (int s = 16; s; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
                    if (lane == 0) sh.m[0][h] = ref, sh.l[0][h] = sum == 0.f ? 0.f : 1.0f / sum;
                }
                __syncthreads();
                for (int idx = tid; idx < nh * (D / 4); idx += kThreads) {
                    const int h = idx / (D / 4), col = idx % (D / 4) * 4;
                    const float ref = sh.m[0][h], inv = sh.l[0][h];
                    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
                    for (int i = 0; i < parts; ++i) {
                        const float f = ex2(__ldcg(part_of(i) + kHeads * D + h) - ref);
                        const float4 x = __ldcg(reinterpret_cast<const float4*>(part_of(i) + h * D + col));
                        a.x += x.x * f; a.y += x.y * f; a.z += x.z * f; a.w += x.w * f;
                    }
                    *reinterpret_cast<float4*>(p.out + ((int64_t)cc.row * p.n_heads + h0 + h) * D + col) =
                        make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv);
                }
            }
        }
        done += n;
        if (done < count) next_item(p.at, p.rows, p.cap, items, cc);
    }
    if constexpr (TILED) {
        if (failed)  // copies in flight must not land after the CTA has gone
            for (int i = 0; i < S; ++i)
                if ((filled >> (8 * i)) & 255) mbar_wait(&sh.full[warp][i], (phase >> i) & 1);
    } else {
        cp_wait<0>();
    }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
    static const EncodeTiledFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
                       q == cudaDriverEntryPointSuccess
                   ? reinterpret_cast<EncodeTiledFn>(p)
                   : nullptr;
    }();
    return fn;
}

template <int D>
bool encode(CUtensorMap* map, void* base, const KvCache& kv) {
    constexpr int PE = part_elems(D);
    // the stride of a dimension of size 1 is never used, but has to be a legal one
    auto bytes = [](int64_t n, int64_t stride) { return (cuuint64_t)(n > 1 ? stride : (int64_t)D) * 2; };
    const cuuint64_t dims[5] = {PE, (cuuint64_t)kv.page_size, D / PE, (cuuint64_t)kv.n_kv, (cuuint64_t)kv.n_pages};
    const cuuint64_t strides[4] = {(cuuint64_t)kv.token_stride * 2, PE * 2, bytes(kv.n_kv, kv.head_stride),
                                   bytes(kv.n_pages, kv.page_stride)};
    const cuuint32_t box[5] = {PE, kWarpTok, D / PE, 1, 1}, ones[5] = {1, 1, 1, 1, 1};
    return encode_fn()(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 5, base, dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                       PE == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                       CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, class T, bool TILED, bool PACK>
cudaError_t launch_typed(const AttnArgs& a, const CUtensorMap (&maps)[2], int sms, bool pdl, cudaStream_t s) {
    static bool configured[kMaxDevices] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= kMaxDevices || !configured[dev]) {
        e = cudaFuncSetAttribute(attention_kernel<D, T, TILED, PACK>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes(D));
        if (e != cudaSuccess) return e;
        if (dev < kMaxDevices) configured[dev] = true;
    }
    const int64_t tiles = (int64_t)a.rows * a.n_kv * a.head_groups * ((a.cap + kTileTok - 1) / kTileTok);
    const int64_t ctas = (int64_t)sms * ctas_per_sm(D);
    return launch_kernel(attention_kernel<D, T, TILED, PACK>, dim3((unsigned)(tiles < ctas ? tiles : ctas)), kThreads,
                         smem_bytes(D), pdl, s, a, maps[0], maps[1]);
}

template <int D, bool TILED>
cudaError_t launch_tiled(const AttnArgs& a, const CUtensorMap (&maps)[2], int sms, bool pdl, cudaStream_t s) {
    if (a.kv.type != kKvBf16) return launch_typed<D, __half, TILED, false>(a, maps, sms, pdl, s);
    return a.group <= 4 ? launch_typed<D, __nv_bfloat16, TILED, true>(a, maps, sms, pdl, s)
                        : launch_typed<D, __nv_bfloat16, TILED, false>(a, maps, sms, pdl, s);
}

template <int D>
cudaError_t launch_dim(const AttnArgs& a, int sms, bool pdl, cudaStream_t s) {
    CUtensorMap maps[2] = {};
    // strides of 2^40 bytes and more do not fit a tensor map
    const bool fits = a.kv.token_stride < (1ll << 39) && a.kv.head_stride < (1ll << 39) && a.kv.page_stride < (1ll << 39);
    if (a.kv.page_size % kWarpTok == 0 && fits && encode_fn() && encode<D>(&maps[0], a.kv.k, a.kv) && encode<D>(&maps[1], a.kv.v, a.kv))
        return launch_tiled<D, true>(a, maps, sms, pdl, s);
    return launch_tiled<D, false>(a, maps, sms, pdl, s);
}

}  // namespace

size_t attention_part_bytes(int sms) {
    size_t most = 0;
    for (int d : {64, 96, 128, 256}) {
        const size_t b = (size_t)sms * ctas_per_sm(d) * 2 * slot_floats(d) * 4;
        most = b > most ? b : most;
    }
    return most;
}
size_t attention_counters(int sms) { return (size_t)sms * max_ctas_per_sm; }

cudaError_t launch_paged_attention(const float* q, int64_t q_stride, int64_t rows, int64_t n_heads, const KvCache& kv,
                                   const KvRows& at, float scale, float* out, float* part, unsigned int* counters,
                                   unsigned int* err, int sms, bool pdl, cudaStream_t s) {
    AttnArgs a{};
    a.q = q;
    a.q_stride = q_stride;
    a.rows = (int)rows;
    a.n_heads = (int)n_heads;
    a.n_kv = (int)kv.n_kv;
    a.group = (int)(n_heads / kv.n_kv);
    a.head_groups = (a.group + kHeads - 1) / kHeads;
    a.kv = kv;
    a.at = at;
    a.page_size = divisor_of((uint32_t)kv.page_size);
    const int64_t cap = at.max_pages * kv.page_size;
    a.cap = (int)(cap < 0x7fffff00 ? cap : 0x7fffff00);
    a.scale = scale * 1.4426950408889634f;
    a.out = out;
    a.part = part;
    a.counters = counters;
    a.err = err;
    switch (kv.head_dim) {
        case 64: return launch_dim<64>(a, sms, pdl, s);
        case 96: return launch_dim<96>(a, sms, pdl, s);
        case 128: return launch_dim<128>(a, sms, pdl, s);
        case 256: return launch_dim<256>(a, sms, pdl, s);
    }
    return cudaErrorInvalidValue;
}

}  // namespace ocl
