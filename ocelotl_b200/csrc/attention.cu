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
// head_dim, 32 tokens of p.v) and joined with rounding f32 adds.  Error against the formula
// in 64 bits, by its norm: bf16 1.4e-7 to 3.1e-7 of the result, f16 2.4e-7 to 5.0e-7 (random
// keys and values, all head_dims, up to 16000 tokens; f32 matrix products 1.3e-7 to 1.3e-6).
//
// Work split: the tiles (4 warps of 32 tokens of one row and k/v head) of all rows, in
// order, are cut into equal runs, one per resident CTA, from the positions in device
// memory -- so one captured launch stays balanced while the lengths grow (paging.cuh has
// the arithmetic).  Each warp streams its own tokens through a private ring of cp.async
// slots, rows gathered from whatever pages they lie in, and needs no barrier inside an
// item.  (Tensor-map copies of 16 tokens, with bounded waits and a second path for other
// page sizes, measured the same: 158 against 155 us for 8 rows of 30000 tokens, 8.9 against
// 9.1 for one of 555; issuing them took a warp as long as the gather.)  A row whose tiles
// lie in several CTAs is joined by the last of them to arrive, in CTA order: the result
// does not depend on which one it is.  Nothing waits on another CTA.
//
// Measured (bf16, 8 k/v heads, head_dim 128, a pass among others): 61 rows of 70 to 16000 tokens,
// 4 heads each, 131 us = 6.0 TB/s; one row of 131000 tokens 91 us = 5.9 TB/s, one of 555 7.4 us.
#include <type_traits>

#include "device.cuh"
#include "internal.cuh"

namespace ocl {

namespace {

constexpr int kHeads = 8;   // query heads of one k/v head worked on together
constexpr int kBoxTok = 16; // tokens kept together: those of one p.v MMA

// How the 8 rows of a piece's MMA rows are used:
enum Mode {
    kPlain,   // the query heads of a row (kHeads at a time)
    kPacked,  // bf16, at most 4 of them: two pieces side by side
    kShared,  // those of several rows of one sequence: 8, 4 or 2 rows of 1, 2 or 4 heads
};
// Tokens a warp takes at a time.  32 halve the work a token costs besides its MMAs
// (maximum, rescaling, waits, look-ups) and give a warp twice the independent MMAs; at
// head_dim 256 they would not leave three slots to each of 8 warps.
constexpr int warp_tok(int d) { return d == 256 ? 16 : 32; }
// Warps and ring.  Up to head_dim 128 four warps, each with a ring of slots that hold the
// keys and the values of its tokens: a tile takes about as long as HBM takes to bring it.
// At head_dim 256 a tile takes a warp twice as long and eight are wanted; their rings have
// separate slots for keys and values, so that three of 8 KB keep copies under way
// (6 rows of 900 to 6000 tokens, 4 k/v heads of 8: 25.6 us with four warps, 22.9 with
// eight; at head_dim 128 both changes lose: 64 ragged rows 123 us, 143 and 129; sixteen warps
// at 256, two to the halves of 16 tokens' elements: 64 rows of 1000 tokens 63 us, of eight 55).
constexpr bool split_slots(int d) { return d == 256; }
constexpr int warps(int d) { return d == 256 ? 8 : 4; }
constexpr int slots(int d) { return d == 96 ? 4 : 3; }
// CTAs of w warps that an SM holds.  With one warp a CTA, items are not shared by warps
// (many_items below).
constexpr int ctas_per_sm(int d, int w) { return w > 1 ? (d == 64 ? 2 : 1) : d == 64 ? 8 : d == 256 ? 5 : 4; }
constexpr int max_ctas_per_sm = 8;
constexpr int tile_tok(int d, int w) { return w * warp_tok(d); }
// A box of 16 tokens of k or v is kept as parts of 64 elements (32 for head_dim 96): a part is
// 16 rows of 128 (64) bytes, its 16-byte chunks exclusive-or'ed with the row.
constexpr int part_elems(int d) { return d % 64 == 0 ? 64 : 32; }
constexpr int part_bytes(int d) { return kBoxTok * part_elems(d) * 2; }
constexpr int box_bytes(int d) { return kBoxTok * d * 2; }
constexpr int half_bytes(int d) { return warp_tok(d) * d * 2; }  // keys or values of a warp's tokens
constexpr int slot_bytes(int d) { return (split_slots(d) ? 1 : 2) * half_bytes(d); }
constexpr int merge_cols(int d) { return d == 256 ? 64 : d; }
constexpr bool q_in_smem(int d) { return d > 128; }
constexpr int q_bytes(int d) { return q_in_smem(d) ? d / 16 * 32 * 24 : 0; }
constexpr int slot_floats(int d) { return kHeads * d + 2 * kHeads; }

template <int W>
struct Shared {  // behind the ring, the merge buffer and the q fragments
    uint32_t scan[W], longest[W];
    Cursor first;
    uint32_t edge[2];
    int last_in;
    uint32_t valid[W][4];  // a bit per token of a tile of the warp, by the tile's number in the run modulo 4
    float m[W][kHeads], l[W][kHeads], top[W][kHeads];
};
constexpr int ring_bytes(int d, int w) { return w * slots(d) * slot_bytes(d); }
constexpr int merge_bytes(int d, int w) { return w * kHeads * merge_cols(d) * 4; }
constexpr int shared_bytes(int w) { return (int)(w == 8 ? sizeof(Shared<8>) : w == 4 ? sizeof(Shared<4>) : sizeof(Shared<1>)); }
constexpr int smem_bytes(int d, int w) { return ring_bytes(d, w) + merge_bytes(d, w) + q_bytes(d) + shared_bytes(w); }
constexpr bool fits(int d, int w) { return ctas_per_sm(d, w) * (smem_bytes(d, w) + 1024) <= 228 * 1024; }
static_assert(fits(64, 4) && fits(96, 4) && fits(128, 4) && fits(256, 8) && fits(64, 1) && fits(96, 1) && fits(128, 1) && fits(256, 1),
              "CTAs per SM");

struct AttnArgs {
    const float* q;
    int64_t q_stride;
    int rows, n_heads, n_kv, group, head_groups;
    KvCache kv;
    KvRows at;
    Divisor page_size;
    int cap;      // tokens a row of the block table can hold
    float scale;  // in units of log2
    int snap;     // tiles that a cut moves at most to reach an item's edge
    int head_shift;  // kShared: query heads of a row, as a power of two
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

template <int V>
__device__ __forceinline__ void load_cg(float (&x)[V], const float* p) {
    if constexpr (V == 4) {
        const float4 t = __ldcg(reinterpret_cast<const float4*>(p));
        x[0] = t.x; x[1] = t.y; x[2] = t.z; x[3] = t.w;
    } else if constexpr (V == 2) {
        const float2 t = __ldcg(reinterpret_cast<const float2*>(p));
        x[0] = t.x; x[1] = t.y;
    } else {
        x[0] = __ldcg(p);
    }
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

// x, or NaN where it is infinite.  An infinite key or value meets each piece of its other
// factor by itself, so the sum is an infinity or NaN by the signs of low-order pieces: either
// becomes NaN, so that a score of minus infinity does not leave its token out silently.
__device__ __forceinline__ float finite_or_nan(float x) { return fmaf(x, 0.f, x); }

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

// Whether one of eight 16-bit elements is an infinity or a NaN.
template <class T>
__device__ __forceinline__ bool not_finite(uint4 w, T) {
    constexpr uint32_t kLow = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u, kHigh = kLow << 16;
    bool odd = false;
    for (const uint32_t x : {w.x, w.y, w.z, w.w}) odd |= (x & kLow) == kLow || (x & kHigh) == kHigh;
    return odd;
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
// of o.
//
// SHARE: an item has several rows of one sequence, which read its tokens together: from
// shared memory, the L2 and HBM once for all of them.  Each row has its own length; in the
// tiles where one ends, its scores are masked, and values that it does not see are zeroed
// in shared memory before its p.v (0 * NaN would not be 0), longest row first.
template <int D, class T, int MODE, int W>
__global__ void __launch_bounds__(32 * W, ctas_per_sm(D, W)) attention_kernel(const AttnArgs p) {
    constexpr int kWarps = W, kThreads = 32 * kWarps;
    constexpr bool PACK = MODE == kPacked, SHARE = MODE == kShared;
    constexpr int S = slots(D), KS = D / 16, NT = D / 8, C = D / 8, N = kPieces<T>;
    constexpr int WT = warp_tok(D), TT = tile_tok(D, W), H = WT / kBoxTok;  // H boxes of 16 tokens a slot
    constexpr uint32_t kAll = 0xffffffffu >> (32 - WT);
    constexpr int kBox = box_bytes(D), kHalf = half_bytes(D), kSlot = slot_bytes(D), kPart = part_bytes(D);
    constexpr int CP2 = part_elems(D) / 16;
    constexpr bool SPLIT = split_slots(D), QS = q_in_smem(D);
    constexpr int MC = merge_cols(D), kRows = PACK ? 4 : kHeads;
    constexpr bool THIRD = N == 3 && !PACK;               // third pieces of two k steps in one fragment
    constexpr int QV = THIRD ? 3 : 2;                     // 16-byte vectors of q's pieces per two k steps
    constexpr int XP = QS ? KS / 2 / kWarps : KS / 2;     // pairs of k steps that a warp cuts up
    static_assert(!QS || KS / 2 % kWarps == 0, "pairs of k steps by warp");
    extern __shared__ __align__(1024) unsigned char smem[];
    float* merge_o = reinterpret_cast<float*>(smem + ring_bytes(D, W));
    uint4* q_frag = reinterpret_cast<uint4*>(smem + ring_bytes(D, W) + merge_bytes(D, W));
    using Sh = Shared<W>;
    Sh& sh = *reinterpret_cast<Sh*>(smem + ring_bytes(D, W) + merge_bytes(D, W) + q_bytes(D));

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c4 = lane & 3;
    const int items = p.n_kv * p.head_groups;
    grid_wait();

    // ---- this CTA's run: the rows' units summed over the threads, then its two cuts
    // located, one by either half of the CTA (which both sum all rows)
    constexpr int kSides = kWarps > 1 ? 2 : 1, kHalfThreads = kThreads / kSides, kHalfWarps = kWarps / kSides;
    const int side = warp / kHalfWarps, most = (p.rows + kHalfThreads - 1) / kHalfThreads;
    const int per = SHARE ? (most + p.at.together - 1) & -p.at.together : most;
    const int r0 = min(tid % kHalfThreads * per, p.rows), r1 = min(r0 + per, p.rows);
    uint32_t mine = 0, longest = 0;
    int first_tokens = 0;
    if constexpr (!SHARE) {
#pragma unroll 4
        for (int r = r0; r < r1; ++r) {
            const int tokens = row_tokens(p.at, p.cap, r), tiles = tiles_of(tokens, TT);
            if (r == r0) first_tokens = tokens;
            if (tiles) mine += item_units(tiles);
            longest = max(longest, (uint32_t)tiles);
        }
    } else {
        int seq = 0, tokens = 0;  // of the item so far
        auto item_ends = [&]() {
            const int tiles = tiles_of(tokens, TT);
            if (tiles) mine += item_units(tiles);
            longest = max(longest, (uint32_t)tiles);
            tokens = 0;
        };
#pragma unroll 4
        for (int r = r0; r < r1; ++r) {
            const int n = row_tokens(p.at, p.cap, r), of = p.at.seqs[r];
            if ((r & (p.at.together - 1)) == 0 || of != seq) item_ends();
            tokens = max(tokens, n);
            seq = of;
        }
        item_ends();
    }
    mine *= items;
    longest = __reduce_max_sync(0xffffffffu, longest);
    uint32_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t t = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += t;
    }
    if (lane == 31) sh.scan[warp] = upto, sh.longest[warp] = longest;
    __syncthreads();
    uint32_t total = 0;
#pragma unroll
    for (int w = 0; w < kHalfWarps; ++w) {
        if (w < warp % kHalfWarps) upto += sh.scan[w];
        total += sh.scan[w];
        longest = max(longest, sh.longest[w]);
    }
    // Pieces of an item cost their join: about a twentieth of a tile's time each, so the
    // longest item is cut into no more than sqrt(20 * tiles) of them (one row of 2000 tokens,
    // head_dim 256: 15.0 us with sqrt(10 * tiles), 12.8, 12.8 with sqrt(40 * tiles)).
    // Items of one or two tiles are left
    // whole (200 tokens: 8.9 us cut in two, 7.0 whole).
    const Runs runs = runs_of(total, gridDim.x, max(1u, (uint32_t)(sqrtf(0.05f * (float)longest) + 0.999f)),
                              longest <= 2 ? max(p.snap, 1) : p.snap);
    const uint32_t cta = blockIdx.x;
    const bool active = total > 0 && cta < runs.P;
    for (int i = side; i < 2; i += kSides) {
        const uint32_t cut = run_cut(runs, cta + i);
        uint32_t at = upto - mine;
        if (active && cut >= at && cut < upto) {
            for (int r = r0;;) {
                int next = r + 1;
                const int tokens = SHARE ? item_tokens(p.at, p.cap, p.rows, r, next) : r == r0 ? first_tokens : row_tokens(p.at, p.cap, r);
                const int tiles = tiles_of(tokens, TT);
                const uint32_t all = tiles ? item_units(tiles) : 0, off = cut - at;
                if (off < all * items) {
                    const uint32_t item = off / all, u = off - item * all, moved = moved_cut(runs, u, tiles);
                    sh.edge[i] = cut - u + moved;
                    if (i == 0) sh.first = {r, next, (int)item, tokens, tiles, moved ? (int)moved - kItemCost : 0, 0, cut - u};
                    break;
                }
                at += all * items;
                r = next;
            }
        }
    }
    __syncthreads();
    uint32_t end = 0;
    Cursor ld = {};  // the tile to load next
    if (active) {
        end = cta + 1 == runs.P ? total : sh.edge[1];
        if (sh.edge[0] < end) {
            ld = sh.first;
            if (ld.tile == ld.tiles) next_item(p.at, p.rows, p.cap, items, TT, end, ld);
            else set_stop(ld, end);
        }
    }
    Cursor cc = ld;  // the item to compute next

    unsigned char* ring = smem + warp * S * kSlot;
    const uint32_t n_pages = (uint32_t)p.kv.n_pages;  // below 2^31
    const T* kbase = static_cast<const T*>(p.kv.k);
    const T* vbase = static_cast<const T*>(p.kv.v);

    // The place of token lane % WT of the warp's tokens of the tile at `ld`, looked up one
    // tile ahead of its loads.
    const int32_t* pages = p.at.table + (ld.tile < ld.stop ? sequence_of(p.at, ld.row) * p.at.table_stride : 0);
    int page = -1, in_page = 0;
    auto look_up = [&]() {  // only starts the table's load: what it names is checked when it is used
        const int tok = ld.tile * TT + warp * WT + lane % WT;
        if (ld.tile < ld.stop && tok < ld.tokens) {
            const uint32_t nth = quotient((uint32_t)tok, p.page_size);
            in_page = (int)((uint32_t)tok - nth * p.page_size.d);
            page = pages[nth];
        }
    };
    // Loads: 4 lanes a row, 64 bytes of it at a time, 8 rows together; the row's place comes
    // from the lane that looked it up.  Rows without a place are zeros.
    constexpr int CG = C / 4;
    const int rq = lane >> 2, cq = lane & 3;
    int dst_at[CP2 == 4 ? 2 : 1];  // where this lane's chunk of an even / odd run of 4 goes
    dst_at[0] = chunk_at<D>(cq, rq);
    if constexpr (CP2 == 4) dst_at[1] = chunk_at<D>(4 + cq, rq);
    bool values = false;   // SPLIT: the next load is of the tile's values
    int64_t place = 0;     // this lane's token's, in elements; -1: none
    uint32_t have_ld = 0;  // the tile's tokens that have a place
    uint32_t full = 0;     // bit s: slot s holds (SPLIT: the keys of) all of the warp's tokens; else sh.valid says which
    int loaded = 0;
    auto load = [&](int slot) {
        if (ld.tile < ld.stop) {
            if (!SPLIT || !values) {
                const int head = p.head_groups == 1 ? ld.item : ld.item / p.head_groups;
                const bool mine = ld.tile * TT + warp * WT + lane % WT < ld.tokens, ok = (uint32_t)page < n_pages;
                place = mine && ok ? (int64_t)page * p.kv.page_stride + (int64_t)in_page * p.kv.token_stride +
                                         (int64_t)head * p.kv.head_stride
                                   : -1;
                if (__all_sync(0xffffffffu, mine && ok)) {
                    have_ld = kAll;
                    full |= 1u << slot;
                } else {
                    have_ld = __ballot_sync(0xffffffffu, mine && ok) & kAll;
                    if (mine && !ok && ld.item == 0 && lane < WT) atomicAdd(p.err, 1u);
                    if (lane == 0) sh.valid[warp][loaded & 3] = have_ld;
                    full &= ~(1u << slot);
                }
                ++loaded;
            }
            if (have_ld) {
                const uint32_t dst = smem_u32(ring + slot * kSlot);
                const T* from = SPLIT && values ? vbase : kbase;
#pragma unroll
                for (int rg = 0; rg < WT / 8; ++rg) {
                    const int64_t row = __shfl_sync(0xffffffffu, place, rg * 8 + rq);
                    const int bytes = row < 0 ? 0 : 16;
                    const int64_t el = (row < 0 ? 0 : row) + cq * 8;
                    const uint32_t to = dst + rg / 2 * kBox + rg % 2 * 8 * part_elems(D) * 2;
#pragma unroll
                    for (int cg = 0; cg < CG; ++cg) {
                        const uint32_t at = to + (CP2 == 4 ? cg / 2 : cg) * kPart + dst_at[CP2 == 4 ? cg % 2 : 0];
                        cp_async16(at, from + el + cg * 32, bytes);
                        if constexpr (!SPLIT) cp_async16(at + kHalf, vbase + el + cg * 32, bytes);
                    }
                }
            }
            if (!SPLIT || values) {
                if (++ld.tile == ld.stop && next_item(p.at, p.rows, p.cap, items, TT, end, ld))
                    pages = p.at.table + sequence_of(p.at, ld.row) * p.at.table_stride;
                look_up();
            }
            values = !values;
        }
        cp_commit();
    };
    // lane constants of the operand reads: chunk 2k + hi of this lane's row, per k within a part
    int k_at[CP2], v_at[CP2];
#pragma unroll
    for (int k = 0; k < CP2; ++k) {
        k_at[k] = chunk_at<D>(2 * k + ((lane >> 3) & 1), (lane & 7) + ((lane >> 4) << 3));
        v_at[k] = chunk_at<D>(2 * k + (lane >> 4), lane & 15);
    }

    // q of the query heads of the item at `cc`, f32: loaded ahead of its use, with what each
    // of its rows sees.  With the fragments in shared memory a warp has only those k steps
    // that it cuts up.
    float2 x[XP][2][2];
    int sees = 0, least = 0;  // tokens that the row of this lane's q sees, and the fewest that one of the rows sees
    auto load_q = [&]() {
        const int kvh = p.head_groups == 1 ? cc.item : cc.item / p.head_groups, hg = cc.item - kvh * p.head_groups;
        const int nh = min(kHeads, p.group - hg * kHeads);
        const int member = SHARE ? g >> p.head_shift : 0, hq = SHARE ? g & ((1 << p.head_shift) - 1) : PACK ? g & 3 : g;
        const bool used = hq < nh && (!SHARE || member < cc.next - cc.row);
        const float* qr = p.q + (int64_t)(cc.row + member) * p.q_stride + (int64_t)(kvh * p.group + hg * kHeads + hq) * D + c4 * 2;
        if constexpr (SHARE) {
            sees = used ? row_tokens(p.at, p.cap, cc.row + member) : 0;
            least = __reduce_min_sync(0xffffffffu, used ? sees : 0x7fffffff);
        }
#pragma unroll
        for (int i = 0; i < XP; ++i)
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    x[i][k][j] = used ? *reinterpret_cast<const float2*>(qr + (2 * (QS ? i * kWarps + warp : i) + k) * 16 + j * 8)
                                      : make_float2(0.f, 0.f);
    };

    look_up();
    if (cc.tile < cc.stop) load_q();
#pragma unroll
    for (int s = 0; s < S - 1; ++s) load(s);

    // rows without tokens are zeros; rows whose place is out of range are counted
    for (int r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const int tokens = row_tokens(p.at, p.cap, r), pos = p.at.positions[r];
        if (tid == 0 && pos >= 0 && pos >= tokens) atomicAdd(p.err, 1u);
        if (tokens == 0)
            for (int i = tid; i < p.n_heads * D; i += kThreads) p.out[(int64_t)r * p.n_heads * D + i] = 0.f;
    }
    if (cc.tile >= cc.stop) return;

    // A fragments of q: [k][0..3] = rows g, g + 8 at (k = 2c, 2c+1), then at (2c+8, 2c+9).  The
    // third pieces of two k steps share one fragment, in rows 0-7 and 8-15: each step's MMA
    // reads its own half of the result.
    uint32_t qa[QS ? 1 : KS / 2][4 * QV];
    int at_slot = 0, computed = 0;  // the ring's next slot, and the tiles of the run behind it
    // The next slot, its copies landed; the load that refills the one before it is started.
    auto arrive = [&]() {
        const int cur = at_slot;
        at_slot = at_slot + 1 == S ? 0 : at_slot + 1;
        cp_wait<S - 2>();
        __syncwarp();  // every lane's copies are in, and every lane has read the slot before
        load(cur == 0 ? S - 1 : cur - 1);
        return cur;
    };
    for (;;) {
        // ---- one item, or this run's piece of it: query heads h0..h0+nh of a row
        const int row = cc.row, tiles = cc.stop - cc.tile;
        const bool whole = tiles == cc.tiles;
        const int kvh = p.head_groups == 1 ? cc.item : cc.item / p.head_groups, hg = cc.item - kvh * p.head_groups;
        const int h0 = kvh * p.group + hg * kHeads, nh = min(kHeads, p.group - hg * kHeads), item_rows = cc.next - cc.row;
        float scale = p.scale;
        if constexpr (N == 2) {
            // f16 pieces: bring the head's largest |q| into [2^7, 2^8)
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < XP; ++i)
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int j = 0; j < 2; ++j) top = fmaxf(top, fmaxf(fabsf(x[i][k][j].x), fabsf(x[i][k][j].y)));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            if constexpr (QS && kWarps > 1) {
                if (c4 == 0) sh.top[warp][g] = top;
                __syncthreads();
#pragma unroll
                for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sh.top[w][g]);
            }
            const int e = max(-126, min(126, 134 - (int)((__float_as_uint(top) >> 23) & 255)));
            const float up = __uint_as_float((uint32_t)(127 + e) << 23);
            scale *= __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
            for (int i = 0; i < XP; ++i)
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int j = 0; j < 2; ++j) x[i][k][j].x *= up, x[i][k][j].y *= up;
        }
#pragma unroll
        for (int i = 0; i < XP; ++i) {
            uint32_t f[4 * QV];
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    uint32_t w[N];
                    cut<N, T>(w, x[i][k][j].x, x[i][k][j].y);
                    f[4 * k + 2 * j] = PACK && g >= 4 ? w[N - 1] : w[0];
                    f[4 * k + 2 * j + 1] = PACK && g >= 4 ? 0u : w[1];
                    if constexpr (THIRD) f[8 + 2 * j + k] = w[2];
                }
#pragma unroll
            for (int v = 0; v < QV; ++v) {
                if constexpr (!QS) qa[i][4 * v] = f[4 * v], qa[i][4 * v + 1] = f[4 * v + 1], qa[i][4 * v + 2] = f[4 * v + 2], qa[i][4 * v + 3] = f[4 * v + 3];
                else q_frag[((i * kWarps + warp) * QV + v) * 32 + lane] = make_uint4(f[4 * v], f[4 * v + 1], f[4 * v + 2], f[4 * v + 3]);
            }
        }
        __syncthreads();  // q_frag is written; the previous item's merge buffers are read

        float o[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t) o[t][0] = o[t][1] = 0.f;
        float m = -INFINITY, l = 0.f;  // running maximum (scaled, less kShift) and this lane's part of the sum

        for (int t = 0; t < tiles; ++t) {
            const uint32_t have = (full >> at_slot) & 1 ? kAll : sh.valid[warp][computed & 3];  // bit per token
            ++computed;
            uint32_t base = smem_u32(ring + arrive() * kSlot);
            if (have == 0) {
                if constexpr (SPLIT) arrive();
                continue;
            }
            const int t0 = (cc.tile + t) * TT + warp * WT;  // the first token
            const bool ragged = SHARE && t0 + WT > least;   // one of the rows ends in these

            // ---- s = q . k: two 8-token MMA columns a box
            float acc[H][2][2][4], low[H][2][2][4];
#pragma unroll
            for (int k = 0; k < KS; k += 2) {
                uint32_t a[4 * QV];
                if constexpr (QS) {
#pragma unroll
                    for (int v = 0; v < QV; ++v) {
                        const uint4 f = q_frag[(k / 2 * QV + v) * 32 + lane];
                        a[4 * v] = f.x, a[4 * v + 1] = f.y, a[4 * v + 2] = f.z, a[4 * v + 3] = f.w;
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 4 * QV; ++i) a[i] = qa[k / 2][i];
                }
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int h = 0; h < H; ++h) {
                        uint32_t b[4];
                        ldmatrix4(b, base + h * kBox + (k + i) / CP2 * kPart + k_at[(k + i) % CP2]);
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            if (k == 0) mma0(acc[h][j][i], a[4 * i], a[4 * i + 1], a[4 * i + 2], a[4 * i + 3], b[2 * j], b[2 * j + 1], T());
                            else mma(acc[h][j][i], a[4 * i], a[4 * i + 1], a[4 * i + 2], a[4 * i + 3], b[2 * j], b[2 * j + 1], T());
                            if constexpr (THIRD) {
                                if (k == 0) mma0(low[h][j][i], a[8], a[9], a[10], a[11], b[2 * j], b[2 * j + 1], T());
                                else mma(low[h][j][i], a[8], a[9], a[10], a[11], b[2 * j], b[2 * j + 1], T());
                            }
                        }
                    }
            }
            float s[H][4];
#pragma unroll
            for (int h = 0; h < H; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int j = i >> 1, e = i & 1;
                    s[h][i] = acc[h][j][0][e + 2] + acc[h][j][1][e + 2];
                    if constexpr (THIRD) s[h][i] += low[h][j][0][e] + low[h][j][1][e + 2];
                    s[h][i] += acc[h][j][0][e] + acc[h][j][1][e];
                    if constexpr (PACK) s[h][i] += __shfl_xor_sync(0xffffffffu, s[h][i], 16);
                    s[h][i] = finite_or_nan(s[h][i]);
                }
            if (have != kAll || ragged) {
#pragma unroll
                for (int h = 0; h < H; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int tok = 16 * h + 8 * (i >> 1) + 2 * c4 + (i & 1);
                        if (!((have >> tok) & 1) || (SHARE && t0 + tok >= sees)) s[h][i] = -INFINITY;
                    }
            }
            float top = -INFINITY;
#pragma unroll
            for (int h = 0; h < H; ++h) top = fmaxf(top, fmaxf(fmaxf(s[h][0], s[h][1]), fmaxf(s[h][2], s[h][3])));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const float m_new = fmaxf(m, top * scale - kShift<T>);
            const float ref = m_new == -INFINITY ? 0.f : m_new;
            const float alpha = ex2(m - ref);
            m = m_new;
            // ---- p, in pieces
            uint32_t pa[H][2][N];
            float more = 0.f;
#pragma unroll
            for (int h = 0; h < H; ++h) {
                float w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = ex2(fmaf(s[h][i], scale, -ref));
                more += (w[0] + w[1]) + (w[2] + w[3]);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    cut<N, T>(pa[h][j], w[2 * j], w[2 * j + 1]);
                    if constexpr (PACK) {
                        pa[h][j][0] = g >= 4 ? pa[h][j][2] : pa[h][j][0];
                        pa[h][j][1] = g >= 4 ? 0u : pa[h][j][1];
                    }
                }
            }
            l = fmaf(l, alpha, more);

            // ---- o = o * alpha + p . v; with `some` for the rows that see `only` of these tokens
            const uint32_t v_at_slot = SPLIT ? arrive() * kSlot : base - smem_u32(ring) + kHalf;
            base = smem_u32(ring) + v_at_slot;
            auto add_values = [&](auto some, int only) {
                const bool mine = !decltype(some)::value || min(sees - t0, WT) == only;
#pragma unroll
                for (int c = 0; c < NT; c += 2) {
                    float d[2][4];
#pragma unroll
                    for (int h = 0; h < H; ++h) {
                        uint32_t b[4];
                        ldmatrix4_t(b, base + h * kBox + c / 2 / CP2 * kPart + v_at[c / 2 % CP2]);
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            if constexpr (THIRD) {
                                if (h == 0) mma0(d[j], pa[h][0][2], 0u, pa[h][1][2], 0u, b[2 * j], b[2 * j + 1], T());
                                else mma(d[j], pa[h][0][2], 0u, pa[h][1][2], 0u, b[2 * j], b[2 * j + 1], T());
                            }
                            if (h == 0 && !THIRD) mma0(d[j], pa[h][0][0], pa[h][0][1], pa[h][1][0], pa[h][1][1], b[2 * j], b[2 * j + 1], T());
                            else mma(d[j], pa[h][0][0], pa[h][0][1], pa[h][1][0], pa[h][1][1], b[2 * j], b[2 * j + 1], T());
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            if (mine) o[c + j][e] = fmaf(o[c + j][e], alpha, d[j][e] + d[j][e + 2]);
                }
            };
            if constexpr (!SHARE) {
                add_values(std::false_type(), 0);
            } else {
                // Weights of 0 leave out what a row does not see, but for infinities and NaN.
                const int first = max(0, least - t0);
                unsigned char* const v_rows = ring + v_at_slot;
                auto value_at = [&](int i) {  // i-th 16 bytes of the rows that not all see
                    const int tok = first + i / C;
                    return reinterpret_cast<uint4*>(v_rows + tok / kBoxTok * kBox + chunk_at<D>(i % C, tok % kBoxTok));
                };
                bool odd = false;
                if (ragged)
                    for (int i = lane; i < (WT - first) * C; i += 32) odd |= not_finite(*value_at(i), T());
                if (!__any_sync(0xffffffffu, odd)) {
                    add_values(std::false_type(), 0);
                } else {
                    // the rows that see most of these tokens first; then the values that no other sees are zeroed
                    const int n = min(sees - t0, WT);
                    for (int only = __reduce_max_sync(0xffffffffu, n); only > 0;) {
                        add_values(std::true_type(), only);
                        __syncwarp();
                        only = __reduce_max_sync(0xffffffffu, n < only ? n : 0);
                        for (int i = lane + max(0, only - first) * C; i < (WT - first) * C; i += 32) *value_at(i) = make_uint4(0, 0, 0, 0);
                        __syncwarp();
                    }
                }
            }
        }

        uint32_t c0 = cta, c1 = cta;
        if (!whole) item_runs(runs, cc.begin, cc.tiles, c0, c1);
        next_item(p.at, p.rows, p.cap, items, TT, end, cc);
        const bool more = cc.tile < cc.stop;
        if (more) load_q();

        // ---- join the warps
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        if (c4 == 0) sh.m[warp][g] = m, sh.l[warp][g] = l;
        if (MC < D && !more) {  // the ring is free
            cp_wait<0>();
            __syncthreads();
        }
        // the row (from the item's first on) and query head that MMA row h holds; false: none
        auto holds = [&](int h, int& member, int& head) {
            member = SHARE ? h >> p.head_shift : 0;
            head = SHARE ? h & ((1 << p.head_shift) - 1) : h;
            return head < nh && (!SHARE || member < item_rows);
        };
        float* slot = p.part + (size_t)(2 * cta + (cta == c0 ? 1 : 0)) * slot_floats(D);
        auto merge = [&](auto columns, float* buffer) {  // so many columns at a time
            constexpr int kCols = decltype(columns)::value;
#pragma unroll
            for (int col0 = 0; col0 < D; col0 += kCols) {
                if (col0) __syncthreads();  // the previous columns are read
#pragma unroll
                for (int t = 0; t < kCols / 8; ++t)
                    *reinterpret_cast<float2*>(buffer + (warp * kHeads + g) * kCols + ((t * 8 + c4 * 2) ^ ((g & 3) << 3))) =
                        make_float2(o[col0 / 8 + t][0], o[col0 / 8 + t][1]);
                __syncthreads();
#pragma unroll
                for (int i = 0; i < (kRows * kCols / 4 + kThreads - 1) / kThreads; ++i) {
                    const int idx = i * kThreads + tid, h = idx / (kCols / 4), col = idx % (kCols / 4) * 4;
                    if (idx >= kRows * kCols / 4) break;
                    float top = -INFINITY;
#pragma unroll
                    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sh.m[w][h]);
                    const float ref = top == -INFINITY ? 0.f : top;
                    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
                    float sum = 0.f;
#pragma unroll
                    for (int w = 0; w < kWarps; ++w) {
                        const float f = ex2(sh.m[w][h] - ref);
                        float4 x = *reinterpret_cast<const float4*>(buffer + (w * kHeads + h) * kCols + (col ^ ((h & 3) << 3)));
                        if constexpr (PACK) {  // h + 4 has the same swizzle
                            const float4 z = *reinterpret_cast<const float4*>(buffer + (w * kHeads + h + 4) * kCols + (col ^ ((h & 3) << 3)));
                            x.x += z.x; x.y += z.y; x.z += z.z; x.w += z.w;
                        }
                        sum += sh.l[w][h] * f;
                        a.x += x.x * f; a.y += x.y * f; a.z += x.z * f; a.w += x.w * f;
                    }
                    int member, head;
                    if (!holds(h, member, head)) continue;
                    if (whole) {
                        const float inv = sum == 0.f ? 0.f : 1.0f / sum;
                        *reinterpret_cast<float4*>(p.out + ((int64_t)(row + member) * p.n_heads + h0 + head) * D + col0 + col) =
                            make_float4(finite_or_nan(a.x * inv), finite_or_nan(a.y * inv), finite_or_nan(a.z * inv), finite_or_nan(a.w * inv));
                    } else {
                        __stcg(reinterpret_cast<float4*>(slot + h * D + col0 + col), a);
                        if (col0 + col == 0) {
                            __stcg(slot + kHeads * D + h, top);
                            __stcg(slot + kHeads * D + kHeads + h, sum);
                        }
                    }
                }
            }
        };
        if constexpr (MC < D) {
            if (more) merge(std::integral_constant<int, MC>(), merge_o);
            else merge(std::integral_constant<int, D>(), reinterpret_cast<float*>(smem));
        } else {
            merge(std::integral_constant<int, MC>(), merge_o);
        }
        if (!whole) {
            __syncthreads();
            if (tid == 0) {
                unsigned int before;  // releases this CTA's part, acquires those of the CTAs before
                asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(p.counters + c0) : "memory");
                sh.last_in = before == c1 - c0;
                if (sh.last_in) p.counters[c0] = 0;
            }
            __syncthreads();
            if (sh.last_in) {
                // ---- this CTA is the last one of the item: join all, in CTA order
                // A warp takes a head, two together where there are as many: lane i holds the maximum
                // and the sum of the i-th CTA, then every lane adds its columns, B CTAs' loads in flight.
                const int parts = (int)(c1 - c0) + 1;
                const float* first = p.part + (size_t)(2 * c0 + 1) * slot_floats(D);
                const float* rest = p.part + (size_t)(2 * c0) * slot_floats(D);
                auto part_of = [&](int i) { return i == 0 ? first : rest + (size_t)(2 * i) * slot_floats(D); };
                constexpr int V = D % 128 == 0 ? 4 : D == 64 ? 2 : 1, L = D / (32 * V);  // floats a load, loads a lane
                constexpr int U = kRows >= 2 * kWarps ? 2 : 1, B = D == 96 ? 4 : 16 / L / U;
                for (int n = warp; n < kRows; n += U * kWarps) {
                    int h[U];
                    int64_t to[U];  // -1: not a head of the item
                    float top[U], sum[U], weight[U], acc[U][L][V] = {};
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        int member, head;
                        h[u] = n + u * kWarps;
                        to[u] = holds(h[u], member, head) ? ((int64_t)(row + member) * p.n_heads + h0 + head) * D + lane * V : -1;
                        top[u] = -INFINITY, sum[u] = weight[u] = 0.f;
                    }
                    for (int i0 = 0; i0 < parts; i0 += 32) {
                        float m_i[U], l_i[U];
#pragma unroll
                        for (int u = 0; u < U; ++u) {
                            m_i[u] = -INFINITY, l_i[u] = 0.f;
                            if (i0 + lane < parts) {
                                m_i[u] = __ldcg(part_of(i0 + lane) + kHeads * D + h[u]);
                                l_i[u] = __ldcg(part_of(i0 + lane) + kHeads * D + kHeads + h[u]);
                            }
                        }
                        const int n32 = min(32, parts - i0);
                        for (int b = 0; b < n32; b += B) {
                            float part_o[U][B][L][V];
#pragma unroll
                            for (int i = 0; i < B; ++i) {
                                const float* from = part_of(i0 + min(b + i, n32 - 1));
#pragma unroll
                                for (int u = 0; u < U; ++u)
#pragma unroll
                                    for (int j = 0; j < L; ++j) load_cg<V>(part_o[u][i][j], from + h[u] * D + lane * V + j * 32 * V);
                            }
#pragma unroll
                            for (int u = 0; u < U; ++u) {
                                if (b == 0) {  // the maximum over these CTAs, behind the loads
                                    float t = m_i[u];
#pragma unroll
                                    for (int s = 16; s; s >>= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, s));
                                    t = fmaxf(t, top[u]);
                                    const float ref = t == -INFINITY ? 0.f : t, less = ex2(top[u] - ref);
                                    top[u] = t;
                                    weight[u] = ex2(m_i[u] - ref);
                                    sum[u] = fmaf(sum[u], less, l_i[u] * weight[u]);
#pragma unroll
                                    for (int j = 0; j < L; ++j)
#pragma unroll
                                        for (int e = 0; e < V; ++e) acc[u][j][e] *= less;
                                }
#pragma unroll
                                for (int i = 0; i < B; ++i) {
                                    const float f = __shfl_sync(0xffffffffu, weight[u], (b + i) & 31);
                                    const bool in = b + i < n32;
#pragma unroll
                                    for (int j = 0; j < L; ++j)
#pragma unroll
                                        for (int e = 0; e < V; ++e) acc[u][j][e] = fmaf(in ? part_o[u][i][j][e] : 0.f, in ? f : 0.f, acc[u][j][e]);
                                }
                            }
                        }
                    }
#pragma unroll
                    for (int u = 0; u < U; ++u) {
#pragma unroll
                        for (int s = 16; s; s >>= 1) sum[u] += __shfl_xor_sync(0xffffffffu, sum[u], s);
                        const float inv = sum[u] == 0.f ? 0.f : 1.0f / sum[u];
                        if (to[u] < 0) continue;
#pragma unroll
                        for (int j = 0; j < L; ++j)
#pragma unroll
                            for (int e = 0; e < V; ++e) p.out[to[u] + j * 32 * V + e] = finite_or_nan(acc[u][j][e] * inv);
                    }
                }
            }
        }
        if (!more) break;
    }
    cp_wait<0>();
}

template <int D, class T, int MODE, int W>
cudaError_t launch_typed(AttnArgs a, int sms, bool pdl, cudaStream_t s) {
    constexpr int kSmem = smem_bytes(D, W);
    static bool configured[kMaxDevices] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= kMaxDevices || !configured[dev]) {
        e = cudaFuncSetAttribute(attention_kernel<D, T, MODE, W>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
        if (e != cudaSuccess) return e;
        if (dev < kMaxDevices) configured[dev] = true;
    }
    const int64_t items = (int64_t)a.rows * a.n_kv * a.head_groups, tiles = items * tiles_of(a.cap, tile_tok(D, W));
    if (tiles + items > 0x7fffffff) return cudaErrorInvalidValue;  // the runs' arithmetic; checked by the caller
    const int64_t most = (int64_t)sms * ctas_per_sm(D, W), ctas = tiles + items < most ? tiles + items : most;
    // With about as many items as CTAs, a short item is better left whole than shared (its
    // join takes longer than its tiles: 16 rows of 555 tokens and 8 k/v heads 15.2 -> 11.1
    // us, 230 rows of 5 to 180 tokens 15.3 -> 12.5); with fewer items every cut is wanted (one
    // row of 1000 tokens and 8 k/v heads 9.3 us, with moved cuts 11.7).
    a.snap = 2 * (items / a.at.together) >= ctas ? 2 : 0;
    return launch_kernel(attention_kernel<D, T, MODE, W>, dim3((unsigned)ctas), 32 * W, kSmem, pdl, s, a);
}

// Many items: one warp to each, so that short ones leave no warp idle and need no join of
// warps.  Measured against the wide CTAs, us (k/v heads x rows, tokens):
//   head_dim 128:  8 x 64, 10 11.2 -> 5.9, 100 12.8 -> 10.3, 2000 93 -> 94;  8 x 1000, 10 113 -> 47, 400 324 -> 277
//                  8 x 32, 100 8.4 -> 14.5 (too few: what is not shared by warps is shared by CTAs)
//   head_dim 64:   8 x 64, 100 7.6 -> 14.1;  8 x 128, 100 12.3 -> 9.1, 2000 91 -> 96
//   head_dim 256:  4 x 128, 100 29.7 -> 25.2, 400 66 -> 63, 2000 189 -> 211;  4 x 800, 100 119 -> 78;
//                  4 x 512, 1 to 512 145 -> 161
// so at 64 and 256 only where the block table bounds the lengths.
bool many_items(int d, int64_t items, int cap, int sms) {
    if (d == 64) return items >= 6 * (int64_t)sms && cap <= 256;
    return items >= 3 * (int64_t)sms && (d != 256 || cap <= 256);
}

template <int D, class T, int MODE>
cudaError_t launch_warps(const AttnArgs& a, int sms, bool pdl, cudaStream_t s) {
    if (many_items(D, (int64_t)(a.rows / a.at.together) * a.n_kv * a.head_groups, a.cap, sms)) return launch_typed<D, T, MODE, 1>(a, sms, pdl, s);
    return launch_typed<D, T, MODE, warps(D)>(a, sms, pdl, s);
}

// Several rows of a sequence together: where the rows outnumber the block table's sequences,
// so that some must share one, and the tiles that the table allows are four to a CTA or more.
// Measured without and with, us (sequences x rows of each, tokens):
//   8 k/v heads of 4, head_dim 128, bf16:  6 x 4, 3000 48 -> 38;  64 x 2, 1000 95 -> 65;  1 x 512, 512 87 -> 88;
//                                          8 x 100, 100 53 -> 58
//   8 of 2, head_dim 64:  6 x 4, 3000 27 -> 15;  1 x 512, 512 57 -> 26;  16 x 2, 100 (too few) 5.3 -> 6.8
//   8 of 1, head_dim 128: 1 x 4, 30000 69 -> 34;  8 x 100, 100 50 -> 29
// and 64 x 1, 1000 with no two rows of a sequence 55 -> 64 (8 of 4).  Rows of 5 or more heads
// stay by themselves: two sets of 8 in one warp took as long as two items (4 k/v heads of 8,
// head_dim 256, 6 x 4 of 3000 54 -> 59 us: a warp's instructions are the bound, not its loads).
template <int D, class T>
cudaError_t launch_dim(AttnArgs a, int sms, bool pdl, cudaStream_t s) {
    const int64_t tiles = (int64_t)a.rows * a.n_kv * tiles_of(a.cap, tile_tok(D, warps(D)));
    if (a.group <= 4 && a.at.seqs && a.rows > a.at.n_seqs && tiles >= 4 * sms * ctas_per_sm(D, warps(D))) {
        a.head_shift = a.group > 2 ? 2 : a.group - 1;
        a.at.together = kHeads >> a.head_shift;
        return launch_warps<D, T, kShared>(a, sms, pdl, s);
    }
    if constexpr (kPieces<T> == 3)
        if (a.group <= 4) return launch_warps<D, T, kPacked>(a, sms, pdl, s);
    return launch_warps<D, T, kPlain>(a, sms, pdl, s);
}

template <int D>
cudaError_t launch_type(const AttnArgs& a, int sms, bool pdl, cudaStream_t s) {
    return a.kv.type == kKvBf16 ? launch_dim<D, __nv_bfloat16>(a, sms, pdl, s) : launch_dim<D, __half>(a, sms, pdl, s);
}

}  // namespace

size_t attention_part_bytes(int sms) {
    size_t most = 0;
    for (int d : {64, 96, 128, 256}) {
        for (int w : {1, warps(d)}) {
            const size_t b = (size_t)sms * ctas_per_sm(d, w) * 2 * slot_floats(d) * 4;
            most = b > most ? b : most;
        }
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
        case 64: return launch_type<64>(a, sms, pdl, s);
        case 96: return launch_type<96>(a, sms, pdl, s);
        case 128: return launch_type<128>(a, sms, pdl, s);
        case 256: return launch_type<256>(a, sms, pdl, s);
    }
    return cudaErrorInvalidValue;
}

}  // namespace ocl
