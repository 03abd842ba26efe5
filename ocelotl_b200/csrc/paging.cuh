// paging.cuh -- index arithmetic of the paged cache and of the attention's work
// split, for the kernels and for a host build that checks it without a GPU.
#pragma once
#include <cstdint>

#ifdef __CUDACC__
#define OCL_HD __host__ __device__ __forceinline__
#else
#define OCL_HD inline
#endif

namespace ocl {

// Where the rows of a call stand: row r holds token positions[r] of sequence
// seqs[r] (r itself when seqs is null); a negative position is a padding row.
struct KvRows {
    const int32_t *positions, *seqs, *table;
    int64_t n_seqs, max_pages, table_stride;
};

// The row's sequence, or -1 if the block table has none such.
OCL_HD int64_t sequence_of(const KvRows& at, int64_t row) {
    const int64_t seq = at.seqs ? (int64_t)at.seqs[row] : row;
    return seq >= 0 && seq < at.n_seqs ? seq : -1;
}

// n / d for 0 <= n < 2^31 as a product and a shift (Granlund and Montgomery, Division
// by invariant integers using multiplication): with l = ceil(log2 d) and
// m = floor(2^(31 + l) / d) + 1, m * d exceeds 2^(31 + l) by at most 2^l.
struct Divisor {
    uint32_t d, m;
    int shift;
};
inline Divisor divisor_of(uint32_t d) {
    int l = 0;
    while ((1ull << l) < d) ++l;
    return {d, (uint32_t)(((unsigned long long)1 << (31 + l)) / d + 1), 31 + l};
}
OCL_HD uint32_t quotient(uint32_t n, const Divisor& by) { return (uint32_t)(((unsigned long long)n * by.m) >> by.shift); }

// Page and slot of token `tok` (>= 0) of the sequence with page list `pages`.  False:
// the list has no such token, or names a page that the cache has not.
OCL_HD bool place_of(const int32_t* pages, int64_t max_pages, int64_t n_pages, const Divisor& page_size, int tok, int& page,
                     int& in_page) {
    const uint32_t nth = quotient((uint32_t)tok, page_size);
    if ((int64_t)nth >= max_pages) return false;
    in_page = (int)((uint32_t)tok - nth * page_size.d);
    page = pages[nth];
    return page >= 0 && (int64_t)page < n_pages;
}

// Tokens that a row sees: 0 for a padding row or one without a sequence, at most
// `cap`, what a row of the block table can hold.
OCL_HD int row_tokens(const KvRows& at, int cap, int64_t row) {
    const int pos = at.positions[row];
    if (pos < 0 || sequence_of(at, row) < 0) return 0;
    return pos >= cap ? cap : pos + 1;
}

constexpr int kWarpTok = 16, kTileWarps = 4, kTileTok = kWarpTok * kTileWarps;  // attention: tokens of a tile
OCL_HD int tiles_of(int tokens) { return (tokens + kTileTok - 1) / kTileTok; }

// `total` tiles in P <= total runs: run c is [run_begin(c), run_begin(c + 1)), never
// empty; run_of(t) is the run that tile t lies in.
OCL_HD long long run_begin(long long total, long long P, long long c) { return total * c / P; }
OCL_HD long long run_of(long long total, long long P, long long t) { return ((t + 1) * P - 1) / total; }

// A place in the order of all tiles: by row, item (k/v head and head group), tile.
struct Cursor {
    int row, item, tile, tokens, tiles;
};
OCL_HD void next_item(const KvRows& at, int rows, int cap, int items, Cursor& c) {
    c.tile = 0;
    if (++c.item < items) return;
    c.item = 0;
    c.tokens = 0;
    do {
        ++c.row;
    } while (c.row < rows && (c.tokens = row_tokens(at, cap, c.row)) == 0);
    c.tiles = tiles_of(c.tokens);
}

}  // namespace ocl
