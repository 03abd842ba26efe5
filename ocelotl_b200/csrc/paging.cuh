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
    int together = 1;  // rows that an item may have (see item_tokens); 1 where seqs is null
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
// `cap`, what a row of the block table can hold.  Without branches, so that a thread's
// loads of several rows are under way together.
OCL_HD int row_tokens(const KvRows& at, int cap, int64_t row) {
    const int pos = at.positions[row];
    const bool there = pos >= 0 && sequence_of(at, row) >= 0;
    const int seen = pos < cap ? pos : cap - 1;
    return there ? seen + 1 : 0;
}

// The rows of an item: of each `together` (a power of two) rows from a multiple of it on,
// those that follow one another in the same sequence.  Tokens that the item which starts
// with `row` reads, the most that a row of it sees; `next` is the next item's first row.
OCL_HD int item_tokens(const KvRows& at, int cap, int rows, int row, int& next) {
    int most = row_tokens(at, cap, row);
    next = row + 1;
    if (at.together > 1) {
        const int all = (row | (at.together - 1)) + 1, behind = all < rows ? all : rows, seq = at.seqs[row];
        for (; next < behind && at.seqs[next] == seq; ++next) {
            const int tokens = row_tokens(at, cap, next);
            most = tokens > most ? tokens : most;
        }
    }
    return most;
}

OCL_HD int tiles_of(int tokens, int tile_tok) { return (tokens + tile_tok - 1) / tile_tok; }

// The work of all items (an item: a row and group of heads; its tiles, after kItemCost
// units for what an item costs by itself) in order, cut into P runs, one per CTA.
// Cut c lies on unit c * total / P, up to a unit; one within `snap` tiles of an item's
// edge moves to that edge, so that an item is not shared for a sliver of it, and items
// of up to 2 * snap tiles are never shared.  All in 32 bits: total < 2^31.
constexpr int kItemCost = 1;
struct Runs {
    uint32_t total, P, share, rest;  // total = P * share + rest
    int snap;
};
OCL_HD uint32_t item_units(int tiles) { return (uint32_t)(tiles + kItemCost); }
OCL_HD Runs runs_of(uint32_t total, uint32_t ctas, uint32_t min_share, int snap) {
    Runs r;
    r.total = total;
    r.P = min_share > 1 ? total / min_share : total;
    r.P = r.P < 1 ? 1 : r.P < ctas ? r.P : ctas;
    r.share = total / r.P;
    r.rest = total - r.share * r.P;
    r.snap = snap;
    return r;
}
OCL_HD uint32_t run_cut(const Runs& r, uint32_t c) { return c * r.share + (c < r.rest ? c : r.rest); }
// Largest c whose unmoved cut lies on unit u or before (u < total).
OCL_HD uint32_t run_before(const Runs& r, uint32_t u) {
    const uint32_t wide = r.rest * (r.share + 1);
    return u < wide ? u / (r.share + 1) : r.rest + (u - wide) / r.share;
}
// Where a cut on unit u of an item moves: 0 (its start), item_units (the next one's), or u itself.
OCL_HD uint32_t moved_cut(const Runs& r, uint32_t u, int tiles) {
    const uint32_t low = (uint32_t)(kItemCost + (r.snap < tiles / 2 ? r.snap : tiles / 2)), all = item_units(tiles);
    return u <= low ? 0 : all - u <= (uint32_t)r.snap ? all : u;
}
// First and last run that have a piece of the item that begins on unit `begin`.
OCL_HD void item_runs(const Runs& r, uint32_t begin, int tiles, uint32_t& c0, uint32_t& c1) {
    const int low = kItemCost + (r.snap < tiles / 2 ? r.snap : tiles / 2), high = kItemCost + tiles - r.snap - 1;
    c0 = run_before(r, begin + (uint32_t)low);
    c1 = high <= low ? c0 : run_before(r, begin + (uint32_t)high);
}

// A place in the order of all tiles.
struct Cursor {
    int row, next;   // first row of the item, and of the next one
    int item;        // item of the rows: k/v head and group of query heads
    int tokens, tiles;
    int tile, stop;  // next tile, and where this run's piece of the item ends
    uint32_t begin;  // the item's first unit
};
// `stop` of the item for a run that ends on (moved) unit `end`.
OCL_HD void set_stop(Cursor& c, uint32_t end) {
    const uint32_t behind = end - c.begin;  // > kItemCost
    c.stop = behind >= item_units(c.tiles) ? c.tiles : (int)behind - kItemCost;
}
// On to the next item of the run; without one, tile == stop.  True: on another row.
OCL_HD bool next_item(const KvRows& at, int rows, int cap, int items, int tile_tok, uint32_t end, Cursor& c) {
    c.tile = c.stop = 0;
    c.begin += item_units(c.tiles);
    if (c.begin >= end) return false;
    const bool other = ++c.item == items;
    if (other) {
        c.item = 0;
        c.tokens = 0;
        do {
            c.row = c.next;
        } while (c.row < rows && (c.tokens = item_tokens(at, cap, rows, c.row, c.next)) == 0);
        c.tiles = tiles_of(c.tokens, tile_tok);
    }
    set_stop(c, end);
    return other;
}

}  // namespace ocl
