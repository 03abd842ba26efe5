// Host build of the index arithmetic in ocelotl_b200/csrc/paging.cuh (test_paging_cpu.py).
#include "../ocelotl_b200/csrc/paging.cuh"

using namespace ocl;
constexpr int kTile = 64;

static uint32_t units_of(const KvRows& at, int cap, int items, int rows, int r, int& next) {
    const int tokens = item_tokens(at, cap, rows, r, next);
    return tokens ? item_units(tiles_of(tokens, kTile)) * (uint32_t)items : 0;
}

// Walk every run of the CTAs as the attention kernel does.  For each visited tile
// writes (row, item, tile, cta) to out; returns the number of tiles, or a negative
// code where two runs disagree about an item that they share.
extern "C" long long walk(const int32_t* positions, const int32_t* seqs, long long n_seqs, int rows, int cap, int items,
                          unsigned ctas, unsigned min_share, int snap, int together, int32_t* out, long long room) {
    const KvRows at{positions, seqs, nullptr, n_seqs, 0, 0, together};
    uint32_t total = 0;
    long long tiles = 0;
    for (int r = 0, next; r < rows; r = next) {
        total += units_of(at, cap, items, rows, r, next);
        tiles += (long long)tiles_of(item_tokens(at, cap, rows, r, next), kTile) * items;
    }
    if (!total) return 0;
    const Runs runs = runs_of(total, ctas, min_share, snap);
    if (run_cut(runs, 0) != 0 || run_cut(runs, runs.P) != total) return -9;
    long long seen = 0;
    uint32_t last_end = 0;
    for (uint32_t c = 0; c < runs.P; ++c) {
        uint32_t edge[2];
        Cursor cc{};
        for (int i = 0; i < 2; ++i) {
            const uint32_t cut = run_cut(runs, c + i);
            edge[i] = total;
            uint32_t before = 0;
            for (int r = 0, next; r < rows; r = next) {
                const uint32_t n = units_of(at, cap, items, rows, r, next);
                if (cut < before + n) {
                    Cursor e{};
                    e.row = r;
                    e.tokens = item_tokens(at, cap, rows, r, e.next);
                    e.tiles = tiles_of(e.tokens, kTile);
                    const uint32_t all = item_units(e.tiles), off = cut - before, u = off % all;
                    e.item = (int)(off / all);
                    e.begin = cut - u;
                    const uint32_t moved = moved_cut(runs, u, e.tiles);
                    edge[i] = e.begin + moved;
                    e.tile = moved == 0 ? 0 : (int)moved - kItemCost;  // == tiles: at its end
                    if (i == 0) cc = e;
                    break;
                }
                before += n;
            }
        }
        if (edge[0] != last_end) return -1;
        last_end = edge[1];
        if (edge[0] >= edge[1]) continue;
        if (cc.tile == cc.tiles) next_item(at, rows, cap, items, kTile, edge[1], cc);
        else set_stop(cc, edge[1]);
        int starts = 0, goes_on = 0;  // shared items that this run starts, and that it continues
        while (cc.tile < cc.stop) {
            uint32_t c0, c1;
            item_runs(runs, cc.begin, cc.tiles, c0, c1);
            if (c < c0 || c > c1) return -2;
            if ((c == c0) != (cc.tile == 0)) return -3;          // the first piece starts the item
            if ((c == c1) != (cc.stop == cc.tiles)) return -8;   // the last one ends it
            if (c0 != c1) {
                if (c == c0) ++starts;
                else ++goes_on;
            }
            if ((c0 == c1) != (cc.tile == 0 && cc.stop == cc.tiles)) return -4;
            for (int t = cc.tile; t < cc.stop; ++t, ++seen) {
                if (seen >= room) return -5;
                int32_t* o = out + 4 * seen;
                o[0] = cc.row, o[1] = cc.item, o[2] = t, o[3] = (int32_t)c;
            }
            next_item(at, rows, cap, items, kTile, edge[1], cc);
        }
        if (starts > 1 || goes_on > 1) return -6;  // one workspace slot each
    }
    return seen == tiles && last_end == total ? seen : -7;
}

extern "C" int place(const int32_t* table, long long max_pages, long long stride, long long n_pages, unsigned page_size,
                     long long seq, int tok, int* page, int* in_page) {
    return place_of(table + seq * stride, max_pages, n_pages, divisor_of(page_size), tok, *page, *in_page) ? 1 : 0;
}

// First n of [from, to) in steps whose quotient by d is wrong, or -1.
extern "C" long long wrong_quotient(unsigned d, long long from, long long to, long long step) {
    const Divisor by = divisor_of(d);
    for (long long n = from; n < to; n += step)
        if (quotient((uint32_t)n, by) != (uint32_t)n / d) return n;
    return -1;
}
