// Host build of the index arithmetic in ocelotl_b200/csrc/paging.cuh (test_paging_cpu.py).
#include "../ocelotl_b200/csrc/paging.cuh"

using namespace ocl;

// Walk every run of `ctas` CTAs as the attention kernel does.  For each visited
// tile writes (row, item, tile, cta) to out; returns the number of tiles, or a
// negative code where two runs disagree about an item that they share.
extern "C" long long walk(const int32_t* positions, const int32_t* seqs, long long n_seqs, int rows, int cap, int items,
                          long long ctas, int32_t* out, long long room) {
    const KvRows at{positions, seqs, nullptr, n_seqs, 0, 0};
    long long total = 0;
    for (int r = 0; r < rows; ++r) total += tiles_of(row_tokens(at, cap, r));
    total *= items;
    const long long P = total < ctas ? total : ctas;
    long long seen = 0;
    for (long long c = 0; c < P; ++c) {
        const long long begin = run_begin(total, P, c), end = run_begin(total, P, c + 1);
        if (begin >= end) return -1;
        long long at_row = 0;
        int r = 0;
        for (;; ++r) {
            const long long n = (long long)tiles_of(row_tokens(at, cap, r)) * items;
            if (begin < at_row + n) break;
            at_row += n;
        }
        Cursor cc{r, 0, 0, row_tokens(at, cap, r), 0};
        cc.tiles = tiles_of(cc.tokens);
        cc.item = (int)((begin - at_row) / cc.tiles);
        cc.tile = (int)((begin - at_row) % cc.tiles);
        const long long count = end - begin;
        int starts = 0, goes_on = 0;  // shared items that this run starts, and that it continues
        for (long long done = 0; done < count;) {
            const long long left = count - done, n = cc.tiles - cc.tile < left ? cc.tiles - cc.tile : left;
            const long long b = begin + done - cc.tile, e = b + cc.tiles;
            const long long c0 = run_of(total, P, b), c1 = run_of(total, P, e - 1);
            if (c < c0 || c > c1) return -2;
            if (run_begin(total, P, c0) > b || (c0 + 1 <= P && run_begin(total, P, c0 + 1) <= b)) return -3;
            if (c0 != c1) {
                if (c == c0) ++starts;
                else ++goes_on;
            }
            if ((c0 == c1) != (n == cc.tiles)) return -4;
            for (long long t = 0; t < n; ++t, ++seen) {
                if (seen >= room) return -5;
                int32_t* o = out + 4 * seen;
                o[0] = cc.row, o[1] = cc.item, o[2] = cc.tile + (int)t, o[3] = (int32_t)c;
            }
            done += n;
            if (done < count) next_item(at, rows, cap, items, cc);
        }
        if (starts > 1 || goes_on > 1) return -6;  // one workspace slot each
    }
    return seen == total ? seen : -7;
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
