// Walking the token kernel's line of work (paged_params.h): which work a unit belongs to, which units a group of warps
// takes, and which pieces share a work. Host and device: the CPU tests walk it too.
#pragma once

#include "paged_params.h"

namespace f2k {

F2K_HD int least_of(int a, int b) { return a < b ? a : b; }
F2K_HD unsigned least_of(unsigned a, unsigned b) { return a < b ? a : b; }

struct Where {                                  // the work that a unit belongs to
    int b;
    unsigned seq_begin, work_begin;
    SeqView s;
    SeqWork w;
    int kvh, rt, lo, hi;                        // keys that some row of the tile sees
};

F2K_HD void load_seq(const AttendParams& p, int rows, int unit, Where& x) {
    const PagedBatch& b = p.batch;
    const int cu0 = b.cu ? b.cu[x.b] : x.b, cu1 = b.cu ? b.cu[x.b + 1] : x.b + 1;
    x.s = seq_view(cu0, cu1, b.lens[x.b], b.n_tokens, (long long)b.table_width << p.page_shift);
    x.w = seq_work(x.s, p.group, rows, unit, p.window);
}
F2K_HD unsigned seq_units(const AttendParams& p, const SeqWork& w) {
    return (unsigned)w.row_tiles * (unsigned)w.n_units * (unsigned)p.n_kv_heads;
}
// Moves on to the work of unit u (at or behind the present one).
F2K_HD void find_work(const AttendParams& p, int rows, int unit, unsigned u, Where& x) {
    while (u - x.seq_begin >= seq_units(p, x.w)) {
        x.seq_begin += seq_units(p, x.w);
        ++x.b;
        load_seq(p, rows, unit, x);
    }
    const unsigned work = (u - x.seq_begin) / (unsigned)x.w.n_units;
    x.work_begin = x.seq_begin + work * (unsigned)x.w.n_units;
    x.kvh = (int)(work / (unsigned)x.w.row_tiles);
    x.rt = (int)(work - (unsigned)x.kvh * (unsigned)x.w.row_tiles);
    const int i0 = x.rt * rows / p.group, i1 = least_of(x.s.n_new - 1, (x.rt * rows + rows - 1) / p.group);
    x.lo = visible_keys(x.s, i0, p.window).lo;
    x.hi = visible_keys(x.s, i1, p.window).hi;
}

// The units of one group inside the CTA's piece of the line, work by work.
template <int kRows, int kUnit, int KW>
struct Units {
    Where x;
    unsigned u, end, work_end;                  // work_end: of the present work, or of the CTA's piece
    int kw;
    bool more;

    F2K_HD int key0() const { return (x.w.unit0 + (int)(u - x.work_begin)) * kUnit; }
    // The first needed unit of the work(s) from unit number `at` on.
    F2K_HD void enter(const AttendParams& p, unsigned at) {
        for (;;) {
            more = at < end;
            if (!more) return;
            find_work(p, kRows, kUnit, at, x);
            work_end = least_of(end, x.work_begin + (unsigned)x.w.n_units);
            u = at + (unsigned)kw;
            if (settle()) return;
            at = work_end;
        }
    }
    // Skips units that no row of the tile sees; false at the end of the work.
    F2K_HD bool settle() {
        while (u < work_end) {
            const int k = key0();
            if (k < x.hi && k + kUnit > x.lo) return true;
            u += KW;
        }
        return false;
    }
    F2K_HD void next(const AttendParams& p) {
        u += KW;
        if (!settle()) enter(p, work_end);
    }
};

// Where a piece leaves its rows of a work it has only a part of: the work that it begins in the middle of (at most one), or
// the one that it begins but does not end (at most one).
F2K_HD int share_of(int cta, bool from_start) { return 2 * cta + (from_start ? 1 : 0); }
// How many pieces, from cta - 1 on, share the work x that piece cta begins in; 0 unless cta's is the first cut through it.
F2K_HD int shares_to_join(const Where& x, unsigned total, int n_pieces, int cta) {
    if (cta == 0 || piece_begin(total, n_pieces, cta) <= x.work_begin || piece_begin(total, n_pieces, cta - 1) > x.work_begin) return 0;
    const unsigned long long work_end = x.work_begin + (unsigned)x.w.n_units;
    // the last piece that begins in front of the work's end
    const int last = (int)((work_end * (unsigned)n_pieces + total - 1) / total) - 1;
    return least_of(last, n_pieces - 1) - cta + 2;
}

}  // namespace f2k
