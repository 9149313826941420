// Walking the token kernel's line of work (paged_params.h): which work a unit belongs to, which units a group of warps
// takes, and which pieces share a work. Host and device: the CPU tests walk it too.
//
// A work takes kWorkCost places of the line in front of its units' places: what it costs to begin and end one (its queries,
// the join of the CTA's warps, its rows out), in units. A cut inside those places is a cut in front of the work.
#pragma once

#include "paged_params.h"

namespace f2k {

F2K_HD int least_of(int a, int b) { return a < b ? a : b; }
F2K_HD unsigned least_of(unsigned a, unsigned b) { return a < b ? a : b; }

constexpr unsigned kWorkCost = 8;
// A CTA gets at least so many places. One sequence of 1000 keys, 8 heads: 10.6, 9.7, 9.8 us with 12, 8, 6; 47 sequences of up to
// 18 keys, one head: 10.4, 7.6, 8.8. (A cost of 4: 11.0 and 10.4; 64 sequences of 200 to 8191 keys 125 us, 121 with 8, 123 with 12.)
constexpr int kLeastPlaces = 8;
// Places are counted in 32 bits, and a group's walk steps over the end of the line by up to the groups of a CTA.
constexpr unsigned kMostPlaces = 0xFFFFFF00u;

F2K_HD SeqView seq_of(const PagedBatch& b, int page_shift, int i) {
    return seq_view(b.cu ? b.cu[i] : i, b.cu ? b.cu[i + 1] : i + 1, b.lens[i], b.n_tokens, b.max_new, (long long)b.table_width << page_shift);
}
F2K_HD unsigned seq_places(const AttendParams& p, const SeqWork& w) {
    return (unsigned)w.row_tiles * ((unsigned)w.n_units + kWorkCost) * (unsigned)p.n_kv_heads;
}

struct Where {                                  // the work that a place belongs to
    int b;
    unsigned seq_begin, work_begin, work_end;   // places; the work's units begin at work_begin + kWorkCost
    SeqView s;
    SeqWork w;
    int kvh, rt, lo, hi;                        // keys [lo, hi) that some row of the tile sees

    F2K_HD unsigned first_unit() const { return work_begin + kWorkCost; }
};

// Moves on to the work of place u (at or behind the present one); seq(b) gives a sequence.
template <int kRows, int kUnit, class Seq>
F2K_HD void find_work(const AttendParams& p, const Seq& seq, unsigned u, Where& x) {
    while (u - x.seq_begin >= seq_places(p, x.w)) {
        x.seq_begin += seq_places(p, x.w);
        x.s = seq(++x.b);
        x.w = seq_work(x.s, p.group, kRows, kUnit, p.window);
    }
    const unsigned places = (unsigned)x.w.n_units + kWorkCost, work = (u - x.seq_begin) / places;
    x.work_begin = x.seq_begin + work * places;
    x.work_end = x.work_begin + places;
    x.kvh = (int)(work / (unsigned)x.w.row_tiles);
    x.rt = (int)(work - (unsigned)x.kvh * (unsigned)x.w.row_tiles);
    const int i0 = x.rt * kRows / p.group, i1 = least_of(x.s.n_new - 1, (x.rt * kRows + kRows - 1) / p.group);
    x.lo = visible_keys(x.s, i0, p.window).lo;
    x.hi = visible_keys(x.s, i1, p.window).hi;
}

// The units of group kw of KW inside the CTA's piece [.., end) of the line, work by work.
template <int kRows, int kUnit, int KW>
struct Units {
    Where x;
    unsigned u, end, stop;                      // stop: of the present work, or of the CTA's piece
    int kw;
    bool more;

    F2K_HD int key0() const { return (x.w.unit0 + (int)(u - x.first_unit())) * kUnit; }
    // The work of place `at`; false where the piece ends before the work's first unit.
    template <class Seq>
    F2K_HD bool begin(const AttendParams& p, const Seq& seq, unsigned at) {
        find_work<kRows, kUnit>(p, seq, at, x);
        stop = least_of(end, x.work_end);
        u = (at > x.first_unit() ? at : x.first_unit()) + (unsigned)kw;
        return stop > x.first_unit();
    }
    // Skips units that no row of the tile sees; false at the end of the work.
    F2K_HD bool settle() {
        while (u < stop) {
            const int k = key0();
            if (k < x.hi && k + kUnit > x.lo) return true;
            u += KW;
        }
        return false;
    }
    // The group's first unit at or behind place `at`, and the one after the present one: for fetching ahead over works.
    template <class Seq>
    F2K_HD void enter(const AttendParams& p, const Seq& seq, unsigned at) {
        for (;;) {
            more = at < end;
            if (!more) return;
            begin(p, seq, at);
            if (settle()) return;
            at = stop;
        }
    }
    template <class Seq>
    F2K_HD void next(const AttendParams& p, const Seq& seq) {
        u += KW;
        if (!settle()) enter(p, seq, stop);
    }
};

// Where a piece leaves its rows of a work it has only a part of: the work that it begins in the middle of (at most one), or
// the one that it begins but does not end (at most one).
F2K_HD int share_of(int cta, bool from_start) { return 2 * cta + (from_start ? 1 : 0); }
// How many pieces, from cta - 1 on, share the work x that piece cta begins in; 0 unless cta's is the first cut through it.
F2K_HD int shares_to_join(const Where& x, unsigned total, int n_pieces, int cta) {
    if (cta == 0 || piece_begin(total, n_pieces, cta) <= x.first_unit() || piece_begin(total, n_pieces, cta - 1) > x.first_unit()) return 0;
    // the last piece that begins in front of the work's end
    const int last = (int)(((unsigned long long)x.work_end * (unsigned)n_pieces + total - 1) / total) - 1;
    return least_of(last, n_pieces - 1) - cta + 2;
}

}  // namespace f2k
