// Launch parameters of the paged key/value cache's kernels, and the arithmetic that host and kernels share: where a
// new token lies, which keys a row of queries sees, and how the token kernel's work is cut.
//
// A batch is n_seqs sequences. Sequence b has the new tokens cu[b] .. cu[b+1]-1 of the call's tensors and kv_lens[b]
// keys with them; key j of it is row j % page of page table[b][j / page]. All of that lives in device memory and is
// read by the kernels alone, so that a captured call can be replayed with other lengths.
#pragma once

#include <cstddef>
#include <cstdint>
#include <cuda.h>
#include <vector_types.h>

#ifdef __CUDACC__
#define F2K_HD __host__ __device__ __forceinline__
#else
#define F2K_HD inline
#endif

namespace f2k {

// Bits of a cache handle's status word, beside kStatusWaitExpired.
enum PagedStatus : int {
    kStatusBadPage   = 16,   // a page number outside the cache: its tokens are not written, its keys not attended
    kStatusBadLength = 32,   // a length that the page table cannot hold or below the number of new tokens; rows outside the call's, or more than max_new
    kStatusBadPosition = 64, // a position behind the rotation tables: the token is not written
};

struct PagedBatch {
    const int32_t* cu;               // [n_seqs + 1], nullptr: one new token each
    const int32_t* lens;             // [n_seqs]
    const int32_t* table;            // [n_seqs][table_stride]
    long long table_stride;
    int table_width;                 // pages a row holds
    int n_seqs, n_tokens, max_new;
};

// New tokens of sequence b, first token, and keys, kept inside what the call can hold whatever the device memory says. A sequence
// whose rows do not fit has none: the grids are sized by max_new and n_tokens, so a few rows of it would take the places of the
// sequences behind it, and a part of its rows would stand at positions that are not theirs.
struct SeqView {
    int first, n_new, len;
    bool bad;
};
F2K_HD SeqView seq_view(int cu0, int cu1, int len, int n_tokens, int max_new, long long capacity) {
    SeqView s;
    s.first = cu0 < 0 ? 0 : (cu0 > n_tokens ? n_tokens : cu0);
    const bool fits = cu0 >= 0 && cu1 >= cu0 && cu1 <= n_tokens && cu1 - cu0 <= max_new;
    s.n_new = fits ? cu1 - cu0 : 0;
    s.len = len < 0 ? 0 : (len > capacity ? (int)capacity : len);
    s.bad = !fits || len < s.n_new || len > capacity;
    return s;
}

// Keys [lo, hi) that the new token number i of a sequence sees; empty (hi <= lo) where its position is negative.
struct KeyRange {
    int lo, hi;
};
F2K_HD KeyRange visible_keys(const SeqView& s, int i, int window) {
    KeyRange r;
    r.hi = s.len - s.n_new + i + 1;                     // position + 1
    r.lo = window > 0 && r.hi > window ? r.hi - window : 0;
    return r;
}

// ---- the token kernel's work ---------------------------------------------------------------------------------
// A work is one sequence, key head and tile of `rows` query rows; row r of a tile is new token r / group, query head
// r % group of the key head. A unit is `unit` consecutive keys of one work. All units of the batch stand in one line,
// sequence by sequence, and the grid's CTAs take equal pieces of it, whatever the lengths.
struct SeqWork {
    int row_tiles;        // 0 where the sequence has no new token
    int unit0, n_units;   // units of every row tile: from that of the first key that the first token sees; at least 1
};
F2K_HD SeqWork seq_work(const SeqView& s, int group, int rows, int unit, int window) {
    SeqWork w;
    w.row_tiles = (int)(((long long)s.n_new * group + rows - 1) / rows);
    const KeyRange k = visible_keys(s, 0, window);
    w.unit0 = k.lo / unit;
    const int n = (s.len + unit - 1) / unit - w.unit0;
    w.n_units = n > 1 ? n : 1;
    return w;
}
// First place of the line that CTA c of n takes.
F2K_HD unsigned piece_begin(unsigned total, int n, int c) {
    return (unsigned)((unsigned long long)total * (unsigned)c / (unsigned)n);
}
// CTAs that get places: no more than give each `least`, so that a short batch is not cut finer than it pays.
F2K_HD int pieces(unsigned total, int n_ctas, int least) {
    const unsigned want = total / (unsigned)least;
    return want < 1 ? 1 : (want > (unsigned)n_ctas ? n_ctas : (int)want);
}

struct AppendParams {
    PagedBatch batch;
    const void *q, *k, *v, *gamma_q, *gamma_k;
    const float *cos_tab, *sin_tab, *k_scale, *v_scale;
    void *q_out, *k_pages, *v_pages;
    long long q_stride, k_stride, v_stride, qo_stride;          // token strides, elements
    long long kp_page, kp_head, kp_tok, vp_page, vp_head, vp_tok;
    int n_heads, n_kv_heads, page_shift, n_pages, n_positions, rot_dim, interleaved;
    float eps;
    int* status;
};

// What the join does for the cut in front of a CTA's piece: the shares of n pieces (0: nothing), for `rows` query rows of one
// key head from row0 on of the sequence whose first new token is `first`.
struct alignas(16) JoinJob {
    int n, first, kvh, row0, rows, unused[3];
};

struct AttendParams {
    CUtensorMap tm_k, tm_v;       // [pages][kv heads][128-byte pieces of a row][page][piece]
    PagedBatch batch;
    const void* q;
    void* o;
    float* lse;                   // [n_tokens][n_heads] or nullptr
    const float *k_scale, *v_scale;
    long long q_stride, o_stride;
    int n_heads, n_kv_heads, group, page_shift, n_pages, window;
    float scale_log2;             // scale * log2(e)
    long long wait_limit_clk;
    int* status;
    // token kernel: descriptors of joins, then maxima and sums, then unnormalised rows of the pieces
    JoinJob* ws_join;
    float2* ws_ml;
    float* ws_o;
    int n_ctas;
};

// Element types, as in the C ABI.
enum PagedType { kBf16 = 0, kF16 = 1, kE4m3 = 2 };

// The token kernel's tiling for a cache type and head_dim: keys of a unit.
constexpr int token_unit_keys(int row_bytes) { return row_bytes >= 256 ? 16 : 32; }
constexpr int kPromptTile = 128;  // keys per tile of the prompt kernel

}  // namespace f2k
