// Attention of a sequence's few new tokens over its pages, split over the keys and joined.
//
// With one new token a key and its value are read once and meet `group` query rows: 2 * group flops a byte (16-bit
// cache), so the kernel is bound by reading the cache, and everything serves that:
//
//  * All units (16 or 32 keys of one sequence and key head) of the batch stand in one line and every CTA takes an equal
//    piece of it (token_work.h), so ragged lengths cost nothing and one long sequence spreads over the GPU. A work
//    that a cut goes through is left as unnormalised rows with their maxima and sums, one set per piece, and a
//    second kernel joins the sets in the order of the keys; a whole work is written by the CTA that has it.
//  * A CTA is four warps, two CTAs per SM: one reads while the other begins or ends a work. RW warps share the rows, and the
//    KW = 4 / RW groups of them take every KW-th unit. A group has a ring of K and V boxes of its own, fetched by TMA (one
//    lane of the group's first warp), and no group waits for another before the end of a work.
//  * Keys are the long side of the products: S^T = K Q^T and O^T += V^T P^T as m16n8k16 products of the warp, K and V the
//    16-row operands straight from ldmatrix, eight query rows a column tile. Eight rows hold the heads of most models'
//    groups; a tcgen05 tile would have 128. With rows as the 16-row operand half of every product, register and
//    exponential was spent on rows that do not exist (96 sequences of about 2700 keys, e4m3, 40 heads over 8: 193 us).
//
// Online softmax per warp, raw scores, exponents of 2, fp32; a row's reference only moves when a score exceeds it by 2^8, so
// most units need no maximum across lanes. P is rounded to 16 bits for the product (the tensor cores take no wider operand
// beside a 16-bit V; a second product for what the rounding leaves would double V's), the sum is taken before. Rows
// are masked by key number; values of keys that no row of the tile sees are cleared in registers, so what lies in the
// rest of a page (NaN included) does not matter.
//
// e4m3 caches: the bytes become fp16 in registers (exactly), the products are fp16 ones. A thread's four bytes of K are
// neighbours in head_dim; a contraction may be taken in any order, so Q is laid out to match. bf16 queries are brought
// into fp16's range by a power of two per row. The heads' scales are applied to S and O.
#include "../ptx.cuh"
#include "../attn_params.h"
#include "kv_launch.h"
#include "mma_sync.cuh"
#include "token_work.h"

#include <type_traits>

namespace f2k {

using namespace f2k::ptx;

namespace {

constexpr int kWarps = 4, kThreads = 32 * kWarps, kCtasPerSm = 2;
constexpr uint32_t kRingBytes = 96 * 1024;     // over the groups of a CTA
constexpr int kMostStages = 24;
constexpr int kSeqsHeld = kThreads;            // sequences kept in shared memory; larger batches are looked up where they lie
constexpr float kLazyThreshold = 8.0f;         // log2 units

// NT tiles of eight rows a warp, RW warps over the rows.
template <bool kE4m3, int D, int NT, int RW>
struct Shape {
    static constexpr int kRows = 8 * NT * RW, KW = kWarps / RW;
    static constexpr int kRowBytes = D * (kE4m3 ? 1 : 2);
    static constexpr int kUnit = token_unit_keys(kRowBytes);
    static constexpr int kPiece = kRowBytes < 128 ? kRowBytes : 128;     // bytes of a shared-memory row
    static constexpr uint32_t kTile = kUnit * kRowBytes, kStage = 2 * kTile;   // K or V of a unit; both
    static constexpr int kStages = kRingBytes / kStage, kRing = kStages / KW;
    static_assert(kStages <= kMostStages && kRing >= 3, "stages");
    static constexpr int kSlice = D / 16 / KW;                            // 16-row tiles of O^T that a warp sums up and writes
    static constexpr int kSliceFloats = kSlice * 16 * 8;
    static constexpr uint32_t kSlots = kWarps * (KW - 1) * kSliceFloats;  // floats: every warp's other slices, one row tile
    static constexpr uint32_t kSmem = kRingBytes + kSlots * 4;
};

struct Ctl {
    uint64_t full[kMostStages], empty[kMostStages];
    uint32_t boxes[kMostStages];               // which boxes of the stage hold keys
    float2 ml[kWarps][32];
    unsigned long long scan[kWarps];
    unsigned seq_begin;
    int seq;
    uint32_t abort;
    int first[kSeqsHeld], n_new[kSeqsHeld], len[kSeqsHeld];
};

template <class T, bool kE4m3, int D, int NT, int RW>
__global__ void __launch_bounds__(kThreads, kCtasPerSm)
paged_token_kernel(const __grid_constant__ AttendParams p) {
    using S = Shape<kE4m3, D, NT, RW>;
    using M = std::conditional_t<kE4m3, __half, T>;          // the type of the products
    constexpr int KW = S::KW, kUnit = S::kUnit, kRing = S::kRing, kSteps = D / 16, kBlocks = kUnit / 16;
    extern __shared__ uint8_t smem_raw[];
    __shared__ Ctl ctl;
    const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
    float* slots = reinterpret_cast<float*>(smem_raw + (smem - smem_u32(smem_raw)) + kRingBytes);
    volatile uint32_t* abort_flag = &ctl.abort;

    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int kw = warp / RW, rw = warp % RW;
    if (threadIdx.x < kMostStages) {
        mbar_init(smem_u32(&ctl.full[threadIdx.x]), 1);
        mbar_init(smem_u32(&ctl.empty[threadIdx.x]), RW);
    }
    if (threadIdx.x == 0) ctl.abort = 0;
    fence_mbar_init();
    fence_proxy_async_smem();
    grid_launch_dependents();
    grid_dependency_wait();

    // ---- where this CTA's piece of the line lies: a sum over the sequences, a run of them per thread
    const bool held = p.batch.n_seqs <= kSeqsHeld;
    auto seq = [&](int b) {
        return held ? SeqView{ctl.first[b], ctl.n_new[b], ctl.len[b], false} : seq_of(p.batch, p.page_shift, b);
    };
    const int per = (p.batch.n_seqs + kThreads - 1) / kThreads;
    const int b_first = min(p.batch.n_seqs, (int)threadIdx.x * per), b_last = min(p.batch.n_seqs, b_first + per);
    unsigned long long mine = 0;                              // 64 bits: rows of malformed batches may overlap and add up to anything
    for (int b = b_first; b < b_last; ++b) {
        const SeqView s = seq_of(p.batch, p.page_shift, b);
        if (s.bad) atomicOr(p.status, (int)kStatusBadLength);
        if (held) ctl.first[b] = s.first, ctl.n_new[b] = s.n_new, ctl.len[b] = s.len;
        mine += seq_places(p, seq_work(s, p.group, S::kRows, kUnit, p.window));
    }
    unsigned long long upto = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const unsigned long long v = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += v;
    }
    if (lane == 31) ctl.scan[warp] = upto;
    __syncthreads();
    unsigned long long all_places = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) upto += ctl.scan[w];
        all_places += ctl.scan[w];
    }
    const unsigned total = all_places > kMostPlaces ? 0u : (unsigned)all_places;
    if (all_places > kMostPlaces && threadIdx.x == 0) atomicOr(p.status, (int)kStatusBadLength);
    const int n_pieces = pieces(total, p.n_ctas, kLeastPlaces);
    const int cta = blockIdx.x;
    if (cta >= n_pieces || total == 0) {
        if (threadIdx.x == 0) p.ws_join[cta].n = 0;
        return;
    }
    const unsigned begin = piece_begin(total, n_pieces, cta), end = piece_begin(total, n_pieces, cta + 1);
    if (begin >= upto - mine && begin < upto) {
        unsigned at = (unsigned)(upto - mine);
        for (int b = b_first;; ++b) {
            const unsigned places = seq_places(p, seq_work(seq(b), p.group, S::kRows, kUnit, p.window));
            if (begin - at < places) {
                ctl.seq = b;
                ctl.seq_begin = at;
                break;
            }
            at += places;
        }
    }
    __syncthreads();

    // ---- the group's ring
    using Walk = Units<S::kRows, kUnit, KW>;
    Where start;
    start.b = ctl.seq;
    start.seq_begin = ctl.seq_begin;
    start.s = seq(start.b);
    start.w = seq_work(start.s, p.group, S::kRows, kUnit, p.window);
    const uint32_t ring = smem + kw * kRing * S::kStage;
    const uint32_t full0 = smem_u32(&ctl.full[kw * kRing]), empty0 = smem_u32(&ctl.empty[kw * kRing]);
    const int box_rows = min(kUnit, 1 << p.page_shift);      // 16, or 32
    const int n_boxes = kUnit / box_rows;
    const uint32_t box_bytes = (uint32_t)box_rows * S::kRowBytes;
    bool ok = true;

    Walk ahead;                                               // what is fetched next (the group's first warp)
    int fetched = 0, page[2] = {0, 0};
    bool need[2] = {false, false};
    auto look_up = [&]() {                                    // pages of the unit fetched next: asked for a unit ahead
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int k = ahead.key0() + i * box_rows;
            need[i] = ahead.more && i < n_boxes && k < ahead.x.hi && k + box_rows > ahead.x.lo;
            if (need[i]) page[i] = p.batch.table[ahead.x.b * p.batch.table_stride + (k >> p.page_shift)];
        }
    };
    auto fetch = [&]() {
        if (!ahead.more || !ok) return;
        const int stage = fetched % kRing, use = fetched / kRing;
        if (RW > 1 && use > 0) {
            ok = mbar_wait(empty0 + stage * 8, (use - 1) & 1, abort_flag, p.wait_limit_clk);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) return;
        }
        if (lane == 0) {
            uint32_t have = 0, bytes = 0;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (!need[i]) continue;
                if ((unsigned)page[i] < (unsigned)p.n_pages) have |= 1u << i, bytes += 2 * box_bytes;
                else atomicOr(p.status, (int)kStatusBadPage);
            }
            ctl.boxes[kw * kRing + stage] = have;
            const uint32_t bar = full0 + stage * 8, dst = ring + stage * S::kStage;
            mbar_arrive_expect_tx(bar, bytes);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (!(have >> i & 1u)) continue;
                const int row = (ahead.key0() + i * box_rows) & ((1 << p.page_shift) - 1);
                tma_load_5d(dst + i * box_bytes, &p.tm_k, bar, 0, row, 0, ahead.x.kvh, page[i]);
                tma_load_5d(dst + S::kTile + i * box_bytes, &p.tm_v, bar, 0, row, 0, ahead.x.kvh, page[i]);
            }
        }
        ++fetched;
        ahead.next(p, seq);
        look_up();
    };
    if (rw == 0) {
        ahead.x = start;
        ahead.end = end;
        ahead.kw = kw;
        ahead.enter(p, seq, begin);
        look_up();
    }

    // ---- work by work
    const int g8 = lane >> 2, t4 = lane & 3;                  // rows g8 of an operand's column tile; 2 t4, 2 t4 + 1 of a result's
    int used = 0;                                             // units of the group consumed
    Walk walk;
    walk.x = start;
    walk.end = end;
    walk.kw = kw;
    for (unsigned at = begin; at < end; at = walk.stop) {
        const bool any = walk.begin(p, seq, at);
        const Where& x = walk.x;
        if (at == begin && threadIdx.x == 0)
            p.ws_join[cta] = JoinJob{shares_to_join(x, total, n_pieces, cta), x.s.first, x.kvh, x.rt * S::kRows, x.s.n_new * p.group - x.rt * S::kRows, {0, 0, 0}};
        if (!any) break;                                      // the piece ends before the work's first unit
        const int tile_rows = min(S::kRows, x.s.n_new * p.group - x.rt * S::kRows);
        const bool active = rw * 8 * NT < tile_rows;

        // ---- Q: row n of column tile nt is the tile's row rw * 8 NT + 8 nt + n
        uint32_t qb[NT][kSteps][2];
        float coef[NT][2];
        KeyRange see[NT][2];
        const float scale = kE4m3 ? score_factor(p.scale_log2, p.k_scale, x.kvh) : p.scale_log2;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int r = x.rt * S::kRows + rw * 8 * NT + nt * 8 + g8;
            const int tok = r / p.group, head = x.kvh * p.group + (r - tok * p.group);
            const bool valid = tok < x.s.n_new;
            const T* row = static_cast<const T*>(p.q) + (x.s.first + tok) * p.q_stride + (long long)head * D;
            coef[nt][0] = coef[nt][1] = scale;
            if constexpr (!kE4m3) {
#pragma unroll
                for (int ks = 0; ks < kSteps; ++ks) {
                    qb[nt][ks][0] = valid ? *reinterpret_cast<const uint32_t*>(row + ks * 16 + 2 * t4) : 0u;
                    qb[nt][ks][1] = valid ? *reinterpret_cast<const uint32_t*>(row + ks * 16 + 8 + 2 * t4) : 0u;
                }
            } else {
                uint2 raw[kSteps];
#pragma unroll
                for (int ks = 0; ks < kSteps; ++ks)
                    raw[ks] = valid ? *reinterpret_cast<const uint2*>(row + ks * 16 + 4 * t4) : make_uint2(0u, 0u);
                if constexpr (std::is_same_v<T, __nv_bfloat16>) {
                    float top = 0.f;
#pragma unroll
                    for (int ks = 0; ks < kSteps; ++ks)
                        top = fmaxf(top, fmaxf(fmaxf(fabsf(Half16<T>::lo(raw[ks].x)), fabsf(Half16<T>::hi(raw[ks].x))),
                                               fmaxf(fabsf(Half16<T>::lo(raw[ks].y)), fabsf(Half16<T>::hi(raw[ks].y)))));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    const unsigned f = fp16_row_power(top, scale);
                    const float up = __uint_as_float(f << 23), down = __uint_as_float((254u - f) << 23);
#pragma unroll
                    for (int h = 0; h < 2; ++h) coef[nt][h] *= __shfl_sync(0xffffffffu, down, (2 * t4 + h) * 4);
#pragma unroll
                    for (int ks = 0; ks < kSteps; ++ks) {
                        qb[nt][ks][0] = Half16<M>::pack(Half16<T>::lo(raw[ks].x) * up, Half16<T>::hi(raw[ks].x) * up);
                        qb[nt][ks][1] = Half16<M>::pack(Half16<T>::lo(raw[ks].y) * up, Half16<T>::hi(raw[ks].y) * up);
                    }
                } else {
#pragma unroll
                    for (int ks = 0; ks < kSteps; ++ks) qb[nt][ks][0] = raw[ks].x, qb[nt][ks][1] = raw[ks].y;
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int i = (x.rt * S::kRows + rw * 8 * NT + nt * 8 + 2 * t4 + h) / p.group;
                see[nt][h] = i < x.s.n_new ? visible_keys(x.s, i, p.window) : KeyRange{0, 0};
            }
        }

        // The first units are fetched behind the first queries' loads, whose latency and that of the pages' numbers then run together.
        if (rw == 0 && at == begin)
            for (int i = 0; i < kRing - 1; ++i) fetch();

        float o[NT][kSteps][4], m[NT][2], l[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m[nt][0] = m[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
            for (int i = 0; i < kSteps; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
        }
        // rows see keys [lo_all, hi_all) without exception
        const int i_first = x.rt * S::kRows / p.group, i_last = min(x.s.n_new - 1, (x.rt * S::kRows + S::kRows - 1) / p.group);
        const int lo_all = visible_keys(x.s, i_last, p.window).lo, hi_all = visible_keys(x.s, i_first, p.window).hi;

        for (bool have = walk.settle(); have && ok; walk.u += KW, have = walk.settle()) {
            if (rw == 0) fetch();
            const int stage = used % kRing;
            ok = ok && mbar_wait(full0 + stage * 8, (used / kRing) & 1, abort_flag, p.wait_limit_clk);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            ++used;
            if (active) {
                const int key0 = walk.key0();
                const uint32_t boxes = ctl.boxes[kw * kRing + stage];
                const uint32_t tile_k = ring + stage * S::kStage, tile_v = tile_k + S::kTile;
                // Shared-memory byte of 16-byte chunk `ch` of key `key` of the unit: boxes one behind the other, in each the
                // 128-byte pieces of its rows one behind the other, 16-byte chunks swizzled as the copy wrote them.
                auto at_smem = [&](uint32_t tile, int key, int ch) {
                    const int box = key >= box_rows ? 1 : 0, r = key - box * box_rows;
                    constexpr int kChunks = S::kPiece / 16;
                    const int piece = ch / kChunks, c = ch % kChunks;
                    const int twist = kChunks == 8 ? (r & 7) : ((r >> 1) & 3);
                    return tile + box * box_bytes + (piece * box_rows + r) * S::kPiece + ((c ^ twist) << 4);
                };
                float s[NT][kBlocks][4];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int kb = 0; kb < kBlocks; ++kb) s[nt][kb][0] = s[nt][kb][1] = s[nt][kb][2] = s[nt][kb][3] = 0.f;
                // ---- S^T = K Q^T
                const int key_k = ((lane >> 3 & 1) << 3) + (lane & 7);
                if constexpr (!kE4m3) {
#pragma unroll
                    for (int ks = 0; ks < kSteps; ++ks)
#pragma unroll
                        for (int kb = 0; kb < kBlocks; ++kb) {
                            uint32_t a[4];
                            ldmatrix_x4(a, at_smem(tile_k, kb * 16 + key_k, ks * 2 + (lane >> 4)));
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) Half16<M>::mma(s[nt][kb], a, qb[nt][ks][0], qb[nt][ks][1]);
                        }
                } else {
#pragma unroll
                    for (int ks = 0; ks < kSteps; ks += 2)
#pragma unroll
                        for (int kb = 0; kb < kBlocks; ++kb) {
                            uint32_t r[4];
                            ldmatrix_x4(r, at_smem(tile_k, kb * 16 + key_k, ks + (lane >> 4)));
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                const uint32_t a[4] = {f16x2_of_e4m3x2(r[2 * i]), f16x2_of_e4m3x2(r[2 * i + 1]), f16x2_of_e4m3x2(r[2 * i] >> 16),
                                                       f16x2_of_e4m3x2(r[2 * i + 1] >> 16)};
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt) Half16<M>::mma(s[nt][kb], a, qb[nt][ks + i][0], qb[nt][ks + i][1]);
                            }
                        }
                }
                // ---- mask, reference maximum
                const bool whole = key0 >= lo_all && key0 + kUnit <= hi_all && boxes == (1u << n_boxes) - 1u;
                if (!whole) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int kb = 0; kb < kBlocks; ++kb)
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const int k = kb * 16 + (j >> 1) * 8 + g8, key = key0 + k;
                                const KeyRange& r = see[nt][j & 1];
                                if (!(key >= r.lo && key < r.hi && (boxes >> (k >= box_rows ? 1 : 0) & 1u))) s[nt][kb][j] = -INFINITY;
                            }
                }
                float top[NT][2];
                bool moves = false;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        top[nt][h] = -INFINITY;
#pragma unroll
                        for (int kb = 0; kb < kBlocks; ++kb) top[nt][h] = fmaxf(top[nt][h], fmaxf(s[nt][kb][h], s[nt][kb][2 + h]));
                        moves |= (top[nt][h] - m[nt][h]) * coef[nt][h] > kLazyThreshold || (m[nt][h] == -INFINITY && top[nt][h] > -INFINITY);
                    }
                if (__any_sync(0xffffffffu, moves)) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            float to = top[nt][h];
                            to = fmaxf(to, __shfl_xor_sync(0xffffffffu, to, 4));
                            to = fmaxf(to, __shfl_xor_sync(0xffffffffu, to, 8));
                            to = fmaxf(m[nt][h], fmaxf(to, __shfl_xor_sync(0xffffffffu, to, 16)));
                            const float f = m[nt][h] == to ? 1.f : ex2_approx((m[nt][h] - to) * coef[nt][h]);
                            m[nt][h] = to;
                            l[nt][h] *= f;
#pragma unroll
                            for (int i = 0; i < kSteps; ++i) o[nt][i][h] *= f, o[nt][i][2 + h] *= f;
                        }
                }
                // ---- P^T and its sum
                uint32_t pb[NT][kBlocks][2];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float neg[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) neg[h] = m[nt][h] == -INFINITY ? 0.f : -m[nt][h] * coef[nt][h];
#pragma unroll
                    for (int kb = 0; kb < kBlocks; ++kb)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const float a = ex2_approx(fmaf(s[nt][kb][2 * i], coef[nt][0], neg[0]));
                            const float b = ex2_approx(fmaf(s[nt][kb][2 * i + 1], coef[nt][1], neg[1]));
                            l[nt][0] += a;
                            l[nt][1] += b;
                            pb[nt][kb][i] = movmatrix_trans(Half16<M>::pack(a, b));
                        }
                }
                // ---- O^T += V^T P^T
#pragma unroll
                for (int kb = 0; kb < kBlocks; ++kb) {
                    // Values of keys that no row of the tile sees are not read as numbers: they may be anything.
                    uint32_t keep[2] = {0xFFFFFFFFu, 0xFFFFFFFFu};
                    if (!whole) {
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            uint32_t mask = 0;
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const int k = kb * 16 + i * 8 + 2 * t4 + e, key = key0 + k;
                                if (key >= x.lo && key < x.hi && (boxes >> (k >= box_rows ? 1 : 0) & 1u)) mask |= 0xFFFFu << (16 * e);
                            }
                            keep[i] = mask;
                        }
                    }
                    if constexpr (!kE4m3) {
                        const int key = kb * 16 + (lane >> 4) * 8 + (lane & 7);
#pragma unroll
                        for (int dt = 0; dt < kSteps; ++dt) {
                            uint32_t a[4];
                            ldmatrix_x4_trans(a, at_smem(tile_v, key, dt * 2 + (lane >> 3 & 1)));
                            if (!whole) a[0] &= keep[0], a[1] &= keep[0], a[2] &= keep[1], a[3] &= keep[1];
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) Half16<M>::mma(o[nt][dt], a, pb[nt][kb][0], pb[nt][kb][1]);
                        }
                    } else {
#pragma unroll
                        for (int dt = 0; dt < kSteps; dt += 2) {
                            uint32_t r[4];
                            ldmatrix_x4_trans(r, at_smem(tile_v, kb * 16 + key_k, dt + (lane >> 4)));
                            if (!whole) r[0] &= keep[0], r[1] &= keep[1], r[2] &= keep[0], r[3] &= keep[1];
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                // a word: two keys of two neighbours of head_dim; even ones are rows 0-7 of the tile, odd ones 8-15
                                const uint32_t a[4] = {f16x2_of_e4m3x2(__byte_perm(r[2 * i], 0, 0x4420)), f16x2_of_e4m3x2(__byte_perm(r[2 * i], 0, 0x4431)),
                                                       f16x2_of_e4m3x2(__byte_perm(r[2 * i + 1], 0, 0x4420)), f16x2_of_e4m3x2(__byte_perm(r[2 * i + 1], 0, 0x4431))};
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt) Half16<M>::mma(o[nt][dt + i], a, pb[nt][kb][0], pb[nt][kb][1]);
                            }
                        }
                    }
                }
            }
            __syncwarp();
            if (RW > 1 && lane == 0) mbar_arrive(empty0 + stage * 8);
        }

        // ---- the groups' shares of the work: maxima and sums, then row tile by row tile every warp sums a slice of head_dim up
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                l[nt][h] += __shfl_xor_sync(0xffffffffu, l[nt][h], 4);
                l[nt][h] += __shfl_xor_sync(0xffffffffu, l[nt][h], 8);
                l[nt][h] += __shfl_xor_sync(0xffffffffu, l[nt][h], 16);
                if (m[nt][h] != -INFINITY) m[nt][h] *= coef[nt][h];            // from here on in log2 units
                if (g8 == 0) ctl.ml[warp][nt * 8 + 2 * t4 + h] = make_float2(m[nt][h], l[nt][h]);
            }
        const bool from_start = at <= x.first_unit(), to_end = walk.stop == x.work_end;
        const int share = share_of(cta, from_start);
        const float v_scale = kE4m3 && p.v_scale ? p.v_scale[x.kvh] : 1.f;
        bool stopped = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            // slice k of this warp's O^T, in the order of its registers: a float2 a lane
            auto slot_at = [&](int from_kw, int to_kw, int i, int half) {
                const int other = to_kw < from_kw ? to_kw : to_kw - 1;
                return reinterpret_cast<float2*>(slots + ((from_kw * RW + rw) * (KW - 1) + other) * S::kSliceFloats + i * 128 + half * 64) + lane;
            };
            if (nt > 0) __syncthreads();
#pragma unroll
            for (int k = 0; k < KW; ++k)
                if (k != kw) {
#pragma unroll
                    for (int i = 0; i < S::kSlice; ++i) {
                        const float(&v)[4] = o[nt][k * S::kSlice + i];
                        *slot_at(kw, k, i, 0) = make_float2(v[0], v[1]);
                        *slot_at(kw, k, i, 1) = make_float2(v[2], v[3]);
                    }
                }
            __syncthreads();
            if (nt == 0) stopped = *abort_flag != 0u;          // the same in every thread: nobody waits between the barriers
            // this thread's two rows over the groups
            float all[2], sum[2], f[KW][2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                all[h] = -INFINITY;
#pragma unroll
                for (int k = 0; k < KW; ++k) all[h] = fmaxf(all[h], ctl.ml[k * RW + rw][nt * 8 + 2 * t4 + h].x);
                const float to = all[h] == -INFINITY ? 0.f : all[h];
                sum[h] = 0.f;
#pragma unroll
                for (int k = 0; k < KW; ++k) {
                    const float2 v = ctl.ml[k * RW + rw][nt * 8 + 2 * t4 + h];
                    f[k][h] = ex2_approx(v.x - to);
                    sum[h] += v.y * f[k][h];
                }
            }
            const int row0 = rw * 8 * NT + nt * 8;
            float out_f[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) out_f[h] = from_start && to_end ? v_scale / sum[h] : 1.f;
            // where this thread's words go: row g8 of the row tile
            const int r = row0 + g8, rr = x.rt * S::kRows + r, tok = rr / p.group, head = x.kvh * p.group + (rr - tok * p.group);
            T* dst = static_cast<T*>(p.o) + (long long)(x.s.first + tok) * p.o_stride + (long long)head * D;
#pragma unroll
            for (int i = 0; i < S::kSlice; ++i) {
                const int dt = kw * S::kSlice + i;
                float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < KW; ++k) {
                    float2 a, b;
                    if (k == kw) {
#pragma unroll
                        for (int j = 0; j < KW; ++j)
                            if (j == kw) {
                                const float(&w)[4] = o[nt][j * S::kSlice + i];
                                a = make_float2(w[0], w[1]), b = make_float2(w[2], w[3]);
                            }
                    } else {
                        a = *slot_at(k, kw, i, 0), b = *slot_at(k, kw, i, 1);
                    }
                    v[0] += a.x * f[k][0], v[1] += a.y * f[k][1], v[2] += b.x * f[k][0], v[3] += b.y * f[k][1];
                }
                if (from_start && to_end) {
                    // a row without keys is zero; rows out as 16-bit pairs along head_dim
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[j] = all[j & 1] == -INFINITY ? 0.f : v[j] * out_f[j & 1];
                    const uint32_t a = movmatrix_trans(Half16<T>::pack(v[0], v[1])), b = movmatrix_trans(Half16<T>::pack(v[2], v[3]));
                    if (r < tile_rows) {
                        if constexpr (kE4m3) {
                            *reinterpret_cast<uint2*>(dst + dt * 16 + 4 * t4) = make_uint2(__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632));
                        } else {
                            *reinterpret_cast<uint32_t*>(dst + dt * 16 + 2 * t4) = a;
                            *reinterpret_cast<uint32_t*>(dst + dt * 16 + 8 + 2 * t4) = b;
                        }
                    }
                } else {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int row = row0 + 2 * t4 + h;
                        if (row >= tile_rows) continue;
                        float* ws = p.ws_o + ((long long)share * S::kRows + row) * D + dt * 16;
                        if constexpr (kE4m3) {
                            *reinterpret_cast<float2*>(ws + 2 * g8) = make_float2(v[h], v[2 + h]);
                        } else {
                            ws[g8] = v[h];
                            ws[8 + g8] = v[2 + h];
                        }
                    }
                }
            }
            if (kw == 0 && g8 == 0) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int row = row0 + 2 * t4 + h;
                    if (row >= tile_rows) continue;
                    if (!(from_start && to_end)) {
                        p.ws_ml[share * S::kRows + row] = make_float2(all[h], sum[h]);
                    } else if (p.lse != nullptr) {
                        const int at_row = x.rt * S::kRows + row, i = at_row / p.group;
                        p.lse[(long long)(x.s.first + i) * p.n_heads + x.kvh * p.group + (at_row - i * p.group)] =
                            all[h] == -INFINITY ? -INFINITY : (all[h] + log2f(sum[h])) * 0.69314718055994531f;
                    }
                }
            }
        }
        __syncthreads();
        if (stopped) break;
    }

    if (*abort_flag != 0u) {
        // Leaving early: the copies that are on their way land first (bounded).
        if (rw == 0) {
            volatile uint32_t never = 0;
            for (int i = max(0, fetched - kRing); i < fetched; ++i)
                mbar_wait(full0 + (i % kRing) * 8, (i / kRing) & 1, &never, 40000000ll);
        }
        __syncthreads();
        if (threadIdx.x == 0) atomicOr(p.status, (int)kStatusWaitExpired);
    }
}

// One cut's work: the shares of the pieces c-1, c, ... in the order of their keys. A warp has a row. No shared memory, so that
// its blocks fit beside the token kernel's and stand ready when that ends; the shares' rows are asked for together with
// their maxima.
template <class T, bool kE4m3, int D>
__global__ void __launch_bounds__(128)
paged_join_kernel(const __grid_constant__ AttendParams p, int rows) {
    grid_launch_dependents();
    const int cta = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int row = blockIdx.y * 4 + warp;
    grid_dependency_wait();
    const JoinJob job = p.ws_join[cta];
    if (job.n == 0 || row >= min(rows, job.rows)) return;
    auto share = [&](int j) { return (long long)share_of(cta - 1 + j, j == 0) * rows + row; };
    constexpr int kCols = D / 32, kAhead = 8;
    float all = -INFINITY, sum = 0.f, acc[kCols] = {};
    for (int j0 = 0; j0 < job.n; j0 += 32) {                  // 32 shares at a time, a lane for each one's maximum and sum
        const int n = min(32, job.n - j0);
        float2 ml = lane < n ? p.ws_ml[share(j0 + lane)] : make_float2(-INFINITY, 0.f);
        float top = ml.x;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        const float to = fmaxf(all, top), ref = to == -INFINITY ? 0.f : to;
        const float old = ex2_approx(all - ref), f = ex2_approx(ml.x - ref);
        all = to;
        float part = ml.y * f;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) part += __shfl_xor_sync(0xffffffffu, part, d);
        sum = sum * old + part;
#pragma unroll
        for (int i = 0; i < kCols; ++i) acc[i] *= old;
        for (int j = 0; j < n; j += kAhead) {
            float2 v[kAhead][kCols / 2];
#pragma unroll
            for (int u = 0; u < kAhead; ++u)
                if (j + u < n) {
                    const float* src = p.ws_o + share(j0 + j + u) * D + lane * kCols;
#pragma unroll
                    for (int i = 0; i < kCols / 2; ++i) v[u][i] = reinterpret_cast<const float2*>(src)[i];
                }
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const float w = __shfl_sync(0xffffffffu, f, (j + u) & 31);
                if (j + u < n) {
#pragma unroll
                    for (int i = 0; i < kCols / 2; ++i) acc[2 * i] += w * v[u][i].x, acc[2 * i + 1] += w * v[u][i].y;
                }
            }
        }
    }
    const int rr = job.row0 + row, tok = rr / p.group, head = job.kvh * p.group + (rr - tok * p.group);
    const long long t = job.first + tok;
    const float f = (kE4m3 && p.v_scale ? p.v_scale[job.kvh] : 1.f) / sum;
    uint32_t* dst = reinterpret_cast<uint32_t*>(static_cast<T*>(p.o) + t * p.o_stride + (long long)head * D + lane * kCols);
#pragma unroll
    for (int i = 0; i < kCols; i += 2) dst[i / 2] = all == -INFINITY ? 0u : Half16<T>::pack(acc[i] * f, acc[i + 1] * f);
    if (p.lse != nullptr && lane == 0)
        p.lse[t * p.n_heads + head] = all == -INFINITY ? -INFINITY : (all + log2f(sum)) * 0.69314718055994531f;
}

// The variant for a tile of `rows` rows: f(NT, RW). 64-wide heads have registers for four row tiles a warp, and then read K and
// V from shared memory once for 32 rows.
template <int D, class F>
cudaError_t with_rows(int rows, F&& f) {
    using std::integral_constant;
    constexpr int kWide = D == 64 ? 4 : 2;
    if (rows == 8) return f(integral_constant<int, 1>{}, integral_constant<int, 1>{});
    if (rows == 16) return f(integral_constant<int, 2>{}, integral_constant<int, 1>{});
    if (rows == 32) return f(integral_constant<int, kWide>{}, integral_constant<int, 4 / kWide>{});
    return f(integral_constant<int, kWide>{}, integral_constant<int, 8 / kWide>{});
}

template <class T, bool kE4m3, int D>
cudaError_t prepare() {
    cudaFuncAttributes attr;
    cudaError_t e = cudaFuncGetAttributes(&attr, paged_join_kernel<T, kE4m3, D>);
    for (int rows : {8, 16, 32, 64})
        if (e == cudaSuccess)
            e = with_rows<D>(rows, [](auto nt, auto rw) {
                constexpr int NT = decltype(nt)::value, RW = decltype(rw)::value;
                return cudaFuncSetAttribute(paged_token_kernel<T, kE4m3, D, NT, RW>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                            (int)Shape<kE4m3, D, NT, RW>::kSmem + 1024);
            });
    return e;
}

template <class T, bool kE4m3, int D>
cudaError_t launch(const AttendParams& p, int rows, int used_rows, cudaStream_t stream) {
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.n_ctas);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = stream;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    const cudaError_t e = with_rows<D>(rows, [&](auto nt, auto rw) {
        constexpr int NT = decltype(nt)::value, RW = decltype(rw)::value;
        cfg.dynamicSmemBytes = Shape<kE4m3, D, NT, RW>::kSmem + 1024;
        return cudaLaunchKernelEx(&cfg, paged_token_kernel<T, kE4m3, D, NT, RW>, p);
    });
    if (e != cudaSuccess || p.n_ctas == 1) return e;
    cfg.gridDim = dim3(p.n_ctas, (used_rows + 3) / 4);
    cfg.blockDim = dim3(128);
    cfg.dynamicSmemBytes = 0;
    return cudaLaunchKernelEx(&cfg, paged_join_kernel<T, kE4m3, D>, p, rows);
}

// f(type, e4m3, dim) for the run-time choice.
template <class F>
cudaError_t with_types(PagedType type, PagedType cache, int head_dim, F&& f) {
    auto by_dim = [&](auto t, auto e) {
        return head_dim == 64 ? f(t, e, std::integral_constant<int, 64>{}) : f(t, e, std::integral_constant<int, 128>{});
    };
    auto by_cache = [&](auto t) { return cache == kE4m3 ? by_dim(t, std::true_type{}) : by_dim(t, std::false_type{}); };
    return type == kBf16 ? by_cache(__nv_bfloat16{}) : by_cache(__half{});
}

}  // namespace

int token_rows(long long rows) { return rows <= 8 ? 8 : rows <= 16 ? 16 : rows <= 32 ? 32 : 64; }
int token_ctas(int sms) { return kCtasPerSm * sms; }

cudaError_t paged_token_prepare(PagedType type, PagedType cache, int head_dim) {
    return with_types(type, cache, head_dim, [](auto t, auto e, auto d) { return prepare<decltype(t), decltype(e)::value, decltype(d)::value>(); });
}

cudaError_t paged_token_launch(const AttendParams& p, PagedType type, PagedType cache, int head_dim, int rows, int used_rows,
                               cudaStream_t stream) {
    return with_types(type, cache, head_dim, [&](auto t, auto e, auto d) { return launch<decltype(t), decltype(e)::value, decltype(d)::value>(p, rows, used_rows, stream); });
}

}  // namespace f2k
