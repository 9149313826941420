// Attention of a sequence's few new tokens over its pages, split over the keys and joined.
//
// With one new token a key and its value are read once and meet `group` query rows: 2 * group flops a byte (16-bit
// cache), so the kernel is bound by reading the cache, and everything serves that:
//
//  * All units (16 or 32 keys of one sequence and key head) of the batch stand in one line and every CTA takes an equal
//    piece of it (token_work.h), so ragged lengths cost nothing and one long sequence spreads over the GPU. A work
//    that a cut goes through is left as unnormalised rows with their maxima and sums, one set per piece, and a
//    second kernel joins the sets in the order of the keys; a whole work is written by the CTA that has it.
//  * A CTA is eight warps, one per SM. RW warps share the rows (16 each), and the KW = 8 / RW groups of them take every
//    KW-th unit. A group has a ring of K and V boxes of its own, fetched by TMA (one lane of the group's first warp),
//    192 KB per SM in flight or in use, and no group waits for another before the end of a work.
//  * S = Q K^T and O += P V are m16n8k16 products of the warp with the softmax on their registers: 16 rows are enough
//    for `group` heads, where a tcgen05 tile would have 128, and the row of a 16-key unit is read by ldmatrix once.
//
// Online softmax per warp: maximum, sum and O in fp32, exponents of 2; P is rounded to 16 bits for P V, the sum is
// taken before. Rows are masked by key number; values of keys that no row of the tile sees are cleared in registers, so
// what lies in the rest of a page (NaN included) does not matter.
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

constexpr int kWarps = 8, kThreads = 32 * kWarps;
constexpr int kStagesAll = 24;                 // over the groups of a CTA

template <bool kE4m3, int D, int RW>
struct Shape {
    static constexpr int kRows = 16 * RW, KW = kWarps / RW;
    static constexpr int kRowBytes = D * (kE4m3 ? 1 : 2);
    static constexpr int kUnit = token_unit_keys(kRowBytes);
    static constexpr int kPiece = kRowBytes < 128 ? kRowBytes : 128;     // bytes of a shared-memory row
    static constexpr uint32_t kTile = kUnit * kRowBytes, kStage = 2 * kTile;   // K or V of a unit; both
    static constexpr int kRing = kStagesAll / KW;
    static constexpr int kSlots = kWarps / 2;
    static constexpr uint32_t kSlotFloats = 16 * D;
    static constexpr uint32_t kSmem = kStagesAll * kStage + kSlots * kSlotFloats * 4;
};

struct Ctl {
    uint64_t full[kStagesAll], empty[kStagesAll];
    uint32_t boxes[kStagesAll];                // which boxes of the stage hold keys
    float2 ml[kWarps][16];
    unsigned scan[kWarps];
    unsigned total, seq_begin;
    int seq;
    uint32_t abort;
};

template <class T, bool kE4m3, int D, int RW>
__global__ void __launch_bounds__(kThreads, 1)
paged_token_kernel(const __grid_constant__ AttendParams p) {
    using S = Shape<kE4m3, D, RW>;
    using M = std::conditional_t<kE4m3, __half, T>;          // the type of the products
    constexpr int KW = S::KW, kUnit = S::kUnit, kRing = S::kRing, kSteps = D / 16;
    extern __shared__ uint8_t smem_raw[];
    __shared__ Ctl ctl;
    const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
    float* slots = reinterpret_cast<float*>(smem_raw + (smem - smem_u32(smem_raw)) + kStagesAll * S::kStage);
    volatile uint32_t* abort_flag = &ctl.abort;

    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int kw = warp / RW, rw = warp % RW;
    if (threadIdx.x < kStagesAll) {
        mbar_init(smem_u32(&ctl.full[threadIdx.x]), 1);
        mbar_init(smem_u32(&ctl.empty[threadIdx.x]), RW);
    }
    if (threadIdx.x == 0) ctl.abort = 0;
    fence_mbar_init();
    fence_proxy_async_smem();
    grid_launch_dependents();
    grid_dependency_wait();

    // ---- where this CTA's piece of the line lies: a sum over the sequences, a run of them per thread
    const int per = (p.batch.n_seqs + kThreads - 1) / kThreads;
    const int b_first = min(p.batch.n_seqs, (int)threadIdx.x * per), b_last = min(p.batch.n_seqs, b_first + per);
    unsigned mine = 0;
    for (int b = b_first; b < b_last; ++b) {
        Where x;
        x.b = b;
        load_seq(p, S::kRows, kUnit, x);
        if (x.s.bad) atomicOr(p.status, (int)kStatusBadLength);
        mine += seq_units(p, x.w);
    }
    unsigned upto = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const unsigned v = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += v;
    }
    if (lane == 31) ctl.scan[warp] = upto;
    __syncthreads();
    unsigned total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) upto += ctl.scan[w];
        total += ctl.scan[w];
    }
    const int n_pieces = pieces(total, p.n_ctas, KW);
    const int cta = blockIdx.x;
    if (cta >= n_pieces || total == 0) {
        if (threadIdx.x == 0) p.ws_join[cta] = make_int4(0, 0, 0, 0);
        return;
    }
    const unsigned begin = piece_begin(total, n_pieces, cta), end = piece_begin(total, n_pieces, cta + 1);
    if (begin >= upto - mine && begin < upto) {
        unsigned at = upto - mine;
        for (int b = b_first;; ++b) {
            Where x;
            x.b = b;
            load_seq(p, S::kRows, kUnit, x);
            if (begin - at < seq_units(p, x.w)) {
                ctl.seq = b;
                ctl.seq_begin = at;
                break;
            }
            at += seq_units(p, x.w);
        }
    }
    __syncthreads();

    // ---- the group's ring
    using Walk = Units<S::kRows, kUnit, KW>;
    Where start;
    start.b = ctl.seq;
    start.seq_begin = ctl.seq_begin;
    load_seq(p, S::kRows, kUnit, start);
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
        ahead.next(p);
        look_up();
    };
    if (rw == 0) {
        ahead.x = start;
        ahead.end = end;
        ahead.kw = kw;
        ahead.enter(p, begin);
        look_up();
        for (int i = 0; i < kRing - 1; ++i) fetch();
    }

    // ---- work by work
    const int g8 = lane >> 2, t4 = lane & 3;                  // fragment row and column group
    int used = 0;                                             // units of the group consumed
    Walk walk;
    walk.x = start;
    walk.end = end;
    walk.kw = kw;
    for (unsigned at = begin; at < end;) {
        find_work(p, S::kRows, kUnit, at, walk.x);
        const Where x = walk.x;
        const unsigned work_end = x.work_begin + (unsigned)x.w.n_units;
        walk.work_end = min(end, work_end);
        walk.u = at + (unsigned)kw;
        const int tile_rows = min(S::kRows, x.s.n_new * p.group - x.rt * S::kRows);
        const bool active = rw * 16 < tile_rows;
        if (at == begin && threadIdx.x == 0) p.ws_join[cta] = make_int4(x.b, x.kvh, x.rt, shares_to_join(x, total, n_pieces, cta));

        // rows of this thread: rw * 16 + g8 and + 8
        KeyRange see[2];
        float coef[2];
        uint32_t qa[kSteps][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = x.rt * S::kRows + rw * 16 + g8 + 8 * h;
            const int tok = r / p.group, head = x.kvh * p.group + (r - tok * p.group);
            const bool valid = tok < x.s.n_new;
            see[h] = valid ? visible_keys(x.s, tok, p.window) : KeyRange{0, 0};
            const T* row = static_cast<const T*>(p.q) + (x.s.first + tok) * p.q_stride + (long long)head * D;
            coef[h] = p.scale_log2;
            if constexpr (!kE4m3) {
#pragma unroll
                for (int ks = 0; ks < kSteps; ++ks) {
                    qa[ks][h] = valid ? *reinterpret_cast<const uint32_t*>(row + ks * 16 + 2 * t4) : 0u;
                    qa[ks][2 + h] = valid ? *reinterpret_cast<const uint32_t*>(row + ks * 16 + 8 + 2 * t4) : 0u;
                }
            } else {
                uint2 raw[kSteps];
#pragma unroll
                for (int ks = 0; ks < kSteps; ++ks)
                    raw[ks] = valid ? *reinterpret_cast<const uint2*>(row + ks * 16 + 4 * t4) : make_uint2(0u, 0u);
                if (p.k_scale) coef[h] *= p.k_scale[x.kvh];
                if constexpr (std::is_same_v<T, __nv_bfloat16>) {
                    float top = 0.f;
#pragma unroll
                    for (int ks = 0; ks < kSteps; ++ks)
                        top = fmaxf(top, fmaxf(fmaxf(fabsf(Half16<T>::lo(raw[ks].x)), fabsf(Half16<T>::hi(raw[ks].x))),
                                               fmaxf(fabsf(Half16<T>::lo(raw[ks].y)), fabsf(Half16<T>::hi(raw[ks].y)))));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    // largest element into [2^14, 2^15); an infinite one is left as it is
                    const unsigned e = __float_as_uint(top) >> 23;
                    const unsigned f = e == 255u ? 127u : min(253u, 268u - e);
                    const float up = __uint_as_float(f << 23);
                    coef[h] *= __uint_as_float((254u - f) << 23);
#pragma unroll
                    for (int ks = 0; ks < kSteps; ++ks) {
                        qa[ks][h] = Half16<M>::pack(Half16<T>::lo(raw[ks].x) * up, Half16<T>::hi(raw[ks].x) * up);
                        qa[ks][2 + h] = Half16<M>::pack(Half16<T>::lo(raw[ks].y) * up, Half16<T>::hi(raw[ks].y) * up);
                    }
                } else {
#pragma unroll
                    for (int ks = 0; ks < kSteps; ++ks) qa[ks][h] = raw[ks].x, qa[ks][2 + h] = raw[ks].y;
                }
            }
        }

        float o[D / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
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
                float s[kUnit / 8][4];
#pragma unroll
                for (int i = 0; i < kUnit / 8; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[i][j] = 0.f;
                // ---- S = Q K^T
#pragma unroll
                for (int kb = 0; kb < kUnit / 16; ++kb) {
                    if constexpr (!kE4m3) {
                        const int key = kb * 16 + ((lane >> 4) << 3) + (lane & 7);
#pragma unroll
                        for (int ks = 0; ks < kSteps; ++ks) {
                            uint32_t r[4];
                            ldmatrix_x4(r, at_smem(tile_k, key, ks * 2 + ((lane >> 3) & 1)));
                            Half16<M>::mma(s[2 * kb], qa[ks], r[0], r[1]);
                            Half16<M>::mma(s[2 * kb + 1], qa[ks], r[2], r[3]);
                        }
                    } else {
                        const int key = kb * 16 + (((lane >> 3) & 1) << 3) + (lane & 7);
#pragma unroll
                        for (int ks = 0; ks < kSteps; ks += 2) {
                            uint32_t r[4];
                            ldmatrix_x4(r, at_smem(tile_k, key, ks + (lane >> 4)));
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                Half16<M>::mma(s[2 * kb + (i & 1)], qa[ks + (i >> 1)], f16x2_of_e4m3x2(r[i]), f16x2_of_e4m3x2(r[i] >> 16));
                        }
                    }
                }
                // ---- scale, mask, running maximum
                const bool whole = key0 >= lo_all && key0 + kUnit <= hi_all && boxes == (1u << n_boxes) - 1u;
                float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < kUnit / 8; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        float v = s[i][j] * coef[j >> 1];
                        if (!whole) {
                            const int k = i * 8 + 2 * t4 + (j & 1), key = key0 + k;
                            const bool in = key >= see[j >> 1].lo && key < see[j >> 1].hi && (boxes >> (k >= box_rows ? 1 : 0) & 1u);
                            v = in ? v : -INFINITY;
                        }
                        s[i][j] = v;
                        top[j >> 1] = fmaxf(top[j >> 1], v);
                    }
                float ref[2];
                bool moved = false;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
                    top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
                    moved |= top[h] > m[h];
                }
                if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float to = fmaxf(m[h], top[h]);
                        const float f = to == -INFINITY ? 1.f : ex2_approx(m[h] - to);
                        m[h] = to;
                        l[h] *= f;
#pragma unroll
                        for (int i = 0; i < D / 8; ++i) o[i][2 * h] *= f, o[i][2 * h + 1] *= f;
                    }
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) ref[h] = m[h] == -INFINITY ? 0.f : m[h];
                // ---- P, its sum, and O += P V
#pragma unroll
                for (int kb = 0; kb < kUnit / 16; ++kb) {
                    uint32_t pa[4];
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float a = ex2_approx(s[2 * kb + i][2 * h] - ref[h]), b = ex2_approx(s[2 * kb + i][2 * h + 1] - ref[h]);
                            l[h] += a + b;
                            pa[2 * i + h] = Half16<M>::pack(a, b);
                        }
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
                        const int key = kb * 16 + (((lane >> 3) & 1) << 3) + (lane & 7);
#pragma unroll
                        for (int dt = 0; dt < D / 16; ++dt) {
                            uint32_t r[4];
                            ldmatrix_x4_trans(r, at_smem(tile_v, key, dt * 2 + (lane >> 4)));
                            Half16<M>::mma(o[2 * dt], pa, r[0] & keep[0], r[1] & keep[1]);
                            Half16<M>::mma(o[2 * dt + 1], pa, r[2] & keep[0], r[3] & keep[1]);
                        }
                    } else {
                        const int key = kb * 16 + (((lane >> 3) & 1) << 3) + (lane & 7);
#pragma unroll
                        for (int dt = 0; dt < D / 16; dt += 2) {
                            uint32_t r[4];
                            ldmatrix_x4_trans(r, at_smem(tile_v, key, dt + (lane >> 4)));
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                const uint32_t a = r[2 * i] & keep[0], b = r[2 * i + 1] & keep[1];
                                Half16<M>::mma(o[2 * (dt + i)], pa, f16x2_of_e4m3x2(__byte_perm(a, 0, 0x4420)), f16x2_of_e4m3x2(__byte_perm(b, 0, 0x4420)));
                                Half16<M>::mma(o[2 * (dt + i) + 1], pa, f16x2_of_e4m3x2(__byte_perm(a, 0, 0x4431)), f16x2_of_e4m3x2(__byte_perm(b, 0, 0x4431)));
                            }
                        }
                    }
                }
            }
            __syncwarp();
            if (RW > 1 && lane == 0) mbar_arrive(empty0 + stage * 8);
        }

        // ---- the groups' shares of the work, joined
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
            if (t4 == 0) ctl.ml[warp][g8 + 8 * h] = make_float2(m[h], l[h]);
        }
        constexpr int kHalf = KW / 2;
        // Four neighbouring columns of a slot's row stand together; 8-column runs are moved by the row against bank conflicts.
        auto slot_at = [&](int slot, int row, int col) { return slots + slot * S::kSlotFloats + row * D + (col ^ ((row & 7) << 3)); };
        auto each_pair = [&](auto&& f) {       // f(row, column, value, value) for this thread's elements of O, two neighbours at a time
#pragma unroll
            for (int c = 0; c < D / 16; ++c)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if constexpr (kE4m3) {
                        f(h, c * 16 + 4 * t4, o[2 * c][2 * h], o[2 * c + 1][2 * h]);
                        f(h, c * 16 + 4 * t4 + 2, o[2 * c][2 * h + 1], o[2 * c + 1][2 * h + 1]);
                    } else {
                        f(h, c * 16 + 2 * t4, o[2 * c][2 * h], o[2 * c][2 * h + 1]);
                        f(h, c * 16 + 8 + 2 * t4, o[2 * c + 1][2 * h], o[2 * c + 1][2 * h + 1]);
                    }
                }
        };
        if (kw >= kHalf)
            each_pair([&](int h, int col, float a, float b) {
                *reinterpret_cast<float2*>(slot_at((kw - kHalf) * RW + rw, g8 + 8 * h, col)) = make_float2(a, b);
            });
        __syncthreads();
        if (*abort_flag != 0u) break;                          // the same in every thread: nobody waits between the barriers
        if (kw < kHalf) {
            float mine_f[2], other_f[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float all = -INFINITY;
#pragma unroll
                for (int k = 0; k < KW; ++k) all = fmaxf(all, ctl.ml[k * RW + rw][g8 + 8 * h].x);
                const float to = all == -INFINITY ? 0.f : all;
                mine_f[h] = ex2_approx(m[h] - to);
                other_f[h] = ex2_approx(ctl.ml[(kw + kHalf) * RW + rw][g8 + 8 * h].x - to);
            }
            each_pair([&](int h, int col, float a, float b) {
                float2* s2 = reinterpret_cast<float2*>(slot_at(kw * RW + rw, g8 + 8 * h, col));
                const float2 v = *s2;
                *s2 = make_float2(a * mine_f[h] + v.x * other_f[h], b * mine_f[h] + v.y * other_f[h]);
            });
        }
        __syncthreads();
        // ---- rows out: finished, or a piece's share for the join
        const bool from_start = at == x.work_begin, to_end = walk.work_end == work_end;
        const int share = share_of(cta, from_start);
        const float v_scale = kE4m3 && p.v_scale ? p.v_scale[x.kvh] : 1.f;
        for (int idx = threadIdx.x; idx < tile_rows * (D / 4); idx += kThreads) {
            const int r = idx / (D / 4), col = (idx % (D / 4)) * 4, r16 = r & 15, rwi = r >> 4;
            float all = -INFINITY, sum = 0.f;
#pragma unroll
            for (int k = 0; k < KW; ++k) all = fmaxf(all, ctl.ml[k * RW + rwi][r16].x);
            const float to = all == -INFINITY ? 0.f : all;
#pragma unroll
            for (int k = 0; k < KW; ++k) {
                const float2 v = ctl.ml[k * RW + rwi][r16];
                sum += v.y * ex2_approx(v.x - to);
            }
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int k = 0; k < kHalf; ++k) {
                const float4 v = *reinterpret_cast<const float4*>(slot_at(k * RW + rwi, r16, col));
                acc.x += v.x, acc.y += v.y, acc.z += v.z, acc.w += v.w;
            }
            if (from_start && to_end) {
                const int rr = x.rt * S::kRows + r, tok = rr / p.group, head = x.kvh * p.group + (rr - tok * p.group);
                const long long t = x.s.first + tok;
                const float f = v_scale / sum;                // a row without keys is zero
                *reinterpret_cast<uint2*>(static_cast<T*>(p.o) + t * p.o_stride + (long long)head * D + col) =
                    all == -INFINITY ? make_uint2(0u, 0u) : make_uint2(Half16<T>::pack(acc.x * f, acc.y * f), Half16<T>::pack(acc.z * f, acc.w * f));
                if (p.lse != nullptr && col == 0)
                    p.lse[t * p.n_heads + head] = all == -INFINITY ? -INFINITY : (all + log2f(sum)) * 0.69314718055994531f;
            } else {
                *reinterpret_cast<float4*>(p.ws_o + ((long long)share * S::kRows + r) * D + col) = acc;
                if (col == 0) p.ws_ml[share * S::kRows + r] = make_float2(all, sum);
            }
        }
        __syncthreads();
        at = walk.work_end;
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

// One cut's work: the shares of the pieces c-1, c, ... in the order of their keys. A warp has a row.
template <class T, bool kE4m3, int D>
__global__ void __launch_bounds__(128)
paged_join_kernel(const __grid_constant__ AttendParams p, int rows) {
    extern __shared__ float weights[];                        // [4][n_ctas]
    grid_launch_dependents();
    grid_dependency_wait();
    const int cta = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int4 job = p.ws_join[cta];
    if (job.w == 0) return;
    const int row = blockIdx.y * 4 + warp, rr = job.z * rows + row, tok = rr / p.group;
    Where x;
    x.b = job.x;
    load_seq(p, rows, 16, x);
    if (tok >= x.s.n_new) return;
    auto share = [&](int j) { return share_of(cta - 1 + j, j == 0); };
    float all = -INFINITY;
    for (int j = lane; j < job.w; j += 32) all = fmaxf(all, p.ws_ml[share(j) * rows + row].x);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) all = fmaxf(all, __shfl_xor_sync(0xffffffffu, all, d));
    const float to = all == -INFINITY ? 0.f : all;
    float sum = 0.f, *w = weights + warp * p.n_ctas;
    for (int j = lane; j < job.w; j += 32) {
        const float2 v = p.ws_ml[share(j) * rows + row];
        const float f = ex2_approx(v.x - to);
        w[j] = f;
        sum += v.y * f;
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    __syncwarp();
    constexpr int kCols = D / 32;
    float acc[kCols] = {};
#pragma unroll 8
    for (int j = 0; j < job.w; ++j) {
        const float* src = p.ws_o + ((long long)share(j) * rows + row) * D + lane * kCols;
        const float f = w[j];
#pragma unroll
        for (int i = 0; i < kCols; i += 2) {
            const float2 v = *reinterpret_cast<const float2*>(src + i);
            acc[i] += f * v.x;
            acc[i + 1] += f * v.y;
        }
    }
    const int head = job.y * p.group + (rr - tok * p.group);
    const long long t = x.s.first + tok;
    const float f = (kE4m3 && p.v_scale ? p.v_scale[job.y] : 1.f) / sum;
    uint32_t* dst = reinterpret_cast<uint32_t*>(static_cast<T*>(p.o) + t * p.o_stride + (long long)head * D + lane * kCols);
#pragma unroll
    for (int i = 0; i < kCols; i += 2) dst[i / 2] = all == -INFINITY ? 0u : Half16<T>::pack(acc[i] * f, acc[i + 1] * f);
    if (p.lse != nullptr && lane == 0)
        p.lse[t * p.n_heads + head] = all == -INFINITY ? -INFINITY : (all + log2f(sum)) * 0.69314718055994531f;
}

template <class T, bool kE4m3, int D, int RW>
cudaError_t prepare_one() {
    return cudaFuncSetAttribute(paged_token_kernel<T, kE4m3, D, RW>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                (int)Shape<kE4m3, D, RW>::kSmem + 1024);
}
template <class T, bool kE4m3, int D>
cudaError_t prepare_rows() {
    cudaFuncAttributes attr;
    cudaError_t e = prepare_one<T, kE4m3, D, 1>();
    if (e == cudaSuccess) e = prepare_one<T, kE4m3, D, 2>();
    if (e == cudaSuccess) e = prepare_one<T, kE4m3, D, 4>();
    if (e == cudaSuccess) e = cudaFuncGetAttributes(&attr, paged_join_kernel<T, kE4m3, D>);
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
    cfg.dynamicSmemBytes = Shape<kE4m3, D, 1>::kSmem + 1024;   // the same for 16, 32 and 64 rows
    cfg.stream = stream;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, rows == 16 ? paged_token_kernel<T, kE4m3, D, 1>
                                             : rows == 32 ? paged_token_kernel<T, kE4m3, D, 2> : paged_token_kernel<T, kE4m3, D, 4>, p);
    if (e != cudaSuccess || p.n_ctas == 1) return e;
    cfg.gridDim = dim3(p.n_ctas, (used_rows + 3) / 4);
    cfg.blockDim = dim3(128);
    cfg.dynamicSmemBytes = 4 * sizeof(float) * p.n_ctas;
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

int token_rows(long long rows) { return rows <= 16 ? 16 : rows <= 32 ? 32 : 64; }

cudaError_t paged_token_prepare(PagedType type, PagedType cache, int head_dim) {
    return with_types(type, cache, head_dim, [](auto t, auto e, auto d) { return prepare_rows<decltype(t), decltype(e)::value, decltype(d)::value>(); });
}

cudaError_t paged_token_launch(const AttendParams& p, PagedType type, PagedType cache, int head_dim, int rows, int used_rows,
                               cudaStream_t stream) {
    return with_types(type, cache, head_dim, [&](auto t, auto e, auto d) { return launch<decltype(t), decltype(e)::value, decltype(d)::value>(p, rows, used_rows, stream); });
}

}  // namespace f2k
