// Causal attention of prompts over a paged cache, head_dim 64 or 128, for sm_100a.
//
// A tile is 128 query rows of one sequence and key head: 128 / group new tokens with the `group` query heads of the key
// head side by side (fewer rows where group does not divide 128), so a key and its value are read once for all heads
// that share them, and the rows of a tile see nearly the same keys. A CTA walks the 128-key tiles between the first key
// that its first token sees and the last that its last one sees, in one of two forms:
//
//   pair    two neighbouring query tiles, every key tile meets both: half the reads of the other form;
//   split   one query tile, its even key tiles for one softmax group and its odd ones for the other, joined at the end
//           through shared memory: CTAs half as long, for batches that do not fill the GPU with pairs, and for the odd last
//           tile of a sequence. (One group on all key tiles leaves the special-function unit and the tensor pipe idle
//           half the time: 1024 tokens behind 15001, 16 heads of 64, 154 us.)
//
// Roles as in the joint-attention kernel (attn_fwd_sm100.cu): warps 0-3 / 4-7 the softmax groups (one thread per row),
// warps 8 and 10 the loaders of K and V, warp 9 the tcgen05 issuer, P from tensor memory, lazily moved reference maxima. With
// head_dim 128 tensor memory has one S buffer, which the groups use in turn; with 64 each has its own (Columns), and a step of
// both groups takes 2900 clk, of which the special-function unit has work for 2048 (1024 a group); with one buffer a
// group waited another 900 to 1200 for its S. P is rounded to 16 bits in front of its product, as there; its sum is taken
// before. What differs from that kernel:
//
//  * A loader brings a key tile in page by page: a lane per page and 128-byte piece of head_dim looks its page up (a
//    tile ahead) and issues its own TMA box. Rows of V that no query of the CTA may see - the rest of the last page,
//    pages in front of a window, pages outside the cache - hold anything, and 0 * NaN is NaN in a product, so the loader
//    waits for such a tile and clears them before it hands the tile over. That is the last tile, or the first ones of a
//    window. (A row that some queries of the CTA see stays for all of them.) K and V have a ring and a loader each: K of the tile after next may come in as soon as S is done with its slot.
//  * Q is fetched by the softmax groups themselves (the rows of a tile are a gather once group is not a power of two).
//  * Scores are masked by key number, in tensor memory, only in tiles that some row of the warp does not see whole.
//
// e4m3 caches: a tile comes in as bytes into the second half of its slot, and its loader turns it into fp16 (exactly) in place,
// row by row, before it hands it over; rows of V to be cleared are written as zeros then. The products are fp16 ones; bf16
// queries are brought into fp16's range by a power of two per row, which goes into the row's exponent factor with the
// head's scale of K. (8192 tokens 582 us; 6.6 ms in the token kernel, which converts in registers for every 64 rows anew.)
//
// Long tiles first, inside a sequence: its first CTAs are its last tiles, which see the most keys. The sequences stand in the
// batch's order, so a batch starts its longest CTAs where its longest prompt stands (8 prompts of 60 to 3000 tokens: 93 us with
// the longest first, 100 with it last, 109 with it in the middle).
#include "../attn_params.h"
#include "../barrier_look.h"
#include "../ptx.cuh"
#include "../softmax_row.cuh"
#include "kv_launch.h"
#include "mma_sync.cuh"

#include <cstddef>
#include <type_traits>

namespace f2k {

using namespace f2k::ptx;

namespace {

constexpr int kThreads = 384, kLoadK = 8, kMmaWarp = 9, kLoadV = 10;
constexpr int kRows = 128, kKeys = kPromptTile;
constexpr uint32_t kPieceBytes = 128 * 128;             // 128 rows of 128 bytes
constexpr uint32_t kTmemCols = 512;
constexpr float kLazyThreshold = 8.0f;                  // log2 units
constexpr int kPParts = 2;
// Registers a thread, softmax groups and the other warps, of the 384 * 168 a CTA is launched with; the e4m3 loaders convert.
// Every variant spills a little (24 to 40 bytes of stack; 72 to 88 bytes loaded with 16-bit caches, 120 to 184 with e4m3).
// (e4m3 with 208 for the softmax: 8192 tokens 567 instead of 580 us, but with head_dim 64 1024 behind 15001 170 instead of 156.)
template <bool kE4m3>
constexpr int kRegsSoftmax = kE4m3 ? 216 : 224;
template <bool kE4m3>
constexpr int kRegsOther = (384 * 168 - 256 * kRegsSoftmax<kE4m3>) / 128 / 8 * 8;

constexpr int kMostStages = 4;
// Tensor memory: S and O in fp32, P two values a column.
template <int D>
struct Columns {
    static constexpr bool kOwnS = D == 64;
    static __host__ __device__ constexpr uint32_t s(int t) { return kOwnS ? 128 * t : 0; }
    static __host__ __device__ constexpr uint32_t p(int t) { return (kOwnS ? 256 : 128) + 64 * t; }
    static __host__ __device__ constexpr uint32_t o(int t) { return (kOwnS ? 384 : 256) + D * t; }
};

template <int D>
constexpr int kStages = D == 64 ? 4 : 2;                // tiles of K, and of V, in flight or in use: 64 KB each

struct Ctl {
    uint64_t q_full[2];
    uint64_t s_free[2];                                 // S is in registers; one buffer: [0]
    uint64_t p_full[2][kPParts];
    uint64_t joined;                                    // split form: group 1 has left its share (these: four arrivals each)
    uint64_t full[2][kMostStages];                      // [K, V][slot]
    uint64_t empty[2][kMostStages];
    uint64_t raw[2][kMostStages];                       // e4m3: the bytes are there
    uint64_t s_full[2];
    uint64_t pv_done[2];
    uint64_t drain;
    uint64_t clean;                                     // a V tile that has to be cleared in part has arrived
    uint32_t tmem_base;
    uint32_t abort;
    int2 see[2][kRows];                                 // [group][row]: keys that the row sees
    float row_scale[2][kRows];                          // e4m3 with bf16 queries: what a row of S is multiplied by
};

struct WarpBarriers {                                   // the MMA warp's side of barrier_look.h
    volatile uint32_t* abort_flag;
    long long limit;
    __device__ __forceinline__ bool test(uint32_t bar_a, uint32_t par_a, uint32_t bar_b, uint32_t par_b) const {
        return bar_a == bar_b ? mbar_test(bar_a, par_a) : mbar_test2(bar_a, par_a, bar_b, par_b);
    }
    __device__ __forceinline__ bool all(bool pred) const { return __all_sync(0xffffffffu, pred) != 0; }
    __device__ __forceinline__ bool wait(uint32_t bar, uint32_t par) const { return all(mbar_wait(bar, par, abort_flag, limit)); }
};

// 16 scores -> 8 packed pairs of T and the sum of the unrounded values (softmax_row.cuh has it for bf16).
template <class T>
__device__ __forceinline__ void exp_chunk(const uint32_t* s, uint32_t* pk, float c, float neg_mc, float (&sum)[4]) {
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
        float x0, x1, x2, x3;
        fma2(x0, x1, __uint_as_float(s[i + 0]), __uint_as_float(s[i + 1]), c, c, neg_mc, neg_mc);
        fma2(x2, x3, __uint_as_float(s[i + 2]), __uint_as_float(s[i + 3]), c, c, neg_mc, neg_mc);
        const float p0 = ex2_approx(x0), p1 = ex2_approx(x1), p2 = ex2_approx(x2), p3 = ex2_approx(x3);
        add2(sum[0], sum[1], sum[0], sum[1], p0, p1);
        add2(sum[2], sum[3], sum[2], sum[3], p2, p3);
        pk[i / 2 + 0] = Half16<T>::pack(p0, p1);
        pk[i / 2 + 1] = Half16<T>::pack(p2, p3);
    }
}

// The work of CTA `slot` (of one key head): sequence and first tile. Sequences one behind the other, in each the last
// tiles first. False: there is none.
struct Job {
    SeqView s;
    int b, tile0;
    bool two;
};
__device__ __forceinline__ bool find_job(const AttendParams& p, int tokens_per_tile, int per_cta, int slot, int lane, Job& job) {
    const PagedBatch& b = p.batch;
    int before = 0;
    for (int b0 = 0; b0 < b.n_seqs; b0 += 32) {
        const int i = b0 + lane;
        SeqView s{0, 0, 0, false};
        if (i < b.n_seqs) s = seq_view(b.cu ? b.cu[i] : i, b.cu ? b.cu[i + 1] : i + 1, b.lens[i], b.n_tokens, b.max_new, (long long)b.table_width << p.page_shift);
        if (s.bad && lane == i - b0) atomicOr(p.status, (int)kStatusBadLength);
        const int tiles = (s.n_new + tokens_per_tile - 1) / tokens_per_tile, ctas = (tiles + per_cta - 1) / per_cta;
        int upto = ctas;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, upto, d);
            if (lane >= d) upto += v;
        }
        const unsigned here = __ballot_sync(0xffffffffu, slot < before + upto);
        if (here != 0) {
            const int src = __ffs(here) - 1;
            const int nth = slot - before - __shfl_sync(0xffffffffu, upto - ctas, src);      // CTA of the sequence
            const int n = __shfl_sync(0xffffffffu, ctas, src), all = __shfl_sync(0xffffffffu, tiles, src);
            job.b = b0 + src;
            job.s.first = __shfl_sync(0xffffffffu, s.first, src);
            job.s.n_new = __shfl_sync(0xffffffffu, s.n_new, src);
            job.s.len = __shfl_sync(0xffffffffu, s.len, src);
            job.tile0 = (n - 1 - nth) * per_cta;
            job.two = per_cta == 2 && job.tile0 + 1 < all;
            return true;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    return false;
}

// Shared memory of a tile's Q, and later of its rows on their way out: there 16 bytes apart, against bank conflicts.
template <int D>
constexpr uint32_t kQArea = kRows * (D * 2 + 16);
template <int D>
constexpr int kSmemBytes = 2 * (int)kQArea<D> + 2 * kStages<D> * (D / 64) * (int)kPieceBytes + 1024;

// One row of e4m3, LPR lanes of 16 bytes, to fp16: lane c writes elements 16c .. 16c + 15 of the row.
struct Row16 {
    uint4 lo, hi;
};
__device__ __forceinline__ Row16 f16_of_e4m3x16(const uint4& v) {
    Row16 r;
    r.lo = make_uint4(f16x2_of_e4m3x2(v.x), f16x2_of_e4m3x2(v.x >> 16), f16x2_of_e4m3x2(v.y), f16x2_of_e4m3x2(v.y >> 16));
    r.hi = make_uint4(f16x2_of_e4m3x2(v.z), f16x2_of_e4m3x2(v.z >> 16), f16x2_of_e4m3x2(v.w), f16x2_of_e4m3x2(v.w >> 16));
    return r;
}

template <class T, bool kE4m3, int D>
__global__ void __launch_bounds__(kThreads, 1)
paged_prompt_kernel(const __grid_constant__ AttendParams p, const int per_cta) {
    constexpr int kPieces = D / 64;                     // 128-byte pieces of a row
    constexpr uint32_t kTileBytes = kPieces * kPieceBytes;
    constexpr int kSlots = kStages<D>;
    constexpr bool kOwnS = Columns<D>::kOwnS;
    constexpr uint32_t kQBytes = kQArea<D>, kSmemQ = 0, kSmemRing = 2 * kQBytes;      // K slots, then V slots
    using M = std::conditional_t<kE4m3, __half, T>;     // the type of the products
    constexpr uint32_t kFormat = std::is_same_v<M, __nv_bfloat16> ? 1u : 0u;
    constexpr uint32_t kRowBytes = kE4m3 ? D : 128;     // of a piece as it comes in
    extern __shared__ uint8_t smem_raw[];
    __shared__ Ctl ctl_;
    Ctl* ctl = &ctl_;
    const uint32_t raw_addr = smem_u32(smem_raw);
    const uint32_t smem = (raw_addr + 1023u) & ~1023u;
    volatile uint32_t* abort_flag = &ctl->abort;
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0);
    const int lane = threadIdx.x & 31;
    const long long wait_limit = p.wait_limit_clk;

    grid_launch_dependents();
    if (warp == kLoadK) {
        constexpr int kBars = offsetof(Ctl, tmem_base) / sizeof(uint64_t), kPerWarp = offsetof(Ctl, full) / sizeof(uint64_t);
        for (int i = lane; i < kBars; i += 32) mbar_init(smem_u32(ctl) + i * 8, i < kPerWarp ? 4 : 1);    // a group's four warps arrive, or one thread
        if (lane == 0) ctl->abort = 0;
        fence_mbar_init();
        fence_proxy_async_smem();
    }
    if (warp == kMmaWarp) {
        tmem_alloc(smem_u32(&ctl->tmem_base), kTmemCols);
        tmem_relinquish();
    }
    grid_dependency_wait();
    const int kvh = blockIdx.x % p.n_kv_heads;
    const int per_tile = kRows / p.group;               // new tokens of a tile
    Job job;
    const bool any = find_job(p, per_tile, per_cta, blockIdx.x / p.n_kv_heads, lane, job);
    // Keys that some row of the CTA sees, and the key tiles they lie in.
    const bool pair = any && job.two;
    int lo = 0, hi = 0;
    if (any) {
        lo = visible_keys(job.s, job.tile0 * per_tile, p.window).lo;
        hi = visible_keys(job.s, min(job.s.n_new, (job.tile0 + (pair ? 2 : 1)) * per_tile) - 1, p.window).hi;
    }
    const int key00 = lo / kKeys * kKeys;
    const int n_kv = hi > key00 ? (hi - key00 + kKeys - 1) / kKeys : 0;
    // Step i of group t is key tile `tile_of(t, i)`, i < steps(t).
    auto steps = [&](int t) { return pair ? n_kv : (n_kv + 1 - t) >> 1; };
    auto tile_of = [&](int t, int i) { return pair ? i : 2 * i + t; };
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    constexpr uint32_t tmem = 0;                        // all columns are taken: the allocation starts at 0
    if (*reinterpret_cast<volatile uint32_t*>(&ctl->tmem_base) != tmem) ctl->abort = 1;

    if (warp >= 8) {
        setmaxnreg_dec<kRegsOther<kE4m3>>();
        if (warp == kLoadK || warp == kLoadV) {
            // ------------------------------ loaders: a lane per page and piece ------------------------------
            const int kv = warp == kLoadK ? 0 : 1;
            const int box_rows = min(kKeys, 1 << p.page_shift), n_boxes = kKeys / box_rows, box_shift = min(p.page_shift, 7);
            const int box = lane & 7, piece = lane >> 3;
            const bool mine = box < n_boxes && piece < (kE4m3 ? 1 : kPieces);
            const uint32_t all_boxes = (1u << n_boxes) - 1u;
            const int32_t* row = p.batch.table + (any ? job.b : 0) * p.batch.table_stride;
            const CUtensorMap* map = kv == 0 ? &p.tm_k : &p.tm_v;
            auto needed = [&](int j) {
                const int k = key00 + j * kKeys + box * box_rows;
                return mine && j < n_kv && k < hi && k + box_rows > lo;
            };
            auto look_up = [&](int j) { return needed(j) ? row[(key00 + j * kKeys + box * box_rows) >> p.page_shift] : 0; };
            // e4m3: tile j, which has come in, to fp16 where it lies. Rows go up: what row r's 256 (128) bytes of fp16 are written over has
            // been read before (its own bytes, or rows of its batch or below it). Tiles to be cleared in part have a loop of their own
            // (one loop with a test 732 us for 8192 tokens, apart 605, with eight rows a lane at a time instead of four 582).
            auto convert = [&](int j, uint32_t boxes) -> bool {
                const int slot = j % kSlots, base = key00 + j * kKeys;
                if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&ctl->raw[kv][slot]), (j / kSlots) & 1, abort_flag, wait_limit))) return false;
                const bool clear = kv == 1 && (base < lo || base + kKeys > hi || boxes != all_boxes);
                const uint32_t dst = smem + kSmemRing + (kv * kSlots + slot) * kTileBytes, in = dst + kTileBytes / 2;
                constexpr int kLanes = D / 16, kAtOnce = 32 / kLanes, kBatch = 8;      // lanes of a row, rows of the warp at once
                const int ch = lane % kLanes;
                auto rows = [&](auto clears) {
#pragma unroll 1
                    for (int r0 = lane / kLanes; r0 < kKeys; r0 += kAtOnce * kBatch) {
                        uint4 v[kBatch];
#pragma unroll
                        for (int u = 0; u < kBatch; ++u) {
                            const int r = r0 + u * kAtOnce, twist = D == 128 ? (r & 7) : ((r >> 1) & 3);
                            v[u] = ld_shared_v4(in + r * D + ((ch ^ twist) << 4));
                            if constexpr (decltype(clears)::value) {
                                const int key = base + r;
                                if (!(key >= lo && key < hi && (boxes >> (r >> box_shift) & 1u))) v[u] = make_uint4(0, 0, 0, 0);
                            }
                        }
                        __syncwarp();
#pragma unroll
                        for (int u = 0; u < kBatch; ++u) {
                            const int r = r0 + u * kAtOnce;
                            const Row16 w = f16_of_e4m3x16(v[u]);
                            const uint32_t at = dst + (ch >> 2) * kPieceBytes + r * 128;
                            st_shared_v4(at + (((2 * ch & 7) ^ (r & 7)) << 4), w.lo);
                            st_shared_v4(at + (((2 * ch + 1 & 7) ^ (r & 7)) << 4), w.hi);
                        }
                        __syncwarp();
                    }
                };
                if (clear) rows(std::true_type{});
                else rows(std::false_type{});
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&ctl->full[kv][slot]));
                return true;
            };
            uint32_t came_boxes = 0;                          // e4m3: of the tile that is to be converted next
            int converted = 0;
            // On the way out j is the number of tiles whose copies report to `raw` or `full`. (Counted apart: 1.4 % of the whole, in registers.)
            int next_page = look_up(0), cleaned = 0, j = 0;
            bool ok = true;
            for (; j < n_kv; ++j) {
                const int slot = j % kSlots, base = key00 + j * kKeys, page = next_page;
                next_page = look_up(j + 1);
                const bool wanted = needed(j), good = wanted && (unsigned)page < (unsigned)p.n_pages;
                if (wanted && !good) atomicOr(p.status, (int)kStatusBadPage);
                const uint32_t boxes = __ballot_sync(0xffffffffu, good) & 0xFFu;
                if constexpr (kE4m3) {
                    // The tile before is converted while this one's slot is still in use, or its copy on its way.
                    const bool free = j < kSlots || mbar_test(smem_u32(&ctl->empty[kv][slot]), ((j / kSlots) & 1) ^ 1u);
                    if (converted < j && !__all_sync(0xffffffffu, free)) {
                        if (!(ok = convert(converted, came_boxes))) break;
                        ++converted;
                    }
                }
                if (j >= kSlots) {
                    ok = mbar_wait(smem_u32(&ctl->empty[kv][slot]), ((j / kSlots) & 1) ^ 1u, abort_flag, wait_limit);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                }
                const bool clear = kv == 1 && (base < lo || base + kKeys > hi || boxes != all_boxes);
                const uint32_t full = smem_u32(&ctl->full[kv][slot]);
                const uint32_t bar = kE4m3 ? smem_u32(&ctl->raw[kv][slot]) : clear ? smem_u32(&ctl->clean) : full;
                const uint32_t dst = smem + kSmemRing + (kv * kSlots + slot) * kTileBytes, in = dst + (kE4m3 ? kTileBytes / 2 : 0);
                if (lane == 0) {
                    mbar_arrive_expect_tx(bar, (uint32_t)__popc(boxes) * (kE4m3 ? 1 : kPieces) * (uint32_t)box_rows * kRowBytes);
                }
                __syncwarp();
                if (good) {
                    const int first = (base + box * box_rows) & ((1 << p.page_shift) - 1);
                    tma_load_5d(in + piece * kPieceBytes + box * box_rows * kRowBytes, map, bar, 0, first, piece, kvh, page);
                }
                if constexpr (kE4m3) {
                    if (converted < j) {
                        if (!(ok = convert(converted, came_boxes))) {
                            ++j;                              // this tile's copies are on their way
                            break;
                        }
                        ++converted;
                    }
                    came_boxes = boxes;
                    continue;
                }
                if (clear) {
                    ok = mbar_wait(bar, cleaned & 1, abort_flag, wait_limit);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    ++cleaned;
                    for (int r = lane >> 3; r < kKeys; r += 4) {
                        const int key = base + r;
                        if (key >= lo && key < hi && (boxes >> (r >> box_shift) & 1u)) continue;
#pragma unroll
                        for (int i = 0; i < kPieces; ++i) st_shared_v4(dst + i * kPieceBytes + r * 128 + (lane & 7) * 16, make_uint4(0, 0, 0, 0));
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(full);
                }
            }
            if (kE4m3 && ok && converted < n_kv) ok = convert(converted, came_boxes);
            if (!ok) {
                // Leaving early: let the copies this warp started land first (bounded), the present tile's among them.
                volatile uint32_t never = 0;
                if (kv == 1 && !kE4m3) mbar_wait(smem_u32(&ctl->clean), cleaned & 1, &never, 4000000ll);
                for (int i = max(0, j - kSlots); i < j; ++i)
                    mbar_wait(smem_u32(kE4m3 ? &ctl->raw[kv][i % kSlots] : &ctl->full[kv][i % kSlots]), (i / kSlots) & 1, &never, 40000000ll);
            }
        } else if (warp == kMmaWarp) {
            // ------------------------------ MMA issuer, converged ------------------------------
            constexpr uint32_t idesc_s = umma_idesc_16(kRows, kKeys, false, kFormat), idesc_o = umma_idesc_16(kRows, D, true, kFormat);
            bool ok = true;
            const uint64_t q0_desc = umma_smem_desc(smem + kSmemQ, 16, 1024), q1_desc = umma_smem_desc(smem + kSmemQ + (pair ? kQBytes : 0), 16, 1024);
            const uint64_t k_desc0 = umma_smem_desc(smem + kSmemRing, 16, 1024);
            const uint64_t v_desc0 = umma_smem_desc(smem + kSmemRing + kSlots * kTileBytes, kPieceBytes, 1024);
            const uint32_t bar_full0 = smem_u32(&ctl->full[0][0]), bar_empty0 = smem_u32(&ctl->empty[0][0]), bar_free = smem_u32(&ctl->s_free[0]);
            // Every wait is looked at ahead, in front of the MMAs before it; a look at a barrier that the warp has seen complete
            // before (the second group's at a tile of a pair) costs nothing more.
            auto slot_off16 = [&](int j) { return (uint32_t)(j % kSlots) * (kTileBytes >> 4); };
            const WarpBarriers bars{abort_flag, wait_limit};
            auto peek = [&](auto... bar_and_parity) { return look_at(bars, bar_and_parity...); };
            auto finish = [&](const Look& l) { return f2k::finish(bars, l); };
            auto bar_full = [&](int kv, int j) { return bar_full0 + (kv * kMostStages + j % kSlots) * 8; };
            auto par_full = [&](int j) { return (uint32_t)(j / kSlots) & 1u; };
            auto release = [&](int kv, int j) { umma_commit(bar_empty0 + (kv * kMostStages + j % kSlots) * 8); };
            auto bar_p = [&](int t, int part) { return smem_u32(&ctl->p_full[t][part]); };
            // With one S buffer the order is S0_0, then S1_i, P1 V_(i-1), S0_(i+1), P0 V_i: S0_i is use 2i of the buffer and S1_i use
            // 2i + 1, and a use waits for the release of the one before. The two forms are compiled apart: this warp's instructions are what a tile
            // costs (with `pair` looked at as it goes the pair form took 6 % longer).
            auto run = [&](auto form) {
                constexpr bool kPair = decltype(form)::value;
                auto tile = [](int t, int i) { return kPair ? i : 2 * i + t; };
                const int n0 = kPair ? n_kv : (n_kv + 1) >> 1, n1 = kPair ? n_kv : n_kv >> 1;
                // S_t of step i: K's tile (seen before where the other group of a pair had it), and the S buffer read: its own, step
                // i - 1; or the one that both use.
                auto look_s = [&](int t, int i) {
                    const int j = tile(t, i);
                    const uint32_t free = bar_free + (kOwnS ? t * 8 : 0), par = kOwnS ? (uint32_t)(i - 1) & 1u : t == 1 ? 0u : 1u;
                    if (kPair && t == 1) return peek(free, par);
                    return peek(bar_full(0, j), par_full(j), free, par);
                };
                auto look_p = [&](int t, int i) {
                    const int j = tile(t, i);
                    if (kPair && t == 1) return peek(bar_p(1, 0), (uint32_t)i & 1u);   // V_i is there
                    return peek(bar_full(1, j), par_full(j), bar_p(t, 0), (uint32_t)i & 1u);
                };
                auto issue_s = [&](int t, int i) {
                    tc_fence_after_sync();
                    const int j = tile(t, i);
                    const uint64_t q = t == 0 ? q0_desc : q1_desc, k = k_desc0 + slot_off16(j);
                    const uint32_t d = tmem + (t == 0 ? Columns<D>::s(0) : Columns<D>::s(1));
                    if constexpr (kPieces == 2) umma_ss_x8(d, q, k, idesc_s);
                    else umma_ss_x4(d, q, k, idesc_s);
                    umma_commit(smem_u32(&ctl->s_full[t]));
                    if (t == 1 || !kPair) release(0, j);
                };
                // O_t (+)= P_t V_j, half by half as the softmax group hands P over; `next` takes the look at what follows.
                auto issue_pv = [&](int t, int i, const Look& first, auto&& next) -> bool {
                    const int j = tile(t, i);
                    const uint32_t d = tmem + (t == 0 ? Columns<D>::o(0) : Columns<D>::o(1)), a = tmem + (t == 0 ? Columns<D>::p(0) : Columns<D>::p(1));
                    const uint64_t v = v_desc0 + slot_off16(j);
                    if (!finish(first)) return false;
                    const Look half = peek(bar_p(t, 1), (uint32_t)i & 1u);
                    tc_fence_after_sync();
                    umma_ts_x4(d, a, v, idesc_o, i > 0 ? 1u : 0u);
                    if (!finish(half)) return false;
                    next();
                    tc_fence_after_sync();
                    umma_ts_x4(d, a + 32, v + 4 * (2048 >> 4), idesc_o, 1u);
                    umma_commit(smem_u32(&ctl->pv_done[t]));
                    if (t == 1 || !kPair) release(1, j);
                    return true;
                };
                Look s_look{}, p_look{};
                if (n0 > 0) {
                    ok = bars.wait(smem_u32(&ctl->q_full[0]), 0) && bars.wait(bar_full(0, 0), 0);
                    if (ok) issue_s(0, 0);
                    if (ok && kPair) ok = bars.wait(smem_u32(&ctl->q_full[1]), 0);
                }
                if constexpr (kOwnS) {
                    // S0_0, S1_0, then S0_(i+1), P0 V_i, S1_(i+1), P1 V_i.
                    if (ok && n1 > 0) {
                        if (!kPair) ok = bars.wait(bar_full(0, tile(1, 0)), par_full(tile(1, 0)));
                        if (ok) issue_s(1, 0);
                    }
                    if (n0 > 1) s_look = look_s(0, 1);
                    for (int i = 0; i < n0 && ok; ++i) {
                        if (i + 1 < n0) {
                            if (!(ok = finish(s_look))) break;
                            p_look = look_p(0, i);
                            issue_s(0, i + 1);
                        } else {
                            p_look = look_p(0, i);
                        }
                        if (!(ok = issue_pv(0, i, p_look, [&] { if (i + 1 < n1) s_look = look_s(1, i + 1); }))) break;
                        if (i >= n1) break;
                        if (i + 1 < n1) {
                            if (!(ok = finish(s_look))) break;
                            p_look = look_p(1, i);
                            issue_s(1, i + 1);
                        } else {
                            p_look = look_p(1, i);
                        }
                        if (!(ok = issue_pv(1, i, p_look, [&] { if (i + 2 < n0) s_look = look_s(0, i + 2); }))) break;
                    }
                    return;
                }
                if (n1 > 0) s_look = look_s(1, 0);
                for (int i = 0; i < n0 && ok; ++i) {
                    if (i < n1) {
                        if (!(ok = finish(s_look))) break;
                        if (i > 0) p_look = look_p(1, i - 1);
                        issue_s(1, i);
                    } else if (i > 0 && i - 1 < n1) {
                        p_look = look_p(1, i - 1);
                    }
                    auto look_next_s0 = [&] {
                        if (i + 1 < n0) s_look = look_s(0, i + 1);
                    };
                    if (i > 0 && i - 1 < n1) {
                        if (!(ok = issue_pv(1, i - 1, p_look, look_next_s0))) break;
                    } else {
                        look_next_s0();
                    }
                    if (i + 1 < n0) {
                        if (!(ok = finish(s_look))) break;
                    }
                    p_look = look_p(0, i);
                    if (i + 1 < n0) issue_s(0, i + 1);
                    if (!(ok = issue_pv(0, i, p_look, [&] { if (i + 1 < n1) s_look = look_s(1, i + 1); }))) break;
                }
                if (ok && n0 > 0 && n1 == n0) ok = issue_pv(1, n1 - 1, look_p(1, n1 - 1), [] {});
            };
            if (pair) run(std::true_type{});
            else run(std::false_type{});
            if (!ok) {
                // Leaving early: until the MMAs already issued retire (bounded), so tensor memory is idle when freed.
                volatile uint32_t never = 0;
                __syncwarp();
                umma_commit(smem_u32(&ctl->drain));
                mbar_wait(smem_u32(&ctl->drain), 0, &never, 40000000ll);
            }
        }
    } else if (any) {
        // ------------------------------ softmax groups ------------------------------
        setmaxnreg_inc<kRegsSoftmax<kE4m3>>();
        const int t = warp >> 2;
        const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t tS = tmem + lane_base + Columns<D>::s(t), tP = tmem + lane_base + Columns<D>::p(t), tO = tmem + lane_base + Columns<D>::o(t);
        float c = kE4m3 ? score_factor(p.scale_log2, p.k_scale, kvh) : p.scale_log2;        // of this thread's row
        const int tok0 = (job.tile0 + (pair ? t : 0)) * per_tile, rows = min(per_tile, job.s.n_new - tok0) * p.group;
        constexpr int kChunks = D / 8;                  // 16-byte chunks of a row
        const uint32_t q_tile = smem + kSmemQ + (pair ? t : 0) * kQBytes;
        // Row r of a tile is token r / group: by a multiplication (r < 128, group <= 128), a division per row cost more than the row.
        const uint32_t over_group = (65536u + (uint32_t)p.group - 1u) / (uint32_t)p.group;
        auto token_of = [&](int r) { return (int)((uint32_t)r * over_group >> 16); };
        constexpr int kAtOnce = 32 / kChunks;           // rows that a warp reads or writes at once
        const int ch = lane % kChunks, first_row = (warp & 3) * 32 + lane / kChunks;
        if (t == 0 || pair) {   // Q rows to shared memory as the MMA reads them: 128-byte pieces, chunks swizzled by row. All loads first.
            const T* q = static_cast<const T*>(p.q) + (long long)(job.s.first + tok0) * p.q_stride + (long long)kvh * p.group * D + ch * 8;
            uint4 v[kChunks];
#pragma unroll
            for (int i = 0; i < kChunks; ++i) {
                const int r = first_row + i * kAtOnce, tok = token_of(r);
                v[i] = make_uint4(0, 0, 0, 0);
                if (r < rows) v[i] = *reinterpret_cast<const uint4*>(q + tok * p.q_stride + (r - tok * p.group) * D);
            }
            if constexpr (kE4m3 && std::is_same_v<T, __nv_bfloat16>) {
#pragma unroll
                for (int i = 0; i < kChunks; ++i) {
                    using H = Half16<T>;
                    uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
                    float top = 0.f;
#pragma unroll
                    for (int k = 0; k < 4; ++k) top = fmaxf(top, fmaxf(fabsf(H::lo(w[k])), fabsf(H::hi(w[k]))));
#pragma unroll
                    for (int d = 1; d < kChunks; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                    const unsigned f = fp16_row_power(top, c);
                    const float up = __uint_as_float(f << 23);
#pragma unroll
                    for (int k = 0; k < 4; ++k) w[k] = Half16<M>::pack(H::lo(w[k]) * up, H::hi(w[k]) * up);
                    v[i] = make_uint4(w[0], w[1], w[2], w[3]);
                    if (ch == 0) ctl->row_scale[t][first_row + i * kAtOnce] = __uint_as_float((254u - f) << 23);
                }
            }
#pragma unroll
            for (int i = 0; i < kChunks; ++i) {
                const int r = first_row + i * kAtOnce;
                st_shared_v4(q_tile + (ch >> 3) * kPieceBytes + r * 128 + (((ch & 7) ^ (r & 7)) << 4), v[i]);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&ctl->q_full[t]));
        }
        const int r = (warp & 3) * 32 + lane;
        // Steps [clean0, clean1) have nothing to mask in this warp. What a row sees is kept in shared memory: the other steps read
        // it there, and these need its registers (rows that do not exist see everything and end nowhere).
        int clean0, clean1;
        {
            KeyRange see{0, 0x7fffffff};
            if (r < rows) see = visible_keys(job.s, tok0 + token_of(r), p.window);
            ctl->see[t][r] = make_int2(see.lo, see.hi);
            const int lo_max = __reduce_max_sync(0xffffffffu, see.lo), hi_min = __reduce_min_sync(0xffffffffu, see.hi);
            const int first = max(0, (lo_max - key00 + kKeys - 1) / kKeys), end = hi_min <= key00 ? 0 : min(n_kv, (hi_min - key00) / kKeys);
            clean0 = pair ? first : (first + 1 - t) >> 1;
            clean1 = pair ? end : (end + 1 - t) >> 1;
        }
        // The other steps' scores are masked where they lie, in tensor memory, chunk by chunk of 32 keys and only the chunks that
        // are cut, in front of the step proper: with the masks inside it, behind a test, every step paid for them in registers
        // and order of instructions (8192 tokens 499 us, without any masks 443; the step compiled twice, 523 to 540).
        const int box_shift = min(p.page_shift, 7);
        auto hide = [&](int tile, uint32_t bad) {
            const int base = key00 + tile * kKeys;
            const int2 see = ctl->see[t][(warp & 3) * 32 + lane];
            const int first = see.x - base, end = see.y - base;
#pragma unroll 1
            for (int from = 0; from < kKeys; from += 32) {
                if (bad == 0u && !__any_sync(0xffffffffu, end < from + 32 || first > from)) continue;
                uint32_t v[32];
                tmem_ld_x32(tS + from, v);
                const bool bad0 = bad >> (from >> box_shift) & 1u, bad1 = bad >> ((from + 16) >> box_shift) & 1u;
                const int lo0 = bad0 ? from + 16 : first, hi1 = bad1 ? from + 16 : end;      // either half of the chunk may be gone
                tmem_wait_ld();
#pragma unroll
                for (int k = 0; k < 16; ++k)
                    if (from + k < lo0 || from + k >= end) v[k] = __float_as_uint(-INFINITY);
#pragma unroll
                for (int k = 16; k < 32; ++k)
                    if (from + k < first || from + k >= hi1) v[k] = __float_as_uint(-INFINITY);
                tmem_st_x32(tS + from, v);
            }
            tmem_wait_st();
        };
        // Pages outside the cache: whether there are any is looked up once, while the first key tile is on its way, and which
        // only where there are. (A word in shared memory, written by the loader and read every step, cost 4 to 8 % of the whole,
        // the MMAs' operands keeping shared memory busy; a step's pages looked up a step ahead by the warp itself, 5 %.)
        const int32_t* pages = p.batch.table + job.b * p.batch.table_stride;
        bool strays = false;
#pragma unroll 4
        for (int k = (lo >> p.page_shift) + lane; k < (hi + (1 << p.page_shift) - 1) >> p.page_shift; k += 32)
            strays |= (unsigned)pages[k] >= (unsigned)p.n_pages;
        strays = __any_sync(0xffffffffu, strays);
        auto bad_pages = [&](int tile) {
            const int k = key00 + tile * kKeys + (lane << box_shift);
            const bool bad = lane < kKeys >> box_shift && k < hi && k + (1 << box_shift) > lo && (unsigned)pages[k >> p.page_shift] >= (unsigned)p.n_pages;
            return __ballot_sync(0xffffffffu, bad);
        };
        float m_ref = -INFINITY, l_sum = 0.0f;
        if constexpr (kE4m3 && std::is_same_v<T, __nv_bfloat16>) {
            if (t == 1 && !pair) {                      // the rows are group 0's
                const bool came = __all_sync(0xffffffffu, mbar_wait(smem_u32(&ctl->q_full[0]), 0, abort_flag, wait_limit));
                if (came) c *= ctl->row_scale[0][r];
            } else {
                c *= ctl->row_scale[t][r];              // written by this warp in front of the __syncwarp above
            }
        }
        bool ok = true;
        const int n = steps(t);
        for (int i = 0; i < n; ++i) {
            ok = mbar_wait(smem_u32(&ctl->s_full[t]), i & 1, abort_flag, wait_limit);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after_sync();
            if (i < clean0 || i >= clean1 || strays) hide(tile_of(t, i), strays ? bad_pages(tile_of(t, i)) : 0u);

            uint32_t s[128];
            float mx[kMaxChains];
            {
                uint32_t(&s0)[32] = *reinterpret_cast<uint32_t(*)[32]>(&s[0]);
                uint32_t(&s1)[32] = *reinterpret_cast<uint32_t(*)[32]>(&s[32]);
                uint32_t(&s2)[32] = *reinterpret_cast<uint32_t(*)[32]>(&s[64]);
                uint32_t(&s3)[32] = *reinterpret_cast<uint32_t(*)[32]>(&s[96]);
                tmem_ld_x32(tS + 0, s0);
                tmem_ld_x32(tS + 32, s1);
                tmem_wait_ld();
                tmem_ld_x32(tS + 64, s2);
                tmem_ld_x32(tS + 96, s3);
                row_max64<true>(&s[0], mx);
                tmem_wait_ld();
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&ctl->s_free[kOwnS ? t : 0]));
            }
            row_max64<false>(&s[64], mx);
            const float m_tile = row_max_finish(mx);
            const bool pv_seen = i == 0 || mbar_test(smem_u32(&ctl->pv_done[t]), (i - 1) & 1);

            const bool need = (m_tile - m_ref) * c > kLazyThreshold;
            if (__any_sync(0xffffffffu, need)) {
                const float m_new = fmaxf(m_ref, m_tile);
                const float f = m_new == -INFINITY ? 1.0f : ex2_approx((m_ref - m_new) * c);
                l_sum *= f;
                m_ref = m_new;
                if (i > 0) {
                    ok = mbar_wait(smem_u32(&ctl->pv_done[t]), (i - 1) & 1, abort_flag, wait_limit);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    tc_fence_after_sync();
#pragma unroll
                    for (int q = 0; q < D / 32; ++q) {
                        uint32_t o[32];
                        tmem_ld_x32(tO + q * 32, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
                        tmem_st_x32(tO + q * 32, o);
                    }
                }
            }
            // A row that has seen no key yet has the reference 0: its weights are 2^-inf = 0.
            const float neg_mc = m_ref == -INFINITY ? 0.0f : -m_ref * c;
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
            int pending = -1;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                uint32_t pk[16];
                exp_chunk<M>(&s[q * 32], pk, c, neg_mc, sum);
                if (pending >= 0) {
                    tmem_wait_st();
                    tc_fence_before_sync();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&ctl->p_full[t][0]) + pending * 8);
                    pending = -1;
                }
                exp_chunk<M>(&s[q * 32 + 16], pk + 8, c, neg_mc, sum);
                if (q == 0 && !__all_sync(0xffffffffu, pv_seen)) {
                    ok = mbar_wait(smem_u32(&ctl->pv_done[t]), (i - 1) & 1, abort_flag, wait_limit);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                }
                if (q == 0) tc_fence_after_sync();
                tmem_st_x16(tP + q * 16, pk);
                if ((q + 1) % (4 / kPParts) == 0) pending = (q + 1) / (4 / kPParts) - 1;
            }
            if (!ok) break;
            tmem_wait_st();
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&ctl->p_full[t][kPParts - 1]));
            l_sum += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        }

        // ------------------------------ epilogue ------------------------------
        // Rows are parked over the group's Q. The last product stands behind the Q of all four warps; without a step nothing does, and
        // a warp that is ahead would park its zeros where its neighbour still stores Q.
        if (ok && (n > 0 || t == 0 || pair)) {
            ok = n > 0 ? mbar_wait(smem_u32(&ctl->pv_done[t]), (n - 1) & 1, abort_flag, wait_limit)
                       : mbar_wait(smem_u32(&ctl->q_full[t]), 0, abort_flag, wait_limit);
            ok = __all_sync(0xffffffffu, ok);
        }
        // Split form: group 1 leaves its rows, in fp32, with their references and sums where the key tiles were (once no MMA reads
        // them any more), and group 0 takes them in.
        constexpr uint32_t kShareRow = D * 4 + 16;
        const uint32_t share = smem + kSmemRing + r * kShareRow;
        const bool joins = !pair && n_kv > 1;
        float other = 0.0f;                                  // factor of group 1's row
        if (ok && joins) {
            if (t == 1) {
                ok = mbar_wait(smem_u32(&ctl->pv_done[0]), (steps(0) - 1) & 1, abort_flag, wait_limit);
                ok = __all_sync(0xffffffffu, ok);
                if (ok) {
                    tc_fence_after_sync();
#pragma unroll
                    for (int q = 0; q < D / 32; ++q) {
                        uint32_t o[32];
                        tmem_ld_x32(tO + q * 32, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int k = 0; k < 32; k += 4) st_shared_v4(share + (q * 32 + k) * 4, make_uint4(o[k], o[k + 1], o[k + 2], o[k + 3]));
                    }
                    st_shared_v4(share + D * 4, make_uint4(__float_as_uint(m_ref), __float_as_uint(l_sum), 0u, 0u));
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&ctl->joined));
                }
            } else {
                ok = mbar_wait(smem_u32(&ctl->joined), 0, abort_flag, wait_limit);
                ok = __all_sync(0xffffffffu, ok);
            }
        }
        if (ok && (t == 0 || pair)) {
            tc_fence_after_sync();
            float mine = 1.0f;
            if (joins) {
                const uint4 v = ld_shared_v4(share + D * 4);
                const float m1 = __uint_as_float(v.x), m = fmaxf(m_ref, m1);
                if (m != -INFINITY) {
                    mine = ex2_approx((m_ref - m) * c);
                    other = ex2_approx((m1 - m) * c);
                }
                l_sum = l_sum * mine + __uint_as_float(v.y) * other;
                m_ref = m;
            }
            const bool none = l_sum == 0.0f && m_ref == -INFINITY;      // a row that sees no key is zero
            const float inv = (kE4m3 && p.v_scale != nullptr ? p.v_scale[kvh] : 1.0f) / l_sum;
            mine *= inv;
            other *= inv;
            // Rows go out through the shared memory of the tile's Q (no MMA reads it any more), a bulk copy each: 16-byte stores by
            // half-warps kept the CTA 6000 to 7000 clk.
            const uint32_t park = q_tile + r * (D * 2 + 16);
#pragma unroll
            for (int q = 0; q < D / 32; ++q) {
                uint32_t o[32];
                if (n > 0) {
                    tmem_ld_x32(tO + q * 32, o);
                    tmem_wait_ld();
                }
#pragma unroll
                for (int k = 0; k < 32; k += 8) {
                    float x[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(o[k + e]) * mine;
                    if (joins) {
#pragma unroll
                        for (int e = 0; e < 8; e += 4) {
                            const uint4 w = ld_shared_v4(share + (q * 32 + k + e) * 4);
                            x[e] += __uint_as_float(w.x) * other, x[e + 1] += __uint_as_float(w.y) * other;
                            x[e + 2] += __uint_as_float(w.z) * other, x[e + 3] += __uint_as_float(w.w) * other;
                        }
                    }
                    uint4 v = make_uint4(Half16<T>::pack(x[0], x[1]), Half16<T>::pack(x[2], x[3]), Half16<T>::pack(x[4], x[5]), Half16<T>::pack(x[6], x[7]));
                    if (none) v = make_uint4(0, 0, 0, 0);
                    st_shared_v4(park + (q * 4 + (k >> 3)) * 16, v);
                }
            }
            fence_proxy_async_smem();
            if (r < rows) {
                const int tok = token_of(r), head = kvh * p.group + (r - tok * p.group);
                const long long at = job.s.first + tok0 + tok;
                bulk_store(static_cast<T*>(p.o) + at * p.o_stride + (long long)head * D, park, D * 2);
                bulk_commit();
                if (p.lse != nullptr) p.lse[at * p.n_heads + head] = none ? -INFINITY : (m_ref * c + log2f(l_sum)) * 0.69314718055994531f;
                bulk_wait_read<0>();
            }
        }
    }

    __syncwarp();
    tc_fence_before_sync();
    __syncthreads();
    if (threadIdx.x == 0 && *abort_flag != 0u) atomicOr(p.status, (int)kStatusWaitExpired);
    if (warp == kMmaWarp) {
        tc_fence_after_sync();
        tmem_dealloc(tmem, kTmemCols);
    }
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

cudaError_t paged_prompt_prepare(PagedType type, PagedType cache, int head_dim) {
    return with_types(type, cache, head_dim, [](auto t, auto e, auto d) {
        return cudaFuncSetAttribute(paged_prompt_kernel<decltype(t), decltype(e)::value, decltype(d)::value>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    kSmemBytes<decltype(d)::value>);
    });
}

cudaError_t paged_prompt_launch(const AttendParams& p, PagedType type, PagedType cache, int head_dim, int max_new, int sms, cudaStream_t stream) {
    // CTAs that the sequences can need: their tiles rounded up, whatever the lengths.
    const int per_tile = kRows / p.group;
    auto ctas = [&](int per_cta) {
        const long long step = (long long)per_tile * per_cta;
        const long long by_tokens = p.batch.n_tokens / step + p.batch.n_seqs, by_most = (max_new + step - 1) / step * p.batch.n_seqs;
        return (by_tokens < by_most ? by_tokens : by_most) * p.n_kv_heads;
    };
    const int per_cta = ctas(2) >= sms ? 2 : 1;
    if (ctas(per_cta) > 0x7fffffffll) return cudaErrorInvalidConfiguration;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas(per_cta));
    cfg.blockDim = dim3(kThreads);
    cfg.stream = stream;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return with_types(type, cache, head_dim, [&](auto t, auto e, auto d) {
        cfg.dynamicSmemBytes = kSmemBytes<decltype(d)::value>;
        return cudaLaunchKernelEx(&cfg, paged_prompt_kernel<decltype(t), decltype(e)::value, decltype(d)::value>, p, per_cta);
    });
}

}  // namespace f2k
