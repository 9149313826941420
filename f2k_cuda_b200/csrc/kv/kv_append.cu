// New tokens into the paged cache: per-head RMSNorm and position rotation of Q and K on the way (both optional),
// K and V to the rows of their sequence's pages, Q to the attention's input.
//
// With y = x rsqrt(mean x^2 + eps) g, element i < r/2 of a row and its partner (i + r/2, or the neighbour in the
// interleaved form) become  y_a cos - y_b sin,  y_b cos + y_a sin  with the angle of the token's position; elements
// from r on stay. fp32 arithmetic, one rounding to the type stored.
//
// Bound: memory, and close behind it instructions. So a lane holds both halves of its pairs (16 elements: 16-byte chunks j
// and j + r/16 of a row, two neighbouring chunks where nothing is apart), no element crosses lanes but the sum of squares,
// a token's angles and gains are multiplied once for a set of four rows, and the arithmetic is packed pairs of fp32: 5274
// tokens of 32 + 2 x 8 heads, bf16, 27.9 us = 4.7 TB/s, 20000 tokens 5.6 TB/s (a lane per chunk, partners by shuffles, gain and
// angle apart: 43 us). The call's items are dealt out in equal runs to as many blocks as are resident; a block looks its
// tokens' sequences, positions and pages up 32 at a time, in shared memory. Tried: the next item's rows on their way while
// this one is worked on 39 us (128 registers and spills), two rows a team at a time 31, five blocks an SM 31 (spills).
// A few tokens (a decoding step) are bound by latency instead: there a team has one row (8 tokens: 3.2 us).
#include "../ptx.cuh"
#include "kv_launch.h"
#include "mma_sync.cuh"

#include <type_traits>

namespace f2k {

namespace {

constexpr int kBlock = 128, kBlocksPerSm = 4;

struct Token {
    long long k_at, v_at;      // element offset of the token's row of head 0
    int pos;                   // -1: leave the token alone
};

// The sequence of a token: the last one that begins at or before it (empty sequences before it are passed over).
__device__ __forceinline__ int sequence_of(const int32_t* cu, int n_seqs, int token) {
    int lo = 0, hi = n_seqs;                          // cu[lo] <= token < cu[hi] for the well-formed
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (cu[mid] <= token) lo = mid;
        else hi = mid;
    }
    return lo;
}

__device__ Token look_up(const AppendParams& p, int t) {
    Token r{0, 0, -1};
    const PagedBatch& b = p.batch;
    int seq, cu0, cu1;
    if (b.cu == nullptr) {
        seq = t, cu0 = t, cu1 = t + 1;
        if (t >= b.n_seqs) return r;
    } else {
        seq = sequence_of(b.cu, b.n_seqs, t);
        cu0 = b.cu[seq], cu1 = b.cu[seq + 1];
        if (t < cu0 || t >= cu1) return r;            // behind the last sequence
    }
    const SeqView s = seq_view(cu0, cu1, b.lens[seq], b.n_tokens, b.max_new, (long long)b.table_width << p.page_shift);
    const int pos = s.len - s.n_new + (t - s.first);
    if (s.bad || pos < 0) {
        atomicOr(p.status, (int)kStatusBadLength);
        return r;
    }
    if (p.rot_dim > 0 && pos >= p.n_positions) {
        atomicOr(p.status, (int)kStatusBadPosition);
        return r;
    }
    const int page = b.table[seq * b.table_stride + (pos >> p.page_shift)];
    if ((unsigned)page >= (unsigned)p.n_pages) {
        atomicOr(p.status, (int)kStatusBadPage);
        return r;
    }
    const int row = pos & ((1 << p.page_shift) - 1);
    r.k_at = page * p.kp_page + row * p.kp_tok;
    r.v_at = page * p.vp_page + row * p.vp_tok;
    r.pos = pos;
    return r;
}

struct Pair { float x, y; };                   // packed arithmetic works on these
__device__ __forceinline__ Pair mul(Pair a, Pair b) {
    Pair d;
    asm("{\n\t.reg .b64 ra, rb, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tmul.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ Pair fma(Pair a, Pair b, Pair c) {
    Pair d;
    ptx::fma2(d.x, d.y, a.x, a.y, b.x, b.y, c.x, c.y);
    return d;
}
// A lane's 16 elements of a row as x0, x1 so that x0[i] and x1[i] are a rotation's pairs: the two chunks, or (interleaved) the
// even and the odd elements of both.
template <class T, bool kInter>
__device__ __forceinline__ void unpack(const uint4 (&v)[2], Pair (&x0)[4], Pair (&x1)[4]) {
    const uint32_t w[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        using H = Half16<T>;
        x0[i] = kInter ? Pair{H::lo(w[2 * i]), H::lo(w[2 * i + 1])} : Pair{H::lo(w[i]), H::hi(w[i])};
        x1[i] = kInter ? Pair{H::hi(w[2 * i]), H::hi(w[2 * i + 1])} : Pair{H::lo(w[4 + i]), H::hi(w[4 + i])};
    }
}
// Elements 2i, 2i + 1 of the 16.
template <bool kInter>
__device__ __forceinline__ Pair in_order(const Pair (&x0)[4], const Pair (&x1)[4], int i) {
    if (kInter) return i & 1 ? Pair{x0[i >> 1].y, x1[i >> 1].y} : Pair{x0[i >> 1].x, x1[i >> 1].x};
    return i < 4 ? x0[i] : x1[i - 4];
}
__device__ __forceinline__ void load8(const float* p, Pair (&f)[4]) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    f[0] = Pair{a.x, a.y}, f[1] = Pair{a.z, a.w}, f[2] = Pair{b.x, b.y}, f[3] = Pair{b.z, b.w};
}

// An item is kSet rows of one kind (Q, K or V) and token, taken by a team of lanes, kAhead rows loaded at a time. A block takes an
// equal run of the call's items; kTokens: tokens looked up at a time.
template <class T, bool kE4m3, int kDim, bool kInter, int kSet>
__global__ void __launch_bounds__(kBlock, kBlocksPerSm)
kv_append_kernel(const __grid_constant__ AppendParams p) {
    constexpr int kLanes = kDim / 16, kTeams = kBlock / kLanes, kTokens = 32, kAhead = kSet < 4 ? kSet : 4;
    __shared__ Token tokens[kTokens];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int sub = threadIdx.x % kLanes, team = threadIdx.x / kLanes;
    const uint32_t mates = ((1u << kLanes) - 1u) << (threadIdx.x & 31 & ~(kLanes - 1));
    const int H = p.n_heads, G = p.n_kv_heads;
    const int q_sets = (H + kSet - 1) / kSet, k_sets = (G + kSet - 1) / kSet, sets = q_sets + 2 * k_sets;
    // This lane's two chunks of a row: lanes below `turning` rotate, by the angles 8 sub .. 8 sub + 7.
    const int turning = p.rot_dim >> 4;
    const bool apart = !kInter && sub < turning;
    const int c0 = apart ? sub : 2 * sub, c1 = apart ? sub + turning : 2 * sub + 1;
    const long long items = (long long)p.batch.n_tokens * sets;
    const long long first_item = items * blockIdx.x / gridDim.x, end_item = items * (blockIdx.x + 1) / gridDim.x;
    const int t_end = (int)((end_item + sets - 1) / sets);

    const T* src = nullptr;
    int kind = 0, row0 = 0, n_rows = 0;                       // of the present item; kind: 0 Q, 1 K, 2 V; n_rows 0: none left
    uint4 raw[kAhead][2];
    auto load = [&](int first) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (first + u < n_rows) {
                raw[u][0] = reinterpret_cast<const uint4*>(src + (first + u) * kDim)[c0];
                raw[u][1] = reinterpret_cast<const uint4*>(src + (first + u) * kDim)[c1];
            }
    };
    int t = (int)(first_item / sets), set = (int)(first_item - (long long)t * sets) + team;
    const int t_first = t;
    auto begin_item = [&]() {                                 // needs no look-up: rows of the call's tensors
        while (set >= sets) set -= sets, ++t;
        n_rows = 0;
        if ((long long)t * sets + set >= end_item) return;
        kind = set < q_sets ? 0 : set < q_sets + k_sets ? 1 : 2;
        row0 = (set - (kind == 0 ? 0 : kind == 1 ? q_sets : q_sets + k_sets)) * kSet;
        n_rows = min(kSet, (kind == 0 ? H : G) - row0);
        src = static_cast<const T*>(kind == 0 ? p.q : kind == 1 ? p.k : p.v) + t * (kind == 0 ? p.q_stride : kind == 1 ? p.k_stride : p.v_stride) + row0 * kDim;
        load(0);
    };
    begin_item();
    for (int t0 = t_first; t0 < t_end; t0 += kTokens) {
        if (t0 > t_first) __syncthreads();
        if (threadIdx.x < kTokens)
            tokens[threadIdx.x] = t0 + (int)threadIdx.x < t_end ? look_up(p, t0 + threadIdx.x) : Token{0, 0, -1};
        __syncthreads();
        for (; n_rows > 0 && t < t0 + kTokens; set += kTeams, begin_item()) {
            const Token tk = tokens[t - t0];
            if (tk.pos < 0) continue;
            // y0 = (x0 a0 + x1 b0) / rms, y1 = (x1 a1 + x0 b1) / rms: gains times cosines and sines.
            const T* gamma = static_cast<const T*>(kind == 0 ? p.gamma_q : kind == 1 ? p.gamma_k : nullptr);
            const bool turns = kind != 2 && sub < turning, norm = gamma != nullptr, as_is = kind == 2 || (!norm && p.rot_dim == 0);
            Pair a0[4], a1[4], b0[4], b1[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) a0[i] = a1[i] = Pair{1.f, 1.f};
            if (norm) {
                const uint4 g[2] = {reinterpret_cast<const uint4*>(gamma)[c0], reinterpret_cast<const uint4*>(gamma)[c1]};
                unpack<T, kInter>(g, a0, a1);
            }
            if (turns) {
                const long long at = (long long)tk.pos * (p.rot_dim >> 1) + 8 * sub;
                Pair c[4], s[4];
                load8(p.cos_tab + at, c);
                load8(p.sin_tab + at, s);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    b0[i] = mul(a1[i], Pair{-s[i].x, -s[i].y});
                    b1[i] = mul(a0[i], s[i]);
                    a0[i] = mul(a0[i], c[i]);
                    a1[i] = mul(a1[i], c[i]);
                }
            }
            // where the rows go: elements of the type stored
            const long long dst_head = kind == 0 ? kDim : kind == 1 ? p.kp_head : p.vp_head;
            const long long dst_at = (kind == 0 ? t * p.qo_stride : kind == 1 ? tk.k_at : tk.v_at) + row0 * dst_head;
            void* base = kind == 0 ? p.q_out : kind == 1 ? p.k_pages : p.v_pages;
#pragma unroll 1
            for (int first = 0; first < n_rows; first += kAhead) {
                if (first > 0) load(first);
#pragma unroll
                for (int u = 0; u < kAhead; ++u) {
                    if (first + u >= n_rows) break;          // the same for the whole team
                    const long long at = dst_at + (first + u) * dst_head;
                    if (as_is && !(kE4m3 && kind != 0)) {
                        uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(base) + at);
                        dst[c0] = raw[u][0];
                        dst[c1] = raw[u][1];
                        continue;
                    }
                    Pair x0[4], x1[4];
                    unpack<T, kInter>(raw[u], x0, x1);
                    if (!as_is) {
                        Pair over_rms{1.f, 1.f};
                        if (norm) {
                            Pair ss = mul(x0[0], x0[0]), s2 = mul(x1[0], x1[0]);
#pragma unroll
                            for (int i = 1; i < 4; ++i) ss = fma(x0[i], x0[i], ss), s2 = fma(x1[i], x1[i], s2);
                            float sum = (ss.x + s2.x) + (ss.y + s2.y);
#pragma unroll
                            for (int d = kLanes / 2; d > 0; d >>= 1) sum += __shfl_xor_sync(mates, sum, d);
                            over_rms.x = over_rms.y = rsqrtf(sum * (1.0f / kDim) + p.eps);
                        }
                        if (turns) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const Pair y = fma(x0[i], a0[i], mul(x1[i], b0[i]));
                                x1[i] = mul(fma(x1[i], a1[i], mul(x0[i], b1[i])), over_rms);
                                x0[i] = mul(y, over_rms);
                            }
                        } else {
#pragma unroll
                            for (int i = 0; i < 4; ++i) x0[i] = mul(mul(x0[i], a0[i]), over_rms), x1[i] = mul(mul(x1[i], a1[i]), over_rms);
                        }
                    }
                    uint32_t w[8];
                    if (kE4m3 && kind != 0) {
                        // over the head's scale, to nearest even, beyond +-448 saturated, NaN kept
                        const float* scale = kind == 2 ? p.v_scale : p.k_scale;
                        const float over = scale ? 1.0f / scale[row0 + first + u] : 1.0f;
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const Pair v = mul(in_order<kInter>(x0, x1, i), Pair{over, over});
                            w[i] = __nv_cvt_float2_to_fp8x2(make_float2(v.x, v.y), __NV_SATFINITE, __NV_E4M3);
                        }
                        uint2* dst = reinterpret_cast<uint2*>(static_cast<uint8_t*>(base) + at);
                        dst[c0] = make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
                        dst[c1] = make_uint2(w[4] | w[5] << 16, w[6] | w[7] << 16);
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const Pair v = in_order<kInter>(x0, x1, i);
                            w[i] = Half16<T>::pack(v.x, v.y);
                        }
                        uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(base) + at);
                        dst[c0] = make_uint4(w[0], w[1], w[2], w[3]);
                        dst[c1] = make_uint4(w[4], w[5], w[6], w[7]);
                    }
                }
            }
        }
    }
}

template <class T, bool kE4m3, int kDim, bool kInter>
cudaError_t launch(const AppendParams& p, int sms, cudaStream_t stream) {
    constexpr int kTeams = kBlock / (kDim / 16), kMany = 4;
    const int H = p.n_heads, G = p.n_kv_heads;
    const long long n = p.batch.n_tokens, rows = n * (H + 2 * G), sets = n * ((H + kMany - 1) / kMany + 2 * ((G + kMany - 1) / kMany));
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(kBlock);
    cfg.stream = stream;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    // While every row can have a team of its own on the GPU at once, it gets one; beyond, four rows a team, and as many blocks as
    // are resident.
    const long long most = (long long)kBlocksPerSm * sms;
    if (rows <= most * kTeams) {
        cfg.gridDim = dim3((unsigned)((rows + kTeams - 1) / kTeams));
        return cudaLaunchKernelEx(&cfg, kv_append_kernel<T, kE4m3, kDim, kInter, 1>, p);
    }
    const long long blocks = (sets + kTeams - 1) / kTeams;
    cfg.gridDim = dim3((unsigned)(blocks < most ? blocks : most));
    return cudaLaunchKernelEx(&cfg, kv_append_kernel<T, kE4m3, kDim, kInter, kMany>, p);
}

}  // namespace

cudaError_t kv_append_prepare(PagedType type, PagedType cache, int head_dim, bool interleaved) {
    cudaFuncAttributes attr;
    auto load = [&](auto t, auto e, auto d, auto i) {
        using T = decltype(t);
        constexpr bool kE = decltype(e)::value, kI = decltype(i)::value;
        const cudaError_t r = cudaFuncGetAttributes(&attr, kv_append_kernel<T, kE, decltype(d)::value, kI, 1>);
        return r == cudaSuccess ? cudaFuncGetAttributes(&attr, kv_append_kernel<T, kE, decltype(d)::value, kI, 4>) : r;
    };
    auto by_pairs = [&](auto t, auto e, auto d) { return interleaved ? load(t, e, d, std::true_type{}) : load(t, e, d, std::false_type{}); };
    auto by_dim = [&](auto t, auto e) {
        return head_dim == 64 ? by_pairs(t, e, std::integral_constant<int, 64>{}) : by_pairs(t, e, std::integral_constant<int, 128>{});
    };
    auto by_cache = [&](auto t) { return cache == kE4m3 ? by_dim(t, std::true_type{}) : by_dim(t, std::false_type{}); };
    return type == kBf16 ? by_cache(__nv_bfloat16{}) : by_cache(__half{});
}

cudaError_t kv_append_launch(const AppendParams& p, PagedType type, PagedType cache, int head_dim, int sms, cudaStream_t stream) {
    auto by_dim = [&](auto t, auto e) {
        using T = decltype(t);
        constexpr bool kE = decltype(e)::value;
        if (p.interleaved) return head_dim == 64 ? launch<T, kE, 64, true>(p, sms, stream) : launch<T, kE, 128, true>(p, sms, stream);
        return head_dim == 64 ? launch<T, kE, 64, false>(p, sms, stream) : launch<T, kE, 128, false>(p, sms, stream);
    };
    auto by_cache = [&](auto t) { return cache == kE4m3 ? by_dim(t, std::true_type{}) : by_dim(t, std::false_type{}); };
    return type == kBf16 ? by_cache(__nv_bfloat16{}) : by_cache(__half{});
}

}  // namespace f2k
