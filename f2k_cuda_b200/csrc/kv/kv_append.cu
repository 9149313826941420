// New tokens into the paged cache: per-head RMSNorm and position rotation of Q and K on the way (both optional),
// K and V to the rows of their sequence's pages, Q to the attention's input.
//
// With y = x rsqrt(mean x^2 + eps) g, element i < r/2 of a row and its partner (i + r/2, or the neighbour in the
// interleaved form) become  y_a cos - y_b sin,  y_b cos + y_a sin  with the angle of the token's position; elements
// from r on stay. fp32 arithmetic, one rounding to the type stored.
//
// Bound: memory. A head row is D / 8 lanes of one 16-byte load each; a team of lanes takes kAhead rows at a time, loads
// first. A block takes kTokens tokens and looks their sequence, position and page up once, in shared memory. A few
// tokens (a decoding step) are bound by the latency of one block instead: there a block has one token and the
// grid's second dimension spreads its rows.
#include "kv_launch.h"
#include "mma_sync.cuh"

#include <type_traits>

namespace f2k {

namespace {

constexpr int kBlock = 256;

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
    const SeqView s = seq_view(cu0, cu1, b.lens[seq], b.n_tokens, (long long)b.table_width << p.page_shift);
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

template <class T>
__device__ __forceinline__ void unpack(const uint4& v, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) f[2 * i] = Half16<T>::lo(w[i]), f[2 * i + 1] = Half16<T>::hi(w[i]);
}
template <class T>
__device__ __forceinline__ uint4 packed(const float (&f)[8]) {
    return make_uint4(Half16<T>::pack(f[0], f[1]), Half16<T>::pack(f[2], f[3]), Half16<T>::pack(f[4], f[5]), Half16<T>::pack(f[6], f[7]));
}
// Eight values divided by the head's scale, as e4m3: to nearest even, beyond +-448 saturated, NaN kept.
__device__ __forceinline__ uint2 packed_e4m3(const float (&f)[8], float scale) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        w[i] = __nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(f[2 * i], scale), __fdiv_rn(f[2 * i + 1], scale)), __NV_SATFINITE, __NV_E4M3);
    return make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
}

template <class T, bool kE4m3, int kDim, int kTokens, int kAhead>
__global__ void __launch_bounds__(kBlock)
kv_append_kernel(const __grid_constant__ AppendParams p) {
    constexpr int kLanes = kDim / 8, kTeams = kBlock / kLanes;
    __shared__ Token tokens[kTokens];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int t0 = blockIdx.x * kTokens;
    if (threadIdx.x < kTokens) {
        const int t = t0 + threadIdx.x;
        tokens[threadIdx.x] = t < p.batch.n_tokens ? look_up(p, t) : Token{0, 0, -1};
    }
    __syncthreads();

    const int sub = threadIdx.x % kLanes, team = threadIdx.x / kLanes;
    const uint32_t mates = (kLanes == 32 ? 0xFFFFFFFFu : ((1u << kLanes) - 1u)) << (threadIdx.x & 31 & ~(kLanes - 1));
    const int H = p.n_heads, G = p.n_kv_heads, rows = H + 2 * G;
    const int r8 = p.rot_dim >> 3;                      // lanes that rotate
    const int sets = (rows + kAhead - 1) / kAhead;      // sets of kAhead rows of one token
    for (int item = blockIdx.y * kTeams + team; item < sets * kTokens; item += gridDim.y * kTeams) {
        const int ti = item / sets, row0 = (item - ti * sets) * kAhead;
        const Token tk = tokens[ti];
        if (tk.pos < 0) continue;
        const long long t = t0 + ti;
        const T* src[kAhead];
        uint4 raw[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int row = row0 + u;
            src[u] = row < H ? static_cast<const T*>(p.q) + t * p.q_stride + row * kDim
                   : row < H + G ? static_cast<const T*>(p.k) + t * p.k_stride + (row - H) * kDim
                                 : static_cast<const T*>(p.v) + t * p.v_stride + (row - H - G) * kDim;
            if (row < rows) raw[u] = reinterpret_cast<const uint4*>(src[u])[sub];
        }
        float cs[8], sn[8];
        if (row0 < H + G && sub < r8) {
            const int half = p.rot_dim >> 1;
            if (p.interleaved) {
                const float4 c = reinterpret_cast<const float4*>(p.cos_tab + (long long)tk.pos * half)[sub];
                const float4 s = reinterpret_cast<const float4*>(p.sin_tab + (long long)tk.pos * half)[sub];
                cs[0] = c.x, cs[1] = c.y, cs[2] = c.z, cs[3] = c.w;
                sn[0] = s.x, sn[1] = s.y, sn[2] = s.z, sn[3] = s.w;
            } else {
                const int at = 2 * (2 * sub < r8 ? sub : sub - (r8 >> 1));
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float4 c = reinterpret_cast<const float4*>(p.cos_tab + (long long)tk.pos * half)[at + i];
                    const float4 s = reinterpret_cast<const float4*>(p.sin_tab + (long long)tk.pos * half)[at + i];
                    cs[4 * i] = c.x, cs[4 * i + 1] = c.y, cs[4 * i + 2] = c.z, cs[4 * i + 3] = c.w;
                    sn[4 * i] = s.x, sn[4 * i + 1] = s.y, sn[4 * i + 2] = s.z, sn[4 * i + 3] = s.w;
                }
            }
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int row = row0 + u;
            if (row >= rows) break;                      // the same for the whole team
            const bool is_q = row < H, is_v = row >= H + G;
            const int head = is_q ? row : is_v ? row - H - G : row - H;
            float x[8];
            uint4 y16 = raw[u];
            if (!is_v || kE4m3) unpack<T>(raw[u], x);
            if (!is_v) {
                const void* gamma = is_q ? p.gamma_q : p.gamma_k;
                if (gamma != nullptr) {
                    float g[8], ss = 0.f;
                    unpack<T>(static_cast<const uint4*>(gamma)[sub], g);
#pragma unroll
                    for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
                    for (int d = kLanes / 2; d > 0; d >>= 1) ss += __shfl_xor_sync(mates, ss, d);
                    const float rrms = rsqrtf(ss * (1.0f / kDim) + p.eps);
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[i] = x[i] * rrms * g[i];
                }
                if (p.rot_dim > 0) {
                    if (p.interleaved) {
                        if (sub < r8) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const float a = x[2 * i], b = x[2 * i + 1];
                                x[2 * i] = fmaf(a, cs[i], -(b * sn[i]));
                                x[2 * i + 1] = fmaf(b, cs[i], a * sn[i]);
                            }
                        }
                    } else {
                        const bool first = 2 * sub < r8;
                        const int mate = sub >= r8 ? sub : first ? sub + (r8 >> 1) : sub - (r8 >> 1);
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float other = __shfl_sync(mates, x[i], mate, kLanes);
                            if (sub < r8) x[i] = fmaf(x[i], cs[i], first ? -(other * sn[i]) : other * sn[i]);
                        }
                    }
                }
                if (gamma != nullptr || p.rot_dim > 0) y16 = packed<T>(x);
            }
            if (is_q) {
                reinterpret_cast<uint4*>(static_cast<T*>(p.q_out) + t * p.qo_stride + head * kDim)[sub] = y16;
                continue;
            }
            const long long at = (is_v ? tk.v_at + head * p.vp_head : tk.k_at + head * p.kp_head) + sub * 8;
            void* base = is_v ? p.v_pages : p.k_pages;
            if constexpr (kE4m3) {
                const float* scale = is_v ? p.v_scale : p.k_scale;
                *reinterpret_cast<uint2*>(static_cast<uint8_t*>(base) + at) = packed_e4m3(x, scale ? scale[head] : 1.0f);
            } else {
                *reinterpret_cast<uint4*>(static_cast<T*>(base) + at) = y16;
            }
        }
    }
}

template <class T, bool kE4m3, int kDim>
cudaError_t launch(const AppendParams& p, cudaStream_t stream) {
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return e;
    constexpr int kTeams = kBlock / (kDim / 8), kMany = 8;
    const int rows = p.n_heads + 2 * p.n_kv_heads, n = p.batch.n_tokens;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(kBlock);
    cfg.stream = stream;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    // While every row can have a team of its own on the GPU at once, it gets one.
    if ((long long)n * ((rows + kTeams - 1) / kTeams) <= 4ll * sms) {
        cfg.gridDim = dim3(n, (rows + kTeams - 1) / kTeams);
        return cudaLaunchKernelEx(&cfg, kv_append_kernel<T, kE4m3, kDim, 1, 1>, p);
    }
    cfg.gridDim = dim3((n + kMany - 1) / kMany);
    return cudaLaunchKernelEx(&cfg, kv_append_kernel<T, kE4m3, kDim, kMany, 4>, p);
}

}  // namespace

cudaError_t kv_append_launch(const AppendParams& p, PagedType type, PagedType cache, int head_dim, cudaStream_t stream) {
    auto by_dim = [&](auto t, auto e) {
        using T = decltype(t);
        return head_dim == 64 ? launch<T, decltype(e)::value, 64>(p, stream) : launch<T, decltype(e)::value, 128>(p, stream);
    };
    auto by_cache = [&](auto t) { return cache == kE4m3 ? by_dim(t, std::true_type{}) : by_dim(t, std::false_type{}); };
    return type == kBf16 ? by_cache(__nv_bfloat16{}) : by_cache(__half{});
}

}  // namespace f2k
