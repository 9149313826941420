// The paged key/value cache behind the C ABI (include/f2k_attn.h): argument checks, tensor maps, workspace, launches.
#include "f2k_attn.h"

#include "../attn_params.h"
#include "../handle_device.h"
#include "kv_launch.h"
#include "token_work.h"

#include <cmath>
#include <cstdio>
#include <cstring>
#include <new>
#include <string>

using namespace f2k;

struct f2k_kv {
    f2k_kv_config cfg{};
    float         scale = 0.f;
    bool          valid = false;
    std::string   err;
    int           device = -1, sms = 0, page_shift = 0;
    int*          d_status = nullptr;
    long long     wait_clk = 0;
    CUtensorMap   token_k, token_v, prompt_k, prompt_v;
};

namespace {

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                   const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                   CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

int fail(f2k_kv* h, int code, std::string msg) {
    h->err = std::move(msg);
    return code;
}
int fail_cuda(f2k_kv* h, const char* what, cudaError_t e) { return fail(h, F2K_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e)); }

bool misaligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }

// A cache array as [pages][kv heads][128-byte pieces of a row][tokens of a page][piece]: the rows of a box stand one
// behind the other, 128 (or 64) bytes each, which is how the kernels read a piece of head_dim. A box has `rows` tokens and
// `pieces` pieces (0: all).
int encode_pages(f2k_kv* h, CUtensorMap* map, void* base, long long page, long long head, long long tok, int rows, int pieces) {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    const cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q);
    if (e != cudaSuccess || q != cudaDriverEntryPointSuccess || fn == nullptr) return fail_cuda(h, "cuTensorMapEncodeTiled", e);
    const f2k_kv_config& c = h->cfg;
    const cuuint64_t es = c.cache_type == F2K_E4M3 ? 1 : 2, row = c.head_dim * es, piece = row < 128 ? row : 128;
    const cuuint64_t dims[5] = {piece / es, (cuuint64_t)c.page_size, row / piece, (cuuint64_t)c.n_kv_heads, (cuuint64_t)c.n_pages};
    const cuuint64_t strides[4] = {tok * es, piece, head * es, page * es};
    const cuuint32_t box[5] = {(cuuint32_t)(piece / es), (cuuint32_t)rows, (cuuint32_t)(pieces ? pieces : row / piece), 1, 1}, step[5] = {1, 1, 1, 1, 1};
    const CUresult r = reinterpret_cast<EncodeTiledFn>(fn)(
        map, es == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 5, base, dims, strides, box, step,
        CU_TENSOR_MAP_INTERLEAVE_NONE, piece == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r == CUDA_SUCCESS) return F2K_OK;
    char buf[96];
    std::snprintf(buf, sizeof buf, "cuTensorMapEncodeTiled failed for the pages (CUresult %d)", (int)r);
    return fail(h, F2K_ERR_CUDA, buf);
}

// What append and attend ask of a batch. Returns the batch as the kernels take it.
int check_batch(f2k_kv* h, const f2k_kv_batch* b, PagedBatch& out) {
    if (!b) return fail(h, F2K_ERR_INVALID, "null batch");
    if (b->n_seqs < 0 || b->n_tokens < 0) return fail(h, F2K_ERR_INVALID, "negative number of sequences or tokens");
    if (b->n_seqs == 0 || b->n_tokens == 0) return F2K_OK;
    if (b->max_new <= 0 || b->table_width <= 0) return fail(h, F2K_ERR_INVALID, "max_new and table_width must be positive");
    const long long stride = b->table_stride ? b->table_stride : b->table_width;
    if (stride < b->table_width && b->n_seqs > 1) return fail(h, F2K_ERR_INVALID, "table_stride is below table_width");
    if (((long long)b->table_width << h->page_shift) > 0x7fffff00ll) return fail(h, F2K_ERR_INVALID, "a table row holds more than 2^31 - 256 tokens");
    if (!b->kv_lens || !b->page_table) return fail(h, F2K_ERR_INVALID, "null length or page table pointer");
    if (misaligned(b->kv_lens, 4) || misaligned(b->page_table, 4) || misaligned(b->cu_seqlens, 4))
        return fail(h, F2K_ERR_INVALID, "lengths and page table must be 4-byte aligned");
    if (!b->cu_seqlens && b->n_tokens < b->n_seqs) return fail(h, F2K_ERR_INVALID, "fewer tokens than sequences without cu_seqlens");
    out = PagedBatch{b->cu_seqlens, b->kv_lens, b->page_table, stride, b->table_width, b->n_seqs, b->n_tokens, b->max_new};
    return F2K_OK;
}

int check_ready(f2k_kv* h) {
    if (!h || !h->valid) return F2K_ERR_INVALID;
    return check_current_device(h->device, h->err);
}

// A tensor's token stride: dense where it is 0.
int take_stride(f2k_kv* h, long long given, int heads, const char* name, long long& out) {
    const long long dense = (long long)heads * h->cfg.head_dim;
    out = given ? given : dense;
    if (out < dense || out % 8 != 0) return fail(h, F2K_ERR_INVALID, std::string(name) + " stride must be a multiple of 8 and hold a token's heads");
    return F2K_OK;
}

// A call in place reads and writes a row at the same time: with other strides rows would be written before they are read.
int check_in_place(f2k_kv* h, const void* in, long long in_stride, const void* out, long long out_stride, int n_tokens, const char* names) {
    if (in != out || in_stride == out_stride || n_tokens == 1) return F2K_OK;
    return fail(h, F2K_ERR_INVALID, std::string(names) + " are the same memory with different strides");
}

struct Workspace {
    size_t join, ml, o, bytes;
};
Workspace workspace_of(const f2k_kv* h, int rows) {
    auto up = [](size_t x) { return (x + 255) / 256 * 256; };
    Workspace w;
    const size_t ctas = token_ctas(h->sms), shares = 2 * ctas;
    w.join = 0;
    w.ml = up(sizeof(JoinJob) * ctas);
    w.o = w.ml + up(shares * rows * sizeof(float2));
    w.bytes = w.o + shares * rows * h->cfg.head_dim * sizeof(float);
    return w;
}
int group_of(const f2k_kv* h) { return h->cfg.n_heads / h->cfg.n_kv_heads; }
// Which kernel attends. Up to 64 query rows a sequence and key head the token kernel can take all of them at once, split over
// the keys; its time grows with the rows from 16 on (head_dim 128; 32 with 64). The prompt kernel's does not, but it has one
// CTA a sequence and key head then. 16-bit caches, us, token kernel / prompt kernel: 16 sequences of about 27000 keys, 8 key
// heads, 16 rows 278 / 303, 32 rows 488 / 307, 64 rows 1032 / 323; of 16000 keys, 64 rows: 2 sequences 96 / 133, 4 sequences
// 171 / 134; 32 rows: 4 sequences 87 / 133, 8 sequences 159 / 135. head_dim 64, 192 CTAs: 32 rows 39 / 41, 64 rows 56 / 41.
// e4m3, where the prompt kernel is bound by turning bytes into fp16: 32 rows, 16 sequences of about 27000 keys 348 / 555;
// 36 and 64 rows alike, of 16000 keys: 8 sequences 224 / 279, 10 sequences 275 / 279, 16 sequences 430 / 282; head_dim 64,
// 8 sequences 126 / 152, of 1000 keys 24 / 17.
// More than 64 rows always go to the prompt kernel, few sequences behind many keys too, where its CTAs leave most of the GPU idle: one
// sequence of 32000 keys, 8 key heads, 64 rows 96 us here, 68 rows 263 there; one key head, 64 rows 48, 80 rows 250.
bool takes_prompt_kernel(const f2k_kv* h, const f2k_kv_batch* b) {
    const long long rows = (long long)b->max_new * group_of(h);
    if (b->max_new == 1 || rows <= 16) return false;
    if (rows > 64) return true;
    const long long ctas = (long long)b->n_seqs * h->cfg.n_kv_heads;
    if (h->cfg.cache_type == F2K_E4M3) return rows > 32 && ctas >= 80;
    return rows * h->cfg.head_dim > 2048 && rows * ctas >= 2048;
}
int rows_of(const f2k_kv* h, const f2k_kv_batch* b) { return token_rows((long long)b->max_new * group_of(h)); }

}  // namespace

extern "C" {

int f2k_kv_create(const f2k_kv_config* cfg, f2k_kv** out) {
    if (!out) return F2K_ERR_INVALID;
    *out = nullptr;
    f2k_kv* h = new (std::nothrow) f2k_kv();
    if (!h) return F2K_ERR_CUDA;
    *out = h;
    if (!cfg) return fail(h, F2K_ERR_INVALID, "null config");
    f2k_kv_config& c = h->cfg;
    c = *cfg;
    if (c.n_heads <= 0 || c.n_kv_heads <= 0 || c.head_dim <= 0 || c.page_size <= 0 || c.n_pages <= 0)
        return fail(h, F2K_ERR_INVALID, "PagedKV: zero/negative dim");
    if (c.n_heads % c.n_kv_heads != 0) return fail(h, F2K_ERR_INVALID, "n_heads must be a multiple of n_kv_heads");
    if (group_of(h) > 128) return fail(h, F2K_ERR_UNSUPPORTED, "more than 128 query heads per key head");
    if (c.n_heads > 65535) return fail(h, F2K_ERR_UNSUPPORTED, "more than 65535 heads");
    if (c.head_dim != 64 && c.head_dim != 128) return fail(h, F2K_ERR_UNSUPPORTED, "head_dim must be 64 or 128");
    for (h->page_shift = 4; h->page_shift < 8 && (1 << h->page_shift) != c.page_size;) ++h->page_shift;
    if ((1 << h->page_shift) != c.page_size) return fail(h, F2K_ERR_UNSUPPORTED, "page_size must be 16, 32, 64, 128 or 256");
    if (c.type != F2K_BF16 && c.type != F2K_F16) return fail(h, F2K_ERR_UNSUPPORTED, "type must be bf16 or f16");
    if (c.cache_type != c.type && c.cache_type != F2K_E4M3) return fail(h, F2K_ERR_UNSUPPORTED, "the cache's type must be that of K and V, or e4m3");
    if (c.cache_type != F2K_E4M3 && (c.k_scale || c.v_scale)) return fail(h, F2K_ERR_INVALID, "scales belong to an e4m3 cache");
    if (c.rot_dim < 0 || c.rot_dim > c.head_dim || c.rot_dim % 16 != 0) return fail(h, F2K_ERR_INVALID, "rot_dim must be a multiple of 16 up to head_dim");
    if (c.window < 0) return fail(h, F2K_ERR_INVALID, "window must not be negative");
    if (std::isnan(c.scale) || std::isinf(c.scale)) return fail(h, F2K_ERR_INVALID, "scale must be finite");
    if (!c.k_pages || !c.v_pages) return fail(h, F2K_ERR_INVALID, "null page pointer");
    if (misaligned(c.k_pages, 16) || misaligned(c.v_pages, 16)) return fail(h, F2K_ERR_INVALID, "pages must be 16-byte aligned");
    if (misaligned(c.k_scale, 4) || misaligned(c.v_scale, 4)) return fail(h, F2K_ERR_INVALID, "scales must be 4-byte aligned");
    auto strides = [&](long long& page, long long& head, long long& tok) {
        if (page == 0 && head == 0 && tok == 0) {
            tok = c.head_dim;
            head = tok * c.page_size;
            page = head * c.n_kv_heads;
        }
        const long long unit = c.cache_type == F2K_E4M3 ? 16 : 8, most = 1ll << 39;
        for (long long s : {page, head, tok})
            if (s <= 0 || s % unit != 0 || s >= most) return false;
        return tok >= c.head_dim && (c.n_kv_heads == 1 || head >= c.head_dim) && (c.n_pages == 1 || page >= c.head_dim);
    };
    if (!strides(c.k_page_stride, c.k_head_stride, c.k_token_stride) || !strides(c.v_page_stride, c.v_head_stride, c.v_token_stride))
        return fail(h, F2K_ERR_INVALID, "page, head and token strides must be positive multiples of 16 bytes and hold a row");
    h->scale = c.scale > 0.f ? c.scale : 1.0f / std::sqrt((float)c.head_dim);

    cudaError_t e = cudaGetDevice(&h->device);
    if (e != cudaSuccess) return fail_cuda(h, "cudaGetDevice", e);
    int major = 0;
    e = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, h->device);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&h->sms, cudaDevAttrMultiProcessorCount, h->device);
    if (e != cudaSuccess) return fail_cuda(h, "cudaDeviceGetAttribute", e);
    if (major != 10) return fail(h, F2K_ERR_UNSUPPORTED, "this library contains sm_100a code only (needs a B200-class GPU)");
    // The pages are read and written for as long as the handle lives: they have to be where its kernels run.
    for (const void* x : {(const void*)c.k_pages, (const void*)c.v_pages, (const void*)c.k_scale, (const void*)c.v_scale}) {
        cudaPointerAttributes a{};
        if (x == nullptr) continue;
        e = cudaPointerGetAttributes(&a, x);
        if (e != cudaSuccess) return fail_cuda(h, "cudaPointerGetAttributes", e);
        if (a.type != cudaMemoryTypeManaged && (a.type != cudaMemoryTypeDevice || a.device != h->device))
            return fail(h, F2K_ERR_INVALID, "pages and scales must lie in the current device's memory");
    }
    e = paged_token_prepare((PagedType)c.type, (PagedType)c.cache_type, c.head_dim);
    if (e == cudaSuccess) e = kv_append_prepare((PagedType)c.type, (PagedType)c.cache_type, c.head_dim, c.interleaved != 0);
    if (e == cudaSuccess) e = paged_prompt_prepare((PagedType)c.type, (PagedType)c.cache_type, c.head_dim);
    if (e != cudaSuccess) return fail_cuda(h, "kernel load", e);
    const int unit = token_unit_keys(c.head_dim * (c.cache_type == F2K_E4M3 ? 1 : 2));
    const int rows = unit < c.page_size ? unit : c.page_size;
    int rc = encode_pages(h, &h->token_k, c.k_pages, c.k_page_stride, c.k_head_stride, c.k_token_stride, rows, 0);
    if (rc == F2K_OK) rc = encode_pages(h, &h->token_v, c.v_pages, c.v_page_stride, c.v_head_stride, c.v_token_stride, rows, 0);
    if (rc == F2K_OK) {
        const int most = c.page_size < kPromptTile ? c.page_size : kPromptTile;
        rc = encode_pages(h, &h->prompt_k, c.k_pages, c.k_page_stride, c.k_head_stride, c.k_token_stride, most, 1);
        if (rc == F2K_OK) rc = encode_pages(h, &h->prompt_v, c.v_pages, c.v_page_stride, c.v_head_stride, c.v_token_stride, most, 1);
    }
    if (rc != F2K_OK) return rc;
    e = cudaMalloc(reinterpret_cast<void**>(&h->d_status), kStatusBytes);
    if (e != cudaSuccess) return fail_cuda(h, "cudaMalloc(status)", e);
    e = cudaMemset(h->d_status, 0, kStatusBytes);
    if (e != cudaSuccess) return fail_cuda(h, "cudaMemset(status)", e);
    h->valid = true;
    return F2K_OK;
}

void f2k_kv_destroy(f2k_kv* h) {
    if (!h) return;
    if (h->d_status) cudaFree(h->d_status);
    delete h;
}

const char* f2k_kv_last_error(const f2k_kv* h) { return h ? h->err.c_str() : "no handle"; }

int f2k_kv_append(f2k_kv* h, const f2k_kv_batch* batch, const f2k_kv_append_args* args, void* stream) {
    if (const int rc = check_ready(h)) return rc;
    const f2k_kv_config& c = h->cfg;
    AppendParams p{};
    if (const int rc = check_batch(h, batch, p.batch)) return rc;
    if (!args) return fail(h, F2K_ERR_INVALID, "null arguments");
    const f2k_kv_append_args& a = *args;
    if (p.batch.n_seqs == 0) return F2K_OK;
    if (!a.q || !a.k || !a.v || !a.q_out) return fail(h, F2K_ERR_INVALID, "null tensor pointer");
    if (!a.gamma_q != !a.gamma_k) return fail(h, F2K_ERR_INVALID, "one gain without the other");
    if (c.rot_dim > 0 && (!a.cos_table || !a.sin_table || a.n_positions <= 0)) return fail(h, F2K_ERR_INVALID, "null rotation table");
    const void* pointers[8] = {a.q, a.k, a.v, a.q_out, a.gamma_q, a.gamma_k, a.cos_table, a.sin_table};
    for (const void* x : pointers)
        if (misaligned(x, 16)) return fail(h, F2K_ERR_INVALID, "tensors, gains and tables must be 16-byte aligned");
    if (const int rc = take_stride(h, a.q_stride, c.n_heads, "q", p.q_stride)) return rc;
    if (const int rc = take_stride(h, a.k_stride, c.n_kv_heads, "k", p.k_stride)) return rc;
    if (const int rc = take_stride(h, a.v_stride, c.n_kv_heads, "v", p.v_stride)) return rc;
    if (const int rc = take_stride(h, a.q_out_stride, c.n_heads, "q_out", p.qo_stride)) return rc;
    if (const int rc = check_in_place(h, a.q, p.q_stride, a.q_out, p.qo_stride, p.batch.n_tokens, "q and q_out")) return rc;
    p.q = a.q, p.k = a.k, p.v = a.v, p.gamma_q = a.gamma_q, p.gamma_k = a.gamma_k, p.cos_tab = a.cos_table, p.sin_tab = a.sin_table;
    p.k_scale = c.k_scale, p.v_scale = c.v_scale, p.q_out = a.q_out, p.k_pages = c.k_pages, p.v_pages = c.v_pages;
    p.kp_page = c.k_page_stride, p.kp_head = c.k_head_stride, p.kp_tok = c.k_token_stride;
    p.vp_page = c.v_page_stride, p.vp_head = c.v_head_stride, p.vp_tok = c.v_token_stride;
    p.n_heads = c.n_heads, p.n_kv_heads = c.n_kv_heads, p.page_shift = h->page_shift, p.n_pages = c.n_pages;
    p.n_positions = a.n_positions, p.rot_dim = c.rot_dim, p.interleaved = c.interleaved, p.eps = a.eps, p.status = h->d_status;
    const cudaError_t e = kv_append_launch(p, (PagedType)c.type, (PagedType)c.cache_type, c.head_dim, h->sms, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? F2K_OK : fail_cuda(h, "append launch", e);
}

size_t f2k_kv_workspace_bytes(const f2k_kv* h, const f2k_kv_batch* batch) {
    if (!h || !h->valid || !batch || batch->max_new <= 0 || takes_prompt_kernel(h, batch)) return 0;
    return workspace_of(h, rows_of(h, batch)).bytes;
}

int f2k_kv_attend(f2k_kv* h, const f2k_kv_batch* batch, const f2k_kv_attend_args* args, void* stream) {
    if (const int rc = check_ready(h)) return rc;
    const f2k_kv_config& c = h->cfg;
    AttendParams p{};
    if (const int rc = check_batch(h, batch, p.batch)) return rc;
    if (!args) return fail(h, F2K_ERR_INVALID, "null arguments");
    const f2k_kv_attend_args& a = *args;
    if (p.batch.n_seqs == 0) return F2K_OK;
    if (!a.q || !a.o) return fail(h, F2K_ERR_INVALID, "null tensor pointer");
    if (misaligned(a.q, 16) || misaligned(a.o, 16)) return fail(h, F2K_ERR_INVALID, "q and o must be 16-byte aligned");
    if (misaligned(a.lse, 4)) return fail(h, F2K_ERR_INVALID, "lse must be 4-byte aligned");
    if (const int rc = take_stride(h, a.q_stride, c.n_heads, "q", p.q_stride)) return rc;
    if (const int rc = take_stride(h, a.o_stride, c.n_heads, "o", p.o_stride)) return rc;
    if (const int rc = check_in_place(h, a.q, p.q_stride, a.o, p.o_stride, p.batch.n_tokens, "q and o")) return rc;
    p.q = a.q, p.o = a.o, p.lse = a.lse, p.k_scale = c.k_scale, p.v_scale = c.v_scale;
    p.n_heads = c.n_heads, p.n_kv_heads = c.n_kv_heads, p.group = group_of(h), p.page_shift = h->page_shift, p.n_pages = c.n_pages;
    p.window = c.window, p.scale_log2 = h->scale * 1.4426950408889634f, p.status = h->d_status;
    p.wait_limit_clk = h->wait_clk > 0 ? h->wait_clk : kDefaultWaitClk;

    if (takes_prompt_kernel(h, batch)) {
        p.tm_k = h->prompt_k;
        p.tm_v = h->prompt_v;
        const cudaError_t e = paged_prompt_launch(p, (PagedType)c.type, (PagedType)c.cache_type, c.head_dim, batch->max_new, h->sms, static_cast<cudaStream_t>(stream));
        return e == cudaSuccess ? F2K_OK : fail_cuda(h, "attention launch", e);
    }
    const int rows = rows_of(h, batch);
    const Workspace ws = workspace_of(h, rows);
    if (!a.workspace || a.workspace_bytes < ws.bytes) return fail(h, F2K_ERR_WORKSPACE, "workspace smaller than f2k_kv_workspace_bytes");
    if (misaligned(a.workspace, 16)) return fail(h, F2K_ERR_INVALID, "workspace must be 16-byte aligned");
    // The kernel counts units in 32 bits.
    const int unit = token_unit_keys(c.head_dim * (c.cache_type == F2K_E4M3 ? 1 : 2));
    const long long keys = (long long)batch->table_width << h->page_shift;
    const double tiles = (double)batch->n_tokens * p.group / rows + batch->n_seqs;
    if (tiles * c.n_kv_heads * (double)(keys / unit + 1 + kWorkCost) >= (double)kMostPlaces)
        return fail(h, F2K_ERR_UNSUPPORTED, "the batch could hold 2^32 pieces of work: make two calls of it");
    uint8_t* w = static_cast<uint8_t*>(a.workspace);
    p.ws_join = reinterpret_cast<JoinJob*>(w + ws.join);
    p.ws_ml = reinterpret_cast<float2*>(w + ws.ml);
    p.ws_o = reinterpret_cast<float*>(w + ws.o);
    p.n_ctas = token_ctas(h->sms);
    p.tm_k = h->token_k;
    p.tm_v = h->token_v;
    const long long used = (long long)batch->max_new * p.group;
    const cudaError_t e = paged_token_launch(p, (PagedType)c.type, (PagedType)c.cache_type, c.head_dim, rows,
                                             used < rows ? (int)used : rows, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? F2K_OK : fail_cuda(h, "attention launch", e);
}

int f2k_kv_device_status(f2k_kv* h, int* status_out) {
    if (!h || !h->valid) return F2K_ERR_INVALID;
    int st = 0;
    const OnDevice here(h->device);
    if (here.error != cudaSuccess) return fail_cuda(h, "cudaSetDevice", here.error);
    cudaError_t e = cudaDeviceSynchronize();
    if (e == cudaSuccess) e = cudaMemcpy(&st, h->d_status, sizeof st, cudaMemcpyDeviceToHost);
    if (e == cudaSuccess && st != 0) e = cudaMemset(h->d_status, 0, sizeof st);
    if (e != cudaSuccess) return fail_cuda(h, "status", e);
    if (status_out) *status_out = st;
    if (st == 0) return F2K_OK;
    std::string msg;
    if (st & kStatusWaitExpired) msg += "a bounded wait inside a kernel expired; ";
    if (st & kStatusBadPage) msg += "a page number outside the cache; ";
    if (st & kStatusBadLength) msg += "lengths that do not fit the call or the page table; ";
    if (st & kStatusBadPosition) msg += "a position behind the rotation tables; ";
    return fail(h, F2K_ERR_DEVICE, msg.substr(0, msg.size() - 2));
}

int f2k_kv_set_wait_limits(f2k_kv* h, long long in_cta_clk) {
    if (!h || !h->valid) return F2K_ERR_INVALID;
    if (in_cta_clk < 0) return fail(h, F2K_ERR_INVALID, "wait limits must not be negative");
    h->wait_clk = in_cta_clk;
    return F2K_OK;
}

}  // extern "C"
