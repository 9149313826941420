"""What the paged cache refuses, on the CPU: the C entry points with a fake CUDA runtime (nothing that is refused reaches a
launch, and a handle's calls are refused while another device is current), and the Python mirror's checks of tensors."""
import ctypes as C
import subprocess
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parent.parent
CSRC = ROOT / "f2k_cuda_b200" / "csrc"
CUDA = Path("/usr/local/cuda/include")

PROGRAM = r"""
#include "f2k_attn.h"
#include "kv/kv_launch.h"
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <cstring>
static int current = 0, work = 0, synchronised = -1, status_word = 0;
static CUresult fake_encode(CUtensorMap*, CUtensorMapDataType, cuuint32_t rank, void*, const cuuint64_t* dims, const cuuint64_t* strides,
                            const cuuint32_t* box, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle swizzle, CUtensorMapL2promotion,
                            CUtensorMapFloatOOBfill) {
    // what the driver would refuse, and what the kernels count on: a box's rows are 64 or 128 bytes and as wide as its swizzle
    for (unsigned i = 0; i + 1 < rank; ++i) if (strides[i] % 16 || strides[i] >= 1ull << 40) return CUDA_ERROR_INVALID_VALUE;
    for (unsigned i = 0; i < rank; ++i) if (box[i] == 0 || box[i] > 256 || dims[i] == 0) return CUDA_ERROR_INVALID_VALUE;
    return swizzle == CU_TENSOR_MAP_SWIZZLE_128B || swizzle == CU_TENSOR_MAP_SWIZZLE_64B ? CUDA_SUCCESS : CUDA_ERROR_INVALID_VALUE;
}
extern "C" {
cudaError_t cudaGetDevice(int* d) { *d = current; return cudaSuccess; }
cudaError_t cudaSetDevice(int d) { current = d; return cudaSuccess; }
cudaError_t cudaDeviceGetAttribute(int* v, cudaDeviceAttr a, int) { *v = a == cudaDevAttrComputeCapabilityMajor ? 10 : 148; return cudaSuccess; }
cudaError_t cudaDeviceSynchronize() { synchronised = current; return cudaSuccess; }
cudaError_t cudaMalloc(void** p, size_t n) { *p = std::calloc(1, n); return cudaSuccess; }
cudaError_t cudaFree(void* p) { std::free(p); return cudaSuccess; }
cudaError_t cudaMemset(void* p, int v, size_t n) { std::memset(p, v, n); return cudaSuccess; }
cudaError_t cudaMemcpy(void* d, const void* s, size_t n, cudaMemcpyKind) { std::memcpy(d, s, n); return cudaSuccess; }
static int memory_type = cudaMemoryTypeDevice, memory_device = -1;      // -1: the current one
cudaError_t cudaPointerGetAttributes(cudaPointerAttributes* a, const void*) {
    a->type = (cudaMemoryType)memory_type;
    a->device = memory_device < 0 ? current : memory_device;
    return cudaSuccess;
}
const char* cudaGetErrorString(cudaError_t) { return "fake"; }
cudaError_t cudaGetDriverEntryPoint(const char*, void** fn, unsigned long long, cudaDriverEntryPointQueryResult* q) {
    *fn = reinterpret_cast<void*>(fake_encode);
    *q = cudaDriverEntryPointSuccess;
    return cudaSuccess;
}
}
static int launched_kernel = 0, launched_rows = 0;       // 1 append, 2 token, 3 prompt
static int* last_status;
namespace f2k {
cudaError_t kv_append_prepare(PagedType, PagedType, int, bool) { return cudaSuccess; }
cudaError_t kv_append_launch(const AppendParams& p, PagedType, PagedType, int, int, cudaStream_t) { ++work; launched_kernel = 1; last_status = p.status; return cudaSuccess; }
int token_rows(long long rows) { return rows <= 8 ? 8 : rows <= 16 ? 16 : rows <= 32 ? 32 : 64; }
int token_ctas(int sms) { return 2 * sms; }
cudaError_t paged_token_prepare(PagedType, PagedType, int) { return cudaSuccess; }
cudaError_t paged_token_launch(const AttendParams& p, PagedType, PagedType, int, int rows, int used, cudaStream_t) {
    if (used > rows) std::exit(9);
    ++work; launched_kernel = 2; launched_rows = rows; last_status = p.status; return cudaSuccess;
}
cudaError_t paged_prompt_prepare(PagedType, PagedType, int) { return cudaSuccess; }
cudaError_t paged_prompt_launch(const AttendParams& p, PagedType, PagedType, int, int, int, cudaStream_t) { ++work; launched_kernel = 3; last_status = p.status; return cudaSuccess; }
}
alignas(256) static unsigned char mem[1 << 12];
static float* fl = reinterpret_cast<float*>(mem);
static f2k_kv_config good() {
    f2k_kv_config c{};
    c.n_heads = 8; c.n_kv_heads = 2; c.head_dim = 128; c.page_size = 16; c.n_pages = 10; c.type = F2K_BF16; c.cache_type = F2K_BF16; c.rot_dim = 128;
    c.k_pages = c.v_pages = mem;
    return c;
}
static int bad = 0;
template <class F>
static void create(const char* what, int want, F change) {
    f2k_kv_config c = good();
    change(c);
    f2k_kv* h = nullptr;
    const int rc = f2k_kv_create(&c, &h);
    const char* msg = f2k_kv_last_error(h);
    if (rc != want || !h || (want && !*msg)) { std::printf("create, %s: %d '%s'\n", what, rc, msg); ++bad; }
    const f2k_kv_batch b{1, 1, 1, 1, 0, nullptr, reinterpret_cast<int32_t*>(mem), reinterpret_cast<int32_t*>(mem)};
    f2k_kv_append_args a{mem, mem, mem, nullptr, nullptr, fl, fl, mem, 0, 0, 0, 0, 8, 1e-6f};
    work = 0;
    if (want && (f2k_kv_append(h, &b, &a, nullptr) == F2K_OK || work)) { std::printf("%s: a failed handle appends\n", what); ++bad; }
    f2k_kv_destroy(h);
}
int main() {
    create("good", F2K_OK, [](auto&) {});
    create("no heads", F2K_ERR_INVALID, [](auto& c) { c.n_heads = 0; });
    create("negative pages", F2K_ERR_INVALID, [](auto& c) { c.n_pages = -1; });
    create("heads no multiple", F2K_ERR_INVALID, [](auto& c) { c.n_heads = 7; });
    create("129 heads a key head", F2K_ERR_UNSUPPORTED, [](auto& c) { c.n_heads = 258; });
    create("128 heads a key head", F2K_OK, [](auto& c) { c.n_heads = 256; });
    for (int d : {32, 96, 256}) create("head_dim", F2K_ERR_UNSUPPORTED, [&](auto& c) { c.head_dim = d; c.rot_dim = 0; });
    create("head_dim 64", F2K_OK, [](auto& c) { c.head_dim = 64; c.rot_dim = 64; });
    for (int s : {1, 8, 24, 48, 512}) create("page size", F2K_ERR_UNSUPPORTED, [&](auto& c) { c.page_size = s; });
    for (int s : {16, 32, 64, 128, 256}) create("page size", F2K_OK, [&](auto& c) { c.page_size = s; });
    create("e4m3 queries", F2K_ERR_UNSUPPORTED, [](auto& c) { c.type = c.cache_type = F2K_E4M3; });
    create("no such type", F2K_ERR_UNSUPPORTED, [](auto& c) { c.type = 7; });
    create("another cache", F2K_ERR_UNSUPPORTED, [](auto& c) { c.cache_type = F2K_F16; });
    create("e4m3 cache", F2K_OK, [](auto& c) { c.cache_type = F2K_E4M3; c.k_scale = c.v_scale = fl; });
    create("scales of a bf16 cache", F2K_ERR_INVALID, [](auto& c) { c.k_scale = fl; });
    for (int r : {-16, 8, 72, 144}) create("rot_dim", F2K_ERR_INVALID, [&](auto& c) { c.rot_dim = r; });
    create("window", F2K_ERR_INVALID, [](auto& c) { c.window = -1; });
    create("scale", F2K_ERR_INVALID, [](auto& c) { c.scale = NAN; });
    create("no pages", F2K_ERR_INVALID, [](auto& c) { c.v_pages = nullptr; });
    create("misaligned pages", F2K_ERR_INVALID, [](auto& c) { c.k_pages = mem + 8; });
    create("one stride", F2K_ERR_INVALID, [](auto& c) { c.k_token_stride = 128; });
    create("token stride below a row", F2K_ERR_INVALID, [](auto& c) { c.k_token_stride = 64; c.k_head_stride = c.k_page_stride = 4096; });
    create("odd stride", F2K_ERR_INVALID, [](auto& c) { c.k_token_stride = 132; c.k_head_stride = c.k_page_stride = 4096; });
    create("e4m3 stride of 8", F2K_ERR_INVALID, [](auto& c) { c.cache_type = F2K_E4M3; c.k_token_stride = 136; c.k_head_stride = c.k_page_stride = 4096; });
    create("tokens before heads", F2K_OK, [](auto& c) { c.k_token_stride = 256; c.k_head_stride = 128; c.k_page_stride = 4096; });
    memory_type = cudaMemoryTypeUnregistered;
    create("host memory", F2K_ERR_INVALID, [](auto&) {});
    memory_type = cudaMemoryTypeDevice; memory_device = 3;
    create("another device's memory", F2K_ERR_INVALID, [](auto&) {});
    memory_type = cudaMemoryTypeManaged;
    create("managed memory", F2K_OK, [](auto&) {});
    memory_type = cudaMemoryTypeDevice; memory_device = -1;
    if (f2k_kv_create(nullptr, nullptr) != F2K_ERR_INVALID) { std::printf("null out\n"); ++bad; }

    current = 1;
    f2k_kv_config c = good();
    f2k_kv* h = nullptr;
    if (f2k_kv_create(&c, &h)) { std::printf("create\n"); return 1; }
    int32_t* ip = reinterpret_cast<int32_t*>(mem);
    const f2k_kv_batch b0{3, 5, 2, 4, 0, ip, ip, ip};
    const f2k_kv_append_args a0{mem, mem, mem, nullptr, nullptr, fl, fl, mem, 0, 0, 0, 0, 8, 1e-6f};
    const size_t ws = f2k_kv_workspace_bytes(h, &b0);
    const f2k_kv_attend_args t0{mem, mem, nullptr, 0, 0, mem, ws};
    auto call = [&](const char* what, int want, int kernel, auto change) {
        f2k_kv_batch b = b0; f2k_kv_append_args a = a0; f2k_kv_attend_args t = t0;
        change(b, a, t);
        for (int which = 1; which <= 2; ++which) {
            if (kernel && !(kernel & which)) continue;
            work = 0;
            const int rc = which == 1 ? f2k_kv_append(h, &b, &a, nullptr) : f2k_kv_attend(h, &b, &t, nullptr);
            if (rc != want || (work != 0) != (want == F2K_OK && b.n_seqs && b.n_tokens)) {
                std::printf("%s %s: %d, %d launches '%s'\n", which == 1 ? "append" : "attend", what, rc, work, f2k_kv_last_error(h)); ++bad;
            }
        }
    };
    using B = f2k_kv_batch; using A = f2k_kv_append_args; using T = f2k_kv_attend_args;
    call("good", F2K_OK, 0, [](B&, A&, T&) {});
    call("no sequences", F2K_OK, 0, [](B& b, A&, T&) { b.n_seqs = 0; });
    call("no tokens", F2K_OK, 0, [](B& b, A&, T&) { b.n_tokens = 0; });
    call("negative tokens", F2K_ERR_INVALID, 0, [](B& b, A&, T&) { b.n_tokens = -1; });
    call("max_new 0", F2K_ERR_INVALID, 0, [](B& b, A&, T&) { b.max_new = 0; });
    call("width 0", F2K_ERR_INVALID, 0, [](B& b, A&, T&) { b.table_width = 0; });
    call("stride below width", F2K_ERR_INVALID, 0, [](B& b, A&, T&) { b.table_stride = 3; });
    call("a row of 2^31 tokens", F2K_ERR_INVALID, 0, [](B& b, A&, T&) { b.table_width = 1 << 27; });
    call("no lengths", F2K_ERR_INVALID, 0, [](B& b, A&, T&) { b.kv_lens = nullptr; });
    call("no table", F2K_ERR_INVALID, 0, [](B& b, A&, T&) { b.page_table = nullptr; });
    call("odd lengths", F2K_ERR_INVALID, 0, [&](B& b, A&, T&) { b.kv_lens = reinterpret_cast<int32_t*>(mem + 2); });
    call("more sequences than tokens", F2K_ERR_INVALID, 0, [](B& b, A&, T&) { b.cu_seqlens = nullptr; b.n_tokens = 2; });
    call("one token each", F2K_OK, 0, [](B& b, A&, T&) { b.cu_seqlens = nullptr; b.max_new = 1; });
    call("no q", F2K_ERR_INVALID, 0, [](B&, A& a, T& t) { a.q = nullptr; t.q = nullptr; });
    call("no output", F2K_ERR_INVALID, 0, [](B&, A& a, T& t) { a.q_out = nullptr; t.o = nullptr; });
    call("misaligned q", F2K_ERR_INVALID, 0, [](B&, A& a, T& t) { a.q = mem + 4; t.q = mem + 4; });
    call("stride below the heads", F2K_ERR_INVALID, 0, [](B&, A& a, T& t) { a.q_stride = t.q_stride = 512; });
    call("odd stride", F2K_ERR_INVALID, 0, [](B&, A& a, T& t) { a.q_out_stride = t.o_stride = 1028; });
    call("wide rows", F2K_OK, 0, [](B&, A& a, T& t) { a.q_stride = t.q_stride = a.q_out_stride = t.o_stride = 4096; a.k_stride = a.v_stride = 512; });
    call("k stride", F2K_ERR_INVALID, 1, [](B&, A& a, T&) { a.k_stride = 128; });
    call("one gain", F2K_ERR_INVALID, 1, [](B&, A& a, T&) { a.gamma_q = mem; });
    call("misaligned gain", F2K_ERR_INVALID, 1, [](B&, A& a, T&) { a.gamma_q = mem; a.gamma_k = mem + 2; });
    call("no table of sines", F2K_ERR_INVALID, 1, [](B&, A& a, T&) { a.sin_table = nullptr; });
    call("no positions", F2K_ERR_INVALID, 1, [](B&, A& a, T&) { a.n_positions = 0; });
    call("misaligned table", F2K_ERR_INVALID, 1, [](B&, A& a, T&) { a.cos_table = fl + 1; });
    call("misaligned lse", F2K_ERR_INVALID, 2, [](B&, A&, T& t) { t.lse = reinterpret_cast<float*>(mem + 2); });
    call("no workspace", F2K_ERR_WORKSPACE, 2, [](B&, A&, T& t) { t.workspace = nullptr; });
    call("small workspace", F2K_ERR_WORKSPACE, 2, [](B&, A&, T& t) { t.workspace_bytes -= 1; });
    call("misaligned workspace", F2K_ERR_INVALID, 2, [](B&, A&, T& t) { t.workspace = mem + 8; });
    call("a prompt needs none", F2K_OK, 2, [](B& b, A&, T& t) { b.max_new = 100; t.workspace = nullptr; t.workspace_bytes = 0; });
    call("2^32 units", F2K_ERR_UNSUPPORTED, 2, [](B& b, A&, T&) { b.n_seqs = 1 << 20; b.n_tokens = 1 << 20; b.table_width = 1 << 16; });
    if (f2k_kv_append(h, &b0, nullptr, nullptr) != F2K_ERR_INVALID || f2k_kv_append(h, nullptr, &a0, nullptr) != F2K_ERR_INVALID ||
        f2k_kv_attend(h, &b0, nullptr, nullptr) != F2K_ERR_INVALID || f2k_kv_append(nullptr, &b0, &a0, nullptr) != F2K_ERR_INVALID ||
        f2k_kv_workspace_bytes(nullptr, &b0) != 0 || f2k_kv_device_status(nullptr, nullptr) != F2K_ERR_INVALID) { std::printf("null\n"); ++bad; }
    if (f2k_kv_set_wait_limits(h, -1) != F2K_ERR_INVALID || f2k_kv_set_wait_limits(h, 5) != F2K_OK) { std::printf("limits\n"); ++bad; }

    // which kernel, and with how many rows (group 4)
    auto takes = [&](int max_new, int seqs, int kernel, int rows) {
        f2k_kv_batch b = b0; f2k_kv_attend_args t = t0;
        b.max_new = max_new; b.n_seqs = seqs; b.n_tokens = seqs * max_new;
        t.workspace_bytes = 1 << 30;
        if (f2k_kv_attend(h, &b, &t, nullptr) || launched_kernel != kernel || (kernel == 2 && launched_rows != rows)) {
            std::printf("max_new %d, %d sequences: kernel %d, rows %d\n", max_new, seqs, launched_kernel, launched_rows); ++bad;
        }
        if (kernel == 3 && f2k_kv_workspace_bytes(h, &b) != 0) { std::printf("a prompt's workspace\n"); ++bad; }
    };
    takes(1, 1, 2, 8); takes(2, 100, 2, 8); takes(3, 1, 2, 16); takes(4, 100, 2, 16); takes(8, 31, 2, 32); takes(8, 32, 3, 0); takes(16, 15, 2, 64);
    takes(16, 16, 3, 0); takes(17, 1, 3, 0);

    current = 0; work = 0;
    if (f2k_kv_append(h, &b0, &a0, nullptr) != F2K_ERR_INVALID || f2k_kv_attend(h, &b0, &t0, nullptr) != F2K_ERR_INVALID || work ||
        !std::strstr(f2k_kv_last_error(h), "made on device 1, device 0 is current")) { std::printf("another device: %s\n", f2k_kv_last_error(h)); ++bad; }
    int st = 1;
    if (f2k_kv_device_status(h, &st) != F2K_OK || st != 0 || synchronised != 1 || current != 0) { std::printf("status\n"); ++bad; }
    *last_status = 16 + 32 + 64;
    if (f2k_kv_device_status(h, &st) != F2K_ERR_DEVICE || st != 112 || !std::strstr(f2k_kv_last_error(h), "page number") ||
        !std::strstr(f2k_kv_last_error(h), "lengths") || !std::strstr(f2k_kv_last_error(h), "rotation")) { std::printf("status word: %s\n", f2k_kv_last_error(h)); ++bad; }
    if (f2k_kv_device_status(h, &st) != F2K_OK || st != 0) { std::printf("status is not cleared\n"); ++bad; }
    f2k_kv_destroy(h);
    f2k_kv_destroy(nullptr);

    // over an e4m3 cache (2 key heads here) up to 32 rows stay, and so do more rows of fewer than 80 pairs of sequence and key head
    c = good();
    c.cache_type = F2K_E4M3;
    if (f2k_kv_create(&c, &h)) { std::printf("create e4m3\n"); return 1; }
    takes(8, 100, 2, 32); takes(9, 39, 2, 64); takes(9, 40, 3, 0); takes(16, 39, 2, 64); takes(16, 40, 3, 0); takes(17, 1, 3, 0);
    f2k_kv_destroy(h);
    return bad;
}
"""


def test_c_entry_points(tmp_path):
    if not (CUDA / "cuda.h").exists():
        pytest.skip("no CUDA headers")
    src, exe = tmp_path / "refusals.cpp", tmp_path / "refusals"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", str(ROOT / "include"), "-I", str(CSRC), "-I", str(CUDA), "-x", "c++", str(src),
                    str(CSRC / "kv" / "paged_kv.cu"), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr


class _Lib:
    """Stands in for the library: keeps what it is called with."""

    def __init__(self):
        self.calls = []

    def f2k_kv_create(self, cfg, out):
        return 0

    def f2k_kv_destroy(self, h):
        pass

    def f2k_kv_append(self, *args):
        self.calls.append(args)
        return 0

    f2k_kv_attend = f2k_kv_append


@pytest.fixture
def kv(monkeypatch):
    from f2k_cuda_b200 import paged
    monkeypatch.setattr(paged, "lib", _Lib())
    monkeypatch.setattr(paged, "stream_handle", lambda s: 0 if s is None else s)
    pages = torch.zeros(6, 2, 16, 64, dtype=torch.bfloat16)
    return paged.PagedKV(paged.PagedKV.Config(4, 2, 64, 16, 6, rot_dim=32), pages, pages.clone())


def _args():
    from f2k_cuda_b200.paged import PagedBatch
    q, k = torch.zeros(3, 4, 64, dtype=torch.bfloat16), torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    g, t = torch.ones(64, dtype=torch.bfloat16), torch.zeros(40, 16)
    batch = PagedBatch(torch.ones(3, dtype=torch.int32), torch.zeros(3, 2, dtype=torch.int32))
    return {"Q": q, "K": k, "V": k, "gammas": (g, g), "tables": (t, t), "eps": 1e-6, "Q_out": q, "batch": batch}


@pytest.mark.parametrize("change", [
    {"Q": torch.zeros(3, 4, 64)}, {"K": torch.zeros(3, 4, 64, dtype=torch.bfloat16)}, {"V": torch.zeros(2, 2, 64, dtype=torch.bfloat16)},
    {"Q_out": torch.zeros(3, 4, 128, dtype=torch.bfloat16)}, {"Q": torch.zeros(3, 64, 4, dtype=torch.bfloat16).transpose(1, 2)},
    {"Q": torch.zeros(3, 8, 64, dtype=torch.bfloat16)[:, ::2]}, {"gammas": (torch.ones(64), torch.ones(64))},
    {"gammas": (torch.ones(32, dtype=torch.bfloat16),) * 2}, {"tables": (torch.zeros(40, 32),) * 2},
    {"tables": (torch.zeros(40, 16), torch.zeros(39, 16))}, {"tables": (torch.zeros(40, 16).double(),) * 2}], ids=range(11))
def test_append_checks_its_tensors(kv, change):
    from f2k_cuda_b200 import paged
    with pytest.raises(TypeError):
        kv.append(**{**_args(), **change})
    assert not paged.lib.calls


@pytest.mark.parametrize("name", ["Q", "K", "V", "Q_out", "gammas", "tables", "batch"])
def test_tensors_of_another_device_are_refused(kv, name):
    """A handle of GPU 0 (the tests' tensors are on the CPU: index -1): each tensor alone on another device. Tensors that
    are right get a stand-in that says it is on GPU 0."""
    from f2k_cuda_b200 import paged

    class There:
        def __init__(self, t):
            self.t = t

        def get_device(self):
            return 0

        def __getattr__(self, n):
            return getattr(self.t, n)

    kv._index = 0
    a = _args()
    there = {k: There(v) for k, v in a.items() if isinstance(v, torch.Tensor)} | {"gammas": tuple(map(There, a["gammas"])), "tables": tuple(map(There, a["tables"])),
                                                                                  "eps": a["eps"], "batch": a["batch"]}
    a["batch"].index = 0
    assert kv.append(**there)
    if name == "batch":
        a["batch"].index = 1
    with pytest.raises(TypeError):
        kv.append(**{**there, name: a[name]})
    assert len(paged.lib.calls) == 1


def test_arguments_arrive_as_the_header_says(kv):
    """The packed arguments, read back through the C structures of include/f2k_attn.h."""
    from f2k_cuda_b200 import paged

    class Append(C.Structure):
        _fields_ = [(n, C.c_void_p) for n in ("q", "k", "v", "gamma_q", "gamma_k", "cos", "sin", "q_out")] + \
            [(n, C.c_longlong) for n in ("qs", "ks", "vs", "qos")] + [("n_positions", C.c_int), ("eps", C.c_float)]

    class Attend(C.Structure):
        _fields_ = [(n, C.c_void_p) for n in ("q", "o", "lse")] + [("qs", C.c_longlong), ("os", C.c_longlong), ("ws", C.c_void_p), ("ws_bytes", C.c_size_t)]

    assert C.sizeof(Append) == paged._APPEND.size and C.sizeof(Attend) == paged._ATTEND.size
    a = _args()
    wide = torch.zeros(3, 1000, dtype=torch.bfloat16)
    a["Q"], a["V"] = wide[:, :256].unflatten(1, (4, 64)), wide[:, 400:528].unflatten(1, (2, 64))
    assert kv.append(**a, stream=7)
    h, batch, at, stream = paged.lib.calls[0]
    got = Append.from_address(at)
    ptr = lambda t: t.data_ptr()  # noqa: E731
    assert (got.q, got.k, got.v, got.q_out) == tuple(map(ptr, (a["Q"], a["K"], a["V"], a["Q_out"]))) and stream == 7
    assert (got.gamma_q, got.cos, got.sin) == (ptr(a["gammas"][0]), ptr(a["tables"][0]), ptr(a["tables"][1]))
    assert (got.qs, got.ks, got.vs, got.qos) == (1000, 0, 1000, 0) and got.n_positions == 40 and abs(got.eps - 1e-6) < 1e-12
    assert batch._obj.n_tokens == 3 and batch._obj.n_seqs == 3 and batch._obj.table_width == 2 and batch._obj.cu_seqlens is None
    ws, lse = torch.zeros(64, dtype=torch.uint8), torch.zeros(3, 4)
    assert kv.attend(a["Q"], a["Q_out"], a["batch"], ws, lse=lse, stream=0)
    got = Attend.from_address(paged.lib.calls[1][2])
    assert (got.q, got.o, got.lse, got.qs, got.os, got.ws, got.ws_bytes) == (ptr(a["Q"]), ptr(a["Q_out"]), ptr(lse), 1000, 0, ptr(ws), 64)
    assert kv.append(**{**a, "gammas": (None, None)}) and Append.from_address(paged.lib.calls[2][2]).gamma_q is None


def test_attend_checks_its_tensors(kv):
    from f2k_cuda_b200 import paged
    a = _args()
    ok = dict(Q=a["Q"], O=a["Q_out"], batch=a["batch"], workspace=None)
    for change in ({"Q": a["K"]}, {"O": a["Q"].float()}, {"lse": torch.zeros(3, 2)}, {"lse": torch.zeros(3, 4).double()},
                   {"workspace": torch.zeros(8, 8)[:, :4]}):
        with pytest.raises(TypeError):
            kv.attend(**{**ok, **change})
    assert not paged.lib.calls


def test_expanded_tensors_are_refused(kv):
    """A stride of 0 means dense to the C functions: an expanded view would be read far behind its memory."""
    from f2k_cuda_b200 import paged
    a = _args()
    for name, heads in (("Q", 4), ("K", 2), ("V", 2), ("Q_out", 4)):
        with pytest.raises(TypeError):
            kv.append(**{**a, name: torch.zeros(1, heads, 64, dtype=torch.bfloat16).expand(3, -1, -1)})
    with pytest.raises(TypeError):
        kv.append(**{**a, "Q": torch.zeros(600, dtype=torch.bfloat16).as_strided((3, 4, 64), (128, 64, 1))})
    with pytest.raises(TypeError):
        kv.attend(torch.zeros(1, 4, 64, dtype=torch.bfloat16).expand(3, -1, -1), a["Q_out"], a["batch"], None)
    lens = torch.ones(3, dtype=torch.int32)
    for args in ((lens, torch.zeros(1, 2, dtype=torch.int32).expand(3, -1)), (lens[:1].expand(3), torch.zeros(3, 2, dtype=torch.int32))):
        with pytest.raises(TypeError):
            paged.PagedBatch(*args)
    cfg = paged.PagedKV.Config(4, 2, 64, 16, 6, rot_dim=32)
    pages = torch.zeros(6, 2, 16, 64, dtype=torch.bfloat16)
    for view in (pages[:1].expand(6, -1, -1, -1), pages[:, :1].expand(-1, 2, -1, -1), pages[:1, :1, :1].expand(6, 2, 16, -1)):
        with pytest.raises(TypeError):
            paged.PagedKV(cfg, view, pages)
    assert not paged.lib.calls


def test_strides_of_single_pages_and_heads():
    """A dimension of one element may have any stride; the library gets that of a dense array."""
    from f2k_cuda_b200.paged import _strides
    one = torch.zeros(4096).as_strided((1, 1, 16, 64), (0, 0, 128, 1))
    assert _strides(one) == [1024, 1024, 128]
    assert _strides(torch.zeros(3, 16, 2, 64).transpose(1, 2)) == [2048, 64, 128]


def test_batches_and_caches_check_theirs(kv):
    from f2k_cuda_b200.paged import PagedBatch, PagedKV
    lens, table = torch.ones(3, dtype=torch.int32), torch.zeros(3, 2, dtype=torch.int32)
    for args in ((lens.long(), table), (lens, table[:2]), (lens, table, lens), (lens, table.T), (lens, table, None, 2), (lens[None], table),
                 (lens, table.float())):
        with pytest.raises(TypeError):
            PagedBatch(*args)
    pages, cfg = torch.zeros(6, 2, 16, 64, dtype=torch.float16), dict(n_heads=4, n_kv_heads=2, head_dim=64, page_size=16, n_pages=6, dtype=torch.float16)
    scale = torch.ones(2)
    for args in ((pages[:5], pages), (pages, pages.bfloat16()), (pages.float(), pages.float()), (pages.transpose(2, 3), pages),
                 (pages, pages, scale[:1], None), (pages, pages, scale.double(), None)):
        with pytest.raises(TypeError):
            PagedKV(PagedKV.Config(**cfg), *args)
    with pytest.raises(TypeError):
        PagedKV(PagedKV.Config(**{**cfg, "dtype": torch.float32}), pages, pages)
