"""Calls in place, at the C entry points with the fake CUDA runtime of the refusals' tests: the same memory for Q and the result
goes with the same stride only."""
import subprocess

import pytest

from tests.test_paged_refusals import CSRC, CUDA, PROGRAM, ROOT

MAIN = r"""
int main() {
    f2k_kv_config c = good();
    f2k_kv* h = nullptr;
    if (f2k_kv_create(&c, &h)) return 1;
    int32_t* ip = reinterpret_cast<int32_t*>(mem);
    f2k_kv_batch b{3, 5, 2, 4, 0, ip, ip, ip};
    const size_t ws = f2k_kv_workspace_bytes(h, &b);
    auto call = [&](const void* q, long long q_stride, void* out, long long out_stride, int want) {
        const f2k_kv_append_args a{q, mem, mem, nullptr, nullptr, fl, fl, out, q_stride, 0, 0, out_stride, 8, 1e-6f};
        const f2k_kv_attend_args t{q, out, nullptr, q_stride, out_stride, mem, ws};
        for (int which = 0; which < 2; ++which) {
            work = 0;
            const int rc = which ? f2k_kv_attend(h, &b, &t, nullptr) : f2k_kv_append(h, &b, &a, nullptr);
            if (rc != want || (work != 0) != (want == F2K_OK) || (want && !std::strstr(f2k_kv_last_error(h), "different strides"))) {
                std::printf("%s, strides %lld and %lld: %d '%s'\n", which ? "attend" : "append", q_stride, out_stride, rc, f2k_kv_last_error(h)); ++bad;
            }
        }
    };
    call(mem, 0, mem, 0, F2K_OK);
    call(mem, 0, mem, 1024, F2K_OK);              // 8 heads of 128: dense
    call(mem, 4096, mem, 4096, F2K_OK);
    call(mem, 4096, mem, 0, F2K_ERR_INVALID);
    call(mem, 0, mem, 2048, F2K_ERR_INVALID);
    call(mem, 4096, mem + 16, 0, F2K_OK);         // other memory
    b.n_seqs = b.n_tokens = 1;                    // one row: its stride says nothing
    call(mem, 4096, mem, 0, F2K_OK);
    f2k_kv_destroy(h);
    return bad;
}
"""


def test_in_place_needs_one_stride(tmp_path):
    if not (CUDA / "cuda.h").exists():
        pytest.skip("no CUDA headers")
    src, exe = tmp_path / "in_place.cpp", tmp_path / "in_place"
    src.write_text(PROGRAM[:PROGRAM.index("int main()")] + MAIN)
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", str(ROOT / "include"), "-I", str(CSRC), "-I", str(CUDA), "-x", "c++", str(src),
                    str(CSRC / "kv" / "paged_kv.cu"), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
