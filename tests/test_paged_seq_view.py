"""What the kernels take of a sequence, on the CPU: rows that do not fit are no rows, the others are as the offsets say, and
the sequences together never have more rows than the call, so that each finds its place in a grid sized by the call."""
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "f2k_cuda_b200" / "csrc"
CUDA = Path("/usr/local/cuda/include")

PROGRAM = r"""
#include "kv/paged_params.h"
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>
using namespace f2k;
#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); std::exit(1); } } while (0)
int main() {
    SeqView s = seq_view(5, 8, 40, 10, 3, 64);
    CHECK(s.first == 5 && s.n_new == 3 && s.len == 40 && !s.bad);
    s = seq_view(5, 9, 40, 10, 3, 64);                       // one more than max_new
    CHECK(s.n_new == 0 && s.bad);
    s = seq_view(8, 11, 40, 10, 3, 64);                      // a row behind the call's
    CHECK(s.n_new == 0 && s.bad);
    s = seq_view(-1, 1, 40, 10, 3, 64);                      // one in front
    CHECK(s.n_new == 0 && s.bad);
    s = seq_view(6, 5, 40, 10, 3, 64);
    CHECK(s.n_new == 0 && s.bad);
    s = seq_view(5, 8, 2, 10, 3, 64);                        // fewer keys than new tokens: the rows are there
    CHECK(s.first == 5 && s.n_new == 3 && s.len == 2 && s.bad);
    s = seq_view(5, 8, 65, 10, 3, 64);
    CHECK(s.n_new == 3 && s.len == 64 && s.bad);
    s = seq_view(5, 8, -7, 10, 3, 64);
    CHECK(s.n_new == 3 && s.len == 0 && s.bad);
    s = seq_view(4, 4, 0, 10, 3, 64);
    CHECK(s.first == 4 && s.n_new == 0 && s.len == 0 && !s.bad);
    s = seq_view(2147483647, -2147483647 - 1, 1, 10, 3, 64);
    CHECK(s.n_new == 0 && s.bad);
    std::mt19937 r(3);
    for (int i = 0; i < 20000; ++i) {
        // offsets that ascend, of which some sequences are too long or end behind the call's rows
        const int n = 1 + r() % 9, max_new = 1 + r() % 12, n_tokens = 1 + r() % 60;
        std::vector<int> cu{(int)(r() % 4) - 2};
        for (int b = 0; b < n; ++b) cu.push_back(cu.back() + r() % 16);
        long long tiles = 0, rows = 0;
        const int step = 1 + r() % 8;
        for (int b = 0; b < n; ++b) {
            const SeqView v = seq_view(cu[b], cu[b + 1], 20, n_tokens, max_new, 64);
            CHECK(v.first >= 0 && v.n_new >= 0 && v.n_new <= max_new && v.first + v.n_new <= n_tokens);
            if (!v.bad) CHECK(v.first == cu[b] && v.n_new == cu[b + 1] - cu[b]);
            rows += v.n_new;
            tiles += (v.n_new + step - 1) / step;
        }
        const long long by_tokens = n_tokens / step + n, by_most = (long long)((max_new + step - 1) / step) * n;
        CHECK(rows <= n_tokens && tiles <= by_tokens && tiles <= by_most);
    }
    return 0;
}
"""


def test_rows_that_do_not_fit_are_none(tmp_path):
    if not (CUDA / "cuda.h").exists():
        pytest.skip("no CUDA headers")
    src, exe = tmp_path / "view.cpp", tmp_path / "view"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover", "-I", str(CSRC), "-I", str(CUDA), str(src),
                    "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
