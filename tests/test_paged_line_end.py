"""The end of the longest line of work that the token kernel takes, walked on the CPU: a group's step over the end of the line
must not come out at its beginning."""
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "f2k_cuda_b200" / "csrc"
CUDA = Path("/usr/local/cuda/include")

PROGRAM = r"""
#include "kv/token_work.h"
#include <cstdio>
#include <vector>
using namespace f2k;
int main() {
    // Sequences of one token and one head, as long as can be; the last one fills the line up to the limit exactly.
    constexpr int kUnit = 16, KW = 4, kLen = 0x7fffff00;
    AttendParams p{};
    p.page_shift = 8; p.group = 1; p.n_kv_heads = 1;
    std::vector<int> cu{0}, lens;
    unsigned long long line = 0, last = 0;
    while (line < kMostPlaces) {
        const unsigned long long left = kMostPlaces - line, whole = kLen / kUnit + kWorkCost;
        last = line;
        lens.push_back(left >= whole + kWorkCost + 1 || left == whole ? kLen : left > whole ? kLen - 100 * kUnit : (int)(left - kWorkCost) * kUnit);
        line += lens.back() / kUnit + kWorkCost;
        cu.push_back(cu.back() + 1);
    }
    if (line != kMostPlaces) { std::printf("line %llu\n", line); return 1; }
    const int n = (int)lens.size();
    p.batch = PagedBatch{cu.data(), lens.data(), nullptr, 0x7fffff, 0x7fffff, n, n, 1};
    auto seq = [&](int b) { return seq_of(p.batch, p.page_shift, b); };
    const unsigned total = (unsigned)line;
    for (int kw = 0; kw < KW; ++kw) {
        Units<8, kUnit, KW> a;
        a.x.b = n - 1; a.x.seq_begin = (unsigned)last; a.x.s = seq(n - 1); a.x.w = seq_work(a.x.s, 1, 8, kUnit, 0);
        a.end = total; a.kw = kw;
        const unsigned begin = total - 40;
        long long steps = 0;
        for (a.enter(p, seq, begin); a.more; a.next(p, seq)) {
            if (a.u < begin || a.u >= total || ++steps > 10) { std::printf("group %d at place %u of %u..%u\n", kw, a.u, begin, total); return 1; }
        }
        if (steps != 10) { std::printf("group %d: %lld units\n", kw, steps); return 1; }
    }
    return 0;
}
"""


def test_the_line_does_not_wrap(tmp_path):
    if not (CUDA / "cuda.h").exists():
        pytest.skip("no CUDA headers")
    src, exe = tmp_path / "line.cpp", tmp_path / "line"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", str(CSRC), "-I", str(CUDA), str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr
