"""The token kernel's line of work, walked on the CPU as the kernel's groups of warps walk it: every key that some row of a
tile sees is taken exactly once, in order; pieces of the line are equal; the pieces that share a work leave their rows
in places of their own and the join finds all of them; nothing leaves the table, whatever the lengths say."""
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
CSRC = ROOT / "f2k_cuda_b200" / "csrc"
CUDA = Path("/usr/local/cuda/include")

PROGRAM = r"""
#include "kv/token_work.h"
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>
#include <set>
#include <tuple>
#include <vector>
using namespace f2k;
#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s (case %d)\n", __LINE__, #x, case_no); std::exit(1); } } while (0)
static int case_no;

template <int kRows, int kUnit, int KW>
static void one(std::mt19937& r, bool wild) {
    auto pick = [&](int lo, int hi) { return (int)(lo + r() % (unsigned)(hi - lo + 1)); };
    AttendParams p{};
    p.page_shift = pick(4, 8);
    p.group = pick(1, 9);
    p.n_kv_heads = pick(1, 5);
    p.window = pick(0, 2) ? 0 : pick(1, 200);
    const int n = pick(1, 9), width = pick(1, 8);
    const long long capacity = (long long)width << p.page_shift;
    std::vector<int32_t> cu{0}, lens;
    for (int b = 0; b < n; ++b) {
        const int n_new = pick(0, 3) ? pick(0, 3) : pick(0, 60);
        cu.push_back(cu.back() + n_new);
        lens.push_back((int)(capacity < n_new ? capacity : pick(n_new, (int)capacity)));
    }
    const int n_tokens = cu.back() + pick(0, 3);
    if (wild) for (auto* v : {&cu, &lens}) for (auto& x : *v) if (!pick(0, 2)) x = (int)(r() - (1u << 31)) >> pick(0, 30);
    p.batch = PagedBatch{cu.data(), lens.data(), nullptr, width, width, n, n_tokens, 60};
    const int n_ctas = pick(1, 12);

    auto seq = [&](int b) { return seq_of(p.batch, p.page_shift, b); };
    unsigned total = 0;
    std::vector<unsigned> start;
    for (int b = 0; b < n; ++b) {
        start.push_back(total);
        total += seq_places(p, seq_work(seq(b), p.group, kRows, kUnit, p.window));
    }
    start.push_back(total);
    if (total == 0) return;
    const int n_pieces = pieces(total, n_ctas, kLeastPlaces);
    CHECK(piece_begin(total, n_pieces, 0) == 0 && piece_begin(total, n_pieces, n_pieces) == total);
    using Id = std::tuple<int, int, int>;                       // sequence, head, row tile
    std::map<Id, std::set<int>> keys;                           // units taken
    std::map<Id, std::vector<int>> shares;                      // in the order of the pieces
    std::set<int> share_used;
    std::map<Id, std::vector<int>> joined;
    std::map<Id, int> whole;
    for (int c = 0; c < n_pieces; ++c) {
        const unsigned begin = piece_begin(total, n_pieces, c), end = piece_begin(total, n_pieces, c + 1);
        CHECK(end > begin);
        int b0 = 0;
        while (start[b0 + 1] <= begin) ++b0;
        Where first; first.b = b0; first.seq_begin = start[b0];
        first.s = seq(b0);
        first.w = seq_work(first.s, p.group, kRows, kUnit, p.window);
        for (int kw = 0; kw < KW; ++kw) {
            // the fetching warp's walk and the consuming one's have to be the same
            std::vector<std::pair<Id, int>> fetched, used;
            Units<kRows, kUnit, KW> a;
            a.x = first; a.end = end; a.kw = kw;
            for (a.enter(p, seq, begin); a.more; a.next(p, seq)) {
                CHECK(a.x.b < n && a.x.kvh < p.n_kv_heads && a.x.rt < a.x.w.row_tiles);
                CHECK(a.key0() >= 0 && a.key0() < a.x.hi && a.x.hi <= capacity);
                fetched.push_back({Id{a.x.b, a.x.kvh, a.x.rt}, a.key0()});
            }
            Units<kRows, kUnit, KW> w;
            w.x = first; w.end = end; w.kw = kw;
            for (unsigned at = begin; at < end; at = w.stop) {
                const bool any = w.begin(p, seq, at);
                if (kw == 0 && at == begin) {
                    const int m = shares_to_join(w.x, total, n_pieces, c);
                    if (m) {
                        const Id id{w.x.b, w.x.kvh, w.x.rt};
                        CHECK(joined.count(id) == 0 && m >= 2);
                        for (int j = 0; j < m; ++j) joined[id].push_back(share_of(c - 1 + j, j == 0));
                    }
                }
                if (!any) { CHECK(w.stop == end); break; }
                const Id id{w.x.b, w.x.kvh, w.x.rt};
                for (bool have = w.settle(); have; w.u += KW, have = w.settle()) used.push_back({id, w.key0()});
                if (kw == 0) {
                    const bool from_start = at <= w.x.first_unit(), to_end = w.stop == w.x.work_end;
                    if (from_start && to_end) ++whole[id];
                    else {
                        const int s = share_of(c, from_start);
                        CHECK(s >= 0 && s < 2 * n_ctas && share_used.insert(s).second);
                        shares[id].push_back(s);
                    }
                }
            }
            CHECK(fetched == used);
            for (auto& [id, k] : used) CHECK(keys[id].insert(k).second);
        }
    }
    CHECK(shares == joined);
    for (int b = 0; b < n; ++b) {
        Where x;
        x.s = seq(b);
        x.w = seq_work(x.s, p.group, kRows, kUnit, p.window);
        CHECK(x.s.first >= 0 && x.s.n_new >= 0 && x.s.first + x.s.n_new <= n_tokens && x.s.len >= 0 && x.s.len <= capacity);
        for (int h = 0; h < p.n_kv_heads; ++h)
            for (int rt = 0; rt < x.w.row_tiles; ++rt) {
                const Id id{b, h, rt};
                CHECK(whole[id] + (int)joined.count(id) == 1);
                std::set<int> want;
                for (int row = rt * kRows; row < (rt + 1) * kRows && row / p.group < x.s.n_new; ++row) {
                    const KeyRange k = visible_keys(x.s, row / p.group, p.window);
                    for (int j = k.lo; j < k.hi; ++j) want.insert(j / kUnit * kUnit);
                }
                for (int k : want) CHECK(keys[id].count(k));
                for (int k : keys[id]) CHECK(want.count(k));
            }
    }
}
int main() {
    std::mt19937 r(7);
    for (case_no = 0; case_no < 800; ++case_no) {
        const bool wild = case_no % 3 == 2;
        switch (case_no % 4) {
            case 0: one<8, 16, 4>(r, wild); break;
            case 1: one<16, 32, 4>(r, wild); break;
            case 2: one<32, 16, 2>(r, wild); break;
            default: one<64, 16, 1>(r, wild);
        }
    }
    return 0;
}
"""


def test_every_key_is_taken_once_and_every_share_joined(tmp_path):
    if not (CUDA / "cuda.h").exists():
        pytest.skip("no CUDA headers")
    src, exe = tmp_path / "plan.cpp", tmp_path / "plan"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover", "-I", str(CSRC), "-I", str(CUDA), str(src),
                    "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
