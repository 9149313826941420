"""The order of the prompt kernel's accesses to shared memory where reading shows it and no run does for certain: what is
written over what, and which wait stands between the two."""
import re
from pathlib import Path

import pytest

TEXT = re.sub(r"//[^\n]*", "", (Path(__file__).resolve().parent.parent / "f2k_cuda_b200" / "csrc" / "kv" / "paged_prompt_sm100.cu").read_text())


@pytest.mark.parametrize("dim", [64, 128])
def test_rows_are_parked_behind_the_group_s_queries(dim):
    """Row r goes out from r * (2 dim + 16) of the tile's Q area, where other warps than r's have their rows of Q: every path
    from the queries' stores to the first parked row leads through a barrier that all four warps arrive at."""
    q_row = lambda r: {(piece * 128 * 128 + r * 128 + i) for piece in range(dim // 64) for i in range(128)}  # noqa: E731
    parked = lambda r: {r * (dim * 2 + 16) + i for i in range(dim * 2)}  # noqa: E731
    assert any(parked(r) & q_row(o) for r in range(32) for o in range(32, 128))             # so a wait is needed
    epilogue = TEXT[TEXT.index("l_sum += (sum[0] + sum[1]) + (sum[2] + sum[3]);"):]
    before = epilogue[:epilogue.index("const uint32_t park")]
    wait = re.search(r"if \(ok && \(n > 0 \|\| t == 0 \|\| pair\)\) \{\s*ok = n > 0 \? mbar_wait\(smem_u32\(&ctl->pv_done\[t\]\).*?"
                     r": mbar_wait\(smem_u32\(&ctl->q_full\[t\]\), 0,.*?ok = __all_sync", before, re.S)
    assert wait, "no wait in front of the parked rows of a tile without a key"
    assert "if (ok && (t == 0 || pair))" in before[wait.end():]


def test_a_loader_that_leaves_early_waits_for_every_copy_it_started():
    """The places where the loader's loop over the tiles j can be left: in front of tile j's copies with j tiles started; behind
    them with j + 1, counted before the loop is left. (A 16-bit tile that is cleared in part reports to a barrier of its own, which
    is waited for in any case.) What is waited for on the way out are the last tiles counted, as many as there are slots."""
    loader = TEXT[TEXT.index("int next_page = look_up(0)"):TEXT.index("constexpr uint32_t idesc_s")]
    assert "for (; j < n_kv; ++j) {" in loader
    copies = loader.index("tma_load_5d(")
    cleared = loader.index("ok = mbar_wait(bar, cleaned & 1")
    before, behind = loader[:copies], loader[copies:cleared]
    assert before.count("break;") == 2 and "++j;" not in before
    assert re.sub(r"\s+", " ", behind).count("break;") == 1
    assert "if (!(ok = convert(converted, came_boxes))) { ++j; break; }" in re.sub(r"\s+", " ", behind)
    way_out = loader[loader.index("volatile uint32_t never"):]
    assert "mbar_wait(smem_u32(&ctl->clean), cleaned & 1, &never" in way_out
    assert "for (int i = max(0, j - kSlots); i < j; ++i)" in way_out
