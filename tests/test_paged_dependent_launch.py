"""The paged cache's kernels may start while the kernel in front of them still runs: each waits for it before its first access
to memory, in every thread, and none reads through the read-only path or through pointers that promise no alias."""
import re
from pathlib import Path

import pytest

KV = Path(__file__).resolve().parent.parent / "f2k_cuda_b200" / "csrc" / "kv"
SOURCES = sorted(KV.glob("*.cu"))
KERNELS = [(f.name, m.group(0)) for f in SOURCES for m in re.finditer(r"__global__.*?\n}\n", re.sub(r"//[^\n]*", "", f.read_text()), re.S)]


def test_the_kernels_are_found():
    assert sorted(f for f, _ in KERNELS) == ["kv_append.cu", "paged_prompt_sm100.cu", "paged_token.cu", "paged_token.cu"]


@pytest.mark.parametrize("file,text", KERNELS, ids=[f"{f}-{i}" for i, (f, _) in enumerate(KERNELS)])
def test_they_wait_before_they_read(file, text):
    for word in ("__ldg", "__restrict__", "ld.global.nc"):
        assert word not in text
    wait = min(text.index(w) for w in ("grid_dependency_wait", "griddepcontrol.wait") if w in text)
    before = text[:wait]
    for access in ("batch.", "p.q", "p.status", "ws_", "return"):      # no look at the call's memory, no way past the wait
        assert access not in before.split("{", 1)[1], f"{file}: {access} in front of the wait"
