"""Paged key/value cache on the GPU: batches at the edges of what a call may hold, and calls that leave early."""
import pytest
import torch

from tests._paged import Problem

pytestmark = pytest.mark.gpu
BF, HF, E4 = torch.bfloat16, torch.float16, torch.float8_e4m3fn
TYPES = [(BF, BF), (HF, HF), (BF, E4), (HF, E4)]
NAMES = {BF: "bf16", HF: "f16", E4: "e4m3"}
ids = lambda v: NAMES.get(v, None) if isinstance(v, torch.dtype) else None  # noqa: E731


@pytest.mark.parametrize("dtype,cache", TYPES, ids=ids)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("seqs,new", [(2, 300), (8, 700)], ids=["one tile a CTA", "two"])
def test_prompts_whose_tiles_see_no_key(dtype, cache, dim, seqs, new):
    """Sequences of no keys with many new tokens: every row is zero, whatever the queries are, every time."""
    p = Problem([new] * seqs, [new] * seqs, 32, 8, dim, 64, dtype, cache, seed=dim + seqs)
    p.lens_t.zero_()
    p.q.fill_(3.0)
    for _ in range(10):
        p.o.fill_(9.0)
        p.lse.fill_(9.0)
        p.attend()
        assert not p.o.any() and (p.lse == -torch.inf).all()
    assert p.kv.device_status() == 32
