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


@pytest.mark.parametrize("dtype,cache", [(BF, BF), (HF, E4)], ids=ids)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("news,lens", [([1] * 4, [9000, 20, 300, 5000]), ([16] * 8, [16, 500, 4000, 60, 700, 20, 900, 3000]),
                                       ([400, 3, 130], [2000, 50, 130]), ([900] * 8, [900, 2000, 1000, 901, 950, 4000, 1800, 900])],
                         ids=["tokens", "drafts", "a tile", "two tiles"])
def test_short_wait_limits(dtype, cache, dim, news, lens):
    """A limit of a few clocks: the call is right, or ends and says that a wait ran out, and the next one is right. (A wait looks
    at its limit after 256 misses, and a miss suspends the thread for long, so that none of these waits runs out here.)"""
    p = Problem(news, lens, 16, 4, dim, 32, dtype, cache, 700, seed=dim + len(news))
    for limit in (1, 3000, 0):
        assert p.kv.set_wait_limits(limit)
        p.o.fill_(9.0)
        p.attend()
        status = p.kv.device_status()
        assert status in (0, 1) if limit else status == 0
        if status == 0:
            p.check_attend()
