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


def _call(p, max_new=None, rows=None):
    """Append and attend with another max_new, or the first `rows` rows of the tensors only; outputs filled with 9."""
    import f2k_cuda_b200 as f2k
    p.batch = f2k.PagedBatch(p.lens_t, p.table, p.cu, max_new or max(p.news))
    p.ws = torch.empty(p.kv.workspace_size_bytes(p.batch), dtype=torch.uint8, device="cuda").fill_(0xAA)
    n = rows or p.T
    p.o.fill_(9.0)
    p.lse.fill_(9.0)
    assert p.kv.attend(p.q[:n], p.o[:n], p.batch, p.ws, lse=p.lse[:n]), p.kv.last_error()
    assert p.kv.device_status() == 32


# sequence 1 or 0 has more new tokens than max_new says; the rule picks the kernel by max_new
TOO_MANY = [([1000, 100, 100], 0, 100), ([100, 1000, 100, 7], 1, 100), ([3, 1, 1], 0, 1), ([1, 70, 1], 1, 1), ([4, 30, 3], 1, 4)]


@pytest.mark.parametrize("news,wrong,max_new", TOO_MANY, ids=[str(i) for i in range(len(TOO_MANY))])
@pytest.mark.parametrize("dtype,cache", [(BF, BF), (HF, E4)], ids=ids)
@pytest.mark.parametrize("behind", [0, 6000])
def test_a_sequence_with_more_new_tokens_than_max_new(news, wrong, max_new, dtype, cache, behind):
    """None of its rows is written; the other sequences, those behind it too, are attended as ever."""
    p = Problem(news, [n + behind for n in news], 8, 2, 128, 16, dtype, cache, seed=sum(news))
    _call(p, max_new)
    first = sum(news[:wrong])
    assert (p.o[first:first + news[wrong]] == 9.0).all() and (p.lse[first:first + news[wrong]] == 9.0).all()
    p.news[wrong] = 0
    p.check_attend()


@pytest.mark.parametrize("news,rows", [([40, 90, 60], 160), ([1, 2, 1], 3), ([2, 1, 4], 5)], ids=["prompts", "token", "drafts"])
@pytest.mark.parametrize("dtype,cache", [(BF, BF), (HF, E4)], ids=ids)
def test_a_sequence_with_rows_behind_the_call_s(news, rows, dtype, cache):
    """Its first rows lie inside the call's tensors; where they would be in the sequence says the part that does not."""
    p = Problem(news, [n + 700 for n in news], 8, 2, 64, 16, dtype, cache, seed=sum(news))
    _call(p, rows=rows)
    first = sum(news[:2])
    assert (p.o[first:] == 9.0).all() and (p.lse[first:] == 9.0).all()
    p.news[2] = 0
    p.check_attend()


def test_a_sequence_with_rows_in_front_of_the_call_s():
    p = Problem([30, 50, 20], [200, 300, 100], 8, 2, 128, 16, BF, seed=41)
    p.cu[0] = -8
    _call(p)
    assert (p.o[:30] == 9.0).all()
    p.news[0] = 0
    p.check_attend()


@pytest.mark.parametrize("dtype", [BF, HF], ids=ids)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("k_scale", [1.0, 1e-8, 1e-30, 1e-44])
@pytest.mark.parametrize("news,lens", [([1, 3, 2], [500, 40, 9000]), ([200, 3, 70], [200, 50, 900]), ([600] * 6, [600, 700, 800, 601, 900, 600])],
                         ids=["tokens", "a tile", "two tiles"])
def test_rows_of_zeros_over_e4m3(dtype, dim, k_scale, news, lens):
    """Queries of nothing, or next to nothing: the mean of the values that the row sees, however small the keys' scale is."""
    p = Problem(news, lens, 16, 4, dim, 32, dtype, E4, window=300, scales=True, seed=dim)
    p.k_scale.fill_(k_scale)
    p.q[::2] = 0
    p.q[1::4, ::3] = 0
    p.q[1::4, 1::3] *= 1e-38 if dtype is BF else 2.0 ** -20
    p.attend()
    p.check_attend()
    assert p.kv.device_status() == 0


def test_small_scales_of_the_scores_over_e4m3():
    for scale in (1e-20, 1e-38, 1e-45):
        for news, lens in (([1, 2], [500, 300]), ([100, 300], [200, 300])):
            p = Problem(news, lens, 8, 2, 128, 16, BF, E4, scales=True, scale=scale, seed=5)
            p.k_scale.fill_(0.5)
            p.q[0] = 0
            p.attend()
            p.check_attend()


@pytest.mark.parametrize("news,lens", [([1, 3, 2], [5000, 70, 900]), ([40, 200, 1], [2000, 200, 5])], ids=["tokens", "prompts"])
def test_a_layer_in_place_in_wider_rows(news, lens):
    """Q, K and V are columns of one projection; Q is turned where it stands, and its rows become the attention's."""
    p = Problem(news, lens, 8, 2, 128, 16, BF, rot=128, gap=520, seed=51)
    angle = torch.rand(max(lens), 64, generator=p.gen, device="cuda") * 100
    tables = angle.cos(), angle.sin()
    apart, o = torch.empty(p.T, 8, 128, device="cuda", dtype=BF), torch.empty(p.T, 8, 128, device="cuda", dtype=BF)
    assert p.kv.append(p.q, p.k, p.v, (None, None), tables, 1e-6, apart, p.batch)
    assert p.kv.attend(apart, o, p.batch, p.ws, lse=p.lse)
    assert p.kv.append(p.q, p.k, p.v, (None, None), tables, 1e-6, p.q, p.batch)
    assert torch.equal(p.q, apart)
    assert p.kv.attend(p.q, p.q, p.batch, p.ws, lse=p.lse)
    assert torch.equal(p.q, o) and p.kv.device_status() == 0
    assert not p.kv.append(p.q, p.k, p.v, (None, None), tables, 1e-6, p.q.as_strided((p.T, 8, 128), (1024, 128, 1)), p.batch)
    assert "different strides" in p.kv.last_error()


@pytest.mark.parametrize("order", ["longest last", "longest first", "longest in the middle"])
@pytest.mark.parametrize("dim,heads,kv_heads", [(128, 8, 2), (64, 4, 4)])
def test_ragged_prompts_in_any_order(order, dim, heads, kv_heads):
    news = {"longest last": [40, 130, 333, 700, 1500], "longest first": [1500, 700, 333, 130, 40],
            "longest in the middle": [130, 700, 1500, 333, 40]}[order]
    p = Problem(news, [n + 77 * b for b, n in enumerate(news)], heads, kv_heads, dim, 64, BF, seed=dim)
    p.attend()
    p.check_attend()


@pytest.mark.parametrize("cache", [HF, E4], ids=ids)
def test_more_prompts_than_lanes(cache):
    """A CTA finds its sequence 32 at a time; some have no new token, one is long."""
    gen = torch.Generator().manual_seed(8)
    news = torch.randint(0, 90, (70,), generator=gen).tolist()
    news[45] = 600
    p = Problem(news, [n + 13 * b % 200 for b, n in enumerate(news)], 8, 4, 64, 16, HF, cache, seed=9)
    p.attend()
    p.check_attend()


# one sequence of `new` tokens behind `past` keys, and one beside it
BATCHES = [(8, 300), (200, 150), (900, 100)]


@pytest.mark.parametrize("new,past", BATCHES, ids=["drafts", "a tile", "two tiles"])
@pytest.mark.parametrize("window", [0, 90])
@pytest.mark.parametrize("cache", [BF, E4], ids=ids)
@pytest.mark.parametrize("value", [float("nan"), float("inf")], ids=["nan", "inf"])
def test_values_that_are_not_finite_inside_a_sequence(new, past, window, cache, value):
    """One element of one key and one value, in the middle of a sequence's new tokens. The key is nothing to tokens that do not
    see it. The value reaches tokens that see it, in its own column, and at most such as lie within 255 tokens of one
    that does: never another column, key head or sequence."""
    if cache is E4 and value == float("inf"):
        pytest.skip("e4m3 has no infinity")
    p = Problem([new, new], [past + new] * 2, 8, 2, 64, 32, BF, cache, window, seed=new + window)
    at = past + new // 2
    pos = torch.arange(past, past + new, device="cuda")
    sees = (pos >= at) & (pos < at + window if window else True)
    page, row = int(p.table[0, at // 32]), at % 32

    def out(pages, x):
        pages[page, 1, row, 5] = x
        p.attend()
        assert p.kv.device_status() == 0
        return p.o.clone(), p.lse.clone()

    (o0, l0), (o1, l1) = out(p.k_pages, 0.0), out(p.k_pages, value)
    # Rows of a warp move their references together, so the same answers may be rounded in other places: against the formula.
    p.k_pages[page, 1, row, 5] = 0.0
    mixed = [torch.cat([torch.where(sees.view(-1, *[1] * (x.dim() - 1)), x[:new], y[:new]), y[new:]]) for x, y in ((o0, o1), (l0, l1))]
    p.check_attend(*mixed)
    assert torch.equal(o0[new:], o1[new:]) and torch.equal(o0[:, :4], o1[:, :4])
    if value != value:
        assert torch.isnan(o1[:new][sees][:, 4:]).all()
    out(p.k_pages, 0.0)
    (o0, l0), (o1, l1) = out(p.v_pages, 0.0), out(p.v_pages, value)
    assert torch.equal(l0, l1) and torch.equal(o0[new:], o1[new:]) and torch.equal(o0[:, :4], o1[:, :4])
    others = [c for c in range(64) if c != 5]
    assert torch.equal(o0[..., others], o1[..., others])
    assert not torch.isfinite(o1[:new][sees][:, 4:, 5]).any()
    last = at + window - 1 if window else past + new
    far = (pos < at - 255) | (pos > last + 255)
    assert torch.equal(o0[:new][far], o1[:new][far])
