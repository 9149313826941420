"""Paged key/value cache on the GPU: appending and attention against the formulas in 64 bits, at the lengths, layouts and
masks where they can go wrong."""
import pytest
import torch

from tests._paged import HALF, Problem, rotate

pytestmark = pytest.mark.gpu
BF, HF, E4 = torch.bfloat16, torch.float16, torch.float8_e4m3fn
TYPES = [(BF, BF), (HF, HF), (BF, E4), (HF, E4)]
NAMES = {BF: "bf16", HF: "f16", E4: "e4m3"}
ids = lambda v: NAMES.get(v, None) if isinstance(v, torch.dtype) else None  # noqa: E731

# one new token each: no key before it, inside and at the ends of units, tiles and pages, many of them, an idle sequence
LENS = [1, 2, 15, 16, 17, 31, 33, 64, 127, 128, 129, 300, 1000]


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype,cache", TYPES, ids=ids)
@pytest.mark.parametrize("page", [16, 64, 256])
def test_single_tokens(dtype, cache, dim, page):
    p = Problem([1] * len(LENS), LENS, 8, 2, dim, page, dtype, cache, scales=cache is E4, seed=dim + page)
    p.attend()
    p.check_attend()
    assert p.kv.device_status() == 0


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (6, 2), (7, 1), (16, 1), (17, 1), (32, 1), (40, 1), (64, 1), (128, 1), (32, 8)])
@pytest.mark.parametrize("cache", [BF, E4], ids=ids)
def test_head_groups(heads, kv_heads, cache):
    p = Problem([1, 1, 1], [5, 70, 513], heads, kv_heads, 128, 32, BF, cache, scales=cache is E4, seed=heads)
    p.attend()
    p.check_attend()


@pytest.mark.parametrize("dtype,cache", TYPES, ids=ids)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("window", [0, 1, 20, 100])
def test_several_new_tokens(dtype, cache, dim, window):
    """Drafts and short prompts, sequences without a new token, empty sequences, rows that see nothing."""
    p = Problem([4, 0, 3, 9, 1, 2, 0, 7], [4, 0, 40, 200, 1, 333, 50, 61], 6, 2, dim, 32, dtype, cache, window, scales=cache is E4,
                pad=3, gap=24, seed=window + dim)
    p.o.fill_(9.0)
    p.attend()
    p.check_attend()
    assert (p.o[-3:] == 9.0).all() and (p.lse[-3:] == 7.0).all()     # behind the last sequence
    assert p.kv.device_status() == 0


@pytest.mark.parametrize("seqs", [39, 40])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("window", [0, 50])
def test_drafts_over_e4m3_on_both_sides_of_the_rule(seqs, dim, window):
    """9 to 16 tokens of 4 query heads a key head: below 80 pairs of sequence and key head the token kernel, else the prompts'."""
    news = [9 + b % 8 for b in range(seqs)]
    p = Problem(news, [n + 37 * b % 400 for b, n in enumerate(news)], 8, 2, dim, 32, BF, E4, window, scales=True, pad=2, seed=seqs + dim)
    assert (p.ws.numel() == 0) == (seqs == 40)
    p.o.fill_(9.0)
    p.attend()
    p.check_attend()
    assert (p.o[-2:] == 9.0).all() and (p.lse[-2:] == 7.0).all() and p.kv.device_status() == 0


@pytest.mark.parametrize("cache", [HF, E4], ids=ids)
@pytest.mark.parametrize("lens", [[20000], [9000, 1], [4097, 12000, 300]])
def test_long_caches_are_split_and_joined(cache, lens):
    p = Problem([1] * len(lens), lens, 8, 2, 128, 64, HF, cache, seed=len(lens))
    p.attend()
    p.check_attend()
    first = p.o.clone(), p.lse.clone()
    p.o.fill_(3.0)
    p.attend()
    assert torch.equal(first[0], p.o) and torch.equal(first[1], p.lse)      # the same bits every time


@pytest.mark.parametrize("n_seqs", [257, 700])
def test_many_sequences(n_seqs):
    """More sequences than the CTA has threads; ragged, some without a new token."""
    gen = torch.Generator().manual_seed(n_seqs)
    lens = torch.randint(1, 70, (n_seqs,), generator=gen).tolist()
    news = [min(n, int(x)) for n, x in zip(lens, torch.randint(0, 3, (n_seqs,), generator=gen))]
    p = Problem(news, lens, 4, 2, 64, 16, BF, seed=n_seqs)
    p.attend()
    p.check_attend()


@pytest.mark.parametrize("dtype,cache", [(BF, BF), (HF, E4)], ids=ids)
def test_cache_with_tokens_before_heads(dtype, cache):
    """Pages as [page][token][head][dim]: the strides come from the views."""
    p = Problem([1, 2, 5], [77, 300, 31], 8, 4, 128, 32, dtype, cache, token_major=True, seed=3)
    assert p.k_pages.stride(2) == 4 * 128
    p.attend()
    p.check_attend()


# prompts: tiles of 128 rows, one or two a CTA, behind cached keys or not, sequences without a token among them
PROMPTS = [([64], [64]), ([128], [128]), ([33], [33]), ([300], [300]), ([129, 0, 65, 1, 256], [129, 7, 65, 200, 256]),
           ([70, 90], [1000, 90]), ([200, 3], [457, 3])]


@pytest.mark.parametrize("news,lens", PROMPTS, ids=[str(i) for i in range(len(PROMPTS))])
@pytest.mark.parametrize("dtype,cache", TYPES, ids=ids)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv_heads,page", [(8, 2, 16), (2, 2, 64), (3, 1, 128), (14, 2, 32), (4, 1, 256)])
def test_prompts(news, lens, dtype, cache, dim, heads, kv_heads, page):
    p = Problem(news, lens, heads, kv_heads, dim, page, dtype, cache, scales=cache is E4, pad=5, gap=8, seed=sum(lens) + dim + heads)
    p.o.fill_(9.0)
    p.attend()
    p.check_attend()
    assert (p.o[-5:] == 9.0).all() and (p.lse[-5:] == 7.0).all()
    assert p.kv.device_status() == 0


@pytest.mark.parametrize("window", [1, 50, 128, 300])
@pytest.mark.parametrize("heads,dim,page,cache", [(4, 128, 16, BF), (2, 64, 128, BF), (12, 128, 64, BF), (4, 128, 32, E4), (6, 64, 16, E4)], ids=ids)
def test_prompts_with_a_window(window, heads, dim, page, cache):
    """Pages in front of the window are gone: their entries in the table are outside the cache."""
    p = Problem([500, 40, 130], [500, 900, 700], heads, 2, dim, page, BF, cache, window=window, seed=window)
    for b, (n, m) in enumerate(zip(p.news, p.lens)):
        gone = max(0, m - n + 1 - window) // page
        p.table[b, :gone] = -1
    p.attend()
    assert p.kv.device_status() == 0
    p.table = p.table.clamp(min=0)                      # any page: the formula masks those keys
    for pages in (p.k_pages, p.v_pages):
        pages.copy_(pages.float().nan_to_num(0.0).to(pages.dtype))
    p.check_attend()


@pytest.mark.parametrize("cache", [None, E4], ids=ids)
def test_many_prompts_two_tiles_a_cta(cache):
    p = Problem([700, 513, 650, 40, 0, 333], [700, 513, 1200, 40, 3, 2000], 32, 8, 128, 16, BF, cache, seed=21)
    p.attend()
    p.check_attend()
    p = Problem([700, 513, 650], [700, 513, 1200], 30, 10, 64, 16, HF, cache, seed=22)
    p.attend()
    p.check_attend()


def test_one_more_head_group_than_rows():
    p = Problem([2, 5], [100, 300], 100, 1, 64, 16, BF, seed=23)          # 100 query heads a key head: a token a tile
    p.attend()
    p.check_attend()


def test_prompts_with_fewer_keys_than_tokens():
    """Tokens at negative positions see nothing: zero, and a report."""
    p = Problem([200, 300, 70], [200, 300, 70], 4, 2, 128, 16, HF, seed=24)
    p.lens = [0, 120, 70]
    p.lens_t.copy_(torch.tensor(p.lens, dtype=torch.int32))
    p.attend()
    assert p.kv.device_status() == 32
    p.check_attend()


@pytest.mark.parametrize("cache", [HF, E4], ids=ids)
@pytest.mark.parametrize("dim", [64, 128])
def test_prompt_with_a_page_outside_the_cache(cache, dim):
    p = Problem([150], [400], 4, 2, dim, 32, HF, cache, seed=25)
    whole = [p.keys(0, x) for x in (p.k_pages, p.v_pages)]
    p.table[0, 3] = 10 ** 6                             # keys 96 .. 127
    p.attend()
    assert p.kv.device_status() == 16
    keep = torch.tensor([j for j in range(400) if not 96 <= j < 128], device="cuda")
    q = p.q[-1].double().unflatten(0, (2, 2))
    w = torch.softmax(q @ whole[0][:, keep].mT * p.scale, -1)
    assert ((w @ whole[1][:, keep]).flatten(0, 1) - p.o[-1].double()).abs().max() < 4 * HALF[HF] * whole[1][:, keep].abs().max()
    assert torch.isfinite(p.o).all()


def test_queries_in_place():
    p = Problem([1, 3, 40], [500, 70, 2000], 8, 2, 128, 16, BF, seed=4)
    q = p.q.clone()
    assert p.kv.attend(p.q, p.q, p.batch, p.ws, lse=p.lse)
    out, p.q = p.q, q
    p.check_attend(out)


def test_scores_far_apart():
    """Scores of some hundreds: weights that are one or nothing; the maximum moves often."""
    p = Problem([1, 2], [3000, 500], 8, 2, 128, 16, HF, scale=8.0, seed=5)
    p.attend()
    p.check_attend()


def test_bad_pages_and_lengths_are_reported():
    p = Problem([1, 1, 1], [100, 40, 64], 4, 2, 64, 16, HF, seed=6)
    good = p.table.clone()
    p.table[0, 2] = -5
    p.attend()
    assert p.kv.device_status() == 16 and "page number" in p.kv.last_error()
    assert torch.isfinite(p.o).all()
    assert p.kv.device_status() == 0
    # sequence 0 without keys 32 .. 47
    p.table.copy_(good)
    k, v = p.keys(0, p.k_pages), p.keys(0, p.v_pages)
    keep = torch.tensor([j for j in range(100) if not 32 <= j < 48], device="cuda")
    q = p.q[0].double().unflatten(0, (2, 2))
    w = torch.softmax(q @ k[:, keep].mT / 8, -1)
    assert ((w @ v[:, keep]).flatten(0, 1) - p.o[0].double()).abs().max() < 4 * HALF[HF] * v[:, keep].abs().max()
    for lens in ([-1, 40, 64], [100, 40, 10 ** 9], [100, 0, 64]):
        p.lens_t.copy_(torch.tensor(lens, dtype=torch.int32))
        p.attend()
        assert p.kv.device_status() & 32 and "lengths" in p.kv.last_error()
    p.lens_t.copy_(torch.tensor([100, 40, 64], dtype=torch.int32))
    for cu in ([0, 1, 2, 1000], [0, -7, 2, 3], [2, 1, 0, 3]):
        p.cu.copy_(torch.tensor(cu, dtype=torch.int32))
        p.attend()
        assert p.kv.device_status() & 32
    p.cu.copy_(torch.tensor([0, 2, 3, 3], dtype=torch.int32))           # two new tokens where max_new says one
    p.attend()
    assert p.kv.device_status() == 32
    p.cu.copy_(torch.arange(4, dtype=torch.int32))
    p.attend()
    p.check_attend()


@pytest.mark.parametrize("dtype,cache", TYPES, ids=ids)
@pytest.mark.parametrize("dim,rot,interleaved,norm", [(128, 128, False, True), (128, 64, True, False), (64, 16, False, True),
                                                      (64, 64, True, True), (128, 0, False, False), (64, 0, False, True),
                                                      (128, 48, False, False)])
@pytest.mark.parametrize("news,lens", [([1, 1, 1], [1, 17, 400]), ([70, 0, 33, 1], [70, 5, 49, 300]), ([900, 300], [1000, 300])])
def test_append(dtype, cache, dim, rot, interleaved, norm, news, lens):
    p = Problem(news, lens, 6, 2, dim, 32, dtype, cache, rot=rot, interleaved=interleaved, scales=cache is E4, pad=2, gap=16,
                seed=dim + rot + len(news))
    gen, n_pos = p.gen, max(lens)
    angle = torch.rand(n_pos, max(1, rot // 2), generator=gen, device="cuda") * 100
    tables = (angle.cos(), angle.sin()) if rot else (None, None)
    gains = tuple((0.5 + torch.rand(dim, generator=gen, device="cuda")).to(dtype) for _ in range(2)) if norm else (None, None)
    before_k, before_v = p.k_pages.clone(), p.v_pages.clone()
    q_out = p.rows(6).fill_(5.0)
    assert p.kv.append(p.q, p.k, p.v, gains, tables, 1e-5, q_out, p.batch), p.kv.last_error()
    assert p.kv.device_status() == 0
    n = sum(news)
    seq = torch.repeat_interleave(torch.arange(len(news)), torch.tensor(news)).cuda()
    pos = torch.cat([torch.arange(m - k, m) for k, m in zip(news, lens)]).cuda()
    page, row = p.table[seq, pos // p.P].long(), pos % p.P
    step, tiny = HALF[cache], {BF: 0.0, HF: 2.0 ** -25, E4: 2.0 ** -10}

    def want(x, gain):
        x = x[:n].double()
        if gain is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-5) * gain.double()
        y = rotate(x, tables[0][pos], tables[1][pos], rot, interleaved) if rot else x
        # fp32 sums and products in front of the rounding: 2^-20 of the pair's size
        return y, 2.0 ** -20 * (x.abs() + x.abs().amax(-1, keepdim=True))

    for got, x, gain, t, u, scale in ((q_out[:n], p.q, gains[0], dtype, HALF[dtype], None), (p.k_pages[page, :, row], p.k, gains[1], cache, step, p.k_scale),
                                      (p.v_pages[page, :, row], p.v, None, cache, step, p.v_scale)):
        y, noise = want(x, gain) if x is not p.v else (x[:n].double(), 0.0)
        if scale is not None:
            y, noise = y / scale.double()[:, None], noise / scale.double()[:, None]
        if t is E4:
            y = y.clamp(-448, 448)
        off = (got.double() - y).abs() / (1.001 * u * y.abs() + tiny[t] + noise + 1e-30)
        assert off.max() <= 1, f"{off.max():.3g} times the tolerance"
    # everything else as it was
    touched = torch.zeros_like(p.used)
    touched[page, row] = True
    raw = lambda t: t.transpose(1, 2)[~touched].contiguous().view(torch.uint8)  # noqa: E731
    assert torch.equal(raw(p.k_pages), raw(before_k)) and torch.equal(raw(p.v_pages), raw(before_v))
    assert (q_out[n:] == 5.0).all()


def test_append_reports_what_does_not_fit():
    p = Problem([1, 1, 2], [10, 20, 40], 4, 2, 64, 16, BF, rot=64, seed=8)
    cos = sin = torch.ones(30, 32, device="cuda")
    before = p.k_pages.clone()
    assert p.kv.append(p.q, p.k, p.v, (None, None), (cos, sin), 1e-6, p.q, p.batch)
    assert p.kv.device_status() == 64 and "rotation" in p.kv.last_error()      # positions 38, 39
    changed = (p.k_pages.view(torch.int16) != before.view(torch.int16)).any(-1).any(1).sum()
    assert changed == 2
    cos = sin = torch.ones(40, 32, device="cuda")
    p.table[2, 2] = p.k_pages.shape[0]
    assert p.kv.append(p.q, p.k, p.v, (None, None), (cos, sin), 1e-6, p.q, p.batch)
    assert p.kv.device_status() == 16
    p.lens_t[1] = 0
    p.lens_t[0] = 2 ** 30
    assert p.kv.append(p.q, p.k, p.v, (None, None), (cos, sin), 1e-6, p.q, p.batch)
    assert p.kv.device_status() == 16 + 32


def test_append_values_that_e4m3_cannot_hold():
    p = Problem([3], [3], 2, 1, 64, 16, HF, E4, seed=9)
    p.v[0, 0, :4] = torch.tensor([1e4, -1e4, float("inf"), float("nan")], device="cuda")
    assert p.kv.append(p.q, p.k, p.v, (None, None), (None, None), 1e-6, p.q, p.batch)
    got = p.v_pages[int(p.table[0, 0]), 0, 0, :4].float().tolist()
    assert got[:3] == [448.0, -448.0, 448.0] and got[3] != got[3]


def _layer(p, gains, tables):
    assert p.kv.append(p.q, p.k, p.v, gains, tables, 1e-6, p.q, p.batch), p.kv.last_error()
    p.attend()


@pytest.mark.parametrize("dtype,cache", TYPES, ids=ids)
def test_prompts_then_tokens(dtype, cache):
    """A layer as a program runs it: prompts, then tokens one by one; every step against the formula over what the cache holds,
    and the last against one call that appends everything at once."""
    import f2k_cuda_b200 as f2k
    prompts, steps = [37, 1, 130], 4
    full = [n + steps for n in prompts]
    p = Problem(full, full, 8, 2, 128, 16, dtype, cache, rot=128, seed=10)
    angle = torch.arange(200, device="cuda")[:, None] * 10.0 ** -torch.linspace(0, 4, 64, device="cuda")
    tables, gains = (angle.cos(), angle.sin()), tuple(torch.ones(128, device="cuda", dtype=dtype) for _ in range(2))
    q, k, v = p.q.clone(), p.k.clone(), p.v.clone()
    _layer(p, gains, tables)
    p.check_attend()
    at_once, k_once = p.o.clone(), p.k_pages.clone()
    p.k_pages.fill_(float("nan"))
    p.v_pages.fill_(float("nan"))
    begin = p.cu.tolist()
    last = []
    for step in range(steps + 1):
        p.news = prompts if step == 0 else [1] * 3
        p.lens = [n + step for n in prompts]
        rows = torch.cat([torch.arange(m - n, m) + begin[b] for b, (n, m) in enumerate(zip(p.news, p.lens))]).cuda()
        p.q, p.k, p.v = q[rows].clone(), k[rows].clone(), v[rows].clone()
        p.T = len(rows)
        p.o, p.lse = torch.empty_like(p.q), torch.empty(p.T, 8, device="cuda")
        p.cu = torch.tensor([0] + torch.tensor(p.news).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
        p.lens_t = torch.tensor(p.lens, dtype=torch.int32, device="cuda")
        p.batch = f2k.PagedBatch(p.lens_t, p.table, p.cu if step < 2 else None, max(p.news))
        p.ws = torch.empty(p.kv.workspace_size_bytes(p.batch), dtype=torch.uint8, device="cuda")
        _layer(p, gains, tables)
        p.check_attend()
        last = rows
    assert p.kv.device_status() == 0
    same = p.used[:, None, :, None].expand(p.k_pages.shape)
    assert torch.equal(p.k_pages.float()[same], k_once.float()[same])       # the cache is the same, bit for bit
    a, b = p.o.double(), at_once[last].double()
    # both within the tolerance of check_attend of the same value: P and O rounded, on each side
    assert (a - b).abs().max() <= 2 * 2 * HALF[dtype] * 1.1 * p.v_pages.float()[same].abs().max()


def test_captured_and_replayed_with_other_lengths():
    p = Problem([1, 1, 1, 1], [300, 20, 64, 1000], 8, 2, 128, 16, BF, rot=64, seed=11)
    tables = tuple(torch.rand(1000, 32, device="cuda") for _ in range(2))
    q = p.q.clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        p.attend()                                           # loads the kernels
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p.q.copy_(q)
        _layer(p, (None, None), tables)
    for lens in ([300, 20, 64, 1000], [299, 1, 17, 3], [5, 20, 33, 999]):
        p.lens = lens
        p.lens_t.copy_(torch.tensor(lens, dtype=torch.int32))
        p.o.zero_()
        graph.replay()
        p.check_attend()
    assert p.kv.device_status() == 0


@pytest.fixture(scope="module")
def late_copy(tmp_path_factory):
    """late_copy(dst, src): a copy that lets its successor start at once and writes some 0.3 ms later."""
    import ctypes as C
    import subprocess
    from pathlib import Path

    from f2k_cuda_b200.build import NVCC_FLAGS, _nvcc
    so = tmp_path_factory.mktemp("late") / "late_copy.so"
    subprocess.run([_nvcc(), *NVCC_FLAGS, "-shared", str(Path(__file__).parent / "cpp" / "late_copy.cu"), "-o", str(so)], check=True)
    lib = C.CDLL(str(so))
    lib.late_copy.argtypes = [C.c_void_p, C.c_void_p, C.c_longlong, C.c_longlong, C.c_void_p]

    def copy(dst, src):
        assert dst.is_contiguous() and src.is_contiguous() and dst.nbytes == src.nbytes and dst.nbytes % 16 == 0
        assert lib.late_copy(dst.data_ptr(), src.data_ptr(), dst.nbytes, 600_000, torch.cuda.current_stream().cuda_stream) == 0
    return copy


@pytest.mark.parametrize("late", ["q", "lens_t", "cu", "table", "k_pages", "v_pages"])
@pytest.mark.parametrize("news,lens", [([1] * 4, [300, 20, 64, 1000]), ([200, 1, 40, 60], [300, 20, 64, 1000])], ids=["tokens", "prompts"])
def test_attend_behind_a_late_writer(late_copy, late, news, lens):
    """Every input may be written by the kernel in front while this one's blocks already stand ready."""
    p = Problem(news + [0] * 3, lens + [0] * 3, 8, 2, 128, 16, BF, seed=30)        # 7 sequences: 8 offsets; lengths padded below
    import f2k_cuda_b200 as f2k
    room = torch.zeros(8, dtype=torch.int32, device="cuda")
    room[:7] = p.lens_t
    table = torch.zeros(8, p.table.shape[1], dtype=torch.int32, device="cuda")
    table[:7] = p.table
    tensors = {"q": p.q, "lens_t": room, "cu": p.cu, "table": table, "k_pages": p.k_pages, "v_pages": p.v_pages}
    batch = f2k.PagedBatch(room[:7], table[:7], p.cu, max(news))
    right = tensors[late].clone()
    wrong = torch.zeros_like(right)
    tensors[late].copy_(wrong)
    torch.cuda.synchronize()
    late_copy(tensors[late], right)
    assert p.kv.attend(p.q, p.o, batch, p.ws, lse=p.lse)
    p.check_attend()
    assert p.kv.device_status() == 0


@pytest.mark.parametrize("late", ["q", "k", "lens_t", "table", "cos", "gain"])
def test_append_behind_a_late_writer(late_copy, late):
    import f2k_cuda_b200 as f2k
    p = Problem([70, 1, 33, 8], [70, 9, 100, 8], 8, 2, 128, 16, BF, rot=128, seed=31)
    cos, sin = torch.rand(128, 64, device="cuda"), torch.rand(128, 64, device="cuda")
    gain = torch.rand(128, device="cuda").to(BF)
    expect = [torch.empty_like(p.q), torch.empty_like(p.q)]
    tensors = {"q": p.q, "k": p.k, "lens_t": p.lens_t, "table": p.table, "cos": cos, "gain": gain}
    caches = []
    for i in range(2):
        p.k_pages.fill_(3.0)
        right = tensors[late].clone()
        if i:
            tensors[late].zero_()
            torch.cuda.synchronize()
            late_copy(tensors[late], right)
        assert p.kv.append(p.q, p.k, p.v, (gain, gain), (cos, sin), 1e-6, expect[i], p.batch)
        caches.append(p.k_pages.clone())
    assert p.kv.device_status() == 0
    assert torch.equal(expect[0], expect[1]) and torch.equal(caches[0], caches[1])


def test_two_streams_with_a_workspace_each():
    a = Problem([1] * 3, [3000, 200, 900], 8, 2, 128, 16, BF, seed=12)
    b = Problem([2] * 3, [5000, 100, 700], 8, 2, 128, 16, BF, seed=13)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for p, s in zip((a, b), streams):
            p.attend(stream=s)
    torch.cuda.synchronize()
    a.check_attend()
    b.check_attend()


def test_one_handle_two_calls_one_workspace():
    """Two calls in a row of one stream share a workspace; the second is another batch."""
    import f2k_cuda_b200 as f2k
    p = Problem([1] * 4, [2000, 30, 1500, 64], 8, 2, 128, 16, HF, seed=14)
    part = f2k.PagedBatch(p.lens_t[2:], p.table[2:], p.cu[2:], 1)           # rows 2, 3 of the same tensors
    o2, lse2 = torch.zeros_like(p.o), torch.zeros_like(p.lse)
    p.attend()
    assert p.kv.attend(p.q, o2, part, p.ws, lse=lse2)
    p.check_attend()
    assert torch.equal(o2[:2], torch.zeros_like(o2[:2]))
    whole, p.news, p.lens, p.table, p.cu = p, p.news[2:], p.lens[2:], p.table[2:], p.cu[2:]
    p.check_attend(o2, lse2)
