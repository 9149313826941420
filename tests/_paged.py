"""Batches of a paged cache for the tests, and its operators from their formulas in 64 bits."""
import math

import torch

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float8_e4m3fn: 2.0 ** -4}   # half a step, relative


class Problem:
    """`news` new tokens and `lens` keys (with them) of every sequence; pages in random order, everything that no key lies in
    filled with NaN; `pad` rows behind the last sequence."""

    def __init__(self, news, lens, heads=4, kv_heads=2, dim=128, page=16, dtype=torch.bfloat16, cache=None, window=0, rot=0,
                 interleaved=False, scales=False, token_major=False, pad=0, seed=0, gap=0, scale=0.0, n_pages=None):
        import f2k_cuda_b200 as f2k
        self.news, self.lens, self.H, self.G, self.D, self.P = list(news), list(lens), heads, kv_heads, dim, page
        self.dtype, self.ct, self.window, self.rot, self.interleaved = dtype, cache or dtype, window, rot, interleaved
        gen = self.gen = torch.Generator(device="cuda").manual_seed(seed)
        self.scale = scale or dim ** -0.5
        B, width = len(self.lens), max(1, -(-max(self.lens) // page))
        n_pages = n_pages or sum(-(-n // page) for n in self.lens) + 2
        order = torch.randperm(n_pages, generator=gen, device="cuda").tolist()
        table = torch.full((B, width), 2 ** 30, dtype=torch.int32)          # entries no key needs are outside the cache
        shape = (n_pages, page, kv_heads, dim) if token_major else (n_pages, kv_heads, page, dim)
        self.used = torch.zeros(n_pages, page, dtype=torch.bool, device="cuda")
        for b, n in enumerate(self.lens):
            for j in range(-(-n // page)):
                table[b, j] = order.pop()
                self.used[int(table[b, j]), :min(page, n - j * page)] = True
        self.table, self.lens_t = table.cuda(), torch.tensor(self.lens, dtype=torch.int32, device="cuda")
        self.cu = torch.tensor([0] + torch.tensor(self.news).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
        self.T = sum(self.news) + pad

        def pages():
            x = torch.randn(shape, generator=gen, device="cuda")
            if token_major:
                x = x.transpose(1, 2)
            x = torch.where(self.used[:, None, :, None], x, float("nan")).to(self.ct)
            return x.transpose(1, 2).contiguous().transpose(1, 2) if token_major else x

        self.k_pages, self.v_pages = pages(), pages()
        self.k_scale = self.v_scale = None
        if scales:
            self.k_scale, self.v_scale = (0.25 + torch.rand(kv_heads, generator=gen, device="cuda") for _ in range(2))
        self.kv = f2k.PagedKV(f2k.PagedKV.Config(heads, kv_heads, dim, page, n_pages, rot, interleaved, window, scale, dtype),
                              self.k_pages, self.v_pages, self.k_scale, self.v_scale)
        assert self.kv.ok(), self.kv.last_error()
        self.batch = f2k.PagedBatch(self.lens_t, self.table, self.cu, max(1, max(self.news)))
        self.gap = gap
        self.q, self.k, self.v = self.rows(heads), self.rows(kv_heads), self.rows(kv_heads)
        self.o, self.lse = self.rows(heads), torch.full((self.T, heads), 7.0, device="cuda")
        self.ws = torch.empty(self.kv.workspace_size_bytes(self.batch), dtype=torch.uint8, device="cuda").fill_(0xAA)

    def rows(self, heads):
        """[tokens, heads, dim], token rows `gap` elements apart."""
        wide = torch.randn(self.T, heads * self.D + self.gap, generator=self.gen, device="cuda").to(self.dtype)
        return wide[:, :heads * self.D].unflatten(1, (heads, self.D))

    def attend(self, **more):
        assert self.kv.attend(self.q, self.o, self.batch, self.ws, lse=self.lse, **more), self.kv.last_error()

    def keys(self, b, pages):
        """[kv heads, keys, dim] of sequence b in 64 bits."""
        n = self.lens[b]
        x = pages[self.table[b, :-(-n // self.P)].long()].transpose(1, 2).double().flatten(0, 1)[:n].transpose(0, 1)
        s = self.k_scale if pages is self.k_pages else self.v_scale
        return x if s is None else x * s.double()[:, None, None]

    def check_attend(self, o=None, lse=None):
        """Outputs against the formula. With w the softmax weights and A = sum w |v|: the weights are rounded by at most half
        a step u each (u A), the output by u |o|; a score s = scale sum q k is off by less than 2^-20 scale sum |q k| =: d
        (fp32 sums of at most 128 products, the exponent's rounding included), which changes weights by a factor within
        e^(+-2 d); 2^-20 A covers the fp32 sums over the keys (blocks of 16 keys added one after the other) and the
        approximate exponent. fp16 weights below 2^-14 of the largest are off by up to 2^-25 of it each."""
        o, lse = self.o if o is None else o, self.lse if lse is None else lse
        u = HALF[self.dtype]
        uw = HALF[torch.float16] if self.ct is torch.float8_e4m3fn else u
        begin, group = self.cu.tolist(), self.H // self.G
        for b, (n, m) in enumerate(zip(self.news, self.lens)):
            if n == 0:
                continue
            k, v = self.keys(b, self.k_pages), self.keys(b, self.v_pages)
            q = self.q[begin[b]:begin[b + 1]].double().transpose(0, 1).unflatten(0, (self.G, group))       # [G, g, n, D]
            pos = torch.arange(m - n, m, device="cuda")[:, None]
            j = torch.arange(m, device="cuda")[None]
            seen = (j <= pos) & (j > pos - self.window if self.window else True)
            x = (q @ k.mT[:, None] * self.scale).masked_fill(~seen, -math.inf)
            d = ((q.abs() @ k.abs().mT[:, None]).masked_fill(~seen, 0).amax(-1) * self.scale * 2.0 ** -20) if m else torch.zeros_like(x.sum(-1))
            want_lse = torch.logsumexp(x, -1)
            none = want_lse == -math.inf
            w = torch.exp(x - torch.where(none, 0.0, want_lse)[..., None])
            want, mass = w @ v[:, None], w @ v.abs()[:, None]
            tiny = 2.0 ** -25 * v.abs().sum(1)[:, None, None] * torch.exp(x.amax(-1, keepdim=True) - torch.where(none, 0.0, want_lse)[..., None]).nan_to_num(0) \
                if uw == HALF[torch.float16] and m else 0.0
            tol = 1.01 * (uw + 2 * d[..., None] + 2.0 ** -20) * mass + 1.01 * u * want.abs() + tiny + 1e-30
            if self.dtype is torch.float16:
                tol = tol + 2.0 ** -25
            got = o[begin[b]:begin[b + 1]].double().transpose(0, 1).unflatten(0, (self.G, group))
            got_lse = lse[begin[b]:begin[b + 1]].double().T.unflatten(0, (self.G, group))
            assert torch.isfinite(got).all(), f"sequence {b}: {int((~torch.isfinite(got)).sum())} values are not finite"
            off = (got - want).abs() / tol
            assert off.max() <= 1, f"sequence {b} (new {n}, keys {m}): {off.max():.3g} times the tolerance at {divmod(int(off.argmax()), self.D)}"
            assert torch.equal(got_lse[none], torch.full_like(got_lse[none], -math.inf)) and not got[none].any()
            off = ((got_lse - want_lse)[~none].abs() / (d + 2.0 ** -20 + 2.0 ** -23 * want_lse.abs())[~none])
            assert off.numel() == 0 or off.max() <= 1, f"sequence {b}: lse {off.max():.3g} times its tolerance"


def rotate(x, cos, sin, rot, interleaved):
    """[tokens, heads, dim] in 64 bits, cos and sin [tokens, rot / 2]."""
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    c, s = cos[:, None].double(), sin[:, None].double()
    y = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2) if interleaved else torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([y, x[..., rot:]], -1)
