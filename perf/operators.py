"""Performance cases of the paged key/value cache: appending to it, and attention over it for single tokens and prompts.

A case names what is called ("op") and its sizes:

  append   PagedKV.append    new tokens of a batch of sequences: per-head RMSNorm and rotation of Q and K on the way,
                             K and V into the sequences' pages
  attend   PagedKV.attend    the new tokens' queries over the pages of their sequences, causal
  layer    both, one after the other, as a decoder layer calls them

A batch is `seqs` sequences; each has between new_lo and new_hi new tokens behind between past_lo and past_hi cached
ones (drawn by lens_seed over their logarithm; the first sequence has the most of both). Pages are scattered over the
cache at random. K and V of a cached token, and the projections of a new one, are N(0, 1) as after QK-norm; pages hold
values of earlier sequences where no token lies.
"""
import numpy as np
import torch

own = False

EPS = 1e-6
THETA = 1e6
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn}
SIZES = {"bf16": 2, "f16": 2, "e4m3": 1}


def _case(name, op, seqs, new, past, heads=32, kv_heads=8, dim=128, page=16, dtype="bf16", cache=None, rot=None,
          interleaved=False, norm=True, window=0, lse=False, lens_seed=1):
    c = {"op": op, "seqs": seqs, "new_lo": new[0], "new_hi": new[1], "past_lo": past[0], "past_hi": past[1],
         "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype, "cache": cache or dtype,
         "rot": dim if rot is None else rot, "interleaved": interleaved, "norm": norm, "window": window, "lse": lse,
         "lens_seed": lens_seed}
    return {"name": name, **c} if name else c


def listed():
    return [
        # One decoding step of eight requests: a launch and a few rows.
        _case("append_8_tokens", "append", 8, (1, 1), (100, 900)),
        # Prompts of a batch, ragged, as the prompt phase writes them.
        _case("append_prompts", "append", 6, (77, 3500), (0, 0), page=64),
        # The same into an 8-bit cache: five query heads a key head, 64 wide, a quarter of each head turned in
        # neighbouring pairs, no QK-norm.
        _case("append_prompts_e4m3", "append", 40, (100, 2000), (0, 300), heads=20, kv_heads=4, dim=64, page=32, dtype="f16",
              cache="e4m3", rot=16, interleaved=True, norm=False),
        # One request, one token: latency.
        _case("token_1x1000", "attend", 1, (1, 1), (999, 999)),
        # A serving batch in the middle of its answers.
        _case("tokens_64_ragged", "attend", 64, (1, 1), (200, 8191)),
        # Long contexts: reading the cache is all there is.
        _case("tokens_16x32k", "attend", 16, (1, 1), (20000, 32767), page=64),
        # An 8-bit cache under five query heads a key head.
        _case("tokens_96_e4m3", "attend", 96, (1, 1), (1000, 6000), heads=40, dtype="f16", cache="e4m3", page=32),
        # Four drafted tokens of each request verified at once, in a layer with a window, 64-wide heads.
        _case("verify_24x4_window", "attend", 24, (4, 4), (500, 16000), heads=64, dim=64, page=32, dtype="f16", window=2048,
              lse=True),
        # One prompt as long as the image model's text stream.
        _case("prompt_512", "attend", 1, (512, 512), (0, 0)),
        # Prompts of a batch, ragged, three query heads a key head.
        _case("prompts_8_ragged", "attend", 8, (60, 3000), (0, 0), heads=24, dtype="f16", page=32),
        # The largest: one long prompt.
        _case("prompt_8192", "attend", 1, (8192, 8192), (0, 0), page=64),
        # A piece of a long prompt behind what is cached already; a key head for every query head, 64 wide.
        _case("prompt_chunk_1024", "attend", 1, (1024, 1024), (15001, 15001), heads=16, kv_heads=16, dim=64, page=128, lse=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    """Another case of the same ranges: 1 to 96 sequences, 1 to 8192 new tokens, up to 32768 keys, 1 to 64 heads, 1 to 16 query
    heads a key head."""
    while True:
        op, kind = rng.choice([("append", "tokens"), ("append", "prompts"), ("attend", "tokens"), ("attend", "tokens"), ("attend", "tokens"),
                               ("attend", "drafts"), ("attend", "prompts"), ("attend", "prompts"), ("attend", "chunks"), ("layer", "tokens"),
                               ("layer", "prompts")])
        kv_heads = rng.choice([1, 2, 4, 8, 8, 8, 16])
        group = rng.choice([1, 2, 3, 4, 4, 4, 5, 7, 8, 16])
        dtype = rng.choice(["bf16", "bf16", "f16"])
        dim = rng.choice([64, 128, 128])
        rot = rng.choice([dim, dim, dim // 2])
        seqs = _log_int(rng, 1, 96)
        if kind in ("tokens", "drafts"):
            n = 1 if kind == "tokens" else rng.randint(2, 8)
            new = (n, n)
            past_hi = _log_int(rng, 16, 32767)
            past = (_log_int(rng, 1, past_hi), past_hi)
        else:
            seqs = min(seqs, 12)
            new_hi = _log_int(rng, 40, 8192)
            new = (_log_int(rng, max(1, new_hi // 30), new_hi), new_hi)
            past = (0, 0) if kind == "prompts" else (0, _log_int(rng, 100, 20000))
        c = _case(None, op, seqs, new, past, kv_heads * group, kv_heads, dim, rng.choice([16, 16, 32, 64, 128, 256]), dtype,
                  "e4m3" if rng.random() < 0.25 else dtype, rot, rng.random() < 0.3, rng.random() < 0.7,
                  rng.choice([0, 0, 0, _log_int(rng, 64, 4096)]), rng.random() < 0.3, rng.randint(1, 10 ** 6))
        w, n = work(c), _lens(c)
        scores = seqs * c["heads"] * float(n[0].max()) * float(n[1].max())
        if c["heads"] <= 64 and w["bytes"] <= 2.0e9 and w["flops"] <= 5.4e11 and scores <= 2.0e9 \
                and seqs * float(n[1].max()) * kv_heads * dim <= 6e8:
            return c


def _lens(c):
    """New tokens and keys (new ones included) of every sequence."""
    r = np.random.RandomState(c["lens_seed"])

    def spread(lo, hi):
        n = np.exp(r.uniform(np.log(lo + 1), np.log(hi + 1), c["seqs"])).round().astype(np.int64) - 1
        n[0] = hi
        return np.clip(n, lo, hi)

    new = spread(c["new_lo"], c["new_hi"])
    return new, spread(c["past_lo"], c["past_hi"]) + new


def prepare(case, seed):
    c = case
    new, lens = _lens(c)
    B, H, G, D, P = c["seqs"], c["heads"], c["kv_heads"], c["dim"], c["page"]
    T = int(new.sum())
    width = int(-(-lens.max() // P))
    n_pages = int((-(-lens // P)).sum()) + 3
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dt, ct = TYPES[c["dtype"]], TYPES[c["cache"]]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", dtype=torch.float32 if ct is not dt else dt, generator=gen)

    def cache():
        out = torch.empty(n_pages, G, P, D, device="cuda", dtype=ct)
        out.copy_(normal(n_pages, G, P, D))
        return out

    order = torch.randperm(n_pages, device="cuda", generator=gen).to(torch.int32)
    have = torch.from_numpy(-(-lens // P)).cuda()
    first = have.cumsum(0) - have
    col = torch.arange(width, device="cuda")
    table = torch.where(col[None] < have[:, None], order[(first[:, None] + col[None]).clamp(max=n_pages - 1)], 0).to(torch.int32)

    s = {"case": c, "B": B, "T": T, "max_new": int(new.max()), "max_len": int(lens.max()), "width": width,
         "k_pages": cache(), "v_pages": cache(), "table": table,
         "lens": torch.from_numpy(lens.astype(np.int32)).cuda(),
         "cu": torch.from_numpy(np.concatenate([[0], new.cumsum()]).astype(np.int32)).cuda(),
         "q": normal(T, H, D).to(dt), "k": normal(T, G, D).to(dt), "v": normal(T, G, D).to(dt),
         "q_out": torch.empty(T, H, D, device="cuda", dtype=dt), "o": torch.empty(T, H, D, device="cuda", dtype=dt),
         "lse": torch.empty(T, H, device="cuda") if c["lse"] else None, "gains": (None, None), "scales": (None, None)}
    if c["norm"]:
        s["gains"] = tuple((0.9 + 0.2 * torch.rand(D, device="cuda", generator=gen)).to(dt) for _ in range(2))
    if c["cache"] == "e4m3" and c["op"] == "attend":     # what the rows of each head were divided by
        s["scales"] = tuple(0.5 + torch.rand(G, device="cuda", generator=gen) for _ in range(2))
    if c["op"] == "append" or c["op"] == "layer":
        freq = THETA ** (-torch.arange(c["rot"] // 2, device="cuda", dtype=torch.float64) * 2 / c["rot"])
        angle = torch.arange(s["max_len"], device="cuda", dtype=torch.float64)[:, None] * freq
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    if own:
        import f2k_cuda_b200 as f2k
        s["kv"] = kv = f2k.PagedKV(f2k.PagedKV.Config(H, G, D, P, n_pages, rot_dim=c["rot"], interleaved=c["interleaved"],
                                                      window=c["window"], dtype=dt), s["k_pages"], s["v_pages"], *s["scales"])
        if not kv.ok():
            raise RuntimeError(kv.last_error())
        s["batch"] = f2k.PagedBatch(s["lens"], table, None if new.max() == 1 and new.min() == 1 else s["cu"], s["max_new"])
        s["workspace"] = torch.empty(kv.workspace_size_bytes(s["batch"]), dtype=torch.uint8, device="cuda")
    return s


def _places(s):
    """Sequence, number inside it and position of every new token."""
    tok = torch.arange(s["T"], device="cuda")
    cu = s["cu"].long()
    seq = torch.searchsorted(cu, tok, right=True) - 1
    inside = tok - cu[seq]
    return seq, inside, s["lens"].long()[seq] - (cu[seq + 1] - cu[seq]) + inside


def _turned(x, gain, cos, sin, c):
    """RMSNorm of every head row and the rotation, in 32 bits."""
    if gain is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * gain.float()
    r = c["rot"]
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if c["interleaved"] else (x[..., :r // 2], x[..., r // 2:r])
    cos, sin = cos[:, None], sin[:, None]
    y = [a * cos - b * sin, b * cos + a * sin]
    y = torch.stack(y, -1).flatten(-2) if c["interleaved"] else torch.cat(y, -1)
    return torch.cat([y, x[..., r:]], -1)


def _plain_append(s):
    c = s["case"]
    seq, _, pos = _places(s)
    page, row = s["table"][seq, pos // c["page"]].long(), pos % c["page"]
    cos, sin = s["cos"][pos], s["sin"][pos]
    q = _turned(s["q"].float(), s["gains"][0], cos, sin, c)
    k, v = _turned(s["k"].float(), s["gains"][1], cos, sin, c), s["v"]
    if c["cache"] == "e4m3":
        k, v = k.clamp(-448, 448), v.float().clamp(-448, 448)
    s["k_pages"][page, :, row] = k.to(s["k_pages"].dtype)
    s["v_pages"][page, :, row] = v.to(s["v_pages"].dtype)
    return q.to(s["q"].dtype)


def _plain_attend(s, q):
    """Queries padded to [sequence, head, token], pages gathered, a full matrix of scores, in 32 bits."""
    c = s["case"]
    B, H, G, D, N = s["B"], c["heads"], c["kv_heads"], c["dim"], s["max_new"]
    seq, inside, pos = _places(s)
    gather = lambda x: x[s["table"].long()].transpose(1, 2).reshape(B, G, -1, D).float()  # noqa: E731
    k, v = gather(s["k_pages"]), gather(s["v_pages"])
    if s["scales"][0] is not None:
        k, v = k * s["scales"][0][:, None, None], v * s["scales"][1][:, None, None]
    key = torch.arange(k.shape[2], device="cuda")
    v = torch.where((key < s["lens"][:, None])[:, None, :, None], v, 0.0)
    padded = torch.zeros(B, N, H, D, device="cuda")
    padded[seq, inside] = q.float()
    at = torch.full((B, N), -1, device="cuda", dtype=torch.int64)
    at[seq, inside] = pos
    seen = key <= at[..., None]
    if c["window"]:
        seen &= key > at[..., None] - c["window"]
    x = padded.view(B, N, G, H // G, D).permute(0, 2, 3, 1, 4).reshape(B, G, H // G * N, D)
    x = (x * D ** -0.5) @ k.transpose(-1, -2)
    x = x.view(B, G, H // G, N, -1).masked_fill_(~seen[:, None, None], float("-inf"))
    top = x.amax(-1, keepdim=True)
    x = x.sub_(torch.where(top == float("-inf"), 0.0, top)).exp_()
    total = x.sum(-1, keepdim=True)
    o = (x.view(B, G, H // G * N, -1) @ v).view(B, G, H // G, N, D) / torch.where(total == 0, 1.0, total)
    o = o.permute(0, 3, 1, 2, 4).reshape(B, N, H, D)[seq, inside].to(q.dtype)
    if not c["lse"]:
        return o
    return o, (top + total.log())[..., 0].permute(0, 3, 1, 2).reshape(B, N, H)[seq, inside]


def run(s):
    op = s["case"]["op"]
    if not own:
        if op == "append":
            return _plain_append(s), s["k_pages"], s["v_pages"]
        if op == "attend":
            return _plain_attend(s, s["q"])
        return _plain_attend(s, _plain_append(s)), s["k_pages"], s["v_pages"]
    kv, ok, q = s["kv"], True, s["q"]
    if op != "attend":
        ok = kv.append(q, s["k"], s["v"], s["gains"], (s["cos"], s["sin"]), EPS, s["q_out"], s["batch"])
        q = s["q_out"]
    if op != "append":
        ok = ok and kv.attend(q, s["o"], s["batch"], s["workspace"], lse=s["lse"])
    if not ok:
        raise RuntimeError(kv.last_error())
    if op == "append":
        return s["q_out"], s["k_pages"], s["v_pages"]
    o = (s["o"], s["lse"]) if s["case"]["lse"] else s["o"]
    return o if op == "attend" else (o, s["k_pages"], s["v_pages"])


def work(case):
    """append: Q, K and V read once and written once. attend: Q read, O written, every row of K and V that some query of
    the sequence sees read once; two products a query head and visible key."""
    c = case
    new, lens = _lens(c)
    H, G, D, size = c["heads"], c["kv_heads"], c["dim"], SIZES[c["cache"]]
    T, W = float(new.sum()), c["window"]
    total, flops = 0.0, 0.0
    if c["op"] != "attend":
        tables = float(min(T, lens.max())) * c["rot"] * 4
        total += T * H * D * 4 + T * G * D * 2 * (2 + size) + tables
        flops += T * (H + G) * D * 8
    if c["op"] != "append":
        seen = np.minimum(lens, W + new - 1) if W else lens
        total += T * H * D * 4 + float(seen.sum()) * G * D * 2 * size
        flops += 4.0 * H * D * float(sum(_visible(int(n), int(m), W) for n, m in zip(new, lens)))
    return {"bytes": total, "flops": flops}


def _visible(new, length, window):
    """Keys seen by the last `new` tokens of a sequence, added up."""
    n = np.arange(length - new + 1, length + 1)
    return (np.minimum(n, window) if window else n).sum()


def exact(case, seed):
    """What run() gives, from the formulas in 64 bits, a sequence and a head at a time. Attention is over what the cache
    holds, in its type."""
    c, s = case, prepare(case, seed)
    new, lens = _lens(c)
    H, G, D, P, r = c["heads"], c["kv_heads"], c["dim"], c["page"], c["rot"]
    K, V, q = s["k_pages"].double(), s["v_pages"].double(), s["q"].double()
    begin = np.concatenate([[0], new.cumsum()])

    def spin(x, gain, positions):
        if gain is not None:
            x = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / D + EPS) * gain.double()
        freq = torch.tensor([THETA ** (-2.0 * i / r) for i in range(r // 2)], dtype=torch.float64, device="cuda")
        z = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), positions[:, None, None].double() * freq)
        y = x.clone()
        if c["interleaved"]:
            w = torch.complex(x[..., 0:r:2].contiguous(), x[..., 1:r:2].contiguous()) * z
            y[..., 0:r:2], y[..., 1:r:2] = w.real, w.imag
        else:
            w = torch.complex(x[..., :r // 2].contiguous(), x[..., r // 2:r].contiguous()) * z
            y[..., :r // 2], y[..., r // 2:r] = w.real, w.imag
        return y

    if c["op"] != "attend":
        turned = torch.empty_like(q)
        for b in range(len(new)):
            rows = slice(int(begin[b]), int(begin[b + 1]))
            pos = torch.arange(int(lens[b] - new[b]), int(lens[b]), device="cuda")
            where = s["table"][b].long()[pos // P]
            turned[rows] = spin(q[rows], s["gains"][0], pos)
            K[where, :, pos % P] = spin(s["k"][rows].double(), s["gains"][1], pos)
            V[where, :, pos % P] = s["v"][rows].double()
        if c["op"] == "append":
            return turned, K, V
        written = K, V
        q, K, V = (x.to(like.dtype).double() for x, like in ((turned, s["q"]), (K, s["k_pages"]), (V, s["v_pages"])))
    o = torch.zeros(s["T"], H, D, dtype=torch.float64, device="cuda")
    lse = torch.full((s["T"], H), -float("inf"), dtype=torch.float64, device="cuda")
    for b in range(len(new)):
        n, m = int(new[b]), int(lens[b])
        pages = s["table"][b, :-(-m // P)].long()
        pos = torch.arange(m - n, m, device="cuda")[:, None]
        j = torch.arange(m, device="cuda")[None]
        hidden = (j > pos) | ((j <= pos - c["window"]) if c["window"] else False)
        for g in range(G):
            keys, values = (x[pages, g].reshape(-1, D)[:m] for x in (K, V))
            if s["scales"][0] is not None:
                keys, values = keys * s["scales"][0][g].double(), values * s["scales"][1][g].double()
            for h in range(g * (H // G), (g + 1) * (H // G)):
                x = (q[int(begin[b]):int(begin[b + 1]), h] @ keys.T / D ** 0.5).masked_fill_(hidden, -float("inf"))
                t = torch.logsumexp(x, -1)
                o[int(begin[b]):int(begin[b + 1]), h] = torch.exp(x - t[:, None]) @ values
                lse[int(begin[b]):int(begin[b + 1]), h] = t
    out = (o, lse) if c["lse"] else o
    return out if c["op"] == "attend" else (out, *written)
