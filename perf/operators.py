"""The paged 4-bit KV cache's operators as cases that can be timed.

A serving program with many requests keeps their keys and values in pages of
16 to 128 tokens, 4 bits a channel with one fp16 scale per (token, key head).
Each step it lays out the batch on the GPU (`paged_batch`: pages taken from
the free list, slots and positions of the new tokens), and for every layer
writes the new rows (`paged_append`), attends over the pages
(`paged_attention`, one new token per request or ragged chunks of them) and,
where a prompt is continued by other kernels or its cache is copied, reads
rows back (`paged_gather`).

Head shapes are 32 query / 8 key heads, 64 / 8 and 32 / 2 of dimension 128,
and the same counts of dimension 64.  Keys are Gaussian with offsets ~ N(0, 2)
per (key head, channel); pages are scattered over the pool.  `draw` spreads
cases of the same paths over 1 to 1024 requests, contexts of none to 32768
tokens, both 16-bit types, page sizes of 16 to 128 and sliding windows.

    cache   int8 [pages, key heads, page, D / 2] codes (the even channel in
            the low nibble), fp16 [pages, key heads, page] scales
    scale = fp16(max(amax |x|, 1e-5) / 7), code = round_half_even(x / scale)
    out_i = sum_j softmax_j(sm q_i . k_j) v_j over the visible keys j <= pos_i
            (and j > pos_i - window), k_j and v_j = code * scale
"""

import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
MOST_KEYS = 16 * 32768 * 8             # requests * context * key heads of the largest decode case
MOST_PAIRS = 32 * 2 * 8192 * 8192      # heads * requests * chunk * keys of the largest chunk case, padded


def listed():
    return [
        # a decode step of a small batch: the layout of its batch, launch latency and little else
        dict(name="batch_decode_r24", path="batch", requests=24, page=64, ctx_lo=300, ctx_hi=32000, new_lo=1, new_hi=1,
             tokens=24),
        # a step with prompts in it, padded to the token count of a captured graph
        dict(name="batch_mixed_r1000", path="batch", requests=1000, page=16, ctx_lo=1, ctx_hi=9000, new_lo=1, new_hi=700,
             tokens=150000),
        # a decode step's new rows into one layer's pages, read back
        dict(name="append_t16", path="append", tokens=16, padded=16, kv_heads=8, dim=128, page=64, dtype="bf16"),
        # an 8K prompt's rows, slices of a fused projection
        dict(name="append_t8k", path="append", tokens=8192, padded=8192, kv_heads=8, dim=128, page=64, dtype="bf16"),
        # chunks of several prompts of an fp16 model with heads of 64, padded rows behind them
        dict(name="append_t30k_d64", path="append", tokens=30011, padded=30720, kv_heads=8, dim=64, page=16, dtype="fp16"),
        # one user, 8K context
        dict(name="decode_r1_8k", path="attend", requests=1, decodes=1, ctx_lo=8191, ctx_hi=8191, new_lo=1, new_hi=1,
             q_heads=32, kv_heads=8, dim=128, page=64, window=0, dtype="bf16", lse=False),
        # continuous batching: contexts of 700 to 32000 tokens
        dict(name="decode_r48_ragged", path="attend", requests=48, decodes=48, ctx_lo=700, ctx_hi=32000, new_lo=1, new_hi=1,
             q_heads=32, kv_heads=8, dim=128, page=16, window=0, dtype="bf16", lse=False),
        # a full batch of the longest contexts: HBM bandwidth
        dict(name="decode_r16_32k", path="attend", requests=16, decodes=16, ctx_lo=32767, ctx_hi=32767, new_lo=1, new_hi=1,
             q_heads=32, kv_heads=8, dim=128, page=64, window=0, dtype="bf16", lse=False),
        # 16 query heads on each of two key heads of 64 channels, fp16, a sliding window, many short requests
        dict(name="decode_r200_d64_window", path="attend", requests=200, decodes=200, ctx_lo=100, ctx_hi=13000, new_lo=1,
             new_hi=1, q_heads=32, kv_heads=2, dim=64, page=32, window=4096, dtype="fp16", lse=False),
        # a 2K chunk of a prompt whose first 8K tokens are in the cache
        dict(name="chunk_2k_at_8k", path="attend", requests=1, decodes=0, ctx_lo=8192, ctx_hi=8192, new_lo=2048, new_hi=2048,
             q_heads=32, kv_heads=8, dim=128, page=64, window=0, dtype="bf16", lse=True),
        # chunks next to decode steps in one call, odd sizes
        dict(name="mixed_r12", path="attend", requests=12, decodes=8, ctx_lo=37, ctx_hi=9001, new_lo=33, new_hi=515,
             q_heads=64, kv_heads=8, dim=128, page=32, window=0, dtype="bf16", lse=False),
        # two whole prompts of up to 8K tokens, fp16
        dict(name="prompts_r2_8k", path="attend", requests=2, decodes=0, ctx_lo=0, ctx_hi=0, new_lo=5003, new_hi=8192,
             q_heads=32, kv_heads=8, dim=128, page=128, window=0, dtype="fp16", lse=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    path = rng.choice(["batch", "append", "decode", "decode", "chunk", "chunk"])
    page = rng.choice([16, 16, 32, 64, 128])
    if path == "batch":
        lo, hi = sorted((_log_int(rng, 1, 16000), _log_int(rng, 1, 16000)))
        n = _log_int(rng, 1, 1000)
        new = _log_int(rng, 1, 700)
        c = dict(path="batch", requests=n, page=page, ctx_lo=lo, ctx_hi=hi, new_lo=1, new_hi=new)
        c["tokens"] = sum(_lengths(n, 1, new, 1)) + rng.choice([0, rng.randint(1, 500)])
        return c
    q_heads, kv_heads = rng.choice([(32, 8), (32, 8), (64, 8), (32, 2)])
    c = dict(kv_heads=kv_heads, dim=rng.choice([128, 128, 64]), page=page, dtype=rng.choice(["bf16", "bf16", "fp16"]))
    if path == "append":
        n = _log_int(rng, 1, 30000)
        return dict(c, path="append", tokens=n, padded=n + rng.choice([0, rng.randint(1, 300)]))
    c.update(path="attend", q_heads=q_heads, window=rng.choice([0, 0, 0, _log_int(rng, 64, 8192)]), lse=rng.random() < 0.3)
    if path == "decode":
        hi = _log_int(rng, 64, 32000)
        n = _log_int(rng, 1, min(256, MOST_KEYS // (2 * hi * kv_heads)))
        return dict(c, requests=n, decodes=n, ctx_lo=_log_int(rng, 1, hi), ctx_hi=hi, new_lo=1, new_hi=1)
    hi = _log_int(rng, 2, 4000)
    ctx = rng.choice([0, _log_int(rng, 1, 16000)])
    n = _log_int(rng, 1, max(1, min(16, MOST_PAIRS // (2 * q_heads * hi * (hi + ctx)))))
    return dict(c, requests=n, decodes=rng.choice([0, rng.randint(0, n - 1)]), ctx_lo=min(ctx, _log_int(rng, 1, 16000)),
                ctx_hi=ctx, new_lo=_log_int(rng, 1, hi), new_hi=hi)


# ---------------------------------------------------------------------------
# sizes, the same for every seed
# ---------------------------------------------------------------------------


def _lengths(n, lo, hi, salt):
    """n lengths of lo to hi, spread over their logarithm in no order."""
    if n == 1 or lo >= hi or lo == 0:
        return [hi] * n
    return [int(round(lo * (hi / lo) ** ((i * 0.6180339887 + 0.37 * salt) % 1.0))) for i in range(n)]


def _requests(c):
    """(tokens in the cache before, new tokens) of each request."""
    n = c["requests"]
    ctx = _lengths(n, c["ctx_lo"], c["ctx_hi"], 0)
    new = _lengths(n, c["new_lo"], c["new_hi"], 1)
    for i in range(c.get("decodes", 0)):
        new[i] = 1
    return ctx, new


def _pages(tokens, page):
    return -(-tokens // page)


def work(c):
    if c["path"] == "batch":
        ctx, new = _requests(c)
        taken = sum(_pages(a + b, c["page"]) - _pages(a, c["page"]) for a, b in zip(ctx, new))
        held = sum(_pages(a + b, c["page"]) - a // c["page"] for a, b in zip(ctx, new))
        return dict(bytes=8 * len(ctx) + 4 * taken + 4 * taken + 4 * (held - taken) + 8 * len(ctx) + 16 * c["tokens"], flops=0)
    if c["path"] == "append":
        rows = 2 * c["kv_heads"]
        cache = c["tokens"] * rows * (c["dim"] // 2 + 2)
        return dict(bytes=c["tokens"] * rows * 2 * c["dim"] + cache + c["padded"] * (8 + rows * 2 * c["dim"]), flops=0)
    ctx, new = _requests(c)
    keys, pairs = 0, 0
    for a, b in zip(ctx, new):
        w = c["window"] or a + b
        first = max(0, a - w + 1)
        keys += a + b - first
        pairs += sum(min(w, a + i + 1) for i in range(b))
    rows = sum(new) * c["q_heads"]
    return dict(bytes=keys * c["kv_heads"] * (c["dim"] + 4) + rows * c["dim"] * 4 + 4 * _pages(keys, c["page"])
                + (4 * rows if c["lse"] else 0), flops=4 * c["dim"] * c["q_heads"] * pairs)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def _pool(g, pages, heads, page, dim, offset):
    """Codes and scales of Gaussian rows for every slot of a pool."""
    x = torch.randn(pages, heads, page, dim, generator=g, device="cuda")
    if offset is not None:
        x += offset[:, None, :]
    scale = (x.abs().amax(-1).clamp(min=1e-5) / 7).half()
    x /= scale.float()[..., None]
    code = x.round_().clamp_(-8, 7).to(torch.int8) & 15
    return code[..., 0::2] | (code[..., 1::2] << 4), scale


def _table(g, held, width, pages):
    """A block table of scattered pages, -1 behind each row's last, and the pages left over."""
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    held = torch.tensor(held, device="cuda")
    at = torch.arange(width, device="cuda")
    first = held.cumsum(0) - held
    table = order[(first[:, None] + at).clamp(max=pages - 1)]
    table[at >= held[:, None]] = -1
    return table, order[int(held.sum()):].contiguous()


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case=dict(c))
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    if c["path"] == "batch":
        ctx, new = _requests(c)
        held = [_pages(a, c["page"]) for a in ctx]
        total = [_pages(a + b, c["page"]) for a, b in zip(ctx, new)]
        s["table"], s["free"] = _table(g, held, max(total) + 3, sum(total) + 50)
        s["ctx"], s["new"] = i32(ctx), i32(new)
        return s
    h, d, page, dt = c["kv_heads"], c["dim"], c["page"], TYPES[c["dtype"]]
    offset = math.sqrt(2.0) * torch.randn(h, d, generator=g, device="cuda")
    if c["path"] == "append":
        pages = _pages(c["tokens"], page) + 5
        s["kp"], s["ks"] = _pool(g, pages, h, page, d, offset)
        s["vp"], s["vs"] = _pool(g, pages, h, page, d, None)
        x = torch.randn(c["padded"], 6, h, d, generator=g, device="cuda")      # q (4 per key head), k and v of one projection
        x[:, 4] += offset
        x = x.to(dt)
        s["k"], s["v"] = x[:, 4], x[:, 5]
        order = torch.randperm(pages, generator=g, device="cuda")
        t = torch.arange(c["padded"], device="cuda")
        slots = order[(t // page).clamp(max=pages - 1)] * page + t % page
        s["slots"] = torch.where(t < c["tokens"], slots, -1)
        return s
    ctx, new = _requests(c)
    total = [_pages(a + b, page) for a, b in zip(ctx, new)]
    pages = sum(total) + 3
    s["table"], _ = _table(g, total, max(total) + 1, pages)
    s["kp"], s["ks"] = _pool(g, pages, h, page, d, offset)
    s["vp"], s["vs"] = _pool(g, pages, h, page, d, None)
    s["q"] = torch.randn(sum(new), c["q_heads"], d, generator=g, device="cuda").to(dt)
    s["lens"] = i32([a + b for a, b in zip(ctx, new)])
    s["cu"] = None if max(new) == 1 else i32([0] + torch.tensor(new).cumsum(0).tolist())
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------


def _own_run(s):
    import hyquant_amd as hq
    c = s["case"]
    if c["path"] == "batch":
        b = hq.paged_batch(s["ctx"], s["new"], s["table"], s["free"], c["page"], c["tokens"])
        return dict(table=s["table"], cu=b.cu_seqlens, lens=b.seq_lens, slots=b.slots, positions=b.positions,
                    used=b.pages_used)
    if c["path"] == "append":
        hq.paged_append(s["k"], s["v"], s["slots"], s["kp"], s["vp"], s["ks"], s["vs"])
        k, v = hq.paged_gather(s["slots"], s["kp"], s["vp"], s["ks"], s["vs"], dtype=s["k"].dtype)
        return dict(k=k, v=v, k_scale=s["ks"], v_scale=s["vs"])
    if c["lse"]:
        out, lse = hq.paged_attention(s["q"], s["kp"], s["vp"], s["ks"], s["vs"], s["table"], s["lens"], s["cu"],
                                      window=c["window"], return_lse=True)
        return dict(out=out, lse=lse)
    return dict(out=hq.paged_attention(s["q"], s["kp"], s["vp"], s["ks"], s["vs"], s["table"], s["lens"], s["cu"],
                                       window=c["window"]))


def run(s):
    if own:
        return _own_run(s)
    path = s["case"]["path"]
    return _plain_batch(s) if path == "batch" else _plain_append(s) if path == "append" else _plain_attend(s)


def _plain_batch(s):
    c, table, free = s["case"], s["table"], s["free"]
    page, n = c["page"], c["requests"]
    ctx, new = s["ctx"].long(), s["new"].long()
    lens = ctx + new
    old = (ctx + page - 1) // page
    need = (lens + page - 1) // page - old
    first = need.cumsum(0) - need
    at = torch.arange(table.shape[1], device="cuda")
    take = first[:, None] + at - old[:, None]
    fresh = (at >= old[:, None]) & (at < (old + need)[:, None])
    table.copy_(torch.where(fresh, free[take.clamp(0, len(free) - 1)], table))
    cu = torch.zeros(n + 1, dtype=torch.int64, device="cuda")
    cu[1:] = new.cumsum(0)
    t = torch.arange(c["tokens"], device="cuda")
    ends = torch.zeros(c["tokens"] + 1, dtype=torch.int64, device="cuda").index_add_(0, cu[1:], torch.ones_like(new))
    r = ends.cumsum(0)[:-1].clamp(max=n - 1)
    live = t < cu[-1]
    pos = torch.where(live, ctx[r] + t - cu[r], 0)
    slots = table[r, pos // page].long() * page + pos % page
    return dict(table=table, cu=cu.int(), lens=lens.int(), slots=torch.where(live, slots, -1),
                positions=torch.where(live, pos, -1), used=need.sum().int().reshape(1))


def _quantise(x):
    x = x.float()
    scale = (x.abs().amax(-1).clamp(min=1e-5) / 7).half()
    code = torch.round(x / scale.float()[..., None]).clamp(-8, 7).to(torch.int8) & 15
    return code[..., 0::2] | (code[..., 1::2] << 4), scale


def _unpack(packed):
    """fp32 codes of packed rows."""
    low, high = (packed << 4) >> 4, packed >> 4
    return torch.stack((low, high), -1).flatten(-2).float()


def _plain_append(s):
    c = s["case"]
    n, page = c["tokens"], c["page"]
    slots = s["slots"][:n]
    at, off = slots // page, slots % page
    out = {}
    for name in "kv":
        codes, scales, x = s[name + "p"], s[name + "s"], s[name]
        codes[at, :, off], scales[at, :, off] = _quantise(x[:n])
        row = torch.zeros(c["padded"], c["kv_heads"], c["dim"], dtype=x.dtype, device="cuda")
        row[:n] = (_unpack(codes[at, :, off]) * scales[at, :, off].float()[..., None]).to(x.dtype)
        out[name] = row
    return dict(out, k_scale=s["ks"], v_scale=s["vs"])


def _plain_attend(s):
    c, q, table, lens = s["case"], s["q"], s["table"], s["lens"].long()
    n, hk, d = c["requests"], c["kv_heads"], c["dim"]
    rep, size = c["q_heads"] // hk, table.shape[1] * c["page"]
    new = max(_requests(c)[1])
    first = s["cu"][:-1].long() if s["cu"] is not None else torch.arange(n, device="cuda")
    count = s["cu"][1:].long() - first if s["cu"] is not None else torch.ones_like(first)

    def rows(codes, scales):
        at = table.clamp(min=0).long()
        x = _unpack(codes[at]) * scales[at].float()[..., None]              # [request, page, head, token, channel]
        return x.transpose(1, 2).reshape(n, hk, size, d)

    i, j = torch.arange(new, device="cuda"), torch.arange(size, device="cuda")
    at = (first[:, None] + i).clamp(max=len(q) - 1)                         # [request, new token]
    pos = lens[:, None] - count[:, None] + i
    seen = j <= pos[..., None]
    if c["window"]:
        seen &= j > pos[..., None] - c["window"]
    x = q.float()[at].reshape(n, new, hk, rep, d).permute(0, 2, 1, 3, 4).reshape(n, hk, new * rep, d) * d ** -0.5
    p = (x @ rows(s["kp"], s["ks"]).transpose(-1, -2)).reshape(n, hk, new, rep, size)
    p.masked_fill_(~seen[:, None, :, None], -math.inf)
    top = p.amax(-1, keepdim=True)
    p.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    y = (p.reshape(n, hk, new * rep, size) @ rows(s["vp"], s["vs"])).reshape(n, hk, new, rep, d) / total
    y = y.permute(0, 2, 1, 3, 4).reshape(n, new, hk * rep, d).to(q.dtype)
    live = torch.zeros(len(q) + 1, dtype=torch.int64, device="cuda")        # the padded row of each token
    flat = torch.where(i < count[:, None], at, len(q)).flatten()
    live[flat] = torch.arange(n * new, device="cuda")
    out = dict(out=y.reshape(n * new, hk * rep, d)[live[:-1]])
    if c["lse"]:
        lse = (top + total.log()).squeeze(-1).permute(0, 2, 1, 3).reshape(n * new, hk * rep)
        out["lse"] = lse[live[:-1]]
    return out


# ---------------------------------------------------------------------------
# the definition in 64 bits, request by request
# ---------------------------------------------------------------------------


def _exact_rows(x):
    """The values that rows are held as."""
    x = x.double()
    scale = (x.abs().amax(-1, keepdim=True).clamp(min=1e-5) / 7.0).half().double()
    return torch.clamp(torch.round(x / scale), -8, 7) * scale, scale[..., 0]


def _exact_values(codes, scales):
    u = codes.to(torch.int16) & 255
    u = torch.cat(((u % 16)[..., None], (u // 16)[..., None]), -1).reshape(*codes.shape[:-1], -1)
    return (u - 16 * (u > 7)).double() * scales.double()[..., None]


def exact(c, seed):
    s = prepare(c, seed)
    if c["path"] == "batch":
        table, free = s["table"].cpu().numpy().copy(), s["free"].cpu().tolist()
        page, used, cu, slots, positions, lens = c["page"], 0, [0], [], [], []
        for r, (a, b) in enumerate(zip(*_requests(c))):
            for p in range(_pages(a, page), _pages(a + b, page)):
                table[r, p] = free[used]
                used += 1
            positions += range(a, a + b)
            slots += [int(table[r, p // page]) * page + p % page for p in range(a, a + b)]
            cu.append(cu[-1] + b)
            lens.append(a + b)
        pad = [-1] * (c["tokens"] - len(slots))
        return dict(table=torch.from_numpy(table), cu=torch.tensor(cu, dtype=torch.int32),
                    lens=torch.tensor(lens, dtype=torch.int32), slots=torch.tensor(slots + pad),
                    positions=torch.tensor(positions + pad), used=torch.tensor([used], dtype=torch.int32))
    if c["path"] == "append":
        out = {}
        for name in "kv":
            value, scale = _exact_rows(s[name])
            value[c["tokens"]:] = 0
            pool = s[name + "s"].double().transpose(1, 2).reshape(-1, c["kv_heads"])
            pool[s["slots"][:c["tokens"]]] = scale[:c["tokens"]]
            out[name] = value
            out[name + "_scale"] = pool.reshape(-1, c["page"], c["kv_heads"]).transpose(1, 2)
        return out
    ctx, new = _requests(c)
    rep, d, first = c["q_heads"] // c["kv_heads"], c["dim"], 0
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.empty(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    for r, (a, b) in enumerate(zip(ctx, new)):
        n = a + b
        pages = s["table"][r, :_pages(n, c["page"])].long()
        k, v = (_exact_values(s[x + "p"][pages], s[x + "s"][pages]).transpose(0, 1).reshape(c["kv_heads"], -1, d)[:, :n]
                for x in "kv")
        for t in range(0, b, 1024):
            m = min(1024, b - t)
            pos = torch.arange(a + t, a + t + m, device="cuda")[:, None]
            key = torch.arange(n, device="cuda")
            hidden = (key > pos) | (key <= pos - c["window"]) if c["window"] else key > pos
            for h in range(c["q_heads"]):
                z = s["q"][first + t:first + t + m, h].double() @ k[h // rep].t() / math.sqrt(d)
                z[hidden] = -math.inf
                out[first + t:first + t + m, h] = torch.softmax(z, -1) @ v[h // rep]
                lse[first + t:first + t + m, h] = torch.logsumexp(z, -1)
        first += b
    return dict(out=out, lse=lse) if c["lse"] else dict(out=out)
