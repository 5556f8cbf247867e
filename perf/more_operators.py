"""Position rotation, rotated appends and the paged 8-bit cache as cases that can be timed.

Between a layer's projections and its attention a decoder normalises the
queries and keys of each head (some models), rotates them by their positions
and puts the keys and values into the cache.  `qk_norm_rope` does the first two
in one pass; `paged_rope_append` does all three for a serving program whose
cache is paged, in 4 bits with a scale per (token, key head) or in 8 bits with a
scale per (block of 16 tokens, key head).  `paged8_attention` reads the 8-bit
pages: one new token per request, or ragged chunks of them.

Head shapes are 32 query / 8 key heads, 64 / 8 and 32 / 2 of dimension 128,
and the same counts of dimension 64.  Queries and keys are Gaussian, keys with
offsets ~ N(0, 2) per (key head, channel); norm weights lie around 1, angles are
position * 500000^(-2i / rotated channels); pages are scattered over the pool.
`draw` spreads cases of the same paths over 1 to 1024 requests, 1 to 30000
tokens, contexts of none to 32768, both 16-bit types, pages of 16 to 128, both
orders of the rotated pairs, heads rotated in part and sliding windows.

    norm      y = x / sqrt(mean(x^2) + eps) * w over a head's channels
    rotation  (a, b) -> (a cos - b sin, b cos + a sin) for the channel pairs
              (i, i + R/2), or (2i, 2i + 1), of the first R channels
    4 bits    scale = fp16(max(amax, 1e-5) / 7) of a row, code =
              round_half_even(x / scale), x before any rounding to 16 bits
    8 bits    scale = 2^e, the smallest with max(amax, 1e-5) <= 127 2^e over
              the block's new rows, and at least the block's scale before
              where rows of it stay: those become round_half_even(code * old / new);
              code = round_half_even(x / scale)
    out_i = sum_j softmax_j(sm q_i . k_j) v_j over the visible keys j <= pos_i
            (and j > pos_i - window), k_j and v_j = code * scale
"""

import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
BLOCK = 16                             # tokens of an 8-bit scale
EPS = 1e-6
MOST_ROWS = 32764 * 72                 # tokens * heads of the largest rotation
MOST_KEYS = 16 * 32768 * 8             # requests * context * key heads of the largest decode case
MOST_PAIRS = 32 * 2048 * 10240         # heads * requests * chunk * keys of the largest chunk case, padded


def listed():
    return [
        # a decode step of 16 requests, heads normalised: launch latency
        dict(name="rotate_t16", path="rotate", batch=1, length=16, q_heads=64, kv_heads=8, dim=128, rotary=128,
             interleaved=False, norm=True, positions=True, dtype="bf16"),
        # four prompts of a batch as a model's own attention module has them, an odd length
        dict(name="rotate_b4_8191", path="rotate", batch=4, length=8191, q_heads=64, kv_heads=8, dim=128, rotary=128,
             interleaved=False, norm=True, positions=False, dtype="bf16"),
        # a decode step's new rows of one layer into 4-bit pages
        dict(name="append4_r48", path="append", bits=4, requests=48, ctx_lo=700, ctx_hi=32000, new_lo=1, new_hi=1, pad=0,
             q_heads=32, kv_heads=8, dim=128, rotary=128, interleaved=False, norm=True, page=16, dtype="bf16"),
        # an 8K prompt into 4-bit pages, slices of a fused projection
        dict(name="append4_8k", path="append", bits=4, requests=1, ctx_lo=0, ctx_hi=0, new_lo=8191, new_hi=8191, pad=0,
             q_heads=64, kv_heads=8, dim=128, rotary=128, interleaved=False, norm=True, page=64, dtype="bf16"),
        # 200 decode steps into 8-bit pages, blocks that are partly filled
        dict(name="append8_r200", path="append", bits=8, requests=200, ctx_lo=100, ctx_hi=13000, new_lo=1, new_hi=1, pad=0,
             q_heads=32, kv_heads=8, dim=128, rotary=128, interleaved=False, norm=False, page=64, dtype="bf16"),
        # chunks of many prompts into 8-bit pages, heads of 64 rotated in half, fp16, padded rows behind them
        dict(name="append8_r60_d64", path="append", bits=8, requests=60, ctx_lo=37, ctx_hi=9001, new_lo=33, new_hi=1501,
             pad=300, q_heads=32, kv_heads=8, dim=64, rotary=32, interleaved=True, norm=False, page=32, dtype="fp16"),
        # one user, 8K context
        dict(name="decode8_r1_8k", path="attend", requests=1, decodes=1, ctx_lo=8191, ctx_hi=8191, new_lo=1, new_hi=1,
             q_heads=32, kv_heads=8, dim=128, page=64, window=0, dtype="bf16", lse=False),
        # continuous batching: contexts of 700 to 32000 tokens
        dict(name="decode8_r48_ragged", path="attend", requests=48, decodes=48, ctx_lo=700, ctx_hi=32000, new_lo=1, new_hi=1,
             q_heads=32, kv_heads=8, dim=128, page=16, window=0, dtype="bf16", lse=False),
        # a full batch of the longest contexts: HBM bandwidth
        dict(name="decode8_r16_32k", path="attend", requests=16, decodes=16, ctx_lo=32767, ctx_hi=32767, new_lo=1, new_hi=1,
             q_heads=32, kv_heads=8, dim=128, page=64, window=0, dtype="bf16", lse=False),
        # 16 query heads on each of two key heads of 64 channels, fp16, a sliding window, many short requests
        dict(name="decode8_r200_d64_window", path="attend", requests=200, decodes=200, ctx_lo=100, ctx_hi=13000, new_lo=1,
             new_hi=1, q_heads=32, kv_heads=2, dim=64, page=32, window=4096, dtype="fp16", lse=False),
        # a 2K chunk of a prompt whose first 8K tokens are in the cache
        dict(name="chunk8_2k_at_8k", path="attend", requests=1, decodes=0, ctx_lo=8192, ctx_hi=8192, new_lo=2048, new_hi=2048,
             q_heads=32, kv_heads=8, dim=128, page=64, window=0, dtype="bf16", lse=True),
        # chunks next to decode steps in one call, odd sizes, fp16
        dict(name="mixed8_r12", path="attend", requests=12, decodes=8, ctx_lo=37, ctx_hi=9001, new_lo=33, new_hi=515,
             q_heads=64, kv_heads=8, dim=128, page=32, window=0, dtype="fp16", lse=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    path = rng.choice(["rotate", "append", "append", "decode", "decode", "chunk", "chunk"])
    page = rng.choice([16, 16, 32, 64, 128])
    q_heads, kv_heads = rng.choice([(32, 8), (32, 8), (64, 8), (32, 2)])
    dim = rng.choice([128, 128, 64])
    c = dict(q_heads=q_heads, kv_heads=kv_heads, dim=dim, dtype=rng.choice(["bf16", "bf16", "fp16"]))
    if path in ("rotate", "append"):
        c.update(rotary=rng.choice([dim, dim, dim // 2]), interleaved=rng.random() < 0.3, norm=rng.random() < 0.5)
    if path == "rotate":
        batch = rng.choice([1, 1, rng.randint(2, 8)])
        length = _log_int(rng, 1, MOST_ROWS // (batch * (q_heads + kv_heads)) // 2)
        return dict(c, path="rotate", batch=batch, length=length, positions=rng.random() < 0.5)
    if path == "append":
        bits = rng.choice([4, 8, 8])
        hi = rng.choice([1, _log_int(rng, 2, 3000)])
        n = _log_int(rng, 1, min(400, 30000 // hi))
        ctx = rng.choice([0, _log_int(rng, 1, 16000)])
        return dict(c, path="append", bits=bits, requests=n, ctx_lo=min(ctx, _log_int(rng, 1, 16000)), ctx_hi=ctx,
                    new_lo=_log_int(rng, 1, hi), new_hi=hi, pad=rng.choice([0, rng.randint(1, 300)]), page=page)
    c.update(path="attend", page=page, window=rng.choice([0, 0, 0, _log_int(rng, 64, 8192)]), lse=rng.random() < 0.3)
    if path == "decode":
        hi = _log_int(rng, 64, 32000)
        n = _log_int(rng, 1, min(256, MOST_KEYS // (2 * hi * kv_heads)))
        return dict(c, requests=n, decodes=n, ctx_lo=_log_int(rng, 1, hi), ctx_hi=hi, new_lo=1, new_hi=1)
    hi = _log_int(rng, 2, 3000)
    ctx = rng.choice([0, _log_int(rng, 1, 16000)])
    n = _log_int(rng, 1, max(1, min(16, MOST_PAIRS // (q_heads * hi * (hi + ctx)))))
    if n * q_heads * hi * (hi + ctx) > MOST_PAIRS:
        hi = max(2, MOST_PAIRS // (q_heads * (3000 + ctx)))
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
    hq, hk, d = c["q_heads"], c["kv_heads"], c["dim"]
    if c["path"] == "rotate":
        n = c["batch"] * c["length"]
        rows = n * (hq + hk)
        # rows in and out, a table row per position, positions
        return dict(bytes=rows * d * 4 + c["length"] * c["rotary"] * 4 + (8 * n if c["positions"] else 0),
                    flops=rows * (3 * c["rotary"] + (4 * d if c["norm"] else 0)))
    ctx, new = _requests(c)
    if c["path"] == "append":
        n = sum(new)
        held = 2 * hk * (n * (d // 2 + 2) if c["bits"] == 4 else n * d + 4 * sum(_pages(a + b, BLOCK) - a // BLOCK for a, b in zip(ctx, new)))
        read = n if c["bits"] == 4 else sum(b + a % BLOCK for a, b in zip(ctx, new))
        # rows in, q out, the cache's new rows, a table row per token, slots and positions, rows read back
        return dict(bytes=n * (hq + 2 * hk) * d * 2 + (n + c["pad"]) * (hq * d * 2 + 16) + held + n * c["rotary"] * 4 + read * 2 * hk * d * 2,
                    flops=n * (hq + hk) * (3 * c["rotary"] + (4 * d if c["norm"] else 0)) + 2 * n * hk * d * 3)
    keys, pairs = 0, 0
    for a, b in zip(ctx, new):
        w = c["window"] or a + b
        first = max(0, a - w + 1)
        keys += a + b - first
        pairs += sum(min(w, a + i + 1) for i in range(b))
    rows = sum(new) * hq
    return dict(bytes=keys * hk * 2 * d + keys // BLOCK * hk * 8 + rows * d * 4 + 4 * _pages(keys, c["page"]) + (4 * rows if c["lse"] else 0),
                flops=4 * d * hq * pairs)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def _pool4(g, pages, heads, page, dim, offset):
    """4-bit codes and scales of Gaussian rows for every slot of a pool."""
    x = torch.randn(pages, heads, page, dim, generator=g, device="cuda")
    if offset is not None:
        x += offset[:, None, :]
    scale = (x.abs().amax(-1).clamp(min=1e-5) / 7).half()
    x /= scale.float()[..., None]
    code = x.round_().clamp_(-8, 7).to(torch.int8) & 15
    return code[..., 0::2] | (code[..., 1::2] << 4), scale


def _pool8(g, pages, heads, page, dim, offset):
    """8-bit codes and block scales of Gaussian rows for every slot of a pool."""
    x = torch.randn(pages, heads, page, dim, generator=g, device="cuda")
    if offset is not None:
        x += offset[:, None, :]
    x = x.reshape(pages, heads, page // BLOCK, BLOCK * dim)
    scale = torch.exp2(torch.ceil(torch.log2(x.abs().amax(-1) / 127)))
    x /= scale[..., None]
    return x.round_().clamp_(-127, 127).to(torch.int8).reshape(pages, heads, page, dim), scale


def _table(g, held, width, pages):
    """A block table of scattered pages, -1 behind each row's last."""
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    held = torch.tensor(held, device="cuda")
    at = torch.arange(width, device="cuda")
    table = order[((held.cumsum(0) - held)[:, None] + at).clamp(max=pages - 1)]
    table[at >= held[:, None]] = -1
    return table


def _angles(rows, rotary):
    """cos and sin of every position below `rows`, fp32 from 64-bit angles."""
    f = 500000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device="cuda") / rotary)
    a = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * f
    return a.cos().float(), a.sin().float()


def _rows(g, c, tokens, parts):
    """Token rows of a fused projection: query heads, key heads and (parts 2) value heads."""
    x = torch.randn(tokens, c["q_heads"] + parts * c["kv_heads"], c["dim"], generator=g, device="cuda")
    x[:, c["q_heads"]:c["q_heads"] + c["kv_heads"]] += math.sqrt(2.0) * torch.randn(c["kv_heads"], c["dim"], generator=g, device="cuda")
    return x.to(TYPES[c["dtype"]])


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case=dict(c))
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    hq, h, d, dt = c["q_heads"], c["kv_heads"], c["dim"], TYPES[c["dtype"]]
    if c["path"] != "attend":
        s["wq"] = s["wk"] = None
        if c["norm"]:
            s["wq"], s["wk"] = ((1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(dt) for _ in range(2))
    if c["path"] == "rotate":
        n = c["batch"] * c["length"]
        x = _rows(g, c, n, 1)
        s["positions"] = None
        if c["positions"]:             # tokens of a serving step: each at its own place
            s["cos"], s["sin"] = _angles(32768, c["rotary"])
            s["positions"] = torch.randint(0, 32768, (n,), generator=g, device="cuda")
        else:                          # a batch of prompts from position 0
            x = x.reshape(c["batch"], c["length"], hq + h, d)
            s["cos"], s["sin"] = _angles(c["length"], c["rotary"])
        s["q"], s["k"] = x[..., :hq, :], x[..., hq:, :]
        return s
    ctx, new = _requests(c)
    page = c["page"]
    total = [_pages(a + b, page) for a, b in zip(ctx, new)]
    pages = sum(total) + 3
    table = _table(g, total, max(total) + 1, pages)
    offset = math.sqrt(2.0) * torch.randn(h, d, generator=g, device="cuda")
    pool = _pool4 if c.get("bits") == 4 else _pool8
    s["kp"], s["ks"] = pool(g, pages, h, page, d, offset)
    s["vp"], s["vs"] = pool(g, pages, h, page, d, None)
    if c["path"] == "append":
        n = sum(new)
        x = _rows(g, c, n + c["pad"], 2)
        s["q"], s["k"], s["v"] = x[:, :hq], x[:, hq:hq + h], x[:, hq + h:]
        s["cos"], s["sin"] = _angles(max(a + b for a, b in zip(ctx, new)), c["rotary"])

        def tokens(first, count, pad):
            """(slot, position) of `count` tokens of each request from `first`, -1 behind them."""
            first, count = torch.tensor(first, device="cuda"), torch.tensor(count, device="cuda")
            r = torch.repeat_interleave(torch.arange(len(first), device="cuda"), count)
            pos = torch.arange(len(r), device="cuda") - (count.cumsum(0) - count)[r] + first[r]
            tail = torch.full((pad,), -1, dtype=torch.int64, device="cuda")
            return torch.cat((table[r, pos // page].long() * page + pos % page, tail)), torch.cat((pos, tail))

        s["slots"], s["positions"] = tokens(ctx, new, c["pad"])
        # what the call may change: the new rows, and those that share a block with them
        keep = [a % BLOCK if c["bits"] == 8 else 0 for a in ctx]
        s["changed"], _ = tokens([a - k for a, k in zip(ctx, keep)], [b + k for b, k in zip(new, keep)], 0)
        return s
    s["table"] = table
    s["q"] = torch.randn(sum(new), hq, d, generator=g, device="cuda").to(dt)
    s["lens"] = i32([a + b for a, b in zip(ctx, new)])
    s["cu"] = None if max(new) == 1 else i32([0] + torch.tensor(new).cumsum(0).tolist())
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------


def _own_run(s):
    import hyquant_amd as hq
    c = s["case"]
    if c["path"] == "rotate":
        q, k = hq.qk_norm_rope(s["q"], s["k"], s["cos"], s["sin"], s["positions"], q_weight=s["wq"], k_weight=s["wk"], eps=EPS,
                               interleaved=c["interleaved"])
        return dict(q=q, k=k)
    pool = (s["kp"], s["vp"], s["ks"], s["vs"])
    if c["path"] == "append":
        q = hq.paged_rope_append(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["positions"], s["slots"], *pool, q_weight=s["wq"],
                                 k_weight=s["wk"], eps=EPS, interleaved=c["interleaved"])
        gather = hq.paged_gather if c["bits"] == 4 else hq.paged8_gather
        k, v = gather(s["changed"], *pool, dtype=q.dtype)
        return dict(q=q, k=k, v=v, k_scale=s["ks"], v_scale=s["vs"])
    if c["lse"]:
        out, lse = hq.paged8_attention(s["q"], *pool, s["table"], s["lens"], s["cu"], window=c["window"], return_lse=True)
        return dict(out=out, lse=lse)
    return dict(out=hq.paged8_attention(s["q"], *pool, s["table"], s["lens"], s["cu"], window=c["window"]))


def run(s):
    if own:
        return _own_run(s)
    path = s["case"]["path"]
    return _plain_rotate(s) if path == "rotate" else _plain_append(s) if path == "append" else _plain_attend(s)


def _turn(x, w, cos, sin, c):
    """Rows x [..., heads, D] normalised and rotated; cos and sin broadcast against [..., heads, R / 2]."""
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.to(x.dtype)
    r = c["rotary"]
    y = x.clone()
    first, second = (slice(0, r, 2), slice(1, r, 2)) if c["interleaved"] else (slice(0, r // 2), slice(r // 2, r))
    a, b = x[..., first], x[..., second]
    y[..., first] = a * cos - b * sin
    y[..., second] = b * cos + a * sin
    return y


def _plain_rotate(s):
    c = s["case"]
    cos, sin = s["cos"], s["sin"]
    if s["positions"] is not None:
        cos, sin = cos[s["positions"]], sin[s["positions"]]
    cos, sin = cos[..., None, :], sin[..., None, :]
    return {n: _turn(s[n].float(), s["w" + n], cos, sin, c).to(s[n].dtype) for n in "qk"}


def _unpack(packed):
    """Codes of packed rows."""
    low, high = (packed << 4) >> 4, packed >> 4
    return torch.stack((low, high), -1).flatten(-2)


def _exponent(amax):
    """The smallest e with max(amax, 1e-5) <= 127 2^e."""
    f, x = torch.frexp(amax.clamp(min=1e-5))
    return x - 7 + (f > 127 / 128)


def _plain_append(s):
    c = s["case"]
    slots = s["slots"][:sum(_requests(c)[1])]
    n, page, h, d = len(slots), c["page"], c["kv_heads"], c["dim"]
    at, off = slots // page, slots % page
    cos, sin = s["cos"][s["positions"][:n]][:, None], s["sin"][s["positions"][:n]][:, None]
    q = torch.zeros(s["q"].shape, dtype=s["q"].dtype, device="cuda")
    q[:n] = _turn(s["q"][:n].float(), s["wq"], cos, sin, c).to(q.dtype)
    # (codes lie next to borders: 64 bits)
    values = dict(k=_turn(s["k"][:n].double(), s["wk"], cos.double(), sin.double(), c), v=s["v"][:n].double())
    out = dict(q=q)
    changed = s["changed"]
    for name in "kv":
        codes, scales, x = s[name + "p"], s[name + "s"], values[name]
        if c["bits"] == 4:
            scale = (x.abs().amax(-1).clamp(min=1e-5) / 7).half()
            code = torch.round(x / scale.double()[..., None]).clamp(-8, 7).to(torch.int8) & 15
            codes[at, :, off], scales[at, :, off] = code[..., 0::2] | (code[..., 1::2] << 4), scale
            held, by = _unpack(codes[changed // page, :, changed % page]), scales[changed // page, :, changed % page]
        else:
            # all blocks of the pool, block = slot // 16
            pool = codes.reshape(-1, h, page // BLOCK, BLOCK, d).transpose(1, 2).reshape(-1, h, BLOCK, d)
            old = torch.frexp(scales.transpose(1, 2).reshape(-1, h))[1].long() - 1
            block = slots // BLOCK
            first = torch.full((len(pool),), BLOCK, device="cuda").scatter_reduce(0, block, slots % BLOCK, "amin")
            need = torch.full((len(pool), h), -1000, device="cuda")
            need = need.scatter_reduce(0, block[:, None].expand(-1, h), _exponent(x.abs().amax(-1)).long(), "amax")
            touched = (first < BLOCK)[:, None]
            e = torch.where(touched, torch.maximum(need, torch.where(first[:, None] > 0, old, -1000)), old)
            stays = touched[..., None] & (torch.arange(BLOCK, device="cuda") < first[:, None, None])
            again = torch.round(pool.float() * torch.exp2((old - e).float())[..., None, None]).to(torch.int8)
            pool = torch.where(stays[..., None], again, pool)
            pool[block, :, slots % BLOCK] = torch.round(x * torch.exp2(-e[block].double())[..., None]).to(torch.int8)
            codes.copy_(pool.reshape(-1, page // BLOCK, h, BLOCK, d).transpose(1, 2).reshape(codes.shape))
            scales.copy_(torch.exp2(e.float()).reshape(-1, page // BLOCK, h).transpose(1, 2))
            held, by = pool[changed // BLOCK, :, changed % BLOCK], scales.transpose(1, 2).reshape(-1, h)[changed // BLOCK]
        out[name] = (held.float() * by.float()[..., None]).to(q.dtype)
        out[name + "_scale"] = scales
    return out


def _plain_attend(s):
    c, q, table, lens = s["case"], s["q"], s["table"], s["lens"].long()
    n, hk, d = c["requests"], c["kv_heads"], c["dim"]
    rep, size = c["q_heads"] // hk, table.shape[1] * c["page"]
    new = max(_requests(c)[1])
    first = s["cu"][:-1].long() if s["cu"] is not None else torch.arange(n, device="cuda")
    count = s["cu"][1:].long() - first if s["cu"] is not None else torch.ones_like(first)

    def rows(codes, scales):
        at = table.clamp(min=0).long()
        x = codes[at].float().unflatten(3, (-1, BLOCK)) * scales[at][..., None, None]     # [request, page, head, block, token, channel]
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
# the definition in 64 bits
# ---------------------------------------------------------------------------


def _exact_turn(x, w, cos, sin, c):
    """As a product of complex numbers: channel pairs times cos + i sin."""
    x = x.double()
    if w is not None:
        x = w.double() * x / torch.sqrt(torch.mean(torch.square(x), -1, keepdim=True) + EPS)
    r, turn = c["rotary"], torch.complex(cos.double(), sin.double())
    part, rest = x[..., :r], x[..., r:]
    pairs = part.unflatten(-1, (r // 2, 2)) if c["interleaved"] else part.unflatten(-1, (2, r // 2)).transpose(-1, -2)
    z = torch.view_as_real(torch.complex(pairs[..., 0], pairs[..., 1]) * turn)
    z = z if c["interleaved"] else z.transpose(-1, -2)
    return torch.cat((z.flatten(-2), rest), -1)


def _exact_append(c, s):
    ctx, new = _requests(c)
    n = sum(new)
    at = s["positions"][:n]
    cos, sin = s["cos"][at].unsqueeze(1), s["sin"][at].unsqueeze(1)
    q = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    q[:n] = _exact_turn(s["q"][:n], s["wq"], cos, sin, c)
    rows = dict(k=_exact_turn(s["k"][:n], s["wk"], cos, sin, c), v=s["v"][:n].double())
    out = dict(q=q)
    slots, page, h = s["slots"][:n], c["page"], c["kv_heads"]
    if c["bits"] == 4:
        for name in "kv":
            x = rows[name]
            scale = (x.abs().amax(-1).clamp(min=1e-5) / 7.0).half()
            pool = s[name + "s"].transpose(1, 2).reshape(-1, h)
            pool[slots] = scale
            out[name] = torch.clamp(torch.round(x / scale.double()[..., None]), -8, 7) * scale.double()[..., None]
            out[name + "_scale"] = pool.reshape(-1, page, h).transpose(1, 2).double()
        return out
    # request by request, its blocks padded to whole ones
    for name in "kv":
        per_block = s[name + "s"].transpose(1, 2).reshape(-1, h).double()
        rows_of = s[name + "p"].transpose(1, 2).reshape(-1, h, c["dim"])
        values, t, u = [], 0, 0
        for a, b in zip(ctx, new):
            keep = a % BLOCK
            mine = s["changed"][u:u + keep + b]
            block = mine[::BLOCK] // BLOCK
            before = per_block[block[0]]                                    # [heads]
            kept = rows_of[mine[:keep]].double() * before[:, None]
            x = torch.nn.functional.pad(rows[name][t:t + b], (0, 0, 0, 0, keep, -(keep + b) % BLOCK))
            x = x.unflatten(0, (-1, BLOCK))                                 # [blocks, tokens, heads, channels]
            most = x.abs().amax((1, 3)).clamp(min=1e-5)
            scale = torch.exp2(torch.ceil(torch.log2(most / 127.0)))
            scale = torch.where(scale * 127.0 < most, 2 * scale, torch.where(scale * 63.5 >= most, scale / 2, scale))
            if keep:
                scale[0] = torch.maximum(scale[0], before)
                x[0, :keep] = kept
            per_block[block] = scale
            values.append((torch.round(x / scale[:, None, :, None]) * scale[:, None, :, None]).flatten(0, 1)[:keep + b])
            t, u = t + b, u + keep + b
        out[name] = torch.cat(values)
        out[name + "_scale"] = per_block.reshape(-1, page // BLOCK, h).transpose(1, 2)
    return out


def exact(c, seed):
    s = prepare(c, seed)
    if c["path"] == "rotate":
        if s["positions"] is not None:
            s["cos"], s["sin"] = s["cos"][s["positions"]], s["sin"][s["positions"]]
        return {n: _exact_turn(s[n], s["w" + n], s["cos"].unsqueeze(-2), s["sin"].unsqueeze(-2), c) for n in "qk"}
    if c["path"] == "append":
        return _exact_append(c, s)
    ctx, new = _requests(c)
    rep, d, first = c["q_heads"] // c["kv_heads"], c["dim"], 0
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.empty(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    for r, (a, b) in enumerate(zip(ctx, new)):
        n = a + b
        pages = s["table"][r, :_pages(n, c["page"])].long()
        k, v = ((s[x + "p"][pages].double() * s[x + "s"][pages].double().repeat_interleave(BLOCK, 2)[..., None]).transpose(0, 1)
                .reshape(c["kv_heads"], -1, d)[:, :n] for x in "kv")
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
