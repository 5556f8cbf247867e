"""The paged 4-bit cache's operators on the GPU against plain references in 64
bits: batch layout, append and read-back, attention over block tables, and
whole steps of them together."""

import math

import pytest
import torch

import hyquant_amd as hq
from tests import paged_util as U

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _cu(new):
    return _i32([0] + torch.tensor(new, dtype=torch.int64).cumsum(0).tolist())


# ---------------------------------------------------------------------------
# batch layout
# ---------------------------------------------------------------------------


def _batch_reference(ctx, new, table, free, page, T):
    table = [row[:] for row in table]
    width = len(table[0]) if table else 0
    used, cu, slots, positions = 0, [0], [], []
    for r, (a, b) in enumerate(zip(ctx, new)):
        for col in range(-(-a // page), -(-(a + b) // page)):
            if col < width:
                table[r][col] = free[used] if used < len(free) else -1
            used += 1
        for p in range(a, a + b):
            page_id = table[r][p // page] if p // page < width else -1
            slots.append(page_id * page + p % page if page_id >= 0 else -1)
            positions.append(p)
        cu.append(cu[-1] + b)
    slots, positions = slots[:T], positions[:T]
    pad = [-1] * (T - len(slots))
    return table, cu, [a + b for a, b in zip(ctx, new)], slots + pad, positions + pad, used


@pytest.mark.parametrize("R,page,ctx_hi,new_hi,pad", [(1, 16, 0, 1, 0), (1, 64, 5000, 1, 3), (3, 16, 40, 33, 0), (65, 32, 500, 1, 7),
                                                      (257, 16, 300, 50, 11), (1000, 128, 2000, 9, 0), (4, 256, 3000, 2500, 100)])
@pytest.mark.parametrize("short", [False, True])
def test_batch_layout(R, page, ctx_hi, new_hi, pad, short):
    g = torch.Generator().manual_seed(R * 7 + page)
    ctx = torch.randint(0, ctx_hi + 1, (R,), generator=g).tolist()
    new = torch.randint(0, new_hi + 1, (R,), generator=g).tolist()
    new[0] = max(new[0], 1)
    need = [-(-(a + b) // page) for a, b in zip(ctx, new)]
    taken = sum(n - -(-a // page) for n, a in zip(need, ctx))
    width = max(need) + (1 if not short else 0)
    width = max(1, width - (1 if short and max(need) > 1 else 0))          # short: the longest row misses a column
    held = sum(min(-(-a // page), width) for a in ctx)
    ids = torch.randperm(held + taken + 5, generator=g).tolist()
    table, at = [], 0
    for a in ctx:
        h = min(-(-a // page), width)
        table.append(ids[at:at + h] + [-7] * (width - h))                  # entries behind the held ones: anything
        at += h
    free = ids[at:at + taken + 3] if not short else ids[at:at + taken // 2]
    T = sum(new) + pad
    t = _i32(table)
    b = hq.paged_batch(_i32(ctx), _i32(new), t, _i32(free), page, T)
    want = _batch_reference(ctx, new, table, free, page, T)
    for got, exp in zip((t, b.cu_seqlens, b.seq_lens, b.slots, b.positions, b.pages_used), want[:5] + ([want[5]],)):
        assert got.tolist() == exp
    # again: the entries are the same
    b2 = hq.paged_batch(_i32(ctx), _i32(new), t, _i32(free), page, T)
    assert t.tolist() == want[0] and torch.equal(b2.slots, b.slots)


def test_batch_layout_truncated_tokens_and_empty():
    t = _i32([[4, -1, -1]])
    b = hq.paged_batch(_i32([10]), _i32([20]), t, _i32([9, 8]), 16, 7)      # 7 of the 20 tokens
    assert b.slots.tolist() == [4 * 16 + 10 + i for i in range(6)] + [9 * 16] and b.pages_used.tolist() == [1]
    b = hq.paged_batch(_i32([]), _i32([]), torch.empty(0, 4, dtype=torch.int32, device="cuda"), _i32([1]), 16, 3)
    assert b.cu_seqlens.tolist() == [0] and b.slots.tolist() == [-1] * 3 and b.pages_used.tolist() == [0]
    b = hq.paged_batch(_i32([5, 3]), _i32([0, 0]), _i32([[1], [2]]), _i32([]), 16, 0)
    assert b.cu_seqlens.tolist() == [0, 0, 0] and b.seq_lens.tolist() == [5, 3]
    b = hq.paged_batch(_i32([-5, 3]), _i32([2, -4]), _i32([[1], [2]]), _i32([6]), 16, 2)      # negative lengths count as 0
    assert b.cu_seqlens.tolist() == [0, 2, 2] and b.seq_lens.tolist() == [2, 3] and b.slots.tolist() == [96, 97]


def test_batch_layout_most_requests():
    R = 16384
    new = torch.randint(0, 3, (R,), generator=torch.Generator().manual_seed(0), dtype=torch.int32)
    ctx = torch.randint(0, 60, (R,), generator=torch.Generator().manual_seed(1), dtype=torch.int32)
    t = torch.randint(0, 1000, (R, 4), dtype=torch.int32, generator=torch.Generator().manual_seed(2))
    free = torch.arange(5000, 5000 + R, dtype=torch.int32)
    T = int(new.sum())
    want = _batch_reference(ctx.tolist(), new.tolist(), t.tolist(), free.tolist(), 16, T)
    td = t.cuda()
    b = hq.paged_batch(ctx.cuda(), new.cuda(), td, free.cuda(), 16, T)
    for got, exp in zip((td, b.cu_seqlens, b.seq_lens, b.slots, b.positions, b.pages_used), want[:5] + ([want[5]],)):
        assert got.tolist() == exp
    with pytest.raises(ValueError, match="16384"):
        hq.paged_batch(torch.zeros(R + 1, dtype=torch.int32, device="cuda"), torch.zeros(R + 1, dtype=torch.int32, device="cuda"),
                       torch.zeros(R + 1, 1, dtype=torch.int32, device="cuda"), _i32([]), 16, 0)


# ---------------------------------------------------------------------------
# append and read back
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("T,H,D,page", [(1, 8, 128, 64), (5, 1, 64, 16), (37, 3, 128, 16), (300, 2, 64, 256), (1000, 8, 128, 32)])
def test_append_and_gather(dtype, T, H, D, page):
    g = _gen(T + D)
    pages = -(-T // page) + 3
    pool = U.make_pool(g, pages, H, page, D, "cuda")
    before = [x.clone() for x in pool]
    qkv = torch.randn(T, 3, H, D, generator=g, device="cuda")
    qkv[0, 1] *= 1e-7                                    # a row under the smallest scale
    if T > 2:
        qkv[1, 1] *= 3000.0
        qkv[2, 2] = 0.0
    qkv = qkv.to(dtype)
    k, v = qkv[:, 1], qkv[:, 2]                          # strided views
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:T]
    if T > 4:
        slots[3], slots[4] = -1, pages * page            # outside the pool: not written
    hq.paged_append(k, v, slots, *pool)
    ok = (slots >= 0) & (slots < pages * page)
    at, off = slots[ok] // page, slots[ok] % page
    for x, codes, scales, codes0, scales0 in ((k, pool[0], pool[2], before[0], before[2]), (v, pool[1], pool[3], before[1], before[3])):
        want_c, want_s = hq.quantize_per_token(x[ok].reshape(-1, 1, D).contiguous(), 4)
        codes0[at, :, off], scales0[at, :, off] = want_c.reshape(-1, H, D // 2), want_s.reshape(-1, H)
        assert torch.equal(codes, codes0) and torch.equal(scales.view(torch.int16), scales0.view(torch.int16))
    for out_dtype in (BF16, FP16):
        gk, gv = hq.paged_gather(slots, *pool, dtype=out_dtype)
        for got, codes, scales in ((gk, pool[0], pool[2]), (gv, pool[1], pool[3])):
            want = torch.zeros(T, H, D, dtype=torch.float64, device="cuda")
            want[ok] = U.values(codes[at, :, off], scales[at, :, off])
            assert torch.equal(got, want.float().to(out_dtype))      # the products are exact in fp32
    # the dequantiser of the D-stage cache gives the same fp16 values
    d = hq.dequantize_per_token(pool[0].reshape(-1, page, D // 2), pool[2].reshape(-1, page), D, 4).reshape(pages, H, page, D)
    assert torch.equal(d[at, :, off], hq.paged_gather(slots, *pool, dtype=FP16)[0][ok])


def test_append_empty_and_misaligned_rows():
    g = _gen(3)
    pool = U.make_pool(g, 2, 2, 16, 128, "cuda")
    before = [x.clone() for x in pool]
    e = torch.empty(0, 2, 128, dtype=BF16, device="cuda")
    hq.paged_append(e, e, torch.empty(0, dtype=torch.int64, device="cuda"), *pool)
    k, v = hq.paged_gather(torch.empty(0, dtype=torch.int64, device="cuda"), *pool)
    assert k.shape == (0, 2, 128) and all(torch.equal(a, b) for a, b in zip(pool, before))
    flat = torch.randn(3 * 2 * 128 + 1, generator=g, device="cuda").to(BF16)
    x = flat[1:].reshape(3, 2, 128)                      # rows at odd addresses: copied
    slots = torch.tensor([5, 17, 30], device="cuda")
    hq.paged_append(x, x, slots, *pool)
    c, s = U.quantise(x)
    assert torch.equal(pool[0][slots // 16, :, slots % 16], c) and torch.equal(pool[3][slots // 16, :, slots % 16], s)


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------


def _attend(dtype, D, H, G, page, seq, new, window=0, seed=0, sm_scale=None, lse=True, decode=False, pad=0):
    g = _gen(seed)
    table, pages = U.make_table(g, seq, page, "cuda")
    pool = U.make_pool(g, pages, H, page, D, "cuda")
    T = sum(new) + pad
    q = torch.randn(T, H * G, D, generator=g, device="cuda").to(dtype)
    got = hq.paged_attention(q, *pool, table, _i32(seq), None if decode else _cu(new), sm_scale=sm_scale, window=window, return_lse=lse)
    out, got_lse = got if lse else (got, None)
    ref, ref_lse, tol = U.reference(q[:sum(new)], pool, table, seq, new, window, sm_scale)
    n = sum(new)
    U.check(out[:n], ref, tol)
    assert torch.equal(out[n:], torch.zeros_like(out[n:]))
    if lse:
        empty = torch.isinf(ref_lse)
        assert torch.equal(torch.isinf(got_lse[:n]), empty) and bool((got_lse[n:] == -math.inf).all())
        # lse: a score's error (a few 1e-5 at the tests' sizes, see paged_util) and fp32 roundings
        err = (got_lse[:n].double() - ref_lse)[~empty].abs()
        x = q[:n].double().abs().sum(-1).max() if n else torch.tensor(0.0)
        sm = D ** -0.5 if sm_scale is None else abs(sm_scale)
        d = (D + 16) * 2.0 ** -24 * sm * 15 * float(x) * float(pool[2].double().max())
        lim = d + (max(seq) / 16 + 64) * 2.0 ** -23 + 2.0 ** -22 * ref_lse[~empty].abs()
        assert bool((err <= lim).all()), float((err / lim).max())
    return out


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,G", [(8, 4), (2, 16), (1, 1), (3, 7)])
@pytest.mark.parametrize("page", [16, 64])
def test_attention_decode(dtype, D, H, G, page):
    seq = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 500, 1000, 2049, 0]
    _attend(dtype, D, H, G, page, seq, [1] * len(seq), decode=True)


@pytest.mark.parametrize("dtype,D,H,G,page,seq", [(BF16, 128, 8, 4, 64, [8192]), (FP16, 128, 8, 4, 16, [32768, 3]),
                                                  (BF16, 128, 2, 8, 128, [20001, 7, 12345]), (FP16, 64, 8, 4, 256, [30011]),
                                                  (BF16, 128, 1, 16, 32, [4097] * 3)])
@pytest.mark.parametrize("window", [0, 1000])
def test_attention_decode_long(dtype, D, H, G, page, seq, window):
    _attend(dtype, D, H, G, page, seq, [1] * len(seq), window=window, decode=True)


def test_attention_decode_many_requests():
    g = torch.Generator().manual_seed(5)
    seq = torch.randint(0, 300, (1500,), generator=g).tolist()
    _attend(BF16, 128, 2, 4, 16, seq, [1] * len(seq), decode=True, lse=False)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D,H,G,page", [(128, 8, 4, 64), (64, 2, 16, 16), (128, 2, 8, 32), (128, 1, 3, 128), (64, 4, 1, 64)])
@pytest.mark.parametrize("window", [0, 1, 50, 300])
def test_attention_ragged(dtype, D, H, G, page, window):
    new = [1, 5, 0, 33, 64, 1, 130, 2, 17]
    seq = [900, 5, 40, 133, 64, 1, 515, 3, 17]
    _attend(dtype, D, H, G, page, seq, new, window=window, pad=5)


@pytest.mark.parametrize("dtype,D,H,G,page,seq,new,window", [
    (BF16, 128, 8, 4, 64, [2500], [700], 0), (FP16, 128, 2, 8, 16, [1300, 4000], [1300, 77], 0),
    (BF16, 128, 1, 5, 32, [3001], [1001], 0), (FP16, 64, 4, 4, 128, [2000, 100, 5000], [2000, 100, 1], 0),
    (BF16, 64, 8, 4, 16, [6000, 700], [600, 700], 1024), (BF16, 128, 8, 8, 256, [20000], [40], 0)])
def test_attention_chunks(dtype, D, H, G, page, seq, new, window):
    _attend(dtype, D, H, G, page, seq, new, window=window)


def test_attention_rows_without_keys():
    # more new tokens than cached ones: the first rows are before position 0
    out = _attend(BF16, 128, 2, 4, 16, [3, 0, 40], [10, 4, 60])
    assert torch.equal(out[:7], torch.zeros_like(out[:7])) and torch.equal(out[10:14], torch.zeros_like(out[10:14]))
    # no pages at all
    pool = U.make_pool(_gen(0), 0, 2, 16, 128, "cuda")
    q = torch.randn(3, 8, 128, generator=_gen(1), device="cuda").to(BF16)
    out, lse = hq.paged_attention(q, *pool, _i32([[0], [1], [2]]), _i32([5, 6, 7]), return_lse=True)
    assert torch.equal(out, torch.zeros_like(out)) and bool((lse == -math.inf).all())
    out = hq.paged_attention(q, *pool, torch.empty(3, 0, dtype=torch.int32, device="cuda"), _i32([5, 6, 7]))
    assert torch.equal(out, torch.zeros_like(out))
    # no request, no token
    out, lse = hq.paged_attention(q, *pool, torch.empty(0, 1, dtype=torch.int32, device="cuda"), _i32([]), _i32([0]), return_lse=True)
    assert torch.equal(out, torch.zeros_like(out)) and bool((lse == -math.inf).all())
    assert hq.paged_attention(q[:0], *pool, torch.empty(0, 1, dtype=torch.int32, device="cuda"), _i32([])).shape == (0, 8, 128)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_attention_scale_and_magnitudes(dtype):
    _attend(dtype, 128, 2, 4, 16, [333, 70], [1, 20], sm_scale=0.03)
    _attend(dtype, 128, 2, 4, 16, [333, 70], [1, 20], sm_scale=-0.05)
    _attend(dtype, 64, 2, 4, 16, [333, 70], [1, 20], sm_scale=0.0)
    # query rows of very different size, all in one tile, and large scores
    g = _gen(11)
    table, pages = U.make_table(g, [200], 16, "cuda")
    pool = U.make_pool(g, pages, 1, 16, 128, "cuda", scale=30.0)
    q = torch.randn(1, 16, 128, generator=g, device="cuda") * torch.logspace(-12, 1, 16, base=2, device="cuda")[None, :, None]
    q = q.to(dtype)
    out = hq.paged_attention(q, *pool, table, _i32([200]))
    ref, _, tol = U.reference(q, pool, table, [200], [1])
    U.check(out, ref, tol)


@pytest.mark.parametrize("new", [[1, 1], [40, 3]])
def test_attention_masked_places_hold_anything(new):
    """Scales of NaN and infinity where no row may look (rows behind a
    sequence's end, other pages) change nothing; those that only later rows
    see leave the earlier ones alone."""
    g = _gen(4)
    seq, page, H, G, D = [77, 50], 32, 2, 4, 128
    table, pages = U.make_table(g, seq, page, "cuda")
    pool = U.make_pool(g, pages, H, page, D, "cuda")
    q = torch.randn(sum(new), H * G, D, generator=g, device="cuda").to(BF16)
    cu = _cu(new) if max(new) > 1 else None
    want = hq.paged_attention(q, *pool, table, _i32(seq), cu)
    live = torch.zeros(pages, page, dtype=torch.bool, device="cuda")
    for r, n in enumerate(seq):
        for j in range(n):
            live[table[r, j // page], j % page] = True
    for bad in (float("nan"), float("inf"), float("-inf")):
        dirty = [x.clone() for x in pool]
        for s in dirty[2:]:
            s.masked_fill_(~live[:, None], bad)
        for c in dirty[:2]:
            c.masked_fill_(~live[:, None, :, None], 127)
        t = table.clone()
        t[t < 0] = 12345678
        assert torch.equal(hq.paged_attention(q, *dirty, t, _i32(seq), cu), want)
        if max(new) > 1:                                 # the last key of request 0: only its last row sees it
            for s in dirty[2:]:
                s[table[0, 76 // page], :, 76 % page] = bad
            got = hq.paged_attention(q, *dirty, t, _i32(seq), cu)
            assert torch.equal(got[:39], want[:39]) and torch.equal(got[40:], want[40:])


def test_attention_nan_query_row_stays_alone():
    g = _gen(6)
    table, pages = U.make_table(g, [100], 16, "cuda")
    pool = U.make_pool(g, pages, 2, 16, 128, "cuda")
    q = torch.randn(9, 8, 128, generator=g, device="cuda").to(BF16)
    want = hq.paged_attention(q, *pool, table, _i32([100]), _cu([9]))
    for bad in (float("nan"), float("inf")):
        x = q.clone()
        x[4, 3, 7] = bad
        got = hq.paged_attention(x, *pool, table, _i32([100]), _cu([9]))
        assert bool(torch.isnan(got[4, 3]).any())
        got[4, 3] = want[4, 3]
        assert torch.equal(got, want)


@pytest.mark.parametrize("new", [[1, 1, 1], [1, 70, 9]])
def test_attention_pages_outside_the_pool(new):
    """Their keys are left out, as paged_util.reference leaves them out."""
    g = _gen(8)
    seq, page = [300, 400, 129], 16
    table, pages = U.make_table(g, seq, page, "cuda")
    table[0, 3], table[0, 18], table[1, 0], table[1, 7], table[2] = -1, pages, 2 ** 31 - 1, -2 ** 31, pages + 5
    pool = U.make_pool(g, pages, 2, page, 128, "cuda")
    q = torch.randn(sum(new), 8, 128, generator=g, device="cuda").to(BF16)
    out, lse = hq.paged_attention(q, *pool, table, _i32(seq), _cu(new) if max(new) > 1 else None, return_lse=True)
    ref, ref_lse, tol = U.reference(q, pool, table, seq, new)
    U.check(out, ref, tol)
    assert bool((lse[-new[2]:] == -math.inf).all()) and bool((out[-new[2]:] == 0).all())


def test_attention_lengths_past_the_table_and_bad_cu():
    g = _gen(9)
    seq, page = [64, 48], 16
    table, pages = U.make_table(g, seq, page, "cuda", spare=8)
    table[0, 4], table[1, 3:] = pages - 1, torch.tensor([pages - 2, pages - 3], dtype=torch.int32, device="cuda")
    pool = U.make_pool(g, pages, 2, page, 128, "cuda")
    q = torch.randn(2, 8, 128, generator=g, device="cuda").to(BF16)
    a = hq.paged_attention(q, *pool, table, _i32([10 ** 9, -4]))           # 80 tokens in a row of the table; none
    b = hq.paged_attention(q, *pool, table, _i32([80, 0]))
    assert torch.equal(a, b) and bool((b[1] == 0).all())
    # offsets outside the tokens are clamped; nothing outside the outputs is written
    big = torch.full((6, 8, 128), 3.0, dtype=BF16, device="cuda")
    for cu in ([-5, 1, 900], [0, 2 ** 31 - 1, -2 ** 31], [2, 1, 0], [7, 8, 9]):
        hq.paged_attention(q, *pool, table, _i32([64, 48]), _i32(cu), out=big[2:4])
        assert bool((big[:2] == 3.0).all()) and bool((big[4:] == 3.0).all())


def test_attention_strides_and_out():
    g = _gen(10)
    seq, new, page, H, G, D = [200, 65, 130], [1, 65, 9], 32, 2, 4, 128
    T, pad = sum(new), 4
    table, pages = U.make_table(g, seq, page, "cuda")
    pool = U.make_pool(g, pages, H, page, D, "cuda")
    wide = torch.full((3, table.shape[1] + 7), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    # K and V of a page side by side, one layer of three
    codes = torch.zeros(3, pages, 2, H, page, D // 2, dtype=torch.int8, device="cuda")
    scales = torch.zeros(3, pages, 2, H, page, dtype=torch.float16, device="cuda")
    codes[1, :, 0], codes[1, :, 1], scales[1, :, 0], scales[1, :, 1] = pool
    view = (codes[1, :, 0], codes[1, :, 1], scales[1, :, 0], scales[1, :, 1])
    qkv = torch.randn(T + pad, H * G + 2 * H, D, generator=g, device="cuda").to(BF16)
    q = qkv[:, :H * G]
    want = hq.paged_attention(q.contiguous(), *pool, table, _i32(seq), _cu(new))
    ref, _, tol = U.reference(q[:T], pool, table, seq, new)
    U.check(want[:T], ref, tol)
    out = torch.full((H * G, T + pad, D), 7.0, dtype=BF16, device="cuda").transpose(0, 1)
    got = hq.paged_attention(q, *view, wide[:, :table.shape[1]], _i32(seq), _cu(new), out=out)
    assert got is out and torch.equal(out[:T], want[:T]) and bool((out[T:] == 7.0).all())
    odd = torch.randn((T + pad) * H * G * D + 1, generator=g, device="cuda").to(BF16)[1:].reshape(T + pad, H * G, D)
    odd.copy_(q)                                         # rows at odd addresses: copied
    assert torch.equal(hq.paged_attention(odd, *pool, table, _i32(seq), _cu(new)), want)
    heads = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(hq.paged_attention(heads, *pool, table, _i32(seq), _cu(new)), want)


def test_attention_pool_past_32_bits():
    """Pages whose codes start beyond 4 GiB and scales beyond 2^31 elements' bytes."""
    g = _gen(12)
    page, H, D = 64, 8, 128
    pages = 5 * 2 ** 30 // (H * page * D // 2)
    seq, new = [500, 130], [1, 30]
    kp, vp = (torch.empty(pages, H, page, D // 2, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.empty(pages, H, page, dtype=torch.float16, device="cuda") for _ in range(2))
    table, used = U.make_table(g, seq, page, "cuda", spare=0)
    small = U.make_pool(g, used, H, page, D, "cuda")
    high = torch.where(table >= 0, table + (pages - used), table)
    for big, x in zip((kp, vp, ks, vs), small):
        big[pages - used:] = x
    q = torch.randn(sum(new), 32, D, generator=g, device="cuda").to(BF16)
    want = hq.paged_attention(q, *small, table, _i32(seq), _cu(new))
    assert torch.equal(hq.paged_attention(q, kp, vp, ks, vs, high, _i32(seq), _cu(new)), want)
    slots = torch.tensor([(pages - 1) * page + 63, (pages - used) * page], device="cuda")
    x = torch.randn(2, H, D, generator=g, device="cuda").to(BF16)
    hq.paged_append(x, x, slots, kp, vp, ks, vs)
    c, s = U.quantise(x)
    assert torch.equal(kp[slots // page, :, slots % page], c) and torch.equal(vs[slots // page, :, slots % page], s)
    k, _ = hq.paged_gather(slots, kp, vp, ks, vs)
    assert torch.equal(k, U.values(c, s).float().to(BF16))


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------


def _step(b, page, q, k, v, pool, table, **kw):
    hq.paged_append(k, v, b.slots, *pool)
    return hq.paged_attention(q, *pool, table, b.seq_lens, b.cu_seqlens, **kw)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_steps_together(dtype):
    """Prompts, a chunk beside decode steps, a request that joins late: the
    cache and the outputs of every step against 64 bits."""
    g = _gen(20)
    page, H, G, D, pages = 16, 2, 4, 128, 80
    pool = U.make_pool(g, pages, H, page, D, "cuda")
    table = torch.full((3, 20), -1, dtype=torch.int32, device="cuda")
    free = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    ctx, rows = [0, 0, 0], [[], [], []]
    for new in ([100, 37, 0], [1, 1, 64], [1, 30, 1], [1, 1, 1], [1, 1, 1]):
        T = sum(new) + 3
        q, k, v = (torch.randn(T, h, D, generator=g, device="cuda").to(dtype) for h in (H * G, H, H))
        b = hq.paged_batch(_i32(ctx), _i32(new), table, free, page, T)
        free = free[int(b.pages_used):]
        out = _step(b, page, q, k, v, pool, table)
        at = 0
        for r, n in enumerate(new):
            rows[r].append((k[at:at + n], v[at:at + n]))
            at += n
        ctx = [a + n for a, n in zip(ctx, new)]
        for r in range(3):                               # the cache holds every row that was appended
            if ctx[r]:
                j = torch.arange(ctx[r], device="cuda")
                for i in (0, 1):
                    c, s = U.quantise(torch.cat([x[i] for x in rows[r]]))
                    ids = table[r, j // page].long()
                    assert torch.equal(pool[i][ids, :, j % page], c) and torch.equal(pool[2 + i][ids, :, j % page], s)
        ref, _, tol = U.reference(q[:sum(new)], pool, table, ctx, new)
        U.check(out[:sum(new)], ref, tol)


@pytest.mark.parametrize("decode", [False, True])
def test_captured_steps(decode):
    """A graph of a whole step replayed with other lengths, with eager work in
    between, and two graphs replayed on two streams at once."""
    g = _gen(21)
    page, H, G, D, R, T = 16, 2, 4, 128, 4, 4 if decode else 200
    pages = 650
    lens = [[1000, 20, 300, 5], [1, 2, 3, 4], [2000, 1500, 15, 16]]
    news = [[1] * 4] * 3 if decode else [[1, 100, 30, 60], [50, 0, 1, 2], [1, 1, 100, 90]]
    pools = [U.make_pool(_gen(22 + i), pages, H, page, D, "cuda") for i in range(2)]
    table = torch.randperm(4 * 150, generator=g, device="cuda").to(torch.int32).reshape(4, 150) % 600
    free = torch.arange(600, 650, dtype=torch.int32, device="cuda")
    qs, ks, vs = (torch.randn(T, h, D, generator=g, device="cuda").to(BF16) for h in (H * G, H, H))
    ctx, new = [_i32([0] * 4) for _ in range(2)], [_i32([1] * 4) for _ in range(2)]

    def step(i):
        b = hq.paged_batch(ctx[i], new[i], table[:], free, page, T)
        hq.paged_append(ks, vs, b.slots, *pools[i])
        return hq.paged_attention(qs, *pools[i], table, b.seq_lens, None if decode else b.cu_seqlens)

    keep, keep_table = [[x.clone() for x in p] for p in pools], table.clone()

    def reset():
        for p, k in zip(pools, keep):
            for a, b in zip(p, k):
                a.copy_(b)
        table.copy_(keep_table)

    def lengths(i, s):
        new[i].copy_(_i32(news[s]))
        ctx[i].copy_(_i32([max(a - b, 0) for a, b in zip(lens[s], news[s])]))

    step(0)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(step(i))
        graphs.append(gr)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in (0, 1, 2, 0, 2):
        want = []
        for i in range(2):
            reset()
            lengths(i, (s + i) % 3)
            want.append(step(i).clone())
        for i in range(2):                               # one after the other
            reset()
            lengths(i, (s + i) % 3)
            outs[i].fill_(9.0)
            graphs[i].replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[i], want[i])
        reset()
        if not decode:
            continue
        # at once (a decode step within a page takes none, so the shared table does not change)
        table0 = table.clone()
        for i in range(2):
            lengths(i, 0)
        want = [step(i).clone() for i in range(2)]
        torch.cuda.synchronize()
        assert torch.equal(table, table0)
        for st, gr in zip(streams, graphs):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_calls_on_two_streams():
    g = _gen(30)
    seq, page = [3000, 500, 17], 32
    table, pages = U.make_table(g, seq, page, "cuda")
    pool = U.make_pool(g, pages, 2, page, 128, "cuda")
    q = [torch.randn(3, 8, 128, generator=g, device="cuda").to(BF16) for _ in range(2)]
    want = [hq.paged_attention(x, *pool, table, _i32(seq)) for x in q]
    lens = _i32(seq)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        got = []
        for st, x in zip(streams, q):
            with torch.cuda.stream(st):
                got += [hq.paged_attention(x, *pool, table, lens) for _ in range(3)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got[:3], [want[0]] * 3)) and all(torch.equal(a, want[1]) for a in got[3:])


def test_repeat_is_bit_equal():
    g = _gen(31)
    seq, new = [5000, 300, 900], [1, 300, 64]
    table, pages = U.make_table(g, seq, 16, "cuda")
    pool = U.make_pool(g, pages, 8, 16, 128, "cuda")
    q = torch.randn(sum(new), 32, 128, generator=g, device="cuda").to(BF16)
    a = [hq.paged_attention(q, *pool, table, _i32(seq), _cu(new), return_lse=True) for _ in range(5)]
    assert all(torch.equal(x[0], a[0][0]) and torch.equal(x[1], a[0][1]) for x in a[1:])


# ---------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------


def test_refusals():
    g = _gen(40)
    pool = U.make_pool(g, 4, 2, 16, 128, "cuda")
    kp, vp, ks, vs = pool
    table, lens = _i32([[0, 1], [2, 3]]), _i32([20, 30])
    q = torch.randn(2, 8, 128, generator=g, device="cuda").to(BF16)
    k = torch.randn(2, 2, 128, generator=g, device="cuda").to(BF16)
    slots = torch.tensor([0, 1], device="cuda")
    ok = dict(q=q, k_pages=kp, v_pages=vp, k_scale=ks, v_scale=vs, block_table=table, seq_lens=lens)
    for change, word in ((dict(q=q.float()), "bf16 or fp16"), (dict(q=q[:, :7]), "multiple"), (dict(q=q[0]), "q must be"),
                         (dict(q=q.cpu()), "GPU"), (dict(q=q[..., :64]), "q must be"), (dict(k_pages=kp.float()), "k_pages"),
                         (dict(v_scale=vs.float()), "v_scale"), (dict(k_scale=ks[:3]), "shapes"), (dict(seq_lens=lens.long()), "seq_lens"),
                         (dict(block_table=table.long()), "block_table"), (dict(block_table=table[:1]), "requests"),
                         (dict(q=q[:1]), "cu_seqlens"), (dict(cu_seqlens=_i32([0, 2])), "cu_seqlens"), (dict(window=-1), "window"),
                         (dict(seq_lens=lens.cpu()), "cpu"), (dict(out=q[:1]), "out"), (dict(out=q.half()), "out"),
                         (dict(sm_scale=float("nan")), "sm_scale"), (dict(sm_scale=float("inf")), "sm_scale"),
                         (dict(v_pages=vp.transpose(0, 1).contiguous().transpose(0, 1)), "strides"),
                         (dict(block_table=table.t().contiguous().t()), "block_table")):
        with pytest.raises(ValueError, match=word):
            hq.paged_attention(**{**ok, **change})
    odd = U.make_pool(g, 2, 2, 24, 128, "cuda")
    with pytest.raises(ValueError, match="page size"):
        hq.paged_attention(q, *odd, table, lens)
    with pytest.raises(ValueError, match="head dim"):
        hq.paged_append(k[..., :96], k[..., :96], slots, *(x[..., :48] if x.dim() == 4 else x for x in pool))
    for args, word in (((k.float(), k.float(), slots), "bf16 or fp16"), ((k, k.half(), slots), "one dtype"), ((k, k[:1], slots), "must be"),
                       ((k, k, slots.int()), "slots"), ((k, k, slots[:1]), "slots"), ((k[:, :1], k[:, :1], slots), "must be")):
        with pytest.raises(ValueError, match=word):
            hq.paged_append(*args, *pool)
    with pytest.raises(ValueError, match="bf16 or fp16"):
        hq.paged_gather(slots, *pool, dtype=torch.float32)
    for args, word in (((lens.long(), lens, table, lens, 16, 4), "context_lens"), ((lens, lens[:1], table, lens, 16, 4), "requests"),
                       ((lens, lens, table, lens, 48, 4), "page size"), ((lens, lens, table, lens, 16, -1), "num_tokens"),
                       ((lens, lens, table.long(), lens, 16, 4), "block_table")):
        with pytest.raises(ValueError, match=word):
            hq.paged_batch(*args)


@pytest.mark.parametrize("R", [65, 200, 256, 257, 400])
@pytest.mark.parametrize("decode", [True, False])
def test_attention_batches_of_long_and_short_requests(R, decode):
    """Schedules on both sides of 64 and 256 requests, with tiles that are cut
    and tiles that are not, in both kinds of tiles."""
    g = torch.Generator().manual_seed(R)
    seq = torch.randint(1, 60, (R,), generator=g).tolist()
    new = [1] * R
    seq[3], seq[R // 2], seq[-1], seq[7] = 9000, 5003, 2500, 0
    if not decode:
        new = [min(n, s) for n, s in zip(torch.randint(0, 9, (R,), generator=g).tolist(), seq)]
        new[3], new[R // 2], new[-1] = 300, 2, 70
    else:
        new[7] = 1
    _attend(BF16, 64, 2, 4, 16, seq, new, decode=decode, seed=R, pad=0 if decode else 5)


@pytest.mark.parametrize("R", [5, 70, 300])
@pytest.mark.parametrize("G", [4, 32])
def test_attention_offsets_that_do_not_ascend(R, G):
    """More tiles than tokens: rows of such calls are unspecified, memory around the outputs is not touched."""
    g = _gen(R)
    seq, page, T = [600] * R, 16, 40
    table = torch.zeros(R, 40, dtype=torch.int32, device="cuda")
    pool = U.make_pool(g, 4, 2, page, 64, "cuda")
    q = torch.randn(T, 2 * G, 64, generator=g, device="cuda").to(BF16)
    big = torch.full((T + 8, 2 * G, 64), 3.0, dtype=BF16, device="cuda")
    for cu in ([0, T] * (R // 2 + 1), [T, 0] * (R // 2 + 1), [0, 2 ** 31 - 1, -2 ** 31] * (R // 3 + 1)):
        hq.paged_attention(q, *pool, table, _i32(seq), _i32(cu[:R + 1]), out=big[4:-4])
        assert bool((big[:4] == 3.0).all()) and bool((big[-4:] == 3.0).all())
    # and a call after them is as ever
    _attend(BF16, 64, 2, G, page, [600, 30], [10, 3])


@pytest.mark.parametrize("pad", [0, 9])
def test_attention_more_heads_than_a_short_tile(pad):
    """32 query heads on a key head: no tile of 16 rows, and tables too short for any tile to be cut."""
    for R in (1, 3, 70, 300):
        _attend(FP16, 128, 2, 32, 32, [33 + r % 7 for r in range(R)], [1 + r % 3 for r in range(R)], pad=pad, seed=R)
        _attend(BF16, 64, 1, 20, 16, [20] * R, [1] * R, decode=True, seed=R)


def test_native_and_checked_calls_agree(monkeypatch):
    """The C++ form of the calls and the Python form launch the same kernels."""
    from hyquant_amd import decode_d_stage as dd
    g = _gen(50)
    seq, new, page, H, G, D = [700, 65, 0, 130], [1, 65, 0, 9], 16, 2, 4, 64
    table, pages = U.make_table(g, seq, page, "cuda")
    T, pad = sum(new), 3
    ctx = [s - n for s, n in zip(seq, new)]
    pool = U.make_pool(g, pages, H, page, D, "cuda")
    q = torch.randn(T + pad, H * G, D, generator=g, device="cuda").to(FP16)
    kv = torch.randn(2, T + pad, H, D, generator=g, device="cuda").to(FP16)
    free = torch.arange(pages, dtype=torch.int32, device="cuda")

    def calls():
        t, p = torch.full_like(table, -1), tuple(x.clone() for x in pool)
        b = hq.paged_batch(_i32(ctx), _i32(new), t, free, page, T + pad)
        hq.paged_append(kv[0], kv[1], b.slots, *p)
        rows = hq.paged_gather(b.slots, *p, dtype=FP16)
        o = hq.paged_attention(q, *p, table, b.seq_lens, b.cu_seqlens, sm_scale=0.2, window=90, return_lse=True)
        d = hq.paged_attention(q[:4], *p, table, b.seq_lens)
        return (t, *p, *b, *rows, *o, d)

    native = calls()
    assert dd._FX
    monkeypatch.setattr(dd, "_FX", False)
    for i, (x, y) in enumerate(zip(native, calls())):
        assert x.dtype == y.dtype and torch.equal(x, y), i


def test_window_past_32_bits_and_shared_outputs():
    g = _gen(51)
    table, pages = U.make_table(g, [100, 40], 16, "cuda")
    pool = U.make_pool(g, pages, 2, 16, 64, "cuda")
    q = torch.randn(2, 8, 64, generator=g, device="cuda").to(BF16)
    lens = _i32([100, 40])
    want = hq.paged_attention(q, *pool, table, lens)
    for window in (1 << 30, 2 ** 31 - 1, 2 ** 33 + 5):
        assert torch.equal(hq.paged_attention(q, *pool, table, lens, window=window), want)
    row = torch.empty(1, 8, 64, dtype=BF16, device="cuda")
    for out in (q, row.expand(2, 8, 64), row.view(-1).as_strided((2, 8, 64), (64, 32, 1)), row[:, :1].expand(1, 8, 64).expand(2, 8, 64)):
        with pytest.raises(ValueError, match="share memory"):
            hq.paged_attention(q, *pool, table, lens, out=out)
    with pytest.raises(ValueError, match="num_tokens"):
        hq.paged_batch(lens, lens, table, lens, 16, 1 << 31)


@pytest.mark.parametrize("dtype,D,H,G,seq,window", [(BF16, 128, 8, 4, [8192], 0), (FP16, 64, 2, 16, [9000, 3, 700, 0, 5001], 0),
                                                    (BF16, 128, 1, 1, [20000], 0), (FP16, 128, 3, 7, [4000] * 70, 1500),
                                                    (BF16, 64, 4, 9, [100 + 90 * i for i in range(300)], 0),
                                                    (BF16, 128, 2, 13, [6000, 11, 2000], 0)])
def test_pieces_joined_by_either_launch(dtype, D, H, G, seq, window, monkeypatch):
    """A cut request's pieces are added up by its last workgroup, or by a launch
    of their own where a call has no counters: the same bits, also lse, and
    the counters are zero again."""
    from hyquant_amd import paged
    g = _gen(60)
    table, pages = U.make_table(g, seq, 16, "cuda")
    pool = U.make_pool(g, pages, H, 16, D, "cuda")
    q = torch.randn(len(seq), H * G, D, generator=g, device="cuda").to(dtype)
    lens = _i32(seq)
    got = [hq.paged_attention(q, *pool, table, lens, window=window, return_lse=True) for _ in range(3)]
    torch.cuda.synchronize()
    assert paged._counts and all(bool((c == 0).all()) for c in paged._counts.values())
    monkeypatch.setattr(paged, "_counters", lambda *_: 0)
    out, lse = hq.paged_attention(q, *pool, table, lens, window=window, return_lse=True)
    for o, x in got:
        assert torch.equal(o, out) and torch.equal(x, lse)
    ref, ref_lse, tol = U.reference(q, pool, table, seq, [1] * len(seq), window)
    U.check(out, ref, tol)


def test_captured_decode_replayed_beside_eager_calls():
    """A graph captured on a stream that has arrival counters leaves them alone:
    its replays on another stream run beside eager calls on that one."""
    from hyquant_amd import paged
    g = _gen(70)
    seq, H, G, D = [9000, 5000, 3001], 2, 8, 128
    table, pages = U.make_table(g, seq, 16, "cuda")
    pool = U.make_pool(g, pages, H, 16, D, "cuda")
    lens = _i32(seq)
    qa, qb = (torch.randn(3, H * G, D, generator=g, device="cuda").to(BF16) for _ in range(2))
    want_a, want_b = (hq.paged_attention(x, *pool, table, lens).clone() for x in (qa, qb))
    torch.cuda.synchronize()
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(s):
        hq.paged_attention(qa, *pool, table, lens)
    torch.cuda.synchronize()
    assert (0, s.cuda_stream) in paged._counts
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        captured = [hq.paged_attention(qa, *pool, table, lens) for _ in range(4)]
    for _ in range(5):
        for x in captured:
            x.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(t):
            graph.replay()
        with torch.cuda.stream(s):
            eager = [hq.paged_attention(qb, *pool, table, lens) for _ in range(8)]
        torch.cuda.synchronize()
        assert all(torch.equal(x, want_a) for x in captured) and all(torch.equal(x, want_b) for x in eager)
    assert all(bool((c == 0).all()) for c in paged._counts.values())
