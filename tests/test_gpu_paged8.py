"""Attention over the paged 8-bit cache on the GPU against the definition in 64
bits, its masks and what hidden places may hold, whole steps together, and its
refusals."""

import math

import pytest
import torch

import hyquant_amd as hq
from tests import paged8_util as U
from tests import paged_bounds as B
from tests.paged_util import make_table

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _cu(new):
    return _i32([0] + torch.tensor(new, dtype=torch.int64).cumsum(0).tolist())


def _compare(got, q, pool, table, seq, new, window=0, sm_scale=None, what=""):
    """Value by value, and whole outputs' norms and roundings."""
    out, lse = got
    n = sum(new)
    ref, ref_lse, tol, lse_tol, E = U.reference(q[:n], pool, table, seq, new, window, sm_scale)
    U.check(out[:n], ref, tol, what)
    assert torch.equal(out[n:], torch.zeros_like(out[n:]))
    if ref.norm() > 0:
        B.check(out[:n], ref, E, what)
    if lse is not None:
        empty = torch.isinf(ref_lse)
        assert torch.equal(torch.isinf(lse[:n]), empty) and bool((lse[n:] == -math.inf).all())
        err = (lse[:n].double() - ref_lse)[~empty].abs()
        assert bool((err <= lse_tol[~empty]).all()), float((err / lse_tol[~empty]).max())


def _attend(dtype, D, H, G, page, seq, new, window=0, seed=0, sm_scale=None, lse=True, decode=False, pad=0, scale=1.0, amp=1.0):
    g = _gen(seed)
    table, pages = make_table(g, seq, page, "cuda")
    pool = U.make_pool(g, pages, H, page, D, "cuda", scale)
    T = sum(new) + pad
    q = (amp * torch.randn(T, H * G, D, generator=g, device="cuda")).to(dtype)
    got = hq.paged8_attention(q, *pool, table, _i32(seq), None if decode else _cu(new), sm_scale=sm_scale, window=window, return_lse=lse)
    _compare(got if lse else (got, None), q, pool, table, seq, new, window, sm_scale)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,G", [(8, 4), (2, 16), (1, 1), (3, 7)])
@pytest.mark.parametrize("page", [16, 64])
def test_decode(dtype, D, H, G, page):
    seq = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 500, 1000, 2049, 0]
    _attend(dtype, D, H, G, page, seq, [1] * len(seq), decode=True)


@pytest.mark.parametrize("dtype,D,H,G,page,seq", [(BF16, 128, 8, 4, 64, [8192]), (FP16, 128, 8, 4, 16, [32768, 3]),
                                                  (BF16, 128, 2, 8, 128, [20001, 7, 12345]), (FP16, 64, 8, 4, 256, [30011]),
                                                  (BF16, 128, 1, 16, 32, [4097] * 3), (FP16, 128, 8, 4, 64, [9000] * 48)])
@pytest.mark.parametrize("window", [0, 1000])
def test_decode_long(dtype, D, H, G, page, seq, window):
    _attend(dtype, D, H, G, page, seq, [1] * len(seq), window=window, decode=True, amp=2.0)


@pytest.mark.parametrize("R", [65, 200, 257, 1500])
@pytest.mark.parametrize("decode", [True, False])
def test_many_requests(R, decode):
    g = torch.Generator().manual_seed(R)
    seq = torch.randint(1, 60, (R,), generator=g).tolist()
    new = [1] * R
    seq[3], seq[R // 2], seq[-1], seq[7] = 9000, 5003, 2500, 0
    if not decode:
        new = [min(n, s) for n, s in zip(torch.randint(0, 9, (R,), generator=g).tolist(), seq)]
        new[3], new[R // 2], new[-1] = 300, 2, 70
    _attend(BF16, 64, 2, 4, 16, seq, new, decode=decode, seed=R, pad=0 if decode else 5)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D,H,G,page", [(128, 8, 4, 64), (64, 2, 16, 16), (128, 2, 8, 32), (128, 1, 3, 128), (64, 4, 1, 64), (128, 1, 32, 16)])
@pytest.mark.parametrize("window", [0, 1, 50, 300])
def test_ragged(dtype, D, H, G, page, window):
    new = [1, 5, 0, 33, 64, 1, 130, 2, 17]
    seq = [900, 5, 40, 133, 64, 1, 515, 3, 17]
    _attend(dtype, D, H, G, page, seq, new, window=window, pad=5)


@pytest.mark.parametrize("dtype,D,H,G,page,seq,new,window", [
    (BF16, 128, 8, 4, 64, [2500], [700], 0), (FP16, 128, 2, 8, 16, [1300, 4000], [1300, 77], 0),
    (BF16, 128, 1, 5, 32, [3001], [1001], 0), (FP16, 64, 4, 4, 128, [2000, 100, 5000], [2000, 100, 1], 0),
    (BF16, 64, 8, 4, 16, [6000, 700], [600, 700], 1024), (BF16, 128, 8, 8, 256, [20000], [40], 0)])
def test_chunks(dtype, D, H, G, page, seq, new, window):
    _attend(dtype, D, H, G, page, seq, new, window=window, amp=2.0)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("sm", [0.03, -0.05, 0.0, 1.0])
def test_score_scales(dtype, sm):
    _attend(dtype, 128, 2, 4, 16, [333, 70], [1, 20], sm_scale=sm)
    _attend(dtype, 64, 2, 4, 16, [333, 70], [1, 1], sm_scale=sm, decode=True)


@pytest.mark.parametrize("new", [[1, 1], [40, 30]])
@pytest.mark.parametrize("spread", [4, 30])
def test_block_scales_and_query_rows_far_apart(new, spread):
    """Blocks' scales 2^-spread to 2^spread of each other, K's so that scores stay
    moderate; query rows from 2^-30 to 2 side by side, that single out keys."""
    g = _gen(11)
    seq, page, H, G, D = [600, 211], 32, 2, 4, 128
    table, pages = make_table(g, seq, page, "cuda")
    pool = list(U.make_pool(g, pages, H, page, D, "cuda"))
    pool[2] = pool[2] * torch.exp2(torch.randint(-3, 2, pool[2].shape, generator=g, device="cuda").float())
    pool[3] = torch.exp2(torch.randint(-spread, spread + 1, pool[3].shape, generator=g, device="cuda").float())
    T = sum(new)
    q = torch.randn(T, H * G, D, generator=g, device="cuda") * torch.logspace(-30, 1, T * H * G, base=2, device="cuda").reshape(T, H * G, 1)
    for r in range(len(seq)):            # the last token's heads look for one key each
        k, _, sk, _, _ = U.held(pool, table[r], seq[r])
        for h in range(H * G):
            key = (37 * h + 5) % seq[r]
            q[sum(new[:r + 1]) - 1, h] = 3 * (k[h // G, key] * sk[h // G, key]).float()
    for dtype in (BF16, FP16) if spread < 9 else (BF16,):                   # (127 * 2^30 is no fp16 number)
        x = q.to(dtype)
        got = hq.paged8_attention(x, *pool, table, _i32(seq), _cu(new) if max(new) > 1 else None, return_lse=True)
        _compare(got, x, pool, table, seq, new)


@pytest.mark.parametrize("new", [[1], [30]])
def test_extreme_codes_and_scales(new):
    """Codes of -128 (which no append writes) and the largest and smallest scales."""
    g = _gen(12)
    table, pages = make_table(g, [100], 16, "cuda")
    pool = list(U.make_pool(g, pages, 2, 16, 64, "cuda"))
    pool[0][0], pool[1][:] = -128, torch.where(pool[1] % 3 == 0, -128, pool[1]).to(torch.int8)
    q = torch.randn(sum(new), 8, 64, generator=g, device="cuda").to(BF16)
    cu = _cu(new) if max(new) > 1 else None
    for sv in (2.0 ** -40, 2.0 ** 48):
        pool[3] = torch.full_like(pool[3], sv)
        got = hq.paged8_attention(q, *pool, table, _i32([100]), cu, return_lse=True)
        _compare(got, q, pool, table, [100], new)
    pool[3] = torch.ones_like(pool[3])
    for sk, x in ((2.0 ** -40, q * 2.0 ** 30), (2.0 ** 48, q * 2.0 ** -50)):
        pool[2] = torch.full_like(pool[2], sk)
        got = hq.paged8_attention(x, *pool, table, _i32([100]), cu, return_lse=True)
        _compare(got, x, pool, table, [100], new)


def test_rows_without_keys():
    # more new tokens than cached ones: the first rows are before position 0
    _attend(BF16, 128, 2, 4, 16, [3, 0, 40], [10, 4, 60])
    pool = U.make_pool(_gen(0), 0, 2, 16, 128, "cuda")                      # no pages at all
    q = torch.randn(3, 8, 128, generator=_gen(1), device="cuda").to(BF16)
    out, lse = hq.paged8_attention(q, *pool, _i32([[0], [1], [2]]), _i32([5, 6, 7]), return_lse=True)
    assert torch.equal(out, torch.zeros_like(out)) and bool((lse == -math.inf).all())
    out = hq.paged8_attention(q, *pool, torch.empty(3, 0, dtype=torch.int32, device="cuda"), _i32([5, 6, 7]))
    assert torch.equal(out, torch.zeros_like(out))
    out, lse = hq.paged8_attention(q, *pool, torch.empty(0, 1, dtype=torch.int32, device="cuda"), _i32([]), _i32([0]), return_lse=True)
    assert torch.equal(out, torch.zeros_like(out)) and bool((lse == -math.inf).all())
    assert hq.paged8_attention(q[:0], *pool, torch.empty(0, 1, dtype=torch.int32, device="cuda"), _i32([])).shape == (0, 8, 128)


@pytest.mark.parametrize("new", [[1, 1], [40, 3]])
@pytest.mark.parametrize("which", [2, 3])
def test_masked_places_hold_anything(new, which):
    """Scales that are not finite, zero or negative in blocks that no row sees
    change nothing; a row that sees one is NaN, the others are as ever."""
    g = _gen(4)
    seq, page, H, G, D = [77, 50], 32, 2, 4, 128
    table, pages = make_table(g, seq, page, "cuda")
    pool = U.make_pool(g, pages, H, page, D, "cuda")
    q = torch.randn(sum(new), H * G, D, generator=g, device="cuda").to(BF16)
    cu = _cu(new) if max(new) > 1 else None
    want, want_lse = hq.paged8_attention(q, *pool, table, _i32(seq), cu, return_lse=True)
    live = torch.zeros(pages, page, dtype=torch.bool, device="cuda")
    for r, n in enumerate(seq):
        for j in range(n):
            live[table[r, j // page], j % page] = True
    blocks = live.reshape(pages, page // 16, 16).any(-1)
    for bad in (math.nan, math.inf, -math.inf, 0.0, -1.0, 2.0 ** -41, 2.0 ** 49):
        dirty = [x.clone() for x in pool]
        for s in dirty[2:]:
            s.masked_fill_(~blocks[:, None], bad)
        for c in dirty[:2]:
            c.masked_fill_(~live[:, None, :, None], -128)
        t = table.clone()
        t[t < 0] = 12345678
        got, lse = hq.paged8_attention(q, *dirty, t, _i32(seq), cu, return_lse=True)
        assert torch.equal(got, want) and torch.equal(lse, want_lse)
        dirty[which][table[0, 76 // page], 1, 76 % page // 16] = bad       # the last block of request 0, keys 64 to 76, one head
        got, lse = hq.paged8_attention(q, *dirty, t, _i32(seq), cu, return_lse=True)
        hit = torch.zeros(sum(new), H * G, dtype=torch.bool, device="cuda")
        sees = [i for i in range(new[0]) if seq[0] - new[0] + i >= 64]
        hit[sees, G:] = True
        assert bool(got[hit].isnan().all()) and bool(lse[hit].isnan().all())
        assert torch.equal(got[~hit], want[~hit]) and torch.equal(lse[~hit], want_lse[~hit])


def test_nan_query_row_stays_alone():
    g = _gen(6)
    table, pages = make_table(g, [100], 16, "cuda")
    pool = U.make_pool(g, pages, 2, 16, 128, "cuda")
    for m in (9, 1):
        q = torch.randn(m, 8, 128, generator=g, device="cuda").to(BF16)
        want = hq.paged8_attention(q, *pool, table, _i32([100]), _cu([m]))
        for bad in (math.nan, math.inf):
            x = q.clone()
            x[m // 2, 3, 7] = bad
            got = hq.paged8_attention(x, *pool, table, _i32([100]), _cu([m]))
            assert bool(torch.isnan(got[m // 2, 3]).any())
            got[m // 2, 3] = want[m // 2, 3]
            assert torch.equal(got, want)


@pytest.mark.parametrize("new", [[1, 1, 1], [1, 70, 9]])
def test_pages_outside_the_pool(new):
    g = _gen(8)
    seq, page = [300, 400, 129], 16
    table, pages = make_table(g, seq, page, "cuda")
    table[0, 3], table[0, 18], table[1, 0], table[1, 7], table[2] = -1, pages, 2 ** 31 - 1, -2 ** 31, pages + 5
    pool = U.make_pool(g, pages, 2, page, 128, "cuda")
    q = torch.randn(sum(new), 8, 128, generator=g, device="cuda").to(BF16)
    got = hq.paged8_attention(q, *pool, table, _i32(seq), _cu(new) if max(new) > 1 else None, return_lse=True)
    _compare(got, q, pool, table, seq, new)
    assert bool((got[1][-new[2]:] == -math.inf).all()) and bool((got[0][-new[2]:] == 0).all())


def test_lengths_past_the_table_and_bad_cu():
    g = _gen(9)
    seq, page = [64, 48], 16
    table, pages = make_table(g, seq, page, "cuda", spare=8)
    table[0, 4], table[1, 3:] = pages - 1, torch.tensor([pages - 2, pages - 3], dtype=torch.int32, device="cuda")
    pool = U.make_pool(g, pages, 2, page, 128, "cuda")
    q = torch.randn(2, 8, 128, generator=g, device="cuda").to(BF16)
    a = hq.paged8_attention(q, *pool, table, _i32([10 ** 9, -4]))          # 80 tokens in a row of the table; none
    b = hq.paged8_attention(q, *pool, table, _i32([80, 0]))
    assert torch.equal(a, b) and bool((b[1] == 0).all())
    big = torch.full((6, 8, 128), 3.0, dtype=BF16, device="cuda")
    for cu in ([-5, 1, 900], [0, 2 ** 31 - 1, -2 ** 31], [2, 1, 0], [7, 8, 9]):
        hq.paged8_attention(q, *pool, table, _i32([64, 48]), _i32(cu), out=big[2:4])
        assert bool((big[:2] == 3.0).all()) and bool((big[4:] == 3.0).all())


def test_strides_out_and_repeats():
    g = _gen(10)
    seq, new, page, H, G, D = [200, 65, 130], [1, 65, 9], 32, 2, 4, 128
    T, pad = sum(new), 4
    table, pages = make_table(g, seq, page, "cuda")
    pool = U.make_pool(g, pages, H, page, D, "cuda")
    wide = torch.full((3, table.shape[1] + 7), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    codes = torch.zeros(3, pages, 2, H, page, D, dtype=torch.int8, device="cuda")       # K and V of a page side by side, one layer of three
    scales = torch.zeros(3, pages, 2, H, page // 16, device="cuda")
    codes[1, :, 0], codes[1, :, 1], scales[1, :, 0], scales[1, :, 1] = pool
    view = (codes[1, :, 0], codes[1, :, 1], scales[1, :, 0], scales[1, :, 1])
    qkv = torch.randn(T + pad, H * G + 2 * H, D, generator=g, device="cuda").to(BF16)
    q = qkv[:, :H * G]
    want = hq.paged8_attention(q.contiguous(), *pool, table, _i32(seq), _cu(new))
    _compare((want, None), q, pool, table, seq, new)
    out = torch.full((H * G, T + pad, D), 7.0, dtype=BF16, device="cuda").transpose(0, 1)
    got = hq.paged8_attention(q, *view, wide[:, :table.shape[1]], _i32(seq), _cu(new), out=out)
    assert got is out and torch.equal(out[:T], want[:T]) and bool((out[T:] == 7.0).all())
    odd = torch.randn((T + pad) * H * G * D + 1, generator=g, device="cuda").to(BF16)[1:].reshape(T + pad, H * G, D)
    odd.copy_(q)                                         # rows at odd addresses: copied
    assert torch.equal(hq.paged8_attention(odd, *pool, table, _i32(seq), _cu(new)), want)
    for _ in range(3):
        assert torch.equal(hq.paged8_attention(q, *pool, table, _i32(seq), _cu(new)), want)
    for window in (1 << 30, 2 ** 31 - 1, 2 ** 33 + 5):
        assert torch.equal(hq.paged8_attention(q, *pool, table, _i32(seq), _cu(new), window=window), want)


def test_pool_past_32_bits():
    """Pages whose codes start beyond 4 GiB."""
    g = _gen(12)
    page, H, D = 64, 8, 128
    pages = 5 * 2 ** 30 // (H * page * D)
    seq, new = [500, 130], [1, 30]
    kp, vp = (torch.empty(pages, H, page, D, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.empty(pages, H, page // 16, device="cuda") for _ in range(2))
    table, used = make_table(g, seq, page, "cuda", spare=0)
    small = U.make_pool(g, used, H, page, D, "cuda")
    high = torch.where(table >= 0, table + (pages - used), table)
    for big, x in zip((kp, vp, ks, vs), small):
        big[pages - used:] = x
    q = torch.randn(sum(new), 32, D, generator=g, device="cuda").to(BF16)
    want = hq.paged8_attention(q, *small, table, _i32(seq), _cu(new))
    assert torch.equal(hq.paged8_attention(q, kp, vp, ks, vs, high, _i32(seq), _cu(new)), want)


@pytest.mark.parametrize("R", [5, 70, 300])
@pytest.mark.parametrize("G", [4, 32])
def test_offsets_that_do_not_ascend(R, G):
    """More tiles than tokens: rows of such calls are unspecified, memory around the outputs is not touched."""
    g = _gen(R)
    seq, page, T = [600] * R, 16, 40
    table = torch.zeros(R, 40, dtype=torch.int32, device="cuda")
    pool = U.make_pool(g, 4, 2, page, 64, "cuda")
    q = torch.randn(T, 2 * G, 64, generator=g, device="cuda").to(BF16)
    big = torch.full((T + 8, 2 * G, 64), 3.0, dtype=BF16, device="cuda")
    for cu in ([0, T] * (R // 2 + 1), [T, 0] * (R // 2 + 1), [0, 2 ** 31 - 1, -2 ** 31] * (R // 3 + 1)):
        hq.paged8_attention(q, *pool, table, _i32(seq), _i32(cu[:R + 1]), out=big[4:-4])
        assert bool((big[:4] == 3.0).all()) and bool((big[-4:] == 3.0).all())
    _attend(BF16, 64, 2, G, page, [600, 30], [10, 3])    # and a call after them is as ever


@pytest.mark.parametrize("dtype,D,H,G,seq,window", [(BF16, 128, 8, 4, [8192], 0), (FP16, 64, 2, 16, [9000, 3, 700, 0, 5001], 0),
                                                    (BF16, 128, 1, 1, [20000], 0), (FP16, 128, 3, 7, [4000] * 70, 1500),
                                                    (BF16, 64, 4, 9, [100 + 90 * i for i in range(300)], 0)])
def test_pieces_joined_by_either_launch(dtype, D, H, G, seq, window, monkeypatch):
    """A cut request's pieces are added up by its last workgroup, or by a launch of
    their own where a call has no counters: the same bits, also beside calls on
    the 4-bit cache, whose counters they are."""
    from hyquant_amd import paged
    from tests import paged_util as U4
    g = _gen(60)
    table, pages = make_table(g, seq, 16, "cuda")
    pool = U.make_pool(g, pages, H, 16, D, "cuda")
    pool4 = U4.make_pool(g, pages, H, 16, D, "cuda")
    q = torch.randn(len(seq), H * G, D, generator=g, device="cuda").to(dtype)
    lens = _i32(seq)
    got = []
    for _ in range(3):
        got.append(hq.paged8_attention(q, *pool, table, lens, window=window, return_lse=True))
        hq.paged_attention(q, *pool4, table, lens, window=window)
    torch.cuda.synchronize()
    assert paged._counts and all(bool((c == 0).all()) for c in paged._counts.values())
    monkeypatch.setattr(paged, "_counters", lambda *_: 0)
    out, lse = hq.paged8_attention(q, *pool, table, lens, window=window, return_lse=True)
    for o, x in got:
        assert torch.equal(o, out) and torch.equal(x, lse)
    _compare((out, lse), q, pool, table, seq, [1] * len(seq), window)


@pytest.mark.parametrize("dtype,interleaved,norm", [(BF16, False, True), (FP16, True, False)])
def test_steps_together(dtype, interleaved, norm):
    """A serving program's steps: prompts, a chunk beside decode steps, a request
    that joins late.  Layout, rotated append and attention, cache and outputs of
    every step against 64 bits."""
    from tests import rope_util as R
    g = _gen(20)
    page, H, G, D, pages = 32, 2, 4, 128, 40
    pool = tuple(torch.zeros(pages, H, page, D, dtype=torch.int8, device="cuda") for _ in range(2)) + tuple(
        torch.zeros(pages, H, page // 16, device="cuda") for _ in range(2))
    mine = [x.cpu().clone() for x in pool]
    table = torch.full((3, 10), -1, dtype=torch.int32, device="cuda")
    free = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    cos, sin = R.tables(300, D, device="cuda")
    qw, kw = (torch.randn(D, generator=g, device="cuda").to(dtype) if norm else None for _ in range(2))
    ctx = [0, 0, 0]
    for new in ([100, 37, 0], [1, 1, 64], [1, 30, 1], [1, 1, 1], [1, 1, 1]):
        T = sum(new) + 3
        x = torch.randn(T, H * G + 2 * H, D, generator=g, device="cuda").to(dtype)
        q, k, v = x[:, :H * G], x[:, H * G:-H], x[:, -H:]
        b = hq.paged_batch(_i32(ctx), _i32(new), table, free, page, T)
        free = free[int(b.pages_used):]
        turned = hq.paged_rope_append(q, k, v, cos, sin, b.positions, b.slots, *pool, q_weight=qw, k_weight=kw, interleaved=interleaved)
        out, lse = hq.paged8_attention(turned, *pool, table, b.seq_lens, b.cu_seqlens, return_lse=True)
        at = b.positions.clamp(min=0)
        ref, big = R.turn(q, cos[at], sin[at], qw, 1e-6, interleaved)
        live = b.positions >= 0
        assert bool(((turned.double() - ref).abs() <= R.tolerance(ref, big, dtype))[live].all()) and not turned[~live].any()
        rows = R.turn(k, cos[at], sin[at], kw, 1e-6, interleaved)[0].cpu(), v.double().cpu()
        for i in range(2):
            R.append8(mine[i], mine[2 + i], rows[i], b.slots.tolist())
            assert torch.equal(mine[i], pool[i].cpu()) and torch.equal(mine[2 + i], pool[2 + i].cpu())
        ctx = [a + n for a, n in zip(ctx, new)]
        _compare((out, lse), turned, pool, table, ctx, new)


@pytest.mark.parametrize("decode", [False, True])
def test_captured_steps(decode):
    """A graph of a whole step replayed with other lengths, with eager calls in
    between, and two graphs replayed on two streams at once."""
    from tests import rope_util as R
    g = _gen(21)
    page, H, G, D, T = 16, 2, 4, 128, 4 if decode else 200
    pages = 650
    lens = [[1000, 20, 300, 5], [1, 2, 3, 4], [2000, 1500, 15, 16]]
    news = [[1] * 4] * 3 if decode else [[1, 100, 30, 5], [1, 0, 1, 2], [1, 1, 15, 16]]
    cos, sin = R.tables(2500, D, device="cuda")
    pools = [U.make_pool(_gen(22 + i), pages, H, page, D, "cuda") for i in range(2)]
    table = torch.randperm(600, generator=g, device="cuda").to(torch.int32).reshape(4, 150)
    free = torch.arange(600, 650, dtype=torch.int32, device="cuda")
    x = torch.randn(T, H * G + 2 * H, D, generator=g, device="cuda").to(BF16)
    ctx, new = [_i32([0] * 4) for _ in range(2)], [_i32([1] * 4) for _ in range(2)]
    tables = [table.clone() for _ in range(2)]

    def step(i):
        b = hq.paged_batch(ctx[i], new[i], tables[i], free, page, T)
        q = hq.paged_rope_append(x[:, :H * G], x[:, H * G:-H], x[:, -H:], cos, sin, b.positions, b.slots, *pools[i])
        return hq.paged8_attention(q, *pools[i], tables[i], b.seq_lens, None if decode else b.cu_seqlens)

    keep = [[t.clone() for t in p] for p in pools]

    def reset(s):
        for i in range(2):
            for a, b in zip(pools[i], keep[i]):
                a.copy_(b)
            tables[i].copy_(table)
            k = (s + i) % 3
            new[i].copy_(_i32(news[k]))
            ctx[i].copy_(_i32([max(a - b, 0) for a, b in zip(lens[k], news[k])]))

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
        reset(s)
        want = [step(i).clone() for i in range(2)]
        cache = [[t.clone() for t in p] for p in pools]
        for together in (False, True):
            reset(s)
            for o in outs:
                o.fill_(9.0)
            torch.cuda.synchronize()
            for st, gr in zip(streams, graphs):
                with torch.cuda.stream(st if together else streams[0]):
                    gr.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs, want))
            assert all(torch.equal(a, b) for p, c in zip(pools, cache) for a, b in zip(p, c))


def test_calls_on_two_streams():
    g = _gen(30)
    seq, page = [3000, 500, 17], 32
    table, pages = make_table(g, seq, page, "cuda")
    pool = U.make_pool(g, pages, 2, page, 128, "cuda")
    q = [torch.randn(3, 8, 128, generator=g, device="cuda").to(BF16) for _ in range(2)]
    lens = _i32(seq)
    want = [hq.paged8_attention(x, *pool, table, lens) for x in q]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        got = []
        for st, x in zip(streams, q):
            with torch.cuda.stream(st):
                got += [hq.paged8_attention(x, *pool, table, lens) for _ in range(3)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, want[0]) for a in got[:3]) and all(torch.equal(a, want[1]) for a in got[3:])


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
                         (dict(v_scale=vs.half()), "v_scale"), (dict(k_scale=ks[:3]), "shapes"), (dict(seq_lens=lens.long()), "seq_lens"),
                         (dict(block_table=table.long()), "block_table"), (dict(block_table=table[:1]), "requests"),
                         (dict(q=q[:1]), "cu_seqlens"), (dict(cu_seqlens=_i32([0, 2])), "cu_seqlens"), (dict(window=-1), "window"),
                         (dict(seq_lens=lens.cpu()), "cpu"), (dict(out=q[:1]), "out"), (dict(out=q.half()), "out"), (dict(out=q), "share memory"),
                         (dict(sm_scale=float("nan")), "sm_scale"), (dict(sm_scale=float("inf")), "sm_scale"),
                         (dict(v_pages=vp.transpose(0, 1).contiguous().transpose(0, 1)), "strides")):
        with pytest.raises(ValueError, match=word):
            hq.paged8_attention(**{**ok, **change})
    for args, word in (((k.float(), k.float(), slots), "bf16 or fp16"), ((k, k.half(), slots), "one dtype"), ((k, k[:1], slots), "must be"),
                       ((k, k, slots.int()), "slots"), ((k, k, slots[:1]), "slots"), ((k[:, :1], k[:, :1], slots), "must be")):
        with pytest.raises(ValueError, match=word):
            hq.paged8_append(*args, *pool)
    with pytest.raises(ValueError, match="bf16 or fp16"):
        hq.paged8_gather(slots, *pool, dtype=torch.float32)
    with pytest.raises(ValueError, match="k_scale"):     # a 4-bit pool's scales
        hq.paged8_append(k, k, slots, kp, vp, ks.half(), vs.half())
    cos = torch.zeros(4, 64, device="cuda")
    for args, word in (((q, k, k.half(), cos, cos, slots, slots), "v must"), ((q, k, k[:, :1], cos, cos, slots, slots), "must be"),
                       ((q, k, k, cos, cos, slots.int(), slots), "positions"), ((q, k, k, cos, cos, slots, slots[:1]), "slots"),
                       ((q, k, k, cos.cpu(), cos, slots, slots), "cos"), ((q.float(), k, k, cos, cos, slots, slots), "bf16 or fp16")):
        with pytest.raises(ValueError, match=word):
            hq.paged_rope_append(*args, *pool)
