"""Calls of the paged operators at the edges of what they allow."""

import math

import pytest
import torch

import hyquant_amd as hq
from hyquant_amd import decode_d_stage as dd
from tests import paged_util as U

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _cu(new):
    return _i32([0] + torch.tensor(new, dtype=torch.int64).cumsum(0).tolist())


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("G,R", [(1, 2), (4, 2), (4, 300)])
def test_largest_windows_and_rows_before_position_0(native, G, R, monkeypatch):
    """More new tokens than cached ones under windows that hide nothing: the same
    as without a window, in short tiles and long ones and by both forms of the call."""
    if not native:
        monkeypatch.setattr(dd, "_FX", False)
    g, page = _gen(1), 16
    seq, new = [5, 40] + [7] * (R - 2), [10, 300] + [12] * (R - 2)
    table, pages = U.make_table(g, seq, page, "cuda")
    pool = U.make_pool(g, pages, 2, page, 64, "cuda")
    q = torch.randn(sum(new), 2 * G, 64, generator=g, device="cuda").to(BF16)
    want, want_lse = hq.paged_attention(q, *pool, table, _i32(seq), _cu(new), return_lse=True)
    assert bool((want[5:10] != 0).any(-1).all()) and bool(torch.isfinite(want_lse[5:10]).all())
    for window in (1 << 20, (1 << 30) - 1, 1 << 30, (1 << 31) - 257, (1 << 31) - 2, (1 << 31) - 1, 1 << 40):
        out, lse = hq.paged_attention(q, *pool, table, _i32(seq), _cu(new), window=window, return_lse=True)
        assert torch.equal(out, want) and torch.equal(lse, want_lse), window


def test_batch_layout_of_most_tokens():
    """Token tensors of 2^31 - 1 entries, nearly all of them padding."""
    T = 2 ** 31 - 1
    table = _i32([[3, -1], [7, -1]])
    b = hq.paged_batch(_i32([14, 0]), _i32([4, 2]), table, _i32([5, 9]), 16, T)
    assert b.slots.shape == b.positions.shape == (T,)
    assert b.slots[:8].tolist() == [62, 63, 80, 81, 144, 145, -1, -1] and b.positions[:8].tolist() == [14, 15, 16, 17, 0, 1, -1, -1]
    for x in (b.slots, b.positions):
        for part in x[6:].split(1 << 28):
            assert bool((part == -1).all())
    assert table.tolist() == [[3, 5], [9, -1]] and b.cu_seqlens.tolist() == [0, 4, 6] and b.pages_used.tolist() == [2]


@pytest.mark.parametrize("native", [True, False])
def test_batch_tables_whose_rows_share_memory(native, monkeypatch):
    if not native:
        monkeypatch.setattr(dd, "_FX", False)
    lens, free = _i32([3, 3]), _i32([5, 6, 7, 8])
    flat = torch.full((8,), -1, dtype=torch.int32, device="cuda")
    for table in (flat[:4].expand(2, 4), flat.as_strided((2, 4), (3, 1))):
        with pytest.raises(ValueError, match="share memory"):
            hq.paged_batch(lens, lens, table, free, 16, 6)
    assert bool((flat == -1).all())
    b = hq.paged_batch(lens[:1], lens[:1], flat[:4].expand(1, 4), free, 16, 3)      # one row shares it with none
    assert b.slots.tolist() == [-1] * 3                                               # (its held page is entry -1)
    b = hq.paged_batch(lens, lens, flat.as_strided((2, 1), (1, 1)), free, 16, 6)
    assert b.cu_seqlens.tolist() == [0, 3, 6]


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("D,seq,new,window", [(128, [700, 90], [1, 1], 0), (128, [700, 90], [65, 40], 0), (64, [9000, 300], [80, 80], 0),
                                              (64, [9000, 300], [1, 1], 500), (128, [30, 200], [40, 200], 64)])
def test_v_scales_that_are_not_finite(bad, D, seq, new, window):
    """A row that sees one is NaN, in short requests, long ones and cut ones; its lse
    does not depend on V, and other rows and heads are left alone."""
    g, page, H, G = _gen(3), 16, 2, 4
    table, pages = U.make_table(g, seq, page, "cuda")
    pool = U.make_pool(g, pages, H, page, D, "cuda")
    q = torch.randn(sum(new), H * G, D, generator=g, device="cuda").to(BF16)
    want, want_lse = hq.paged_attention(q, *pool, table, _i32(seq), _cu(new), window=window, return_lse=True)
    at = max(seq[0] - new[0] // 2 - 5, 0)                # request 0's key of head 1
    vs = pool[3].clone()
    vs[table[0, at // page], 1, at % page] = bad
    out, lse = hq.paged_attention(q, *pool[:3], vs, table, _i32(seq), _cu(new), window=window, return_lse=True)
    pos = seq[0] - new[0] + torch.arange(new[0], device="cuda")
    sees = (pos >= at) & ((pos < at + window) if window else True)
    assert bool(sees.any())
    hit = torch.zeros(sum(new), H * G, dtype=torch.bool, device="cuda")
    hit[:new[0], G:] = sees[:, None]
    assert bool(torch.isnan(out[hit]).all()) and torch.equal(out[~hit], want[~hit]) and torch.equal(lse[~hit], want_lse[~hit])
    # (the rows' references differ: fp32 roundings of m and log2 l)
    assert bool(((lse - want_lse)[hit].abs() <= 2.0 ** -20 * (1 + want_lse[hit].abs())).all())


def _decode_setup(seed=4):
    g, seq, page, H, G, D = _gen(seed), [9000, 5000, 3001], 16, 2, 8, 128
    table, pages = U.make_table(g, seq, page, "cuda")
    pool = U.make_pool(g, pages, H, page, D, "cuda")
    q = torch.randn(3, H * G, D, generator=g, device="cuda").to(BF16)
    return q, pool, table, _i32(seq)


def test_arrivals_left_behind_do_not_count(monkeypatch):
    """What a call leaves in the counters whose lengths were changed while it ran
    (arrivals, but not the last one) does no harm to the calls after it."""
    from hyquant_amd import paged
    q, pool, table, lens = _decode_setup()
    qs = [q, 3 * q, -q]                                  # (other memory and other values from call to call)
    with monkeypatch.context() as m:
        m.setattr(paged, "_counters", lambda *_: 0)
        want = [hq.paged_attention(x, *pool, table, lens) for x in qs]
    assert torch.equal(hq.paged_attention(q, *pool, table, lens), want[0])
    stream = torch.cuda.current_stream().cuda_stream
    words = paged._counts[(0, stream)].view(torch.int64)
    for left in (1, 2, 5, 30, 200):
        words.fill_(left)                                # (of the call before the first)
        got = [hq.paged_attention(x, *pool, table, lens) for x in qs]
        assert all(torch.equal(x, y) for x, y in zip(got, want)), left
        for x in got:
            x.fill_(7.0)                                 # (the next calls get this memory)
    words.zero_()


def test_streams_of_others_have_no_counters():
    """A handle that torch does not own may come back for another stream: its calls
    take the form without state."""
    from hyquant_amd import paged
    q, pool, table, lens = _decode_setup()
    want = hq.paged_attention(q, *pool, table, lens)
    torch.cuda.synchronize()
    own = torch.cuda.Stream()
    other = torch.cuda.ExternalStream(own.cuda_stream)
    known = (0, own.cuda_stream) in paged._counts        # (torch hands its streams out in turn)
    with torch.cuda.stream(other):
        got = [hq.paged_attention(q, *pool, table, lens) for _ in range(4)]
    torch.cuda.synchronize()
    assert ((0, own.cuda_stream) in paged._counts) == known
    assert all(torch.equal(x, want) for x in got)
    with torch.cuda.stream(own):                         # and torch's stream has them after all
        got = [hq.paged_attention(q, *pool, table, lens) for _ in range(4)]
    torch.cuda.synchronize()
    assert (0, own.cuda_stream) in paged._counts and all(torch.equal(x, want) for x in got)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [64, 128])
def test_append_rows_that_are_not_finite(dtype, D):
    """Rows with NaN and infinities among their channels: quantize_per_token's codes and scales all the same."""
    g, H, page = _gen(6), 2, 16
    x = torch.randn(40, H, D, generator=g, device="cuda")
    x[0, 0, 3], x[1, 1, D - 1], x[2, 0, 0], x[3] = math.nan, math.inf, -math.inf, math.nan
    x[4, 1, 5], x[4, 1, 6], x[5, 0, 7], x[5, 0, 8] = math.nan, math.inf, math.inf, -math.inf
    x = x.to(dtype)
    pool = tuple(t.clone() for t in U.make_pool(g, 4, H, page, D, "cuda"))
    slots = torch.randperm(4 * page, generator=g, device="cuda")[:40]
    hq.paged_append(x, x, slots, *pool)
    c, s = hq.quantize_per_token(x.reshape(-1, 1, D).contiguous(), 4)
    for i in (0, 1):
        assert torch.equal(pool[i][slots // page, :, slots % page], c.reshape(40, H, D // 2))
        assert torch.equal(pool[2 + i][slots // page, :, slots % page].view(torch.int16), s.reshape(40, H).view(torch.int16))


@pytest.mark.parametrize("native", [True, False])
def test_one_token_of_a_buffer_of_odd_pitch(native, monkeypatch):
    """The stride of a dimension of one is no stride: one token's rows of a buffer
    whose rows are no multiple of 16 bytes, as inputs and as out."""
    if not native:
        monkeypatch.setattr(dd, "_FX", False)
    g, H, G, D, page = _gen(8), 2, 4, 64, 16
    pool = U.make_pool(g, 3, H, page, D, "cuda")
    buf = torch.randn(6, 2 * H * D + H * G * D + 6, generator=g, device="cuda").to(BF16)
    at = 4                                               # (a row at a 16-byte address: 4 * 774 * 2 bytes)
    assert buf[at].data_ptr() % 16 == 0 and buf.stride(0) % 8
    k, v, q = (x.view(6, -1, D)[at:at + 1] for x in buf[:, :-6].split([H * D, H * D, H * G * D], 1))
    assert q.stride(0) % 8 and q.is_contiguous()
    slots = torch.tensor([20], device="cuda")
    hq.paged_append(k, v, slots, *pool)
    c, s = U.quantise(k.clone())
    assert torch.equal(pool[0][1, :, 4], c[0]) and torch.equal(pool[2][1, :, 4], s[0])
    table, lens = _i32([[2, 1]]), _i32([21])
    want = hq.paged_attention(q.clone(memory_format=torch.contiguous_format) + 0, *pool, table, lens)
    assert torch.equal(hq.paged_attention(q, *pool, table, lens), want)
    wide = torch.zeros(6, H * G * D + 2, dtype=BF16, device="cuda")
    out = wide[:, :-2].view(6, H * G, D)[at:at + 1]
    assert out.stride(0) % 4 and hq.paged_attention(q, *pool, table, lens, out=out) is out and torch.equal(out, want)
    assert bool((wide[:at] == 0).all()) and bool((wide[at + 1:] == 0).all())


def test_tables_of_one_column():
    """Whatever the stride of a table's only column says."""
    g = _gen(10)
    pool = U.make_pool(g, 4, 2, 16, 64, "cuda")
    q = torch.randn(3, 4, 64, generator=g, device="cuda").to(BF16)
    lens, flat = _i32([5, 16, 9]), _i32([3, 0, 2])
    want = hq.paged_attention(q, *pool, flat[:, None].contiguous(), lens)
    column = flat[None].t()
    assert column.stride() == (1, 3) and torch.equal(hq.paged_attention(q, *pool, column, lens), want)
    assert hq.paged_batch(lens - 1, torch.ones_like(lens), column, flat, 16, 3).slots.tolist() == [52, 15, 40]
