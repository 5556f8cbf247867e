"""Rotation, rotated appends and the 8-bit pages' append on the GPU against 64-bit
references: rotated rows within their own rounding and 32 bits' error, codes and
scales exactly."""

import math

import pytest
import torch

import hyquant_amd as hq
from tests import rope_util as U

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF, HF, FL = torch.bfloat16, torch.float16, torch.float32


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(g, *shape, dtype=BF, scale=1.0):
    return (scale * torch.randn(*shape, generator=g)).to(dtype).to(DEV)


def check(out, ref, big, what=""):
    ref, big = ref.to(DEV), big.to(DEV)
    tol = U.tolerance(ref, big, out.dtype)
    err = (out.double() - ref).abs()
    assert out.shape == ref.shape
    assert bool((err <= tol).all()), (what, float((err / tol).max()))


@pytest.mark.parametrize("dtype,dim,rotary,interleaved,norm,table", [
    (BF, 128, 128, False, True, FL), (BF, 128, 128, False, False, BF), (HF, 128, 64, False, True, FL), (HF, 64, 64, True, True, FL),
    (BF, 64, 32, True, False, HF), (BF, 64, 16, False, True, FL), (HF, 128, 96, True, False, FL), (BF, 128, 112, False, True, BF)])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1), (1, 7, 5, 3), (3, 13, 8, 2), (2, 33, 32, 8)])
def test_rotation(dtype, dim, rotary, interleaved, norm, table, shape):
    B, N, HQ, HK = shape
    g = gen(B * 100 + N + dim)
    q, k = randn(g, B, N, HQ, dim, dtype=dtype), randn(g, B, N, HK, dim, dtype=dtype, scale=3.0)
    qw, kw = (randn(g, dim, dtype=w) if norm else None for w in (dtype, FL))
    cos, sin = U.tables(N + 3, rotary, table, device=DEV)
    qo, ko = hq.qk_norm_rope(q, k, cos, sin, q_weight=qw, k_weight=kw, interleaved=interleaved)
    for x, y, w in ((q, qo, qw), (k, ko, kw)):
        assert y.is_contiguous() and y.dtype == dtype
        check(y, *U.turn(x, cos[:N], sin[:N], w, 1e-6, interleaved))
    # the same tokens by positions, in another order
    at = torch.randperm(B * N, generator=g).to(DEV)
    pos = torch.arange(N, device=DEV).repeat(B)[at]
    qp, kp = hq.qk_norm_rope(q.flatten(0, 1)[at], k.flatten(0, 1)[at], cos, sin, pos, q_weight=qw, k_weight=kw, interleaved=interleaved)
    assert torch.equal(qp, qo.flatten(0, 1)[at]) and torch.equal(kp, ko.flatten(0, 1)[at])


def test_rotation_of_rows_past_32_bits():
    """More than 2^31 values in and out."""
    T, HQ, HK, D = 240000, 64, 8, 128
    x = torch.empty(T, HQ + HK, D, dtype=BF, device=DEV)
    some = torch.tensor([0, 1, T // 2, T - 17, T - 1], device=DEV)
    x[some] = randn(gen(8), len(some), HQ + HK, D)
    cos, sin = U.tables(T, D, device=DEV)
    q, k = hq.qk_norm_rope(x[:, :HQ], x[:, HQ:], cos, sin)
    check(q[some], *U.turn(x[some, :HQ], cos[some], sin[some]))
    check(k[some], *U.turn(x[some, HQ:], cos[some], sin[some]))


def test_rotation_takes_strides_and_tables_of_each_sequence():
    g = gen(1)
    B, N, HQ, HK, D = 2, 11, 6, 2, 128
    x = randn(g, B, N, HQ + 2 * HK, D)
    table = torch.randn(B, N, D, generator=g).to(DEV)                     # as a model's embedding gives it: both halves
    cos, sin = table.cos(), table.sin()
    want = [U.turn(t, cos[..., :D // 2], sin[..., :D // 2])[0] for t in (x[:, :, :HQ], x[:, :, HQ:HQ + HK])]
    odd = torch.zeros(B, N, HQ + 2 * HK, D + 4, dtype=BF, device=DEV)       # rows that are not 16-byte aligned
    odd[..., 2:D + 2] = x
    turned = x.transpose(1, 2).contiguous().transpose(1, 2)                 # [B, heads, N, D] memory
    apart = x.transpose(2, 3).contiguous().transpose(2, 3)                  # channels apart
    outs = []
    for y in (x, odd[..., 2:D + 2], turned, apart):
        outs.append(hq.qk_norm_rope(y[:, :, :HQ], y[:, :, HQ:HQ + HK], cos[..., :D // 2], sin[..., :D // 2]))
        for o, w, t in zip(outs[-1], want, (x[:, :, :HQ], x[:, :, HQ:HQ + HK])):
            check(o, w, U.turn(t, cos[..., :D // 2], sin[..., :D // 2])[1])
    for o in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(o, outs[0]))
    one = hq.qk_norm_rope(x[:1, :, :HQ], x[:1, :, HQ:HQ + HK], cos[:1, :, :D // 2], sin[:1, :, :D // 2])
    assert torch.equal(one[0], outs[0][0][:1])
    # one table for both
    both = hq.qk_norm_rope(x[:, :, :HQ], x[:, :, HQ:HQ + HK], cos[:1, :, :D // 2], sin[:1, :, :D // 2])
    assert torch.equal(both[0][0], outs[0][0][0]) and not torch.equal(both[0][1], outs[0][0][1])


def test_rotation_without_heads_tokens_or_position():
    cos, sin = U.tables(4, 64, device=DEV)
    e = lambda *s: torch.empty(*s, dtype=BF, device=DEV)  # noqa: E731
    q, k = hq.qk_norm_rope(e(0, 4, 64), e(0, 2, 64), cos, sin)
    assert q.shape == (0, 4, 64) and k.shape == (0, 2, 64)
    x = randn(gen(2), 3, 4, 64)
    q, k = hq.qk_norm_rope(x, e(3, 0, 64), cos, sin)
    assert k.shape == (3, 0, 64)
    check(q, *U.turn(x, cos[:3], sin[:3]))
    q, k = hq.qk_norm_rope(x, x, cos, sin, torch.tensor([1, -1, 4], device=DEV))
    check(q[:1], *U.turn(x[:1], cos[1:2], sin[1:2]))
    assert not q[1:].any() and not k[1:].any()


def test_rotation_of_values_that_are_not_finite_stays_in_their_rows():
    cos, sin = U.tables(8, 128, device=DEV)
    x = randn(gen(3), 8, 4, 128)
    w = torch.ones(128, device=DEV)
    clean = hq.qk_norm_rope(x, x, cos, sin, q_weight=w, k_weight=w)
    y = x.clone()
    y[3, 1, 5], y[5, 2, 70] = math.inf, math.nan
    q, k = hq.qk_norm_rope(y, y, cos, sin, q_weight=w, k_weight=w)
    hit = torch.zeros(8, 4, dtype=torch.bool, device=DEV)
    hit[3, 1] = hit[5, 2] = True
    assert torch.equal(q[~hit], clean[0][~hit]) and torch.equal(k[~hit], clean[1][~hit])
    assert q[hit].isnan().any(-1).all()
    zero = torch.zeros(1, 1, 128, dtype=BF, device=DEV)
    q, _ = hq.qk_norm_rope(zero, zero, cos, sin, q_weight=w, k_weight=w)
    assert not q.any()


@pytest.mark.parametrize("eps", [1e-6, 0.0])
def test_norms_of_rows_of_any_magnitude(eps):
    """bf16 rows from 1e-30 to 1e37: their squares are no 32-bit numbers."""
    g = gen(7)
    scale = torch.logspace(-30, 37, 24).reshape(24, 1, 1)
    x = (torch.randn(24, 3, 64, generator=g) * scale).clamp(-3e38, 3e38).to(BF).to(DEV)
    w = randn(g, 64, dtype=FL)
    cos, sin = U.tables(24, 64, device=DEV)
    q, k = hq.qk_norm_rope(x, x, cos, sin, q_weight=w, k_weight=w, eps=eps)
    check(q, *U.turn(x, cos, sin, w, eps))
    assert torch.equal(q, k)
    pool = U.pool8(g, 2, 3, 16, 64, DEV)
    want = pool[0].cpu().clone(), pool[2].cpu().clone()
    hq.paged_rope_append(x, x, x.clamp(-1, 1), cos, sin, as_long(list(range(24))), as_long(list(range(24))), *pool, q_weight=w, k_weight=w, eps=eps)
    U.append8(*want, U.turn(x, cos, sin, w, eps)[0].cpu(), list(range(24)))
    assert torch.equal(pool[0].cpu(), want[0]) and torch.equal(pool[2].cpu(), want[1])


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("norm", [False, True])
def test_appended_keys_that_are_not_finite_or_hardly(bits, norm):
    """Rows with an infinity or NaN have scales that are not finite, in their own
    block alone; rows next to fp32's largest number, and products past it, have
    their codes."""
    g = gen(17)
    T, H, D, page = 64, 2, 64, 16
    x = randn(g, T, H, D)
    x[3, 0, 7], x[20, 1, 40] = math.inf, math.nan
    if norm:
        x[36] = (x[36].float() * 1e38).clamp(-3e38, 3e38).to(BF)          # the inverse root is no normal fp32 number
    w = (1 + 0.1 * torch.randn(D, generator=g)).to(DEV) if norm else None
    cos, sin = U.tables(T, D, device=DEV)
    if norm:
        cos[50], sin[50] = 3e38, -3e38   # sums of products past fp32, small in the cache no more than there
    pool = U.pool8(g, T // 16, H, page, D, DEV) if bits == 8 else (
        tuple(torch.zeros(T // 16, H, page, D // 2, dtype=torch.int8, device=DEV) for _ in range(2)) +
        tuple(torch.zeros(T // 16, H, page, dtype=HF, device=DEV) for _ in range(2)))
    want = [t.cpu().clone() for t in pool]
    at, v = as_long(list(range(T))), randn(g, T, H, D)
    hq.paged_rope_append(x, x, v, cos, sin, at, at, *pool, q_weight=w, k_weight=w)
    y = U.turn(x, cos, sin, w)[0].cpu()
    if bits == 8:
        U.append8(want[0], want[2], y, list(range(T)))
        bad = want[2].isnan()
        good = ~bad.repeat_interleave(16, -1)
        assert torch.equal(pool[2].cpu().isnan(), bad) and int(bad.sum()) == (4 if norm else 2)
    else:
        for t in range(T):
            c, sc = U.codes4(y[t])
            want[0][t // page, :, t % page], want[2][t // page, :, t % page] = c, sc
        bad = ~want[2].isfinite()
        good = ~bad
        assert torch.equal(~pool[2].cpu().isfinite(), bad) and int(bad.sum()) == (4 if norm else 2)
    assert torch.equal(pool[0].cpu()[good], want[0][good])
    assert torch.equal(pool[2].cpu()[~bad], want[2][~bad])


def test_rotation_by_far_rows_of_a_table():
    """A table past 2^31 values."""
    rows = (1 << 28) + 5
    cos = torch.zeros(rows, 8, device=DEV)
    sin = torch.zeros(rows, 8, device=DEV)
    cos[-1] = 0.6
    sin[-1] = 0.8
    x = randn(gen(4), 2, 1, 64)
    q, _ = hq.qk_norm_rope(x, x, cos, sin, torch.tensor([rows - 1, 0], device=DEV))
    check(q[:1], *U.turn(x[:1], cos[-1:], sin[-1:]))
    check(q[1:], *U.turn(x[1:], cos[:1], sin[:1]))


# ---- appends ----

def layout(g, contexts, news, page, pad=0):
    """(pages, slots, positions) of requests in scattered pages."""
    need = [-(-(a + b) // page) for a, b in zip(contexts, news)]
    order = torch.randperm(sum(need) + 2, generator=g).tolist()
    slots, positions, at = [], [], 0
    for a, b, n in zip(contexts, news, need):
        slots += [order[at + p // page] * page + p % page for p in range(a, a + b)]
        positions += range(a, a + b)
        at += n
    return sum(need) + 2, slots + [-1] * pad, positions + [-1] * pad


def as_long(v):
    return torch.tensor(v, dtype=torch.int64, device=DEV)


REQUESTS = [([0], [1]), ([5], [1]), ([15, 16, 31, 0], [1, 1, 1, 1]), ([3], [40]), ([0, 7, 30], [16, 9, 35]), ([9, 2, 0, 14, 1], [5, 31, 33, 2, 15])]


@pytest.mark.parametrize("dtype,dim,page", [(BF, 128, 16), (HF, 64, 32), (BF, 64, 256), (HF, 128, 64)])
@pytest.mark.parametrize("contexts,news", REQUESTS)
def test_append8(dtype, dim, page, contexts, news):
    g = gen(len(news) * 10 + dim + page)
    H = 3
    pages, slots, _ = layout(g, contexts, news, page, pad=3)
    pool = U.pool8(g, pages, H, page, dim, DEV)
    want = [t.cpu().clone() for t in pool]
    T = len(slots)
    x = randn(g, T, 4, H, dim, dtype=dtype, scale=2.0)
    x[:, 1] *= 2.0 ** torch.randint(-6, 6, (T, H, 1), generator=g).to(DEV)
    k, v = x[:, 1], x[:, 3]
    hq.paged8_append(k, v, as_long(slots), *pool)
    U.append8(want[0], want[2], k.double().cpu(), slots)
    U.append8(want[1], want[3], v.double().cpu(), slots)
    for a, b in zip(pool, want):
        assert torch.equal(a.cpu(), b)
    for out_type in (BF, HF):
        ko, vo = hq.paged8_gather(as_long(slots + [pages * page]), *pool, dtype=out_type)
        assert not ko[-4:].any() and not vo[-4:].any()
        for o, codes, scales in ((ko, *want[0::2]), (vo, *want[1::2])):
            all_rows = U.values8(codes, scales)
            ref = torch.stack([all_rows[s // page, :, s % page] for s in slots[:-3]])
            assert torch.equal(o[:-4].cpu(), ref.float().to(out_type))


@pytest.mark.parametrize("step", [1, 3, 16])
def test_append8_token_by_token_keeps_values_within_a_step(step):
    """A block filled by tokens of rising magnitude: every value is within one
    step of the block's last scale of what was appended (half a step for each
    rounding, each step at most half the next where a scale grew)."""
    g = gen(step)
    H, D, page = 2, 64, 32
    pool = U.pool8(g, 3, H, page, D, DEV)
    want = [t.cpu().clone() for t in pool]
    x = randn(g, 32, H, D) * (1.3 ** torch.arange(32, device=DEV)).to(BF)[:, None, None]
    for t in range(0, 32, step):
        n = min(step, 32 - t)
        slots = list(range(page + t, page + t + n))
        hq.paged8_append(x[t:t + n], x[t:t + n], as_long(slots), *pool)
        U.append8(want[0], want[2], x[t:t + n].double().cpu(), slots)
    assert torch.equal(pool[0].cpu(), want[0]) and torch.equal(pool[2].cpu(), want[2])
    held, scale = U.values8(pool[0], pool[2])[1].transpose(0, 1), pool[2][1].double().repeat_interleave(16, -1).t()
    assert bool(((held - x.double()).abs() <= scale[..., None]).all())


def test_append8_holes_strange_scales_and_values():
    g = gen(9)
    H, D, page = 1, 64, 16
    pool = U.pool8(g, 8, H, page, D, DEV)
    pool[2][0, 0, 0], pool[2][1, 0, 0], pool[2][2, 0, 0], pool[2][3, 0, 0] = 0.0, 0.3, math.nan, -1.0
    want = [t.cpu().clone() for t in pool]
    x = randn(g, 8, H, D)
    x[4, 0, 3], x[5, 0, 60] = math.inf, math.nan
    x[6] = 0
    x[7, 0, 0] = 1e30
    slots = [3, 16 + 4, 32 + 1, 48 + 15, 64, 80, 96, 112]
    hq.paged8_append(x, x, as_long(slots), *pool)
    U.append8(want[0], want[2], x.double().cpu(), slots)
    assert torch.equal(pool[2].cpu().isnan(), want[2].isnan())
    assert pool[2].cpu().isnan().flatten().tolist() == [False, False, True, True, True, True, False, True]
    good = ~want[2].isnan().flatten()
    assert torch.equal(pool[0].cpu()[good], want[0][good]) and torch.equal(pool[2].cpu()[good], want[2][good])
    k, _ = hq.paged8_gather(as_long([64 + 2, 96]), *pool)
    assert k[0].isnan().all() and not k[1].any()


@pytest.mark.parametrize("rope", [False, True])
def test_append8_slots_out_of_order_touch_their_own_blocks_alone(rope):
    """Slots of a block that are not neighbours, or descend, leave anything in that
    block; the others are as ever."""
    g = gen(10)
    H, D, page, pages = 2, 128, 32, 6
    pool = U.pool8(g, pages, H, page, D, DEV)
    want = [t.cpu().clone() for t in pool]
    wild = [5, 40, 6, 41, 3, 42, 4] + list(range(79, 63, -1)) + [7, 8, 9] * 7            # blocks 0, 2 and 4
    fine = list(range(96, 130)) + list(range(145, 160))
    slots = wild + fine
    x = randn(g, len(slots), H, D)
    if rope:
        cos, sin = torch.ones(1, D // 2, device=DEV), torch.zeros(1, D // 2, device=DEV)
        hq.paged_rope_append(x, x, x, cos, sin, as_long([0] * len(slots)), as_long(slots), *pool)
    else:
        hq.paged8_append(x, x, as_long(slots), *pool)
    U.append8(want[0], want[2], x[len(wild):].double().cpu(), fine)
    blocks = lambda t: t.cpu().reshape(pages, H, page // 16, -1)  # noqa: E731
    for a, b in ((pool[0], want[0]), (pool[2], want[2])):
        a, b = blocks(a).transpose(1, 2).reshape(pages * 2, H, -1), blocks(b).transpose(1, 2).reshape(pages * 2, H, -1)
        for i in range(pages * 2):
            if i not in (0, 2, 4):
                assert torch.equal(a[i], b[i]), i


def test_append8_pool_inside_a_larger_allocation_past_32_bits():
    H, D, page = 2, 128, 64
    pages = (1 << 31) // (2 * H * page * D) + 70
    big = torch.empty(pages, 2 * H, page, D, dtype=torch.int8, device=DEV)           # K and V heads side by side
    big[-1] = 0
    scales = torch.zeros(pages, 2 * H, page // 16, device=DEV)
    pool = big[:, :H], big[:, H:], scales[:, :H], scales[:, H:]
    g = gen(5)
    x = randn(g, 20, 2, H, D)
    slots = [(pages - 1) * page + 30 + i for i in range(20)]
    want = torch.zeros(1, H, page, D, dtype=torch.int8), torch.zeros(1, H, page // 16)
    hq.paged8_append(x[:, 0], x[:, 1], as_long(slots), *pool)
    for at, (c, s) in ((0, pool[0::2]), (1, pool[1::2])):
        codes, sc = (t.clone() for t in want)
        U.append8(codes, sc, x[:, at].double().cpu(), [30 + i for i in range(20)])
        assert torch.equal(c[-1].cpu(), codes[0]) and torch.equal(s[-1].cpu(), sc[0])
    k, v = hq.paged8_gather(as_long(slots), *pool)
    assert torch.equal(k.double().cpu(), U.values8(pool[0][-1].cpu(), pool[2][-1].cpu())[:, 30:50].transpose(0, 1))


@pytest.mark.parametrize("dtype,dim,rotary,interleaved,norm,page", [
    (BF, 128, 128, False, True, 16), (HF, 64, 32, True, False, 64), (BF, 64, 64, False, True, 32), (HF, 128, 96, False, True, 16)])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("contexts,news", REQUESTS[1:])
def test_rope_append(bits, dtype, dim, rotary, interleaved, norm, page, contexts, news):
    g = gen(bits + len(news) + dim + page)
    HQ, H = 6, 2
    pages, slots, positions = layout(g, contexts, news, page, pad=2)
    T = len(slots)
    x = randn(g, T, HQ + 2 * H, dim, dtype=dtype, scale=1.5)
    q, k, v = x[:, :HQ], x[:, HQ:HQ + H], x[:, HQ + H:]
    qw, kw = (randn(g, dim, dtype=dtype) if norm else None for _ in range(2))
    cos, sin = U.tables(max(positions) + 1, rotary, device=DEV)
    if T > 6:
        positions[T // 2] = len(cos)         # outside the table: nothing is written
    if bits == 8:
        pool = U.pool8(g, pages, H, page, dim, DEV)
    else:
        pool = tuple(torch.randint(-128, 127, (pages, H, page, dim // 2), generator=g, dtype=torch.int8).to(DEV) for _ in range(2)) + tuple(
            torch.rand(pages, H, page, generator=g).half().to(DEV) for _ in range(2))
    want = [t.cpu().clone() for t in pool]
    qo = hq.paged_rope_append(q, k, v, cos, sin, as_long(positions), as_long(slots), *pool, q_weight=qw, k_weight=kw, interleaved=interleaved)
    ok = torch.tensor([0 <= p < len(cos) for p in positions])
    at = as_long([p if o else 0 for p, o in zip(positions, ok)])
    ref, big = U.turn(q, cos[at], sin[at], qw, 1e-6, interleaved)
    check(qo[ok.to(DEV)], ref[ok.to(DEV)], big[ok.to(DEV)])
    assert not qo[~ok.to(DEV)].any()
    again, _ = hq.qk_norm_rope(q, k, cos, sin, as_long(positions), q_weight=qw, k_weight=kw, interleaved=interleaved)
    assert torch.equal(again, qo)
    rows = U.turn(k, cos[at], sin[at], kw, 1e-6, interleaved)[0].cpu(), v.double().cpu()
    live = [s if o else -1 for s, o in zip(slots, ok)]
    for i, r in enumerate(rows):
        codes, scales = want[i], want[2 + i]
        if bits == 8:
            U.append8(codes, scales, r, slots, ok.tolist())
            hole = slots[T // 2]                 # (its row holds anything)
            if not ok[T // 2]:
                codes[hole // page, :, hole % page] = pool[i][hole // page, :, hole % page].cpu()
        else:
            c, s = U.codes4(r)
            for t, slot in enumerate(live):
                if slot >= 0:
                    codes[slot // page, :, slot % page], scales[slot // page, :, slot % page] = c[t], s[t]
        assert torch.equal(pool[i].cpu(), codes) and torch.equal(pool[2 + i].cpu(), scales)


@pytest.mark.parametrize("bits", [4, 8])
def test_rope_append_at_position_zero_is_the_plain_append(bits):
    """A rotation by nothing leaves the rows: the codes are paged_append's and paged8_append's."""
    g = gen(bits)
    T, H, D, page = 37, 2, 128, 16
    cos, sin = U.tables(1, D, device=DEV)
    pages, slots, _ = layout(g, [0], [T], page)
    x = randn(g, T, 2 * H, D)
    k, v = x[:, :H], x[:, H:]
    new = lambda: (tuple(torch.zeros(pages, H, page, D // 2, dtype=torch.int8, device=DEV) for _ in range(2)) + tuple(  # noqa: E731
        torch.zeros(pages, H, page, dtype=HF, device=DEV) for _ in range(2)) if bits == 4 else
        tuple(torch.zeros(pages, H, page, D, dtype=torch.int8, device=DEV) for _ in range(2)) + tuple(
        torch.zeros(pages, H, page // 16, device=DEV) for _ in range(2)))
    a, b = new(), new()
    q = hq.paged_rope_append(x, k, v, cos, sin, as_long([0] * T), as_long(slots), *a)
    (hq.paged_append if bits == 4 else hq.paged8_append)(k, v, as_long(slots), *b)
    assert torch.equal(q, x) and all(torch.equal(s, t) for s, t in zip(a, b))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("interleaved", [False, True])
def test_keys_next_to_the_borders_of_their_codes(bits, interleaved):
    """Keys rotated by 2^-32: values on the border between two codes move by less
    than 32 bits hold, and fall on their own side of it; the largest values of a row
    that lie on the border between two scales, too."""
    D, H, page, T = 64, 2, 16, 48
    g = gen(13)
    cos, sin = torch.ones(1, D // 2, device=DEV), torch.full((1, D // 2), 2.0 ** -32, device=DEV)
    most = 7 if bits == 4 else 127
    x = torch.randint(-most, most, (T, H, D), generator=g).float() + 0.5                 # borders of a scale of one
    x[..., 5] = most
    x[T // 2:, :, 40] = -most
    x = x.to(BF).to(DEV)                 # (at most 8 bits: exact)
    pool = U.pool8(g, T // 16, H, page, D, DEV) if bits == 8 else (
        tuple(torch.zeros(T // 16, H, page, D // 2, dtype=torch.int8, device=DEV) for _ in range(2)) +
        tuple(torch.zeros(T // 16, H, page, dtype=HF, device=DEV) for _ in range(2)))
    want = [t.cpu().clone() for t in pool]
    at, slots = as_long([0] * T), list(range(T))
    hq.paged_rope_append(x, x, x, cos, sin, at, as_long(slots), *pool, interleaved=interleaved)
    y = U.turn(x, cos[at], sin[at], None, 1e-6, interleaved)[0].cpu()
    if bits == 8:
        U.append8(want[0], want[2], y, slots)
    else:
        c, sc = U.codes4(y)
        for t in slots:
            want[0][t // page, :, t % page], want[2][t // page, :, t % page] = c[t], sc[t]
    assert torch.equal(pool[0].cpu(), want[0]) and torch.equal(pool[2].cpu(), want[2])


def test_rope_append_of_nothing_and_into_nothing():
    cos, sin = U.tables(4, 64, device=DEV)
    pool = U.pool8(gen(0), 2, 2, 16, 64, DEV)
    before = [t.clone() for t in pool]
    e = lambda h: torch.empty(0, h, 64, dtype=BF, device=DEV)  # noqa: E731
    none = torch.empty(0, dtype=torch.int64, device=DEV)
    assert hq.paged_rope_append(e(4), e(2), e(2), cos, sin, none, none, *pool).shape == (0, 4, 64)
    hq.paged8_append(e(2), e(2), none, *pool)
    empty = tuple(t[:0] for t in pool)
    x = randn(gen(1), 3, 2, 64)
    q = hq.paged_rope_append(x, x, x, cos, sin, as_long([0, 1, 2]), as_long([0, 1, 2]), *empty)
    check(q, *U.turn(x, cos[:3], sin[:3]))
    hq.paged8_append(x, x, as_long([0, 1, 2]), *empty)
    k, _ = hq.paged8_gather(as_long([0, 1]), *empty)
    assert not k.any()
    assert all(torch.equal(a, b) for a, b in zip(pool, before))


def test_captured_rope_append_follows_what_it_is_replayed_with():
    """A captured step replayed with other positions, slots and rows, on another
    stream than the eager calls between the replays."""
    g = gen(6)
    T, HQ, H, D, page, pages = 5, 8, 2, 128, 16, 40
    cos, sin = U.tables(pages * page, D, device=DEV)
    x = randn(g, T, HQ + 2 * H, D)
    pos, slots = as_long([0] * T), as_long([-1] * T)
    pool = U.pool8(g, pages, H, page, D, DEV)
    eager = tuple(t.clone() for t in pool)
    call = lambda p: hq.paged_rope_append(x[:, :HQ], x[:, HQ:HQ + H], x[:, HQ + H:], cos, sin, pos, slots, *p)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(pool)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = call(pool)
    for step in range(4):
        at = [(3 * r + r * page + step) for r in range(T)]
        pos.copy_(as_long(at))
        slots.copy_(as_long([(7 * r % pages) * page + a % page for r, a in enumerate(at)]))
        x.copy_(randn(g, *x.shape))
        graph.replay()
        want = call(eager)
        torch.cuda.synchronize()
        assert torch.equal(q, want) and all(torch.equal(a, b) for a, b in zip(pool, eager))


def test_gradients_are_refused():
    cos, sin = U.tables(4, 64, device=DEV)
    x = randn(gen(0), 2, 2, 64)
    pool = U.pool8(gen(0), 1, 2, 16, 64, DEV)
    with pytest.raises(ValueError, match="gradients"):
        hq.qk_norm_rope(x.clone().requires_grad_(), x, cos, sin)
    with pytest.raises(ValueError, match="gradients"):
        hq.paged_rope_append(x, x.clone().requires_grad_(), x, cos, sin, as_long([0, 1]), as_long([0, 1]), *pool)
    with torch.no_grad():
        hq.qk_norm_rope(x.clone().requires_grad_(), x, cos, sin)


@pytest.mark.parametrize("bits", [4, 8])
def test_native_and_checked_calls_agree(bits, monkeypatch):
    """The C++ form of the calls and the Python form launch the same kernels."""
    from hyquant_amd import decode_d_stage as dd
    from tests import paged8_util, paged_util
    g = gen(50)
    T, HQ, H, D, page, pages = 41, 8, 2, 64, 32, 6
    x = randn(g, T, HQ + 2 * H, D, dtype=HF)
    q, k, v = x[:, :HQ], x[:, HQ:HQ + H], x[:, HQ + H:]
    w = randn(g, D, dtype=HF)
    cos, sin = U.tables(T, 32, device=DEV)
    dev_gen = torch.Generator(device="cuda").manual_seed(1)
    pool = (paged_util if bits == 4 else paged8_util).make_pool(dev_gen, pages, H, page, D, "cuda")
    slots, pos = as_long(list(range(30, 30 + T))), as_long(list(range(T)))
    table, lens = torch.arange(4, dtype=torch.int32, device=DEV)[None], torch.tensor([71], dtype=torch.int32, device=DEV)
    cu = torch.tensor([0, T], dtype=torch.int32, device=DEV)

    def calls():
        p = tuple(t.clone() for t in pool)
        out = hq.qk_norm_rope(q, k, cos, sin, q_weight=w, interleaved=True) + hq.qk_norm_rope(q[None], k[None], cos[None], sin[None], k_weight=w.float())
        out += (hq.paged_rope_append(q, k, v, cos, sin, pos, slots, *p, q_weight=w, k_weight=w, eps=1e-5),)
        out += tuple(t.clone() for t in p)
        (hq.paged_append if bits == 4 else hq.paged8_append)(v, k, slots, *p)
        out += p + (hq.paged_gather if bits == 4 else hq.paged8_gather)(slots, *p, dtype=HF)
        attend = hq.paged_attention if bits == 4 else hq.paged8_attention
        return out + attend(q, *p, table, lens, cu, sm_scale=0.2, window=90, return_lse=True) + (attend(q[:1], *p, table, lens),)

    native = calls()
    assert dd._FX
    monkeypatch.setattr(dd, "_FX", False)
    for i, (a, b) in enumerate(zip(native, calls())):
        assert a.dtype == b.dtype and torch.equal(a, b), i
