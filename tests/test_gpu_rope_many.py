"""Rotations and rotated appends of as many rows as a lane group's four heads are
taken from, with head counts that four does not divide: against 64 bits, and the same
bits as the same tokens in calls that take one head at a time."""

import pytest
import torch

import hyquant_amd as hq
from tests import rope_util as U
from tests.test_gpu_rope import BF, DEV, FL, HF, as_long, check, gen, layout, randn

pytestmark = pytest.mark.gpu

CASES = [(BF, 128, 6, 3, 128, False, True, FL), (HF, 64, 5, 1, 32, True, False, HF), (BF, 64, 6, 3, 64, False, True, BF),
         (HF, 128, 5, 1, 96, True, True, FL), (BF, 128, 7, 2, 64, False, False, FL), (BF, 64, 1, 2, 16, True, True, FL)]


def tokens(dim, heads):
    """A token count just above that from which four heads are taken: 8192 wavefronts of 512 / dim rows."""
    return 8192 * 64 // (dim // 8) // heads + 13


def weights(g, norm, dim, dtype):
    return [(1 + 0.3 * torch.randn(dim, generator=g)).to(dtype).to(DEV) if norm else None for _ in range(2)]


@pytest.mark.parametrize("dtype,dim,HQ,HK,rotary,interleaved,norm,table", CASES)
def test_rotation(dtype, dim, HQ, HK, rotary, interleaved, norm, table):
    g = gen(dim + HQ)
    T = tokens(dim, HQ + HK)
    x = randn(g, T, HQ + HK + 1, dim, dtype=dtype, scale=2.0)
    q, k = x[:, :HQ], x[:, HQ:HQ + HK]
    qw, kw = weights(g, norm, dim, dtype)
    cos, sin = U.tables(500, rotary, table, device=DEV)
    pos = torch.randint(0, 500, (T,), generator=g).to(DEV)
    out = torch.rand(T, generator=g).to(DEV) < 0.02
    out[-1] = out[0] = True
    pos[out] = torch.where(torch.arange(T, device=DEV) % 2 == 0, -1, 500)[out]
    kws = dict(q_weight=qw, k_weight=kw, interleaved=interleaved)
    qo, ko = hq.qk_norm_rope(q, k, cos, sin, pos, **kws)
    at = pos[~out]
    for a, b, w in ((q, qo, qw), (k, ko, kw)):
        check(b[~out], *U.turn(a[~out], cos[at], sin[at], w, 1e-6, interleaved))
        assert not b[out].any()
    cut = list(range(0, T, 977)) + [T]
    for a, b in zip(cut, cut[1:]):
        qs, ks = hq.qk_norm_rope(q[a:b], k[a:b], cos, sin, pos[a:b], **kws)
        assert torch.equal(qs, qo[a:b]) and torch.equal(ks, ko[a:b])


@pytest.mark.parametrize("dtype,dim,HQ,HK,rotary,interleaved,norm,table", CASES)
@pytest.mark.parametrize("tables", [1, 3])
def test_rotation_of_a_batch(dtype, dim, HQ, HK, rotary, interleaved, norm, table, tables):
    g = gen(dim + HQ + tables)
    B = 3
    N = tokens(dim, HQ + HK) // B + 1
    x = randn(g, B, HQ + HK, N, dim, dtype=dtype).transpose(1, 2)
    q, k = x[:, :, :HQ], x[:, :, HQ:]
    qw, kw = weights(g, norm, dim, dtype)
    angle = torch.randn(tables, N + 2, rotary // 2, generator=g, dtype=torch.float64)
    cos, sin = angle.cos().to(table).to(DEV), angle.sin().to(table).to(DEV)
    kws = dict(q_weight=qw, k_weight=kw, interleaved=interleaved)
    qo, ko = hq.qk_norm_rope(q, k, cos, sin, **kws)
    c, s = (t[:, :N].expand(B, N, rotary // 2) for t in (cos, sin))
    for a, b, w in ((q, qo, qw), (k, ko, kw)):
        check(b, *U.turn(a, c, s, w, 1e-6, interleaved))
    for b in range(B):
        t = b if tables > 1 else 0
        qs, ks = hq.qk_norm_rope(q[b], k[b], cos[t], sin[t], **kws)
        assert torch.equal(qs, qo[b]) and torch.equal(ks, ko[b])


@pytest.mark.parametrize("dtype,dim,HQ,HK,rotary,interleaved,norm,table", CASES)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("chunks", [False, True])
def test_rope_append(bits, chunks, dtype, dim, HQ, HK, rotary, interleaved, norm, table):
    """A decode step's scattered tokens, or chunks of requests with contexts, padded behind."""
    g = gen(dim + HQ + bits + chunks)
    T, page = tokens(dim, HQ + 2 * HK), 32
    if chunks:
        news = []
        while sum(news) < T - 5:
            news.append(min(1 + int(torch.randint(0, 400, (1,), generator=g)), T - 5 - sum(news)))
        contexts = torch.randint(0, 90, (len(news),), generator=g).tolist()
    else:
        news, contexts = [1] * (T - 5), torch.randint(0, 30, (T - 5,), generator=g).tolist()
    pages, slots, positions = layout(g, contexts, news, page, pad=5)
    x = randn(g, T, HQ + 2 * HK, dim, dtype=dtype, scale=1.5)
    q, k, v = x[:, :HQ], x[:, HQ:HQ + HK], x[:, HQ + HK:]
    qw, kw = weights(g, norm, dim, dtype)
    cos, sin = U.tables(max(positions) + 1, rotary, table, device=DEV)
    for t in range(7, T, 311):
        positions[t] = len(cos)              # outside the table: nothing is written
    if bits == 8:
        pool = U.pool8(g, pages, HK, page, dim, DEV)
    else:
        pool = tuple(torch.randint(-128, 127, (pages, HK, page, dim // 2), generator=g, dtype=torch.int8).to(DEV) for _ in range(2)) + tuple(
            torch.rand(pages, HK, page, generator=g).half().to(DEV) for _ in range(2))
    want = [t.cpu().clone() for t in pool]
    pos, at = as_long(positions), as_long(slots)
    kws = dict(q_weight=qw, k_weight=kw, interleaved=interleaved)
    qo = hq.paged_rope_append(q, k, v, cos, sin, pos, at, *pool, **kws)
    ok = torch.tensor([0 <= p < len(cos) for p in positions])
    on = ok.to(DEV)
    row = torch.where(on, pos, 0)
    ref, big = U.turn(q, cos[row], sin[row], qw, 1e-6, interleaved)
    check(qo[on], ref[on], big[on])
    assert not qo[~on].any()
    cut = list(range(0, T, 499)) + [T]
    for a, b in zip(cut, cut[1:]):
        assert torch.equal(hq.qk_norm_rope(q[a:b], k[a:b], cos, sin, pos[a:b], **kws)[0], qo[a:b])
    rows = U.turn(k, cos[row], sin[row], kw, 1e-6, interleaved)[0].cpu(), v.double().cpu()
    for i, r in enumerate(rows):
        codes, scales = want[i], want[2 + i]
        got = pool[i].cpu()
        if bits == 8:
            U.append8(codes, scales, r, slots, ok.tolist())
            for t, s in enumerate(slots):
                if s >= 0 and not ok[t]:     # (its row holds anything)
                    codes[s // page, :, s % page] = got[s // page, :, s % page]
        else:
            c, sc = U.codes4(r)
            live = torch.tensor([t for t, s in enumerate(slots) if s >= 0 and ok[t]])
            where = torch.tensor(slots)[live]
            codes[where // page, :, where % page], scales[where // page, :, where % page] = c[live], sc[live]
        assert torch.equal(got, codes) and torch.equal(pool[2 + i].cpu(), scales)
