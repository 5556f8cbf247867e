"""Rows, pages and scales behind the 2^32nd element of their tensors, in and out."""

import pytest
import torch

import hyquant_amd as hq
from tests import rope_util as U
from tests.test_gpu_rope import BF, DEV, HF, as_long, check, gen, randn

pytestmark = pytest.mark.gpu
WIDE = 1 << 32


@pytest.fixture(autouse=True)
def give_back():
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("batch", [1, 2])
def test_rotation(batch):
    """More than 2^32 values of q in and out."""
    HQ, HK, D = 64, 8, 128
    T = WIDE // (HQ * D) + 300
    x = torch.empty(T, HQ + HK, D, dtype=BF, device=DEV)
    some = torch.tensor([0, 1, T // 2, WIDE // (HQ * D) - 1, WIDE // (HQ * D), T - 17, T - 1], device=DEV)
    x[some] = randn(gen(8), len(some), HQ + HK, D)
    cos, sin = U.tables(50, D, device=DEV)
    pos = torch.arange(T, device=DEV) % 50
    shape = (T,) if batch == 1 else (batch, T // batch)
    y = x.view(*shape, HQ + HK, D)
    q, k = hq.qk_norm_rope(y[..., :HQ, :], y[..., HQ:, :], cos, sin, pos)
    assert q.numel() > WIDE and x.numel() > WIDE
    at = pos[some]
    check(q.view(T, HQ, D)[some], *U.turn(x[some, :HQ], cos[at], sin[at]))
    check(k.view(T, HK, D)[some], *U.turn(x[some, HQ:], cos[at], sin[at]))


@pytest.mark.parametrize("bits", [4, 8])
def test_append_and_read_back(bits):
    """Rows whose stride carries the last ones past 2^32 values, into pages whose codes and
    scales lie past 2^32."""
    H, D, page, T = 2, 64, 16, 20
    per = D // 2 if bits == 4 else D
    pages = WIDE // (2 * H * page * per) + 3
    codes = torch.empty(pages, 2 * H, page, per, dtype=torch.int8, device=DEV)            # K and V heads side by side
    wide = torch.empty(pages, -(-WIDE // pages) + 8, dtype=HF if bits == 4 else torch.float32, device=DEV)
    n = page if bits == 4 else 1
    scales = wide[:, :2 * H * n].view(pages, 2 * H, n)
    for i in (pages - 2, pages - 1):
        codes[i] = 0
        scales[i] = 0
    pool = codes[:, :H], codes[:, H:], scales[:, :H], scales[:, H:]
    assert pool[0].stride(0) * (pages - 2) > WIDE - 2 * codes[0].numel() and pool[2].stride(0) * (pages - 1) > WIDE
    rows = torch.empty(T, 1 << 28, dtype=BF, device=DEV)[:, :3 * H * D].view(T, 3 * H, D)
    assert rows.stride(0) * (T - 1) > WIDE
    rows.copy_(randn(gen(bits), T, 3 * H, D))
    q, k, v = rows[:, :H], rows[:, H:2 * H], rows[:, 2 * H:]
    cos, sin = U.tables(T, D, device=DEV)
    slots = [(pages - 2) * page + 7 + i for i in range(T)]
    at = as_long(list(range(T)))
    qo = hq.paged_rope_append(q, k, v, cos, sin, at, as_long(slots), *pool)
    check(qo, *U.turn(q, cos, sin))
    turned = U.turn(k, cos, sin)[0].cpu(), v.double().cpu()

    def expect(r, i):
        c, s = torch.zeros(2, H, page, per, dtype=torch.int8), torch.zeros(2, H, n, dtype=wide.dtype)
        here = [7 + j for j in range(T)]
        if bits == 8:
            U.append8(c, s, r, here)
        else:
            for t, (code, sc) in zip(here, zip(*U.codes4(r))):
                c[t // page, :, t % page], s[t // page, :, t % page] = code, sc
        assert torch.equal(pool[i][-2:].cpu(), c) and torch.equal(pool[2 + i][-2:].cpu(), s)

    for i, r in enumerate(turned):
        expect(r, i)
    gather, append = (hq.paged_gather, hq.paged_append) if bits == 4 else (hq.paged8_gather, hq.paged8_append)
    small = tuple(t[-2:].clone() for t in pool)
    for a, b in zip(gather(as_long(slots), *pool), gather(as_long([7 + j for j in range(T)]), *small)):
        assert torch.equal(a, b) and bool((a != 0).any())
    if bits == 8:
        for i in (pages - 2, pages - 1):
            codes[i] = 0
            scales[i] = 0
        append(k, v, as_long(slots), *pool)
        for i, r in enumerate((k.double().cpu(), v.double().cpu())):
            expect(r, i)
