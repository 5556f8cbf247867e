"""8-bit blocks that a rejected draft was appended to: what it does to the accepted
tokens of the block, and the two ways back."""

import math

import pytest
import torch

import hyquant_amd as hq
from tests import rope_util as U
from tests.test_gpu_rope import BF, DEV, as_long, gen, randn

pytestmark = pytest.mark.gpu


def append(pool, x, first, rope):
    slots = as_long(list(range(first, first + len(x))))
    if rope:                             # (a rotation by nothing)
        D = x.shape[-1]
        cos, sin = torch.ones(1, D // 2, device=DEV), torch.zeros(1, D // 2, device=DEV)
        hq.paged_rope_append(x, x, x, cos, sin, torch.zeros_like(slots), slots, *pool)
    else:
        hq.paged8_append(x, x, slots, *pool)


def equal_rows(a, b, upto):
    """The scales, and the codes before token `upto` of the one page that is used."""
    return all(torch.equal(s[1, :, :upto], t[1, :, :upto]) for s, t in zip(a[:2], b[:2])) and all(
        torch.equal(s[1], t[1]) for s, t in zip(a[2:], b[2:]))


@pytest.mark.parametrize("rope", [False, True])
@pytest.mark.parametrize("kept", [1, 7, 8, 9, 15])
def test_a_large_draft_coarsens_the_accepted_tokens_of_its_block(kept, rope):
    g = gen(kept)
    H, D, page = 2, 64, 16
    pool = U.pool8(g, 2, H, page, D, DEV)
    x, draft, after = randn(g, kept, H, D), randn(g, 16 - kept, H, D, scale=40.0), randn(g, 16 - kept, H, D)
    append(pool, x, page, rope)
    once = [t.clone() for t in pool]
    want = [t.cpu().clone() for t in pool]
    append(pool, draft, page + kept, rope)
    append(pool, after, page + kept, rope)
    for rows in (draft, after):
        U.append8(want[0], want[2], rows.double().cpu(), list(range(page + kept, 2 * page)))
    assert torch.equal(pool[0].cpu(), want[0]) and torch.equal(pool[2].cpu(), want[2])
    assert bool((pool[2][1] > once[2][1]).all())        # the scale stays the draft's
    rows = lambda p: U.values8(p[0], p[2])[1, :, :kept].transpose(0, 1)  # noqa: E731
    step = pool[2][1].double()[None]
    assert bool(((rows(pool) - x.double()).abs() <= step).all())

    # the two ways back: the block as it was before the draft, or its tokens again from its first slot
    clean = [t.clone() for t in once]
    append(clean, after, page + kept, rope)
    back = [t.clone() for t in pool]
    for t, was in zip(back, once):
        t[1].copy_(was[1])
    append(back, after, page + kept, rope)
    assert equal_rows(back, clean, page)
    both = torch.cat([x, after])
    append(pool, both, page, rope)
    fresh = U.pool8(gen(1), 2, H, page, D, DEV)
    append(fresh, both, page, rope)
    assert equal_rows(pool, fresh, page)


@pytest.mark.parametrize("rope", [False, True])
@pytest.mark.parametrize("value", [math.inf, math.nan, -1e30])
@pytest.mark.parametrize("kept", [1, 9, 15])
def test_a_draft_that_is_not_finite_leaves_the_accepted_codes(kept, value, rope):
    """The block's scale is NaN, and stays it while tokens from before stay; their codes are
    untouched, so that the old scale is the way back."""
    g = gen(kept)
    H, D, page = 2, 128, 32
    pool = U.pool8(g, 2, H, page, D, DEV)
    x, draft, after = randn(g, kept, H, D), randn(g, 1, H, D), randn(g, 16 - kept, H, D)
    draft[0, :, 70] = value
    append(pool, x, page, rope)
    once = [t.clone() for t in pool]
    append(pool, draft, page + kept, rope)
    assert pool[2][1, :, 0].isnan().all() and pool[3][1, :, 0].isnan().all()
    assert torch.equal(pool[0][1, :, :kept], once[0][1, :, :kept]) and torch.equal(pool[1][1, :, :kept], once[1][1, :, :kept])
    append(pool, after, page + kept, rope)
    assert pool[2][1, :, 0].isnan().all() and pool[3][1, :, 0].isnan().all()
    assert torch.equal(pool[0][1, :, :kept], once[0][1, :, :kept]) and torch.equal(pool[1][1, :, :kept], once[1][1, :, :kept])
    pool[2].copy_(once[2])
    pool[3].copy_(once[3])
    append(pool, after, page + kept, rope)
    append(once, after, page + kept, rope)
    assert equal_rows(pool, once, 16)
    k, _ = hq.paged8_gather(as_long(list(range(page, page + kept))), *pool, dtype=BF)
    assert bool(((k.double() - x.double()).abs() <= pool[2][1, :, :1].double()[None]).all())
