"""Norms of rows so small that their inverse root is no 32-bit number."""

import pytest
import torch

import hyquant_amd as hq
from tests import rope_util as U
from tests.test_gpu_rope import BF, DEV, FL, as_long, check, gen, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("eps", [0.0, 1e-80, 1e-300])
def test_norms_of_subnormal_rows(dim, eps):
    """bf16 rows from 1e-40 (subnormal numbers, most channels zero) to 1e-30, with an eps that
    is none or no 32-bit number: normalised they are of order one."""
    g = gen(dim)
    T, H = 21, 3
    scale = torch.logspace(-40, -30, T).reshape(T, 1, 1)
    x = (torch.randn(T, H, dim, generator=g).double() * scale).to(BF)
    x[0, 0] = 0
    x[0, 0, 5] = 2.0 ** -133                # the smallest bf16 number alone
    x[1, :, ::2] = 0
    x[:, :, 7] += (x == 0).all(-1).to(BF) * 2.0 ** -133
    x = x.to(DEV)
    assert bool((x != 0).any(-1).all())
    w = randn(g, dim, dtype=FL)
    cos, sin = U.tables(T, dim, device=DEV)
    q, k = hq.qk_norm_rope(x, x, cos, sin, q_weight=w, k_weight=w, eps=eps)
    check(q, *U.turn(x, cos, sin, w, eps))
    assert torch.equal(q, k)
    pool = U.pool8(g, 2, H, 16, dim, DEV)
    want = pool[0].cpu().clone(), pool[2].cpu().clone()
    at = as_long(list(range(T)))
    assert torch.equal(hq.paged_rope_append(x, x, x, cos, sin, at, at, *pool, q_weight=w, k_weight=w, eps=eps), q)
    U.append8(*want, U.turn(x, cos, sin, w, eps)[0].cpu(), list(range(T)))
    assert torch.equal(pool[0].cpu(), want[0]) and torch.equal(pool[2].cpu(), want[1])


def test_norms_of_the_largest_rows():
    """bf16 rows next to the largest number: the inverse root is a subnormal 32-bit number."""
    g = gen(2)
    x = torch.full((4, 2, 128), 3.3e38).to(BF) * torch.sign(torch.randn(4, 2, 128, generator=g)).to(BF)
    x[1] = (x[1].float() * torch.rand(2, 128, generator=g)).to(BF)
    x = x.to(DEV)
    w = randn(g, 128, dtype=FL)
    cos, sin = U.tables(4, 128, device=DEV)
    q, _ = hq.qk_norm_rope(x, x, cos, sin, q_weight=w, k_weight=w)
    check(q, *U.turn(x, cos, sin, w, 1e-6))
