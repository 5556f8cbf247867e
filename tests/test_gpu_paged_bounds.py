"""The paged attention's precision over whole rows, against bounds that do not
grow past the outputs themselves (paged_bounds)."""

import pytest
import torch

import hyquant_amd as hq
from tests import paged_bounds as B
from tests import paged_util as U

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("D,R,n", [(128, 64, 32768), (64, 100, 32768), (128, 48, 9000)])
def test_fp16_rows_that_are_not_cut(D, R, n):
    """So many requests that one workgroup takes a request's whole context: the
    codes' offset in its sums costs an fp16 output nothing."""
    g, H, G, page = _gen(1), 8, 4, 64
    row, pages = U.make_table(g, [n], page, "cuda")
    pool = U.make_pool(g, pages, H, page, D, "cuda")
    q = torch.randn(R, H * G, D, generator=g, device="cuda").to(FP16)
    out = hq.paged_attention(q, *pool, row.expand(R, -1), _i32([n] * R))
    for r in (0, R - 1):
        ref, E = B.rows(q[r:r + 1], pool, row[0], n)
        B.check(out[r:r + 1], ref, E, f"request {r}")
