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


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D,H,G,seq", [(128, 8, 4, [8192]), (64, 2, 16, [4096] * 40), (128, 8, 1, [300, 2000, 20000]), (64, 4, 8, [17, 1000])])
@pytest.mark.parametrize("window", [0, 700])
def test_short_requests_round_their_outputs_alone(dtype, D, H, G, seq, window):
    """Requests of at most 16 rows: a weight keeps 16 bits, so that the output's own
    rounding is all that counts, of either type."""
    g, page = _gen(2), 16
    table, pages = U.make_table(g, seq, page, "cuda")
    pool = U.make_pool(g, pages, H, page, D, "cuda")
    for amp in (1.0, 3.0):
        q = (amp * torch.randn(len(seq), H * G, D, generator=g, device="cuda")).to(dtype)
        out = hq.paged_attention(q, *pool, table, _i32(seq), window=window)
        some = sorted({0, len(seq) // 2, len(seq) - 1})
        refs = [B.rows(q[r:r + 1], pool, table[r], seq[r], window) for r in some]
        B.check(out[some], torch.cat([x for x, _ in refs]), torch.cat([x for _, x in refs]), f"requests {some}, queries of {amp}")
