"""How many rows a rotation takes: as many as a launch has threads for, queries and
keys alike."""

import pytest
import torch

import hyquant_amd as hq
from tests import rope_util as U
from tests.test_gpu_rope import BF, DEV, check, gen, randn

pytestmark = pytest.mark.gpu


def test_many_key_heads():
    """160 million rows of keys, 1.3e9 threads: a launch holds 4.3e9."""
    HQ, HK, D = 1, 64, 64
    T = 2500000
    x = torch.empty(T, HQ + HK, D, dtype=BF, device=DEV)
    some = torch.tensor([0, T // 2, T - 1], device=DEV)
    x[some] = randn(gen(1), len(some), HQ + HK, D)
    cos, sin = U.tables(50, D, device=DEV)
    pos = torch.arange(T, device=DEV) % 50
    q, k = hq.qk_norm_rope(x[:, :HQ], x[:, HQ:], cos, sin, pos)
    at = pos[some]
    check(q[some], *U.turn(x[some, :HQ], cos[at], sin[at]))
    check(k[some], *U.turn(x[some, HQ:], cos[at], sin[at]))
    del x, q, k
    torch.cuda.empty_cache()
