"""Appends into 8-bit pages with tokens between those of a block that have no slot,
as rejected tokens of a step or the padding of a batch have none: they write
nothing, and the others of the block are one run, however far apart they are."""

import pytest
import torch

import hyquant_amd as hq
from tests import rope_util as U
from tests.test_gpu_rope import BF, DEV, HF, as_long, gen, randn

pytestmark = pytest.mark.gpu


def step(g, gaps, page, lone):
    """(pages, slots) of appends into blocks of random rows, in scattered pages; before each token
    a gap of one of `gaps` lengths stands with probability `lone`."""
    blocks = torch.randperm(4 * page // 16 * 4, generator=g)[:14].tolist()
    slots = []
    for i, b in enumerate(blocks):
        first = int(torch.randint(0, 16, (1,), generator=g)) if i % 3 else 0
        last = int(torch.randint(first, 16, (1,), generator=g)) if i % 4 else 15
        for r in range(first, last + 1):
            if float(torch.rand(1, generator=g)) < lone:
                slots += [-1] * gaps[int(torch.randint(0, len(gaps), (1,), generator=g))]
            slots.append(16 * b + r)
    return 4 * page // 16 * 4 * 16 // page, slots


GAPS = [((1,), 0.2), ((1, 2, 3), 0.9), ((15, 16, 17), 0.2), ((1, 63, 64, 65), 0.15), ((500, 1030), 0.1), ((1, 20000), 0.03)]


@pytest.mark.parametrize("dtype,dim,page", [(BF, 128, 16), (HF, 64, 64)])
@pytest.mark.parametrize("gaps,lone", GAPS)
@pytest.mark.parametrize("tail", [0, 5, 700])
def test_gaps_do_not_part_a_block(dtype, dim, page, gaps, lone, tail):
    g = gen(len(gaps) + gaps[-1] + dim + tail)
    H, HQ = 2, 3
    pages, slots = step(g, gaps, page, lone)
    slots = [-1] * (tail // 2) + slots + [-1] * tail
    slots = [s if s >= 0 else (-1, pages * page, -(1 << 40))[i % 3] for i, s in enumerate(slots)]       # all of them outside the pool
    T = len(slots)
    x = randn(g, T, HQ + 2 * H, dim, dtype=dtype)
    x[:, HQ:] *= (2.0 ** torch.randint(-4, 5, (T, 2 * H, 1), generator=g)).to(dtype).to(DEV)
    q, k, v = x[:, :HQ], x[:, HQ:HQ + H], x[:, HQ + H:]
    pool = U.pool8(g, pages, H, page, dim, DEV)
    at = [t for t, s in enumerate(slots) if 0 <= s < pages * page]
    some, held = as_long(at), [slots[t] for t in at]

    plain = [t.clone() for t in pool]
    hq.paged8_append(k, v, as_long(slots), *plain)
    for i, rows in enumerate((k, v)):
        codes, scales = pool[i].cpu().clone(), pool[2 + i].cpu().clone()
        U.append8(codes, scales, rows[some].double().cpu(), held)
        assert torch.equal(plain[i].cpu(), codes) and torch.equal(plain[2 + i].cpu(), scales)

    # rotated: positions outside the table among those with a slot, and any for the others
    cos, sin = U.tables(300, dim, device=DEV)
    pos = torch.randint(0, 300, (T,), generator=g)
    out = torch.rand(T, generator=g) < 0.1
    pos[out] = -1
    turned = [t.clone() for t in pool]
    qo = hq.paged_rope_append(q, k, v, cos, sin, pos.to(DEV), as_long(slots), *turned)
    again, _ = hq.qk_norm_rope(q, k, cos, sin, pos.to(DEV))
    assert torch.equal(qo, again)
    live = ~out[at]
    row = pos.clamp(min=0).to(DEV)[some]
    for i, rows in enumerate((U.turn(k[some], cos[row], sin[row])[0].cpu(), v[some].double().cpu())):
        codes, scales = pool[i].cpu().clone(), pool[2 + i].cpu().clone()
        U.append8(codes, scales, rows, held, live.tolist())
        got = turned[i].cpu()
        for s, yes in zip(held, live.tolist()):
            if not yes:                  # (its row holds anything)
                codes[s // page, :, s % page] = got[s // page, :, s % page]
        assert torch.equal(got, codes) and torch.equal(turned[2 + i].cpu(), scales)


@pytest.mark.parametrize("page", [16, 128])
def test_a_block_filled_around_a_gap_is_the_block_filled_at_once(page):
    """The same rows with and without tokens between them, in eager calls and in a captured one
    that is replayed with other slots."""
    g = gen(3)
    H, D, T = 2, 64, 90
    x = randn(g, T, H, D) * (2.0 ** torch.randint(-5, 6, (T, H, 1), generator=g)).to(BF).to(DEV)
    slots = as_long([-1] * T)
    base = U.pool8(g, 128 // page * 2, H, page, D, DEV)
    pool = [t.clone() for t in base]
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        hq.paged8_append(x, x, slots, *pool)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        hq.paged8_append(x, x, slots, *pool)
    for i in range(6):
        keep = torch.rand(T, generator=g) < 0.2 + 0.15 * i
        keep[0] = True
        n = int(keep.sum())
        where = torch.full((T,), -1)
        where[keep] = torch.arange(5 + i, 5 + i + n)
        slots.copy_(where)
        for a, b in zip(pool, base):
            a.copy_(b)
        graph.replay()
        want = [t.clone() for t in base]
        rows = x[keep.to(DEV)]
        hq.paged8_append(rows, rows, as_long(list(range(5 + i, 5 + i + n))), *want)
        eager = [t.clone() for t in base]
        hq.paged8_append(x, x, slots, *eager)
        torch.cuda.synchronize()
        for a, b, c in zip(pool, want, eager):
            assert torch.equal(a, b) and torch.equal(c, b), i
