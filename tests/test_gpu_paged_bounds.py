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


LONG = dict(weight=2.0 ** -11, floor=2.0 ** -21)         # requests of more than 16 rows


def _v_scales(kind, shape, g):
    """Factors of the V rows' magnitudes [pages, heads, page]."""
    u = torch.rand(shape, generator=g, device="cuda")
    if kind == "some":                                   # 2^-6 to 2^6
        return torch.exp2(12 * u - 6)
    if kind == "all":                                    # what fp16 scales hold
        return torch.exp2(30 * u - 16)
    if kind == "spikes":                                 # few tokens are far larger
        return torch.where(u < 0.02, 2.0 ** 14, 2.0 ** -10)
    if kind == "holes":                                  # few tokens are far smaller
        return torch.where(u < 0.02, 2.0 ** -16, 2.0 ** 12)
    if kind == "zeros":                                  # some tokens count for nothing, whatever their weight
        return torch.ones_like(u)
    ramp = torch.arange(shape[0] * shape[2], device="cuda").reshape(shape[0], 1, shape[2]) / (shape[0] * shape[2])
    return torch.exp2(28 * (ramp if kind == "rising" else 1 - ramp) - 15).expand(shape)


@pytest.mark.parametrize("kind", ["some", "all", "spikes", "holes", "rising", "falling", "zeros"])
@pytest.mark.parametrize("dtype,D,H,G,seq,new,window", [
    (BF16, 128, 2, 4, [1000, 40], [300, 20], 0), (FP16, 64, 2, 8, [700, 33], [40, 33], 0), (BF16, 64, 1, 4, [6000], [60], 0),
    (BF16, 128, 2, 4, [900], [100], 90), (BF16, 128, 2, 4, [3000, 50], [1, 1], 0), (BF16, 64, 2, 4, [3000, 50], [4, 3], 200)])
def test_v_rows_of_different_magnitudes(kind, dtype, D, H, G, seq, new, window):
    """V scales that differ between tokens, up to all that fp16 holds; queries that
    pick single keys out, whatever their scale, among them."""
    g, page = _gen(5), 16
    pages = sum(-(-n // page) for n in seq)
    table = torch.full((len(seq), max(-(-n // page) for n in seq)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for r, n in enumerate(seq):                          # pages in order: the ramps run along the sequences
        table[r, :-(-n // page)] = torch.arange(at, at - (-n // page), dtype=torch.int32, device="cuda")
        at += -(-n // page)
    k, v = (torch.randn(pages, H, page, D, generator=g, device="cuda") for _ in range(2))
    kc, ks = U.quantise(k)
    vc, vs = U.quantise(v * _v_scales(kind, (pages, H, page), g)[..., None])
    assert bool(torch.isfinite(vs.float()).all())
    if kind == "zeros":
        vs[torch.rand(vs.shape, generator=g, device="cuda") < 0.3] = 0.0
    pool = (kc, vc, ks, vs)
    q = torch.randn(sum(new), H, G, D, generator=g, device="cuda")
    first = 0
    for r, (n, m) in enumerate(zip(seq, new)):           # every second token looks for one key that it sees
        for i in range(0, m, 2):
            pos = n - m + i
            lo = max(0, pos - window + 1) if window else 0
            j = lo + int(torch.randint(0, pos - lo + 1, (1,), generator=g, device="cuda"))
            q[first + i] = 4 * k[table[r, j // page].long(), :, j % page][:, None]
        first += m
    q = q.reshape(-1, H * G, D).to(dtype)
    out = hq.paged_attention(q, *pool, table, _i32(seq), _i32([0] + torch.tensor(new).cumsum(0).tolist()), window=window)
    first = 0
    for r, (n, m) in enumerate(zip(seq, new)):
        short = m * G <= 16
        ref, E = B.rows(q[first:first + m], pool, table[r], n, window, **({} if short else LONG))
        got = out[first:first + m]
        B.check(got, ref, E, f"{kind}, request {r}")
        # row by row: rows of small values do not hide behind rows of large ones
        lim = 1.2 * (ref.to(dtype).double() - ref).norm(dim=-1) + E.norm(dim=-1) + 2.0 ** -60
        worst = ((got.double() - ref).norm(dim=-1) / lim).max()
        print(f"{kind}, request {r}: rows at most {float(worst):.3g} of their limit")
        assert worst <= 1, (kind, r, float(worst))
        first += m


def _check_rows(out, pool, table, seq, new, q, window, G, what):
    """Every request's outputs together and row by row (rows of small values do not
    hide behind rows of large ones)."""
    first = 0
    for r, (n, m) in enumerate(zip(seq, new)):
        x = q[first:first + m]
        ref, E = B.rows(x, pool, table[r], n, window, **({} if m * G <= 16 else LONG))
        got = out[first:first + m]
        B.check(got, ref, E, f"{what}, request {r}")
        lim = 1.2 * (ref.to(out.dtype).double() - ref).norm(dim=-1) + E.norm(dim=-1) + 2.0 ** -60
        worst = ((got.double() - ref).norm(dim=-1) / lim).max()
        assert worst <= 1, (what, r, float(worst))
        first += m


@pytest.mark.parametrize("dtype,D,H,G,page,seq,new,window", [
    (FP16, 128, 8, 4, 16, [32768, 3], [1, 1], 0), (BF16, 128, 8, 4, 64, [8192], [1], 0), (BF16, 128, 2, 8, 128, [20001, 7, 12345], [1] * 3, 0),
    (FP16, 64, 8, 4, 256, [30011], [1], 0), (BF16, 128, 8, 4, 64, [9000] * 48, [1] * 48, 0), (FP16, 128, 8, 4, 32, [20001], [1], 5000),
    (BF16, 64, 2, 4, 16, [700] * 300, [1] * 300, 0), (BF16, 128, 8, 8, 256, [20000], [40], 0), (FP16, 128, 2, 8, 16, [9000, 4000], [30, 77], 0),
    (BF16, 64, 4, 4, 64, [12000, 300], [64, 200], 3000), (FP16, 64, 2, 32, 32, [5000] * 3, [1] * 3, 0)])
def test_each_row_finds_its_key(dtype, D, H, G, page, seq, new, window):
    """Every second row looks for one key, at the edges of tiles, pages and steps and
    at random places of long contexts: reading another key's codes, scales or page in
    its place would be the whole of such a row's output."""
    g = _gen(7)
    table, pages = U.make_table(g, seq, page, "cuda")
    k, v = (torch.randn(pages, H, page, D, generator=g, device="cuda") for _ in range(2))
    (kc, ks), (vc, vs) = U.quantise(k), U.quantise(v)
    pool = (kc, vc, ks, vs)
    q = torch.randn(sum(new), H, G, D, generator=g, device="cuda")
    rnd = torch.randint(0, 1 << 30, (sum(new), H, G), generator=g, device="cuda").tolist()
    first = 0
    for r, (n, m) in enumerate(zip(seq, new)):
        at, who = [], []
        for i in range(m):
            pos = n - m + i
            lo = max(0, pos - window + 1) if window else 0
            edges = sorted({min(max(e, lo), pos) for b in (0, 16, 32, 64, page, 128, 256, 384, 1024, 4096, n // 2 // 32 * 32, n // page * page, lo, pos)
                            for e in (b - 1, b, b + 1)})
            for h in range(H):
                for a in range(G):
                    x = rnd[first + i][h][a]
                    if (i + h + a) % 2 == 0:
                        at.append(edges[x % len(edges)] if x & 1 << 20 else lo + x % (pos - lo + 1))
                        who.append((first + i, h, a))
        at, who = torch.tensor(at, device="cuda"), torch.tensor(who, device="cuda")
        q[who[:, 0], who[:, 1], who[:, 2]] = (6 if D == 64 else 4) * k[table[r, at // page].long(), who[:, 1], at % page]
        first += m
    q = q.reshape(-1, H * G, D).to(dtype)
    out = hq.paged_attention(q, *pool, table, _i32(seq), None if max(new) == 1 else _i32([0] + torch.tensor(new).cumsum(0).tolist()), window=window)
    some = range(len(seq)) if len(seq) < 10 else (0, len(seq) // 2, len(seq) - 1)
    if max(new) == 1:
        for r in some:
            _check_rows(out[r:r + 1], pool, table[r:r + 1], seq[r:r + 1], [1], q[r:r + 1], window, G, f"row {r}")
    else:
        _check_rows(out, pool, table, seq, new, q, window, G, "rows")


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D,H,G,page,seq,new,window", [
    (128, 8, 4, 64, [2500], [700], 0), (128, 2, 8, 16, [1300, 4000], [1300, 77], 0), (64, 8, 4, 16, [6000, 700], [600, 700], 1024),
    (128, 8, 8, 256, [20000], [40], 0), (64, 2, 32, 32, [3000] * 4, [1] * 4, 0), (128, 2, 4, 32, [17, 9000], [17, 5], 0)])
def test_longer_requests_round_weights_to_11_bits(dtype, D, H, G, page, seq, new, window):
    """Requests of more than 16 rows: half a step of fp16 for a weight, no more."""
    g = _gen(8)
    table, pages = U.make_table(g, seq, page, "cuda")
    pool = U.make_pool(g, pages, H, page, D, "cuda")
    for amp in (1.0, 3.0):
        q = (amp * torch.randn(sum(new), H * G, D, generator=g, device="cuda")).to(dtype)
        out = hq.paged_attention(q, *pool, table, _i32(seq), _i32([0] + torch.tensor(new).cumsum(0).tolist()), window=window)
        _check_rows(out, pool, table, seq, new, q, window, G, f"queries of {amp}")


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D,H,G,page,seq,new,spread", [(128, 2, 8, 16, [900, 77], [1, 1], 60), (64, 2, 3, 32, [300], [5], 60), (64, 1, 1, 16, [7], [9], 60),
                                                       (128, 2, 4, 16, [700, 90], [70, 20], 60), (64, 1, 16, 64, [9000], [40], 60),
                                                       (64, 2, 4, 32, [400, 60], [90, 70], 11), (128, 2, 4, 32, [400], [90], 5), (128, 1, 32, 16, [1000], [1], 40)])
def test_query_rows_of_very_different_magnitude(dtype, D, H, G, page, seq, new, spread):
    """Rows of one request, tokens or heads, that are 2^120 times others (2^28 in
    fp16): each row's output is its own."""
    spread = spread if dtype == BF16 else min(spread, 14)
    g = _gen(9)
    table, pages = U.make_table(g, seq, page, "cuda")
    pool = U.make_pool(g, pages, H, page, D, "cuda")
    q = torch.randn(sum(new), H * G, D, generator=g, device="cuda").clamp(-3.9, 3.9)
    e = torch.randint(-spread, spread + 1, q.shape[:2], generator=g, device="cuda")
    e = torch.where(torch.rand(e.shape, generator=g, device="cuda") < 0.6, 0, e)
    q = (q * torch.exp2(e.float())[..., None]).to(dtype)
    assert bool(torch.isfinite(q.float()).all())
    cu = None if max(new) == 1 else _i32([0] + torch.tensor(new).cumsum(0).tolist())
    out = hq.paged_attention(q, *pool, table, _i32(seq), cu)
    _check_rows(out, pool, table, seq, new, q, 0, G, "rows")
