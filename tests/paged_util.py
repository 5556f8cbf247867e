"""Pools, block tables and 64-bit references of the paged 4-bit cache's tests."""

import math

import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def quantise(x):
    """quantize_per_token's 4-bit codes (packed) and scales, in plain torch."""
    x = x.float()
    scale = (x.abs().amax(-1).clamp(min=1e-5) / 7).half()
    code = torch.round(x / scale.float()[..., None]).clamp(-8, 7).to(torch.int8) & 15
    return code[..., 0::2] | (code[..., 1::2] << 4), scale


def values(codes, scales):
    """float64 values of packed rows."""
    x = codes.to(torch.int16) & 255
    x = torch.stack((x & 15, x >> 4), -1).flatten(-2)
    return (x - 16 * (x >= 8)).double() * scales.double()[..., None]


def make_pool(g, pages, heads, page, dim, dev, scale=1.0):
    """Random codes and scales: ((k codes, v codes), (k scales, v scales))."""
    out = [quantise(scale * torch.randn(pages, heads, page, dim, generator=g, device=dev)) for _ in range(2)]
    return out[0][0], out[1][0], out[0][1], out[1][1]


def make_table(g, seq_lens, page, dev, spare=2):
    """A table of scattered distinct pages (-1 behind each row's last) and the pool's size."""
    need = [-(-max(n, 0) // page) for n in seq_lens]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    table = torch.full((len(seq_lens), max(need + [0]) + 1), -1, dtype=torch.int32, device=dev)
    at = 0
    for r, n in enumerate(need):
        table[r, :n] = order[at:at + n]
        at += n
    return table, pages


def reference(q, pool, table, seq_lens, new_lens, window=0, sm_scale=None):
    """(out, lse, tol): the definition in 64 bits, request by request, and the
    error allowed to each output.

    The tolerance counts, for a row with weights p_j = exp(s_j) and mean
    magnitude A = sum p |v| / sum p:
      - the output's own rounding, half a step of its type times |out|;
      - the weights' rounding, half a step of bf16 (fp16 models carry them as a
        sum of two bf16 numbers: its square) times A;
      - scores: sums of D exact fp32 products of magnitude at most
        15 |q_d| scale each, and a few roundings more; an error d of a score
        moves a weight by d, numerator and denominator alike: 2 d A;
      - exp2 and the fp32 sums over n keys: (n / 16 + 64) 2^-23 of A, and of
        the codes' offset 136 + 8 times the V scales' weighted mean."""
    kp, vp, ks, vs = pool
    T, HQ, D = q.shape
    N, H, P, _ = kp.shape
    G = HQ // H
    sm = D ** -0.5 if sm_scale is None else sm_scale
    dev = q.device
    out = torch.zeros(T, HQ, D, dtype=torch.float64, device=dev)
    lse = torch.full((T, HQ), -math.inf, dtype=torch.float64, device=dev)
    tol = torch.zeros(T, HQ, D, dtype=torch.float64, device=dev)
    half = HALF_STEP[q.dtype]
    weight = 2.0 ** -8 if q.dtype == torch.bfloat16 else 2.0 ** -16
    first = 0
    for r, (n, m) in enumerate(zip(seq_lens, new_lens)):
        n = max(n, 0)
        if m == 0:
            continue
        keys = torch.arange(n, device=dev)
        ids = table[r][keys // P].long()
        good = (ids >= 0) & (ids < N)
        ids = ids.clamp(0, max(N - 1, 0))
        pos = n - m + torch.arange(m, device=dev)
        seen = (keys[None] <= pos[:, None]) & good[None]
        if window:
            seen &= keys[None] > pos[:, None] - window
        for h in range(H):
            if N == 0 or n == 0:
                continue
            sk, sv = ks[ids, h, keys % P], vs[ids, h, keys % P]
            k, v = values(kp[ids, h, keys % P], sk), values(vp[ids, h, keys % P], sv)
            sv, sk = sv.double(), sk.double()
            used = seen.any(0)                   # what no row sees may hold anything
            k, v = torch.where(used[:, None], k, 0.0), torch.where(used[:, None], v, 0.0)
            sk, sv = torch.where(used, sk, 0.0), torch.where(used, sv, 0.0)
            x = q[first:first + m, h * G:(h + 1) * G].double()
            s = (x.reshape(m * G, D) @ k.t()).reshape(m, G, n) * sm
            s = s.masked_fill(~seen[:, None], -math.inf)
            top = s.amax(-1, keepdim=True)
            live = torch.isfinite(top)
            p = torch.where(live, torch.exp(s - torch.where(live, top, 0.0)), 0.0)
            total = p.sum(-1, keepdim=True)
            w = p / torch.where(total > 0, total, 1.0)
            flat = w.reshape(m * G, n)
            out[first:first + m, h * G:(h + 1) * G] = (flat @ v).reshape(m, G, D)
            lse[first:first + m, h * G:(h + 1) * G] = torch.where(total > 0, top + total.log(), -math.inf).squeeze(-1)
            A = (flat @ v.abs()).reshape(m, G, D)
            vbar = (flat @ sv).reshape(m, G, 1)
            d = (D + 16) * 2.0 ** -24 * abs(sm) * 15 * x.abs().sum(-1, keepdim=True) * sk.max()
            acc = (n / 16 + 64) * 2.0 ** -23
            tol[first:first + m, h * G:(h + 1) * G] = (weight + 2 * d + acc) * A + acc * 144 * vbar
        first += m
    tol += half * out.abs() + torch.finfo(q.dtype).smallest_normal * half * 2
    return out, lse, tol


def check(out, ref, tol, what=""):
    err = (out.double() - ref).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} values off, the worst by "
                           f"{float((err / tol.clamp(min=1e-300))[bad].max()):.3g} times its tolerance")
