"""Pools and 64-bit references of the paged 8-bit cache's attention tests."""

import math

import torch

BLOCK = 16
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# what a weight times its V scale is held in: the sum of two fp16 numbers, each rounded
# towards zero (requests of at most 16 rows), or one fp16 number
WEIGHT = {True: 2.0 ** -20, False: 2.0 ** -11}
# fp16's subnormal steps: 2^-24 of a number whose row's largest is at least 2^6 (rounded towards
# zero, or to half of it)
FLOOR = 2.0 ** -30


def make_pool(g, pages, heads, page, dim, dev, scale=1.0):
    """Codes and power-of-two scales of Gaussian rows (times `scale`, which may be a tensor
    [pages, heads, page / 16])."""
    out = []
    for _ in range(2):
        x = torch.randn(pages, heads, page // BLOCK, BLOCK * dim, generator=g, device=dev)
        s = torch.exp2(torch.ceil(torch.log2(x.abs().amax(-1) / 127))) if pages else x.new_zeros(0, heads, page // BLOCK)
        code = (x / s[..., None]).round().clamp(-127, 127).to(torch.int8).reshape(pages, heads, page, dim)
        out.append((code, s * scale))
    return out[0][0], out[1][0], out[0][1].contiguous(), out[1][1].contiguous()


def held(pool, table_row, n):
    """(k, v codes [H, n, D] float64, their scales [H, n], which keys' pages are in the pool) of a request."""
    kp, vp, ks, vs = pool
    N, _, P, _ = kp.shape
    j = torch.arange(n, device=kp.device)
    ids = table_row[j // P].long()
    good = (ids >= 0) & (ids < N)
    ids = ids.clamp(0, max(N - 1, 0))
    k, v = (x[ids, :, j % P].transpose(0, 1).double() for x in (kp, vp))
    sk, sv = (x[ids, :, j % P // BLOCK].transpose(0, 1).double() for x in (ks, vs))
    return k, v, sk, sv, good


def reference(q, pool, table, seq_lens, new_lens, window=0, sm_scale=None):
    """(out, lse, tol, lse_tol, E): the definition in 64 bits, request by request; the error
    allowed to each output and lse, and to an output if roundings of different keys are
    independent (a few standard deviations, without the output's own rounding).

    For a row with scores s_j, weights w_j (their sum 1), A = sum w |v|, W = max w v_scale:
      - a weight's rounding, WEIGHT of it, and FLOOR W for each key's code;
      - a score is an fp32 sum of D exact products of magnitude at most 255 |q_d| scale
        (codes enter with an offset of 128) in 16 + D roundings of 2^-24: d; its exponent adds
        log2 of the V scale and the row's reference: 6 roundings of 2^-24 of their magnitudes,
        below 2^-22 (|s| + 64); an error of a score moves numerator and denominator: twice;
      - exp2, log2 and the reciprocal (2^-22), and fp32 sums over n keys: (n / 16 + 64) 2^-23
        of sums that carry 128 + 128 times the weights between two takings-off."""
    T, HQ, D = q.shape
    H = pool[0].shape[1]
    G = HQ // H
    sm = D ** -0.5 if sm_scale is None else sm_scale
    dev = q.device
    out, tol, E = (torch.zeros(T, HQ, D, dtype=torch.float64, device=dev) for _ in range(3))
    lse = torch.full((T, HQ), -math.inf, dtype=torch.float64, device=dev)
    lse_tol = torch.zeros(T, HQ, dtype=torch.float64, device=dev)
    half = HALF_STEP[q.dtype]
    first = 0
    for r, (n, m) in enumerate(zip(seq_lens, new_lens)):
        n = max(n, 0)
        if m == 0:
            continue
        if n and pool[0].shape[0]:
            K, V, SK, SV, good = held(pool, table[r], n)
            weight = WEIGHT[m * G <= 16]
            keys = torch.arange(n, device=dev)
            pos = n - m + torch.arange(m, device=dev)
            seen = (keys[None] <= pos[:, None]) & good[None]
            if window:
                seen &= keys[None] > pos[:, None] - window
            used = seen.any(0)                   # what no row sees may hold anything
            hide = ~seen[:, None].expand(m, G, n).reshape(m * G, n)
            for h in range(H):
                sk, sv = (torch.where(used, x[h], 0.0) for x in (SK, SV))
                code = V[h]
                v = code * sv[:, None]
                x = q[first:first + m, h * G:(h + 1) * G].double().reshape(m * G, D)
                s = (x @ (K[h] * sk[:, None]).t() * sm).masked_fill(hide, -math.inf)
                none = hide.all(-1, keepdim=True)
                w = torch.softmax(s, -1).masked_fill(none, 0.0)
                A, W = w @ v.abs(), (w * sv).amax(-1, keepdim=True)
                xs = x.abs().sum(-1, keepdim=True)
                d = (D + 16) * 2.0 ** -24 * abs(sm) * 255 * xs * sk.max()
                top = torch.where(none, 0.0, s.masked_fill(hide, 0.0).abs().amax(-1, keepdim=True))
                d = d + 2.0 ** -22 * (top * 1.45 + 64)
                acc = (n / 16 + 64) * 2.0 ** -23
                at = slice(first, first + m), slice(h * G, (h + 1) * G)
                out[at] = (w @ v).reshape(m, G, D)
                lse[at] = torch.where(none, -math.inf, torch.logsumexp(s, -1, keepdim=True)).reshape(m, G)
                tol[at] = ((weight + 2 * d + 2.0 ** -21 + acc) * A + acc * 256 * (w @ sv[:, None])
                           + FLOOR * W * ((~hide).double() @ code.abs())).reshape(m, G, D)
                lse_tol[at] = (2 * d + acc + 2.0 ** -21 + 2.0 ** -22 * lse[at].reshape(m * G, 1).nan_to_num(0, 0, 0).abs()).reshape(m, G)
                size = 255 * abs(sm) * xs * sk
                eps = weight ** 2 + (4 * 2.0 ** -24 * size) ** 2 + (2.0 ** -22 * (top * 1.45 + 64)) ** 2
                g = torch.nn.functional.pad(w * sv, (0, -n % 32)).reshape(m * G, -1, 32).sum(-1)
                var = ((eps * w * w) @ (v * v) + (FLOOR * W) ** 2 * ((~hide).double() @ (code * code))
                       + (256 * 6 * 2.0 ** -24) ** 2 * g.square().sum(-1, keepdim=True))
                E[at] = (3 * var.sqrt()).reshape(m, G, D)
        first += m
    tol += half * out.abs() + torch.finfo(q.dtype).smallest_normal * half * 2
    return out, lse, tol, lse_tol, E


def check(out, ref, tol, what=""):
    err = (out.double() - ref).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} values off, the worst by "
                           f"{float((err / tol.clamp(min=1e-300))[bad].max()):.3g} times its tolerance")
