"""64-bit references of the rotation and of the 8-bit pages, in plain torch."""

import math

import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
BLOCK = 16


def tables(rows, rotary, dtype=torch.float32, base=10000.0, device="cpu"):
    """cos and sin [rows, rotary / 2] of positions 0 .. rows - 1."""
    f = base ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)
    a = torch.arange(rows, dtype=torch.float64)[:, None] * f
    return a.cos().to(dtype).to(device), a.sin().to(dtype).to(device)


def turn(x, cos, sin, w=None, eps=1e-6, interleaved=False):
    """(rows, bound) in 64 bits: x [..., heads, D] rotated by cos, sin [..., R / 2], and the sum of
    the magnitudes that each value is made of."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()
    c, s = cos.double().unsqueeze(-2), sin.double().unsqueeze(-2)
    r = 2 * cos.shape[-1]
    y, big = x.clone(), x.abs()
    at = [slice(0, r, 2), slice(1, r, 2)] if interleaved else [slice(0, r // 2), slice(r // 2, r)]
    a, b = x[..., at[0]], x[..., at[1]]
    y[..., at[0]], y[..., at[1]] = a * c - b * s, b * c + a * s
    big[..., at[0]], big[..., at[1]] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    return y, big


def tolerance(ref, big, dtype):
    """Half a step of the output's type, and the 32-bit arithmetic before it: a
    norm's sum of squares (at most 128 terms in a tree of 8 + 4 additions, 12
    roundings, half of which reach its root), the root, the reciprocal, two
    products, the rotation's two products and sum, each half a step of 2^-24 of
    the magnitudes: below 16 in all."""
    half = HALF_STEP[dtype]
    return half * ref.abs() + torch.finfo(dtype).smallest_normal * half * 2 + 16 * 2.0 ** -24 * (1 + half) * big


def codes4(x):
    """Codes (packed) and scales of rows in 64 bits."""
    scale = (x.abs().amax(-1).clamp(min=1e-5) / 7).float().half()
    code = torch.round(x / scale.double()[..., None]).clamp(-8, 7).to(torch.int8) & 15
    return code[..., 0::2] | (code[..., 1::2] << 4), scale


def exponent(amax):
    """The smallest e with max(amax, 1e-5) <= 127 2^e."""
    e = math.ceil(math.log2(max(amax, 1e-5) / 127))
    while 127 * 2.0 ** e < max(amax, 1e-5):
        e += 1
    while 127 * 2.0 ** (e - 1) >= max(amax, 1e-5):
        e -= 1
    return e


def append8(codes, scales, x, slots, live=None):
    """The rows x [T, H, D] (float64) into a pool of codes [N, H, P, D] and scales
    [N, H, P / 16] on the CPU, in place, block by block; `live`: which tokens
    write (the others of a block leave no gap between its rows)."""
    N, H, P, D = codes.shape
    runs, last = [], None
    for t, s in enumerate(slots):
        block = s // BLOCK if 0 <= s < N * P else None
        if block is not None and block == last:
            runs[-1].append(t)
        elif block is not None:
            runs.append([t])
        last = block
    runs = [[t for t in run if live is None or live[t]] for run in runs]
    for run in filter(None, runs):
        page, off = slots[run[0]] // P, slots[run[0]] % P
        b, kept = off // BLOCK, off % BLOCK
        for h in range(H):
            new = torch.stack([x[t, h] for t in run])
            rows = codes[page, h, b * BLOCK:(b + 1) * BLOCK]
            old = float(scales[page, h, b]) if kept else 0.0
            if not bool(torch.isfinite(new).all()) or not (new.abs().max() <= 127 * 2.0 ** 40) or not (0 <= old <= 2.0 ** 41):
                scales[page, h, b] = math.nan
                continue
            s = 2.0 ** exponent(float(new.abs().max()))
            while s < old:
                s *= 2
            if kept:
                rows[:kept] = torch.round(rows[:kept].double() * (old / s)).to(torch.int8)
            for t in run:
                rows[slots[t] % BLOCK] = torch.round(x[t, h] / s).to(torch.int8)
            scales[page, h, b] = s


def values8(codes, scales):
    """float64 values of a pool's rows."""
    return codes.double() * scales.double().repeat_interleave(BLOCK, -1)[..., None]


def pool8(g, pages, heads, page, dim, device="cpu"):
    """Random codes and power-of-two scales: k codes, v codes, k scales, v scales."""
    code = [torch.randint(-127, 128, (pages, heads, page, dim), generator=g, dtype=torch.int8) for _ in range(2)]
    scale = [2.0 ** torch.randint(-9, -3, (pages, heads, page // BLOCK), generator=g).float() for _ in range(2)]
    return tuple(t.to(device) for t in code + scale)
