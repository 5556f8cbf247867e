"""Error bounds of the paged attention's tests that hold for whole rows.

paged_util.reference allows each output its worst case, which grows with the
number of keys while a mean over many keys shrinks.  Here rounding errors of
different keys count as independent, as they are: an output's error before its
own rounding is at most a few standard deviations,

    E_i = 3 sqrt(sum_j (eps_j w_j v_ij)^2 + sum_j (floor max W code_ij)^2 + acc^2)

  eps_j   relative error of a weight: half a step of what holds it (`weight`),
          and its score's error: a score is a sum of products exact in fp32 of
          magnitude at most 15 |q_d| scale each, 16 roundings of 2^-24 of their
          sum's magnitude.  Half a step counts as the standard deviation (a
          rounding's own is 1 / sqrt(3) of that).
  acc     fp32 sums.  A 16-row tile's running sum carries at most 143 times the
          weights W of the 96 keys whose offset has not been taken off; each
          product over 32 keys rounds it 4 times.  Over all steps
          143 2^-24 sqrt(4 sum (g_1 + g_2 + g_3)^2) <= 143 2^-24 6 sqrt(sum g^2),
          g the sums of W = w_j v_scale_j over 32 keys.
  floor   (256-row tiles) a weight times its V scale is an fp16 number, the row's
          largest at least 2^5: below 2^-14 the step is 2^-24, so that half of it
          is 2^-30 of the largest; 2^-21 where the row's scale follows 16 keys whose
          V scales lie within a factor of 2^9 and so may be that much too high.

and the output is the correctly rounded value wherever that error does not reach
over the middle between two values: it does in a share E_i / step_i of cases.
"""

import torch

from tests import paged_util as U


def rows(q, pool, table_row, n, window=0, sm_scale=None, weight=2.0 ** -16, floor=0.0):
    """(out, E) of one request's new tokens q [m, HQ, D], the last of its n tokens."""
    kp, vp, ks, vs = pool
    m, HQ, D = q.shape
    N, H, P, _ = kp.shape
    G = HQ // H
    sm = D ** -0.5 if sm_scale is None else sm_scale
    j = torch.arange(n, device=q.device)
    ids = table_row[j // P].long()
    pos = n - m + torch.arange(m, device=q.device)
    hide = j[None] > pos[:, None]
    if window:
        hide = hide | (j[None] <= pos[:, None] - window)
    hide = hide[:, None].expand(m, G, n).reshape(m * G, n)
    out, E = (torch.zeros(m, HQ, D, dtype=torch.float64, device=q.device) for _ in range(2))
    for h in range(H):
        sk, sv = ks[ids, h, j % P], vs[ids, h, j % P]
        k, v = U.values(kp[ids, h, j % P], sk), U.values(vp[ids, h, j % P], sv)
        x = q[:, h * G:(h + 1) * G].double().reshape(m * G, D)
        s = (x @ k.t() * sm).masked_fill(hide, float("-inf"))
        w = torch.softmax(s, -1).masked_fill(hide.all(-1, keepdim=True), 0.0)      # (a row without keys is zero)
        size = 15 * abs(sm) * x.abs().sum(-1, keepdim=True) * sk.double()
        eps = weight ** 2 + (4 * 2.0 ** -24 * size) ** 2
        W = w * sv.double().abs()
        code = U.values(vp[ids, h, j % P], torch.ones_like(sv))
        var = (eps * w * w) @ (v * v) + (floor * W.amax(-1, keepdim=True)) ** 2 * ((~hide).double() @ (code * code))
        g = torch.nn.functional.pad(W, (0, -n % 32)).reshape(m * G, -1, 32).sum(-1)
        acc = 143 * 6 * 2.0 ** -24 * g.square().sum(-1, keepdim=True).sqrt()
        out[:, h * G:(h + 1) * G] = (w @ v).reshape(m, G, D)
        E[:, h * G:(h + 1) * G] = (3 * (var + acc * acc).sqrt()).reshape(m, G, D)
    return out, E


def check(out, ref, E, what=""):
    """The error's norm, and how many outputs are not the correctly rounded value."""
    best = ref.to(out.dtype)
    err, rounding = (out.double() - ref).norm(), (best.double() - ref).norm()
    lim = 1.1 * rounding + E.norm()                      # (a tenth for the spread of the roundings over a few thousand outputs)
    f = torch.finfo(out.dtype)
    step = f.eps * torch.exp2(torch.floor(torch.log2(ref.abs().clamp(min=f.smallest_normal))))
    share = (E / step).clamp(max=1.0).sum()
    wrong = (out != best).sum()
    print(f"{what}: error {float(err / ref.norm()):.3g}, rounding {float(rounding / ref.norm()):.3g}, limit {float(lim / ref.norm()):.3g}; "
          f"{int(wrong)} of {out.numel()} not the nearest, limit {float(share):.0f}")
    assert err <= lim, f"{what}: error {float(err):.3g} of {float(ref.norm()):.3g}, limit {float(lim):.3g}"
    assert wrong <= share + 5 * share.sqrt() + 5, f"{what}: {int(wrong)} of {out.numel()} outputs are not the nearest value, limit {float(share):.0f}"
