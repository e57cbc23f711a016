"""How far an attention row may be off: its error against float64, row by row and
relative to what the roundings of the kernels predict for that row.

For out = sum_j p_j v_j, p = softmax(x), small errors dx_j of the logits and dw_j
(relative) of the weights move a channel by

    do = sum_j p_j (dx_j + dw_j) (v_j - out),

since the weights are divided by their own sum, plus the output's rounding.
Roundings are independent of the values, so over a row's channels

    mean do^2 = mean_c [ sum_j p_j^2 (s_j^2 + w_j^2) (v_jc - out_c)^2 + o_c^2 ]

with s, w, o the root mean squares of the errors of logits, weights and output. A
rounding to t is off by at most u = eps(t) / 2 relative to the value, by u / sqrt(3)
in the root mean square at most (uniform over a step, the value at the step's lower
end). That gives

  16 bits   s_j^2 = sum_c q_c^2 (k_c^2 + (2^-13 scale_c)^2) 2^-22 / 3 for cached tokens (keys
            rounded to float16; the dequantisation in float32, of terms up to 160 scale, is
            off by 2^-17 scale at most, 2^-24 scale in units of the factor outside), 0 for
            drafts; w = u / sqrt(3); o_c = u / sqrt(3) |out_c|
  float32   s_j = 2^-24 / sqrt(3) sqrt(d / 8 + 6) (|x_j| + 2 sqrt(sum_c q_c^2 k_c^2)): as many
            additions one after another, of partial sums of that size; w_j = 2^-22 + 2^-23 (max x
            - x_j): the bound of ex2 and the rounding of its argument; o_c = 2^-24 / sqrt(3)
            sqrt(n / 64 + 16) (|out_c| + sqrt(sum_j p_j^2 v_jc^2)): a warp's additions

A row passes where the root mean square of its error is below 6 of these (a row whose
weight lies on two tokens has one error for all channels, so single errors, normally
distributed, count: 6 of them are exceeded once in 5e8 rows), plus 2^-22 of its largest
value for what float32 sums add in 16 bits.
"""

import math

import torch

FACTOR = 6.0


def expected(q, k, v, scale, cached, seen, dtype):
    """(out, rms) of rows q [T, H, G, D] over tokens k / v [n, H, D] in float64, rms [T, H, G]
    the predicted root mean square of a row's error. ``scale`` [n, H, D]: the keys' quantisation
    step (0 for drafts), ``cached`` [n] bool, ``seen`` [T, n] bool."""
    n, d = k.shape[0], k.shape[2]
    kt, vt = k.permute(1, 2, 0), v.permute(1, 0, 2)                   # [H, D, n], [H, n, D]
    x = torch.einsum("thgd,hdn->thgn", q, kt)
    x = x.masked_fill(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
    out = torch.einsum("thgn,hnd->thgd", p, vt)
    qk2 = torch.einsum("thgd,hdn->thgn", q * q, kt * kt)
    if dtype == torch.float32:
        size = torch.where(torch.isinf(x), torch.zeros_like(x), x.abs()) + 2 * qk2.sqrt()
        s2 = (2.0 ** -24) ** 2 / 3 * (d / 8 + 6) * size ** 2
        w2 = (2.0 ** -22 + 2.0 ** -23 * torch.where(p > 0, top - x, torch.zeros_like(x))) ** 2
        walk = torch.einsum("thgn,hnd->thgd", p * p, vt * vt).sqrt()
        o2 = ((2.0 ** -24) ** 2 / 3 * (n / 64 + 16) * (out.abs() + walk) ** 2).mean(-1)
    else:
        u = torch.finfo(dtype).eps / 2
        st = scale.permute(1, 2, 0)
        qs2 = torch.einsum("thgd,hdn->thgn", q * q, (2.0 ** -13 * st) ** 2)
        s2 = (qk2 + qs2) * 2.0 ** -22 / 3 * cached
        w2 = u * u / 3
        o2 = (u * u / 3 * out ** 2).mean(-1)
    e = p * p * (s2 + w2)
    a, b, c = torch.einsum("thgn,hnd->thgd", e, vt * vt), torch.einsum("thgn,hnd->thgd", e, vt), e.sum(-1)
    spread = (a - 2 * out * b + out ** 2 * c[..., None]).clamp(min=0).mean(-1)
    return out, (spread + o2).sqrt()


def excess(got, out, rms):
    """Largest error of a row over what it may be (passes up to 1)."""
    err = (got.double() - out).square().mean(-1).sqrt()
    room = FACTOR * rms + 2.0 ** -22 * out.abs().amax(-1)
    assert torch.isfinite(got).all()
    return float((err / room.clamp(min=1e-30)).max()) if err.numel() else 0.0
