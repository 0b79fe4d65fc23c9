"""The serving operators in 64 bits, written from their formulas, for the tests."""
import math

import torch

GROUP = 32


def unit(dtype):
    """Half a step of rounding to `dtype`, relative."""
    return torch.finfo(dtype).eps / 2


def norm_rope(x, *, eps=None, weight=None, positions=None, inv_freq=None):
    """x [B, H, T, D]; positions [B, T]; inv_freq: D / 2 numbers."""
    y = x.double()
    if eps is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps)
        if weight is not None:
            y = y * weight.double()
    if inv_freq is None:
        return y
    angle = positions.double()[:, None, :, None] * torch.tensor(list(inv_freq), dtype=torch.float64, device=x.device)
    a, b = y[..., 0::2], y[..., 1::2]
    return torch.stack([a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()], dim=-1).flatten(-2)


def attention(q, k, v, *, scale, causal):
    """One sequence: q [nq, Hq, D], k, v [nk, Hkv, D] -> o, lse [Hq, nq], and sum_j p_j |v_j| and max_j sum_d |q k| scale, which error bounds need."""
    q, k, v = q.double(), k.double(), v.double()
    nq, hq, nk, rep = q.shape[0], q.shape[1], k.shape[0], q.shape[1] // max(1, k.shape[1])
    k, v = k.repeat_interleave(rep, 1), v.repeat_interleave(rep, 1)
    s = torch.einsum("ihd,jhd->hij", q, k) * scale
    size = torch.einsum("ihd,jhd->hij", q.abs(), k.abs()) * abs(scale)
    if causal:
        seen = torch.arange(nk, device=q.device)[None] <= torch.arange(nq, device=q.device)[:, None] + (nk - nq)
        s = s.masked_fill(~seen, -math.inf)
        size = size.masked_fill(~seen, 0)
    if nk == 0:
        z = torch.zeros(nq, hq, q.shape[2], dtype=torch.float64, device=q.device)
        return z, torch.full((hq, nq), -math.inf, dtype=torch.float64, device=q.device), z, torch.zeros(hq, nq, dtype=torch.float64, device=q.device)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
    l = p.sum(-1, keepdim=True)
    p = p / torch.where(l == 0, torch.ones_like(l), l)
    lse = (torch.where(m == -math.inf, torch.zeros_like(m), m) + torch.log(l))[..., 0]
    return torch.einsum("hij,jhd->ihd", p, v), lse, torch.einsum("hij,jhd->ihd", p, v.abs()), size.amax(-1)


def quantise(x, exponent=0):
    """Values that rows x [..., D] are held as in the 4-bit cache."""
    y = x.double().unflatten(-1, (-1, GROUP)) * 2.0 ** -exponent
    odd = ~torch.isfinite(y).all(-1)
    m = torch.where(torch.isfinite(y), y.abs(), torch.zeros_like(y)).amax(-1)
    s = (m / 7).clamp(max=448.0)
    step = torch.exp2(torch.floor(torch.log2(s.clamp(min=2.0 ** -6))) - 3)
    s = (torch.round(s / step) * step).clamp(max=448.0)
    c = torch.where(s[..., None] > 0, torch.floor(y.abs() / torch.where(s > 0, s, torch.ones_like(s))[..., None] + 0.5).clamp(max=7), torch.zeros_like(y))
    got = torch.sign(y) * c * s[..., None] * 2.0 ** exponent
    return torch.where(odd[..., None], torch.full_like(got, math.nan), got).flatten(-2)


def attention_bound(o, weighted, size, *, dtype, weights, D, v):
    """How far a kernel's output may be from 64 bits, element by element: weights rounded to `weights` (each off by half a step, so that the sum moves by at
    most that share of sum p |v|) and the result rounded to `dtype`; and fp32 scores, off by at most D + 8 roundings of 2^-23 of sum |q k| scale (tensor cores
    truncate), which moves each weight by twice that share.

    Weights in fp16 have a smallest step as well, 2^-24: the kernels give the largest weight of the moment 2^7 or more, so that rounding to that step moves a
    weight of the normalised sum by at most 2^-25 / 2^7 = 2^-32, and the result by 2^-32 of sum |v| over the keys (v, [keys, heads of o, D])."""
    score = (D + 8) * 2.0 ** -23 * size.transpose(0, 1)[..., None] + 2.0 ** -20
    floor = 2.0 ** -32 * v.double().abs().sum(0).repeat_interleave(o.shape[1] // v.shape[1], 0) if weights == torch.float16 else 0
    return unit(dtype) * o.abs() + (unit(weights) + 2 * score) * weighted * (1 + unit(dtype)) + floor + 2.0 ** -30


def lse_bound(lse, size, D):
    return (D + 8) * 2.0 ** -23 * size + 2.0 ** -20 * (1 + torch.where(torch.isfinite(lse), lse.abs(), torch.zeros_like(lse)))


def check(got, want, bound, what):
    got = got.double()
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    bad = ~(same | ((got - want).abs() <= bound))
    if bad.any():
        at = tuple(int(i) for i in bad.nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} values out of bounds, first at {at}: {float(got[at])} for {float(want[at])}, bound "
                             f"{float(bound[at] if bound.numel() > 1 else bound)}")
