"""Plain 64-bit forms of the group-affine cache's operators (torch, CPU), and how far a kernel may be from them.

Words are LSB-first; a group's bias is its least value, its scale a
(2^bits - 1)-th of its range (a difference and a division in f32) rounded to
the vectors' dtype, its codes the number of half steps that x - bias (in f32)
reaches.
"""
import math

import torch

LOWEST = torch.finfo(torch.float32).min


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def quantize(x, bits, group):
    """(words as int64, params (..., groups, 2) in x's dtype) of CPU vectors."""
    n = 2 ** bits - 1
    g = x.unflatten(-1, (-1, group))
    lo, hi = g.min(-1).values, g.max(-1).values
    # the range and its division are f32 operations, in halves so that the range stays finite
    scale = ((hi.float() * 0.5 - lo.float() * 0.5) / n * 2.0).to(x.dtype)
    scale = torch.where(scale.double() < 2.0 ** -100, torch.zeros_like(scale), scale)
    # x - lo in f32, taken in halves: exact beyond f32's range too
    away = (g.float() * 0.5 - lo.float()[..., None] * 0.5).double() * 2
    step = scale.double()[..., None]
    codes = torch.floor(away / torch.where(step > 0, step, torch.ones_like(step)) + 0.5).clamp(0, n)
    codes = torch.where(step > 0, codes, torch.zeros_like(codes))
    bad = ~torch.isfinite(g).all(-1)
    codes = torch.where(bad[..., None], torch.zeros_like(codes), codes)
    nan = torch.full_like(scale, math.nan)
    params = torch.stack([torch.where(bad, nan, scale), torch.where(bad, nan, lo)], -1)
    per = 32 // bits
    c = codes.long().flatten(-2).unflatten(-1, (-1, per))
    return (c << torch.arange(0, 32, bits)).sum(-1), params


def values(words, params, bits, group):
    """f64 values that int64 words and params stand for."""
    c = (words.long()[..., None] >> torch.arange(0, 32, bits)) & (2 ** bits - 1)
    c = c.flatten(-2).unflatten(-1, (-1, group)).double()
    return (c * params[..., 0, None].double() + params[..., 1, None].double()).flatten(-2)


def words_of(codes):
    """A uint32 tensor's values as int64 on the CPU."""
    return codes.view(torch.int32).cpu().long() & 0xFFFFFFFF


def attention(q, k, v, scale, causal=False, seq_lens=None, seq_starts=None, mask=None):
    """(out, scores, weights) in f64 of q (B, Hq, L, Dk) over k, v (B, Hkv, T, .); mask broadcasts to (B, Hq, L, T)."""
    B, Hq, L, _ = q.shape
    Hkv, T = k.shape[1], k.shape[2]
    k, v = (t.double().repeat_interleave(Hq // Hkv, 1) for t in (k, v))
    end = torch.full((B,), T) if seq_lens is None else torch.as_tensor(seq_lens).long()
    start = torch.zeros(B).long() if seq_starts is None else torch.as_tensor(seq_starts).long()
    t = torch.arange(T)
    held = (t >= start[:, None]) & (t < end[:, None])
    s = torch.matmul(q.double(), torch.nan_to_num(k, nan=0.0).transpose(-1, -2)) * scale
    if mask is not None:
        m = torch.as_tensor(mask)
        if m.dtype == torch.bool:
            s = torch.where(m, s, torch.full_like(s, LOWEST))
        else:
            s = torch.where(torch.isneginf(m), torch.full_like(s, -math.inf), (s + m.double()).clamp_min(LOWEST))
    if causal:
        last = end[:, None] - L + torch.arange(L)
        hidden = (t > last[..., None])[:, None] & ~torch.isneginf(s)
        s = torch.where(hidden, torch.full_like(s, LOWEST), s)
    s = torch.where(held[:, None, None], s, torch.full_like(s, -math.inf))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isneginf(top), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = torch.where(total > 0, p / torch.where(total > 0, total, torch.ones_like(total)), torch.zeros_like(p))
    return torch.matmul(p, torch.where(torch.isnan(v), torch.zeros_like(v), v)), s, p


def attention_tolerance(q, k_params, k_bits, v, want, p, scale, dtype, group, rounded):
    """How far a kernel's output may be from ``want`` (B, Hq, L, Dv), element by element.

    Scores: q and codes meet exactly (or q off by 2^-27 of its row's largest); a
    sum of D products in f32 is off by at most (D / 4 + 8) * 2^-24 of the sum of
    their magnitudes, where a code may be carried as 128 + c (4 bits) or
    1024 + c (8 bits) and the group's sum taken off again.  A score's
    error dS moves a weight by 2 dS of itself at most (numerator and sum) while
    dS is small.  ``rounded``: keys, weights and values go through f16 (many
    query rows); independent roundings of half a step u add up to at most 6 u
    sqrt(sum of squares).  f16 ends at 2^-24: queries, brought to [1, 2), are off
    by 2^-25 of the row's largest, weights by 2^-25 of a sum of one or more, keys
    and values whose group's largest is 2^-15 or more by 2^-10 of that, a step u
    once more (others, and those past 65504, meet the f32 way).  Otherwise a weight times a scale keeps 16 bits
    (two bf16 pieces, each rounded), of codes up to 143 while in flight.  The
    result is rounded once.
    """
    B, Hq, L, D = q.shape
    R = Hq // k_params.shape[1]
    u = 2.0 ** -11 if rounded and dtype != torch.float32 else 0.0
    if dtype == torch.bfloat16:
        u = 2 * u
    kp = torch.nan_to_num(k_params.double(), nan=0.0, posinf=0.0, neginf=0.0).repeat_interleave(R, 1)
    top = 128 + 15 if k_bits == 4 else 1024 + 255
    size = kp[..., 0].abs() * top + kp[..., 1].abs()                              # (B, Hq, T, groups)
    qa = q.double().abs().unflatten(-1, (-1, group))
    mag = torch.matmul(qa.sum(-1), size.transpose(-1, -2)).amax(-1) * abs(scale)  # (B, Hq, L)
    rms = torch.sqrt(torch.matmul(qa.square().sum(-1), size.square().transpose(-1, -2))).amax(-1) * abs(scale)
    dS = mag * (D / 4 + 8) * 2.0 ** -24 + 6 * u * rms + 2.0 ** -20
    if u:
        dS = dS + 2.0 ** -25 * q.double().abs().amax(-1) * size.sum(-1).amax(-1, keepdim=True) * group * abs(scale)
    vt = torch.nan_to_num(v.double(), nan=0.0, posinf=0.0, neginf=0.0)
    vmax = vt.abs().amax((-1, -2)).repeat_interleave(R, 1)                        # (B, Hq)
    root = p.square().sum(-1).sqrt()
    # two or three roundings of weight and value, then the pieces
    dV = vmax[..., None] * (18 * u * root + 20 * 2.0 ** -16 * root + 2.0 ** -18 + (u > 0) * v.shape[2] * 2.0 ** -25)
    return half_step(dtype) * want.abs() * 1.01 + (2 * dS * vmax[..., None] + dV)[..., None] + 1e-30
