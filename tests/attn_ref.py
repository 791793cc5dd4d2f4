"""Plain 64-bit forms of the operators around the cache, with the rounding that
their kernels may add (imported by test modules only)."""

import math

import torch

# half a step of every type, relative to the value
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def visible(n, m, T, start, window, sinks, device="cpu"):
    """``(T, n)``: what query t of m sees of n keys."""
    p = (n - m + torch.arange(T, device=device))[:, None]
    j = torch.arange(n, device=device)[None]
    low = p - window if window else torch.full_like(p, -1)
    return (torch.arange(T, device=device)[:, None] < m) & (j <= p) & (j >= start) & ((j > low) | (j < start + sinks))


def attention(q, k, v, sees, scale):
    """One sequence: ``q (Hq, T, D)`` over ``k, v (Hkv, n, D)`` under ``sees (T,
    n)``: the output in 64 bits, sum_j p_j |v_j| and the largest sum_i |q_i k_ji|
    of a row (what roundings are relative to).  Hidden places count for nothing,
    whatever they hold; a row that sees nothing gives zeros."""
    g = q.shape[0] // k.shape[0]
    q, k, v = q.double(), k.double().repeat_interleave(g, 0), v.double().repeat_interleave(g, 0)
    hidden = ~sees
    some = sees.any(0)[None, :, None]
    kz = torch.where(some, k, 0.0)
    s = torch.matmul(q, kz.transpose(1, 2).contiguous()) * scale
    s = s.masked_fill(hidden, -math.inf)
    top = s.amax(-1, keepdim=True) if s.shape[-1] else torch.full(s.shape[:-1] + (1,), -math.inf, dtype=s.dtype, device=s.device)
    w = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
    den = w.sum(-1, keepdim=True)
    w = torch.where(den == 0, torch.zeros_like(w), w / torch.where(den == 0, torch.ones_like(den), den))
    vz = torch.where(some, v, 0.0)
    mag = torch.matmul(q.abs(), kz.abs().transpose(1, 2).contiguous()).masked_fill(hidden, 0.0)
    mag = mag.amax(-1, keepdim=True) if mag.shape[-1] else torch.zeros_like(den)
    fin = torch.where(torch.isfinite(vz), vz, 0.0)
    out = torch.matmul(w, fin)
    if not bool(torch.isfinite(vz).all()):
        # infinities and NaN, only into the rows that see them
        odd = torch.where(torch.isfinite(vz), 0.0, vz)
        for j in torch.nonzero((odd != 0).any(0).any(-1)).flatten().tolist():
            out = out + torch.where(sees[None, :, j, None], w[:, :, j, None] * odd[:, j, None, :], 0.0)
    return out, torch.matmul(w, fin.abs()), mag, fin.abs().amax() if vz.numel() else torch.zeros(())


def attention_bound(dtype, want, weighted, mag, vmax, n, D, scale):
    """How far a 16-bit attention with fp32 sums may be off: the output's
    rounding; every weight's rounding to the type (and, in fp16, to a multiple of
    2^-24 where it is small: half a step of that for each of n weights, against a
    sum of at least 1); the scores' sum over D products, each within 2^-23 of
    the products' magnitude, which moves numerator and denominator; exp2, the
    running sums over n weights in 2^-24 steps and the rescales: n / 16 + 64 of
    them in each of numerator and denominator."""
    score = 2 * scale * D * 2.0 ** -23 * mag
    sums = 2 * (n / 16 + 64) * 2.0 ** -24
    low = n * 2.0 ** -25 * float(vmax) if dtype == torch.float16 else 0.0
    tiny = 2.0 ** -25  # fp16 outputs below its normal range
    return HALF[dtype] * want.abs() + (HALF[dtype] * (1 + HALF[dtype]) + score + sums) * weighted + low + tiny
