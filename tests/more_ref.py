"""Plain 64-bit forms of the operators that read less of a coded cache: chosen
groups, received weights, eviction (imported by test modules only)."""

import math

import torch

from attn_ref import HALF, attention


def tokens(seed, B, H, L, D, dtype):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    scale = torch.exp(torch.randn((B, H, 1, D), generator=gen, device="cuda"))
    k = (torch.randn((B, H, L, D), generator=gen, device="cuda") * scale).to(dtype)
    v = torch.randn((B, H, L, D), generator=gen, device="cuda").to(dtype)
    return k, v


def make_pool(seed, lens, Hq, H, D=128, room=0, **kw):
    from turboquant_pro_amd import TQKVPool
    top = max(max(lens), 1)
    pool = TQKVPool(n_kv_heads=H, n_q_heads=Hq, head_dim=D, max_batch=len(lens), max_seq_len=top + room, seed=seed, **kw)
    k, v = tokens(seed, len(lens), H, top, D, pool.dtype)
    pool.append(k, v, n_new=lens)
    pool.check()
    return pool


def queries(seed, pool, T):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn((pool.max_batch, T, pool.n_q_heads, pool.head_dim), generator=gen,
                       device="cuda").to(pool.dtype).transpose(1, 2)


def cached(pool, b):
    """Keys and values (H, n, D) of sequence b as the cache holds them."""
    H, D, ng = pool.n_kv_heads, pool.head_dim, pool.n_groups(b)
    ks, vs = [], []
    if ng:
        k, v = pool.dequant_groups([(b, g) for g in range(ng)])
        ks, vs = ([x.permute(1, 0, 2, 3).reshape(H, -1, D).double()] for x in (k, v))
    hk, hv = pool.hot_window_tokens(b)
    return torch.cat(ks + [hk.double()], 1), torch.cat(vs + [hv.double()], 1)


def listed(pool, b, groups, T, m):
    """``(H, T, n)``: what query t of m sees of sequence b with ``groups (H, T or 1, K)``."""
    n, G, ng = pool.lengths[b], pool.group_tokens, pool.n_groups(b)
    j = torch.arange(n, device="cuda")
    p = (n - m + torch.arange(T, device="cuda"))[:, None]
    of = torch.where(j < ng * G, j // G, -1)
    pick = groups.long()
    pick = torch.where((pick >= 0) & (pick < ng), pick, -2)
    inside = (of == -1) | (of[None, None, None] == pick[..., None]).any(2)
    return inside & (j <= p) & (torch.arange(T, device="cuda")[:, None] < m)


def coefficient(mag, n, D):
    """What the scores' sums (fp32, their operands fp16 pairs: 32 units in the last
    place and one a product) and the sums of weights may move a weight by, relative to
    it: numerator and denominator."""
    return 2 * D ** -0.5 * mag * (32 + D) * 2.0 ** -24 + (n / 16 + 64) * 2.0 ** -23


def check_rows(out, q, k, v, sees, what=""):
    """One sequence and kv head's rows ``out, q (gq, T, D)`` over ``k, v (n, D)`` under
    ``sees (T, n)``.  The kernels round the value centroids to fp16, which the rotation
    spreads over the channels (half a step of sum p |v|_2), and the output.  Returns
    the squared distance and size."""
    n, D = k.shape
    scale = 1.0 / math.sqrt(D)
    want, _, mag, _ = attention(q, k[None], v[None], sees, scale)
    size = attention(q, k[None], v.norm(dim=-1, keepdim=True).expand_as(v)[None].contiguous(), sees, scale)[0]
    half = HALF[torch.float16]
    tol = half * want.abs() + (coefficient(mag, n, D) + half) * size + 2.0 ** -25
    got = out.double()
    assert torch.isfinite(got).all(), what
    err = (got - want).abs()
    assert bool((err <= tol).all()), f"{what}: {float((err - tol).max()):.3e} past the bound"
    assert bool((out[:, ~sees.any(1)] == 0).all()), f"{what}: rows that see nothing"
    return float(err.square().sum()), float(want.square().sum())


def check_listed(pool, out, q, groups, q_lens=None, what=""):
    B, Hq, T, D = q.shape
    H = pool.n_kv_heads
    gq = Hq // H
    off = tot = 0.0
    assert out.shape == q.shape and out.dtype == q.dtype
    for b in range(B):
        m = T if q_lens is None else q_lens[b]
        if pool.lengths[b] == 0:
            assert bool((out[b] == 0).all())
            continue
        k, v = cached(pool, b)
        sees = listed(pool, b, groups[b], T, m)
        for h in range(H):
            s = slice(h * gq, (h + 1) * gq)
            e, w = check_rows(out[b, s], q[b, s], k[h], v[h], sees[h], f"{what} seq {b} head {h}")
            off, tot = off + e, tot + w
    # random roundings do not add up as the bound allows: together 2^-10 of the output
    assert math.sqrt(off / max(tot, 1e-30)) <= 2.0 ** -10, what


def chosen(pool, q, top, first, last, spread, q_lens=None):
    """The groups of every query from the definition, in 64 bits on the host."""
    B, Hq, T, D = q.shape
    H, G = pool.n_kv_heads, pool.group_tokens
    gq = Hq // H
    got = torch.full((B, H, T, top), -1, dtype=torch.int32)
    steps = (2 ** pool.key_bits - 1) / 2 if pool.key_grid == "uniform" else None
    for b in range(B):
        n, ng = pool.lengths[b], pool.n_groups(b)
        m = T if q_lens is None else q_lens[b]
        slots = pool.group_table[b, :ng].long()
        mean, scale = pool.gmean[slots].double().cpu(), pool.gscale[slots].double().cpu()
        mid, half = (mean, scale) if steps is None else (mean + scale * steps, scale * steps)
        for h in range(H):
            for t in range(m):
                p = n - m + t
                c = min(ng, p // G + 1) if p >= 0 else 0
                x = q[b, h * gq:(h + 1) * gq, t].double().cpu()
                s = ((x[:, None] * mid[None, :c, h]).sum(-1) + spread * (x.abs()[:, None] * half[None, :c, h]).sum(-1))
                s = torch.where(s.isnan().any(0), torch.full((), math.nan, dtype=s.dtype), s.amax(0)).tolist() if c else []
                pick = [g for g in range(c) if g < first or g >= c - last] if c > top else list(range(c))
                rest = sorted((g for g in range(c) if g not in set(pick)),
                              key=lambda g: (0, 0.0, g) if math.isnan(s[g]) else (1, -s[g], g))
                pick = sorted(pick + rest[:top - len(pick)])
                got[b, h, t, :len(pick)] = torch.tensor(pick, dtype=torch.int32)
    return got
