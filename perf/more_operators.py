"""What is measured of the operators that read less of a long coded cache.

Kinds of cases, all over a ``TQKVPool`` (4-bit asym-NF4 keys with an fp16
side-list, PolarQuant values, an uncoded hot window, paged):

* ``choose``  every query picks the coded groups that it attends by a score of
  their scales and zero points, and attends them and the uncoded tokens
  (``TQKVPool.select_groups``, then ``attend(groups=...)``);
* ``weigh``   attention that adds up the weight which every coded group received
  (``attend(weights=...)``);
* ``evict``   the groups of little weight leave the cache (``TQKVPool.evict``);
* ``shared``  a batch whose sequences begin with the same tokens, held once
  (``TQKVPool.share_prefix``, then ``attend``).

``run`` computes them in plain torch, or with ``own`` calls the framework.
``exact`` restates them in 64 bits from the unpacked codes.
"""

from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

sys.path.insert(1, os.path.join(os.getcwd(), "turboquant-pro_amd"))

own = False

# Lloyd-Max N(0,1) levels and NormalFloat-4 levels: the formats' tables
LLOYD_MAX = {
    2: (-1.510, -0.453, 0.453, 1.510),
    3: (-1.748, -1.050, -0.500, -0.069, 0.069, 0.500, 1.050, 1.748),
    4: (-2.401, -1.844, -1.437, -1.099, -0.800, -0.524, -0.262, -0.066,
        0.066, 0.262, 0.524, 0.800, 1.099, 1.437, 1.844, 2.401),
}
NF4 = (-1.0, -0.6961928009986877, -0.5250730514526367, -0.39491748809814453, -0.28444138169288635,
       -0.18477343022823334, -0.09105003625154495, 0.0, 0.07958029955625534, 0.16093020141124725,
       0.24611230194568634, 0.33791524171829224, 0.44070982933044434, 0.5626170039176941,
       0.7229568362236023, 1.0)


def _case(name, kind, **kw):
    case = dict(name=name, kind=kind, batch=16, q_heads=32, kv_heads=8, head_dim=128, length=32768, q_len=1,
                ragged=False, page=32, hot_window=512, value_bits=3, outliers=0.02)
    if kind == "choose":
        case.update(top=16, first=1, last=1, spread=1.0)
    elif kind == "weigh":
        case.update(window=0, sinks=0)
    elif kind == "evict":
        case.update(keep=64, first=1, last=1)
    else:
        case.update(prefix=32768)
    case.update(kw)
    return case


def listed():
    return [
        # the serving step at full context: an eighth of the cache's groups
        _case("choose_b16_32k", "choose"),
        # one long conversation: 64 groups of 511
        _case("choose_b1_128k", "choose", batch=1, length=131072, top=64, value_bits=4),
        # groups of 32 tokens, 7 query heads a kv head, ragged, three queries to verify
        _case("choose_fine_ragged", "choose", batch=8, q_heads=28, kv_heads=4, length=6001, q_len=3, ragged=True,
              page=16, hot_window=64, top=24, first=2, last=2, spread=0.5),
        # head_dim 256 (16 / 8 heads)
        _case("choose_d256", "choose", batch=8, q_heads=16, head_dim=256, length=8192, value_bits=4, top=8, last=0),
        # the serving step that keeps the groups' weights
        _case("weigh_b16_32k", "weigh"),
        # one short conversation: latency
        _case("weigh_b1_4k", "weigh", batch=1, length=4096, value_bits=4),
        # a verification step of four queries, head_dim 64, windowed, ragged, no side-list
        _case("weigh_d64_ragged", "weigh", batch=5, q_heads=16, kv_heads=4, head_dim=64, length=5003, q_len=4,
              ragged=True, value_bits=2, outliers=0.0, window=2001, sinks=4),
        # half of a full cache leaves it
        _case("evict_b16_32k", "evict", ragged=True),
        # two conversations, groups of 24 tokens, a ring whose places move
        _case("evict_b2_small", "evict", batch=2, kv_heads=2, q_heads=2, length=3001, page=24, hot_window=47, keep=37,
              first=3, last=4),
        # one long document asked about by 32 users
        _case("shared_b32_32k", "shared", batch=32, length=34000),
        # a short system prompt of a large batch
        _case("shared_b64_2k", "shared", batch=64, prefix=2048, length=2500, ragged=True, value_bits=4),
        # head_dim 256 (16 / 8 heads), three queries to verify
        _case("shared_d256_verify", "shared", batch=6, q_heads=16, head_dim=256, prefix=8192, length=9001, q_len=3,
              ragged=True, value_bits=4),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(["choose", "choose", "weigh", "weigh", "evict", "shared", "shared"])
    D = rng.choice([64, 128, 128, 128, 256])
    H = rng.choice([1, 2, 4, 8, 8])
    Hq = H * rng.choice([1, 2, 4, 7, 8])
    B = _log(rng, 1, 32)
    W, page = rng.choice([(512, 32), (512, 32), (512, 16), (256, 32), (64, 32), (48, 24), (47, 12)])
    T = 1 if rng.random() < 0.6 else _log(rng, 2, 8)
    # cached cells: no more than half of the largest listed case's
    top = max(700, min(65536, 16 * 32768 * 8 * 128 // (2 * B * H * D)))
    L = _log(rng, 100, top)
    kw = dict(batch=B, q_heads=Hq, kv_heads=H, head_dim=D, length=L, q_len=min(T, L), ragged=rng.random() < 0.4,
              page=page, hot_window=W, value_bits=rng.choice([2, 3, 3, 4]), outliers=rng.choice([0.02, 0.02, 0.0]))
    groups = max(1, _groups(L, W))
    if kind == "choose":
        pick = _log(rng, 1, max(2, min(128, groups // 2)))
        first, last = rng.choice([0, 0, 1, 2]), rng.choice([0, 1, 1, 3])
        kw.update(top=max(pick, first + last), first=first, last=last, spread=rng.choice([0.0, 0.5, 1.0, 1.0]))
        while kw["q_len"] * kw["top"] * W * B * Hq > 1 << 24 and kw["q_len"] > 1:
            kw["q_len"] -= 1
    elif kind == "weigh":
        kw.update(window=rng.choice([0, 0, _log(rng, 1, 8192)]), sinks=rng.choice([0, 4, _log(rng, 1, 300)]))
        while B * Hq * kw["q_len"] * L > 16 * 32 * 32768 and kw["q_len"] > 1:
            kw["q_len"] -= 1
    elif kind == "evict":
        kw.update(q_len=1, keep=_log(rng, 8, max(9, groups)), first=rng.choice([0, 1, 3]), last=rng.choice([0, 1, 4]))
    else:
        prefix = _log(rng, 100, L)
        kw.update(prefix=prefix, length=prefix + kw["q_len"] + _log(rng, 1, 2000))
        while B * Hq * kw["q_len"] * L > 32 * 32 * 32768 // 2 and kw["q_len"] > 1:
            kw["q_len"] -= 1
    case = _case("", kind, **kw)
    del case["name"]
    return case


# ------------------------------------------------------------------ inputs --
def _gen(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return gen


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _groups(length, W):
    G = (W + 1) // 2
    return 0 if length <= W else (length - (W + 1)) // G + 1


def _low(case):
    return case["prefix"] + case["q_len"] if case["kind"] == "shared" else case["q_len"]


def _lengths(case):
    """Every sequence's length: the case's, or ragged up to it."""
    if not case["ragged"]:
        return [case["length"]] * case["batch"]
    rng = np.random.default_rng(case["batch"] * 7919 + case["length"])
    low = max(_low(case), (case["length"] + 2) // 3)
    return [int(n) for n in rng.integers(low, case["length"] + 1, size=case["batch"])]


def _rotation(seed, D):
    gauss = np.random.default_rng(seed).standard_normal((D, D)).astype(np.float32)
    return np.ascontiguousarray(np.linalg.qr(gauss)[0])


class _Form:
    """A pool's numbers: groups, pages and side-list of the case."""

    def __init__(self, case):
        self.W, self.P = case["hot_window"], case["page"]
        self.G = (self.W + 1) // 2
        self.groups = max(1, _groups(case["length"], self.W))
        self.per_group = self.G // self.P
        self.pages = self.groups * self.per_group
        self.k_out = max(1, round(self.G * case["outliers"])) if case["outliers"] else 0
        # the pool's capacity: four times the nominal side-list, at most the group
        self.cap = min(self.G * case["head_dim"], 4 * self.k_out * case["head_dim"])
        self.tiled = case["head_dim"] == 128 and self.P % 16 == 0 and self.G % 32 == 0
        # coded groups that all sequences share
        self.shared = _groups(case["prefix"], self.W) if case["kind"] == "shared" else 0


def _coded(case, seed):
    """A cache's contents, unpacked: codes, scales, side-list, norms, hot window,
    (sequence, group, head, ...); a shared group is the first sequence's."""
    f, gen = _Form(case), _gen(seed)
    B, H, D, G, ng = case["batch"], case["kv_heads"], case["head_dim"], f.G, f.groups
    c = {}
    nf4 = torch.tensor(NF4, device="cuda")
    cut = (nf4[1:] + nf4[:-1]) / 2 * 2.9
    lm = torch.tensor(LLOYD_MAX[case["value_bits"]], device="cuda")
    vcut = (lm[1:] + lm[:-1]) / 2
    big = torch.rand((B, 1, H, D), generator=gen, device="cuda").argsort(-1) < max(1, round(0.02 * D))
    chan = torch.exp(_randn(gen, B, 1, H, D)) * torch.where(big, 10.0, 1.0)
    # neighbouring tokens are alike: a group has a direction of its own
    c["scale"] = 2.9 * chan * torch.exp(0.1 * _randn(gen, B, ng, H, D))
    c["mean"] = 0.3 * chan * _randn(gen, B, ng, H, D)
    c["kcode"] = torch.zeros((B, ng, H, G, D), dtype=torch.uint8, device="cuda")
    c["vcode"] = torch.zeros_like(c["kcode"])
    for b in range(B):
        own_from = f.shared if b else 0
        n = ng - own_from
        if n:
            c["kcode"][b, own_from:] = torch.bucketize(_randn(gen, n, H, G, D), cut, out_int32=True)
            c["vcode"][b, own_from:] = torch.bucketize(_randn(gen, n, H, G, D), vcut, out_int32=True)
    c["vnorm"] = math.sqrt(D) * (1.0 + 0.1 * _randn(gen, B, ng, H, G)).clamp(0.5, 2.0)
    c["hot_k"] = (chan.transpose(1, 2) * _randn(gen, B, H, f.W, D)).half()
    c["hot_v"] = _randn(gen, B, H, f.W, D).half()
    if f.k_out:
        # k_out distinct tokens of every channel; entries in (token, channel) order
        first = torch.randint(0, G, (B, ng, H, D, 1), generator=gen, device="cuda")
        tok = (first + torch.arange(f.k_out, device="cuda") * (G // f.k_out)) % G
        at = (tok * D + torch.arange(D, device="cuda")[:, None]).flatten(-2).sort(-1).values
        val = c["scale"].gather(-1, at % D) * (1.0 + 0.2 * _randn(gen, *at.shape))
        c["at"], c["val"] = at, val.clamp(-6e4, 6e4).half()
        c["kcode"].view(B, ng, H, G * D).scatter_(-1, at, 7)  # (the zero level stands there)
    if f.shared:
        for x in c.values():
            if x.shape[1] == ng and x.dim() >= 4 and x is not c["hot_k"] and x is not c["hot_v"]:
                x[1:, :f.shared] = x[:1, :f.shared]
    c["table"] = torch.randperm(B * f.pages, generator=gen, device="cuda").int().view(B, f.pages)
    c["q"] = _randn(gen, B, case["q_heads"], case["q_len"], D).half()
    # what attention leaves: little on most groups, much on a few
    c["weights"] = torch.exp(2.0 * _randn(gen, B, H, ng))
    c["lens"] = _lengths(case)
    return c


def _pack_stream(code, bits):
    """Codes ``(..., n)`` as a little-endian bit stream of ``n * bits / 8`` bytes."""
    x = code.view(*code.shape[:-1], -1, 8).int()
    word = sum(x[..., i] << (bits * i) for i in range(8))
    return torch.stack([(word >> (8 * i)) & 255 for i in range(bits)], -1).to(torch.uint8).flatten(-2)


class _State:
    pass


def prepare(case, seed):
    s = _State()
    s.case = case
    f, c = _Form(case), _coded(case, seed)
    B, H, D, G, P, ng, vb = (case["batch"], case["kv_heads"], case["head_dim"], f.G, f.P, f.groups,
                             case["value_bits"])
    s.form = f
    s.kcodes = torch.zeros((H, B * f.pages, P, D // 2), dtype=torch.uint8, device="cuda")
    s.vcodes = torch.zeros((H, B * f.pages, P, D * vb // 8), dtype=torch.uint8, device="cuda")
    s.vnorm = torch.zeros((H, B * f.pages, P), device="cuda")
    rev = torch.tensor([int(format(i, "04b")[::-1], 2) for i in range(16)], dtype=torch.uint8, device="cuda")
    for b in range(B):
        g0 = f.shared if b else 0
        at = c["table"][b, g0 * f.per_group:].long()
        if not len(at):
            continue
        k = rev[c["kcode"][b, g0:].transpose(0, 1).int()]
        s.kcodes[:, at] = ((k[..., 0::2] << 4) | k[..., 1::2]).reshape(H, -1, P, D // 2)
        v = c["vcode"][b, g0:].transpose(0, 1)
        if f.tiled:  # units of 4 tokens x 8 channels, a channel's tokens side by side
            v = v.reshape(H, -1, P // 16, 4, 4, 16, 8).permute(0, 1, 2, 3, 5, 6, 4).contiguous().flatten(-2)
        s.vcodes[:, at] = _pack_stream(v.contiguous(), vb).reshape(H, -1, P, D * vb // 8)
        s.vnorm[:, at] = c["vnorm"][b, g0:].transpose(0, 1).reshape(H, -1, P)
    s.gscale, s.gmean = c["scale"].view(B * ng, H, D), c["mean"].view(B * ng, H, D)
    s.ocount = torch.zeros((B * ng, H, 8), dtype=torch.int32, device="cuda")
    s.oent = torch.zeros((B * ng, H, max(f.cap, 1)), dtype=torch.int32, device="cuda")
    if f.k_out:
        at = c["at"].view(B * ng, H, -1)
        bits = c["val"].view(torch.int16).int().view(at.shape)
        s.oent[..., :at.shape[-1]] = at.int() | (bits << 16)
        s.ocount[:] = (at[..., None] // D < 32 * torch.arange(1, 9, device="cuda")).sum(-2)
    s.hot_k, s.hot_v, s.q, s.lens = c["hot_k"], c["hot_v"], c["q"], c["lens"]
    s.weights = c["weights"]
    s.seq_lens = torch.tensor(s.lens, dtype=torch.int32, device="cuda")
    s.weights *= torch.arange(ng, device="cuda") < torch.tensor([_groups(n, f.W) for n in s.lens],
                                                                device="cuda")[:, None, None]
    s.table, s.slots = c["table"], torch.arange(B * ng, dtype=torch.int32, device="cuda").view(B, ng)
    own_table = s.table.cpu().numpy()
    if f.shared:
        s.table, s.slots = s.table.clone(), s.slots.clone()
        s.table[:, :f.shared * f.per_group] = s.table[0, :f.shared * f.per_group]
        s.slots[:, :f.shared] = s.slots[0, :f.shared]
    pi = _rotation(seed, D)
    s.pi = torch.from_numpy(pi).cuda()
    s.cent = (torch.tensor(LLOYD_MAX[vb], dtype=torch.float64) / math.sqrt(D)).float().cuda()
    s.pool = None
    if own:  # the pool that a serving program keeps, holding this cache
        from turboquant_pro_amd import TQKVPool
        p = s.pool = TQKVPool(n_kv_heads=H, n_q_heads=case["q_heads"], head_dim=D, max_batch=B,
                              max_seq_len=case["length"], hot_window=f.W, value_bits=vb,
                              outlier_frac=case["outliers"], page_tokens=P, rotation=(pi, pi.T),
                              block_table=own_table, input_dtype="float16")
        for name in ("kcodes", "vcodes", "vnorm", "gscale", "gmean", "ocount", "oent", "hot_k", "hot_v"):
            getattr(p, name).copy_(getattr(s, name).view(getattr(p, name).shape))
        if case["kind"] == "shared":  # the prefix in the first sequence, then in all
            p.lengths = [case["prefix"]] + [0] * (B - 1)
            p.seq_lens.copy_(torch.tensor(p.lengths, dtype=torch.int32))
            p.share_prefix(0)
            p.hot_k.copy_(s.hot_k)
            p.hot_v.copy_(s.hot_v)
        p.seq_lens.copy_(s.seq_lens)
        p.lengths = list(s.lens)
    return s


# ------------------------------------------------------------- plain forms --
def _dense(s, b, h, g):
    """fp32 keys and values ``(..., G, D)`` of the groups ``g`` of heads ``h`` of
    sequences ``b`` (index tensors of one shape)."""
    case, f = s.case, s.form
    D, G, P, vb = case["head_dim"], f.G, f.P, case["value_bits"]
    t = torch.arange(G, device="cuda")
    page = s.table.long()[b[..., None], g[..., None] * f.per_group + t // P]
    off = t % P
    hh = h[..., None]
    # keys: four bits a code, most significant first, the even channel above
    byte = s.kcodes[hh, page, off].int()
    code = torch.stack([byte >> 4, byte & 15], -1).flatten(-2)
    code = ((code & 1) << 3) | ((code & 2) << 1) | ((code & 4) >> 1) | ((code & 8) >> 3)
    slot = s.slots.long()[b, g]
    k = s.gmean[slot, h][..., None, :] + s.gscale[slot, h][..., None, :] * torch.tensor(NF4, device="cuda")[code]
    if f.k_out:
        ent = s.oent[slot, h]
        real = torch.arange(ent.shape[-1], device="cuda") < s.ocount[slot, h, 7][..., None]
        val = (ent >> 16).to(torch.int16).view(torch.float16).float()
        k = torch.cat([k.flatten(-2), torch.zeros_like(val[..., :1])], -1)  # (one place for what is no entry)
        k = k.scatter(-1, torch.where(real, (ent & 0xFFFF).long(), G * D), val)[..., :-1].unflatten(-1, (G, D))
    # values: a little-endian stream a token, or a unit of 4 tokens x 8 channels
    if f.tiled:
        unit = s.vcodes.view(case["kv_heads"], -1, P // 16, 4, 16, 4, vb)[hh, page, off // 16, off % 16 // 4]
    else:
        unit = s.vcodes.view(case["kv_heads"], -1, P, D // 8, vb)[hh, page, off]
    word = (unit.long() << (8 * torch.arange(vb, device="cuda"))).sum(-1)
    code = (word[..., None] >> (vb * torch.arange(8, device="cuda"))) & ((1 << vb) - 1)
    if f.tiled:
        code = code.reshape(*code.shape[:-3], 16, 8, 4)
        code = code.gather(-1, (t % 4).view(G, 1, 1, 1).expand(*code.shape[:-1], 1))
    v = (s.cent[code.reshape(*page.shape, D)] @ s.pi) * s.vnorm[hh, page, off][..., None]
    return k, v


def _hot(s):
    """fp32 keys and values of the rings in token order, ``(B, H, W, D)``, and their tokens ``(B, W)``."""
    f = s.form
    length = s.seq_lens.long()
    ng = torch.where(length <= f.W, 0, torch.div(length - (f.W + 1), f.G, rounding_mode="floor") + 1)
    t = (ng * f.G)[:, None] + torch.arange(f.W, device="cuda")
    at = (t % f.W)[:, None, :, None].expand(-1, s.hot_k.shape[1], -1, s.hot_k.shape[-1])
    return s.hot_k.float().gather(2, at), s.hot_v.float().gather(2, at), t, ng


def _softmax(score):
    """Rows' softmax; a row without a visible token: zeros."""
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    den = p.sum(-1, keepdim=True)
    return p / torch.where(den == 0, 1.0, den)


def _plain_choose(s):
    case, f = s.case, s.form
    B, Hq, H, T, D, G, K = (case["batch"], case["q_heads"], case["kv_heads"], case["q_len"], case["head_dim"], f.G,
                            case["top"])
    gq, NG = Hq // H, f.groups
    hot_k, hot_v, hot_t, ng = _hot(s)
    p = s.seq_lens.long()[:, None] - T + torch.arange(T, device="cuda")          # (B, T)
    # scores next to one another decide which group is chosen: 64 bits
    meta = s.slots.long()
    mid = s.gmean[meta].permute(0, 2, 3, 1).double().reshape(B * H, D, NG)
    half = s.gscale[meta].permute(0, 2, 3, 1).double().reshape(B * H, D, NG) * case["spread"]
    q = s.q.double().reshape(B * H, gq * T, D)
    score = (torch.bmm(q, mid.contiguous()) + torch.bmm(q.abs(), half.contiguous())).view(B, H, gq, T, NG).amax(2)
    g = torch.arange(NG, device="cuda")
    count = torch.minimum(ng[:, None], torch.div(p, G, rounding_mode="floor") + 1).clamp(min=0)[:, None, :, None]
    always = (g < case["first"]) | (g >= count - case["last"])
    score = torch.where(g < count, torch.where(always, math.inf, score), -math.inf)
    order = score.sort(dim=-1, descending=True, stable=True).indices[..., :K]
    pick = torch.where(order < count, order, NG).sort(-1).values
    if pick.shape[-1] < K:
        pick = torch.cat([pick, torch.full_like(pick[..., :1], NG).expand(B, H, T, K - pick.shape[-1])], -1)
    groups = torch.where(pick < NG, pick, -1)
    # attention over what was picked and the uncoded tokens, a query at a time
    live = groups >= 0
    bi = torch.arange(B, device="cuda")[:, None, None].expand(B, H, K)
    hi = torch.arange(H, device="cuda")[None, :, None].expand(B, H, K)
    out = torch.empty((B, Hq, T, D), dtype=torch.float16, device="cuda")
    for t in range(T):
        gt = torch.where(live[:, :, t], groups[:, :, t], 0)
        k, v = _dense(s, bi, hi, gt)
        k, v = k.reshape(B, H, K * G, D), v.reshape(B, H, K * G, D)
        pos = (gt[..., None] * G + torch.arange(G, device="cuda")).flatten(2)
        sees = live[:, :, t].repeat_interleave(G, -1) & (pos <= p[:, t, None, None])
        sees = torch.cat([sees, (hot_t <= p[:, t, None])[:, None].expand(B, H, f.W)], -1)
        k, v = torch.cat([k, hot_k], 2), torch.cat([v, hot_v], 2)
        score = torch.matmul(s.q[:, :, t].float().view(B, H, gq, D), k.transpose(2, 3).contiguous()) / math.sqrt(D)
        w = _softmax(torch.where(sees[:, :, None], score, -math.inf))
        out[:, :, t] = torch.matmul(w, v).view(B, Hq, D)
    return {"groups": groups.int(), "out": out}


def _whole(s, g0):
    """fp32 keys and values of every sequence's groups from ``g0`` on and of its
    ring, ``(B, H, n, D)``, their tokens ``(B, n)`` and whether they exist."""
    case, f = s.case, s.form
    B, H, D, G, NG = case["batch"], case["kv_heads"], case["head_dim"], f.G, f.groups - g0
    hot_k, hot_v, hot_t, ng = _hot(s)
    k = torch.empty((B, H, NG * G + f.W, D), device="cuda")
    v = torch.empty_like(k)
    hi, gi = torch.meshgrid(torch.arange(H, device="cuda"), g0 + torch.arange(NG, device="cuda"), indexing="ij")
    for b in range(B):
        kb, vb = _dense(s, torch.full_like(hi, b), hi, gi)
        k[b, :, :NG * G], v[b, :, :NG * G] = kb.reshape(H, NG * G, D), vb.reshape(H, NG * G, D)
    k[:, :, NG * G:], v[:, :, NG * G:] = hot_k, hot_v
    pos = g0 * G + torch.arange(NG * G, device="cuda")
    live = torch.cat([pos < (ng * G)[:, None], hot_t < s.seq_lens[:, None]], 1)
    return k, v, torch.cat([pos.expand(B, -1), hot_t], 1), live


def _plain_weigh(s):
    case, f = s.case, s.form
    B, Hq, H, T, D = case["batch"], case["q_heads"], case["kv_heads"], case["q_len"], case["head_dim"]
    k, v, pos, live = _whole(s, 0)
    p = (s.seq_lens.long()[:, None] - T + torch.arange(T, device="cuda"))[..., None]
    j, window = pos[:, None], case["window"] or 1 << 30
    sees = live[:, None] & (j <= p) & ((j > p - window) | (j < case["sinks"]))
    score = torch.matmul(s.q.float().view(B, H, -1, D), k.transpose(2, 3).contiguous()) / math.sqrt(D)
    score = torch.where(sees[:, None, None], score.view(B, H, Hq // H, T, -1), -math.inf)
    w = _softmax(score)
    out = torch.matmul(w.view(B, H, -1, k.shape[2]), v).view(B, Hq, T, D)
    got = w.sum((2, 3), dtype=torch.float64)[..., :f.groups * f.G].view(B, H, f.groups, f.G).sum(-1)
    return {"out": out.half(), "weights": got.float()}


def _plain_evict(s):
    case, f = s.case, s.form
    B, NG, keep = case["batch"], f.groups, case["keep"]
    length = s.seq_lens.long()
    ng = torch.where(length <= f.W, 0, torch.div(length - (f.W + 1), f.G, rounding_mode="floor") + 1)[:, None]
    g = torch.arange(NG, device="cuda")
    score = s.weights.double().sum(1)
    always = (g < case["first"]) | (g >= ng - case["last"])
    score = torch.where(g < ng, torch.where(always, math.inf, score), -math.inf)
    rank = torch.empty((B, NG), dtype=torch.long, device="cuda")
    rank.scatter_(1, score.sort(dim=-1, descending=True, stable=True).indices, g.expand(B, -1))
    stays = (g < ng) & (rank < keep)
    # what stays in order, then what leaves, then the places without a group
    order = torch.where(stays, 0, torch.where(g < ng, 1, 2)).sort(dim=-1, stable=True).indices
    n = stays.sum(-1, keepdim=True)
    kept = torch.where(g < n, order, -1)[:, :keep]
    if kept.shape[1] < keep:
        kept = torch.cat([kept, torch.full_like(kept[:, :1], -1).expand(B, keep - kept.shape[1])], 1)
    gone = (ng - n) * f.G
    pages = (order[..., None] * f.per_group + torch.arange(f.per_group, device="cuda")).flatten(1)
    weights = s.weights.gather(2, order[:, None].expand_as(s.weights)) * (g < n)[:, None]
    at = ((torch.arange(f.W, device="cuda") + gone) % f.W)[:, None, :, None].expand_as(s.hot_k)
    return {"kept": kept.int(), "groups": s.slots.gather(1, order), "pages": s.table.gather(1, pages),
            "lengths": (length - gone[:, 0]).int(), "weights": weights, "hot_k": s.hot_k.gather(2, at),
            "hot_v": s.hot_v.gather(2, at)}


def _plain_shared(s):
    case, f = s.case, s.form
    B, Hq, H, T, D, G = case["batch"], case["q_heads"], case["kv_heads"], case["q_len"], case["head_dim"], f.G
    gq = Hq // H
    k, v, pos, live = _whole(s, f.shared)
    p = (s.seq_lens.long()[:, None] - T + torch.arange(T, device="cuda"))[..., None]
    sees = live[:, None] & (pos[:, None] <= p)
    score = torch.matmul(s.q.float().view(B, H, gq * T, D), k.transpose(2, 3).contiguous()) / math.sqrt(D)
    score = torch.where(sees[:, None, None], score.view(B, H, gq, T, -1), -math.inf).view(B, H, gq * T, -1)
    if f.shared:  # the prefix once for all sequences
        hi, gi = torch.meshgrid(torch.arange(H, device="cuda"), torch.arange(f.shared, device="cuda"), indexing="ij")
        pk, pv = _dense(s, torch.zeros_like(hi), hi, gi)
        pk, pv = pk.reshape(H, -1, D), pv.reshape(H, -1, D)
        q = s.q.float().view(B, H, gq * T, D).transpose(0, 1).reshape(H, -1, D)
        first = torch.bmm(q, pk.transpose(1, 2).contiguous()) / math.sqrt(D)
        first = first.view(H, B, gq, T, -1)
        seen = torch.arange(f.shared * G, device="cuda") <= p
        first = torch.where(seen[:, None], first, -math.inf).view(H, B, gq * T, -1).transpose(0, 1)
        w = _softmax(torch.cat([first, score], -1))
        out = torch.matmul(w[..., f.shared * G:], v)
        w = w[..., :f.shared * G].transpose(0, 1).reshape(H, B * gq * T, -1)
        out = out + torch.bmm(w, pv).view(H, B, gq * T, D).transpose(0, 1)
    else:
        out = torch.matmul(_softmax(score), v)
    return {"out": out.reshape(B, Hq, T, D).half()}


def run(s):
    case, p = s.case, s.pool
    if not own:
        return {"choose": _plain_choose, "weigh": _plain_weigh, "evict": _plain_evict,
                "shared": _plain_shared}[case["kind"]](s)
    if case["kind"] == "choose":
        groups = p.select_groups(s.q, case["top"], first=case["first"], last=case["last"], spread=case["spread"])
        return {"groups": groups, "out": p.attend(s.q, groups=groups)}
    if case["kind"] == "weigh":
        weights = torch.zeros_like(s.weights)
        out = p.attend(s.q, window=case["window"] or None, sinks=case["sinks"], weights=weights)
        return {"out": out, "weights": weights}
    if case["kind"] == "shared":
        return {"out": p.attend(s.q)}
    # (an eviction changes the pool: it is put back as it was before each)
    p.lengths = list(s.lens)
    p.seq_lens.copy_(s.seq_lens)
    p.block_table.copy_(s.table)
    p.group_table.copy_(s.slots)
    p.hot_k.copy_(s.hot_k)
    p.hot_v.copy_(s.hot_v)
    weights = s.weights.clone()
    kept = p.evict(weights, case["keep"], first=case["first"], last=case["last"])
    return {"kept": kept, "groups": p.group_table, "pages": p.block_table, "lengths": p.seq_lens, "weights": weights,
            "hot_k": p.hot_k, "hot_v": p.hot_v}


# -------------------------------------------------------------------- work --
def work(case):
    f = _Form(case)
    D, H, Hq, T, G, W, B = (case["head_dim"], case["kv_heads"], case["q_heads"], case["q_len"], f.G, f.W,
                            case["batch"])
    group = H * (G * (D // 2 + D * case["value_bits"] // 8 + 4) + 8 * D + 4 * f.k_out * D)  # bytes of a coded group
    nbytes = flops = 0
    for n in _lengths(case):
        ng = _groups(n, W)
        hot = n - ng * G
        if case["kind"] == "evict":
            left = min(ng, case["keep"])
            nbytes += 2 * 4 * (H * f.groups + f.groups * (1 + f.per_group))
            nbytes += 2 * 2 * 2 * H * W * D if (ng - left) * G % W else 0
            flops += H * ng
            continue
        nbytes += 2 * Hq * T * D * 2
        if case["kind"] == "choose":
            some = min(ng, case["top"])
            nbytes += H * ng * 8 * D + some * group + H * hot * 2 * D * 2
            flops += 4 * T * Hq * D * (ng + some * G + hot)
        elif case["kind"] == "weigh":
            p = np.arange(n - T, n)
            low = np.maximum(p - (case["window"] or 1 << 30) + 1, 0)
            first = np.minimum(case["sinks"], low)
            tokens = int(n - low[0] + min(case["sinks"], int(low[0])))
            hot = min(hot, tokens)
            nbytes += (tokens - hot) * group // G + H * hot * 2 * D * 2 + 8 * H * f.groups
            flops += 4 * Hq * D * int((p + 1 - low + first).sum())
        else:
            nbytes += (ng - f.shared) * group + H * hot * 2 * D * 2
            flops += 4 * T * Hq * D * n
    return {"bytes": nbytes + f.shared * group, "flops": flops}


# ------------------------------------------------------------------- exact --
def _unpacked(c, f, case, seed, b, groups, heads=slice(None)):
    """64-bit keys and values ``(H, n, G, D)`` of some groups of a sequence."""
    D = case["head_dim"]
    level = torch.tensor(NF4, dtype=torch.float32, device="cuda").double()
    cent = (torch.tensor(LLOYD_MAX[case["value_bits"]], dtype=torch.float64) / math.sqrt(D)).float().double().cuda()
    pi = torch.from_numpy(_rotation(seed, D)).cuda().double()

    def take(name):
        return c[name][b][groups][:, heads].transpose(0, 1)

    k = take("mean")[:, :, None].double() + take("scale")[:, :, None].double() * level[take("kcode").int()]
    if f.k_out:
        k = k.flatten(2).scatter(2, take("at"), take("val").double()).view(k.shape)
    return k, cent[take("vcode").int()] @ pi * take("vnorm").double()[..., None]


def _attend_rows(q, k, v, hidden):
    """A kv head in 64 bits: the weights and the result of ``q (r, D)`` over ``k, v (n, D)``."""
    a = (q.double() @ k.T) * q.shape[-1] ** -0.5
    a = a.masked_fill(hidden, -math.inf)
    none = hidden.all(-1)
    a[none] = 0.0
    w = torch.softmax(a, -1)
    w[none] = 0.0
    return w, w @ v


def exact(case, seed):
    c, f = _coded(case, seed), _Form(case)
    B, Hq, H, T, D, G, W, NG = (case["batch"], case["q_heads"], case["kv_heads"], case["q_len"], case["head_dim"],
                                f.G, f.W, f.groups)
    gq = Hq // H
    if case["kind"] == "evict":
        got = {x: [] for x in ("kept", "groups", "pages", "lengths", "weights", "hot_k", "hot_v")}
        for b, n in enumerate(c["lens"]):
            ng = _groups(n, W)
            total = [math.fsum(x) for x in c["weights"][b].T.double().cpu().tolist()]
            stays = set(range(min(case["first"], ng))) | set(range(max(0, ng - case["last"]), ng))
            rest = sorted((g for g in range(ng) if g not in stays), key=lambda g: (-total[g], g))
            forced = sorted(stays)[:case["keep"]]
            stays = sorted(forced + rest[:max(0, case["keep"] - len(forced))]) if ng > case["keep"] else list(range(ng))
            order = stays + [g for g in range(ng) if g not in set(stays)] + list(range(ng, NG))
            at = torch.tensor(order, device="cuda")
            gone = (ng - len(stays)) * G
            got["kept"].append(torch.tensor(stays + [-1] * (case["keep"] - len(stays)), device="cuda"))
            got["groups"].append(b * NG + at)
            got["pages"].append(c["table"][b].view(NG, f.per_group)[at].flatten())
            got["lengths"].append(torch.tensor(n - gone, device="cuda"))
            w = c["weights"][b][:, at].double()
            w[:, len(stays):] = 0.0
            got["weights"].append(w)
            for x in ("hot_k", "hot_v"):
                got[x].append(torch.roll(c[x][b], -(gone % W), 1).double())
        return {x: torch.stack(y) for x, y in got.items()}
    out = torch.zeros((B, Hq, T, D), dtype=torch.float64, device="cuda")
    groups = torch.full((B, H, T, case.get("top", 1)), -1, dtype=torch.long, device="cuda")
    weights = torch.zeros((B, H, NG), dtype=torch.float64, device="cuda")
    for b, n in enumerate(c["lens"]):
        ng = _groups(n, W)
        hot = torch.arange(ng * G, n, device="cuda")
        hk, hv = c["hot_k"][b][:, hot % W].double(), c["hot_v"][b][:, hot % W].double()
        p = n - T + torch.arange(T, device="cuda")
        if case["kind"] == "choose":
            for h in range(H):
                mid, half = c["mean"][b, :ng, h].double(), c["scale"][b, :ng, h].double()
                q = c["q"][b, h * gq:(h + 1) * gq].double()
                for t in range(T):
                    count = min(ng, (n - T + t) // G + 1)
                    s = ((q[:, t, None] * mid).sum(-1) + case["spread"] * (q[:, t, None].abs() * half).sum(-1)).amax(0)
                    s = s[:count].tolist()
                    pick = [g for g in range(count) if g < case["first"] or g >= count - case["last"]][:case["top"]]
                    rest = sorted((g for g in range(count) if g not in set(pick)), key=lambda g: (-s[g], g))
                    pick = sorted(pick + rest[:case["top"] - len(pick)])
                    groups[b, h, t, :len(pick)] = torch.tensor(pick, dtype=torch.long, device="cuda")
                    k, v = _unpacked(c, f, case, seed, b, pick, slice(h, h + 1))
                    pos = torch.cat([torch.arange(g * G, (g + 1) * G, device="cuda") for g in pick] + [hot])
                    k = torch.cat([k.reshape(-1, D), hk[h]])
                    v = torch.cat([v.reshape(-1, D), hv[h]])
                    out[b, h * gq:(h + 1) * gq, t] = _attend_rows(q[:, t], k, v, (pos > n - T + t).expand(gq, -1))[1]
            continue
        k, v = _unpacked(c, f, case, seed, b, slice(0, ng))
        pos = torch.arange(n, device="cuda")
        hidden = pos > p[:, None]
        if case["kind"] == "weigh":
            window = case["window"] or 1 << 40
            hidden = hidden | ((p[:, None] - pos >= window) & (pos >= case["sinks"]))
        for h in range(H):
            for i in range(h * gq, (h + 1) * gq):
                w, o = _attend_rows(c["q"][b, i], torch.cat([k[h].reshape(-1, D), hk[h]]),
                                    torch.cat([v[h].reshape(-1, D), hv[h]]), hidden)
                out[b, i] = o
                weights[b, h, :ng] += w[:, :ng * G].sum(0).view(ng, G).sum(-1)
    if case["kind"] == "choose":
        return {"groups": groups, "out": out}
    return {"out": out, "weights": weights} if case["kind"] == "weigh" else {"out": out}
