"""norm_rope against its formula in 64 bits: types, head layouts, rotary widths,
pair orders, far positions, one token to long ones, strides and alignment."""

import pytest

torch = pytest.importorskip("torch")

from attn_ref import HALF  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU visible")


def formula(qkv, Hq, Hkv, inv, pos, qw, kw, eps, off, interleaved, scale):
    """q, k, v in 64 bits, and each value's pair magnitude."""
    B, T, C = qkv.shape
    D = C // (Hq + 2 * Hkv)
    R = 2 * inv.shape[0]
    p = pos.double() if pos.dim() == 2 else pos.double()[:, None] + torch.arange(T, dtype=torch.float64, device=pos.device)
    ang = p[..., None] * inv.double()
    cos, sin = (ang.cos() * scale)[:, None], (ang.sin() * scale)[:, None]
    x = qkv.double().view(B, T, Hq + 2 * Hkv, D).transpose(1, 2)
    out, size = [], []
    for part, w in ((x[:, :Hq], qw), (x[:, Hq:Hq + Hkv], kw), (x[:, Hq + Hkv:], "v")):
        if isinstance(w, str):
            out.append(part)
            size.append(part.abs())
            continue
        if w is not None:
            part = part / (part.square().mean(-1, keepdim=True) + eps).sqrt() * (w.double() + off)
        y, m = part.clone(), part.abs().clone()
        a = part[..., 0:R:2] if interleaved else part[..., :R // 2]
        b = part[..., 1:R:2] if interleaved else part[..., R // 2:R]
        ra, rb, h = a * cos - b * sin, b * cos + a * sin, (a.abs() + b.abs()) * scale
        if interleaved:
            y[..., 0:R:2], y[..., 1:R:2], m[..., 0:R:2], m[..., 1:R:2] = ra, rb, h, h
        else:
            y[..., :R // 2], y[..., R // 2:R], m[..., :R // 2], m[..., R // 2:R] = ra, rb, h, h
        out.append(y)
        size.append(m)
    return out, size


def check(got, want, size, dtype, D, what=""):
    # fp32 on the way: the mean of D squares in D / 8 + 5 steps of 2^-24 (its root
    # halves them), root, quotient, three products and the fused sum; the angle's
    # fraction (pi 2^-24) and the sine's two last places
    calc = ((D / 8 + 5) / 2 + 12) * 2.0 ** -24
    for name, g, w, m in zip("qkv", got, want, size):
        tol = HALF[dtype] * w.abs() + calc * (1 + 2.0 ** -8) * m + 2.0 ** -25
        err = (g.double() - w).abs()
        assert g.dtype == dtype and bool((err <= tol).all()), f"{what} {name}: {float((err - tol).max()):.3e} past the bound"


@pytest.mark.parametrize("D,R,Hq,Hkv,B,T,dtype,out,norm,off,inter", [
    (128, 128, 32, 8, 16, 1, torch.bfloat16, torch.float16, True, 0.0, False),
    (128, 128, 32, 8, 1, 1, torch.float16, None, True, 0.0, False),
    (128, 64, 28, 4, 2, 37, torch.bfloat16, None, True, 1.0, False),
    (128, 32, 7, 1, 3, 5, torch.float32, torch.float16, False, 0.0, True),
    (64, 64, 4, 4, 2, 129, torch.float16, torch.float32, True, 0.0, False),
    (64, 32, 3, 1, 1, 70, torch.float32, None, True, 1.0, True),
    (64, 16, 8, 8, 1, 3, torch.bfloat16, torch.bfloat16, True, 0.0, False),
    (256, 256, 16, 8, 2, 33, torch.bfloat16, torch.float16, True, 1.0, False),
    (256, 128, 2, 1, 5, 9, torch.float32, torch.bfloat16, True, 0.0, True),
    (256, 0, 1, 1, 1, 1, torch.float16, None, True, 0.0, False),
    (128, 128, 8, 0, 2, 3, torch.float16, None, True, 0.0, False),
    (128, 128, 0, 8, 2, 3, torch.float16, None, True, 0.0, False),
    (128, 128, 32, 8, 2, 2500, torch.bfloat16, torch.float16, True, 0.0, False),
])
def test_norm_rope_against_the_formula(D, R, Hq, Hkv, B, T, dtype, out, norm, off, inter):
    from turboquant_pro_amd import norm_rope
    print(f"[rope] D={D} R={R} {Hq}/{Hkv} B={B} T={T} {dtype} -> {out}", flush=True)
    gen = torch.Generator(device="cuda").manual_seed(D + R + T)
    qkv = (3.0 * torch.randn((B, T, (Hq + 2 * Hkv) * D), generator=gen, device="cuda")).to(dtype)
    qw = (torch.randn(D, generator=gen, device="cuda") * 0.3 + 1.0 - off).to(dtype) if norm else None
    kw = (torch.randn(D, generator=gen, device="cuda") * 0.3 + 1.0 - off).float() if norm else None
    inv = (10000.0 ** (-torch.arange(R // 2, dtype=torch.float64) / max(R // 2, 1))).float().cuda()
    for pos in (torch.randint(0, 1 << 20, (B,), generator=gen, device="cuda", dtype=torch.int32),
                torch.randint(0, 1 << 20, (B, T), generator=gen, device="cuda"),
                torch.zeros((B,), dtype=torch.int64, device="cuda")):
        got = norm_rope(qkv, Hq, Hkv, inv, pos, q_weight=qw, k_weight=kw, eps=1e-5, weight_offset=off, interleaved=inter,
                        rope_scale=1.25, dtype=out)
        assert [tuple(x.shape) for x in got] == [(B, Hq, T, D), (B, Hkv, T, D), (B, Hkv, T, D)]
        want, size = formula(qkv, Hq, Hkv, inv, pos, qw, kw, 1e-5, off, inter, 1.25)
        check(got, want, size, out or dtype, D)


def test_norm_rope_strided_misaligned_and_one_sided():
    from turboquant_pro_amd import norm_rope
    print("[rope] strides", flush=True)
    D, Hq, Hkv, B, T = 128, 4, 2, 3, 6
    C = (Hq + 2 * Hkv) * D
    gen = torch.Generator(device="cuda").manual_seed(3)
    wide = torch.randn((T, B, C + 40), generator=gen, device="cuda").half()
    inv = (10000.0 ** (-torch.arange(64, dtype=torch.float64) / 64)).float().cuda()
    pos = torch.tensor([0, 77, 131071], dtype=torch.int32, device="cuda")
    w = torch.rand(D + 1, generator=gen, device="cuda").half()[1:]  # two bytes off an aligned start
    for x in (wide.transpose(0, 1)[..., 8:C + 8],      # sequences inside, a 16-byte start
              wide.transpose(0, 1)[..., 3:C + 3],      # no 16-byte start
              wide.transpose(0, 1)[..., :C].contiguous().expand(B, T, C)):
        got = norm_rope(x, Hq, Hkv, inv, pos, q_weight=w)
        want, size = formula(x, Hq, Hkv, inv, pos, w, None, 1e-6, 0.0, False, 1.0)
        check(got, want, size, torch.float16, D, "strided")
    # nothing to do
    q, k, v = norm_rope(wide.transpose(0, 1)[:0, :, :C], Hq, Hkv, inv, pos[:0])
    assert q.numel() == k.numel() == v.numel() == 0
    q, k, v = norm_rope(wide[:0, :, :C].transpose(0, 1), Hq, Hkv, inv, pos)
    assert tuple(q.shape) == (B, Hq, 0, D)


def test_norm_rope_non_finite_rows_stay_their_own():
    """An infinity or a NaN reaches the head that holds it and no other."""
    from turboquant_pro_amd import norm_rope
    print("[rope] non-finite", flush=True)
    D, Hq, Hkv, B, T = 128, 8, 2, 2, 5
    x = torch.randn((B, T, (Hq + 2 * Hkv) * D), device="cuda").half()
    inv = (10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32)).float().cuda()
    pos = torch.tensor([5, 9], dtype=torch.int32, device="cuda")
    w = torch.ones(D, device="cuda").half()
    clean = norm_rope(x, Hq, Hkv, inv, pos, q_weight=w, k_weight=w)
    y = x.clone()
    y[0, 2, 3 * D + 5] = float("nan")               # query head 3
    y[1, 4, (Hq + 1) * D + 100] = float("inf")      # key head 1
    y[1, 0, (Hq + Hkv) * D + 7] = float("-inf")     # value head 0
    got = norm_rope(y, Hq, Hkv, inv, pos, q_weight=w, k_weight=w)
    for g, c, (b, h, t) in zip(got, clean, ((0, 3, 2), (1, 1, 4), (1, 0, 0))):
        keep = torch.ones(g.shape[:3], dtype=torch.bool, device="cuda")
        keep[b, h, t] = False
        assert torch.equal(g[keep], c[keep])
        assert not torch.isfinite(g[b, h, t]).all()
    assert torch.isnan(got[0][0, 3, 2]).all()
    assert got[2][1, 0, 0, 7] == float("-inf") and torch.isfinite(got[2][1, 0, 0]).sum() == D - 1


def test_norm_rope_on_another_stream_and_in_a_graph():
    from turboquant_pro_amd import norm_rope
    print("[rope] stream, graph", flush=True)
    D, Hq, Hkv, B, T = 128, 32, 8, 4, 1
    x = torch.randn((B, T, (Hq + 2 * Hkv) * D), device="cuda").half()
    inv = (10000.0 ** (-torch.arange(64, dtype=torch.float64) / 64)).float().cuda()
    pos = torch.tensor([5, 9, 0, 1000], dtype=torch.int32, device="cuda")
    want = [y.clone() for y in norm_rope(x, Hq, Hkv, inv, pos)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = norm_rope(x, Hq, Hkv, inv, pos)
    side.synchronize()
    assert all(torch.equal(g, w) for g, w in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = norm_rope(x, Hq, Hkv, inv, pos)
    for step in range(4):
        pos.add_(step)
        x.mul_(-1.0)
        graph.replay()
        torch.cuda.synchronize()
        eager = norm_rope(x, Hq, Hkv, inv, pos)
        assert all(torch.equal(g, w) for g, w in zip(out, eager)), step
