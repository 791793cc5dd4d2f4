"""The operators around the cache where offsets pass 32 bits and where one sequence is
very long."""

import math

import pytest

torch = pytest.importorskip("torch")

from attn_ref import attention, attention_bound, visible  # noqa: E402
from test_gpu_attend import make_pool, queries  # noqa: E402
from test_gpu_attend_large import check, is_dense  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU visible")


@pytest.mark.parametrize("T,window", [(1, None), (70, 3000)])
def test_keys_past_32_bits(T, window):
    """Keys and values of 2^31 elements and more: the last head's, the last tokens'."""
    from turboquant_pro_amd import window_attention
    print(f"[long] window T={T}", flush=True)
    L, H, D = 2200000, 8, 128
    gen = torch.Generator(device="cuda").manual_seed(1)
    k = torch.empty((1, L, H, D), dtype=torch.float16, device="cuda")
    k.normal_(generator=gen)
    v = torch.empty_like(k).normal_(generator=gen)
    q = torch.randn((1, H, T, D), generator=gen, device="cuda").half()
    assert k.numel() > 1 << 31
    for kk, vv in ((k.transpose(1, 2), v.transpose(1, 2)), (k.view(1, H, L, D), v.view(1, H, L, D))):
        out = window_attention(q, kk, vv, window=window, sinks=3)
        h = H - 1
        if window is None:  # (one query: every key)
            kh, vh, sees = kk[0, h:], vv[0, h:], torch.ones((1, L), dtype=torch.bool, device="cuda")
        else:  # the first tokens, and those that the window reaches
            at = torch.cat([torch.arange(3), torch.arange(L - T - window, L)]).cuda()
            kh, vh = kk[0, h:][:, at], vv[0, h:][:, at]
            p = (L - T + torch.arange(T, device="cuda"))[:, None]
            sees = (at <= p) & ((at > p - window) | (at < 3))
        want, weighted, mag, vmax = attention(q[0, h:], kh, vh, sees, 1.0 / math.sqrt(D))
        tol = attention_bound(q.dtype, want, weighted, mag, vmax, kh.shape[1], D, 1.0 / math.sqrt(D))
        assert bool(((out[0, h:].double() - want).abs() <= tol).all())


@pytest.mark.parametrize("D,form", [(128, dict()), (64, dict(value_bits=4)), (256, dict(key_grid="uniform", key_bits=3))])
def test_codes_past_32_bits(D, form):
    """The last sequence of a pool whose codes and side-lists pass 4 GiB."""
    print(f"[long] codes D={D}", flush=True)
    from turboquant_pro_amd import TQKVPool
    B, H, L = 16, 8, 700000 * 128 // D
    pool = TQKVPool(n_kv_heads=H, n_q_heads=2 * H, head_dim=D, max_batch=B, max_seq_len=L, seed=2, **form)
    assert pool.kcodes.numel() > (1 << 32) or pool.key_bits < 4
    assert pool.oent.numel() * 4 > 1 << 31
    gen = torch.Generator(device="cuda").manual_seed(3)
    lens = [0] * (B - 2) + [40, 2600]
    k, v = (torch.randn((B, H, 2600, D), generator=gen, device="cuda").half() for _ in range(2))
    pool.append(k, v, n_new=lens)
    for T in (1, 5, 65):
        q = queries(T, pool, T)
        for window, sinks in ((None, 0), (900, 5)):
            check(pool, pool.attend(q, window=window, sinks=sinks), q, window, sinks, 1.0 / math.sqrt(D), what=f"T={T}")


def test_rows_past_32_bits():
    """norm_rope over 2^31 elements and more: the last tokens as in a call of their own."""
    from turboquant_pro_amd import norm_rope
    print("[long] rope", flush=True)
    Hq, H, D, T = 8, 2, 128, 1450000
    rows = torch.empty((1, T, (Hq + 2 * H) * D), dtype=torch.float16, device="cuda")
    rows.normal_(generator=torch.Generator(device="cuda").manual_seed(4))
    assert rows.numel() > 1 << 31
    inv = (10000.0 ** (-torch.arange(64, dtype=torch.float64) / 64)).float().cuda()
    w = torch.linspace(0.5, 1.5, D, device="cuda")
    out = norm_rope(rows, Hq, H, inv, torch.tensor([7], device="cuda"), q_weight=w, k_weight=w)
    last = norm_rope(rows[:, -50:], Hq, H, inv, torch.tensor([7 + T - 50], device="cuda"), q_weight=w, k_weight=w)
    for a, b in zip(out, last):
        assert torch.equal(a[:, :, -50:], b)


def test_a_head_too_long_to_reconstruct():
    """More tokens than a GiB of reconstructed keys and values holds: the codes are
    attended by a chunk too."""
    print("[long] head", flush=True)
    n, T = 1500000, 65
    pool = make_pool(5, [n], 2, 1)
    assert is_dense(pool, T) and 6 * 128 * n > 1 << 30
    q = queries(5, pool, T)
    out = pool.attend(q)
    # the last queries alone stand where they stood in the chunk
    last = pool.attend(q[:, :, -5:].contiguous())
    # (both on the codes; their splits differ, so the order of fp32 sums does)
    assert float((last - out[:, :, -5:]).abs().max()) <= 2.0 ** -10 * float(out.abs().max())
    ks, vs = [], []
    for g0 in range(0, pool.n_groups(0), 500):
        k, v = pool.dequant_groups([(0, g) for g in range(g0, min(g0 + 500, pool.n_groups(0)))])
        ks.append(k[:, 0].reshape(-1, 128))
        vs.append(v[:, 0].reshape(-1, 128))
    hk, hv = pool.hot_window_tokens(0)
    k, v = (torch.cat(x + [y[0].float()]).double()[None] for x, y in ((ks, hk), (vs, hv)))
    for i in (0, 1, 33, 64):
        sees = visible(n, T, T, 0, None, 0, "cuda")[i:i + 1]
        want = attention(q[0, :, i:i + 1], k, v, sees, 128 ** -0.5)[0]
        err = (out[0, :, i:i + 1].double() - want)
        # random roundings of half a step of fp16 each: together 2^-10 of the output
        assert float(err.norm()) <= 2.0 ** -10 * float(want.norm())
