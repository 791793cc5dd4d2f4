"""Sliding-window layers of a HuggingFace model on the GPU: decode steps over the
codes of the window's tokens, prefills and chunks through window_attention, and
everything else through SDPA as before."""

import pytest

torch = pytest.importorskip("torch")
pytest.importorskip("transformers")

from attn_ref import HALF, attention  # noqa: E402
from test_hf_window_cpu import window_mask  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU visible")


def rows(gen, *shape, dtype=torch.float16):
    return torch.randn(shape, generator=gen, device="cuda").to(dtype)


def counted(monkeypatch):
    """Counts the calls of the kernels' entry points."""
    from turboquant_pro_amd import TQKVPool
    from turboquant_pro_amd import hf_cache as HC
    calls = {"attend": 0, "decode": 0, "window": 0}

    def wrap(key, real):
        def f(*a, **kw):
            calls[key] += 1
            return real(*a, **kw)
        return f

    monkeypatch.setattr(TQKVPool, "attend", wrap("attend", TQKVPool.attend))
    monkeypatch.setattr(TQKVPool, "decode", wrap("decode", TQKVPool.decode))
    monkeypatch.setattr(HC, "window_attention", wrap("window", HC.window_attention))
    return calls


@pytest.mark.parametrize("D,Hq,H,dtype", [(128, 8, 2, "float16"), (128, 4, 4, "bfloat16"), (256, 4, 1, "float16"),
                                          (64, 8, 2, "float16")])
def test_windowed_layer(D, Hq, H, dtype, monkeypatch):
    from turboquant_pro_amd.hf_cache import TurboQuantLayer, tqk_attention
    print(f"[hf window] D={D} {Hq}/{H} {dtype}", flush=True)
    calls = counted(monkeypatch)
    dt, B, L, window, scaling = getattr(torch, dtype), 2, 900, 300, 0.8 * D ** -0.5
    gen = torch.Generator(device="cuda").manual_seed(7)
    layer = TurboQuantLayer(hot_window=128, value_bits=4, n_q_heads=Hq, max_cache_len=2048, fused_decode=True)
    module = torch.nn.Module()
    module.num_key_value_groups = Hq // H

    def close(out, q, k, v, mask, what):
        """Within half a step of the type for the scores' keys and queries, the
        weights, the values and the output, as the kernels' own tests have it."""
        half = HALF[dt] + (HALF[torch.float16] if dt == torch.bfloat16 else 0.0)
        assert out.dtype == dt and out.is_contiguous()
        for b in range(B):
            sees = mask[b, 0]
            want, weighted, mag, vmax = attention(q[b], k[b].double(), v[b].double(), sees, scaling)
            size = attention(q[b], k[b].double(), v[b].double().norm(dim=-1, keepdim=True).expand_as(v[b]).contiguous(),
                             sees, scaling)[0]
            tol = 2 * half * want.abs() + (4 * scaling * mag * half + 2 * half) * size + 4 * half * weighted + 2.0 ** -24
            err = (out[b].transpose(0, 1).double() - want).abs()
            assert bool((err <= tol).all()), f"{what}: {float((err - tol).max()):.2e} past the bound"

    for T in (L, 70, 1, 1):  # a prefill, a chunk, two steps
        q, k, v = (rows(gen, B, h, T, D, dtype=dt) for h in (Hq, H, H))
        kk, vv = layer.update(k, v)
        n = layer.get_seq_length()
        mask = window_mask(T, n, window, B).cuda()
        before = dict(calls)
        out, _ = tqk_attention(module, q, kk, vv, mask, scaling=scaling, sliding_window=window)
        assert calls["attend"] - before["attend"] == (T == 1) and calls["window"] - before["window"] == (T > 1)
        assert out.shape == (B, T, Hq, D)
        dk, dv = layer.dense(torch.float32)
        if T > 1:
            dk, dv = dk.to(dt), dv.to(dt)
        close(out, q, dk, dv, mask, f"T={T}")
        # a padded batch, no window named, soft-capped scores: SDPA on the dense cache
        before = dict(calls)
        padded = mask.clone()
        padded[1, :, :, :n - 50] = False
        for m, kw in ((padded, dict(sliding_window=window)), (mask, {}),
                      (mask, dict(sliding_window=window, softcap=30.0)) if T > 1 else (mask, {})):
            out, _ = tqk_attention(module, q, kk, vv, m, scaling=scaling, **kw)
            xk, xv = layer.dense()
            want = torch.nn.functional.scaled_dot_product_attention(
                q, xk.repeat_interleave(Hq // H, 1), xv.repeat_interleave(Hq // H, 1), attn_mask=m, scale=scaling)
            live = m.any(-1)[:, 0, :, None, None]
            assert float(torch.where(live, (out - want.transpose(1, 2)).abs(), 0.0).max()) <= 2.0 ** -5
        assert calls["attend"] == before["attend"] and calls["window"] == before["window"]
    # a window that reaches over the whole cache: the mask lets everything through
    before = dict(calls)
    q, k, v = (rows(gen, B, h, 1, D, dtype=dt) for h in (Hq, H, H))
    kk, vv = layer.update(k, v)
    n = layer.get_seq_length()
    tqk_attention(module, q, kk, vv, window_mask(1, n, 5000, B).cuda(), scaling=scaling, sliding_window=5000)
    assert calls["decode"] == before["decode"] + 1


def test_gradients_stay_with_sdpa(monkeypatch):
    from turboquant_pro_amd.hf_cache import tqk_attention
    print("[hf window] gradients", flush=True)
    calls = counted(monkeypatch)
    gen = torch.Generator(device="cuda").manual_seed(8)
    q, k, v = (rows(gen, 1, 2, 40, 64).requires_grad_() for _ in range(3))
    out, _ = tqk_attention(torch.nn.Module(), q, k, v, window_mask(40, 40, 9).cuda(), scaling=0.125, sliding_window=9)
    out.float().sum().backward()
    assert calls["window"] == 0 and all(x.grad is not None and bool(torch.isfinite(x.grad).all()) for x in (q, k, v))
