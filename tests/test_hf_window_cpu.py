"""The HuggingFace attention function's sliding-window masks: which ones are a
window's, and that CPU tensors, gradients and other masks stay with SDPA."""

import pytest

torch = pytest.importorskip("torch")
pytest.importorskip("transformers")


def window_mask(T, L, window, B=1):
    at, p = torch.arange(L), torch.arange(L - T, L)[:, None]
    return ((at <= p) & (at > p - window)).expand(B, 1, T, L).clone()


def test_mask_is_window():
    from turboquant_pro_amd.hf_cache import _mask_is_window
    for T, L, window in ((1, 9, 3), (4, 9, 3), (9, 9, 3), (9, 9, 1), (5, 9, 20), (1, 1, 1)):
        m = window_mask(T, L, window, 2)
        assert _mask_is_window(m, L, window)
        assert _mask_is_window(torch.where(m, 0.0, float("-inf")), L, window)
        assert not _mask_is_window(m, L + 1, window)
        assert not _mask_is_window(m[:, 0], L, window)
        if 1 < window < L:
            assert not _mask_is_window(m, L, window - 1)
        m[1, 0, -1, -1] = False  # a padded sequence's
        assert not _mask_is_window(m, L, window)
    assert not _mask_is_window(None, 9, 3)


def test_cpu_tensors_run_sdpa():
    from turboquant_pro_amd.hf_cache import tqk_attention
    gen = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(1, 2, 7, 64, generator=gen) for _ in range(3))
    m = window_mask(7, 7, 3)
    out, _ = tqk_attention(torch.nn.Module(), q, k, v, m, scaling=0.125, sliding_window=3)
    want = torch.nn.functional.scaled_dot_product_attention(q, k, v, attn_mask=m, scale=0.125)
    assert torch.equal(out, want.transpose(1, 2).contiguous())
