"""Masks that look like a sliding window's and are not (no GPU needed)."""

import pytest

torch = pytest.importorskip("torch")
pytest.importorskip("transformers")

from test_hf_window_cpu import window_mask  # noqa: E402


def test_a_finite_bias_is_no_window():
    """Zeros inside the window and a finite bias outside it: those keys still count."""
    from turboquant_pro_amd.hf_cache import _mask_is_window
    m = window_mask(4, 9, 3)
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        for hidden in (-1.0, -1e-3, -10000.0, 1.0, float("inf"), float("nan")):
            assert not _mask_is_window(torch.where(m, 0.0, hidden).to(dtype), 9, 3), (dtype, hidden)
        for hidden in (float("-inf"), torch.finfo(dtype).min):
            assert _mask_is_window(torch.where(m, 0.0, hidden).to(dtype), 9, 3), (dtype, hidden)
            one = torch.where(m, 0.0, hidden).to(dtype)
            one[0, 0, 1, 8] = -2.0
            assert not _mask_is_window(one, 9, 3)
    # the lowest value of the model's type in a mask of another
    assert _mask_is_window(torch.where(m, 0.0, torch.finfo(torch.bfloat16).min).float(), 9, 3)
    assert not _mask_is_window(torch.where(m, 0, -1), 9, 3)
