"""window_attention over keys and values that end where their memory ends: last tiles
of one row and of one row less than whole, tokens far apart."""

import pytest

torch = pytest.importorskip("torch")

from test_gpu_window_attention import check, inputs  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU visible")


@pytest.mark.parametrize("D,dtype", [(64, torch.float16), (128, torch.bfloat16), (256, torch.float16)])
@pytest.mark.parametrize("L", [1, 31, 65, 127, 129])
@pytest.mark.parametrize("T", [1, 40])
def test_the_last_tile_ends_with_the_memory(D, dtype, L, T):
    from turboquant_pro_amd import window_attention
    print(f"[window] tail D={D} L={L} T={T} {dtype}", flush=True)
    T = min(T, L)
    q, k, v = inputs(L, 1, 4, 2, D, T, L, dtype)
    # (token, head) rows of a buffer of their own, 512 rows a token, at its end
    wide = [torch.full((L, 512, D), float("nan"), dtype=dtype, device="cuda") for _ in range(2)]
    for w, x in zip(wide, (k, v)):
        w[:, -2:] = x[0].transpose(0, 1)
    ks, vs = (w[:, -2:].transpose(0, 1)[None] for w in wide)
    for window in (None, 20):
        out = window_attention(q, ks, vs, window=window)
        check(out, q, k, v, window, 0, what=f"window={window}")
        assert torch.equal(out, window_attention(q, k, v, window=window))
