"""Calls of the HuggingFace attention function with a window's mask that the kernels do
not take: they run SDPA, as without a window."""

import pytest

torch = pytest.importorskip("torch")
pytest.importorskip("transformers")

from test_gpu_hf_window import counted, rows  # noqa: E402
from test_hf_window_cpu import window_mask  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU visible")


def module(groups=1):
    m = torch.nn.Module()
    m.num_key_value_groups = groups
    return m


def sdpa(q, k, v, mask, scale):
    g = q.shape[1] // k.shape[1]
    return torch.nn.functional.scaled_dot_product_attention(
        q, k.repeat_interleave(g, 1), v.repeat_interleave(g, 1), attn_mask=mask, scale=scale).transpose(1, 2)


@pytest.mark.parametrize("scaling,dv", [(0.0, 64), (-0.125, 64), (0.125, 128)])
@torch.no_grad()
def test_scales_and_value_widths_stay_with_sdpa(scaling, dv, monkeypatch):
    """A scale that is not positive, values of another width than the keys'."""
    from turboquant_pro_amd.hf_cache import tqk_attention
    print(f"[hf window] scaling={scaling} dv={dv}", flush=True)
    calls = counted(monkeypatch)
    gen = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = rows(gen, 2, 4, 900, 64), rows(gen, 2, 2, 900, 64), rows(gen, 2, 2, 900, dv)
    mask = window_mask(900, 900, 90, 2).cuda()
    out, _ = tqk_attention(module(2), q, k, v, mask, scaling=scaling, sliding_window=90)
    assert calls["window"] == 0 and calls["attend"] == 0
    # (two calls of one library: the same up to the order of its sums)
    assert float((out - sdpa(q, k, v, mask, scaling)).abs().max()) <= 2.0 ** -9


@pytest.mark.parametrize("scaling", [0.0, -0.125])
@torch.no_grad()
def test_scales_of_a_coded_layer_stay_with_sdpa(scaling, monkeypatch):
    from turboquant_pro_amd.hf_cache import TurboQuantLayer, tqk_attention
    print(f"[hf window] layer scaling={scaling}", flush=True)
    calls = counted(monkeypatch)
    gen = torch.Generator(device="cuda").manual_seed(4)
    layer = TurboQuantLayer(hot_window=64, value_bits=4, n_q_heads=4, max_cache_len=512, fused_decode=True)
    layer.update(rows(gen, 2, 2, 200, 64), rows(gen, 2, 2, 200, 64))
    q = rows(gen, 2, 4, 1, 64)
    kk, vv = layer.update(rows(gen, 2, 2, 1, 64), rows(gen, 2, 2, 1, 64))
    mask = window_mask(1, 201, 50, 2).cuda()
    out, _ = tqk_attention(module(2), q, kk, vv, mask, scaling=scaling, sliding_window=50)
    assert calls["attend"] == 0
    k, v = layer.dense()
    assert float((out - sdpa(q, k, v, mask, scaling)).abs().max()) <= 2.0 ** -9


@torch.no_grad()
def test_a_captured_prefill_stays_with_sdpa(monkeypatch):
    """The mask is read on the host, which a capture cannot wait for."""
    from turboquant_pro_amd.hf_cache import tqk_attention
    print("[hf window] capture", flush=True)
    calls = counted(monkeypatch)
    gen = torch.Generator(device="cuda").manual_seed(5)
    q, k, v = (rows(gen, 1, 2, 900, 64) for _ in range(3))
    mask = window_mask(900, 900, 90).cuda()
    want, _ = tqk_attention(module(), q, k, v, mask, scaling=0.125, sliding_window=90)
    assert calls["window"] == 1
    sdpa(q, k, v, mask, 0.125)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _ = tqk_attention(module(), q, k, v, mask, scaling=0.125, sliding_window=90)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        # (both round a value of at most 4 to fp16, weights and sums before it)
        assert float((out - want).abs().max()) <= 2.0 ** -8
    assert calls["window"] == 1


@pytest.mark.parametrize("B,Hq,T,L,kernel", [(1, 8, 64, 64, False), (1, 32, 256, 256, False), (1, 8, 1, 1024, False),
                                             (1, 8, 2, 1024, True), (1, 8, 1, 1500, True), (8, 32, 300, 300, True)])
@torch.no_grad()
def test_short_calls_stay_with_sdpa(B, Hq, T, L, kernel, monkeypatch):
    """Where reading the mask costs more than the kernel gains, SDPA's time is kept;
    the result is the same either way."""
    from turboquant_pro_amd.hf_cache import tqk_attention
    print(f"[hf window] B={B} Hq={Hq} T={T} L={L}", flush=True)
    calls = counted(monkeypatch)
    gen = torch.Generator(device="cuda").manual_seed(6)
    q, k, v = rows(gen, B, Hq, T, 128), rows(gen, B, Hq // 4, L, 128), rows(gen, B, Hq // 4, L, 128)
    mask = window_mask(T, L, L // 3, B).cuda()
    out, _ = tqk_attention(module(4), q, k, v, mask, scaling=128 ** -0.5, sliding_window=L // 3)
    assert calls["window"] == kernel
    # (values of at most 5: their weights' and the output's roundings to fp16)
    assert float((out - sdpa(q, k, v, mask, 128 ** -0.5)).abs().max()) <= 2 * 5 * 2.0 ** -11 * 2


@torch.no_grad()
def test_one_mask_row_for_every_query_stays_with_sdpa(monkeypatch):
    """A mask row that is broadcast over the queries is no window of each of them, though
    it is the last one's."""
    from turboquant_pro_amd.hf_cache import tqk_attention
    print("[hf window] one mask row", flush=True)
    calls = counted(monkeypatch)
    gen = torch.Generator(device="cuda").manual_seed(7)
    q, k, v = rows(gen, 2, 4, 70, 64), rows(gen, 2, 2, 1000, 64), rows(gen, 2, 2, 1000, 64)
    mask = window_mask(1, 1000, 90, 2).cuda()
    out, _ = tqk_attention(module(2), q, k, v, mask, scaling=0.125, sliding_window=90)
    assert calls["window"] == 0
    # (two calls of one library: the same up to the order of its sums)
    assert float((out - sdpa(q, k, v, mask, 0.125)).abs().max()) <= 2.0 ** -9


@torch.no_grad()
def test_a_layer_without_the_query_heads_stays_with_sdpa(monkeypatch):
    """A cache made without the model's config: its windowed steps run on dense keys and
    values, as they did."""
    from turboquant_pro_amd.hf_cache import TurboQuantLayer, tqk_attention
    print("[hf window] no config", flush=True)
    calls = counted(monkeypatch)
    gen = torch.Generator(device="cuda").manual_seed(8)
    layer = TurboQuantLayer(hot_window=64, value_bits=4, max_cache_len=512, fused_decode=True)
    layer.update(rows(gen, 2, 2, 200, 64), rows(gen, 2, 2, 200, 64))
    q = rows(gen, 2, 8, 1, 64)
    kk, vv = layer.update(rows(gen, 2, 2, 1, 64), rows(gen, 2, 2, 1, 64))
    mask = window_mask(1, 201, 50, 2).cuda()
    out, _ = tqk_attention(module(4), q, kk, vv, mask, scaling=0.125, sliding_window=50)
    assert calls["attend"] == 0
    k, v = layer.dense()
    # (two calls of one library: the same up to the order of its sums)
    assert float((out - sdpa(q, k, v, mask, 0.125)).abs().max()) <= 2.0 ** -9
