"""A sliding-window model run over a TurboQuantCache: prefill, chunk and steps on the
windowed kernels against SDPA on the same cache's dense keys and values."""

import pytest

torch = pytest.importorskip("torch")
transformers = pytest.importorskip("transformers")

from test_gpu_hf_window import counted  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU visible")


@pytest.mark.parametrize("D,dtype", [(64, torch.float16), (128, torch.bfloat16)])
@torch.no_grad()
def test_a_windowed_model(D, dtype, monkeypatch):
    from transformers import MistralConfig, MistralForCausalLM
    from turboquant_pro_amd import hf_cache as HC
    print(f"[hf window model] D={D} {dtype}", flush=True)
    torch.manual_seed(5)
    layers, steps = 2, 8
    cfg = MistralConfig(vocab_size=256, hidden_size=8 * D, intermediate_size=256, num_hidden_layers=layers,
                        num_attention_heads=8, num_key_value_heads=2, head_dim=D, sliding_window=200,
                        max_position_embeddings=4096)
    model = MistralForCausalLM(cfg).to("cuda", dtype).eval()
    ids = torch.randint(0, 256, (2, 1100 + steps)).cuda()
    calls = counted(monkeypatch)

    def run(implementation, fused):
        HC._register()
        model.set_attn_implementation(implementation)
        cache = HC.TurboQuantCache(config=cfg, hot_window=256, fused_decode=fused)
        cuts = [0, 1000, 1100] + [1101 + i for i in range(steps)]
        return torch.stack([model(ids[:, a:b], past_key_values=cache).logits[:, -1] for a, b in zip(cuts, cuts[1:])]).float()

    dense = run("sdpa", False)
    assert calls == {"attend": 0, "decode": 0, "window": 0}
    fused = run(HC.ATTN_IMPLEMENTATION, True)
    assert calls == {"attend": steps * layers, "decode": 0, "window": 2 * layers}
    # (two layers of 16-bit roundings, as the model test without a window has it)
    assert float((fused - dense).abs().max()) <= 2e-2 * float(dense.abs().max())
    out = HC.enable_turboquant_cache(model).generate(ids[:, :300], max_new_tokens=5, do_sample=False)
    assert out.shape == (2, 305)
