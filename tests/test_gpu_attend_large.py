"""TQKVPool.attend on queries and keys near fp16's largest values: queries times
group scales, rotated queries and reconstructed keys that no fp16 holds."""

import pytest

torch = pytest.importorskip("torch")

from attn_ref import HALF, attention, visible  # noqa: E402
from test_gpu_attend import cached, queries  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU visible")


def is_dense(pool, T):
    """Whether the queries go over reconstructed keys and values."""
    return not pool.f32 and T * (pool.n_q_heads // pool.n_kv_heads) > 128


def check(pool, out, q, window, sinks, scale, q_lens=None, what=""):
    """Against 64 bits, with the roundings of the path taken, for fp16 caches: the
    output's; value centroids, and Pi in a chunk, half a step each of sum p |v|_2;
    weights, and in a chunk the reconstructed values, half a step each of sum p |v|,
    and of fp16's smallest where a weight is small; the scores' products and sums in
    fp32, 32 + D units in the last place, in numerator and denominator; PolarQuant
    keys' centroids (a chunk's) half a step of |q|_2 |k|_2, at head_dim 256 Pi's too.
    Together 2^-10 of the output: random roundings do not add up as the bound allows."""
    B, Hq, T, D = q.shape
    dense, h = is_dense(pool, T), HALF[torch.float16]
    off = tot = 0.0
    assert out.dtype == q.dtype == torch.float16 and out.shape == q.shape
    for b in range(B):
        n, m = pool.lengths[b], T if q_lens is None else q_lens[b]
        sees = visible(n, m, T, 0, window, sinks, "cuda")
        assert bool((out[b][:, ~sees.any(1)] == 0).all()), f"{what} seq {b}: a row that sees nothing"
        if n == 0:
            continue
        k, v = cached(pool, b)
        want, weighted, mag, vmax = attention(q[b], k, v, sees, scale)
        size, _, _, longest = attention(q[b], k, v.norm(dim=-1, keepdim=True).expand_as(v).contiguous(), sees, scale)
        score = 2 * scale * mag * (32 + D) * 2.0 ** -24
        if dense and pool.key_grid == "polar":
            parts = 2 if D == 256 else 1
            score = score + 2 * scale * parts * h * q[b].double().norm(dim=-1, keepdim=True) * k.norm(dim=-1).max()
        tol = (h * want.abs() + (score + (n / 16 + 64) * 2.0 ** -23 + (2 if dense else 1) * h) * size
               + (2 if dense else 1) * h * weighted + n * 2.0 ** -25 * longest + 2.0 ** -25)
        got = out[b].double()
        assert bool(torch.isfinite(got).all()), f"{what} seq {b}: not finite"
        err = (got - want).abs()
        assert bool((err <= tol).all()), f"{what} seq {b}: {float((err - tol).max()):.3e} past the bound"
        off += float(err.square().sum())
        tot += float(want.square().sum())
    assert (off / max(tot, 1e-30)) ** 0.5 <= 2.0 ** -10, f"{what} rel {(off / max(tot, 1e-30)) ** 0.5:.2e}"


def pool_of(k, v, Hq, **form):
    from turboquant_pro_amd import TQKVPool
    B, H, L, D = k.shape
    pool = TQKVPool(n_kv_heads=H, n_q_heads=Hq, head_dim=D, max_batch=B, max_seq_len=L, seed=3, **form)
    pool.append(k, v)
    pool.check()
    return pool


def randn(seed, *shape):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


FORMS = [(64, 8, 2, dict(value_bits=4)), (128, 8, 2, dict()), (128, 4, 4, dict(value_bits=2, page_tokens=16)),
         (128, 4, 2, dict(hot_window=48, page_tokens=24)), (256, 4, 1, dict(value_bits=4)),
         (128, 8, 1, dict(key_grid="uniform", key_bits=3)), (64, 4, 2, dict(key_grid="uniform", key_bits=2))]


@pytest.mark.parametrize("D,Hq,H,form", FORMS)
@pytest.mark.parametrize("T", [1, 6, None])
def test_queries_times_group_scales_past_fp16(D, Hq, H, form, T):
    """q * scale of a channel reaches 10^6 (an fp16 pair holds 131008): the scores,
    and with them who wins, are the formula's; groups of small and large scales."""
    T = 128 * H // Hq + 1 if T is None else T
    print(f"[attend] large products D={D} {Hq}/{H} T={T} {form}", flush=True)
    L = 1500
    grow = torch.exp2(torch.arange(L, device="cuda") * 13.0 / L - 1.0).floor()  # 1/2 .. 4096 along the tokens
    k = (randn(1, 2, H, L, D) * 0.8 * grow[:, None]).half()
    k[:, :, ::7] = (randn(2, 2, H, len(range(0, L, 7)), D) * 3000).half()  # (every group has a large scale)
    pool = pool_of(k, randn(3, 2, H, L, D).half(), Hq, **form)
    q = (40.0 * queries(4, pool, T)).half()
    assert 160 * float(pool.gscale.max()) > 2 * 131008
    for scale in (2.0 ** -20, 2.0 ** -24):
        pool.desc.sm_scale = scale
        for window, sinks in ((None, 0), (700, 5)):
            check(pool, pool.attend(q, window=window, sinks=sinks), q, window, sinks, scale, what=f"{scale} {window}")


@pytest.mark.parametrize("D,bits", [(64, 4), (128, 3), (256, 2), (256, 4)])
@pytest.mark.parametrize("T", [1, None])
def test_rotated_queries_past_fp16(D, bits, T):
    """PolarQuant keys: a query that one row of the rotation gathers to 10^6."""
    T = 65 if T is None else T
    print(f"[attend] large rotated queries D={D} T={T}", flush=True)
    k, v = (2.0 * randn(5, 1, 2, 900, D)).half(), randn(6, 1, 2, 900, D).half()
    pool = pool_of(k, v, 4, key_grid="polar", key_bits=bits, value_bits=bits, hot_window=128)
    q = (3000.0 * queries(7, pool, T)).half()
    q[:, 1] = (60000.0 * torch.sign(pool.pi_t[:, 3])).half()
    q[:, 2] = (60000.0 * torch.sign(pool.pi_t[:, D - 1])).half()
    assert float((q[0, 1].float() @ pool.pi_t).abs().max()) > 131008
    scale = 2.0 ** -18
    pool.desc.sm_scale = scale
    for window, sinks in ((None, 0), (300, 5)):
        check(pool, pool.attend(q, window=window, sinks=sinks), q, window, sinks, scale, what=f"{window}")


@pytest.mark.parametrize("D,Hq,H,form", [(64, 4, 2, dict()), (128, 4, 2, dict(outlier_frac=0.0)), (256, 2, 1, dict()),
                                         (128, 4, 2, dict(key_grid="polar", key_bits=3, value_bits=3)),
                                         (64, 4, 2, dict(key_grid="polar", key_bits=2, value_bits=2)),
                                         (256, 4, 2, dict(key_grid="polar", key_bits=4, value_bits=4))])
@pytest.mark.parametrize("T", [1, None])
def test_keys_reconstructed_past_fp16(D, Hq, H, form, T):
    """Keys near 65504 whose code stands for more (an NF4 level above them, or a rotated
    centroid; a uniform grid ends at the group's largest key): the formula's result, of
    few queries and of a chunk."""
    T = 128 * H // Hq + 1 if T is None else T
    print(f"[attend] large keys D={D} T={T} {form}", flush=True)
    L = 1100
    u = torch.rand((1, H, L, D), generator=torch.Generator(device="cuda").manual_seed(8), device="cuda")
    share = torch.linspace(0.3, 0.95, D, device="cuda")
    up = torch.rand((1, H, L, D), generator=torch.Generator(device="cuda").manual_seed(9), device="cuda") < share
    k = torch.where(up, 52000 + 13504 * u, -62000 + 14000 * u).half()
    assert bool(torch.isfinite(k).all())
    pool = pool_of(k, randn(10, 1, H, L, D).half(), Hq, hot_window=128, **form)
    assert float(cached(pool, 0)[0].abs().max()) > 65520
    q = queries(11, pool, T)
    scale = 2.0 ** -18
    pool.desc.sm_scale = scale
    for window, sinks in ((None, 0), (300, 5)):
        check(pool, pool.attend(q, window=window, sinks=sinks), q, window, sinks, scale, what=f"{window}")
