"""Infinities and NaN among values that queries do see, under weights that no 16-bit or
32-bit number holds beside the largest: an infinity times any positive weight."""

import pytest

torch = pytest.importorskip("torch")

from attn_ref import visible  # noqa: E402
from test_gpu_attend import make_pool, queries  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU visible")


INF, NAN = float("inf"), float("nan")
# (token, channel, value): alone, both signs of one channel, a NaN beside an infinity
ODD = [(3, 5, INF), (40, 9, -INF), (41, 11, INF), (90, 11, -INF), (60, 20, NAN), (61, 20, INF), (130, 33, NAN)]


def same_kind(got, clean, sees, heads, odd, what):
    """``got (Hq, T, D)``: in a channel where a row sees odd values their sum (every
    weight of the formula is positive, though 64 bits hold some as zero beside weights
    e^700 times as large), every other result as without them."""
    want = clean.double().clone()
    for ch in {c for _, c, _ in odd}:
        for t in range(sees.shape[0]):
            seen = [x for at, c, x in odd if c == ch and bool(sees[t, at])]
            if seen:
                want[heads, t, ch] = sum(seen)
    assert torch.equal(got.double().isnan(), want.isnan()), what
    assert torch.equal(got.double().nan_to_num(0.0, INF, -INF), want.nan_to_num(0.0, INF, -INF)), what


@pytest.mark.parametrize("D,dtype", [(64, torch.float16), (128, torch.bfloat16), (128, torch.float16), (256, torch.float16)])
@pytest.mark.parametrize("T,L", [(1, 300), (1, 9000), (250, 700), (40, 5000)])
@pytest.mark.parametrize("spread", [1.0, 5.0, 40.0])
def test_window_attention(D, dtype, T, L, spread):
    from turboquant_pro_amd import window_attention
    print(f"[visible] D={D} {dtype} T={T} L={L} spread={spread}", flush=True)
    gen = torch.Generator(device="cuda").manual_seed(L)
    q = torch.randn((1, 4, T, D), generator=gen, device="cuda").to(dtype)
    k = (spread * torch.randn((1, 2, L, D), generator=gen, device="cuda")).to(dtype)
    v = torch.randn((1, 2, L, D), generator=gen, device="cuda").to(dtype)
    for window in (None, 200):
        clean = window_attention(q, k, v, window=window)
        odd = {(base + at, (ch + base) % D): x for base in (0, L - 250) for at, ch, x in ODD}
        odd = [(at, ch, x) for (at, ch), x in odd.items()]
        bad = v.clone()
        for at, ch, x in odd:
            bad[0, 1, at, ch] = x
        got = window_attention(q, k, bad, window=window)
        same_kind(got[0], clean[0], visible(L, T, T, 0, window, 0), [2, 3], odd, f"window={window}")


def attend(D, Hq, H, dtype, T, spread):
    print(f"[visible] attend D={D} {Hq}/{H} {dtype} T={T} spread={spread}", flush=True)
    pool = make_pool(61, [1500, 700], Hq, H, D, input_dtype=dtype)
    q = (spread * queries(61, pool, T)).to(pool.dtype)
    for window in (None, 250):
        clean = pool.attend(q, window=window).clone()
        keep = pool.hot_v.clone()
        for b in range(2):
            for at, ch, x in ODD:
                pool.hot_v[b, H - 1, (pool.lengths[b] - 1 - at) % pool.hot_window, ch] = x
        got = pool.attend(q, window=window)
        for b in range(2):
            n = pool.lengths[b]
            same_kind(got[b], clean[b], visible(n, T, T, 0, window, 0), list(range(Hq - Hq // H, Hq)),
                      [(n - 1 - at, ch, x) for at, ch, x in ODD], f"{b} window={window}")
        pool.hot_v.copy_(keep)


@pytest.mark.parametrize("D,Hq,H", [(64, 4, 2), (128, 8, 2), (256, 4, 2)])
@pytest.mark.parametrize("spread", [1.0, 5.0, 40.0])
def test_attend_chunks(D, Hq, H, spread):
    """Uncoded values of a chunk over reconstructed keys and values."""
    attend(D, Hq, H, "float16", 128 * H // Hq + 1, spread)


@pytest.mark.parametrize("D,Hq,H", [(64, 4, 2), (128, 8, 2), (256, 4, 2)])
@pytest.mark.parametrize("T", [1, 7])
@pytest.mark.parametrize("spread", [1.0, 5.0, 40.0])
def test_attend_few(D, Hq, H, T, spread):
    """Over the codes: weights that another wave's, split's or later block's scores
    leave behind by more than fp32 holds."""
    attend(D, Hq, H, "float16", T, spread)


@pytest.mark.parametrize("D,Hq,H", [(64, 4, 2), (128, 4, 2), (256, 2, 1)])
@pytest.mark.parametrize("T", [1, 7])
@pytest.mark.parametrize("spread", [1.0, 5.0, 40.0])
def test_attend_fp32_caches(D, Hq, H, T, spread):
    attend(D, Hq, H, "float32", T, spread)
