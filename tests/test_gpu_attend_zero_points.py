"""TQKVPool.attend over caches whose groups' zero points come from elsewhere than the
tokens (symmetric, sparse, a key bias), and fp32 caches with more queries than one
launch takes."""

import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import test_gpu_attend as A  # noqa: E402
from test_gpu_attend import make_pool, queries  # noqa: E402
from test_gpu_attend_large import check  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU visible")


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("zero", ["symmetric", "sparse", "bias"])
@pytest.mark.parametrize("outliers", [0.0, 0.03])
def test_zero_points(D, zero, outliers):
    print(f"[attend] zero point {zero} D={D} {outliers}", flush=True)
    Hq, H = 8, 2
    form = dict(zero_point=zero, outlier_frac=outliers, hot_window=128)
    if zero != "symmetric":
        form["rope_theta"] = 10000.0
    if zero == "bias":
        form["k_bias"] = np.random.default_rng(2).standard_normal((H, D)).astype(np.float32)
    pool = make_pool(51, [1100, 400], Hq, H, D, **form)
    for T in (1, 32, 33):
        q = queries(T, pool, T)
        for window, sinks in ((None, 0), (300, 4)):
            check(pool, pool.attend(q, window=window, sinks=sinks), q, window, sinks, 1.0 / math.sqrt(D), what=f"T={T}")


def test_more_queries_than_a_launch_of_an_fp32_cache():
    print("[attend] fp32 launches", flush=True)
    pool = make_pool(52, [900, 300, 700], 2, 2, 64, input_dtype="float32", hot_window=64)
    T = 1500  # (4500 queries: 4096 in a launch; more than the tokens there are)
    q = queries(52, pool, T)
    for window, sinks in ((None, 0), (100, 3)):
        A.check(pool, pool.attend(q, window=window, sinks=sinks), q, window, sinks, what=f"{window}")
