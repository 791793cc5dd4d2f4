"""TQKVPool.attend in every instance of its kernels: head dims, tiled and plain value
rows, value widths, key grids and widths; few queries and a chunk."""

import math

import pytest

torch = pytest.importorskip("torch")

from test_gpu_attend import make_pool, queries  # noqa: E402
from test_gpu_attend_large import check, is_dense  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU visible")


@pytest.mark.parametrize("keys", ["nf4", "uniform4", "uniform3", "uniform2", "polar"])
@pytest.mark.parametrize("vb", [2, 3, 4])
@pytest.mark.parametrize("D,page", [(64, 32), (128, 32), (128, 8), (256, 32)])
def test_instance(D, page, vb, keys):
    print(f"[attend] instance D={D} page={page} V{vb} {keys}", flush=True)
    form = dict(value_bits=vb, hot_window=128, page_tokens=page)
    if keys == "polar":
        form.update(key_grid="polar", key_bits=vb)
    elif keys != "nf4":
        form.update(key_grid="uniform", key_bits=int(keys[-1]))
    pool = make_pool(71, [900, 333], 8, 2, D, **form)
    assert pool.tiled == (D == 128 and page == 32)
    for T in (1, 6, 33):
        assert is_dense(pool, T) == (T == 33)
        q = queries(T, pool, T)
        for window, sinks in ((None, 0), (250, 3)):
            check(pool, pool.attend(q, window=window, sinks=sinks), q, window, sinks, 1.0 / math.sqrt(D),
                  what=f"T={T} window={window}")
