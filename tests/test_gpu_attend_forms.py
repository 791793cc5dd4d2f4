"""TQKVPool.attend on both sides of the count of rows (queries times query heads of a
kv head) from which keys and values are reconstructed, for every form of the cache:
the first count past 128 rows and the last one before, under the bound of the path
that is taken."""

import math

import pytest

torch = pytest.importorskip("torch")

import test_gpu_attend as A  # noqa: E402
import test_gpu_attend_edges as E  # noqa: E402
from test_gpu_attend import make_pool, queries  # noqa: E402
from test_gpu_attend_large import check, is_dense  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU visible")


def polar(bits):
    return dict(key_grid="polar", key_bits=bits, value_bits=bits)


FORMS = [([1500, 900], 32, 8, 128, dict()), ([1400, 40], 7, 1, 128, dict(value_bits=2, page_tokens=16)),
         ([700, 150], 4, 2, 128, dict(hot_window=48, page_tokens=24)),
         ([1500, 900], 2, 1, 128, dict(key_grid="uniform", key_bits=3, outlier_frac=0.0)),
         ([900, 500], 6, 2, 128, dict(key_grid="uniform", key_bits=3, value_bits=4, hot_window=64)),
         ([900, 500], 5, 1, 64, dict(key_grid="uniform", key_bits=3, outlier_frac=0.05)),
         ([900, 300], 8, 1, 256, dict(key_grid="uniform", key_bits=2, hot_window=64)),
         ([1500, 900], 4, 4, 128, polar(2)), ([1500, 900], 4, 4, 128, polar(3)), ([1500, 900], 8, 2, 128, polar(4)),
         ([700, 150], 4, 2, 128, dict(hot_window=48, page_tokens=24, **polar(3))),
         ([900, 600], 8, 1, 64, polar(2)), ([900, 600], 4, 2, 64, polar(3)), ([900, 600], 3, 1, 64, polar(4)),
         ([900, 600], 4, 1, 256, polar(2)), ([900, 600], 8, 4, 256, polar(3)), ([900, 600], 2, 2, 256, polar(4)),
         ([2100, 600], 4, 1, 64, dict(value_bits=4)), ([2100, 600], 16, 8, 256, dict(value_bits=3))]


@pytest.mark.parametrize("lens,Hq,H,D,form", FORMS)
def test_both_sides_of_the_count(lens, Hq, H, D, form):
    print(f"[attend] forms {lens} {Hq}/{H} D={D} {form}", flush=True)
    pool = make_pool(41, lens, Hq, H, D, **form)
    few = 128 * H // Hq
    for T in (few, few + 1):
        assert is_dense(pool, T) == (T > few)
        q = queries(T, pool, T)
        for window, sinks in ((None, 0), (1, 0), (300, 4), (600, 257), (20, 33)):
            out = pool.attend(q, window=window, sinks=sinks)
            check(pool, out, q, window, sinks, 1.0 / math.sqrt(D), what=f"T={T} window={window} sinks={sinks}")
            assert torch.equal(out, pool.attend(q, window=window, sinks=sinks))


@pytest.mark.parametrize("D,form", [(128, dict()), (64, dict(key_grid="uniform", key_bits=3)), (128, polar(3)),
                                    (256, dict())])
def test_ragged_chunks(D, form):
    """Lengths of zero and one, fewer tokens than queries, no queries at all, on the
    reconstructing side."""
    print(f"[attend] ragged chunks D={D} {form}", flush=True)
    pool = make_pool(42, [0, 1, 4, 600, 1100, 530, 70], 8, 2, D, **form)
    T, m = 33, [33, 3, 33, 33, 7, 0, 33]
    q = queries(T, pool, T)
    ql = torch.tensor(m, dtype=torch.int32, device="cuda")
    for window, sinks in ((None, 0), (200, 3), (1, 1)):
        out = pool.attend(q, window=window, sinks=sinks, q_lens=ql)
        check(pool, out, q, window, sinks, 1.0 / math.sqrt(D), m, f"{window}")
        check(pool, pool.attend(q, window=window, sinks=sinks), q, window, sinks, 1.0 / math.sqrt(D), None, f"{window}")


@pytest.mark.parametrize("D,Hq,H", [(64, 4, 1), (128, 8, 2), (256, 4, 2)])
def test_infinities_that_some_rows_of_a_chunk_see(D, Hq, H):
    E.test_infinities_that_some_queries_see(D, Hq, H, "float16", 128 * H // Hq + 1)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_what_no_row_of_a_chunk_sees_is_not_read(D):
    A.test_what_no_query_sees_is_not_read(D, "float16", 33)


@pytest.mark.parametrize("form", [dict(), polar(3)])
def test_a_captured_chunk(form):
    """A chunk over reconstructed keys and values, captured, replayed between eager
    calls on queries that change."""
    print(f"[attend] captured chunk {form}", flush=True)
    pool = make_pool(43, [3000, 900], 8, 2, **form)
    q, other = queries(43, pool, 40), queries(44, pool, 50)
    graph = torch.cuda.CUDAGraph()
    pool.attend(q, window=700, sinks=4)
    with torch.cuda.graph(graph):
        out = pool.attend(q, window=700, sinks=4)
    for i in range(4):
        q.mul_(-0.9)
        graph.replay()
        pool.attend(other, window=100 + i)
        torch.cuda.synchronize()
        assert torch.equal(out, pool.attend(q, window=700, sinks=4)), i
        out.zero_()


@pytest.mark.parametrize("Hq,H", [(3, 1), (7, 1), (10, 2)])
@pytest.mark.parametrize("D", [64, 128])
def test_odd_head_counts_of_fp32_caches(Hq, H, D):
    print(f"[attend] fp32 {Hq}/{H} D={D}", flush=True)
    pool = make_pool(45, [900, 300], Hq, H, D, input_dtype="float32")
    for T in (1, 5):
        q = queries(T, pool, T)
        for window, sinks in ((None, 0), (200, 4)):
            A.check(pool, pool.attend(q, window=window, sinks=sinks), q, window, sinks, what=f"T={T}")
