"""Sizes at the limits of the operators that read less of a coded cache: lists, queries
and rings larger than one launch or column takes."""

import pytest

torch = pytest.importorskip("torch")

from more_ref import make_pool  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU visible")


def test_a_number_of_groups_past_32_bits_is_refused():
    """... and not taken for its lowest 32 bits: the pool's lengths stay its tables'."""
    print("[limits] keep", flush=True)
    pool = make_pool(1, [1500], 2, 1)
    weights = torch.zeros((1, 1, pool.max_groups), device="cuda")
    for keep in (2 ** 24 + 1, 2 ** 32 + 2):
        with pytest.raises(ValueError):
            pool.evict(weights, keep)
    assert pool.lengths == [1500] == pool.seq_lens.tolist()
