"""TQKVPool.attend where the reconstruction of every sequence at once would pass its
bound: slices of sequences, and of one sequence's kv heads."""

import pytest

torch = pytest.importorskip("torch")

from test_gpu_attend import check, make_pool, queries  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU visible")


@pytest.mark.parametrize("lens,D,q_lens", [([90000], 256, None), ([70000, 300, 69000], 128, [129, 40, 77])])
def test_slices(lens, D, q_lens):
    print(f"[attend] slices {lens} D={D}", flush=True)
    T = 129  # (one query head a kv head: the first count that is reconstructed)
    pool = make_pool(31, lens, 8, 8, D)
    q = queries(31, pool, T)
    ql = None if q_lens is None else torch.tensor(q_lens, dtype=torch.int32, device="cuda")
    out = pool.attend(q, q_lens=ql)
    check(pool, out, q, None, 0, q_lens, "slices")
    # a head's result does not go by the slice it is in: as with its own queries alone
    for h in (0, 7):
        q2 = torch.zeros_like(q)
        q2[:, h] = q[:, h]
        assert torch.equal(pool.attend(q2, q_lens=ql)[:, h], out[:, h])
