"""Sizes at the limits of the operators that read less of a coded cache: lists, queries
and rings larger than one launch or column takes."""

import pytest

torch = pytest.importorskip("torch")

from more_ref import make_pool, queries  # noqa: E402

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


def test_choices_for_more_queries_than_a_launch():
    """2^21 rows, two slices of queries: every one's choice from its definition in 64 bits."""
    print("[limits] queries", flush=True)
    B, H, T, top = 64, 8, 4096, 3
    pool = make_pool(2, [T] * (B - 1) + [2000], H, H, 64, outlier_frac=0.0)
    q = queries(3, pool, T)
    got = pool.select_groups(q, top)
    G = pool.group_tokens
    assert B * H * T > (2 ** 31 - 1) // 1024
    for b in (0, 31, B - 1):
        ng, n = pool.n_groups(b), pool.lengths[b]
        slots = pool.group_table[b, :ng].long()
        mid, half = (x[slots].double().permute(1, 2, 0).contiguous() for x in (pool.gmean, pool.gscale))  # (H, D, ng)
        x = q[b].double().contiguous()
        score = torch.matmul(x, mid) + torch.matmul(x.abs(), half)  # (H, T, ng)
        p = (n - T + torch.arange(T, device="cuda"))[:, None]
        g = torch.arange(ng, device="cuda")
        c = torch.where(p >= 0, torch.clamp(p // G + 1, max=ng), 0)
        score = torch.where((g < 1) | (g >= c - 1), torch.inf, score).masked_fill(g >= c, -torch.inf)
        order = score.sort(dim=-1, descending=True, stable=True).indices[..., :top]
        want = torch.where(torch.arange(top, device="cuda") < c, order, ng).sort(-1).values
        want = torch.where(want == ng, -1, want)
        assert torch.equal(got[b].long(), want), f"sequence {b}"
    # the same of fewer queries, in one launch
    assert torch.equal(pool.select_groups(q[:, :, -300:], top), got[:, :, -300:])
