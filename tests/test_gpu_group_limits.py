"""Sizes at the limits of the operators that read less of a coded cache: lists, queries
and rings larger than one launch or column takes."""

import pytest

torch = pytest.importorskip("torch")

from attn_ref import visible  # noqa: E402
from more_ref import cached, check_rows, listed, make_pool, queries  # noqa: E402

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


@pytest.mark.parametrize("per_query", [True, False])
def test_lists_for_more_rows_than_a_launch(per_query):
    """More than 2^22 workgroups, two slices of queries: rows of both against 64 bits, the
    last queries as a call of their own."""
    print(f"[limits] lists {per_query}", flush=True)
    # (one list for all queries: eight rows a workgroup)
    B, H, T = (1024, 8, 520) if per_query else (8192, 8, 520)
    hot, D = (64, 64) if per_query else (2, 64)
    lens = [600 - (b % 3) * 30 for b in range(B)] if per_query else [5 + b % 3 for b in range(B)]
    pool = make_pool(4, lens, H, H, D, hot_window=hot, outlier_frac=0.0)
    q = queries(5, pool, T)
    gen = torch.Generator(device="cuda").manual_seed(6)
    most = max(pool.n_groups(b) for b in range(B))
    groups = torch.randint(-1, most // 2, (B, H, T if per_query else 1, 2), generator=gen, device="cuda", dtype=torch.int32)
    groups[..., 1] += (groups[..., 1] >= 0).int() * (most // 2)  # (no group twice, which would count twice)
    assert B * H * (T if per_query else T // 8) > 2 ** 22
    out = pool.attend(q, groups=groups)
    for b in (0, 1, 517, B - 1):
        k, v = cached(pool, b)
        sees = listed(pool, b, groups[b], T, T)
        for h in (0, H - 1):
            check_rows(out[b, h:h + 1], q[b, h:h + 1], k[h], v[h], sees[h], f"seq {b} head {h}")
    few = groups[:, :, -40:] if per_query else groups
    assert torch.equal(pool.attend(q[:, :, -40:], groups=few), out[:, :, -40:])


def test_weights_of_more_rows_than_a_launch():
    """A coded group at most, 2^22 workgroups and more."""
    print("[limits] weights", flush=True)
    B, H, T = 1500, 5, 600
    pool = make_pool(7, [70 - b % 9 for b in range(B)], 5 * H, H, 64, hot_window=64, outlier_frac=0.0)
    assert B * H * T > 2 ** 22 and max(pool.n_groups(b) for b in range(B)) == 1
    q = queries(8, pool, T)
    weights = torch.zeros((B, H, pool.max_groups), device="cuda")
    out = pool.attend(q, weights=weights)
    again = torch.zeros_like(weights)
    assert torch.equal(pool.attend(q[:, :, -70:], weights=again), out[:, :, -70:])
    # (queries before the first token have no weights; sums of other slices: fp32's steps)
    assert torch.allclose(weights, again, rtol=2.0 ** -20, atol=0)
    for b in (0, 4, B - 1):
        k, v = cached(pool, b)
        sees = visible(pool.lengths[b], T, T, 0, None, 0, "cuda")
        for h in (0, H - 1):
            s = slice(5 * h, 5 * h + 5)
            check_rows(out[b, s], q[b, s], k[h], v[h], sees, f"seq {b} head {h}")
