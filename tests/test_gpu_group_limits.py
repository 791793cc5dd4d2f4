"""Sizes at the limits of the operators that read less of a coded cache: lists, queries
and rings larger than one launch or column takes."""

import pytest

torch = pytest.importorskip("torch")

from attn_ref import visible  # noqa: E402
from more_ref import cached, check_rows, listed, make_pool, queries, tokens  # noqa: E402

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


def ringed(ring, lens, Hq, H, D, room, **kw):
    """A pool whose rings are longer than the hot window."""
    import ctypes

    from turboquant_pro_amd import TQKVPool
    pool = TQKVPool(n_kv_heads=H, n_q_heads=Hq, head_dim=D, max_batch=len(lens), max_seq_len=max(lens) + room, seed=3, **kw)
    pool.hot_k, pool.hot_v = (torch.full((len(lens), H, ring, D), 7.0, dtype=pool.dtype, device="cuda") for _ in range(2))
    pool.ptrs.hot_k, pool.ptrs.hot_v, pool.desc.hot_ring = pool.hot_k.data_ptr(), pool.hot_v.data_ptr(), ring
    assert pool.ptrs.hot_k == ctypes.c_void_p(pool.hot_k.data_ptr()).value
    k, v = tokens(3, len(lens), H, max(lens), D, pool.dtype)
    pool.append(k, v, n_new=lens)
    pool.check()
    return pool


@pytest.mark.parametrize("ring,D,form", [(512, 128, dict()), (513, 128, dict()), (1024, 64, dict()), (2048, 128, dict()),
                                         (4096, 128, dict()), (4095, 64, dict()), (4096, 256, dict(input_dtype="float32")),
                                         (100, 64, dict(hot_window=64))])
def test_evictions_turn_rings_of_any_length(ring, D, form):
    """Columns of 128 to 16 bytes: the cache after evictions and appends as with a ring of
    the hot window's size."""
    print(f"[limits] ring {ring} D={D} {form}", flush=True)
    lens, H = [2900, 1500, 40], 2
    one, two = ringed(ring, lens, 2 * H, H, D, 1500, **form), make_pool(3, lens, 2 * H, H, D, room=1500, **form)
    gen = torch.Generator(device="cuda").manual_seed(9)
    for step in range(3):
        weights = torch.rand((3, H, one.max_groups), generator=gen, device="cuda")
        other = weights.clone()
        keep = (9, 5, 3)[step]
        assert torch.equal(one.evict(weights, keep), two.evict(other, keep))
        assert torch.equal(weights, other) and one.lengths == two.lengths
        for i in range(2):
            for b, (x, y) in enumerate(zip(zip(*one.dense()), zip(*two.dense()))):
                n = one.lengths[b]
                assert torch.equal(x[0][:, :n], y[0][:, :n]) and torch.equal(x[1][:, :n], y[1][:, :n]), f"step {step} seq {b}"
            q = queries(step, one, 1)
            assert torch.equal(one.attend(q), two.attend(q))
            k, v = tokens(20 + step, 3, H, 400, D, one.dtype)
            one.append(k, v, n_new=[400, 37, 1])
            two.append(k, v, n_new=[400, 37, 1])


@pytest.mark.parametrize("D,Hq,H,form", [(128, 8, 2, dict()), (64, 4, 4, dict(hot_window=64)), (256, 7, 1, dict(value_bits=4))])
def test_infinite_values_of_uncoded_tokens(D, Hq, H, form):
    """Their channel of the rows that see them, however small their weight is; a row that
    does not see them, and every other number, stays as it is."""
    print(f"[limits] infinities D={D} {Hq}/{H}", flush=True)
    pool, gq, T = make_pool(10, [1500, 700], Hq, H, D, **form), Hq // H, 3
    q = queries(11, pool, T)
    q[..., 3] = 1.0
    groups = pool.select_groups(q, 2)
    b, h, token = 1, H - 1, pool.lengths[1] - 2  # (the first query stands before it)
    at = token % pool.hot_window
    pool.hot_k[b, h, at] = 0.0
    pool.hot_k[b, h, at, 3] = -60000.0
    pool.hot_v[b, h, at, 11] = 0.0

    def runs():
        w = torch.zeros((2, H, pool.max_groups), device="cuda")
        return [pool.attend(q, groups=groups), pool.attend(q, weights=w), pool.attend(q, window=9, sinks=3, weights=w)], w

    want, weights = runs()
    for x in (float("inf"), float("-inf"), float("nan")):
        pool.hot_v[b, h, at, 11] = x
        got, w = runs()
        assert torch.equal(w, weights)
        for y, was in zip(got, want):
            rows = y[b, h * gq:(h + 1) * gq, 1:, 11].clone()
            assert bool((rows.isnan() if x != x else rows == x).all())
            y[b, h * gq:(h + 1) * gq, 1:, 11] = was[b, h * gq:(h + 1) * gq, 1:, 11]
            assert torch.equal(y, was)
