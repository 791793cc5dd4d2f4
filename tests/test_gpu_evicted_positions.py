"""Positions of what an eviction leaves: ``position_start`` of exported groups, through
appends, further evictions, growth, a shared prefix, a restore and a reset; a restored
sequence counts on from where it was."""

import pytest

torch = pytest.importorskip("torch")

from more_ref import cached, make_pool, queries, tokens  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU visible")


def starts(pool, b):
    return [pool.export_group(b, g)["position_start"] for g in range(pool.n_groups(b))]


def evicted(pool, want, seed, keep, **kw):
    """Evict by random weights; ``want``: every sequence's groups' positions, which follow."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    weights = torch.rand((pool.max_batch, pool.n_kv_heads, pool.max_groups), generator=gen, device="cuda")
    kept = pool.evict(weights, keep, **kw).tolist()
    return [[x[g] for g in row if g >= 0] for x, row in zip(want, kept)]


def grow(pool, want, seed, new):
    k, v = tokens(seed, pool.max_batch, pool.n_kv_heads, max(new), pool.head_dim, pool.dtype)
    pool.append(k, v, n_new=new)
    G = pool.group_tokens
    return [x + [g * G + pool.evicted_tokens[b] for g in range(len(x), pool.n_groups(b))] for b, x in enumerate(want)]


FORMS = [
    ([5000, 1300, 700, 0], 4, 2, 128, dict()),
    ([700, 150], 4, 2, 128, dict(hot_window=47, page_tokens=12)),
    ([900, 300], 2, 2, 64, dict(key_grid="polar", key_bits=3, value_bits=3, hot_window=64)),
    ([900, 300], 2, 1, 256, dict(input_dtype="float32", hot_window=64)),
]


@pytest.mark.parametrize("lens,Hq,H,D,form", FORMS)
def test_groups_keep_their_positions(lens, Hq, H, D, form):
    print(f"[positions] {lens} {Hq}/{H} D={D} {form}", flush=True)
    pool = make_pool(3, lens, Hq, H, D, room=1500, **form)
    G, n = pool.group_tokens, len(lens)
    want = [[g * G for g in range(pool.n_groups(b))] for b in range(n)]
    assert [starts(pool, b) for b in range(n)] == want
    for step, (share, kw) in enumerate(((0.9, {}), (0.5, dict(first=0, last=2)), (0.6, dict(first=2, last=0)))):
        keep = max(int(share * max(len(x) for x in want)), 2)
        want = evicted(pool, want, step, keep, **kw)
        assert [starts(pool, b) for b in range(n)] == want, f"eviction {step}"
        # (few sequences' tokens with the launch, and a longer chunk)
        for i, new in enumerate(([G + 1 + b for b in range(n)], [3 * G - b for b in range(n)])):
            want = grow(pool, want, 10 * step + i, new)
            assert [starts(pool, b) for b in range(n)] == want, f"append {step}"
    big = pool.grown(pool.max_seq_len + 3000)
    assert [starts(big, b) for b in range(n)] == want
    want = grow(big, want, 99, [2 * G] * n)
    want = evicted(big, want, 98, 3)
    assert [starts(big, b) for b in range(n)] == want
    pool.reset()
    k, v = tokens(5, n, H, 2 * pool.hot_window + G, D, pool.dtype)
    pool.append(k, v)
    assert [starts(pool, b) for b in range(n)] == [[g * G for g in range(pool.n_groups(b))] for b in range(n)]


def test_a_prefix_shared_after_an_eviction():
    print("[positions] shared", flush=True)
    pool = make_pool(4, [0, 3000, 0], 8, 2, room=1500)
    want = evicted(pool, [[], [g * 256 for g in range(pool.n_groups(1))], []], 1, 5)
    pool.share_prefix(1)
    want = [want[1]] * 3
    assert [starts(pool, b) for b in range(3)] == want
    want = grow(pool, want, 7, [600, 900, 300])
    assert [starts(pool, b) for b in range(3)] == want
    want = evicted(pool, want, 2, pool._shared + 1, first=0)
    assert [starts(pool, b) for b in range(3)] == want


@pytest.mark.parametrize("last", [0, 1])
def test_a_restored_sequence_counts_on(last):
    """Exported groups and hot tokens into another pool: queries, keys and positions go on
    as in the pool that they came from."""
    print(f"[positions] restore {last}", flush=True)
    from turboquant_pro_amd import TQKVPool
    pool = make_pool(5, [3000, 1900], 8, 2, room=1500)
    want = evicted(pool, [[g * 256 for g in range(pool.n_groups(b))] for b in range(2)], 3, 4, last=last)
    gen = torch.Generator(device="cuda").manual_seed(6)
    rows = torch.randn((2, 700, 12 * 128), generator=gen, device="cuda").half()
    inv = (10000.0 ** (-torch.arange(64, dtype=torch.float64) / 64)).float().cuda()
    other = TQKVPool(n_kv_heads=2, n_q_heads=8, max_batch=2, max_seq_len=4500,
                     rotation=(pool.pi.cpu().numpy(), pool.pi_t.cpu().numpy()))
    for b in range(2):
        groups = [(x, x) for x in (pool.export_group(b, g) for g in range(pool.n_groups(b)))]
        hot = pool.hot_window_tokens(b)
        if any(x["position_start"] != g * 256 for g, (x, _) in enumerate(groups)):
            with pytest.raises(ValueError):
                other.load_sequence(b, groups, *hot)
        for bad in (-256, 100, 2 ** 31, 256 * (groups[-1][0]["position_start"] // 256 - len(groups))):
            with pytest.raises(ValueError):
                other.load_sequence(b, groups, *hot, evicted_tokens=bad)
        for bad in ([dict(x, position_start=None) for x, _ in groups], [x for x, _ in groups][::-1]):
            with pytest.raises(ValueError):
                other.load_sequence(b, [(x, x) for x in bad], *hot, evicted_tokens=pool.evicted_tokens[b])
        assert other.lengths[b] == 0
        other.load_sequence(b, groups, *hot, evicted_tokens=pool.evicted_tokens[b])
    assert other.lengths == pool.lengths and other.evicted_tokens == pool.evicted_tokens
    assert [starts(other, b) for b in range(2)] == want == [starts(pool, b) for b in range(2)]
    for x in (rows, rows[:, :1].contiguous()):
        assert torch.equal(pool.append_qkv(x, inv), other.append_qkv(x, inv))
    assert [starts(other, b) for b in range(2)] == [starts(pool, b) for b in range(2)]
    for b in range(2):
        assert len(starts(pool, b)) > len(want[b])
        for x, y in zip(cached(pool, b), cached(other, b)):
            assert torch.equal(x, y)
    q = queries(7, pool, 1)
    assert torch.equal(pool.attend(q), other.attend(q))


def test_a_whole_sequence_is_restored_as_ever():
    """No tokens lost: with positions, without them, or with another writer's zeros."""
    print("[positions] whole", flush=True)
    from turboquant_pro_amd import TQKVPool
    pool = make_pool(8, [1500], 4, 2)
    groups = [pool.export_group(0, g) for g in range(pool.n_groups(0))]
    for kind in (groups, [{k: v for k, v in x.items() if k != "position_start"} for x in groups],
                 [dict(x, position_start=0) for x in groups]):
        for kw in ({}, dict(evicted_tokens=0)):
            other = TQKVPool(n_kv_heads=2, n_q_heads=4, max_batch=1, max_seq_len=1500,
                             rotation=(pool.pi.cpu().numpy(), pool.pi_t.cpu().numpy()))
            other.load_sequence(0, [(x, x) for x in kind], *pool.hot_window_tokens(0), **kw)
            assert other.evicted_tokens == [0] and starts(other, 0) == starts(pool, 0)
            for x, y in zip(cached(pool, 0), cached(other, 0)):
                assert torch.equal(x, y)


def test_inference_mode():
    """Evictions and shares inside of it, appends, exports and resets outside."""
    print("[positions] inference mode", flush=True)
    pool = make_pool(9, [0, 2600], 4, 2, room=1500)
    with torch.inference_mode():
        want = evicted(pool, [[], [g * 256 for g in range(pool.n_groups(1))]], 1, 4)
        pool.share_prefix(1)
    want = grow(pool, [want[1]] * 2, 3, [700, 300])
    assert [starts(pool, b) for b in range(2)] == want
    q = queries(1, pool, 1)
    with torch.inference_mode():
        got = pool.attend(q)
        want = grow(pool, want, 4, [300, 700])
    assert torch.isfinite(got).all() and [starts(pool, b) for b in range(2)] == want
    assert torch.isfinite(grown_out := pool.grown(9000).attend(q)).all() and grown_out.shape == got.shape
    pool.reset()
    assert pool.lengths == [0, 0]
