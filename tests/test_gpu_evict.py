"""TQKVPool.evict: which groups stay, against the definition on the host; the cache after
it against its own groups and tokens before, appends and attention that go on from it."""

import math

import pytest

torch = pytest.importorskip("torch")

from more_ref import cached, check_rows, make_pool, queries, tokens  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU visible")


def kept_groups(weights, b, ng, keep, first, last):
    if ng <= keep:
        return list(range(ng))
    total = weights[b].double().sum(0).tolist()
    pick = [g for g in range(ng) if g < first or g >= ng - last]
    rest = sorted((g for g in range(ng) if g not in set(pick)),
                  key=lambda g: (0, 0.0, g) if math.isnan(total[g]) else (1, -total[g], g))
    return sorted(pick + rest[:keep - len(pick)])


def some_weights(seed, pool):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    w = torch.exp(2 * torch.randn((pool.max_batch, pool.n_kv_heads, pool.max_groups), generator=gen, device="cuda"))
    for b in range(pool.max_batch):
        w[b, :, pool.n_groups(b):] = 0.0
    return w


def state(pool):
    """Every sequence's keys and values in order, its group count."""
    return [(cached(pool, b) if pool.lengths[b] else None, pool.n_groups(b)) for b in range(pool.max_batch)]


def check_eviction(pool, weights, keep, first=1, last=1):
    before, w0, lens, gone0 = state(pool), weights.clone(), list(pool.lengths), pool.evicted_tokens
    slots0 = pool.group_table.clone()
    kept = pool.evict(weights, keep, first=first, last=last)
    G = pool.group_tokens
    assert kept.shape == (pool.max_batch, keep) and kept.dtype == torch.int32
    for b, (kv, ng) in enumerate(before):
        want = kept_groups(w0, b, ng, keep, max(first, pool._shared), last)
        assert kept[b].tolist() == want + [-1] * (keep - len(want))
        gone = ng - len(want)
        assert pool.lengths[b] == lens[b] - gone * G == int(pool.seq_lens[b]) and pool.n_groups(b) == len(want)
        assert pool.evicted_tokens[b] == gone0[b] + gone * G
        assert sorted(pool.group_table[b].tolist()) == sorted(slots0[b].tolist())
        assert torch.equal(weights[b, :, :len(want)].nan_to_num(-1.0), w0[b][:, want].nan_to_num(-1.0))
        assert bool((weights[b, :, len(want):] == 0).all())
        if kv is None:
            continue
        at = torch.tensor([g * G + i for g in want for i in range(G)] + list(range(ng * G, lens[b])), device="cuda")
        for got, was in zip(cached(pool, b), kv):
            assert torch.equal(got, was[:, at])
    return kept


FORMS = [
    ([5000, 1300, 700, 0, 5], 8, 2, 128, dict()),
    ([2600, 900], 4, 4, 128, dict(hot_window=64, page_tokens=16)),
    ([700, 150], 4, 2, 128, dict(hot_window=47, page_tokens=12)),
    ([300, 81], 2, 1, 64, dict(hot_window=7, page_tokens=4)),
    ([2100, 600], 8, 8, 256, dict(value_bits=4)),
    ([1500, 900], 4, 4, 128, dict(key_grid="polar", key_bits=3, value_bits=3)),
    ([1500, 900], 4, 1, 256, dict(input_dtype="float32")),
    ([1500, 900], 4, 1, 128, dict(key_grid="uniform", key_bits=2, hot_window=63, page_tokens=8)),
]


@pytest.mark.parametrize("lens,Hq,H,D,form", FORMS)
def test_what_stays_and_where(lens, Hq, H, D, form):
    """Again and again, with appends between: rings turned, tables reordered twice."""
    print(f"[evict] {lens} {Hq}/{H} D={D} {form}", flush=True)
    pool = make_pool(3, lens, Hq, H, D, room=1200, **form)
    G = pool.group_tokens
    most = max(pool.n_groups(b) for b in range(len(lens)))
    for step, (keep, first, last) in enumerate(((most, 1, 1), (most - 1, 1, 1), (max(most // 2, 3), 2, 1),
                                                (max(most // 3, 2), 0, 2), (1, 0, 0), (0, 0, 0))):
        weights = some_weights(step, pool)
        if step == 2:
            weights[:, :, 2:4] = float("nan")
            weights[:, :, :] = torch.where(weights.isnan(), weights, weights.round())  # ties too
        check_eviction(pool, weights, keep, first, last)
        # what is appended next lands behind what stayed
        before = state(pool)
        new = [min(2 * G + 3 * b, pool.max_seq_len - pool.lengths[b]) for b in range(len(lens))]
        k, v = tokens(100 + step, len(lens), H, max(new), D, pool.dtype)
        held = [(pool.n_groups(b), pool.lengths[b]) for b in range(len(lens))]
        pool.append(k, v, n_new=new)
        pool.check()
        for b, (kv, ng) in enumerate(before):
            got = cached(pool, b)
            if kv is not None:
                for x, was in zip(got, kv):
                    assert torch.equal(x[:, :ng * G], was[:, :ng * G])
            hot = torch.arange(pool.n_groups(b) * G, pool.lengths[b])
            mine = hot >= held[b][1]
            at = (hot[mine] - held[b][1]).cuda()
            assert torch.equal(got[0][:, hot[mine].cuda()], k[b][:, at].double())
            assert torch.equal(got[1][:, hot[mine].cuda()], v[b][:, at].double())


def test_attention_goes_on_over_what_stayed():
    """Weights added up by a step, an eviction, and the next steps and decodes."""
    print("[evict] run", flush=True)
    pool = make_pool(5, [4000, 2500, 600], 16, 4, room=800)
    weights = torch.zeros((3, 4, pool.max_groups), device="cuda")
    for step in range(4):
        k, v = tokens(200 + step, 3, 4, 150, 128, torch.float16)
        pool.append(k, v)
        q = queries(300 + step, pool, 1)
        pool.attend(q, weights=weights)
        check_eviction(pool, weights, 6)
        out = pool.attend(q)
        dec = pool.decode(q[:, :, 0].contiguous())
        assert float((out[:, :, 0].float() - dec).abs().max()) <= 2.0 ** -9 * float(dec.abs().max())
        for b in range(3):
            kk, vv = cached(pool, b)
            sees = torch.ones((1, pool.lengths[b]), dtype=torch.bool, device="cuda")
            for h in range(4):
                check_rows(out[b, 4 * h:4 * h + 4], q[b, 4 * h:4 * h + 4], kk[h], vv[h], sees, f"step {step} seq {b}")


def test_positions_count_on():
    """append_qkv rotates by the tokens seen, not by those that are left."""
    print("[evict] positions", flush=True)
    from turboquant_pro_amd import norm_rope
    pool = make_pool(6, [2000, 900], 8, 2, room=50)
    weights = some_weights(6, pool)
    pool.evict(weights, 2)
    assert pool.evicted_tokens == [2000 - pool.lengths[0], 900 - pool.lengths[1]] and pool.lengths[0] < 2000
    gen = torch.Generator(device="cuda").manual_seed(6)
    rows = torch.randn((2, 3, 12 * 128), generator=gen, device="cuda").half()
    inv = (10000.0 ** (-torch.arange(64, dtype=torch.float64) / 64)).float().cuda()
    first = torch.tensor([2000, 900], dtype=torch.int32, device="cuda")
    want, k, _ = norm_rope(rows, 8, 2, inv, first)
    assert torch.equal(pool.append_qkv(rows, inv), want)
    assert torch.equal(pool.hot_window_tokens(0)[0][:, -3:], k[0])
    assert torch.equal(pool.append_qkv(rows, inv), norm_rope(rows, 8, 2, inv, first + 3)[0])
    grown = None
    try:
        grown = pool.grown(8000)
    except ValueError:
        pytest.fail("a pool with its own tables grows")
    assert grown.evicted_tokens == pool.evicted_tokens
    for b in range(2):
        for x, y in zip(cached(pool, b), cached(grown, b)):
            assert torch.equal(x, y)
    pool.reset()
    assert pool.evicted_tokens == [0, 0]
    assert torch.equal(pool.append_qkv(rows, inv), norm_rope(rows, 8, 2, inv, torch.zeros_like(first))[0])


def test_reset_gives_the_tables_back():
    print("[evict] reset", flush=True)
    pool = make_pool(7, [5000], 4, 2)
    tables = pool.block_table.clone(), pool.group_table.clone()
    pool.evict(some_weights(1, pool), 5)
    pool.evict(some_weights(2, pool), 3)
    assert not torch.equal(pool.group_table, tables[1])
    pool.reset()
    assert torch.equal(pool.block_table, tables[0]) and torch.equal(pool.group_table, tables[1])


def test_many_groups():
    """More groups than a workgroup's registers hold."""
    print("[evict] many", flush=True)
    pool = make_pool(8, [140000, 9000], 1, 1, 64, hot_window=15, page_tokens=8, outlier_frac=0.0)
    assert pool.n_groups(0) > 1024 * 16
    for keep in (12000, 1000, 7):
        check_eviction(pool, some_weights(keep, pool), keep)


def test_refusals():
    print("[evict] refusals", flush=True)
    pool = make_pool(11, [1300, 800], 8, 2)
    good = torch.zeros((2, 2, pool.max_groups), device="cuda")
    for kw in (dict(keep=1), dict(keep=-1, first=0, last=0), dict(keep=3, first=-1), dict(keep=3, last=-1),
               dict(keep=3, first=3, last=1)):
        with pytest.raises(ValueError):
            pool.evict(good, **kw)
    for bad in (good.double(), good[:1], good[..., :-1], good.cpu(), good.transpose(0, 1)):
        with pytest.raises(ValueError):
            pool.evict(bad, 3)
    with pytest.raises(NotImplementedError):
        pool.evict(good.clone().requires_grad_(), 3)
    import numpy as np
    bias = make_pool(11, [1300], 8, 2, zero_point="bias", rope_theta=10000.0, k_bias=np.zeros((2, 128), np.float32))
    with pytest.raises(NotImplementedError):
        bias.evict(torch.zeros((1, 2, bias.max_groups), device="cuda"), 3)
    assert pool.lengths == [1300, 800] and pool.evicted_tokens == [0, 0]
