"""TQKVPool.share_prefix and the attention over a prefix that all sequences share,
against 64 bits over the cache's own reconstruction; appends, evictions and resets of
such a pool, captured steps."""

import math

import pytest

torch = pytest.importorskip("torch")

from attn_ref import visible  # noqa: E402
from more_ref import cached, check_rows, queries, tokens  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU visible")


def shared_pool(seed, prefix, more, Hq, H, D=128, source=0, room=0, **kw):
    """A prefix of the source's, shared, then ``more[b]`` tokens of each sequence."""
    from turboquant_pro_amd import TQKVPool
    B = len(more)
    pool = TQKVPool(n_kv_heads=H, n_q_heads=Hq, head_dim=D, max_batch=B, max_seq_len=prefix + max(more) + room, seed=seed,
                    **kw)
    k, v = tokens(seed, B, H, prefix, D, pool.dtype)
    pool.append(k, v, n_new=[prefix if b == source else 0 for b in range(B)])
    pool.share_prefix(source)
    if max(more):
        k2, v2 = tokens(seed + 1, B, H, max(more), D, pool.dtype)
        pool.append(k2, v2, n_new=more)
    pool.check()
    return pool


def read_once(pool, T):
    """Whether a step of T queries reads the prefix once, through the first sequence's
    table: it then takes no notice of what the others' say of the prefix."""
    if not pool._shared_step(T, 0, max(pool.lengths)):
        return False
    q, keep = queries(T, pool, T), pool.block_table.clone()
    pages = pool._shared * pool.group_tokens // pool.page_tokens
    want = pool.attend(q)
    pool.block_table[1:, :pages] = keep[1:, :pages].flip(1)
    got = pool.attend(q)
    pool.block_table.copy_(keep)
    return torch.equal(got, want)


def check(pool, out, q, q_lens=None, what="", only=None):
    B, Hq, T, D = q.shape
    H = pool.n_kv_heads
    gq = Hq // H
    off = tot = 0.0
    for b in range(B) if only is None else only:
        n, m = pool.lengths[b], T if q_lens is None else q_lens[b]
        k, v = cached(pool, b)
        sees = visible(n, m, T, 0, None, 0, "cuda")
        for h in range(H):
            s = slice(h * gq, (h + 1) * gq)
            e, w = check_rows(out[b, s], q[b, s], k[h], v[h], sees, f"{what} seq {b} head {h}")
            off, tot = off + e, tot + w
    # random roundings do not add up as the bound allows: together 2^-10 of the output
    assert math.sqrt(off / max(tot, 1e-30)) <= 2.0 ** -10, what


FORMS = [
    # prefix, tokens of each after it, Hq, H, D, form
    (2600, [700, 3, 0, 1400], 32, 8, 128, dict()),
    (5000, [600, 20, 300, 1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 13, 14, 15], 8, 2, 128, dict(value_bits=4)),
    (1300, [200, 80], 7, 1, 128, dict(hot_window=64, page_tokens=16, value_bits=2)),
    (700, [100, 31], 4, 2, 128, dict(hot_window=47, page_tokens=12)),
    (900, [600, 90], 4, 4, 128, dict(key_grid="polar", key_bits=3, value_bits=3)),
    (2100, [90, 600], 4, 1, 64, dict(value_bits=4)),
    (2100, [90, 600, 7], 16, 8, 256, dict(value_bits=3)),
    (900, [300, 9], 8, 1, 256, dict(key_grid="uniform", key_bits=2, hot_window=64)),
    (900, [300, 9], 2, 1, 64, dict(key_grid="uniform", key_bits=3, outlier_frac=0.0, hot_window=64)),
]


@pytest.mark.parametrize("prefix,more,Hq,H,D,form", FORMS)
def test_attention_over_a_shared_prefix(prefix, more, Hq, H, D, form):
    print(f"[shared] {prefix} {more} {Hq}/{H} D={D} {form}", flush=True)
    pool = shared_pool(3, prefix, more, Hq, H, D, **form)
    assert pool._shared > 0
    for T in (1, 3, 16):
        q = queries(T, pool, T)
        assert pool._shared_step(T, 0, max(pool.lengths)) == (T * Hq // H <= 128 and pool.key_grid != "polar")
        out = pool.attend(q)
        check(pool, out, q, what=f"T={T}")
        assert torch.equal(out, pool.attend(q))
        assert torch.equal(out, pool.attend(q, window=10 ** 6))
        ql = [(b + T) % (T + 1) for b in range(len(more))]
        check(pool, pool.attend(q, q_lens=torch.tensor(ql, dtype=torch.int32, device="cuda")), q, ql, f"ragged T={T}")


ONCE = [
    # prefix, sequences, Hq, H, D, form: batches that read the prefix once
    (4000, 64, 32, 8, 128, dict()),
    (4000, 64, 8, 8, 128, dict(value_bits=4, outlier_frac=0.1)),
    (4000, 90, 56, 8, 128, dict(value_bits=2, hot_window=64)),
    (1400, 90, 16, 8, 128, dict(key_grid="uniform", key_bits=3, hot_window=47, page_tokens=12)),
    (1400, 90, 16, 8, 128, dict(value_bits=2, hot_window=48, page_tokens=8)),
    (1400, 90, 16, 8, 128, dict(value_bits=4, hot_window=15, page_tokens=4, outlier_frac=0.5)),
    (4000, 90, 32, 8, 64, dict(value_bits=4)),
    (4000, 90, 16, 8, 64, dict(value_bits=3, hot_window=64)),
    (4000, 90, 16, 8, 64, dict(value_bits=2, key_grid="uniform", key_bits=4, outlier_frac=0.0)),
    (4000, 40, 16, 8, 256, dict(value_bits=3)),
    (4000, 40, 8, 8, 256, dict(value_bits=4, outlier_frac=0.1)),
    (4000, 40, 32, 8, 256, dict(value_bits=2, key_grid="uniform", key_bits=2, hot_window=100, page_tokens=10)),
]


@pytest.mark.parametrize("prefix,B,Hq,H,D,form", ONCE)
def test_a_prefix_read_once(prefix, B, Hq, H, D, form):
    """One and several queries, rows past a workgroup's, tiles and blocks that end short."""
    print(f"[shared] once {prefix} x {B} {Hq}/{H} D={D} {form}", flush=True)
    more = [(37 * b) % 130 + 3 for b in range(B)]
    pool = shared_pool(3, prefix, more, Hq, H, D, **form)
    only = [0, 1, 31, B - 1]
    for T in (1, 3):
        q = queries(T, pool, T)
        assert read_once(pool, T) or (T > 1 and Hq // H < 7)  # (few rows a sequence: 16 go together for each)
        out = pool.attend(q)
        check(pool, out, q, what=f"T={T}", only=only)
        assert torch.equal(out, pool.attend(q))
        ql = [(b + T) % (T + 1) for b in range(B)]
        check(pool, pool.attend(q, q_lens=torch.tensor(ql, dtype=torch.int32, device="cuda")), q, ql, f"ragged T={T}", only)
    # as each sequence for itself, but for the roundings of weights and centroids
    q = queries(5, pool, 1)
    got, pool._shared = pool.attend(q).float(), 0
    want = pool.attend(q).float()
    assert float((got - want).abs().max()) <= 2.0 ** -8 * float(want.abs().max())


def test_a_shared_pool_holds_what_separate_ones_do():
    """Codes, windows, decodes and chunks as without sharing."""
    print("[shared] as separate", flush=True)
    from turboquant_pro_amd import TQKVPool
    prefix, more = 3000, [400, 900, 30]
    for source in (0, 2):
        pool = shared_pool(4, prefix, more, 8, 2, source=source)
        k, v = tokens(4, 3, 2, prefix, 128, torch.float16)
        k2, v2 = tokens(5, 3, 2, max(more), 128, torch.float16)
        other = TQKVPool(n_kv_heads=2, n_q_heads=8, max_batch=3, max_seq_len=prefix + 900, seed=4)
        other.append(k[source].expand(3, -1, -1, -1), v[source].expand(3, -1, -1, -1))
        other.append(k2, v2, n_new=more)
        for b in range(3):
            assert pool.lengths[b] == other.lengths[b]
            for x, y in zip(cached(pool, b), cached(other, b)):
                assert torch.equal(x, y)
        q = queries(4, pool, 1)
        assert torch.equal(pool.decode(q[:, :, 0].contiguous()), other.decode(q[:, :, 0].contiguous()))
        assert torch.equal(pool.attend(q, window=500, sinks=3), other.attend(q, window=500, sinks=3))
        q = queries(5, pool, 60)
        assert torch.equal(pool.attend(q), other.attend(q))
        grown = pool.grown(9000)
        assert torch.equal(grown.attend(q), other.attend(q)) and grown._shared == 0


def test_queries_inside_the_prefix_and_short_prefixes():
    print("[shared] inside", flush=True)
    pool = shared_pool(5, 1500, [0, 0, 0], 8, 2, hot_window=64)
    for T in (1, 10, 32):
        q = queries(T, pool, T)
        check(pool, pool.attend(q), q, what=f"T={T}")
    short = shared_pool(5, 40, [3, 0, 700], 8, 2, hot_window=64)
    assert short._shared == 0
    q = queries(5, short, 3)
    check(short, short.attend(q), q)
    one = shared_pool(5, 700, [3], 8, 2, hot_window=64)
    check(one, one.attend(queries(1, one, 1)), queries(1, one, 1))


def test_appends_evictions_and_resets():
    print("[shared] life", flush=True)
    pool = shared_pool(6, 2000, [100, 200], 8, 2, room=3000)
    S, G = pool._shared, pool.group_tokens
    first = [x[:, :S * G].clone() for x in cached(pool, 0)]
    for step in range(3):
        k, v = tokens(60 + step, 2, 2, 700, 128, torch.float16)
        pool.append(k, v, n_new=[700, 500])
        for b in range(2):
            for x, was in zip(cached(pool, b), first):
                assert torch.equal(x[:, :S * G], was)
        weights = torch.rand((2, 2, pool.max_groups), device="cuda")
        kept = pool.evict(weights, S + 2, first=0, last=1)
        assert kept[:, :S].tolist() == [list(range(S))] * 2
        q = queries(step, pool, 2)
        assert pool._shared_step(2, 0, max(pool.lengths))
        check(pool, pool.attend(q), q, what=f"step {step}")
    with pytest.raises(ValueError):
        pool.evict(weights, S, first=0, last=1)
    with pytest.raises(ValueError):
        pool.import_group(1, 0, values=dict(vpacked=None, vnorms=None))
    with pytest.raises(ValueError):
        pool.share_prefix(0)
    tables = pool.block_table.clone()
    pool.reset()
    assert pool._shared == 0 and not torch.equal(tables, pool.block_table)
    k, v = tokens(70, 2, 2, 1500, 128, torch.float16)
    pool.append(k, v)
    q = queries(7, pool, 1)
    check(pool, pool.attend(q), q, what="after reset")


def test_captured_steps_share_nothing():
    """Two graphs of two pools' steps, replayed in turn with eager work between."""
    print("[shared] graphs", flush=True)
    pools = [shared_pool(8 + i, 1500, [300, 5, 60], 8, 2) for i in range(2)]
    qs = [queries(80 + i, p, 1) for i, p in enumerate(pools)]
    weights = [torch.zeros((3, 2, p.max_groups), device="cuda") for p in pools]
    eager = []
    for p, q, w in zip(pools, qs, weights):
        groups = p.select_groups(q, 3)
        eager.append((p.attend(q).clone(), groups.clone(), p.attend(q, groups=groups).clone()))
        p.attend(q, weights=w)
    want = [w.clone() for w in weights]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    for p, q, w in zip(pools, qs, weights):
        w.zero_()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            a = p.attend(q)
            groups = p.select_groups(q, 3)
            b = p.attend(q, groups=groups)
            w.zero_()
            p.attend(q, weights=w)
        graphs.append(g)
        outs.append((a, groups, b))
    for _ in range(3):
        for i in (0, 1):
            graphs[i].replay()
            pools[1 - i].attend(qs[1 - i])
        torch.cuda.synchronize()
        for i in (0, 1):
            for x, y in zip(outs[i], eager[i]):
                assert torch.equal(x, y)
            assert torch.equal(weights[i], want[i])
        torch.rand(1000, device="cuda").sort()
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError):
        with torch.cuda.graph(g, stream=side):
            pools[0].evict(weights[0], pools[0].max_groups)


def test_another_stream():
    print("[shared] streams", flush=True)
    pool = shared_pool(9, 1500, [300, 5], 8, 2)
    q = queries(9, pool, 1)
    want, groups = pool.attend(q), pool.select_groups(q, 3)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append((pool.attend(q), pool.select_groups(q, 3), pool.attend(q, groups=groups)))
    torch.cuda.synchronize()
    for a, b, c in got:
        assert torch.equal(a, want) and torch.equal(b, groups) and torch.equal(c, got[0][2])


def test_refusals():
    print("[shared] refusals", flush=True)
    from turboquant_pro_amd import TQKVPool
    pool = TQKVPool(n_kv_heads=2, n_q_heads=8, max_batch=3, max_seq_len=2000, seed=1)
    for bad in (0, -1, 3):
        with pytest.raises(ValueError):
            pool.share_prefix(bad)
    k, v = tokens(1, 3, 2, 700, 128, torch.float16)
    pool.append(k, v, n_new=[700, 1, 0])
    with pytest.raises(ValueError):
        pool.share_prefix(0)
    f32 = shared_pool(2, 900, [40, 2], 4, 2, input_dtype="float32", hot_window=64)
    q = queries(1, f32, 1)
    out = f32.attend(q)
    for b in range(2):
        kk, vv = cached(f32, b)
        s = torch.softmax(q[b].double().view(2, 2, 128) @ kk.transpose(1, 2) / math.sqrt(128), -1)
        want = (s @ vv).view(4, 1, 128)
        assert float((out[b].double() - want).abs().max()) <= 1e-5 * float(want.abs().max())
