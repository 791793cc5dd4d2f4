"""A prefix that is read once for all sequences, in every way that its steps are used:
which batches it is read once for, captured and replayed steps, other streams,
evictions, growth and resets, numbers that are not finite."""

import pytest

torch = pytest.importorskip("torch")

from more_ref import make_pool, queries, tokens  # noqa: E402
from test_gpu_shared_prefix import ONCE, check, read_once, shared_pool  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU visible")


def once_pool(seed, B=64, prefix=4000, Hq=32, H=8, D=128, room=0, **kw):
    return shared_pool(seed, prefix, [(37 * b) % 130 + 3 for b in range(B)], Hq, H, D, room=room, **kw)


# one, three and sixteen queries of every form there (the time of each sequence for itself
# against that of the prefix's workgroups in rounds of 256)
@pytest.mark.parametrize("form,want", list(zip(ONCE, [
    (True, True, True), (True, True, False), (True, True, True), (True, False, False), (True, False, False),
    (True, True, True), (True, False, False), (True, False, False), (True, False, False), (True, True, True),
    (True, True, True), (True, True, True)])))
def test_which_steps_read_the_prefix_once(form, want):
    prefix, B, Hq, H, D, kw = form
    print(f"[once] {prefix} x {B} {Hq}/{H} D={D} {kw}", flush=True)
    pool = shared_pool(3, prefix, [16 + b % 3 for b in range(B)], Hq, H, D, **kw)
    got = tuple(read_once(pool, T) for T in (1, 3, 16))
    assert got == tuple(x and T * Hq // H <= 128 for x, T in zip(want, (1, 3, 16)))


@pytest.mark.parametrize("T", [1, 2])
def test_captured_steps_share_nothing(T):
    """Two graphs of two pools' steps, replayed in turn with eager work between."""
    print(f"[once] graphs T={T}", flush=True)
    pools = [once_pool(8), once_pool(9, 40, Hq=16, D=256, value_bits=4)]
    qs = [queries(80 + i, p, T) for i, p in enumerate(pools)]
    assert all(read_once(p, T) for p in pools)
    eager = [p.attend(q).clone() for p, q in zip(pools, qs)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    for p, q in zip(pools, qs):
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(p.attend(q))
        graphs.append(g)
    for _ in range(3):
        for i in (0, 1):
            graphs[i].replay()
            assert torch.equal(pools[1 - i].attend(qs[1 - i]), eager[1 - i])
        torch.cuda.synchronize()
        for x, y in zip(outs, eager):
            assert torch.equal(x, y)
        for x in outs:
            x.fill_(7.0)
        torch.rand(1000, device="cuda").sort()
    # new queries in the captured ones' place
    qs[0].copy_(queries(90, pools[0], T))
    graphs[0].replay()
    assert torch.equal(outs[0], pools[0].attend(qs[0]))


def test_streams_side_by_side():
    print("[once] streams", flush=True)
    pools = [once_pool(10), once_pool(11, 90, Hq=16, D=64, value_bits=3, hot_window=64)]
    assert all(read_once(p, 1) for p in pools)
    qs = [queries(9 + i, p, 1) for i, p in enumerate(pools)]
    want = [p.attend(q) for p, q in zip(pools, qs)]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for p, q, y in zip(pools, qs, want):
            with torch.cuda.stream(torch.cuda.Stream()):
                got.append((p.attend(q), y))
    torch.cuda.synchronize()
    for x, y in got:
        assert torch.equal(x, y)


def test_appends_evictions_growth_and_resets():
    print("[once] life", flush=True)
    pool = once_pool(6, room=2500)
    B, S, only = 64, pool._shared, [0, 5, 33, 63]
    for step in range(3):
        k, v = tokens(60 + step, B, 8, 700, 128, torch.float16)
        pool.append(k, v, n_new=[700 - 9 * (b % 40) for b in range(B)])
        weights = torch.rand((B, 8, pool.max_groups), device="cuda")
        kept = pool.evict(weights, S + 1, first=0, last=step % 2)
        assert kept[:, :S].tolist() == [list(range(S))] * B
        for T in (1, 2):
            assert read_once(pool, T)
            q = queries(step, pool, T)
            check(pool, pool.attend(q), q, what=f"step {step} T={T}", only=only)
    q = queries(7, pool, 1)
    want = pool.attend(q)
    grown = pool.grown(pool.max_seq_len + 1000)
    assert grown._shared == 0 and float((grown.attend(q) - want).abs().max()) <= 2.0 ** -8 * float(want.abs().max())
    tables = pool.block_table.clone()
    pool.reset()
    assert not torch.equal(tables, pool.block_table) and not pool._shared_step(1, 0, 1)
    k, v = tokens(70, B, 8, 900, 128, torch.float16)
    pool.append(k, v)
    check(pool, pool.attend(q), q, what="after reset", only=only)


@pytest.mark.parametrize("D,Hq,form", [(128, 32, dict()), (64, 32, dict(value_bits=4)), (256, 16, dict(value_bits=4))])
def test_a_prefix_that_lost_groups(D, Hq, form):
    """Shared after an eviction: the first sequence's table is in another order."""
    print(f"[once] evicted prefix D={D}", flush=True)
    B, source = 90, 7
    pool = make_pool(12, [9000 if b == source else 0 for b in range(B)], Hq, 8, D, room=200, **form)
    gen = torch.Generator(device="cuda").manual_seed(1)
    pool.evict(torch.rand((B, 8, pool.max_groups), generator=gen, device="cuda"), 14)
    pool.share_prefix(source)
    k, v = tokens(13, B, 8, 130, D, torch.float16)
    pool.append(k, v, n_new=[(37 * b) % 130 + 1 for b in range(B)])
    assert pool._shared == 14 and read_once(pool, 1)
    q = queries(14, pool, 1)
    check(pool, pool.attend(q), q, only=[0, source, B - 1])


@pytest.mark.parametrize("D,Hq,form", [(128, 32, dict()), (256, 16, dict(value_bits=4))])
def test_numbers_that_are_not_finite(D, Hq, form):
    """A NaN of the prefix's levels or norms takes its kv head's rows, of all sequences;
    an infinite value of a sequence's own tokens its channel of that sequence's rows,
    however small its weight; every other number stays as it is."""
    print(f"[once] not finite D={D}", flush=True)
    B, gq = 64, Hq // 8
    pool = once_pool(15, B, Hq=Hq, D=D, **form)
    q = queries(16, pool, 1)
    q[..., 3] = 1.0
    assert read_once(pool, 1)
    # a hot token that nobody gives a weight that 64 bits hold
    b, h, at = 40, 5, (pool.lengths[40] - 2) % pool.hot_window
    pool.hot_k[b, h, at] = 0.0
    pool.hot_k[b, h, at, 3] = -60000.0
    pool.hot_v[b, h, at, 11] = 0.0
    want = pool.attend(q)
    for x in (float("inf"), float("-inf"), float("nan")):
        pool.hot_v[b, h, at, 11] = x
        got = pool.attend(q)
        rows = got[b, h * gq:(h + 1) * gq, 0, 11].clone()
        assert bool(torch.equal(rows.isnan(), torch.full_like(rows, x).isnan())) and bool(((rows == x) | rows.isnan()).all())
        got[b, h * gq:(h + 1) * gq, 0, 11] = want[b, h * gq:(h + 1) * gq, 0, 11]
        assert torch.equal(got, want)
    pool.hot_v[b, h, at, 11] = 0.0
    slot, (phys, off) = int(pool.group_table[0, 2]), pool._rows(0, 3)
    for kind, where in (("scale", pool.gscale[slot, 6]), ("mean", pool.gmean[slot, 6]), ("norm", pool.vnorm[6, phys[:1], off[:1]])):
        was = where.clone()
        if kind == "norm":
            pool.vnorm[6, phys[:1], off[:1]] = float("nan")
        else:
            where[9] = float("nan")
        got = pool.attend(q)
        assert bool(got[:, 6 * gq:7 * gq].isnan().all()), kind
        got[:, 6 * gq:7 * gq] = want[:, 6 * gq:7 * gq]
        assert torch.equal(got, want), kind
        if kind == "norm":
            pool.vnorm[6, phys[:1], off[:1]] = was
        else:
            where.copy_(was)
    assert torch.equal(pool.attend(q), want)
