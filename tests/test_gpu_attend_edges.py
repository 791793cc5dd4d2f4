"""TQKVPool.attend where it can go wrong: infinities that only some queries see,
hot windows smaller than a block of tokens, first tokens that reach into the hot
window, side-lists longer than a wave takes at once, runs of more blocks than a
wave's tables hold, head dims by query counts, both sides of the number of queries
from which keys and values are reconstructed, several calls under way at once."""

import pytest

torch = pytest.importorskip("torch")

from test_gpu_attend import cached, check, make_pool, queries  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU visible")


@pytest.mark.parametrize("D,Hq,H,dtype", [(64, 4, 1, "float16"), (128, 8, 2, "float16"), (128, 3, 3, "float16"),
                                          (256, 4, 2, "float16"), (128, 4, 2, "float32")])
@pytest.mark.parametrize("T", [1, 2, 4, 9])
def test_infinities_that_some_queries_see(D, Hq, H, dtype, T):
    """An infinity or a NaN in an uncoded value or key changes the rows that see
    its token, there as the formula has it, and no other."""
    print(f"[attend] some see D={D} {Hq}/{H} T={T}", flush=True)
    window, sinks = 90, 2
    pool = make_pool(21, [700, 640], Hq, H, D, input_dtype=dtype)
    q = queries(21, pool, T)
    want = pool.attend(q, window=window, sinks=sinks).clone()
    for bad in (float("inf"), float("-inf"), float("nan")):
        for back in (1, T, window, window + T - 1, window + T):  # tokens from the end: 1 is the last
            for what in ("hot_v", "hot_k"):
                x = getattr(pool, what)
                keep = x.clone()
                ch = 5 * back % D
                for b in range(2):
                    x[b, H - 1, (pool.lengths[b] - back) % pool.hot_window, ch] = bad
                got = pool.attend(q, window=window, sinks=sinks)
                x.copy_(keep)
                t = torch.arange(T)
                sees = (T - t <= back) & (back < window + T - t)  # (query t stands T - t from the end)
                for b in range(2):
                    heads = torch.arange(Hq) // (Hq // H) == H - 1
                    assert torch.equal(got[b][~heads], want[b][~heads])
                    assert torch.equal(got[b][:, ~sees], want[b][:, ~sees])
                    hit, clean = got[b][heads][:, sees], want[b][heads][:, sees]
                    if what == "hot_v":
                        one = torch.zeros(D, dtype=torch.bool)
                        one[ch] = True
                        assert torch.equal(hit[..., ~one], clean[..., ~one])
                        assert bool((hit[..., one] == bad).all()) or (bad != bad and bool(hit[..., one].isnan().all()))
                    elif bad != bad:
                        assert bool(hit.isnan().all())


@pytest.mark.parametrize("hot,page,D", [(1, 1, 128), (7, 1, 128), (24, 12, 64), (31, 16, 128), (40, 20, 256),
                                        (64, 32, 128), (96, 48, 128), (130, 65, 128), (512, 8, 128)])
def test_small_hot_windows_and_pages(hot, page, D):
    """Groups shorter than a block of 32 tokens and no multiple of it, pages that
    end inside a tile, windows and first tokens across the hot window's start."""
    print(f"[attend] hot {hot} page {page} D={D}", flush=True)
    pool = make_pool(22, [3 * hot + 70, hot + 1, hot, 2], 4, 2, D, hot_window=hot, page_tokens=page)
    for T in (1, 2, 5):
        q = queries(T, pool, T)
        for window, sinks in ((None, 0), (1, 0), (2, 1), (hot + 3, 0), (33, hot + 40), (5, 3 * hot + 60), (1, 10 ** 6)):
            out = pool.attend(q, window=window, sinks=sinks)
            check(pool, out, q, window, sinks, what=f"T={T} window={window} sinks={sinks}")


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("key", [dict(), dict(key_grid="uniform", key_bits=3), dict(key_grid="uniform", key_bits=2)])
def test_long_side_lists(D, key):
    """More side-list entries in a block of tokens than a wave brings at once."""
    print(f"[attend] lists D={D} {key}", flush=True)
    for frac in (0.03, 0.2):
        pool = make_pool(23, [1500, 800], 4, 1, D, outlier_frac=frac, **key)
        for T in (1, 6):
            q = queries(T, pool, T)
            for window, sinks in ((None, 0), (700, 40)):
                check(pool, pool.attend(q, window=window, sinks=sinks), q, window, sinks, what=f"{frac} T={T}")


@pytest.mark.parametrize("D,lens", [(128, [17100, 16900] + [60] * 30), (64, [17100, 16900] + [60] * 30),
                                    (128, [20000]), (128, [9000 - 150 * i for i in range(40)])])
def test_long_runs(D, lens):
    """Runs past the 64 blocks whose table entries a wave holds at once (as many
    heads as workgroups fit: no splits), and many splits of one sequence."""
    print(f"[attend] long runs D={D} {len(lens)}", flush=True)
    pool = make_pool(24, lens, 8, 8, D)
    for T in (1, 2):
        q = queries(T, pool, T)
        out = pool.attend(q)
        check(pool, out, q, None, 0, what=f"T={T}")
        assert torch.equal(out, pool.attend(q, window=10 ** 9, sinks=7))


@pytest.mark.parametrize("D,Hq,H,T", [(64, 8, 1, 16), (64, 8, 1, 17), (128, 8, 2, 32), (128, 8, 2, 33), (128, 4, 4, 128),
                                      (128, 4, 4, 129), (256, 4, 1, 32), (256, 4, 1, 33)])
def test_both_sides_of_the_query_count(D, Hq, H, T):
    """As many rows as are attended on the codes, and the first count past it;
    what no query sees hidden in both."""
    print(f"[attend] rows D={D} {Hq}/{H} T={T}", flush=True)
    pool = make_pool(25, [1900, 700, 90], Hq, H, D)
    q = queries(25, pool, T)
    for window, sinks in ((None, 0), (250, 3), (30, 0)):
        out = pool.attend(q, window=window, sinks=sinks)
        check(pool, out, q, window, sinks, what=f"window={window}")
        if window is not None:
            first = 1900 - T - window + 1
            G = pool.group_tokens
            keep = pool.vnorm.clone(), pool.gscale.clone()
            for g in range(pool.n_groups(0)):
                t = torch.arange(g * G, (g + 1) * G, device="cuda")
                hidden = (t < first) & (t >= sinks)
                phys, off = pool._rows(0, g)
                pool.vnorm[:, phys[hidden], off[hidden]] = float("inf")
                if bool(hidden.all()):
                    pool.gscale[int(pool.group_table[0, g])] = float("nan")
            again = pool.attend(q, window=window, sinks=sinks)
            pool.vnorm.copy_(keep[0])
            pool.gscale.copy_(keep[1])
            assert torch.equal(again, out)


def test_calls_at_once():
    """Calls on three streams over one pool, their workspaces apart, and one on
    queries that the stream before still writes."""
    print("[attend] at once", flush=True)
    pool = make_pool(26, [7000, 3000, 64], 32, 8)
    args = [dict(window=2000, sinks=4), dict(), dict(window=64)]
    qs = [queries(i, pool, T) for i, T in enumerate((1, 40, 3))]
    want = [pool.attend(q, **a).clone() for q, a in zip(qs, args)]
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for s, q, a in zip(streams, qs, args):
            with torch.cuda.stream(s):
                got.append(pool.attend(q * 1.0, **a))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert torch.equal(g, w)


def test_a_captured_step_between_other_calls():
    """A captured step replayed after calls of other sizes on the same pool."""
    print("[attend] capture", flush=True)
    pool = make_pool(27, [2000, 900], 8, 2)
    q, more = queries(27, pool, 1), queries(28, pool, 40)
    want = pool.attend(q, window=700, sinks=4).clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = pool.attend(q, window=700, sinks=4)
    for i in range(3):
        graph.replay()
        pool.attend(more, window=100 + i)
        pool.attend(more[:, :, :5])
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
        out.zero_()


@pytest.mark.parametrize("D,Hq,H,T", [(64, 8, 1, 50), (128, 8, 2, 100), (256, 4, 1, 90)])
def test_chunks_keep_what_rounding_keys_leaves(D, Hq, H, T):
    """A chunk's reconstructed keys are fp16 pairs: with keys of large scores the
    result is as close as on the codes, 2^-10 together (the weights', values' and
    output's roundings, each at most 2^-11 and rarely near it)."""
    from test_gpu_attend import attention, visible
    print(f"[attend] pairs D={D} T={T}", flush=True)
    pool = make_pool(29, [2300, 1200], Hq, H, D, value_bits=4)
    q = (3.0 * queries(29, pool, T)).half()
    out = pool.attend(q, window=900, sinks=4)
    check(pool, out, q, 900, 4, what="pairs")
    off = tot = 0.0
    for b in range(2):
        k, v = cached(pool, b)
        sees = visible(pool.lengths[b], T, T, 0, 900, 4, "cuda")
        want = attention(q[b], k, v, sees, D ** -0.5)[0]
        off += float((out[b].double() - want).square().sum())
        tot += float(want.square().sum())
    assert (off / tot) ** 0.5 <= 2.0 ** -10
