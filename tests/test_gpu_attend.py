"""TQKVPool.attend (windowed attention of one or more new queries over the coded
cache) and append_qkv against 64-bit attention over the cache's own
reconstruction: key and value forms, head layouts, hot windows, pages, ragged
lengths, queries before the first token, hidden infinities, streams, graphs."""

import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from attn_ref import HALF, attention, visible  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU visible")


def tokens(seed, B, H, L, D, dtype):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    scale = torch.exp(torch.randn((B, H, 1, D), generator=gen, device="cuda"))
    k = (torch.randn((B, H, L, D), generator=gen, device="cuda") * scale).to(dtype)
    v = torch.randn((B, H, L, D), generator=gen, device="cuda").to(dtype)
    return k, v


def make_pool(seed, lens, Hq, H, D=128, **kw):
    from turboquant_pro_amd import TQKVPool
    pool = TQKVPool(n_kv_heads=H, n_q_heads=Hq, head_dim=D, max_batch=len(lens), max_seq_len=max(max(lens), 1), seed=seed,
                    **kw)
    k, v = tokens(seed, len(lens), H, max(max(lens), 1), D, pool.dtype)
    pool.append(k, v, n_new=lens)
    pool.check()
    return pool


def cached(pool, b):
    """Keys and values (H, n, D) of sequence b as the cache holds them."""
    H, D, ng = pool.n_kv_heads, pool.head_dim, pool.n_groups(b)
    ks, vs = [], []
    if ng:
        k, v = pool.dequant_groups([(b, g) for g in range(ng)])
        ks, vs = ([x.permute(1, 0, 2, 3).reshape(H, -1, D).double()] for x in (k, v))
    hk, hv = pool.hot_window_tokens(b)
    return torch.cat(ks + [hk.double()], 1), torch.cat(vs + [hv.double()], 1)


def check(pool, out, q, window, sinks, q_lens=None, what=""):
    """The split kernels round the value centroids to fp16 (half a step of each,
    which the rotation spreads over the channels: half a step of sum p |v|_2) and
    carry the rest as fp16 pairs or fp32 (32 units in the last place of fp32 of
    the scores' products, and of the weights and sums).  Over reconstructed keys
    and values these are rounded to fp16 too, and the weights."""
    B, Hq, T, D = q.shape
    scale = 1.0 / math.sqrt(D)
    dtype = q.dtype
    assert out.dtype == dtype and out.shape == q.shape
    dense = dtype == torch.float16 and T > 8
    off = tot = 0.0
    for b in range(B):
        n, m = pool.lengths[b], T if q_lens is None else q_lens[b]
        sees = visible(n, m, T, 0, window, sinks, "cuda")
        if n == 0:
            assert bool((out[b] == 0).all())
            continue
        k, v = cached(pool, b)
        want, weighted, mag, vmax = attention(q[b], k, v, sees, scale)
        size = attention(q[b], k, v.norm(dim=-1, keepdim=True).expand_as(v).contiguous(), sees, scale)[0]
        half = HALF[torch.float16] if dtype == torch.float16 else 0.0
        score = 2 * scale * mag * (HALF[torch.float16] if dense else 0.0) + 2 * scale * mag * (32 + D) * 2.0 ** -24
        tol = HALF[dtype] * want.abs() + (score + (n / 16 + 64) * 2.0 ** -23) * size + half * size
        if dense:
            tol = tol + (2 * half) * weighted + n * 2.0 ** -25 * vmax
        if dtype == torch.float16:
            tol = tol + 2.0 ** -25
        got = out[b].double()
        assert torch.isfinite(got).all(), f"{what} seq {b}"
        err = (got - want).abs()
        assert bool((err <= tol).all()), f"{what} seq {b}: {float((err - tol).max()):.3e} past the bound"
        empty = ~sees.any(1)
        assert bool((out[b][:, empty] == 0).all())
        off += float(err.square().sum())
        tot += float(want.square().sum())
    # random roundings do not add up as the bound allows: together 2^-9 of the
    # output (2^-10 where keys keep their 32 bits, 2^-15 for fp32 caches)
    rel = math.sqrt(off / max(tot, 1e-30))
    assert rel <= (2.0 ** -15 if dtype == torch.float32 else 2.0 ** -9 if dense else 2.0 ** -10), f"{what} rel {rel:.2e}"


def queries(seed, pool, T):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn((pool.max_batch, T, pool.n_q_heads, pool.head_dim), generator=gen,
                       device="cuda").to(pool.dtype).transpose(1, 2)


FORMS = [
    # lens, Hq, H, D, pool form
    ([5000, 1300, 700], 32, 8, 128, dict()),
    ([2600, 513], 8, 2, 128, dict(value_bits=4)),
    ([1400, 40], 7, 1, 128, dict(value_bits=2, page_tokens=16)),
    ([1500, 900], 2, 1, 128, dict(key_grid="uniform", key_bits=3, outlier_frac=0.0)),
    ([1500, 900], 4, 4, 128, dict(key_grid="polar", key_bits=3, value_bits=3)),
    ([1500, 900], 8, 1, 128, dict(hot_window=64, value_bits=3)),
    ([700, 150], 4, 2, 128, dict(hot_window=48, page_tokens=24)),
    ([2100, 600], 4, 1, 64, dict(value_bits=4)),
    ([2100, 600], 16, 8, 256, dict(value_bits=3)),
    ([900, 300], 8, 1, 256, dict(key_grid="uniform", key_bits=2, hot_window=64)),
    ([1700, 700], 4, 1, 128, dict(input_dtype="float32")),
    ([900, 200], 2, 2, 256, dict(input_dtype="float32", hot_window=64)),
]


@pytest.mark.parametrize("lens,Hq,H,D,form", FORMS)
def test_attend_against_the_reconstructed_cache(lens, Hq, H, D, form):
    print(f"[attend] {lens} {Hq}/{H} D={D} {form}", flush=True)
    pool = make_pool(3, lens, Hq, H, D, **form)
    for T in (1, 3, 33):
        q = queries(T, pool, T)
        for window, sinks in ((None, 0), (1, 0), (300, 4), (600, 257), (20, 33), (100000, 2)):
            out = pool.attend(q, window=window, sinks=sinks)
            check(pool, out, q, window, sinks, what=f"T={T} window={window} sinks={sinks}")
            assert torch.equal(out, pool.attend(q, window=window, sinks=sinks))


def test_attend_without_a_window_is_decode():
    """One query over the whole cache: the decode's result, rounded."""
    print("[attend] decode", flush=True)
    pool = make_pool(4, [3000, 700], 32, 8)
    q = queries(4, pool, 1)
    got, want = pool.attend(q)[:, :, 0].float(), pool.decode(q[:, :, 0].contiguous())
    # two roundings of the centroids apart, and the output's
    assert float((got - want).abs().max()) <= 2.0 ** -9 * float(want.abs().max())


def test_ragged_queries_and_short_sequences():
    """Lengths of zero and one, fewer tokens than queries, fewer queries than rows."""
    print("[attend] ragged", flush=True)
    for dtype, D in (("float16", 128), ("float16", 64), ("float32", 128)):
        pool = make_pool(5, [0, 1, 4, 600, 1100, 530], 8, 2, D, input_dtype=dtype)
        for T, m in ((6, [0, 1, 6, 2, 6, 0]), (20, [20, 3, 20, 20, 7, 1])):
            q = queries(T, pool, T)
            ql = torch.tensor(m, dtype=torch.int32, device="cuda")
            for window, sinks in ((None, 0), (200, 3)):
                check(pool, pool.attend(q, window=window, sinks=sinks, q_lens=ql), q, window, sinks, m, f"{dtype} T={T}")
                check(pool, pool.attend(q, window=window, sinks=sinks), q, window, sinks, None, f"{dtype} T={T}")
    empty = make_pool(5, [0], 8, 2)
    q = queries(1, empty, 2)
    assert bool((empty.attend(q, window=4) == 0).all())
    assert empty.attend(q[:, :, :0]).shape == (1, 8, 0, 128)


def test_out_strides_and_refusals():
    print("[attend] out", flush=True)
    pool = make_pool(6, [1300, 800], 8, 2)
    for T in (1, 40):
        q = queries(T, pool, T)
        want = pool.attend(q, window=300, sinks=4)
        big = torch.full((2, T + 1, 9, 136), 7.0, dtype=torch.float16, device="cuda")
        view = big[:, :T, :8, :128].transpose(1, 2)
        assert pool.attend(q.contiguous(), window=300, sinks=4, out=view) is view
        assert torch.equal(view, want)
        big[:, :T, :8, :128] = 7.0
        assert bool((big == 7.0).all())
    q = queries(1, pool, 1)
    for bad in (dict(window=0), dict(sinks=-1), dict(q_lens=torch.zeros(2, device="cuda")),
                dict(q_lens=torch.zeros(2, dtype=torch.int32)), dict(out=torch.empty_like(q).float()),
                dict(out=torch.empty((2, 8, 1, 128), dtype=torch.float16))):
        with pytest.raises(ValueError):
            pool.attend(q, **bad)
    for x in (q.float(), q[:, :4], q[:1], q[..., :64], q[:, :, 0], q.cpu()):
        with pytest.raises(ValueError):
            pool.attend(x)


@pytest.mark.parametrize("D,dtype", [(128, "float16"), (256, "float16"), (128, "float32")])
@pytest.mark.parametrize("T", [1, 30])
def test_what_no_query_sees_is_not_read(D, dtype, T):
    """NaN in every norm, scale and hot token that no query sees leaves the
    result as it was."""
    print(f"[attend] hidden D={D} {dtype} T={T}", flush=True)
    pool = make_pool(7, [3000, 2000], 8, 2, D, input_dtype=dtype)
    for window, sinks in ((900, 5), (100, 0), (100, 300)):
        q = queries(T, pool, T)
        want = pool.attend(q, window=window, sinks=sinks).clone()
        keep = {n: getattr(pool, n).clone() for n in ("gscale", "vnorm", "hot_k", "hot_v")}
        for b in range(2):
            L, G, ng = pool.lengths[b], pool.group_tokens, pool.n_groups(b)
            first = L - T - window + 1
            for g in range(ng):
                t = torch.arange(g * G, (g + 1) * G, device="cuda")
                hidden = (t < first) & (t >= sinks)
                phys, off = pool._rows(b, g)
                pool.vnorm[:, phys[hidden], off[hidden]] = float("nan")
                if bool(hidden.all()):
                    pool.gscale[int(pool.group_table[b, g])] = float("nan")
            t = torch.arange(L - pool.hot_length(b), L, device="cuda")
            hidden = t[(t < first) & (t >= sinks)] % pool.hot_window
            for x in (pool.hot_k, pool.hot_v):
                x[b][:, hidden] = float("nan")
                unused = torch.ones(pool.hot_window, dtype=torch.bool, device="cuda")
                unused[t % pool.hot_window] = False
                x[b][:, unused] = float("inf")
        got = pool.attend(q, window=window, sinks=sinks)
        for n, x in keep.items():
            getattr(pool, n).copy_(x)
        assert torch.equal(got, want), (window, sinks)


def test_attend_on_another_stream_and_in_graphs():
    """Two captured steps of one pool (their workspaces apart) replayed between
    eager ones, on queries that change; one more on a second stream."""
    print("[attend] stream, graphs", flush=True)
    pool = make_pool(8, [6000, 1500], 32, 8)
    q1, q2 = queries(1, pool, 1), queries(2, pool, 20)
    args = dict(window=1000, sinks=4)
    want = pool.attend(q1, **args), pool.attend(q2, **args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = pool.attend(q1, **args)
    with_main = pool.attend(q2, **args)
    side.synchronize()
    assert torch.equal(got, want[0]) and torch.equal(with_main, want[1])
    graphs = []
    for q in (q1, q2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = pool.attend(q, **args)
        graphs.append((g, q, out))
    for step in range(4):
        for g, q, out in graphs:
            q.mul_(-0.9)
            g.replay()
        torch.randn(1 << 18, device="cuda").sum().item()
        for g, q, out in graphs:
            assert torch.equal(out, pool.attend(q, **args)), step


@pytest.mark.parametrize("dtype", ["float16", "float32"])
def test_a_serving_run(dtype):
    """append_qkv and attend as a model uses them: a prompt in two chunks, then
    token by token, against norm, rotation, append and attention apart."""
    from turboquant_pro_amd import TQKVPool, norm_rope
    print(f"[attend] run {dtype}", flush=True)
    B, Hq, H, D, window, sinks = 2, 8, 2, 128, 400, 4
    gen = torch.Generator(device="cuda").manual_seed(11)
    pools = [TQKVPool(n_kv_heads=H, n_q_heads=Hq, max_batch=B, max_seq_len=1200, seed=1, input_dtype=dtype)
             for _ in range(2)]
    inv = (10000.0 ** (-torch.arange(64, dtype=torch.float64) / 64)).float().cuda()
    w = (1.0 + 0.1 * torch.randn(D, generator=gen, device="cuda")).bfloat16()
    at = [0, 0]
    for T, n_new in ((700, [700, 333]), (300, [100, 300]), (1, None), (1, None), (3, None)):
        rows = torch.randn((B, T, (Hq + 2 * H) * D), generator=gen, device="cuda").bfloat16()
        q = pools[0].append_qkv(rows, inv, q_weight=w, k_weight=w, n_new=n_new)
        pos = torch.tensor(at, device="cuda")[:, None] + torch.arange(T, device="cuda")
        q2, k2, v2 = norm_rope(rows, Hq, H, inv, pos, q_weight=w, k_weight=w, dtype=pools[1].dtype)
        pools[1].append(k2, v2, n_new=n_new)
        at = [a + (T if n_new is None else n) for a, n in zip(at, n_new or [T, T])]
        assert torch.equal(q, q2) and pools[0].lengths == at == pools[1].lengths
        ql = None if n_new is None else torch.tensor(n_new, dtype=torch.int32, device="cuda")
        out = pools[0].attend(q, window=window, sinks=sinks, q_lens=ql)
        assert torch.equal(out, pools[1].attend(q2, window=window, sinks=sinks, q_lens=ql))
        check(pools[0], out, q, window, sinks, n_new, f"T={T}")
    for a, b in ((p.export_group(0, 0) for p in pools),):
        assert all(np.array_equal(a[k], b[k]) for k in ("kpacked", "vpacked", "vnorms"))
    with pytest.raises(ValueError):
        pools[0].append_qkv(rows[..., :-8], inv)
