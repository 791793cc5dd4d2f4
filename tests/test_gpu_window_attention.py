"""window_attention against its formula in 64 bits: windows and first tokens,
ragged lengths, left padding, rows that see nothing, lengths of zero and one,
strides, infinities and NaN in hidden places, splits over a long axis, streams
and graphs."""

import math

import pytest

torch = pytest.importorskip("torch")

from attn_ref import attention, attention_bound, visible  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU visible")


def inputs(seed, B, Hq, Hkv, D, T, L, dtype):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randn((B, T, Hq, D), generator=gen, device="cuda").to(dtype).transpose(1, 2)
    k = (2.0 * torch.randn((B, Hkv, L, D), generator=gen, device="cuda")).to(dtype)
    v = torch.randn((B, Hkv, L, D), generator=gen, device="cuda").to(dtype)
    return q, k, v


def check(out, q, k, v, window, sinks, scale=None, lens=None, q_lens=None, starts=None, what=""):
    B, Hq, T, D = q.shape
    L = k.shape[2]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    assert out.dtype == q.dtype and out.shape == q.shape
    for b in range(B):
        n = L if lens is None else lens[b]
        m = T if q_lens is None else q_lens[b]
        sees = visible(n, m, T, 0 if starts is None else starts[b], window, sinks, "cuda")
        want, weighted, mag, vmax = attention(q[b], k[b, :, :n], v[b, :, :n], sees, scale)
        tol = attention_bound(q.dtype, want, weighted, mag, vmax, n, D, scale)
        got = out[b].double()
        fine = torch.isfinite(want)
        assert torch.equal(torch.isfinite(got), fine), f"{what} seq {b}: other places finite"
        err = torch.where(fine, (got - want).abs(), torch.zeros_like(want))
        bad = err > torch.where(fine, tol, torch.ones_like(tol))
        assert not bool(bad.any()), f"{what} seq {b}: {int(bad.sum())} off, worst {float(err[bad].max()):.3e}"
        empty = ~sees.any(1)
        assert bool((out[b][:, empty] == 0).all()), f"{what} seq {b}: a row that sees nothing is not zero"


CASES = [
    # B, Hq, Hkv, D, T, L, window, sinks, dtype
    (1, 1, 1, 128, 1, 1, None, 0, torch.float16),
    (2, 8, 2, 128, 1, 700, 64, 4, torch.bfloat16),
    (1, 32, 8, 128, 1, 5000, None, 0, torch.float16),
    (2, 7, 1, 128, 5, 130, 33, 1, torch.float16),
    (1, 8, 2, 128, 257, 257, None, 0, torch.bfloat16),
    (2, 8, 2, 128, 200, 461, 100, 4, torch.float16),
    (1, 4, 4, 64, 300, 300, 64, 130, torch.bfloat16),
    (1, 3, 1, 64, 97, 1000, 1, 0, torch.float16),
    (2, 4, 2, 256, 150, 333, 77, 65, torch.bfloat16),
    (1, 16, 8, 256, 64, 2500, 1024, 3, torch.float16),
    (1, 12, 1, 128, 40, 64, None, 7, torch.bfloat16),
    (3, 2, 2, 128, 64, 64, 4000, 0, torch.float16),
    (1, 8, 8, 128, 1025, 1025, 512, 4, torch.bfloat16),
    (1, 40, 1, 64, 3, 129, 128, 0, torch.float16),
]


@pytest.mark.parametrize("B,Hq,Hkv,D,T,L,window,sinks,dtype", CASES)
def test_window_attention_against_the_formula(B, Hq, Hkv, D, T, L, window, sinks, dtype):
    from turboquant_pro_amd import window_attention
    print(f"[window] {B} x {Hq}/{Hkv} D={D} T={T} L={L} window={window} sinks={sinks} {dtype}", flush=True)
    q, k, v = inputs(T + L, B, Hq, Hkv, D, T, L, dtype)
    out = window_attention(q, k, v, window=window, sinks=sinks)
    check(out, q, k, v, window, sinks)
    again = window_attention(q, k, v, window=window, sinks=sinks)
    assert torch.equal(out, again)


@pytest.mark.parametrize("D,dtype", [(128, torch.float16), (64, torch.bfloat16), (256, torch.float16)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (50, 4), (17, 200)])
def test_ragged_lengths_padding_and_empty_rows(D, dtype, window, sinks):
    """Lengths of zero and one, more queries than keys, padding past a window or
    past every key: rows that see nothing are zero."""
    from turboquant_pro_amd import window_attention
    print(f"[window] ragged D={D} window={window} sinks={sinks}", flush=True)
    T, L = 70, 200
    lens, q_lens, starts = [200, 1, 0, 30, 133, 64, 200], [70, 1, 5, 70, 0, 33, 70], [0, 0, 0, 3, 9, 64, 180]
    q, k, v = inputs(9, len(lens), 8, 2, D, T, L, dtype)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    out = window_attention(q, k, v, window=window, sinks=sinks, kv_lens=ints(lens), q_lens=ints(q_lens),
                           kv_starts=ints(starts))
    check(out, q, k, v, window, sinks, None, lens, q_lens, starts)
    one = window_attention(q[:, :, :1], k, v, window=window, sinks=sinks, kv_lens=ints(lens), kv_starts=ints(starts))
    check(one, q[:, :, :1], k, v, window, sinks, None, lens, None, starts, "one query")
    out = window_attention(q, k[:, :, :0], v[:, :, :0], window=window, sinks=sinks)
    assert bool((out == 0).all())


def test_out_scale_and_strides():
    from turboquant_pro_amd import window_attention
    print("[window] strides", flush=True)
    B, Hq, Hkv, D, T, L = 2, 8, 2, 128, 50, 90
    q, k, v = inputs(4, B, Hq, Hkv, D, T, L, torch.float16)
    # keys and values of one (B, L, 2, Hkv, D) buffer, an output inside a larger one
    kv = torch.stack([k, v], 0).permute(1, 3, 0, 2, 4).contiguous()
    ks, vs = kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
    big = torch.full((B, T + 2, Hq + 1, D + 8), 7.0, dtype=torch.float16, device="cuda")
    view = big[:, 1:T + 1, :Hq, :D].transpose(1, 2)
    got = window_attention(q, ks, vs, window=33, sinks=2, scale=0.5, out=view)
    assert got is view
    check(view, q, k, v, 33, 2, 0.5)
    big[:, 1:T + 1, :Hq, :D] = 7.0
    assert bool((big == 7.0).all())  # nothing written around it
    # a start off 16 bytes is copied, not misread
    flat = torch.empty(k.numel() + 3, dtype=torch.float16, device="cuda")
    flat[3:] = k.reshape(-1)
    off = flat[3:].view(k.shape)
    check(window_attention(q, off, v, window=33), q, k, v, 33, 0)
    # one kv head shared by a broadcast batch
    check(window_attention(q, k[:1].expand(B, -1, -1, -1), v[:1].expand(B, -1, -1, -1)), q, k[:1].expand(B, -1, -1, -1),
          v[:1].expand(B, -1, -1, -1), None, 0)
    with pytest.raises(ValueError):
        window_attention(q, k, v, out=torch.empty((B, Hq, D, T), dtype=torch.float16, device="cuda").transpose(2, 3))


@pytest.mark.parametrize("T", [1, 90])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_infinities_and_nan_in_hidden_places(T, dtype):
    """What stands in a hidden key or value reaches no row that does not see
    it, and every row that does."""
    from turboquant_pro_amd import window_attention
    print(f"[window] hidden T={T}", flush=True)
    B, Hq, Hkv, D, L, window, sinks = 2, 4, 2, 128, 300, 60, 5
    q, k, v = inputs(12, B, Hq, Hkv, D, T, L, dtype)
    lens, starts = [280, 300], [11, 0]
    args = dict(window=window, sinks=sinks, kv_lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
                kv_starts=torch.tensor(starts, dtype=torch.int32, device="cuda"))
    clean = window_attention(q, k, v, **args)
    for x in (k, v):  # past the length, in the padding, between first tokens and window
        x[0, :, 280:] = float("nan")
        x[0, :, :11] = float("inf")
        x[0, :, 17:100] = float("nan")
        x[1, :, 6:100] = float("-inf")
    assert torch.equal(window_attention(q, k, v, **args), clean)
    check(clean, q, k, v, window, sinks, None, lens, None, starts)
    if T == 1:
        return
    # seen by some rows of a tile and hidden to others
    v[0, 1, 250, 3] = float("nan")
    v[1, 0, 299, 100] = float("inf")
    v[1, 1, 215, 64:70] = float("-inf")
    k[1, 1, 262, 5] = float("nan")
    out = window_attention(q, k, v, **args)
    check(out, q, k, v, window, sinks, None, lens, None, starts)
    assert not bool(torch.isfinite(out[0, 2:, 60:]).all())


def test_extreme_scores():
    """Scores of the type's largest values, rising and falling along the keys,
    and rows whose every visible score is the same."""
    from turboquant_pro_amd import window_attention
    print("[window] extreme", flush=True)
    B, Hq, Hkv, D, T, L = 1, 4, 1, 128, 64, 256
    q, k, v = inputs(5, B, Hq, Hkv, D, T, L, torch.float16)
    ramp = torch.linspace(-200.0, 200.0, L, device="cuda")
    k[0, 0] = (ramp[:, None] * torch.ones(D, device="cuda")).half()
    q[0, 0], q[0, 1], q[0, 2] = 1.0, -1.0, 0.0
    check(window_attention(q, k, v, window=100, sinks=4), q, k, v, 100, 4)
    check(window_attention(q, k, v, scale=1e-30), q, k, v, None, 0, 1e-30)


def test_on_another_stream_and_in_a_graph():
    """Two captured calls (a split one among them) replayed with eager work
    between, on inputs that change."""
    from turboquant_pro_amd import window_attention
    print("[window] stream, graph", flush=True)
    q, k, v = inputs(7, 2, 8, 2, 128, 3, 3000, torch.float16)
    q2, k2, v2 = inputs(8, 1, 8, 2, 64, 80, 500, torch.bfloat16)
    lens = torch.tensor([3000, 700], dtype=torch.int32, device="cuda")
    want = window_attention(q, k, v, window=2000, sinks=4, kv_lens=lens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = window_attention(q, k, v, window=2000, sinks=4, kv_lens=lens)
    side.synchronize()
    assert torch.equal(got, want)
    graphs = []
    for args in (dict(window=2000, sinks=4, kv_lens=lens), dict(kv_lens=lens)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = window_attention(q, k, v, **args), window_attention(q2, k2, v2, window=100)
        graphs.append((g, out, args))
    for step in range(4):
        q.mul_(-1.25)
        lens.sub_(step)
        for g, out, args in graphs:
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out[0], window_attention(q, k, v, **args)), step
            assert torch.equal(out[1], window_attention(q2, k2, v2, window=100)), step
        torch.randn(1 << 18, device="cuda").sum().item()
