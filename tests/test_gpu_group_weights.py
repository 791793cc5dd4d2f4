"""TQKVPool.attend(weights=...): the weight that every coded group received, against
64-bit attention over the cache's own reconstruction, and the output as without it."""

import pytest

torch = pytest.importorskip("torch")

from attn_ref import visible  # noqa: E402
from more_ref import cached, check_rows, coefficient, make_pool, queries  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU visible")


def check_weights(pool, out, weights, before, q, window, sinks, q_lens=None, what=""):
    """Every weight within the scores' and sums' roundings of its row's (relative), the
    sum rounded once."""
    B, Hq, T, D = q.shape
    H, G = pool.n_kv_heads, pool.group_tokens
    gq = Hq // H
    for b in range(B):
        n, m, ng = pool.lengths[b], T if q_lens is None else q_lens[b], pool.n_groups(b)
        assert torch.equal(weights[b, :, ng:], before[b, :, ng:]), what
        if n == 0:
            continue
        k, v = cached(pool, b)
        sees = visible(n, m, T, 0, window, sinks, "cuda")
        for h in range(H):
            s = slice(h * gq, (h + 1) * gq)
            check_rows(out[b, s], q[b, s], k[h], v[h], sees, f"{what} seq {b} head {h}")
            x = q[b, s].double()
            hidden = ~sees
            score = (x @ k[h].T * D ** -0.5).masked_fill(hidden, -torch.inf)
            score[:, hidden.all(-1)] = 0.0
            w = torch.softmax(score, -1).masked_fill(hidden, 0.0)
            mag = (x.abs() @ k[h].abs().T).masked_fill(hidden, 0.0).amax(-1, keepdim=True)
            w = w[..., :ng * G].view(gq, T, ng, G).sum(-1)
            want = w.sum((0, 1)) + before[b, h, :ng].double()
            tol = (w * coefficient(mag, n, D)).sum((0, 1)) + 2.0 ** -23 * want.abs() + 1e-37
            err = (weights[b, h, :ng].double() - want).abs()
            assert bool((err <= tol).all()), f"{what} seq {b} head {h}: {float((err - tol).max()):.3e} past the bound"


FORMS = [
    ([5000, 1300, 700], 32, 8, 128, dict()),
    ([2600, 513], 8, 2, 128, dict(value_bits=4)),
    ([1400, 40], 7, 1, 128, dict(value_bits=2, page_tokens=16, hot_window=64)),
    ([1500, 900], 4, 4, 128, dict(key_grid="polar", key_bits=3, value_bits=3)),
    ([700, 150], 4, 2, 128, dict(hot_window=47, page_tokens=12)),
    ([2100, 600], 4, 1, 64, dict(value_bits=4)),
    ([2100, 600], 16, 8, 256, dict(value_bits=3)),
    ([900, 300], 8, 1, 256, dict(key_grid="uniform", key_bits=2, hot_window=64)),
]


@pytest.mark.parametrize("lens,Hq,H,D,form", FORMS)
def test_weights_against_the_reconstructed_cache(lens, Hq, H, D, form):
    print(f"[weights] {lens} {Hq}/{H} D={D} {form}", flush=True)
    pool = make_pool(3, lens, Hq, H, D, **form)
    gen = torch.Generator(device="cuda").manual_seed(1)
    for T in (1, 3, 40):
        q = queries(T, pool, T)
        for window, sinks in ((None, 0), (1, 0), (300, 4), (600, 257), (20, 33)):
            before = torch.rand((len(lens), H, pool.max_groups), generator=gen, device="cuda")
            weights = before.clone()
            out = pool.attend(q, window=window, sinks=sinks, weights=weights)
            check_weights(pool, out, weights, before, q, window, sinks, what=f"T={T} window={window} sinks={sinks}")
            again = before.clone()
            assert torch.equal(out, pool.attend(q, window=window, sinks=sinks, weights=again))
            assert torch.equal(weights, again)


def test_ragged_queries_and_short_sequences():
    print("[weights] ragged", flush=True)
    for D in (128, 64):
        pool = make_pool(6, [0, 1, 4, 600, 1100, 530], 8, 2, D, hot_window=64)
        for T, m in ((6, [0, 1, 6, 2, 6, 0]), (200, [200, 3, 20, 200, 7, 150])):
            q = queries(T, pool, T)
            ql = torch.tensor(m, dtype=torch.int32, device="cuda")
            for window, sinks in ((None, 0), (70, 3)):
                zero = torch.zeros((6, 2, pool.max_groups), device="cuda")
                weights = zero.clone()
                out = pool.attend(q, window=window, sinks=sinks, q_lens=ql, weights=weights)
                check_weights(pool, out, weights, zero, q, window, sinks, m, f"T={T}")


def test_queries_in_slices():
    """More queries than the blocks' sums of one slice take: rows and slices end apart."""
    print("[weights] slices", flush=True)
    # 32 query heads of one sequence, 2047 blocks: 512 KiB a query, 512 queries a slice
    pool = make_pool(7, [66000], 32, 8)
    q = queries(7, pool, 515)
    zero = torch.zeros((1, 8, pool.max_groups), device="cuda")
    weights = zero.clone()
    out = pool.attend(q, weights=weights)
    check_weights(pool, out, weights, zero, q, None, 0)


def test_infinite_and_missing_numbers():
    """A NaN key's group makes its rows NaN, as their softmax is; other heads keep theirs."""
    print("[weights] nan", flush=True)
    pool = make_pool(8, [1500], 4, 2)
    q = queries(8, pool, 1)
    zero = torch.zeros((1, 2, pool.max_groups), device="cuda")
    want = zero.clone()
    pool.attend(q, weights=want)
    pool.gmean[int(pool.group_table[0, 1]), 0] = float("nan")
    got = zero.clone()
    out = pool.attend(q, weights=got)
    ng = pool.n_groups(0)
    assert bool(out[0, :2].isnan().all()) and bool(got[0, 0, :ng].isnan().all())
    assert torch.equal(got[0, 1], want[0, 1])


def test_refusals():
    print("[weights] refusals", flush=True)
    pool = make_pool(11, [1300, 800], 8, 2)
    q = queries(11, pool, 2)
    good = torch.zeros((2, 2, pool.max_groups), device="cuda")
    for bad in (good.double(), good[:1], good[..., :-1], good.cpu(), good.transpose(0, 1),
                torch.zeros((2, 2, 2 * pool.max_groups), device="cuda")[..., ::2]):
        with pytest.raises(ValueError):
            pool.attend(q, weights=bad)
    with pytest.raises(NotImplementedError):
        pool.attend(q, weights=good.clone().requires_grad_())
    f32 = make_pool(11, [700], 4, 1, input_dtype="float32")
    with pytest.raises(NotImplementedError):
        f32.attend(queries(1, f32, 1), weights=torch.zeros((1, 1, f32.max_groups), device="cuda"))
