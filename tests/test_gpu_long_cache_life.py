"""The operators of a long cache together, as a conversation uses them: a prompt shared
by a batch, its tokens projected and rotated into the cache, dense steps that keep
account of the groups' weights, sparse steps over chosen groups, evictions between, and
windows, decodes and resets after them.  Every result against the reconstructed cache."""

import math

import pytest

torch = pytest.importorskip("torch")

from attn_ref import visible  # noqa: E402
from more_ref import cached, check_listed, check_rows, chosen, coefficient, queries, tokens  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU visible")


def check_whole(pool, out, q, window=0, what=""):
    gq, T, off, tot = pool.n_q_heads // pool.n_kv_heads, q.shape[2], 0.0, 0.0
    for b in range(pool.max_batch):
        k, v = cached(pool, b)
        sees = visible(pool.lengths[b], T, T, 0, window, 0, "cuda")
        for h in range(pool.n_kv_heads):
            s = slice(h * gq, (h + 1) * gq)
            e, w = check_rows(out[b, s], q[b, s], k[h], v[h], sees, f"{what} seq {b} head {h}")
            off, tot = off + e, tot + w
    assert math.sqrt(off / tot) <= 2.0 ** -10, what


def softmax_of_groups(pool, b, q):
    """``(H, n_groups)``: the weights that sequence b's last queries give every group, in
    64 bits, and what they may be off by, relative to them."""
    H, G, ng, n = pool.n_kv_heads, pool.group_tokens, pool.n_groups(b), pool.lengths[b]
    gq, T = pool.n_q_heads // H, q.shape[2]
    k, x = cached(pool, b)[0], q[b].double().view(H, gq * T, -1)
    sees = visible(n, T, T, 0, None, 0, "cuda")
    s = x @ k.transpose(1, 2) / math.sqrt(q.shape[3])
    off = coefficient(float((x.abs() @ k.abs().transpose(1, 2)).max()), n, q.shape[3])
    p = torch.softmax(s.masked_fill(~sees.repeat(gq, 1), -math.inf), -1)
    return p.sum(1)[:, :ng * G].view(H, ng, G).sum(-1), off


@pytest.mark.parametrize("D,Hq,H,form", [(128, 8, 2, dict(value_bits=3)), (128, 4, 4, dict(value_bits=4, hot_window=100)),
                                         (64, 6, 2, dict(value_bits=4)), (256, 4, 1, dict(key_grid="uniform"))])
def test_a_conversation(D, Hq, H, form):
    print(f"[life] D={D} {form}", flush=True)
    from turboquant_pro_amd import TQKVPool
    B, prompt = 3, 4000
    gen = torch.Generator(device="cuda").manual_seed(D + Hq)
    pool = TQKVPool(n_kv_heads=H, n_q_heads=Hq, head_dim=D, max_batch=B, max_seq_len=prompt + 2500, seed=3, **form)
    inv = 10000.0 ** (-torch.arange(0, D, 2, device="cuda", dtype=torch.float64) / D)
    inv = inv.float()
    G = pool.group_tokens

    def rows(T):
        return torch.randn((B, T, (Hq + 2 * H) * D), generator=gen, device="cuda").half()

    pool.append_qkv(rows(prompt), inv, n_new=[0, prompt, 0])
    pool.share_prefix(1)
    S = pool._shared
    weights = torch.zeros((B, H, pool.max_groups), device="cuda")
    total = [prompt] * B
    for turn in range(3):
        new = [300 + 10 * turn, 1, 700]
        pool.append_qkv(rows(max(new)), inv, n_new=new)
        total = [n + x for n, x in zip(total, new)]
        assert [n + x for n, x in zip(pool.lengths, pool.evicted_tokens)] == total
        for step in range(2):
            q = pool.append_qkv(rows(1), inv)
            total = [n + 1 for n in total]
            # dense, sparse and accounted steps over one state of the cache
            dense = pool.attend(q)
            check_whole(pool, dense, q, what=f"turn {turn} dense")
            top = S // 2 + 2
            groups = pool.select_groups(q, top, first=1, last=2)
            assert torch.equal(groups.cpu(), chosen(pool, q, top, 1, 2, 1.0))
            check_listed(pool, pool.attend(q, groups=groups), q, groups, what=f"turn {turn} sparse")
            before = weights.clone()
            counted = pool.attend(q, weights=weights)
            check_whole(pool, counted, q, what=f"turn {turn} counted")
            for b in range(B):
                got = weights[b].double() - before[b].double()
                want, off = softmax_of_groups(pool, b, q)
                # (and half a step of the sum, which is held in fp32)
                tol = off * want + 2.0 ** -24 * (before[b, :, :pool.n_groups(b)].double() + (1 + off) * want) + 1e-30
                assert bool(((got[:, :pool.n_groups(b)] - want).abs() <= tol).all())
                assert bool((got[:, pool.n_groups(b):] == 0).all())
        keep = S + 2 - (turn == 2)
        mass = weights.double().sum(1)
        counts = [pool.n_groups(b) for b in range(B)]
        kept = pool.evict(weights, keep, last=1).cpu()
        for b in range(B):
            want = list(range(counts[b]))
            if counts[b] > keep:
                free = sorted(range(S, counts[b] - 1), key=lambda g: (-float(mass[b, g]), g))
                want = sorted(list(range(S)) + free[:keep - S - 1] + [counts[b] - 1])
            assert kept[b].tolist() == want + [-1] * (keep - len(want))
            assert torch.allclose(weights[b].double().sum(0)[:len(want)], mass[b, want], rtol=1e-6, atol=0)
        q = queries(turn, pool, 3)
        check_whole(pool, pool.attend(q), q, what=f"turn {turn} after")
        check_whole(pool, pool.attend(q, window=G + 7), q, window=G + 7, what=f"turn {turn} window")
        q = queries(turn, pool, 1)
        # (the decode's own rounding of keys and weights: within a few halves' steps of the attention)
        one, two = pool.decode(q[:, :, 0].contiguous()).double(), pool.attend(q)[:, :, 0].double()
        assert float((one - two).norm() / two.norm()) <= 2.0 ** -8
    pool.reset()
    assert pool.evicted_tokens == [0] * B and pool._shared == 0
    pool.append_qkv(rows(900), inv, n_new=[900, 20, 0])
    q = queries(9, pool, 1)
    out = pool.attend(q)
    assert bool((out[2] == 0).all())
    groups = pool.select_groups(q, 2)
    check_listed(pool, pool.attend(q, groups=groups), q, groups, what="after reset")


def test_a_callers_table_with_a_page_twice_is_not_evicted():
    """The page that one place frees would be written while another one reads it."""
    print("[life] pages twice", flush=True)
    import numpy as np
    from turboquant_pro_amd import TQKVPool
    for twice in (False, True):
        table = np.arange(48, dtype=np.int32)[::-1].reshape(2, 24).copy()
        if twice:
            table[1, :4] = table[0, :4]
        pool = TQKVPool(n_kv_heads=2, n_q_heads=4, max_batch=2, max_seq_len=2000, page_tokens=64, block_table=table, seed=1)
        k, v = tokens(1, 2, 2, 2000, 128, torch.float16)
        pool.append(k, v, n_new=[2000, 100] if twice else [2000, 1500])
        weights = torch.rand((2, 2, pool.max_groups), device="cuda")
        if twice:
            with pytest.raises(NotImplementedError):
                pool.evict(weights, 2)
            assert pool.lengths == [2000, 100] and pool.evicted_tokens == [0, 0]
        else:
            want = [torch.stack([x[:, :256] for x in cached(pool, b)]) for b in range(2)]
            pool.evict(weights, 2)
            for b in range(2):
                assert torch.equal(torch.stack([x[:, :256] for x in cached(pool, b)]), want[b])
