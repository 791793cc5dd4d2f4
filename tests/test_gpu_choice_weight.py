"""How much of the softmax weight the choice of groups keeps, with a side-list and
without one: what lies in the levels is kept, a value of the side-list is not looked at."""

import math

import pytest

torch = pytest.importorskip("torch")

from more_ref import cached, check_listed  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU visible")


def kept_weight(pool, q, groups):
    """Of sequence 0's single query: the softmax weight of the listed groups and the
    uncoded tokens, ``(Hq,)``, in 64 bits."""
    k, G, ng = cached(pool, 0)[0], pool.group_tokens, pool.n_groups(0)
    gq, D = pool.n_q_heads // pool.n_kv_heads, pool.head_dim
    p = torch.softmax((q[0, :, 0].double()[:, None] * k.repeat_interleave(gq, 0)).sum(-1) / math.sqrt(D), -1)
    of = torch.arange(k.shape[1], device="cuda") // G
    chosen = (of >= ng) | (of == groups[0, :, 0, :, None]).any(1).repeat_interleave(gq, 0)
    return (p * chosen).sum(-1)


@pytest.mark.parametrize("D,form", [(128, dict()), (128, dict(outlier_frac=0.0)), (128, dict(key_grid="uniform", key_bits=3)),
                                    (64, dict()), (256, dict(outlier_frac=0.1)), (128, dict(hot_window=64))])
@pytest.mark.parametrize("spread", [0.0, 1.0])
def test_groups_that_a_query_looks_for_are_chosen(D, form, spread):
    """Four groups whose every key scores 30 above the others' centre, the scores'
    deviation 1: the others' 9000 tokens have a weight of at most 9000 e^(10 - 30), their
    best and the four groups' worst 5 deviations off; levels off by at most a few tenths."""
    print(f"[choice] D={D} {form} spread={spread}", flush=True)
    from turboquant_pro_amd import TQKVPool
    gen = torch.Generator(device="cuda").manual_seed(D)
    H, L = 2, 9000
    pool = TQKVPool(n_kv_heads=H, n_q_heads=H, head_dim=D, max_batch=1, max_seq_len=L, seed=1, **form)
    G = pool.group_tokens
    q = torch.randn((1, H, 1, D), generator=gen, device="cuda").half()
    k = torch.randn((1, H, L, D), generator=gen, device="cuda")
    want = [3, 7, 8, 20]
    along = q.float() / q.float().square().sum(-1, keepdim=True) * 30 * math.sqrt(D)
    for g in want:
        k[:, :, g * G:(g + 1) * G] += along
    pool.append(k.half(), torch.randn((1, H, L, D), generator=gen, device="cuda").half())
    groups = pool.select_groups(q, 6, first=1, last=1, spread=spread)
    assert groups[0, :, 0].tolist() == [[0] + want + [pool.n_groups(0) - 1]] * H
    assert float(kept_weight(pool, q, groups).min()) >= 1 - 1e-4
    check_listed(pool, pool.attend(q, groups=groups), q, groups)


LEVELS = [dict(), dict(outlier_frac=0.1), dict(key_grid="uniform", key_bits=3), dict(key_grid="uniform", key_bits=2),
          dict(zero_point="symmetric"), dict(zero_point="sparse", rope_theta=10000.0), dict(hot_window=47)]


@pytest.mark.parametrize("form", LEVELS)
def test_levels_reach_over_every_value(form):
    """A group's levels end at its channels' largest deviations, the side-list's values
    among them: with spread=1 the score is a bound on the products with all its keys."""
    print(f"[choice] levels {form}", flush=True)
    from turboquant_pro_amd import TQKVPool
    gen = torch.Generator(device="cuda").manual_seed(3)
    H, D, L = 2, 128, 1500
    k = (torch.randn((1, H, L, D), generator=gen, device="cuda") + torch.randn((D,), generator=gen, device="cuda")).half()
    k[:, :, 100::170] *= 20.0
    pool = TQKVPool(n_kv_heads=H, n_q_heads=H, head_dim=D, max_batch=1, max_seq_len=L, seed=1, **form)
    pool.append(k, k.clone())
    G, ng = pool.group_tokens, pool.n_groups(0)
    slots = pool.group_table[0, :ng].long()
    mean, scale = pool.gmean[slots].double(), pool.gscale[slots].double()
    steps = 2 ** pool.key_bits - 1
    lo, hi = (mean, mean + steps * scale) if pool.key_grid == "uniform" else (mean - scale, mean + scale)
    x = k[0, :, :ng * G].double().view(H, ng, G, D).transpose(0, 1)
    # (ends from differences and quotients in fp32: a few of its half steps of what they are made of)
    off = 4 * 2.0 ** -24 * (mean.abs() + (steps if pool.key_grid == "uniform" else 1) * scale)[:, :, None]
    assert bool((x >= lo[:, :, None] - off).all()) and bool((x <= hi[:, :, None] + off).all())


@pytest.mark.parametrize("frac", [0.02, 0.0])
def test_a_single_large_value_is_found(frac):
    """One token that takes the softmax by one channel, in the side-list or coded (its
    level then off by at most 14 of 200, 5 of the products): its group is chosen."""
    print(f"[choice] one value {frac}", flush=True)
    from turboquant_pro_amd import TQKVPool
    gen = torch.Generator(device="cuda").manual_seed(5)
    H, D, L, token = 1, 128, 6000, 2000
    k = torch.randn((1, H, L, D), generator=gen, device="cuda")
    q = torch.randn((1, H, 1, D), generator=gen, device="cuda").half()
    q[..., 17] = 4.0
    k[0, 0, token, 17] = 200.0  # (70 above the others' centre, of a deviation of 1.1)
    pool = TQKVPool(n_kv_heads=H, n_q_heads=H, head_dim=D, max_batch=1, max_seq_len=L, seed=1, outlier_frac=frac)
    pool.append(k.half(), torch.randn((1, H, L, D), generator=gen, device="cuda").half())
    groups = pool.select_groups(q, 3)
    assert token // pool.group_tokens in groups.flatten().tolist()
    assert float(kept_weight(pool, q, groups).min()) >= 1 - 1e-9
    check_listed(pool, pool.attend(q, groups=groups), q, groups)


def test_an_imported_side_list_may_lie_outside():
    """Its values past the levels are not looked at by the choice; a list has them."""
    print("[choice] imported", flush=True)
    from turboquant_pro_amd import TQKVPool
    gen = torch.Generator(device="cuda").manual_seed(6)
    H, D, L, mine = 1, 128, 6000, 9
    k = torch.randn((1, H, L, D), generator=gen, device="cuda")
    k[:, :, mine * 256:(mine + 1) * 256] *= 0.5  # (half of the others' bound)
    q = torch.randn((1, H, 1, D), generator=gen, device="cuda").half()
    q[..., 17] = 4.0
    pool = TQKVPool(n_kv_heads=H, n_q_heads=H, head_dim=D, max_batch=1, max_seq_len=L, seed=1)
    pool.append(k.half(), torch.randn((1, H, L, D), generator=gen, device="cuda").half())
    group = pool.export_group(0, mine)
    at = int((group["outlier_idx"] % D == 17).nonzero()[0][0])
    group["outlier_val"][at] = 200.0
    pool.import_group(0, mine, keys=group)
    groups = pool.select_groups(q, 4)
    assert mine not in groups.flatten().tolist() and float(kept_weight(pool, q, groups).min()) <= 1e-9
    groups[..., 1] = mine
    assert float(kept_weight(pool, q, groups).min()) >= 1 - 1e-9
    check_listed(pool, pool.attend(q, groups=groups), q, groups)
