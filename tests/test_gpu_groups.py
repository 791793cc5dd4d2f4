"""TQKVPool.select_groups and attend(groups=...): the choice against its definition on
the host, attention over listed groups against 64 bits; key and value forms, head
layouts, group sizes, ragged queries, lists with holes and strides."""

import pytest

torch = pytest.importorskip("torch")

from more_ref import check_listed, chosen, make_pool, queries  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU visible")


FORMS = [
    # lens, Hq, H, D, pool form
    ([5000, 1300, 700], 32, 8, 128, dict()),
    ([2600, 513], 8, 2, 128, dict(value_bits=4)),
    ([1400, 40], 7, 1, 128, dict(value_bits=2, page_tokens=16, hot_window=64)),
    ([1500, 900], 2, 1, 128, dict(key_grid="uniform", key_bits=3, outlier_frac=0.0, hot_window=128)),
    ([1500, 900], 8, 1, 128, dict(hot_window=64, zero_point="symmetric")),
    ([700, 150], 4, 2, 128, dict(hot_window=47, page_tokens=12)),
    ([2100, 600], 4, 1, 64, dict(value_bits=4)),
    ([2100, 600], 16, 8, 256, dict(value_bits=3)),
    ([900, 300], 8, 1, 256, dict(key_grid="uniform", key_bits=2, hot_window=64)),
    ([900, 300], 5, 5, 64, dict(hot_window=7, page_tokens=2)),
]


@pytest.mark.parametrize("lens,Hq,H,D,form", FORMS)
def test_chosen_groups_and_attention_over_them(lens, Hq, H, D, form):
    print(f"[groups] {lens} {Hq}/{H} D={D} {form}", flush=True)
    pool = make_pool(3, lens, Hq, H, D, **form)
    for T in (1, 3, 21):
        q = queries(T, pool, T)
        for top, first, last, spread in ((1, 0, 0, 1.0), (3, 1, 1, 0.0), (6, 2, 3, 0.5), (500, 1, 1, 1.0)):
            groups = pool.select_groups(q, top, first=first, last=last, spread=spread)
            want = chosen(pool, q, top, first, last, spread)
            assert torch.equal(groups.cpu(), want), f"T={T} top={top}"
            out = pool.attend(q, groups=groups)
            check_listed(pool, out, q, groups, what=f"T={T} top={top}")
            assert torch.equal(out, pool.attend(q, groups=groups))


def test_polar_keys_take_listed_groups():
    print("[groups] polar", flush=True)
    pool = make_pool(4, [1500, 900], 4, 4, key_grid="polar", key_bits=3, value_bits=3)
    q = queries(4, pool, 2)
    groups = torch.tensor([0, 2, 1], dtype=torch.int32, device="cuda").expand(2, 4, 1, 3)
    check_listed(pool, pool.attend(q, groups=groups), q, groups)
    with pytest.raises(NotImplementedError):
        pool.select_groups(q, 2)


def test_all_groups_are_the_whole_cache():
    print("[groups] all", flush=True)
    pool = make_pool(5, [3000, 700, 100], 32, 8)
    for T in (1, 5):
        q = queries(5, pool, T)
        got, want = pool.attend(q, groups=pool.select_groups(q, pool.max_groups)).float(), pool.attend(q).float()
        # two roundings of the weighted centroids apart, and the output's
        assert float((got - want).abs().max()) <= 2.0 ** -9 * float(want.abs().max())


def test_ragged_queries_and_short_sequences():
    """Lengths of zero and one, fewer tokens than queries, fewer queries than rows; a
    query inside a coded group that is not listed sees nothing."""
    print("[groups] ragged", flush=True)
    for D in (128, 64):
        pool = make_pool(6, [0, 1, 4, 600, 1100, 530], 8, 2, D, hot_window=64)
        for T, m in ((6, [0, 1, 6, 2, 6, 0]), (200, [200, 3, 20, 200, 7, 150])):
            q = queries(T, pool, T)
            ql = torch.tensor(m, dtype=torch.int32, device="cuda")
            groups = pool.select_groups(q, 4, q_lens=ql)
            assert torch.equal(groups.cpu(), chosen(pool, q, 4, 1, 1, 1.0, m))
            check_listed(pool, pool.attend(q, groups=groups, q_lens=ql), q, groups, m, f"T={T}")
            one = torch.tensor([3, 0], dtype=torch.int32, device="cuda").expand(6, 2, 1, 2)
            check_listed(pool, pool.attend(q, groups=one, q_lens=ql), q, one, m, f"one list T={T}")
            check_listed(pool, pool.attend(q, groups=one), q, one, None, f"one list T={T}")
            none = one[..., :0]
            check_listed(pool, pool.attend(q, groups=none), q, none, None, f"no list T={T}")


def test_lists_with_holes_orders_and_strides():
    print("[groups] lists", flush=True)
    pool = make_pool(7, [2600, 1300], 8, 2, hot_window=64)
    q = queries(7, pool, 4)
    gen = torch.Generator().manual_seed(1)
    groups = torch.stack([torch.randperm(90, generator=gen)[:70] for _ in range(2 * 2 * 4)]).view(2, 2, 4, 70).int() - 5
    groups[..., 1::7] = -1
    groups[..., 3] = 2 ** 31 - 1
    groups[..., 5] = -2 ** 31
    groups = groups.cuda()
    out = pool.attend(q, groups=groups)
    check_listed(pool, out, q, groups)
    wide = torch.full((2, 4, 2, 141), -1, dtype=torch.int32, device="cuda")
    wide[..., 1::2] = groups.transpose(1, 2)
    assert torch.equal(pool.attend(q, groups=wide[..., 1::2].transpose(1, 2)), out)
    pad = torch.full((2, 2, 5, 77), -1, dtype=torch.int32, device="cuda")
    pad[:, :, 1:, 3:73] = groups
    assert torch.equal(pool.attend(q, groups=pad[:, :, 1:, 3:73]), out)
    big = torch.full((2, 5, 9, 136), 7.0, dtype=torch.float16, device="cuda")
    view = big[:, :4, :8, :128].transpose(1, 2)
    assert pool.attend(q.contiguous(), groups=groups, out=view) is view and torch.equal(view, out)
    big[:, :4, :8, :128] = 7.0
    assert bool((big == 7.0).all())


def test_what_is_not_listed_is_not_read():
    """NaN in every scale, norm and code's place of the other groups."""
    print("[groups] hidden", flush=True)
    pool = make_pool(8, [3000, 2000], 8, 2)
    q = queries(8, pool, 2)
    groups = pool.select_groups(q, 3)[:, :1, :1].expand(2, 2, 1, 3).contiguous()
    want = pool.attend(q, groups=groups).clone()
    for b in range(2):
        for g in set(range(pool.n_groups(b))) - set(groups[b].flatten().tolist()):
            phys, off = pool._rows(b, g)
            pool.vnorm[:, phys, off] = float("nan")
            pool.gscale[int(pool.group_table[b, g])] = float("nan")
    assert torch.equal(pool.attend(q, groups=groups), want)


def test_scores_that_are_no_numbers_ties_and_infinities():
    print("[groups] ties", flush=True)
    pool = make_pool(9, [3000], 4, 2)
    q = queries(9, pool, 2)
    pool.gscale[:] = pool.gscale[0].clone()
    pool.gmean[:] = pool.gmean[0].clone()
    ng = pool.n_groups(0)
    want = chosen(pool, q, 4, 1, 1, 1.0)
    assert want[0, 0, 1].tolist() == [0, 1, 2, ng - 1]
    assert torch.equal(pool.select_groups(q, 4).cpu(), want)
    pool.gmean[5, 1, 7] = float("nan")
    pool.gscale[7, :, 9] = float("inf")
    pool.gmean[3, 0] = -pool.gmean[3, 0]
    for top in (3, 5):
        assert torch.equal(pool.select_groups(q, top).cpu(), chosen(pool, q, top, 1, 1, 1.0))
    assert 5 in pool.select_groups(q, 3)[0, 1, 0].tolist()


@pytest.mark.parametrize("length,hot_window", [(40000, 15), (150000, 15)])
def test_many_groups(length, hot_window):
    """More groups than one wave, and than a workgroup's registers, hold."""
    print(f"[groups] many {length}", flush=True)
    pool = make_pool(10, [length], 2, 1, 64, hot_window=hot_window, page_tokens=8, outlier_frac=0.0)
    q = queries(10, pool, 1)
    for top in (2, 100, 2000):
        groups = pool.select_groups(q, top)
        assert torch.equal(groups.cpu(), chosen(pool, q, top, 1, 1, 1.0))
        check_listed(pool, pool.attend(q, groups=groups), q, groups, what=f"top={top}")


def test_refusals():
    print("[groups] refusals", flush=True)
    pool = make_pool(11, [1300, 800], 8, 2)
    q = queries(11, pool, 2)
    for bad in (dict(top=0), dict(top=2, first=2, last=1), dict(top=3, first=-1), dict(top=3, last=-1),
                dict(top=3, spread=-1.0), dict(top=3, spread=float("nan")), dict(top=3, spread=float("inf")),
                dict(top=3, q_lens=torch.zeros(2, dtype=torch.int32)), dict(top=3, q_lens=torch.zeros(2, device="cuda"))):
        with pytest.raises(ValueError):
            pool.select_groups(q, **bad)
    for x in (q.float(), q[:, :4], q[:1], q[..., :64], q[:, :, 0], q.cpu()):
        with pytest.raises(ValueError):
            pool.select_groups(x, 3)
    groups = pool.select_groups(q, 3)
    for bad in (groups.long(), groups[:1], groups[:, :1], groups[:, :, 0], groups.cpu(), groups.expand(2, 2, 2, 3)[:, :, :, None],
                torch.cat([groups, groups], 2)):
        with pytest.raises(ValueError):
            pool.attend(q, groups=bad)
    for bad in (dict(window=4), dict(sinks=1), dict(weights=torch.zeros((2, 2, pool.max_groups), device="cuda"))):
        with pytest.raises(ValueError):
            pool.attend(q, groups=groups, **bad)
    f32 = make_pool(11, [700], 4, 1, input_dtype="float32")
    q = queries(1, f32, 1)
    with pytest.raises(NotImplementedError):
        f32.select_groups(q, 2)
    with pytest.raises(NotImplementedError):
        f32.attend(q, groups=torch.zeros((1, 1, 1, 1), dtype=torch.int32, device="cuda"))
