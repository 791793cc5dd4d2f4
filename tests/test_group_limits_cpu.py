"""Sizes at which the entry points over chosen groups, received weights, a shared prefix
and eviction take a call and from which on they refuse it (no GPU needed; every right
call has a workspace one byte short, refused last)."""

import pytest

torch = pytest.importorskip("torch")

from test_group_refusals_cpu import MANY, Call  # noqa: E402


@pytest.mark.parametrize("ring,want", [(512, "EWORKSPACE"), (513, "EWORKSPACE"), (1024, "EWORKSPACE"),
                                       (4096, "EWORKSPACE"), (4097, "EUNSUPPORTED")])
@pytest.mark.parametrize("cache", [dict(), dict(input_f32=1), dict(head_dim=64), dict(head_dim=256)])
def test_rings_that_fit_a_column(ring, want, cache):
    """16 bytes of every row of a ring go through 64 KiB at a time."""
    c = Call({**cache, "hot_ring": ring})
    assert c.evict()[1] == getattr(c.N, "TQK_" + want)


@pytest.mark.parametrize("heads,ring,columns", [(8, 4096, 16), (8, 512, 2), (64, 513, 4)])
def test_more_rings_than_a_launch_are_refused_first(heads, ring, columns):
    """... before tables, lengths and weights are rewritten."""
    most = (2 ** 31 - 1) // 256 // (heads * 2 * columns)
    cache = {**MANY, "n_kv_heads": heads, "n_q_heads": heads, "hot_ring": ring}
    for batch, want in ((min(most, 65535), "EWORKSPACE"), (most + 1, "EINVAL")):
        c = Call(cache)
        assert c.evict(batch=batch)[1] == getattr(c.N, "TQK_" + want), batch


@pytest.mark.parametrize("n,want", [(1 << 24, "EWORKSPACE"), ((1 << 24) + 1, "EINVAL"), (2 ** 31 - 1, "EINVAL")])
def test_lists_past_their_counters_are_refused(n, want):
    """A thread's next place in a list of nearly 2^31 entries would pass 32 bits."""
    c = Call()
    assert c.select(top=n)[1] == c.evict(keep=n)[1] == getattr(c.N, "TQK_" + want)


@pytest.mark.parametrize("batch,q_len,max_len", [(64, 4096, 4096), (128, 2048, 2048), (1, 1 << 22, 700), (16, 1 << 20, 600),
                                                 (64, 4096, 512)])
def test_choices_for_any_number_of_queries(batch, q_len, max_len):
    """More rows than a launch takes go in slices of queries."""
    c = Call({**MANY, "n_kv_heads": 8, "n_q_heads": 8})
    need, rc = c.select(batch=batch, q_len=q_len, max_len=max_len)
    groups = max(0, (max_len - 257) // 256)  # (512 tokens stay uncoded at first, then more than 256)
    assert rc == c.N.TQK_EWORKSPACE
    slice_ = min(q_len, (2 ** 21 - 1) // (8 * batch), (256 << 20) // (64 * batch * groups) if groups else q_len)
    assert need == 8 * batch * groups * 8 * slice_ + 16


@pytest.mark.parametrize("heads,batch,max_len,want", [(1, (1 << 21) - 1, 700, "EWORKSPACE"), (1, 1 << 21, 700, "EINVAL"),
                                                      (64, 1 << 14, 2048, "EWORKSPACE"), (64, 1 << 16, 32768, "EINVAL"),
                                                      (16, 1 << 16, 28672, "EWORKSPACE"), (16, 1 << 16, 32768 + 512, "EINVAL")])
def test_choices_for_any_batch_up_to_a_launch(heads, batch, max_len, want):
    """The size of a workspace is given exactly where the call is taken (16 x 65536 pairs:
    110 groups make 7 x 2^20 workgroups, 128 make 2^23)."""
    c = Call({**MANY, "n_kv_heads": heads, "n_q_heads": heads})
    need, rc = c.select(batch=batch, max_len=max_len)
    assert rc == getattr(c.N, "TQK_" + want) and (need > 0) == (want == "EWORKSPACE")


def test_weights_of_more_rows_than_a_launch():
    """Short caches, many queries: slices of 2^22 workgroups (one query of 8 heads each), one split."""
    cache = {**MANY, "n_kv_heads": 8, "n_q_heads": 64}
    for batch, q_len, slice_ in ((2048, 512, 256), (1024, 512, 512), (1024, 513, 512), (3, 512, 512)):
        c = Call(cache, dict(batch=batch, q_len=q_len, max_len=512))
        need, rc = c.weights()
        assert rc == c.N.TQK_EWORKSPACE
        # (a split's sums of 130 floats a row; blocks: none)
        assert need == 256 + batch * 64 * slice_ * 130 * 4 * (1 if batch > 3 else (need - 256) // (batch * 64 * slice_ * 520))


@pytest.mark.parametrize("kind", ["groups", "weights", "shared"])
@pytest.mark.parametrize("batch,q_len,heads", [(1 << 22, 1, 2), (1 << 20, 2, 8), (4096, 256, 8), (1 << 19, 1, 8), (1 << 13, 7, 8),
                                               (1024, 512, 8), (65535, 60, 1), (1 << 16, 1, 1), (64, 1 << 17, 1)])
def test_a_workspace_is_given_where_the_call_is_taken(kind, batch, q_len, heads):
    c = Call({**MANY, "n_kv_heads": heads, "n_q_heads": heads * 8}, dict(batch=batch, q_len=q_len))
    need, rc = getattr(c, kind)()
    assert (need > 0) == (rc == c.N.TQK_EWORKSPACE) and rc in (c.N.TQK_EWORKSPACE, c.N.TQK_EINVAL)
    rows, pairs = batch * heads * 8 * q_len, batch * heads
    if kind == "groups":
        assert (need > 0) == (rows < 2 ** 30 and pairs <= 2 ** 22)
    elif kind == "weights":
        assert (need > 0) == (rows < 2 ** 30 and pairs <= 65535)
