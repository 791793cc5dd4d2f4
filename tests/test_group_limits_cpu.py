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
