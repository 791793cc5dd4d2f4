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
