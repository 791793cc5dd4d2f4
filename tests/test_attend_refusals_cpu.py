"""What tqk_attend and TQKVPool.attend refuse before any GPU work (no GPU needed)."""

import ctypes

import pytest

torch = pytest.importorskip("torch")

from test_ops_cpu import _lib  # noqa: E402

CACHE = dict(head_dim=128, key_bits=4, value_bits=4, n_kv_heads=2, n_q_heads=8, hot_window=512, group_tokens=256,
             page_tokens=64, hot_ring=512, max_groups_per_seq=6, max_pages_per_seq=24, n_pages=24, outlier_cap=64,
             outliers_per_channel=2, sm_scale=0.1)


def attend_desc(N, **kw):
    t = N.AttendDesc(**{**dict(batch=1, q_len=4, max_len=2000, window=300, sinks=1, out_type=1), **kw})
    t.q_stride[:] = t.o_stride[:] = [1024] * 3
    return t


@pytest.mark.parametrize("q_len", [1, 64])
def test_a_side_list_without_room_is_refused(q_len):
    """Outliers but a capacity of none: a load of an entry would have no place to go."""
    N, lib = _lib()
    buf = ctypes.create_string_buffer(512)
    at = (ctypes.addressof(buf) + 15) & ~15
    p = N.CachePtrs(**{name: at for name, _ in N.CachePtrs._fields_})
    for cap, outliers, want in ((0, 2, N.TQK_EINVAL), (0, 0, N.TQK_EWORKSPACE), (1, 2, N.TQK_EWORKSPACE)):
        d = N.CacheDesc(**{**CACHE, "outlier_cap": cap, "outliers_per_channel": outliers})
        t = attend_desc(N, q_len=q_len)
        assert lib.tqk_attend(ctypes.byref(d), ctypes.byref(p), ctypes.byref(t), at, at, None, at, at, 0, None) == want
        need = lib.tqk_attend_workspace_bytes(ctypes.byref(d), ctypes.byref(t))
        assert (need == 0) == (want == N.TQK_EINVAL)


@pytest.mark.parametrize("batch,heads,D,max_len,window", [(16, 8, 128, 131072, 0), (16, 8, 128, 131072, 131000),
                                                          (1, 8, 256, 1 << 19, 0), (1, 2, 128, 1 << 21, 0),
                                                          (64, 8, 64, 32768, 20000), (5, 8, 128, 70000, 0)])
@pytest.mark.parametrize("q_len", [33, 129, 512])
def test_a_chunk_s_workspace_is_bounded(batch, heads, D, max_len, window, q_len):
    """Keys and values reconstructed at a time stay within a GiB (and the splits of the
    attention over them within 512 workgroups' rows and numbers), whatever the batch."""
    N, lib = _lib()
    d = N.CacheDesc(**{**CACHE, "head_dim": D, "n_kv_heads": heads, "n_q_heads": 4 * heads, "max_groups_per_seq": 1 << 14,
                       "max_pages_per_seq": 1 << 16, "n_pages": 1 << 22})
    need = lib.tqk_attend_workspace_bytes(ctypes.byref(d), ctypes.byref(attend_desc(
        N, batch=batch, q_len=q_len, max_len=max_len, window=window)))
    assert 0 < need <= (1 << 30) + 512 * 128 * (D + 2) * 4 + 512


@pytest.mark.parametrize("q_len", [1, 64])
def test_page_pools_past_32_bits_are_refused(q_len):
    """A head's rows are held in 32 bits by the fp16 caches' kernels."""
    N, lib = _lib()
    buf = ctypes.create_string_buffer(512)
    at = (ctypes.addressof(buf) + 15) & ~15
    p = N.CachePtrs(**{name: at for name, _ in N.CachePtrs._fields_})
    for pages, f32, want in ((1 << 25, 0, N.TQK_EUNSUPPORTED), ((1 << 25) - 1, 0, N.TQK_EWORKSPACE),
                             (1 << 25, 1, N.TQK_EWORKSPACE)):
        d = N.CacheDesc(**{**CACHE, "n_pages": pages, "input_f32": f32})
        t = attend_desc(N, q_len=q_len)
        assert lib.tqk_attend(ctypes.byref(d), ctypes.byref(p), ctypes.byref(t), at, at, None, at, at, 0, None) == want
