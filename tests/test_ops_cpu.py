"""Refusals of the operators around the cache: every wrong call is an error
before any GPU work (no GPU needed)."""

import ctypes
import os

import pytest

torch = pytest.importorskip("torch")


def _call_rope(**kw):
    from turboquant_pro_amd import norm_rope
    a = dict(qkv=torch.zeros(2, 3, 12 * 128, dtype=torch.float16), n_q_heads=8, n_kv_heads=2,
             inv_freq=torch.ones(64), positions=torch.zeros(2, dtype=torch.int32))
    a.update(kw)
    return norm_rope(a.pop("qkv"), a.pop("n_q_heads"), a.pop("n_kv_heads"), a.pop("inv_freq"), a.pop("positions"), **a)


@pytest.mark.parametrize("kw,error", [
    (dict(qkv=torch.zeros(3, 12 * 128, dtype=torch.float16)), ValueError),
    (dict(qkv=torch.zeros(2, 3, 12 * 128 + 8, dtype=torch.float16)), ValueError),
    (dict(qkv=torch.zeros(2, 3, 12 * 96, dtype=torch.float16)), NotImplementedError),
    (dict(qkv=torch.zeros(2, 3, 12 * 128, dtype=torch.float64)), ValueError),
    (dict(dtype=torch.int8), ValueError),
    (dict(n_q_heads=0, n_kv_heads=0), ValueError),
    (dict(n_q_heads=-1), ValueError),
    (dict(inv_freq=torch.ones(65)), ValueError),
    (dict(inv_freq=torch.ones(20)), NotImplementedError),
    (dict(inv_freq=torch.ones(64, dtype=torch.float64)), ValueError),
    (dict(inv_freq=torch.ones(2, 32)), ValueError),
    (dict(positions=torch.zeros(3, dtype=torch.int32)), ValueError),
    (dict(positions=torch.zeros(2)), ValueError),
    (dict(positions=torch.zeros(2, 4, dtype=torch.int64)), ValueError),
    (dict(q_weight=torch.ones(64, dtype=torch.float16)), ValueError),
    (dict(k_weight=torch.ones(128, dtype=torch.bfloat16)), ValueError),
    (dict(), RuntimeError),  # a right call on CPU tensors: there is no CPU form
])
def test_norm_rope_refusals(kw, error):
    with pytest.raises(error):
        _call_rope(**kw)


def _call_window(**kw):
    from turboquant_pro_amd import window_attention
    h = torch.float16
    a = dict(q=torch.zeros(2, 8, 3, 128, dtype=h), k=torch.zeros(2, 2, 9, 128, dtype=h),
             v=torch.zeros(2, 2, 9, 128, dtype=h))
    a.update(kw)
    return window_attention(a.pop("q"), a.pop("k"), a.pop("v"), **a)


@pytest.mark.parametrize("kw,error", [
    (dict(q=torch.zeros(8, 3, 128, dtype=torch.float16)), ValueError),
    (dict(v=torch.zeros(2, 2, 8, 128, dtype=torch.float16)), ValueError),
    (dict(k=torch.zeros(2, 3, 9, 128, dtype=torch.float16), v=torch.zeros(2, 3, 9, 128, dtype=torch.float16)), ValueError),
    (dict(k=torch.zeros(1, 2, 9, 128, dtype=torch.float16), v=torch.zeros(1, 2, 9, 128, dtype=torch.float16)), ValueError),
    (dict(k=torch.zeros(2, 2, 9, 128, dtype=torch.bfloat16)), ValueError),
    (dict(q=torch.zeros(2, 8, 3, 96, dtype=torch.float16), k=torch.zeros(2, 2, 9, 96, dtype=torch.float16),
          v=torch.zeros(2, 2, 9, 96, dtype=torch.float16)), NotImplementedError),
    (dict(q=torch.zeros(2, 8, 3, 128), k=torch.zeros(2, 2, 9, 128), v=torch.zeros(2, 2, 9, 128)), NotImplementedError),
    (dict(window=0), ValueError),
    (dict(window=-4), ValueError),
    (dict(sinks=-1), ValueError),
    (dict(scale=0.0), ValueError),
    (dict(scale=float("nan")), ValueError),
    (dict(scale=float("inf")), ValueError),
    (dict(kv_lens=torch.zeros(2, dtype=torch.int64)), ValueError),
    (dict(q_lens=torch.zeros(3, dtype=torch.int32)), ValueError),
    (dict(kv_starts=torch.zeros(2)), ValueError),
    (dict(out=torch.zeros(2, 8, 3, 64, dtype=torch.float16)), ValueError),
    (dict(out=torch.zeros(2, 8, 3, 128, dtype=torch.bfloat16)), ValueError),
    (dict(), RuntimeError),
])
def test_window_attention_refusals(kw, error):
    with pytest.raises(error):
        _call_window(**kw)


def _lib():
    from turboquant_pro_amd import _native as N
    if not os.path.exists(N.LIB_PATH):
        pytest.skip("libtqk.so not built (run __graft_entry__.build())")
    return N, N.lib()


def test_rope_abi_status_codes():
    N, lib = _lib()
    buf = ctypes.create_string_buffer(512)
    at = (ctypes.addressof(buf) + 15) & ~15

    def rc(qkv=at, q=at, w=None, **kw):
        base = dict(batch=1, tokens=1, n_q_heads=4, n_kv_heads=2, head_dim=128, rotary_dim=128, in_type=1, out_type=1,
                    weight_type=1, eps=1e-6, rope_scale=1.0)
        base.update(kw)
        d = N.RopeDesc(**base)
        return lib.tqk_norm_rope(ctypes.byref(d), qkv, at, at, w, w, q, at, at, None)

    assert lib.tqk_norm_rope(None, at, at, at, None, None, at, at, at, None) == N.TQK_EINVAL
    assert rc(head_dim=96) == N.TQK_EUNSUPPORTED
    assert rc(rotary_dim=24) == N.TQK_EUNSUPPORTED
    assert rc(weight_type=2) == N.TQK_EUNSUPPORTED
    for bad in (dict(batch=-1), dict(tokens=-1), dict(n_q_heads=-1), dict(in_type=3), dict(out_type=-1),
                dict(rotary_dim=144), dict(pos_i64=2), dict(interleaved=2), dict(pos_per_token=-1),
                dict(token_stride=4), dict(qkv=at + 2), dict(q=None), dict(qkv=None), dict(w=at + 8)):
        assert rc(**bad) == N.TQK_EINVAL, bad
    assert rc(batch=0, qkv=None) == N.TQK_OK  # nothing to do


def test_attention_abi_status_codes():
    N, lib = _lib()
    buf = ctypes.create_string_buffer(512)
    at = (ctypes.addressof(buf) + 15) & ~15

    def desc(**kw):
        base = dict(batch=1, n_q_heads=8, n_kv_heads=2, head_dim=128, q_len=4, kv_len=9, window=3, sinks=1, type=1,
                    sm_scale=0.1)
        base.update(kw)
        stride = base.pop("stride", 1024)
        d = N.AttnDesc(**base)
        for s in (d.q_stride, d.k_stride, d.v_stride, d.o_stride):
            s[:] = [stride] * 3
        return d

    def rc(q=at, ws=0, n=0, **kw):
        return lib.tqk_attention(ctypes.byref(desc(**kw)), q, at, at, None, None, None, at, ws, n, None)

    assert lib.tqk_attention(None, at, at, at, None, None, None, at, None, 0, None) == N.TQK_EINVAL
    assert rc(head_dim=80) == N.TQK_EUNSUPPORTED
    assert rc(type=0) == N.TQK_EUNSUPPORTED
    for bad in (dict(batch=-1), dict(q_len=-1), dict(kv_len=-1), dict(window=-1), dict(sinks=-1), dict(n_kv_heads=3),
                dict(n_kv_heads=0), dict(sm_scale=0.0), dict(sm_scale=float("nan")), dict(sm_scale=-1.0),
                dict(stride=4), dict(q=at + 4), dict(q=None), dict(q_len=1 << 29), dict(batch=1 << 30)):
        assert rc(**bad) == N.TQK_EINVAL, bad
    assert rc(batch=0, q=None) == N.TQK_OK
    # a long context with few queries is split, and needs its workspace
    need = lib.tqk_attention_workspace_bytes(ctypes.byref(desc(kv_len=1 << 20, window=0)))
    assert need >= 2 * 8 * 4 * 130 * 4
    assert rc(kv_len=1 << 20, window=0) == N.TQK_EWORKSPACE
    assert rc(kv_len=1 << 20, window=0, ws=at, n=need - 1) == N.TQK_EWORKSPACE
    assert lib.tqk_attention_workspace_bytes(ctypes.byref(desc(q_len=1 << 29))) == 0


def test_attend_abi_status_codes():
    N, lib = _lib()
    buf = ctypes.create_string_buffer(512)
    at = (ctypes.addressof(buf) + 15) & ~15
    cache = dict(head_dim=128, key_bits=4, value_bits=4, n_kv_heads=2, n_q_heads=8, hot_window=512, group_tokens=256,
                 page_tokens=64, hot_ring=512, max_groups_per_seq=6, max_pages_per_seq=24, n_pages=24, outlier_cap=64,
                 outliers_per_channel=2, sm_scale=0.1)

    def desc(**kw):
        base = dict(batch=1, q_len=4, max_len=2000, window=300, sinks=1, out_type=1)
        base.update(kw)
        stride = base.pop("stride", 1024)
        t = N.AttendDesc(**base)
        t.q_stride[:] = t.o_stride[:] = [stride] * 3
        return t

    def rc(q=at, out=at, ws=at, n=0, c=(), none=None, **kw):
        d = N.CacheDesc(**{**cache, **dict(c)})
        p = N.CachePtrs(**{name: at for name, _ in N.CachePtrs._fields_ if name != none})
        return lib.tqk_attend(ctypes.byref(d), ctypes.byref(p), ctypes.byref(desc(**kw)), q, at, None, out, ws, n, None)

    d = N.CacheDesc(**cache)
    assert lib.tqk_attend(None, None, ctypes.byref(desc()), at, at, None, at, at, 0, None) == N.TQK_EINVAL
    assert lib.tqk_attend(ctypes.byref(d), None, None, at, at, None, at, at, 0, None) == N.TQK_EINVAL
    assert rc(c=dict(head_dim=96)) == N.TQK_EUNSUPPORTED
    assert rc(c=dict(n_q_heads=32)) == N.TQK_EUNSUPPORTED  # 16 query heads a kv head
    assert rc(out_type=2) == N.TQK_EUNSUPPORTED
    for bad in (dict(batch=-1), dict(q_len=-1), dict(max_len=-1), dict(window=-1), dict(sinks=-1), dict(stride=4),
                dict(q=at + 8), dict(out=at + 2), dict(q=None), dict(out=None), dict(q_len=1 << 29),
                dict(batch=25), dict(max_len=1 << 16), dict(c=dict(max_pages_per_seq=20)), dict(c=dict(sm_scale=0.0)),
                dict(c=dict(sm_scale=float("nan"))), dict(none="knorm", c=dict(key_grid=2, outliers_per_channel=0)),
                *(dict(none=x) for x in ("kcodes", "gscale", "gmean", "ocount", "oent", "vcodes", "vnorm", "hot_k",
                                         "hot_v", "block_table", "group_table", "vcent", "pi", "pi_t"))):
        assert rc(**bad) == N.TQK_EINVAL, bad
    assert rc(batch=0, q=None) == N.TQK_OK and rc(q_len=0, q=None) == N.TQK_OK
    for q_len in (4, 64):  # over the codes; over reconstructed keys and values
        need = lib.tqk_attend_workspace_bytes(ctypes.byref(d), ctypes.byref(desc(q_len=q_len)))
        assert need > 0
        for ws, n in ((at, need - 1), (at + 8, need), (None, need)):
            assert rc(q_len=q_len, ws=ws, n=n) == N.TQK_EWORKSPACE
    assert lib.tqk_attend_workspace_bytes(ctypes.byref(d), ctypes.byref(desc(window=-1))) == 0


def test_gradients_are_refused():
    x = torch.zeros(2, 3, 12 * 128, dtype=torch.float16, requires_grad=True)
    q = torch.zeros(2, 8, 3, 128, dtype=torch.float16, requires_grad=True)
    with pytest.raises(NotImplementedError, match="backward"):
        _call_rope(qkv=x)
    with pytest.raises(NotImplementedError, match="backward"):
        _call_window(q=q)
    with torch.no_grad():  # no gradient asked: refused for the CPU tensors only
        with pytest.raises(RuntimeError, match="GPU"):
            _call_rope(qkv=x)
        with pytest.raises(RuntimeError, match="GPU"):
            _call_window(q=q)
