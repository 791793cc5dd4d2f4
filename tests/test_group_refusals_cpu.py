"""What the entry points over chosen groups, received weights, a shared prefix and
eviction refuse before any GPU work (no GPU needed)."""

import ctypes

import pytest

torch = pytest.importorskip("torch")

from test_attend_refusals_cpu import CACHE  # noqa: E402
from test_ops_cpu import _lib  # noqa: E402

# (max_len 2000, hot window 512, groups of 256: 6 coded groups at most)
STEP = dict(batch=2, q_len=1, max_len=2000, window=0, sinks=0, out_type=1)
MANY = dict(max_groups_per_seq=1 << 15, max_pages_per_seq=1 << 17, n_pages=1 << 22)


class Call:
    """One call with every pointer to a host buffer that is never reached."""

    def __init__(self, cache=None, step=None, stride=1024, null=(), shift=()):
        self.N, self.lib = _lib()
        self.buf = ctypes.create_string_buffer(512)
        self.at = (ctypes.addressof(self.buf) + 15) & ~15
        self.d = self.N.CacheDesc(**{**CACHE, **(cache or {})})
        self.p = self.N.CachePtrs(**{n: None if n in null else self.at for n, _ in self.N.CachePtrs._fields_})
        self.t = self.N.AttendDesc(**{**STEP, **(step or {})})
        self.t.q_stride[:] = self.t.o_stride[:] = [stride] * 3
        self.null, self.shift = null, shift

    def ptr(self, name):
        return None if name in self.null else self.at + (4 if name in self.shift else 0)

    def groups(self, n=2, ws=1 << 40, per_query=False):
        l = self.N.GroupList(n)
        l.stride[:] = [64, 32, 8 if per_query else 0]
        d, t, l = ctypes.byref(self.d), ctypes.byref(self.t), ctypes.byref(l)
        need = self.lib.tqk_attend_groups_workspace_bytes(d, t, l)
        return need, self.lib.tqk_attend_groups(
            d, ctypes.byref(self.p), t, l, self.ptr("q"), self.ptr("lens"), None, self.ptr("groups"), self.ptr("out"),
            self.ptr("ws"), min(ws, max(need - 1, 0)), None)

    def weights(self, ws=1 << 40):
        d, t = ctypes.byref(self.d), ctypes.byref(self.t)
        need = self.lib.tqk_attend_weights_workspace_bytes(d, t)
        return need, self.lib.tqk_attend_weights(d, ctypes.byref(self.p), t, self.ptr("q"), self.ptr("lens"), None,
                                                 self.ptr("out"), self.ptr("weights"), self.ptr("ws"),
                                                 min(ws, max(need - 1, 0)), None)

    def shared(self, n=3, ws=1 << 40):
        d, t = ctypes.byref(self.d), ctypes.byref(self.t)
        need = self.lib.tqk_attend_shared_workspace_bytes(d, t, n)
        return need, self.lib.tqk_attend_shared(d, ctypes.byref(self.p), t, n, self.ptr("q"), self.ptr("lens"), None,
                                                self.ptr("out"), self.ptr("ws"), min(ws, max(need - 1, 0)), None)

    def select(self, **kw):
        s = self.N.SelectDesc(**{**dict(batch=2, q_len=1, max_len=2000, top=4, first=1, last=1, spread=1.0), **kw})
        s.q_stride[:] = list(self.t.q_stride)
        d, s = ctypes.byref(self.d), ctypes.byref(s)
        need = self.lib.tqk_select_groups_workspace_bytes(d, s)
        return need, self.lib.tqk_select_groups(d, ctypes.byref(self.p), s, self.ptr("q"), self.ptr("lens"), None,
                                                self.ptr("groups"), self.ptr("ws"), max(need - 1, 0), None)

    def evict(self, batch=2, keep=4, first=1, last=1, own_tables=True):
        d = ctypes.byref(self.d)
        need = self.lib.tqk_evict_groups_workspace_bytes(d, max(batch, 1))
        other = 0 if own_tables else 64
        return need, self.lib.tqk_evict_groups(
            d, ctypes.byref(self.p), batch, keep, first, last, self.ptr("weights"), self.ptr("lens"),
            None if "block_table" in self.null else self.at + other,
            None if "group_table" in self.null else self.at + other, self.ptr("kept"), self.ptr("ws"),
            max(need - 1, 0), None)


KINDS = ("groups", "weights", "shared")


# (every right call here has a workspace one byte short: refused last, before any launch)
@pytest.mark.parametrize("kind", KINDS + ("select", "evict"))
def test_a_short_workspace_is_refused(kind):
    for cache in ({}, dict(head_dim=64), dict(head_dim=256)):
        c = Call(cache, stride=2048)
        need, rc = getattr(c, kind)()
        assert need > 0 and rc == c.N.TQK_EWORKSPACE
        c = Call(cache, null=("ws",))
        assert getattr(c, kind)()[1] == c.N.TQK_EWORKSPACE
        c = Call(cache, shift=("ws",))
        assert getattr(c, kind)()[1] == c.N.TQK_EWORKSPACE


@pytest.mark.parametrize("kind,names", [
    ("groups", ("q", "lens", "groups", "out", "kcodes", "vcodes", "vnorm", "oent", "ocount", "hot_k", "hot_v", "gscale",
                "gmean", "block_table", "group_table", "vcent", "pi", "pi_t")),
    ("weights", ("q", "lens", "weights", "out", "kcodes", "hot_v", "gscale", "pi_t")),
    ("shared", ("q", "lens", "out", "vcodes", "hot_k", "gmean", "group_table")),
    ("select", ("q", "lens", "groups", "gscale", "gmean", "group_table")),
    ("evict", ("weights", "lens", "kept", "hot_k", "hot_v", "block_table", "group_table"))])
def test_missing_buffers_are_refused(kind, names):
    for name in names:
        c = Call(null=(name,))
        assert getattr(c, kind)()[1] == c.N.TQK_EINVAL, name


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("cache,step,stride,shift,want", [
    ({}, dict(batch=-1), 1024, (), "EINVAL"),
    ({}, dict(q_len=-1), 1024, (), "EINVAL"),
    ({}, dict(max_len=-1), 1024, (), "EINVAL"),
    ({}, dict(max_len=2100), 1024, (), "EINVAL"),        # past the tables
    ({}, dict(out_type=2), 1024, (), "EUNSUPPORTED"),
    ({}, dict(q_len=1 << 28, batch=24), 1024, (), "EINVAL"),
    (MANY, dict(q_len=1 << 20, batch=128), 1024, (), "EINVAL"),  # rows past 2^30
    ({}, {}, 1020, (), "EINVAL"),                        # rows between 16-byte borders
    ({}, {}, 1024, ("q",), "EINVAL"),
    ({}, {}, 1024, ("out",), "EINVAL"),
    (dict(input_f32=1), {}, 1024, (), "EUNSUPPORTED"),
    (dict(n_pages=1 << 25), {}, 1024, (), "EUNSUPPORTED"),
    (dict(outlier_cap=0), {}, 1024, (), "EINVAL"),
    (dict(n_q_heads=9), {}, 1024, (), "EINVAL"),
    (dict(head_dim=96), {}, 1024, (), "EUNSUPPORTED"),
])
def test_wrong_steps_are_refused(kind, cache, step, stride, shift, want):
    c = Call(cache, step, stride, shift=shift)
    need, rc = getattr(c, kind)()
    assert rc == getattr(c.N, "TQK_" + want)
    assert need == 0 or shift


def test_windows_belong_to_weights():
    for step in (dict(window=300), dict(sinks=1)):
        for kind in ("groups", "shared"):
            c = Call(step=step)
            assert getattr(c, kind)() == (0, c.N.TQK_EINVAL)
        c = Call(step=step)
        assert c.weights()[1] == c.N.TQK_EWORKSPACE


def test_lists():
    c = Call()
    for n in (-1, (1 << 24) + 1):
        assert c.groups(n) == (0, c.N.TQK_EINVAL)
    assert c.groups(0)[1] == c.N.TQK_EWORKSPACE
    c = Call(null=("groups",))  # (a list of none needs no entries)
    assert c.groups(0)[1] == c.N.TQK_EWORKSPACE
    # the splits are those of groups that there are, however long the list
    c = Call(MANY, dict(max_len=32768))
    most = c.groups(1 << 24)[0]
    assert most == c.groups(126)[0] > 0
    # no list but the lengths: nothing to do without queries or sequences
    for step in (dict(batch=0), dict(q_len=0)):
        c = Call(step=step, null=("q", "lens", "groups", "out", "ws"))
        for kind in KINDS:
            assert getattr(c, kind)() == (0, c.N.TQK_OK)


def test_shared_groups_are_coded_ones():
    c = Call()
    for n in (0, -1, 7):
        assert c.shared(n) == (0, c.N.TQK_EINVAL)
    assert c.shared(6)[1] == c.N.TQK_EWORKSPACE
    c = Call(dict(key_grid=2, outliers_per_channel=0))
    assert c.shared() == (0, c.N.TQK_EUNSUPPORTED)
    assert c.groups()[1] == c.weights()[1] == c.N.TQK_EWORKSPACE


def test_weights_of_many_sequences():
    """A workgroup row a (sequence, kv head) of the sums."""
    c = Call({**MANY, "n_kv_heads": 8, "n_q_heads": 8}, dict(batch=8192))
    assert c.weights()[1] == c.N.TQK_EINVAL
    c = Call({**MANY, "n_kv_heads": 8, "n_q_heads": 8}, dict(batch=8191))
    assert c.weights()[1] == c.N.TQK_EWORKSPACE


@pytest.mark.parametrize("batch,q_len,max_len", [(16, 2000, 131072), (1, 1 << 20, 32768), (64, 1, 1 << 20), (3, 77, 700)])
def test_the_blocks_sums_are_bounded(batch, q_len, max_len):
    """256 MiB of blocks' maxima and sums beside a slice's partial results, or one query's."""
    c = Call({**MANY, "n_q_heads": 8, "n_kv_heads": 1}, dict(batch=batch, q_len=q_len, max_len=max_len))
    need, rc = c.weights()
    blocks = (max_len - 512 + 255) // 256 * 8
    one = batch * 8 * blocks * 8
    slice_ = max(min(q_len, (256 << 20) // one), 1)
    assert 0 < need <= one * slice_ + 64 * batch * 8 * slice_ * (128 + 2) * 4 + batch * 8 * slice_ * 8 + 256
    assert rc == c.N.TQK_EWORKSPACE


@pytest.mark.parametrize("kw,want", [
    (dict(top=0), "EINVAL"), (dict(first=-1), "EINVAL"), (dict(last=-1), "EINVAL"), (dict(first=3, last=2), "EINVAL"),
    (dict(first=2 ** 31 - 1, last=2 ** 31 - 1), "EINVAL"), (dict(spread=-0.5), "EINVAL"),
    (dict(spread=float("nan")), "EINVAL"), (dict(spread=float("inf")), "EINVAL"), (dict(batch=-1), "EINVAL"),
    (dict(q_len=-1), "EINVAL"), (dict(max_len=2100), "EINVAL"), (dict(first=4, last=0), "EWORKSPACE"),
    (dict(first=0, last=0), "EWORKSPACE"), (dict(top=1 << 24), "EWORKSPACE"), (dict(spread=0.0), "EWORKSPACE")])
def test_choices(kw, want):
    c = Call()
    need, rc = c.select(**kw)
    assert rc == getattr(c.N, "TQK_" + want) and (need > 0) == (want == "EWORKSPACE")


def test_choices_of_other_caches():
    for cache in (dict(input_f32=1), dict(key_grid=2, outliers_per_channel=0)):
        c = Call(cache)
        assert c.select() == (0, c.N.TQK_EUNSUPPORTED)
    c = Call(stride=1020)
    assert c.select() == (0, c.N.TQK_EINVAL)
    c = Call(shift=("q",))
    assert c.select()[1] == c.N.TQK_EINVAL
    # scores in slices of 256 MiB of queries
    c = Call(MANY)
    assert c.select(q_len=1 << 20, max_len=1 << 20, batch=2)[0] <= (256 << 20) + 16
    for kw in (dict(batch=0), dict(q_len=0)):
        c = Call(null=("q", "lens", "groups", "ws"))
        assert c.select(**kw) == (0, c.N.TQK_OK)


@pytest.mark.parametrize("kw,want", [
    (dict(batch=-1), "EINVAL"), (dict(batch=65536), "EINVAL"), (dict(keep=-1, first=0, last=0), "EINVAL"),
    (dict(first=-1), "EINVAL"), (dict(last=-1), "EINVAL"), (dict(keep=1), "EINVAL"),
    (dict(first=2 ** 31 - 1, last=2 ** 31 - 1, keep=5), "EINVAL"), (dict(own_tables=False), "EINVAL"),
    (dict(keep=0, first=0, last=0), "EWORKSPACE"), (dict(keep=2), "EWORKSPACE")])
def test_evictions(kw, want):
    c = Call()
    assert c.evict(**kw)[1] == getattr(c.N, "TQK_" + want)


def test_evictions_of_other_caches():
    c = Call(dict(zero_point=2), null=())
    assert c.evict()[1] == c.N.TQK_EUNSUPPORTED
    c = Call(dict(max_pages_per_seq=23))  # (a page short of six groups)
    assert c.evict()[1] == c.N.TQK_EINVAL
    c = Call(shift=("kept",), null=())
    assert c.evict()[1] == c.N.TQK_EWORKSPACE
    for cache, want in ((dict(hot_window=4096, hot_ring=4096, group_tokens=2048), "EWORKSPACE"),
                        (dict(hot_window=4097, hot_ring=4097, group_tokens=2049), "EUNSUPPORTED"),
                        (dict(input_f32=1), "EWORKSPACE")):
        c = Call(cache)
        rc = c.evict()[1]
        if c.lib.tqk_check_desc(ctypes.byref(c.d)) == c.N.TQK_OK:
            assert rc == getattr(c.N, "TQK_" + want)
        else:
            assert rc not in (c.N.TQK_OK, c.N.TQK_EHIP)
    c = Call(null=("weights", "lens", "kept", "ws"))
    assert c.evict(batch=0)[1] == c.N.TQK_OK
