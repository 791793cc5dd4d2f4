"""Calls of the operators around the cache that would be answered without what was
asked for: gradients, forward-mode tangents, outputs that share places (no GPU needed)."""

import pytest

torch = pytest.importorskip("torch")

from test_ops_cpu import _call_rope, _call_window  # noqa: E402


def pool_without_a_gpu():
    """A pool's numbers alone: what attend checks before any GPU work."""
    from turboquant_pro_amd import TQKVPool
    pool = object.__new__(TQKVPool)
    pool.max_batch, pool.n_q_heads, pool.n_kv_heads, pool.head_dim = 2, 8, 2, 128
    pool.dtype, pool.input_dtype, pool.f32 = torch.float16, "float16", False
    pool.kcodes = torch.empty(1, dtype=torch.uint8, device="meta")
    return pool


def query(T=3):
    return torch.zeros(2, 8, T, 128, dtype=torch.float16)


def test_attend_refuses_gradients():
    pool = pool_without_a_gpu()
    with pytest.raises(NotImplementedError, match="backward"):
        pool.attend(query().requires_grad_())
    with pytest.raises(NotImplementedError, match="backward"):
        pool.attend(query(), out=query().requires_grad_())
    with torch.no_grad(), pytest.raises(ValueError, match="is on cpu"):  # no gradient asked: refused for its place
        pool.attend(query().requires_grad_())


def test_tangents_are_refused():
    import torch.autograd.forward_ad as fwd
    rows = torch.zeros(2, 3, 12 * 128, dtype=torch.float16)
    kv = torch.zeros(2, 2, 9, 128, dtype=torch.float16)
    with fwd.dual_level():
        for call in (lambda: _call_rope(qkv=fwd.make_dual(rows, rows)),
                     lambda: _call_rope(q_weight=fwd.make_dual(torch.ones(128), torch.ones(128))),
                     lambda: _call_window(q=fwd.make_dual(query(), query())),
                     lambda: _call_window(v=fwd.make_dual(kv, kv)),
                     lambda: pool_without_a_gpu().attend(fwd.make_dual(query(), query()))):
            with pytest.raises(NotImplementedError, match="backward"):
                call()
            with torch.no_grad(), pytest.raises(NotImplementedError, match="backward"):
                call()
        with pytest.raises(RuntimeError, match="GPU"):  # none carried: refused for the CPU tensors only
            _call_window()


def outputs():
    """Outputs that write one place twice, then ones that do not."""
    e = lambda *s: torch.empty(s, dtype=torch.float16)  # noqa: E731
    bad = [e(1, 8, 3, 128).expand(2, -1, -1, -1), e(2, 1, 3, 128).expand(-1, 8, -1, -1), e(2, 8, 1, 128).expand(-1, -1, 3, -1),
           e(8 * 3 * 2 * 128).as_strided((2, 8, 3, 128), (8 * 2 * 128, 2 * 128, 64, 1)),
           e(4 * 8 * 3 * 128).as_strided((2, 8, 3, 128), (1024, 384, 128, 1))]
    good = [e(2, 8, 3, 128), e(2, 3, 8, 128).transpose(1, 2), e(3, 2, 8, 136)[..., :128].permute(1, 2, 0, 3),
            e(2, 12, 5, 128)[:, 2:10, 1:4]]
    return bad, good


def test_outputs_that_overlap_themselves():
    bad, good = outputs()
    for out in bad:
        with pytest.raises(ValueError, match="share memory"):
            _call_window(out=out)
        with pytest.raises(ValueError, match="share memory"):
            pool_without_a_gpu().attend(query(), out=out)
    for out in good:
        with pytest.raises(RuntimeError, match="GPU"):
            _call_window(out=out)
        with pytest.raises(ValueError, match="is on cpu"):
            pool_without_a_gpu().attend(query(), out=out)
    one = torch.empty((1, 8, 1, 128), dtype=torch.float16)  # dimensions of one: any stride
    with pytest.raises(RuntimeError, match="GPU"):
        _call_window(q=query()[:1, :, :1], k=torch.zeros(1, 2, 9, 128, dtype=torch.float16),
                     v=torch.zeros(1, 2, 9, 128, dtype=torch.float16), out=one.as_strided((1, 8, 1, 128), (0, 128, 0, 1)))


def test_append_qkv_refuses_rows_of_another_device():
    """Rows, and positions beside them, that are not on the pool's device."""
    pool = pool_without_a_gpu()
    pool.seq_lens, pool.device = torch.zeros(2, dtype=torch.int32), torch.device("meta")
    rows = torch.zeros(2, 3, 12 * 128, dtype=torch.float16)
    with pytest.raises(ValueError, match="the pool on"):
        pool.append_qkv(rows, torch.ones(64), positions=torch.zeros(2, dtype=torch.int32))
