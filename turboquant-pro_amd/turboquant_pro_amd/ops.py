"""The model step's operators around the cache: head norms with the position
rotation (:func:`norm_rope`) and attention over dense keys and values with a
sliding window and first tokens that stay visible (:func:`window_attention`).

Both run hand-written gfx950 kernels behind ``include/tqk.h`` on the current
stream of their tensors' device; they have no CPU form and no backward pass.  ``TQKVPool.append_qkv``
and ``TQKVPool.attend`` are their counterparts on a coded cache.
"""

from __future__ import annotations

import ctypes
import functools
import math

from . import _native as N
from .codebooks import HEAD_DIMS


def _torch():
    import torch
    return torch


@functools.lru_cache(None)
def _types():
    torch = _torch()
    return {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def _on_gpu(what, *tensors):
    """The one GPU that every given tensor is on."""
    dev = tensors[0].device
    if dev.type != "cuda":
        raise RuntimeError(f"{what} runs on a ROCm GPU (gfx950); got a tensor on {dev}")
    for t in tensors[1:]:
        if t is not None and t.device != dev:
            raise ValueError(f"{what}: tensors on {dev} and {t.device}")
    return dev


def needs_grad(*tensors):
    """Whether a gradient or a forward-mode tangent is asked of any of the tensors
    (None: none)."""
    torch = _torch()
    fwd = torch.autograd.forward_ad
    dual = getattr(fwd, "_current_level", 0) >= 0  # (inside a dual level: rare, and dear to ask every tensor)
    for t in tensors:
        if t is not None and ((t.requires_grad and torch.is_grad_enabled())
                              or (dual and fwd.unpack_dual(t).tangent is not None)):
            return True
    return False


class on_device:
    """Makes ``dev`` the current device for a launch, where it is not."""

    def __init__(self, dev):
        torch = _torch()
        self.guard = None if torch.cuda.current_device() == dev.index else torch.cuda.device(dev)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def stream_of(dev):
    """The current stream of ``dev`` as the C ABI takes it (the handle alone: the
    stream object of ``torch.cuda.current_stream`` costs a small call 2 us)."""
    return _torch()._C._cuda_getCurrentRawStream(dev.index)


def _is_aligned(x):
    if x.is_contiguous() and x.shape[-1] % 8 == 0 and x.data_ptr() % 16 == 0:
        return True  # (the usual case, without a walk over the strides)
    el = x.element_size()
    return (x.stride(-1) == 1 or x.shape[-1] == 1) and x.data_ptr() % 16 == 0 and all(
        s % 8 == 0 and s * el % 16 == 0 for s, n in zip(x.stride()[:-1], x.shape[:-1]) if n > 1)


def aligned(x):
    """``x`` with its last dimension contiguous, 16-byte rows and a 16-byte
    start: itself, or a copy."""
    if _is_aligned(x):
        return x
    return x.contiguous() if not x.is_contiguous() else x.clone()


def check_out(out, like):
    """A given output: of the queries' shape and type, channels side by side,
    rows of whole 16 bytes and a 16-byte start, no two rows in one place."""
    if tuple(out.shape) != tuple(like.shape) or out.dtype != like.dtype:
        raise ValueError(f"out is {tuple(like.shape)} {like.dtype}, not {tuple(out.shape)} {out.dtype}")
    if not _is_aligned(out):
        raise ValueError("out needs channels side by side, rows of whole 16 bytes and a 16-byte start")
    if out.is_contiguous():
        return
    extent = out.shape[-1]
    for s, n in sorted((s, n) for s, n in zip(out.stride()[:-1], out.shape[:-1]) if n > 1):
        if s < extent:  # (a dimension lies inside the next one's step)
            raise ValueError(f"out: rows share memory (strides {tuple(out.stride())})")
        extent += s * (n - 1)


def _check_rope(qkv, n_q_heads, n_kv_heads, inv_freq, positions, q_weight, k_weight, dtype):
    """Shapes and types of a :func:`norm_rope` call: (B, T, D, out dtype)."""
    torch = _torch()
    types = _types()
    n_q_heads, n_kv_heads = int(n_q_heads), int(n_kv_heads)
    if n_q_heads < 0 or n_kv_heads < 0 or n_q_heads + n_kv_heads == 0:
        raise ValueError("norm_rope needs query or key/value heads")
    heads = n_q_heads + 2 * n_kv_heads
    if qkv.dim() != 3 or qkv.shape[2] % heads:
        raise ValueError(f"norm_rope expects (B, T, {heads} * head_dim) rows, got {tuple(qkv.shape)}")
    B, T, D = int(qkv.shape[0]), int(qkv.shape[1]), int(qkv.shape[2]) // heads
    if D not in HEAD_DIMS:
        raise NotImplementedError(f"head_dim {D}: the gfx950 kernels serve {HEAD_DIMS}")
    dtype = qkv.dtype if dtype is None else dtype
    if qkv.dtype not in types or dtype not in types:
        raise ValueError(f"norm_rope takes and gives fp32, fp16 or bf16, not {qkv.dtype} and {dtype}")
    if inv_freq.dim() != 1 or inv_freq.dtype != torch.float32:
        raise ValueError("inv_freq is a 1-D fp32 tensor, one frequency for each rotated pair")
    if 2 * inv_freq.shape[0] > D:
        raise ValueError(f"{inv_freq.shape[0]} rotated pairs do not fit head_dim {D}")
    if inv_freq.shape[0] % 8:
        raise NotImplementedError(f"{inv_freq.shape[0]} rotated pairs: the gfx950 kernel takes multiples of 8")
    if positions.dtype not in (torch.int32, torch.int64) or tuple(positions.shape) not in ((B,), (B, T)):
        raise ValueError(f"positions are int32 or int64 of shape ({B},) (of first tokens) or ({B}, {T}), "
                         f"not {positions.dtype} {tuple(positions.shape)}")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None and (tuple(w.shape) != (D,) or w.dtype not in (qkv.dtype, torch.float32)):
            raise ValueError(f"{name} is ({D},) in the rows' type or fp32, not {tuple(w.shape)} {w.dtype}")
    return B, T, D, dtype


def norm_rope(qkv, n_q_heads: int, n_kv_heads: int, inv_freq, positions, *, q_weight=None, k_weight=None,
              eps: float = 1e-6, weight_offset: float = 0.0, interleaved: bool = False, rope_scale: float = 1.0,
              dtype=None):
    """Queries, keys and values of new tokens from their projection rows.

    ``qkv`` ``(B, T, (Hq + 2 Hkv) * D)`` fp32, fp16 or bf16: the query heads,
    then the key heads, then the value heads of a token.  Queries are
    normalised per head by ``x * rsqrt(mean(x^2) + eps) * (q_weight +
    weight_offset)`` when ``q_weight`` ``(D,)`` is given, keys likewise; then
    the first ``2 * len(inv_freq)`` channels are rotated by ``position *
    inv_freq`` in pairs ``(i, i + R/2)`` (``interleaved``: ``(2i, 2i + 1)``)
    and scaled by ``rope_scale``; values are only converted.  ``positions``:
    ``(B, T)``, or ``(B,)`` for the position of every sequence's first token
    (int32 or int64).  Computed in fp32, the angles in 64 bits, and rounded
    once to ``dtype`` (the rows' by default).

    Returns ``q (B, Hq, T, D)``, ``k`` and ``v`` ``(B, Hkv, T, D)``: what
    ``TQKVPool.append`` and ``TQKVPool.attend`` take."""
    torch = _torch()
    B, T, D, dtype = _check_rope(qkv, n_q_heads, n_kv_heads, inv_freq, positions, q_weight, k_weight, dtype)
    if needs_grad(qkv, q_weight, k_weight):
        raise NotImplementedError("norm_rope has no backward pass: call it under torch.no_grad()")
    dev = _on_gpu("norm_rope", qkv, inv_freq, positions, q_weight, k_weight)
    types = _types()
    if q_weight is not None and k_weight is not None and q_weight.dtype != k_weight.dtype:
        q_weight, k_weight = q_weight.float(), k_weight.float()
    w = q_weight if q_weight is not None else k_weight
    qkv, inv_freq, positions = aligned(qkv), inv_freq.contiguous(), positions.contiguous()
    q_weight = None if q_weight is None else aligned(q_weight)
    k_weight = None if k_weight is None else aligned(k_weight)
    q = torch.empty((B, n_q_heads, T, D), dtype=dtype, device=dev)
    k = torch.empty((B, n_kv_heads, T, D), dtype=dtype, device=dev)
    v = torch.empty_like(k)
    if B * T:
        d = N.RopeDesc(B, T, n_q_heads, n_kv_heads, D, 2 * inv_freq.shape[0], bool(interleaved), types[qkv.dtype],
                       types[dtype], 0 if w is None else types[w.dtype], positions.dtype == torch.int64,
                       positions.dim() == 2, qkv.stride(0) if B > 1 else 0, qkv.stride(1) if T > 1 else 0,
                       eps, weight_offset, rope_scale)
        with on_device(dev):
            N.check(N.lib().tqk_norm_rope(ctypes.byref(d), qkv.data_ptr(), positions.data_ptr(), inv_freq.data_ptr(),
                                          None if q_weight is None else q_weight.data_ptr(),
                                          None if k_weight is None else k_weight.data_ptr(),
                                          q.data_ptr(), k.data_ptr(), v.data_ptr(), stream_of(dev)), "norm_rope")
    return q, k, v


def window_args(window, sinks):
    """``window`` (None: 0) and ``sinks`` as whole numbers of the C ABI."""
    if window is not None and int(window) < 1:
        raise ValueError("window is at least 1 token (the query's own), or None")
    if int(sinks) < 0:
        raise ValueError("sinks is not negative")
    top = 2 ** 31 - 1  # (a longer window or more sinks than an int32 length: all keys)
    return 0 if window is None or int(window) > top else int(window), min(int(sinks), top)


def strides_of(x):
    """Batch, head and token strides for the C ABI (of a size of one: 0)."""
    (b, h, t, _), (sb, sh, st, _) = x.shape, x.stride()
    return sb if b > 1 else 0, sh if h > 1 else 0, st if t > 1 else 0


def lengths_arg(x, B, name):
    if x is None:
        return None
    torch = _torch()
    if tuple(x.shape) != (B,) or x.dtype != torch.int32:
        raise ValueError(f"{name} is ({B},) int32, not {tuple(x.shape)} {x.dtype}")
    return x.contiguous()


def window_attention(q, k, v, *, window: int | None = None, sinks: int = 0, scale: float | None = None,
                     kv_lens=None, q_lens=None, kv_starts=None, out=None):
    """Causal attention over dense keys and values with a sliding window and
    first tokens that stay visible.

    ``q`` ``(B, Hq, T, D)``, ``k`` and ``v`` ``(B, Hkv, L, D)``, fp16 or bf16,
    any strides; query head i reads kv head ``i // (Hq / Hkv)``.  The queries
    are a sequence's last: with ``n = kv_lens[b]`` keys (L) and ``m =
    q_lens[b]`` queries (T), query t stands at ``p = n - m + t`` and sees the
    keys j of ``[start, p]``, ``start = kv_starts[b]`` (0; a left-padded
    batch's first tokens), with ``j > p - window`` (every one with None) or
    ``j < start + sinks``.  Lengths are int32 ``(B,)`` tensors on the device.

    Returns ``(B, Hq, T, D)`` in the inputs' type, ``out`` where given (any
    strides of whole 16 bytes that keep its rows apart; it shares no memory
    with ``k`` and ``v``), else laid out ``(B, T, Hq, D)`` as the output
    projection reads it.  A query that sees nothing and rows ``t >= m`` get
    zeros.  ``scale``: ``1/sqrt(D)`` by default, positive."""
    torch = _torch()
    types = _types()
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3]:
        raise ValueError(f"window_attention expects q (B, Hq, T, D) and k, v (B, Hkv, L, D), got {tuple(q.shape)}, "
                         f"{tuple(k.shape)} and {tuple(v.shape)}")
    B, Hq, T, D = q.shape
    _, Hkv, L, _ = k.shape
    if Hkv < 1 or Hq < 1 or Hq % Hkv:
        raise ValueError(f"{Hq} query heads are no multiple of {Hkv} kv heads")
    if D not in HEAD_DIMS:
        raise NotImplementedError(f"head_dim {D}: the gfx950 kernels serve {HEAD_DIMS}")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"q, k and v are of one type, not {q.dtype}, {k.dtype} and {v.dtype}")
    if types.get(q.dtype, 0) == 0:
        raise NotImplementedError(f"window_attention takes fp16 or bf16, not {q.dtype}")
    window, sinks = window_args(window, sinks)
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not scale > 0.0 or not math.isfinite(scale):
        raise ValueError(f"scale is positive and finite, not {scale}")
    kv_lens, q_lens, kv_starts = (lengths_arg(kv_lens, B, "kv_lens"), lengths_arg(q_lens, B, "q_lens"),
                                  lengths_arg(kv_starts, B, "kv_starts"))
    if out is not None:
        check_out(out, q)
    if needs_grad(q, k, v, out):
        raise NotImplementedError("window_attention has no backward pass: call it under torch.no_grad()")
    dev = _on_gpu("window_attention", q, k, v, kv_lens, q_lens, kv_starts, out)
    q, k, v = aligned(q), aligned(k), aligned(v)
    if out is None:
        out = torch.empty((B, T, Hq, D), dtype=q.dtype, device=dev).transpose(1, 2)
    if B * T == 0:
        return out
    d = N.AttnDesc(B, Hq, Hkv, D, T, L, window, sinks, types[q.dtype], scale)
    d.q_stride[:], d.k_stride[:], d.v_stride[:], d.o_stride[:] = map(strides_of, (q, k, v, out))
    lib = N.lib()
    with on_device(dev):
        need = lib.tqk_attention_workspace_bytes(ctypes.byref(d))
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        N.check(lib.tqk_attention(ctypes.byref(d), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                                  *(None if x is None else x.data_ptr() for x in (kv_lens, q_lens, kv_starts)),
                                  out.data_ptr(), None if ws is None else ws.data_ptr(), need, stream_of(dev)),
                "window_attention")
    return out
