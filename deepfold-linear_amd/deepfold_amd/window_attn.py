"""Attention over a sliding window and a few first tokens, its rolling cache and its
single-token form, on MI355X.

* ``flash_window_attn``: for whole sequences, forward and backward (``dfl_window_attn_*``).
  Query i stands at position t = i + N - M and sees the keys t - window < j <= t (with
  ``causal=False``: |t - j| < window) and the first ``n_sink`` keys (causal: up to t), so
  its cost is linear in the length.  Fewer key heads than query heads are shared, a
  learned bias by relative position (``rel_pos_bias``'s tables) is formed in the kernels.
* ``window_cache_fill`` / ``window_decode_attn``: the same attention one token at a time
  (``dfl_window_cache_fill``, ``dfl_window_decode``), over a rolling cache of n_sink + window
  slots that a prompt fills.  The caches are tensors of the inputs' type, or hold 8 or 4 bits an
  element (``quantized_cache``; ``dfl_lowbit_cache_fill``, ``dfl_lowbit_decode``).  A whole run::

      o = flash_window_attn(Q, K, V, mask, window=W, n_sink=s)          # the prompt
      window_cache_fill(K, V, lengths, k_cache, v_cache, n_sink=s)      # caches (B, Hk, s + W, d)
      while ...:
          o = window_decode_attn(q, k, v, k_cache, v_cache, lengths, n_sink=s)
          lengths += 1

* ``window_cache_read``: what a cache holds, in the order of the positions (``dfl_window_cache_read``).
  A prompt in chunks: each one's rows attend to the cache's and to its own::

      Kp, Vp, m = window_cache_read(k_cache, v_cache, lengths, D, n_sink=s)
      o = flash_window_attn(Q, torch.cat((Kp, K), 2), torch.cat((Vp, V), 2), torch.cat((m, mask), 1), window=W, n_sink=s)
      window_cache_fill(K, V, chunk, k_cache, v_cache, n_sink=s, starts=lengths)   # chunk: rows of each sample
      lengths += chunk

  Chunks of at most ``window`` rows are right from any lengths on (0 too); longer ones where the caches hold the n_sink
  first tokens already: those that come with a chunk stand at its rows, not at the first n_sink, and are seen no further
  than the window.

Where ``flash_atom_attn`` has fixed windows of 32 queries and 128 keys, here the window
moves with the query.  The reference has no counterpart.  bf16 runs on bf16 MFMA with fp32
sums, any other type in fp32, as in the other attention ops; CPU tensors raise.
"""

from __future__ import annotations

import ctypes
import math

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._attn import _compute_dtype, _unit_inner
from .quantized_cache import QuantizedCache, groups_of
from .rel_pos_bias import edge_array

MAX_HEAD_DIM = 128
MAX_SINK = 128
MAX_SLOTS = 1 << 28  # window and rows of a chunk of caches in few bits
EXACT_KEYS = 256  # rows of at most this many keys need no remainder of o (csrc/window_geometry.h)


def _check_window(what, window, n_sink):
    if window < 1:
        raise ValueError(f"{what}: window={window} must be positive")
    if not 0 <= n_sink <= MAX_SINK:
        raise ValueError(f"{what}: n_sink={n_sink} outside [0, {MAX_SINK}]")


def _scale(what, scale, d):
    if scale is None:
        return 1.0 / math.sqrt(d)
    scale = float(scale)
    if not 1e-30 <= scale <= 1e30:
        raise ValueError(f"{what}: scale={scale} outside [1e-30, 1e30]")
    return scale


def _fwd_params(dt, q, k, v, mask, tab, arr, window, n_sink, causal, scale, o, lse):
    B, H, M, d = q.shape
    return _lib.WindowAttnParams(
        _lib.DFL_BF16 if dt == torch.bfloat16 else _lib.DFL_F32, q.data_ptr(), k.data_ptr(), v.data_ptr(),
        *q.stride()[:3], *k.stride()[:3], *v.stride()[:3], _lib.ptr(mask), _lib.ptr(tab),
        None if arr is None else ctypes.addressof(arr), 0 if arr is None else len(arr), B, H, k.shape[1], M,
        k.shape[2], d, window, n_sink, int(causal), scale, o.data_ptr(), _lib.ptr(lse))


def _forward(q, k, v, table, mask, arr, window, n_sink, causal, scale, train):
    dev = _lib.require_gpu(q, k, v, table, mask)
    dt = _compute_dtype(q)
    qc, kc, vc = (_unit_inner(t.detach().to(dt)) for t in (q, k, v))
    tab = None if table is None else table.detach().to(torch.float32).contiguous()
    mk = None if mask is None else mask.detach().to(torch.float32).contiguous()
    B, H, M, d = qc.shape
    o = torch.empty(B, H, M, d, dtype=dt, device=dev)
    lse = torch.empty(B, H, M, dtype=torch.float32, device=dev) if train else None
    # (without it the backward forms D from the products, as it does for rows of so few keys in any case)
    keys = min((window if causal else 2 * window - 1) + n_sink, kc.shape[2])
    rest = torch.empty_like(o) if train and dt == torch.bfloat16 and keys > EXACT_KEYS else None
    p = _fwd_params(dt, qc, kc, vc, mk, tab, arr, window, n_sink, causal, scale, o, lse)
    p.o_rest = _lib.ptr(rest)
    lib = _lib.load()
    with _lib.on_device(dev):
        rc = _lib.timed_launch("window_attn_fwd", dev, lambda: lib.dfl_window_attn_fwd(
            ctypes.byref(p), ctypes.c_void_p(_lib.stream_handle(dev))))
    _lib.check(rc, "dfl_window_attn_fwd")
    return (qc, kc, vc, tab, mk, o, rest, lse), (o if dt == q.dtype else o.to(q.dtype))


class WindowAttnFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, table, mask, arr, window, n_sink, causal, scale):
        saved, out = _forward(q, k, v, table, mask, arr, window, n_sink, causal, scale, True)
        ctx.save_for_backward(*saved)
        ctx.meta = (arr, window, n_sink, causal, scale, q.dtype, k.dtype, v.dtype,
                    None if table is None else table.dtype)
        ctx.set_materialize_grads(False)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_o):
        none = (None,) * 6
        if grad_o is None:
            return (None,) * 4 + none
        qc, kc, vc, tab, mk, o, rest, lse = ctx.saved_tensors
        arr, window, n_sink, causal, scale, qdt, kdt, vdt, tdt = ctx.meta
        need = ctx.needs_input_grad
        dev, dt = qc.device, qc.dtype
        B, H, M, d = qc.shape
        Hk, N = kc.shape[1], kc.shape[2]
        go = grad_o.to(dt).contiguous()
        dq = torch.empty(B, H, M, d, dtype=dt, device=dev)
        dk = torch.empty(B, Hk, N, d, dtype=dt, device=dev)
        dv = torch.empty(B, Hk, N, d, dtype=dt, device=dev)
        dtab = torch.empty_like(tab) if tab is not None and need[3] else None
        p = _fwd_params(dt, qc, kc, vc, mk, tab, arr, window, n_sink, causal, scale, o, lse)
        p.grad_o, p.dq, p.dk, p.dv, p.drel_table = (go.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                                                    _lib.ptr(dtab))
        p.o_rest = _lib.ptr(rest)
        lib = _lib.load()
        # a workspace of the call's own: calls on other streams and captured graphs cannot share it
        ws = torch.empty(lib.dfl_window_attn_workspace_size(B, H, Hk, M, N, d, window, n_sink, int(causal), p.n_edges),
                         dtype=torch.uint8, device=dev)
        with _lib.on_device(dev):
            rc = _lib.timed_launch("window_attn_bwd", dev, lambda: lib.dfl_window_attn_bwd(
                ctypes.byref(p), ctypes.c_void_p(ws.data_ptr()), ws.numel(),
                ctypes.c_void_p(_lib.stream_handle(dev))))
        _lib.check(rc, "dfl_window_attn_bwd")
        cast = lambda t, to: t if t is None or t.dtype == to else t.to(to)
        return (cast(dq, qdt) if need[0] else None, cast(dk, kdt) if need[1] else None,
                cast(dv, vdt) if need[2] else None, cast(dtab, tdt), *none)


def flash_window_attn(
    Q: torch.Tensor,
    K: torch.Tensor,
    V: torch.Tensor,
    mask: torch.Tensor | None = None,
    *,
    window: int,
    n_sink: int = 0,
    causal: bool = True,
    scale: float | None = None,
    rel_table: torch.Tensor | None = None,
    rel_edges=None,
) -> torch.Tensor:
    """Attention over a sliding window and the first ``n_sink`` tokens (module docstring).

    Q (B,H,M,D) or (H,M,D); K, V (B,Hk,N,D) or (Hk,N,D) with H a multiple of Hk (query head h reads key head
    h // (H // Hk)), M <= N, D <= 128, any strides.  mask (B,N) or (N,), 0 = masked: a masked key reaches nothing,
    whatever its values, and rows of masked queries are zero, as is a row that sees no key.  (A key that only the
    window or the table hides is ordinary data: a NaN or infinity in its V may reach queries nearby, and one in the
    gradient of a query's row the keys nearby.)  ``scale`` defaults to
    D ** -0.5 and is positive.  ``rel_table`` with ``rel_edges``: scores get table[h, bucket(j - t)], see
    ``rel_pos_bias``, whose ``bidirectional`` is ``not causal`` here; an entry of -inf (or below -1e30) takes its keys out.

    Returns O with the shape and dtype of Q; gradients to Q, K, V and rel_table."""
    if not Q.dim() == K.dim() == V.dim() or Q.dim() not in (3, 4):
        raise ValueError("flash_window_attn: Q, K, V must be (B,H,M,D) / (B,Hk,N,D), or the same without B")
    unbatched = Q.dim() == 3
    if unbatched:
        Q, K, V = Q.unsqueeze(0), K.unsqueeze(0), V.unsqueeze(0)
        mask = None if mask is None else mask.unsqueeze(0)
    B, H, M, d = Q.shape
    Hk, N = K.shape[1], K.shape[2]
    if K.shape != (B, Hk, N, d) or V.shape != K.shape:
        raise ValueError(f"flash_window_attn: K {tuple(K.shape)} and V {tuple(V.shape)} do not fit Q {tuple(Q.shape)}")
    if Hk < 1 or H % Hk:
        raise ValueError(f"flash_window_attn: {H} query heads are no multiple of {Hk} key heads")
    if not 1 <= d <= MAX_HEAD_DIM:
        raise ValueError(f"flash_window_attn: head dim {d} outside [1, {MAX_HEAD_DIM}]")
    if M > N:
        raise ValueError(f"flash_window_attn: {M} queries for {N} keys")
    if mask is not None and mask.shape != (B, N):
        raise ValueError(f"flash_window_attn: mask {tuple(mask.shape)} must be ({B}, {N})")
    window, n_sink, causal = min(int(window), 1 << 28), int(n_sink), bool(causal)
    _check_window("flash_window_attn", window, n_sink)
    if (rel_table is None) != (rel_edges is None):
        raise ValueError("flash_window_attn: give rel_table and rel_edges together")
    arr = None if rel_table is None else edge_array(rel_table, rel_edges, H, not causal)
    scale = _scale("flash_window_attn", scale, d)
    if not (Q.is_floating_point() and K.is_floating_point() and V.is_floating_point()):
        raise TypeError("flash_window_attn: Q, K, V must be floating point")
    if B == 0 or H == 0 or M == 0:
        _lib.require_gpu(Q, K, V)
        raise ValueError("flash_window_attn: empty batch, heads or queries")
    if _lib.recording() or torch.is_grad_enabled() and (
            Q.requires_grad or K.requires_grad or V.requires_grad or (rel_table is not None and rel_table.requires_grad)):
        O = WindowAttnFn.apply(Q, K, V, rel_table, mask, arr, window, n_sink, causal, scale)
    else:
        O = _forward(Q, K, V, rel_table, mask, arr, window, n_sink, causal, scale, False)[1]
    return O.squeeze(0) if unbatched else O


def _meet(shape, stride, apart):
    """Whether two tensors of one shape and stride, ``apart`` elements between their first, have an element in common.
    Each stride reaches over the extents below it (``_check_caches``), so the difference of two elements is, widest stride
    first, the quotient or the next in that dimension."""
    rest = {apart}
    for s, n in sorted(zip(stride, shape), reverse=True):
        if n > 1:
            rest = {r - c * s for r in rest for c in (r // s, r // s + 1) if -n < c < n}
    return 0 in rest


def _extent(what, c, inner):
    """Elements from the first to the last of a cache's (B,Hk,n) rows of ``inner`` elements; every row a memory of its own:
    strides that can hold the extents below them."""
    if c.is_contiguous():
        return c.numel()
    at = inner
    for s, n in sorted((s, n) for s, n in zip(c.stride()[:3], c.shape[:3]) if n > 1):
        if s < at:
            raise ValueError(f"{what}: the cache's slots overlap (strides {c.stride()})")
        at = s * (n - 1) + at
    return at


def _check_caches(what, k_cache, v_cache, B, Hk, d, dtype, n_sink):
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape:
        raise ValueError(f"{what}: k_cache and v_cache must be (B,Hk,n_sink + window,D) alike")
    if k_cache.shape[0] != B or k_cache.shape[1] != Hk or k_cache.shape[3] != d:
        raise ValueError(f"{what}: cache {tuple(k_cache.shape)} does not fit ({B}, {Hk}, *, {d})")
    if k_cache.dtype != dtype or v_cache.dtype != dtype or dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"{what}: caches and inputs must all be bf16 or all fp32, got {k_cache.dtype}, "
                        f"{v_cache.dtype} and {dtype}")
    extent = []  # elements from a cache's first to its last
    for c in (k_cache, v_cache):
        if c.stride(3) != 1 and d > 1:
            raise ValueError(f"{what}: the caches' last dimension must be contiguous")
        extent.append(_extent(what, c, d))
    apart, odd = divmod(v_cache.data_ptr() - k_cache.data_ptr(), k_cache.element_size())
    if -extent[1] < apart < extent[0] and (
            odd or k_cache.stride() != v_cache.stride() or _meet(k_cache.shape, k_cache.stride(), apart)):
        raise ValueError(f"{what}: k_cache and v_cache share memory, or interleave with different strides")
    window = k_cache.shape[2] - n_sink
    _check_window(what, window, n_sink)
    return window


def _check_codes(what, k_cache, v_cache, B, Hk, d, n_sink):
    """The window of two caches in few bits, whose four tensors have no element in common."""
    bits, groups, regions = k_cache.bits, groups_of(d), []
    if bits not in (4, 8) or v_cache.bits != bits:
        raise ValueError(f"{what}: k_cache and v_cache must both hold 8 or both 4 bits, got {bits} and {v_cache.bits}")
    slots = k_cache.codes.shape[2] if k_cache.codes.dim() == 4 else 0
    shape, exp_shape = (B, Hk, slots, groups * 4 * bits), (B, Hk, groups)
    for codes, exps, _ in (k_cache, v_cache):
        if codes.dtype != torch.uint8 or exps.dtype != torch.uint8:
            raise TypeError(f"{what}: a quantized cache's codes and exponents must be uint8")
        es = exps.shape
        if codes.shape != shape or len(es) != 4 or es[:3] != exp_shape:
            raise ValueError(f"{what}: quantized cache {tuple(codes.shape)}, {tuple(es)} does not fit "
                             f"({B}, {Hk}, *, {d}) in {bits} bits")
        if es[3] < slots or es[3] % 4:
            raise ValueError(f"{what}: {es[3]} exponents a group for {slots} slots: need a multiple of 4, as many at least")
        for t, unit in ((codes, 16), (exps, 4)):
            at = t.data_ptr()
            if t.is_contiguous():
                size, fine = t.numel(), True
            else:
                fine = t.stride(3) == 1 and all(s % unit == 0 for s, n in zip(t.stride(), t.shape[:3]) if n > 1)
                size = _extent(what, t, t.shape[3])
            if at % unit or not fine:
                raise ValueError(f"{what}: a quantized cache's rows must be contiguous, {unit}-byte aligned")
            regions.append((at, at + size, t))
    regions.sort(key=_address)
    if regions[0][1] > regions[1][0] or regions[1][1] > regions[2][0] or regions[2][1] > regions[3][0]:
        for i, (a0, a1, s) in enumerate(regions):
            for b0, b1, t in regions[i + 1:]:
                if a0 < b1 and b0 < a1 and (s.shape != t.shape or s.stride() != t.stride() or
                                            _meet(s.shape, s.stride(), b0 - a0)):
                    raise ValueError(f"{what}: codes or exponents of the caches share memory")
    window = slots - n_sink
    _check_window(what, window, n_sink)
    if window > MAX_SLOTS:
        raise ValueError(f"{what}: window={window} above {MAX_SLOTS}")
    return window


def _address(region):
    return region[0]


def _same_kind(what, k_cache, v_cache):
    """Whether the caches are in few bits."""
    few = isinstance(k_cache, QuantizedCache)
    if few != isinstance(v_cache, QuantizedCache):
        raise TypeError(f"{what}: k_cache and v_cache must be of one kind")
    return few


def _check_lengths(what, lengths, B, name="lengths"):
    if lengths.shape != (B,) or lengths.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{what}: {name} must be ({B},) int32 or int64")


def _lengths(lengths):
    return _lib.to_int32(lengths).contiguous()


def _no_grad_inputs(what, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad(), or train with flash_window_attn")


def _codes_of(codes, exps):
    return _lib.LowbitCache(codes.data_ptr(), exps.data_ptr(), *codes.stride()[:3], *exps.stride()[:3])


def _dtype_of(t):
    return _lib.DFL_BF16 if t.dtype == torch.bfloat16 else _lib.DFL_F32


def _fill(K, V, lengths, k_cache, v_cache, n_sink, starts=None):
    B, Hk, N, d = K.shape
    dev, at = K.device, _lengths(lengths)
    start = None if starts is None else _lengths(starts)
    k, v = _unit_inner(K.detach()), _unit_inner(V.detach())
    p = _lib.WindowCacheFillParams(
        _dtype_of(K), k.data_ptr(), v.data_ptr(), *k.stride()[:3],
        *v.stride()[:3], at.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), *k_cache.stride()[:3],
        *v_cache.stride()[:3], B, Hk, N, d, k_cache.shape[2] - n_sink, n_sink)
    lib = _lib.load()
    with _lib.on_device(dev):
        if start is None:
            rc = _lib.timed_launch("window_cache_fill", dev, lambda: lib.dfl_window_cache_fill(
                ctypes.byref(p), ctypes.c_void_p(_lib.stream_handle(dev))))
        else:
            rc = _lib.timed_launch("window_cache_fill", dev, lambda: lib.dfl_window_cache_append(
                ctypes.byref(p), ctypes.c_void_p(start.data_ptr()), ctypes.c_void_p(_lib.stream_handle(dev))))
    _lib.check(rc, "dfl_window_cache_fill")
    torch.autograd.graph.increment_version((k_cache, v_cache))


def _fill_codes(K, V, lengths, starts, kc, ke, vc, ve, bits, n_sink):
    B, Hk, N, d = K.shape
    dev, at = K.device, _lengths(lengths)
    start = None if starts is None else _lengths(starts)
    k, v = _unit_inner(K), _unit_inner(V)
    p = _lib.LowbitCacheFillParams(
        _dtype_of(K), bits, k.data_ptr(), v.data_ptr(), *k.stride()[:3], *v.stride()[:3], at.data_ptr(), _lib.ptr(start),
        _codes_of(kc, ke), _codes_of(vc, ve), B, Hk, N, d, kc.shape[2] - n_sink, n_sink)
    lib = _lib.load()
    with _lib.on_device(dev):
        rc = _lib.timed_launch("window_cache_fill", dev, lambda: lib.dfl_lowbit_cache_fill(
            ctypes.byref(p), _lib.stream_handle(dev)))
    _lib.check(rc, "dfl_lowbit_cache_fill")
    torch.autograd.graph.increment_version((kc, ke, vc, ve))


def _read(lengths, kc, ke, vc, ve, bits, d, n_sink, dtype):
    B, Hk, S = kc.shape[:3]
    dev, at = kc.device, _lengths(lengths)
    if bits:
        caches = _codes_of(kc, ke), _codes_of(vc, ve)
    else:
        caches = [_lib.LowbitCache(c.data_ptr(), None, *c.stride()[:3]) for c in (kc, vc)]
    k, v = (torch.empty(B, Hk, S, d, dtype=dtype, device=dev) for _ in range(2))
    mask = torch.empty(B, S, dtype=torch.float32, device=dev)
    p = _lib.WindowCacheReadParams(_dtype_of(k), bits, *caches, at.data_ptr(), k.data_ptr(), v.data_ptr(), mask.data_ptr(),
                                   B, Hk, d, S - n_sink, n_sink)
    lib = _lib.load()
    with _lib.on_device(dev):
        rc = _lib.timed_launch("window_cache_read", dev, lambda: lib.dfl_window_cache_read(
            ctypes.byref(p), _lib.stream_handle(dev)))
    _lib.check(rc, "dfl_window_cache_read")
    return k, v, mask


def _decode_codes(q, k, v, kc, ke, vc, ve, lengths, rel_table, arr, bits, n_sink, scale):
    B, H, d = q.shape
    Hk, window = k.shape[1], kc.shape[2] - n_sink
    dev, at = q.device, _lengths(lengths)
    tab = None if rel_table is None else rel_table.detach().to(torch.float32).contiguous()
    q, k, v = _unit_inner(q), _unit_inner(k), _unit_inner(v)
    o = torch.empty(B, H, d, dtype=q.dtype, device=dev)
    lib = _lib.load()
    nbytes = lib.dfl_lowbit_decode_workspace_size(B, H, Hk, d, window, n_sink)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    p = _lib.LowbitDecodeParams(
        _dtype_of(q), bits, q.data_ptr(), k.data_ptr(), v.data_ptr(), *q.stride()[:2], *k.stride()[:2], *v.stride()[:2],
        _codes_of(kc, ke), _codes_of(vc, ve), at.data_ptr(), _lib.ptr(tab),
        None if arr is None else ctypes.addressof(arr), 0 if arr is None else len(arr), B, H, Hk, d, window, n_sink,
        scale, o.data_ptr())
    with _lib.on_device(dev):
        rc = _lib.timed_launch("window_decode_attn", dev, lambda: lib.dfl_lowbit_decode(
            ctypes.byref(p), _lib.ptr(ws), nbytes, _lib.stream_handle(dev)))
    _lib.check(rc, "dfl_lowbit_decode")
    torch.autograd.graph.increment_version((kc, ke, vc, ve))
    return o


def _decode(q, k, v, k_cache, v_cache, lengths, rel_table, arr, n_sink, scale):
    B, H, d = q.shape
    Hk, window = k.shape[1], k_cache.shape[2] - n_sink
    dev, at = q.device, _lengths(lengths)
    tab = None if rel_table is None else rel_table.detach().to(torch.float32).contiguous()
    q, k, v = _unit_inner(q.detach()), _unit_inner(k.detach()), _unit_inner(v.detach())
    o = torch.empty(B, H, d, dtype=q.dtype, device=dev)
    lib = _lib.load()
    nbytes = lib.dfl_window_decode_workspace_size(B, H, Hk, d, window, n_sink)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    p = _lib.WindowDecodeParams(
        _lib.DFL_BF16 if q.dtype == torch.bfloat16 else _lib.DFL_F32, q.data_ptr(), k.data_ptr(), v.data_ptr(),
        *q.stride()[:2], *k.stride()[:2], *v.stride()[:2], k_cache.data_ptr(), v_cache.data_ptr(),
        *k_cache.stride()[:3], *v_cache.stride()[:3], at.data_ptr(), _lib.ptr(tab),
        None if arr is None else ctypes.addressof(arr), 0 if arr is None else len(arr), B, H, Hk, d, window, n_sink,
        scale, o.data_ptr())
    with _lib.on_device(dev):
        rc = _lib.timed_launch("window_decode_attn", dev, lambda: lib.dfl_window_decode(
            ctypes.byref(p), ctypes.c_void_p(_lib.ptr(ws)), nbytes, ctypes.c_void_p(_lib.stream_handle(dev))))
    _lib.check(rc, "dfl_window_decode")
    torch.autograd.graph.increment_version((k_cache, v_cache))
    return o


class _CacheFillFn(torch.autograd.Function):
    """A fill as a node of a trace, without a gradient."""

    @staticmethod
    def forward(ctx, *args):
        _fill(*args)


class _DecodeFn(torch.autograd.Function):
    """A token's step as a node of a trace, without a gradient."""

    @staticmethod
    def forward(ctx, *args):
        return _decode(*args)


class _FillCodesFn(torch.autograd.Function):
    """A fill of caches in few bits as a node of a trace, without a gradient."""

    @staticmethod
    def forward(ctx, *args):
        _fill_codes(*args)


class _DecodeCodesFn(torch.autograd.Function):
    """A token's step over caches in few bits as a node of a trace, without a gradient."""

    @staticmethod
    def forward(ctx, *args):
        return _decode_codes(*args)


class _CacheReadFn(torch.autograd.Function):
    """A reading of a cache as a node of a trace, without a gradient."""

    @staticmethod
    def forward(ctx, *args):
        return _read(*args)


def window_cache_fill(
    K: torch.Tensor,
    V: torch.Tensor,
    lengths: torch.Tensor,
    k_cache: torch.Tensor | QuantizedCache,
    v_cache: torch.Tensor | QuantizedCache,
    *,
    n_sink: int = 0,
    starts: torch.Tensor | None = None,
) -> None:
    """Copies a prompt's keys and values into the rolling caches, in place.

    K, V (B,Hk,N,D), any strides, in memory of their own; lengths (B,) int32 or int64: rows 0 .. lengths[b] - 1 are the
    prompt (above N counts as N, below 1 leaves the sample's caches alone).  k_cache, v_cache
    (B,Hk,n_sink + window,D): position p < n_sink goes to slot p, any other to slot n_sink + (p - n_sink) % window, the
    last of those that share one; slots that no position of the prompt belongs to keep what they hold.  The two caches
    may interleave in one buffer, but have no element in common.

    ``starts`` (B,) int32 or int64: the rows are a later chunk, row i at position starts[b] + i (below 0 leaves the
    sample's caches alone; above 2^31 - 1 counts as that).  Both caches may be in 8 or 4 bits
    (``quantized_cache``); K and V are then bf16 or fp32 and rounded to codes as they are written."""
    what = "window_cache_fill"
    if K.dim() != 4 or K.shape != V.shape:
        raise ValueError(f"{what}: K and V must be (B,Hk,N,D) alike")
    B, Hk, N, d = K.shape
    n_sink = int(n_sink)
    if _same_kind(what, k_cache, v_cache):
        (kc, ke, bits), (vc, ve, _) = k_cache, v_cache
        _no_grad_inputs(what, K, V)
        _lib.require_gpu(K, V, lengths, starts, kc, ke, vc, ve)
        if V.dtype != K.dtype or K.dtype not in (torch.bfloat16, torch.float32):
            raise TypeError(f"{what}: K and V must both be bf16 or both fp32, got {K.dtype} and {V.dtype}")
        if not 1 <= d <= MAX_HEAD_DIM or not 1 <= N <= MAX_SLOTS:
            raise ValueError(f"{what}: K {tuple(K.shape)} is empty, or its head dim above {MAX_HEAD_DIM} or rows above "
                             f"{MAX_SLOTS}")
        _check_codes(what, k_cache, v_cache, B, Hk, d, n_sink)
    else:
        _no_grad_inputs(what, K, V, k_cache, v_cache)
        _lib.require_gpu(K, V, lengths, starts, k_cache, v_cache)
        if V.dtype != K.dtype:
            raise TypeError(f"{what}: K is {K.dtype}, V is {V.dtype}")
        _check_caches(what, k_cache, v_cache, B, Hk, d, K.dtype, n_sink)
    _check_lengths(what, lengths, B)
    if starts is not None:
        _check_lengths(what, starts, B, "starts")
    if isinstance(k_cache, QuantizedCache):
        run = _FillCodesFn.apply if _lib.recording() else _fill_codes
        run(K, V, lengths, starts, kc, ke, vc, ve, bits, n_sink)
    else:
        run = _CacheFillFn.apply if _lib.recording() else _fill
        run(K, V, lengths, k_cache, v_cache, n_sink, starts)


def window_cache_read(
    k_cache: torch.Tensor | QuantizedCache,
    v_cache: torch.Tensor | QuantizedCache,
    lengths: torch.Tensor,
    D: int,
    *,
    n_sink: int = 0,
    dtype: torch.dtype | None = None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """What the rolling caches hold, in the order of the positions: K, V (B,Hk,n_sink + window,D) and a mask
    (B,n_sink + window) fp32, as the first keys of ``flash_window_attn`` for the rows that follow (module docstring).

    lengths (B,) int32 or int64: the number of positions that each sample's caches have taken.  Row j < n_sink is position
    j, any other row position lengths[b] - (n_sink + window) + j: the last ``window`` positions end with the last row.  Rows
    that have no such position (short sequences, lengths below 1) are zero and masked: 0.  The caches may be tensors
    (``dtype`` is theirs) or in few bits (``dtype`` bf16 or fp32, by default bf16, in which every code is
    exact).  The rows that follow may be more than ``window`` only where lengths[b] >= n_sink (module docstring).  Distances
    between the first tokens and the others are those of the rows, not of the positions: a table of relative biases that
    goes on beyond the window sees them nearer.  No gradient."""
    what = "window_cache_read"
    n_sink = int(n_sink)
    if _same_kind(what, k_cache, v_cache):
        (kc, ke, bits), (vc, ve, _) = k_cache, v_cache
        dtype = torch.bfloat16 if dtype is None else dtype
    else:
        kc, ke, vc, ve, bits = k_cache, None, v_cache, None, 0
        dtype = kc.dtype if dtype is None else dtype
        _no_grad_inputs(what, kc, vc)
    _lib.require_gpu(kc, ke, vc, ve, lengths)
    if kc.dim() != 4:
        raise ValueError(f"{what}: caches must be (B,Hk,n_sink + window,*)")
    B, Hk = kc.shape[:2]
    if not 1 <= D <= MAX_HEAD_DIM or B < 1 or Hk < 1:
        raise ValueError(f"{what}: D={D} outside [1, {MAX_HEAD_DIM}], or no samples or heads")
    if bits:
        if dtype not in (torch.bfloat16, torch.float32):
            raise TypeError(f"{what}: dtype {dtype} is neither bf16 nor fp32")
        _check_codes(what, k_cache, v_cache, B, Hk, D, n_sink)
    else:
        _check_caches(what, kc, vc, B, Hk, D, dtype, n_sink)
    _check_lengths(what, lengths, B)
    run = _CacheReadFn.apply if _lib.recording() else _read
    return run(lengths, kc, ke, vc, ve, bits, int(D), n_sink, dtype)


def window_decode_attn(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    k_cache: torch.Tensor | QuantizedCache,
    v_cache: torch.Tensor | QuantizedCache,
    lengths: torch.Tensor,
    *,
    n_sink: int = 0,
    scale: float | None = None,
    rel_table: torch.Tensor | None = None,
    rel_edges=None,
) -> torch.Tensor:
    """One token of each sample against its rolling cache (module docstring): ``flash_window_attn``'s causal
    attention for the query at position lengths[b].

    q (B,H,D); k, v (B,Hk,D) the token's own key and value, which enter k_cache, v_cache (B,Hk,n_sink + window,D) in
    place at position lengths[b], the number of tokens that the sample's cache has taken so far; lengths (B,) int32 or
    int64, below 2^31 (above counts as 2^31 - 1), on the device, not changed by the call; a sample with
    lengths[b] < 0 has no token: its output is zero and its caches stay as they are.  All of q, k, v and the caches in bf16
    or all in fp32.  The table has one direction (len(rel_edges) + 1 buckets).  No gradient.  Returns o (B,H,D).

    Both caches may be in 8 or 4 bits (``quantized_cache``): the token's own key and value are rounded to codes and
    enter, and count, as their codes stand; q, k and v are bf16 or fp32 and only the result is rounded to their type.
    Where a slot in use holds a group with an infinity or NaN, all heads that read it are NaN."""
    what = "window_decode_attn"
    if q.dim() != 3 or k.dim() != 3 or k.shape != v.shape:
        raise ValueError(f"{what}: q must be (B,H,D), k and v (B,Hk,D)")
    few = _same_kind(what, k_cache, v_cache)
    if few:
        (kc, ke, bits), (vc, ve, _) = k_cache, v_cache
        _no_grad_inputs(what, q, k, v, rel_table)
        _lib.require_gpu(q, k, v, kc, ke, vc, ve, lengths, rel_table)
    else:
        _no_grad_inputs(what, q, k, v, k_cache, v_cache, rel_table)
        _lib.require_gpu(q, k, v, k_cache, v_cache, lengths, rel_table)
    B, H, d = q.shape
    Hk = k.shape[1]
    if k.shape[0] != B or k.shape[2] != d or Hk < 1 or H % Hk:
        raise ValueError(f"{what}: k {tuple(k.shape)} does not fit q {tuple(q.shape)}")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"{what}: q is {q.dtype}, k {k.dtype}, v {v.dtype}")
    n_sink = int(n_sink)
    if few:
        if q.dtype not in (torch.bfloat16, torch.float32):
            raise TypeError(f"{what}: q, k and v must be bf16 or fp32, got {q.dtype}")
        if not 1 <= d <= MAX_HEAD_DIM or B < 1 or H < 1:
            raise ValueError(f"{what}: q {tuple(q.shape)} is empty, or its head dim above {MAX_HEAD_DIM}")
        _check_codes(what, k_cache, v_cache, B, Hk, d, n_sink)
    else:
        _check_caches(what, k_cache, v_cache, B, Hk, d, q.dtype, n_sink)
    _check_lengths(what, lengths, B)
    if (rel_table is None) != (rel_edges is None):
        raise ValueError(f"{what}: give rel_table and rel_edges together")
    arr = None if rel_table is None else edge_array(rel_table, rel_edges, H, False)
    if few:
        run = _DecodeCodesFn.apply if _lib.recording() else _decode_codes
        return run(q, k, v, kc, ke, vc, ve, lengths, rel_table, arr, bits, n_sink, _scale(what, scale, d))
    run = _DecodeFn.apply if _lib.recording() else _decode
    return run(q, k, v, k_cache, v_cache, lengths, rel_table, arr, n_sink, _scale(what, scale, d))
