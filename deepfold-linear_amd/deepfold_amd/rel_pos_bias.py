"""Learned bias by buckets of the relative position, on MI355X.

``rel_pos_bias`` forms bias[h, i, j] = table[h, bucket(k_pos[j] - q_pos[i])] from the
positions, without an (N, N) array of buckets, and gives the table its gradient; the bias
goes into ``flash_diffusion_attn(pair_bias=...)`` (its kernels add a dense bias) or any
other attention.  ``flash_window_attn`` and ``window_decode_attn`` take the same table
and edges and form the bias inside their kernels.

Buckets: ``edges`` is an ascending tuple of whole numbers in [1, 2048].  With
rel = key position - query position and mag = |rel| (``bidirectional``) or max(-rel, 0),
the bucket is the number of edges <= mag; ``bidirectional`` gives keys behind the query a
second set of len(edges) + 1 buckets (the first of these is in use only where edges[0] > 1).
So the table is (H, 2 (len(edges) + 1)) or (H, len(edges) + 1), at most 96 buckets.
``tuple(range(1, 33))`` clips at a distance of 32; ``relative_bucket_edges`` makes buckets
that widen with the distance.

The reference has no such operator: its 68-bin bias (flash_diffusion_attn.py:440-473) reads
bins that the caller made.
"""

from __future__ import annotations

import ctypes
import functools

import torch
from torch.autograd.function import once_differentiable

from . import _lib

MAX_BUCKETS = 96
MAX_EDGE = 2048


def relative_bucket_edges(n_buckets: int, max_distance: int, bidirectional: bool = True) -> tuple[int, ...]:
    """Edges of ``n_buckets`` buckets (half of them for each direction with ``bidirectional``): the first
    half of a direction's buckets hold one distance each, e of them, the rest grow in equal ratios and the last
    one begins before ``max_distance``: bucket e + k holds the distances d with (d / e)^L >= (max_distance / e)^k,
    L buckets in all.  Whole-number arithmetic throughout: no rounding decides a border."""
    side = n_buckets // 2 if bidirectional else n_buckets
    if side < 2 or n_buckets > MAX_BUCKETS:
        raise ValueError(f"relative_bucket_edges: n_buckets={n_buckets} leaves {side} buckets a direction "
                         f"(at least 2) or is above {MAX_BUCKETS}")
    exact = max(1, side // 2)
    L = side - exact
    if not exact < max_distance <= MAX_EDGE:
        raise ValueError(f"relative_bucket_edges: max_distance={max_distance} outside ({exact}, {MAX_EDGE}]")
    edges = list(range(1, exact + 1))
    for k in range(1, L):
        d = max(edges[-1] + 1, int(exact * (max_distance / exact) ** (k / L)) - 2)
        while d ** L * exact ** k < max_distance ** k * exact ** L:  # d^L e^k >= m^k e^L
            d += 1
        edges.append(d)
    if edges[-1] > MAX_EDGE:
        raise ValueError(f"relative_bucket_edges: {n_buckets} buckets do not fit below distance {MAX_EDGE}")
    return tuple(edges)


@functools.lru_cache(maxsize=256)
def _edge_array(edges: tuple, bidirectional: bool):
    """The C array of checked edges (by value; read by the library during the call)."""
    n = (len(edges) + 1) * (2 if bidirectional else 1)
    if not edges or n > MAX_BUCKETS:
        raise ValueError(f"edges: {len(edges)} edges give {n} buckets; need at least one edge and at most "
                         f"{MAX_BUCKETS} buckets")
    if any(int(e) != e for e in edges):
        raise ValueError("edges: whole numbers are needed")
    if edges[0] < 1 or edges[-1] > MAX_EDGE or any(b <= a for a, b in zip(edges, edges[1:])):
        raise ValueError(f"edges must ascend within [1, {MAX_EDGE}]")
    return (ctypes.c_int * len(edges))(*(int(e) for e in edges)), n


def edge_array(table: torch.Tensor, edges, H: int, bidirectional: bool):
    arr, n = _edge_array(tuple(edges), bool(bidirectional))
    if table.dim() != 2 or table.shape[0] != H or table.shape[1] != n:
        raise ValueError(f"table: expected ({H}, {n}) for {len(arr)} edges, got {tuple(table.shape)}")
    if not table.is_floating_point():
        raise TypeError(f"table: unsupported dtype {table.dtype}")
    return arr


def _positions(t, name, dims):
    if t.is_floating_point() or t.is_complex() or t.dtype == torch.bool:
        raise TypeError(f"rel_pos_bias: {name} must hold integers, got {t.dtype}")
    if t.dim() != 2 or t.shape[1] != dims:
        raise ValueError(f"rel_pos_bias: {name} must be (B, {dims}) or ({dims},)")
    return _lib.to_int32(t.detach()).contiguous()


class _RelPosBias(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, arr, both, qp, kp, B, M, N, dt):
        dev = _lib.require_gpu(table, qp, kp)
        H = table.shape[0]
        tab = table.detach().to(torch.float32).contiguous()
        out = torch.empty(B, H, M, N, dtype=dt, device=dev)
        p = _lib.RelBiasParams(_lib.DFL_BF16 if dt == torch.bfloat16 else _lib.DFL_F32, tab.data_ptr(),
                               ctypes.addressof(arr), len(arr), int(both), _lib.ptr(qp), _lib.ptr(kp), B, H, M, N,
                               out.data_ptr())
        lib = _lib.load()
        with _lib.on_device(dev):
            rc = _lib.timed_launch("rel_bias_fwd", dev, lambda: lib.dfl_rel_bias_fwd(
                ctypes.byref(p), ctypes.c_void_p(_lib.stream_handle(dev))))
        _lib.check(rc, "dfl_rel_bias_fwd")
        ctx.save_for_backward(qp, kp)
        ctx.meta = (arr, both, table.shape, table.dtype)
        ctx.set_materialize_grads(False)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        none = (None,) * 8
        if grad is None:
            return (None, *none)
        qp, kp = ctx.saved_tensors
        arr, both, shape, tdt = ctx.meta
        dev = grad.device
        g = grad.contiguous()
        B, H, M, N = g.shape
        dtab = torch.empty(shape, dtype=torch.float32, device=dev)
        lib = _lib.load()
        ws = torch.empty(lib.dfl_rel_bias_workspace_size(B, H, M, N, len(arr), int(both)), dtype=torch.uint8, device=dev)
        p = _lib.RelBiasParams(_lib.DFL_BF16 if g.dtype == torch.bfloat16 else _lib.DFL_F32, None,
                               ctypes.addressof(arr), len(arr), int(both), _lib.ptr(qp), _lib.ptr(kp), B, H, M, N,
                               None, g.data_ptr(), dtab.data_ptr())
        with _lib.on_device(dev):
            rc = _lib.timed_launch("rel_bias_bwd", dev, lambda: lib.dfl_rel_bias_bwd(
                ctypes.byref(p), ctypes.c_void_p(ws.data_ptr()), ws.numel(),
                ctypes.c_void_p(_lib.stream_handle(dev))))
        _lib.check(rc, "dfl_rel_bias_bwd")
        return (dtab if tdt == torch.float32 else dtab.to(tdt), *none)


def rel_pos_bias(
    table: torch.Tensor,
    edges,
    n_query: int,
    n_key: int | None = None,
    *,
    q_pos: torch.Tensor | None = None,
    k_pos: torch.Tensor | None = None,
    bidirectional: bool = True,
    dtype: torch.dtype | None = None,
) -> torch.Tensor:
    """Bias by buckets of the relative position (module docstring), with gradient to ``table``.

    table (H, buckets); query i stands at position i + n_key - n_query and key j at j, or, with
    ``q_pos`` (B, n_query) / (n_query,) and ``k_pos`` (B, n_key) / (n_key,) integers, where those say (one of them
    alone stands for both if n_query == n_key).  Positions are held in 32 bits: one beyond them stands at their end, so
    shift a sample's positions into [-2^31, 2^31) first (only differences count).  Returns (H, n_query, n_key), or
    (B, H, n_query, n_key) with batched positions, contiguous, in ``dtype`` (bf16 or fp32;
    default: the table's if it is one of them)."""
    M = int(n_query)
    N = M if n_key is None else int(n_key)
    if M < 1 or N < 1:
        raise ValueError(f"rel_pos_bias: n_query={M}, n_key={N} must be positive")
    if table.dim() != 2:
        raise ValueError("rel_pos_bias: table must be (H, buckets)")
    arr = edge_array(table, edges, table.shape[0], bidirectional)
    dt = dtype if dtype is not None else (torch.bfloat16 if table.dtype == torch.bfloat16 else torch.float32)
    if dt not in (torch.bfloat16, torch.float32):
        raise TypeError(f"rel_pos_bias: unsupported dtype {dt} (bf16 or fp32)")
    B, batched = 1, False
    if q_pos is not None or k_pos is not None:
        if (q_pos is None or k_pos is None) and M != N:
            raise ValueError("rel_pos_bias: give q_pos and k_pos where n_query != n_key")
        q_pos = k_pos if q_pos is None else q_pos
        k_pos = q_pos if k_pos is None else k_pos
        batched = q_pos.dim() == 2 or k_pos.dim() == 2
        q_pos = _positions(q_pos if q_pos.dim() == 2 else q_pos.unsqueeze(0), "q_pos", M)
        k_pos = _positions(k_pos if k_pos.dim() == 2 else k_pos.unsqueeze(0), "k_pos", N)
        B = max(q_pos.shape[0], k_pos.shape[0])
        if min(q_pos.shape[0], k_pos.shape[0]) not in (1, B):
            raise ValueError("rel_pos_bias: q_pos and k_pos have different batch sizes")
        q_pos, k_pos = q_pos.expand(B, M).contiguous(), k_pos.expand(B, N).contiguous()
    out = _RelPosBias.apply(table, arr, bool(bidirectional), q_pos, k_pos, B, M, N, dt)
    return out if batched else out.squeeze(0)
