"""Float64 forms of the sequence operators: the relative position bias by buckets, attention
over a sliding window and a few first tokens (with its gradients written out), and the
rolling cache with its single-token attention.

``attention`` also returns, for every result, how far a kernel may be off that keeps sums in
fp32 and rounds probabilities and score gradients once to the operand type: worst-case sums of
half steps, elementwise.  With u the operands' half step (2^-8 for bf16; fp32 operands are not
rounded, u = 0), w the results' half step and e the bound of the fp32 arithmetic itself:

* scores: a dot product of d terms, the scale and the bias, each term off by at most 2^-24 of its
  size, so a probability is off by e = 2 (d + 8) 2^-24 max(scale |q|.|k| + |bias|) + (n + 32) 2^-24
  of itself (numerator and sum; n keys summed, 32 for exp2, the reference and the division);
* o: (u + e) sum p |v| + w |o|; dv: (u + e) sum p |do| + w |dv|;
* D = do.o: from the stored o, sum |do| err(o), or as the sum of p dp (kernels do so where a row tile
  sees few keys): e' sum p |do|.|v| with e' = 2 e + (n + d) 2^-24; the larger of the two is used;
  With ``remainder`` the tighter bound of a D that does not know the stored o's rounding: what the forward kept
  is sum p~ v / sum p~ of the rounded probabilities p~ = p (1 + eps_j), |eps_j| <= u, in two roundings of the
  operand type (the first o's own; the second, of what is left of it, at most 2 u |o| before and so 2 u u |o| off).  As
  sum p~ dp / sum p~ - D = sum p eps (dp - D) / (1 + sum p eps), that D is off by u / (1 - u) sum p |dp - D| +
  2 u u sum |do| |o| + e' sum p |do|.|v|;
* ds = p (dp - D): e' p (|do|.|v| + sum p |do|.|v|) + p err(D);
* dq, dk: sums of (u |ds| + err(ds)) against |k|, |q|, plus (n + 8) 2^-24 of sum |ds| |k|, plus w of the result;
* dtable: sums of err(ds) and (n + 8) 2^-24 |ds| by bucket, plus its own rounding.
"""

from __future__ import annotations

import math

import torch

U32 = 2.0 ** -24


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def bucket(edges, bidirectional, rel):
    """Bucket of every relative position (key - query)."""
    mag = rel.abs() if bidirectional else (-rel).clamp(min=0)
    b = sum(((mag >= e).long() for e in edges), torch.zeros_like(rel))
    return b + (rel > 0).long() * (len(edges) + 1) if bidirectional else b


def rel_bias(table, edges, rel, bidirectional):
    """rel (..., M, N) -> (..., H, M, N) in float64."""
    return torch.movedim(table.double()[:, bucket(edges, bidirectional, rel)], 0, -3)


def rel_bias_grad(grad, edges, rel, bidirectional, n_buckets):
    """grad (B, H, M, N), rel (B or 1, M, N) -> (dtable (H, buckets), sum of |grad| by bucket)."""
    b = bucket(edges, bidirectional, rel).unsqueeze(1)
    g = grad.double()
    cols = [torch.where(b == n, g, 0.0) for n in range(n_buckets)]
    return (torch.stack([c.sum((0, 2, 3)) for c in cols], 1),
            torch.stack([c.abs().sum((0, 2, 3)) for c in cols], 1))


def visible(M, N, window, n_sink, causal, mask, B, device=None):
    """(B, M, N): whether query i (at position i + N - M) sees key j."""
    t = torch.arange(M, device=device)[:, None] + N - M
    j = torch.arange(N, device=device)[None, :]
    if causal:
        see = (j <= t) & ((t - j < window) | (j < n_sink))
    else:
        see = ((t - j).abs() < window) | (j < n_sink)
    see = see.expand(B, M, N)
    if mask is not None:
        ok = mask != 0
        see = see & ok[:, None, :] & ok[:, N - M:, None]
    return see


def _by_group(x, Hk):
    """(B, H, ...) summed over the query heads of each key head."""
    return x.reshape(x.shape[0], Hk, x.shape[1] // Hk, *x.shape[2:]).sum(2)


def attention(q, k, v, *, window, n_sink=0, causal=True, mask=None, scale=None, table=None, edges=None, grad=None,
              operand=torch.float32, result=torch.float32, table_dtype=torch.float32, remainder=False):
    """Values and bounds: {"o", "dq", "dk", "dv", "dtable"} -> (float64 value, elementwise bound)."""
    q, k, v = q.double(), k.double(), v.double()
    B, H, M, d = q.shape
    Hk, N = k.shape[1], k.shape[2]
    G = H // Hk
    scale = d ** -0.5 if scale is None else scale
    see = visible(M, N, window, n_sink, causal, mask, B, q.device)
    if mask is not None:  # masked rows reach nothing, whatever they hold
        ok = (mask != 0)[:, None, :, None]
        k, v = torch.where(ok, k, 0.0), torch.where(ok, v, 0.0)
        q = torch.where(ok[:, :, N - M:], q, 0.0)
    kk, vv = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    s = (q @ kk.transpose(-1, -2)) * scale
    size = (q.abs() @ kk.abs().transpose(-1, -2)) * abs(scale)
    rel = torch.arange(N)[None, :] - torch.arange(M)[:, None] - (N - M)
    if table is not None:
        b = rel_bias(table, edges, rel, not causal)
        s = s + b
        size = size + torch.where(b > -1e30, b.abs(), 0.0)
        see = see[:, None] & (b > -1e30)
    else:
        see = see[:, None].expand(B, H, M, N)
    s = torch.where(see, s, -math.inf)
    top = s.amax(-1, keepdim=True)
    ex = torch.where(see, torch.exp(s - torch.where(top > -math.inf, top, 0.0)), 0.0)
    total = ex.sum(-1, keepdim=True)
    p = ex / torch.where(total > 0, total, 1.0)
    o = p @ vv

    u = half_step(operand) if operand == torch.bfloat16 else 0.0
    w = half_step(result)
    n = float(see.sum(-1).max())
    e = 2 * (d + 8) * U32 * float(torch.where(see, size, 0.0).max()) + (n + 32) * U32
    e2 = 2 * e + (n + d) * U32
    out = {"o": (o, (u + e) * (p @ vv.abs()) + w * o.abs())}
    if grad is None:
        return out
    g = grad.double()
    if mask is not None:
        g = torch.where(ok[:, :, N - M:], g, 0.0)
    dp, dpa = g @ vv.transpose(-1, -2), g.abs() @ vv.abs().transpose(-1, -2)
    D, Da = (p * dp).sum(-1, keepdim=True), (p * dpa).sum(-1, keepdim=True)
    ds = p * (dp - D)
    dD = torch.maximum((g.abs() * out["o"][1]).sum(-1, keepdim=True), e2 * Da)
    if remainder:
        dD = u / (1 - u) * ds.abs().sum(-1, keepdim=True) + 2 * u * u * (g.abs() * o.abs()).sum(-1, keepdim=True) + e2 * Da
    eds = e2 * p * (dpa + Da) + p * dD
    a = ds.abs()
    soft = u * a + eds + (n + 8) * U32 * a
    dq = ds @ kk * scale
    dk = _by_group(ds.transpose(-1, -2) @ q * scale, Hk)
    dv = _by_group(p.transpose(-1, -2) @ g, Hk)
    rows = float(see.sum(-2).max()) * G
    out["dq"] = (dq, soft @ kk.abs() * abs(scale) + w * dq.abs())
    out["dk"] = (dk, _by_group((soft + rows * U32 * a).transpose(-1, -2) @ q.abs() * abs(scale), Hk) + w * dk.abs())
    out["dv"] = (dv, _by_group(((u + e + rows * U32) * p).transpose(-1, -2) @ g.abs(), Hk) + w * dv.abs())
    if table is not None:
        dt, _ = rel_bias_grad(ds, edges, rel[None], not causal, table.shape[1])
        err, _ = rel_bias_grad(eds, edges, rel[None], not causal, table.shape[1])
        mag, _ = rel_bias_grad(a, edges, rel[None], not causal, table.shape[1])
        out["dtable"] = (dt, err + (n + rows + 64) * U32 * mag + half_step(table_dtype) * dt.abs())
    return out


def slot(p, n_sink, window):
    return p if p < n_sink else n_sink + (p - n_sink) % window


def fill(k, v, lengths, k_cache, v_cache, n_sink):
    """The caches after the prompt, as new tensors."""
    kc, vc = k_cache.clone(), v_cache.clone()
    window = kc.shape[2] - n_sink
    for b in range(k.shape[0]):
        for p in range(min(int(lengths[b]), k.shape[2])):  # in order: the last of those that share a slot stays
            kc[b, :, slot(p, n_sink, window)] = k[b, :, p]
            vc[b, :, slot(p, n_sink, window)] = v[b, :, p]
    return kc, vc


def decode(q, k, v, k_cache, v_cache, lengths, n_sink, *, scale=None, table=None, edges=None, operand=torch.float32,
           result=torch.float32):
    """(o, bound), and the caches with the token in."""
    kc, vc = k_cache.clone(), v_cache.clone()
    B, H, d = q.shape
    Hk, window = kc.shape[1], kc.shape[2] - n_sink
    o, bound = torch.zeros(B, H, d, dtype=torch.float64), torch.zeros(B, H, d, dtype=torch.float64)
    for b in range(B):
        t = int(lengths[b])
        if t < 0:
            continue
        kc[b, :, slot(t, n_sink, window)] = k[b]
        vc[b, :, slot(t, n_sink, window)] = v[b]
        held = {}
        for p in range(max(0, t + 1 - 4 * (n_sink + window)), t + 1):
            held[slot(p, n_sink, window)] = p
        for p in range(min(n_sink, t + 1)):
            held[p] = p
        at = sorted(held)
        pos = torch.tensor([held[x] for x in at])
        kk, vv = kc[b][:, at].double(), vc[b][:, at].double()
        for h in range(H):
            g = h // (H // Hk)
            s = kk[g] @ q[b, h].double() * (d ** -0.5 if scale is None else scale)
            size = kk[g].abs() @ q[b, h].double().abs() * abs(d ** -0.5 if scale is None else scale)
            if table is not None:
                bias = table[h].double()[bucket(edges, False, pos - t)]
                s, size = s + bias, size + torch.where(bias > -1e30, bias.abs(), 0.0)
                s = torch.where(bias > -1e30, s, -math.inf)
            top = s.max()
            ex = torch.exp(s - top) if top > -math.inf else torch.zeros_like(s)
            p = ex / ex.sum().clamp(min=1e-300)
            o[b, h] = p @ vv[g]
            u = half_step(operand) if operand == torch.bfloat16 else 0.0
            e = 2 * (d + 8) * U32 * float(size.max()) + (len(at) + 32) * U32
            bound[b, h] = (u + e) * (p @ vv[g].abs()) + half_step(result) * o[b, h].abs()
    return o, bound, kc, vc
