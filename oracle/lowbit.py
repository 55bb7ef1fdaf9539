"""Float64 forms of the operators of a layer served in few bits: rolling caches in 8 or 4 bits (codes, values, copies and
readings of them, one token's attention over them) and products in 8-bit integers.

Codes, exponents, values, integer sums and scales are exact: powers of two are searched among all of them by their defining
inequality, codes among all codes by distance.  ``decode`` and ``linear`` also return how far a kernel may be off that keeps
sums in fp32:

* a score is a sum of d products that are exact in fp32 (fp32 queries: of three parts, 3 d products), the scale and the bias,
  each step off by at most 2^-24 of its size; a weight is off by e = 2 (3 d + 8) 2^-24 max(scale |q|.|k| + |bias|) +
  (n + 32) 2^-24 of itself (numerator and sum; n keys summed, 32 for exp2, the reference and the division);
* a weight enters its products as two bf16 numbers (bf16 results: the second, of a remainder of at most 2^-8 of it, is off by
  2^-8 of that) or three (fp32): u = 2^-16 or 2^-24;
* a weight, formed against a reference that no score passes by more than 2^8, may vanish where it or its last part lies below
  the smallest normal number 2^-126; the largest weight is at least 1 then, so each is off by f = 2^-125 of their sum, which
  counts beside the relative errors only where the rest of a sum is as small (a dominant key whose element is 0);
* o: (u + e) sum w |v| + f sum |v| + (half a step of the result's type) |o|;
* y = sum s_w s_x + b: the sum's conversion, two products and the sum with b, 2^-24 each of |sum s_w s_x| + |y|, and half
  a step of the result.
"""

from __future__ import annotations

import torch

from .window import U32, bucket, half_step, slot

GROUP = 32
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def groups_of(d):
    return -(-d // GROUP)


def grouped(x):
    """(..., d) -> (..., groups, 32) in float64, filled up with zeros."""
    d = x.shape[-1]
    out = torch.zeros(*x.shape[:-1], groups_of(d) * GROUP, dtype=torch.float64)
    out[..., :d] = x.double()
    return out.unflatten(-1, (-1, GROUP))


def exponent(amax, bits):
    """The byte of each group by its largest magnitude; 255 where that is no finite number."""
    top = 248 if bits == 8 else 252
    step = 2.0 ** (torch.arange(1, top + 1, dtype=torch.float64) - 127)
    fits = amax[..., None] < 127.5 * step if bits == 8 else amax[..., None] <= 7 * step
    e = torch.where(fits.any(-1), fits.to(torch.uint8).argmax(-1) + 1, top)  # the first that fits
    return torch.where(torch.isfinite(amax), e, 255)


def encode(x, bits):
    """Codes as they lie in memory (..., bytes) and exponent bytes (..., groups), uint8."""
    g = grouped(x)
    e = exponent(torch.where(g.isnan(), float("inf"), g.abs()).amax(-1), bits)
    y = torch.where((e == 255)[..., None], 0.0, g) / torch.where(e == 255, 1.0, 2.0 ** (e.double() - 127))[..., None]
    if bits == 8:
        n = torch.floor(y)
        up = (y - n > 0.5) | ((y - n == 0.5) & (n.remainder(2) == 1))
        code = (n + up.double()).clamp(-127, 127).to(torch.int8).view(torch.uint8).flatten(-2)
    else:
        grid = torch.tensor(E2M1, dtype=torch.float64)
        far = (y.abs()[..., None] - grid).abs()
        # of two equally near codes the even one: its distance counts a little less
        far = far - 1e-9 * (torch.arange(8) % 2 == 0).double() * (far == far.amin(-1, keepdim=True)).double()
        code = far.argmin(-1) + 8 * torch.signbit(y).long()
        code = torch.where((e == 255)[..., None], 0, code).flatten(-2)
        code = (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8)
    return code, e.to(torch.uint8)


def values(code, e, d, bits):
    """float64 rows (..., d) of codes (..., bytes) and exponent bytes (..., groups)."""
    if bits == 8:
        v = code.view(torch.int8).double()
    else:
        nib = torch.stack((code & 15, code >> 4), -1).flatten(-2).long()
        v = torch.tensor(E2M1, dtype=torch.float64)[nib & 7] * (1 - 2 * (nib >> 3)).double()
    scale = torch.where(e == 255, float("nan"), 2.0 ** (e.double() - 127))
    return (v.unflatten(-1, (-1, GROUP)) * scale[..., None]).flatten(-2)[..., :d]


def cache_values(cache, d):
    """float64 (B,Hk,S,d) of a cache (codes, exponents (B,Hk,groups,n), bits)."""
    codes, exps, bits = cache
    return values(codes, exps[..., :codes.shape[2]].transpose(-1, -2), d, bits)


def fill(k, v, lengths, starts, k_cache, v_cache, n_sink):
    """The caches (codes, exponents, bits) after a chunk, as new tensors."""
    out = [(c.clone(), e.clone(), bits) for c, e, bits in (k_cache, v_cache)]
    new = [encode(x, c[2]) for x, c in zip((k, v), out)]
    window = out[0][0].shape[2] - n_sink
    for b in range(k.shape[0]):
        start = 0 if starts is None else int(starts[b])
        if start < 0:
            continue
        for i in range(min(int(lengths[b]), k.shape[2])):  # in order: the last of those that share a slot stays
            s = slot(start + i, n_sink, window)
            for (codes, exps, _), (code, e) in zip(out, new):
                codes[b, :, s], exps[b, :, :, s] = code[b, :, i], e[b, :, i]
    return out


def read(k_rows, v_rows, lengths, n_sink):
    """(K, V, mask) of caches whose rows (B,Hk,S,d) are given, in the order of the positions."""
    B, _, S, _ = k_rows.shape
    window = S - n_sink
    K, V, mask = torch.zeros_like(k_rows), torch.zeros_like(v_rows), torch.zeros(B, S, dtype=torch.float64)
    for b in range(B):
        n = int(lengths[b])
        for j in range(S):
            p = j if j < n_sink else n - S + j
            if p < n and p >= (0 if j < n_sink else n_sink):
                s = slot(p, n_sink, window)
                K[b, :, j], V[b, :, j], mask[b, j] = k_rows[b, :, s], v_rows[b, :, s], 1
    return K, V, mask


def held_slots(t, S, n_sink):
    """The slots in use once position t is in, and their positions."""
    window = S - n_sink
    at = {p: p for p in range(min(n_sink, t + 1))}
    for p in range(max(n_sink, t + 1 - window), t + 1):
        at[slot(p, n_sink, window)] = p
    slots = sorted(at)
    return slots, torch.tensor([at[s] for s in slots])


def decode(q, k, v, k_cache, v_cache, lengths, n_sink, *, scale=None, table=None, edges=None, result=torch.float32):
    """(o, bound), and the caches with the token in."""
    B, H, d = q.shape
    Hk, S = k.shape[1], k_cache[0].shape[2]
    kc, vc = fill(k[:, :, None], v[:, :, None], (lengths >= 0).long(), lengths, k_cache, v_cache, n_sink)
    kr, vr = cache_values(kc, d), cache_values(vc, d)
    scale = d ** -0.5 if scale is None else scale
    o, bound = torch.zeros(B, H, d, dtype=torch.float64), torch.zeros(B, H, d, dtype=torch.float64)
    u = 2.0 ** -16 if result == torch.bfloat16 else 2.0 ** -24
    for b in range(B):
        t = int(lengths[b])
        if t < 0:
            continue
        slots, pos = held_slots(t, S, n_sink)
        for h in range(H):
            kk, vv = kr[b, h // (H // Hk), slots], vr[b, h // (H // Hk), slots]
            s, size = kk @ q[b, h].double() * scale, kk.abs() @ q[b, h].double().abs() * scale
            if table is not None:
                bias = table[h].double()[bucket(edges, False, pos - t)]
                size = size + torch.where(bias > -1e30, bias.abs(), 0.0)
                s = torch.where(bias > -1e30, s + bias, -float("inf"))
            ex = torch.exp(s - s.max()) if s.max() > -float("inf") else torch.zeros_like(s)
            w = ex / ex.sum().clamp(min=1e-300)
            if bool(kk.isnan().any() | vv.isnan().any()):
                w = w * float("nan")
            o[b, h] = w @ vv
            e = 2 * (3 * d + 8) * U32 * float(size.max()) + (len(slots) + 32) * U32
            bound[b, h] = (u + e) * (w @ vv.abs()) + 2.0 ** -125 * vv.abs().sum(0) + half_step(result) * o[b, h].abs()
    return o, bound, kc, vc


def rows(x):
    """Codes (M,K) int8 and scale (M,) fp32 of rows."""
    xd = x.double()
    top = xd.abs().amax(-1)
    fine = torch.isfinite(top)
    scale = (torch.where(fine, top, 1.0) / 127).to(torch.float32).clamp(min=2.0 ** -100)
    y = torch.where(fine[:, None], xd, 0.0) / scale.double()[:, None]
    n = torch.floor(y)
    # the quotient's distance to a tie, from the exact remainder: (n + 1/2) s fits float64 exactly, and so does x
    over = torch.where(fine[:, None], xd, 0.0) - (n + 0.5) * scale.double()[:, None]
    up = (over > 0) | ((over == 0) & (n.remainder(2) == 1))
    code = (n + up.double()).to(torch.int8)
    return code, torch.where(fine, scale, float("nan"))


def linear(x, codes, scale, bias, result):
    """(y, bound)."""
    a, s = rows(x)
    total = (a.double() @ codes.double().T) * scale.double() * s.double()[:, None]
    y = total if bias is None else total + bias.double()
    return y, 4 * U32 * (total.abs() + y.abs()) + half_step(result) * y.abs()
