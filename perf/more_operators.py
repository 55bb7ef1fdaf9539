"""The operators of a layer served in few bits that this framework is timed and checked on.

Three operators: a rolling cache held in 8 or 4 bits, quantised as it is written and read
back in the order of its positions (``window_cache_fill``, ``window_cache_read``), one
token's attention over such a cache (``window_decode_attn``), and the product of tokens
and weights in 8-bit integers with a scale for each token and each row of the weights
(``int8_linear``).

Caches: groups of 32 elements of a row share a power of two, 2 ** (E - 127) with the byte E;
a code is an integer from -127 to 127 (8 bits), or one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 with a
sign (4 bits, the even element in a byte's low half).  E is the lowest, from 1 on, at which
the group's largest magnitude rounds to a code.  All of this is exact in 32 bits.

``run`` with ``own`` false is the plain form: elementary torch operations in 32 bits (64 for
the quotients of ``int8_linear``'s codes, which may lie next to a border), rounded once at
the end.  ``exact`` restates each operator in float64.
"""

import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
GROUP = 32


def listed():
    return [
        # a short prompt of one small layer into its cache and back: latency counts
        dict(name="cache_small", op="cache", B=1, Hk=4, N=150, d=32, dtype="f32", window=64, sinks=1, bits=8, later=False),
        # a ragged batch of prompts into 4-bit caches, read back as the first keys of their next chunks
        dict(name="cache_batch", op="cache", B=32, Hk=8, N=2048, d=128, dtype="bf16", window=1024, sinks=4, bits=4,
             later=False),
        # later chunks of long prompts, odd lengths, into caches that have gone round already
        dict(name="cache_chunk", op="cache", B=8, Hk=8, N=1021, d=64, dtype="bf16", window=2048, sinks=4, bits=8, later=True),
        # one token of one sequence: latency counts
        dict(name="decode_one", op="decode", B=1, H=16, Hk=4, d=64, dtype="bf16", window=1024, sinks=4, bits=4, buckets=0,
             far=0, full=True),
        # one token of each of a few sequences of any length, with the bias
        dict(name="decode_table", op="decode", B=8, H=16, Hk=16, d=32, dtype="f32", window=500, sinks=1, bits=8, buckets=32,
             far=128, full=False),
        # one token of each of a large batch, full caches
        dict(name="decode_batch", op="decode", B=32, H=32, Hk=8, d=128, dtype="bf16", window=4096, sinks=4, bits=4,
             buckets=0, far=0, full=True),
        # one token of one very long sequence
        dict(name="decode_long", op="decode", B=1, H=32, Hk=8, d=128, dtype="bf16", window=131068, sinks=4, bits=8,
             buckets=0, far=0, full=True),
        # a projection of one token: the weights are all that is read
        dict(name="linear_token", op="linear", M=1, K=4096, N=4096, dtype="bf16", bias=False),
        # one decoding step of a batch
        dict(name="linear_step", op="linear", M=32, K=4096, N=4096, dtype="bf16", bias=True),
        # a trunk-sized projection of one short chain
        dict(name="linear_small", op="linear", M=97, K=512, N=512, dtype="f32", bias=True),
        # odd sizes throughout
        dict(name="linear_odd", op="linear", M=777, K=1000, N=1333, dtype="f32", bias=True),
        # a projection of a long prompt
        dict(name="linear_prompt", op="linear", M=8192, K=4096, N=4096, dtype="bf16", bias=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: any of the operators, sizes spread over the logarithm of their range."""
    op = rng.choice(["cache", "decode", "decode", "linear", "linear"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op == "linear":
        c = dict(op=op, M=_log(rng, 1, 8192), K=_log(rng, 48, 6000), N=_log(rng, 48, 6000), dtype=dtype,
                 bias=rng.random() < 0.5)
        if rng.random() < 0.5:  # widths of models, rather than any
            c["K"], c["N"] = (max(64, x // 64 * 64) for x in (c["K"], c["N"]))
        while c["M"] * c["K"] * c["N"] > 8192 * 4096 * 4096:
            c["M"] //= 2
        return c
    H, Hk = rng.choice([(4, 4), (8, 8), (8, 2), (16, 16), (16, 4), (12, 4), (8, 1), (32, 8), (16, 1)])
    d, bits = rng.choice([24, 32, 64, 80, 96, 128]), rng.choice([4, 4, 8])
    sinks = rng.choice([0, 1, 4, 16, 50])
    if op == "cache":
        c = dict(op=op, B=rng.choice([1, 2, 8, 16]), Hk=Hk, N=_log(rng, 1, 4000), d=d, dtype=dtype,
                 window=_log(rng, 1, 4096), sinks=sinks, bits=bits, later=rng.random() < 0.5)
        while c["B"] > 1 and c["B"] * Hk * max(c["N"], c["window"]) * d > 32 * 8 * 2048 * 64:
            c["B"] //= 2
        return c
    c = dict(op=op, B=rng.choice([1, 2, 5, 16, 32]), H=H, Hk=Hk, d=d, dtype=dtype, window=_log(rng, 1, 20000), sinks=sinks,
             bits=bits, buckets=rng.choice([16, 32, 64, 90]) if rng.random() < 0.4 else 0, far=_log(rng, 96, 1000),
             full=rng.random() < 0.6)
    while c["B"] > 1 and c["B"] * H * c["window"] * d > 32 * 32 * 4096 * 64:
        c["B"] //= 2
    return c


def _edges(count, far):
    """Ascending distances at which the bucket goes up: half of them one by one, the rest in equal ratios up to ``far``."""
    exact = count // 2
    edges = list(range(1, exact + 1))
    for k in range(1, count - exact):
        edges.append(max(edges[-1] + 1, int(math.ceil(exact * (far / exact) ** (k / (count - exact)) - 1e-9))))
    return tuple(edges)


def _up(n, to):
    return -(-n // to) * to


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    rnd = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    s = dict(case)
    if case["op"] == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        s["x"] = (rnd(M, K) * torch.exp(rnd(M, 1))).to(dt)  # tokens of different sizes
        w = rnd(N, K) * K ** -0.5
        scale = (w.abs().amax(1).double() / 127).float()
        codes = torch.zeros(N, _up(K, 16), dtype=torch.int8, device=dev)  # rows of whole 16-byte pieces
        codes[:, :K] = torch.round(w.double() / scale.double()[:, None]).to(torch.int8)
        s["codes"], s["scale"] = codes[:, :K], scale
        s["bias"] = rnd(N).to(dt) if case["bias"] else None
        return s
    B, Hk, d, bits = case["B"], case["Hk"], case["d"], case["bits"]
    S = case["sinks"] + case["window"]
    lengthwise = torch.arange(B, device=dev)
    for name in ("k", "v"):  # what the cache holds: rows whose channels are of different sizes, as a layer's keys are
        size = torch.exp(0.5 * rnd(Hk, 1, d))
        rows = rnd(B, Hk, S, d) * size
        s[name + "c"], s[name + "s"] = _quantise(rows.to(dt), bits)
        pad = torch.zeros(B, Hk, s[name + "s"].shape[2], _up(S, 16), dtype=torch.uint8, device=dev)
        pad[..., :S] = s[name + "s"]
        s[name + "s"] = pad
        new = rnd(B, Hk, case["N"], d) if case["op"] == "cache" else rnd(B, Hk, 1, d)
        s[name] = (new * size).to(dt) if case["op"] == "cache" else (new * size).to(dt)[:, :, 0].contiguous()
    if case["op"] == "cache":
        s["lengths"] = (case["N"] - lengthwise * case["N"] // (2 * B)).to(torch.int32)
        s["starts"] = None
        if case["later"]:
            s["starts"] = torch.randint(1, 3 * S + 1, (B,), generator=g, device=dev).to(torch.int32)
        s["held"] = s["lengths"] if s["starts"] is None else s["lengths"] + s["starts"]
        return s
    s["q"] = rnd(B, case["H"], d).to(dt)
    if case["buckets"]:
        s["edges"] = _edges(case["buckets"], case["far"])
        s["table"] = rnd(case["H"], len(s["edges"]) + 1).to(dt)
    if case["full"]:  # long past the window
        at = S + torch.randint(0, 3 * S, (B,), generator=g, device=dev)
    else:  # any length, none at all among them; -1: a row of the batch that no sequence uses
        at = torch.randint(0, 2 * S, (B,), generator=g, device=dev)
        at[B // 2:] //= 4
        at[B - 1] = -1 if B > 2 else 0
    s["lengths"] = at.to(torch.int32)
    return s


def _grouped(x):
    """(..., groups, 32), the last group filled up with zeros."""
    d = x.shape[-1]
    x = torch.nn.functional.pad(x, (0, _up(d, GROUP) - d))
    return x.reshape(*x.shape[:-1], -1, GROUP)


def _power(e):
    """2 ** e as fp32, -126 <= e <= 127."""
    return ((e + 127) << 23).to(torch.int32).view(torch.float32)


def _quantise(x, bits):
    """Rows x (B,Hk,n,d) as codes (B,Hk,n,bytes) and exponent bytes (B,Hk,groups,n)."""
    x = _grouped(x.float())
    top = x.abs().amax(-1).contiguous().view(torch.int32)
    e, m = (top >> 23) - 127, top & 0x7FFFFF
    up = (m > 0x600000) if bits == 4 else (m >= 0x7F0000)
    odd = e == 128  # an infinity or NaN in the group
    e = (e - (2 if bits == 4 else 6) + (up & (e < 127)).int()).clamp(-126, 125)
    y = torch.where(odd[..., None], torch.zeros_like(x), x) * _power(-e)[..., None]
    a = y.abs()
    if bits == 4:
        code = torch.where(a < 2, torch.round(2 * a), torch.where(a < 4, torch.round(a) + 2, torch.round(a / 2) + 4))
        code = code.clamp(max=7).to(torch.int32) + 8 * torch.signbit(y).int()
        code = code.flatten(-2)
        code = (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8)
    else:
        code = torch.round(y).clamp(-127, 127).to(torch.int8).flatten(-2).view(torch.uint8)
    byte = torch.where(odd, 255, e + 127).to(torch.uint8)
    return code, byte.transpose(-1, -2).contiguous()


def _values(code, byte, d):
    """fp32 rows (B,Hk,n,d) of codes (B,Hk,n,bytes) and exponent bytes (B,Hk,groups,n)."""
    groups = byte.shape[2]
    if code.shape[-1] == groups * GROUP:
        v = code.view(torch.int8).float()
    else:
        levels = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=code.device)
        levels = torch.cat((levels, -levels))
        v = levels[torch.stack((code & 15, code >> 4), -1).flatten(-2).int()]
    e = byte.transpose(-1, -2).contiguous().int() - 127
    scale = torch.where(e == 128, torch.full_like(e, 0, dtype=torch.float32) / 0, _power(e.clamp(-126, 127)))
    return (v.unflatten(-1, (groups, GROUP)) * scale[..., None]).flatten(-2)[..., :d]


def _held(s, last):
    """Position that each slot of the rolling cache holds once position ``last`` (B,) is the latest; below 0: none."""
    slot = torch.arange(s["sinks"] + s["window"], device=last.device)[None, :]
    last = last[:, None].long()
    turn = torch.div(last - slot, s["window"], rounding_mode="floor").clamp(min=0)
    return torch.where(slot <= last, torch.where(slot < s["sinks"], slot, slot + turn * s["window"]), -1)


def _cache_plain(s):
    S, W, sinks = s["sinks"] + s["window"], s["window"], s["sinks"]
    held = s["held"].long()
    at = _held(s, held - 1)
    row = at if s["starts"] is None else at - s["starts"].long()[:, None]
    new = (at >= 0) & (row >= 0)
    row = row.clamp(min=0)[:, None, :, None].expand(-1, s["Hk"], -1, s["d"])
    out = []
    # the order of the positions: the first tokens, then the last `window` positions
    j = torch.arange(S, device=held.device)[None, :]
    p = torch.where(j < sinks, j.expand(s["B"], -1), held[:, None] - S + j)
    there = torch.where(j < sinks, j < held[:, None], p >= sinks)
    slot = torch.where(p < sinks, p, sinks + (p - sinks) % W).clamp(min=0)
    slot = slot[:, None, :, None].expand(-1, s["Hk"], -1, s["d"])
    for name in ("k", "v"):
        code, byte = _quantise(torch.gather(s[name], 2, row), s["bits"])
        s[name + "c"].copy_(torch.where(new[:, None, :, None], code, s[name + "c"]))
        s[name + "s"][..., :S] = torch.where(new[:, None, None, :], byte, s[name + "s"][..., :S])
        rows = torch.gather(_values(s[name + "c"], s[name + "s"][..., :S], s["d"]), 2, slot)
        out.append(torch.where(there[:, None, :, None], rows, torch.zeros_like(rows)).to(DTYPES[s["dtype"]]))
    return [*out, there.float()]


def _bucket(s, mag):
    """Bucket of each distance (query minus key)."""
    edges = torch.tensor(s["edges"], device=mag.device)
    lut = (torch.arange(s["edges"][-1] + 1, device=mag.device)[:, None] >= edges).sum(1)
    return lut[mag.clamp(0, s["edges"][-1])]


def _decode_plain(s):
    t = s["lengths"].long()
    S, G = s["sinks"] + s["window"], s["H"] // s["Hk"]
    slot = torch.where(t < s["sinks"], t, s["sinks"] + (t - s["sinks"]) % s["window"]).clamp(min=0)
    b = torch.arange(s["B"], device=t.device)
    on = (t >= 0)[:, None, None]
    rows = []
    for name in ("k", "v"):
        code, byte = _quantise(s[name][:, :, None], s["bits"])
        codes, bytes_ = s[name + "c"], s[name + "s"]
        codes[b, :, slot] = torch.where(on, code[:, :, 0], codes[b, :, slot])
        bytes_[b, :, :, slot] = torch.where(on, byte[..., 0], bytes_[b, :, :, slot])
        rows.append(_values(codes, bytes_[..., :S], s["d"]))
    at = _held(s, t)
    q = s["q"].float().reshape(s["B"], s["Hk"], G, s["d"])
    score = (rows[0] @ q.transpose(-1, -2).contiguous()).transpose(-1, -2) * s["d"] ** -0.5
    if s["buckets"]:
        bias = s["table"].float()[:, _bucket(s, t[:, None] - at)].transpose(0, 1)
        score = score + bias.reshape(s["B"], s["Hk"], G, S)
    score = score.masked_fill((at < 0)[:, None, None, :], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-1e30))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    o = (p @ rows[1]).reshape(s["B"], s["H"], s["d"])
    # (the caches as they are held: codes and exponents are exact functions of the rows)
    return [o.to(s["q"].dtype), s["kc"], s["ks"], s["vc"], s["vs"]]


def _linear_plain(s):
    x = s["x"].double()
    scale = (x.abs().amax(1, keepdim=True) / 127).float().clamp(min=2.0 ** -100)
    a = torch.round(x / scale.double()).float()
    y = (a @ s["codes"].float().t().contiguous()) * scale * s["scale"][None, :]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return [y.to(s["x"].dtype)]


def _own(s):
    root = os.path.join(os.getcwd(), "deepfold-linear_amd")  # the package lies one folder below the root
    if root not in sys.path:
        sys.path.insert(0, root)
    import deepfold_amd as df

    if s["op"] == "linear":
        return [df.int8_linear(s["x"], s["codes"], s["scale"], s["bias"])]
    kc, vc = (df.QuantizedCache(s[n + "c"], s[n + "s"], s["bits"]) for n in ("k", "v"))
    if s["op"] == "cache":
        df.window_cache_fill(s["k"], s["v"], s["lengths"], kc, vc, n_sink=s["sinks"], starts=s["starts"])
        return list(df.window_cache_read(kc, vc, s["held"], s["d"], n_sink=s["sinks"], dtype=DTYPES[s["dtype"]]))
    o = df.window_decode_attn(s["q"], s["k"], s["v"], kc, vc, s["lengths"], n_sink=s["sinks"],
                              rel_table=s.get("table"), rel_edges=s.get("edges"))
    return [o, s["kc"], s["ks"], s["vc"], s["vs"]]


def run(state):
    if own:
        return _own(state)
    return {"cache": _cache_plain, "decode": _decode_plain, "linear": _linear_plain}[state["op"]](state)


def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        return {"bytes": M * K * e + N * K + 4 * N + M * N * e + (N * e if case["bias"] else 0), "flops": 2 * M * N * K}
    B, Hk, d = case["B"], case["Hk"], case["d"]
    S, dp = case["sinks"] + case["window"], _up(d, GROUP)
    held = dp * case["bits"] // 8 + dp // GROUP  # bytes of a row in the cache
    if case["op"] == "cache":
        # rows written (about min(S, length) of them), then a whole cache's read and given out
        new = sum(min(S, case["N"] - b * case["N"] // (2 * B)) for b in range(B))
        rows = B * S if case["later"] else new
        return {"bytes": 2 * Hk * (new * (d * e + held) + rows * held + B * S * d * e) + 4 * B * S, "flops": 0}
    # about half of a cache that is not full is in use
    rows = B * S if case["full"] else max(1, B * S // 2)
    return {"bytes": 2 * rows * Hk * held + 2 * B * (case["H"] + Hk) * d * e, "flops": 4 * rows * case["H"] * d}


def _two_to(e):
    """2 ** e in float64, of whole e: the bits themselves (a device's power function may be off by one)."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _exact_step(amax, bits):
    """The step of groups with these largest magnitudes, in float64."""
    _, e = torch.frexp(amax)
    e = e.to(torch.int64) - (3 if bits == 4 else 7)  # amax in [4, 8) or [64, 128) steps
    step = _two_to(e.clamp(min=-1000))
    over = amax > 7 * step if bits == 4 else amax >= 127.5 * step
    top = e == (125 if bits == 4 else 121)  # the largest exponent of 32 bits: it is not raised
    step = torch.where(over & ~top, 2 * step, step)
    return step.clamp(min=2.0 ** -126)


def _exact_values(x, bits):
    """What rows x stand for once they are held in the cache, in float64."""
    d = x.shape[-1]
    full = torch.zeros(*x.shape[:-1], _up(d, GROUP), dtype=torch.float64, device=x.device)
    full[..., :d] = x
    g = full.unflatten(-1, (-1, GROUP))
    step = _exact_step(g.abs().amax(-1, keepdim=True), bits)
    a = g.abs() / step
    if bits == 8:
        n = torch.floor(a)
        frac = a - n
        n = (n + ((frac > 0.5) | ((frac == 0.5) & (n % 2 == 1))).double()).clamp(max=127)
    else:
        code = torch.zeros_like(a)
        for i, mid in enumerate((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)):  # halfway: to the even code
            code += ((a > mid) | ((a == mid) & (i % 2 == 1))).double()
        n = torch.where(code < 4, code / 2, torch.where(code < 6, code - 2, 2 * code - 8))
    return (torch.sign(g) * n * step).flatten(-2)[..., :d]


def _exact_held(codes, exps, d, bits):
    """float64 rows of what a cache holds, codes (..., n, bytes) and exponent bytes (..., groups, n)."""
    if bits == 8:
        v = codes.view(torch.int8).double()
    else:
        mag = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=codes.device)
        half = torch.empty(*codes.shape, 2, dtype=torch.long, device=codes.device)
        half[..., 0], half[..., 1] = codes % 16, torch.div(codes, 16, rounding_mode="floor")
        v = (mag[half % 8] * (1 - 2 * (half // 8))).flatten(-2)
    scale = _two_to(exps.long() - 127).transpose(-1, -2).repeat_interleave(GROUP, -1)
    return (v * scale)[..., :d]


def exact(case, seed):
    s = prepare(case, seed)
    dev = torch.device("cuda")
    if case["op"] == "linear":
        x, w = s["x"].double(), s["codes"].double() * s["scale"].double()[:, None]
        step = torch.clamp((x.abs().amax(1) / 127).float(), min=2.0 ** -100).double()[:, None]
        y = (torch.round(x / step) * step) @ w.t().contiguous()
        return [y if s["bias"] is None else y + s["bias"].double()]
    B, Hk, d, bits, W, first = case["B"], case["Hk"], case["d"], case["bits"], case["window"], case["sinks"]
    S = first + W
    place = lambda p: p if p < first else first + (p - first) % W  # noqa: E731
    if case["op"] == "cache":
        lengths, starts = s["lengths"].tolist(), [0] * B if s["starts"] is None else s["starts"].tolist()
        out = [torch.zeros(B, Hk, S, d, dtype=torch.float64, device=dev) for _ in range(2)]
        mask = torch.zeros(B, S, dtype=torch.float64, device=dev)
        for b in range(B):
            total = lengths[b] + starts[b]
            where = [p for p in range(min(first, total))] + list(range(max(first, total - W), total))
            row = [p if p < first else p - total + S for p in where]
            old = [i for i, p in enumerate(where) if p < starts[b]]
            new = [i for i, p in enumerate(where) if p >= starts[b]]
            mask[b, row] = 1
            for o, name in zip(out, ("k", "v")):
                slots = [place(where[i]) for i in old]
                o[b][:, [row[i] for i in old]] = _exact_held(s[name + "c"][b][:, slots], s[name + "s"][b][:, :, slots], d, bits)
                rows = s[name][b].double()[:, [where[i] - starts[b] for i in new]]
                o[b][:, [row[i] for i in new]] = _exact_values(rows, bits)
        return [*out, mask]
    H, G = case["H"], case["H"] // Hk
    o = torch.zeros(B, H, d, dtype=torch.float64, device=dev)
    lengths = s["lengths"].tolist()
    for b in range(B):
        n = lengths[b]
        if n < 0:
            continue
        where = list(range(min(first, n))) + list(range(max(first, n - W + 1), n))
        slots = torch.tensor([place(p) for p in where], dtype=torch.long, device=dev)
        kk, vv = (torch.cat((_exact_held(s[x + "c"][b][:, slots], s[x + "s"][b][:, :, slots], d, bits),
                             _exact_values(s[x][b].double(), bits)[:, None]), 1) for x in ("k", "v"))
        for h in range(H):
            score = (kk[h // G] * s["q"][b, h].double()).sum(-1) / math.sqrt(d)
            if case["buckets"]:
                gap = n - torch.tensor(where + [n], device=dev)
                score = score + s["table"][h].double()[sum((gap >= x).long() for x in s["edges"])]
            w = torch.exp(score - score.max())
            o[b, h] = (w[:, None] * vv[h // G]).sum(0) / w.sum()
    return [o, None, None, None, None]
