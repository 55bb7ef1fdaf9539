"""The sequence operators that this framework is timed and checked on.

Four operators: the learned bias by buckets of the relative position (``rel_pos_bias``,
with its gradient), attention over a sliding window and a few first tokens
(``flash_window_attn``, forward and training), the copy of a prompt into the rolling cache
that such attention needs (``window_cache_fill``) and its single-token form over that cache
(``window_decode_attn``).

``run`` with ``own`` false is the plain form: elementary torch operations in 32 bits (64
for the long sums of the table's gradient), rounded once at the end.  ``exact`` restates
each operator in float64, with the gradients written out.
"""

import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # the bias of one small layer, for a short chain: latency counts
        dict(name="bias_small", op="bias", B=1, H=8, M=97, N=97, buckets=32, far=128, both=True, dtype="f32",
             table="f32", chains=False),
        # the pair bias of the diffusion transformer's 1024 tokens, in training
        dict(name="bias_pair", op="bias", B=1, H=16, M=1024, N=1024, buckets=32, far=128, both=True, dtype="bf16",
             table="f32", chains=False),
        # a batch of complexes, residue numbers with gaps and chain breaks, odd length, in training
        dict(name="bias_chains", op="bias", B=4, H=16, M=777, N=777, buckets=64, far=500, both=True, dtype="f32",
             table="f32", chains=True),
        # inference of one small layer: a short chain, both directions, with the bias
        dict(name="window_small", op="window", B=1, H=4, Hk=4, M=150, N=150, d=32, dtype="f32", window=64, sinks=1,
             causal=False, buckets=32, far=64, ragged=False, train=False),
        # training of a trunk-sized layer on a padded batch, both directions, bias and its gradient
        dict(name="window_train", op="window", B=2, H=16, Hk=16, M=1021, N=1021, d=64, dtype="bf16", window=129,
             sinks=4, causal=False, buckets=32, far=128, ragged=True, train=True),
        # training on long sequences: shared key heads, causal, wide window
        dict(name="window_gqa", op="window", B=1, H=16, Hk=4, M=4096, N=4096, d=128, dtype="bf16", window=1024,
             sinks=4, causal=True, buckets=0, far=0, ragged=False, train=True),
        # the longest prompt, read in one pass
        dict(name="window_long", op="window", B=1, H=32, Hk=8, M=8192, N=8192, d=128, dtype="bf16", window=2048,
             sinks=4, causal=True, buckets=32, far=128, ragged=False, train=False),
        # a short prompt into its cache
        dict(name="fill_small", op="fill", B=1, Hk=4, N=150, d=32, dtype="f32", window=64, sinks=1),
        # a ragged batch of prompts into their caches
        dict(name="fill_batch", op="fill", B=32, Hk=8, N=2048, d=128, dtype="bf16", window=1024, sinks=4),
        # one token of one sequence: latency counts
        dict(name="decode_one", op="decode", B=1, H=16, Hk=4, d=64, dtype="bf16", window=1024, sinks=4, buckets=0,
             far=0, full=True),
        # one token of each of a few sequences of any length, with the bias
        dict(name="decode_table", op="decode", B=8, H=16, Hk=16, d=32, dtype="f32", window=500, sinks=1, buckets=32,
             far=128, full=False),
        # one token of each of a large batch, full caches
        dict(name="decode_batch", op="decode", B=32, H=32, Hk=8, d=128, dtype="bf16", window=4096, sinks=4,
             buckets=0, far=0, full=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: any of the operators, sizes spread over the logarithm of their range."""
    op = rng.choice(["bias", "window", "window", "window", "fill", "decode", "decode"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    buckets = rng.choice([16, 32, 64, 90])
    far = _log(rng, 48, 1000)
    if op == "bias":
        c = dict(op=op, B=rng.choice([1, 2, 4]), H=rng.choice([4, 8, 16]), M=_log(rng, 1, 1500), N=_log(rng, 8, 1500),
                 buckets=buckets, far=far, both=rng.random() < 0.6, dtype=dtype, table=rng.choice(["f32", dtype]),
                 chains=rng.random() < 0.5)
        if not c["chains"]:
            c["B"] = 1
        while c["B"] * c["H"] * c["M"] * c["N"] > (1 << 25):
            c["N"] = c["N"] // 2
        return c
    H, Hk = rng.choice([(4, 4), (8, 8), (8, 2), (16, 16), (16, 4), (12, 4), (8, 1), (32, 8)])
    d = rng.choice([24, 32, 64, 80, 128])
    window, sinks = _log(rng, 1, 2048), rng.choice([0, 1, 4, 16, 50])
    if op == "window":
        N = _log(rng, 1, 4096)
        c = dict(op=op, B=rng.choice([1, 2, 4]), H=H, Hk=Hk, M=N if rng.random() < 0.7 else _log(rng, 1, N), N=N, d=d,
                 dtype=dtype, window=window, sinks=sinks, causal=rng.random() < 0.6,
                 buckets=buckets if rng.random() < 0.5 else 0, far=far, ragged=rng.random() < 0.4,
                 train=rng.random() < 0.6)
        while c["B"] > 1 and c["B"] * c["H"] * c["M"] * c["N"] > (1 << 28):
            c["B"] //= 2
        while c["H"] * c["M"] * c["N"] > (1 << 28):
            c["M"], c["N"] = c["M"] // 2, c["N"] // 2
        c["M"] = max(1, c["M"])
        return c
    if op == "fill":
        return dict(op=op, B=rng.choice([1, 2, 8, 16]), Hk=Hk, N=_log(rng, 1, 3000), d=d, dtype=dtype, window=window,
                    sinks=sinks)
    return dict(op=op, B=rng.choice([1, 2, 5, 16, 32]), H=H, Hk=Hk, d=d, dtype=dtype, window=2 * window, sinks=sinks,
                buckets=buckets if rng.random() < 0.5 else 0, far=far, full=rng.random() < 0.6)


def _edges(count, far, both):
    """Ascending magnitudes at which the bucket goes up: half of them one by one, the rest in equal
    ratios up to ``far``, in whole numbers."""
    side = count // 2 if both else count
    exact = max(1, side // 2)
    edges = list(range(1, exact + 1))
    for k in range(1, side - exact):
        edges.append(max(edges[-1] + 1, int(math.ceil(exact * (far / exact) ** (k / (side - exact)) - 1e-9))))
    return tuple(edges)


def _both(case):
    return case["both"] if case["op"] == "bias" else not case["causal"] if case["op"] == "window" else False


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    rnd = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    s = dict(case)
    if case["op"] == "bias" or case.get("buckets"):
        s["edges"] = _edges(case["buckets"], case["far"], _both(case))
        heads = (len(s["edges"]) + 1) * (2 if _both(case) else 1)
        s["table"] = rnd(case["H"], heads).to(DTYPES[case["table"]] if case["op"] == "bias" else dt)
    if case["op"] == "bias":
        B, H, M, N = case["B"], case["H"], case["M"], case["N"]
        s["q_pos"] = s["k_pos"] = None
        if case["chains"]:
            # residue numbers that go up by one, now and then by a gap, and start again with each chain
            step = 1 + (torch.rand(B, max(M, N), generator=g, device=dev) < 0.02) * torch.randint(
                1, 40, (B, max(M, N)), generator=g, device=dev)
            pos = torch.cumsum(step, 1)
            s["k_pos"] = (pos % 400)[:, :N].to(torch.int32).contiguous()
            s["q_pos"] = (pos % 400)[:, :M].to(torch.int32).contiguous()
        s["table"].requires_grad_(True)
        s["go"] = rnd(*((B, H, M, N) if case["chains"] else (H, M, N))).to(dt)
        return s
    B, Hk, d = case["B"], case["Hk"], case["d"]
    if case["op"] == "window":
        H, M, N = case["H"], case["M"], case["N"]
        s["q"], s["k"], s["v"] = rnd(B, H, M, d).to(dt), rnd(B, Hk, N, d).to(dt), rnd(B, Hk, N, d).to(dt)
        s["mask"] = None
        if case["ragged"]:
            s["mask"] = torch.zeros(B, N, device=dev)
            for b in range(B):
                s["mask"][b, :N - N // 85 - b * N // (2 * B)] = 1.0
        if case["train"]:
            for t in ("q", "k", "v", "table"):
                if s.get(t) is not None:
                    s[t].requires_grad_(True)
            s["go"] = rnd(B, H, M, d).to(dt)
        return s
    S = case["sinks"] + case["window"]
    if case["op"] == "fill":
        s["k"], s["v"] = rnd(B, Hk, case["N"], d).to(dt), rnd(B, Hk, case["N"], d).to(dt)
        s["lengths"] = torch.tensor([case["N"] - b * case["N"] // (2 * B) for b in range(B)], dtype=torch.int32,
                                    device=dev)
        s["kc"], s["vc"] = torch.zeros(B, Hk, S, d, device=dev, dtype=dt), torch.zeros(B, Hk, S, d, device=dev, dtype=dt)
        return s
    H = case["H"]
    s["q"], s["k"], s["v"] = rnd(B, H, d).to(dt), rnd(B, Hk, d).to(dt), rnd(B, Hk, d).to(dt)
    s["kc"], s["vc"] = rnd(B, Hk, S, d).to(dt), rnd(B, Hk, S, d).to(dt)
    if case["full"]:  # long past the window
        at = S + torch.randint(0, 3 * S, (B,), generator=g, device=dev)
    else:  # any length, none at all among them; -1: a row of the batch that no sequence uses
        at = torch.randint(0, 2 * S, (B,), generator=g, device=dev)
        at[B // 2:] //= 4
        at[B - 1] = -1 if B > 2 else 0
    s["lengths"] = at.to(torch.int32)
    return s


def _bucket(s, rel):
    """Bucket of each relative position (key minus query)."""
    edges = torch.tensor(s["edges"], device=rel.device)
    lut = (torch.arange(s["edges"][-1] + 1, device=rel.device)[:, None] >= edges).sum(1)
    mag = rel.abs() if _both(s) else (-rel).clamp(min=0)
    b = lut[mag.clamp(max=s["edges"][-1])]
    return b + (rel > 0) * (len(s["edges"]) + 1) if _both(s) else b


def _table_grad(s, bucket, g):
    """(H, buckets): the sums over each bucket of g (H, ..., N); a row's in 32 bits, those of all rows in 64."""
    n, rows = bucket.shape[-1], bucket.numel() // bucket.shape[-1]
    hit = (bucket.reshape(rows, n, 1) == torch.arange(s["table"].shape[1], device=g.device)).float()
    g = g.reshape(g.shape[0], rows, n).transpose(0, 1).float().contiguous()
    return (g @ hit).double().sum(0).to(s["table"].dtype)


def _bias_plain(s):
    ar = lambda n: torch.arange(n, device=s["table"].device)  # noqa: E731
    if s["chains"]:
        bucket = _bucket(s, s["k_pos"].long()[:, None, :] - s["q_pos"].long()[:, :, None])
        out = s["table"].detach().float()[:, bucket].transpose(0, 1)
        grad = s["go"].transpose(0, 1)
    else:
        bucket = _bucket(s, ar(s["N"])[None, :] - ar(s["M"])[:, None] - (s["N"] - s["M"]))
        out = s["table"].detach().float()[:, bucket]
        grad = s["go"]
    return out.to(DTYPES[s["dtype"]]).contiguous(), _table_grad(s, bucket, grad)


def _visible(s, t, j):
    """Whether a query at position t sees a key at position j, without the mask."""
    near = ((t - j < s["window"]) & (j <= t)) if s["causal"] else ((t - j).abs() < s["window"])
    first = (j < s["sinks"]) & (j <= t) if s["causal"] else (j < s["sinks"])
    return near | first


def _window_plain(s):
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    M, N, G = s["M"], s["N"], s["H"] // s["Hk"]
    t = torch.arange(M, device=q.device)[:, None] + (N - M)
    j = torch.arange(N, device=q.device)[None, :]
    seen = _visible(s, t, j)[None, None]
    if s["mask"] is not None:
        seen = seen & (s["mask"] != 0)[:, None, None, :] & (s["mask"][:, N - M:] != 0)[:, None, :, None]
    score = q @ k.repeat_interleave(G, 1).transpose(-1, -2).contiguous() * s["d"] ** -0.5
    bias = None
    if s["buckets"]:
        bucket = _bucket(s, j - t)
        bias = s["table"].detach().float()[:, bucket]
        if s["train"]:
            bias.requires_grad_(True)
        score = score + bias
    score = score.masked_fill(~seen, -math.inf)
    p = torch.exp(score - score.detach().amax(-1, keepdim=True).clamp(min=-1e30))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    o = p @ v.repeat_interleave(G, 1)
    if not s["train"]:
        return [o.to(s["q"].dtype)]
    wrt = [s["q"], s["k"], s["v"]] + ([bias] if bias is not None else [])
    grads = list(torch.autograd.grad(o, wrt, s["go"].float()))
    if bias is not None:
        grads[3] = _table_grad(s, bucket, grads[3])
    return [o.detach().to(s["q"].dtype)] + grads


def _held(s, last):
    """Position that each slot of the rolling cache holds once position ``last`` (B,) is the latest; below 0: none."""
    slot = torch.arange(s["sinks"] + s["window"], device=last.device)[None, :]
    last = last[:, None].long()
    turn = torch.div(last - slot, s["window"], rounding_mode="floor").clamp(min=0)
    return torch.where(slot <= last, torch.where(slot < s["sinks"], slot, slot + turn * s["window"]), -1)


def _fill_plain(s):
    at = _held(s, s["lengths"] - 1)
    rows = at.clamp(min=0)[:, None, :, None].expand(-1, s["Hk"], -1, s["d"])
    used = (at >= 0)[:, None, :, None]
    for cache, new in ((s["kc"], s["k"]), (s["vc"], s["v"])):
        cache.copy_(torch.where(used, torch.gather(new, 2, rows), cache))
    return [s["kc"], s["vc"]]


def _decode_plain(s):
    t = s["lengths"].long()
    G = s["H"] // s["Hk"]
    slot = torch.where(t < s["sinks"], t, s["sinks"] + (t - s["sinks"]) % s["window"]).clamp(min=0)
    b = torch.arange(s["B"], device=t.device)
    on = (t >= 0)[:, None, None]
    for cache, new in ((s["kc"], s["k"]), (s["vc"], s["v"])):
        cache[b, :, slot] = torch.where(on, new, cache[b, :, slot])
    at = _held(s, t)
    score = (s["kc"].float().repeat_interleave(G, 1) @ s["q"].float()[..., None])[..., 0] * s["d"] ** -0.5
    if s["buckets"]:
        score = score + s["table"].float()[:, _bucket(s, at - t[:, None])].transpose(0, 1)
    score = score.masked_fill((at < 0)[:, None, :], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-1e30))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    o = (p[:, :, None, :] @ s["vc"].float().repeat_interleave(G, 1))[:, :, 0]
    return [o.to(s["q"].dtype), s["kc"], s["vc"]]


def _own(s):
    root = os.path.join(os.getcwd(), "deepfold-linear_amd")  # the package lies one folder below the root
    if root not in sys.path:
        sys.path.insert(0, root)
    import deepfold_amd as df

    table, edges = s.get("table"), s.get("edges")
    if s["op"] == "bias":
        out = df.rel_pos_bias(table, edges, s["M"], s["N"], q_pos=s["q_pos"], k_pos=s["k_pos"],
                              bidirectional=s["both"], dtype=DTYPES[s["dtype"]])
        return [out, torch.autograd.grad(out, table, s["go"])[0]]
    if s["op"] == "window":
        o = df.flash_window_attn(s["q"], s["k"], s["v"], s["mask"], window=s["window"], n_sink=s["sinks"],
                                 causal=s["causal"], rel_table=table, rel_edges=edges)
        if not s["train"]:
            return [o]
        wrt = [s["q"], s["k"], s["v"]] + ([table] if table is not None else [])
        return [o] + list(torch.autograd.grad(o, wrt, s["go"]))
    if s["op"] == "fill":
        df.window_cache_fill(s["k"], s["v"], s["lengths"], s["kc"], s["vc"], n_sink=s["sinks"])
        return [s["kc"], s["vc"]]
    o = df.window_decode_attn(s["q"], s["k"], s["v"], s["kc"], s["vc"], s["lengths"], n_sink=s["sinks"],
                              rel_table=table, rel_edges=edges)
    return [o, s["kc"], s["vc"]]


def run(state):
    if own:
        return _own(state)
    plain = {"bias": _bias_plain, "window": _window_plain, "fill": _fill_plain, "decode": _decode_plain}
    return plain[state["op"]](state)


def _pairs(case, n_masked=0):
    """Visible (query, key) pairs of one head of one sample."""
    M, N, w, s, total = case["M"], case["N"], case["window"], case["sinks"], 0
    for i in range(M):
        t = i + N - M
        lo, hi = max(0, t - w + 1), (t if case["causal"] else min(N - 1, t + w - 1))
        total += hi - lo + 1 + min(s, lo) + (0 if case["causal"] else max(0, s - max(hi + 1, lo, 0)))
    return total


def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "bias":
        n = (case["B"] if case["chains"] else 1) * case["H"] * case["M"] * case["N"]
        return {"bytes": 2 * n * e, "flops": n}
    B, Hk, d = case["B"], case["Hk"], case["d"]
    if case["op"] == "window":
        qo, kv = B * case["H"] * case["M"] * d * e, B * Hk * case["N"] * d * e
        pairs = B * case["H"] * _pairs(case)
        if case["train"]:  # q, k, v, dO read, o, dq, dk, dv written; seven products, the forward's two among them
            return {"bytes": 4 * qo + 4 * kv, "flops": 14 * d * pairs}
        return {"bytes": 2 * qo + 2 * kv, "flops": 4 * d * pairs}
    S = case["sinks"] + case["window"]
    if case["op"] == "fill":
        rows = sum(min(S, case["N"] - b * case["N"] // (2 * B)) for b in range(B))
        return {"bytes": 4 * rows * Hk * d * e, "flops": 0}
    # about half of a cache that is not full is in use
    rows = B * S if case["full"] else max(1, B * S // 2)
    return {"bytes": 2 * rows * Hk * d * e + 2 * B * (case["H"] + Hk) * d * e, "flops": 4 * rows * case["H"] * d}


def _exact_bucket(edges, both, rel):
    mag = rel.abs() if both else torch.clamp(-rel, min=0)
    out = torch.zeros_like(rel)
    for x in edges:
        out += mag >= x
    return out + (rel > 0).to(rel.dtype) * (len(edges) + 1) if both else out


def _exact_sums(bucket, g, n):
    return torch.stack([(g * (bucket == b)).sum() for b in range(n)])


def _exact_softmax(score):
    top = score.amax(-1, keepdim=True)
    e = torch.where(torch.isneginf(score), torch.zeros_like(score), torch.exp(score - torch.nan_to_num(top, neginf=0.0)))
    return e / e.sum(-1, keepdim=True).clamp(min=1e-300)


def exact(case, seed):
    s = prepare(case, seed)
    dev = torch.device("cuda")
    f64 = lambda x: None if x is None else x.detach().double()  # noqa: E731
    edges, both, table = s.get("edges"), _both(case), f64(s.get("table"))
    if case["op"] == "bias":
        H, M, N = case["H"], case["M"], case["N"]
        if case["chains"]:
            rel = s["k_pos"].long()[:, None, :] - s["q_pos"].long()[:, :, None]
        else:
            rel = torch.arange(N, device=dev)[None, None, :] - (torch.arange(M, device=dev) + N - M)[None, :, None]
        bucket = _exact_bucket(edges, both, rel)
        out = torch.stack([table[h][bucket] for h in range(H)], 1)
        go = f64(s["go"]).reshape(out.shape)
        grad = torch.stack([_exact_sums(bucket, go[:, h], table.shape[1]) for h in range(H)])
        return [out.reshape(s["go"].shape), grad]
    if case["op"] == "window":
        B, H, Hk, M, N, d = (case[x] for x in ("B", "H", "Hk", "M", "N", "d"))
        q, k, v, go = f64(s["q"]), f64(s["k"]), f64(s["v"]), f64(s.get("go"))
        t = (torch.arange(M, device=dev) + N - M)[:, None]
        j = torch.arange(N, device=dev)[None, :]
        gone = (j > t) if case["causal"] else torch.zeros(M, N, dtype=torch.bool, device=dev)
        far = torch.maximum(t - j, j - t) >= case["window"]
        gone = gone | (far & (j >= case["sinks"]))
        bucket = _exact_bucket(edges, both, j - t) if table is not None else None
        o, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
        dt = None if table is None else torch.zeros_like(table)
        for b in range(B):
            hide = gone
            if s["mask"] is not None:
                hide = gone | (s["mask"][b] == 0)[None, :] | (s["mask"][b, N - M:] == 0)[:, None]
            for h in range(H):
                kk, vv = k[b, h * Hk // H], v[b, h * Hk // H]
                score = q[b, h] @ kk.T / math.sqrt(d)
                if table is not None:
                    score = score + table[h][bucket]
                p = _exact_softmax(torch.where(hide, torch.full_like(score, -math.inf), score))
                o[b, h] = p @ vv
                if not case["train"]:
                    continue
                dp = go[b, h] @ vv.T
                ds = p * (dp - (p * dp).sum(-1, keepdim=True))
                dv[b, h * Hk // H] += p.T @ go[b, h]
                dq[b, h] = ds @ kk / math.sqrt(d)
                dk[b, h * Hk // H] += ds.T @ q[b, h] / math.sqrt(d)
                if dt is not None:
                    dt[h] += _exact_sums(bucket, ds, table.shape[1])
        return ([o, dq, dk, dv] + ([dt] if dt is not None else [])) if case["train"] else [o]
    B, Hk, W, first = case["B"], case["Hk"], case["window"], case["sinks"]
    kc, vc = f64(s["kc"]), f64(s["vc"])
    lengths = s["lengths"].tolist()
    if case["op"] == "fill":
        for b in range(B):
            n = lengths[b]
            where = [p for p in range(n) if p < first or p >= n - W]
            to = [p if p < first else first + (p - first) % W for p in where]
            kc[b][:, to] = f64(s["k"][b][:, where])
            vc[b][:, to] = f64(s["v"][b][:, where])
        return [kc, vc]
    H, d = case["H"], case["d"]
    o = torch.zeros(B, H, d, dtype=torch.float64, device=dev)
    for b in range(B):
        n = lengths[b]
        if n < 0:
            continue
        where = [p for p in range(n + 1) if p < first or p > n - W]
        to = [p if p < first else first + (p - first) % W for p in where]
        kc[b][:, to[-1]], vc[b][:, to[-1]] = f64(s["k"][b]), f64(s["v"][b])
        kk = kc[b][:, to].repeat_interleave(H // Hk, 0)
        score = (kk * f64(s["q"][b])[:, None, :]).sum(-1) / math.sqrt(d)
        if table is not None:
            score = score + table[:, _exact_bucket(edges, both, torch.tensor(where, device=dev) - n)]
        o[b] = (_exact_softmax(score)[..., None] * vc[b][:, to].repeat_interleave(H // Hk, 0)).sum(1)
    return [o, kc, vc]
