"""The sequence operators on the GPU against their float64 forms (oracle/window.py) on identical inputs.

Every entry of every result is held to the elementwise bound that the oracle derives from half steps of the
operand and result types and from the fp32 arithmetic; copies and look-ups are exact.
"""

import math

import pytest
import torch

from oracle import window as ref

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF, F32 = torch.bfloat16, torch.float32
EDGES = (1, 2, 3, 4, 6, 9, 14, 20, 31)


def rnd(*shape, seed, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def holds(name, got, want, bound):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, name
    off = (got - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), (f"{name}: {int(bad.sum())} of {bad.numel()} entries off, worst {float(off.max()):.3e}, "
                           f"at most {float((off / bound.clamp(min=1e-30)).max()):.2f} times the bound")


def leaf(t):
    return None if t is None else t.to(DEV).requires_grad_(True)


def attention_case(B, H, Hk, M, N, d, dtype, window, n_sink, causal, rel=False, mask=None, scale=None, edges=EDGES, seed=1):
    from deepfold_amd import flash_window_attn

    q, k, v = (rnd(B, h, n, d, seed=seed + i, dtype=dtype) for i, (h, n) in enumerate(((H, M), (Hk, N), (Hk, N))))
    go = rnd(B, H, M, d, seed=seed + 3, dtype=dtype)
    table = rnd(H, (len(edges) + 1) * (1 if causal else 2), seed=seed + 4) if rel else None
    want = ref.attention(q, k, v, window=window, n_sink=n_sink, causal=causal, mask=mask, scale=scale, table=table,
                         edges=edges, grad=go, operand=dtype, result=dtype)
    x = [leaf(t) for t in (q, k, v, table)]
    kw = dict(window=window, n_sink=n_sink, causal=causal, scale=scale, rel_table=x[3], rel_edges=edges if rel else None)
    m = None if mask is None else mask.to(DEV)
    o = flash_window_attn(*x[:3], m, **kw)
    grads = torch.autograd.grad(o, [t for t in x if t is not None], go.to(DEV))
    with torch.no_grad():
        assert torch.equal(flash_window_attn(*x[:3], m, **kw), o)
    holds("o", o, *want["o"])
    for name, g in zip(("dq", "dk", "dv", "dtable"), grads):
        holds(name, g, *want[name])
    return o, grads


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("H,Hk,M,N,d,window,n_sink,rel", [
    (2, 2, 1, 1, 32, 1, 0, True), (2, 1, 2, 2, 24, 5, 1, False), (4, 2, 33, 33, 32, 7, 0, True),
    (3, 3, 64, 64, 64, 64, 4, False), (4, 1, 129, 129, 64, 40, 33, True), (2, 2, 150, 150, 20, 1, 2, True),
    (2, 1, 1, 77, 128, 30, 3, True), (2, 2, 45, 301, 128, 100, 5, False), (4, 2, 300, 300, 80, 31, 100, True),
    (2, 2, 257, 257, 7, 300, 1, True), (1, 1, 130, 260, 1, 64, 0, False), (6, 2, 96, 353, 33, 65, 17, True),
])
def test_attention(H, Hk, M, N, d, window, n_sink, rel, causal, dtype):
    attention_case(2, H, Hk, M, N, d, dtype, window, n_sink, causal, rel)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_long(causal, dtype):
    """Bands of several key tiles (rows past the exact-sum rule), first tokens in chunks, table ranges on both sides of a
    tile, one with the largest distance."""
    attention_case(1, 2, 1, 900, 900, 64, dtype, 400, 4, causal, True)
    attention_case(1, 2, 1, 600, 700, 32, dtype, 333, 128, causal, True, edges=(1, 5, 200, 2048) if causal else (3, 90))
    # the largest table: its sums leave the key tiles one buffer
    attention_case(1, 2, 1, 300, 310, 128, dtype, 290, 4, causal, True,
                   edges=(*range(1, 95), 2048) if causal else (*range(2, 48), 2048))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_masked(causal, dtype):
    """Padded tails, holes, a sample without any token; what lies in masked places (NaN, infinities) reaches nothing."""
    from deepfold_amd import flash_window_attn

    B, H, Hk, N, d = 4, 4, 2, 190, 64
    mask = torch.ones(B, N)
    mask[0, 111:] = 0
    mask[1] = (torch.rand(N, generator=torch.Generator().manual_seed(3)) < 0.6).float()
    mask[2] = 0
    mask[3, :70] = 0
    o, grads = attention_case(B, H, Hk, N, N, d, dtype, 23, 6, causal, True, mask=mask)
    assert not o[2].any() and not any(g[2].any() for g in grads[:3])
    assert not o[0, :, 111:].any() and not grads[1][0, :, 111:].any()

    x = [rnd(B, h, N, d, seed=1 + i, dtype=dtype) for i, h in enumerate((H, Hk, Hk))]
    go = rnd(B, H, N, d, seed=4, dtype=dtype)
    hole = (mask == 0)[:, None, :, None]
    bad = torch.tensor([math.nan, math.inf, -math.inf, 3e38]).repeat(N)[:N].to(dtype).view(1, 1, N, 1)
    y = [leaf(torch.where(hole, bad, t)) for t in x]
    table = leaf(rnd(H, (len(EDGES) + 1) * (1 if causal else 2), seed=5))
    o2 = flash_window_attn(*y, mask.to(DEV), window=23, n_sink=6, causal=causal, rel_table=table, rel_edges=EDGES)
    g2 = torch.autograd.grad(o2, [*y, table], torch.where(hole, bad, go).to(DEV))
    assert torch.equal(o2, o) and all(torch.equal(a, b) for a, b in zip(g2, grads))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_masked_long(dtype):
    """Key tiles whose queries are split over workgroups, with holes in the mask and first tokens among them."""
    mask = (torch.rand(2, 650, generator=torch.Generator().manual_seed(9)) < 0.8).float()
    mask[0, 400:] = 0
    attention_case(2, 4, 1, 650, 650, 64, dtype, 300, 5, True, True, mask=mask)
    attention_case(2, 4, 1, 600, 650, 128, dtype, 300, 5, False, False, mask=mask)


def test_offsets_beyond_32_bits():
    """Samples, and slots of a cache, more than 2^31 elements apart."""
    from deepfold_amd import flash_window_attn, window_cache_fill, window_decode_attn

    far, H, N, d, S = 2**31 + 64, 2, 40, 64, 24
    big = torch.empty(far + 8 * N * d * 4, dtype=BF, device=DEV)
    view = lambda at, *shape: big[at:].as_strided((2, *shape), (far, *torch.empty(shape, device="meta").stride()))
    K, V = view(0, H, N, d), view(H * N * d, H, N, d)
    q, k, v = (rnd(2, H, N, d, seed=s, dtype=BF).to(DEV) for s in (1, 2, 3))
    K.copy_(k), V.copy_(v)
    assert torch.equal(flash_window_attn(q, K, V, window=9, n_sink=2), flash_window_attn(q, k, v, window=9, n_sink=2))
    got, want = [view(2 * H * N * d, H, S, d), view(3 * H * N * d, H, S, d)], [torch.zeros(2, H, S, d, dtype=BF, device=DEV) for _ in "kv"]
    for c in got:
        c.zero_()
    lengths = torch.tensor([N, 7], device=DEV)
    window_cache_fill(K, V, lengths, *got, n_sink=2)
    window_cache_fill(k, v, lengths, *want, n_sink=2)
    o = [window_decode_attn(q[:, :, 0], k[:, :, 1], v[:, :, 1], *c, lengths, n_sink=2) for c in (got, want)]
    assert torch.equal(*o) and all(torch.equal(a, b) for a, b in zip(got, want))
    # slots far apart
    wide = big.as_strided((1, 1, 2, d), (0, 0, far, 1)), big[d:].as_strided((1, 1, 2, d), (0, 0, far, 1))
    near = [torch.zeros(1, 1, 2, d, dtype=BF, device=DEV) for _ in "kv"]
    for a, b in zip(wide, near):
        a.copy_(b)
    for c in (wide, near):
        window_cache_fill(k[:1, :1], v[:1, :1], lengths[:1], *c)
    assert all(torch.equal(a, b) and a.any() for a, b in zip(wide, near))


def test_one_key_rows_have_no_score_gradient():
    """Where every row sees one key, the weights are one and dq, dk and the table's gradient exactly zero."""
    from deepfold_amd import flash_window_attn

    for dtype in (BF, F32):
        for N, window in ((1, 9), (200, 1)):
            x = [leaf(rnd(2, 4, N, 64, seed=s, dtype=dtype)) for s in (1, 2, 3)]
            t = leaf(rnd(4, len(EDGES) + 1, seed=5))
            o = flash_window_attn(*x, window=window, rel_table=t, rel_edges=EDGES)
            # the weight and its sum are one number near 1: bf16 weights are rounded to 1, fp32 keeps the roundings
            # of their product and quotient
            assert ((o - x[2]).abs() <= (0 if dtype == BF else 4 * ref.U32) * x[2].abs()).all()
            dq, dk, dv, dt = torch.autograd.grad(o, [*x, t], torch.ones_like(o) * 0.37)
            assert not dq.any() and not dk.any() and not dt.any()


@pytest.mark.parametrize("low", [-math.inf, torch.finfo(F32).min, -1e9])
def test_table_entries_that_mask(low):
    """An entry of -inf or the type's lowest takes its keys out, also where it leaves a row empty; -1e9 only outweighs."""
    from deepfold_amd import flash_window_attn

    H, N, d, edges = 2, 140, 32, (1, 2, 4)
    x = [rnd(1, H, N, d, seed=s) for s in (1, 2, 3)]
    go = rnd(1, H, N, d, seed=4)
    table = rnd(H, 4, seed=5)
    table[0, 0] = low  # a query's own key
    table[1, 1:] = low
    want = ref.attention(*x, window=50, table=table, edges=edges, grad=go)
    y = [leaf(t) for t in (*x, table)]
    o = flash_window_attn(*y[:3], window=50, rel_table=y[3], rel_edges=edges)
    g = torch.autograd.grad(o, y, go.to(DEV))
    if low == -1e9:  # scores of 1e9 beside ones of order 1 keep no digits: the rows with another key must still be right
        want_o, bound = want["o"][0], 1e-4 * torch.ones(())
        assert ((o.double().cpu() - want_o).abs()[:, 1] <= bound).all() and torch.isfinite(o).all()
        return
    assert not o[0, 0, 0].any()  # row 0 of head 0 sees nothing else
    holds("o", o, *want["o"])
    for name, a in zip(("dq", "dk", "dv", "dtable"), g):
        holds(name, a, *want[name])


def test_strides_and_alignment():
    """Views (projections' heads, a batch expanded, rows one element off alignment) give what copies give."""
    from deepfold_amd import flash_window_attn

    for dtype in (BF, F32):
        B, H, Hk, N, d = 2, 4, 2, 100, 32
        q = rnd(B, N, H, d, seed=1, dtype=dtype).to(DEV).transpose(1, 2)
        kv = rnd(B, N, 2, Hk, d, seed=2, dtype=dtype).to(DEV)
        k, v = kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
        kw = dict(window=20, n_sink=3)
        want = flash_window_attn(q.contiguous(), k.contiguous(), v.contiguous(), **kw)
        assert torch.equal(flash_window_attn(q, k, v, **kw), want)
        off = torch.empty(k.numel() + 1, dtype=dtype, device=DEV)[1:].view(k.shape).copy_(k)
        assert torch.equal(flash_window_attn(q, off, v, **kw), want)
        one = flash_window_attn(q, k[:1].expand(B, Hk, N, d), v[:1].expand(B, Hk, N, d), **kw)
        assert torch.equal(one[0], want[0])
        leaves = [t.detach().requires_grad_(True) for t in (q, off, v)]
        go = rnd(B, N, H, d, seed=3, dtype=dtype).to(DEV).transpose(1, 2)
        got = torch.autograd.grad(flash_window_attn(*leaves, **kw), leaves, go)
        same = [t.detach().contiguous().requires_grad_(True) for t in (q, k, v)]
        ref_g = torch.autograd.grad(flash_window_attn(*same, **kw), same, go.contiguous())
        assert all(torch.equal(a, b) for a, b in zip(got, ref_g))
        # a key shared by the whole batch gets the sum over it, through the expansion's own gradient
        shared = k[:1].detach().clone().requires_grad_(True)
        g1 = torch.autograd.grad(flash_window_attn(q, shared.expand(B, Hk, N, d), v, **kw), shared, go)[0]
        full = shared.detach().expand(B, Hk, N, d).contiguous().requires_grad_(True)
        g2 = torch.autograd.grad(flash_window_attn(q, full, v, **kw), full, go)[0]
        assert torch.equal(g1, g2.sum(0, keepdim=True))


def test_other_types_and_unbatched():
    from deepfold_amd import flash_window_attn

    q, k, v = rnd(4, 50, 32, seed=1), rnd(2, 50, 32, seed=2), rnd(2, 50, 32, seed=3)
    want = flash_window_attn(q.to(DEV), k.to(DEV), v.to(DEV), window=9)
    assert want.shape == (4, 50, 32)
    h = flash_window_attn(q.to(DEV).half(), k.to(DEV).half(), v.to(DEV).half(), window=9)
    assert h.dtype == torch.float16 and (h.float() - want).abs().max() < 0.02
    d = [t.to(DEV).double().requires_grad_(True) for t in (q, k, v)]
    o = flash_window_attn(*d, torch.ones(50, device=DEV, dtype=torch.bool), window=9)
    assert o.dtype == torch.float64 and torch.equal(o.float(), want)
    assert all(g.dtype == torch.float64 for g in torch.autograd.grad(o.sum(), d))
    assert flash_window_attn(*d[:2], d[2].detach(), window=9).requires_grad


# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("both", [True, False])
@pytest.mark.parametrize("H,M,N,edges", [(1, 1, 1, (1,)), (3, 7, 9, EDGES), (4, 65, 64, EDGES), (2, 1, 700, (2, 300, 2048)),
                                         (70, 33, 31, (5,)), (2, 301, 123, tuple(range(1, 48))), (5, 200, 400, EDGES)])
def test_rel_pos_bias(H, M, N, edges, both, dtype):
    from deepfold_amd import rel_pos_bias

    n = (len(edges) + 1) * (2 if both else 1)
    table = rnd(H, n, seed=1)
    rel = torch.arange(N)[None, :] - torch.arange(M)[:, None] - (N - M)
    leaf_t = leaf(table)
    out = rel_pos_bias(leaf_t, edges, M, N, bidirectional=both, dtype=dtype)
    assert torch.equal(out.cpu(), ref.rel_bias(table, edges, rel, both).to(dtype))
    go = rnd(H, M, N, seed=2, dtype=dtype)
    g = torch.autograd.grad(out, leaf_t, go.to(DEV))[0]
    want, size = ref.rel_bias_grad(go[None], edges, rel[None], both, n)
    # a thread's column, the 256 columns and the parts: chains of at most 512 terms each
    holds("dtable", g, want, 1600 * ref.U32 * size + 1e-30)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_rel_pos_bias_of_positions(dtype):
    from deepfold_amd import rel_pos_bias

    B, H, M, N = 3, 4, 50, 77
    g = torch.Generator().manual_seed(4)
    qp = torch.randint(-40, 40, (B, M), generator=g, dtype=torch.int32)
    kp = torch.randint(-40, 40, (B, N), generator=g, dtype=torch.int64)
    qp[0, 0], kp[0, 0], qp[0, 1], kp[0, 1] = 2**31 - 1, -2**31, -2**31, 2**31 - 1  # differences of 33 bits
    table = rnd(H, 2 * (len(EDGES) + 1), seed=1, dtype=dtype)
    rel = kp.long()[:, None, :] - qp.long()[:, :, None]
    t = leaf(table)
    out = rel_pos_bias(t, EDGES, M, N, q_pos=qp.to(DEV), k_pos=kp.to(DEV))
    assert out.dtype == dtype and torch.equal(out.cpu(), ref.rel_bias(table, EDGES, rel, True).to(dtype))
    go = rnd(B, H, M, N, seed=2, dtype=dtype)
    want, size = ref.rel_bias_grad(go, EDGES, rel, True, table.shape[1])
    grad = torch.autograd.grad(out, t, go.to(DEV))[0]
    assert grad.dtype == dtype
    holds("dtable", grad, want, 1600 * ref.U32 * size + ref.half_step(dtype) * want.abs() + 1e-30)
    one = rel_pos_bias(t, EDGES, M, N, q_pos=qp[1].to(DEV), k_pos=kp[1].to(DEV))
    assert one.shape == (H, M, N) and torch.equal(one, out[1])
    own = rel_pos_bias(t, EDGES, M, q_pos=qp.to(DEV))
    assert torch.equal(own.cpu(), ref.rel_bias(table, EDGES, qp.long()[:, None, :] - qp.long()[:, :, None], True).to(dtype))


def test_bias_feeds_the_diffusion_attention():
    """rel_pos_bias into flash_diffusion_attn's pair bias is the window attention whose window reaches everything."""
    from deepfold_amd import flash_diffusion_attn, flash_window_attn, rel_pos_bias

    H, N, d = 4, 150, 32
    q, k, v, go = (rnd(1, H, N, d, seed=s) for s in (1, 2, 3, 4))
    table = rnd(H, 2 * (len(EDGES) + 1), seed=5)
    want = ref.attention(q, k, v, window=N, causal=False, table=table, edges=EDGES, grad=go)
    for way in (0, 1):
        x = [leaf(t) for t in (q, k, v, table)]
        if way:
            o = flash_window_attn(*x[:3], window=N, causal=False, rel_table=x[3], rel_edges=EDGES)
        else:
            o = flash_diffusion_attn(*x[:3], None, None, pair_bias=rel_pos_bias(x[3], EDGES, N).unsqueeze(0))
        grads = torch.autograd.grad(o, x, go.to(DEV))
        for name, g in zip(("o", "dq", "dk", "dv", "dtable"), (o, *grads)):
            scale = float(want[name][0].abs().max())
            # the diffusion attention's own bar
            assert float((g.detach().double().cpu() - want[name][0]).abs().max()) <= 1e-4 * scale, (way, name)


# ---------------------------------------------------------------------------
def caches(B, Hk, S, d, dtype, seed, layout):
    """Cache pairs with marked values, as (B,Hk,S,d) or as views of a (B,S,2,Hk,d) buffer, one element off if odd."""
    if layout == "own":
        return rnd(B, Hk, S, d, seed=seed, dtype=dtype).to(DEV), rnd(B, Hk, S, d, seed=seed + 1, dtype=dtype).to(DEV)
    n = B * S * 2 * Hk * d
    buf = torch.empty(n + 1, dtype=dtype, device=DEV)[1:].view(B, S, 2, Hk, d)
    buf.copy_(rnd(B, S, 2, Hk, d, seed=seed, dtype=dtype))
    return buf[:, :, 0].transpose(1, 2), buf[:, :, 1].transpose(1, 2)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("layout", ["own", "shared"])
@pytest.mark.parametrize("Hk,N,d,window,n_sink", [(2, 1, 8, 1, 0), (2, 50, 64, 7, 3), (3, 40, 24, 64, 4), (1, 300, 128, 130, 0),
                                                  (2, 33, 5, 16, 40)])
def test_cache_fill(Hk, N, d, window, n_sink, layout, dtype):
    from deepfold_amd import window_cache_fill

    lengths = torch.tensor([N, 0, 1, max(1, N - 5), N + 7, -3], dtype=torch.int64)
    B = len(lengths)
    k, v = (rnd(B, N, Hk, d, seed=s, dtype=dtype).transpose(1, 2) for s in (1, 2))
    kc, vc = caches(B, Hk, n_sink + window, d, dtype, 3, layout)
    want = ref.fill(k, v, lengths, kc.cpu(), vc.cpu(), n_sink)
    before = kc._version
    window_cache_fill(k.to(DEV), v.to(DEV), lengths.to(DEV), kc, vc, n_sink=n_sink)
    assert torch.equal(kc.cpu(), want[0]) and torch.equal(vc.cpu(), want[1])
    assert kc._version > before


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("layout", ["own", "shared"])
@pytest.mark.parametrize("H,Hk,d,window,n_sink,rel", [(2, 2, 32, 1, 0, True), (4, 2, 64, 60, 4, False), (3, 1, 24, 200, 1, True),
                                                      (8, 1, 128, 300, 0, True), (10, 2, 80, 65, 70, False),
                                                      (1, 1, 1, 5, 2, True), (16, 1, 64, 1100, 4, True)])
def test_decode(H, Hk, d, window, n_sink, rel, layout, dtype):
    from deepfold_amd import window_decode_attn

    S = n_sink + window
    lengths = torch.tensor([0, S, -1, S - 1, S // 2, 3 * S + 5, 2**31 - 1 - S, 1], dtype=torch.int64)
    if window == 1:  # position 2^31 - 1 - S: the oracle walks back over 4 S positions only
        lengths[6] = 10**9
    B = len(lengths)
    q, k, v = rnd(B, H, d, seed=1, dtype=dtype), rnd(B, Hk, d, seed=2, dtype=dtype), rnd(B, Hk, d, seed=3, dtype=dtype)
    kc, vc = caches(B, Hk, S, d, dtype, 4, layout)
    table = rnd(H, len(EDGES) + 1, seed=6) if rel else None
    want, bound, kw, vw = ref.decode(q, k, v, kc.cpu(), vc.cpu(), lengths, n_sink, table=table, edges=EDGES, operand=dtype,
                                     result=dtype)
    o = window_decode_attn(q.to(DEV), k.to(DEV), v.to(DEV), kc, vc, lengths.to(DEV), n_sink=n_sink,
                           rel_table=None if table is None else table.to(DEV), rel_edges=EDGES if rel else None)
    assert torch.equal(kc.cpu(), kw) and torch.equal(vc.cpu(), vw)
    assert not o[2].any()
    holds("o", o, want, bound)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_prompt_then_tokens(dtype):
    """A run as a user makes it: prompts of different lengths through the attention, into the caches, then token by token;
    every token's output is the row of the attention over the whole sequence."""
    from deepfold_amd import flash_window_attn, window_cache_fill, window_decode_attn

    B, H, Hk, N, d, window, n_sink = 3, 8, 2, 90, 64, 33, 4
    q, k, v = rnd(B, H, N, d, seed=1, dtype=dtype), rnd(B, Hk, N, d, seed=2, dtype=dtype), rnd(B, Hk, N, d, seed=3, dtype=dtype)
    table = rnd(H, len(EDGES) + 1, seed=4)
    want = ref.attention(q, k, v, window=window, n_sink=n_sink, table=table, edges=EDGES, operand=dtype, result=dtype)["o"]
    q, k, v, table = (t.to(DEV) for t in (q, k, v, table))
    kw = dict(n_sink=n_sink, rel_table=table, rel_edges=EDGES)
    start = [5, 60, 1]
    lengths = torch.tensor(start, dtype=torch.int32, device=DEV)
    mask = (torch.arange(N, device=DEV)[None] < lengths[:, None]).float()
    prompt = flash_window_attn(q, k, v, mask, window=window, **kw)
    kc, vc = (torch.full((B, Hk, n_sink + window, d), math.nan, dtype=dtype, device=DEV) for _ in range(2))
    window_cache_fill(k, v, lengths, kc, vc, n_sink=n_sink)
    rows = torch.arange(B, device=DEV)
    got = prompt.clone()
    for _ in range(30):
        at = lengths.long()
        o = window_decode_attn(q[rows, :, at], k[rows, :, at], v[rows, :, at], kc, vc, lengths, **kw)
        got[rows, :, at] = o
        lengths += 1
    for b, s in enumerate(start):
        holds("o", got[b, :, :s + 30], want[0][b, :, :s + 30], want[1][b, :, :s + 30])


def test_graph_replays():
    """A training step and a decoding step captured and replayed with eager work between the replays."""
    from deepfold_amd import flash_window_attn, rel_pos_bias, window_decode_attn

    B, H, Hk, N, d, window, n_sink = 1, 4, 2, 300, 64, 50, 3
    x = [rnd(B, h, N, d, seed=s, dtype=BF).to(DEV) for s, h in ((1, H), (2, Hk), (3, Hk))]
    table, go = rnd(H, 2 * (len(EDGES) + 1), seed=4).to(DEV), rnd(B, H, N, d, seed=5, dtype=BF).to(DEV)
    kc, vc = (torch.zeros(2, Hk, n_sink + window, d, dtype=BF, device=DEV) for _ in range(2))
    tok = [rnd(2, h, d, seed=s, dtype=BF).to(DEV) for s, h in ((6, H), (7, Hk), (8, Hk))]
    lengths = torch.tensor([0, 7], dtype=torch.int32, device=DEV)

    def train():
        y = [t.detach().requires_grad_(True) for t in (*x, table)]
        bias = rel_pos_bias(y[3], EDGES, N)
        o = flash_window_attn(*y[:3], window=window, n_sink=n_sink, causal=False, rel_table=y[3], rel_edges=EDGES)
        return [o, bias, *torch.autograd.grad((o, bias), y, (go, bias.detach()))]

    def decode():
        o = window_decode_attn(*tok, kc, vc, lengths, n_sink=n_sink)
        lengths.add_(1)
        return [o]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        train(), decode()
    s.synchronize()
    kc.zero_(), vc.zero_()
    lengths.copy_(torch.tensor([0, 7]))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        out = train() + decode()
    kc2, vc2, len2 = kc.clone(), vc.clone(), lengths.clone()
    for step in range(4):
        for t in (*x, go, *tok):
            t.copy_(torch.randn(t.shape, generator=torch.Generator().manual_seed(50 + step)).to(BF))
        g.replay()
        got = [t.clone() for t in out]
        torch.cuda.synchronize()
        want = train()
        want.append(window_decode_attn(*tok, kc2, vc2, len2, n_sink=n_sink))
        len2 += 1
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        assert torch.equal(kc, kc2) and torch.equal(lengths, len2)


def test_two_streams_at_once():
    """Calls in flight on two streams share nothing."""
    from deepfold_amd import flash_window_attn, window_decode_attn

    B, H, N, d = 2, 8, 700, 64
    sets = [[rnd(B, H, N, d, seed=10 * i + s, dtype=BF).to(DEV) for s in (1, 2, 3)] for i in range(2)]
    kc = [[rnd(B, H, 600, d, seed=40 + 2 * i + j, dtype=BF).to(DEV) for j in range(2)] for i in range(2)]
    at = torch.tensor([5000, 400], device=DEV, dtype=torch.int32)

    def step(i):
        y = [t.detach().requires_grad_(True) for t in sets[i]]
        o = flash_window_attn(*y, window=90, n_sink=4)
        dec = window_decode_attn(*(t[:, :, 0] for t in sets[i]), *kc[i], at, n_sink=4)
        return [o, dec, *torch.autograd.grad(o, y, torch.ones_like(o))]

    want = [[t.clone() for t in step(i)] for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        got = [None, None]
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = step(i)
        torch.cuda.synchronize()
        for i in range(2):
            assert all(torch.equal(a, b) for a, b in zip(got[i], want[i]))
