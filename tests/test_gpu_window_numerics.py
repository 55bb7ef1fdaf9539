"""The sequence operators on the GPU where their numbers are hard: lengths at the ends of their type, scores that grow
along the sequence, sharp and diffuse rows, long sums.  Bounds as in oracle/window.py."""

import math

import pytest
import torch

from oracle import window as ref
from test_gpu_window import BF, DEV, EDGES, F32, attention_case, holds, leaf, rnd

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, F32])
def test_lengths_at_the_ends_of_their_type(dtype):
    """Beyond N counts as N, below 1 leaves the caches alone, also where 32 bits end."""
    from deepfold_amd import window_cache_fill

    Hk, N, d, window, n_sink = 2, 30, 24, 9, 3
    lengths = torch.tensor([2**32 + 5, 2**31, 2**31 - 1, -2**31, -2**31 - 1, -2**40, 2**62, 4])
    B = len(lengths)
    k, v = rnd(B, Hk, N, d, seed=1, dtype=dtype), rnd(B, Hk, N, d, seed=2, dtype=dtype)
    kc, vc = rnd(B, Hk, n_sink + window, d, seed=3, dtype=dtype), rnd(B, Hk, n_sink + window, d, seed=4, dtype=dtype)
    want = ref.fill(k, v, lengths, kc, vc, n_sink)
    got = kc.to(DEV), vc.to(DEV)
    window_cache_fill(k.to(DEV), v.to(DEV), lengths.to(DEV), *got, n_sink=n_sink)
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])
    short = lengths.clamp(-2**31, 2**31 - 1).to(torch.int32).to(DEV)
    again = kc.to(DEV), vc.to(DEV)
    window_cache_fill(k.to(DEV), v.to(DEV), short, *again, n_sink=n_sink)
    assert torch.equal(again[0], got[0]) and torch.equal(again[1], got[1])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("causal", [True, False])
def test_table_gradient_over_many_tiles(causal, dtype):
    """A wave adds up the diagonals of many tiles in a row, each through the same columns of LDS: the table's gradient at
    every distance (a bucket for each of the first ones), and the same bits from call to call."""
    edges = (*range(1, 90), 400) if causal else (*range(1, 46), 700)
    case = dict(rel=True, edges=edges, seed=21)
    first = attention_case(1, 2, 2, 640, 640, 64, dtype, 640, 0, causal, **case)[1]
    for _ in range(3):
        again = attention_case(1, 2, 2, 640, 640, 64, dtype, 640, 0, causal, **case)[1]
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_bias_gradient_of_many_heads_and_a_large_plane():
    """Where the heads alone fill the card a plane is still cut up: at most 1024 additions a thread in fp32, 256 columns
    added up in a tree of 10, the parts in 64 bits.  Equal addends round the same way each time."""
    from deepfold_amd import rel_pos_bias

    H, M, N = 1024, 512, 2048
    table = torch.zeros(H, 2, device=DEV, requires_grad=True)
    out = rel_pos_bias(table, (700,), M, N, bidirectional=False)
    value = (torch.arange(H, dtype=F32) + 1.3) / 3
    g = torch.autograd.grad(out, table, value.to(DEV)[:, None, None].expand(H, M, N))[0]
    rel = torch.arange(N)[None, :] - torch.arange(M)[:, None] - (N - M)
    far = int((rel <= -700).sum())
    want = value.double()[:, None] * torch.tensor([M * N - far, far]).double()
    holds("dtable", g, want, (1024 + 10 + 1) * ref.U32 * want)


def hard_rows(kind, causal, dtype, d, N=700, H=2, Hk=1):
    """Rows whose outputs are large against their score gradients, among more than 256 keys each."""
    q, k, v = rnd(1, H, N, d, seed=1), rnd(1, Hk, N, d, seed=2), rnd(1, Hk, N, d, seed=3)
    mask = table = None
    if kind == "sharp":  # one key or a few take most of a row
        q = q * 6
    elif kind == "sharper":
        q = q * 14
    elif kind == "offset":  # values with a large common part: the softmax gradient cancels it
        v = v + 9
    elif kind == "masked":  # padding on the left and holes: few keys are left of a wide window
        mask = (torch.rand(1, N, generator=torch.Generator().manual_seed(5)) < 0.02).float()
        mask[0, -3:] = 1
    elif kind == "table":  # entries of -inf leave the three nearest keys (of either side)
        table = rnd(H, 4 * (1 if causal else 2), seed=6)
        table[:, 3::4] = -math.inf
    return [t.to(dtype) for t in (q, k, v)], mask, table


@pytest.mark.parametrize("d", [8, 16, 40, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("kind", ["sharp", "sharper", "offset", "masked", "table", "plain"])
def test_score_gradients_know_no_rounding_of_the_output(kind, causal, d):
    """bf16 rows that see more than 256 places: D is as good as the rounded probabilities, not as the rounded output."""
    (q, k, v), mask, table = hard_rows(kind, causal, BF, d)
    go = rnd(*q.shape, seed=4, dtype=BF)
    kw = dict(window=600, n_sink=3, causal=causal)
    want = ref.attention(q, k, v, mask=mask, table=table, edges=(1, 2, 3), grad=go, operand=BF, result=BF, remainder=True, **kw)
    from deepfold_amd import flash_window_attn

    x = [leaf(t) for t in (q, k, v, table)]
    o = flash_window_attn(*x[:3], None if mask is None else mask.to(DEV), rel_table=x[3],
                          rel_edges=None if table is None else (1, 2, 3), **kw)
    grads = torch.autograd.grad(o, [t for t in x if t is not None], go.to(DEV))
    for name, got in zip(("o", "dq", "dk", "dv", "dtable"), (o, *grads)):
        holds(f"{kind} {name}", got, *want[name])


@pytest.mark.parametrize("kind", ["sharp", "offset", "table"])
def test_backward_without_the_remainder(kind, monkeypatch):
    """A caller of the C entries that kept only o: the backward forms D from the products themselves."""
    from deepfold_amd import flash_window_attn, window_attn

    (q, k, v), mask, table = hard_rows(kind, True, BF, 16)
    go = rnd(*q.shape, seed=4, dtype=BF)
    kw = dict(window=600, n_sink=3)
    want = ref.attention(q, k, v, mask=mask, table=table, edges=(1, 2, 3), grad=go, operand=BF, result=BF, remainder=True, **kw)
    forward = window_attn._forward

    def dropped(*args):
        (*head, rest, lse), out = forward(*args)
        assert rest is not None
        return (*head, None, lse), out

    monkeypatch.setattr(window_attn, "_forward", dropped)
    x = [leaf(t) for t in (q, k, v, table)]
    o = flash_window_attn(*x[:3], rel_table=x[3], rel_edges=None if table is None else (1, 2, 3), **kw)
    grads = torch.autograd.grad(o, [t for t in x if t is not None], go.to(DEV))
    for name, got in zip(("o", "dq", "dk", "dv", "dtable"), (o, *grads)):
        holds(f"{kind} {name}", got, *want[name])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("N", [5, 100, 400])
def test_small_weights_beside_a_dominant_key(N, dtype):
    """One key outweighs the others by far more than fp32 holds beside 1 (e^-20 .. e^-30 each): the others' own gradients
    are small, not zero, in rows of few keys as in rows of many."""
    H, d = 2, 8
    q, k, v = rnd(1, H, N, d, seed=1), rnd(1, H, N, d, seed=2), rnd(1, H, N, d, seed=3)
    q[..., 0] = 8 + q[..., 0].abs()  # against key 0, the first token: scores of 22 and more
    k[:, :, 1:, 0] = 0
    k[:, :, 0, 0] = 8
    q, k, v, go = (t.to(dtype) for t in (q, k, v, rnd(1, H, N, d, seed=4)))
    want = ref.attention(q, k, v, window=N, n_sink=1, grad=go, operand=dtype, result=dtype, remainder=True)
    from deepfold_amd import flash_window_attn

    x = [leaf(t) for t in (q, k, v)]
    o = flash_window_attn(*x, window=N, n_sink=1)
    grads = torch.autograd.grad(o, x, go.to(DEV))
    for name, got in zip(("o", "dq", "dk", "dv"), (o, *grads)):
        holds(name, got, *want[name])
    assert grads[1][:, :, 1:].any()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("scale", [0.01, 0.6, 3.0])
def test_scales(scale, causal, dtype):
    """A scale of the caller's own, in short and long rows, forward and both passes of the backward."""
    attention_case(2, 4, 2, 130, 150, 24, dtype, 40, 3, causal, True, scale=scale)
    attention_case(1, 2, 1, 520, 520, 64, dtype, 400, 4, causal, True, scale=scale)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("growth", [3.0, 14.0, -14.0, 60.0])
def test_scores_that_grow_along_the_sequence(growth, causal, dtype):
    """Each 64 keys raise (or lower) the scores by ``growth`` in log2: the running reference moves up in steps of any size
    (8 and more rescale a row), or stays at the first keys."""
    from deepfold_amd import flash_window_attn

    B, H, Hk, N, d, scale = 1, 4, 2, 450, 16, 0.4
    q, k, v, go = (rnd(B, h, N, d, seed=s) for s, h in ((1, H), (2, Hk), (3, Hk), (4, H)))
    # column 0: q 1, k the wanted score / (scale log2 e)
    q[..., 0] = 1
    k[..., 0] = torch.arange(N) / 64 * growth / (scale * math.log2(math.e))
    q, k, v, go = (t.to(dtype) for t in (q, k, v, go))
    table = rnd(H, (len(EDGES) + 1) * (1 if causal else 2), seed=5)
    # A weight below 2^-126, fp32's smallest normal number, may be zero in the kernel (at a growth of 60 they go down to
    # 2^-420): each of the H / Hk N of a key's rows is then off by 2^-126 times at most |q|, |k| or |do| and |dp - D| <=
    # 2 max |do|.|v|, each taken as its largest, plus as much for the result itself.
    big = max(float(t.abs().max()) for t in (q, k, go)) * (1 + 2 * float(go.double().abs().sum(-1).max() * v.abs().max()))
    tiny = 2.0 ** -126 * (H // Hk * N * N + 1) * big
    for window, n_sink in ((450, 0), (200, 2)):
        kw = dict(window=window, n_sink=n_sink, causal=causal, scale=scale)
        want = ref.attention(q, k, v, table=table, edges=EDGES, grad=go, operand=dtype, result=dtype,
                             remainder=dtype == BF, **kw)
        x = [leaf(t) for t in (q, k, v, table)]
        o = flash_window_attn(*x[:3], rel_table=x[3], rel_edges=EDGES, **kw)
        grads = torch.autograd.grad(o, x, go.to(DEV))
        for name, got in zip(("o", "dq", "dk", "dv", "dtable"), (o, *grads)):
            holds(f"{name} window {window}", got, want[name][0], want[name][1] + tiny)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("scale,growth", [(0.02, 0.0), (2.0, 0.0), (0.5, 20.0), (0.5, -20.0)])
def test_decode_scales_and_growth(scale, growth, dtype):
    from deepfold_amd import window_decode_attn

    B, H, Hk, d, window, n_sink = 3, 8, 2, 48, 700, 2
    S = window + n_sink
    q, k, v = rnd(B, H, d, seed=1), rnd(B, Hk, d, seed=2), rnd(B, Hk, d, seed=3)
    kc, vc = rnd(B, Hk, S, d, seed=4), rnd(B, Hk, S, d, seed=5)
    q[..., 0] = 1
    if growth:
        kc[..., 0] = torch.arange(S) / 64 * growth / (scale * math.log2(math.e))
    lengths = torch.tensor([S - 1, 350, 5 * S])
    table = rnd(H, len(EDGES) + 1, seed=6)
    q, k, v, kc, vc = (t.to(dtype) for t in (q, k, v, kc, vc))
    want, bound, _, _ = ref.decode(q, k, v, kc, vc, lengths, n_sink, scale=scale, table=table, edges=EDGES, operand=dtype,
                                   result=dtype)
    o = window_decode_attn(*(t.to(DEV) for t in (q, k, v, kc, vc, lengths)), n_sink=n_sink, scale=scale,
                           rel_table=table.to(DEV), rel_edges=EDGES)
    holds("o", o, want, bound)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_gradients_beside_an_outweighing_table_entry(dtype):
    """Entries of -1e9, which keep no digits of the scores beside them: heads with other keys are right, all is finite."""
    from deepfold_amd import flash_window_attn

    H, N, d, edges = 2, 140, 32, (1, 2, 4)
    x = [rnd(1, H, N, d, seed=s, dtype=dtype) for s in (1, 2, 3)]
    go, table = rnd(1, H, N, d, seed=4, dtype=dtype), rnd(H, 4, seed=5)
    gone = table.clone()
    table[:, 2:], gone[:, 2:] = -1e9, -math.inf  # a key two or more away: the same weights of zero
    y = [leaf(t) for t in (*x, table)]
    o = flash_window_attn(*y[:3], window=50, rel_table=y[3], rel_edges=edges)
    got = (o, *torch.autograd.grad(o, y, go.to(DEV)))
    want = ref.attention(*x, window=50, table=gone, edges=edges, grad=go, operand=dtype, result=dtype)
    for name, t in zip(("o", "dq", "dk", "dv", "dtable"), got):
        holds(name, t, *want[name])


def test_graph_replays_of_wide_windows():
    """A training step whose rows see more than 256 keys, captured and replayed on new inputs with eager work between."""
    from deepfold_amd import flash_window_attn

    x = [rnd(1, h, 600, 64, seed=s, dtype=BF).to(DEV) for s, h in ((1, 4), (2, 2), (3, 2))]
    go = rnd(1, 4, 600, 64, seed=4, dtype=BF).to(DEV)

    def train():
        y = [t.detach().requires_grad_(True) for t in x]
        o = flash_window_attn(*y, window=400, n_sink=4)
        return [o, *torch.autograd.grad(o, y, go)]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        train()
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        out = train()
    for step in range(3):
        for t in (*x, go):
            t.copy_(torch.randn(t.shape, generator=torch.Generator().manual_seed(70 + step)).to(BF))
        g.replay()
        got = [t.clone() for t in out]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, train()))


@pytest.mark.parametrize("window,n_sink,causal,kept", [(252, 4, True, False), (253, 4, True, True), (126, 5, False, False),
                                                       (127, 4, False, True), (2000, 0, True, True)])
def test_the_remainder_is_kept_where_it_is_used(window, n_sink, causal, kept):
    from deepfold_amd import window_attn

    x = [rnd(1, 2, 400, 64, seed=s, dtype=BF).to(DEV) for s in (1, 2, 3)]
    for train in (True, False):
        saved, _ = window_attn._forward(*x, None, None, None, window, n_sink, causal, 0.1, train)
        assert (saved[6] is not None) == (kept and train)
    saved, _ = window_attn._forward(*(t.float() for t in x), None, None, None, window, n_sink, causal, 0.1, True)
    assert saved[6] is None
