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
