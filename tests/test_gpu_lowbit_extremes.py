"""One token's attention over a few-bit cache at the ends of its range, against the float64 form (oracle/lowbit.py) and its
elementwise bound."""

import pytest
import torch

from oracle import lowbit as ref
from test_gpu_lowbit import BF, DEV, F32, holds, onto, rnd

pytestmark = pytest.mark.gpu


def cache_of(x, bits):
    """A cache on the CPU that holds rows x (B,Hk,S,d)."""
    from deepfold_amd import QuantizedCache

    code, e = ref.encode(x, bits)
    exps = torch.zeros(*e.shape[:2], e.shape[3], -(-x.shape[2] // 4) * 4, dtype=torch.uint8)
    exps[..., :x.shape[2]] = e.transpose(-1, -2)
    return QuantizedCache(code, exps, bits)


def check(q, k, v, keys, values, bits, lengths, n_sink=0, scale=None, table=None, edges=None):
    from deepfold_amd import window_decode_attn

    kc, vc = cache_of(keys, bits), cache_of(values, bits)
    lengths = torch.tensor(lengths)
    want, bound, _, _ = ref.decode(q, k, v, kc, vc, lengths, n_sink, scale=scale, table=table, edges=edges, result=q.dtype)
    o = window_decode_attn(q.to(DEV), k.to(DEV), v.to(DEV), onto(kc), onto(vc), lengths.to(DEV), n_sink=n_sink, scale=scale,
                           rel_table=None if table is None else table.to(DEV), rel_edges=edges)
    assert bool(torch.isfinite(o).all())
    holds("o", o, want, bound)
    return o


def token(B, H, Hk, d, seed, dtype):
    return [rnd(B, h, d, seed=seed + i, dtype=dtype) for i, h in enumerate((H, Hk, Hk))]


BIG = 3.3e38


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("B,H,Hk,d,S", [(1, 4, 1, 64, 100), (2, 2, 2, 32, 3), (1, 16, 1, 128, 1500), (1, 1, 1, 24, 2600), (70, 4, 4, 40, 40)])
def test_values_at_the_end_of_the_range(B, H, Hk, d, S, bits, dtype):
    """Sums of values near 2^128 pass fp32 long before they are divided by the weights' sum."""
    q, k, v = token(B, H, Hk, d, 1, dtype)
    keys, values = rnd(B, Hk, S, d, seed=4), rnd(B, Hk, S, d, seed=5).clamp(-1, 1) * BIG
    lengths = [(3 * S + 7 * b) if b % 3 else S // 2 for b in range(B)]
    check(q, k, v.clamp(-1, 1) * BIG, keys, values, bits, lengths)
    # of one sign, every weight alike: the largest number itself
    top = torch.full((B, Hk, S, d), BIG)
    o = check(torch.zeros_like(q), k, top[:, :, 0].to(dtype), keys, top, bits, lengths)
    assert bool((o > 2.5e38).all())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("bits", [4, 8])
def test_large_values_beside_ordinary_ones(bits, dtype):
    """Large values in some groups, in some slots, of some samples: what does not meet them is as exact as ever."""
    B, H, Hk, d, S = 3, 8, 2, 128, 700
    q, k, v = token(B, H, Hk, d, 1, dtype)
    keys, values = rnd(B, Hk, S, d, seed=4), rnd(B, Hk, S, d, seed=5)
    values[0, :, :, 32:64] *= 2.0**120  # a group of all slots
    values[1, 1, 333] = BIG  # one slot
    keys[1, 1, 333] = 0
    values[2, 0, 500:] *= 2.0**124
    check(q, k, v, keys, values, bits, [5 * S, 3000, 650])
    # the large slot hardly counts: e^-60 and less of the weights
    keys[1, 1] = q[1, 4].float() * 2
    keys[1, 1, 333] = -q[1, 4].float() * 2
    check(q, k, v, keys, values, bits, [5 * S, 3000, 650], scale=0.25)


@pytest.mark.parametrize("S", [1, 2, 31, 64, 1000, 5000])
def test_values_around_the_border(S):
    """Every power of two around the one from which sums are formed otherwise."""
    for bits in (4, 8):
        for power in (*range(88, 120, 3), 127):
            q, k, v = token(1, 4, 1, 32, power, F32)
            keys, values = rnd(1, 1, S, 32, seed=power), rnd(1, 1, S, 32, seed=power + 1).clamp(-1, 1) * 2.0**power
            check(q, k, v.clamp(-1, 1) * 2.0**power, keys, values, bits, [2 * S])


def test_large_values_with_a_table():
    B, H, Hk, d, S = 2, 6, 2, 64, 400
    for dtype in (BF, F32):
        q, k, v = token(B, H, Hk, d, 1, dtype)
        table = rnd(H, 5, seed=9) * 3
        table[2, 1] = -float("inf")
        values = rnd(B, Hk, S, d, seed=5).clamp(-1, 1) * BIG
        check(q, k, v.clamp(-1, 1) * BIG, rnd(B, Hk, S, d, seed=4), values, 8, [399, 1000], n_sink=3, table=table, edges=(1, 7, 32, 100))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("scale", [1.5, 4.0, 2.0**20, 1e30])
def test_queries_times_a_large_scale(scale, bits, dtype):
    """Scores within reach whose queries, times the scale, are not."""
    B, H, Hk, d, S = 2, 4, 1, 64, 100
    q, k, v = token(B, H, Hk, d, 1, dtype)
    keys, values = rnd(B, Hk, S, d, seed=4), rnd(B, Hk, S, d, seed=5)
    small = 2.0**-126  # of the keys; queries as large as bf16 and fp32 have them, if the scale lets the scores stay below 100
    size = min(3.3e38, 2.0**126 / scale)
    check(q.clamp(-1, 1) * size, k * small, v, keys * small, values, bits, [70, 1000], scale=scale)
    check(q.clamp(-1, 1) * 2.0**60, k / 2.0**60 / scale, v, keys / 2.0**60 / scale, values, bits, [70, 1000], scale=scale)


@pytest.mark.parametrize("bits", [4, 8])
def test_the_largest_finite_query(bits):
    """A query's largest element at the end of fp32, its head held to the bound of the others."""
    H, d, S = 4, 32, 60
    q, k, v = token(1, H, 1, d, 1, F32)
    q[0, 1] = 0
    q[0, 1, 0] = torch.finfo(F32).max
    q[0, 2] = -torch.finfo(F32).max
    check(q, k, v, rnd(1, 1, S, d, seed=4), rnd(1, 1, S, d, seed=5), bits, [40], scale=1e-30)
    check(q, k * 1e-38, v, rnd(1, 1, S, d, seed=4) * 1e-38, rnd(1, 1, S, d, seed=5), bits, [40], scale=1.0)
    check(q, k * 1e-38, v, rnd(1, 1, S, d, seed=4) * 1e-38, rnd(1, 1, S, d, seed=5), bits, [40], scale=4.0)


@pytest.mark.parametrize("dtype,bits,d", [(BF, 4, 32), (F32, 8, 16)])
def test_one_head_in_many_splits(dtype, bits, d):
    """One key head of so many slots that its splits (250) pass the join's workgroup: all of them, some without a slot, one
    with a group that is no number."""
    from deepfold_amd import window_decode_attn
    from test_gpu_lowbit import cache

    S = 120000
    q, k, v = token(1, 1, 1, d, 1, dtype)
    kc, vc = (cache(1, 1, S, d, bits, s, odd=False) for s in (4, 5))
    q = q * 4  # (so that the splits' references differ)
    for n in (3 * S + 11, 100001, 62000, 477):
        lengths = torch.tensor([n])
        want, bound, _, _ = ref.decode(q, k, v, kc, vc, lengths, 0, result=dtype)
        o = window_decode_attn(q.to(DEV), k.to(DEV), v.to(DEV), onto(kc), onto(vc), lengths.to(DEV))
        holds(str(n), o, want, bound)
    vc.exponents[0, 0, 0, 100001] = 255
    for n, spoilt in ((100000, False), (100002, True)):
        o = window_decode_attn(q.to(DEV), k.to(DEV), v.to(DEV), onto(kc), onto(vc), torch.tensor([n], device=DEV))
        assert bool(o.isnan().all()) == spoilt and bool(o.isnan().any()) == spoilt
