"""The float64 forms of the few-bit operators (oracle/lowbit.py) against other statements of the same: groups spelled out
element by element, the plain forms of the timed cases, a cache kept as a list of positions."""

import importlib.util
import os
import random

import pytest
import torch

from conftest import ROOT
from oracle import lowbit as ref
from oracle import window as plain_window

BF, F32 = torch.bfloat16, torch.float32


def rnd(*shape, seed, dtype=F32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def wide(*shape, seed, dtype=F32):
    """Numbers of any size, and some that do not count as such."""
    g = torch.Generator().manual_seed(seed)
    bits = torch.randint(-2**31, 2**31, shape, generator=g, dtype=torch.int64).to(torch.int32)
    return bits.view(F32).to(dtype)


@pytest.fixture(scope="module")
def plain():
    spec = importlib.util.spec_from_file_location("more_operators", os.path.join(ROOT, "perf", "more_operators.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_codes_element_by_element():
    """Each code is the nearest of all, each exponent the lowest that serves, by a walk over the groups in Python."""
    for bits in (4, 8):
        grid = [float(n) for n in range(128)] if bits == 8 else list(ref.E2M1)
        x = torch.cat((rnd(40, 32, seed=1), 2.0 ** torch.randint(-126, 120, (40, 1), generator=torch.Generator().manual_seed(2)) *
                       torch.randint(-64, 65, (40, 32), generator=torch.Generator().manual_seed(3)).float() / 4,
                       torch.tensor([[0.0] * 32, [-0.0] * 31 + [1e-45], [7.0] * 32, [127.5] + [63.5, 62.5] * 15 + [0.5],
                                     [3.4e38] * 32, [-1.75 * 2.0**127, 2.0**100] * 16])))
        code, e = ref.encode(x, bits)
        got = ref.values(code, e, 32, bits)
        for row, byte, back in zip(x.double().tolist(), e[:, 0].tolist(), got.tolist()):
            top, step = max(map(abs, row)), 2.0 ** (byte - 127)
            limit = lambda s: top < 127.5 * s if bits == 8 else top <= 7 * s  # noqa: E731
            assert limit(step) or byte == (248 if bits == 8 else 252)
            assert byte == 1 or not limit(step / 2)
            for a, b in zip(row, back):
                near = min(abs(abs(a) - c * step) for c in grid)
                assert abs(a - b) == near, (bits, a, b, step)
                n = [i for i, c in enumerate(grid) if abs(abs(a) - c * step) == near]
                assert len(n) == 1 or abs(b) == grid[[i for i in n if i % 2 == 0][0]] * step


def test_groups_that_are_no_numbers():
    for bits in (4, 8):
        x = torch.ones(3, 70)
        x[0, 3], x[1, 40], x[2, 69] = float("inf"), float("nan"), -float("inf")
        code, e = ref.encode(x, bits)
        assert (e == 255).tolist() == [[True, False, False], [False, True, False], [False, False, True]]
        got = ref.values(code, e, 70, bits)
        for i, (lo, hi) in enumerate(((0, 32), (32, 64), (64, 70))):
            assert got[i, lo:hi].isnan().all() and not got[i, :lo].isnan().any() and not got[i, hi:].isnan().any()
        assert not code[0, :4 * bits].any()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_plain_codes(plain, bits, dtype):
    """The timed cases' plain form makes the same codes, whatever the numbers, and reads them the same way."""
    for seed, make in enumerate((rnd, wide, rnd)):
        for d in (1, 24, 32, 80, 128):
            x = make(2, 3, 40, d, seed=10 * seed + d, dtype=dtype)
            code, e = plain._quantise(x, bits)
            want, we = ref.encode(x, bits)
            assert torch.equal(code, want) and torch.equal(e.transpose(-1, -2), we)
            back = plain._values(code, e, d)
            assert torch.equal(back.double().nan_to_num(nan=123.0), ref.values(want, we, d, bits).nan_to_num(nan=123.0))


def test_plain_rows():
    """quantize_rows' codes by rounded float64 quotients, where these cannot hit a tie by themselves."""
    x = torch.cat((rnd(50, 200, seed=1), rnd(50, 200, seed=2, dtype=BF).float(), wide(50, 200, seed=3)))
    x[5] = 0
    x[6] = torch.arange(200).float() - 73.5  # ties: a largest magnitude of 126.5
    x[7] = torch.arange(200).float() / 2 - 27.5  # (72)
    x[8, :] = 1e-40
    x[9, 0], x[10, 1] = float("inf"), float("nan")
    code, s = ref.rows(x)
    assert s[9].isnan() and s[10].isnan() and not code[9].any() and not code[10].any() and not code[8].any()
    assert s[5] == 2.0 ** -100
    fine = torch.isfinite(x).all(1)
    top = x[fine].double().abs().amax(1)
    assert torch.equal(s[fine], torch.clamp((top / 127).float(), min=2.0 ** -100))
    assert torch.equal(code[fine].double(), torch.round(x[fine].double() / s[fine].double()[:, None]))
    assert code.min() >= -127 and int(code[fine].abs().amax(1)[:5].min()) == 127


def test_cache_as_a_list_of_positions():
    """Fill in chunks, tokens and readings against a list that keeps every position's row."""
    rng = random.Random(3)
    for trial in range(12):
        bits, n_sink, window, d = rng.choice([4, 8]), rng.choice([0, 1, 3]), rng.choice([1, 2, 7]), rng.choice([8, 40])
        S = n_sink + window
        caches = [(torch.zeros(1, 1, S, ref.groups_of(d) * 4 * bits, dtype=torch.uint8),
                   torch.zeros(1, 1, ref.groups_of(d), 16, dtype=torch.uint8), bits) for _ in range(2)]
        every, n = [], 0
        for step in range(4):
            rows = rng.choice([1, 2, 5, 11])
            k, v = rnd(1, 1, rows, d, seed=100 * trial + step), rnd(1, 1, rows, d, seed=100 * trial + step + 50)
            caches = ref.fill(k, v, torch.tensor([rows]), torch.tensor([n]), *caches, n_sink)
            for i in range(rows):
                every.append([ref.values(*ref.encode(x[0, 0, i], bits), d, bits) for x in (k, v)])
            n += rows
            K, V, mask = ref.read(ref.cache_values(caches[0], d), ref.cache_values(caches[1], d), torch.tensor([n]), n_sink)
            for j in range(S):
                p = j if j < n_sink else n - S + j
                there = p < n and (j < n_sink or p >= n_sink)
                assert bool(mask[0, j]) == there
                want = every[p] if there else [torch.zeros(d)] * 2
                assert torch.equal(K[0, 0, j], want[0].double()) and torch.equal(V[0, 0, j], want[1].double())
            slots, pos = ref.held_slots(n - 1, S, n_sink)
            assert sorted(pos.tolist()) == [p for p in range(n) if p < n_sink or p >= n - window]
            assert all(s == ref.slot(int(p), n_sink, window) for s, p in zip(slots, pos))


def test_decode_reads_what_the_codes_stand_for():
    """The few-bit decode is the plain one over a cache of the codes' values."""
    B, H, Hk, d, n_sink, W = 3, 4, 2, 40, 2, 6
    S = n_sink + W
    lengths = torch.tensor([3, -1, 20])
    table, edges = rnd(H, 4, seed=9), (1, 2, 5)
    for bits in (4, 8):
        q, k, v = rnd(B, H, d, seed=1), rnd(B, Hk, d, seed=2), rnd(B, Hk, d, seed=3)
        caches = []
        for s in (4, 5):
            code, e = ref.encode(rnd(B, Hk, S, d, seed=s), bits)
            caches.append((code, e.transpose(-1, -2).contiguous(), bits))
        o, bound, kc, vc = ref.decode(q, k, v, *caches, lengths, n_sink, table=table, edges=edges)
        rows = [ref.cache_values(c, d) for c in caches]
        new = [ref.values(*ref.encode(x, bits), d, bits) for x in (k, v)]
        want, _, kw, vw = plain_window.decode(q, *new, *rows, lengths, n_sink, table=table, edges=edges)
        assert torch.allclose(o, want, atol=1e-12) and not o[1].any() and not bound[1].any()
        assert torch.equal(ref.cache_values(kc, d), kw) and torch.equal(ref.cache_values(vc, d), vw)
