"""Calls whose kernels have more threads than one launch's grid may (2^32 side by side), each held against calls of a few rows
of the same kind."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def memory_back():
    yield
    torch.cuda.empty_cache()


def rnd(*shape, seed, dtype=F32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def test_rows():
    """2^26 rows and more, a wave each: their codes, and the product that takes them."""
    from deepfold_amd import int8_linear, quantize_rows

    P, M, K, N = 4099, (1 << 26) + 70, 8, 3
    part = rnd(P, K, seed=1, dtype=BF).to(DEV)
    x = part.repeat(-(-M // P), 1)[:M]
    x[-1] = 0
    x[-1, 3] = 5.0
    codes, scale = quantize_rows(x)
    want, s = quantize_rows(part)
    at = torch.arange(M, device=DEV) % P
    at[-1] = 0
    same = (codes == want[at]).all(1) & (scale == s[at])
    assert bool(same[:-1].all()) and codes[-1].tolist() == [0, 0, 0, 127, 0, 0, 0, 0] and float(scale[-1]) == float(torch.tensor(5.0) / 127)
    del codes, scale, same
    w, ws = quantize_rows(rnd(N, K, seed=2).to(DEV))
    y, few = int8_linear(x, w, ws), int8_linear(part, w, ws)
    assert torch.equal(y[:-1], few[at[:-1]]) and torch.equal(y[-1:], int8_linear(x[-1:], w, ws))


def test_rows_of_weights():
    """2^27 rows of weights and more, a workgroup for 16."""
    from deepfold_amd import int8_linear

    P, N, K = 4099, (1 << 27) + 45, 16
    g = torch.Generator().manual_seed(1)
    part, ps = torch.randint(-127, 128, (P, K), generator=g).to(torch.int8).to(DEV), torch.rand(P, generator=g).to(DEV)
    reps = -(-N // P)
    codes, scale = part.repeat(reps, 1)[:N], ps.repeat(reps)[:N]
    at = torch.arange(N, device=DEV) % P
    for M in (1, 3):
        x = rnd(M, K, seed=M, dtype=BF).to(DEV)
        assert torch.equal(int8_linear(x, codes, scale), int8_linear(x, part, ps)[:, at])


def test_slots():
    """2^28 slots and more, a workgroup for 16: the window's whole range."""
    from deepfold_amd import quantized_cache, window_cache_fill

    d, n_sink, window, N = 128, 5, 1 << 28, 40
    k, v = rnd(1, 1, N, d, seed=1, dtype=BF).to(DEV), rnd(1, 1, N, d, seed=2, dtype=BF).to(DEV)
    small = [quantized_cache(1, 1, N, d, bits=4, device=DEV) for _ in range(2)]
    rows = torch.tensor([N], device=DEV)
    window_cache_fill(k, v, rows, *small)
    caches = [quantized_cache(1, 1, n_sink + window, d, bits=4, device=DEV) for _ in range(2)]
    start = n_sink + window - 17  # 17 rows in the last slots, the others in the first behind the first tokens
    window_cache_fill(k, v, rows, *caches, n_sink=n_sink, starts=torch.tensor([start], device=DEV))
    slot = torch.cat((torch.arange(start, n_sink + window), n_sink + torch.arange(N - 17))).to(DEV)
    for c, s in zip(caches, small):
        assert torch.equal(c.codes[0, 0, slot], s.codes[0, 0]) and torch.equal(c.exponents[0, 0][:, slot], s.exponents[0, 0][:, :N])
        c.codes[0, 0, slot] = 0
        assert not any(bool(part.any()) for part in c.codes.view(torch.int64).flatten().split(1 << 28))
