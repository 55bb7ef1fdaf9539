"""Products in 8-bit integers on the GPU against their float64 forms (oracle/lowbit.py) on identical inputs: codes and scales
exactly, results to the bound of their few fp32 operations (the integer sums are exact)."""

import math

import pytest
import torch

from oracle import lowbit as ref

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF, F32 = torch.bfloat16, torch.float32


def rnd(*shape, seed, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def weights(N, K, seed):
    """Codes in padded rows whose padding holds anything, and scales."""
    g = torch.Generator().manual_seed(seed)
    whole = torch.randint(-127, 128, (N, -(-K // 16) * 16), generator=g).to(torch.int8)
    return whole[:, :K], torch.rand(N, generator=g) * 0.1 + 1e-3


def onto(codes):
    return torch.empty(0, dtype=codes.dtype).set_(codes.untyped_storage()).to(DEV).as_strided(codes.shape, codes.stride(),
                                                                                             codes.storage_offset())


def holds(got, want, bound):
    want = torch.where(want.to(got.dtype).isinf(), want.to(got.dtype).double(), want)  # beyond the type's range: infinite
    got = got.double().cpu()
    assert got.shape == want.shape and bool((got.isnan() == want.isnan()).all())
    off = torch.where(got == want, 0.0, (got - want).abs()).nan_to_num(nan=0.0)
    bad = ~(off <= bound.nan_to_num(nan=0.0))
    worst = float((off / bound.clamp(min=1e-30)).nan_to_num(nan=0.0).max())
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} off, the worst {worst:.2f} times the bound"


def case(M, K, N, dtype, bias=True, x=None, seed=1):
    from deepfold_amd import int8_linear

    x = rnd(M, K, seed=seed, dtype=dtype) if x is None else x
    codes, scale = weights(N, K, seed + 1)
    b = rnd(N, seed=seed + 2, dtype=dtype) if bias else None
    y = int8_linear(x.to(DEV), onto(codes), scale.to(DEV), None if b is None else b.to(DEV))
    assert y.dtype == dtype
    holds(y, *ref.linear(x, codes, scale, b, dtype))
    return y


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("M,K,N", [(1, 1, 1), (1, 64, 16), (2, 15, 17), (3, 16, 33), (15, 17, 1), (16, 63, 64), (17, 65, 100), (31, 127, 48),
                                   (32, 128, 15), (33, 200, 70), (48, 1000, 31), (64, 512, 129), (65, 48, 64), (65, 513, 200), (97, 512, 512),
                                   (128, 100, 65), (129, 64, 63), (200, 2100, 130), (1, 4097, 20), (5, 9000, 18), (70, 8200, 66),
                                   (5, 4096, 40), (8, 4095, 33), (7, 520, 300), (9, 4096, 17), (6, 100, 4097), (8, 64, 4096), (9, 2048, 50),
                                   (16, 2049, 33), (13, 2047, 4096), (16, 1000, 97), (33, 1024, 40), (17, 1025, 40), (100, 1023, 300),
                                   (2, 20, 12289), (24, 8, 12289), (700, 640, 200)])
def test_linear(M, K, N, dtype):
    case(M, K, N, dtype, bias=(M + K + N) % 2 == 0)


@pytest.mark.parametrize("M,K,N", [(500, 100, 450), (513, 2100, 449), (3100, 33, 60), (66, 700, 1600), (2048, 192, 2048),
                                   (2049, 80, 2177), (4096, 64, 4096), (4100, 130, 4099)])
def test_linear_large_tiles(M, K, N):
    """Products of enough tiles for the larger ones, whole and with ragged edges."""
    case(M, K, N, BF)
    case(M, K, N, F32, bias=False)


@pytest.mark.parametrize("M", [1, 40, 100])
def test_largest_sums(M):
    """131072 products of the largest codes, of one sign: the sum that 32 bits just hold."""
    from deepfold_amd import int8_linear

    K, N = 2**17, 3
    codes = torch.full((N, K), 127, dtype=torch.int8)
    codes[1] = -127
    codes[2, ::2] = -127
    x = torch.full((M, K), 2.0)
    scale = torch.ones(N)
    y = int8_linear(x.to(DEV), codes.to(DEV), scale.to(DEV))
    holds(y, *ref.linear(x, codes, scale, None, F32))
    assert not y[:, 2].any() and (y[:, 0] > 2.6e7).all()


@pytest.mark.parametrize("M,N", [(385, 449), (2048, 2048)])
def test_largest_sums_in_tiles(M, N):
    from deepfold_amd import int8_linear

    K = 2**17 if M < 2048 else 2**12
    codes = torch.full((N, K), 127, dtype=torch.int8, device=DEV)
    codes[1::2] = -127
    y = int8_linear(torch.full((M, K), 2.0, dtype=BF, device=DEV), codes, torch.ones(N, device=DEV))
    want = torch.full((M, N), 127.0 * 127 * K * float(torch.tensor(2.0 / 127)), dtype=torch.float64)
    want[:, 1::2] *= -1
    holds(y, want, want.abs() * (2.0**-9 + 2.0**-20))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("M", [4, 40, 90])
def test_rows_of_every_kind(M, dtype):
    """Zeros, ties, tiny and huge rows, rows that are no numbers: each row's result is its own affair."""
    K = 70
    x = rnd(M, K, seed=1)
    x[0] = 0
    x[1] = torch.arange(K).float() * 2 - 69
    x[1, -1] = 127  # steps of 1: every other element is a whole code
    x[2] = (torch.arange(K).float() - 35) * 2 + 0.5
    x[2, 0] = 127  # (ties)
    x[3] = torch.finfo(F32).max / 2
    for i, make in enumerate((lambda r: r * 1e-38, lambda r: r * 1e30, lambda r: r.index_fill(0, torch.tensor([5]), math.inf),
                              lambda r: r.index_fill(0, torch.tensor([69]), math.nan), lambda r: r * 1e-42)):
        if 4 + i < M:
            x[4 + i] = make(x[4 + i])
    y = case(M, K, 35, dtype, x=x.to(dtype))
    if M > 8:
        assert y[6].isnan().all() and y[7].isnan().all()
        assert not y[torch.arange(M) != 6][:6].isnan().any()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("M,K", [(1, 1), (3, 7), (5, 16), (40, 100), (7, 2048), (9, 2049), (3, 8192), (4, 8200), (2, 131072), (700, 64)])
def test_quantize_rows(M, K, dtype):
    from deepfold_amd import quantize_rows

    g = torch.Generator().manual_seed(M + K)
    x = torch.randint(-2**31, 2**31, (M, K), generator=g).to(torch.int32).view(F32).to(dtype)  # any bits at all
    x[::2] = rnd(M, K, seed=2, dtype=dtype)[::2]
    if K > 100:
        x[0] = (torch.randint(-253, 254, (K,), generator=g).float() / 2).to(dtype)  # ties, if the largest is 127
        x[0, 9] = 127
    codes, scale = quantize_rows(x.to(DEV))
    want, s = ref.rows(x)
    assert codes.shape == (M, K) and codes.dtype == torch.int8 and codes.stride(0) == -(-K // 16) * 16
    assert torch.equal(scale.cpu().nan_to_num(nan=-1.0), s.nan_to_num(nan=-1.0))
    assert torch.equal(codes.cpu(), want)
    whole = torch.empty(0, dtype=torch.int8, device=DEV).set_(codes.untyped_storage()).view(M, -1)
    assert not whole[:, K:].any()


@pytest.mark.parametrize("M", [3, 90])
def test_strides_and_shapes(M):
    from deepfold_amd import int8_linear, quantize_rows

    w = rnd(24, 50, seed=1).to(DEV)
    codes, scale = quantize_rows(w.t().contiguous().t())
    x = rnd(M, 2, 50, seed=2, dtype=BF).to(DEV)
    want = int8_linear(x.reshape(-1, 50).contiguous(), codes, scale)
    assert torch.equal(int8_linear(x, codes, scale), want.view(M, 2, 24))
    assert torch.equal(int8_linear(x[:, 1], codes, scale), want.view(M, 2, 24)[:, 1])
    wide = torch.zeros(M, 2, 61, dtype=BF, device=DEV)
    wide[..., 7:57] = x
    assert torch.equal(int8_linear(wide[..., 7:57], codes, scale), want.view(M, 2, 24))
    assert torch.equal(int8_linear(x[:, 0].t().contiguous().t(), codes, scale), want.view(M, 2, 24)[:, 0])
    assert torch.equal(int8_linear(x[0, 0], codes, scale), want[0])
    assert torch.equal(int8_linear(x[:1, :1].expand(M, 2, 50), codes, scale), want[:1].expand(2 * M, 24).reshape(M, 2, 24))
    assert torch.equal(int8_linear(x, codes[4:20], scale[4:20]), want.view(M, 2, 24)[..., 4:20])


def test_graph_replays_and_streams():
    from deepfold_amd import int8_linear, quantize_rows

    w, x = rnd(300, 256, seed=1).to(DEV), [rnd(m, 256, seed=m, dtype=BF).to(DEV) for m in (1, 30, 200)]
    bias = rnd(300, seed=3, dtype=BF).to(DEV)

    def step():
        codes, scale = quantize_rows(w)
        return [int8_linear(t, codes, scale, bias) for t in x]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        out = step()
    for turn in range(4):
        for t in (w, *x):
            t.copy_(torch.randn(t.shape, generator=torch.Generator().manual_seed(50 + turn)).to(t.dtype))
        g.replay()
        got = [t.clone() for t in out]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))
    codes, scale = quantize_rows(w)
    want = [int8_linear(t, codes, scale) for t in x]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(4):
        got = []
        for t, st in zip(x, streams):
            with torch.cuda.stream(st):
                got.append(int8_linear(t, codes, scale))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_a_layer_in_few_bits(dtype, bits):
    """One token through a served layer: its projection in 8-bit integers, its cache in few bits, the attention over it, the
    projection back; each step against the float64 form of the same step on the step's own inputs."""
    from deepfold_amd import int8_linear, quantize_rows, quantized_cache, window_cache_fill, window_decode_attn
    from oracle.lowbit import decode

    B, C, H, Hk, d, window, n_sink, prompt = 3, 192, 6, 2, 32, 20, 2, 30
    w_in, w_out = rnd((H + 2 * Hk) * d, C, seed=1, scale=C ** -0.5), rnd(C, H * d, seed=2, scale=(H * d) ** -0.5)
    (ci, si), (co, so) = quantize_rows(w_in.to(DEV)), quantize_rows(w_out.to(DEV))
    kc, vc = (quantized_cache(B, Hk, n_sink + window, d, bits=bits, device=DEV) for _ in range(2))
    lengths = torch.tensor([prompt, 7, 0], dtype=torch.int32, device=DEV)
    x = rnd(B, prompt, C, seed=3, dtype=dtype).to(DEV)
    heads = lambda y: y.unflatten(-1, (H + 2 * Hk, d)).transpose(-3, -2) if y.dim() == 3 else y.unflatten(-1, (H + 2 * Hk, d))  # noqa: E731
    y = int8_linear(x, ci, si)
    holds(y.flatten(0, 1), *ref.linear(x.cpu().flatten(0, 1), ci.cpu(), si.cpu(), None, dtype))
    window_cache_fill(*heads(y)[:, H:].split(Hk, 1), lengths, kc, vc, n_sink=n_sink)
    for step in range(3):
        tok = rnd(B, C, seed=10 + step, dtype=dtype).to(DEV)
        q, k, v = heads(int8_linear(tok, ci, si)).split((H, Hk, Hk), 1)
        before = [type(c)(c.codes.cpu(), c.exponents.cpu(), bits) for c in (kc, vc)]
        o = window_decode_attn(q, k, v, kc, vc, lengths, n_sink=n_sink)
        want, bound, _, _ = decode(q.cpu(), k.cpu(), v.cpu(), *before, lengths.cpu(), n_sink, result=dtype)
        holds(o, want, bound)
        out = int8_linear(o.flatten(1), co, so)
        holds(out, *ref.linear(o.flatten(1).cpu(), co.cpu(), so.cpu(), None, dtype))
        lengths += 1
