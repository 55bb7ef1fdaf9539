"""Rolling caches in 8 or 4 bits on the GPU against their float64 forms (oracle/lowbit.py) on identical inputs: codes,
exponents and readings exactly, one token's attention to the elementwise bound that the oracle derives."""

import math

import pytest
import torch

from oracle import lowbit as ref
from oracle import window as plain_ref

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF, F32 = torch.bfloat16, torch.float32
EDGES = (1, 2, 3, 4, 6, 9, 14, 20, 31)


def rnd(*shape, seed, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def odd_rows(B, Hk, N, d, seed, dtype):
    """Rows with everything that a code has to survive: ties, zeros of both signs, tiny, huge and infinite elements."""
    x = rnd(B, Hk, N, d, seed=seed)
    g = torch.Generator().manual_seed(seed + 1)
    kind = torch.randint(0, 9, (B, Hk, N), generator=g)
    ties = torch.randint(-255, 256, (B, Hk, N, d), generator=g).float() / 4
    size = torch.randint(-130, 120, (B, Hk, N, 1), generator=g)
    x = torch.where((kind == 1)[..., None], ties, x)
    x = torch.where((kind == 2)[..., None], torch.where(x > 0, 0.0, -0.0), x)
    x = torch.where((kind == 3)[..., None], x * 2.0 ** size.clamp(-126, 100), x)
    x = torch.where((kind == 4)[..., None], x.clamp(-1, 1) * 3.38e38, x)
    x = torch.where((kind == 5)[..., None], ties * 2.0 ** size.clamp(-126, 100), x)
    at = torch.randint(0, d, (B, Hk, N, 1), generator=g)
    spoilt = x.scatter(-1, at, math.inf)
    x = torch.where((kind == 6)[..., None], spoilt, x)
    spoilt = x.scatter(-1, at, math.nan)
    x = torch.where((kind == 7)[..., None], spoilt, x)
    return x.to(dtype)


def cache(B, Hk, S, d, bits, seed, layout="own", odd=True):
    """A cache on the CPU: codes of ordinary rows, or (odd) any bytes; as one tensor each, or as views with room between."""
    from deepfold_amd import QuantizedCache

    g = torch.Generator().manual_seed(seed)
    row, groups, n = ref.groups_of(d) * 4 * bits, ref.groups_of(d), -(-S // 4) * 4
    if odd:
        code = torch.randint(0, 256, (B, Hk, S, row), generator=g).to(torch.uint8)
        exps = torch.randint(100, 150, (B, Hk, groups, n), generator=g).to(torch.uint8)
    else:
        code, e = ref.encode(rnd(B, Hk, S, d, seed=seed) * torch.exp(rnd(1, Hk, 1, d, seed=seed + 7) / 2), bits)
        exps = torch.randint(0, 256, (B, Hk, groups, n), generator=g).to(torch.uint8)  # (any behind the last slot)
        exps[..., :S] = e.transpose(-1, -2)
    if layout == "own":
        return QuantizedCache(code, exps, bits)
    # (B,S,Hk,..) with gaps of whole 16-byte pieces, one piece into the buffer
    buf = torch.full((B * S * Hk * (row + 16) + 16,), 91, dtype=torch.uint8)
    code2 = buf[16:].view(B, S, Hk, row + 16)[..., :row].permute(0, 2, 1, 3)
    code2.copy_(code)
    ebuf = torch.full((B * groups * Hk * (n + 4) + 4,), 92, dtype=torch.uint8)
    exps2 = ebuf[4:].view(B, groups, Hk, n + 4)[..., :n].permute(0, 2, 1, 3)
    exps2.copy_(exps)
    return QuantizedCache(code2, exps2, bits)


def onto(c):
    """The same on the GPU, layout and surroundings included."""
    from deepfold_amd import QuantizedCache

    def move(t):
        base = torch.empty(0, dtype=t.dtype).set_(t.untyped_storage())
        return base.to(DEV).as_strided(t.shape, t.stride(), t.storage_offset())

    return QuantizedCache(move(c.codes), move(c.exponents), c.bits)


def around(c):
    """Every byte of a cache's storages, in the cache and between its rows."""
    return [torch.empty(0, dtype=torch.uint8, device=t.device).set_(t.untyped_storage()).cpu() for t in (c.codes, c.exponents)]


def same_cache(got, start, want):
    """The rows are `want`; all the bytes between them are what they were."""
    (codes, exps, _), S = want, start.codes.shape[2]
    expect = onto(start)
    expect.codes.copy_(codes.to(DEV))
    expect.exponents[..., :S].copy_(exps[..., :S].to(DEV))
    for a, b in zip(around(got), around(expect)):
        off = int((a != b).sum())
        assert off == 0, f"{off} of {a.numel()} bytes differ"


def holds(name, got, want, bound):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, name
    assert bool((got.isnan() == want.isnan()).all()), f"{name}: NaN in other places"
    off = (got - want).abs().nan_to_num(nan=0.0)
    bad = ~(off <= bound.nan_to_num(nan=0.0))
    assert not bad.any(), (f"{name}: {int(bad.sum())} of {bad.numel()} entries off, worst {float(off.max()):.3e}, "
                           f"at most {float((off / bound.clamp(min=1e-30)).nan_to_num(nan=0.0).max()):.2f} times the bound")


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("layout", ["own", "view"])
@pytest.mark.parametrize("Hk,N,d,window,n_sink", [(2, 1, 8, 1, 0), (2, 50, 64, 7, 3), (3, 40, 24, 64, 4), (1, 300, 128, 130, 0),
                                                  (2, 33, 5, 16, 40), (1, 21, 96, 9, 1), (2, 17, 80, 30, 2), (1, 9, 1, 5, 2)])
def test_fill(Hk, N, d, window, n_sink, layout, bits, dtype):
    from deepfold_amd import window_cache_fill

    lengths = torch.tensor([N, 0, 1, max(1, N - 5), N + 7, -3, N, N, N, 1], dtype=torch.int64)
    starts = torch.tensor([0, 5, 0, 3, n_sink, 2, -1, 1000, 2**31 + 5, n_sink + window - 1], dtype=torch.int64)
    starts[8] = 2**31 - 1 if N == 1 else 2**31 - N // 2  # (the last position that a start can be, positions behind it)
    B = len(lengths)
    k, v = (odd_rows(B, N, Hk, d, s, dtype).transpose(1, 2) for s in (1, 2))
    for start in (None, starts):
        kc, vc = (cache(B, Hk, n_sink + window, d, bits, s, layout) for s in (3, 4))
        got = onto(kc), onto(vc)
        want = ref.fill(k, v, lengths, start, kc, vc, n_sink)
        before = got[0].codes._version
        window_cache_fill(k.to(DEV), v.to(DEV), lengths.to(DEV), *got, n_sink=n_sink, starts=None if start is None else start.to(DEV))
        for c, s, w in zip(got, (kc, vc), want):
            same_cache(c, s, w)
        assert got[0].codes._version > before


@pytest.mark.parametrize("dtype", [BF, F32])
def test_fill_any_numbers(dtype):
    """Rows of random bits, at every alignment of their first element."""
    from deepfold_amd import window_cache_fill

    B, Hk, N, d = 2, 3, 65, 64
    g = torch.Generator().manual_seed(5)
    for bits in (4, 8):
        for shift in (0, 1, 4):
            kv = []
            for _ in range(2):
                x = torch.randint(-2**31, 2**31, (B * Hk * N * d + 8,), generator=g).to(torch.int32).view(F32).to(dtype)
                kv.append(x[shift:shift + B * Hk * N * d].view(B, Hk, N, d))
            kc, vc = (cache(B, Hk, N, d, bits, s) for s in (3, 4))
            got = onto(kc), onto(vc)
            lengths = torch.tensor([N, N - 1])
            want = ref.fill(*kv, lengths, None, kc, vc, 0)
            moved = [torch.cat((t.new_zeros(shift), t.flatten())).to(DEV)[shift:].view(t.shape) for t in kv]
            window_cache_fill(*moved, lengths.to(DEV), *got)
            for c, s, w in zip(got, (kc, vc), want):
                same_cache(c, s, w)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_plain_caches_in_chunks(dtype):
    """`starts` for caches of the inputs' type, and their reading."""
    from deepfold_amd import window_cache_fill, window_cache_read

    B, Hk, d, n_sink, window = 3, 2, 24, 3, 10
    kc, vc = (rnd(B, Hk, n_sink + window, d, seed=s, dtype=dtype) for s in (1, 2))
    g = [c.to(DEV) for c in (kc, vc)]
    starts = torch.tensor([0, 5, 40])
    for step, n in enumerate((7, 1, 20)):
        k, v = (rnd(B, n, Hk, d, seed=10 * step + s, dtype=dtype).transpose(1, 2) for s in (3, 4))
        lengths = torch.tensor([n, n - 1, n])
        for b in range(B):
            for i in range(int(lengths[b])):
                s = plain_ref.slot(int(starts[b]) + i, n_sink, window)
                kc[b, :, s], vc[b, :, s] = k[b, :, i], v[b, :, i]
        window_cache_fill(k.to(DEV), v.to(DEV), lengths.to(DEV), *g, n_sink=n_sink, starts=starts.to(DEV))
        assert torch.equal(g[0].cpu(), kc) and torch.equal(g[1].cpu(), vc)
        starts += lengths
        want = ref.read(kc.double(), vc.double(), starts, n_sink)
        got = window_cache_read(*g, starts.to(DEV), d, n_sink=n_sink)
        assert got[0].dtype == dtype and all(torch.equal(a.double().cpu(), b) for a, b in zip(got, want))
    # one start for all at None is the fill that there was
    a, b = [t.clone() for t in g], [t.clone() for t in g]
    zero = torch.zeros(B, dtype=torch.int32, device=DEV)
    window_cache_fill(k.to(DEV), v.to(DEV), lengths.to(DEV), *a, n_sink=n_sink)
    window_cache_fill(k.to(DEV), v.to(DEV), lengths.to(DEV), *b, n_sink=n_sink, starts=zero)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    far = torch.full((B,), -2**40, device=DEV)
    window_cache_fill(k.to(DEV), v.to(DEV), lengths.to(DEV), *b, n_sink=n_sink, starts=far)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("out", [BF, F32])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("layout", ["own", "view"])
@pytest.mark.parametrize("Hk,d,window,n_sink", [(2, 8, 1, 0), (1, 64, 7, 3), (2, 24, 30, 4), (1, 128, 70, 0), (2, 5, 6, 40), (1, 96, 9, 1),
                                                (1, 80, 30, 2), (2, 1, 5, 2)])
def test_read(Hk, d, window, n_sink, layout, bits, out):
    from deepfold_amd import window_cache_read

    S = n_sink + window
    lengths = torch.tensor([0, S, -1, S - 1, S // 2, 3 * S + 5, 2**31 - 1, 1, 2**40, -2**31])
    B = len(lengths)
    kc, vc = (cache(B, Hk, S, d, bits, s, layout) for s in (3, 4))
    for c in (kc, vc):  # groups that are no numbers among the others, and the ends of the exponents
        c.exponents[::2, :, :, ::3] = 255
        c.exponents[1::2, :, :, ::5] = 1
        c.exponents[1::2, :, :, 1::5] = 248
    K, V, mask = window_cache_read(onto(kc), onto(vc), lengths.to(DEV), d, n_sink=n_sink, dtype=out)
    want = ref.read(ref.cache_values(kc, d), ref.cache_values(vc, d), lengths.clamp(max=2**31 - 1), n_sink)
    assert K.dtype == V.dtype == out
    for a, b in zip((K, V, mask), want):  # (any byte is a code here: -128 times the highest power rounds to infinity)
        a, b = a.double().cpu(), b.to(out).double()
        same = (a == b) | (a.isnan() & b.isnan())
        assert a.shape == b.shape and bool(same.all()), int((~same).sum())


DECODES = [(2, 2, 32, 1, 0, True), (4, 2, 64, 60, 4, False), (3, 1, 24, 200, 1, True), (8, 1, 128, 300, 0, True),
           (10, 2, 80, 65, 70, False), (1, 1, 1, 5, 2, True), (16, 1, 64, 1100, 4, True), (9, 1, 96, 500, 1, False),
           (17, 1, 128, 140, 3, True), (40, 1, 40, 97, 0, False), (12, 4, 128, 1500, 4, False)]


def decode_case(H, Hk, d, window, n_sink, rel, bits, dtype, layout, lengths, scale=None, size=1.0):
    from deepfold_amd import window_decode_attn

    B, S = len(lengths), n_sink + window
    q = rnd(B, H, d, seed=1, dtype=dtype, scale=size)
    k, v = rnd(B, Hk, d, seed=2, dtype=dtype), rnd(B, Hk, d, seed=3, dtype=dtype)
    kc, vc = (cache(B, Hk, S, d, bits, s, layout, odd=False) for s in (4, 5))
    for b, n in enumerate(lengths.tolist()):  # what is not in use is anything at all
        for c in (kc, vc):
            if n < S - 1:
                c.exponents[b, :, :, max(0, n + 1):S] = 255
                c.codes[b, :, max(0, n + 1):] = 133
            if n >= 0:  # the token's own slot holds what it held
                own = plain_ref.slot(n, n_sink, window)
                c.exponents[b, :, :, own], c.codes[b, :, own] = 255, 77
    table = rnd(H, len(EDGES) + 1, seed=6) if rel else None
    want, bound, kw, vw = ref.decode(q, k, v, kc, vc, lengths, n_sink, scale=scale, table=table, edges=EDGES, result=dtype)
    got = onto(kc), onto(vc)
    at = lengths.to(DEV)
    o = window_decode_attn(q.to(DEV), k.to(DEV), v.to(DEV), *got, at, n_sink=n_sink, scale=scale,
                           rel_table=None if table is None else table.to(DEV), rel_edges=EDGES if rel else None)
    assert o.dtype == dtype and torch.equal(at.cpu(), lengths)
    for c, s, w in zip(got, (kc, vc), (kw, vw)):
        same_cache(c, s, w)
    holds("o", o, want, bound)
    return o


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("layout", ["own", "view"])
@pytest.mark.parametrize("H,Hk,d,window,n_sink,rel", DECODES)
def test_decode(H, Hk, d, window, n_sink, rel, layout, bits, dtype):
    S = n_sink + window
    lengths = torch.tensor([0, S, -1, S - 1, S // 2, 3 * S + 5, 10**9, 1, min(31, S), 32, -2**31])
    o = decode_case(H, Hk, d, window, n_sink, rel, bits, dtype, layout, lengths)
    assert not o[2].any() and not o[-1].any()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("bits", [4, 8])
def test_decode_lengths(bits, dtype):
    """Every length around a block of slots and around the end of the cache, in caches of one split and of several."""
    for window, n_sink in ((70, 2), (330, 1)):
        S = n_sink + window
        lengths = torch.tensor([*range(0, 4), *range(14, 20), *range(29, 36), *range(62, 68), 127, 128, 129, *range(S - 3, S + 3),
                                2**31 - 1 - S])
        decode_case(4, 2, 64, window, n_sink, False, bits, dtype, "own", lengths[lengths < 3 * S])


@pytest.mark.parametrize("dtype,bits", [(BF, 4), (F32, 8)])
@pytest.mark.parametrize("B,H,Hk,d,window,n_sink", [(129, 4, 2, 24, 45, 3), (86, 3, 3, 64, 300, 0), (100, 3, 3, 8, 1600, 1),
                                                    (150, 6, 3, 8, 1600, 0)])
def test_decode_many_sequences(B, H, Hk, d, window, n_sink, bits, dtype):
    """More samples and key heads than CUs, with short and long caches, as many as fill the CUs again and fewer."""
    lengths = torch.randint(-1, 3 * window, (B,), generator=torch.Generator().manual_seed(B))
    decode_case(H, Hk, d, window, n_sink, False, bits, dtype, "own", lengths)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("bits", [4, 8])
def test_decode_sharp_scores(bits, dtype):
    """Scores that differ by hundreds, in both directions along the cache: references that move, weights that vanish."""
    lengths = torch.tensor([400, 1000, 77])
    decode_case(6, 2, 64, 396, 4, True, bits, dtype, "own", lengths, scale=2.0, size=4.0)
    decode_case(6, 2, 64, 396, 4, False, bits, dtype, "own", lengths, scale=1e-30)


def test_decode_scores_that_grow():
    """Keys along the query, larger and larger: every block moves the reference by more than its slack."""
    from deepfold_amd import QuantizedCache, window_decode_attn

    B, H, d, S = 1, 2, 32, 1600
    q = torch.ones(B, H, d)
    k = torch.ones(B, 1, S, d) * torch.arange(S).float()[None, None, :, None] / 10
    v = rnd(B, 1, S, d, seed=1)
    for flip in (False, True):
        kk = k.flip(2) if flip else k
        caches = []
        for x in (kk, v):
            code, e = ref.encode(x, 8)
            exps = torch.zeros(B, 1, 1, S, dtype=torch.uint8)
            exps[..., :S] = e.transpose(-1, -2)
            caches.append(QuantizedCache(code, exps, 8))
        lengths = torch.tensor([S + 3])
        tok = torch.ones(B, 1, d), torch.ones(B, 1, d)
        want, bound, _, _ = ref.decode(q, *tok, *caches, lengths, 0)
        o = window_decode_attn(q.to(DEV), *(t.to(DEV) for t in tok), *(onto(c) for c in caches), lengths.to(DEV))
        holds("o", o, want, bound)


def test_decode_table_entries():
    """An entry of -inf (or far below all scores) takes its keys out; where it takes all, the row is zero."""
    from deepfold_amd import window_decode_attn

    B, H, d, S, edges = 2, 3, 32, 100, (1, 5, 40)
    q, k, v = rnd(B, H, d, seed=1), rnd(B, 1, d, seed=2), rnd(B, 1, d, seed=3)
    lengths = torch.tensor([250, 3])
    for low in (-math.inf, torch.finfo(F32).min, -1e35):
        table = torch.zeros(H, 4)
        table[0, 0], table[0, 2], table[1] = low, low, low
        kc, vc = (cache(B, 1, S, d, 4, s, odd=False) for s in (4, 5))
        want, bound, _, _ = ref.decode(q, k, v, kc, vc, lengths, 0, table=table, edges=edges)
        o = window_decode_attn(q.to(DEV), k.to(DEV), v.to(DEV), onto(kc), onto(vc), lengths.to(DEV), rel_table=table.to(DEV),
                               rel_edges=edges)
        assert not o[:, 1].any()
        holds("o", o, want, bound)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("where", ["k", "v", "own k", "own v"])
def test_decode_of_what_is_no_number(where, bits):
    """A group of E = 255 in a slot in use: NaN for every head that reads it, and for no other sample or key head."""
    from deepfold_amd import window_decode_attn

    B, H, Hk, d, S = 2, 6, 2, 70, 300
    q, k, v = (rnd(B, h, d, seed=s, dtype=BF) for s, h in ((1, H), (2, Hk), (3, Hk)))
    kc, vc = (cache(B, Hk, S, d, bits, s, odd=False) for s in (4, 5))
    lengths = torch.tensor([290, 1000])
    if where == "own k":
        k[1, 0, 69] = math.inf
    elif where == "own v":
        v[1, 0, 3] = math.nan
    else:
        (kc if where == "k" else vc).exponents[1, 0, 1, 201] = 255
    o = window_decode_attn(q.to(DEV), k.to(DEV), v.to(DEV), onto(kc), onto(vc), lengths.to(DEV))
    assert o[1, :3].isnan().all() and not o[0].isnan().any() and not o[1, 3:].isnan().any()


def test_decode_queries_that_are_no_numbers():
    """A NaN in a query is its own head's affair; the largest finite query has no infinite part."""
    from deepfold_amd import window_decode_attn

    B, H, d, S = 1, 4, 32, 60
    for dtype in (BF, F32):
        q, k, v = rnd(B, H, d, seed=1, dtype=dtype), rnd(B, 1, d, seed=2, dtype=dtype), rnd(B, 1, d, seed=3, dtype=dtype)
        kc, vc = (cache(B, 1, S, d, 4, s, odd=False) for s in (4, 5))
        clean = window_decode_attn(*(t.to(DEV) for t in (q, k, v)), onto(kc), onto(vc), torch.tensor([40], device=DEV))
        q[0, 2, 7] = math.nan
        o = window_decode_attn(*(t.to(DEV) for t in (q, k, v)), onto(kc), onto(vc), torch.tensor([40], device=DEV))
        assert o[0, 2].isnan().all() and torch.equal(o[0, [0, 1, 3]], clean[0, [0, 1, 3]])
    q = torch.zeros(1, 1, d)
    q[0, 0, 0] = torch.finfo(F32).max
    lengths = torch.tensor([40])
    kc, vc = (cache(B, 1, S, d, 8, s, odd=False) for s in (4, 5))
    want, bound, _, _ = ref.decode(q, k, v, kc, vc, lengths, 0, scale=1e-30)
    o = window_decode_attn(*(t.to(DEV) for t in (q, k, v)), onto(kc), onto(vc), lengths.to(DEV), scale=1e-30)
    assert torch.isfinite(o).all()


def test_a_long_cache():
    """Offsets of codes and of exponents beyond 32 bits: 3 GB of codes between a sample's heads."""
    from deepfold_amd import QuantizedCache, window_cache_fill, window_cache_read, window_decode_attn

    Hk, d, S, bits = 2, 128, 40, 4
    apart = 3 << 30
    buf = torch.empty(apart + S * 64, dtype=torch.uint8, device=DEV)
    ebuf = torch.empty(apart + 4 * S, dtype=torch.uint8, device=DEV)
    kc = QuantizedCache(buf.as_strided((1, Hk, S, 64), (apart, apart, 64, 1)), ebuf.as_strided((1, Hk, 4, S), (apart, apart, S, 1)), bits)
    vc = QuantizedCache(*(t.clone(memory_format=torch.contiguous_format) for t in kc[:2]), bits)
    small = [QuantizedCache(*(t.clone(memory_format=torch.contiguous_format) for t in c[:2]), bits) for c in (kc, vc)]
    k, v = rnd(1, Hk, S, d, seed=1, dtype=BF).to(DEV), rnd(1, Hk, S, d, seed=2, dtype=BF).to(DEV)
    q = rnd(1, 4, d, seed=3, dtype=BF).to(DEV)
    lengths = torch.tensor([S], device=DEV)
    out = []
    for a, b in ((kc, vc), small):
        window_cache_fill(k, v, lengths, a, b)
        o = window_decode_attn(q, k[:, :, 0], v[:, :, 0], a, b, lengths)
        out.append((o, *window_cache_read(a, b, lengths + 1, d), *(t.clone() for t in (a.codes, a.exponents))))
    assert all(torch.equal(x, y) for x, y in zip(*out))


def test_chunks_before_the_first_tokens():
    """Chunks as long as the window for samples without, with a part of and with all of the first tokens, then a longer one."""
    from deepfold_amd import flash_window_attn, quantized_cache, window_cache_fill, window_cache_read

    B, H, Hk, d, window, n_sink, bits = 4, 4, 2, 32, 20, 4, 8
    kc, vc = (quantized_cache(B, Hk, n_sink + window, d, bits=bits, device=DEV) for _ in range(2))
    held = [[torch.zeros(Hk, 0, d) for _ in range(B)] for _ in range(2)]
    lengths = torch.zeros(B, dtype=torch.int32, device=DEV)
    for step, rows in enumerate(([0, 2, 3, 4], [window] * 4, [2 * window + 1, 2 * window + 1, 7, 0])):
        n = max(rows)
        q, k, v = (rnd(B, h, n, d, seed=20 * step + i) for i, h in enumerate((H, Hk, Hk)))
        chunk = torch.tensor(rows, device=DEV, dtype=torch.int32)
        mine = (torch.arange(n, device=DEV)[None] < chunk[:, None]).float()
        kp, vp, m = window_cache_read(kc, vc, lengths, d, n_sink=n_sink, dtype=F32)
        o = flash_window_attn(q.to(DEV), torch.cat((kp, k.to(DEV)), 2), torch.cat((vp, v.to(DEV)), 2), torch.cat((m, mine), 1),
                              window=window, n_sink=n_sink)
        window_cache_fill(k.to(DEV), v.to(DEV), chunk, kc, vc, n_sink=n_sink, starts=lengths)
        for b in range(B):
            if rows[b]:
                whole = [torch.cat((h[b], x[b, :, :rows[b]]), 1)[None] for h, x in zip(held, (k, v))]
                want = plain_ref.attention(q[b:b + 1, :, :rows[b]], *whole, window=window, n_sink=n_sink, operand=F32, result=F32)["o"]
                holds("chunk", o[b:b + 1, :, :rows[b]], *want)
            for h, x in zip(held, (k, v)):
                h[b] = torch.cat((h[b], ref.values(*ref.encode(x[b], bits), d, bits)[:, :rows[b]].to(F32)), 1)
        lengths += chunk


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_chunks_then_tokens(dtype, bits):
    """A prompt in chunks, then tokens, as a user makes it: every chunk attends to what the cache gives back and to itself,
    every token to the cache.  Each step is held against the float64 attention over the rows that it is to see."""
    from deepfold_amd import flash_window_attn, quantized_cache, window_cache_fill, window_cache_read, window_decode_attn

    B, H, Hk, d, window, n_sink = 2, 8, 2, 64, 33, 4
    kc, vc = (quantized_cache(B, Hk, n_sink + window, d, bits=bits, device=DEV) for _ in range(2))
    held = [[[] for _ in range(B)] for _ in range(2)]  # the rows (Hk,d) that entered, as their codes stand, by sample
    lengths = torch.zeros(B, dtype=torch.int32, device=DEV)
    for step, n in enumerate((20, 50, 7)):
        q, k, v = (rnd(B, h, n, d, seed=10 * step + i, dtype=dtype) for i, h in enumerate((H, Hk, Hk)))
        chunk = torch.tensor([n, n - 3], device=DEV, dtype=torch.int32)
        mine = (torch.arange(n, device=DEV)[None] < chunk[:, None]).float()
        kp, vp, m = window_cache_read(kc, vc, lengths, d, n_sink=n_sink, dtype=dtype)
        o = flash_window_attn(q.to(DEV), torch.cat((kp, k.to(DEV)), 2), torch.cat((vp, v.to(DEV)), 2), torch.cat((m, mine), 1),
                              window=window, n_sink=n_sink)
        window_cache_fill(k.to(DEV), v.to(DEV), chunk, kc, vc, n_sink=n_sink, starts=lengths)
        for b in range(B):  # against all positions in a row: those before as held, the chunk's own as given
            rows = int(chunk[b])
            before = [torch.stack(h[b], 1).to(dtype) if h[b] else torch.zeros(Hk, 0, d, dtype=dtype) for h in held]
            whole = [torch.cat((x, y[b, :, :rows]), 1)[None] for x, y in zip(before, (k, v))]
            want = plain_ref.attention(q[b:b + 1, :, :rows], *whole, window=window, n_sink=n_sink, operand=dtype, result=dtype)["o"]
            holds("chunk", o[b:b + 1, :, :rows], *want)
            for h, x in zip(held, (k, v)):
                h[b] += ref.values(*ref.encode(x[b], bits), d, bits)[:, :rows].unbind(1)
        lengths += chunk
    for step in range(6):
        q, k, v = (rnd(B, h, d, seed=100 + 10 * step + i, dtype=dtype) for i, h in enumerate((H, Hk, Hk)))
        before = [type(kc)(c.codes.cpu(), c.exponents.cpu(), bits) for c in (kc, vc)]
        want, bound, _, _ = ref.decode(q, k, v, *before, lengths.cpu(), n_sink, result=dtype)
        o = window_decode_attn(q.to(DEV), k.to(DEV), v.to(DEV), kc, vc, lengths, n_sink=n_sink)
        holds("token", o, want, bound)
        lengths += 1
        for h, x in zip(held, (k, v)):
            for b in range(B):
                h[b].append(ref.values(*ref.encode(x[b], bits), d, bits))
    # what the cache holds are the codes of what entered
    K, V, mask = window_cache_read(kc, vc, lengths, d, n_sink=n_sink, dtype=F32)
    for b in range(B):
        for got, h in zip((K, V), held):
            want = torch.stack(h[b][:n_sink] + h[b][len(h[b]) - window:], 1)
            assert torch.equal(got[b].double().cpu(), want)
    assert mask.all()


def test_graph_replays():
    """A token's whole step captured and replayed, with eager work between: the caches move on as in the eager run."""
    from deepfold_amd import quantized_cache, window_cache_fill, window_cache_read, window_decode_attn

    B, H, Hk, d, window, n_sink = 2, 8, 2, 64, 300, 3
    tok = [rnd(B, h, d, seed=s, dtype=BF).to(DEV) for s, h in ((6, H), (7, Hk), (8, Hk))]
    rows = [rnd(B, Hk, 5, d, seed=s, dtype=BF).to(DEV) for s in (9, 10)]
    n = torch.tensor([5, 4], dtype=torch.int32, device=DEV)

    def start():
        return [quantized_cache(B, Hk, n_sink + window, d, bits=b, device=DEV) for b in (4, 4, 8, 8)] + [
            torch.tensor([0, 290], dtype=torch.int32, device=DEV)]

    def step(a, b, c, e, at):
        o = [window_decode_attn(*tok, x, y, at, n_sink=n_sink) for x, y in ((a, b), (c, e))]
        for x, y in ((a, b), (c, e)):
            window_cache_fill(*rows, n, x, y, n_sink=n_sink, starts=at + 1)
        at.add_(6)
        return [*o, *window_cache_read(a, b, at, d, n_sink=n_sink), *window_cache_read(c, e, at, d, n_sink=n_sink)]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(*start())
    s.synchronize()
    mine, eager = start(), start()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        out = step(*mine)
    for c, e in zip(mine, start()):  # (a capture runs nothing)
        assert torch.equal(c[0] if isinstance(c, tuple) else c, e[0] if isinstance(e, tuple) else e)
    for turn in range(5):
        for t in (*tok, *rows):
            t.copy_(torch.randn(t.shape, generator=torch.Generator().manual_seed(50 + turn)).to(BF))
        g.replay()
        got = [t.clone() for t in out]
        torch.cuda.synchronize()
        want = step(*eager)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        for a, b in zip(mine[:4], eager[:4]):
            assert torch.equal(a.codes, b.codes) and torch.equal(a.exponents, b.exponents)


def test_two_streams_at_once():
    """Calls in flight on two streams share nothing."""
    from deepfold_amd import window_decode_attn

    B, H, Hk, d, S = 2, 8, 2, 128, 2000
    sets = [[rnd(B, h, d, seed=10 * i + s, dtype=BF).to(DEV) for s, h in ((1, H), (2, Hk), (3, Hk))] for i in range(2)]
    caches = [[onto(cache(B, Hk, S, d, 4, 40 + 2 * i + j, odd=False)) for j in range(2)] for i in range(2)]
    at = torch.tensor([5000, 400], device=DEV, dtype=torch.int32)
    want = [window_decode_attn(*sets[i], *caches[i], at).clone() for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(4):
        got = [None, None]
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = window_decode_attn(*sets[i], *caches[i], at)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_strided_tokens():
    """Queries, keys and values as views of one projection's result, and transposed ones."""
    from deepfold_amd import window_decode_attn

    B, H, Hk, d, S = 3, 4, 2, 32, 50
    x = rnd(B, (H + 2 * Hk) * d, seed=1, dtype=BF).to(DEV)
    q, k, v = x.view(B, H + 2 * Hk, d).split((H, Hk, Hk), 1)
    at = torch.tensor([100, 3, 49], device=DEV)
    caches = [[onto(cache(B, Hk, S, d, 4, 4 + j, odd=False)) for j in range(2)] for _ in range(3)]
    want = window_decode_attn(q.contiguous(), k.contiguous(), v.contiguous(), *caches[0], at)
    assert torch.equal(window_decode_attn(q, k, v, *caches[1], at), want)
    spread = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]  # the last dimension apart
    assert torch.equal(window_decode_attn(*spread, *caches[2], at), want)
    for c in caches[1:]:
        assert torch.equal(c[0].codes, caches[0][0].codes) and torch.equal(c[1].exponents, caches[0][1].exponents)
