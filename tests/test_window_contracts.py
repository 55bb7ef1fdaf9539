"""CPU checks of the sequence operators' wrappers with the launches replaced by copies: what a trace
records and what forward-mode differentiation sees.  And of the C entries' sizes."""

import contextlib
import ctypes
import subprocess
import sys

import pytest
import torch
from torch.autograd import forward_ad

import deepfold_amd as df
from deepfold_amd import _lib


END = 2**31


def test_integers_beyond_32_bits_stay_at_the_end():
    """Lengths and positions are held in 32 bits: what does not fit is the largest or lowest, not another number."""
    from deepfold_amd import rel_pos_bias, window_attn

    x = torch.tensor([0, -1, 5, END - 1, END, END + 5, 2 * END + 5, -END, -END - 1, 2**62, -2**62])
    want = x.clamp(-END, END - 1).to(torch.int32)
    assert torch.equal(window_attn._lengths(x), want)
    assert torch.equal(window_attn._lengths(x[::2]), want[::2]) and window_attn._lengths(x[::2]).is_contiguous()
    short = x[:4].to(torch.int32)
    assert window_attn._lengths(short).data_ptr() == short.data_ptr()
    module = sys.modules["deepfold_amd.rel_pos_bias"]
    assert torch.equal(module._positions(x[None], "q_pos", len(x))[0], want)
    assert rel_pos_bias is module.rel_pos_bias
    for dtype in (torch.int16, torch.uint8, torch.int8):
        assert module._positions(torch.tensor([[0, 7, 100]], dtype=dtype), "q_pos", 3).tolist() == [[0, 7, 100]]


def test_caches_that_share_memory_are_refused():
    """k_cache and v_cache must not have an element in common; interleaved ones (a view of keys and values) are taken.
    The answer is held against the sets of addresses."""
    import random

    from deepfold_amd import window_attn

    rng, seen = random.Random(3), [0, 0]
    for _ in range(600):
        n, hk, slots, d = rng.choice([1, 2, 3]), rng.choice([1, 2]), rng.choice([1, 2, 5]), rng.choice([1, 2, 4])
        order, stride, at = rng.sample(range(3), 3), [0, 0, 0], d
        for dim in order:  # nested strides in any order, with gaps now and then
            stride[dim] = at + rng.choice([0, 0, d, 3])
            at = stride[dim] * ((n, hk, slots)[dim] - 1) + at
        buf = torch.zeros(4 * at + 64)
        shape, first = (n, hk, slots, d), at + 8
        a, b = (buf.as_strided(shape, (*stride, 1), first), buf.as_strided(shape, (*stride, 1), first + rng.randint(-at, at)))
        where = [set((x.storage_offset() + sum(i * s for i, s in zip(ix, x.stride()))) for ix in
                     torch.cartesian_prod(*map(torch.arange, shape)).tolist()) for x in (a, b)]
        shared = bool(where[0] & where[1])
        seen[shared] += 1
        if shared:
            with pytest.raises(ValueError, match="share memory"):
                window_attn._check_caches("t", a, b, n, hk, d, torch.float32, 0)
        else:
            assert window_attn._check_caches("t", a, b, n, hk, d, torch.float32, 0) == slots
    assert min(seen) > 50
    kc = torch.zeros(2, 2, 6, 8)
    with pytest.raises(ValueError, match="share memory"):
        window_attn._check_caches("t", kc[:, :, :5], kc[:, :, 1:], 2, 2, 8, torch.float32, 1)
    # the same storage, one behind the other
    assert window_attn._check_caches("t", kc[:1], kc[1:], 1, 2, 8, torch.float32, 1) == 5


class Copies:
    """In place of the library: each launch copies its first input to what it writes (o = q, cache = k / v)."""

    calls = 0

    def dfl_window_attn_fwd(self, ref, stream):
        p = ref._obj
        ctypes.memmove(p.o, p.q, 4 * p.B * p.H * p.M * p.d)
        self.calls += 1
        return 0

    def dfl_window_cache_fill(self, ref, stream):
        p = ref._obj
        n = 4 * p.B * p.Hk * p.N * p.d
        ctypes.memmove(p.k_cache, p.k, n), ctypes.memmove(p.v_cache, p.v, n)
        self.calls += 1
        return 0

    def dfl_window_decode_workspace_size(self, *sizes):
        return 0

    def dfl_window_decode(self, ref, ws, size, stream):
        p = ref._obj
        ctypes.memmove(p.o, p.q, 4 * p.B * p.H * p.d)
        ctypes.memmove(p.k_cache, p.k, 4 * p.d), ctypes.memmove(p.v_cache, p.v, 4 * p.d)
        self.calls += 1
        return 0


@pytest.fixture
def copies(monkeypatch):
    lib = Copies()
    monkeypatch.setattr(_lib, "require_gpu", lambda *t: torch.device("cpu"))
    monkeypatch.setattr(_lib, "load", lambda: lib)
    monkeypatch.setattr(_lib, "stream_handle", lambda dev: 0)
    monkeypatch.setattr(_lib, "timed_launch", lambda what, dev, f: f())
    monkeypatch.setattr(_lib, "on_device", lambda dev: contextlib.nullcontext())
    return lib


B, H, N, D, W = 2, 2, 5, 4, 4  # N = W + 1 slots: the copies fill a cache exactly


def rows(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def token(*x):
    return [t[:, :, 0].contiguous() for t in x]


def step(q, k, v, kc, vc, lengths):
    """A prompt, its cache and one token."""
    o = df.flash_window_attn(q, k, v, window=W, n_sink=1)
    df.window_cache_fill(k, v, lengths, kc, vc, n_sink=1)
    return o, df.window_decode_attn(*token(q, k, v), kc, vc, lengths, n_sink=1)


def inputs(seed):
    x = [rows(seed + i, B, H, N, D) for i in range(3)]
    return [*x, torch.zeros(B, H, N, D), torch.zeros(B, H, N, D), torch.full((B,), N, dtype=torch.int64)]


def test_a_trace_holds_the_launches(copies):
    """A traced program runs the kernels on its own inputs, writes its caches, and returns no memory of the trace's."""
    traced = torch.jit.trace(step, tuple(inputs(1)), check_trace=False)
    assert str(traced.graph).count("^WindowAttnFn") == 1
    for seed in (10, 20):
        got, want, before = inputs(seed), inputs(seed), copies.calls
        o, dec = traced(*got)
        assert copies.calls == before + 3
        o2, dec2 = step(*want)
        assert torch.equal(o, o2) and torch.equal(o, got[0])
        assert torch.equal(dec, dec2) and torch.equal(dec, got[0][:, :, 0])
        assert torch.equal(got[3], want[3]) and torch.equal(got[4], want[4]) and got[3].any()


def test_forward_mode_is_refused(copies):
    """Inputs with tangents raise, as in the other attention calls; inputs without them still run."""
    with forward_ad.dual_level():
        for at in range(3):
            x = inputs(1)
            x[at] = forward_ad.make_dual(x[at], torch.ones_like(x[at]))
            with pytest.raises(NotImplementedError):
                df.flash_window_attn(*x[:3], window=W)
        for at in (0, 1, 3, 4):
            x = inputs(1)
            x[at] = forward_ad.make_dual(x[at], torch.ones_like(x[at]))
            with pytest.raises(NotImplementedError):
                df.window_decode_attn(*token(*x[:3]), *x[3:], n_sink=1)
            if at:
                with pytest.raises(NotImplementedError):
                    df.window_cache_fill(x[1], x[2], x[5], x[3], x[4], n_sink=1)
        x = inputs(1)
        table = forward_ad.make_dual(torch.zeros(H, 3), torch.ones(H, 3))
        with pytest.raises(NotImplementedError):
            df.window_decode_attn(*token(*x[:3]), *x[3:], n_sink=1, rel_table=table,
                                  rel_edges=(1, 2))
        o, dec = step(*x)
        assert torch.equal(o, x[0]) and torch.equal(dec, x[0][:, :, 0])


SIZES = """
import ctypes, sys
lib = ctypes.CDLL(sys.argv[1])
I = ctypes.c_int
for name, n in (("dfl_window_decode_workspace_size", 6), ("dfl_window_attn_workspace_size", 10), ("dfl_rel_bias_workspace_size", 6)):
    f = getattr(lib, name)
    f.restype, f.argtypes = ctypes.c_size_t, [I] * n
for call in sys.argv[2:]:
    name, *args = call.split(",")
    print(getattr(lib, "dfl_" + name)(*map(int, args)))
"""


def test_workspace_sizes_of_refused_arguments():
    """A size asked for what the entry itself refuses is 0, whatever the numbers; in a process of its own, as a division
    by zero would end it."""
    top = 2**31 - 1
    refused = [("window_decode", 1, 2, 4, 64, 128, 0), ("window_decode", 1, 3, 2, 64, 4096, 0),
               ("window_decode", 1, 2, 2, 64, top, 1), ("window_decode", 1, 2, 2, 64, 4096, 129),
               ("window_decode", 2**30, 2**30, 2**30, 64, 4096, 0), ("window_decode", 1 << 22, 1, 1, 64, 4096, 4),
               ("window_attn", 1, 2, 4, 64, 64, 64, 16, 0, 1, 0), ("window_attn", 1, 2, 2, 1, top, 64, 16, 0, 1, 0),
               ("window_attn", 2**30, 2**30, 2**30, 8, 8, 64, 16, 0, 1, 0), ("window_attn", 1, 2, 2, 8, 8, 64, 16, 129, 1, 0),
               ("window_attn", 1, 2, 2, 8, 8, 64, 16, 0, 1, top), ("window_attn", 1, 2, 2, 8, 8, 64, 16, 0, 0, 48),
               ("rel_bias", 1, 1, 8, 8, top, 1), ("rel_bias", 65536, 1, 8, 8, 3, 1), ("rel_bias", 1, 1, 8, 8, 96, 0)]
    taken = [("window_decode", 1, 2, 2, 64, 4096, 128), ("window_attn", 1, 2, 2, 8, 8, 64, top, 128, 0, 47),
             ("rel_bias", 1, 1, 8, 8, 95, 0)]
    calls = [f"{name}_workspace_size," + ",".join(map(str, a)) for name, *a in refused + taken]
    run = subprocess.run([sys.executable, "-c", SIZES, _lib.LIB_PATH, *calls], capture_output=True, text=True)
    assert run.returncode == 0, (run.returncode, run.stderr[-500:])
    got = list(map(int, run.stdout.split()))
    assert got[:len(refused)] == [0] * len(refused)
    assert all(n > 0 for n in got[len(refused):])


def test_entries_refuse_head_counts_that_wrap_around():
    """B * H of 2^60: the products formed from it would be 0 in 64 bits."""
    lib, fake, n = _lib.load(), 4096, 1 << 30
    p = _lib.WindowAttnParams(dtype=_lib.DFL_BF16, q=fake, k=fake, v=fake, B=n, H=n, Hk=n, M=8, N=8, d=64, window=4, causal=1,
                              scale=1.0, o=fake)
    assert lib.dfl_window_attn_fwd(ctypes.byref(p), None) < 0 and "too large" in lib.dfl_last_error().decode()
    p = _lib.WindowDecodeParams(dtype=_lib.DFL_BF16, q=fake, k=fake, v=fake, k_cache=fake, v_cache=fake, lengths=fake, B=n, H=n,
                                Hk=n, d=64, window=8, scale=1.0, o=fake)
    assert lib.dfl_window_decode(ctypes.byref(p), None, 0, None) < 0 and "too large" in lib.dfl_last_error().decode()


def test_bias_gradient_chains_are_bounded():
    """The workspace holds one sum a bucket for each part of a plane: a thread of a part adds up at most 1024 elements in
    fp32, however large the plane and however many heads there are."""
    lib = _lib.load()
    for heads in (1, 3, 64, 1000, 1024, 4096, 65535):
        for m, n in ((1, 7), (97, 97), (512, 512), (777, 777), (1, 2**20), (4096, 4096), (16384, 16384), (2**17 + 1, 2**13 + 3)):
            size = lib.dfl_rel_bias_workspace_size(1, heads, m, n, 47, 1)
            parts = size // (heads * 96 * 4)
            assert m * n / (256 * parts) <= 1024, (heads, m, n, parts)
            assert parts <= max(1, 1024 // heads, m * n // 2**18 + m * n // 2**23 + 2), (heads, m, n, parts)
