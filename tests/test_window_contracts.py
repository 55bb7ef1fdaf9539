"""CPU checks of the sequence operators' wrappers with the launches replaced by copies: what a trace
records and what forward-mode differentiation sees."""

import contextlib
import ctypes

import pytest
import torch
from torch.autograd import forward_ad

import deepfold_amd as df
from deepfold_amd import _lib


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
