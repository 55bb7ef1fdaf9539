"""CPU checks of the few-bit operators' host side: parameter blocks, what the C entries and the wrappers refuse, what a trace
records (launches replaced).  No kernel runs here."""

import contextlib
import ctypes
import os
import re
import subprocess

import pytest
import torch
from torch.autograd import forward_ad

import deepfold_amd as df
from conftest import ROOT
from deepfold_amd import _lib, window_attn

BF, F32 = torch.bfloat16, torch.float32
FAKE = 4096  # an address that is never read


def test_struct_layout_matches_c(tmp_path):
    header = os.path.join(ROOT, "include", "dfl_lowbit.h")
    mirrors = {"dfl_lowbit_cache": _lib.LowbitCache, "dfl_lowbit_cache_fill_params": _lib.LowbitCacheFillParams,
               "dfl_window_cache_read_params": _lib.WindowCacheReadParams, "dfl_lowbit_decode_params": _lib.LowbitDecodeParams,
               "dfl_quantize_rows_params": _lib.QuantizeRowsParams, "dfl_int8_linear_params": _lib.Int8LinearParams}
    text = re.sub(r"/\*.*?\*/", "", open(header).read(), flags=re.S)
    assert set(re.findall(r"\} (\w+);", text)) == set(mirrors)
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{header}"', "int main(void) {"]
    for name, cls in mirrors.items():
        lines.append(f'  printf("{name} size %zu\\n", sizeof({name}));')
        lines += [f'  printf("{name} {f} %zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    (tmp_path / "probe.c").write_text("\n".join(lines + ["  return 0;", "}"]))
    subprocess.run(["gcc", "-std=c99", "-o", tmp_path / "probe", tmp_path / "probe.c"], check=True)
    out = subprocess.run([tmp_path / "probe"], capture_output=True, text=True, check=True).stdout
    layout = {tuple(line.split()[:2]): int(line.split()[2]) for line in out.splitlines()}
    for name, cls in mirrors.items():
        assert ctypes.sizeof(cls) == layout[name, "size"], name
        for f, _ in cls._fields_:
            assert getattr(cls, f).offset == layout[name, f], (name, f)


def codes(**kw):
    return _lib.LowbitCache(**{**dict(codes=FAKE, exponents=FAKE, stride_b=256, stride_h=128, stride_n=64, exp_stride_b=64,
                                      exp_stride_h=64, exp_stride_g=8192), **kw})


def fill_params(**kw):
    return _lib.LowbitCacheFillParams(**{**dict(dtype=0, bits=4, k=FAKE, v=FAKE, lengths=FAKE, k_cache=codes(), v_cache=codes(), B=2,
                                                Hk=2, N=8, d=64, window=8, n_sink=1), **kw})


def read_params(**kw):
    return _lib.WindowCacheReadParams(**{**dict(dtype=0, bits=4, k_cache=codes(), v_cache=codes(), lengths=FAKE, k=FAKE, v=FAKE,
                                                mask=FAKE, B=2, Hk=2, d=64, window=8, n_sink=1), **kw})


def decode_params(**kw):
    return _lib.LowbitDecodeParams(**{**dict(dtype=0, bits=4, q=FAKE, k=FAKE, v=FAKE, k_cache=codes(), v_cache=codes(), lengths=FAKE,
                                             B=2, H=4, Hk=2, d=64, window=4096, n_sink=1, scale=1.0, o=FAKE), **kw})


def rows_params(**kw):
    return _lib.QuantizeRowsParams(**{**dict(dtype=0, x=FAKE, x_stride=64, M=4, K=60, codes=FAKE, code_stride=64, scale=FAKE), **kw})


def linear_params(**kw):
    return _lib.Int8LinearParams(**{**dict(dtype=0, x=FAKE, x_stride=64, w=FAKE, w_stride=64, w_scale=FAKE, y=FAKE, M=4, K=60, N=8),
                                    **kw})


SHAPE = [dict(dtype=2), dict(B=0), dict(Hk=0), dict(d=0), dict(d=129), dict(window=0), dict(window=2**31 - 1), dict(n_sink=-1),
         dict(n_sink=129)]
CODES = [dict(bits=5), dict(bits=16), dict(k_cache=codes(codes=None)), dict(v_cache=codes(exponents=None)),
         dict(k_cache=codes(codes=FAKE + 8)), dict(v_cache=codes(stride_n=68)), dict(k_cache=codes(stride_b=-8)),
         dict(v_cache=codes(exp_stride_g=6)), dict(k_cache=codes(exponents=FAKE + 2))]


@pytest.mark.parametrize("entry,make,bad", [
    ("fill", fill_params, SHAPE + CODES + [dict(N=0), dict(N=2**30), dict(B=70000, Hk=1), dict(k=None), dict(lengths=None),
                                           dict(B=2**30, Hk=2**30)]),
    ("read", read_params, SHAPE + CODES + [dict(mask=None), dict(k=None), dict(lengths=None), dict(B=70000, Hk=1),
                                           dict(bits=0, v_cache=codes(codes=None)), dict(bits=1)]),
    ("decode", decode_params, SHAPE + CODES + [dict(H=3), dict(H=0), dict(scale=0.0), dict(scale=float("nan")), dict(q=None), dict(o=None),
                                               dict(rel_table=FAKE), dict(n_edges=2), dict(n_edges=96, rel_table=FAKE, rel_edges=FAKE),
                                               dict(n_edges=-1, rel_table=FAKE), dict(B=2**30, H=2**30, Hk=2**30),
                                               dict(k_cache=codes(stride_n=16)), dict(v_cache=codes(stride_n=1 << 26)),
                                               dict(k_cache=codes(exp_stride_g=4096)), dict(v_cache=codes(exp_stride_g=1 << 30))]),
    ("rows", rows_params, [dict(dtype=2), dict(M=0), dict(M=2**31), dict(K=0), dict(K=2**17 + 1), dict(x=None), dict(codes=None),
                           dict(scale=None), dict(code_stride=48), dict(code_stride=72), dict(codes=FAKE + 4)]),
    ("linear", linear_params, [dict(dtype=2), dict(M=0), dict(K=0), dict(N=0), dict(M=-1), dict(K=2**17 + 1, w_stride=2**18), dict(x=None),
                               dict(w=None), dict(w_scale=None), dict(y=None), dict(w_stride=48), dict(w_stride=72),
                               dict(w=FAKE + 8), dict(M=2**31 - 1, N=2**31 - 1), dict(M=2**31 - 255), dict(N=2**31 - 1)]),
])
def test_entries_refuse(entry, make, bad):
    """Every refusal comes before any launch (the pointers are no memory)."""
    lib = _lib.load()
    call = {"fill": lambda p: lib.dfl_lowbit_cache_fill(ctypes.byref(p), None),
            "read": lambda p: lib.dfl_window_cache_read(ctypes.byref(p), None),
            "decode": lambda p: lib.dfl_lowbit_decode(ctypes.byref(p), FAKE, 1 << 40, None),
            "rows": lambda p: lib.dfl_quantize_rows(ctypes.byref(p), None),
            "linear": lambda p: lib.dfl_int8_linear(ctypes.byref(p), FAKE, 1 << 60, None)}[entry]
    for kw in bad:
        assert call(make(**kw)) < 0, kw
        assert lib.dfl_last_error(), kw
    null = {"fill": lambda: lib.dfl_lowbit_cache_fill(None, None), "read": lambda: lib.dfl_window_cache_read(None, None),
            "decode": lambda: lib.dfl_lowbit_decode(None, None, 0, None), "rows": lambda: lib.dfl_quantize_rows(None, None),
            "linear": lambda: lib.dfl_int8_linear(None, None, 0, None)}[entry]
    assert null() < 0


def test_workspaces():
    """Sizes of what the entries refuse are 0; a workspace one byte short is refused."""
    lib = _lib.load()
    top = 2**31 - 1
    for a in ((1, 2, 4, 64, 128, 0), (1, 3, 2, 64, 128, 0), (1, 2, 2, 64, top, 1), (1, 2, 2, 64, 128, 129), (0, 1, 1, 64, 128, 0),
              (2**30, 2**30, 2**30, 64, 128, 0), (1, 2, 2, 129, 128, 0), (1 << 22, 1, 1, 64, 4096, 4), (1, 2, 2, 64, 0, 4)):
        assert lib.dfl_lowbit_decode_workspace_size(*a) == 0, a
    for a in ((0, 64, 64), (64, 0, 64), (64, 64, 0), (-1, 64, 64), (4, 2**17 + 1, 4), (top, -5, 1)):
        assert lib.dfl_int8_linear_workspace_size(*a) == 0, a
    assert lib.dfl_int8_linear_workspace_size(top, 2**17, 1) > top * 2**17
    need = lib.dfl_lowbit_decode_workspace_size(2, 4, 2, 64, 4096, 1)
    assert need > 0
    assert lib.dfl_lowbit_decode(ctypes.byref(decode_params()), FAKE, need - 1, None) < 0
    assert b"workspace too small" in lib.dfl_last_error()
    assert lib.dfl_lowbit_decode(ctypes.byref(decode_params()), None, need, None) < 0
    assert lib.dfl_int8_linear_workspace_size(4, 60, 8) == 0  # (few tokens: none is needed)
    for a in ((8, 4096, 8), (16, 2048, 8), (100, 1024, 8)):
        assert lib.dfl_int8_linear_workspace_size(*a) == 0, a
    for a in ((8, 4097, 8), (9, 2049, 8), (17, 1025, 8), (1, 64, 2**20)):
        assert lib.dfl_int8_linear_workspace_size(*a) > 0, a
    need = lib.dfl_int8_linear_workspace_size(9, 4100, 8)
    assert lib.dfl_int8_linear(ctypes.byref(linear_params(M=9, K=4100, x_stride=4104, w_stride=4112)), FAKE, need - 1, None) < 0
    assert b"workspace too small" in lib.dfl_last_error()
    assert lib.dfl_int8_linear(ctypes.byref(linear_params(M=9, K=4100, x_stride=4104, w_stride=4112)), FAKE + 8, need, None) < 0
    assert lib.dfl_int8_linear(ctypes.byref(linear_params(M=9, K=4100, x_stride=4104, w_stride=4112)), None, need, None) < 0


class Launches:
    """In place of the library: counts the calls and writes what is simple to tell (q into o, ones into y, ...)."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        if name.endswith("workspace_size"):
            return lambda *a: 256
        assert name.startswith("dfl_")

        def call(ref, *rest):
            p = ref._obj
            if name == "dfl_lowbit_decode":
                ctypes.memmove(p.o, p.q, 4 * p.B * p.H * p.d)
            elif name == "dfl_window_cache_read":
                for out in (p.k, p.v):
                    ctypes.memset(out, 0, 4 * p.B * p.Hk * (p.window + p.n_sink) * p.d)
                ctypes.memset(p.mask, 0, 4 * p.B * (p.window + p.n_sink))
            elif name == "dfl_int8_linear":
                ctypes.memmove(p.y, p.x, 4 * p.M * p.N)
            elif name == "dfl_quantize_rows":
                ctypes.memset(p.codes, 1, p.M * p.code_stride), ctypes.memset(p.scale, 0, 4 * p.M)
            elif name == "dfl_lowbit_cache_fill":
                ctypes.memset(p.k_cache.codes, 7, 16)
            self.calls.append(name)
            return 0

        return call


@pytest.fixture
def launches(monkeypatch):
    lib = Launches()
    monkeypatch.setattr(_lib, "require_gpu", lambda *t: torch.device("cpu"))
    monkeypatch.setattr(_lib, "load", lambda: lib)
    monkeypatch.setattr(_lib, "stream_handle", lambda dev: 0)
    monkeypatch.setattr(_lib, "timed_launch", lambda what, dev, f: f())
    monkeypatch.setattr(_lib, "on_device", lambda dev: contextlib.nullcontext())
    return lib


B, H, Hk, N, D, W = 2, 4, 2, 5, 40, 6


def cache(bits=4, slots=W + 1, b=B, hk=Hk, d=D):
    return df.quantized_cache(b, hk, slots, d, bits=bits, device="cpu")


def token(dtype=F32):
    return torch.ones(B, H, D, dtype=dtype), torch.ones(B, Hk, D, dtype=dtype), torch.ones(B, Hk, D, dtype=dtype)


def rows(dtype=F32):
    return torch.ones(B, Hk, N, D, dtype=dtype), torch.ones(B, Hk, N, D, dtype=dtype)


LENGTHS = torch.full((B,), N)


def test_a_cache_as_it_is_made():
    for bits, d, row in ((4, 128, 64), (8, 128, 128), (4, 80, 48), (8, 24, 32), (4, 1, 16)):
        c = df.quantized_cache(2, 3, 21, d, bits=bits, device="cpu")
        assert c.codes.shape == (2, 3, 21, row) and c.exponents.shape == (2, 3, -(-d // 32), 32) and c.bits == bits
        assert not c.codes.any() and not c.exponents.any()
    for kw in (dict(bits=2), dict(bits=8, slots=0), dict(bits=8, d=0), dict(bits=8, b=0)):
        with pytest.raises(ValueError):
            cache(**kw)


def test_calls_that_are_taken(launches):
    kc, vc = cache(), cache()
    before = kc.codes._version, kc.exponents._version, vc.codes._version, vc.exponents._version
    df.window_cache_fill(*rows(), LENGTHS, kc, vc, n_sink=1)
    df.window_cache_fill(*rows(BF), LENGTHS, kc, vc, n_sink=1, starts=LENGTHS.int())
    assert all(a > b for a, b in zip((kc.codes._version, kc.exponents._version, vc.codes._version, vc.exponents._version), before))
    K, V, mask = df.window_cache_read(kc, vc, LENGTHS, D, n_sink=1, dtype=F32)
    assert K.shape == V.shape == (B, Hk, W + 1, D) and mask.shape == (B, W + 1)
    q, k, v = token()
    assert torch.equal(df.window_decode_attn(q, k, v, kc, vc, LENGTHS, n_sink=1), q)
    plain = torch.zeros(B, Hk, W + 1, D)
    df.window_cache_fill(*rows(), LENGTHS, plain, plain.clone(), n_sink=1, starts=LENGTHS)
    df.window_cache_fill(*rows(), LENGTHS, plain, plain.clone(), n_sink=1)
    assert df.window_cache_read(plain, plain.clone(), LENGTHS, D, n_sink=1)[0].dtype == F32
    assert launches.calls == ["dfl_lowbit_cache_fill"] * 2 + ["dfl_window_cache_read", "dfl_lowbit_decode", "dfl_window_cache_append",
                                                             "dfl_window_cache_fill", "dfl_window_cache_read"]


def test_wrappers_refuse(launches):
    """Each refusal before any launch."""
    kc, vc, other = cache(), cache(), cache(8)
    plain = torch.zeros(B, Hk, W + 1, D)
    q, k, v = token()
    K, V = rows()

    def odd(c, **kw):
        return c._replace(**kw)

    shifted = torch.zeros(B * Hk * (W + 1) * 32 + 8, dtype=torch.uint8)[8:].view(B, Hk, W + 1, 32)
    calls = [
        (TypeError, lambda: df.window_cache_fill(K, V, LENGTHS, kc, plain, n_sink=1)),
        (ValueError, lambda: df.window_cache_fill(K, V, LENGTHS, kc, other, n_sink=1)),
        (ValueError, lambda: df.window_cache_fill(K, V, LENGTHS, kc, kc, n_sink=1)),
        (ValueError, lambda: df.window_cache_fill(K, V, LENGTHS, kc, odd(vc, exponents=kc.exponents), n_sink=1)),
        (ValueError, lambda: df.window_cache_fill(K, V, LENGTHS, odd(kc, bits=8), odd(vc, bits=8), n_sink=1)),
        (ValueError, lambda: df.window_cache_fill(K, V, LENGTHS, odd(kc, bits=3), odd(vc, bits=3), n_sink=1)),
        (TypeError, lambda: df.window_cache_fill(K, V, LENGTHS, odd(kc, codes=kc.codes.view(torch.int8)), vc, n_sink=1)),
        (ValueError, lambda: df.window_cache_fill(K, V, LENGTHS, odd(kc, codes=shifted), vc, n_sink=1)),
        (ValueError, lambda: df.window_cache_fill(K, V, LENGTHS, odd(kc, exponents=kc.exponents[..., :4]), vc, n_sink=1)),
        (ValueError, lambda: df.window_cache_fill(K, V, LENGTHS, odd(kc, exponents=kc.exponents[..., 1:]), vc, n_sink=1)),
        (ValueError, lambda: df.window_cache_fill(K, V, LENGTHS, odd(kc, codes=kc.codes[:1].expand(B, -1, -1, -1)), vc, n_sink=1)),
        (ValueError, lambda: df.window_cache_fill(K[:, :1], V[:, :1], LENGTHS, kc, vc, n_sink=1)),
        (ValueError, lambda: df.window_cache_fill(K, V, LENGTHS, kc, vc, n_sink=W + 1)),
        (ValueError, lambda: df.window_cache_fill(K, V, LENGTHS, kc, vc, n_sink=-1)),
        (ValueError, lambda: df.window_cache_fill(K, V, LENGTHS[:1], kc, vc, n_sink=1)),
        (ValueError, lambda: df.window_cache_fill(K, V, LENGTHS, kc, vc, n_sink=1, starts=LENGTHS[:1])),
        (ValueError, lambda: df.window_cache_fill(K, V, LENGTHS, kc, vc, n_sink=1, starts=LENGTHS.float())),
        (ValueError, lambda: df.window_cache_fill(K, V[:, :, :1], LENGTHS, kc, vc, n_sink=1)),
        (ValueError, lambda: df.window_cache_fill(K[:, :, :0], V[:, :, :0], LENGTHS, kc, vc, n_sink=1)),
        (ValueError, lambda: df.window_cache_fill(*[K[:, :, :1].expand(B, Hk, 2**32 + 5, D)] * 2, LENGTHS, kc, vc, n_sink=1)),
        (ValueError, lambda: df.window_cache_read(*[df.QuantizedCache(
            torch.empty(1, 1, 1, 16, dtype=torch.uint8).expand(1, 1, 2**32 + 5, 16),
            torch.empty(1, 1, 1, 1, dtype=torch.uint8).expand(1, 1, 1, 2**32 + 8), 4)] * 2, LENGTHS[:1], 8)),
        (TypeError, lambda: df.window_cache_fill(K, V.to(BF), LENGTHS, kc, vc, n_sink=1)),
        (TypeError, lambda: df.window_cache_fill(K.half(), V.half(), LENGTHS, kc, vc, n_sink=1)),
        (RuntimeError, lambda: df.window_cache_fill(K.clone().requires_grad_(), V, LENGTHS, kc, vc, n_sink=1)),
        (TypeError, lambda: df.window_cache_read(kc, plain, LENGTHS, D, n_sink=1)),
        (TypeError, lambda: df.window_cache_read(kc, vc, LENGTHS, D, n_sink=1, dtype=torch.float16)),
        (TypeError, lambda: df.window_cache_read(plain, plain.clone(), LENGTHS, D, n_sink=1, dtype=BF)),
        (ValueError, lambda: df.window_cache_read(plain, plain, LENGTHS, D, n_sink=1)),
        (ValueError, lambda: df.window_cache_read(kc, vc, LENGTHS, 65, n_sink=1)),
        (ValueError, lambda: df.window_cache_read(kc, vc, LENGTHS, 0, n_sink=1)),
        (ValueError, lambda: df.window_cache_read(kc, vc, LENGTHS[:1], D, n_sink=1)),
        (ValueError, lambda: df.window_decode_attn(q, k, v, kc, other, LENGTHS, n_sink=1)),
        (TypeError, lambda: df.window_decode_attn(q, k, v, plain, vc, LENGTHS, n_sink=1)),
        (TypeError, lambda: df.window_decode_attn(q.half(), k.half(), v.half(), kc, vc, LENGTHS, n_sink=1)),
        (TypeError, lambda: df.window_decode_attn(q, k.to(BF), v, kc, vc, LENGTHS, n_sink=1)),
        (ValueError, lambda: df.window_decode_attn(q[:, :3], k, v, kc, vc, LENGTHS, n_sink=1)),
        (ValueError, lambda: df.window_decode_attn(q[:, :0], k, v, kc, vc, LENGTHS, n_sink=1)),
        (ValueError, lambda: df.window_decode_attn(q, k, v, kc, vc, LENGTHS, n_sink=1, scale=0.0)),
        (ValueError, lambda: df.window_decode_attn(q, k, v, kc, vc, LENGTHS, n_sink=1, rel_table=torch.zeros(H, 3))),
        (RuntimeError, lambda: df.window_decode_attn(q.clone().requires_grad_(), k, v, kc, vc, LENGTHS, n_sink=1)),
    ]
    for i, (error, call) in enumerate(calls):
        with pytest.raises(error):
            call()
            pytest.fail(f"call {i} was taken")
    assert not launches.calls


def test_int8_wrappers_refuse(launches):
    x, w, s = torch.ones(3, 20), torch.zeros(4, 32, dtype=torch.int8), torch.ones(4)
    calls = [
        (ValueError, lambda: df.quantize_rows(x[0])), (ValueError, lambda: df.quantize_rows(x[:0])),
        (ValueError, lambda: df.quantize_rows(x[:, :0])), (ValueError, lambda: df.quantize_rows(torch.ones(1, 1).expand(1, 2**17 + 1))),
        (TypeError, lambda: df.quantize_rows(x.half())), (TypeError, lambda: df.quantize_rows(x.long())),
        (RuntimeError, lambda: df.quantize_rows(x.clone().requires_grad_())),
        (TypeError, lambda: df.int8_linear(x, w[:, :20].float(), s)), (TypeError, lambda: df.int8_linear(x.double(), w[:, :20], s)),
        (ValueError, lambda: df.int8_linear(x, w, s)), (ValueError, lambda: df.int8_linear(x, w[:, :20], s[:3])),
        (ValueError, lambda: df.int8_linear(x, w[:, :20], s.double())), (ValueError, lambda: df.int8_linear(x[:0], w[:, :20], s)),
        (ValueError, lambda: df.int8_linear(x, w[:, :20], s, torch.ones(3))),
        (ValueError, lambda: df.int8_linear(x, w[:, :20], s, torch.ones(4, dtype=torch.int8))),
        # rows that are not 16-byte aligned, or whose last piece lies behind the storage
        (ValueError, lambda: df.int8_linear(x, w[:, :20].contiguous(), s)), (ValueError, lambda: df.int8_linear(x, w[:, 8:28], s)),
        (ValueError, lambda: df.int8_linear(x, torch.zeros(3 * 32 + 20, dtype=torch.int8).as_strided((4, 20), (32, 1)), s)),
        (ValueError, lambda: df.int8_linear(x, torch.zeros(20, dtype=torch.int8)[None], s[:1])),
        (ValueError, lambda: df.int8_linear(x, w.t()[:20].t()[:, ::1].t().contiguous().t(), s)),
        (RuntimeError, lambda: df.int8_linear(x.clone().requires_grad_(), w[:, :20], s)),
        (ValueError, lambda: df.int8_linear(x[:1].expand(2**31, 20), w[:, :20], s)),
        (RuntimeError, lambda: df.int8_linear(x, w[:, :20], s, torch.ones(4).requires_grad_())),
    ]
    for i, (error, call) in enumerate(calls):
        with pytest.raises(error):
            call()
            pytest.fail(f"call {i} was taken")
    assert not launches.calls
    # what is taken: whole rows, views of them, one row, a batch of any shape
    assert df.int8_linear(torch.ones(2, 3, 32), w, s).shape == (2, 3, 4)
    assert df.int8_linear(x, torch.zeros(1, 32, dtype=torch.int8)[:, :20], s[:1]).shape == (3, 1)
    assert df.int8_linear(x[0], w[:, :20], s).shape == (4,)
    assert df.int8_linear(x, w.flatten()[:20].view(1, 20), s[:1]).shape == (3, 1)  # (one row in a longer storage)
    codes, scale = df.quantize_rows(x)
    assert codes.shape == (3, 20) and codes.stride() == (32, 1) and scale.shape == (3,)
    assert df.int8_linear(torch.ones(5, 20), codes, scale).shape == (5, 3)


def test_cpu_tensors_are_refused():
    kc, vc = cache(), cache()
    for call in (lambda: df.window_cache_fill(*rows(), LENGTHS, kc, vc, n_sink=1),
                 lambda: df.window_cache_read(kc, vc, LENGTHS, D, n_sink=1),
                 lambda: df.window_decode_attn(*token(), kc, vc, LENGTHS, n_sink=1),
                 lambda: df.quantize_rows(torch.ones(2, 16)),
                 lambda: df.int8_linear(torch.ones(2, 16), torch.zeros(2, 16, dtype=torch.int8), torch.ones(2))):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


def test_caches_that_share_memory(launches):
    """Interleaved caches (keys and values side by side) are taken, any common byte is not."""
    both = torch.zeros(B, Hk, W + 1, 2, 32, dtype=torch.uint8)
    exps = torch.zeros(B, Hk, 2, 2, 16, dtype=torch.uint8)
    kc = df.QuantizedCache(both[:, :, :, 0], exps[:, :, 0], 4)
    vc = df.QuantizedCache(both[:, :, :, 1], exps[:, :, 1], 4)
    window = window_attn._check_codes("t", kc, vc, B, Hk, D, 1)
    assert window == W
    for a, b in ((kc, vc._replace(codes=both[:, :, :, 0])), (kc, vc._replace(exponents=exps[:, :, 0])), (kc, kc)):
        with pytest.raises(ValueError, match="share memory"):
            window_attn._check_codes("t", a, b, B, Hk, D, 1)
    flat = torch.zeros(4096, dtype=torch.uint8)
    inside = df.QuantizedCache(flat[:B * Hk * (W + 1) * 32].view(B, Hk, W + 1, 32), flat[512:512 + B * Hk * 32].view(B, Hk, 2, 16), 4)
    with pytest.raises(ValueError, match="share memory"):
        window_attn._check_codes("t", inside, vc, B, Hk, D, 1)


def run(K, V, q, k, v, lengths, kc, ke, vc, ve, x, w, s):
    keys, vals = df.QuantizedCache(kc, ke, 4), df.QuantizedCache(vc, ve, 4)
    df.window_cache_fill(K, V, lengths, keys, vals, n_sink=1)
    o = df.window_decode_attn(q, k, v, keys, vals, lengths, n_sink=1)
    first = df.window_cache_read(keys, vals, lengths, D, n_sink=1, dtype=F32)[0]
    return o, first, df.int8_linear(x, w, s), df.quantize_rows(x)[0]


def test_a_trace_holds_the_launches(launches):
    def inputs():
        (kc, ke, _), (vc, ve, _) = cache(), cache()
        return (*rows(), *token(), LENGTHS.clone(), kc, ke, vc, ve, torch.rand(4, 16), torch.zeros(16, 16, dtype=torch.int8), torch.ones(16))

    traced = torch.jit.trace(run, inputs(), check_trace=False)
    before = len(launches.calls)
    x = inputs()
    o, first, y, codes = traced(*x)
    assert launches.calls[before:] == ["dfl_lowbit_cache_fill", "dfl_lowbit_decode", "dfl_window_cache_read", "dfl_int8_linear",
                                       "dfl_quantize_rows"]
    assert torch.equal(o, x[2]) and torch.equal(y, x[10]) and (x[6].flatten()[:16] == 7).all()


def test_forward_mode_is_refused(launches):
    dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
    kc, vc, (q, k, v), (K, V) = cache(), cache(), token(), rows()
    w, s, x = torch.zeros(16, 16, dtype=torch.int8), torch.ones(16), torch.ones(4, 16)
    with forward_ad.dual_level():
        for call in (lambda: df.window_cache_fill(dual(K), V, LENGTHS, kc, vc, n_sink=1),
                     lambda: df.window_decode_attn(dual(q), k, v, kc, vc, LENGTHS, n_sink=1),
                     lambda: df.window_decode_attn(q, k, dual(v), kc, vc, LENGTHS, n_sink=1),
                     lambda: df.window_cache_read(dual(K), V, LENGTHS, D),
                     lambda: df.int8_linear(dual(x), w, s), lambda: df.int8_linear(x, w, dual(s)), lambda: df.quantize_rows(dual(x))):
            with pytest.raises(NotImplementedError):
                call()
        assert torch.equal(df.window_decode_attn(q, k, v, kc, vc, LENGTHS, n_sink=1), q)
