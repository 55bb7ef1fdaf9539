"""CPU checks of the float64 forms of the sequence operators (oracle/window.py) against loops and
differences, of the bucket edges, and of what the operators and the C ABI refuse."""

import ctypes
import math
import os
import re
import subprocess

import pytest
import torch

from conftest import ROOT
from oracle import window as ref

EDGES = (1, 2, 3, 5, 9)


def rnd(*shape, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)


def loop_attention(q, k, v, window, n_sink, causal, mask, table, scale):
    B, H, M, d = q.shape
    Hk, N = k.shape[1], k.shape[2]
    o = torch.zeros_like(q)
    for b in range(B):
        for h in range(H):
            for i in range(M):
                t, seen = i + N - M, []
                for j in range(N):
                    near = t - window < j <= t if causal else abs(t - j) < window
                    first = j < n_sink and (j <= t or not causal)
                    if (near or first) and (mask is None or (mask[b, j] and mask[b, t])):
                        s = float(q[b, h, i] @ k[b, h // (H // Hk), j]) * scale
                        if table is not None:
                            mag = abs(j - t) if not causal else max(t - j, 0)
                            n = sum(mag >= e for e in EDGES) + (len(EDGES) + 1 if not causal and j > t else 0)
                            s += float(table[h, n])
                        if s > -1e30:
                            seen.append((s, j))
                if not seen:
                    continue
                top = max(s for s, _ in seen)
                w = [math.exp(s - top) for s, _ in seen]
                o[b, h, i] = sum(x * v[b, h // (H // Hk), j] for x, (_, j) in zip(w, seen)) / sum(w)
    return o


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("M,N,window,n_sink,masked", [(7, 7, 3, 0, False), (5, 9, 2, 2, True), (1, 6, 1, 0, False),
                                                      (8, 8, 50, 3, True), (1, 1, 1, 1, False)])
def test_attention_against_loops_and_differences(M, N, window, n_sink, masked, causal):
    B, H, Hk, d = 2, 4, 2, 3
    q, k, v, go = rnd(B, H, M, d, seed=1), rnd(B, Hk, N, d, seed=2), rnd(B, Hk, N, d, seed=3), rnd(B, H, M, d, seed=4)
    table = rnd(H, (len(EDGES) + 1) * (1 if causal else 2), seed=5)
    mask = torch.ones(B, N)
    if masked:
        mask[0, N // 2:] = 0
        mask[1, 0] = 0
    kw = dict(window=window, n_sink=n_sink, causal=causal, mask=mask if masked else None, scale=0.7, edges=EDGES)
    got = ref.attention(q, k, v, table=table, grad=go, **kw)
    want = loop_attention(q, k, v, window, n_sink, causal, mask if masked else None, table, 0.7)
    assert torch.allclose(got["o"][0], want, rtol=1e-12, atol=1e-12)
    step = 1e-6
    for name, x in (("dq", q), ("dk", k), ("dv", v), ("dtable", table)):
        flat = x.view(-1)
        for e in range(0, flat.numel(), max(1, flat.numel() // 17)):
            keep = float(flat[e])
            sums = []
            for sign in (1, -1):
                flat[e] = keep + sign * step
                sums.append(float((ref.attention(q, k, v, table=table, **kw)["o"][0] * go).sum()))
            flat[e] = keep
            # central differences: error step^2 of the third derivative, 1e-16 / step of the rounding
            assert abs((sums[0] - sums[1]) / (2 * step) - float(got[name][0].reshape(-1)[e])) < 1e-7, name


def test_rel_bias_and_its_gradient():
    H, M, N = 2, 4, 6
    table = rnd(H, 2 * (len(EDGES) + 1), seed=1)
    rel = torch.randint(-12, 13, (3, M, N), generator=torch.Generator().manual_seed(2))
    out = ref.rel_bias(table, EDGES, rel, True)
    g = rnd(3, H, M, N, seed=3)
    dt, _ = ref.rel_bias_grad(g, EDGES, rel, True, table.shape[1])
    want = torch.zeros_like(table)
    for b in range(3):
        for i in range(M):
            for j in range(N):
                r = int(rel[b, i, j])
                n = sum(abs(r) >= e for e in EDGES) + (len(EDGES) + 1 if r > 0 else 0)
                assert torch.equal(out[b, :, i, j], table[:, n])
                want[:, n] += g[b, :, i, j]
    assert torch.allclose(dt, want, rtol=1e-13, atol=1e-13)


@pytest.mark.parametrize("n_sink,window", [(0, 4), (2, 3), (3, 1)])
def test_decode_is_the_last_row_of_the_attention(n_sink, window):
    """A prompt of every length, filled and then continued, gives the rows of the whole attention."""
    B, H, Hk, N, d = 1, 4, 2, 11, 3
    q, k, v = rnd(B, H, N, d, seed=1), rnd(B, Hk, N, d, seed=2), rnd(B, Hk, N, d, seed=3)
    table = rnd(H, len(EDGES) + 1, seed=4)
    want = ref.attention(q, k, v, window=window, n_sink=n_sink, table=table, edges=EDGES)["o"][0]
    for start in range(N):
        zero = torch.zeros(B, Hk, n_sink + window, d, dtype=torch.float64)
        kc, vc = ref.fill(k, v, [start], zero, zero, n_sink)
        for t in range(start, N):
            o, _, kc, vc = ref.decode(q[:, :, t], k[:, :, t], v[:, :, t], kc, vc, [t], n_sink, table=table, edges=EDGES)
            assert torch.allclose(o, want[:, :, t], rtol=1e-12, atol=1e-12)


@pytest.mark.parametrize("n,far,both", [(32, 128, True), (32, 128, False), (16, 1000, True), (90, 500, True), (4, 3, True),
                                        (2, 2, False), (96, 2048, False)])
def test_bucket_edges(n, far, both):
    from fractions import Fraction

    from deepfold_amd import relative_bucket_edges

    edges = relative_bucket_edges(n, far, both)
    side = n // 2 if both else n
    exact = max(1, side // 2)
    assert len(edges) == side - 1 and list(edges[:exact]) == list(range(1, exact + 1))
    assert all(b > a for a, b in zip(edges, edges[1:])) and edges[-1] < max(far, edges[-2] + 2 if len(edges) > 1 else 2)
    for k, e in enumerate(edges[exact:], 1):  # the first distance at or past the k-th ratio, or pushed by the one before
        L = side - exact
        past = lambda d: Fraction(d, exact) ** L >= Fraction(far, exact) ** k
        assert past(e) and (not past(e - 1) or e == edges[exact + k - 2] + 1)


def test_refusals_of_arguments():
    """What the wrappers refuse they refuse before any tensor reaches the GPU: CPU tensors serve."""
    import deepfold_amd as df

    q, k = torch.zeros(1, 4, 6, 8), torch.zeros(1, 2, 6, 8)
    t6 = torch.zeros(4, 6)
    att = df.flash_window_attn
    for err, call in (
            (ValueError, lambda: att(q, k, k, window=0)),
            (ValueError, lambda: att(q, k, k, window=4, n_sink=-1)),
            (ValueError, lambda: att(q, k, k, window=4, n_sink=129)),
            (ValueError, lambda: att(q, torch.zeros(1, 3, 6, 8), torch.zeros(1, 3, 6, 8), window=4)),
            (ValueError, lambda: att(q, k[:, :, :4], k[:, :, :4], window=4)),
            (ValueError, lambda: att(q, k, k[..., :4], window=4)),
            (ValueError, lambda: att(q[0], k, k, window=4)),
            (ValueError, lambda: att(q, k, k, torch.ones(1, 5), window=4)),
            (ValueError, lambda: att(q, k, k, window=4, rel_table=t6)),
            (ValueError, lambda: att(q, k, k, window=4, rel_table=t6, rel_edges=(1, 2))),
            (ValueError, lambda: att(q, k, k, window=4, rel_table=t6, rel_edges=(1, 2, 2, 3, 4))),
            (ValueError, lambda: att(q, k, k, window=4, rel_table=t6, rel_edges=(0, 1, 2, 3, 4))),
            (ValueError, lambda: att(q, k, k, window=4, rel_table=t6, rel_edges=(1, 2, 3, 4, 2049))),
            (ValueError, lambda: att(q, k, k, window=4, causal=False, rel_table=t6, rel_edges=(1, 2, 3, 4, 5))),
            (ValueError, lambda: att(q, k, k, window=4, rel_table=torch.zeros(4, 97), rel_edges=tuple(range(1, 97)))),
            (TypeError, lambda: att(q, k, k, window=4, rel_table=t6.int(), rel_edges=(1, 2, 3, 4, 5))),
            (TypeError, lambda: att(q.int(), k.int(), k.int(), window=4)),
            (ValueError, lambda: att(torch.zeros(1, 1, 1, 129), torch.zeros(1, 1, 1, 129), torch.zeros(1, 1, 1, 129),
                                     window=4)),
            (ValueError, lambda: att(q, k, k, window=4, scale=-1.0)),
            (ValueError, lambda: att(q, k, k, window=4, scale=0)),
            (ValueError, lambda: att(q, k, k, window=4, scale=math.nan)),
            (RuntimeError, lambda: att(q, k, k, window=4)),
            (ValueError, lambda: df.rel_pos_bias(t6, (1, 2, 3), 4)),
            (ValueError, lambda: df.rel_pos_bias(t6, (1, 2), 0)),
            (ValueError, lambda: df.rel_pos_bias(t6, (), 4)),
            (TypeError, lambda: df.rel_pos_bias(t6, (1, 2), 4, dtype=torch.float16)),
            (TypeError, lambda: df.rel_pos_bias(t6, (1, 2), 4, q_pos=torch.zeros(4))),
            (ValueError, lambda: df.rel_pos_bias(t6, (1, 2), 4, 5, q_pos=torch.zeros(4, dtype=torch.int32))),
            (ValueError, lambda: df.rel_pos_bias(t6, (1, 2), 4, 5, q_pos=torch.zeros(2, 4, dtype=torch.int32),
                                                 k_pos=torch.zeros(3, 5, dtype=torch.int32))),
            (ValueError, lambda: df.relative_bucket_edges(3, 128)),
            (ValueError, lambda: df.relative_bucket_edges(32, 8)),
            (ValueError, lambda: df.relative_bucket_edges(200, 128))):
        with pytest.raises(err):
            call()


def test_refusals_of_caches():
    import deepfold_amd as df
    from deepfold_amd import window_attn as wa

    kc, vc = torch.zeros(2, 2, 5, 8), torch.zeros(2, 2, 5, 8)
    ok = lambda a, b, **kw: wa._check_caches("t", a, b, 2, 2, 8, kw.get("dtype", torch.float32), kw.get("n_sink", 1))
    assert ok(kc, vc) == 4
    both = torch.zeros(2, 5, 2, 2, 8)  # keys and values side by side, slots outermost: a layout of its own
    assert ok(both[:, :, :, 0].transpose(1, 2), both[:, :, :, 1].transpose(1, 2)) == 4
    for err, a, b, kw in ((ValueError, kc, vc, dict(n_sink=5)), (TypeError, kc, vc, dict(dtype=torch.bfloat16)),
                          (ValueError, kc, kc, {}), (ValueError, kc[:, :, :, :7], vc[:, :, :, :7], {}),
                          (ValueError, kc[:1], vc[:1], {}), (ValueError, kc[:1].expand(2, 2, 5, 8), vc, {}),
                          (ValueError, kc.transpose(2, 3).contiguous().transpose(2, 3), vc, {}),
                          (TypeError, kc.half(), vc.half(), dict(dtype=torch.float16))):
        with pytest.raises(err):
            ok(a, b, **kw)
    q, k, n = torch.zeros(2, 4, 8), torch.zeros(2, 2, 8), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU"):
        df.window_decode_attn(q, k, k, kc, vc, n, n_sink=1)
    with pytest.raises(RuntimeError, match="GPU"):
        df.window_cache_fill(torch.zeros(2, 2, 3, 8), torch.zeros(2, 2, 3, 8), n, kc, vc, n_sink=1)
    with pytest.raises(RuntimeError, match="no gradient"):
        df.window_decode_attn(q.requires_grad_(True), k, k, kc, vc, n, n_sink=1)


def test_parameter_blocks_match_the_header():
    from deepfold_amd import _lib

    header = os.path.join(ROOT, "include", "dfl_window.h")
    text = re.sub(r"/\*.*?\*/", "", open(header).read(), flags=re.S)
    mirrors = {"dfl_window_attn_params": _lib.WindowAttnParams,
               "dfl_window_cache_fill_params": _lib.WindowCacheFillParams,
               "dfl_window_decode_params": _lib.WindowDecodeParams, "dfl_rel_bias_params": _lib.RelBiasParams}
    bodies = {name: body for body, name in re.findall(r"typedef struct \w+ \{(.*?)\} (\w+);", text, flags=re.S)}
    assert set(bodies) == set(mirrors)
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{header}"', "int main(void) {"]
    for name, cls in mirrors.items():
        lines.append(f'printf("%zu", sizeof({name}));')
        lines += [f'printf(" %zu", offsetof({name}, {f}));' for f, _ in cls._fields_]
        lines.append('printf("\\n");')
    src = os.path.join(os.environ.get("TMPDIR", "/tmp"), f"dfl_window_probe_{os.getpid()}")
    try:
        open(src + ".c", "w").write("\n".join(lines + ["return 0; }"]))
        subprocess.run(["gcc", "-std=c99", "-o", src, src + ".c"], check=True)
        got = subprocess.run([src], capture_output=True, text=True, check=True).stdout.splitlines()
    finally:
        for f in (src, src + ".c"):
            if os.path.exists(f):
                os.remove(f)
    for line, (name, cls) in zip(got, mirrors.items()):
        size, *at = map(int, line.split())
        assert ctypes.sizeof(cls) == size, name
        assert [getattr(cls, f).offset for f, _ in cls._fields_] == at, name
        declared = [n.strip(" *") for d in bodies[name].split(";") if d.strip()
                    for n in re.sub(r"^\s*(const\s+)?(long long|\w+)\s*\**", "", d.strip()).split(",")]
        assert [f for f, _ in cls._fields_] == declared, name


def test_c_entries_refuse():
    """Argument errors of the C entries come before any GPU call: the pointers are never read."""
    from deepfold_amd import _lib

    lib = _lib.load()
    fake = 4096
    edges, flat = (ctypes.c_int * 3)(1, 2, 4), (ctypes.c_int * 2)(3, 3)
    good = dict(dtype=_lib.DFL_BF16, q=fake, k=fake, v=fake, B=1, H=4, Hk=2, M=8, N=8, d=64, window=4, n_sink=0, causal=1,
                scale=1.0, o=fake)
    for bad, text in ((dict(dtype=7), "dtype"), (dict(Hk=3), "multiple"), (dict(d=129), "head dim"), (dict(M=9), "M <= N"),
                      (dict(window=0), "window"), (dict(n_sink=129), "n_sink"), (dict(q=None), "NULL"), (dict(scale=0.0), "scale"), (dict(scale=math.inf), "scale"),
                      (dict(rel_table=fake), "together"),
                      (dict(rel_table=fake, rel_edges=ctypes.addressof(flat), n_edges=2), "ascend"),
                      (dict(N=1 << 29, M=1), "M <= N"), (dict(B=1 << 21), "too large")):
        p = _lib.WindowAttnParams(**{**good, **bad})
        assert lib.dfl_window_attn_fwd(ctypes.byref(p), None) < 0
        assert text in lib.dfl_last_error().decode(), bad
    p = _lib.WindowAttnParams(**good)
    assert lib.dfl_window_attn_bwd(ctypes.byref(p), fake, 1 << 30, None) < 0
    grads = dict(lse=fake, grad_o=fake, dq=fake, dk=fake, dv=fake)
    p = _lib.WindowAttnParams(**good, **grads)
    need = lib.dfl_window_attn_workspace_size(1, 4, 2, 8, 8, 64, 4, 0, 1, 0)
    assert lib.dfl_window_attn_bwd(ctypes.byref(p), fake, need - 1, None) < 0
    assert "workspace too small" in lib.dfl_last_error().decode()
    p = _lib.WindowAttnParams(**good, **grads, drel_table=fake)
    assert lib.dfl_window_attn_bwd(ctypes.byref(p), fake, need, None) < 0
    assert lib.dfl_window_attn_fwd(None, None) < 0
    f = _lib.WindowCacheFillParams(dtype=1, k=fake, v=fake, lengths=fake, k_cache=fake, v_cache=fake, B=70000, Hk=1, N=4,
                                   d=8, window=4, n_sink=0)
    assert lib.dfl_window_cache_fill(ctypes.byref(f), None) < 0 and "65535" in lib.dfl_last_error().decode()
    d = _lib.WindowDecodeParams(dtype=1, q=fake, k=fake, v=fake, k_cache=fake, v_cache=fake, lengths=fake, B=1, H=2, Hk=2,
                                d=64, window=4096, n_sink=4, scale=1.0, o=fake)
    need = lib.dfl_window_decode_workspace_size(1, 2, 2, 64, 4096, 4)
    assert need > 0 and lib.dfl_window_decode(ctypes.byref(d), fake, need - 1, None) < 0
    r = _lib.RelBiasParams(dtype=0, rel_table=fake, rel_edges=ctypes.addressof(edges), n_edges=3, rel_both=1, q_pos=fake,
                           B=1, H=2, M=4, N=4, out=fake)
    assert lib.dfl_rel_bias_fwd(ctypes.byref(r), None) < 0 and "together" in lib.dfl_last_error().decode()
