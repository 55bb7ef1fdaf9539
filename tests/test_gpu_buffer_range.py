"""What gfx950 takes to be outside a raw buffer: the rule that keeps the few-bit decode's loads (csrc/lowbit_decode.hip) inside
its caches, whose results show nothing of it.  All addresses lie in one allocation, whatever the rule."""

import ctypes
import os

import pytest
import torch

from conftest import PKG_ROOT

pytestmark = pytest.mark.gpu


def probe(memory, base, size, lanes, scalars):
    lib = ctypes.CDLL(os.path.join(PKG_ROOT, "deepfold_amd", "libdfl_peaks.so"))
    lib.dfl_probe_buffer_range.argtypes = [ctypes.c_void_p, ctypes.c_int, *[ctypes.c_void_p] * 2, ctypes.c_int, ctypes.c_void_p]
    assert len(lanes) == 64 and base + int(lanes.max()) + int(scalars.max()) + 16 <= memory.numel()
    out = torch.full((len(scalars), 64, 5), -1, dtype=torch.int32, device=memory.device)
    ld, sd = (t.to(torch.uint32).to(memory.device) for t in (lanes, scalars))
    torch.cuda.synchronize()
    assert lib.dfl_probe_buffer_range(memory.data_ptr() + base, size, ld.data_ptr(), sd.data_ptr(), len(scalars), out.data_ptr()) == 0
    return out.cpu()


@pytest.mark.parametrize("size", [0, 16, 64, 68, 1000, 4096, 28 * 4112, 1 << 20])
def test_a_load_is_outside_by_both_offsets(size):
    """Lane and scalar offset count together, dword by dword; a scalar offset beyond the size leaves nothing inside."""
    memory = torch.randint(1, 256, (8 << 20,), generator=torch.Generator().manual_seed(size)).to(torch.uint8)
    near = [0, 4, 16, 60, 64, 100, size // 2 // 4 * 4, *(size + k for k in range(-64, 72, 4))]
    lanes = sorted({x for x in near if 0 <= x})[:60]
    lanes = torch.tensor(lanes + [1 << 20, 3 << 20] + [0] * (62 - len(lanes)), dtype=torch.int64)
    scalars = torch.tensor([0, 16, 64, 1024, 4112, *(max(0, size + k) for k in (-1024, -64, -16, -4, 0, 4, 16, 64, 1024)), 1 << 20, 3 << 20,
                            (4 << 20) - 16], dtype=torch.int64)
    base = 1 << 19
    at = lanes[None, :] + scalars[:, None]
    out = probe(memory.to("cuda:0"), base, size, lanes, scalars)
    dwords = memory.view(torch.int32)
    for i in range(4):
        want = torch.where(at + 4 * i + 4 <= size, dwords[(base + at + 4 * i) // 4], 0)
        assert torch.equal(out[..., i], want), i
    want = torch.where(at + 1 <= size, memory[base + at].int(), 0)
    assert torch.equal(out[..., 4], want)


def test_a_lane_that_reads_nothing():
    """A lane offset of 2^31 is outside with every scalar offset."""
    top = 1 << 31
    memory = torch.full((top + (1 << 26),), 7, dtype=torch.uint8, device="cuda:0")
    lanes = torch.full((64,), top, dtype=torch.int64) + 16 * torch.arange(64)
    scalars = torch.tensor([0, 16, 1024, 4096, 1 << 20, 1 << 25], dtype=torch.int64)
    for size in (0, 64, 1 << 20, 1 << 30, (1 << 31) - 4):
        assert not probe(memory, 0, size, lanes, scalars).any(), size
