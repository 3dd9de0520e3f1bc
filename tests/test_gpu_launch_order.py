"""A call's lengths and row ids in stream order: the kernel just ahead of a decode may
write them, and may let the decode's kernels launch long before it does."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from barellm_b200 import ops
from fp8_helpers import filled, i32
from oracle import fp8_oracle as f8

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32

LENS = [1 + (b * 97) % 1900 for b in range(40)]
LENS = [n + 1 if n & 0xFF in (0x7F, 0x80, 0xFF) else n for n in LENS]  # (their bytes are codes of numbers)
ROWS = [(b * 7 + 3) % 40 for b in range(40)]


class LateWriter:
    """int32 values that a kernel of this library writes: the last codes of one long
    block, quantised from the values that these codes stand for.  One warp writes the
    block front to back, hundreds of microseconds after it has let the next kernel launch."""

    def __init__(self, device, values, tokens=16384):
        want = np.asarray(values, dtype=np.int32).view(np.uint8)
        assert not np.isnan(f8.VALUES[want]).any()
        codes = np.zeros(tokens * 16, dtype=np.uint8)
        codes[0] = 0x7E  # the largest code: the block's scale is 1
        codes[-len(want):] = want
        x = torch.from_numpy(f8.VALUES[codes].astype(np.float32)).to(device).view(1, 1, tokens, 16)
        self.pools = [torch.zeros((1, 1, 1, tokens, 16), dtype=torch.uint8, device=device).view(ops.FP8_DTYPE) for _ in range(2)]
        scales = [torch.ones((1, 1, 1), device=device) for _ in range(2)]
        self.args = (*self.pools, *scales, 0, i32([0], device).view(1, 1), i32([0], device), x, x)
        self.values = self.pools[0].view(torch.uint8).view(-1)[-len(want):].view(torch.int32)

    def write(self):
        ops.paged_append_fp8(*self.args)


@pytest.mark.parametrize("before", [0, 1900])
@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("kind", ["fp8", "fp8_f32", "bf16"])
def test_lengths_written_by_the_kernel_just_ahead(cuda, native_lib, kind, captured, before):
    hkv, hq, d, most = 2, 8, 128, 1920
    dtype = F32 if kind == "fp8_f32" else BF16
    table_lens = [1900 + 20] * 40  # (every row's table covers the longest)
    pool, table, bt = filled(cuda, table_lens, hkv, 16, d, dtype, layers=1, layer=0)
    q = torch.randn(40, hq, d, generator=torch.Generator().manual_seed(3)).to(dtype).to(cuda)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    if kind == "bf16":
        g = torch.Generator(device=cuda).manual_seed(4)
        cache = [torch.randn(pool.dev[0].shape, generator=g, device=cuda).to(BF16) for _ in range(2)]
        ws = torch.zeros(ops.decode_workspace_bytes(40, hq, d, 16, most), dtype=torch.uint8, device=cuda)
        call = lambda seq, rows: ops.paged_decode(q, *cache, 0, bt, seq, most, row_ids=rows, ws=ws, err=err)
    else:
        ws = torch.zeros(ops.decode_fp8_workspace_bytes(40, hq, d, most), dtype=torch.uint8, device=cuda)
        call = lambda seq, rows: ops.paged_decode_fp8(q, *pool.args, 0, bt, seq, most, row_ids=rows, ws=ws, err=err)
    want = call(i32(LENS, cuda), i32(ROWS, cuda)).clone()
    late = LateWriter(cuda, LENS + ROWS)
    seq, rows = late.values[:40], late.values[40:]

    def step():
        late.write()
        return call(seq, rows)

    if captured:
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            out = step()
    for _ in range(5):
        late.pools[0].view(torch.uint8).zero_()
        seq.fill_(before)
        if captured:
            graph.replay()
        else:
            out = step()
        torch.cuda.synchronize()
        assert seq.tolist() == LENS and rows.tolist() == ROWS
        assert torch.equal(out, want)
    assert int(err) == 0


@pytest.mark.parametrize("captured", [False, True])
def test_lengths_that_grow_on_the_device(cuda, native_lib, captured):
    """A serving step that counts its lengths up on the device, then attends."""
    lens = [1 + (b * 61) % 700 for b in range(50)]
    pool, table, bt = filled(cuda, [n + 8 for n in lens], 2, 16, 128, BF16, layers=1, layer=0)
    q = torch.randn(50, 8, 128, generator=torch.Generator().manual_seed(5)).to(BF16).to(cuda)
    seq = i32(lens, cuda)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)

    def step():
        seq.add_(1)
        return ops.paged_decode_fp8(q, *pool.args, 0, bt, seq, 720, err=err)

    if captured:
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            out = step()
        torch.cuda.synchronize()
        seq.copy_(i32(lens, cuda))
    for n in range(1, 6):
        if captured:
            graph.replay()
        else:
            out = step()
        got = out.clone()
        want = ops.paged_decode_fp8(q, *pool.args, 0, bt, i32([x + n for x in lens], cuda), 720)
        assert torch.equal(got, want)
    assert int(err) == 0


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("most", [500, 1920, 6000])
def test_lengths_written_just_ahead_of_a_small_call(cuda, native_lib, most, captured):
    """Calls without a plan: rows of one chunk, rows joined within clusters, rows joined by a kernel."""
    lens, order = [min(n, most) for n in (300, 1500, 1, 777)], [2, 0, 3, 1]
    pool, table, bt = filled(cuda, [1920] * 4, 2, 16, 128, BF16, layers=1, layer=0)
    q = torch.randn(4, 8, 128, generator=torch.Generator().manual_seed(3)).to(BF16).to(cuda)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    call = lambda seq, rows: ops.paged_decode_fp8(q, *pool.args, 0, bt, seq, most, row_ids=rows, err=err)
    want = call(i32(lens, cuda), i32(order, cuda)).clone()
    late = LateWriter(cuda, lens + order)
    seq, rows = late.values[:4], late.values[4:]
    if captured:
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            late.write()
            out = call(seq, rows)
    for _ in range(5):
        late.pools[0].view(torch.uint8).zero_()
        if captured:
            graph.replay()
        else:
            late.write()
            out = call(seq, rows)
        assert torch.equal(out, want)
    assert int(err) == 0
