"""Scratch memory in stream order, 16-bit decode: a workspace may be what the kernel
before the call still reads (an append's tokens, freed since)."""

from __future__ import annotations

import pytest
import torch

from barellm_b200 import ops

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.mark.parametrize("n", [1, 40])
def test_a_workspace_may_be_what_the_append_read(cuda, native_lib, n):
    batch, hkv, bs, d, per_row = 300, 8, 16, 128, 10
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)
    lens = [(b * 7) % 90 for b in range(batch)]
    g = torch.Generator(device=cuda).manual_seed(n)
    pools = [torch.randn(1, batch * per_row, hkv, bs, d, generator=g, device=cuda).to(BF16) for _ in range(2)]
    bt = torch.randperm(batch * per_row, generator=g, device=cuda).to(torch.int32).view(batch, per_row)
    q = torch.randn(batch, 2 * hkv, d, generator=g, device=cuda).to(BF16)
    start, seq, off = i32(lens), i32([x + n for x in lens]), i32([b * n for b in range(batch + 1)])
    bytes_kv = batch * n * hkv * d * 2
    need = ops.decode_workspace_bytes(batch, 2 * hkv, d, bs, 512)
    last = (bytes_kv - 20 * n * hkv * d * 2) // 256 * 256  # the scratch begins at the tokens that are appended last
    buf = torch.zeros(last + max(need, bytes_kv - last), dtype=torch.uint8, device=cuda)
    k = buf[:bytes_kv].view(BF16).view(1, batch * n, hkv, d).transpose(1, 2)
    tokens = torch.randn(k.shape, generator=g, device=cuda).to(BF16)
    clean = [p.clone() for p in pools]
    ops.paged_append(*clean, 0, bt, start, tokens, tokens, new_offsets=off, max_new_tokens=n)
    want = ops.paged_decode(q, *clean, 0, bt, seq, 512)
    for _ in range(20):
        k.copy_(tokens)
        got = [p.clone() for p in pools]
        ops.paged_append(*got, 0, bt, start, k, k, new_offsets=off, max_new_tokens=n)
        out = ops.paged_decode(q, *got, 0, bt, seq, 512, ws=buf[last:])
        assert all(torch.equal(a, b) for a, b in zip(got, clean))
        assert torch.equal(out, want)


def test_records_that_are_no_plan_are_skipped(cuda, native_lib):
    """A workspace whose header is a plan's and whose records are not: rows and chunks outside the batch, also
    chunks whose first block overflows 32 bits, are flagged and skipped; the other rows keep their results."""
    from barellm_b200 import _native as nat

    batch, n, hkv, hq = 20, 700, 2, 8
    g = torch.Generator(device=cuda).manual_seed(0)
    pools = [torch.randn(1, batch * 44, hkv, 16, 128, generator=g, device=cuda).to(BF16) for _ in range(2)]
    bt = torch.randperm(batch * 44, generator=g, device=cuda).to(torch.int32).view(batch, 44)
    q = torch.randn(batch, hq, 128, generator=g, device=cuda).to(BF16)
    seq = torch.full((batch,), n, dtype=torch.int32, device=cuda)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    ws = torch.zeros(ops.decode_workspace_bytes(batch, hq, 128, 16, n), dtype=torch.uint8, device=cuda)
    call = lambda out, ready: ops.paged_decode(q, *pools, 0, bt, seq, n, ws=ws, plan_ready=ready, out=out, err=err)
    want = call(torch.empty_like(q), False).clone()
    good, words = ws.clone(), ws.view(torch.int32)
    units = words[512 // 4:][:2 * 2 * batch].view(2 * batch, 2)  # row, chunk
    assert words[0] == 2 * batch and sorted(units[:, 0].tolist()) == sorted(2 * list(range(batch)))
    for field, value in ((0, batch), (0, -1), (0, 2 ** 31 - 1), (1, -1), (1, 2), (1, 2 ** 26), (1, 2 ** 27), (1, 2 ** 31 - 1)):
        for record in (0, 2 * batch - 1):
            ws.copy_(good)
            hit = int(units[record, 0])
            units[record, field] = value
            out = torch.full_like(want, 9.0)
            err.zero_()
            call(out, True)
            assert int(err) & nat.BL_DEVERR_WORKSPACE, (field, value)
            others = [b for b in range(batch) if b != hit]
            assert torch.equal(out[others], want[others]), (field, value)
    ws.copy_(good)
    err.zero_()
    assert torch.equal(call(torch.empty_like(q), True), want) and int(err) == 0
