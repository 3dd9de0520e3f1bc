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
