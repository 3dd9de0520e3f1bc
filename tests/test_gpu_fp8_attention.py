"""Decode and chunked prefill over 8-bit pages against float64 attention on the
stored values; the bounds follow from the kernels' arithmetic
(fp8_helpers.attention_bound)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from barellm_b200 import _native as nat
from barellm_b200 import ops
from fp8_helpers import Pool, assert_within, attention_bound, filled, i32
from oracle import fp8_oracle as f8

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def check_decode(out, q, pool, table, lens, layer, scale=None):
    eps = 2.0 ** -11 if q.dtype is not F32 else 0.0  # P in fp16 on the tensor cores
    qn, got = q.double().cpu().numpy(), out.double().cpu().numpy()
    for b, n in enumerate(lens):
        k, v = (f8.read(c, s, layer, table[b], n) for c, s in zip(pool.codes, pool.scales))
        want, spread, reach, flat = f8.attention(qn[b][:, None], k, v, scale)
        assert_within(got[b][:, None], want, attention_bound(want, spread, reach, flat, qn[b][:, None], q.dtype, eps, n))


SHAPES = [  # hq, hkv, bs, d
    (16, 8, 16, 128), (32, 8, 16, 128), (8, 8, 16, 128), (16, 1, 16, 128), (12, 4, 16, 128), (20, 2, 32, 128), (8, 2, 48, 128),
    (16, 8, 16, 64), (9, 1, 16, 64), (8, 2, 16, 256), (11, 1, 32, 256), (12, 4, 8, 128), (4, 2, 16, 80), (6, 3, 5, 3), (2, 1, 1, 256),
]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("hq,hkv,bs,d", SHAPES)
def test_decode(cuda, native_lib, dtype, hq, hkv, bs, d):
    lens = [1, 0, 15, 16, 17, 31, 33, 511, 512, 513, 1100]
    pool, table, bt = filled(cuda, lens, hkv, bs, d, dtype, seed=hq * 7 + d)
    q = torch.randn(len(lens), hq, d, generator=torch.Generator().manual_seed(d)).to(dtype).to(cuda)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    out = ops.paged_decode_fp8(q, *pool.args, 1, bt, i32(lens, cuda), 1100, err=err)
    assert int(err) == 0
    assert bool((out[1] == 0).all())
    check_decode(out, q, pool, table, lens, 1)


@pytest.mark.parametrize("max_len", [5, 512])
def test_decode_short_rows_and_no_rows(cuda, native_lib, max_len):
    """Calls whose rows all fit one chunk have no join kernel; empty rows are zeros there too."""
    lens = [0, 5, 1, 0, max_len]
    pool, table, bt = filled(cuda, lens, 8, 16, 128, BF16)
    q = torch.randn(5, 16, 128, device=cuda).to(BF16)
    out = torch.full((5, 16, 128), 9.0, dtype=BF16, device=cuda)
    ops.paged_decode_fp8(q, *pool.args, 1, bt, i32(lens, cuda), max_len, out=out)
    check_decode(out, q, pool, table, lens, 1)
    out.fill_(9.0)
    ops.paged_decode_fp8(q, *pool.args, 1, bt, i32([0] * 5, cuda), max_len, out=out)
    assert bool((out == 0).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_decode_long_row(cuda, native_lib, dtype):
    lens = [20000, 3]
    pool, table, bt = filled(cuda, lens, 2, 16, 128, dtype, layers=1, layer=0)
    q = torch.randn(2, 8, 128, device=cuda).to(dtype)
    out = ops.paged_decode_fp8(q, *pool.args, 0, bt, i32(lens, cuda), 20000)
    check_decode(out, q, pool, table, lens, 0)


@pytest.mark.parametrize("d", [16, 48, 80, 96, 112, 144, 208, 240])
@pytest.mark.parametrize("pad", [0, 4, 1])
def test_decode_head_dims_between(cuda, native_lib, d, pad):
    """Head dims that are multiples of 16: the columns behind them are neither read as values nor written."""
    lens = [3, 0, 512, 1100, 40]
    pool, table, bt = filled(cuda, lens, 2, 16, d, BF16)
    q = torch.full((len(lens), 6, d + pad), float("nan"), dtype=BF16, device=cuda)[..., :d]
    q.copy_(torch.randn(len(lens), 6, d, generator=torch.Generator().manual_seed(d)).to(BF16))
    whole = torch.full((len(lens), 6, d + pad), 9.0, dtype=BF16, device=cuda)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    ops.paged_decode_fp8(q, *pool.args, 1, bt, i32(lens, cuda), 1100, out=whole[..., :d], err=err)
    assert int(err) == 0
    check_decode(whole[..., :d], q, pool, table, lens, 1)
    assert bool((whole[..., d:] == 9.0).all())


@pytest.mark.parametrize("spread", [4.0, 12.0])
def test_decode_scales_far_apart(cuda, native_lib, spread):
    """Blocks whose V scales differ by many binades: the running reference moves up, and small blocks are added apart."""
    rs = np.random.RandomState(int(spread))
    n, h, d = 700, 2, 128
    pool = Pool(cuda, 1, 50, h, 16, d)
    table = pool.table([n])
    bt = torch.from_numpy(table).to(cuda)
    size = np.exp2(np.repeat(rs.uniform(-spread, spread, (h, 44)), 16, axis=1)[:, :n, None])
    k = rs.randn(1, h, n, d).astype(np.float32)
    v = (rs.randn(h, n, d) * size).astype(np.float32)[None]
    v[0, 0, 96:112] = 0.0  # a block of zeros has the smallest scale there is
    ops.paged_append_fp8(*pool.args, 0, bt, i32([0], cuda), torch.from_numpy(k).to(cuda), torch.from_numpy(v).to(cuda))
    pool.download()
    for dtype in (BF16, F16, F32):
        q = (3 * torch.randn(1, 8, d, generator=torch.Generator().manual_seed(1))).to(dtype).to(cuda)
        check_decode(ops.paged_decode_fp8(q, *pool.args, 0, bt, i32([n], cuda), n), q, pool, table, [n], 0)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("bs,d", [(8, 64), (8, 128), (8, 256), (8, 80), (24, 128), (40, 64), (72, 128)])
def test_decode_blocks_of_eights(cuda, native_lib, dtype, bs, d):
    """A 16-token tile that lies in two blocks; rows that end in either of them, stale NaN codes behind."""
    lens = [1, 7, 8, 9, 0, 15, 16, 17, 24, 25, 40, 505, 511, 513, 521, 1100]
    pool, table, bt = filled(cuda, lens, 2, bs, d, dtype, seed=bs + d)
    q = torch.randn(len(lens), 8, d, generator=torch.Generator().manual_seed(d)).to(dtype).to(cuda)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    out = ops.paged_decode_fp8(q, *pool.args, 1, bt, i32(lens, cuda), 1100, err=err)
    assert int(err) == 0
    check_decode(out, q, pool, table, lens, 1)
    for b in (3, 13):  # alone and in the batch
        one = ops.paged_decode_fp8(q[b:b + 1], *pool.args, 1, bt[b:b + 1], i32(lens[b:b + 1], cuda), lens[b])
        assert torch.equal(one, out[b:b + 1])


@pytest.mark.parametrize("bs", [8, 24])
def test_decode_scales_far_apart_within_a_tile(cuda, native_lib, bs):
    rs = np.random.RandomState(bs)
    n, h, d = 700, 2, 128
    pool = Pool(cuda, 1, 100, h, bs, d)
    table = pool.table([n])
    bt = torch.from_numpy(table).to(cuda)
    size = np.exp2(np.repeat(rs.uniform(-12, 12, (h, 100)), bs, axis=1)[:, :n, None])
    k = rs.randn(1, h, n, d).astype(np.float32)
    v = (rs.randn(h, n, d) * size).astype(np.float32)[None]
    v[0, 0, 8 * bs:9 * bs] = 0.0
    ops.paged_append_fp8(*pool.args, 0, bt, i32([0], cuda), torch.from_numpy(k).to(cuda), torch.from_numpy(v).to(cuda))
    pool.download()
    for dtype in (BF16, F16):
        q = (3 * torch.randn(1, 8, d, generator=torch.Generator().manual_seed(1))).to(dtype).to(cuda)
        check_decode(ops.paged_decode_fp8(q, *pool.args, 0, bt, i32([n], cuda), n), q, pool, table, [n], 0)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("factor", [0.0, 2.0 ** -40, 30.0])
def test_decode_q_magnitudes(cuda, native_lib, dtype, factor):
    """q of any magnitude (bf16 reaches far past fp16), sharp softmaxes, a head of zeros."""
    pool, table, bt = filled(cuda, [600], 2, 16, 128, dtype)
    q = torch.randn(1, 4, 128, generator=torch.Generator().manual_seed(2))
    q[0, 1] *= 2.0 ** 10
    q[0, 2] = 0
    q[0, 3, ::3] *= 2.0 ** -9
    q = (q * factor).to(dtype).to(cuda)
    check_decode(ops.paged_decode_fp8(q, *pool.args, 1, bt, i32([600], cuda), 600), q, pool, table, [600], 1)
    scale = 0.7
    out = ops.paged_decode_fp8(q, *pool.args, 1, bt, i32([600], cuda), 600, scale=scale)
    check_decode(out, q, pool, table, [600], 1, scale)


def test_decode_nan_in_the_cache_reaches_its_head_only(cuda, native_lib):
    pool, table, bt = filled(cuda, [40, 40], 2, 16, 128, BF16)
    x = torch.randn(2, 2, 1, 128, device=cuda).to(BF16)
    x[0, 1, 0, 7] = float("nan")
    for which in (0, 1):  # K, then V
        p, t, b = filled(cuda, [40, 40], 2, 16, 128, BF16)
        kv = [torch.randn_like(x), torch.randn_like(x)]
        kv[which] = x
        ops.paged_append_fp8(*p.args, 1, b, i32([39, 39], cuda), *kv)
        q = torch.randn(2, 4, 128, device=cuda).to(BF16)
        nan = torch.isnan(ops.paged_decode_fp8(q, *p.args, 1, b, i32([40, 40], cuda), 40))
        want = torch.zeros_like(nan)
        if which == 0:
            want[0, 2:] = True
        else:
            want[0, 2:, 7] = True
        assert torch.equal(nan, want)


def test_decode_layouts_plan_reuse_and_batch_invariance(cuda, native_lib):
    lens = [900, 1, 513, 40, 2000, 16]
    pool, table, bt = filled(cuda, lens, 8, 16, 128, BF16)
    q = torch.randn(6, 32, 128, device=cuda).to(BF16)
    seq = i32(lens, cuda)
    base = ops.paged_decode_fp8(q, *pool.args, 1, bt, seq, 2000)
    # every row alone, bit for bit
    for b in range(6):
        alone = ops.paged_decode_fp8(q[b:b + 1], *pool.args, 1, bt[b:b + 1], seq[b:b + 1], lens[b])
        assert torch.equal(alone[0], base[b])
    # row indirection
    rows = i32([4, 0, 2], cuda)
    assert torch.equal(ops.paged_decode_fp8(q[[4, 0, 2]], *pool.args, 1, bt, seq[[4, 0, 2]], 2000, row_ids=rows), base[[4, 0, 2]])
    # [B, Hq, 1, D] views, strided and misaligned q and out
    wide = torch.zeros(6, 32, 3, 131, dtype=BF16, device=cuda)
    wide[:, :, 1, 1:129] = q
    out = torch.zeros(6, 40, 1, 130, dtype=BF16, device=cuda)
    ops.paged_decode_fp8(wide[:, :, 1:2, 1:129], *pool.args, 1, bt, seq, 2000, out=out[:, 4:36, :, 1:129])
    assert torch.equal(out[:, 4:36, 0, 1:129], base)
    out[:, 4:36, :, 1:129] = 0
    assert not bool(out.any())
    # the plan of one layer serves the next
    ws = torch.empty(ops.decode_fp8_workspace_bytes(6, 32, 128, 2000), dtype=torch.uint8, device=cuda)
    assert torch.equal(ops.paged_decode_fp8(q, *pool.args, 1, bt, seq, 2000, ws=ws), base)
    assert torch.equal(ops.paged_decode_fp8(q, *pool.args, 1, bt, seq, 2000, ws=ws, plan_ready=True), base)


@pytest.mark.parametrize("lens,hkv", [
    ([1 + (b * 29) % 70 for b in range(1500)], 8),  # dozens of items a CTA, most with steps for some of its warps only
    ([(b * b * 131) % 2100 for b in range(200)], 4),  # full chunks, partial ones of every size, empty rows
], ids=["short", "ragged"])
def test_decode_many_items(cuda, native_lib, lens, hkv):
    pool, table, bt = filled(cuda, lens, hkv, 16, 128, BF16, layers=1, layer=0)
    q = torch.randn(len(lens), 2 * hkv, 128, generator=torch.Generator().manual_seed(0)).to(BF16).to(cuda)
    seq, err = i32(lens, cuda), torch.zeros(1, dtype=torch.int32, device=cuda)
    out = ops.paged_decode_fp8(q, *pool.args, 0, bt, seq, max(lens), err=err)
    assert int(err) == 0
    pick = list(range(0, len(lens), 23))
    check_decode(out[pick], q[pick], pool, table[pick], [lens[i] for i in pick], 0)
    # which CTA takes which item does not change a bit
    for _ in range(10):
        assert torch.equal(ops.paged_decode_fp8(q, *pool.args, 0, bt, seq, max(lens), err=err), out)
    assert int(err) == 0


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("hq,hkv,bs,d", [(16, 8, 16, 128), (4, 4, 16, 64), (20, 2, 8, 256), (5, 1, 16, 80)])
@pytest.mark.parametrize("max_len", [513, 1024, 1025, 2500, 4096])
def test_decode_small_calls_join_their_chunks(cuda, native_lib, dtype, hq, hkv, bs, d, max_len):
    """Small calls of up to eight chunks a row: rows of one chunk, of all, of none beside one another; the same bits as
    with a plan, and as the row alone."""
    lens = [max_len] if hkv == 8 else [max_len, 1, 512]
    pool, table, bt = filled(cuda, lens, hkv, bs, d, dtype, seed=d + max_len)
    q = torch.randn(len(lens), hq, d, generator=torch.Generator().manual_seed(d)).to(dtype).to(cuda)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    out = torch.full((len(lens), hq, d + 2), 9.0, dtype=dtype, device=cuda)
    ops.paged_decode_fp8(q, *pool.args, 1, bt, i32(lens, cuda), max_len, out=out[..., :d], err=err)
    check_decode(out[..., :d], q, pool, table, lens, 1)
    assert bool((out[..., d:] == 9.0).all())
    for bound in (4097, 60000):  # a cluster would be too large; a plan
        assert torch.equal(ops.paged_decode_fp8(q, *pool.args, 1, bt, i32(lens, cuda), bound, err=err), out[..., :d])
    for b, n in enumerate(lens):
        assert torch.equal(ops.paged_decode_fp8(q[b:b + 1], *pool.args, 1, bt[b:b + 1], i32([n], cuda), n, err=err), out[b:b + 1, :, :d])
    lens[-1] = 0
    assert bool((ops.paged_decode_fp8(q, *pool.args, 1, bt, i32(lens, cuda), max_len, err=err)[-1] == 0).all())
    assert int(err) == 0
    # a row longer than the bound is reported
    ops.paged_decode_fp8(q[:1], *pool.args, 1, bt[:1], i32([max_len], cuda), 512 if max_len <= 1024 else 1024, err=err)
    assert int(err) == nat.BL_DEVERR_WORKSPACE


@pytest.mark.parametrize("batch", [1, 33, 700])
@pytest.mark.parametrize("hq,hkv,bs,d", [(16, 8, 16, 128), (4, 4, 8, 64), (20, 2, 16, 256)])
def test_decode_rows_of_one_chunk(cuda, native_lib, batch, hq, hkv, bs, d):
    """Rows of 0..512 tokens, fewer and more of them than CTAs: no join, the same bits as in a call that has one."""
    lens = [(b * 97) % 514 if b % 5 else 0 for b in range(1, batch + 1)]
    lens = [min(n, 512) for n in lens]
    lens[0] = 512
    pool, table, bt = filled(cuda, lens, hkv, bs, d, BF16, seed=batch + d, layers=1, layer=0)
    q = torch.randn(batch, hq, d, generator=torch.Generator().manual_seed(d)).to(BF16).to(cuda)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    out = torch.full((batch, hq, d), 9.0, dtype=BF16, device=cuda)
    ops.paged_decode_fp8(q, *pool.args, 0, bt, i32(lens, cuda), 512, out=out, err=err)
    assert int(err) == 0
    pick = list(range(0, batch, 1 + batch // 40))
    check_decode(out[pick], q[pick], pool, table[pick], [lens[i] for i in pick], 0)
    assert torch.equal(ops.paged_decode_fp8(q, *pool.args, 0, bt, i32(lens, cuda), 513, err=err), out)
    rows = i32(range(batch - 1, -1, -1), cuda)
    turned = ops.paged_decode_fp8(q.flip(0), *pool.args, 0, bt, i32(lens[::-1], cuda), 512, row_ids=rows, err=err)
    assert torch.equal(turned.flip(0), out) and int(err) == 0
    ops.paged_decode_fp8(q, *pool.args, 0, bt, i32([0] * batch, cuda), 512, out=out, err=err)
    assert bool((out == 0).all()) and int(err) == 0
    # a row longer than the bound is reported (its table would hold it), the others are not touched by it
    if bs == 16:
        wide = torch.cat([bt, bt[:, :1]], dim=1)
        more = ops.paged_decode_fp8(q, *pool.args, 0, wide, i32([513] + lens[1:], cuda), 512, err=err)
        assert int(err) == nat.BL_DEVERR_WORKSPACE
        assert torch.equal(more[1:], turned.flip(0)[1:])


def test_decode_reports_what_it_cannot_do(cuda, native_lib):
    pool, table, bt = filled(cuda, [40, 600], 2, 16, 128, BF16)
    q = torch.randn(2, 4, 128, device=cuda).to(BF16)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)

    def word(**kw):
        err.zero_()
        a = dict(bt=bt, seq=i32([40, 600], cuda), n=600, ws=None, plan_ready=False) | kw
        ops.paged_decode_fp8(q, *pool.args, 1, a["bt"], a["seq"], a["n"], ws=a["ws"], plan_ready=a["plan_ready"], err=err)
        return int(err)

    assert word() == 0
    bad = bt.clone()
    bad[1, 3] = 1 << 20
    assert word(bt=bad) == nat.BL_DEVERR_BLOCK_ID
    assert word(bt=bt[:, :20].contiguous()) & nat.BL_DEVERR_TABLE
    assert word(n=100) & nat.BL_DEVERR_WORKSPACE  # a row longer than max_seq_len
    # a plan that was never made, or made for another call (40 rows: more items than a call without a plan takes)
    lens = [600] * 40
    pool, table, bt = filled(cuda, lens, 2, 16, 128, BF16)
    q, seq = torch.randn(40, 4, 128, device=cuda).to(BF16), i32(lens, cuda)
    ws = torch.zeros(ops.decode_fp8_workspace_bytes(40, 4, 128, 600), dtype=torch.uint8, device=cuda)

    def planned(n):
        err.zero_()
        ops.paged_decode_fp8(q[:n], *pool.args, 1, bt, seq[:n], 600, ws=ws, plan_ready=True, err=err)
        return int(err)

    assert planned(40) == nat.BL_DEVERR_WORKSPACE
    ops.paged_decode_fp8(q, *pool.args, 1, bt, seq, 600, ws=ws)
    assert planned(40) == 0 and planned(39) == nat.BL_DEVERR_WORKSPACE


@pytest.mark.parametrize("batch", [1, 9, 32, 33])
def test_decode_small_and_large_calls_agree(cuda, native_lib, batch):
    """Calls with and without a plan, on both sides of the border, and the reuse of a plan by many layers' calls."""
    lens = [(37 * b * b) % 1500 for b in range(batch)]
    pool, table, bt = filled(cuda, lens, 2, 16, 128, BF16)
    q, seq = torch.randn(batch, 8, 128, device=cuda).to(BF16), i32(lens, cuda)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    ws = torch.empty(ops.decode_fp8_workspace_bytes(batch, 8, 128, 60000), dtype=torch.uint8, device=cuda)
    small = ops.paged_decode_fp8(q, *pool.args, 1, bt, seq, 1500, err=err)
    check_decode(small, q, pool, table, lens, 1)
    for n in range(6):  # a bound of 60000 tokens needs a plan
        assert torch.equal(ops.paged_decode_fp8(q, *pool.args, 1, bt, seq, 60000, ws=ws, plan_ready=n > 0, err=err), small)
    assert int(err) == 0


def prefill_case(device, prefixes, chunks, hq, hkv, bs, d, dtype, seed=0):
    lens = [p + c for p, c in zip(prefixes, chunks)]
    pool, table, bt = filled(device, lens, hkv, bs, d, dtype, seed=seed)
    n = sum(chunks)
    q = torch.randn(n, hq, d, generator=torch.Generator().manual_seed(seed)).to(dtype).to(device).unsqueeze(0).transpose(1, 2)
    off = i32(np.concatenate([[0], np.cumsum(chunks)]), device)
    return pool, table, bt, lens, q, off


def check_prefill(out, q, pool, table, lens, chunks, layer, scale=None, tc=True):
    eps = torch.finfo(q.dtype).eps / 2 if tc else 0.0  # P in the element type on the tensor cores
    got, qn, at = out.double().cpu().numpy()[0], q.double().cpu().numpy()[0], 0
    for b, (n, c) in enumerate(zip(lens, chunks)):
        k, v = (f8.read(x, s, layer, table[b], n) for x, s in zip(pool.codes, pool.scales))
        want, spread, reach, flat = f8.attention(qn[:, at:at + c], k, v, scale)
        bound = attention_bound(want, spread, reach, flat, qn[:, at:at + c], q.dtype, eps, n)
        assert_within(got[:, at:at + c], want, bound)
        at += c


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("hq,hkv,bs,d", SHAPES)
def test_prefill(cuda, native_lib, dtype, hq, hkv, bs, d):
    prefixes, chunks = [0, 0, 5, 130, 16, 700], [1, 33, 1, 70, 200, 40]
    pool, table, bt, lens, q, off = prefill_case(cuda, prefixes, chunks, hq, hkv, bs, d, dtype, seed=hq + d)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    total = sum(-(-n // bs) for n in lens)
    out = ops.paged_prefill_fp8(q, *pool.args, 1, bt, i32(lens, cuda), max(lens), total_blocks=total, q_offsets=off,
                                max_q_len=max(chunks), err=err)
    assert int(err) == 0
    # (16-bit shapes of these dims run on the tensor cores, with P rounded to the element type)
    check_prefill(out, q, pool, table, lens, chunks, 1, tc=dtype is not F32 and d % 8 == 0)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("hq,hkv,bs,d", [(8, 2, 16, 256), (6, 2, 8, 144), (3, 3, 5, 192), (10, 1, 48, 208)])
@pytest.mark.parametrize("pad", [0, 3])
def test_prefill_wide_heads(cuda, native_lib, dtype, hq, hkv, bs, d, pad):
    """Head dims above 128: rows of (token, head) pairs that end inside a tile, more queries than tokens, strided q and out."""
    prefixes, chunks = [0, 3, 200, 64, 63, 0], [1, 40, 7, 130, 65, 300]
    pool, table, bt, lens, _, off = prefill_case(cuda, prefixes, chunks, hq, hkv, bs, d, dtype, seed=hq + d)
    total = sum(chunks)
    q = torch.full((1, total, hq, d + pad), float("nan"), dtype=dtype, device=cuda)[..., :d].transpose(1, 2)
    q.copy_(torch.randn(1, hq, total, d, generator=torch.Generator().manual_seed(d)).to(dtype))
    whole = torch.full((1, total + 2, hq, d + pad), 9.0, dtype=dtype, device=cuda)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    out = whole[:, :total, :, :d].transpose(1, 2)
    ops.paged_prefill_fp8(q, *pool.args, 1, bt, i32(lens, cuda), max(lens), total_blocks=sum(-(-n // bs) for n in lens),
                          q_offsets=off, max_q_len=max(chunks), out=out, err=err)
    assert int(err) == 0
    check_prefill(out, q, pool, table, lens, chunks, 1)
    assert bool((whole[..., d:] == 9.0).all()) and bool((whole[:, total:] == 9.0).all())
    # queries that see no key are zeros
    short = [n if b != 5 else 2 for b, n in enumerate(lens)]
    ops.paged_prefill_fp8(q, *pool.args, 1, bt, i32(short, cuda), max(lens), q_offsets=off, max_q_len=max(chunks), out=out, err=err)
    assert int(err) == 0 and bool((out[:, :, sum(chunks[:5]):-2] == 0).all()) and not bool((out[:, :, -2:] == 0).all())


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_prefill_wide_heads_rectangular(cuda, native_lib, dtype):
    """[B, Hq, T, D] queries, rows by row_ids, a row whose table ends early, a captured call, another stream."""
    lens, t, hq, hkv, d = [40, 300, 70], 37, 8, 2, 256
    pool, table, bt = filled(cuda, lens, hkv, 16, d, dtype)
    q = torch.randn(3, hq, t, d, generator=torch.Generator().manual_seed(0)).to(dtype).to(cuda)
    rows = i32([2, 0, 1], cuda)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    seq = i32([lens[2], lens[0], lens[1]], cuda)
    args = dict(row_ids=rows, err=err)
    out = ops.paged_prefill_fp8(q, *pool.args, 1, bt, seq, 300, **args)
    for i, b in enumerate((2, 0, 1)):
        check_prefill(out[i:i + 1], q[i:i + 1], pool, table[b:b + 1], [lens[b]], [t], 1)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        again = ops.paged_prefill_fp8(q, *pool.args, 1, bt, seq, 300, **args)
    again.fill_(5.0)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(again, out) and int(err) == 0
    ops.paged_prefill_fp8(q, *pool.args, 1, bt[:, :10].contiguous(), seq, 300, **args)
    assert int(err) == nat.BL_DEVERR_TABLE
    err.zero_()
    bad = bt.clone()
    bad[1, 3] = 10 ** 6
    wrong = ops.paged_prefill_fp8(q, *pool.args, 1, bad, seq, 300, **args)
    assert int(err) == nat.BL_DEVERR_BLOCK_ID and torch.equal(wrong[:2], out[:2])


@pytest.mark.parametrize("d", [128, 80])
def test_prefill_leaves_tokens_of_no_row(cuda, native_lib, d):
    """A packed q with room behind its last row: those outputs stay as they were; narrow, strided q and out."""
    chunks, lens = [5, 20], [30, 20]
    pool, table, bt = filled(cuda, lens, 2, 16, d, BF16)
    q = torch.randn(1, 40, 8, d + 4, device=cuda).to(BF16)[..., :d].transpose(1, 2)
    out = torch.full((1, 40, 8, d + 4), 3.0, dtype=BF16, device=cuda)
    view = out[..., :d].transpose(1, 2)
    ops.paged_prefill_fp8(q, *pool.args, 1, bt, i32(lens, cuda), 30, q_offsets=i32([0, 5, 25], cuda), max_q_len=20, out=view)
    check_prefill(view[:, :, :25], q[:, :, :25], pool, table, lens, chunks, 1)
    assert bool((out[:, 25:] == 3).all()) and bool((out[..., d:] == 3).all())


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F16, 64), (F32, 128)])
def test_prefill_queries_that_see_no_key(cuda, native_lib, dtype, d):
    """More queries than tokens: the first ones see nothing and get zeros; an empty row gets zeros throughout."""
    chunks, lens = [40, 7, 300, 5], [13, 0, 2, 5]
    pool, table, bt = filled(cuda, lens, 2, 16, d, dtype)
    q = torch.randn(1, 8, sum(chunks), d, device=cuda).to(dtype)
    off = i32(np.concatenate([[0], np.cumsum(chunks)]), cuda)
    out = torch.full_like(q, 5.0)
    ops.paged_prefill_fp8(q, *pool.args, 1, bt, i32(lens, cuda), 13, q_offsets=off, max_q_len=300, out=out)
    # (16-bit shapes of these dims run on the tensor cores, with P rounded to the element type)
    check_prefill(out, q, pool, table, lens, chunks, 1, tc=dtype is not F32 and d % 8 == 0)
    assert bool((out[0, :, :27] == 0).all()) and bool((out[0, :, 40:47] == 0).all())


def test_prefill_rectangular_strided_and_bounds(cuda, native_lib):
    lens, t = [50, 300, 33], 33
    pool, table, bt = filled(cuda, lens, 8, 16, 128, BF16)
    q = torch.randn(3, 16, t, 128, device=cuda).to(BF16)
    seq = i32(lens, cuda)
    base = ops.paged_prefill_fp8(q, *pool.args, 1, bt, seq, 300)
    assert base.shape == q.shape and base.transpose(1, 2).is_contiguous()
    packed = torch.cat(list(q), dim=1).unsqueeze(0)
    check_prefill(torch.cat(list(base), dim=1).unsqueeze(0), packed, pool, table, lens, [t] * 3, 1)
    # a larger bound, its own workspace and row indirection change nothing
    ws = torch.empty(64 << 20, dtype=torch.uint8, device=cuda)
    assert torch.equal(ops.paged_prefill_fp8(q[[2, 0]], *pool.args, 1, bt, seq[[2, 0]], 1000, row_ids=i32([2, 0], cuda), ws=ws), base[[2, 0]])
    # odd strides take the kernel that reads single elements
    wide = torch.zeros(3, 16, t, 131, dtype=BF16, device=cuda)
    wide[..., 1:129] = q
    out = torch.zeros(3, 16, t, 131, dtype=BF16, device=cuda)
    ops.paged_prefill_fp8(wide[..., 1:129], *pool.args, 1, bt, seq, 300, out=out[..., 2:130])
    check_prefill(torch.cat(list(out[..., 2:130]), dim=1).unsqueeze(0), packed, pool, table, lens, [t] * 3, 1)
    assert not bool(out[..., :2].any()) and not bool(out[..., 130:].any())
    with pytest.raises(ValueError, match="workspace"):
        ops.paged_prefill_fp8(q, *pool.args, 1, bt, seq, 300, ws=ws[:1024])


def test_prefill_reports_what_it_cannot_do(cuda, native_lib):
    for dtype in (BF16, F32):
        pool, table, bt = filled(cuda, [40, 600], 2, 16, 128, dtype)
        q = torch.randn(2, 4, 8, 128, device=cuda).to(dtype)
        err = torch.zeros(1, dtype=torch.int32, device=cuda)

        def word(table, n, **kw):
            err.zero_()
            ops.paged_prefill_fp8(q, *pool.args, 1, table, i32([40, 600], cuda), n, err=err, **kw)
            return int(err)

        assert word(bt, 600) == 0
        bad = bt.clone()
        bad[1, 3] = -7
        assert word(bad, 600) & nat.BL_DEVERR_BLOCK_ID
        assert word(bt[:, :20].contiguous(), 600) & nat.BL_DEVERR_TABLE
        if dtype is BF16:  # the bounds size the expanded pages
            assert word(bt, 100) & nat.BL_DEVERR_WORKSPACE
            assert word(bt, 600, total_blocks=5) & nat.BL_DEVERR_WORKSPACE


def test_refusals(cuda, native_lib):
    pool, table, bt = filled(cuda, [40, 20], 2, 16, 128, BF16)
    q = torch.randn(2, 4, 128, device=cuda).to(BF16)
    seq = i32([40, 20], cuda)
    k = torch.randn(2, 2, 1, 128, device=cuda).to(BF16)
    kc, vc, ks, vs = pool.args

    def bad(fn, exc=ValueError):
        with pytest.raises(exc):
            fn()

    dec = lambda **kw: ops.paged_decode_fp8(kw.pop("q", q), kw.pop("kc", kc), vc, kw.pop("ks", ks), vs, kw.pop("layer", 1),
                                            kw.pop("bt", bt), kw.pop("seq", seq), kw.pop("n", 40), **kw)
    dec()
    bad(lambda: dec(q=q.cpu()), RuntimeError)
    bad(lambda: dec(kc=kc.view(torch.uint8)))
    bad(lambda: dec(ks=ks.double()))
    bad(lambda: dec(ks=ks[:, :, :1]))
    bad(lambda: dec(layer=2), IndexError)
    bad(lambda: dec(bt=bt.long()))
    bad(lambda: dec(bt=bt[:1]))
    bad(lambda: dec(seq=seq[:1]))
    bad(lambda: dec(seq=seq.long()))
    bad(lambda: dec(q=q[:, :3]))
    bad(lambda: dec(q=q[..., ::2]))
    bad(lambda: dec(q=q.double()))
    bad(lambda: dec(n=0))
    bad(lambda: dec(scale=0.0))
    bad(lambda: dec(scale=float("nan")))
    bad(lambda: dec(plan_ready=True))
    bad(lambda: dec(out=torch.empty(2, 4, 128, device=cuda)))
    bad(lambda: dec(row_ids=i32([0], cuda)))
    bad(lambda: dec(err=torch.zeros(1, device=cuda)))
    app = lambda key, value, start=i32([0, 0], cuda), **kw: ops.paged_append_fp8(*pool.args, 1, bt, start, key, value, **kw)
    bad(lambda: app(k, k[:1]))
    bad(lambda: app(k.float(), k))
    bad(lambda: app(k[:, :1], k[:, :1]))
    bad(lambda: app(k[:, :, :0], k[:, :, :0]))
    bad(lambda: app(k, k, start=i32([0], cuda)))
    bad(lambda: app(k[:1], k[:1], new_offsets=i32([0, 1, 1], cuda)))
    pre = lambda **kw: ops.paged_prefill_fp8(kw.pop("q", q.unsqueeze(2)), *pool.args, 1, bt, seq, kw.pop("n", 40), **kw)
    pre()
    bad(lambda: pre(n=0))
    bad(lambda: pre(ws=torch.empty(64, dtype=torch.uint8, device=cuda)))
    bad(lambda: pre(total_blocks=0))
    bad(lambda: pre(q=q))
    bad(lambda: pre(scale=-1.0))
    bad(lambda: ops.paged_gather_fp8(*pool.args, 1, bt, seq, 0, dtype=BF16))
    bad(lambda: ops.paged_gather_fp8(*pool.args, 1, bt, seq, 4, dtype=torch.float64))


def test_graphs_streams_and_concurrent_calls(cuda, native_lib):
    """A serving step captured twice (two graphs, own scratch each), replayed together on two streams with new inputs."""
    lens = [700, 30, 1500]
    steps = []
    for seed in (1, 2):
        pool, table, bt = filled(cuda, [n + 8 for n in lens], 8, 16, 128, BF16, seed=seed)
        g = torch.Generator(device=cuda).manual_seed(seed)
        mk = lambda *s: torch.randn(*s, generator=g, device=cuda).to(BF16)
        steps.append(dict(pool=pool, bt=bt, k=mk(3, 8, 1, 128), v=mk(3, 8, 1, 128), q=mk(3, 16, 128), q2=mk(3, 16, 4, 128),
                          start=i32(lens, cuda), seq=i32([n + 1 for n in lens], cuda)))

    for s in steps:
        s["pair"] = s["pool"].free[:2]  # blocks in no row's table

    def run(s):
        ops.paged_append_fp8(*s["pool"].args, 1, s["bt"], s["start"], s["k"], s["v"])
        a = ops.paged_decode_fp8(s["q"], *s["pool"].args, 1, s["bt"], s["seq"], 1600)
        b = ops.paged_prefill_fp8(s["q2"], *s["pool"].args, 1, s["bt"], s["seq"], 1600)
        c = ops.paged_gather_fp8(*s["pool"].args, 1, s["bt"], s["seq"], 1501, dtype=BF16)
        ops.copy_blocks(*s["pool"].args[:2], [s["pair"][0]], [s["pair"][1]], key_scale=s["pool"].args[2], value_scale=s["pool"].args[3])
        return a, b, *c

    graphs = []
    for s in steps:
        run(s)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = run(s)
        graphs.append((graph, outs))
    streams = [torch.cuda.Stream() for _ in steps]
    for rep in range(3):
        for s in steps:
            for name in ("k", "v", "q", "q2"):
                s[name].copy_(torch.randn_like(s[name]))
        torch.cuda.synchronize()
        for (graph, _), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        got = [[o.clone() for o in outs] for _, outs in graphs]
        for s, g in zip(steps, got):
            for x, y in zip(run(s), g):
                assert torch.equal(x, y)


@pytest.mark.parametrize("n", [1, 40])
def test_a_workspace_may_be_what_the_kernel_before_read(cuda, native_lib, n):
    """In stream order an append's tokens are free for the next call's scratch: the plan is written only then."""
    batch, hkv, d = 300, 8, 128
    lens = [n + (b * 7) % 90 for b in range(batch)]
    pool, table, bt = filled(cuda, [x + n for x in lens], hkv, 16, d, BF16, layers=1, layer=0)
    q = torch.randn(batch, 2 * hkv, d, device=cuda).to(BF16)
    seq, start = i32([x + n for x in lens], cuda), i32(lens, cuda)
    off = i32([b * n for b in range(batch + 1)], cuda)
    bytes_kv = batch * n * hkv * d * 2
    need = ops.decode_fp8_workspace_bytes(batch, 2 * hkv, d, 512)
    last = (bytes_kv - 20 * n * hkv * d * 2) // 256 * 256  # the scratch begins at the tokens that are appended last
    buf = torch.zeros(last + max(need, bytes_kv - last), dtype=torch.uint8, device=cuda)
    k = buf[:bytes_kv].view(BF16).view(1, batch * n, hkv, d).transpose(1, 2)
    g = torch.Generator(device=cuda).manual_seed(n)
    tokens = torch.randn(k.shape, generator=g, device=cuda).to(BF16)
    clean = [c.clone() for c in pool.args]
    ops.paged_append_fp8(*clean, 0, bt, start, tokens, tokens, new_offsets=off, max_new_tokens=n)
    want = ops.paged_decode_fp8(q, *clean, 0, bt, seq, 512)
    for _ in range(20):
        k.copy_(tokens)
        got = [c.clone() for c in pool.args]
        ops.paged_append_fp8(*got, 0, bt, start, k, k, new_offsets=off, max_new_tokens=n)
        out = ops.paged_decode_fp8(q, *got, 0, bt, seq, 512, ws=buf[last:])
        for a, b in zip(got, clean):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        assert torch.equal(out, want)


@pytest.mark.parametrize("max_len", [512, 1300])
def test_calls_in_a_row_share_a_workspace(cuda, native_lib, max_len):
    """Plans of different batches written over one another, call after call."""
    lens = [(b * 53) % max_len + 1 for b in range(120)]
    pool, table, bt = filled(cuda, lens, 4, 16, 128, BF16, layers=1, layer=0)
    q = torch.randn(120, 8, 128, device=cuda).to(BF16)
    seq, err = i32(lens, cuda), torch.zeros(1, dtype=torch.int32, device=cuda)
    want = ops.paged_decode_fp8(q, *pool.args, 0, bt, seq, max_len)
    ws = torch.empty(ops.decode_fp8_workspace_bytes(120, 8, 128, max_len), dtype=torch.uint8, device=cuda)
    outs = []
    for i in range(60):
        n = 120 - (i % 3) * 25
        outs.append((n, ops.paged_decode_fp8(q[:n], *pool.args, 0, bt[:n], seq[:n], max_len, ws=ws, err=err)))
    assert all(torch.equal(o, want[:n]) for n, o in outs) and int(err) == 0


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F16, 128), (F16, 64), (BF16, 256), (F16, 144), (BF16, 12), (F32, 128)])
@pytest.mark.parametrize("pad", [0, 2])
def test_prefill_queries_that_see_no_key_beside_nan(cuda, native_lib, dtype, d, pad):
    """They are zeros even where the keys that later queries of their tile see hold NaN."""
    chunks, lens = [40, 300], [13, 150]
    pool, table, bt = filled(cuda, lens, 2, 16, d, dtype)
    q = torch.randn(1, sum(chunks), 8, d, device=cuda).to(dtype).transpose(1, 2)
    off = i32([0, 40, 340], cuda)
    whole = torch.full((1, sum(chunks), 8, d + pad), 5.0, dtype=dtype, device=cuda)
    out = whole[..., :d].transpose(1, 2)
    for which in pool.dev:  # K, then V too: the rows' first tokens, of one head
        which.view(torch.uint8)[1, bt[:, 0].long(), 1, 2, :] = 0x7F
        ops.paged_prefill_fp8(q, *pool.args, 1, bt, i32(lens, cuda), 150, q_offsets=off, max_q_len=300, out=out)
        assert bool((out[0, :, :27] == 0).all()) and bool((out[0, :, 40:190] == 0).all())
        assert bool(out[0, 4:, 39].isnan().all()) and not bool(out[0, :4].isnan().any())


def far_bound(want, spread, reach, flat, q, k, v, dtype, eps, k_scales, v_scales, scale):
    """attention_bound, and what fp16 operands add where scales lie far apart (fp8.cuh,
    half_unit).  A K or V element is kept to 2^-25 of its unit, 2^-7 of the largest
    scale: a score moves by 2^-25 unit sum |q| scale (a weight by twice its expm1, as
    there), an output by 2^-25 unit.  A weight below 2^-14 of the largest is kept to 2^-25 of
    that, and the weights' sum is at least the largest: 2^-25 sum |v| over the keys."""
    err = attention_bound(want, spread, reach, flat, q, dtype, eps, k.shape[1])
    if dtype is F16:
        g = q.shape[0] // k.shape[0]
        unit = lambda s: np.repeat(s.max(axis=0), g)[:, None, None] * 2.0 ** -7
        move = 2.0 ** -25 * unit(k_scales) * np.abs(q).sum(axis=2, keepdims=True) * scale
        err = err + 2 * np.expm1(2 * move) * spread + 2.0 ** -25 * unit(v_scales)
    if dtype is not F32:
        err = err + 2.0 ** -25 * np.repeat(np.abs(v).sum(axis=1), q.shape[0] // v.shape[0], axis=0)[:, None]
    return err


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("hq,hkv,bs,d", [(8, 2, 16, 128), (6, 2, 16, 128), (4, 2, 32, 64), (8, 2, 16, 256), (4, 2, 8, 144), (4, 2, 16, 36),
                                          (8, 2, 4, 128), (10, 2, 5, 64)])  # (the last two: rows of more than 128 blocks)
@pytest.mark.parametrize("k_exp,q_exp,v_exp,v_spread,scale", [(17, -17, 16, 0.0, None), (-22, 12, 0, 0.0, 64.0), (0, 0, -4, 12.0, None),
                                                              (-60, 12, 3, 4.0, 2.0 ** 44)], ids=["large", "small", "apart", "tiny"])
def test_prefill_values_far_from_one(cuda, native_lib, dtype, hq, hkv, bs, d, k_exp, q_exp, v_exp, v_spread, scale):
    """A pool filled from fp32: K and V past fp16's range, below its normal numbers, and V whose blocks lie far apart."""
    rs = np.random.RandomState(100 + d + k_exp)
    n, c = 700, 90
    pool = Pool(cuda, 1, -(-n // bs) + 3, hkv, bs, d)
    table = pool.table([n])
    bt = torch.from_numpy(table).to(cuda)
    size = np.exp2(np.repeat(rs.uniform(-v_spread, v_spread, (hkv, n // 16 + 1)), 16, axis=1)[:, :n, None])
    k = (rs.randn(1, hkv, n, d) * 2.0 ** k_exp).astype(np.float32)
    v = (rs.randn(1, hkv, n, d) * size * 2.0 ** v_exp).astype(np.float32)
    ops.paged_append_fp8(*pool.args, 0, bt, i32([0], cuda), torch.from_numpy(k).to(cuda), torch.from_numpy(v).to(cuda))
    pool.download()
    q = (torch.randn(1, hq, c, d, generator=torch.Generator().manual_seed(1)) * 2.0 ** q_exp).to(dtype).to(cuda)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    out = ops.paged_prefill_fp8(q, *pool.args, 0, bt, i32([n], cuda), n, scale=scale, err=err)
    assert int(err) == 0
    kd, vd = (f8.read(x, s, 0, table[0], n) for x, s in zip(pool.codes, pool.scales))
    qn = q.double().cpu().numpy()[0]
    want, spread, reach, flat = f8.attention(qn, kd, vd, scale)
    eps = torch.finfo(dtype).eps / 2 if dtype is not F32 and d % 8 == 0 else 0.0
    used, scale_d = table[0][table[0] >= 0], scale or 1 / np.sqrt(d)
    bound = far_bound(want, spread, reach, flat, qn, kd, vd, dtype, eps, *(s[0][used] for s in pool.scales), scale_d)
    assert_within(out.double().cpu().numpy()[0], want, bound)
    # the decode of the last token stays within the same bound
    got = ops.paged_decode_fp8(q[:, :, -1].contiguous(), *pool.args, 0, bt, i32([n], cuda), n, scale=scale)
    bound = far_bound(*(x[:, -1:] for x in (want, spread, reach, flat, qn)), kd, vd, dtype, 2.0 ** -11 if dtype is not F32 else 0.0,
                      *(s[0][used] for s in pool.scales), scale_d)
    assert_within(got.double().cpu().numpy()[0][:, None], want[:, -1:], bound)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("hq,hkv,bs,d", [(8, 2, 16, 128), (6, 2, 4, 128), (8, 2, 16, 256)])
@pytest.mark.parametrize("exps", [[17, 0, -18, 2], [17, 0, -13, 2]])  # (-18: q holds infinities in fp16)
def test_prefill_rows_and_heads_of_different_magnitudes(cuda, native_lib, dtype, hq, hkv, bs, d, exps):
    """Each row's KV heads have units of their own; empty rows, queries that see nothing, rows by row_ids, a captured call."""
    rs = np.random.RandomState(d + bs)
    lens, chunks = [600, 0, 33, 520], [40, 3, 50, 17]
    pool = Pool(cuda, 1, sum(-(-n // bs) for n in lens) + 3, hkv, bs, d)
    table = pool.table(lens)
    bt = torch.from_numpy(table).to(cuda)
    tokens = [[rs.randn(hkv, n, d) * 2.0 ** (e + np.array([0, -9]))[:, None, None] for n, e in zip(lens, exps)] for _ in range(2)]
    off = i32(np.concatenate([[0], np.cumsum(lens)]), cuda)
    k, v = (torch.from_numpy(np.concatenate(x, axis=1).astype(np.float32)).to(cuda).unsqueeze(0) for x in tokens)
    ops.paged_append_fp8(*pool.args, 0, bt, i32([0] * 4, cuda), k, v * 0.25, new_offsets=off, max_new_tokens=max(lens))
    pool.download()
    order = [2, 0, 3, 1]  # of the queries' rows in the table
    g = torch.Generator().manual_seed(7)
    qs = [torch.randn(hq, chunks[r], d, generator=g) * 2.0 ** -exps[r] for r in order]
    q = torch.cat(qs, dim=1).to(dtype).to(cuda).unsqueeze(0)
    q_off = i32(np.concatenate([[0], np.cumsum([chunks[r] for r in order])]), cuda)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    call = lambda: ops.paged_prefill_fp8(q, *pool.args, 0, bt, i32_lens, 600, q_offsets=q_off, max_q_len=50, row_ids=rows, err=err)
    i32_lens, rows = i32([lens[r] for r in order], cuda), i32(order, cuda)
    out = call()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        again = call()
    again.fill_(5.0)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(again.view(torch.int16), out.view(torch.int16)) and int(err) == 0
    at, got = 0, out.double().cpu().numpy()[0]
    for r in order:
        kd, vd = (f8.read(x, s, 0, table[r], lens[r]) for x, s in zip(pool.codes, pool.scales))
        qn = q[0, :, at:at + chunks[r]].double().cpu().numpy()
        want, spread, reach, flat = f8.attention(qn, kd, vd)
        used = table[r][:-(-lens[r] // bs)]
        scales = [s[0][used] if len(used) else np.ones((1, hkv)) for s in pool.scales]
        bound = far_bound(want, spread, reach, flat, qn, kd, vd, dtype, torch.finfo(dtype).eps / 2, *scales, 1 / np.sqrt(d))
        bound[:, :max(0, chunks[r] - lens[r])] = 0.0  # no key: zeros (the terms above may be inf * 0)
        assert_within(got[:, at:at + chunks[r]], want, bound)
        at += chunks[r]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("use_rows", [False, True])
def test_decode_skips_records_that_are_no_plan(cuda, native_lib, dtype, use_rows):
    """A workspace whose header is a plan's and whose records are not: the kernel checks each before it
    follows it (rows, chunks whose tokens overflow, lengths), flags it, and leaves its output."""
    batch, n = 40, 700
    pool, table, bt = filled(cuda, [n] * batch, 2, 16, 128, dtype)
    q, seq = torch.randn(batch, 4, 128, device=cuda).to(dtype), i32([n] * batch, cuda)
    rows = i32([(7 * b + 3) % batch for b in range(batch)], cuda) if use_rows else None
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    ws = torch.zeros(ops.decode_fp8_workspace_bytes(batch, 4, 128, n), dtype=torch.uint8, device=cuda)
    call = lambda out, ready: ops.paged_decode_fp8(q, *pool.args, 1, bt, seq, n, row_ids=rows, ws=ws, plan_ready=ready, out=out, err=err)
    want = call(None, False).clone()
    good = ws.clone()
    words = ws.view(torch.int32)
    units = words[(256 + 256) // 4:][:4 * 80].view(80, 4)  # row, chunk, len, part
    assert words[0] == 80 and units[:, 2].tolist() == [n] * 80 and sorted(units[:, 0].tolist()) == sorted(2 * list(range(batch)))
    for field, value in ((0, 10 ** 6), (0, -1), (1, 2 ** 22), (1, 2 ** 23), (1, 2 ** 31 - 1), (1, -1), (1, 2), (2, 2 ** 30), (2, 0),
                         (2, -5)):
        for record in (0, 79):
            ws.copy_(good)
            hit = int(units[record, 0])
            units[record, field] = value
            out = torch.full_like(want, 9.0)
            err.zero_()
            call(out, True)
            assert int(err) & nat.BL_DEVERR_WORKSPACE, (field, value)
            others = [b for b in range(batch) if b != hit]
            assert torch.equal(out[others], want[others]), (field, value)
    if dtype is BF16:  # the counter of claims (the other kernel has none)
        err.zero_()
        ws.copy_(good)
        words[4:6] = -10 ** 6
        call(torch.empty_like(want), True)
        assert int(err) & nat.BL_DEVERR_WORKSPACE
    err.zero_()
    ws.copy_(good)
    assert torch.equal(call(None, True), want) and int(err) == 0
