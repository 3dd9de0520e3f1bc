"""8-bit cache on the GPU: append, gather and page copies against the float64
oracle.  All three are exact: codes, scales and gathered values are compared
for equality."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from barellm_b200 import _native as nat
from barellm_b200 import ops
from fp8_helpers import Pool, cache_values, i32
from oracle import fp8_oracle as f8

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def oracle_append(pool, layer, table, starts, ks, vs):
    for b, (s, k, v) in enumerate(zip(starts, ks, vs)):
        f8.append(pool.codes[0], pool.scales[0], layer, table[b], s, k)
        f8.append(pool.codes[1], pool.scales[1], layer, table[b], s, v)


def gpu_append(pool, layer, bt, starts, ks, vs, dtype, **kw):
    """Packed append of per-row [H, n, D] arrays."""
    off = np.concatenate([[0], np.cumsum([k.shape[1] for k in ks])]).astype(np.int32)
    cat = [torch.from_numpy(np.concatenate(x, axis=1)).to(dtype).to(pool.device).unsqueeze(0) for x in (ks, vs)]
    ops.paged_append_fp8(*pool.args, layer, bt, i32(starts, pool.device), *cat, new_offsets=i32(off, pool.device),
                         max_new_tokens=int(np.diff(off).max()), **kw)


def rounded(x, dtype):
    return torch.from_numpy(np.ascontiguousarray(x)).to(dtype).double().numpy()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hkv,bs,d", [(8, 16, 128), (2, 16, 64), (1, 16, 256), (3, 8, 80), (2, 32, 128), (2, 5, 3), (1, 1, 1),
                                      (2, 24, 12), (5, 16, 129)])
def test_append_equals_oracle(cuda, native_lib, dtype, hkv, bs, d):
    rs = np.random.RandomState(hkv * 1000 + bs * 10 + d)
    starts = [0, 1, bs - 1, bs, bs + bs // 2, 3 * bs, 7]
    new = [1, 1, 2, bs, 2 * bs + 3, 5 * bs, 40]
    pool = Pool(cuda, 2, sum(-(-(s + n) // bs) for s, n in zip(starts, new)) + 3, hkv, bs, d)
    table = pool.table([s + n for s, n in zip(starts, new)])
    bt = torch.from_numpy(table).to(cuda)
    hist = [cache_values(rs, hkv, s, d) for s in starts]
    for layer in (0, 1):
        first = [(b, h) for b, h in enumerate(hist) if h.shape[1]]
        rows = i32([b for b, _ in first], cuda)
        if first:
            ks = [rounded(h, dtype).astype(np.float32) for _, h in first]
            gpu_append(pool, layer, bt, [0] * len(first), ks, [2 * k for k in ks], dtype, row_ids=rows)
            oracle_append(pool, layer, table[[b for b, _ in first]], [0] * len(first), ks, [2 * k for k in ks])
        ks = [cache_values(rs, hkv, n, d) * 2.0 ** rs.randint(-6, 7) for n in new]
        vs = [cache_values(rs, hkv, n, d) for n in new]
        gpu_append(pool, layer, bt, starts, ks, vs, dtype)
        oracle_append(pool, layer, table, starts, [rounded(k, dtype) for k in ks], [rounded(v, dtype) for v in vs])
    pool.assert_equal()


@pytest.mark.parametrize("batch", [2, 31, 33, 64, 1100])
@pytest.mark.parametrize("bs,first", [(16, 0), (16, 37), (1, 2), (5, 0), (64, 5)])
def test_append_rows_of_very_different_lengths(cuda, native_lib, batch, bs, first):
    """A few long chunks among short and empty ones, the first token of the packed axis not row 0's, tokens of no row behind."""
    rs = np.random.RandomState(batch + bs)
    new = [int(n) for n in rs.choice([0, 0, 1, 2, 7], batch)]
    new[0], new[batch // 2], new[-1] = 130, 0, 75
    starts = [int(x) for x in rs.randint(0, 2 * bs + 2, batch)]
    pool = Pool(cuda, 1, sum(-(-(s + n) // bs) for s, n in zip(starts, new)) + 3, 2, bs, 8)
    table = pool.table([s + n for s, n in zip(starts, new)])
    bt = torch.from_numpy(table).to(cuda)
    k, v = (torch.from_numpy(rs.randn(1, 2, first + sum(new) + 3, 8).astype(np.float32)).to(cuda) for _ in range(2))
    off = first + np.concatenate([[0], np.cumsum(new)])
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    ops.paged_append_fp8(*pool.args, 0, bt, i32(starts, cuda), k, v, new_offsets=i32(off, cuda), max_new_tokens=max(new), err=err)
    kn, vn = k[0].double().cpu().numpy(), v[0].double().cpu().numpy()
    pick = [b for b in range(batch) if new[b]]
    oracle_append(pool, 0, table[pick], [starts[b] for b in pick], [kn[:, off[b]:off[b + 1]] for b in pick],
                  [vn[:, off[b]:off[b + 1]] for b in pick])
    assert int(err) == 0
    pool.assert_equal()


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_token_by_token_raises_scales(cuda, native_lib, dtype):
    """Magnitudes that grow and shrink inside a block: old codes are rounded to each raised scale, in order."""
    rs = np.random.RandomState(3)
    pool = Pool(cuda, 1, 6, 2, 16, 128)
    table = pool.table([40, 20])
    bt = torch.from_numpy(table).to(cuda)
    for t in range(40):
        size = 2.0 ** ((t * 7) % 19 - 9)
        rows = [0, 1] if t < 20 else [0]
        ks = [(rs.randn(2, 1, 128) * size).astype(np.float32) for _ in rows]
        vs = [(rs.randn(2, 1, 128) / size).astype(np.float32) for _ in rows]
        gpu_append(pool, 0, bt, [t] * len(rows), ks, vs, dtype, row_ids=i32(rows, cuda))
        oracle_append(pool, 0, table[rows], [t] * len(rows), [rounded(k, dtype) for k in ks], [rounded(v, dtype) for v in vs])
        pool.assert_equal()


def test_append_extremes(cuda, native_lib):
    """Zeros, infinities, NaN, the largest and the smallest magnitudes, and ties."""
    pool = Pool(cuda, 1, 16, 1, 16, 32)
    table = pool.table([16] * 8)
    bt = torch.from_numpy(table).to(cuda)
    rs = np.random.RandomState(0)
    base = rs.randn(1, 16, 32).astype(np.float32)
    rows = [np.zeros_like(base), base * 1e30, base * 1e-37, base.copy(), base.copy(), np.full_like(base, -0.0),
            np.where(rs.rand(*base.shape) < 0.5, 3.38e38, -1.5).astype(np.float32),
            ((f8.POSITIVE[:-1] + f8.POSITIVE[1:]) / 2)[rs.randint(0, 126, base.shape)].astype(np.float32)]
    rows[3][0, 2, 5], rows[3][0, 4, 1], rows[3][0, 0, 0] = np.inf, -np.inf, np.nan
    rows[4][:] = np.inf
    rows[7][0, 0, 0] = 448.0
    gpu_append(pool, 0, bt, [0] * 8, rows, rows, torch.float32)
    oracle_append(pool, 0, table, [0] * 8, [r.astype(np.float64) for r in rows], [r.astype(np.float64) for r in rows])
    # values below the smallest normal fp32 may be flushed on the way: they are zero codes either way
    pool.assert_equal()


@pytest.mark.parametrize("layout", ["bhtd", "bthd", "odd"])
def test_append_rectangular_and_strided(cuda, native_lib, layout):
    rs = np.random.RandomState(5)
    b, h, t, d = 3, 4, 19, 128
    starts = [0, 16, 21]
    pool = Pool(cuda, 1, 16, h, 16, d)
    table = pool.table([s + t for s in starts])
    bt = torch.from_numpy(table).to(cuda)
    full = torch.from_numpy(rs.randn(b, t, h, d + 3).astype(np.float32)).to(torch.bfloat16).to(cuda)
    x = full[..., :d].contiguous().transpose(1, 2) if layout == "bthd" else (
        full[..., :d].transpose(1, 2).contiguous() if layout == "bhtd" else full[..., 1:d + 1].transpose(1, 2))
    y = (x * 3).clone(memory_format=torch.contiguous_format)
    pool.scales[0][:] = pool.scales[1][:] = 2.0 ** -8
    for s in pool.dev_scales:
        s.fill_(2.0 ** -8)
    ops.paged_append_fp8(*pool.args, 0, bt, i32(starts, cuda), x, y)
    oracle_append(pool, 0, table, starts, list(x.double().cpu().numpy()), list(y.double().cpu().numpy()))
    pool.assert_equal()


def test_append_reports_bad_blocks_and_writes_nothing_there(cuda, native_lib):
    pool = Pool(cuda, 1, 4, 2, 16, 64)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    x = torch.randn(1, 2, 20, 64, device=cuda)
    for table, bit in (([[4, 1]], nat.BL_DEVERR_BLOCK_ID), ([[-1, 1]], nat.BL_DEVERR_BLOCK_ID)):
        err.zero_()
        ops.paged_append_fp8(*pool.args, 0, i32(table[0], cuda).view(1, 2), i32([0], cuda), x, x, err=err)
        assert int(err) == bit
        oracle_append(pool, 0, np.array([[0, 1]]), [16], [x[0, :, 16:].double().cpu().numpy()], [x[0, :, 16:].double().cpu().numpy()])
        pool.assert_equal()
    err.zero_()
    ops.paged_append_fp8(*pool.args, 0, i32([3], cuda).view(1, 1), i32([16], cuda), x, x, err=err)
    assert int(err) == nat.BL_DEVERR_TABLE
    ops.paged_append_fp8(*pool.args, 0, i32([3], cuda).view(1, 1), i32([-5], cuda), x, x, err=err)
    assert int(err) == nat.BL_DEVERR_TABLE
    pool.assert_equal()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hkv,bs,d", [(8, 16, 128), (2, 16, 64), (1, 32, 256), (3, 8, 80), (2, 5, 3), (2, 16, 129)])
def test_gather_equals_oracle(cuda, native_lib, dtype, hkv, bs, d):
    lens = [1, bs - 1 or 1, bs, 3 * bs + 1, 0, 50]
    rs = np.random.RandomState(1)
    pool = Pool(cuda, 2, sum(-(-n // bs) for n in lens) + 2, hkv, bs, d)
    table = pool.table(lens)
    bt = torch.from_numpy(table).to(cuda)
    hist = [cache_values(rs, hkv, n, d) for n in lens]
    gpu_append(pool, 1, bt, [0] * len(lens), hist, [h * 100 for h in hist], torch.float32)
    pool.download()
    top = float(torch.finfo(dtype).max)
    k, v = ops.paged_gather_fp8(*pool.args, 1, bt, i32(lens, cuda), 50 + bs, dtype=dtype)
    for b, n in enumerate(lens):
        for got, codes, scales in ((k, pool.codes[0], pool.scales[0]), (v, pool.codes[1], pool.scales[1])):
            want = np.zeros((hkv, 50 + bs, d))
            want[:, :n] = f8.read(codes, scales, 1, table[b], n)[:, :50 + bs]  # a row may be longer than the read
            want = torch.from_numpy(np.clip(want, -top, top)).to(dtype)
            assert torch.equal(got[b].cpu(), want)
    # strided outputs without zero fill: behind the length nothing is written
    ko = torch.full((len(lens), 60, hkv, d), 7.0, dtype=dtype, device=cuda).transpose(1, 2)
    vo = torch.full((len(lens), 60, hkv, d), 7.0, dtype=dtype, device=cuda).transpose(1, 2)
    ops.paged_gather_fp8(*pool.args, 1, bt, i32(lens, cuda), 60, dtype=dtype, out=(ko, vo), zero_fill=False)
    for b, n in enumerate(lens):
        m = min(n, 50)
        assert torch.equal(ko[b, :, :m], k[b, :, :m]) and torch.equal(vo[b, :, :m], v[b, :, :m])
        assert bool((ko[b, :, n:] == 7).all()) and bool((vo[b, :, n:] == 7).all())


def test_gather_saturates_and_keeps_nan(cuda, native_lib):
    pool = Pool(cuda, 1, 1, 1, 16, 32)
    bt = i32([0], cuda).view(1, 1)
    x = torch.full((1, 1, 16, 32), 65504.0, dtype=torch.float16, device=cuda)
    x[0, 0, 1] = -65504.0
    x[0, 0, 2, 3] = float("nan")
    ops.paged_append_fp8(*pool.args, 0, bt, i32([0], cuda), x, x)
    k, _ = ops.paged_gather_fp8(*pool.args, 0, bt, i32([16], cuda), 16, dtype=torch.float16)
    assert float(k[0, 0, 0, 0]) == 65504.0 and float(k[0, 0, 1, 0]) == -65504.0
    assert bool(torch.isnan(k[0, 0, 2, 3])) and int(torch.isnan(k).sum()) == 1
    k, _ = ops.paged_gather_fp8(*pool.args, 0, bt, i32([16], cuda), 16, dtype=torch.float32)
    assert float(k[0, 0, 0, 0]) == 65536.0


def test_gather_reports_bad_blocks(cuda, native_lib):
    pool = Pool(cuda, 1, 2, 1, 16, 32)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    ops.paged_gather_fp8(*pool.args, 0, i32([9], cuda).view(1, 1), i32([3], cuda), 3, dtype=torch.float32, err=err)
    assert int(err) == nat.BL_DEVERR_BLOCK_ID
    err.zero_()
    ops.paged_gather_fp8(*pool.args, 0, i32([1], cuda).view(1, 1), i32([17], cuda), 17, dtype=torch.float32, err=err)
    assert int(err) == nat.BL_DEVERR_TABLE


@pytest.mark.parametrize("dtype", [ops.FP8_DTYPE, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape,pairs", [((3, 40, 8, 16, 128), 17), ((1, 9, 1, 1, 3), 4), ((2, 2500, 2, 4, 8), 1203), ((5, 3, 7, 5, 17), 1),
                                         ((2, 6, 16, 64, 256), 3)])
def test_copy_blocks(cuda, native_lib, dtype, shape, pairs):
    rs = np.random.RandomState(pairs)
    raw = [torch.from_numpy(rs.randint(0, 256, (*shape[:-1], shape[-1] * dtype.itemsize)).astype(np.uint8)).to(cuda) for _ in range(2)]
    kc, vc = (r.view(dtype) for r in raw)
    scales = [torch.rand(shape[:3], device=cuda) for _ in range(2)] if dtype is ops.FP8_DTYPE else [None, None]
    want = [t.clone() for t in raw + [s for s in scales if s is not None]]
    ids = rs.permutation(shape[1])[: 2 * pairs]
    src, dst = ids[:pairs].tolist(), ids[pairs:].tolist()
    if pairs > 1:
        src[1] = src[0]  # a block may be read more than once
    for w in want:
        w[:, dst] = w[:, src]
    ops.copy_blocks(kc, vc, src, np.asarray(dst), key_scale=scales[0], value_scale=scales[1])
    for got, w in zip(raw + [s for s in scales if s is not None], want):
        assert torch.equal(got, w)


def test_copy_blocks_refusals_copy_nothing(cuda, native_lib):
    kc = torch.randn(2, 6, 2, 16, 8, device=cuda)
    vc = kc + 1
    before = kc.clone()
    for src, dst in (([0, 1], [2, 2]), ([0, 1], [1, 2]), ([4], [4]), ([0], [6]), ([-1], [2]), ([0, 1], [2]), ([0.5], [2]),
                     ([1 << 40], [2]), ([[0, 1]], [[2, 3]]), ([True], [2])):
        with pytest.raises(ValueError):
            ops.copy_blocks(kc, vc, src, dst)
    with pytest.raises(ValueError, match="scales"):
        ops.copy_blocks(kc, vc, [0], [1], key_scale=torch.ones(2, 6, 2, device=cuda), value_scale=torch.ones(2, 6, 2, device=cuda))
    f = torch.zeros((2, 6, 2, 16, 8), dtype=torch.uint8, device=cuda).view(ops.FP8_DTYPE)
    with pytest.raises(ValueError, match="scales"):
        ops.copy_blocks(f, f.clone(), [0], [1])
    ops.copy_blocks(kc, vc, [], [])
    assert torch.equal(kc, before)


def test_offsets_past_32_bits(cuda, native_lib):
    """A pool of more than 2^32 codes: the last blocks are appended to, read, copied and attended to."""
    shape = (2, 132000, 8, 16, 128)  # 4.3e9 codes in K
    kc = torch.empty(shape, dtype=ops.FP8_DTYPE, device=cuda)
    vc = torch.empty(shape, dtype=ops.FP8_DTYPE, device=cuda)
    ks, vs = (torch.ones(shape[:3], device=cuda) for _ in range(2))
    n = 40
    bt = i32([131999, 131990, 131995], cuda).view(1, 3)
    x = torch.randn(1, 8, n, 128, device=cuda).to(torch.bfloat16)
    ops.paged_append_fp8(kc, vc, ks, vs, 1, bt, i32([0], cuda), x, x)
    small = Pool(cuda, 1, 3, 8, 16, 128)
    sbt = i32([0, 1, 2], cuda).view(1, 3)
    ops.paged_append_fp8(*small.args, 0, sbt, i32([0], cuda), x, x)
    q = torch.randn(1, 16, 128, device=cuda).to(torch.bfloat16)
    q2 = torch.randn(1, 16, 5, 128, device=cuda).to(torch.bfloat16)
    ops.copy_blocks(kc, vc, [131995], [131998], key_scale=ks, value_scale=vs)
    for table in (bt, i32([131999, 131990, 131998], cuda).view(1, 3)):
        got = ops.paged_gather_fp8(kc, vc, ks, vs, 1, table, i32([n], cuda), n, dtype=torch.bfloat16)
        want = ops.paged_gather_fp8(*small.args, 0, sbt, i32([n], cuda), n, dtype=torch.bfloat16)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert torch.equal(ops.paged_decode_fp8(q, kc, vc, ks, vs, 1, table, i32([n], cuda), n),
                           ops.paged_decode_fp8(q, *small.args, 0, sbt, i32([n], cuda), n))
        assert torch.equal(ops.paged_prefill_fp8(q2, kc, vc, ks, vs, 1, table, i32([n], cuda), n),
                           ops.paged_prefill_fp8(q2, *small.args, 0, sbt, i32([n], cuda), n))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("step", [0.7, 1.0, 3.5])
def test_stored_values_stay_near_the_appended_ones(cuda, native_lib, dtype, step):
    """Blocks whose scale is raised with almost every token, against the values that were appended.

    The first rounding is off by at most 2^-4 |x| or 2^-10 of the scale of then; every raise
    rounds to at most 2^-10 of the new scale, at least twice the one before: together
    2^-4 |x| + 2^-9 of the block's scale.  A block that is filled at once is off by half a step."""
    rs = np.random.RandomState(int(10 * step))
    bs, n, d = 16, 48, 64
    pool = Pool(cuda, 1, 7, 2, bs, d)
    table = pool.table([n, n])
    bt = torch.from_numpy(table).to(cuda)
    x = rounded(rs.randn(2, n, d) * 2.0 ** (step * (np.arange(n) % bs - 15) + 2)[None, :, None] * np.exp(rs.randn(2, n, d)), dtype)
    for t in range(n):
        new = x[:, t:t + 1].astype(np.float32)
        gpu_append(pool, 0, bt, [t], [new], [new], dtype, row_ids=i32([0], cuda))
    whole = x.astype(np.float32)
    gpu_append(pool, 0, bt, [0], [whole], [whole], dtype, row_ids=i32([1], cuda))
    pool.download()
    for codes, scales in zip(pool.codes, pool.scales):
        for row, raised in ((0, True), (1, False)):
            got = f8.read(codes, scales, 0, table[row], n)
            s = np.repeat(scales[0][table[row]].T.astype(np.float64), bs, axis=1)[..., None]
            half = np.maximum(2.0 ** -4 * np.abs(x), 2.0 ** -10 * s)
            bound = 2.0 ** -4 * np.abs(x) + 2.0 ** -9 * s if raised else half
            assert (np.abs(got - x) <= bound).all()
            assert not raised or (np.abs(got - x) > half).any()  # (roundings on the way do add up)
        np.testing.assert_array_equal(scales[0][table[0]], scales[0][table[1]])  # the scale does not depend on the steps
