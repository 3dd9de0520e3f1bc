"""8-bit cache, host side (no GPU): the oracle's number format against torch's
e4m3 conversion, and the argument checks of the C entry points, which answer
before anything is launched."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from barellm_b200 import _native as nat
from barellm_b200 import ops
from oracle import fp8_oracle as f8


def test_oracle_code_values_are_torchs():
    got = torch.arange(256, dtype=torch.int32).to(torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(got, f8.VALUES)


def test_oracle_encodes_as_torch_does():
    rs = np.random.RandomState(0)
    mid = (f8.POSITIVE[:-1] + f8.POSITIVE[1:]) / 2  # ties
    x = np.concatenate([rs.randn(50000) * 2.0 ** rs.randint(-12, 9, 50000), mid, -mid, f8.VALUES[:127], [0.0, -0.0, 448.0, -448.0]])
    x = x.astype(np.float32)
    want = torch.from_numpy(x).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    np.testing.assert_array_equal(f8.encode(x), want)
    np.testing.assert_array_equal(f8.encode([np.inf, -np.inf, 1e9, np.nan]), [0x7E, 0xFE, 0x7E, 0x7F])


@pytest.mark.parametrize("amax,scale", [(0.0, 2.0 ** -100), (448.0, 1.0), (448.0001, 2.0), (224.0, 0.5), (1.0, 2.0 ** -8),
                                        (3.3e38, 2.0 ** 119)])
def test_scale_rule(amax, scale):
    assert f8.needed_scale(amax) == scale


def fake_layer(**kw) -> nat.Fp8Layer:
    """A layer whose pointers are never followed: the checks under test refuse it first."""
    p = dict(k_pool=4096, v_pool=8192, num_layers=2, num_blocks=8, num_kv_heads=2, block_size=16, head_dim=128,
             dtype=nat.BL_BF16, layer=1, block_tables=4096, bt_stride=4, bt_width=4, row_ids=None)
    scales = dict(k_scale=4096, v_scale=4096)
    for k, v in kw.items():
        (scales if k in scales else p)[k] = v
    return nat.Fp8Layer(nat.PagedLayer(**p), scales["k_scale"], scales["v_scale"])


BAD_LAYERS = [
    (dict(k_pool=None), nat.BL_ERR_ARG, "pool pointers"),
    (dict(k_pool=4100), nat.BL_ERR_ARG, "16-byte aligned"),
    (dict(k_scale=None), nat.BL_ERR_ARG, "scale pointers"),
    (dict(layer=2), nat.BL_ERR_ARG, "layer index"),
    (dict(dtype=7), nat.BL_ERR_DTYPE, "dtype"),
    (dict(head_dim=257), nat.BL_ERR_ARG, "head_dim"),
    (dict(block_size=1 << 20), nat.BL_ERR_ARG, "block_size"),
    (dict(block_tables=None), nat.BL_ERR_ARG, "block_tables"),
    (dict(bt_stride=3), nat.BL_ERR_ARG, "stride"),
]


def entry_points(layer):
    app = nat.AppendFp8Args(layer=layer, k_new=4096, v_new=4096, start_pos=4096, batch=1, max_new_tokens=1)
    gat = nat.GatherFp8Args(layer=layer, seq_lens=4096, batch=1, k_out=4096, v_out=4096, max_len=1)
    dec = nat.DecodeFp8Args(layer=layer, q=4096, out=4096, seq_lens=4096, batch=1, num_q_heads=4, scale=1.0, max_seq_len=16,
                            workspace=4096, workspace_bytes=1 << 30)
    pre = nat.PrefillFp8Args(layer=layer, q=4096, out=4096, seq_lens=4096, batch=1, num_q_heads=4, max_q_len=2, scale=1.0,
                             total_q_len=2, max_seq_len=16, total_blocks=1, workspace=4096, workspace_bytes=1 << 30)
    return {"bl_paged_append_fp8": app, "bl_paged_gather_fp8": gat, "bl_paged_decode_fp8": dec, "bl_paged_prefill_fp8": pre}


@pytest.mark.parametrize("change,rc,text", BAD_LAYERS, ids=[t for _, _, t in BAD_LAYERS])
def test_bad_layers_are_refused(native_lib, change, rc, text):
    for name, args in entry_points(fake_layer(**change)).items():
        assert getattr(native_lib, name)(ctypes.byref(args), None) == rc, name
        assert text in nat.last_error(), (name, nat.last_error())


@pytest.mark.parametrize("name,change,rc", [
    ("bl_paged_append_fp8", dict(k_new=None), nat.BL_ERR_ARG),
    ("bl_paged_append_fp8", dict(v_new=4097), nat.BL_ERR_ARG),
    ("bl_paged_append_fp8", dict(batch=0), nat.BL_ERR_ARG),
    ("bl_paged_append_fp8", dict(batch=65536), nat.BL_ERR_ARG),
    ("bl_paged_append_fp8", dict(max_new_tokens=0), nat.BL_ERR_ARG),
    ("bl_paged_gather_fp8", dict(max_len=0), nat.BL_ERR_ARG),
    ("bl_paged_gather_fp8", dict(k_out=4097), nat.BL_ERR_ARG),
    ("bl_paged_decode_fp8", dict(num_q_heads=3), nat.BL_ERR_ARG),
    ("bl_paged_decode_fp8", dict(max_seq_len=0), nat.BL_ERR_ARG),
    ("bl_paged_decode_fp8", dict(workspace=None), nat.BL_ERR_CAPACITY),
    ("bl_paged_decode_fp8", dict(workspace_bytes=100), nat.BL_ERR_CAPACITY),
    ("bl_paged_decode_fp8", dict(workspace=4100), nat.BL_ERR_ARG),
    ("bl_paged_decode_fp8", dict(q=4097), nat.BL_ERR_ARG),
    ("bl_paged_prefill_fp8", dict(max_q_len=0), nat.BL_ERR_ARG),
    ("bl_paged_prefill_fp8", dict(total_blocks=0), nat.BL_ERR_ARG),
    ("bl_paged_prefill_fp8", dict(total_q_len=1), nat.BL_ERR_ARG),
    ("bl_paged_prefill_fp8", dict(workspace_bytes=100), nat.BL_ERR_CAPACITY),
    ("bl_paged_prefill_fp8", dict(num_q_heads=5), nat.BL_ERR_ARG),
])
def test_bad_arguments_are_refused(native_lib, name, change, rc):
    args = entry_points(fake_layer())[name]
    for k, v in change.items():
        setattr(args, k, v)
    assert getattr(native_lib, name)(ctypes.byref(args), None) == rc, nat.last_error()
    assert getattr(native_lib, name)(None, None) == nat.BL_ERR_ARG


@pytest.mark.parametrize("src,dst,text", [
    ([0, 1], [2, 2], "written twice"),
    ([0, 1], [1, 2], "read and written"),
    ([3], [3], "read and written"),
    ([0], [8], "outside the pool"),
    ([-1], [2], "outside the pool"),
    (list(range(8)) + [0], [0] * 9, "more pairs"),
    (list(range(40)), list(range(50, 89)) + [50], "written twice"),  # (many pairs are checked another way)
    (list(range(40)), list(range(50, 89)) + [7], "read and written"),
    (list(range(40)), list(range(61, 101)), "outside the pool"),
])
def test_bad_copy_pairs_are_refused(native_lib, src, dst, text):
    s, d = np.asarray(src, dtype=np.int64), np.asarray(dst, dtype=np.int64)
    blocks = 8 if len(src) < 40 else 100
    a = nat.CopyBlocksArgs(4096, 4096, None, None, 2, blocks, 2, 16, 128, 2, s.ctypes.data, d.ctypes.data, len(src))
    assert native_lib.bl_copy_blocks(ctypes.byref(a), None) == nat.BL_ERR_ARG
    assert text in nat.last_error()


def test_packed_arguments_are_the_structures(native_lib):
    """The byte strings that ops passes are the ctypes structures, field for field."""
    rs = np.random.RandomState(0)
    for name, cls in nat.STRUCTS.items():
        if not hasattr(nat, "pack_" + name[3:]):
            continue
        pack = getattr(nat, "pack_" + name[3:])

        def fields(c):
            for f, t in c._fields_:
                if issubclass(t, ctypes.Structure):
                    yield from ((f + "." + g, u) for g, u in fields(t))
                else:
                    yield f, t

        vals = [float(rs.randint(1, 100)) if t is ctypes.c_float else int(rs.randint(1, 1 << 30)) for _, t in fields(cls)]
        data = pack(*vals)
        assert len(data) == ctypes.sizeof(cls), name
        got = cls.from_buffer_copy(data)
        for (path, _), v in zip(fields(cls), vals):
            x = got
            for part in path.split("."):
                x = getattr(x, part)
            assert x == v, (name, path)


def test_copy_of_nothing_is_nothing(native_lib):
    a = nat.CopyBlocksArgs(4096, 4096, None, None, 2, 8, 2, 16, 128, 2, None, None, 0)
    assert native_lib.bl_copy_blocks(ctypes.byref(a), None) == nat.BL_OK
    a = nat.CopyBlocksArgs(4096, 4096, 4096, None, 2, 8, 2, 16, 128, 2, None, None, 0)
    assert native_lib.bl_copy_blocks(ctypes.byref(a), None) == nat.BL_ERR_ARG


def test_workspace_sizes(native_lib):
    # 64 rows of at most one chunk: a plan, no partials
    assert ops.decode_fp8_workspace_bytes(64, 16, 128, 512) < 4096
    assert ops.decode_fp8_workspace_bytes(64, 16, 128, 513) >= 64 * 2 * 16 * 129 * 4
    assert ops.decode_fp8_workspace_bytes(0, 16, 128, 512) == 0
    f = native_lib.bl_paged_prefill_fp8_workspace_bytes
    one = f(nat.BL_BF16, 4, 16, 8, 128, 16, 500, 1000, 40)
    assert one >= 2 * 40 * 8 * 16 * 128 * 2
    assert f(nat.BL_BF16, 4, 24, 8, 128, 16, 500, 1000, 40) > 2 * one  # group 3: every KV head three times
    # narrower heads: q and out widened to 128 dims as well
    assert f(nat.BL_BF16, 4, 16, 8, 64, 16, 500, 1000, 40) >= one + 2 * 500 * 16 * 128 * 2
    assert f(nat.BL_F32, 4, 16, 8, 128, 16, 500, 1000, 40) == 0
    assert f(nat.BL_BF16, 4, 16, 8, 256, 16, 500, 1000, 40) == 0
    assert f(nat.BL_BF16, 4, 16, 8, 12, 16, 500, 1000, 40) == 0


def test_cpu_tensors_are_refused():
    kc = torch.zeros((1, 2, 1, 16, 64), dtype=torch.float8_e4m3fn)
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        ops.copy_blocks(kc, kc, [0], [1])


def test_small_decode_calls_need_no_scratch(native_lib):
    """(64 blocks of 2 KV heads: what fits 148 SMs at once and has at most 8 chunks a row)"""
    def need(dtype=nat.BL_BF16, **kw):
        a = entry_points(fake_layer(dtype=dtype))["bl_paged_decode_fp8"]
        a.workspace, a.workspace_bytes = None, 0
        for k, v in kw.items():
            setattr(a, k, v)
        n = native_lib.bl_paged_decode_fp8_scratch_bytes(ctypes.byref(a))
        if n:
            assert n == native_lib.bl_paged_decode_fp8_workspace_bytes(a.batch, a.num_q_heads, a.layer.kv.head_dim, a.max_seq_len)
            assert native_lib.bl_paged_decode_fp8(ctypes.byref(a), None) == nat.BL_ERR_CAPACITY
        return n
    assert need(max_seq_len=16) == need(max_seq_len=4096) == need(max_seq_len=512, batch=8) == 0
    assert need(max_seq_len=4097) and need(max_seq_len=512, batch=33) and need(max_seq_len=4096, batch=32)
    assert need(dtype=nat.BL_F32, max_seq_len=16) and need(max_seq_len=0) == need(num_q_heads=3) == 0
    assert native_lib.bl_paged_decode_fp8_scratch_bytes(None) == 0


@pytest.mark.parametrize("ids", [[3, 1, 2], (3, 1, 2), np.array([3, 1, 2], dtype=np.int32), np.array([3, 0, 1, 0, 2, 0])[::2],
                                 np.array([3, 1, 2], dtype=np.uint8), range(3, 0, -1)])
def test_block_ids_of_any_host_sequence(ids):
    owner, at, n = ops._block_ids(ids, "src")
    got = list((ctypes.c_int64 * n).from_address(at))
    assert got == [int(i) for i in ids]
    assert ops._block_ids([], "src")[2] == ops._block_ids(np.zeros(0), "src")[2] == 0


@pytest.mark.parametrize("ids", [[1.5], [True, 2], [1, 2.0], [[1, 2]], ["a"], (None,), [2 ** 70], np.array([1.0]), np.array([[1, 2]])])
def test_what_is_no_block_id_is_refused(ids):
    with pytest.raises(ValueError, match="dst must be a sequence of block ids"):
        ops._block_ids(ids, "dst")
