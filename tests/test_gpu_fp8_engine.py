"""The 8-bit cache as a serving engine uses it: the cache classes, the attention
backend, forked requests and the engine's steps, together."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from barellm_b200 import (BatchKVCache, BlockPool, CudaPagedAttentionBackend, KVCacheManager, PackedBatchKVCache, PagedKVCache,
                          ops)
from barellm_b200.engine import PagedEngine, Qwen3Shape, apply_rope, random_qwen3, rope_cos_sin
from fp8_helpers import assert_within, attention_bound
from oracle import fp8_oracle as f8

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn


class Req:
    def __init__(self, rid, n):
        self.id, self.seq_len = rid, n


def setup(device, dtype, *, layers=2, blocks=96, hkv=2, bs=16, d=128):
    cache = PagedKVCache(layers, blocks, hkv, bs, d, dtype=dtype, device=device, kv_dtype=F8)
    return cache, KVCacheManager(bs, BlockPool(blocks), cache)


def values(cache, rid, layer):
    """A request's cached K and V, float64, as the oracle reads the device's codes."""
    pages = cache.request_pages[rid]
    n = int(pages.layer_seq_lens[layer])
    ids = [b.block_id for b in pages.blocks]
    return [f8.read(c.view(torch.uint8).cpu().numpy(), s.cpu().numpy(), layer, ids, n)
            for c, s in ((cache.key_cache, cache.key_scale), (cache.value_cache, cache.value_scale))]


def check_rows(cache, rids, layer, out, q):
    """out / q: [B, Hq, T, D] of the rows' last T tokens."""
    eps = torch.finfo(q.dtype).eps / 2 if q.shape[2] > 1 else 2.0 ** -11
    for b, rid in enumerate(rids):
        k, v = values(cache, rid, layer)
        qn = q[b].double().cpu().numpy()
        want, spread, reach, flat = f8.attention(qn, k, v)
        assert_within(out[b].double().cpu().numpy(), want,
                      attention_bound(want, spread, reach, flat, qn, q.dtype, eps, k.shape[1]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_steps_of_a_batch(cuda, native_lib, dtype):
    """Packed chunked prefill, then decode steps, every layer; the backend's outputs against the codes in the pool."""
    cache, man = setup(cuda, dtype)
    be = CudaPagedAttentionBackend()
    g = torch.Generator(device=cuda).manual_seed(0)
    mk = lambda *s: torch.randn(*s, generator=g, device=cuda).to(dtype)
    rids, lens = ["a", "b", "c"], [70, 16, 1]
    for r, n in zip(rids, lens):
        assert man.allocate_request(Req(r, n + 8))
    done = [0, 0, 0]
    for part in (0.5, 1.0):  # two chunks each
        chunk = [max(1, int(n * part) - d) if int(n * part) > d else 0 for n, d in zip(lens, done)]
        live = [i for i, c in enumerate(chunk) if c]
        packed = PackedBatchKVCache([man.get_cache(Req(rids[i], 0)) for i in live], [chunk[i] for i in live])
        total = sum(chunk)
        for layer in range(2):
            q, k, v = mk(1, 8, total, 128), mk(1, 2, total, 128), mk(1, 2, total, 128)
            out = be.attend(q, k, v, packed.layer(layer), 4)
            at = 0
            for i in live:
                check_rows(cache, [rids[i]], layer, out[:, :, at:at + chunk[i]], q[:, :, at:at + chunk[i]])
                at += chunk[i]
        done = [d + c for d, c in zip(done, chunk)]
    assert done == lens
    for step in range(5):
        batch = BatchKVCache([man.get_cache(Req(r, 0)) for r in rids])
        for layer in range(2):
            q, k, v = mk(3, 8, 1, 128), mk(3, 2, 1, 128), mk(3, 2, 1, 128)
            out = be.attend(q, k, v, batch.layer(layer), 4)
            assert out.shape == q.shape
            check_rows(cache, rids, layer, out, q)
    # several tokens a row at once, one request alone, and the dense read
    batch = BatchKVCache([man.get_cache(Req(r, 0)) for r in rids])
    q, k, v = mk(3, 8, 3, 128), mk(3, 2, 3, 128), mk(3, 2, 3, 128)
    check_rows(cache, rids, 0, be.attend(q, k, v, batch.layer(0), 4), q)
    kd, vd = BatchKVCache([man.get_cache(Req(r, 0)) for r in rids]).layer(0).read()
    for b, r in enumerate(rids):
        kw, vw = values(cache, r, 0)
        n = kw.shape[1]
        assert torch.equal(kd[b, :, :n].double().cpu(), torch.from_numpy(kw)) and not bool(kd[b, :, n:].any())
        assert torch.equal(vd[b, :, :n].double().cpu(), torch.from_numpy(vw))
        one = man.get_cache(Req(r, 0)).layer(0)
        assert torch.equal(one.read()[0][0], kd[b, :, :n])
    for t in (1, 2):
        one = man.get_cache(Req("b", 0)).layer(1)
        q, k, v = mk(1, 8, t, 128), mk(1, 2, t, 128), mk(1, 2, t, 128)
        check_rows(cache, ["b"], 1, be.attend(q, k, v, one, 4), q)
    cache.check_device_errors()


@pytest.mark.parametrize("kind", ["batch", "packed", "single"])
def test_prepped_append_is_norm_rope_append(cuda, native_lib, kind):
    """attend_prepped leaves the same codes and outputs as attend of the prepared q and k."""
    dtype = torch.bfloat16
    g = torch.Generator(device=cuda).manual_seed(1)
    mk = lambda *s: torch.randn(*s, generator=g, device=cuda).to(dtype)
    rids, lens = (["a", "b"], [9, 30]) if kind != "single" else (["a"], [20])
    qw, kw = 1 + mk(128) / 8, 1 + mk(128) / 8
    results = []
    x = None
    for prepped in (False, True):
        cache, man = setup(cuda, dtype)
        be = CudaPagedAttentionBackend()
        for r, n in zip(rids, lens):
            assert man.allocate_request(Req(r, n + 4))
        views = [man.get_cache(Req(r, 0)) for r in rids]
        if kind == "packed":
            b, t, layer = 1, sum(lens), PackedBatchKVCache(views, lens).layer(1)
        elif kind == "batch":
            b, t, layer = 2, 3, BatchKVCache(views).layer(1)
        else:
            b, t, layer = 1, 20, views[0].layer(1)
        if x is None:
            x = mk(b, t, 8, 128).transpose(1, 2), mk(b, t, 2, 128).transpose(1, 2), mk(b, t, 2, 128).transpose(1, 2)
            pos = torch.arange(t, device=cuda).unsqueeze(0).expand(b, t)
            cos, sin = rope_cos_sin(128, 1e4, pos, dtype)
        q, k, v = x
        if prepped:
            out = be.attend_prepped(q, k, v, qw, kw, 1e-6, cos, sin, layer, 4)
        else:
            # the same kernel into a plain scratch pool gives the prepared q and k
            kp = torch.empty((1, b, 2, t, 128), dtype=dtype, device=cuda)
            qp = ops.qk_norm_rope_append(q, k, v, qw, kw, cos, sin, 1e-6, kp, torch.empty_like(kp), 0,
                                         torch.arange(b, dtype=torch.int32, device=cuda).view(b, 1),
                                         torch.zeros(b, dtype=torch.int32, device=cuda))
            norm = lambda y, w: (y.float() * torch.rsqrt(y.float().pow(2).mean(-1, keepdim=True) + 1e-6) * w).to(dtype)
            assert (kp[0].float() - apply_rope(norm(k, kw), cos, sin).float()).abs().max() < 0.1  # (it is that key)
            out = be.attend(qp, kp[0], v, layer, 4)
        results.append((out, cache))
    (o0, c0), (o1, c1) = results
    assert torch.equal(o0, o1)
    for r in rids:
        for a, b in zip(values(c0, r, 1), values(c1, r, 1)):
            np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("kv_dtype", [F8, torch.bfloat16])
def test_forked_requests_go_their_own_ways(cuda, native_lib, kv_dtype):
    """Children of a fork continue exactly as requests that were built alone, and
    leave their parent as it was; compaction moves pages under them."""
    dtype = torch.bfloat16
    cache = PagedKVCache(3, 64, 2, 16, 128, dtype=dtype, device=cuda, kv_dtype=kv_dtype)
    pool = BlockPool(64)
    man = KVCacheManager(16, pool, cache)
    g = torch.Generator(device=cuda).manual_seed(2)
    mk = lambda n, size=1.0: [(size * torch.randn(1, 2, n, 128, generator=g, device=cuda)).to(dtype) for _ in range(2)]

    def append(rid, kv):
        n = int(cache.request_pages[rid].layer_seq_lens[0]) if rid in cache.request_pages else 0
        assert man.allocate_request(Req(rid, n + kv[0].shape[2]))
        for layer in range(3):
            man.get_cache(Req(rid, 0)).layer(layer).append_only(kv[0], kv[1])

    def read(rid):
        return [t for layer in range(3) for t in man.get_cache(Req(rid, 0)).layer(layer).read()]

    for n in (37, 32):  # a partly filled last block, and none
        prompt = mk(n)
        more = {c: mk(20, 4.0 ** i) for i, c in enumerate("xyz")}  # larger tokens raise the copied block's scale
        append("p", prompt)
        before = read("p")
        for c in "xy":
            assert man.fork_request("p", c)
        append("x", more["x"])
        append("y", more["y"])
        assert man.fork_request("x", "z")
        append("z", more["z"])
        for a, b in zip(read("p"), before):
            assert torch.equal(a, b)
        want = {}
        for c, parts in (("x", [prompt, more["x"]]), ("y", [prompt, more["y"]]), ("z", [prompt, more["x"], more["z"]])):
            for p in parts:
                append("alone", p)
            want[c] = read("alone")
            man.free_request("alone")
            for a, b in zip(read(c), want[c]):
                assert torch.equal(a, b)
        man.free_request("p")
        assert man.compact() > 0 or n == 32  # (the second time the low blocks are the ones in use)
        for c in "xyz":
            for a, b in zip(read(c), want[c]):
                assert torch.equal(a, b)
        assert max(b.block_id for c in "xyz" for b in man.request_id_to_blocks[c]) == 64 - pool.num_free - 1
        append("x", mk(5))
        for c in "yz":
            for a, b in zip(read(c), want[c]):
                assert torch.equal(a, b)
            man.free_request(c)
        man.free_request("x")
        assert pool.num_free == 64 and not pool.extra_holders
    cache.check_device_errors()


def test_engine_runs_on_an_eight_bit_cache(cuda, native_lib):
    """Prefill in chunks and decode, eager and as a captured graph: the same tokens, the pool empty at the end."""
    shape = Qwen3Shape(vocab_size=512, hidden_size=256, intermediate_size=512, head_dim=128, num_layers=3, num_heads=8,
                       num_kv_heads=2)
    model = random_qwen3(shape, dtype=torch.bfloat16, device=cuda, seed=3)
    rs = np.random.RandomState(0)
    prompts = [rs.randint(0, 512, n).tolist() for n in (5, 130, 33, 64)]
    outs = []
    for graph in (False, True):
        eng = PagedEngine(model, 64, prefill_tokens=96, kv_dtype=F8)
        outs.append(eng.generate(prompts, 24, use_graph=graph))
        assert eng.pool.num_free == 64
    assert outs[0] == outs[1]
    assert all(len(o) == 24 for o in outs[0])
    # the first token needs no decode step: it agrees with the 16-bit cache unless the logits nearly tie
    full = PagedEngine(model, 64, prefill_tokens=96).generate(prompts, 24)
    assert sum(a[0] == b[0] for a, b in zip(outs[0], full)) >= 3
