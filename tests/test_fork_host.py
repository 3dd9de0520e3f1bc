"""Forking, freeing and compacting requests: block accounting on the host (page
copies are recorded instead of made)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from barellm_b200 import BlockPool, KVCacheManager, PagedKVCache


class Req:
    def __init__(self, rid, n):
        self.id, self.seq_len = rid, n


class Recorder(PagedKVCache):
    """A pool whose page contents are one number per block."""

    def __init__(self, *a, **kw):
        super().__init__(*a, **kw)
        self.content = {}
        self.copies = []

    def copy_blocks(self, src, dst):
        assert len(set(dst)) == len(dst) and not set(src) & set(dst)
        self.copies.append((list(src), list(dst)))
        for a, b in zip(src, dst):
            self.content[b] = self.content.get(a)


def make(blocks=16, bs=4, layers=2):
    cache = Recorder(num_layers=layers, max_blocks=blocks, num_kv_heads=1, block_size=bs, head_dim=2)
    pool = BlockPool(blocks)
    return cache, pool, KVCacheManager(bs, pool, cache)


def grow(cache, man, rid, n, tag):
    """Registers ``n`` cached tokens for ``rid``, as an append would."""
    assert man.allocate_request(Req(rid, n))
    for i, b in enumerate(man.request_id_to_blocks[rid]):
        cache.content.setdefault(b.block_id, (tag, i))
    cache.request_pages[rid].layer_seq_lens[:] = n


def ids(man, rid):
    return [b.block_id for b in man.request_id_to_blocks[rid]]


def test_fork_shares_full_blocks_and_copies_the_last():
    cache, pool, man = make()
    grow(cache, man, "a", 10, "a")  # blocks of 4, 4, 2 tokens
    a = ids(man, "a")
    assert man.fork_request("a", "b")
    b = ids(man, "b")
    assert b[:2] == a[:2] and b[2] not in a
    assert cache.copies == [([a[2]], [b[2]])]
    assert (cache.request_pages["b"].layer_seq_lens == 10).all()
    assert cache.request_pages["b"].block_table.tolist() == b
    assert pool.num_free == 16 - 4
    # both grow on their own
    assert man.allocate_request(Req("a", 13)) and man.allocate_request(Req("b", 13))
    assert set(ids(man, "a")) & set(ids(man, "b")) == set(a[:2])
    # a block returns with its last holder, in any order
    man.free_request("a")
    assert pool.num_free == 16 - 4
    man.free_request("b")
    assert sorted(pool.free_ids) == list(range(16)) and not pool.extra_holders


def test_fork_at_a_block_border_copies_nothing():
    cache, pool, man = make()
    grow(cache, man, "a", 8, "a")
    assert man.fork_request("a", "b") and man.fork_request("a", "c") and man.fork_request("c", "d")
    assert cache.copies == [] and pool.num_free == 14
    assert ids(man, "a") == ids(man, "b") == ids(man, "c") == ids(man, "d")
    for rid in "cadb":
        assert pool.num_free == 14
        man.free_request(rid)
    assert pool.num_free == 16


def test_fork_leaves_spare_blocks_to_their_owner():
    cache, pool, man = make()
    grow(cache, man, "a", 6, "a")
    assert man.allocate_request(Req("a", 16))  # two blocks ahead of its tokens
    assert man.fork_request("a", "b")
    assert len(ids(man, "b")) == 2 and len(ids(man, "a")) == 4
    man.free_request("a")
    man.free_request("b")
    assert sorted(pool.free_ids) == list(range(16))


def test_fork_of_an_empty_request():
    cache, pool, man = make()
    assert man.allocate_request(Req("a", 0))
    assert man.fork_request("a", "b")
    assert ids(man, "b") == [] and cache.copies == []


def test_fork_refusals_change_nothing():
    cache, pool, man = make(blocks=3)
    with pytest.raises(KeyError):
        man.fork_request("a", "b")
    grow(cache, man, "a", 10, "a")
    with pytest.raises(ValueError, match="already exists"):
        man.fork_request("a", "a")
    assert not man.fork_request("a", "b")  # no block for the copy
    assert "b" not in man.request_id_to_blocks and "b" not in cache.request_pages and not pool.extra_holders
    cache.request_pages["a"].layer_seq_lens[1] = 11
    with pytest.raises(ValueError, match="between steps"):
        man.fork_request("a", "b")


def test_a_failed_copy_returns_its_block():
    cache, pool, man = make()
    grow(cache, man, "a", 10, "a")

    def fail(src, dst):
        raise RuntimeError("no device")

    cache.copy_blocks = fail
    with pytest.raises(RuntimeError, match="no device"):
        man.fork_request("a", "b")
    assert pool.num_free == 13 and not pool.extra_holders and "b" not in man.request_id_to_blocks


def test_compact_moves_blocks_in_use_to_the_low_end():
    rs = np.random.RandomState(1)
    cache, pool, man = make(blocks=64)
    want = {}
    for i in range(12):
        grow(cache, man, f"r{i}", int(rs.randint(1, 20)), f"r{i}")
    assert man.fork_request("r3", "f") and man.fork_request("f", "g")
    for i in (0, 2, 5, 6, 9, 11):
        man.free_request(f"r{i}")
    for rid in man.request_id_to_blocks:
        want[rid] = [cache.content[i] for i in ids(man, rid)]
    used = {i for rid in want for i in ids(man, rid)}
    moved = man.compact()
    assert moved == sum(i >= len(used) for i in used) > 0
    after = {i for rid in want for i in ids(man, rid)}
    assert after == set(range(len(used)))
    assert pool.free_ids == list(range(len(used), 64))
    for rid in want:
        assert [cache.content[i] for i in ids(man, rid)] == want[rid]
        assert cache.request_pages[rid].block_table.tolist() == ids(man, rid)
    assert man.compact() == 0
    for rid in list(want):
        man.free_request(rid)
    assert sorted(pool.free_ids) == list(range(64)) and not pool.extra_holders


def test_compact_refuses_blocks_it_does_not_know():
    cache, pool, man = make()
    grow(cache, man, "a", 3, "a")
    pool.allocate(2)
    with pytest.raises(ValueError, match="outside this manager"):
        man.compact()


def test_eight_bit_cache_construction():
    kw = dict(num_layers=2, max_blocks=3, num_kv_heads=2, block_size=4, head_dim=8)
    c = PagedKVCache(**kw, dtype=torch.bfloat16, kv_dtype=torch.float8_e4m3fn)
    assert c.quantized and c.dtype is torch.bfloat16 and c.key_cache.dtype is torch.float8_e4m3fn
    assert c.key_scale.shape == c.value_scale.shape == (2, 3, 2) and len(c.pools) == 4
    p = PagedKVCache(**kw, dtype=torch.float16, kv_dtype=torch.float16)
    assert not p.quantized and p.key_scale is None and len(p.pools) == 2
    with pytest.raises(ValueError, match="kv_dtype"):
        PagedKVCache(**kw, dtype=torch.float16, kv_dtype=torch.int8)
    with pytest.raises(ValueError, match="head_dim"):
        PagedKVCache(**dict(kw, head_dim=257), dtype=torch.float16, kv_dtype=torch.float8_e4m3fn)
