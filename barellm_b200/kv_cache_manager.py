"""Per-request block accounting on top of a BlockPool shard.

Contract of the reference's KVCacheManager (src/barellm/engine/kv_cache_manager.py:8-45):
``allocate_request`` tops a request up to ``ceil(seq_len / block_size)``
blocks and registers the (grown) list with the paged cache; it returns False,
allocating nothing, when the shard lacks free blocks.  ``free_request`` returns
the blocks and drops the request's pages.

``fork_request`` and ``compact`` have no counterpart there: several requests
that continue from one prefix (parallel samples, beams), and moving the pages in
use to the low end of the pool.
"""

from __future__ import annotations

from typing import Protocol

from .block_pool import BlockPool, KVCacheBlock
from .paged_kv_cache import PagedKVCache, PagedKVCacheView, check


class HasSeqLen(Protocol):
    id: str

    @property
    def seq_len(self) -> int: ...


class KVCacheManager:
    def __init__(self, block_size: int, block_pool: BlockPool, paged_kv_cache: PagedKVCache) -> None:
        self.block_size = block_size
        self.block_pool = block_pool
        self.paged_kv_cache = paged_kv_cache
        self.request_id_to_blocks: dict[str, list[KVCacheBlock]] = {}

    def blocks_needed(self, seq_len: int) -> int:
        return -(-seq_len // self.block_size)

    def get_cache(self, req: HasSeqLen) -> PagedKVCacheView:
        if req.id not in self.request_id_to_blocks:
            raise KeyError(f"Unknown request: {req.id}")
        return self.paged_kv_cache.get_cache(req.id)

    def allocate_request(self, req: HasSeqLen) -> bool:
        owned = self.request_id_to_blocks.get(req.id, [])
        missing = max(self.blocks_needed(req.seq_len) - len(owned), 0)
        if not self.block_pool.can_allocate(missing):
            return False
        grown = owned + self.block_pool.allocate(missing)
        self.request_id_to_blocks[req.id] = grown
        self.paged_kv_cache.register_request(req.id, grown)
        return True

    def free_request(self, request_id: str) -> None:
        blocks = self.request_id_to_blocks.pop(request_id, None)
        if blocks is not None:
            self.block_pool.free(blocks)
        self.paged_kv_cache.unregister_request(request_id)

    def fork_request(self, request_id: str, new_id: str) -> bool:
        """Registers ``new_id`` with the tokens that ``request_id`` has cached.

        Full blocks are shared (no token is ever written to a full block again);
        a partly filled last block is copied, since both requests go on writing
        to theirs.  False, changing nothing, when the pool lacks a block for that
        copy.  Call it between steps, when every layer holds the same tokens."""
        if request_id not in self.request_id_to_blocks:
            raise KeyError(f"Unknown request: {request_id}")
        check(new_id not in self.request_id_to_blocks, f"request already exists: {new_id}")
        lens = self.paged_kv_cache.request_pages[request_id].layer_seq_lens
        n = int(lens[0])
        check(bool((lens == n).all()), "a request can be forked between steps only: its layers hold different lengths")
        owned = self.request_id_to_blocks[request_id]
        full, rest = divmod(n, self.block_size)
        if not self.block_pool.can_allocate(1 if rest else 0):
            return False
        tail = self.block_pool.allocate(1) if rest else []
        if rest:
            try:
                self.paged_kv_cache.copy_blocks([owned[full].block_id], [tail[0].block_id])
            except Exception:
                self.block_pool.free(tail)
                raise
        self.block_pool.share(owned[:full])
        self.request_id_to_blocks[new_id] = owned[:full] + tail
        self.paged_kv_cache.register_request(new_id, self.request_id_to_blocks[new_id])
        self.paged_kv_cache.request_pages[new_id].layer_seq_lens[:] = n
        return True

    def compact(self) -> int:
        """Moves the blocks in use to the lowest ids, so that the free ones are
        the pool's end; returns how many were moved.  Requests keep their
        contents and lengths, their block tables are updated in place (on the
        current stream, behind the copies).  Every block in use must be held by
        this manager's requests."""
        pool = self.block_pool
        used = {b.block_id for blocks in self.request_id_to_blocks.values() for b in blocks}
        check(len(used) + len(pool.free_ids) == len(pool.blocks), "blocks are held outside this manager")
        src = sorted(i for i in used if i >= len(used))
        dst = sorted(i for i in pool.free_ids if i < len(used))
        if not src:
            return 0
        self.paged_kv_cache.copy_blocks(src, dst)
        moved = dict(zip(src, dst))
        pool.extra_holders = {moved.get(i, i): n for i, n in pool.extra_holders.items()}
        pool.free_ids = list(range(len(used), len(pool.blocks)))
        for request_id, blocks in self.request_id_to_blocks.items():
            if any(b.block_id in moved for b in blocks):
                blocks = [pool.blocks[moved.get(b.block_id, b.block_id)] for b in blocks]
                self.request_id_to_blocks[request_id] = blocks
                self.paged_kv_cache.register_request(request_id, blocks)
        return len(src)
