"""Free list of physical KV blocks, one per GPU shard.

Same contract as the reference's BlockPool (src/barellm/engine/block_pool.py:9-28):
``allocate(n)`` hands out the most recently freed / highest ids first and
returns ``[]`` when the pool cannot satisfy the request; ``free`` returns blocks
to the top of the stack.  Keeping that order keeps block tables identical to
the reference's for the same sequence of calls.

Blocks may have several holders (requests forked from one another): ``share``
adds one, and ``free`` returns a block to the stack when its last holder frees
it.
"""

from __future__ import annotations

from dataclasses import dataclass


@dataclass(slots=True)
class KVCacheBlock:
    block_id: int


class BlockPool:
    def __init__(self, max_blocks: int) -> None:
        self.blocks = [KVCacheBlock(i) for i in range(max_blocks)]
        # stack of free ids; the top of the stack is the end of the list
        self.free_ids: list[int] = list(range(max_blocks))
        self.extra_holders: dict[int, int] = {}  # block id -> holders beyond the first

    @property
    def num_free(self) -> int:
        return len(self.free_ids)

    def can_allocate(self, num_blocks: int) -> bool:
        return num_blocks <= len(self.free_ids)

    def allocate(self, num_blocks: int) -> list[KVCacheBlock]:
        if num_blocks > len(self.free_ids):
            return []
        if num_blocks <= 0:
            return []
        taken = self.free_ids[-num_blocks:]
        del self.free_ids[-num_blocks:]
        return [self.blocks[i] for i in reversed(taken)]

    def share(self, blocks: list[KVCacheBlock]) -> None:
        """Adds a holder to each block; ``free`` has to be called once more for it."""
        for b in blocks:
            self.extra_holders[b.block_id] = self.extra_holders.get(b.block_id, 0) + 1

    def free(self, blocks: list[KVCacheBlock]) -> None:
        if not self.extra_holders:
            self.free_ids.extend(b.block_id for b in blocks)
            return
        for b in blocks:
            n = self.extra_holders.get(b.block_id, 0)
            if n > 1:
                self.extra_holders[b.block_id] = n - 1
            elif n == 1:
                del self.extra_holders[b.block_id]
            else:
                self.free_ids.append(b.block_id)
