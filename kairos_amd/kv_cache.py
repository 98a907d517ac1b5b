"""A paged key-value cache of one decoder layer, in fp16, or quantised to 8 or 4 bits as it is written.

The pages of all sequences lie in one tensor; a page table (int32 [batch, pages a sequence], shared by the layers) says
which of them hold a sequence, in order.  int8 keeps one fp16 scale a row of head_dim elements, int4 a scale and an offset: at
head_dim 128 a token's key and value of one head take 512, 260 and 136 bytes in the three kinds."""
import torch

from . import ops


class PagedKVCache:
    """kind: 'f16', 'int8' or 'int4'; page_size: tokens a page, a multiple of 32; head_dim 64, 128 or 256.

    append() writes tokens (turning keys and queries by their positions on the way), attend() is the attention of one new
    token a sequence, read() hands back what the cache holds.  The methods add nothing to ops.kv_append, ops.paged_attention and
    ops.kv_read: `data` may be passed to those directly."""

    def __init__(self, num_pages, kv_heads, head_dim, kind="f16", page_size=64, device="cuda"):
        if int(page_size) <= 0 or int(page_size) % ops.KV_TILE:
            raise ValueError(f"PagedKVCache: page_size must be a positive multiple of {ops.KV_TILE}, got {page_size}")
        if int(num_pages) <= 0 or int(kv_heads) <= 0:
            raise ValueError(f"PagedKVCache: num_pages and kv_heads must be positive, got {num_pages} and {kv_heads}")
        self.kind, self.page_size, self.head_dim, self.kv_heads = kind, int(page_size), int(head_dim), int(kv_heads)
        self.data = torch.empty((int(num_pages), self.kv_heads, self.page_size // ops.KV_TILE, ops.kv_tile_bytes(head_dim, kind)),
                                dtype=torch.uint8, device=device)

    @property
    def bytes_per_token(self):
        """Of one token's keys and values, all heads."""
        return self.kv_heads * self.data.shape[-1] / ops.KV_TILE

    def append(self, page_table, start, k, v, table=None, q=None, interleaved=False, count=None, want_k=False):
        return ops.kv_append(self.data, page_table, start, k, v, table, q, interleaved, count, want_k)

    def read(self, page_table, start, length, count=None):
        return ops.kv_read(self.data, page_table, start, length, count)

    def attend(self, q, page_table, lens, scale=None, window=0):
        return ops.paged_attention(q, self.data, page_table, lens, scale, window)
