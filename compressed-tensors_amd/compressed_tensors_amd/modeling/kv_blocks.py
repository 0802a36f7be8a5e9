"""A KV cache that holds its tokens in 8 bits: blocks of tokens with a scale per block and
head, the calls that plan, fill and read it, and `BlockKVCache`, which keeps them together
for the layers of a model.

The reference's cache quantizes and dequantizes what it is given and keeps 16 bits
(modeling/kvcache.py:41-96, `QuantizedKVCache`); codes and scales here follow the same
`calculate_qparams` rules, and there is no counterpart of the block cache in it.
"""
import ctypes
from typing import List, NamedTuple, Optional, Tuple

import torch
from torch import Tensor

from compressed_tensors_amd import _lib

__all__ = ["BlockKVCache", "KVBlocks", "KVPlan", "append_kv_blocks", "attend_kv_blocks", "plan_kv_blocks"]

_INPUTS = (torch.bfloat16, torch.float16)
_CODES = (torch.float8_e4m3fn, torch.int8)


class KVBlocks(NamedTuple):
    """One layer's pool.  Positions of a block that no token was written to may hold anything."""

    key: Tensor          # [blocks, kv_heads, block_size, head_dim] float8_e4m3fn or int8
    value: Tensor        # [blocks, kv_heads, head_dim, block_size], tokens innermost
    key_scale: Tensor    # [blocks, kv_heads] float32
    value_scale: Tensor  # [blocks, kv_heads] float32

    @classmethod
    def allocate(cls, num_blocks: int, kv_heads: int, head_dim: int, block_size: int = 64,
                 dtype: torch.dtype = torch.float8_e4m3fn, device="cuda") -> "KVBlocks":
        """an empty pool (scales of one; codes are whatever the memory held)"""
        codes = [torch.empty(shape, dtype=dtype, device=device)
                 for shape in ((num_blocks, kv_heads, block_size, head_dim), (num_blocks, kv_heads, head_dim, block_size))]
        scales = [torch.ones((num_blocks, kv_heads), dtype=torch.float32, device=device) for _ in codes]
        blocks = cls(*codes, *scales)
        _describe(blocks)
        return blocks


class KVPlan(NamedTuple):
    """What `plan_kv_blocks` returns: the state after the step and where its tokens go."""

    seq_lens: Tensor     # int32 [requests]
    query_start: Tensor  # int32 [requests + 1]
    slots: Tensor        # int64 [total_tokens]
    block_table: Tensor  # int32 [requests, width]
    free_blocks: Tensor  # int32 [capacity]
    num_free: Tensor     # int32 [1]
    status: Tensor       # int32 [1]


def _describe(blocks: KVBlocks) -> _lib.KVBlocksC:
    """the pool as the library takes it, checked"""
    key, value, key_scale, value_scale = blocks
    if key.ndim != 4:
        raise ValueError(f"expected keys [blocks, heads, block size, head dim], got {tuple(key.shape)}")
    n, heads, size, dim = key.shape
    if value.shape != (n, heads, dim, size):
        raise ValueError(f"expected values {(n, heads, dim, size)}, got {tuple(value.shape)}")
    if key_scale.shape != (n, heads) or value_scale.shape != (n, heads):
        raise ValueError(f"expected scales {(n, heads)}, got {tuple(key_scale.shape)} and {tuple(value_scale.shape)}")
    if key.dtype not in _CODES or value.dtype is not key.dtype:
        raise NotImplementedError(f"codes must be float8_e4m3fn or int8, got {key.dtype} and {value.dtype}")
    if key_scale.dtype is not torch.float32 or value_scale.dtype is not torch.float32:
        raise ValueError(f"scales must be float32, got {key_scale.dtype} and {value_scale.dtype}")
    if dim not in (64, 128, 256):
        raise NotImplementedError(f"head_dim must be 64, 128 or 256, got {dim}")
    if size % 16 or not 16 <= size <= 256:
        raise NotImplementedError(f"block_size must be a multiple of 16 up to 256, got {size}")
    if not (key.is_contiguous() and value.is_contiguous() and key_scale.is_contiguous() and value_scale.is_contiguous()):
        raise ValueError("the tensors of a pool must be contiguous")
    return _lib.KVBlocksC(key.data_ptr(), value.data_ptr(), key_scale.data_ptr(), value_scale.data_ptr(),
                          n, heads, dim, size, _lib.dtype_code(key.dtype))


def _ints(name: str, t: Tensor, dtype: torch.dtype, count: Optional[int] = None) -> Tensor:
    """`t`, contiguous, after a check that it is a list of `count` (None: any number) integers"""
    if t.dtype is not dtype or t.ndim != 1 or (count is not None and t.shape[0] != count):
        raise ValueError(f"{name}: expected {dtype} [{'*' if count is None else count}], got {t.dtype} {tuple(t.shape)}")
    return t.contiguous()


def plan_kv_blocks(seq_lens: Tensor, new_tokens: Tensor, block_table: Tensor, free_blocks: Tensor,
                   num_free: Tensor, *, block_size: int, total_tokens: int) -> KVPlan:
    """The bookkeeping of one serving step, on the GPU and without waiting for it.

    Request r holds `seq_lens[r]` tokens in the blocks `block_table[r]` names and gains
    `new_tokens[r]`; a negative number ends it: its blocks go back and its length becomes 0.
    `free_blocks[:num_free]` is a stack of free blocks.  What ended requests return is pushed
    first, so it is used again in the same step; blocks are popped in request order.

    `total_tokens` is the length of `slots`: the sum of the new tokens, or more (a padded
    batch: the rest is -1).  `status` is 0, or the step did not fit and changed nothing (every
    slot is -1): a positive number of missing blocks, -1 for a request longer than its table
    row, -2 for more than `total_tokens` tokens, -3 for a free list that cannot be.  The
    inputs stay as they are; all tensors int32 on one GPU."""
    lens = _ints("seq_lens", seq_lens, torch.int32)
    requests = lens.shape[0]
    add = _ints("new_tokens", new_tokens, torch.int32, requests)
    free = _ints("free_blocks", free_blocks, torch.int32)
    count = _ints("num_free", num_free, torch.int32, 1)
    if block_table.dtype is not torch.int32 or block_table.ndim != 2 or block_table.shape[0] != requests:
        raise ValueError(f"block_table: expected {torch.int32} [{requests}, *], got {block_table.dtype} {tuple(block_table.shape)}")
    width, capacity = block_table.shape[1], free.shape[0]
    if total_tokens < 0 or block_size < 1 or width < 1:
        raise ValueError(f"bad sizes: {total_tokens} tokens, blocks of {block_size}, {width} table columns")
    index = _lib.gpu_index(lens, add, block_table, free, count)
    if not _lib.is_current(index):
        with torch.cuda.device(index):
            return plan_kv_blocks(lens, add, block_table, free, count, block_size=block_size, total_tokens=total_tokens)
    table = block_table.contiguous()
    # one allocation for the 32-bit outputs
    lens_out, start, table_out, free_out, count_out, status = lens.new_empty(
        2 * requests + requests * width + capacity + 3).split_with_sizes(
            (requests, requests + 1, requests * width, capacity, 1, 1))
    slots = torch.empty(total_tokens, dtype=torch.int64, device=lens.device)
    _lib.check(_lib.load().ctmi_kv_plan(
        lens.data_ptr(), add.data_ptr(), table.data_ptr(), free.data_ptr(), count.data_ptr(), requests, width,
        capacity, total_tokens, block_size, lens_out.data_ptr(), start.data_ptr(), slots.data_ptr(),
        table_out.data_ptr(), free_out.data_ptr(), count_out.data_ptr(), status.data_ptr(),
        _lib.stream_of_index(index)))
    return KVPlan(lens_out, start, slots, table_out.view(requests, width), free_out, count_out, status)


def append_kv_blocks(key: Tensor, value: Tensor, blocks: KVBlocks, slots: Tensor, *, dynamic: bool = True) -> None:
    """Write new keys and values [tokens, kv_heads, head_dim] into the pool, in place.

    `slots[t]` is block * block_size + position of token t; one outside the pool (-1) skips the
    token.  Tokens of one block stand next to each other in rising order and a slot is named
    once, as `plan_kv_blocks` gives them.  Where slots are left out, or tokens skipped, inside a
    block, its runs of consecutive slots are written one after the other, as by calls of their own.

    dynamic: the scale of a block and head is the largest new |x| over half the range of the
    codes (448 or 127.5), never below fp32's eps, and never falls while the block fills; where
    it grows, the block's older codes are rewritten to it.  A block whose first position is
    a new token's starts afresh.  Otherwise the scales are the caller's and x / scale
    saturates.  Forward only."""
    c = _describe(blocks)
    if key.ndim != 3 or value.shape != key.shape or key.shape[1] != c.kv_heads or key.shape[2] != c.head_dim:
        raise ValueError(f"expected keys and values [tokens, {c.kv_heads}, {c.head_dim}], got "
                         f"{tuple(key.shape)} and {tuple(value.shape)}")
    if key.dtype not in _INPUTS or value.dtype is not key.dtype:
        raise NotImplementedError(f"keys and values must be bfloat16 or float16, got {key.dtype} and {value.dtype}")
    if _lib.differentiated(key, value):
        raise NotImplementedError("append_kv_blocks has no backward and no forward-mode derivative: call it under "
                                  "torch.no_grad() with plain tensors")
    slots = _ints("slots", slots, torch.int64, key.shape[0])
    index = _lib.gpu_index(key, value, slots, *blocks)
    if not _lib.is_current(index):
        with torch.cuda.device(index):
            return append_kv_blocks(key, value, blocks, slots, dynamic=dynamic)
    key, value = _aligned(key), _aligned(value)
    (kt, kh, _), (vt, vh, _) = key.stride(), value.stride()
    _lib.check(_lib.load().ctmi_kv_append(
        key.data_ptr(), value.data_ptr(), _lib.dtype_code(key.dtype), kt, kh, vt, vh, slots.data_ptr(), key.shape[0],
        ctypes.byref(c), int(dynamic), _lib.stream_of_index(index)))


def _aligned(t: Tensor) -> Tensor:
    """`t` [tokens, heads, dim], or a copy if its heads do not start at 16-byte boundaries"""
    token, head, inner = t.stride()
    if inner == 1 and head % 8 == 0 and token % 8 == 0 and token < 1 << 22 and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def attend_kv_blocks(query: Tensor, blocks: KVBlocks, block_table: Tensor, seq_lens: Tensor,
                     query_start: Optional[Tensor] = None, *, max_query: Optional[int] = None,
                     max_seq: Optional[int] = None, softmax_scale: Optional[float] = None,
                     out: Optional[Tensor] = None) -> Tensor:
    """Causal attention of new tokens over the pool.

    query [tokens, q_heads, head_dim]; request r's queries are the tokens
    `query_start[r]:query_start[r + 1]` (None: one each), the last of its `seq_lens[r]` keys,
    which are in the pool already.  Query i of n sees the keys up to position seq_lens[r] - n +
    i; one that sees none gives zeros.  q_heads is a multiple of the pool's heads: neighbouring
    query heads share one.  `softmax_scale` defaults to head_dim ** -0.5.

    `max_query` and `max_seq`, the longest request's queries and keys, choose the launch, and
    with more than 64 queries x heads a kv head how many bits a softmax weight keeps on its way
    into bfloat16 outputs (11, else 24); any values give the right result.  Without `max_query`
    a batch of no more tokens than requests is taken for a decode step, any other for prompts,
    and a batch of very different requests is better left without it; `max_seq` defaults to the
    table's width.  Rows of
    tokens outside every request (a padded batch) keep what `out` holds; without `out` they are
    zeros.  Forward only."""
    c = _describe(blocks)
    if query.ndim != 3 or query.shape[2] != c.head_dim or query.shape[1] < 1 or query.shape[1] % c.kv_heads:
        raise ValueError(f"expected queries [tokens, a multiple of {c.kv_heads}, {c.head_dim}], got {tuple(query.shape)}")
    if query.dtype not in _INPUTS:
        raise NotImplementedError(f"queries must be bfloat16 or float16, got {query.dtype}")
    if _lib.differentiated(query):
        raise NotImplementedError("attend_kv_blocks has no backward and no forward-mode derivative: call it under "
                                  "torch.no_grad() with plain tensors")
    lens = _ints("seq_lens", seq_lens, torch.int32)
    requests, (tokens, heads, dim) = lens.shape[0], query.shape
    if block_table.dtype is not torch.int32 or block_table.ndim != 2 or block_table.shape[0] != requests:
        raise ValueError(f"block_table: expected {torch.int32} [{requests}, *], got {block_table.dtype} {tuple(block_table.shape)}")
    width = block_table.shape[1]
    if query_start is not None:
        query_start = _ints("query_start", query_start, torch.int32, requests + 1)
    elif tokens != requests:
        raise ValueError(f"without query_start every request has one token: got {tokens} tokens for {requests} requests")
    if out is not None:
        if out.shape != query.shape or out.dtype is not query.dtype or not out.is_contiguous() or out.data_ptr() % 16:
            raise ValueError(f"out: expected contiguous {query.dtype} {tuple(query.shape)}, 16-byte aligned")
        if out.untyped_storage().data_ptr() == query.untyped_storage().data_ptr():
            raise ValueError("out must not share the queries' memory")
    index = _lib.gpu_index(query, block_table, lens, query_start, out, *blocks)
    if not _lib.is_current(index):
        with torch.cuda.device(index):
            return attend_kv_blocks(query, blocks, block_table, lens, query_start, max_query=max_query, max_seq=max_seq,
                                    softmax_scale=softmax_scale, out=out)
    table_stride, inner = block_table.stride()
    if inner != 1 or table_stride < width:
        block_table = block_table.contiguous()
        table_stride = width
    query = _aligned(query)
    longest = width * c.block_size
    if max_query is None:
        max_query = 1 if query_start is None else tokens + 1  # more than there are: not known
    else:
        max_query = max(1, min(max_query, tokens))
    max_seq = max(1, longest if max_seq is None else min(max_seq, longest))
    scale = dim ** -0.5 if softmax_scale is None else float(softmax_scale)
    lib = _lib.load()
    call = lib.ctmi_kv_attend
    if out is None:
        if requests == 0:
            return query.new_zeros((tokens, heads, dim))
        out = query.new_empty((tokens, heads, dim))
        if query_start is not None:
            call = lib.ctmi_kv_attend_padded
    tmp_bytes = lib.ctmi_kv_attend_tmp_bytes(tokens, requests, heads, c.kv_heads, dim, max_query, max_seq)
    tmp = torch.empty(tmp_bytes, dtype=torch.uint8, device=out.device) if tmp_bytes else None
    token_stride, head_stride, _ = query.stride()
    _lib.check(call(
        query.data_ptr(), _lib.dtype_code(query.dtype), token_stride, head_stride, out.data_ptr(), tokens, heads,
        ctypes.byref(c), block_table.data_ptr(), table_stride, width, lens.data_ptr(), _lib.ptr(query_start), requests,
        scale, max_query, max_seq, _lib.ptr(tmp), tmp_bytes, _lib.stream_of_index(index)))
    return out


class BlockKVCache:
    """The block cache of a model: a pool per layer, one block table for all of them.

    A serving step is `plan(new_tokens, total)`, then for each layer `update(layer, key,
    value)` and `attend(layer, query)`.  Everything stays on the GPU: nothing here waits for
    it except `check()`.  A step that does not fit changes nothing: `update` then writes
    nothing and `attend` gives zeros, or leaves `out` as it is.  `plan` replaces the cache's
    tensors; a captured graph calls the functions on buffers of its own."""

    def __init__(self, layers: int, num_blocks: int, max_requests: int, max_blocks_per_request: int,
                 kv_heads: int, head_dim: int, block_size: int = 64,
                 dtype: torch.dtype = torch.float8_e4m3fn, device="cuda"):
        self.block_size = block_size
        self.layers: List[KVBlocks] = [KVBlocks.allocate(num_blocks, kv_heads, head_dim, block_size, dtype, device)
                                       for _ in range(layers)]
        self.seq_lens = torch.zeros(max_requests, dtype=torch.int32, device=device)
        self.block_table = torch.full((max_requests, max_blocks_per_request), -1, dtype=torch.int32, device=device)
        # popped from the end: block 0 is the first to be used
        self.free_blocks = torch.arange(num_blocks - 1, -1, -1, dtype=torch.int32, device=device)
        self.num_free = torch.full((1,), num_blocks, dtype=torch.int32, device=device)
        self._step: Optional[KVPlan] = None
        self._longest: Optional[int] = None
        self._calibrated = set()  # layers whose scales do not follow their values

    def set_scales(self, layer: int, key_scale: Tensor, value_scale: Tensor) -> None:
        """scales from calibration for all blocks of a layer: one, or one per kv head, as an
        attention module holds them in `k_scale` / `v_scale` under a symmetric kv_cache_scheme of
        8 bits.  `update` then keeps them and saturates.  For an empty cache."""
        for scale, pool in zip((key_scale, value_scale), self.layers[layer][2:]):
            if scale.numel() not in (1, pool.shape[1]):
                raise ValueError(f"expected one scale or {pool.shape[1]}, got {tuple(scale.shape)}")
            pool.copy_(scale.detach().reshape(1, -1).expand_as(pool))
        self._calibrated.add(layer)

    def plan(self, new_tokens: Tensor, total_tokens: int, max_query: Optional[int] = None) -> KVPlan:
        """take the blocks for this step's tokens; `new_tokens` int32 [max_requests], -1 ends a
        request (plan_kv_blocks)"""
        step = plan_kv_blocks(self.seq_lens, new_tokens, self.block_table, self.free_blocks, self.num_free,
                              block_size=self.block_size, total_tokens=total_tokens)
        self.seq_lens, self.block_table = step.seq_lens, step.block_table
        self.free_blocks, self.num_free = step.free_blocks, step.num_free
        self._step, self._longest = step, max_query
        return step

    def check(self) -> None:
        """wait for the last plan and raise if it did not fit"""
        status = int(self._current().status)
        if status > 0:
            raise RuntimeError(f"the pool is short of {status} blocks")
        if status:
            raise ValueError({-1: "a request is longer than its row of the block table",
                              -2: "the step has more tokens than total_tokens",
                              -3: "the free list is not in order"}[status])

    def update(self, layer: int, key: Tensor, value: Tensor) -> None:
        """store this step's keys and values of one layer, [tokens, kv_heads, head_dim]"""
        append_kv_blocks(key, value, self.layers[layer], self._current().slots, dynamic=layer not in self._calibrated)

    def attend(self, layer: int, query: Tensor, softmax_scale: Optional[float] = None,
               max_seq: Optional[int] = None, out: Optional[Tensor] = None) -> Tensor:
        """attention of this step's queries, [tokens, q_heads, head_dim], over one layer"""
        step = self._current()
        return attend_kv_blocks(query, self.layers[layer], step.block_table, step.seq_lens, step.query_start,
                                max_query=self._longest, max_seq=max_seq, softmax_scale=softmax_scale, out=out)

    def _current(self) -> KVPlan:
        if self._step is None:
            raise ValueError("plan() comes before update(), attend() and check()")
        return self._step
