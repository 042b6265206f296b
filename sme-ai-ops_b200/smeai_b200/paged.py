"""The paged key/value cache over torch device memory (thin wrappers of smeai_paged.h).

A step of a serving loop, per layer where it says so:

    plan.build(cached_len, new_len, free_pages, n_used)             # once a step
    q = append(kv, k, v, plan.slots, q=q, positions=plan.positions, rope=rope)      # per layer
    context = attention(q, kv, plan.block_table, plan.q_start, plan.kv_len, max_new)

All calls queue work on the current stream and neither wait nor keep anything;
with the outputs given, all of them can be captured in a CUDA graph.  A length,
slot, position or page outside its buffer is reported by take_device_error().
"""
from __future__ import annotations

import ctypes

import torch

from . import KV_BF16, KV_F16, KVCache, check, lib
from .q2k import call

_TYPES = {torch.float16: KV_F16, torch.bfloat16: KV_BF16}


def rope_table(n_positions: int, head_dim: int, base: float = 10000.0, device=None) -> torch.Tensor:
    """[n_positions, head_dim] fp32: the cosines of a position's head_dim/2
    angles, then their sines; angles formed in 64 bits."""
    i = torch.arange(0, head_dim, 2, dtype=torch.float64, device=device)
    angle = torch.arange(n_positions, dtype=torch.float64, device=device)[:, None] * base ** (-i / head_dim)
    return torch.cat([angle.cos(), angle.sin()], 1).float().contiguous()


class PagedKV:
    """Pages of keys and values: k, v [n_pages, n_kv_heads, page_size, head_dim],
    fp16 or bf16 (a cache stored page by token by head is passed as its
    transposed view)."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor):
        assert k.dim() == 4 and k.shape == v.shape and k.stride() == v.stride(), "k and v of one shape and layout"
        assert k.is_cuda and k.device == v.device and k.dtype == v.dtype and k.dtype in _TYPES
        assert k.stride(3) == 1 or k.shape[3] == 1, "a head's elements lie next to one another"
        self.k, self.v = k, v
        self.device, self.dtype = k.device, k.dtype
        self.n_pages, self.n_kv_heads, self.page_size, self.head_dim = k.shape
        # the stride of a dimension of one element says nothing
        strides = [st if n > 1 else self.head_dim for n, st in zip(k.shape, k.stride()[:3])]
        self.struct = KVCache(k.data_ptr(), v.data_ptr(), _TYPES[k.dtype], self.page_size, self.n_kv_heads, self.head_dim,
                              self.n_pages, strides[0], strides[1], strides[2])
        self.ref = ctypes.byref(self.struct)
        self._workspace = {}         # bytes of attention()'s workspace, by sizes; few of them, a server's sizes never end

    @classmethod
    def empty(cls, n_pages: int, n_kv_heads: int, page_size: int, head_dim: int, dtype=torch.float16, device=None) -> "PagedKV":
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else device
        shape = (n_pages, n_kv_heads, page_size, head_dim)
        return cls(torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device))


class PagedPlan:
    """Buffers of a step's bookkeeping over a block table [n_req, max_blocks]
    (int32, kept by the caller from step to step): q_start [n_req + 1], kv_len
    [n_req], slots (int64) and positions [n_tokens]."""

    def __init__(self, block_table: torch.Tensor, page_size: int, n_tokens: int):
        assert block_table.dim() == 2 and block_table.dtype == torch.int32 and block_table.is_cuda
        self.block_table, self.page_size, self.n_tokens = block_table, page_size, n_tokens
        self.n_req, self.max_blocks = block_table.shape
        ld_table = _table_stride(block_table)
        dev = block_table.device
        self.device = dev
        self.q_start = torch.zeros(self.n_req + 1, dtype=torch.int32, device=dev)
        self.kv_len = torch.zeros(self.n_req, dtype=torch.int32, device=dev)
        self.slots = torch.full((n_tokens,), -1, dtype=torch.int64, device=dev)
        self.positions = torch.zeros(n_tokens, dtype=torch.int32, device=dev)
        self._out = (block_table.data_ptr(), ld_table, self.max_blocks,
                     self.q_start.data_ptr(), self.kv_len.data_ptr(), self.slots.data_ptr(), self.positions.data_ptr(),
                     n_tokens)

    def build(self, cached_len: torch.Tensor, new_len: torch.Tensor, free_pages: torch.Tensor, n_used: torch.Tensor,
              used_out: torch.Tensor | None = None) -> "PagedPlan":
        """Fills the buffers for requests that hold cached_len tokens and bring
        new_len more; new pages come from free_pages, from index n_used[0] on,
        which advances (in place, or into used_out).  cached_len may be this
        plan's own kv_len (a refused request's length is then gone)."""
        if used_out is None:
            used_out = n_used
        i32, dev, n = torch.int32, self.device, self.n_req
        assert cached_len.dtype == new_len.dtype == free_pages.dtype == n_used.dtype == used_out.dtype == i32
        assert cached_len.device == new_len.device == free_pages.device == n_used.device == used_out.device == dev
        assert cached_len.numel() == new_len.numel() == n and n_used.numel() == used_out.numel() == 1
        assert cached_len.is_contiguous() and new_len.is_contiguous() and free_pages.is_contiguous()
        call(dev, lib().smeai_paged_plan, "paged_plan", cached_len.data_ptr(), new_len.data_ptr(), n, self.page_size,
             free_pages.data_ptr(), free_pages.numel(), n_used.data_ptr(), used_out.data_ptr(), *self._out)
        return self


def _table_stride(table: torch.Tensor) -> int:
    """Entries between a block table's rows."""
    n, blocks = table.shape
    ld, one = table.stride()
    assert (one == 1 or blocks <= 1) and (ld >= blocks or n <= 1), "a table's rows are contiguous and apart"
    return ld if n > 1 else blocks


def _rows(x: torch.Tensor, n: int, heads: int, dim: int, dtype, dev) -> int:
    """The row stride of x [n, heads, dim], a token's heads next to one another."""
    assert x.shape == (n, heads, dim) and x.dtype == dtype and x.device == dev
    st = x.stride()
    assert (st[2] == 1 or dim == 1) and (st[1] == dim or heads == 1), "a token's heads lie next to one another"
    return st[0] if n > 1 else heads * dim        # a single row's stride says nothing


def append(kv: PagedKV, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, q: torch.Tensor | None = None,
           q_out: torch.Tensor | None = None, positions: torch.Tensor | None = None, rope: torch.Tensor | None = None,
           halves: bool = False) -> torch.Tensor | None:
    """Writes k, v (fp32 [n_tokens, n_kv_heads, head_dim], rows of any stride)
    into the tokens' slots (int64, -1: left out), rotated by rope (rope_table;
    element pairs, or halves) at positions (int32) when given, and returns q
    (fp32 [n_tokens, n_heads, head_dim]) rotated the same way, in the cache's type."""
    dev, dim, n = kv.device, kv.head_dim, k.shape[0]
    ld_k, ld_v = _rows(k, n, kv.n_kv_heads, dim, torch.float32, dev), _rows(v, n, kv.n_kv_heads, dim, torch.float32, dev)
    assert slots.dtype == torch.int64 and slots.device == dev and slots.shape == (n,) and slots.is_contiguous()
    heads = ld_q = ld_qo = n_rope = 0
    q_ptr = qo_ptr = pos_ptr = rope_ptr = None
    if q is not None:
        heads = q.shape[1]
        if q_out is None:
            q_out = torch.empty((n, heads, dim), dtype=kv.dtype, device=dev)
        ld_q, ld_qo = _rows(q, n, heads, dim, torch.float32, dev), _rows(q_out, n, heads, dim, kv.dtype, dev)
        q_ptr, qo_ptr = q.data_ptr(), q_out.data_ptr()
    else:
        assert q_out is None
    if rope is not None:
        n_rope, pos_ptr, rope_ptr = rope.shape[0], positions.data_ptr(), rope.data_ptr()
        assert rope.dtype == torch.float32 and rope.device == dev and rope.shape == (n_rope, dim) and rope.is_contiguous()
        assert positions.dtype == torch.int32 and positions.device == dev and positions.shape == (n,) and positions.is_contiguous()
    if n:
        call(dev, lib().smeai_paged_append, "paged_append", kv.ref, k.data_ptr(), ld_k, v.data_ptr(), ld_v, q_ptr, ld_q, heads,
             qo_ptr, ld_qo, n, slots.data_ptr(), pos_ptr, rope_ptr, n_rope, halves)
    return q_out


def attention(q: torch.Tensor, kv: PagedKV, block_table: torch.Tensor, q_start: torch.Tensor, kv_len: torch.Tensor,
              max_new: int, scale: float | None = None, causal: bool = True, out: torch.Tensor | None = None,
              workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Context rows of q [n_tokens, n_heads, head_dim] (the cache's type; rows
    of any stride) over the requests' pages; scale defaults to head_dim ** -0.5.
    Rows outside q_start[0] .. q_start[-1] are not written (without `out` they
    hold anything).  max_new: the largest number of new tokens of a request.
    workspace: uint8 tensor of attention_workspace() bytes, one per call in
    flight; by default it is allocated for this call."""
    dev, dim = kv.device, kv.head_dim
    n, heads = q.shape[0], q.shape[1]
    ld_q = _rows(q, n, heads, dim, kv.dtype, dev)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        ld_out = heads * dim
    else:
        ld_out = _rows(out, n, heads, dim, kv.dtype, dev)
    n_req, max_blocks = block_table.shape
    ld_table = _table_stride(block_table)
    assert block_table.dtype == q_start.dtype == kv_len.dtype == torch.int32
    assert block_table.device == q_start.device == kv_len.device == dev
    assert q_start.shape == (n_req + 1,) and kv_len.shape == (n_req,) and q_start.is_contiguous() and kv_len.is_contiguous()
    if n == 0:
        return out
    ws_ptr, ws_bytes = None, attention_workspace(kv, heads, n, n_req, max_blocks, max_new)
    if workspace is not None:
        assert workspace.dtype == torch.uint8 and workspace.device == dev and workspace.is_contiguous()
        ws_ptr, ws_bytes = workspace.data_ptr(), workspace.numel()
    elif ws_bytes:
        workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
        ws_ptr = workspace.data_ptr()
    call(dev, lib().smeai_paged_attention, "paged_attention", kv.ref, q.data_ptr(), ld_q, heads, n, q_start.data_ptr(),
         kv_len.data_ptr(), n_req, block_table.data_ptr(), ld_table, max_blocks, max_new,
         dim ** -0.5 if scale is None else scale, causal, out.data_ptr(), ld_out, ws_ptr, ws_bytes)
    return out


def attention_workspace(kv: PagedKV, n_heads: int, n_tokens: int, n_req: int, max_blocks: int, max_new: int) -> int:
    """Bytes of attention()'s workspace for a call of these sizes; 0 when the
    table's rows are too short for a request's keys ever to be split."""
    key = (n_heads, n_tokens, n_req, max_blocks, max_new)
    n = kv._workspace.get(key)
    if n is None:
        if len(kv._workspace) >= 64:
            kv._workspace.clear()
        with torch.cuda.device(kv.device):
            n = kv._workspace[key] = lib().smeai_paged_attention_workspace(kv.ref, *key)
    return n


__all__ = ["PagedKV", "PagedPlan", "append", "attention", "attention_workspace", "rope_table"]
