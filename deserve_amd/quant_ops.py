"""Operators of a KV cache held in 8 bits, implemented by the gfx950 kernels behind the C ABI.  No counterpart in the
reference, whose pages have the model's type.

A page of a layer is a record of bytes (PageRecord): the codes of K, then of V, in e4m3, by head and token, and one float32 scale, a
power of two, for each half and head.  A value is code * scale of its block, the tokens of one page and head.  A pool of such pages is
one of main_dtype torch.float8_e4m3fn (kvcache.paged.page_pool); offload, reload and slice swaps move its records as they are, half
the bytes that 16-bit pages are.  A step's work on a layer:

    wrapper.begin_forward(qo_indptr, kv_indptr, kv_indices, kv_last_page_len, num_qo_heads, num_kv_heads, head_dim, page_size,
                          max_qo_len=)
    q = rope_append_quantized(q, k, v, qo_indptr, pages, kv_indices, kv_indptr, kv_last_page_len, page_size, angles)
    out = wrapper.forward(q, pages)

q, k, v and out have the model's type (bfloat16, float16 or float32); a cache is appended to and read in one type.  Steps of
drafted tokens run as in draft_ops, with move_accepted_quantized_rows behind them.  Lengths and tables stay on the device: nothing is
planned on the host or read back, so the calls can be captured into a graph and replayed with other lengths.  Work
is enqueued on the current stream of the tensors' device.
"""
from __future__ import annotations

import ctypes
import functools
import math
from dataclasses import dataclass
from typing import List, Optional

import torch

from deserve_amd import _lib
from deserve_amd.draft_ops import MAX_TREE_ROWS, _call, _check_vector, _on_device, _token_rows

CODE_DTYPE = torch.float8_e4m3fn
INT32_MAX = 2 ** 31 - 1


@dataclass(frozen=True)
class PageRecord:
    """How a page of a layer lies in memory."""
    page_size: int
    n_kv_heads: int
    head_dim: int

    def __post_init__(self) -> None:
        if self.page_size <= 0 or self.n_kv_heads <= 0 or self.head_dim <= 0 or self.head_dim % 8 or self.head_dim > 256:
            raise ValueError(f"pages of {self.page_size} tokens, {self.n_kv_heads} heads of {self.head_dim} dims: sizes must "
                             "be positive, head_dim a multiple of 8 up to 256")

    @property
    def code_bytes(self) -> int:
        return 2 * self.n_kv_heads * self.page_size * self.head_dim

    @property
    def page_bytes(self) -> int:
        return -(-(self.code_bytes + 8 * self.n_kv_heads) // 128) * 128

    def codes(self, pages: torch.Tensor) -> torch.Tensor:
        """A view of (..., page_bytes) uint8 records: (..., 2, Hkv, P, D) codes."""
        return pages[..., : self.code_bytes].view(CODE_DTYPE).unflatten(-1, (2, self.n_kv_heads, self.page_size, self.head_dim))

    def scales(self, pages: torch.Tensor) -> torch.Tensor:
        """A view of (..., page_bytes) uint8 records: (..., 2, Hkv) float32 scales."""
        end = self.code_bytes + 8 * self.n_kv_heads
        return pages[..., self.code_bytes: end].view(torch.float32).unflatten(-1, (2, self.n_kv_heads))

    def values(self, pages: torch.Tensor, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """(..., 2, P, Hkv, D) of dtype: what the records stand for, in the order of pages of that type."""
        x = self.codes(pages).float() * self.scales(pages)[..., None, None]
        return x.transpose(-3, -2).to(dtype)


@functools.lru_cache(maxsize=256)
def _page_bytes(page_size: int, n_kv_heads: int, head_dim: int) -> int:
    return PageRecord(page_size, n_kv_heads, head_dim).page_bytes


def _check_records(name: str, pages: torch.Tensor, page_bytes: int, dims: int) -> None:
    shape = pages.shape
    if len(shape) == dims and pages.dtype is torch.uint8 and shape[-1] == page_bytes and pages.data_ptr() % 16 == 0 and (
            pages.is_contiguous() or (dims == 3 and (shape[0] == 0 or pages[0].is_contiguous()) and pages.stride(0) % 16 == 0)):
        return
    if pages.dtype is torch.uint8 and len(shape) == dims and shape[-1] == page_bytes and pages.data_ptr() % 16:
        raise ValueError(f"{name} must be 16-byte aligned")
    what = "(num_pages, " if dims == 2 else "(L, num_pages, "
    raise ValueError(f"{name} must be a contiguous {what}{page_bytes}) uint8 tensor, got {tuple(shape)} of {pages.dtype}")


def _check_csr(qo_indptr: torch.Tensor, kv_indices: torch.Tensor, kv_indptr: torch.Tensor, kv_last_page_len: torch.Tensor) -> int:
    batch = qo_indptr.numel() - 1
    i32 = torch.int32
    if qo_indptr.dtype is i32 and kv_indptr.dtype is i32 and kv_indices.dtype is i32 and kv_last_page_len.dtype is i32 and \
            qo_indptr.dim() == kv_indptr.dim() == kv_indices.dim() == kv_last_page_len.dim() == 1 and \
            qo_indptr.is_contiguous() and kv_indptr.is_contiguous() and kv_indices.is_contiguous() and \
            kv_last_page_len.is_contiguous() and 0 <= batch <= kv_last_page_len.numel() and kv_indptr.numel() == batch + 1:
        return batch
    _check_vector("qo_indptr", qo_indptr, i32, 1)
    _check_vector("kv_indptr", kv_indptr, i32, batch + 1)
    _check_vector("kv_indices", kv_indices, i32, 0)
    _check_vector("kv_last_page_len", kv_last_page_len, i32, batch)
    raise ValueError("qo_indptr and kv_indptr disagree about the batch")


def rope_append_quantized(q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor, qo_indptr: torch.Tensor,
                          pages: torch.Tensor, kv_indices: torch.Tensor, kv_indptr: torch.Tensor,
                          kv_last_page_len: torch.Tensor, page_size: int, rope_table: Optional[torch.Tensor] = None, *,
                          out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """In place on ``pages`` (num_pages, page_bytes) uint8, one layer: the n_b new tokens of request b become the last n_b of its
    kv_len_b = (npages_b - 1) * P + last_b tokens, k rotated; returns the rotated q.  q, k, v (tokens, heads, D) may be parts of one
    projection's output, and rope_table and out are as in draft_ops.rope_append_slots; without rope_table q (may be None) comes back as it is.
    A block's scale is the least power of two that its largest value takes to 448 or less, never less than that of the tokens it
    holds already, whose codes are rounded anew where it grows.  A token with a value that is no finite number makes no number of the rows
    that see it, and nothing else.  A request whose arrays contradict themselves, or a page that the pool does not have,
    takes no rows.  No page takes rows of two requests, or of two entries of a table."""
    if k.dim() != 3:
        raise ValueError(f"k must be (tokens, heads, D), got {tuple(k.shape)}")
    nnz, hkv, dim = k.shape
    dtype = k.dtype
    _check_records("pages", pages, _page_bytes(page_size, hkv, dim), 2)
    code = _lib.dtype_code(dtype)
    k, k_stride = _token_rows("k", k, dtype, hkv, dim, nnz)
    v, v_stride = _token_rows("v", v, dtype, hkv, dim, nnz)
    batch = _check_csr(qo_indptr, kv_indices, kv_indptr, kv_last_page_len)
    result, q_stride, heads = q, 0, hkv
    if rope_table is not None:
        if q is None:
            raise ValueError("rope_table rotates q and k: q is missing")
        q, q_stride = _token_rows("q", q, dtype, None, dim, nnz)
        heads = q.shape[1]
        table = rope_table.shape
        if rope_table.dtype is not torch.float32 or len(table) != 2 or table[1] != dim or table[0] < nnz or \
                not rope_table.is_contiguous() or rope_table.data_ptr() % 16:
            raise ValueError(f"rope_table must be a contiguous, 16-byte aligned float32 ({nnz}, {dim}) tensor")
        if out is None:
            result = torch.empty_like(q, memory_format=torch.contiguous_format)
        elif out.shape != q.shape or out.dtype is not dtype or not out.is_contiguous() or out.data_ptr() % 16:
            raise ValueError("out must be contiguous, 16-byte aligned and of q's shape and dtype")
        else:
            result = out
    elif out is not None:
        raise ValueError("out is for the rotated q: rope_table is missing")
    rotated = rope_table is not None
    index = _on_device(pages, k, v, qo_indptr, kv_indices, kv_indptr, kv_last_page_len, rope_table, q if rotated else None, out)
    num_pages, at = pages.shape[0], pages.data_ptr()
    if nnz == 0 or (not rotated and (batch == 0 or num_pages == 0)):
        return result
    if batch == 0 or num_pages == 0:
        # no row is kept and q is rotated all the same: one request that has none, over a table without entries
        qo_indptr = kv_indptr = kv_last_page_len = k.new_zeros((2,), dtype=torch.int32)
        kv_indices, batch, num_pages, at = kv_indptr[:0], 1, 1, result.data_ptr()
    rows = _lib.QuantRows(qo_indptr.data_ptr(), kv_indices.data_ptr(), kv_indptr.data_ptr(), kv_last_page_len.data_ptr(),
                          kv_indices.numel(), batch, nnz, num_pages, page_size, hkv, dim)
    _call("rope_append_quantized", index, _lib.lib().dskv_rope_append_quant, ctypes.byref(rows),
          result.data_ptr() if rotated else None, at, q.data_ptr() if rotated else None, k.data_ptr(), v.data_ptr(),
          q_stride, k_stride, v_stride, _lib.ptr(rope_table), heads, code)
    return result


class BatchQuantizedWithPagedKVCacheWrapper:
    """Attention of a step's rows over pages of 8-bit K/V, with the begin_forward / forward / end_forward protocol of paged_ops:
    one row per request (decode), chains or trees of drafted tokens, chunks of prompts, or all of them together.  begin_forward plans
    nothing and reads nothing back: the kernels take lengths and tables from the device, so a captured step can be replayed with others.
    workspace_buffer: scratch of a forward while it runs; forwards that may run at the same time, on two streams, need a wrapper over
    a workspace of its own each (two over one are both wrong, and so may later ones be until reset).  Making one waits for the device's current stream, once, and is not for a capture."""

    def __init__(self, workspace_buffer: torch.Tensor, kv_layout: str = "HND") -> None:
        if kv_layout != "HND":
            raise ValueError("8-bit pages hold their tokens by head: only the HND layout is implemented")
        self._workspace = workspace_buffer
        # what the parts of a request count themselves in with: zero between launches, and kept for good, also where more heads
        # ask for more words (captured launches hold their address); one list for all copies (another), the longest behind
        self._all_counters: List[torch.Tensor] = []
        self._counters = self._zeros(_lib.lib().dskv_quant_attn_counters(1))
        self._step: Optional[_lib.QuantStep] = None
        self._held: tuple = ()

    def _zeros(self, n: int) -> torch.Tensor:
        device = self._workspace.device
        if device.type != "cuda":
            return torch.zeros((n,), dtype=torch.int32)
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a wrapper for 8-bit pages is made, or first given so many kv heads, outside of a capture")
        with torch.cuda.device(device):
            zeros = torch.zeros((n,), dtype=torch.int32, device=device)
            torch.cuda.current_stream().synchronize()        # whatever stream uses them first
        self._all_counters.append(zeros)
        return zeros

    def another(self) -> "BatchQuantizedWithPagedKVCacheWrapper":
        """For a step planned beside this wrapper's, over the same workspace; costs nothing."""
        other = object.__new__(type(self))
        other.__dict__.update(self.__dict__, _step=None, _held=())
        return other

    def reset(self) -> None:
        """Sets back what parts count themselves in with, of this wrapper and its copies: for a program in which two forwards have run at
        the same time over one workspace, which leaves it off zero.  On the current stream, behind all of their forwards."""
        for counters in self._all_counters:
            counters.zero_()

    def begin_forward(self, qo_indptr: torch.Tensor, paged_kv_indptr: torch.Tensor, paged_kv_indices: torch.Tensor,
                      paged_kv_last_page_len: torch.Tensor, num_qo_heads: int, num_kv_heads: int, head_dim: int,
                      page_size: int, *, max_qo_len: int, min_qo_len: int = 0, masks: Optional[torch.Tensor] = None) -> None:
        """The index tensors (int32) are read by every forward, on the device: they stay as they are until the last one has run.
        max_qo_len: no request has more rows (of one that has, the further ones are left out).  min_qo_len: none has fewer, a
        hint that saves a launch where all have many; 0 is always right.
        masks (tokens) int64, bit j: the row sees new row j of its request, at most MAX_TREE_ROWS rows a request;
        None: it sees the rows up to itself."""
        batch = _check_csr(qo_indptr, paged_kv_indices, paged_kv_indptr, paged_kv_last_page_len)
        page_bytes = _page_bytes(page_size, num_kv_heads, head_dim)
        if masks is not None:
            _check_vector("masks", masks, torch.int64, 0)
            if max_qo_len > MAX_TREE_ROWS:
                raise ValueError(f"masks hold {MAX_TREE_ROWS} rows a request, max_qo_len is {max_qo_len}")
        if num_qo_heads <= 0 or num_qo_heads % num_kv_heads:
            raise ValueError(f"num_qo_heads {num_qo_heads} must be a multiple of num_kv_heads {num_kv_heads}")
        if max_qo_len < 0 or min_qo_len < 0:
            raise ValueError("max_qo_len and min_qo_len must not be negative")
        _on_device(qo_indptr, paged_kv_indptr, paged_kv_indices, paged_kv_last_page_len, masks, self._workspace)
        if num_kv_heads > 512 and self._counters.numel() < (need := _lib.lib().dskv_quant_attn_counters(num_kv_heads)):
            made = self._all_counters[-1]                # perhaps by a copy
            self._counters = made if made.numel() >= need else self._zeros(need)
        counters = self._counters
        self._held = (qo_indptr, paged_kv_indptr, paged_kv_indices, paged_kv_last_page_len, masks, page_bytes, counters)
        workspace = self._workspace
        self._step = _lib.QuantStep((
            qo_indptr.data_ptr(), paged_kv_indptr.data_ptr(), paged_kv_indices.data_ptr(),
            paged_kv_last_page_len.data_ptr(), None if masks is None else masks.data_ptr(), workspace.data_ptr(),
            workspace.numel() * workspace.element_size(), paged_kv_indices.numel(), batch, 0, min(max_qo_len, INT32_MAX),
            num_qo_heads, num_kv_heads, head_dim, page_size), counters.data_ptr(), counters.numel(), min(min_qo_len, INT32_MAX))

    def forward(self, q: torch.Tensor, pages: torch.Tensor, sm_scale: Optional[float] = None, *,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """q (tokens, Hq, D), one row for every row of the step; rows behind the last request's are left out of the
        result (as they were in out).  K and V of the new rows are in the pages (num_pages, page_bytes) uint8.  A row that sees
        nothing gets zeros.  256 times a request's tokens times the largest magnitude in V is under 2 ** 128 (1e27 for any length).
        sm_scale: positive; None: D ** -0.5.  out: optional result tensor (contiguous, q's shape and dtype)."""
        if self._step is None:
            raise RuntimeError("forward over 8-bit pages called before begin_forward")
        s = self._step.step
        _check_records("pages", pages, self._held[5], 2)
        dtype = q.dtype
        code = _lib.dtype_code(dtype)
        q, q_stride = _token_rows("q", q, dtype, s.n_qo_heads, s.head_dim, None)
        nnz, masks = q.shape[0], self._held[4]
        if masks is not None and masks.numel() < nnz:
            raise ValueError(f"masks hold {masks.numel()} rows, q has {nnz}")
        if sm_scale is not None and not sm_scale > 0:
            raise ValueError(f"sm_scale must be positive, not {sm_scale}")
        fresh = out is None
        if fresh:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        elif out.shape != q.shape or out.dtype is not dtype or not out.is_contiguous() or out.data_ptr() % 16:
            raise ValueError("out must be contiguous, 16-byte aligned and of q's shape and dtype")
        index = _on_device(q, pages, None if fresh else out, self._held[0])
        if pages.shape[0] == 0:
            raise ValueError("the pool has no pages")
        step = _lib.QuantStep.from_buffer_copy(self._step)      # calls from several threads do not share it
        inner = step.step
        inner.nnz, inner.num_pages, inner.dtype = nnz, pages.shape[0], code
        inner.sm_scale = 1.0 / math.sqrt(s.head_dim) if sm_scale is None else sm_scale
        _call("forward over 8-bit pages", index, _lib.lib().dskv_quant_attn, ctypes.byref(step), out.data_ptr(), q.data_ptr(),
              q_stride, pages.data_ptr())
        return out

    def end_forward(self) -> None:
        self._step, self._held = None, ()


def move_accepted_quantized_rows(pages: torch.Tensor, qo_indptr: torch.Tensor, kv_indices: torch.Tensor, kv_indptr: torch.Tensor,
                                 kv_last_page_len: torch.Tensor, path: torch.Tensor, counts: torch.Tensor, page_size: int,
                                 n_kv_heads: int, head_dim: int) -> None:
    """In place on ``pages`` (L, num_pages, page_bytes) uint8, layers possibly apart: K/V of the rows of every request's walk
    (draft_ops.verify_drafts) to where its sequence goes on, row j of the walk from the request's new row path[j] to its new row j, in all
    layers; the tables are those of the step that was verified.  The scale of a block that rows move into grows where they need it.
    Accepted chains are there already."""
    _check_records("pages", pages, _page_bytes(page_size, n_kv_heads, head_dim), 3)
    batch = _check_csr(qo_indptr, kv_indices, kv_indptr, kv_last_page_len)
    _check_vector("path", path, torch.int32, 0)
    _check_vector("counts", counts, torch.int32, batch)
    index = _on_device(pages, qo_indptr, kv_indices, kv_indptr, kv_last_page_len, path, counts)
    layers, num_pages, _ = pages.shape
    if layers == 0 or num_pages == 0 or path.numel() == 0:
        return
    rows = _lib.QuantRows(qo_indptr.data_ptr(), kv_indices.data_ptr(), kv_indptr.data_ptr(), kv_last_page_len.data_ptr(),
                          kv_indices.numel(), batch, path.numel(), num_pages, page_size, n_kv_heads, head_dim)
    _call("move_accepted_quantized_rows", index, _lib.lib().dskv_move_quant_rows, ctypes.byref(rows), pages.data_ptr(),
          pages.stride(0), layers, path.data_ptr(), counts.data_ptr())
