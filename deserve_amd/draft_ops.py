"""Operators of a step that verifies drafted tokens over the paged cache, implemented by the gfx950 kernels behind
the C ABI.  No counterpart in the reference, whose decode step gives every request one token for one pass
over its context.

Request b brings n_b rows to such a step.  Row 0 is the last token it was given, whose K/V the cache does not hold
yet; the others are drafted tokens that form a chain or a tree behind it, a row's parent having a smaller index:

    tables = build_step_tables(page_tables, kv_lens, qo_lens, page_size, max_tokens=, max_pages=, parents=)
    wrapper.begin_forward(*tables.csr, num_qo_heads, num_kv_heads, head_dim, page_size, max_qo_len=, masks=tables.masks)
    angles = tables.rope_table(head_dim, theta)                                # for all layers
    per layer:  q = rope_append_slots(q, k, v, tables.slots, pages, angles);  out = wrapper.forward(q, pages)
    verdict = verify_drafts(target_probs, tokens, uniforms, tables.qo_indptr, parents=)
    move_accepted_rows(pool.pages, tables.slots, tables.qo_indptr, verdict.path, verdict.counts)
    kv_lens += verdict.counts

A stage runs them through execution.exec.BatchVerify.  Lengths, tables and verdicts stay on the device: nothing is planned on the host or read back, so the calls can be captured into
a graph and replayed with other lengths.  Work is enqueued on the current stream of the tensors' device.
"""
from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from deserve_amd import _lib

MAX_TREE_ROWS = _lib.MAX_TREE_ROWS


# (the functions behind torch.cuda.current_device() and current_stream(), whose own work costs a short step half of
# its host time)
_current_device = torch._C._cuda_getDevice
_raw_stream = torch._C._cuda_getCurrentRawStream


def _on_device(first: torch.Tensor, *others: Optional[torch.Tensor]) -> int:
    """Index of the device that all of them are on: the kernels read device memory only, and one device's."""
    index = first.get_device()
    if index < 0 or not first.is_cuda:
        raise ValueError(f"tensors must be on the GPU, got one on {first.device}")
    for t in others:
        if t is not None and t.get_device() != index:
            raise ValueError(f"tensors on different devices: {first.device} and {t.device}")
    return index


def _call(what: str, index: int, fn, *args) -> None:
    """Enqueues on the current stream of device `index`, whichever device is the current one."""
    if index == _current_device():
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc:
        _lib.check(rc, what)


def _check_vector(name: str, t: torch.Tensor, dtype: torch.dtype, least: int) -> None:
    if t.dtype is not dtype or t.dim() != 1 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous one-dimensional {dtype} tensor")
    if t.numel() < least:
        raise ValueError(f"{name} holds {t.numel()} entries, {least} are needed")


@dataclass
class StepTables:
    """What build_step_tables writes, all on the device."""
    qo_indptr: torch.Tensor            # (batch + 1) int32
    kv_page_indptr: torch.Tensor       # (batch + 1) int32
    kv_page_indices: torch.Tensor      # (max_pages) int32; behind kv_page_indptr[batch] as it was
    kv_last_page_lens: torch.Tensor    # (batch) int32
    positions: torch.Tensor            # (max_tokens) int32; 0 behind the last row
    slots: torch.Tensor                # (max_tokens) int64: page id * page_size + place in the page; -1 behind the last row
    masks: Optional[torch.Tensor]      # (max_tokens) int64, bit j: is row j or descends from it; None without parents

    @classmethod
    def empty(cls, batch: int, max_tokens: int, max_pages: int, device: torch.device, tree: bool) -> "StepTables":
        # one allocation; the 64-bit arrays first
        words = [2 * max_tokens, 2 * max_tokens if tree else 0, batch + 1, batch + 1, max_pages, batch, max_tokens]
        slots, masks, qo_indptr, kv_indptr, indices, last, positions = \
            torch.empty((sum(words),), dtype=torch.int32, device=device).split_with_sizes(words)
        return cls(qo_indptr, kv_indptr, indices, last, positions, slots.view(torch.int64),
                   masks.view(torch.int64) if tree else None)

    @property
    def csr(self) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
        """In the order in which the wrappers' begin_forward takes them."""
        return self.qo_indptr, self.kv_page_indptr, self.kv_page_indices, self.kv_last_page_lens

    def rope_table(self, head_dim: int, rope_theta: float = 1e4) -> torch.Tensor:
        """(max_tokens, head_dim) floats, row t = cosines | sines of the angles of row t's position: what
        rope_append_slots rotates by, the same for every layer of the step."""
        table = torch.empty((self.positions.shape[0], head_dim), dtype=torch.float32, device=self.positions.device)
        _call("rope table", _on_device(table), _lib.lib().dskv_rope_table, table.data_ptr(), self.positions.data_ptr(),
              table.shape[0], head_dim, float(rope_theta))
        return table


def build_step_tables(page_tables: torch.Tensor, kv_lens: torch.Tensor, qo_lens: torch.Tensor, page_size: int, *,
                      max_tokens: int, max_pages: int, rows: Optional[torch.Tensor] = None,
                      parents: Optional[torch.Tensor] = None, out: Optional[StepTables] = None) -> StepTables:
    """Block tables (CSR), slot map, positions and tree masks of a step, built on the GPU from lengths that live there.

    page_tables (R, W) int32, rows of page ids (a row may be part of a longer one); request b owns row rows[b]
    (None: row b).  kv_lens, qo_lens (batch) int32: tokens cached before the step, new rows of the step.
    parents int32, ragged by the rows as they follow one another: index of a row's parent within its request
    (anything outside [0, own index): none), at most MAX_TREE_ROWS rows a request; None: rows follow one another.
    max_tokens, max_pages: sizes of the arrays by row and by page.
    A request that contradicts itself or its table (negative lengths, more tokens than its row of the table holds,
    no such row, too many rows for a tree) gets no rows and no pages; so does the first that does not
    fit max_tokens or max_pages, with all behind it: its entries of qo_indptr tell."""
    if page_tables.dtype is not torch.int32 or page_tables.dim() != 2 or \
            (page_tables.numel() > 0 and (page_tables.stride(1) != 1 and page_tables.shape[1] > 1)) or \
            (page_tables.shape[0] > 1 and page_tables.stride(0) < page_tables.shape[1]):
        raise ValueError("page_tables must be int32 (rows, width) with contiguous rows")
    _check_vector("kv_lens", kv_lens, torch.int32, 0)
    _check_vector("qo_lens", qo_lens, torch.int32, 0)
    batch = kv_lens.numel()
    if qo_lens.numel() != batch:
        raise ValueError(f"kv_lens and qo_lens disagree about the batch: {batch} and {qo_lens.numel()}")
    if rows is not None:
        _check_vector("rows", rows, torch.int32, batch)
    if parents is not None:
        _check_vector("parents", parents, torch.int32, 0)
    if page_size <= 0 or max_tokens < 0 or max_pages < 0:
        raise ValueError("page_size must be positive, max_tokens and max_pages not negative")
    if out is None:
        index = _on_device(kv_lens, page_tables, qo_lens, rows, parents)
        out = StepTables.empty(batch, max_tokens, max_pages, kv_lens.device, parents is not None)
    else:
        for name, dtype, n in (("qo_indptr", torch.int32, batch + 1), ("kv_page_indptr", torch.int32, batch + 1),
                               ("kv_page_indices", torch.int32, max_pages), ("kv_last_page_lens", torch.int32, batch),
                               ("positions", torch.int32, max_tokens), ("slots", torch.int64, max_tokens)):
            t = getattr(out, name)
            _check_vector("out." + name, t, dtype, n)
            if t.shape[0] != n:
                raise ValueError(f"out.{name} holds {t.shape[0]} entries, not {n}")
        if (out.masks is None) != (parents is None):
            raise ValueError("out has masks exactly where there are parents")
        if out.masks is not None:
            _check_vector("out.masks", out.masks, torch.int64, max_tokens)
        index = _on_device(kv_lens, page_tables, qo_lens, rows, parents, *out.csr, out.positions, out.slots, out.masks)
    table_rows, width = page_tables.shape
    args = _lib.StepTablesArgs(
        page_tables.data_ptr(), _lib.ptr(rows), kv_lens.data_ptr(), qo_lens.data_ptr(), _lib.ptr(parents),
        out.qo_indptr.data_ptr(), out.kv_page_indptr.data_ptr(), out.kv_last_page_lens.data_ptr(),
        out.kv_page_indices.data_ptr(), out.positions.data_ptr(), out.slots.data_ptr(), _lib.ptr(out.masks),
        page_tables.stride(0) if table_rows > 1 else width, 0 if parents is None else parents.numel(),
        table_rows, width, batch, page_size, max_tokens, max_pages)
    _call("build_step_tables", index, _lib.lib().dskv_step_tables, ctypes.byref(args))
    return out


def _token_rows(name: str, t: torch.Tensor, dtype: torch.dtype, heads: Optional[int], dim: int,
                tokens: Optional[int]) -> Tuple[torch.Tensor, int]:
    """(tokens, heads, dim) with the heads of a token contiguous, and how many elements tokens are apart: they may lie apart, as
    parts of one projection's output do.  Anything else is copied."""
    shape = t.shape
    if len(shape) != 3 or shape[2] != dim or t.dtype is not dtype or (heads is not None and shape[1] != heads) or \
            (tokens is not None and shape[0] != tokens):
        raise ValueError(f"{name} must be ({'tokens' if tokens is None else tokens}, {'heads' if heads is None else heads}, "
                         f"{dim}) of the pool's dtype, got {tuple(shape)} of {t.dtype}")
    n, h, _ = shape
    if t.data_ptr() % 16 == 0:
        if t.is_contiguous():
            return t, h * dim
        step, head, one = t.stride()
        if (dim == 1 or one == 1) and (h == 1 or head == dim):
            if n <= 1:
                return t, h * dim
            if step >= h * dim and step * t.element_size() % 16 == 0:
                return t, step
    return t.clone(memory_format=torch.contiguous_format), h * dim


def rope_append_slots(q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor,
                      paged_kv_data: torch.Tensor, rope_table: Optional[torch.Tensor] = None, *,
                      out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """In place on ``paged_kv_data`` (num_pages, 2, P, Hkv, D): row t's k, rotated, and v go to slots[t]; returns the
    rotated q.  rope_table (tokens, D) float32: cosines | sines of the rows' angles, by row (StepTables.rope_table,
    paged_ops.rope_table), with the arithmetic of apply_rope; None: nothing is rotated and q (may be None) comes back as it is.
    q, k and v may be parts of one projection's output: a token's heads are contiguous, tokens need not be.
    A slot that the pool does not have (-1) is no slot: the row goes nowhere; q is rotated in every row.  The slots of
    a call are distinct.  out: optional tensor for the rotated q, contiguous."""
    if paged_kv_data.dim() != 5 or paged_kv_data.shape[1] != 2 or not paged_kv_data.is_contiguous():
        raise ValueError("paged_kv_data must be a contiguous (num_pages, 2, P, Hkv, D) tensor")
    num_pages, _, page, hkv, dim = paged_kv_data.shape
    dtype = paged_kv_data.dtype
    k, k_stride = _token_rows("k", k, dtype, hkv, dim, None)
    nnz = k.shape[0]
    v, v_stride = _token_rows("v", v, dtype, hkv, dim, nnz)
    _check_vector("slots", slots, torch.int64, nnz)
    result, q_stride, heads = q, 0, hkv
    if rope_table is not None:
        if q is None:
            raise ValueError("rope_table rotates q and k: q is missing")
        q, q_stride = _token_rows("q", q, dtype, None, dim, nnz)
        heads = q.shape[1]
        table = rope_table.shape
        if rope_table.dtype is not torch.float32 or len(table) != 2 or table[1] != dim or table[0] < nnz or not rope_table.is_contiguous() or rope_table.data_ptr() % 16:
            raise ValueError(f"rope_table must be a contiguous, 16-byte aligned float32 ({nnz}, {dim}) tensor")
        if out is None:
            result = torch.empty_like(q, memory_format=torch.contiguous_format)
        elif out.shape != q.shape or out.dtype is not dtype or not out.is_contiguous():
            raise ValueError("out must be contiguous and of q's shape and dtype")
        else:
            result = out
    elif out is not None:
        raise ValueError("out is for the rotated q: rope_table is missing")
    index = _on_device(paged_kv_data, q, k, v, slots, rope_table, result)
    rotated = rope_table is not None
    _call("rope_append_slots", index, _lib.lib().dskv_rope_append_slots, result.data_ptr() if rotated else None,
          paged_kv_data.data_ptr(), num_pages, q.data_ptr() if rotated else None, k.data_ptr(), v.data_ptr(),
          q_stride, k_stride, v_stride, slots.data_ptr(), _lib.ptr(rope_table), nnz, page, heads, hkv, dim,
          _lib.dtype_code(dtype))
    return result


class BatchTreeWithPagedKVCacheWrapper:
    """Attention of the rows of a step over the paged context and over the rows that they descend from, with the
    begin_forward / forward / end_forward protocol of paged_ops.  begin_forward plans nothing and reads nothing back: the kernel
    takes lengths and tables from the device, so a captured step can be replayed with others.
    workspace_buffer: scratch of a forward while it runs (the 128 MiB of exec.get_wrappers hold every usual shape; one that needs
    more is refused); forwards that may run at the same time, on two streams, need one each.
    For requests of up to 1024 rows at head_dim 64 or 128; longer chunks and other dims are right, too, but read the context
    once a row: prompts are the prefill wrapper's."""

    def __init__(self, workspace_buffer: torch.Tensor, kv_layout: str = "NHD") -> None:
        if kv_layout != "NHD":
            raise ValueError("only the NHD page layout is implemented")
        self._workspace = workspace_buffer
        self._step: Optional[_lib.TreeStep] = None
        self._held: tuple = ()

    def begin_forward(self, qo_indptr: torch.Tensor, paged_kv_indptr: torch.Tensor, paged_kv_indices: torch.Tensor,
                      paged_kv_last_page_len: torch.Tensor, num_qo_heads: int, num_kv_heads: int, head_dim: int,
                      page_size: int, *, max_qo_len: int, masks: Optional[torch.Tensor] = None) -> None:
        """The index tensors (int32, as StepTables.csr holds them) are read by every forward, on the device: they stay as
        they are until the last one has run.
        max_qo_len: no request has more rows (of one that has, the further ones are left out).
        masks (tokens) int64, bit j: the row sees new row j of its request, at most MAX_TREE_ROWS rows a request;
        None: it sees the rows up to itself."""
        _check_vector("qo_indptr", qo_indptr, torch.int32, 1)
        batch = qo_indptr.numel() - 1
        _check_vector("paged_kv_indptr", paged_kv_indptr, torch.int32, batch + 1)
        _check_vector("paged_kv_indices", paged_kv_indices, torch.int32, 0)
        _check_vector("paged_kv_last_page_len", paged_kv_last_page_len, torch.int32, batch)
        if paged_kv_indptr.numel() != batch + 1:
            raise ValueError("qo_indptr and paged_kv_indptr disagree about the batch")
        if masks is not None:
            _check_vector("masks", masks, torch.int64, 0)
            if max_qo_len > MAX_TREE_ROWS:
                raise ValueError(f"masks hold {MAX_TREE_ROWS} rows a request, max_qo_len is {max_qo_len}")
        if num_kv_heads <= 0 or num_qo_heads <= 0 or num_qo_heads % num_kv_heads:
            raise ValueError(f"num_qo_heads {num_qo_heads} must be a multiple of num_kv_heads {num_kv_heads}")
        if head_dim <= 0 or head_dim % 8 or head_dim > 256:
            raise ValueError(f"head_dim {head_dim} must be a multiple of 8 up to 256")
        if page_size <= 0 or max_qo_len < 0:
            raise ValueError("page_size must be positive, max_qo_len not negative")
        _on_device(qo_indptr, paged_kv_indptr, paged_kv_indices, paged_kv_last_page_len, masks, self._workspace)
        self._held = (qo_indptr, paged_kv_indptr, paged_kv_indices, paged_kv_last_page_len, masks)
        self._step = _lib.TreeStep(
            qo_indptr.data_ptr(), paged_kv_indptr.data_ptr(), paged_kv_indices.data_ptr(),
            paged_kv_last_page_len.data_ptr(), _lib.ptr(masks), self._workspace.data_ptr(),
            self._workspace.numel() * self._workspace.element_size(), paged_kv_indices.numel(), batch, 0, min(max_qo_len, 2 ** 31 - 1),
            num_qo_heads, num_kv_heads, head_dim, page_size)

    def forward(self, q: torch.Tensor, paged_kv_data: torch.Tensor, sm_scale: Optional[float] = None, *,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """q (tokens, Hq, D), one row for every row of the step; rows behind the last request's are left out of the
        result (as they were in out).  K and V of the new rows are in the pages.  A row that sees nothing
        gets zeros.  out: optional result tensor (contiguous, q's shape and dtype)."""
        if self._step is None:
            raise RuntimeError("tree forward called before begin_forward")
        s = self._step
        page = paged_kv_data.shape
        if len(page) != 5 or page[1:] != (2, s.page_size, s.n_kv_heads, s.head_dim) or not paged_kv_data.is_contiguous():
            raise ValueError(f"paged_kv_data must be a contiguous (num_pages, 2, {s.page_size}, {s.n_kv_heads}, {s.head_dim}) "
                             f"tensor as given to begin_forward, got {tuple(page)}")
        dtype = paged_kv_data.dtype
        q, q_stride = _token_rows("q", q, dtype, s.n_qo_heads, s.head_dim, None)
        nnz, masks = q.shape[0], self._held[4]
        if masks is not None and masks.numel() < nnz:
            raise ValueError(f"masks hold {masks.numel()} rows, q has {nnz}")
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        elif out.shape != q.shape or out.dtype is not dtype or not out.is_contiguous():
            raise ValueError("out must be contiguous and of q's shape and dtype")
        index = _on_device(q, paged_kv_data, out, self._held[0])
        step = _lib.TreeStep.from_buffer_copy(s)      # calls from several threads do not share it
        step.nnz, step.num_pages, step.dtype = nnz, page[0], _lib.dtype_code(dtype)
        step.sm_scale = 1.0 / math.sqrt(s.head_dim) if sm_scale is None else sm_scale
        _call("tree forward", index, _lib.lib().dskv_tree_attn, ctypes.byref(step), out.data_ptr(), q.data_ptr(),
              q_stride, paged_kv_data.data_ptr())
        return out

    def end_forward(self) -> None:
        self._step, self._held = None, ()


@dataclass
class Verdict:
    """What verify_drafts writes, all on the device."""
    counts: torch.Tensor     # (batch) int32: tokens given to the request = rows of its walk
    path: torch.Tensor       # (tokens) int32, ragged: the walk's rows, row 0 first; then -1
    tokens: torch.Tensor     # (tokens) int32, ragged: the tokens given; then -1


def verify_drafts(target_probs: torch.Tensor, tokens: torch.Tensor, uniforms: torch.Tensor, qo_indptr: torch.Tensor, *,
                  parents: Optional[torch.Tensor] = None, draft_probs: Optional[torch.Tensor] = None) -> Verdict:
    """Accepts or refuses drafted tokens so that the tokens given are distributed as the target's own - as its rows say,
    if they sum to 1, the draft's too: R below starts at 1, not at a row's sum.  Rows of fewer bits are off by their rounding.

    target_probs (tokens, vocab): row t the target's probabilities of what follows row t.  tokens, uniforms (int32,
    float32): every row's token and its number from [0, 1); that of a request's row 0 is for the last draw.  From row 0 on the
    children of the row reached are tried in index order and the first that passes is followed:
    with draft_probs (tokens, vocab), for chains: token x, sampled from the draft's row q at its parent, passes if
    u q(x) < p(x), and where it is refused the last token is drawn from max(p - q, 0);
    without, for chains and trees (parents, as in build_step_tables) of proposed tokens: x passes if u R < p(x), R = 1 less
    the probabilities of the tokens refused there before (a token that was refused already does not pass),
    and the last token is drawn from p without the refused ones.
    Where nothing is refused, and where a distribution has no mass left, it is drawn from p.  A draw is the first index
    whose cumulated weight exceeds u times their sum; sums are in 64 bits.  One-hot rows of p verify greedily.
    A request has at most MAX_TREE_ROWS rows; one with more is given no token (counts 0), as one without rows."""
    if target_probs.dim() != 2 or (target_probs.shape[1] > 1 and target_probs.stride(1) != 1) or target_probs.shape[1] == 0:
        raise ValueError("target_probs must be (tokens, vocab) with contiguous rows")
    nnz, vocab = target_probs.shape
    for name, t in (("target_probs", target_probs), ("draft_probs", draft_probs)):
        if t is None:
            continue
        if t.shape != target_probs.shape or t.dtype is not target_probs.dtype or (vocab > 1 and t.stride(1) != 1) or \
                (nnz > 1 and t.stride(0) < vocab):
            raise ValueError(f"{name} must be a ({nnz}, {vocab}) tensor of {target_probs.dtype} with contiguous rows")
    if draft_probs is not None and parents is not None:
        raise ValueError("draft_probs belong to chains, parents to trees of proposed tokens")
    _check_vector("tokens", tokens, torch.int32, nnz)
    _check_vector("uniforms", uniforms, torch.float32, nnz)
    _check_vector("qo_indptr", qo_indptr, torch.int32, 1)
    if parents is not None:
        _check_vector("parents", parents, torch.int32, nnz)
    dtype, batch = _lib.dtype_code(target_probs.dtype), qo_indptr.numel() - 1
    index = _on_device(target_probs, tokens, uniforms, qo_indptr, parents, draft_probs)
    lib = _lib.lib()
    need = lib.dskv_verify_workspace(batch, vocab)
    # workspace and results, from the caching allocator for every call: calls on several streams share nothing
    workspace, counts, path, given = tokens.new_empty((need // 4 + batch + 2 * nnz,)).split_with_sizes((need // 4, batch, nnz, nnz))
    _call("verify_drafts", index, lib.dskv_verify_drafts, counts.data_ptr(), path.data_ptr(), given.data_ptr(),
          target_probs.data_ptr(), target_probs.stride(0) if nnz > 1 else vocab, _lib.ptr(draft_probs),
          0 if draft_probs is None else draft_probs.stride(0) if nnz > 1 else vocab, tokens.data_ptr(), uniforms.data_ptr(),
          qo_indptr.data_ptr(), _lib.ptr(parents), workspace.data_ptr(), need, batch, nnz, vocab, dtype)
    return Verdict(counts, path, given)


def move_accepted_rows(pages: torch.Tensor, slots: torch.Tensor, qo_indptr: torch.Tensor, path: torch.Tensor,
                       counts: torch.Tensor) -> None:
    """In place on ``pages`` (L, num_pages, 2, P, Hkv, D), layers possibly apart: K/V of the rows of every request's walk
    (verify_drafts) to where its sequence goes on, row j of the walk from slots[row path[j]] to slots[row j], in
    all layers.  Accepted chains are there already.  Rows that were refused stay behind the sequence, where the
    next step writes over them."""
    if pages.dim() != 6 or pages.shape[2] != 2 or not (pages.is_contiguous() or pages.shape[0] == 0 or pages[0].is_contiguous()):
        raise ValueError("pages must be (L, num_pages, 2, P, Hkv, D) with contiguous layers")
    layers, num_pages, _, page, hkv, dim = pages.shape
    size = pages.element_size()
    if hkv * dim * size % 16:
        raise ValueError(f"a token's K must be a multiple of 16 bytes, not {hkv * dim * size}")
    _check_vector("qo_indptr", qo_indptr, torch.int32, 1)
    batch = qo_indptr.numel() - 1
    _check_vector("path", path, torch.int32, 0)
    nnz = path.numel()
    _check_vector("slots", slots, torch.int64, nnz)
    _check_vector("counts", counts, torch.int32, batch)
    index = _on_device(pages, slots, qo_indptr, path, counts)
    if layers == 0 or num_pages == 0 or nnz == 0:
        return
    _call("move_accepted_rows", index, _lib.lib().dskv_move_rows, pages.data_ptr(), pages.stride(0) * size, layers,
          num_pages, page, hkv * dim * size, slots.data_ptr(), qo_indptr.data_ptr(), path.data_ptr(), counts.data_ptr(), batch,
          nnz)
