"""Execution-layer objects (deserve_worker/execution/exec.py:20-22,58-243).

``prepare()`` builds the forward context (extending the caches) and plans the
attention; ``step()`` runs ``layer_storage.forward(xs, ctx)`` and closes the
plan.  ``layer_storage`` is whatever owns the layers of this stage: it must
offer ``forward(xs, ctx)``, ``model_args`` (n_heads, n_kv_heads, dim,
page_size) and ``need_sample`` (+ ``sample`` when true); the dense model itself
is outside this package.  The reference's module-level workspace and wrapper
pair become lazily created per-device singletons.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Dict, List, Optional, Sequence, Tuple

import torch

from deserve_amd.draft_ops import (MAX_TREE_ROWS, BatchTreeWithPagedKVCacheWrapper, Verdict, move_accepted_rows,
                                   verify_drafts)
from deserve_amd.execution.result import BatchResult
from deserve_amd.kvcache.paged.kvcache import PagedKVCache
from deserve_amd.model.context.flash import FlashDecodeCtx, FlashPrefillCtx, FlashTreeCtx
from deserve_amd.paged_ops import (BatchDecodeWithPagedKVCacheWrapper,
                                   BatchPrefillWithPagedKVCacheWrapper)
from deserve_amd.task import TaskData

WORKSPACE_BYTES = 128 * 1024 * 1024
_wrappers: Dict[torch.device, Tuple[BatchDecodeWithPagedKVCacheWrapper,
                                    BatchPrefillWithPagedKVCacheWrapper]] = {}


def get_wrappers(device: torch.device):
    """(decode_wrapper, prefill_wrapper) sharing one 128 MiB workspace per device."""
    device = torch.device(device)
    if device not in _wrappers:
        ws = torch.empty(WORKSPACE_BYTES, dtype=torch.uint8, device=device)
        _wrappers[device] = (BatchDecodeWithPagedKVCacheWrapper(ws),
                             BatchPrefillWithPagedKVCacheWrapper(ws))
    return _wrappers[device]


_tree_wrappers: Dict[torch.device, BatchTreeWithPagedKVCacheWrapper] = {}


def get_tree_wrapper(device: torch.device) -> BatchTreeWithPagedKVCacheWrapper:
    """The wrapper for steps of drafted tokens, over the workspace of get_wrappers."""
    device = torch.device(device)
    if device not in _tree_wrappers:
        _tree_wrappers[device] = BatchTreeWithPagedKVCacheWrapper(get_wrappers(device)[0]._workspace)
    return _tree_wrappers[device]


@dataclass
class BatchExec:
    xs: torch.Tensor                 # ragged: one row per token of the batch
    layer_storage: object
    task_datas: List[TaskData]
    kvcaches: List[PagedKVCache]

    def bsz(self) -> int:
        return len(self.task_datas)

    def seqlens(self) -> List[int]:
        return [t.seqlen for t in self.task_datas]

    def total_seqlen(self) -> int:
        return sum(self.seqlens())

    @classmethod
    def merge(cls, execs: Sequence["BatchExec"]):
        return cls(torch.cat([e.xs for e in execs]), execs[0].layer_storage,
                   [t for e in execs for t in e.task_datas],
                   [c for e in execs for c in e.kvcaches])

    def split(self):
        out, pos = [], 0
        for task, cache in zip(self.task_datas, self.kvcaches):
            out.append(type(self)(self.xs[pos: pos + task.seqlen], self.layer_storage, [task],
                                  [cache]))
            pos += task.seqlen
        return out

    def pop(self):
        task, cache = self.task_datas.pop(), self.kvcaches.pop()
        tail = type(self)(self.xs[-task.seqlen:], self.layer_storage, [task], [cache])
        self.xs = self.xs[: -task.seqlen]
        return tail

    def post_process(self, result: torch.Tensor, ignore_eos: bool) -> BatchResult:
        ids = [t.task_id for t in self.task_datas]
        if not getattr(self.layer_storage, "need_sample", False):
            return BatchResult(result, ids, result, list(ids), [], {})
        ongoing_tok, ongoing, all_tok, all_datas, done, probs = self.layer_storage.sample(
            result, self.task_datas, ignore_eos)
        empty = torch.empty(0, dtype=torch.int, device=result.device)
        return BatchResult(torch.cat(ongoing_tok) if ongoing_tok else empty,
                           [t.task_id for t in ongoing],
                           torch.cat(all_tok) if all_tok else empty,
                           [t.task_id for t in all_datas], [t.task_id for t in done],
                           {t.task_id: p for t, p in probs})

    def _shape_kwargs(self) -> dict:
        a = self.layer_storage.model_args
        n_kv = a.n_heads if a.n_kv_heads is None else a.n_kv_heads
        return dict(num_qo_heads=a.n_heads, num_kv_heads=n_kv, head_dim=a.dim // a.n_heads,
                    page_size=a.page_size)


@dataclass
class BatchDecode(BatchExec):
    decode_ctx: Optional[FlashDecodeCtx] = None

    def prepare(self) -> None:
        with torch.inference_mode():
            wrapper, _ = get_wrappers(self.kvcaches[0].pool.main_device)
            # the context's index arrays and the attention work list go up in one kernel
            ctx = FlashDecodeCtx.init_and_plan(self.task_datas, self.kvcaches, wrapper,
                                               **self._shape_kwargs())
            self.decode_ctx = ctx

    def step(self, ignore_eos: bool) -> BatchResult:
        with torch.inference_mode():
            assert self.decode_ctx is not None
            result = self.layer_storage.forward(self.xs, self.decode_ctx)
            self.decode_ctx.decode_wrapper.end_forward()
            return self.post_process(result, ignore_eos)


@dataclass
class BatchPrefill(BatchExec):
    prefill_ctx: Optional[FlashPrefillCtx] = None

    def prepare(self) -> None:
        with torch.inference_mode():
            _, wrapper = get_wrappers(self.kvcaches[0].pool.main_device)
            # metadata and plan in one pinned block, one upload kernel
            self.prefill_ctx = FlashPrefillCtx.init_and_plan(self.task_datas, self.kvcaches, wrapper,
                                                             **self._shape_kwargs())

    def step(self, ignore_eos: bool) -> BatchResult:
        with torch.inference_mode():
            assert self.prefill_ctx is not None
            result = self.layer_storage.forward(self.xs, self.prefill_ctx)
            self.prefill_ctx.prefill_wrapper.end_forward()
            return self.post_process(result, ignore_eos)


@dataclass
class BatchVerify(BatchExec):
    """A step of drafted tokens: the rows of a task are its last token and the drafts behind it, task.seqlen of them,
    MAX_TREE_ROWS at most.
    prepare() and step() run on every stage; the last one makes probabilities of what step() returns and calls
    verify(); accept() with its verdict, on every stage, leaves the cache of the accepted rows in the order of the
    sequence and task.seqlen as what the step has advanced by, for task.step().  No counterpart in the reference."""
    tokens: Optional[torch.Tensor] = None      # int32, one a row; for verify()
    parents: Optional[torch.Tensor] = None     # int32, one a row, within the task (build_step_tables); None: chains
    tree_ctx: Optional[FlashTreeCtx] = None

    @classmethod
    def merge(cls, execs: Sequence["BatchVerify"]) -> "BatchVerify":
        """Chains merged with trees become trees: verify() takes no draft_probs for the step then, and their tokens are
        proposals like the trees' - distributed as the target's all the same, though fewer of them are accepted."""
        whole = super().merge(execs)
        if any(e.tokens is not None for e in execs):
            if any(e.tokens is None for e in execs):
                raise ValueError("some of the steps have tokens, some have none")
            whole.tokens = torch.cat([e.tokens for e in execs])
        if any(e.parents is not None for e in execs):      # a chain is the tree in which each row follows the one in front
            whole.parents = torch.cat([e._parents() for e in execs])
        return whole

    def _parents(self) -> torch.Tensor:
        if self.parents is not None:
            return self.parents
        return torch.cat([torch.arange(-1, n - 1, dtype=torch.int32) for n in self.seqlens()]).to(self.xs.device)

    def split(self) -> List["BatchVerify"]:
        out, pos = super().split(), 0
        for part in out:
            rows = slice(pos, pos + part.total_seqlen())
            part.tokens = None if self.tokens is None else self.tokens[rows]
            part.parents = None if self.parents is None else self.parents[rows]
            pos = rows.stop
        return out

    def pop(self) -> "BatchVerify":
        begin = self.total_seqlen() - self.task_datas[-1].seqlen
        tail = super().pop()
        if self.tokens is not None:
            self.tokens, tail.tokens = self.tokens[:begin], self.tokens[begin:]
        if self.parents is not None:
            self.parents, tail.parents = self.parents[:begin], self.parents[begin:]
        return tail

    def prepare(self) -> None:
        if max(self.seqlens()) > MAX_TREE_ROWS:            # on every stage, before a cache grows for rows that no verdict accepts
            raise ValueError(f"a task has at most {MAX_TREE_ROWS} rows to verify")
        with torch.inference_mode():
            # a wrapper of its own, which costs nothing: a step prepared in between does not change this one
            wrapper = BatchTreeWithPagedKVCacheWrapper(get_tree_wrapper(self.kvcaches[0].pool.main_device)._workspace)
            self.tree_ctx = FlashTreeCtx.init_and_plan(self.task_datas, self.kvcaches, wrapper, parents=self.parents,
                                                       **self._shape_kwargs())

    def step(self, ignore_eos: bool = False) -> BatchResult:
        """The rows of the stage's result; nothing is sampled here."""
        with torch.inference_mode():
            assert self.tree_ctx is not None
            result = self.layer_storage.forward(self.xs, self.tree_ctx)
            self.tree_ctx.tree_wrapper.end_forward()
            ids = [t.task_id for t in self.task_datas]
            return BatchResult(result, ids, result, list(ids), [], {})

    def verify(self, target_probs: torch.Tensor, uniforms: torch.Tensor,
               draft_probs: Optional[torch.Tensor] = None) -> Verdict:
        """draft_ops.verify_drafts over the rows of the step.  draft_probs: for steps of chains only (see merge)."""
        with torch.inference_mode():
            assert self.tree_ctx is not None and self.tokens is not None
            if draft_probs is not None and self.parents is not None:
                raise ValueError("draft_probs belong to chains: trees, and chains merged with trees are verified without")
            if max(self.seqlens()) > MAX_TREE_ROWS:
                raise ValueError(f"a task has at most {MAX_TREE_ROWS} rows to verify")
            if target_probs.shape[0] < self.total_seqlen():      # (the tasks behind them would be given no token)
                raise ValueError(f"{target_probs.shape[0]} rows of probabilities for {self.total_seqlen()} rows")
            return verify_drafts(target_probs, self.tokens, uniforms, self.tree_ctx.indptr, parents=self.parents,
                                 draft_probs=draft_probs)

    def accept(self, verdict: Verdict) -> List[int]:
        """Tokens given to each task; waits for the verdict."""
        with torch.inference_mode():
            assert self.tree_ctx is not None
            ctx = self.tree_ctx
            if self.parents is not None:                    # the rows of an accepted chain are in place
                move_accepted_rows(ctx.page_pool.pages, ctx.tables.slots, ctx.indptr, verdict.path, verdict.counts)
            counts = verdict.counts.tolist()
            for task, n in zip(self.task_datas, counts):
                task.seqlen = n
            return counts
