"""Pools of a caller's own classes, which know nothing of 8-bit pages: what asks a pool for its record takes one without for one of the
model's type."""
from types import SimpleNamespace

import pytest
import torch

from deserve_amd.execution import exec as batches
from deserve_amd.execution import graph as graphs
from deserve_amd.execution.graph import GraphedDecodeStep


def own_pool():
    return SimpleNamespace(main_device=torch.device("cpu"), main_dtype=torch.bfloat16, page_size=16, pages=torch.zeros(1))


def test_captured_steps(monkeypatch):
    pool, said = own_pool(), []
    wrapper = SimpleNamespace(begin_forward=lambda **kw: said.append(kw["data_type"]))
    host = dict.fromkeys(("kv_page_indptr", "kv_last_page_lens", "kv_page_indices"))
    ctx = SimpleNamespace(page_pool=pool, host=host, **host)
    monkeypatch.setattr(graphs.FlashDecodeCtx, "init_paged_decode_ctx", lambda *args: ctx)
    step = GraphedDecodeStep(None, wrapper, 4, 64, torch.device("cpu"), 8, 2, 64, 16)
    assert step._prepare([SimpleNamespace(seqlen=1)], [SimpleNamespace(pool=pool)]) is ctx
    assert said == [torch.bfloat16]
    with pytest.raises(ValueError, match="8 bits"):
        step._prepare([SimpleNamespace(seqlen=1)], [SimpleNamespace(pool=SimpleNamespace(record=1))])


def test_accepted_rows(monkeypatch):
    pool, moved = own_pool(), []
    monkeypatch.setattr(batches, "move_accepted_rows", lambda *args: moved.append(args))
    task = SimpleNamespace(task_id="a", seqlen=3)
    ex = batches.BatchVerify(torch.zeros(3, 4), None, [task], [SimpleNamespace(pool=pool)], parents=torch.tensor([-1, 0, 1], dtype=torch.int32))
    ex.tree_ctx = SimpleNamespace(page_pool=pool, tables=SimpleNamespace(slots=1), indptr=2)
    verdict = SimpleNamespace(path=3, counts=torch.tensor([2]))
    assert ex.accept(verdict) == [2] and task.seqlen == 2
    assert len(moved) == 1 and moved[0][0] is pool.pages
