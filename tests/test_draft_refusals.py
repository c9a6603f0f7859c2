"""Refusals of the drafted-token operators, before anything is launched (all on the CPU)."""
import ctypes
import os
import subprocess
import sys

import pytest
import torch

from deserve_amd.execution.exec import BatchVerify
from deserve_amd.kvcache.paged.kvcache import PagedKVCache
from deserve_amd.kvcache.paged.page_pool import PagePool
from deserve_amd.kvcache.paged.page_table import PageTableAllocator
from deserve_amd.model.context.flash import FlashTreeCtx
from deserve_amd.task import TaskData
from deserve_amd import _lib
from deserve_amd.draft_ops import (BatchTreeWithPagedKVCacheWrapper, StepTables, build_step_tables, move_accepted_rows,
                                   rope_append_slots, verify_drafts)

bf16 = torch.bfloat16


def i32(*x):
    return torch.tensor(x, dtype=torch.int32)


def refused(match, fn, *args, **kw):
    with pytest.raises(ValueError, match=match):
        fn(*args, **kw)


def test_step_tables():
    tables, kv, qo = torch.zeros((3, 4), dtype=torch.int32), i32(1, 2), i32(1, 1)
    kw = dict(max_tokens=4, max_pages=4)
    refused("on the GPU", build_step_tables, tables, kv, qo, 16, **kw)
    refused("page_tables", build_step_tables, tables.long(), kv, qo, 16, **kw)
    refused("page_tables", build_step_tables, tables[0], kv, qo, 16, **kw)
    refused("page_tables", build_step_tables, tables.t(), kv, qo, 16, **kw)
    refused("page_tables", build_step_tables, tables[:1].expand(3, 4), kv, qo, 16, **kw)
    refused("kv_lens", build_step_tables, tables, kv.long(), qo, 16, **kw)
    refused("kv_lens", build_step_tables, tables, i32(1, 2, 3, 4)[::2], qo, 16, **kw)
    refused("disagree", build_step_tables, tables, kv, i32(1), 16, **kw)
    refused("rows holds 1", build_step_tables, tables, kv, qo, 16, rows=i32(1), **kw)
    refused("parents", build_step_tables, tables, kv, qo, 16, parents=torch.zeros(3), **kw)
    refused("page_size", build_step_tables, tables, kv, qo, 0, **kw)
    refused("max_tokens", build_step_tables, tables, kv, qo, 16, max_tokens=-1, max_pages=4)
    out = lambda batch, tokens, pages, tree: StepTables.empty(batch, tokens, pages, torch.device("cpu"), tree)
    refused("on the GPU", build_step_tables, tables, kv, qo, 16, out=out(2, 4, 4, False), **kw)
    refused("out.qo_indptr holds 4", build_step_tables, tables, kv, qo, 16, out=out(3, 4, 4, False), **kw)
    refused("out.positions holds 3", build_step_tables, tables, kv, qo, 16, out=out(2, 3, 4, False), **kw)
    refused("out.kv_page_indices holds 5", build_step_tables, tables, kv, qo, 16, out=out(2, 4, 5, False), **kw)
    refused("masks exactly", build_step_tables, tables, kv, qo, 16, out=out(2, 4, 4, True), **kw)
    refused("masks exactly", build_step_tables, tables, kv, qo, 16, out=out(2, 4, 4, False), parents=i32(0, 0), **kw)


def test_rows_into_slots():
    pages = torch.zeros((4, 2, 16, 8, 64), dtype=bf16)
    q, k, slots, table = torch.zeros((3, 32, 64), dtype=bf16), torch.zeros((3, 8, 64), dtype=bf16), torch.zeros(3).long(), torch.zeros((3, 64))
    refused("on the GPU", rope_append_slots, q, k, k, slots, pages, table)
    refused("paged_kv_data", rope_append_slots, q, k, k, slots, pages[:, 0], table)
    refused("paged_kv_data", rope_append_slots, q, k, k, slots, pages[::2], table)
    refused("k must be", rope_append_slots, q, k.half(), k, slots, pages, table)
    refused("k must be", rope_append_slots, q, k[:, :4], k, slots, pages, table)
    refused("v must be \\(3", rope_append_slots, q, k, k[:2], slots, pages, table)
    refused("q must be \\(3", rope_append_slots, q[:2], k, k, slots, pages, table)
    refused("q is missing", rope_append_slots, None, k, k, slots, pages, table)
    refused("slots", rope_append_slots, q, k, k, slots.int(), pages, table)
    refused("slots holds 2", rope_append_slots, q, k, k, slots[:2], pages, table)
    refused("rope_table", rope_append_slots, q, k, k, slots, pages, table[:, :32])
    refused("rope_table", rope_append_slots, q, k, k, slots, pages, table.double())
    refused("out must be", rope_append_slots, q, k, k, slots, pages, table, out=q[:2])
    refused("out is for", rope_append_slots, q, k, k, slots, pages, out=q)


def test_tree_attention():
    w = BatchTreeWithPagedKVCacheWrapper(torch.empty(16, dtype=torch.uint8))
    with pytest.raises(RuntimeError, match="before begin_forward"):
        w.forward(torch.zeros(1), torch.zeros(1))
    refused("NHD", BatchTreeWithPagedKVCacheWrapper, torch.empty(1), "HND")
    csr = (i32(0, 2), i32(0, 1), i32(0), i32(5))
    begin = lambda csr=csr, hq=32, hkv=8, dim=128, page=16, **kw: w.begin_forward(*csr, hq, hkv, dim, page, **{"max_qo_len": 2, **kw})
    refused("on the GPU", begin)
    refused("qo_indptr", begin, (torch.zeros(2), *csr[1:]))
    refused("paged_kv_indptr holds 1", begin, (csr[0], i32(0), *csr[2:]))
    refused("disagree", begin, (csr[0], i32(0, 1, 2), *csr[2:]))
    refused("last_page_len holds 0", begin, (*csr[:3], i32()))
    refused("masks must", begin, masks=i32(1, 1))
    refused("masks hold 64 rows", begin, masks=torch.zeros(70).long(), max_qo_len=65)
    refused("multiple of num_kv_heads", begin, hq=30)
    refused("head_dim 100", begin, dim=100)
    refused("head_dim 264", begin, dim=264)
    refused("page_size", begin, page=0)
    with pytest.raises(RuntimeError, match="before begin_forward"):
        w.forward(torch.zeros(1), torch.zeros(1))
    # behind a begin_forward on the GPU
    w._step = _lib.TreeStep(batch=1, n_qo_heads=32, n_kv_heads=8, head_dim=128, page_size=16, max_qo_len=2)
    w._held = (*csr, torch.zeros(2).long())
    pages, q = torch.zeros((1, 2, 16, 8, 128), dtype=bf16), torch.zeros((2, 32, 128), dtype=bf16)
    refused("as given to begin_forward", w.forward, q, pages[:, :, :8])
    refused("as given to begin_forward", w.forward, q, torch.zeros((4, 2, 16, 8, 128), dtype=bf16)[::2])
    refused("q must be", w.forward, q.half(), pages)
    refused("q must be", w.forward, q[:, :16], pages)
    refused("masks hold 2 rows, q has 3", w.forward, torch.zeros((3, 32, 128), dtype=bf16), pages)
    refused("out must be", w.forward, q, pages, out=q[:1])
    refused("out must be", w.forward, q, pages, out=q.half())
    refused("on the GPU", w.forward, q, pages)
    w.end_forward()
    with pytest.raises(RuntimeError, match="before begin_forward"):
        w.forward(q, pages)


def test_verify():
    p, tok, u, ptr = torch.rand((4, 10)), i32(1, 2, 3, 4), torch.rand(4), i32(0, 4)
    refused("on the GPU", verify_drafts, p, tok, u, ptr)
    refused("target_probs", verify_drafts, p[0], tok, u, ptr)
    refused("target_probs", verify_drafts, p[:, ::2], tok, u, ptr)
    refused("target_probs", verify_drafts, p[:, :0], tok, u, ptr)
    refused("target_probs", verify_drafts, p[:1].expand(4, 10), tok, u, ptr)
    refused("draft_probs must", verify_drafts, p, tok, u, ptr, draft_probs=p[:3])
    refused("draft_probs must", verify_drafts, p, tok, u, ptr, draft_probs=p.half())
    refused("belong to chains", verify_drafts, p, tok, u, ptr, draft_probs=p, parents=tok)
    refused("tokens", verify_drafts, p, tok.long(), u, ptr)
    refused("tokens holds 3", verify_drafts, p, tok[:3], u, ptr)
    refused("uniforms", verify_drafts, p, tok, u.double(), ptr)
    refused("qo_indptr", verify_drafts, p, tok, u, i32())
    refused("parents holds 2", verify_drafts, p, tok, u, ptr, parents=tok[:2])
    refused("dtype", verify_drafts, p.double(), tok, u, ptr)


def test_move():
    pages = torch.zeros((2, 3, 2, 16, 8, 64), dtype=bf16)
    slots, ptr, path, counts = torch.zeros(4).long(), i32(0, 4), i32(0, 2, -1, -1), i32(2)
    refused("on the GPU", move_accepted_rows, pages, slots, ptr, path, counts)
    refused("pages must", move_accepted_rows, pages[0], slots, ptr, path, counts)
    refused("pages must", move_accepted_rows, pages[:, ::2], slots, ptr, path, counts)
    refused("16 bytes", move_accepted_rows, pages[..., :1, :4].contiguous(), slots, ptr, path, counts)
    refused("slots holds 3", move_accepted_rows, pages, slots[:3], ptr, path, counts)
    refused("path", move_accepted_rows, pages, slots, ptr, path.long(), counts)
    refused("counts holds 0", move_accepted_rows, pages, slots, ptr, path, counts[:0])


def test_the_librarys_own_refusals():
    lib = _lib.lib()
    says = lambda rc, what, code=-1: rc == code and what in _lib.last_error()
    assert says(lib.dskv_step_tables(None, None), "null")
    t = _lib.StepTablesArgs(*[16] * 12, 4, 0, 2, 4, 1, 16, 1, 1)
    for name, value, what in (("batch", -1, "negative"), ("max_pages", -1, "negative"), ("page_size", 0, "page_size"),
                              ("table_stride", 3, "table shape"), ("kv_lens", None, "null"), ("slots", None, "null"),
                              ("kv_page_indices", None, "null"), ("page_tables", None, "page tables"), ("qo_indptr", None, "null")):
        bad = _lib.StepTablesArgs.from_buffer_copy(t)
        setattr(bad, name, value)
        assert says(lib.dskv_step_tables(ctypes.byref(bad), None), what), name
    bad = _lib.StepTablesArgs.from_buffer_copy(t)
    bad.parents, bad.n_parents = None, 3
    assert says(lib.dskv_step_tables(ctypes.byref(bad), None), "parents")

    # q_out, pages, num_pages, q, k, v, strides x3, slots, table, nnz, P, Hq, Hkv, D, dtype, stream
    good = [16, 16, 4, 16, 16, 16, 4096, 1024, 1024, 16, 16, 3, 16, 32, 8, 128, 2, None]
    call = lambda **at: lib.dskv_rope_append_slots(*[at.get("a%d" % i, v) for i, v in enumerate(good)])
    assert call(a11=0) == 0 and says(call(a11=-1), "negative") and says(call(a4=None), "null") and says(call(a16=5), "dtype")
    assert says(call(a15=132), "head_dim") and says(call(a7=1016), "overlap") and says(call(a6=4100), "aligned")
    assert says(call(a3=24), "aligned") and says(call(a2=0), "shape") and says(call(a0=None), "null")

    s = _lib.TreeStep(16, 16, 16, 16, None, None, 0, 1, 2, 4, 2, 32, 8, 128, 16, 4, 2, 0.1)
    attn = lambda step, out=16, q=16, stride=4096, pages=16: lib.dskv_tree_attn(ctypes.byref(step), out, q, stride, pages, None)
    for name, value, what in (("batch", -1, "negative"), ("dtype", 7, "dtype"), ("n_qo_heads", 30, "multiple"), ("head_dim", 12, "head_dim"),
                              ("head_dim", 264, "head_dim"), ("num_pages", 0, "page shape"), ("qo_indptr", None, "null")):
        bad = _lib.TreeStep.from_buffer_copy(s)
        setattr(bad, name, value)
        assert says(attn(bad), what), name
    bad = _lib.TreeStep.from_buffer_copy(s)
    bad.masks, bad.max_qo_len = 16, 65
    assert says(attn(bad), "masks hold 64")
    assert says(attn(s, out=None), "null") and says(attn(s, stride=4088), "overlap") and says(attn(s, stride=4100), "aligned")
    assert says(attn(s, q=8), "aligned") and says(lib.dskv_tree_attn(None, 16, 16, 4096, 16, None), "null")
    for name in ("batch", "nnz", "max_qo_len"):
        empty = _lib.TreeStep.from_buffer_copy(s)
        setattr(empty, name, 0)
        assert attn(empty, out=None, q=None, pages=None) == 0

    # counts, path, tokens, target, stride, draft, stride, tokens, uniforms, indptr, parents, ws, bytes, batch, nnz, vocab, dtype, stream
    good = [16, 16, 16, 16, 100, None, 0, 16, 16, 16, None, 16, 1 << 20, 2, 8, 100, 0, None]
    call = lambda **at: lib.dskv_verify_drafts(*[at.get("a%d" % i, v) for i, v in enumerate(good)])
    assert says(call(a13=-1), "negative") and says(call(a15=0), "vocab") and says(call(a3=None), "null") and says(call(a16=3), "dtype")
    assert says(call(a5=16, a6=100, a10=16), "chains") and says(call(a4=99), "overlap") and says(call(a13=65536), "65535")
    assert says(call(a12=8), "needed", -2) and says(call(a11=None), "needed", -2) and says(call(a11=24), "aligned")
    assert call(a13=0, a14=0) == 0

    good = [16, 1 << 20, 2, 4, 16, 2048, 16, 16, 16, 16, 2, 8, None]
    call = lambda **at: lib.dskv_move_rows(*[at.get("a%d" % i, v) for i, v in enumerate(good)])
    assert call(a10=0) == 0 and call(a2=0) == 0 and says(call(a10=-1), "negative") and says(call(a0=None), "null")
    assert says(call(a5=24), "16") and says(call(a0=24), "aligned") and says(call(a1=4096), "overlap") and says(call(a2=65536), "65535")
    assert says(call(a3=0), "page shape")


def test_steps_of_a_stage():
    pool = PagePool(1, 8, 16, torch.device("cpu"), torch.bfloat16, 2, 128)
    table = PageTableAllocator(4, 256, 16, torch.device("cpu"))
    caches = [PagedKVCache.empty(table, pool) for _ in range(2)]
    tasks = [TaskData("a", 3, 1, 2, 3), TaskData("b", 0, 0, 65, 1)]
    shape = dict(num_qo_heads=4, num_kv_heads=2, head_dim=128, page_size=16)
    plan = lambda n, parents, of=caches: FlashTreeCtx.init_and_plan(tasks[:n], of[:n], None, parents=parents, **shape)
    with pytest.raises(ValueError, match="at most 64 rows"):
        plan(2, torch.zeros(67, dtype=torch.int32))
    with pytest.raises(ValueError, match="parents holds 3 entries for 2 rows"):
        plan(1, torch.zeros(3, dtype=torch.int32))
    other = PagePool(1, 8, 16, torch.device("cpu"), torch.bfloat16, 2, 128)
    with pytest.raises(ValueError, match="over one pool"):
        plan(2, None, [caches[0], PagedKVCache.empty(table, other)])
    assert pool.num_avails == 8                                       # nothing was reserved
    steps = [BatchVerify(torch.zeros(t.seqlen, 1), None, [t], [c]) for t, c in zip(tasks, caches)]
    steps[0].tokens = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="some have none"):
        BatchVerify.merge(steps)
    steps[1].tokens, steps[1].tree_ctx = torch.zeros(65, dtype=torch.int32), object()
    with pytest.raises(ValueError, match="at most 64 rows"):
        steps[1].verify(torch.zeros(65, 8), torch.zeros(65))


def test_steps_regrouped():
    """Chains and trees merged, split and popped keep their tokens and parents."""
    tasks = [TaskData(str(i), 0, 0, n, n) for i, n in enumerate((2, 3, 1))]
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)
    steps = [BatchVerify(torch.zeros(2, 1), None, tasks[:1], [0], i32(7, 8)),
             BatchVerify(torch.ones(4, 1), None, tasks[1:], [1, 2], i32(4, 5, 6, 9), i32(-1, 0, 0, -1))]
    whole = BatchVerify.merge(steps)
    assert whole.tokens.tolist() == [7, 8, 4, 5, 6, 9] and whole.parents.tolist() == [-1, 0, -1, 0, 0, -1]
    assert [(p.tokens.tolist(), p.parents.tolist()) for p in whole.split()] == \
        [([7, 8], [-1, 0]), ([4, 5, 6], [-1, 0, 0]), ([9], [-1])]
    tail = whole.pop()
    assert (tail.tokens.tolist(), tail.parents.tolist()) == ([9], [-1])
    assert (whole.tokens.tolist(), whole.parents.tolist()) == ([7, 8, 4, 5, 6], [-1, 0, -1, 0, 0])
    chains = BatchVerify.merge([steps[0], BatchVerify(torch.ones(3, 1), None, [TaskData("x", 0, 0, 3, 3)], [1], i32(1, 2, 3))])
    assert chains.parents is None and chains.pop().tokens.tolist() == [1, 2, 3]


def test_steps_that_cannot_be_verified_are_refused_before_they_begin():
    """Chains of more rows than a verification takes, and parents of another form: no cache has grown."""
    pool = PagePool(1, 8, 16, torch.device("cpu"), torch.bfloat16, 2, 128)
    table = PageTableAllocator(4, 256, 16, torch.device("cpu"))
    caches = [PagedKVCache.empty(table, pool) for _ in range(2)]
    tasks = [TaskData("a", 3, 1, 2, 3), TaskData("b", 0, 0, 65, 1)]
    for tokens in (None, torch.zeros(67, dtype=torch.int32)):
        with pytest.raises(ValueError, match="at most 64 rows"):
            BatchVerify(torch.zeros(67, 1), None, tasks, caches, tokens).prepare()
    shape = dict(num_qo_heads=4, num_kv_heads=2, head_dim=128, page_size=16)
    for parents in (torch.zeros(2).long(), torch.zeros((1, 2), dtype=torch.int32), torch.zeros(4, dtype=torch.int32)[::2]):
        refused("parents must be", FlashTreeCtx.init_and_plan, tasks[:1], caches[:1], None, parents=parents, **shape)
    assert pool.num_avails == 8 and caches[0].page_table.occupied == caches[1].page_table.occupied == 0


def test_chains_merged_with_trees_are_verified_as_proposals():
    """The draft's distributions are refused for the whole step, in words that say what is left to do."""
    chain = BatchVerify(torch.zeros(2, 1), None, [TaskData("a", 0, 0, 2, 2)], [0], i32(7, 8))
    tree = BatchVerify(torch.ones(3, 1), None, [TaskData("b", 0, 0, 3, 3)], [1], i32(4, 5, 6), i32(-1, 0, 0))
    whole = BatchVerify.merge([chain, tree])
    whole.tree_ctx = object()
    probs = torch.rand((5, 8))
    refused("merged with trees are verified without", whole.verify, probs, torch.rand(5), probs)


def test_a_step_is_verified_by_as_many_rows_as_it_has():
    """Probabilities or tokens of fewer rows would give the tasks behind them no token, not even the target's own."""
    step = BatchVerify(torch.zeros(5, 1), None, [TaskData("a", 0, 0, 2, 2), TaskData("b", 0, 0, 3, 3)], [0, 1], i32(7, 8, 4, 5, 6))
    step.tree_ctx = type("Ctx", (), {"indptr": i32(0, 2, 5)})()
    refused("2 rows of probabilities for 5 rows", step.verify, torch.rand((2, 8)), torch.rand(5))
    refused("uniforms holds 4", step.verify, torch.rand((5, 8)), torch.rand(4))
    step.tokens = step.tokens[:4]
    refused("tokens holds 4", step.verify, torch.rand((5, 8)), torch.rand(5))
    step.tokens = i32(7, 8, 4, 5, 6, 9, 9)                     # padded ones are taken
    refused("on the GPU", step.verify, torch.rand((7, 8)), torch.rand(7))


def test_workspaces_for_any_number_of_rows():
    """max_qo_len as large as its type goes, with every group: an answer, and not the end of the process."""
    code = ("from deserve_amd import _lib\n"
            "for rows in (1 << 24, 1 << 28, 1 << 29, 1 << 30, (1 << 31) - 1):\n"
            "    for group in (1, 4, 16, 32, 64, 128, 256, 512, 1024, 1 << 16):\n"
            "        for dtype in (_lib.F32, _lib.F16, _lib.BF16):\n"
            "            for dim in (64, 128):\n"
            "                assert _lib.lib().dskv_tree_attn_workspace(3, 9, rows, group, 1, dim, dtype) > 0, (rows, group, dtype, dim)\n")
    done = subprocess.run([sys.executable, "-c", code], cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                          capture_output=True, text=True)
    assert done.returncode == 0, (done.returncode, done.stderr[-500:])
