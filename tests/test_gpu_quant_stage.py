"""A stage over 8-bit pages: decode, prefill and mixed steps, drafted tokens, offload and reload, slice swaps and captured steps.
After every step the pages are the append's by its definition, and the results the attention over what they stand for."""
import dataclasses

import numpy as np
import pytest
import torch

from draftutil import Step, attention, random_parents
from quantutil import Records, append, move, near

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
LAYERS, HQ, HKV, DIM = 2, 8, 2, 64
F8 = torch.float8_e4m3fn


def make_pool(pages, page, n=8, dim=DIM):
    from deserve_amd.kvcache.paged.kvcache import PagedKVCache
    from deserve_amd.kvcache.paged.page_pool import GpuPagePool
    from deserve_amd.kvcache.paged.page_table import PageTableAllocator

    pool = GpuPagePool(LAYERS, pages, page, DEV, F8, HKV, dim)
    table = PageTableAllocator(n, 64 * page, page, DEV)
    return pool, [PagedKVCache.empty(table, pool) for _ in range(n)]


def records_of(pool, layer):
    return Records.of_tensor(pool.pages[layer], pool.page_size, pool.n_kv_heads, pool.head_dim)


def step_of(tasks, caches, pool, q, masks=None):
    """The step as the definitions take it; pages and q of one layer come later."""
    kv, n = (np.array([getattr(t, f) for t in tasks], np.int64) for f in ("start_pos", "seqlen"))
    exposed = -(-(kv + n) // pool.page_size)
    ids = np.concatenate([c.page_table.retrieve()[:e].numpy() for c, e in zip(caches, exposed)]).astype(np.int32)
    return Step(kv, n, None, pool.page_size, HQ, HKV, pool.head_dim, "bf16", np.concatenate([[0], np.cumsum(n)]).astype(np.int32),
                np.concatenate([[0], np.cumsum(exposed)]).astype(np.int32), ids, ((kv + n - 1) % pool.page_size + 1).astype(np.int32),
                masks, None, q)


def check(tasks, caches, pool, before, xs, result, masks=None):
    """xs: (q, k, v) by layer; before: records in front of the step."""
    q, k, v = (x.cpu() for x in xs)
    total = q.shape[1]
    for layer in range(LAYERS):
        step = step_of(tasks, caches, pool, q[layer], masks)
        want = append(before[layer], step, k[layer].double().numpy(), v[layer].double().numpy(), 240 * 2.0 ** 120)
        got = records_of(pool, layer)
        used = np.unique(step.kv_page_indices)
        assert np.array_equal(got.codes[used], want.codes[used]) or _same_but_behind(got, want, step)
        values = dataclasses.replace(step, pages=torch.from_numpy(got.values().transpose(0, 1, 3, 2, 4).copy()))
        near(result[layer].view(total, HQ, pool.head_dim), *attention(values))


def _same_but_behind(got, want, step):
    """Codes of every token that there is; signed zeros are alike."""
    for b in range(len(step.kv)):
        _, _, table, length = step.request(b)
        at = np.arange(length)
        x, y = (r.values()[table[at // step.page], :, :, at % step.page] for r in (got, want))
        if not np.array_equal(x, y):
            return False
    return True


def rows_for(gen, total, dim=DIM, scale=1.0):
    return tuple((scale * torch.randn((LAYERS, total, h, dim), generator=gen, device=DEV)).to(torch.bfloat16) for h in (HQ, HKV, HKV))


@pytest.mark.parametrize("page", [16, 8, 5])
def test_steps_of_a_stage(page):
    from deserve_amd.execution.exec import BatchDecode, BatchPrefill
    from deserve_amd.stage import KVStage, StageArgs
    from deserve_amd.task import SamplingParams, TaskData

    pool, caches = make_pool(120, page)
    pool.pages.fill_(0xFF)                                   # memory that nothing was written to
    stage = KVStage(StageArgs(HQ, HKV, HQ * DIM, page, LAYERS), use_rope=False)
    tasks = [TaskData.empty(f"t{i}", n, SamplingParams()) for i, n in enumerate([40, 100, 7, 1])]
    gen = torch.Generator(device="cuda").manual_seed(1)
    plan = [([0, 1, 2], [40, 60, 7]), ([0, 1, 2, 3], [1, 40, 1, 1]), ([0, 1, 2, 3], [1, 1, 1, 1]), ([3, 1], [1, 1]), ([0, 1, 2, 3], [1, 1, 1, 1])]
    for i, (who, seqlens) in enumerate(plan):
        print("[case] stage step", page, who, seqlens, flush=True)
        ts, cs = [tasks[w] for w in who], [caches[w] for w in who]
        for t, n in zip(ts, seqlens):
            t.init(n)
        xs = rows_for(gen, sum(seqlens), scale=[1.0, 5.0, 0.1, 1.0, 20.0][i])
        before = [records_of(pool, layer) for layer in range(LAYERS)]
        kind = BatchDecode if all(n == 1 for n in seqlens) else BatchPrefill
        ex = kind(xs, stage, ts, cs)
        ex.prepare()
        other = kind(xs, stage, ts[:1], cs[:1])              # prepared in between, never run
        other.prepare()
        result = ex.step(True).all_xs
        check(ts, cs, pool, before, xs, result)
        for t in ts:
            t.step()


def test_rotation_through_a_stage():
    """With rotation the stage is the operators one after the other, bit for bit."""
    from deserve_amd.execution.exec import BatchPrefill, get_quantized_wrapper
    from deserve_amd.paged_ops import rope_table
    from deserve_amd.quant_ops import rope_append_quantized
    from deserve_amd.stage import KVStage, StageArgs
    from deserve_amd.task import SamplingParams, TaskData

    pools = [make_pool(40, 16) for _ in range(2)]
    tasks = [TaskData.empty("a", 50, SamplingParams()), TaskData.empty("b", 9, SamplingParams())]
    for t, n in zip(tasks, (50, 9)):
        t.init(n)
    gen = torch.Generator(device="cuda").manual_seed(2)
    xs = rows_for(gen, 59)
    ex = BatchPrefill(xs, KVStage(StageArgs(HQ, HKV, HQ * DIM, 16, LAYERS, 1e4), use_rope=True), tasks, pools[0][1][:2])
    ex.prepare()
    result = ex.step(True).all_xs
    for c, n in zip(pools[1][1], (50, 9)):
        c.extend(n)
    ctx = ex.prefill_ctx
    table = rope_table(ctx.indptr, ctx.offsets, 59, DIM, 1e4)
    pool = pools[1][0]
    w = get_quantized_wrapper(DEV)
    w.begin_forward(ctx.indptr, ctx.kv_page_indptr, ctx.kv_page_indices, ctx.kv_last_page_lens, HQ, HKV, DIM, 16, max_qo_len=50)
    for layer in range(LAYERS):
        q = rope_append_quantized(xs[0][layer], xs[1][layer], xs[2][layer], ctx.indptr, pool.pages[layer], ctx.kv_page_indices,
                                  ctx.kv_page_indptr, ctx.kv_last_page_lens, 16, table)
        out = w.forward(q, pool.pages[layer])
        assert torch.equal(out.view(59, -1).view(torch.int16), result[layer].view(59, -1).view(torch.int16))
        a, b = (records_of(p[0], layer) for p in pools)
        used = ctx.kv_page_indices.cpu().numpy()
        assert np.array_equal(a.scales[used], b.scales[used])


@pytest.mark.parametrize("trees", [True, False])
def test_drafted_tokens_over_8_bit_pages(trees):
    from deserve_amd.draft_ops import Verdict
    from deserve_amd.execution.exec import BatchVerify
    from deserve_amd.stage import KVStage, StageArgs
    from deserve_amd.task import SamplingParams, TaskData

    print("[case] drafted tokens", trees, flush=True)
    rng = np.random.default_rng(4)
    pool, caches = make_pool(80, 16)
    pool.pages.zero_()
    stage = KVStage(StageArgs(HQ, HKV, HQ * DIM, 16, LAYERS), use_rope=False)
    gen = torch.Generator(device="cuda").manual_seed(3)
    tasks = [TaskData("a", 0, 0, 20, 20, SamplingParams()), TaskData("b", 0, 0, 33, 33, SamplingParams()), TaskData("c", 0, 0, 1, 1, SamplingParams())]
    for at in range(4):
        if at:
            for t, n in zip(tasks, ([7, 30, 3], [20, 1, 5], [4, 4, 4])[at - 1]):
                t.seqlen = n
        n = [t.seqlen for t in tasks]
        parents = [random_parents(rng, x, 3) if trees else np.arange(-1, x - 1, dtype=np.int32) for x in n]
        flat = torch.from_numpy(np.concatenate(parents)).to(DEV) if trees else None
        masks = None
        if trees:
            masks = []
            for p in parents:
                own = []
                for i, up in enumerate(p.tolist()):
                    own.append((own[up] if up >= 0 else 0) | 1 << i)
                masks += [w - (1 << 64) if w >> 63 else w for w in own]
            masks = np.array(masks, np.int64)
        xs = rows_for(gen, sum(n), scale=4.0 ** at)
        before = [records_of(pool, layer) for layer in range(LAYERS)]
        ex = BatchVerify(xs, stage, tasks, caches[:3], torch.zeros(sum(n), dtype=torch.int32, device=DEV), flat)
        ex.prepare()
        result = ex.step().all_xs
        check(tasks, caches[:3], pool, before, xs, result, masks)
        path, counts = np.full(sum(n), -1, np.int32), []
        lo = 0
        for p in parents:
            walk = [0]
            while (down := [i for i in range(1, len(p)) if p[i] == walk[-1]]) and rng.random() < 0.9:
                walk.append(int(rng.choice(down)))
            path[lo: lo + len(walk)] = walk
            counts.append(len(walk))
            lo += len(p)
        steps = [step_of(tasks, caches[:3], pool, None) for _ in range(LAYERS)]
        held = [records_of(pool, layer) for layer in range(LAYERS)]
        cuda = lambda a: torch.from_numpy(np.asarray(a, np.int32)).to(DEV)
        assert ex.accept(Verdict(cuda(counts), cuda(path), cuda(path))) == counts
        for layer in range(LAYERS):
            want = move(held[layer], steps[layer], path, np.array(counts)) if trees else held[layer]
            got = records_of(pool, layer)
            assert np.array_equal(got.values(), want.values()), layer
        for t in tasks:
            t.step()


def test_offload_reload_and_slices():
    """Records travel as they are: what a request's pages hold is the same bytes after offload and reload, and after a trip of
    its slice, and its next step continues from there."""
    from deserve_amd.engine.pipeline.processor import PipelineProcessor, StepRequest
    from deserve_amd.stage import KVStage, StageArgs
    from deserve_amd.task import SamplingParams

    print("[case] 8-bit pages through the engine", flush=True)
    P = 16
    stage = KVStage(StageArgs(HQ, HKV, HQ * DIM, P, LAYERS), use_rope=False)
    proc = PipelineProcessor(num_rounds=2, num_pages_main=6, num_pages_swap=12, page_size=P, batch_size=4, layer_storage=stage,
                             num_layers=LAYERS, buddy_height=6, main_dtype=F8, max_context_len=512, n_kv_heads=HKV, head_dim=DIM)
    pool = proc.virtual_page_pool
    assert pool.pages.dtype is torch.uint8 and proc.cpu_chunk_pool.chunks.dtype is torch.uint8
    gen = torch.Generator(device="cuda").manual_seed(5)
    lens = {"a": 50, "b": 33, "c": 70, "d": 40}
    held = {}                                                # values of every request's tokens, by layer

    def tokens(cache, count):
        table, at = cache.page_table.retrieve().numpy(), np.arange(count)
        return [records_of(pool, layer).values()[table[at // P], :, :, at % P] for layer in range(LAYERS)]

    def run(m, ids, seqlens, init=False, **kw):
        xs = rows_for(gen, sum(seqlens))
        caches = proc.microbatches[m].ongoing_paged_kvcaches
        proc.run_step(StepRequest(m, xs, ids, seqlens, init_tasks={t: (lens[t], SamplingParams()) for t in ids} if init else {}, **kw))
        torch.cuda.synchronize()
        result, lo = proc.last_result.all_xs, 0
        for tid, n in zip(ids, seqlens):
            old = held.get(tid)
            count = (0 if old is None else old[0].shape[0]) + n
            now = tokens(caches[tid], count)
            for layer in range(LAYERS):
                if old is not None:                          # rounded anew at most, where a scale grew
                    off = np.abs(now[layer][: count - n] - old[layer])
                    assert (off <= 2.0 ** -10 * np.abs(now[layer]).max() / 128).all()
                k, v = (x[layer, lo: lo + n].float().cpu().numpy() for x in xs[1:])
                new = now[layer][count - n:]
                for i, x in enumerate((k, v)):
                    assert (np.abs(new[:, i] - x) <= np.maximum(2.0 ** -4 * np.abs(x), 2.0 ** -10 * np.abs(now[layer]).max() / 128)).all()
                step = Step(np.array([count - n]), np.array([n]), None, P, HQ, HKV, DIM, "bf16", np.array([0, n], np.int32),
                            np.array([0, -(-count // P)], np.int32), np.arange(-(-count // P), dtype=np.int32),
                            np.array([(count - 1) % P + 1], np.int32), None, None, xs[0][layer, lo: lo + n].cpu())
                pages = np.zeros((-(-count // P) * P, 2, HKV, DIM))
                pages[:count] = now[layer]
                step.pages = torch.from_numpy(pages.reshape(-1, P, 2, HKV, DIM).transpose(0, 2, 1, 3, 4).copy())
                near(result[layer].view(-1, HQ, DIM)[lo: lo + n], *attention(step))
            held[tid] = now
            lo += n
    idle = lambda m, **kw: proc.run_step(StepRequest(m, None, **kw))
    run(0, ["a", "b", "c"], [50, 33, 70], init=True)
    run(1, ["d"], [40], init=True)                           # the slice of round 0 goes out, and comes back
    run(0, ["a", "c"], [1, 1], offload_task_ids=["b"])
    run(1, ["d"], [1])
    run(0, ["a", "b", "c"], [1, 1, 1], reload_task_ids=["b"])
    idle(1)
    run(0, ["a", "b"], [1, 1], cancel_task_ids=["c"])
    used_swap = any(bool(c.isswap[: c.page_table.occupied].any()) for c in proc.microbatches[0].ongoing_paged_kvcaches.values())
    assert used_swap, "the scenario was meant to exercise the swap slices"
    ids = proc.microbatches[0].ongoing_paged_kvcaches["a"].page_table.retrieve()
    gathered = pool.retrieve(ids)
    assert torch.equal(gathered, pool.pages[:, ids.long().to(DEV)])
    assert pool.record.values(gathered).shape == (LAYERS, len(ids), 2, P, HKV, DIM)
    proc.synchronize()


def test_captured_decode_steps():
    """One capture for a batch size, whatever the lengths; the bits of eager steps."""
    from deserve_amd.execution.exec import BatchDecode, get_wrappers
    from deserve_amd.execution.graph import GraphedDecodeStep
    from deserve_amd.quant_ops import BatchQuantizedWithPagedKVCacheWrapper
    from deserve_amd.stage import KVStage, StageArgs
    from deserve_amd.task import SamplingParams, TaskData

    print("[case] captured steps over 8-bit pages", flush=True)
    sides = []
    for _ in range(2):
        pool, caches = make_pool(200, 16)
        pool.pages.view(-1)[:] = torch.arange(pool.pages.numel(), device=DEV, dtype=torch.int64).mul_(2654435761).bitwise_right_shift_(7).to(torch.uint8) & 0x77
        pool.record.scales(pool.pages).fill_(0.25)
        sides.append((pool, caches, [TaskData(f"t{i}", n, 0, 1, n, SamplingParams()) for i, n in enumerate([13, 15, 300, 47, 900])]))
    args = StageArgs(HQ, HKV, HQ * DIM, 16, LAYERS)
    stage = KVStage(args, use_rope=True)
    shape = dict(num_qo_heads=HQ, num_kv_heads=HKV, head_dim=DIM, page_size=16)
    step = GraphedDecodeStep(stage, BatchQuantizedWithPagedKVCacheWrapper(torch.empty(64 << 20, dtype=torch.uint8, device=DEV)),
                             max_batch=8, max_pages=400, device=DEV, **shape)
    gen = torch.Generator(device="cuda").manual_seed(6)
    picks = [[0, 1, 2], [0, 1, 2], [3, 4, 0], [0, 1, 2, 3, 4], [4, 2, 1], [0, 1, 2, 3, 4]]
    for at, pick in enumerate(picks):
        xs = rows_for(gen, len(pick))
        (pe, ce, te), (pg, cg, tg) = sides
        ex = BatchDecode(xs, stage, [te[i] for i in pick], [ce[i] for i in pick])
        ex.prepare()
        want = ex.step(True).all_xs.clone()
        got = step.run(xs, [tg[i] for i in pick], [cg[i] for i in pick]).clone()
        torch.cuda.synchronize()
        assert torch.equal(got.view(torch.int16), want.view(torch.int16)), at
        assert torch.equal(pe.pages, pg.pages), at
        for i in pick:
            te[i].step()
            tg[i].step()
    assert step.captures == 2
    with pytest.raises(ValueError, match="8 bits"):
        GraphedDecodeStep(stage, get_wrappers(DEV)[0], 8, 400, DEV, **shape).run(xs, tg[:1], cg[:1])
