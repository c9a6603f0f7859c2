"""What a stage's steps leave in 8-bit pages, codes and scales, against the append's definition alone: the results are compared with the
attention over the definition's records, too, not over those of the GPU."""
import dataclasses

import numpy as np
import pytest
import torch

from draftutil import attention, random_parents, to_signed
from quantutil import append, move, near
from test_gpu_quant_stage import DEV, DIM, HKV, HQ, LAYERS, make_pool, records_of, rows_for, step_of

pytestmark = pytest.mark.gpu


def touched(step):
    """Pages that hold rows of the step, and the places in them that the sequence has reached."""
    for b in range(len(step.kv)):
        _, _, table, length = step.request(b)
        for p in range(int(step.kv[b]) // step.page, -(-length // step.page)):
            yield table[p], min(step.page, length - p * step.page)


def check(tasks, caches, pool, want, xs, result, masks=None):
    """want: the records in front of the step by layer, from the definition; returns those behind it."""
    q, k, v = (x.cpu() for x in xs)
    out = []
    for layer in range(LAYERS):
        step = step_of(tasks, caches, pool, q[layer], masks)
        out.append(append(want[layer], step, k[layer].double().numpy(), v[layer].double().numpy(), 240 * 2.0 ** 120))
        got = records_of(pool, layer)
        for page, n in touched(step):
            assert np.array_equal(got.scales[page], out[-1].scales[page]), (layer, page)
            assert np.array_equal(got.codes[page, :, :, :n] & 0x7F, out[-1].codes[page, :, :, :n] & 0x7F), (layer, page)
        values = dataclasses.replace(step, pages=torch.from_numpy(out[-1].values().transpose(0, 1, 3, 2, 4).copy()))
        near(result[layer].view(q.shape[1], HQ, pool.head_dim), *attention(values))
    return out


@pytest.mark.parametrize("page", [16, 5])
def test_decode_and_mixed_steps(page):
    from deserve_amd.execution.exec import BatchDecode, BatchPrefill
    from deserve_amd.stage import KVStage, StageArgs
    from deserve_amd.task import SamplingParams, TaskData

    pool, caches = make_pool(120, page)
    pool.pages.zero_()
    want = [records_of(pool, layer) for layer in range(LAYERS)]
    stage = KVStage(StageArgs(HQ, HKV, HQ * DIM, page, LAYERS), use_rope=False)
    tasks = [TaskData.empty(f"t{i}", n, SamplingParams()) for i, n in enumerate([40, 70, 7, 1])]
    gen = torch.Generator(device="cuda").manual_seed(7)
    plan = [([0, 1, 2], [40, 30, 7]), ([0, 1, 2, 3], [1, 40, 1, 1]), ([0, 1, 2, 3], [1] * 4), ([3, 1], [1, 1]), ([0, 1, 2, 3], [1] * 4)]
    for i, (who, seqlens) in enumerate(plan):
        print("[case] records of a step", page, who, seqlens, flush=True)
        ts, cs = [tasks[w] for w in who], [caches[w] for w in who]
        for t, n in zip(ts, seqlens):
            t.init(n)
        xs = rows_for(gen, sum(seqlens), scale=[1.0, 6.0, 0.1, 50.0, 3.0][i])
        kind = BatchDecode if all(n == 1 for n in seqlens) else BatchPrefill
        ex = kind(xs, stage, ts, cs)
        ex.prepare()
        want = check(ts, cs, pool, want, xs, ex.step(True).all_xs)
        for t in ts:
            t.step()


def test_drafted_trees():
    """Trees, all of more columns than the narrow form's, with moves of what was accepted."""
    from deserve_amd.draft_ops import Verdict
    from deserve_amd.execution.exec import BatchVerify
    from deserve_amd.stage import KVStage, StageArgs
    from deserve_amd.task import SamplingParams, TaskData

    print("[case] records of drafted trees", flush=True)
    rng = np.random.default_rng(8)
    pool, caches = make_pool(80, 16)
    pool.pages.zero_()
    want = [records_of(pool, layer) for layer in range(LAYERS)]
    stage = KVStage(StageArgs(HQ, HKV, HQ * DIM, 16, LAYERS), use_rope=False)
    gen = torch.Generator(device="cuda").manual_seed(9)
    tasks = [TaskData("a", 0, 0, 20, 20, SamplingParams()), TaskData("b", 0, 0, 33, 33, SamplingParams())]
    cuda = lambda a: torch.from_numpy(np.asarray(a, np.int32)).to(DEV)
    for at in range(4):
        for t, n in zip(tasks, [(20, 33), (24, 18), (40, 17), (17, 64)][at]):
            t.seqlen = n
        n = [t.seqlen for t in tasks]
        parents = [random_parents(rng, x, 3) for x in n]
        masks = []
        for p in parents:
            own = []
            for i, up in enumerate(p.tolist()):
                own.append((own[up] if up >= 0 else 0) | 1 << i)
            masks += [to_signed(w) for w in own]
        masks = np.array(masks, np.int64)
        xs = rows_for(gen, sum(n), scale=5.0 ** at)
        ex = BatchVerify(xs, stage, tasks, caches[:2], torch.zeros(sum(n), dtype=torch.int32, device=DEV), cuda(np.concatenate(parents)))
        ex.prepare()
        want = check(tasks, caches[:2], pool, want, xs, ex.step().all_xs, masks)
        path, counts, lo = np.full(sum(n), -1, np.int32), [], 0
        for p in parents:
            walk = [0]
            while (down := [i for i in range(1, len(p)) if p[i] == walk[-1]]) and rng.random() < 0.9:
                walk.append(int(rng.choice(down)))
            path[lo: lo + len(walk)] = walk
            counts.append(len(walk))
            lo += len(p)
        step = step_of(tasks, caches[:2], pool, None)
        assert ex.accept(Verdict(cuda(counts), cuda(path), cuda(path))) == counts
        for layer in range(LAYERS):
            want[layer] = move(want[layer], step, path, np.array(counts))
            got = records_of(pool, layer)
            for page, places in touched(step):
                assert np.array_equal(got.scales[page], want[layer].scales[page]), (layer, page)
                assert np.array_equal(got.codes[page, :, :, :places] & 0x7F, want[layer].codes[page, :, :, :places] & 0x7F), (layer, page)
        for t in tasks:
            t.step()


@pytest.mark.parametrize("rows_of", [(24, 18), (24, 3), (1, 1)])
def test_steps_of_trees_say_how_few_rows_a_request_has(rows_of):
    """The hint that leaves out the launch for requests of few rows, where a step has none: from the tasks, of trees and chains."""
    from deserve_amd.execution.exec import BatchVerify
    from deserve_amd.stage import KVStage, StageArgs
    from deserve_amd.task import SamplingParams, TaskData

    pool, caches = make_pool(80, 16)
    stage = KVStage(StageArgs(HQ, HKV, HQ * DIM, 16, LAYERS), use_rope=False)
    tasks = [TaskData(t, 0, 0, n, n, SamplingParams()) for t, n in zip("ab", rows_of)]
    total = sum(rows_of)
    chain = torch.cat([torch.arange(-1, n - 1, dtype=torch.int32) for n in rows_of]).to(DEV)
    for parents in (None, chain):
        ex = BatchVerify(rows_for(torch.Generator(device="cuda").manual_seed(1), total), stage, tasks, caches[:2],
                         torch.zeros(total, dtype=torch.int32, device=DEV), parents)
        ex.prepare()
        assert ex.tree_ctx.tree_wrapper._step.min_qo_len == min(rows_of)
        assert ex.tree_ctx.tree_wrapper._step.step.max_qo_len == max(rows_of)
