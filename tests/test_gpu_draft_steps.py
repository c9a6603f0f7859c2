"""Steps of drafted tokens as a program runs them: tables, append, attention of all layers, verification, accepted rows moved, the
next step on top.  What the cache holds afterwards is what a prefill of the sequences given writes, bit for bit, the
accepted rows' results are the sequence's attention by its definition, and the verdicts are the definition's."""
import numpy as np
import pytest
import torch

from deserve_amd.draft_ops import (build_step_tables, move_accepted_rows, rope_append_slots, verify_drafts)
from deserve_amd.execution.exec import BatchVerify, get_tree_wrapper, get_wrappers
from deserve_amd.kvcache.paged.kvcache import PagedKVCache
from deserve_amd.kvcache.paged.page_pool import GpuPagePool
from deserve_amd.kvcache.paged.page_table import PageTableAllocator
from deserve_amd.model.context.flash import FlashPrefillCtx
from deserve_amd.paged_ops import rope_append_paged_kv_cache
from deserve_amd.stage import PackedKVStage, StageArgs
from deserve_amd.task import TaskData
from draftutil import DTYPES, Step, attention, random_parents, verdict

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
LAYERS, HQ, HKV, DIM, VOCAB, THETA = 3, 8, 2, 128, 24, 10000.0


def _caches(n, pages, page, dtype):
    pool = GpuPagePool(LAYERS, pages, page, torch.device(DEV), dtype, HKV, DIM)
    table = PageTableAllocator(n, 64 * page, page, torch.device(DEV))
    return pool, [PagedKVCache.empty(table, pool) for _ in range(n)]


def _held(pool, cache, tokens):
    """K and V of a sequence's tokens: (layers, 2, tokens, heads, dim)."""
    ids = cache.page_table.retrieve().long().to(DEV)
    rows = pool.pages[:, ids].permute(0, 2, 1, 3, 4, 5).flatten(2, 3)
    return rows[:, :, :tokens]


def _prefill(xs, tasks, caches):
    """Rotated K and V of the tasks' tokens into their caches, by the framework's append for prompts; (rotated q of all
    layers, the step's context)."""
    ctx = FlashPrefillCtx.init_paged_prefill_ctx(tasks, caches, get_wrappers(torch.device(DEV))[1])
    q, k, v = (xs[:, :, a: b].transpose(0, 1).contiguous() for a, b in ((0, HQ), (HQ, HQ + HKV), (HQ + HKV, HQ + 2 * HKV)))
    out = [rope_append_paged_kv_cache(q[i], k[i], v[i], ctx.indptr, ctx.offsets, ctx.page_pool.pages[i], ctx.kv_page_indices,
                                      ctx.kv_page_indptr, ctx.kv_last_page_lens, rope_theta=THETA) for i in range(LAYERS)]
    return out, ctx


def _probs(rng, rows):
    """fp32 rows that put most of their mass on few tokens."""
    w = rng.random((rows, VOCAB)) ** 8
    return torch.from_numpy((w / w.sum(1, keepdims=True)).astype(np.float32))


@pytest.mark.parametrize("dtype,page", [("bf16", 16), ("f16", 3), ("fp32", 16)])
@pytest.mark.parametrize("kind", ["chains", "drafts", "trees"])
def test_steps_leave_what_a_prefill_of_the_sequence_writes(kind, dtype, page):
    print("[case] steps", kind, dtype, page, flush=True)
    rng = np.random.default_rng(11)
    dt = DTYPES[dtype]
    embed = torch.randn(VOCAB, LAYERS, HQ + 2 * HKV, DIM, generator=torch.Generator().manual_seed(3)).to(dt).to(DEV)
    stage = PackedKVStage(StageArgs(HQ, HKV, HQ * DIM, page, LAYERS, THETA))
    prompts = [1, 5, 15, 16, 33]
    pool, caches = _caches(len(prompts), 120, page, dt)
    seqs = [rng.integers(0, VOCAB, n).tolist() for n in prompts]       # the last token has no K and V yet
    tasks = [TaskData(str(i), 0, 0, n, n) for i, n in enumerate(prompts)]
    _prefill(embed[torch.tensor(sum(seqs, []), device=DEV)], tasks, caches)
    seqs = [s + [int(rng.integers(VOCAB))] for s in seqs]
    for t in tasks:
        t.step()
    results = [{} for _ in prompts]        # position -> (layers, heads, dim)
    taken = 0
    for turn in range(5):
        rows = [int(rng.integers(1, 8)) for _ in prompts]
        if turn == 1:
            rows = [1] * len(prompts)
        for t, n in zip(tasks, rows):
            t.init(n)
        indptr = np.concatenate([[0], np.cumsum(rows)])
        target = _probs(rng, sum(rows))
        draft = _probs(rng, sum(rows)) if kind == "drafts" else None
        parents = np.concatenate([random_parents(rng, n, 3) for n in rows]) if kind == "trees" else None
        tokens = np.empty(sum(rows), np.int32)
        for b, n in enumerate(rows):
            for j in range(n):
                up = j - 1 if parents is None else parents[indptr[b] + j]
                source = target if draft is None else draft
                tokens[indptr[b] + j] = seqs[b][-1] if j == 0 else rng.choice(VOCAB, p=(
                    lambda w: w / w.sum())(source[indptr[b] + up].double().numpy()))
        uniforms = rng.random(sum(rows)).astype(np.float32)
        on = lambda a: None if a is None else torch.as_tensor(a).to(DEV)
        batch = BatchVerify(embed[on(tokens).long()], stage, tasks, caches, on(tokens), on(parents))
        if turn == 2:       # as a scheduler regroups it
            batch = BatchVerify.merge(batch.split())
            tail = batch.pop()
            batch = BatchVerify.merge([batch, tail])
        batch.prepare()
        out = batch.step(True).all_xs.view(LAYERS, -1, HQ, DIM)
        said = batch.verify(on(target), on(uniforms), on(draft))
        counts, path, given = verdict(target.double().numpy(), tokens, uniforms, indptr, parents,
                                      None if draft is None else draft.double().numpy())
        assert said.counts.tolist() == counts.tolist()
        assert said.path.tolist() == path.tolist() and said.tokens.tolist() == given.tolist()
        assert batch.accept(said) == counts.tolist()
        for b, task in enumerate(tasks):
            for j in range(counts[b]):
                results[b][len(seqs[b]) - 1 + j] = out[:, indptr[b] + path[indptr[b] + j]]
            seqs[b] += given[indptr[b]: indptr[b] + counts[b]].tolist()
            task.step()
            assert task.start_pos == len(seqs[b]) - 1
        taken += int(sum(counts)) - len(prompts)
    assert taken > 5                        # drafts were accepted

    lens = [len(s) - 1 for s in seqs]
    pool2, caches2 = _caches(len(prompts), 120, page, dt)
    q, ctx = _prefill(embed[torch.tensor(sum((s[:-1] for s in seqs), []), device=DEV)],
                      [TaskData(str(i), 0, 0, n, n) for i, n in enumerate(lens)], caches2)
    csr = [getattr(ctx, f).cpu().numpy() for f in ("indptr", "kv_page_indptr", "kv_page_indices", "kv_last_page_lens")]
    for b, n in enumerate(lens):
        assert torch.equal(_held(pool, caches[b], n), _held(pool2, caches2[b], n)), b
    for layer in range(LAYERS):
        want, bound = attention(Step(np.zeros(len(lens), np.int64), np.array(lens), None, page, HQ, HKV, DIM, dtype, csr[0],
                                     csr[1], csr[2], csr[3], None, pool2.pages[layer].cpu(), q[layer].cpu()))
        for b in range(len(lens)):
            for pos, got in results[b].items():
                off = (got[layer].double().cpu().numpy() - want[csr[0][b] + pos])
                assert (np.abs(off) <= bound[csr[0][b] + pos]).all(), (b, pos, layer)


def test_steps_prepared_ahead_keep_their_own_tables():
    dt = DTYPES["bf16"]
    stage = PackedKVStage(StageArgs(HQ, HKV, HQ * DIM, 16, LAYERS, THETA))
    pool, caches = _caches(2, 40, 16, dt)
    tasks = [TaskData("a", 0, 0, 70, 70), TaskData("b", 0, 0, 20, 20)]
    gen = torch.Generator().manual_seed(9)
    randn = lambda n: torch.randn(n, LAYERS, HQ + 2 * HKV, DIM, generator=gen).to(dt).to(DEV)
    _prefill(randn(90), tasks, caches)
    for t, n in zip(tasks, (6, 3)):
        t.step()
        t.init(n)
    xs = [randn(6), randn(3)]
    steps = lambda: [BatchVerify(x, stage, [t], [c]) for x, t, c in zip(xs, tasks, caches)]
    want = []
    for s in steps():
        s.prepare()
        want.append(s.step().all_xs.clone())
    ahead = steps()
    for s in ahead:
        s.prepare()
    for s, w in zip(ahead, want):
        assert torch.equal(s.step().all_xs, w)


class _Program:
    """Buffers of a step, and the step over them: lengths stay on the device and go on by what was given."""

    def __init__(self, dtype, tree):
        gen = torch.Generator().manual_seed(5)
        self.tree = tree
        self.embed = torch.randn(VOCAB, LAYERS, HQ + 2 * HKV, DIM, generator=gen).to(dtype).to(DEV)
        self.pages = torch.randn(LAYERS, 80, 2, 16, HKV, DIM, generator=gen).to(dtype).to(DEV)
        self.table = torch.randperm(80, generator=gen)[:72].view(4, 18).to(torch.int32).to(DEV)
        self.kv = torch.tensor([40, 0, 100, 15], dtype=torch.int32, device=DEV)
        self.rows = torch.zeros(4, dtype=torch.int32, device=DEV)
        self.tokens = torch.zeros(40, dtype=torch.int32, device=DEV)
        self.parents = torch.zeros(40, dtype=torch.int32, device=DEV)
        self.target = torch.zeros(40, VOCAB, device=DEV)
        self.uniforms = torch.zeros(40, device=DEV)
        self.out = torch.full((LAYERS, 40, HQ, DIM), 7.0, dtype=dtype, device=DEV)
        self.verdict = None

    def load(self, seed):
        rng = np.random.default_rng(seed)
        rows = rng.integers(0, 11, 4)
        rows[seed % 4] = 0
        n = int(rows.sum())
        self.rows.copy_(torch.from_numpy(rows.astype(np.int32)))
        self.tokens.copy_(torch.from_numpy(rng.integers(0, VOCAB, 40).astype(np.int32)))
        parents = np.concatenate([random_parents(rng, int(r), 3) for r in rows])
        self.parents[:n].copy_(torch.from_numpy(parents))
        self.target.copy_(_probs(rng, 40))
        self.uniforms.copy_(torch.from_numpy(rng.random(40).astype(np.float32)))

    def step(self):
        parents = self.parents if self.tree else None
        tables = build_step_tables(self.table, self.kv, self.rows, 16, max_tokens=40, max_pages=72, parents=parents)
        wrapper = get_tree_wrapper(torch.device(DEV))
        wrapper.begin_forward(*tables.csr, HQ, HKV, DIM, 16, max_qo_len=12, masks=tables.masks)
        angles = tables.rope_table(DIM, THETA)
        xs = self.embed[self.tokens.long()]
        for layer in range(LAYERS):
            q = rope_append_slots(xs[:, layer, :HQ], xs[:, layer, HQ: HQ + HKV], xs[:, layer, HQ + HKV:], tables.slots,
                                  self.pages[layer], angles)
            wrapper.forward(q, self.pages[layer], out=self.out[layer])
        self.verdict = verify_drafts(self.target, self.tokens, self.uniforms, tables.qo_indptr, parents=parents)
        move_accepted_rows(self.pages, tables.slots, tables.qo_indptr, self.verdict.path, self.verdict.counts)
        self.kv += self.verdict.counts

    def state(self):
        return [t.clone() for t in (self.pages, self.kv, self.out, self.verdict.counts, self.verdict.path, self.verdict.tokens)]


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_captured_steps_go_on_as_eager_ones(dtype):
    """Two captured programs, which share the workspace, replayed in turn with eager steps of two others between
    them, those on a stream of their own."""
    print("[case] captured steps", dtype, flush=True)
    graphs = [_Program(DTYPES[dtype], tree) for tree in (False, True)]
    eager = [_Program(DTYPES[dtype], tree) for tree in (False, True)]
    side, captured = torch.cuda.Stream(), []
    for p in graphs:
        start = [t.clone() for t in (p.pages, p.kv, p.out)]
        p.load(0)
        p.step()                                   # the library's first calls are made outside
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            p.step()
        for t, was in zip((p.pages, p.kv, p.out), start):
            t.copy_(was)
        captured.append(g)
    for turn in range(6):
        for p, g, other in zip(graphs, captured, eager):
            p.load(turn + 1)
            g.replay()
            got = p.state()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                other.load(turn + 1)
                other.step()
                want = other.state()
            torch.cuda.current_stream().wait_stream(side)
            torch.cuda.synchronize()
            for a, b in zip(got, want):
                assert torch.equal(a, b)
    assert int(graphs[1].kv.sum()) > 155           # tokens were given
