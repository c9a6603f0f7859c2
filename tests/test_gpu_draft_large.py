"""The drafted-token operators at the far end: pages behind 4 GB of a pool, contexts of 10^5 tokens, vocabularies
of more parts than a wave has lanes, table rows and walks longer than what a workgroup takes at once."""
import numpy as np
import pytest
import torch

from deserve_amd.draft_ops import (BatchTreeWithPagedKVCacheWrapper, build_step_tables, move_accepted_rows, rope_append_slots,
                                   verify_drafts)
from deserve_amd.execution.exec import get_tree_wrapper
from draftutil import attention, make_step, verdict

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def forward(step, csr, pages, q, masks, scale=None):
    w = BatchTreeWithPagedKVCacheWrapper(get_tree_wrapper(torch.device(DEV))._workspace)
    w.begin_forward(*csr, step.hq, step.hkv, step.dim, step.page, max_qo_len=int(step.rows.max()), masks=masks)
    return w.forward(q, pages, scale)


def i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(DEV)


@pytest.mark.parametrize("dtype,dim,rows,tree", [("bf16", 128, 5, False), ("bf16", 128, 40, True), ("fp32", 128, 9, True),
                                                 ("f16", 64, 12, True), ("bf16", 80, 6, True)])
def test_pages_behind_4_gb(dtype, dim, rows, tree):
    """The same step over a small pool and over the far pages of one of 9 GB and more: the same bits."""
    print("[case] far pages", dtype, dim, rows, flush=True)
    step = make_step(7, [300, 41], [rows, rows // 2], tree, dim=dim, dtype=dtype)
    on = step.on(DEV)
    page_bytes = on["pages"][0].numel() * on["pages"].element_size()
    far = 9 * 2 ** 30 // page_bytes + 1
    pool = torch.empty((far, *on["pages"].shape[1:]), dtype=on["pages"].dtype, device=DEV)
    n = len(step.kv_page_indices)
    ids = np.where(np.arange(n) % 2 == 0, far - 1 - np.arange(n), 2 + np.arange(n))       # far and near ones in turn
    pool[torch.from_numpy(ids).to(DEV)] = on["pages"][torch.from_numpy(step.kv_page_indices).long().to(DEV)]
    csr = list(on["csr"])
    want = forward(step, csr, on["pages"], on["q"], on["masks"])
    csr[2] = i32(ids)
    assert torch.equal(forward(step, csr, pool, on["q"], on["masks"]), want)
    # appended there, and moved from there
    slots = torch.tensor([(far - 1) * 16 + 3, (far - 1) * 16 + 5, 16 + 2], device=DEV)
    k, v = on["pages"][0, 0, :3].clone(), on["pages"][0, 1, :3].clone()
    rope_append_slots(None, k, v, slots, pool)
    assert torch.equal(pool[far - 1, :, 3], torch.stack([k[0], v[0]])) and torch.equal(pool[far - 1, :, 5], torch.stack([k[1], v[1]]))
    move_accepted_rows(pool[None], slots, i32([0, 3]), i32([0, 2, -1]), i32([2]))
    assert torch.equal(pool[far - 1, :, 5], torch.stack([k[2], v[2]])) and torch.equal(pool[1, :, 2], torch.stack([k[2], v[2]]))


@pytest.mark.parametrize("kv,rows,tree,hq,hkv,dtype", [([200000, 3], [5, 2], False, 4, 1, "bf16"), ([131071], [40], True, 4, 1, "f16"),
                                                       ([70000, 70016], [8, 3], True, 2, 1, "fp32")])
def test_long_contexts(kv, rows, tree, hq, hkv, dtype):
    print("[case] long", kv, rows, dtype, flush=True)
    step = make_step(3, kv, rows, tree, hq=hq, hkv=hkv, dtype=dtype)
    on = step.on(DEV)
    got = forward(step, on["csr"], on["pages"], on["q"], on["masks"]).double().cpu().numpy()
    want, bound = attention(step)
    assert (np.abs(got - want) <= bound).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_vocabularies_of_many_parts(dtype):
    """264 parts of 4096: uniforms that draw from the first, the middle and the last of them."""
    vocab, rows = 264 * 4096 - 5, [3, 1, 2, 1]
    gen = torch.Generator(DEV).manual_seed(2)
    target = torch.softmax(torch.randn((7, vocab), generator=gen, device=DEV), 1).to(dtype)
    draft = torch.softmax(torch.randn((7, vocab), generator=gen, device=DEV), 1).to(dtype)
    indptr = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    tokens = np.array([1, vocab - 1, 70, 5, 9, 300000, 2], np.int32)
    for u in (0.0, 0.31, 0.999999):
        uniforms = np.array([u, 0.9, 0.9, 0.5 * u, u, 0.99, 0.75], np.float32)
        for q in (None, draft):
            got = verify_drafts(target, i32(tokens), torch.from_numpy(uniforms).to(DEV), i32(indptr), draft_probs=q)
            want = verdict(target.double().cpu().numpy(), tokens, uniforms, indptr, None, None if q is None else q.double().cpu().numpy())
            for g, w in zip((got.counts, got.path, got.tokens), want):
                assert np.array_equal(g.cpu().numpy(), w), (u, q is None, g.cpu().numpy(), w)


def test_table_rows_longer_than_a_turn():
    rng = np.random.default_rng(1)
    tables = rng.permutation(3 * 9000).reshape(3, 9000).astype(np.int32)
    kv, qo = np.array([8000, 10, 2047]), np.array([700, 600, 2])
    got = build_step_tables(i32(tables), i32(kv), i32(qo), 1, max_tokens=1302, max_pages=11359)
    ends = np.cumsum(kv + qo)
    assert got.kv_page_indptr.tolist() == [0, *ends.tolist()] and got.qo_indptr.tolist() == [0, 700, 1300, 1302]
    assert np.array_equal(got.kv_page_indices.cpu().numpy(), np.concatenate([tables[b, : kv[b] + qo[b]] for b in range(3)]))
    assert np.array_equal(got.slots.cpu().numpy(), np.concatenate([tables[b, kv[b]: kv[b] + qo[b]] for b in range(3)]))
    assert np.array_equal(got.positions.cpu().numpy(), np.concatenate([np.arange(kv[b], kv[b] + qo[b]) for b in range(3)]))


def test_walks_longer_than_a_turn():
    rng = np.random.default_rng(4)
    pool = torch.randn((2, 60, 2, 16, 2, 64), generator=torch.Generator().manual_seed(1)).half().to(DEV)
    slots = rng.permutation(60 * 16)[:900]
    path = np.concatenate([[0], np.sort(rng.choice(np.arange(1, 900), 600, replace=False)), np.full(299, -1)])
    want = pool.clone()
    for j in range(1, 601):
        want[:, slots[j] // 16, :, slots[j] % 16] = pool[:, slots[path[j]] // 16, :, slots[path[j]] % 16]
    move_accepted_rows(pool, torch.from_numpy(slots).to(DEV), i32([0, 900]), i32(path), i32([601]))
    assert torch.equal(pool, want)


def test_two_forwards_at_once():
    """Two streams, each with a workspace of its own, and verifications beside them."""
    steps = [make_step(5, [900, 70, 2000], [6, 3, 5], False), make_step(6, [500, 1200], [40, 33], True)]
    on = [s.on(DEV) for s in steps]
    wrappers = [BatchTreeWithPagedKVCacheWrapper(torch.empty(128 << 20, dtype=torch.uint8, device=DEV)) for _ in steps]
    for w, s, o in zip(wrappers, steps, on):
        w.begin_forward(*o["csr"], s.hq, s.hkv, s.dim, s.page, max_qo_len=int(s.rows.max()), masks=o["masks"])
    want = [w.forward(o["q"], o["pages"]).clone() for w, o in zip(wrappers, on)]
    gen = torch.Generator(DEV).manual_seed(2)
    target = torch.softmax(torch.randn((12, 50000), generator=gen, device=DEV), 1)
    tokens, uniforms, indptr = i32(np.arange(12)), torch.rand(12, generator=gen, device=DEV), i32([0, 5, 12])
    said = verify_drafts(target, tokens, uniforms, indptr)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in steps]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append((wrappers[i].forward(on[i]["q"], on[i]["pages"]), verify_drafts(target, tokens, uniforms, indptr)))
    torch.cuda.synchronize()
    for i in range(2):
        for out, verdict_ in got[i]:
            assert torch.equal(out, want[i])
            assert torch.equal(verdict_.tokens, said.tokens) and torch.equal(verdict_.counts, said.counts)
