"""Attention over pages of 8-bit K/V: out and bounds are those of the attention over the values that the pages stand for."""
import dataclasses

import numpy as np
import pytest
import torch

from draftutil import DTYPES, attention, make_step
from quantutil import append, as_quantised, near, rows
from test_gpu_tree_attention import CASES as TREE_CASES

CASES = TREE_CASES + [
    ("decode_edges", [0, 1, 14, 15, 16, 30, 31, 32, 62, 63, 64, 126, 127, 128, 255, 256], [1] * 16, False, 16, 32, 8, 128, "bf16"),
    ("decode_64", [int(x) for x in np.random.default_rng(3).integers(1, 700, 64)], [1] * 64, False, 16, 32, 8, 128, "f16"),
    ("decode_page8", [300 + 41 * i for i in range(9)], [1] * 9, False, 8, 64, 8, 128, "bf16"),
    ("decode_page4", [300 + 41 * i for i in range(9)], [1] * 9, False, 4, 8, 8, 128, "bf16"),
    ("decode_page48", [100 + 41 * i for i in range(9)], [1] * 9, False, 48, 8, 8, 128, "f16"),
    ("decode_dim64", [300 + 41 * i for i in range(9)], [1] * 9, False, 16, 16, 8, 64, "bf16"),
    ("decode_long", [9000, 3], [1, 1], False, 16, 8, 2, 128, "bf16"),
    ("decode_fp32", [1, 64, 700, 2000], [1] * 4, False, 16, 16, 4, 128, "fp32"),
    ("decode_fp32_page1", [1, 64, 300], [1, 2, 3], False, 1, 16, 4, 64, "fp32"),
    ("rows_and_chunk", [900, 40, 0, 333, 50], [1, 1, 1, 1, 130], False, 16, 32, 8, 128, "bf16"),
    ("rows_and_chunk_f16_page8", [900, 40, 0, 333, 50], [1, 1, 200, 1, 3], False, 8, 16, 4, 128, "f16"),
    ("rows_and_chunk_dim64", [900, 40, 0, 333, 50], [1, 1, 200, 1, 90], False, 16, 16, 4, 64, "bf16"),
    ("chunk_of_300", [0], [300], False, 16, 8, 2, 128, "bf16"),
    ("chunk_of_700_over_100", [100], [700], False, 16, 4, 1, 128, "f16"),
    ("chunks_page12", [0, 100, 37], [257, 130, 65], False, 12, 8, 2, 128, "bf16"),
    ("chunk_of_1500", [20], [1500], False, 16, 2, 1, 64, "bf16"),
    ("chunk_fp32", [30], [100], False, 16, 4, 2, 128, "fp32"),
]


def case_step(case, seed=11):
    name, kv, n, tree, page, hq, hkv, dim, dtype = case
    return make_step(seed, kv, n, tree, page, hq, hkv, dim, dtype)


def run(step, pages, scale=None, max_qo_len=None, min_qo_len=0, q=None, out=None, workspace=None, masks="own"):
    from deserve_amd.execution.exec import get_quantized_wrapper
    from deserve_amd.quant_ops import BatchQuantizedWithPagedKVCacheWrapper

    on = step.on("cuda")
    w = get_quantized_wrapper(torch.device("cuda", 0)) if workspace is None else BatchQuantizedWithPagedKVCacheWrapper(workspace)
    w.begin_forward(*on["csr"], step.hq, step.hkv, step.dim, step.page, min_qo_len=min_qo_len,
                    max_qo_len=int(step.rows.max()) if max_qo_len is None else max_qo_len, masks=on["masks"] if isinstance(masks, str) else masks)
    q = on["q"] if q is None else q
    return w.forward(q, pages, scale, out=torch.full_like(q, float("nan")) if out is None else out)


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: c[0])
def test_rows_match_the_definition(case):
    print("[case] attention over 8 bits", *case, flush=True)
    step = case_step(case)
    records, values = as_quantised(step, spread=4)
    want, bound = attention(values)
    pages = records.tensor().cuda()
    near(run(step, pages), want, bound)
    # what the pages hold behind a sequence is never looked at
    for b in range(len(step.kv)):
        _, _, table, length = step.request(b)
        if length % step.page:
            records.codes[int(table[-1]), :, :, length % step.page:] = 0x7F
    pages = records.tensor().cuda()
    got = run(step, pages)
    near(got, want, bound)
    assert torch.equal(got, run(step, pages, min_qo_len=int(step.rows.min()))), "the hint changes bits"
    assert torch.equal(got, run(step, pages)), "the same call gives other bits"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim,n", [("bf16", 128, 6), ("f16", 64, 6), ("fp32", 128, 6), ("bf16", 80, 6), ("bf16", 128, 60), ("f16", 128, 60)])
def test_rows_that_see_nothing(dtype, dim, n):
    """Masks of a caller's own: no bit at all, later rows only, all rows."""
    step = make_step(2, [0, 5, 0], [n, 4, 3], True, 16, 16, 4, dim, dtype)
    step.masks[:] = 0
    step.masks[1], step.masks[2], step.masks[n], step.masks[n + 3] = 0b110000, -1, 0b1000, 0
    records, values = as_quantised(step)
    got = run(step, records.tensor().cuda())
    near(got, *attention(values))
    assert (got[0] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("dtype,dim,most", [("bf16", 128, 9), ("f16", 128, 60), ("bf16", 64, 40), ("fp32", 128, 9), ("bf16", 80, 9), ("f16", 64, 12)])
def test_tokens_that_are_none_reach_who_sees_them(dtype, dim, most, tree):
    """Appended NaN and infinities: rows that see the token get no number in its heads, the others are as without it."""
    step = make_step(4, [30, 0, 77], [most, 5, most - 2], tree, 16, 8, 2, dim, dtype)
    records, _ = as_quantised(step)
    k, v = rows(1, step, DTYPES[dtype]), rows(2, step, DTYPES[dtype])
    k[2, 0, 1], v[4, 1, dim - 1], v[most + 5, 0, 3] = float("nan"), float("inf"), float("nan")
    lim = 61440.0 if dtype == "f16" else 240 * 2.0 ** 120
    new = append(records, step, k.double().numpy(), v.double().numpy(), lim)
    got = run(step, new.tensor().cuda()).double().cpu().numpy()
    clean = new.copy()
    clean.codes[new.codes & 127 == 127] = 0
    values = dataclasses.replace(step, pages=torch.from_numpy(clean.values().transpose(0, 1, 3, 2, 4).copy()))
    want, bound = attention(values)
    hit = np.zeros(got.shape, bool)
    for token, head in ((2, 0), (4, 1), (most + 5, 0)):
        for b in range(3):
            lo, hi, _, _ = step.request(b)
            if lo <= token < hi:
                hit[lo:hi, head * 4: head * 4 + 4] |= step.sees(b)[:, int(step.kv[b]) + token - lo][:, None, None]
    assert np.isnan(got[hit]).all()
    assert hit.any() and (~hit).any()
    near(torch.from_numpy(got[~hit]), want[~hit], bound[~hit])


@pytest.mark.gpu
def test_heaviest_on_few_keys():
    """Scores that lie far apart, in every order, with values of very different size in their pages: the running maximum moves often."""
    for dtype in ("bf16", "f16", "fp32"):
        for dim, n in ((128, 3), (64, 3), (128, 50), (64, 50)):
            step = make_step(9, [700, 90], [n, 1], False, 16, 8, 2, dim, dtype)
            step.q.mul_(6 if dtype == "f16" else 9)
            records, values = as_quantised(step, spread=8 if dtype == "f16" else 24)
            near(run(step, records.tensor().cuda()), *attention(values))


@pytest.mark.gpu
@pytest.mark.parametrize("dim,n", [(128, 1), (64, 5), (128, 40), (80, 2)])
def test_tables_that_promise_too_much(dim, n):
    """Entries behind the last, ids outside of the pool, lengths that contradict themselves: no token there, no fault."""
    step = make_step(12, [100, 40, 7], [n, n, n], False, 16, 8, 2, dim, "bf16")
    from deserve_amd.execution.exec import get_quantized_wrapper

    records, _ = as_quantised(step)
    pages = records.tensor().cuda()
    on = step.on("cuda")
    qo, indptr, indices, last = on["csr"]
    ones = torch.ones_like(last)
    for name, csr in {"no entries": (qo, indptr, indices[:0], last), "few entries": (qo, indptr, indices[:3], last),
                      "ids": (qo, indptr, indices + 10 ** 6, last), "negative ids": (qo, indptr, -1 - indices, last),
                      "tables in front": (qo, indptr - 5, indices, last), "tables behind": (qo, indptr + 10 ** 6, indices, last),
                      "last": (qo, indptr, indices, 1000 * ones), "last negative": (qo, indptr, indices, -1000 * ones),
                      "rows behind": (qo + 10 ** 6, indptr, indices, last), "rows in front": (qo - 10 ** 6, indptr, indices, last),
                      "more rows than tokens": (qo, indptr * 0, indices, last)}.items():
        print("[case] bad tables:", name, dim, n, flush=True)
        w = get_quantized_wrapper(torch.device("cuda", 0))
        w.begin_forward(*csr, 8, 2, dim, 16, max_qo_len=n)
        out = torch.full_like(on["q"], 7.0)
        w.forward(on["q"], pages, out=out)
        got = out.cpu()
        if name in ("rows behind", "rows in front"):
            assert (got == 7).all(), name
        elif name in ("no entries", "ids", "negative ids", "more rows than tokens"):
            assert (got == 0).all(), name


@pytest.mark.gpu
def test_rows_behind_stay_and_strides():
    step = make_step(13, [100, 40], [5, 2], False, 16, 8, 2, 128, "bf16")
    records, values = as_quantised(step)
    want, bound = attention(values)
    wide = torch.full((9, 24, 128), float("nan"), dtype=torch.bfloat16, device="cuda")
    wide[:7, 3:11] = step.q.cuda()
    out = torch.full((9, 8, 128), 5.0, dtype=torch.bfloat16, device="cuda")
    got = run(step, records.tensor().cuda(), q=wide[:, 3:11], out=out)
    assert got is out and (out[7:] == 5).all()
    near(out[:7], want, bound)
    fewer = run(step, records.tensor().cuda(), max_qo_len=3)
    near(fewer[:3], want[:3], bound[:3])
    near(fewer[5:], want[5:], bound[5:])
    assert torch.isnan(fewer[3:5]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 30])
def test_replayed_with_other_lengths(n):
    """A captured step of append and attention, replayed with other lengths and tables, with eager work in between."""
    from deserve_amd.quant_ops import BatchQuantizedWithPagedKVCacheWrapper, rope_append_quantized

    steps = [make_step(30 + i, kv, [n, n, 1], False, 16, 8, 2, 128, "bf16") for i, kv in enumerate(([100, 5, 900], [3, 333, 0], [64, 16, 48]))]
    held = [as_quantised(s)[0] for s in steps]
    size = max(len(r.codes) for r in held)
    total = 2 * n + 1
    pages = torch.zeros((size, held[0].tensor().shape[1]), dtype=torch.uint8, device="cuda")
    csr = [torch.zeros(4, dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda"),
           torch.zeros(100, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")]
    q, k, v = (torch.zeros((total, h, 128), dtype=torch.bfloat16, device="cuda") for h in (8, 2, 2))
    out = torch.zeros_like(q)
    w = BatchQuantizedWithPagedKVCacheWrapper(torch.empty(128 << 20, dtype=torch.uint8, device="cuda"))
    w.begin_forward(*csr, 8, 2, 128, 16, max_qo_len=n)

    def step():
        rope_append_quantized(None, k, v, csr[0], pages, csr[2], csr[1], csr[3], 16)
        w.forward(q, pages, out=out)

    def load(i):
        for t, a in zip(csr, steps[i].on("cuda")["csr"]):
            t[: a.numel()] = a
        pages[: len(held[i].codes)] = held[i].tensor().cuda()
        for t, seed, h in ((q, 1, 8), (k, 2, 2), (v, 3, 2)):
            t.copy_(rows(seed + 10 * i, steps[i], torch.bfloat16, heads=h).cuda())
    load(0)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in (1, 0, 2, 2, 1):
        load(i)
        step()
        eager, eager_pages = out.clone(), pages.clone()
        load(i)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and torch.equal(pages, eager_pages), i
