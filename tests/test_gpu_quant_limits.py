"""8-bit pages at the edges of what their calls allow: shapes, lengths, pools, streams, hints, graphs."""
import dataclasses

import numpy as np
import pytest
import torch

from draftutil import attention, make_step
from quantutil import Records, append, as_quantised, move, near, quantise, rows, same
from test_gpu_quant_attention import run

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")

# name, cached, rows, tree, page, q heads, kv heads, dim, type
SHAPES = [
    ("one_kv_head_64", [100, 0, 33], [1, 1, 3], False, 16, 64, 1, 128, "bf16"),
    ("one_kv_head_71", [100, 0, 33], [1, 1, 3], False, 16, 71, 1, 64, "f16"),
    ("one_kv_head_130_fp32", [100, 0], [1, 2], False, 16, 130, 1, 64, "fp32"),
    ("one_kv_head_33", [100, 0, 700], [2, 1, 1], False, 16, 33, 1, 128, "bf16"),
    ("one_kv_head_40_chunk", [100, 0, 700], [1, 50, 1], False, 16, 40, 1, 128, "f16"),
    ("9_rows", [700, 20, 0, 1300], [9, 1, 8, 5], True, 16, 8, 2, 128, "bf16"),
    ("16_rows", [700, 20, 0, 1300], [16, 1, 8, 15], False, 12, 8, 2, 128, "f16"),
    ("12_rows_long", [9000, 3], [12, 9], False, 16, 4, 1, 128, "bf16"),
    ("many_parts_32", [16000], [8], False, 16, 32, 8, 128, "bf16"),
    ("many_parts_20", [9000, 4000], [5, 3], True, 16, 16, 4, 128, "f16"),
    ("many_parts_64_dims_28", [9000], [7], False, 16, 8, 2, 64, "fp32"),
    ("many_parts_64", [6000], [12], False, 16, 32, 8, 128, "f16"),
    ("many_parts_64_dims", [6000, 5000], [9, 40], True, 16, 16, 2, 64, "bf16"),
    ("few_parts_256", [700 + 90 * i for i in range(9)], [40 + i for i in range(9)], True, 16, 16, 2, 128, "bf16"),
    ("kv_heads_600", [37, 5], [1, 2], False, 4, 600, 600, 64, "bf16"),
    ("kv_heads_600_chunk", [9], [70], False, 8, 600, 600, 64, "bf16"),
    ("page_256", [300, 255, 256], [1, 1, 130], False, 256, 8, 2, 128, "bf16"),
    ("page_1000", [1999, 3], [2, 50], False, 1000, 8, 2, 64, "f16"),
    ("64_dims_16_rows", [700, 20, 0], [16, 15, 13], True, 16, 8, 2, 64, "bf16"),
    ("64_dims_16_rows_f16", [700, 20, 0], [16, 15, 13], False, 16, 8, 2, 64, "f16"),
    ("fp32_tiles", [700, 20, 0], [16, 15, 13], True, 16, 8, 2, 64, "fp32"),
    ("fp32_many_short", [3 * i for i in range(90)], [1 + i % 2 for i in range(90)], False, 16, 8, 2, 128, "fp32"),
    ("long_4_waves", [5000], [40], False, 16, 2, 1, 128, "bf16"),
    ("long_8_waves", [9000], [70], False, 12, 2, 1, 128, "f16"),
    ("long_one_row", [70000], [1], False, 16, 2, 1, 128, "bf16"),
    ("long_fp32", [70000], [1], False, 16, 2, 1, 64, "fp32"),
    ("empty_between", [0, 50, 0, 0, 70, 0], [0, 1, 0, 1, 60, 0], False, 16, 8, 2, 128, "bf16"),
]


@pytest.mark.parametrize("case", SHAPES, ids=lambda c: c[0])
def test_shapes(case):
    print("[case] 8-bit shapes", case[0], flush=True)
    step = make_step(21, *case[1:])
    records, values = as_quantised(step, spread=4)
    pages = records.tensor().cuda()
    got = run(step, pages)
    near(got, *attention(values))
    assert torch.equal(got, run(step, pages))


@pytest.mark.parametrize("scale", [0.02, 0.4])
@pytest.mark.parametrize("dim,n", [(128, 2), (128, 60), (128, 14), (80, 2)])
def test_scale_and_hints(dim, n, scale):
    """Another scale; hints that are not kept, which leave out nothing but rows behind max_qo_len."""
    step = make_step(22, [300, 40, 7], [n, 1, n], False, 16, 8, 2, dim, "bf16")
    records, values = as_quantised(step)
    want, bound = attention(values, scale)
    pages = records.tensor().cuda()
    near(run(step, pages, scale), want, bound)
    near(run(step, pages, scale, min_qo_len=10 ** 6), want, bound)
    near(run(step, pages, scale, max_qo_len=10 * n, min_qo_len=n), want, bound)
    most = n - 1
    got, kept = run(step, pages, scale, max_qo_len=most), np.ones(2 * n + 1, bool)
    kept[[n - 1, 2 * n]] = False
    near(got[torch.from_numpy(kept).cuda()], want[kept], bound[kept])
    assert torch.isnan(got[n - 1]).all() and torch.isnan(got[2 * n]).all()


@pytest.mark.parametrize("dtype,dim,n", [("bf16", 128, 2), ("f16", 128, 60), ("bf16", 128, 14), ("bf16", 64, 30), ("fp32", 128, 2), ("bf16", 80, 2)])
def test_rows_of_q_that_are_none(dtype, dim, n):
    """A NaN or an infinity in one head of a row: that head has no number, the others are right."""
    step = make_step(23, [200, 31], [n, 1], False, 16, 8, 2, dim, dtype)
    records, values = as_quantised(step)
    want, bound = attention(values)
    q, hit = step.q.cuda(), np.zeros(want.shape[:2], bool)
    for row, head, value in ((0, 3, "nan"), (1, 4, "inf"), (n, 0, "-inf")):
        q[row, head, row % 7] = float(value)
        hit[row, head] = True
    got = run(step, records.tensor().cuda(), q=q).cpu()
    assert torch.isnan(got[torch.from_numpy(hit)]).all()
    near(got[torch.from_numpy(~hit)], want[~hit], bound[~hit])


@pytest.mark.parametrize("size", [5 << 30, 70 << 30], ids=["5GiB", "70GiB"])
def test_pages_far_behind(size):
    """The last pages of large pools: behind 4 GiB, and behind what 32 bits number in 16 bytes."""
    if torch.cuda.mem_get_info()[0] < size + (4 << 30):
        pytest.skip("not as much memory")
    from deserve_amd.quant_ops import move_accepted_quantized_rows, rope_append_quantized

    steps = [make_step(24, [100, 40, 7], [n, 1, 5], n == 6, 16, 8, 2, 128, "bf16") for n in (1, 6, 60)]
    small = [as_quantised(s)[0] for s in steps]
    record_bytes = small[0].tensor().shape[1]
    pool = torch.empty((size // record_bytes, record_bytes), dtype=torch.uint8, device="cuda")
    for step, records in zip(steps, small):
        values = attention(as_quantised(step)[1])
        near_pages = records.tensor().cuda()
        first = len(pool) - len(near_pages)
        far = pool[first:]
        far.copy_(near_pages)
        on = step.on("cuda")
        qo, indptr, indices, last = on["csr"]
        k, v = rows(1, step, torch.bfloat16), rows(2, step, torch.bfloat16)
        total = int(step.qo_indptr[-1])
        path, counts = torch.zeros(total, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
        path[:3], counts[0] = torch.tensor([0, 2, 4], dtype=torch.int32), 3 if step.rows[0] > 4 else 1
        shifted = dataclasses.replace(step, kv_page_indices=step.kv_page_indices + np.int32(first))
        near(run(shifted, pool), *values)
        for pages, ids in ((near_pages, indices), (pool, indices + first)):
            rope_append_quantized(None, k.cuda(), v.cuda(), qo, pages, ids, indptr, last, 16)
            move_accepted_quantized_rows(pages[None], qo, ids, indptr, last, path.cuda(), counts.cuda(), 16, 2, 128)
        assert torch.equal(far, near_pages)
    del pool, far
    torch.cuda.empty_cache()


def test_steps_on_two_streams():
    """Two wrappers with workspaces of their own, forwards at the same time; and two plans over one workspace, one after the other."""
    from deserve_amd.quant_ops import BatchQuantizedWithPagedKVCacheWrapper

    steps = [make_step(25, [3000, 40], [1, 2], False, 16, 8, 2, 128, "bf16"),
             make_step(26, [2000, 700], [60, 1], False, 16, 8, 2, 128, "bf16")]
    pages = [as_quantised(s)[0].tensor().cuda() for s in steps]
    qs = [s.on("cuda")["q"] for s in steps]
    first = BatchQuantizedWithPagedKVCacheWrapper(torch.empty(128 << 20, dtype=torch.uint8, device="cuda"))
    second = BatchQuantizedWithPagedKVCacheWrapper(torch.empty(128 << 20, dtype=torch.uint8, device="cuda"))
    beside = first.another()
    want = []
    for w, s, p, q in zip((first, beside), steps, pages, qs):
        w.begin_forward(*s.on("cuda")["csr"], 8, 2, 128, 16, max_qo_len=int(s.rows.max()))
    for i in range(3):
        want = [w.forward(q, p) for w, p, q in zip((first, beside), pages, qs)]
    for one, s, p in zip(want, steps, pages):
        assert torch.equal(one, run(s, p))
    second.begin_forward(*steps[1].on("cuda")["csr"], 8, 2, 128, 16, max_qo_len=60)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for i in range(20):
        for j, w in enumerate((first, second)):
            with torch.cuda.stream(streams[j]):
                got[j].append(w.forward(qs[j], pages[j]))
    torch.cuda.synchronize()
    for j in range(2):
        assert all(torch.equal(x, want[j]) for x in got[j])


def test_no_wrapper_in_a_capture():
    from deserve_amd.quant_ops import BatchQuantizedWithPagedKVCacheWrapper

    workspace, x = torch.empty(1 << 20, dtype=torch.uint8, device="cuda"), torch.zeros(4, device="cuda")
    step = make_step(27, [30], [1], False, 4, 520, 520, 64, "bf16")
    made = BatchQuantizedWithPagedKVCacheWrapper(workspace)
    on = step.on("cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x.add_(1)
        with pytest.raises(RuntimeError, match="capture"):
            BatchQuantizedWithPagedKVCacheWrapper(workspace)
        with pytest.raises(RuntimeError, match="capture"):
            made.begin_forward(*on["csr"], 520, 520, 64, 4, max_qo_len=1)
    graph.replay()
    torch.cuda.synchronize()
    assert (x == 1).all()


def test_nothing_to_do():
    step = make_step(28, [30, 5], [2, 1], False, 16, 8, 2, 128, "bf16")
    pages = as_quantised(step)[0].tensor().cuda()
    from deserve_amd.execution.exec import get_quantized_wrapper
    from deserve_amd.quant_ops import move_accepted_quantized_rows, rope_append_quantized

    on, w = step.on("cuda"), get_quantized_wrapper(DEV)
    qo, indptr, indices, last = on["csr"]
    out = torch.full_like(on["q"], 3.0)
    for csr, most in (((qo, indptr, indices, last), 0), ((qo[:1], indptr[:1], indices, last[:0]), 2), ((qo * 0, indptr, indices, last), 2)):
        w.begin_forward(*csr, 8, 2, 128, 16, max_qo_len=most)
        w.forward(on["q"], pages, out=out)
        assert (out == 3).all()
    assert w.forward(on["q"][:0], pages).shape == (0, 8, 128)
    kept = pages.clone()
    k = rows(1, step, torch.bfloat16).cuda()
    for csr in ((qo[:1], indptr[:1], last[:0]), (qo * 0, indptr, last)):
        rope_append_quantized(None, k, k, csr[0], pages, indices, csr[1], csr[2], 16)
    rope_append_quantized(None, k[:0], k[:0], qo, pages, indices, indptr, last, 16)
    zeros = torch.zeros(3, dtype=torch.int32, device="cuda")
    move_accepted_quantized_rows(pages[None], qo, indices, indptr, last, zeros, zeros[:2], 16, 2, 128)
    move_accepted_quantized_rows(pages[None][:0], qo, indices, indptr, last, zeros, zeros[:2], 16, 2, 128)
    assert torch.equal(pages, kept)


def test_append_attention_and_moves_replayed():
    """A captured step of drafted trees - append, attention, moves in two layers - against the definition and the eager step, replayed
    with other lengths, tables and walks, with eager work in between."""
    from deserve_amd.quant_ops import (BatchQuantizedWithPagedKVCacheWrapper, move_accepted_quantized_rows,
                                       rope_append_quantized)

    n, kvs = [6, 9, 1], ([100, 5, 900], [3, 333, 0], [63, 16, 47])
    steps = [make_step(40 + i, kv, n, True, 16, 8, 2, 128, "bf16") for i, kv in enumerate(kvs)]
    held = [[as_quantised(s, seed=layer)[0] for layer in range(2)] for s in steps]
    walks = [([0, 2, 3, 5], [0, 4, 8], [0]), ([0, 1, 2], [0, 1, 5, 6, 7], [0]), ([0], [0, 8], [0])]
    size, total = max(len(h[0].codes) for h in held), sum(n)
    pages = torch.zeros((2, size, held[0][0].tensor().shape[1]), dtype=torch.uint8, device="cuda")
    csr = [torch.zeros(m, dtype=torch.int32, device="cuda") for m in (4, 4, 100, 3)]
    path, counts = torch.zeros(total, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    masks = torch.zeros(total, dtype=torch.int64, device="cuda")
    q, k, v = (torch.zeros((total, h, 128), dtype=torch.bfloat16, device="cuda") for h in (8, 2, 2))
    out = torch.zeros((2,) + q.shape, dtype=torch.bfloat16, device="cuda")
    w = BatchQuantizedWithPagedKVCacheWrapper(torch.empty(128 << 20, dtype=torch.uint8, device="cuda"))
    w.begin_forward(*csr, 8, 2, 128, 16, max_qo_len=9, masks=masks)

    def step():
        for layer in range(2):
            rope_append_quantized(None, k, v, csr[0], pages[layer], csr[2], csr[1], csr[3], 16)
            w.forward(q, pages[layer], out=out[layer])
        move_accepted_quantized_rows(pages, csr[0], csr[2], csr[1], csr[3], path, counts, 16, 2, 128)

    def load(i):
        on = steps[i].on("cuda")
        for t, a in zip(csr, on["csr"]):
            t[: a.numel()] = a
        masks.copy_(on["masks"])
        for layer in range(2):
            pages[layer, : len(held[i][layer].codes)] = held[i][layer].tensor().cuda()
        for t, seed, h in ((q, 1, 8), (k, 2, 2), (v, 3, 2)):
            t.copy_(rows(seed + 10 * i, steps[i], torch.bfloat16, heads=h).cuda())
        path.fill_(-1)
        for b, walk in enumerate(walks[i]):
            lo = int(steps[i].qo_indptr[b])
            path[lo: lo + len(walk)] = torch.tensor(walk, dtype=torch.int32, device="cuda")
            counts[b] = len(walk)
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
        for layer in range(2):
            x = [rows(s + 10 * i, steps[i], torch.bfloat16).double().numpy() for s in (2, 3)]
            want = move(append(held[i][layer], steps[i], *x, 240 * 2.0 ** 120), steps[i], path.cpu().numpy(), counts.cpu().numpy())
            got = Records.of_tensor(pages[layer, : len(want.codes)], 16, 2, 128)
            used = np.unique(steps[i].kv_page_indices)
            same(Records(got.codes[used], got.scales[used]), Records(want.codes[used], want.scales[used]))
        load(i)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and torch.equal(pages, eager_pages), i


@pytest.mark.parametrize("n", [[3, 20, 1], [700, 1, 400]], ids=["few", "many"])
def test_rows_in_front_of_the_first_request(n):
    """Rows that are no request's, in front: the others go where they went without them, in waves of one row and of several."""
    from deserve_amd.quant_ops import rope_append_quantized

    step = make_step(29, [13, 7, 0], n, False, 16, 8, 8, 64, "bf16")
    k, v = (rows(s, step, torch.bfloat16).cuda() for s in (1, 2))
    qo, indptr, indices, last = step.on("cuda")["csr"]
    got = []
    for front in (0, 5):
        pages = as_quantised(step)[0].tensor().cuda()
        x, y = (torch.cat([t[:front] * float("nan"), t]) for t in (k, v))
        rope_append_quantized(None, x, y, qo + front, pages, indices, indptr, last, 16)
        got.append(pages)
    assert torch.equal(*got)


def test_counters_of_a_captured_step_outlive_a_wider_one():
    """A wrapper that is given more heads than its counters are for, after a capture with fewer."""
    from deserve_amd.quant_ops import BatchQuantizedWithPagedKVCacheWrapper

    step, wide = make_step(31, [3000], [1], False, 16, 8, 2, 128, "bf16"), make_step(32, [30], [1], False, 4, 600, 600, 64, "bf16")
    w = BatchQuantizedWithPagedKVCacheWrapper(torch.empty(128 << 20, dtype=torch.uint8, device="cuda"))
    first, on = w._counters.data_ptr(), wide.on("cuda")
    w.begin_forward(*on["csr"], 600, 600, 64, 4, max_qo_len=1)
    w.forward(on["q"], as_quantised(wide)[0].tensor().cuda())
    w.end_forward()
    assert w._counters.data_ptr() != first and first in [t.data_ptr() for t in w._all_counters]
    near(run(step, as_quantised(step)[0].tensor().cuda()), *attention(as_quantised(step)[1]))


@pytest.mark.parametrize("dtype,dim,n", [("bf16", 128, 3), ("f16", 64, 700), ("fp32", 80, 40)])
def test_q_is_rotated_where_no_row_is_kept(dtype, dim, n):
    """An append without requests, and one into a pool without pages: q comes back rotated all the same."""
    from deserve_amd.quant_ops import PageRecord, rope_append_quantized

    step = make_step(33, [0], [n], False, 16, 8, 2, dim, dtype)
    qo, indptr, indices, last = step.on("cuda")["csr"]
    pages = as_quantised(step)[0].tensor().cuda()
    kept = pages.clone()
    k, q = rows(1, step, step.q.dtype).cuda(), step.q.cuda()
    angle = torch.linspace(0, 3, n * dim // 2).view(n, dim // 2)
    table = torch.cat([angle.cos(), angle.sin()], 1).cuda()
    want = rope_append_quantized(q, k, k, qo, pages.clone(), indices, indptr, last, 16, table)
    assert not torch.equal(want, q)
    nan = lambda: torch.full_like(q, float("nan"))
    none = torch.empty((0, PageRecord(16, 2, dim).page_bytes), dtype=torch.uint8, device="cuda")
    for what, csr, pool in (("no requests", (qo[:1], indices, indptr[:1], last[:0]), pages), ("no rows", (qo * 0, indices, indptr, last), pages),
                            ("no pages", (qo, indices, indptr, last), none)):
        out = nan()
        got = rope_append_quantized(q, k, k, csr[0], pool, *csr[1:], 16, table, out=out)
        assert got is out and torch.equal(got, want), what
    assert torch.equal(pages, kept)
    assert rope_append_quantized(q, k, k, qo, none, indices, indptr, last, 16) is q


def test_counters_of_steps_planned_on_copies():
    """Steps of more kv heads than a wrapper's first counters are for, each planned on a copy, as a stage plans them: counters are
    made once, and all copies count in them."""
    from deserve_amd.quant_ops import BatchQuantizedWithPagedKVCacheWrapper

    step = make_step(34, [30], [1], False, 4, 520, 520, 64, "bf16")
    records, values = as_quantised(step)
    pages, on = records.tensor().cuda(), step.on("cuda")
    w = BatchQuantizedWithPagedKVCacheWrapper(torch.empty(128 << 20, dtype=torch.uint8, device="cuda"))
    used = set()
    for heads in (520, 600, 520, 600, 520):
        copy = w.another()
        wide = make_step(35, [9], [1], False, 4, heads, heads, 64, "bf16") if heads != 520 else step
        copy.begin_forward(*wide.on("cuda")["csr"], heads, heads, 64, 4, max_qo_len=1)
        used.add((heads, copy._step.counters))
        if heads == 520:
            near(copy.forward(on["q"], pages), *attention(values))
    assert len(w._all_counters) == 3 and len({c for h, c in used if h == 600}) == 1, (len(w._all_counters), used)


# name, cached, rows, q heads, kv heads, dim, type
LARGE = [("narrow", 300, 1, 8, 2, 128, "bf16"), ("narrow_cut", 3000, 8, 8, 2, 128, "bf16"), ("narrow_64", 700, 3, 8, 2, 64, "bf16"),
         ("fp32", 300, 2, 8, 2, 128, "fp32"), ("fp32_cut", 2000, 1, 8, 2, 64, "fp32"), ("wide_2", 300, 14, 8, 2, 128, "bf16"),
         ("wide_4", 900, 30, 8, 2, 64, "bf16"), ("wide_8", 500, 100, 8, 2, 128, "bf16"), ("plain", 300, 2, 8, 2, 80, "bf16"),
         ("plain_fp32", 300, 2, 8, 2, 256, "fp32"), ("f16", 300, 1, 8, 2, 128, "f16"), ("f16_wide", 300, 60, 8, 2, 128, "f16")]


@pytest.mark.parametrize("case", LARGE, ids=lambda c: c[0])
def test_the_largest_values_that_sums_hold(case):
    """V as large as 256 * tokens * |v| < 2^128 (f16: its pages' largest) allows, under scores that rise from token to token by
    less than what raises a running maximum, so that weights are as large as they get."""
    print("[case] large V", *case, flush=True)
    name, kv, n, hq, hkv, dim, dtype = case
    step = make_step(36, [kv], [n], False, 16, hq, hkv, dim, dtype)
    _, _, table, length = step.request(0)
    pages = step.pages.double()
    # log2 of a weight rises by 7.5 over the tokens
    at = torch.arange(len(table) * 16).double().view(-1, 16)[:, :, None]
    pages[:, 0] *= 0.01
    pages[torch.from_numpy(table).long(), 0, :, :, 0] = (at * (7.5 / length * np.log(2))).expand(-1, -1, hkv)
    step.q.mul_(0.01)
    step.q[..., 0] = float(dim) ** 0.5
    # (0.9: codes are rounded up by 2^-4 at most)
    most = 61440.0 if dtype == "f16" else 0.9 * 2.0 ** 128 / (256 * length)
    pages[:, 1] *= most / pages[:, 1].abs().max()
    records = quantise(pages.numpy())
    values = dataclasses.replace(step, pages=torch.from_numpy(records.values().transpose(0, 1, 3, 2, 4).copy()))
    assert most * 0.9 < values.pages[:, 1].abs().max() <= most / 0.9
    near(run(step, records.tensor().cuda()), *attention(values))


def test_a_captured_step_after_wider_ones():
    """A captured step of cut items, replayed after the wrapper was given more heads than its first counters are for, with other
    tensors where freed memory would be."""
    from deserve_amd.quant_ops import BatchQuantizedWithPagedKVCacheWrapper

    step, wide = make_step(31, [3000], [1], False, 16, 8, 2, 128, "bf16"), make_step(32, [30], [1], False, 4, 600, 600, 64, "bf16")
    records, values = as_quantised(step)
    pages, on, more = records.tensor().cuda(), step.on("cuda"), wide.on("cuda")
    want, bound = attention(values)
    w = BatchQuantizedWithPagedKVCacheWrapper(torch.empty(128 << 20, dtype=torch.uint8, device="cuda"))
    w.begin_forward(*on["csr"], 8, 2, 128, 16, max_qo_len=1)
    out = torch.empty_like(on["q"])
    w.forward(on["q"], pages, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w.forward(on["q"], pages, out=out)
    w.end_forward()
    w.begin_forward(*more["csr"], 600, 600, 64, 4, max_qo_len=1)
    wide_pages = as_quantised(wide)[0].tensor().cuda()
    others = [torch.full((n,), 3, dtype=torch.int32, device="cuda") for n in (1024, 1024, 1200, 2400)]
    for _ in range(3):
        near(w.forward(more["q"], wide_pages), *attention(as_quantised(wide)[1]))
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        near(out, want, bound)
    assert all((x == 3).all() for x in others)


def test_counters_that_are_set_back():
    """What two forwards at the same time may leave in a wrapper's counters is gone after reset, for its copies, too."""
    from deserve_amd.quant_ops import BatchQuantizedWithPagedKVCacheWrapper

    step = make_step(37, [3000, 40], [1, 2], False, 16, 8, 2, 128, "bf16")
    records, values = as_quantised(step)
    pages, on = records.tensor().cuda(), step.on("cuda")
    w = BatchQuantizedWithPagedKVCacheWrapper(torch.empty(128 << 20, dtype=torch.uint8, device="cuda"))
    copy = w.another()
    copy.begin_forward(*on["csr"], 8, 2, 128, 16, max_qo_len=2)
    w._counters.fill_(1)
    w.reset()
    near(copy.forward(on["q"], pages), *attention(values))
    assert not w._counters.any()


@pytest.mark.parametrize("most", [2 ** 31 - 1, 2 ** 31, 2 ** 40, 2 ** 63 - 1])
@pytest.mark.parametrize("dtype,n", [("bf16", 1), ("bf16", 30), ("fp32", 3)])
def test_hints_without_a_bound(dtype, n, most):
    """max_qo_len and min_qo_len as large as a program has numbers: all rows."""
    step = make_step(38, [70, 40], [n, 2], False, 16, 8, 2, 64, dtype)
    records, values = as_quantised(step)
    pages = records.tensor().cuda()
    near(run(step, pages, max_qo_len=most), *attention(values))
    near(run(step, pages, max_qo_len=most, min_qo_len=most), *attention(values))
