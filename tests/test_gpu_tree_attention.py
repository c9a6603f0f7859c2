"""Attention of a step's rows over the paged context and over the rows that they descend from."""
import numpy as np
import pytest
import torch

from draftutil import attention, make_step

CASES = [
    # name, cached tokens, rows, tree, page, Hq, Hkv, D, dtype
    ("one_token", [0], [1], False, 16, 32, 8, 128, "bf16"),
    ("nothing_cached", [0, 0, 0], [5, 64, 1], True, 16, 32, 8, 128, "bf16"),
    ("no_rows_between", [40, 0, 9, 70], [0, 0, 3, 0], False, 16, 32, 8, 128, "f16"),
    ("tile_edges", [14, 15, 16, 30, 31, 32, 33, 62, 63, 64], [1, 2, 1, 2, 1, 1, 3, 2, 1, 5], False, 16, 32, 8, 128, "bf16"),
    ("block_edges", [127, 128, 129, 255, 256, 257, 511], [4, 1, 7, 1, 4, 16, 2], True, 16, 32, 8, 128, "f16"),
    ("column_edges_group4", [50] * 8, [3, 4, 5, 8, 9, 16, 17, 64], True, 16, 32, 8, 128, "bf16"),
    ("column_edges_group7", [33] * 6, [1, 2, 3, 9, 10, 37], True, 8, 28, 4, 128, "bf16"),
    ("group1", [100, 3], [64, 17], True, 16, 8, 8, 128, "f16"),
    ("group32", [70, 200], [5, 64], True, 16, 32, 1, 128, "bf16"),
    ("group40", [70], [9], False, 16, 40, 1, 128, "f16"),
    ("odd_heads", [90, 5], [6, 30], True, 16, 15, 5, 128, "bf16"),
    ("page1", [60, 131], [7, 20], True, 1, 16, 4, 128, "bf16"),
    ("page3", [60, 131], [7, 20], True, 3, 16, 4, 128, "f16"),
    ("page12", [60, 500], [7, 20], False, 12, 16, 4, 128, "bf16"),
    ("page128", [600, 127, 128], [7, 1, 1], True, 128, 16, 4, 128, "bf16"),
    ("dim64", [77, 300], [5, 40], True, 16, 32, 8, 64, "bf16"),
    ("dim64_f16_page4", [1000], [12], False, 4, 12, 4, 64, "f16"),
    ("dim80", [77, 30], [5, 9], True, 16, 8, 2, 80, "bf16"),
    ("dim8", [77], [5], True, 16, 4, 2, 8, "f16"),
    ("dim256", [130, 2], [5, 33], True, 16, 8, 2, 256, "bf16"),
    ("fp32", [77, 300, 0], [5, 40, 1], True, 16, 16, 4, 128, "fp32"),
    ("fp32_dim64", [700], [3], False, 12, 8, 8, 64, "fp32"),
    ("fp32_dim200", [90], [12], True, 16, 4, 4, 200, "fp32"),
    ("long", [3000], [6], False, 16, 8, 2, 128, "bf16"),
    ("long_tree", [2500, 9], [64, 2], True, 16, 16, 2, 128, "f16"),
    ("wide_edges", [0, 31, 32, 33, 95, 96, 127, 128], [17, 33, 64, 20, 31, 32, 5, 18], True, 16, 32, 8, 128, "bf16"),
    ("wide_group8", [70, 1000, 5], [64, 17, 33], True, 16, 64, 8, 128, "f16"),
    ("wide_group7_page3", [70, 500], [30, 64], True, 3, 14, 2, 128, "bf16"),
    ("wide_segments", [2047, 2048, 1023, 1024, 4100], [20, 20, 33, 5, 64], True, 16, 16, 4, 128, "bf16"),
    ("wide_chains", [300, 20], [40, 64], False, 12, 32, 8, 128, "f16"),
    ("wide_two_tiles", [900, 1500, 40, 333], [64, 50, 40, 33], True, 16, 16, 2, 128, "bf16"),
    ("wide_two_tiles_or_one", [900, 1500, 140, 333, 700, 80], [64, 64, 64, 40, 64, 3], True, 16, 16, 1, 128, "f16"),
    ("wide_two_tiles_many", [300 + 37 * i for i in range(11)], [64 - 3 * i for i in range(11)], True, 16, 64, 8, 128, "bf16"),
    ("wide_dim64", [0, 31, 32, 33, 63, 64, 65, 95, 96, 127, 128], [17, 33, 64, 20, 31, 32, 5, 18, 1, 40, 29], True, 16, 32, 8, 64, "bf16"),
    ("wide_dim64_four_waves", [70, 1000, 5, 2047, 2048, 4100], [17, 20, 32, 32, 19, 30], True, 3, 16, 4, 64, "f16"),
    ("wide_dim64_two_tiles", [900, 1500, 40, 333], [64, 50, 40, 33], True, 16, 16, 2, 64, "f16"),
    ("wide_dim64_chains", [300, 20, 2111], [40, 64, 64], False, 12, 32, 8, 64, "bf16"),
    ("many_over_eight_heads", [31 * i for i in range(20)], [1 + i % 6 for i in range(20)], True, 16, 16, 8, 128, "bf16"),
    ("many_short", list(range(70)), [1 + i % 5 for i in range(70)], True, 8, 8, 2, 128, "bf16"),
    ("batch_300", [(7 * i) % 90 for i in range(300)], [i % 4 for i in range(300)], True, 16, 8, 2, 128, "bf16"),
    ("batch_700_fp32", [(5 * i) % 40 for i in range(700)], [(i + 1) % 3 for i in range(700)], False, 8, 2, 1, 64, "fp32"),
    ("batch_300_wide", [(11 * i) % 120 for i in range(300)], [(3 * i) % 25 for i in range(300)], True, 16, 4, 1, 128, "f16"),
    ("batch_530_wide", [(13 * i) % 70 for i in range(530)], [(5 * i) % 41 for i in range(530)], True, 16, 4, 1, 128, "bf16"),
    ("batch_530_wide_two_tiles", [(13 * i) % 70 for i in range(530)], [40 + i % 25 for i in range(530)], False, 16, 8, 1, 64, "bf16"),
    ("many_lengths", [int(x) for x in np.random.default_rng(1).integers(0, 900, 40)], [4] * 40, False, 16, 8, 2, 128, "bf16"),
]


def run(step, on=None, scale=None, max_qo_len=None, masks="own", q=None, out=None):
    from deserve_amd.execution.exec import get_tree_wrapper

    on = on or step.on("cuda")
    w = get_tree_wrapper(torch.device("cuda", 0))
    w.begin_forward(*on["csr"], step.hq, step.hkv, step.dim, step.page,
                    max_qo_len=int(step.rows.max()) if max_qo_len is None else max_qo_len,
                    masks=on["masks"] if isinstance(masks, str) else masks)
    q = on["q"] if q is None else q
    return w.forward(q, on["pages"], scale, out=torch.full_like(q, float("nan")) if out is None else out)


def compare(got, want, bound):
    got = got.double().cpu().numpy()
    assert np.isfinite(got).all()
    off = np.abs(got - want) / bound
    assert off.max() <= 1, (np.unravel_index(off.argmax(), off.shape), off.max())


def case_step(case, seed=11):
    name, kv, rows, tree, page, hq, hkv, dim, dtype = case
    return make_step(seed, kv, rows, tree, page, hq, hkv, dim, dtype)


@pytest.mark.parametrize("case", [c for c in CASES if c[7] == 128 and max(c[1]) < 400], ids=lambda c: c[0])
def test_the_bound_lets_no_row_miss_a_key(case):
    """A row without one of the tokens that it sees (its heaviest) is over its bound somewhere."""
    step = case_step(case)
    want, bound = attention(step)
    for b in range(len(step.kv)):
        lo, hi, table, length = step.request(b)
        if hi == lo or step.sees(b)[-1].sum() < 2:
            continue
        held = step.pages[torch.from_numpy(table).long()].double().numpy()
        k, v = (held[:, i].reshape(-1, step.hkv, step.dim)[:length, 0] for i in (0, 1))
        s = np.where(step.sees(b)[-1], k @ step.q[hi - 1, 0].double().numpy() * step.dim ** -0.5, -np.inf)
        w = np.exp(s - s.max())
        w[w.argmax()] = 0
        assert (np.abs(w @ v / w.sum() - want[hi - 1, 0]) > bound[hi - 1, 0]).any()


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: c[0])
def test_rows_match_the_definition(case):
    print("[case] tree attention", *case, flush=True)
    step = case_step(case)
    on = step.on("cuda")
    compare(run(step, on), *attention(step))
    # what the pages hold behind a sequence is never looked at
    for b in range(len(step.kv)):
        _, _, table, length = step.request(b)
        if length % step.page:
            on["pages"][int(table[-1]), :, length % step.page:] = float("nan")
    got = run(step, on)
    compare(got, *attention(step))
    assert torch.equal(got, run(step, on)), "the same call gives other bits"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim", [("bf16", 128), ("f16", 64), ("fp32", 128), ("bf16", 80)])
def test_rows_that_see_nothing(dtype, dim):
    """Masks of a caller's own: no bit at all, later rows only, all rows."""
    step = make_step(2, [0, 5, 0], [6, 4, 3], True, 16, 16, 4, dim, dtype)
    step.masks = np.array([0, 2, 0, 63, 32, -1, 0, 15, 8, 1, 0, 0, 0], np.int64)
    want, bound = attention(step)
    got = run(step)
    compare(got, want, bound + (want == 0) * 1e-30)
    assert not got[[0, 2, 10, 11, 12]].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim,group", [("bf16", 128, 4), ("f16", 128, 1), ("f16", 128, 6), ("bf16", 128, 8), ("f16", 64, 8), ("bf16", 64, 2), ("fp32", 128, 4), ("fp32", 64, 2), ("bf16", 96, 4)])
def test_infinities_and_nan_in_masked_places(dtype, dim, group):
    """A drafted row whose K and V are no numbers reaches the rows that descend from it and no other."""
    for value in (float("nan"), float("inf"), -float("inf")):
        step = make_step(7, [37, 200, 0], [20, 64, 9], True, 16, 4 * group, 4, dim, dtype)
        want, bound = attention(step)
        on, slots = step.on("cuda"), step.slots()
        broken = {0: [3, 7], 1: [5, 33, 62], 2: [4]}
        hit = np.zeros(len(want), bool)
        for b, rows in broken.items():
            for r in rows:
                at = int(slots[step.qo_indptr[b] + r])
                on["pages"][at // 16, 1, at % 16, :, ::3] = value
                on["pages"][at // 16, 0, at % 16] = float("nan")
                hit[step.qo_indptr[b]: step.qo_indptr[b + 1]] |= step.sees(b)[:, step.kv[b] + r]
        got = run(step, on).double().cpu().numpy()
        off = np.abs(got[~hit] - want[~hit]) / bound[~hit]
        assert off.max() <= 1, (value, off.max())
        assert not np.isfinite(got[hit]).all(2).any()


@pytest.mark.gpu
def test_tokens_apart_scales_and_rows_left_out():
    step = make_step(8, [130, 7, 64], [9, 3, 12], True)
    on = step.on("cuda")
    qkv = torch.randn((24, 48, 128), device="cuda").bfloat16()
    qkv[:, :32] = on["q"]
    for scale in (0.2, 0.0, -0.05):
        compare(run(step, on, scale, q=qkv[:, :32], out=torch.empty_like(on["q"])), *attention(step, scale))
    # a batch padded with rows that belong to nobody, and requests with more rows than max_qo_len
    want, bound = attention(step)
    q = torch.cat([on["q"], torch.full_like(on["q"][:5], float("nan"))])
    masks = torch.cat([on["masks"], on["masks"][:5]])
    out = torch.full_like(q, 7.0)
    run(step, on, q=q, masks=masks, out=out)
    compare(out[:24], want, bound)
    assert (out[24:] == 7).all()
    out.fill_(7.0)
    run(step, on, q=q, masks=masks, max_qo_len=5, out=out)
    left = [5, 6, 7, 8] + list(range(17, 29))
    kept = [i for i in range(24) if i not in left]
    compare(out[kept], want[kept], bound[kept])
    assert (out[left] == 7).all()


@pytest.mark.gpu
def test_chains_longer_than_a_tree():
    for dim, dtype in ((128, "bf16"), (64, "f16"), (128, "fp32")):
        step = make_step(9, [100, 0], [150, 70], False, 16, 16, 4, dim, dtype)
        compare(run(step), *attention(step))
    step = make_step(9, [40, 9], [1100, 3], False, 16, 2, 2)
    compare(run(step), *attention(step))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim,hq", [("bf16", 128, 8), ("bf16", 128, 64), ("fp32", 64, 8), ("f16", 96, 8)])
def test_pages_outside_the_pool_hold_no_tokens(dtype, dim, hq):
    step = make_step(10, [100, 40], [4, 3], True, 16, hq, 2, dim, dtype)
    on = step.on("cuda")
    want_step = make_step(10, [100, 40], [4, 3], True, 16, hq, 2, dim, dtype)
    table = step.kv_page_indices.copy()
    table[[2, 5, 8]] = [-1, step.pages.shape[0], 2 ** 31 - 1]
    on["csr"] = on["csr"][:2] + (torch.from_numpy(table).cuda(),) + on["csr"][3:]
    gone = {0: [2, 5], 1: [8 - int(step.kv_page_indptr[1])]}
    sees = Step_without(want_step, gone)
    compare(run(step, on), *attention(sees))
    # a table that is shorter than its indptr says
    on["csr"] = on["csr"][:2] + (torch.from_numpy(step.kv_page_indices[:8].copy()).cuda(),) + on["csr"][3:]
    compare(run(step, on), *attention(Step_without(want_step, {1: [8 - int(step.kv_page_indptr[1]), 9 - int(step.kv_page_indptr[1])]})))


SHORT = [  # cached tokens, rows, pages that the table has beyond its entries
    ([100], [4], 2 ** 31 - 8), ([100, 9], [4, 3], 3), ([90], [20], 1), ([0], [7], 1), ([33, 40], [2, 30], 2)]


def Step_short(step, beyond):
    """The step whose last request's table claims `beyond` pages more than there are entries."""
    last = len(step.kv) - 1

    class Short(type(step)):
        def claimed(self, b):
            lo, hi, table, length = super().request(b)
            return length + beyond * self.page if b == last else length

        def request(self, b):
            lo, hi, table, length = super().request(b)
            return lo, hi, table, min(self.claimed(b), len(table) * self.page)

        def sees(self, b):
            lo, hi, _, held = self.request(b)
            prior, out = self.claimed(b) - (hi - lo), np.ones((hi - lo, held), bool)
            for i in range(hi - lo):
                for j in range(prior, held):
                    out[i, j] = j - prior <= i if self.masks is None else (int(self.masks[lo + i]) >> (j - prior)) & 1
            return out
    return Short(**vars(step))


def short_tables(dtype, dim, hq, tree):
    for kv, rows, beyond in SHORT:
        step = make_step(12, kv, rows, tree, 16, hq, 2, dim, dtype)
        on = step.on("cuda")
        indptr = step.kv_page_indptr.astype(np.int64)
        indptr[-1] += beyond
        assert indptr[-1] < 2 ** 31
        on["csr"] = (on["csr"][0], torch.from_numpy(indptr.astype(np.int32)).cuda(), *on["csr"][2:])
        print("[case] short table", dtype, dim, hq, tree, kv, rows, beyond, flush=True)
        compare(run(step, on), *attention(Step_short(step, beyond)))
    # a table that begins behind the last entry, or in front of the first, has no pages
    for begin in (len(step.kv_page_indices) + 5, 2 ** 31 - 9, -3):
        on["csr"] = (on["csr"][0], torch.tensor([0, begin, max(begin, 0) + 4], dtype=torch.int32).cuda(), *on["csr"][2:])
        assert not run(step, on)[int(step.qo_indptr[1]):].any(), begin


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim,hq", [("f16", 96, 8), ("fp32", 200, 4), ("bf16", 8, 2)])
@pytest.mark.parametrize("tree", [False, True])
def test_tables_longer_than_their_entries(dtype, dim, hq, tree):
    """Pages that a table promises behind the last entry hold no tokens, however many: those in front of them
    stay cached ones."""
    short_tables(dtype, dim, hq, tree)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim,hq", [("bf16", 128, 8), ("bf16", 128, 16), ("f16", 64, 4), ("f16", 64, 64), ("fp32", 128, 4)])
@pytest.mark.parametrize("tree", [False, True])
def test_tables_longer_than_their_entries_matrix_forms(dtype, dim, hq, tree):
    short_tables(dtype, dim, hq, tree)


def Step_without(step, gone):
    """The step with the given pages of its requests unseen."""
    class Without(type(step)):
        def sees(self, b):
            out = super().sees(b)
            for p in gone.get(b, ()):
                out[:, p * self.page: (p + 1) * self.page] = False
            return out
    return Without(**vars(step))


@pytest.mark.gpu
def test_another_stream_and_replays_with_other_lengths():
    """Captured once, replayed with other lengths, trees and tables in the same arrays; eager work between."""
    from deserve_amd.draft_ops import BatchTreeWithPagedKVCacheWrapper

    steps = [make_step(20 + i, kv, rows, True, 16, 32, 8) for i, (kv, rows) in enumerate(
        [([40, 700, 3, 0], [8, 8, 8, 8]), ([0, 1, 2000, 33], [1, 20, 4, 7]), ([5, 0, 0, 0], [0, 0, 0, 3])])]
    pages = torch.zeros((200, 2, 16, 8, 128), dtype=torch.bfloat16, device="cuda")
    csr = [torch.zeros(n, dtype=torch.int32, device="cuda") for n in (5, 5, 200, 4)]
    masks = torch.zeros(32, dtype=torch.int64, device="cuda")
    q, out = (torch.zeros((32, 32, 128), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    w = BatchTreeWithPagedKVCacheWrapper(torch.empty(128 << 20, dtype=torch.uint8, device="cuda"))

    def load(step):
        on = step.on("cuda")
        for to, t in zip([*csr, masks, q, pages], [*on["csr"], on["masks"], on["q"], on["pages"]]):
            to[: t.shape[0]] = t
        out.fill_(7)

    load(steps[0])
    w.begin_forward(*csr, 32, 8, 128, 16, max_qo_len=20, masks=masks)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        eager = w.forward(q, pages, out=out).clone()
    torch.cuda.current_stream().wait_stream(stream)
    compare(eager[:32], *attention(steps[0]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w.forward(q, pages, out=out)
    for step in (steps[0], steps[1], steps[2], steps[1], steps[0]):
        load(step)
        graph.replay()
        total = int(step.rows.sum())
        compare(out[:total], *attention(step))
        assert (out[total:] == 7).all()
        again = w.forward(q, pages, out=torch.full_like(out, 7))
        assert torch.equal(again, out)
        torch.cuda.synchronize()


# Scores under a maximum: one key in sixteen is ahead of all the others by `bits` powers of two and its V is 0, so that the result is
# the others' alone, as behind a token that a model parks its attention on.
@pytest.mark.gpu
@pytest.mark.parametrize("bits", [14.3, 19.64, 21.9, 27.4])
@pytest.mark.parametrize("dtype,dim,rows,hq", [("f16", 128, 5, 8), ("f16", 128, 40, 8), ("f16", 64, 5, 16), ("f16", 64, 48, 16), ("bf16", 128, 5, 8),
                                               ("bf16", 128, 40, 8), ("fp32", 128, 5, 8), ("f16", 96, 5, 8)])
@pytest.mark.parametrize("size", [1, 4096])
def test_few_keys_far_ahead_of_all_others(dtype, dim, rows, hq, bits, size):
    """The float16 forms hold weights of up to 2^8 to 2^15, so that one that is 2^-22 of a row's largest or more is a normal number,
    and a smaller one off by at most half of float16's smallest step, 2^-25 of 2^8 and so 2^-33 of the largest: the definition's bound and that for every token.
    Results are small here: float16 numbers under 2^-14 lie 2^-24 apart, so that rounding one is off by up to 2^-25, which half a
    step of the value does not hold; with V of some thousands they are normal numbers."""
    print("[case] far ahead", dtype, dim, rows, hq, bits, size, flush=True)
    step = make_step(31, [3000], [rows], False, 16, hq, 2, dim, dtype)
    step.q.zero_()
    step.q[..., 0] = 8
    step.pages[:, 0, :, :, 0] = 0
    step.pages[:, 0, ::16, :, 0] = bits * np.log(2) * dim ** 0.5 / 8
    step.pages[:, 1] = (step.pages[:, 1].abs() + 0.5) * size
    step.pages[:, 1, ::16] = 0
    want, bound = attention(step)
    if dtype == "f16":
        # weights over the largest: 1 for one token in 16, 2^-bits for the others
        _, _, table, length = step.request(0)
        first = np.arange(length) % 16 == 0
        for i in range(rows):
            seen = np.arange(length) <= step.kv[0] + i
            total = (seen & first).sum() + (seen & ~first).sum() * 2.0 ** -(bits + 0.01)
            bound[i] += (seen & ~first).sum() / total * 2.0 ** -33 * float(step.pages[:, 1].max()) + 2.0 ** -25
    compare(run(step), want, bound)


SIDES = [  # name, cached tokens, rows, tree, page, Hq, Hkv, D, dtype: four and eight column tiles (of 256) that walk the same tokens
    ("eight_tiles", [900, 40, 1700], [64, 64, 64], True, 16, 32, 1, 128, "bf16"),
    ("eight_tiles_one_request", [2500], [64], True, 3, 32, 1, 128, "f16"),
    ("eight_tiles_or_seven", [1500, 800, 33], [64, 64, 50], True, 16, 32, 1, 128, "f16"),
    ("eight_tiles_two_heads", [300, 1111], [64, 64], False, 16, 64, 2, 128, "bf16"),
    ("eight_tiles_many", [50 + 7 * i for i in range(36)], [64 - i % 3 for i in range(36)], True, 16, 32, 1, 128, "bf16"),
    ("eight_tiles_dim64", [900, 40, 1700], [64, 64, 64], True, 16, 32, 1, 64, "bf16"),
    ("four_tiles", [900, 40, 1700], [64, 64, 64], True, 16, 16, 1, 128, "f16"),
    ("four_tiles_dim64", [2100, 64], [64, 60], True, 8, 32, 2, 64, "f16"),
]


def side_by_side(step):
    """Column tiles of each request where those of all walk the same tokens, by the launch's rule; else 0."""
    group, shares = step.hq // step.hkv, 256 // step.hkv
    tiles = -(-step.rows * group // 256)
    spans = -(-(step.kv + step.rows) // 32)
    sides = int(tiles.max())
    return sides if shares % (8 * sides) == 0 and 4 * sides * spans.sum() <= 5 * (tiles * spans).sum() else 0


@pytest.mark.gpu
@pytest.mark.parametrize("case", SIDES, ids=lambda c: c[0])
def test_four_and_eight_column_tiles_side_by_side(case):
    print("[case] side by side", *case, flush=True)
    step = case_step(case)
    assert side_by_side(step) == (8 if "eight" in case[0] else 4)
    on = step.on("cuda")
    got = run(step, on)
    compare(got, *attention(step))
    assert torch.equal(got, run(step, on))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim,rows,hq", [("bf16", 128, 40, 16), ("f16", 64, 64, 32), ("f16", 128, 33, 4), ("bf16", 64, 40, 4)])
def test_scales_that_are_not_positive_with_many_columns(dtype, dim, rows, hq):
    """More columns than a wave of the narrow form holds, and a scale under which the wide form's mask would be no mask."""
    step = make_step(14, [130, 700, 0], [rows, 9, rows // 2], True, 16, hq, 2, dim, dtype)
    on = step.on("cuda")
    for scale in (0.0, -0.05, -0.3, 0.05):
        print("[case] scale", dtype, dim, rows, hq, scale, flush=True)
        compare(run(step, on, scale), *attention(step, scale))


@pytest.mark.gpu
@pytest.mark.parametrize("most", [2 ** 31 - 1, 2 ** 31, 2 ** 40, 2 ** 63 - 1])
@pytest.mark.parametrize("dtype,n", [("bf16", 1), ("bf16", 30), ("fp32", 3)])
def test_max_qo_len_without_a_bound(dtype, n, most):
    """As large as a program has numbers: all rows."""
    step = make_step(38, [70, 40], [n, 2], False, 16, 8, 2, 64, dtype)
    compare(run(step, max_qo_len=most), *attention(step))
