"""Block tables, slot map, positions and masks built on the GPU; rows appended and moved by their slots."""
import numpy as np
import pytest
import torch

from draftutil import DTYPES, ancestors, make_step, random_parents, to_signed

pytestmark = pytest.mark.gpu


def dev(a, dtype=np.int32):
    return torch.from_numpy(np.ascontiguousarray(a, dtype)).cuda()


def expected(tables, rows, kv, qo, page, max_tokens, max_pages, parents, before):
    """The arrays by definition; `before`: what kv_page_indices held."""
    batch, width = len(kv), tables.shape[1]
    out = {"qo_indptr": [0], "kv_page_indptr": [0], "kv_last_page_lens": [], "kv_page_indices": before.copy(),
           "positions": np.zeros(max_tokens, np.int32), "slots": np.full(max_tokens, -1, np.int64),
           "masks": np.zeros(max_tokens, np.int64)}
    room = True
    for b in range(batch):
        k, n, r = int(kv[b]), int(qo[b]), int(rows[b]) if rows is not None else b
        if k < 0 or n < 0 or not 0 <= r < len(tables) or k + n > width * page or (parents is not None and n > 64):
            k = n = 0
        t0, p0, pages = out["qo_indptr"][-1], out["kv_page_indptr"][-1], -(-(k + n) // page)
        room = room and t0 + n <= max_tokens and p0 + pages <= max_pages
        if not room:
            k = n = pages = 0
        out["qo_indptr"].append(t0 + n)
        out["kv_page_indptr"].append(p0 + pages)
        out["kv_last_page_lens"].append((k + n - 1) % page + 1 if k + n else 0)
        out["kv_page_indices"][p0: p0 + pages] = tables[r][:pages] if pages else []
        above = ancestors(parents[t0: t0 + n].tolist()) if parents is not None else None
        for i in range(n):
            page_id = int(tables[r][(k + i) // page])
            out["slots"][t0 + i] = page_id * page + (k + i) % page if page_id >= 0 else -1
            out["positions"][t0 + i] = k + (i if above is None else len(above[i]) - 1)
            out["masks"][t0 + i] = 0 if above is None else to_signed(sum(1 << a for a in above[i]))
    return {k: np.asarray(v) for k, v in out.items()}


def check(tables, kv, qo, page, max_tokens, max_pages, rows=None, parents=None, strided=False):
    from deserve_amd.draft_ops import StepTables, build_step_tables

    want = expected(tables, rows, kv, qo, page, max_tokens, max_pages, parents, np.full(max_pages, -7, np.int32))
    out = StepTables.empty(len(kv), max_tokens, max_pages, torch.device("cuda", 0), parents is not None)
    for t in (*out.csr, out.positions, out.slots, out.masks):
        if t is not None:
            t.fill_(-7)
    on = dev(tables)
    if strided:
        on = torch.cat([on, on - 1], 1)[:, : tables.shape[1]]
    got = build_step_tables(on, dev(kv), dev(qo), page, max_tokens=max_tokens, max_pages=max_pages,
                            rows=None if rows is None else dev(rows), parents=None if parents is None else dev(parents), out=out)
    for name, w in want.items():
        if name == "masks" and parents is None:
            assert got.masks is None
            continue
        g = getattr(got, name).cpu().numpy()
        assert g.shape == w.shape and np.array_equal(g, w), (name, np.flatnonzero(g != w)[:5])
    return got


@pytest.mark.parametrize("page", [1, 3, 16, 128])
@pytest.mark.parametrize("batch", [1, 2, 63, 256, 257, 700])
@pytest.mark.parametrize("tree", [False, True])
def test_tables_of_many_batches(page, batch, tree):
    rng = np.random.default_rng(batch * 10 + page)
    kv, qo = rng.integers(0, 300, batch), rng.integers(0, 65, batch)
    kv[rng.random(batch) < 0.2] = 0
    qo[rng.random(batch) < 0.2] = 0
    width = int((kv + qo).max() // page + 2)
    tables = rng.integers(0, 1 << 30, (batch + 5, width)).astype(np.int32) // 64
    parents = np.concatenate([random_parents(rng, int(n), 64) for n in qo]) if tree else None
    rows = rng.permutation(batch + 5)[:batch]
    total, pages = int(qo.sum()), int((-(-(kv + qo) // page)).sum())
    check(tables, kv, qo, page, total + 9, pages + 4, rows, parents, strided=batch % 2 == 1)
    check(tables, kv, qo, page, total, pages, None, parents)


def test_tables_of_nothing():
    check(np.zeros((0, 0), np.int32), [], [], 16, 5, 3)
    check(np.zeros((2, 4), np.int32), [0, 0], [0, 0], 16, 0, 0)
    check(np.zeros((2, 4), np.int32), [0, 0], [0, 0], 16, 4, 4, parents=np.zeros(0, np.int32))
    check(np.arange(8, dtype=np.int32).reshape(2, 4), [64, 3], [0, 1], 16, 4, 6)      # a table row filled to its end


def test_requests_that_contradict_themselves_get_nothing():
    tables = np.arange(24, dtype=np.int32).reshape(6, 4)
    tables[3, 1] = -1                                          # a page not handed out yet: no slot
    kv, qo = [5, -1, 60, 17, 3, 2 ** 31 - 1, 7, 9], [3, 2, 5, 4, -2, 2 ** 31 - 1, 1, 2]
    check(tables, kv, qo, 16, 40, 40, rows=[0, 1, 2, 3, 4, 5, 6, -1])
    parents = np.array([-1, 0, 5, -1, 3, 1, 1] + [0] * 70, np.int32)
    check(np.arange(24, dtype=np.int32).reshape(3, 8), [5, 0, 17], [3, 65, 4], 16, 100, 40, parents=parents)


@pytest.mark.parametrize("max_tokens,max_pages", [(0, 40), (7, 40), (8, 40), (40, 3), (40, 4), (11, 5), (40, 0)])
def test_requests_that_do_not_fit_get_nothing(max_tokens, max_pages):
    tables = np.arange(32, dtype=np.int32).reshape(8, 4)
    check(tables, [5, 17, 0, 40, 0, 1], [3, 5, 0, 4, 0, 2], 16, max_tokens, max_pages)
    rng = np.random.default_rng(3)
    kv, qo = rng.integers(0, 50, 600), rng.integers(0, 9, 600)
    check(rng.integers(0, 99, (600, 4)).astype(np.int32), kv, qo, 16, max_tokens * 60, max_pages * 60)


def test_parents_that_are_none_and_short_parents():
    tables = np.arange(16, dtype=np.int32).reshape(2, 8)
    parents = np.array([-1, -5, 1, 9, 3, 2, -1, 6, 7, 100, 0], np.int32)      # own index, later ones, negative ones
    got = check(tables, [10, 3], [6, 5], 16, 11, 10, parents=parents)
    assert got.masks[:6].tolist() == [1, 2, 6, 8, 24, 38]
    from deserve_amd.draft_ops import build_step_tables

    t = build_step_tables(dev(tables), dev([0]), dev([4]), 16, max_tokens=4, max_pages=1, parents=dev([-1, 0]))
    assert t.masks.tolist() == [1, 3, 4, 8] and t.positions.tolist() == [0, 1, 0, 0]


SHAPES = [  # rows, page, Hq, Hkv, D, dtype
    (1, 16, 32, 8, 128, "bf16"), (5, 8, 32, 8, 128, "f16"), (70, 3, 28, 4, 128, "bf16"), (9, 1, 8, 1, 64, "f16"),
    (33, 16, 64, 8, 128, "fp32"), (6, 12, 6, 6, 8, "bf16"), (7, 16, 5, 1, 4, "fp32"), (4, 4, 40, 40, 256, "fp32")]


@pytest.mark.parametrize("rows,page,hq,hkv,dim,dtype", SHAPES)
@pytest.mark.parametrize("fused", [False, True])
def test_rows_into_slots(rows, page, hq, hkv, dim, dtype, fused):
    """Chain rows have the bits of rope_append_paged_kv_cache, whatever the tokens' strides."""
    from deserve_amd.draft_ops import rope_append_slots
    from deserve_amd.paged_ops import rope_append_paged_kv_cache, rope_table

    print("[case] slots", rows, page, hq, hkv, dim, dtype, fused, flush=True)
    s = make_step(3, [17] * rows, [1] * rows, page=page, hq=hq, hkv=hkv, dim=dim, dtype=dtype)
    on = s.on("cuda")
    qkv = torch.randn((rows, hq + 2 * hkv, dim), generator=torch.Generator().manual_seed(9)).to(DTYPES[dtype]).cuda()
    q, k, v = qkv.split((hq, hkv, hkv), 1)
    if not fused:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    indptr, positions = on["csr"][0], dev([17] * rows)
    want_pages = on["pages"].clone()
    if dim % 8 == 0:
        want = rope_append_paged_kv_cache(q, k, v, indptr, positions, want_pages, on["csr"][2], on["csr"][1], on["csr"][3],
                                          rope_theta=1e4)
        table = rope_table(indptr, positions, rows, dim, 1e4)
    else:
        angle = torch.arange(rows, device="cuda")[:, None] * 0.3 + torch.arange(dim // 2, device="cuda")
        table = torch.cat([angle.cos(), angle.sin()], 1)
        turn = lambda x: torch.view_as_real(torch.view_as_complex(x.reshape(*x.shape[:-1], -1, 2).contiguous()) *
                                            torch.complex(*table.split(dim // 2, 1))[:, None]).flatten(-2)
        want = turn(q)
        for t, at in enumerate(s.slots()):
            want_pages[at // page, 0, at % page], want_pages[at // page, 1, at % page] = turn(k)[t], v[t]
    pages = on["pages"].clone()
    got = rope_append_slots(q, k, v, dev(s.slots(), np.int64), pages, table)
    if dim % 8 == 0:
        as_bits = torch.int32 if dtype == "fp32" else torch.int16
        assert torch.equal(got.view(as_bits), want.view(as_bits)) and torch.equal(pages.view(as_bits), want_pages.view(as_bits))
    else:
        # two products of values up to 8, each rounded, and their sum
        assert (got - want).abs().max() < 8 * 2 ** -22 and (pages - want_pages).abs().max() < 8 * 2 ** -22


def test_rows_without_a_slot_or_a_rotation():
    from deserve_amd.draft_ops import rope_append_slots

    s = make_step(4, [30, 2], [3, 4])
    pages = s.on("cuda")["pages"]
    before = pages.clone()
    k, v = torch.randn((2, 7, 8, 128), device="cuda").bfloat16()
    slots = s.slots()
    bad = slots.copy()
    bad[[1, 3, 5]] = [-1, pages.shape[0] * 16, -(2 ** 40)]
    q = torch.randn((7, 32, 128), device="cuda").bfloat16()
    assert rope_append_slots(q, k, v, dev(bad, np.int64), pages) is q
    assert rope_append_slots(None, k[:0], v[:0], dev(bad, np.int64), pages) is None
    want = before.clone()
    for t in (0, 2, 4, 6):
        want[slots[t] // 16, 0, slots[t] % 16], want[slots[t] // 16, 1, slots[t] % 16] = k[t], v[t]
    assert torch.equal(pages, want)
    # every row of q is rotated, also one without a slot
    half = torch.rand((7, 64), device="cuda")
    got = rope_append_slots(q, k, v, dev([-1] * 7, np.int64), pages, torch.cat([half.cos(), half.sin()], 1))
    turned = torch.view_as_complex(q.double().view(7, 32, 64, 2)) * torch.polar(torch.ones_like(half), half).to(torch.complex128)[:, None]
    assert torch.equal(pages, want) and (got.double() - torch.view_as_real(turned).flatten(-2)).abs().max() < 8 * 2 ** -8


@pytest.mark.parametrize("layers,page,hkv,dim,dtype", [(1, 16, 8, 128, "bf16"), (16, 8, 8, 128, "f16"), (3, 3, 1, 8, "bf16"),
                                                        (2, 1, 32, 128, "fp32"), (5, 32, 5, 64, "f16")])
def test_accepted_rows_move(layers, page, hkv, dim, dtype):
    from deserve_amd.draft_ops import move_accepted_rows

    rng = np.random.default_rng(layers)
    rows = [64, 1, 0, 17, 40, 2, 64]
    s = make_step(5, [40, 3, 9, 0, 100, 15, 31], rows, tree=True, page=page, hq=hkv, hkv=hkv, dim=dim, dtype=dtype)
    slots, path, counts = s.slots(), np.full(sum(rows), -1, np.int32), []
    for b, n in enumerate(rows):
        walk = [0] + sorted(rng.choice(np.arange(1, n), int(rng.integers(0, n)), replace=False).tolist()) if n else []
        path[s.qo_indptr[b]: s.qo_indptr[b] + len(walk)] = walk
        counts.append(len(walk))
    # the layers of a stage, every second one of a larger pool
    pool = torch.randn((2 * layers, *s.pages.shape), generator=torch.Generator().manual_seed(1)).to(DTYPES[dtype]).cuda()
    pages = pool[::2]
    want = pool.clone()
    for b in range(len(rows)):
        f = s.qo_indptr[b]
        for j in range(1, counts[b]):
            to, at = slots[f + j], slots[f + path[f + j]]
            want[::2, to // page, :, to % page] = pool[::2, at // page, :, at % page]
    move_accepted_rows(pages, dev(slots, np.int64), dev(s.qo_indptr), dev(path), dev(counts))
    assert torch.equal(pool, want)


def test_paths_and_slots_that_are_none_move_nothing():
    from deserve_amd.draft_ops import move_accepted_rows

    pool = torch.randn((2, 4, 2, 16, 8, 128), device="cuda").bfloat16()
    before = pool.clone()
    slots, indptr = dev([0, 1, 2, 3, 64, -1], np.int64), dev([0, 6])
    for path in ([0, 6, -1, 2, 1, 0], [0, 1, 2, 3, 4, 5], [0, 4, 5, -1, -1, -1], [0, 100, 2 ** 31 - 1, 0, 0, 0]):
        move_accepted_rows(pool, slots, indptr, dev(path), dev([6]))
        assert torch.equal(pool, before), path
    move_accepted_rows(pool, slots, indptr, dev([0, 2, 3, -1, -1, -1]), dev([-3]))
    move_accepted_rows(pool, slots, dev([0, 7]), dev([0, 2, 3, -1, -1, -1]), dev([3]))       # more rows than there are
    move_accepted_rows(pool, slots, dev([-2, 3]), dev([0, 2, 3, -1, -1, -1]), dev([3]))
    assert torch.equal(pool, before)
    move_accepted_rows(pool, slots, indptr, dev([0, 2, 3, -1, -1, -1]), dev([3]))
    before[:, 0, :, 1], before[:, 0, :, 2] = before[:, 0, :, 2].clone(), before[:, 0, :, 3].clone()
    assert torch.equal(pool, before)
