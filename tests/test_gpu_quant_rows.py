"""Rows into pages of 8-bit K/V, and moved within them."""
import numpy as np
import pytest
import torch

from draftutil import DTYPES, HALF_STEP, make_step, random_parents
from quantutil import Records, VALUES, append, as_quantised, encode, least_scale, move, quantise, rows, same

MOST = {"bf16": 240 * 2.0 ** 120, "fp32": 240 * 2.0 ** 120, "f16": 61440.0}


def test_codes_by_definition():
    """The table, and rounding, against torch's own type."""
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(codes, VALUES, equal_nan=True)
    x = torch.cat([torch.linspace(-448, 448, 9001), 2.0 ** torch.linspace(-14, 8.8, 5000), torch.from_numpy(VALUES).float().nan_to_num(),
                   torch.tensor([2.0 ** -10, 3 * 2.0 ** -10, 1.0625, 1.1875])])
    want = x.to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(encode(x.double().numpy()), want)
    assert least_scale(448.0) == 1 and least_scale(448.1) == 2 and least_scale(0.0) == 2.0 ** -126 and least_scale(224.0) == 0.5


APPENDS = [
    # name, cached tokens, rows, page, Hq, Hkv, D, dtype
    ("one_row", [0], [1], 16, 32, 8, 128, "bf16"),
    ("one_row_inside", [1777], [1], 16, 32, 8, 128, "bf16"),
    ("page_edges", [14, 15, 16, 17, 31, 0, 32], [1, 1, 1, 1, 2, 16, 17], 16, 32, 8, 128, "f16"),
    ("no_rows_between", [40, 0, 9, 70], [0, 0, 3, 0], 16, 32, 8, 128, "bf16"),
    ("page1", [3, 0], [5, 2], 1, 8, 2, 128, "bf16"),
    ("page12", [100, 11, 12], [40, 1, 13], 12, 28, 4, 64, "f16"),
    ("page64_inside", [61, 10], [70, 200], 64, 8, 1, 128, "fp32"),
    ("page128", [100], [300], 128, 8, 2, 64, "bf16"),
    ("odd_heads", [9, 30], [20, 3], 16, 15, 5, 128, "bf16"),
    ("dim8", [5], [30], 16, 4, 2, 8, "f16"),
    ("dim80", [5, 50], [30, 4], 16, 4, 2, 80, "bf16"),
    ("dim256", [17], [9], 8, 4, 2, 256, "bf16"),
    ("dim256_fp32", [17], [9], 8, 4, 2, 256, "fp32"),
    ("batch_300", [(7 * i) % 90 for i in range(300)], [i % 4 for i in range(300)], 8, 4, 2, 64, "bf16"),
    ("batch_70_pages_of_4", [3 * i for i in range(70)], [1 + i % 9 for i in range(70)], 4, 4, 2, 128, "f16"),
    ("long_chunks", [0, 500], [700, 333], 16, 8, 2, 128, "bf16"),
]


def case_step(case, seed=3):
    name, kv, n, page, hq, hkv, dim, dtype = case
    return make_step(seed, kv, n, False, page, hq, hkv, dim, dtype)


def call(step, records, k, v, q=None, table=None, **kw):
    from deserve_amd.quant_ops import rope_append_quantized

    pages = records.tensor().cuda()
    qo, indptr, indices, last = step.on("cuda")["csr"]
    cuda = lambda t: None if t is None else t.cuda()
    out = rope_append_quantized(cuda(q), k.cuda(), v.cuda(), qo, pages, indices, indptr, last, step.page, cuda(table), **kw)
    return pages, out


@pytest.mark.gpu
@pytest.mark.parametrize("case", APPENDS, ids=lambda c: c[0])
@pytest.mark.parametrize("size", [1.0, 37.0, 0.01])
def test_rows_without_rotation_are_exact(case, size):
    """Codes and scales bit for bit; `size` against what the pages hold already lets scales grow, or not."""
    print("[case] append", case, size, flush=True)
    step = case_step(case)
    records, _ = as_quantised(step, spread=6)
    k, v = rows(1, step, DTYPES[step.dtype], size), rows(2, step, DTYPES[step.dtype], 1 / size)
    pages, out = call(step, records, k, v)
    assert out is None
    want = append(records, step, k.double().numpy(), v.double().numpy(), MOST[step.dtype])
    same(Records.of_tensor(pages, step.page, step.hkv, step.dim), want)
    # padding, and pages that take no rows, stay as they are
    used = sorted({int(p) for b in range(len(step.kv)) for p in step.request(b)[2][int(step.kv[b]) // step.page:]})
    rest = np.setdiff1d(np.arange(len(records.codes)), used)
    assert torch.equal(pages[torch.from_numpy(rest)].cpu(), records.tensor()[torch.from_numpy(rest)])
    end = records.codes[0].size + 8 * step.hkv
    assert (pages[:, end:] == 0xA5).all()


@pytest.mark.gpu
@pytest.mark.parametrize("case", APPENDS, ids=lambda c: c[0])
def test_rotated_rows(case):
    """q by the arithmetic of apply_rope; k's codes are within a rounding of the rotation in 64 bits."""
    print("[case] rotated append", case, flush=True)
    step = case_step(case)
    records, _ = as_quantised(step)
    dt, half = DTYPES[step.dtype], step.dim // 2
    k, v, q = rows(1, step, dt, 3.0), rows(2, step, dt), rows(4, step, dt, heads=step.hq)
    at = np.concatenate([np.arange(c, c + n) for c, n in zip(step.kv, step.rows)])
    angle = at[:, None] * 5e5 ** (-np.arange(0, step.dim, 2) / step.dim)
    table = torch.from_numpy(np.concatenate([np.cos(angle), np.sin(angle)], 1)).float()
    pages, out = call(step, records, k, v, q, table)
    cs, sn = (t[:, None].double().numpy() for t in (table[:, :half], table[:, half:]))

    def rotate(x):
        x = x.double().numpy()
        re, im = x[..., 0::2], x[..., 1::2]
        turned = np.stack([re * cs - im * sn, re * sn + im * cs], -1).reshape(x.shape)
        size = np.stack([abs(re * cs) + abs(im * sn), abs(re * sn) + abs(im * cs)], -1).reshape(x.shape)
        return turned, 2.0 ** -23 * size                  # two roundings to 32 bits
    want, off = rotate(q)
    assert (abs(out.double().cpu().numpy() - want) <= off + HALF_STEP[step.dtype] * (abs(want) + off) + 2.0 ** -25).all()
    turned, off = rotate(k)
    got = Records.of_tensor(pages, step.page, step.hkv, step.dim)
    ref = append(records, step, turned, v.double().numpy(), MOST[step.dtype])
    assert np.array_equal(got.scales, ref.scales)
    assert np.array_equal(got.codes[:, 1], ref.codes[:, 1])
    slots = step.slots()
    ids, place = slots // step.page, slots % step.page
    scale = got.scales[ids, 0][..., None]
    value = VALUES[got.codes[ids, 0, :, place]] * scale
    # half a step of the code: 2^-4 of the value, 2^-10 of the scale under 2^-6
    assert (abs(value - turned) <= np.maximum(2.0 ** -4 * abs(turned), 2.0 ** -10 * scale) + 2 * off).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "fp32"])
def test_parts_of_a_projection_and_other_rows(dtype):
    """q, k and v side by side, rows apart; the same bits as from tensors of their own; rows behind the last request."""
    step = make_step(5, [20, 3], [7, 30], False, 16, 8, 2, 64, dtype)
    records, dt = as_quantised(step)[0], DTYPES[dtype]
    total = int(step.qo_indptr[-1])
    gen = torch.Generator().manual_seed(1)
    whole = torch.randn((total + 4, 12, 64), generator=gen).to(dt)
    table = torch.randn((total + 4, 64), generator=gen)
    q, k, v = whole[:, :8], whole[:, 8:10], whole[:, 10:]
    from deserve_amd.quant_ops import rope_append_quantized

    got = []
    for apart in (True, False):
        on = whole.cuda()
        q, k, v = (t if apart else t.contiguous() for t in (on[:, :8], on[:, 8:10], on[:, 10:]))
        pages = records.tensor().cuda()
        qo, indptr, indices, last = step.on("cuda")["csr"]
        out = torch.empty((total + 4, 8, 64), dtype=dt, device="cuda")
        assert rope_append_quantized(q, k, v, qo, pages, indices, indptr, last, 16, table.cuda(), out=out) is out
        got.append((pages.cpu(), out.cpu()))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "fp32"])
def test_values_that_are_none(dtype):
    """Infinities and NaN: in no scale, no number in K, 0 in V; the largest values of a type; rows of zeros; the smallest ones."""
    step = make_step(6, [0, 5, 16, 0, 0], [6, 4, 3, 2, 3], False, 16, 4, 2, 64, dtype)
    records, dt = as_quantised(step)[0], DTYPES[dtype]
    k, v = rows(1, step, dt), rows(2, step, dt)
    k[1, 0, 5], v[3, 1, 60], v[7, 0, 0], k[9, 1, 63] = float("inf"), float("nan"), float("-inf"), float("nan")
    k[10:13, 0] = float("nan")
    k[13, 0, 3], v[13, 0, 3] = torch.finfo(dt).max, torch.finfo(dt).min
    k[14], v[14] = 0, 0
    k[15:], v[15:] = 0, 0
    v[15, 1, 7] = torch.finfo(dt).tiny
    pages, _ = call(step, records, k, v)
    got = Records.of_tensor(pages, 16, 2, 64)
    same(got, append(records, step, k.double().numpy(), v.double().numpy(), MOST[dtype]))
    assert np.isfinite(got.scales).all()
    slots = step.slots()
    none = got.codes[slots // 16, 0, :, slots % 16] & 127 == 127
    assert none.all(2).any(1).nonzero()[0].tolist() == [1, 3, 7, 9, 10, 11, 12] and not (none.any(2) & ~none.all(2)).any()
    assert not (got.codes[slots // 16, 1, :, slots % 16] & 127 == 127).any()
    assert torch.isfinite(torch.from_numpy(got.values()[slots // 16, 1, :, slots % 16]).to(dt)).all()


@pytest.mark.gpu
def test_pages_never_written_and_bad_ones():
    """A block of unwritten memory takes rows; ids that the pool does not have, tables that end early and requests that
    contradict themselves take none."""
    step = make_step(7, [3, 0, 40, 5], [4, 20, 2, 9], False, 16, 4, 2, 64, "bf16")
    from deserve_amd.quant_ops import rope_append_quantized

    k, v = rows(1, step, torch.bfloat16), rows(2, step, torch.bfloat16)
    records = as_quantised(step)[0]
    want = append(records, step, k.double().numpy(), v.double().numpy(), MOST["bf16"])
    for byte in (0x00, 0xFF, 0x7F):
        raw = records.tensor()
        raw[int(step.request(0)[2][0])] = byte
        qo, indptr, indices, last = step.on("cuda")["csr"]
        pages = raw.cuda()
        rope_append_quantized(None, k.cuda(), v.cuda(), qo, pages, indices, indptr, last, 16)
        got = Records.of_tensor(pages, 16, 2, 64)
        at = int(step.request(0)[2][0])
        x = v[:4].double().numpy()
        assert np.array_equal(got.codes[at, 1, :, 3:7], encode(x / got.scales[at, 1, :, None]).transpose(1, 0, 2))
        keep = np.arange(len(got.codes)) != at
        assert np.array_equal(got.codes[keep], want.codes[keep]) and np.array_equal(got.scales[keep], want.scales[keep])
    qo, indptr, indices, last = step.on("cuda")["csr"]
    n = len(records.codes)
    for name, args in {"ids": (qo, torch.where(torch.arange(len(indices), device="cuda") % 2 == 0, n, -1).int(), indptr, last),
                       "no table": (qo, indices[:0], indptr, last), "indptr": (qo, indices, indptr + 100, last),
                       "negative": (qo, indices, indptr - 50, last), "last": (qo, indices, indptr, last * 0),
                       "too many rows": (qo, indices, indptr * 0 + torch.arange(5, device="cuda", dtype=torch.int32), last * 0 + 1),
                       "rows behind": (qo + 1000, indices, indptr, last), "rows in front": (qo - 1000, indices, indptr, last)}.items():
        print("[case] bad tables:", name, flush=True)
        pages = records.tensor().cuda()
        rope_append_quantized(None, k.cuda(), v.cuda(), args[0], pages, args[1], args[2], args[3], 16)
        got = pages.cpu()
        if name == "too many rows":
            continue                                     # (a request of one row has its place there)
        assert torch.equal(got, records.tensor()), name


MOVES = [
    # name, cached tokens, rows, page, Hkv, D, layers, spread
    ("one", [500], [32], 16, 8, 128, 2, 1.0),
    ("scales_apart", [500, 3, 0, 17], [64, 40, 7, 2], 16, 2, 128, 3, 12.0),
    ("pages_of_8", [200, 31], [50, 64], 8, 2, 128, 2, 8.0),
    ("pages_of_1", [9], [40], 1, 2, 64, 1, 8.0),
    ("pages_of_12", [9, 50], [40, 33], 12, 3, 80, 2, 8.0),
    ("dim256", [30], [64], 16, 2, 256, 2, 8.0),
    ("dim8", [30, 1], [64, 9], 16, 2, 8, 2, 8.0),
    ("page64", [60, 63], [64, 64], 64, 1, 64, 1, 8.0),
    ("batch_130", [(5 * i) % 40 for i in range(130)], [i % 20 for i in range(130)], 16, 2, 64, 1, 6.0),
]


def walks(step, seed):
    rng = np.random.default_rng(seed)
    path, counts = np.full(int(step.qo_indptr[-1]), -1, np.int32), []
    for b in range(len(step.kv)):
        lo, hi = int(step.qo_indptr[b]), int(step.qo_indptr[b + 1])
        parents = random_parents(rng, hi - lo, 6)
        walk = [0] if hi > lo else []
        while walk and (next_ := [i for i in range(1, hi - lo) if parents[i] == walk[-1]]):
            walk.append(int(rng.choice(next_)))
        path[lo: lo + len(walk)] = walk
        counts.append(len(walk))
    return path, np.array(counts, np.int32)


@pytest.mark.gpu
@pytest.mark.parametrize("case", MOVES, ids=lambda c: c[0])
def test_moves_by_definition(case):
    print("[case] move", case, flush=True)
    from deserve_amd.quant_ops import move_accepted_quantized_rows

    name, kv, n, page, hkv, dim, layers, spread = case
    step = make_step(8, kv, n, False, page, hkv, hkv, dim, "bf16")
    path, counts = walks(step, 5)
    held = [as_quantised(make_step(20 + i, kv, n, False, page, hkv, hkv, dim, "bf16"), spread, i)[0] for i in range(layers)]
    held[0].codes[:, 0, 0, :, 0] |= 127                  # tokens that an append took for none
    stack = torch.stack([r.tensor() for r in held])
    # layers apart
    pages = torch.full((layers, stack.shape[1] + 2, stack.shape[2]), 0x5A, dtype=torch.uint8, device="cuda")
    pages[:, : stack.shape[1]] = stack.cuda()
    view = pages[:, : stack.shape[1]]
    qo, indptr, indices, last = step.on("cuda")["csr"]
    cuda = lambda a: torch.from_numpy(a).cuda()
    move_accepted_quantized_rows(view, qo, indices, indptr, last, cuda(path), cuda(counts), page, hkv, dim)
    for layer, records in enumerate(held):
        same(Records.of_tensor(view[layer], page, hkv, dim), move(records, step, path, counts))
    assert (pages[:, stack.shape[1]:] == 0x5A).all()
    before = pages.clone()
    for bad in (path * 0, -path, path + 1000, np.full_like(path, 2 ** 31 - 1)):
        move_accepted_quantized_rows(view, qo, indices, indptr, last, cuda(bad), cuda(counts), page, hkv, dim)
    for bad in (counts * 0, counts * 0 + 1, -counts, counts * 0 + 65):
        move_accepted_quantized_rows(view, qo, indices, indptr, last, cuda(path), cuda(bad), page, hkv, dim) if bad.max() <= 1 else None
    move_accepted_quantized_rows(view, qo, indices[:0], indptr, last, cuda(path), cuda(counts), page, hkv, dim)
    move_accepted_quantized_rows(view, qo, indices * 0 - 1, indptr, last, cuda(path), cuda(counts), page, hkv, dim)
    move_accepted_quantized_rows(view, qo, indices * 0 + 10 ** 6, indptr, last, cuda(path), cuda(counts), page, hkv, dim)
    assert torch.equal(pages, before)


def test_quantised_values_are_near():
    x = np.random.default_rng(0).standard_normal((3, 2, 16, 2, 64))
    r = quantise(x)
    off = abs(r.values() - x.transpose(0, 1, 3, 2, 4))
    assert (off <= np.maximum(abs(x.transpose(0, 1, 3, 2, 4)) * 2.0 ** -4, r.scales[..., None, None] * 2.0 ** -10)).all()
