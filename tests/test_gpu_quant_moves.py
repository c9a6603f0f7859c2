"""Moves of accepted rows over pages of 8-bit K/V whose blocks have scales far apart, and walks that move nothing."""
import numpy as np
import pytest
import torch

from draftutil import make_step
from quantutil import Records, move, quantise, same

pytestmark = pytest.mark.gpu


def moved(records, step, path, counts, page, hkv, dim):
    from deserve_amd.quant_ops import move_accepted_quantized_rows

    pages = records.tensor()[None].cuda()
    qo, indptr, indices, last = step.on("cuda")["csr"]
    cuda = lambda a: torch.from_numpy(np.asarray(a, np.int32)).cuda()
    move_accepted_quantized_rows(pages, qo, indices, indptr, last, cuda(path), cuda(counts), page, hkv, dim)
    return Records.of_tensor(pages[0], page, hkv, dim)


@pytest.mark.parametrize("size", [900.0, 3e4, 2.0 ** 60, 2.0 ** 120], ids=["900", "3e4", "2^60", "2^120"])
@pytest.mark.parametrize("dim,page", [(128, 16), (64, 8), (80, 16), (8, 4), (256, 16)])
def test_rows_of_zeros_between_scales_far_apart(dim, page, size):
    """Rows that are zero in a head, out of pages whose values there are large, into blocks of zeros, whose scale is the least there
    is: zeros, in K and in V, beside rows that are none."""
    print("[case] rows of zeros", dim, page, size, flush=True)
    step = make_step(3, [page // 2, 0], [4 * page if 4 * page <= 64 else 64, 40], False, page, 3, 3, dim, "bf16")
    values = step.pages.double().numpy()
    _, _, table, length = step.request(0)
    values[table] *= size
    path, counts = np.full(int(step.qo_indptr[-1]), -1, np.int32), [6, 3]
    path[:6] = [0] + list(range(int(step.rows[0]) - 5, int(step.rows[0])))
    path[int(step.rows[0]): int(step.rows[0]) + 3] = [0, 20, 39]
    at = lambda i: (table[(int(step.kv[0]) + i) // page], (int(step.kv[0]) + i) % page)
    for half, head in ((0, 0), (1, 0), (1, 2)):
        for j in range(1, 6):
            values[at(j)[0], half, :, head] = 0                          # the blocks that rows go to
        for i in path[2:6:2]:
            values[at(int(i))[0], half, at(int(i))[1], head] = 0         # two of the rows
    for i in (path[1], path[3], path[5]):                                # the others, in one head: into zeros, too
        values[at(int(i))[0], 1, at(int(i))[1], 2] = 0
    records = quantise(values)
    records.codes[at(int(path[2]))[0], 0, 0, at(int(path[2]))[1]] = 0x7F     # no number in K
    want = move(records, step, path, counts)
    # the reason of the case: a factor from scale to scale that 32 bits do not hold, of a row that stays zero
    far = [(records.scales[at(int(path[j]))[0], 1, 2], want.scales[at(j)[0], 1, 2]) for j in range(1, 6)]
    assert any(a / b >= 2.0 ** 128 for a, b in far), far
    got = moved(records, step, path, counts, page, 3, dim)
    same(got, want)
    v = got.values()[table][:, 1]
    assert np.isfinite(v).all()


def test_rows_of_the_least_values():
    """Values under the normal numbers of 32 bits, code 1 of the least scale: not taken for zeros."""
    step = make_step(4, [8], [40], False, 16, 2, 2, 64, "bf16")
    records = quantise(step.pages.double().numpy() * 2.0 ** -136)
    assert (records.scales == 2.0 ** -126).all() and (records.codes & 127 == 1).any()
    path, counts = np.full(40, -1, np.int32), [4]
    path[:4] = [0, 20, 30, 39]
    want = move(records, step, path, counts)
    assert not np.array_equal(want.codes & 127, records.codes & 127)
    same(moved(records, step, path, counts, 16, 2, 64), want)


@pytest.mark.parametrize("count", [65, 100, 2 ** 31 - 1])
def test_walks_of_more_rows_than_a_tree_has(count):
    """They move nothing, however few rows their request has; the one beside them goes where it should."""
    print("[case] too long walks", count, flush=True)
    step = make_step(5, [13, 7], [40, 20], False, 16, 2, 2, 64, "bf16")
    records = quantise(step.pages.double().numpy())
    path = np.concatenate([np.arange(0, 80, 2)[:40].clip(max=39), np.arange(0, 40, 2)[:20].clip(max=19)]).astype(np.int32)
    counts = [count, 5]
    want = move(records, step, path, counts)
    first = step.request(0)[2]
    assert np.array_equal(want.codes[first], records.codes[first]) and not np.array_equal(want.codes, records.codes)
    same(moved(records, step, path, counts, 16, 2, 64), want)
