"""The operators of a KV cache held in 8 bits, as a serving stage uses them, one case per kind and size.

A page of a layer is a record of bytes: the codes of K, then of V, by head and token, (2, kv_heads, page, dim) in e4m3, then one
float32 scale for each half and head, a power of two; records begin at multiples of 128 bytes.  A value is code * scale of its block,
the tokens of one page and head.  The kinds of pass:

* ``append``: q and k rotated by their rows' angles; k and v of a step's rows into their pages.  A block's scale is the least
  power of two that its largest value takes to 448 or less, and no less than that of the rows which the block holds already; where it
  grows, those are rounded anew.
* ``attend``: attention of a step's rows over the pages, one row per request (decode), a few (drafted tokens, chains or trees),
  chunks of prompts, or rows and a chunk together.
* ``move``: rows that a verified tree accepted, in all layers, to where the sequence goes on; scales grow as in an append.

A case fixes lengths and trees (``lens`` seeds them); values and the order of the pool's pages come from the seed.
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "fp32": torch.float32}
E4M3 = torch.float8_e4m3fn
MAX_ROWS = 64


def _case(kind, batch, rows_lo, rows_hi, kv_lo, kv_hi, lens, tree=False, dtype="bf16", page=16, q_heads=32, kv_heads=8,
          dim=128, chunk=0, layers=1):
    """batch requests of rows_lo .. rows_hi rows over kv_lo .. kv_hi cached tokens; chunk > 0: rows of the last one."""
    return {"kind": kind, "batch": batch, "rows_lo": rows_lo, "rows_hi": rows_hi, "kv_lo": kv_lo, "kv_hi": kv_hi,
            "lens": lens, "tree": tree, "dtype": dtype, "page": page, "q_heads": q_heads, "kv_heads": kv_heads,
            "dim": dim, "chunk": chunk, "layers": layers}


def listed():
    cases = {
        # One user's decode step: launches count.
        "append_1": _case("append", 1, 1, 1, 1777, 1777, 1),
        # The step of 64 requests with four drafts each, which often begins inside a page.
        "append_64": _case("append", 64, 5, 5, 256, 1024, 2),
        # A large prefill: chunks of 512 tokens in float16, pages of 8 tokens as deployed, a model of 64 heads.
        "append_16_chunks": _case("append", 16, 512, 512, 0, 512, 3, False, "f16", 8, 64),
        # One user's decode step, latency.
        "attend_1": _case("attend", 1, 1, 1, 1777, 1777, 4),
        # The decode step of the framework's benchmark: 64 requests over U[256, 4096].
        "attend_64": _case("attend", 64, 1, 1, 256, 4096, 5),
        # The same with four drafts each, float16, pages of 8 tokens.
        "attend_64_drafts": _case("attend", 64, 5, 5, 256, 4096, 6, False, "f16", 8),
        # Trees of 33 to 64 rows over U[1024, 16384] on a model of 64 heads.
        "attend_16_trees": _case("attend", 16, 33, 64, 1024, 16384, 7, True, q_heads=64),
        # The scheduler's usual step: decode rows and one chunk.
        "attend_75_and_chunk": _case("attend", 76, 1, 1, 256, 2048, 8, chunk=437),
        # The largest: chunks of 512 rows over up to 8192 cached tokens.
        "attend_16_chunks": _case("attend", 16, 512, 512, 0, 8192, 9),
        # Single precision, pages of 12 tokens, 64 dims, a few rows.
        "attend_8_fp32": _case("attend", 8, 3, 12, 300, 700, 10, True, "fp32", 12, 28, 4, 64),
        # A single user's accepted rows in 16 layers.
        "move_1": _case("move", 1, 32, 32, 500, 500, 11, True, layers=16),
        # The same for a batch, in 32 layers.
        "move_64": _case("move", 64, 16, 64, 200, 400, 12, True, page=8, layers=32),
    }
    return [dict(c, name=n) for n, c in cases.items()]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


# No drawn case costs more than the largest listed one.
MOST_BYTES, MOST_FLOPS, MOST_SCORES = 4e8, 5e11, 2.2e9


def draw(rng):
    while True:
        kind, chunk = rng.choice(("append", "append", "attend", "attend", "attend", "move")), 0
        tree, lens = rng.random() < 0.4, rng.randrange(1 << 20)
        rows_lo = _log_int(rng, 1, MAX_ROWS)
        rows_hi = min(MAX_ROWS, rows_lo * rng.randint(1, 4))
        kv_lo = _log_int(rng, 1, 4096)
        kv_hi = min(16384, kv_lo * rng.randint(1, 16))
        q_heads, kv_heads = rng.choice(((32, 8), (64, 8), (32, 32), (28, 4), (8, 1), (40, 8)))
        shape = dict(dtype=rng.choice(("bf16", "bf16", "f16", "fp32")), page=rng.choice((1, 4, 8, 8, 12, 16, 16, 32, 64)),
                     q_heads=q_heads, kv_heads=kv_heads, dim=rng.choice((64, 128, 128)))
        if kind == "append":
            if rng.random() < 0.4:
                rows_lo, rows_hi = rows_hi, min(512, rows_hi * rng.randint(1, 16))
            c = _case(kind, _log_int(rng, 1, 128), rows_lo, rows_hi, min(kv_lo, 512), min(kv_hi, 512), lens, tree, **shape)
        elif kind == "attend":
            batch, which = _log_int(rng, 1, 128), rng.random()
            if which < 0.35:
                rows_lo = rows_hi = 1
                chunk = _log_int(rng, 1, 512) if which < 0.15 else 0
                tree = False
            elif which < 0.55:
                rows_lo, rows_hi, tree = rows_hi, min(700, rows_hi * rng.randint(1, 16)), False
                batch = min(batch, 16)
            c = _case(kind, batch, rows_lo, rows_hi, kv_lo, kv_hi, lens, tree, chunk=chunk, **shape)
        else:
            c = _case(kind, _log_int(rng, 1, 64), max(2, rows_lo), max(2, rows_hi), min(kv_lo, 400), min(kv_hi, 400),
                      lens, True, **dict(shape, dtype="bf16"), layers=rng.choice((1, 16, 32)))
        w, (rows, kv, _) = work(c), _lengths(c)
        padded = max(chunk, c["batch"] * rows_hi) if kind == "attend" else 0
        scores = padded * int((rows + kv).max()) * q_heads
        if w["bytes"] <= MOST_BYTES and w["flops"] <= MOST_FLOPS * (0.01 if c["dtype"] == "fp32" else 1) and scores <= MOST_SCORES:
            return c


def _lengths(case):
    """Rows and cached tokens of every request; for trees the parent of every row (-1: none), else None."""
    rng = np.random.default_rng(case["lens"])
    rows = rng.integers(case["rows_lo"], case["rows_hi"] + 1, case["batch"])
    kv = rng.integers(case["kv_lo"], case["kv_hi"] + 1, case["batch"])
    if case["chunk"]:
        rows[-1] = case["chunk"]
    if not case["tree"]:
        return rows, kv, None
    near = rng.integers(1, 9, int(rows.sum()))
    at = np.concatenate([np.arange(n) for n in rows])
    return rows, kv, np.where(at == 0, -1, np.maximum(at - near, 0)).astype(np.int32)


def _descent(rows, parents):
    """Number of rows that every row sees among its request's own, itself included."""
    if parents is None:
        return np.concatenate([np.arange(1, n + 1) for n in rows])
    depth = np.zeros(len(parents), np.int64)
    first = np.repeat(np.cumsum(rows) - rows, rows)
    for i in range(len(parents)):
        depth[i] = 1 if parents[i] < 0 else depth[first[i] + parents[i]] + 1
    return depth


def _accepted(case):
    """For the moves: (path, counts) of rows that a verification may have accepted, a walk from row 0 down."""
    rows, _, parents = _lengths(case)
    rng = random.Random(case["lens"])
    path, counts, first = np.full(int(rows.sum()), -1, np.int32), [], 0
    for n in rows:
        walk, children = [0], [[] for _ in range(n)]
        for i in range(1, n):
            children[parents[first + i]].append(i)
        while children[walk[-1]]:
            walk.append(rng.choice(children[walk[-1]]))
        path[first: first + len(walk)] = walk
        counts.append(len(walk))
        first += n
    return path, np.array(counts, np.int32)


def _masks(rows, parents):
    """Bit j of a row's word: the row is j or descends from it."""
    masks = np.zeros(len(parents), np.uint64)
    first = np.repeat(np.cumsum(rows) - rows, rows)
    for i in range(len(parents)):
        masks[i] = np.uint64(1) << np.uint64(i - first[i])
        if parents[i] >= 0:
            masks[i] |= masks[first[i] + parents[i]]
    return masks.view(np.int64)


def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _record(case):
    """Bytes of a page's codes and of the page."""
    codes = 2 * case["kv_heads"] * case["page"] * case["dim"]
    return codes, -(-(codes + 8 * case["kv_heads"]) // 128) * 128


def _codes(pages, case):
    """(..., pages, 2, kv_heads, page, dim) e4m3, a view."""
    size = (2, case["kv_heads"], case["page"], case["dim"])
    return pages[..., : _record(case)[0]].view(E4M3).unflatten(-1, size)


def _scales(pages, case):
    """(..., pages, 2, kv_heads) float32, a view."""
    codes = _record(case)[0]
    return pages[..., codes: codes + 8 * case["kv_heads"]].view(torch.float32).unflatten(-1, (2, case["kv_heads"]))


def _needed(most):
    """The least power of two that takes `most` to 448 or less."""
    m, e = torch.frexp(most)
    e = torch.where(most > 0, e - 9 + (m > 0.875).int(), -126).clamp(min=-126)
    return ((e + 127) << 23).view(torch.float32)


def _channels(case, gen):
    """Keys have channels that are larger than others."""
    return torch.exp(0.6 * torch.randn((case["kv_heads"], 1, case["dim"]), generator=gen, device="cuda"))


def _pool(case, lens, gen):
    """Layers of pages that hold keys and values of N(0, 1) - keys times their channels' sizes -, handed out in random order, and the
    CSR arrays of the requests with `lens` tokens each."""
    page = case["page"]
    count = -(-lens // page)
    indptr = np.concatenate([[0], np.cumsum(count)])
    num_pages, (size, stride) = int(indptr[-1]) + 7, _record(case)
    pages = torch.zeros((case["layers"], num_pages, stride), dtype=torch.uint8, device="cuda")
    for layer in pages:
        x = torch.randn((num_pages, 2, case["kv_heads"], page, case["dim"]), generator=gen, device="cuda")
        x[:, 0] *= _channels(case, gen)
        scale = _needed(x.abs().amax((3, 4)))
        _scales(layer, case).copy_(scale)
        _codes(layer, case).copy_((x / scale[..., None, None]).to(E4M3))
    order = torch.randperm(num_pages, generator=gen, device="cuda").to(torch.int32)
    return {"pages": pages, "kv_page_indptr": _dev(indptr.astype(np.int32)),
            "kv_page_indices": order[: int(indptr[-1])].contiguous(),
            "kv_last_page_lens": _dev(((lens - 1) % page + 1).astype(np.int32))}


def prepare(case, seed):
    rows, kv, parents = _lengths(case)
    gen = torch.Generator("cuda").manual_seed(seed)
    total, dtype = int(rows.sum()), DTYPES[case["dtype"]]
    s = {"case": dict(case), "qo_indptr": _dev(np.concatenate([[0], np.cumsum(rows)]).astype(np.int32))}
    s.update(_pool(case, kv + rows, gen))
    randn = lambda *shape: torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
    if case["kind"] == "append":
        # the projection's output: q, k and v heads of a token side by side
        heads, hk = case["q_heads"], case["kv_heads"]
        qkv = randn(total, heads + 2 * hk, case["dim"])
        qkv[:, heads: heads + hk] *= _channels(case, gen)[:, 0]
        qkv = qkv.to(dtype)
        angle = _dev(np.repeat(kv, rows) + _descent(rows, parents) - 1).double()[:, None] * torch.pow(
            5e5, -torch.arange(0, case["dim"], 2, device="cuda", dtype=torch.float64) / case["dim"])
        s.update(q=qkv[:, :heads], k=qkv[:, heads: heads + hk], v=qkv[:, heads + hk:], pages=s["pages"][0],
                 table=torch.cat([angle.cos(), angle.sin()], 1).float())
    elif case["kind"] == "attend":
        s.update(pages=s["pages"][0], q=randn(total, case["q_heads"], case["dim"]).to(dtype),
                 masks=None if parents is None else _dev(_masks(rows, parents)), most_rows=int(rows.max()),
                 fewest_rows=int(rows.min()))
    else:
        path, counts = _accepted(case)
        s.update(path=_dev(path), counts=_dev(counts))
    return s


def run(state):
    return (_own if own else _plain)[state["case"]["kind"]](state)


# ---- the framework's calls


def _own_append(s):
    from deserve_amd.quant_ops import rope_append_quantized

    q = rope_append_quantized(s["q"], s["k"], s["v"], s["qo_indptr"], s["pages"], s["kv_page_indices"], s["kv_page_indptr"],
                              s["kv_last_page_lens"], s["case"]["page"], s["table"])
    return {"q": q, "codes": _codes(s["pages"], s["case"]), "scales": _scales(s["pages"], s["case"])}


def _own_attend(s):
    from deserve_amd.execution.exec import get_quantized_wrapper

    c = s["case"]
    wrapper = get_quantized_wrapper(s["q"].device)
    wrapper.begin_forward(s["qo_indptr"], s["kv_page_indptr"], s["kv_page_indices"], s["kv_last_page_lens"], c["q_heads"],
                          c["kv_heads"], c["dim"], c["page"], max_qo_len=s["most_rows"], min_qo_len=s["fewest_rows"],
                          masks=s["masks"])
    return wrapper.forward(s["q"], s["pages"])


def _own_move(s):
    from deserve_amd.quant_ops import move_accepted_quantized_rows

    c = s["case"]
    move_accepted_quantized_rows(s["pages"], s["qo_indptr"], s["kv_page_indices"], s["kv_page_indptr"], s["kv_last_page_lens"],
                                 s["path"], s["counts"], c["page"], c["kv_heads"], c["dim"])
    return {"codes": _codes(s["pages"], c), "scales": _scales(s["pages"], c)}


_own = {"append": _own_append, "attend": _own_attend, "move": _own_move}


# ---- the plain forms


def _places(s, total):
    """For every new row: page id, place in the page and request; for every request: cached tokens."""
    page, indptr, tables = s["case"]["page"], s["qo_indptr"].long(), s["kv_page_indptr"].long()
    lens = (tables[1:] - tables[:-1] - 1) * page + s["kv_last_page_lens"]
    kv = lens - (indptr[1:] - indptr[:-1])
    rows = torch.arange(total, device=indptr.device)
    req = torch.searchsorted(indptr[1:], rows, right=True)
    at = kv[req] + rows - indptr[req]
    ids = s["kv_page_indices"][tables[req] + torch.div(at, page, rounding_mode="floor")].long()
    return ids, at % page, kv, req


def _plain_append(s):
    def rotate(x):
        x, half = x.float(), x.shape[-1] // 2
        cs, sn = s["table"][:, None, :half], s["table"][:, None, half:]
        re, im = x[..., 0::2], x[..., 1::2]
        return torch.stack([re * cs - im * sn, re * sn + im * cs], -1).flatten(-2)

    c, page = s["case"], s["case"]["page"]
    codes, scales = _codes(s["pages"], c), _scales(s["pages"], c)
    ids, place, kv, _ = _places(s, s["k"].shape[0])
    x = torch.stack([rotate(s["k"]), s["v"].float()], 1)                       # (rows, 2, heads, dim)
    index = ids[:, None, None].expand(-1, 2, c["kv_heads"])
    most = torch.zeros_like(scales).scatter_reduce(0, index, x.abs().amax(3), "amax")
    # the page that a request's rows begin in, with `kept` rows that stay
    kept = kv % page
    first = s["kv_page_indptr"][:-1].long() + torch.div(kv, page, rounding_mode="floor")
    begun = s["kv_page_indices"][first].long()
    old = scales[begun]
    held = torch.zeros_like(scales).index_put((begun,), torch.where(kept[:, None, None] > 0, old, 0.0))
    now = torch.maximum(_needed(most), held)
    stay = torch.arange(page, device=kv.device) < kept[:, None]                   # (batch, page)
    again = codes[begun].float() * (old / now[begun])[..., None, None]
    raw = codes.view(torch.uint8)
    raw[begun] = torch.where(stay[:, None, None, :, None], again.to(E4M3).view(torch.uint8), raw[begun])
    raw[ids, :, :, place] = (x / now[ids][..., None]).to(E4M3).view(torch.uint8)
    touched = torch.zeros(scales.shape[0], dtype=torch.bool, device=kv.device).index_fill(0, ids, True)
    scales.copy_(torch.where(touched[:, None, None], now, scales))
    return {"q": rotate(s["q"]).to(s["q"].dtype), "codes": codes, "scales": scales}


def _plain_attend(s):
    c, last = s["case"], s["case"]["batch"] - 1
    if c["chunk"] == 0 or last == 0:
        return _plain_rows(s, 0, c["batch"], s["most_rows"])
    # (padded to the chunk's rows, the others would be most of the work)
    return torch.cat([_plain_rows(s, 0, last, c["rows_hi"]), _plain_rows(s, last, last + 1, c["chunk"])])


def _plain_rows(s, b0, b1, n):
    """Requests b0 .. b1, of at most n rows."""
    c, dev = s["case"], s["q"].device
    group, hk, dim, page = c["q_heads"] // c["kv_heads"], c["kv_heads"], c["dim"], c["page"]
    rows, kv, _ = _lengths(c)
    total, begin, length = int(rows[b0:b1].sum()), int(rows[:b0].sum()), int((rows + kv)[b0:b1].max())
    q, first = s["q"], s["qo_indptr"][b0:b1, None].long()
    count = s["qo_indptr"][b0 + 1: b1 + 1] - s["qo_indptr"][b0:b1]
    row_of = (first + torch.arange(n, device=dev)).clamp(max=q.shape[0] - 1)
    here = torch.arange(n, device=dev) < count[:, None]
    at = torch.arange(length, device=dev)
    tables = s["kv_page_indptr"]
    kv_lens = (tables[b0 + 1: b1 + 1] - tables[b0:b1] - 1) * page + s["kv_last_page_lens"][b0:b1]
    entry = tables[b0:b1, None] + torch.div(at, page, rounding_mode="floor")
    ids = s["kv_page_indices"][entry.clamp(max=s["kv_page_indices"].shape[0] - 1)].long()
    there = at < kv_lens[:, None]
    new = at - (kv_lens - count)[:, None]                                      # (requests, length): index among the new rows
    if s["masks"] is None:
        sees = new[:, None, :] <= torch.arange(n, device=dev)[None, :, None]
    else:
        sees = (new < 0)[:, None, :] | ((s["masks"][row_of][:, :, None] >> new.clamp(0, 63)[:, None, :]) & 1).bool()
    sees = sees & there[:, None, :]                                            # (requests, n, length)
    raw, scales = _codes(s["pages"], c).view(torch.uint8), _scales(s["pages"], c)
    keys, values = ((raw[ids, i, :, at % page].view(E4M3).float() * scales[ids, i][..., None]).permute(0, 2, 1, 3).contiguous()
                    for i in (0, 1))
    x = q[row_of].float().view(-1, n, hk, group, dim).permute(0, 2, 1, 3, 4).reshape(-1, hk, n * group, dim)
    scores = torch.matmul(x, keys.transpose(2, 3).contiguous()).view(-1, hk, n, group, length) / math.sqrt(dim)
    scores = torch.where(sees[:, None, :, None], scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    weight = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(-1, hk, n * group, length), values).view(-1, hk, n, group, dim)
    out = (out / torch.where(weight == 0, 1.0, weight)).permute(0, 2, 1, 3, 4).reshape(-1, n, hk * group, dim)
    at_row = torch.arange(begin, begin + total, device=dev)
    req = torch.searchsorted(s["qo_indptr"][b0 + 1: b1 + 1].long(), at_row, right=True)
    return out[req, at_row - first[req, 0]].to(q.dtype)


def _plain_move(s):
    c, page = s["case"], s["case"]["page"]
    codes, scales = _codes(s["pages"], c), _scales(s["pages"], c)
    raw = codes.view(torch.uint8)
    ids, place, kv, req = _places(s, s["path"].shape[0])
    rows = torch.arange(ids.shape[0], device=ids.device)
    indptr, path = s["qo_indptr"].long(), s["path"].long()
    j = rows - indptr[req]
    moved = (j >= 1) & (j < s["counts"][req]) & (path > j)
    source = torch.where(moved, indptr[req] + path, rows)
    x = raw[:, ids[source], :, :, place[source]].view(E4M3).float()             # (rows, layers, 2, heads, dim): the indices in front
    x = x * scales[:, ids[source]].transpose(0, 1)[..., None]
    most = torch.where(moved[:, None, None, None], x.abs().amax(4), 0.0)
    index = ids[:, None, None, None].expand_as(most)
    most = torch.zeros_like(scales).transpose(0, 1).scatter_reduce(0, index, most, "amax").transpose(0, 1)
    now = torch.where(most > 0, torch.maximum(scales, _needed(most)), scales)
    # the pages of a request from that of its first new row on; rows of them in front of its length are rounded anew
    tables = s["kv_page_indptr"].long()
    entry = torch.arange(s["kv_page_indices"].shape[0], device=ids.device)
    owner = torch.searchsorted(tables[1:], entry, right=True)
    reach = (entry - tables[owner])[:, None] * page + torch.arange(page, device=ids.device)
    stay = reach < (kv + indptr[1:] - indptr[:-1])[owner, None]                   # (entries, page)
    used = s["kv_page_indices"].long()
    ratio = (scales / now)[:, used]
    again = (codes[:, used].float() * ratio[..., None, None]).to(E4M3).view(torch.uint8)
    grown = (ratio < 1)[..., None, None] & stay[:, None, None, :, None]
    raw[:, used] = torch.where(grown, again, raw[:, used])
    target = now[:, ids].transpose(0, 1)[..., None]
    kept = raw[:, ids, :, :, place]
    raw[:, ids, :, :, place] = torch.where(moved[:, None, None, None, None], (x / target).to(E4M3).view(torch.uint8), kept)
    scales.copy_(now)
    return {"codes": codes, "scales": scales}


_plain = {"append": _plain_append, "attend": _plain_attend, "move": _plain_move}


# ---- the results by definition, request by request, in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "move": _exact_move}[case["kind"]](case, s)


def _least_power(most):
    part, power = torch.frexp(most / 448)                # = part * 2^power, part from [0.5, 1)
    power = torch.where(part == 0.5, power - 1, power).clamp(min=-126)
    power = torch.where(most > 0, power, -126).long()
    return ((power + 1023) << 52).view(torch.float64)


def _exact_append(case, s):
    """Codes as the values before their rounding: x / scale."""
    rows, kv, _ = _lengths(case)
    half, page = case["dim"] // 2, case["page"]
    turn = torch.complex(s["table"][:, :half].double(), s["table"][:, half:].double())[:, None]
    rotate = lambda x: torch.view_as_real(torch.view_as_complex(x.double().reshape(x.shape[:-1] + (half, 2))) * turn).flatten(-2)
    codes, scales = _codes(s["pages"], case).double(), _scales(s["pages"], case).double()
    x = torch.stack([rotate(s["k"]), s["v"].double()], 1)
    table, starts, t = s["kv_page_indices"].tolist(), s["kv_page_indptr"].tolist(), 0
    for b in range(case["batch"]):
        begin, end = int(kv[b]), int(kv[b] + rows[b])
        for p in range(begin // page, (end - 1) // page + 1):
            lo, hi = max(begin, p * page), min(end, (p + 1) * page)
            at, mine = table[starts[b] + p], x[t + lo - begin: t + hi - begin]
            now = _least_power(mine.abs().amax((0, 3)))
            if lo > p * page:
                now = torch.maximum(now, scales[at])
                codes[at, :, :, : lo - p * page] *= (scales[at] / now)[..., None, None]
            codes[at, :, :, lo - p * page: hi - p * page] = (mine / now[None, ..., None]).permute(1, 2, 0, 3)
            scales[at] = now
        t += end - begin
    return {"q": rotate(s["q"]), "codes": codes, "scales": scales}


def _exact_attend(case, s):
    rows, kv, parents = _lengths(case)
    seen = _masks(rows, parents) if parents is not None else None
    group, out, first, begin = case["q_heads"] // case["kv_heads"], [], 0, 0
    for n, cached in zip(rows.tolist(), kv.tolist()):
        length = cached + n
        end = begin + -(-length // case["page"])
        mine = s["pages"][s["kv_page_indices"][begin:end].long()]
        held = _codes(mine, case).double() * _scales(mine, case).double()[..., None, None]
        k, v = (held[:, i].transpose(0, 1).reshape(case["kv_heads"], -1, case["dim"])[:, :length] for i in (0, 1))
        q = s["q"][first: first + n].double().unflatten(1, (-1, group)).permute(1, 2, 0, 3)
        sees = np.ones((n, length), bool)
        if seen is None:
            sees[:, cached:] = np.tril(np.ones((n, n), bool))
        else:
            sees[:, cached:] = (seen[first: first + n, None].view(np.uint64) >> np.arange(n, dtype=np.uint64)) & np.uint64(1)
        score = torch.matmul(q, k.transpose(1, 2).unsqueeze(1).contiguous()) * case["dim"] ** -0.5
        score.masked_fill_(~_dev(sees), -math.inf)
        out.append(torch.matmul(torch.softmax(score, -1), v.unsqueeze(1)).permute(2, 0, 1, 3).flatten(1, 2))
        first, begin = first + n, end
    return torch.cat(out)


def _exact_move(case, s):
    """As _exact_append: codes before their rounding."""
    rows, kv, _ = _lengths(case)
    page, (path, counts) = case["page"], _accepted(case)
    codes, scales = _codes(s["pages"], case).double(), _scales(s["pages"], case).double()
    values = codes * scales[..., None, None]
    table, starts, first = s["kv_page_indices"].tolist(), s["kv_page_indptr"].tolist(), 0
    grew, to, at = scales.clone(), [], []
    for b in range(case["batch"]):
        spot = lambda i: (table[starts[b] + (int(kv[b]) + i) // page], (int(kv[b]) + i) % page)
        pairs = [(spot(j), spot(int(path[first + j]))) for j in range(1, int(counts[b])) if path[first + j] > j]
        to += [p[0] for p in pairs]
        at += [p[1] for p in pairs]
        first += int(rows[b])
    to, at = (torch.tensor(x, dtype=torch.int64).reshape(-1, 2).cuda().unbind(1) for x in (to, at))
    x = values[:, at[0], :, :, at[1]]                                           # (moves, layers, 2, heads, dim)
    for i, p in enumerate(to[0].tolist()):
        most = x[i].abs().amax(3)
        grew[:, p] = torch.maximum(grew[:, p], torch.where(most > 0, _least_power(most), 0.0))
    lens = kv + rows
    for b in range(case["batch"]):
        for p in range(-(-int(lens[b]) // page)):
            of, n = table[starts[b] + p], min(page, int(lens[b]) - p * page)
            codes[:, of, :, :, :n] = values[:, of, :, :, :n] / grew[:, of, ..., None, None]
    codes[:, to[0], :, :, to[1]] = x / grew[:, to[0]].transpose(0, 1)[..., None]
    return {"codes": codes, "scales": grew}


# ---- what a pass cannot do without


def work(case):
    rows, kv, parents = _lengths(case)
    size, total, hk, dim = DTYPES[case["dtype"]].itemsize, int(rows.sum()), case["kv_heads"], case["dim"]
    if case["kind"] == "append":
        blocks = int((-(-(kv + rows) // case["page"]) - kv // case["page"]).sum()) * 2 * hk
        return {"bytes": total * dim * (2 * case["q_heads"] * size + 2 * hk * (size + 1) + 4) + 4 * blocks,
                "flops": total * dim * (3 * (case["q_heads"] + hk) + 4 * hk)}
    if case["kind"] == "attend":
        pages = int((-(-(kv + rows) // case["page"])).sum())
        pairs = int((kv * rows).sum() + _descent(rows, parents).sum())
        return {"bytes": 2 * int((kv + rows).sum()) * hk * dim + 8 * pages * hk + 2 * total * case["q_heads"] * dim * size,
                "flops": 4 * case["q_heads"] * dim * pairs}
    path, counts = _accepted(case)
    first = np.repeat(np.cumsum(rows) - rows, rows)
    moved = int((path > np.arange(total) - first).sum())
    return {"bytes": 4 * moved * case["layers"] * hk * dim + 8 * total, "flops": 4 * moved * case["layers"] * hk * dim}
