"""The operators of a step that verifies drafted tokens, as a serving stage uses them, one case per kind and size.

A request brings ``n`` rows to such a step: row 0 is the last token it was given, whose K/V the cache does not
hold yet, the others are drafted tokens that form a chain or a tree behind it (a row's parent has a smaller
index).  The kinds of pass:

* ``tables``: block tables, slot map, positions and tree masks from the requests' lengths.
* ``append``: q and k rotated by their rows' angles, k and v written to the slots of the map.
* ``attend``: attention of the rows over the paged context and over the rows that they descend from.
* ``verify``: drafted tokens accepted or refused from the target's probabilities and given random
  numbers, and the token behind the accepted ones.
* ``move``: K/V of the accepted rows, in all layers, to the slots where the sequence goes on.

A case fixes lengths and trees (``lens`` seeds them); values and the order of the pool's pages come from the seed.
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "fp32": torch.float32}
MAX_ROWS = 64


def _case(kind, batch, rows_lo, rows_hi, kv_lo, kv_hi, lens, tree, dtype="bf16", page=16, q_heads=32, kv_heads=8,
          dim=128, layers=1, vocab=0, drafts=False):
    """batch requests of rows_lo .. rows_hi rows over kv_lo .. kv_hi cached tokens."""
    return {"kind": kind, "batch": batch, "rows_lo": rows_lo, "rows_hi": rows_hi, "kv_lo": kv_lo, "kv_hi": kv_hi,
            "lens": lens, "tree": tree, "dtype": dtype, "page": page, "q_heads": q_heads, "kv_heads": kv_heads,
            "dim": dim, "layers": layers, "vocab": vocab, "drafts": drafts}


def listed():
    cases = {
        # One user, four drafts: launches count.
        "tables_1": _case("tables", 1, 5, 5, 1777, 1777, 1, False),
        # A large batch of trees over long contexts, pages of 8 tokens as deployed.
        "tables_512_trees": _case("tables", 512, 8, 32, 256, 16384, 2, True, page=8),
        # The usual step of 64 requests with four drafts each.
        "append_64": _case("append", 64, 5, 5, 256, 4096, 3, False),
        # Trees of 64 rows in float16 on a model of 64 heads.
        "append_64_trees": _case("append", 64, 64, 64, 256, 1024, 4, True, "f16", 8, 64),
        # One user's step: 7 MB of K/V, latency.
        "attend_1": _case("attend", 1, 5, 5, 1777, 1777, 5, False),
        # The ordinary step: 64 requests over U[256, 4096], four drafts each.
        "attend_64": _case("attend", 64, 5, 5, 256, 4096, 6, False),
        # The largest: trees of 33 to 64 rows over U[1024, 16384] on a model of 64 heads.
        "attend_16_trees": _case("attend", 16, 33, 64, 1024, 16384, 7, True, q_heads=64),
        # Single precision, pages of 12 tokens, small trees.
        "attend_8_fp32": _case("attend", 8, 3, 12, 300, 700, 8, True, "fp32", 12),
        # Sampling verified against the draft's own distributions.
        "verify_64_drafts": _case("verify", 64, 5, 5, 0, 0, 9, False, "fp32", vocab=128000, drafts=True),
        # Trees of proposed tokens, one user, probabilities in bfloat16.
        "verify_1_tree": _case("verify", 1, 40, 40, 0, 0, 10, True, "bf16", vocab=32003),
        # A single user's accepted rows in 16 layers.
        "move_1": _case("move", 1, 32, 32, 500, 500, 11, True, layers=16),
        # The same for a batch, in 32 layers.
        "move_64": _case("move", 64, 16, 64, 200, 400, 12, True, "f16", 8, layers=32),
    }
    return [dict(c, name=n) for n, c in cases.items()]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


# No drawn case costs more than the largest listed one.
MOST_BYTES, MOST_FLOPS = 6e8, 2.5e11


def draw(rng):
    while True:
        kind = rng.choice(("tables", "append", "attend", "attend", "verify", "move"))
        tree, lens = rng.random() < 0.5, rng.randrange(1 << 20)
        rows_lo = _log_int(rng, 1, MAX_ROWS)
        rows_hi = min(MAX_ROWS, rows_lo * rng.randint(1, 4))
        kv_lo = _log_int(rng, 1, 4096)
        kv_hi = min(16384, kv_lo * rng.randint(1, 16))
        page = rng.choice((1, 4, 8, 8, 12, 16, 16, 32, 64))
        dtype = rng.choice(("bf16", "bf16", "f16", "fp32"))
        q_heads, kv_heads = rng.choice(((32, 8), (64, 8), (32, 32), (28, 4), (8, 1), (40, 8)))
        shape = dict(page=page, dtype=dtype, q_heads=q_heads, kv_heads=kv_heads, dim=rng.choice((64, 128, 128)))
        if kind == "tables":
            c = _case(kind, _log_int(rng, 1, 1024), rows_lo, rows_hi, kv_lo, kv_hi, lens, tree, page=page)
        elif kind == "append":
            c = _case(kind, _log_int(rng, 1, 128), rows_lo, rows_hi, min(kv_lo, 512), min(kv_hi, 512), lens, tree, **shape)
        elif kind == "attend":
            c = _case(kind, _log_int(rng, 1, 128), rows_lo, rows_hi, kv_lo, kv_hi, lens, tree, **shape)
        elif kind == "verify":
            drafts = not tree and rng.random() < 0.7
            c = _case(kind, _log_int(rng, 1, 128), rows_lo, rows_hi, 0, 0, lens, tree, dtype,
                      vocab=_log_int(rng, 100, 160000), drafts=drafts)
            if c["batch"] * rows_hi * c["vocab"] > 64 * 5 * 128000:
                continue
        else:
            c = _case(kind, _log_int(rng, 1, 64), max(2, rows_lo), max(2, rows_hi), min(kv_lo, 400), min(kv_hi, 400),
                      lens, True, dtype if dtype != "fp32" else "bf16", page, layers=rng.choice((1, 16, 32)))
        w = work(c)
        if w["bytes"] <= MOST_BYTES and w["flops"] <= MOST_FLOPS * (0.05 if dtype == "fp32" else 1):
            return c


def _lengths(case):
    """Rows and cached tokens of every request; for trees the parent of every row (-1: none), else None."""
    rng = np.random.default_rng(case["lens"])
    rows = rng.integers(case["rows_lo"], case["rows_hi"] + 1, case["batch"])
    kv = rng.integers(case["kv_lo"], case["kv_hi"] + 1, case["batch"])
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


def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _pool(case, lens, gen, layers=None):
    """A pool whose pages, all N(0, 1), are handed out in random order; the table rows and CSR arrays of the
    requests with `lens` tokens each."""
    page, batch = case["page"], case["batch"]
    pages = -(-lens // page)
    indptr = np.concatenate([[0], np.cumsum(pages)])
    num_pages = int(indptr[-1]) + 7
    order = torch.randperm(num_pages, generator=gen, device="cuda").to(torch.int32)
    width = int(pages.max()) + 1
    at = _dev(indptr[:-1, None] + np.arange(width)[None]).clamp(max=num_pages - 1)
    tables = order[at]
    out = {"page_tables": tables, "kv_page_indices": order[: int(indptr[-1])].contiguous(),
           "kv_page_indptr": _dev(indptr.astype(np.int32)),
           "kv_last_page_lens": _dev(((lens - 1) % page + 1).astype(np.int32))}
    if layers is not None:
        shape = (layers, num_pages, 2, page, case["kv_heads"], case["dim"])
        out["pages"] = torch.randn(shape, generator=gen, device="cuda", dtype=DTYPES[case["dtype"]])
    return out


def _slots(case, rows, kv, tables):
    """Slot of every new row: page * page size + place in the page."""
    req = _dev(np.repeat(np.arange(len(rows)), rows))
    at = _dev(np.concatenate([np.arange(k, k + n) for k, n in zip(kv, rows)]))
    return tables[req, at // case["page"]].long() * case["page"] + at % case["page"]


def _masks(rows, parents):
    """Bit j of a row's word: the row is j or descends from it."""
    masks = np.zeros(len(parents), np.uint64)
    first = np.repeat(np.cumsum(rows) - rows, rows)
    for i in range(len(parents)):
        masks[i] = np.uint64(1) << np.uint64(i - first[i])
        if parents[i] >= 0:
            masks[i] |= masks[first[i] + parents[i]]
    return masks.view(np.int64)


def prepare(case, seed):
    rows, kv, parents = _lengths(case)
    gen = torch.Generator("cuda").manual_seed(seed)
    total, dtype = int(rows.sum()), DTYPES[case["dtype"]]
    randn = lambda *s: torch.randn(s, generator=gen, device="cuda", dtype=torch.float32).to(dtype)
    s = {"case": dict(case), "qo_indptr": _dev(np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)),
         "parents": None if parents is None else _dev(parents)}
    if case["kind"] == "tables":
        s.update(_pool(case, kv + rows, gen), kv_lens=_dev(kv.astype(np.int32)), qo_lens=_dev(rows.astype(np.int32)),
                 rows=torch.randperm(case["batch"], generator=gen, device="cuda").to(torch.int32),
                 max_tokens=total + 3, max_pages=int((-(-(kv + rows) // case["page"])).sum()))
        # request b's pages are in row rows[b] of the tables
        s["page_tables"][s["rows"].long()] = s["page_tables"].clone()
    elif case["kind"] == "append":
        pool = _pool(case, kv + rows, gen, 1)
        # the projection's output: q, k and v heads of a token side by side
        heads, hk = case["q_heads"], case["kv_heads"]
        qkv = randn(total, heads + 2 * hk, case["dim"])
        depth = _descent(rows, parents) - 1
        angle = _dev(np.repeat(kv, rows) + depth).double()[:, None] * torch.pow(
            5e5, -torch.arange(0, case["dim"], 2, device="cuda", dtype=torch.float64) / case["dim"])
        s.update(q=qkv[:, :heads], k=qkv[:, heads: heads + hk], v=qkv[:, heads + hk:], pages=pool["pages"][0],
                 slots=_slots(case, rows, kv, pool["page_tables"]),
                 table=torch.cat([angle.cos(), angle.sin()], 1).float())
    elif case["kind"] == "attend":
        pool = _pool(case, kv + rows, gen, 1)
        s.update(pool, pages=pool["pages"][0], q=randn(total, case["q_heads"], case["dim"]),
                 masks=None if parents is None else _dev(_masks(rows, parents)), max_rows=int(rows.max()))
    elif case["kind"] == "verify":
        s.update(_verify_inputs(case, rows, parents, gen, dtype))
    else:
        pool = _pool(case, kv + rows, gen, case["layers"])
        path, counts = _accepted(case)
        s.update(pages=pool["pages"], slots=_slots(case, rows, kv, pool["page_tables"]), path=_dev(path),
                 counts=_dev(counts))
    return s


def _verify_inputs(case, rows, parents, gen, dtype):
    """A target and a draft model that mostly agree; every drafted token is sampled from the draft at its parent."""
    total, vocab = int(rows.sum()), case["vocab"]
    logits = 4 * torch.randn((total, vocab), generator=gen, device="cuda")
    target = torch.softmax(logits, 1).to(dtype)
    draft = torch.softmax(logits + 0.5 * torch.randn((total, vocab), generator=gen, device="cuda"), 1).to(dtype)
    first = np.repeat(np.cumsum(rows) - rows, rows)
    parent = np.arange(total) - 1 if parents is None else first + parents
    sampled = torch.multinomial(draft.float()[_dev(np.maximum(parent, first))], 1, generator=gen)[:, 0]
    return {"target_probs": target, "draft_probs": draft if case["drafts"] else None,
            "tokens": sampled.to(torch.int32), "uniforms": torch.rand(total, generator=gen, device="cuda")}


def run(state):
    return (_own if own else _plain)[state["case"]["kind"]](state)


# ---- the framework's calls


def _own_tables(s):
    from deserve_amd.draft_ops import build_step_tables

    t = build_step_tables(s["page_tables"], s["kv_lens"], s["qo_lens"], s["case"]["page"], max_tokens=s["max_tokens"],
                          max_pages=s["max_pages"], rows=s["rows"], parents=s["parents"])
    out = {"qo_indptr": t.qo_indptr, "kv_page_indptr": t.kv_page_indptr, "kv_page_indices": t.kv_page_indices,
           "kv_last_page_lens": t.kv_last_page_lens, "positions": t.positions, "slots": t.slots}
    return out if t.masks is None else dict(out, masks=t.masks)


def _own_append(s):
    from deserve_amd.draft_ops import rope_append_slots

    q = rope_append_slots(s["q"], s["k"], s["v"], s["slots"], s["pages"], s["table"])
    return {"q": q, "pages": s["pages"]}


def _own_attend(s):
    from deserve_amd.execution.exec import get_tree_wrapper

    c = s["case"]
    wrapper = get_tree_wrapper(s["q"].device)
    wrapper.begin_forward(s["qo_indptr"], s["kv_page_indptr"], s["kv_page_indices"], s["kv_last_page_lens"],
                          c["q_heads"], c["kv_heads"], c["dim"], c["page"], max_qo_len=s["max_rows"], masks=s["masks"])
    return wrapper.forward(s["q"], s["pages"])


def _own_verify(s):
    from deserve_amd.draft_ops import verify_drafts

    r = verify_drafts(s["target_probs"], s["tokens"], s["uniforms"], s["qo_indptr"], parents=s["parents"],
                      draft_probs=s["draft_probs"])
    return {"counts": r.counts, "path": r.path, "tokens": r.tokens}


def _own_move(s):
    from deserve_amd.draft_ops import move_accepted_rows

    move_accepted_rows(s["pages"], s["slots"], s["qo_indptr"], s["path"], s["counts"])
    return s["pages"]


_own = {"tables": _own_tables, "append": _own_append, "attend": _own_attend, "verify": _own_verify, "move": _own_move}


# ---- the plain forms


def _ancestors(parent, there):
    """(B, n, n): row i is j or descends from it; parent (B, n), -1 for none."""
    n = parent.shape[1]
    up = (parent[:, :, None] == torch.arange(n, device=parent.device)) & there[:, :, None]
    eye = torch.eye(n, device=parent.device)
    return (torch.matrix_power(eye + up.float(), n) > 0) & there[:, :, None]


def _plain_tables(s):
    page, batch, dev = s["case"]["page"], s["case"]["batch"], s["kv_lens"].device
    zero = torch.zeros(1, dtype=torch.int64, device=dev)
    sums = lambda x: torch.cat([zero, x.long().cumsum(0)]).int()
    lens = s["kv_lens"] + s["qo_lens"]
    pages = torch.div(lens + page - 1, page, rounding_mode="floor")
    qo_indptr, kv_indptr = sums(s["qo_lens"]), sums(pages)
    table = s["page_tables"][s["rows"].long()].long()
    at = torch.arange(s["max_pages"], device=dev)
    req = torch.searchsorted(kv_indptr[1:].long(), at, right=True)
    indices = table[req, at - kv_indptr[req]]
    t = torch.arange(s["max_tokens"], device=dev)
    req = torch.searchsorted(qo_indptr[1:].long(), t, right=True)
    there, req = req < batch, req.clamp(max=batch - 1)
    i = t - qo_indptr[req]
    place = s["kv_lens"][req] + i
    slots = table[req, torch.div(place, page, rounding_mode="floor").clamp(max=table.shape[1] - 1)] * page + place % page
    out = {"qo_indptr": qo_indptr, "kv_page_indptr": kv_indptr, "kv_page_indices": indices.int(),
           "kv_last_page_lens": (lens - 1) % page + 1, "slots": torch.where(there, slots, -1)}
    if s["parents"] is None:
        return dict(out, positions=torch.where(there, place, 0).int())
    n = torch.arange(MAX_ROWS, device=dev)
    rows = (qo_indptr[:-1, None] + n).clamp(max=s["parents"].shape[0] - 1).long()
    above = _ancestors(s["parents"][rows], n < s["qo_lens"][:, None])
    masks = (above.long() << n).sum(2)
    inside = i.clamp(max=MAX_ROWS - 1)
    depth = above.sum(2) - 1
    return dict(out, masks=torch.where(there, masks[req, inside], 0),
                positions=torch.where(there, s["kv_lens"][req] + depth[req, inside], 0).int())


def _plain_append(s):
    def rotate(x):
        x, half = x.float(), x.shape[-1] // 2
        cs, sn = s["table"][:, None, :half], s["table"][:, None, half:]
        re, im = x[..., 0::2], x[..., 1::2]
        return torch.stack([re * cs - im * sn, re * sn + im * cs], -1).flatten(-2)

    pages, page = s["pages"], s["case"]["page"]
    at, place = torch.div(s["slots"], page, rounding_mode="floor"), s["slots"] % page
    pages[at, 0, place] = rotate(s["k"]).to(pages.dtype)
    pages[at, 1, place] = s["v"]
    return {"q": rotate(s["q"]).to(pages.dtype), "pages": pages}


def _plain_attend(s):
    c, q, dev = s["case"], s["q"], s["q"].device
    rows, kv, _ = _lengths(c)
    lens, n, length = kv + rows, int(rows.max()), int((kv + rows).max())
    group, hk, dim, page = c["q_heads"] // c["kv_heads"], c["kv_heads"], c["dim"], c["page"]
    first = s["qo_indptr"][:-1, None].long()
    row_of = (first + torch.arange(n, device=dev)).clamp(max=q.shape[0] - 1)
    here = torch.arange(n, device=dev) < (s["qo_indptr"][1:] - s["qo_indptr"][:-1])[:, None]
    at = torch.arange(length, device=dev)
    kv_lens = (s["kv_page_indptr"][1:] - s["kv_page_indptr"][:-1] - 1) * page + s["kv_last_page_lens"]
    entry = s["kv_page_indptr"][:-1, None] + torch.div(at, page, rounding_mode="floor")
    ids = s["kv_page_indices"][entry.clamp(max=s["kv_page_indices"].shape[0] - 1)].long()
    there = at < kv_lens[:, None]
    prior = kv_lens - (s["qo_indptr"][1:] - s["qo_indptr"][:-1])
    new = at - prior[:, None]                                                  # (B, length): index among the new rows
    if s["masks"] is None:
        sees = new[:, None, :] <= torch.arange(n, device=dev)[None, :, None]
    else:
        sees = (new < 0)[:, None, :] | ((s["masks"][row_of][:, :, None] >> new.clamp(0, 63)[:, None, :]) & 1).bool()
    sees = sees & there[:, None, :]                                            # (B, n, length)
    keys, values = (s["pages"][ids, i, at % page].float().permute(0, 2, 1, 3).contiguous() for i in (0, 1))
    x = q[row_of].float().view(-1, n, hk, group, dim).permute(0, 2, 1, 3, 4).reshape(-1, hk, n * group, dim)
    scores = torch.matmul(x, keys.transpose(2, 3).contiguous()).view(-1, hk, n, group, length) / math.sqrt(dim)
    scores = torch.where(sees[:, None, :, None], scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(-1, hk, n * group, length), values).view(-1, hk, n, group, dim)
    out = out / torch.where(total == 0, 1.0, total)
    out = out.permute(0, 2, 1, 3, 4).reshape(-1, n, hk * group, dim)
    return out[here].to(q.dtype)


def _plain_verify(s):
    indptr, dev = s["qo_indptr"].long(), s["qo_indptr"].device
    total, n = s["tokens"].shape[0], s["case"]["rows_hi"]
    i = torch.arange(n, device=dev)
    here = i < (indptr[1:] - indptr[:-1])[:, None]
    row = (indptr[:-1, None] + i).clamp(max=total - 1)
    parent = torch.where(here, (i - 1).expand_as(row) if s["parents"] is None else s["parents"][row].long(), -1)
    child = here & (parent >= 0)
    token, u = s["tokens"][row].long(), s["uniforms"][row].double()
    above = (indptr[:-1, None] + parent.clamp(min=0)).clamp(max=total - 1)
    p = s["target_probs"][above, token].double()
    # earlier children of the same parent, and those of them that first proposed their token
    earlier = (parent[:, :, None] == parent[:, None, :]) & child[:, None, :] & (i[None, :, None] > i[None, None, :])
    again = (earlier & (token[:, :, None] == token[:, None, :])).any(2)
    if s["draft_probs"] is None:
        rest = 1 - (earlier & ~again[:, None, :]).double().matmul(p[:, :, None])[:, :, 0]
        passes = child & ~again & (u * rest < p)
    else:
        passes = child & (u * s["draft_probs"][above, token].double() < p)
    taken = passes & ~(earlier & passes[:, None, :]).any(2) | (here & (i == 0))
    reached = here & ~(_ancestors(parent, here) & ~taken[:, None, :]).any(2)
    counts = reached.sum(1)
    path = torch.where(reached, i, n).sort(1).values                            # accepted rows, then n
    last = path.gather(1, (counts - 1)[:, None])
    at = (indptr[:-1, None] + last)[:, 0]
    w = s["target_probs"][at].double()
    refused = child & (parent == last)
    if s["draft_probs"] is None:
        keep = torch.ones_like(w).scatter_reduce_(1, token, 1.0 - refused.double(), "amin")
        rest = w * keep
    else:
        rest = torch.where(refused.any(1, keepdim=True), (w - s["draft_probs"][at].double()).clamp(min=0), w)
    w = torch.where(rest.sum(1, keepdim=True) > 0, rest, w)
    cum = w.cumsum(1)
    draw = torch.searchsorted(cum, u[:, :1] * cum[:, -1:], right=True)[:, 0].clamp(max=w.shape[1] - 1)
    emitted = token.gather(1, path.roll(-1, 1).clamp(max=n - 1))
    emitted = torch.where(i == (counts - 1)[:, None], draw[:, None], torch.where(i < counts[:, None], emitted, -1))
    path = torch.where(i < counts[:, None], path, -1)
    return {"counts": counts.int(), "path": path[here].int(), "tokens": emitted[here].int()}


def _plain_move(s):
    pages, page, indptr = s["pages"], s["case"]["page"], s["qo_indptr"].long()
    rows = torch.arange(s["path"].shape[0], device=pages.device)
    req = torch.searchsorted(indptr[1:], rows, right=True)
    source = torch.where(rows - indptr[req] < s["counts"][req], indptr[req] + s["path"].long(), rows)
    take = lambda slots: (torch.div(slots, page, rounding_mode="floor"), slots % page)
    (to, to_place), (at, at_place) = take(s["slots"]), take(s["slots"][source])
    pages[:, to, :, to_place] = pages[:, at, :, at_place]
    return pages


_plain = {"tables": _plain_tables, "append": _plain_append, "attend": _plain_attend, "verify": _plain_verify,
          "move": _plain_move}


# ---- the results by definition, request by request, in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    rows, kv, parents = _lengths(case)
    first = np.cumsum(rows) - rows
    return {"tables": _exact_tables, "append": _exact_append, "attend": _exact_attend, "verify": _exact_verify,
            "move": _exact_move}[case["kind"]](case, s, rows, kv, parents, first)


def _exact_tables(case, s, rows, kv, parents, first):
    page, tables, order = case["page"], s["page_tables"].cpu().numpy(), s["rows"].cpu().numpy()
    lens = kv + rows
    used = [tables[order[b]][: -(-int(n) // page)] for b, n in enumerate(lens)]
    tail = s["max_tokens"] - int(rows.sum())
    slots = np.concatenate([tables[order[b]][np.arange(k, k + n) // page].astype(np.int64) * page + np.arange(k, k + n) % page
                            for b, (k, n) in enumerate(zip(kv, rows))] + [np.full(tail, -1)])
    depth = _descent(rows, parents) - 1
    out = {"qo_indptr": np.concatenate([[0], np.cumsum(rows)]), "kv_page_indptr": np.concatenate([[0], np.cumsum([len(u) for u in used])]),
           "kv_page_indices": np.concatenate(used), "kv_last_page_lens": lens - (np.array([len(u) for u in used]) - 1) * page,
           "positions": np.concatenate([np.repeat(kv, rows) + depth, np.zeros(tail, np.int64)])}
    out = {k: v.astype(np.int32) for k, v in out.items()}
    out["slots"] = slots
    if parents is not None:
        out["masks"] = np.concatenate([_masks(rows, parents), np.zeros(tail, np.int64)])
    return out


def _exact_append(case, s, rows, kv, parents, first):
    half = case["dim"] // 2
    turn = torch.complex(s["table"][:, :half].double(), s["table"][:, half:].double())[:, None]
    rotate = lambda x: torch.view_as_real(torch.view_as_complex(x.double().reshape(x.shape[:-1] + (half, 2))) * turn).flatten(-2)
    pages = s["pages"].double()
    flat = pages.transpose(1, 2).reshape(-1, 2, case["kv_heads"], case["dim"])
    flat[s["slots"], 0] = rotate(s["k"])
    flat[s["slots"], 1] = s["v"].double()
    return {"q": rotate(s["q"]), "pages": flat.view(-1, case["page"], 2, case["kv_heads"], case["dim"]).transpose(1, 2).contiguous()}


def _exact_attend(case, s, rows, kv, parents, first):
    seen = _masks(rows, parents) if parents is not None else None
    group, out = case["q_heads"] // case["kv_heads"], []
    begin = np.concatenate([[0], np.cumsum(-(-(kv + rows) // case["page"]))])
    for b in range(case["batch"]):
        n, length = int(rows[b]), int(kv[b] + rows[b])
        held = s["pages"][s["kv_page_indices"][begin[b]: begin[b + 1]].long()].double()
        k, v = (held[:, i].reshape(-1, case["kv_heads"], case["dim"])[:length].transpose(0, 1) for i in (0, 1))
        q = s["q"][first[b]: first[b] + n].double().unflatten(1, (-1, group)).permute(1, 2, 0, 3)
        sees = np.ones((n, length), bool)
        for i in range(n):
            bits = (1 << (i + 1)) - 1 if seen is None else int(seen[first[b] + i]) % (1 << 64)
            sees[i, int(kv[b]):] = [(bits >> j) & 1 for j in range(n)]
        score = torch.matmul(q, k.transpose(1, 2).unsqueeze(1).contiguous()) * case["dim"] ** -0.5
        score.masked_fill_(~_dev(sees), -math.inf)
        out.append(torch.matmul(torch.softmax(score, -1), v.unsqueeze(1)).permute(2, 0, 1, 3).flatten(1, 2))
    return torch.cat(out)


def _exact_verify(case, s, rows, kv, parents, first):
    token, u = s["tokens"].tolist(), s["uniforms"].tolist()
    counts, path, emitted = [], np.full(len(token), -1, np.int32), np.full(len(token), -1, np.int32)
    for b in range(case["batch"]):
        f, n, at, walk = int(first[b]), int(rows[b]), 0, [0]
        up = [-1] + [(j - 1 if parents is None else int(parents[f + j])) for j in range(1, n)]
        while True:
            p = s["target_probs"][f + at].double()
            w, rest, follow = p.clone(), 1.0, -1
            for j in (j for j in range(1, n) if up[j] == at):
                x = token[f + j]
                if s["draft_probs"] is not None:
                    q = s["draft_probs"][f + at].double()
                    if u[f + j] * float(q[x]) < float(p[x]):
                        follow = j
                        break
                    w = (p - q).clamp(min=0)
                else:
                    if float(w[x]) > u[f + j] * rest:
                        follow = j
                        break
                    rest -= float(w[x])
                    w[x] = 0
            if follow < 0:
                break
            at = follow
            walk.append(at)
        w = w if float(w.sum()) > 0 else p
        cum = w.cumsum(0)
        draw = int((cum <= u[f] * cum[-1]).sum())
        path[f: f + len(walk)] = walk
        emitted[f: f + len(walk)] = [token[f + j] for j in walk[1:]] + [min(draw, case["vocab"] - 1)]
        counts.append(len(walk))
    return {"counts": np.array(counts, np.int32), "path": path, "tokens": emitted}


def _exact_move(case, s, rows, kv, parents, first):
    pages = s["pages"].double()
    before, slots = pages.clone(), s["slots"].tolist()
    path, counts = _accepted(case)
    page = case["page"]
    for b, f in enumerate(first):
        for j in range(1, int(counts[b])):
            to, at = slots[f + j], slots[f + int(path[f + j])]
            pages[:, to // page, :, to % page] = before[:, at // page, :, at % page]
    return pages


# ---- what a pass cannot do without


def work(case):
    rows, kv, parents = _lengths(case)
    size, total = DTYPES[case["dtype"]].itemsize, int(rows.sum())
    row = case["dim"] * size
    if case["kind"] == "tables":
        pages = int((-(-(kv + rows) // case["page"])).sum())
        return {"bytes": 24 * case["batch"] + 8 * pages + total * (12 if parents is None else 24), "flops": 0}
    if case["kind"] == "append":
        return {"bytes": total * (2 * (case["q_heads"] + 2 * case["kv_heads"]) * row + 4 * case["dim"] + 8),
                "flops": 3 * total * (case["q_heads"] + case["kv_heads"]) * case["dim"]}
    if case["kind"] == "attend":
        tokens = int((kv + rows).sum())
        pairs = int((kv * rows).sum() + _descent(rows, parents).sum())
        return {"bytes": 2 * tokens * case["kv_heads"] * row + 2 * total * case["q_heads"] * row,
                "flops": 4 * case["q_heads"] * case["dim"] * pairs}
    if case["kind"] == "verify":
        # the distributions at the last accepted rows
        held = case["batch"] * case["vocab"] * (2 if case["drafts"] else 1)
        return {"bytes": held * size + total * 24, "flops": 2 * held}
    _, counts = _accepted(case)
    return {"bytes": 2 * int((counts - 1).sum()) * case["layers"] * 2 * case["kv_heads"] * row + 16 * total, "flops": 0}
