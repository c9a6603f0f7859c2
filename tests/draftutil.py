"""Steps of drafted tokens for the tests: seeded requests with chains or trees over a paged pool, and the operators by
their definitions, request by request in 64 bits."""
from __future__ import annotations

from dataclasses import dataclass
from typing import List, Optional, Sequence

import numpy as np
import torch

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "fp32": torch.float32}
HALF_STEP = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "fp32": 2.0 ** -24}      # of a rounding, over the value


def random_parents(rng, n: int, near: int = 5) -> np.ndarray:
    return np.array([-1] + [max(0, i - int(rng.integers(1, near + 1))) for i in range(1, n)], np.int32)[:n]


def ancestors(parents: Sequence[int]) -> List[List[int]]:
    """Row i's ancestors and itself, from the definition: a value outside [0, i) is no parent."""
    out: List[List[int]] = []
    for i, p in enumerate(parents):
        out.append((out[p] if 0 <= p < i else []) + [i])
    return out


def to_signed(word: int) -> int:
    return word - (1 << 64) if word >= 1 << 63 else word


@dataclass
class Step:
    kv: np.ndarray               # cached tokens
    rows: np.ndarray             # new rows
    parents: Optional[np.ndarray]
    page: int
    hq: int
    hkv: int
    dim: int
    dtype: str
    qo_indptr: np.ndarray
    kv_page_indptr: np.ndarray
    kv_page_indices: np.ndarray
    kv_last: np.ndarray
    masks: Optional[np.ndarray]
    pages: torch.Tensor          # (num_pages, 2, P, Hkv, D), on the CPU
    q: torch.Tensor              # (rows, Hq, D)

    def request(self, b: int):
        """Row range, block table, tokens with the new ones."""
        lo, hi = self.qo_indptr[b], self.qo_indptr[b + 1]
        table = self.kv_page_indices[self.kv_page_indptr[b]: self.kv_page_indptr[b + 1]]
        return int(lo), int(hi), table, int(self.kv[b] + self.rows[b])

    def slots(self) -> np.ndarray:
        out = []
        for b in range(len(self.kv)):
            _, _, table, length = self.request(b)
            at = np.arange(int(self.kv[b]), length)
            out.append(table[at // self.page].astype(np.int64) * self.page + at % self.page)
        return np.concatenate(out) if out else np.zeros(0, np.int64)

    def sees(self, b: int) -> np.ndarray:
        """(rows, tokens) truth values."""
        lo, hi, _, length = self.request(b)
        n, kv = hi - lo, int(self.kv[b])
        out = np.ones((n, length), bool)
        for i in range(n):
            for j in range(n):
                out[i, kv + j] = j <= i if self.masks is None else (int(self.masks[lo + i]) >> j) & 1
        return out

    def on(self, device) -> dict:
        i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(device)
        return {"csr": (i32(self.qo_indptr), i32(self.kv_page_indptr), i32(self.kv_page_indices), i32(self.kv_last)),
                "masks": None if self.masks is None else torch.from_numpy(self.masks).to(device),
                "pages": self.pages.to(device), "q": self.q.to(device)}


def make_step(seed: int, kv, rows, tree: bool = False, page: int = 16, hq: int = 32, hkv: int = 8, dim: int = 128,
              dtype: str = "bf16", parents: Optional[np.ndarray] = None) -> Step:
    rng = np.random.default_rng(seed)
    gen = torch.Generator().manual_seed(seed)
    kv, rows = np.asarray(kv, np.int64), np.asarray(rows, np.int64)
    lens = kv + rows
    pages = -(-lens // page)
    indptr = np.concatenate([[0], np.cumsum(pages)]).astype(np.int32)
    qo = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    num_pages = int(indptr[-1]) + 3
    if tree and parents is None:
        parents = np.concatenate([random_parents(rng, int(n)) for n in rows] + [np.zeros(0, np.int32)])
    masks = None
    if parents is not None:
        masks = np.array([to_signed(sum(1 << a for a in anc)) for b in range(len(kv))
                          for anc in ancestors(parents[qo[b]: qo[b + 1]].tolist())], np.int64)
    randn = lambda *s: torch.randn(s, generator=gen).to(DTYPES[dtype])
    return Step(kv, rows, parents, page, hq, hkv, dim, dtype, qo, indptr,
                rng.permutation(num_pages)[: int(indptr[-1])].astype(np.int32),
                np.where(lens > 0, (lens - 1) % page + 1, 0).astype(np.int32), masks,
                randn(num_pages, 2, page, hkv, dim), randn(int(qo[-1]), hq, dim))


def attention(step: Step, scale: Optional[float] = None):
    """(out, bound), (rows, Hq, D) in 64 bits: the result, and how far a kernel may be from it.

    With u half a step of the type and e one of 32 bits, relative to the value: a score is a sum of D products in
    32 bits, off by at most (D + 2) e times the sum of their magnitudes, and a probability by that much of itself, twice (its own
    and the sum's), by u for its rounding to 16 bits (fp32: none) and by e for each of the tokens summed and each of the few
    steps of an exponential; the output is such a mean of v and is rounded by u of itself.  16-bit types: a tenth more for
    terms of second order."""
    out = np.zeros((int(step.qo_indptr[-1]), step.hq, step.dim))
    bound = np.zeros_like(out)
    u, e, group = HALF_STEP[step.dtype], 2.0 ** -24, step.hq // step.hkv
    scale = step.dim ** -0.5 if scale is None else scale
    for b in range(len(step.kv)):
        lo, hi, table, length = step.request(b)
        if hi == lo:
            continue
        held = step.pages[torch.from_numpy(table).long()].double().numpy()
        k, v = (held[:, i].reshape(-1, step.hkv, step.dim)[:length] for i in (0, 1))
        q, sees = step.q[lo:hi].double().numpy(), step.sees(b)
        for h in range(step.hq):
            s = np.where(sees, q[:, h] @ k[:, h // group].T * scale, -np.inf)
            size = np.abs(q[:, h]) @ np.abs(k[:, h // group]).T * abs(scale)
            off = 2 * (step.dim + 2) * e * np.where(sees, size, 0).max(1) + (length + 16) * e
            top = s.max(1)
            w = np.exp(s - np.where(np.isfinite(top), top, 0)[:, None])
            total = w.sum(1)
            w /= np.where(total > 0, total, 1)[:, None]
            out[lo:hi, h] = w @ v[:, h // group]
            spread = w @ np.abs(v[:, h // group])
            rounding = u * (spread + np.abs(out[lo:hi, h])) * 1.1 if step.dtype != "fp32" else 2 * u * np.abs(out[lo:hi, h])
            bound[lo:hi, h] = rounding + off[:, None] * spread + 1e-7 * spread.max(initial=0)
    return out, bound


def verdict(target, tokens, uniforms, qo_indptr, parents=None, draft=None):
    """(counts, path, tokens) by the definition; target and draft (rows, vocab) float64 arrays, what is no probability 0."""
    clean = lambda a: np.where(np.isfinite(a) & (a > 0), a, 0.0)
    target = clean(target)
    draft = None if draft is None else clean(draft)
    vocab = target.shape[1]
    counts, path, given = [], np.full(len(target), -1, np.int32), np.full(len(target), -1, np.int32)
    for b in range(len(qo_indptr) - 1):
        f, n = int(qo_indptr[b]), int(qo_indptr[b + 1] - qo_indptr[b])
        if n == 0 or n > 64:
            counts.append(0)
            continue
        up = [-1] + [j - 1 if parents is None else int(parents[f + j]) for j in range(1, n)]
        walk = [0]
        while True:
            at = walk[-1]
            p = target[f + at]
            w, rest, refused, follow = p.copy(), 1.0, set(), None
            for j in [j for j in range(at + 1, n) if up[j] == at]:
                x = int(tokens[f + j])
                px = p[x] if 0 <= x < vocab else 0.0
                if draft is not None:
                    qx = draft[f + at, x] if 0 <= x < vocab else 0.0
                    if float(uniforms[f + j]) * qx < px:
                        follow = j
                        break
                    w = np.maximum(p - draft[f + at], 0)
                else:
                    if x not in refused:
                        if float(uniforms[f + j]) * rest < px:
                            follow = j
                            break
                        rest -= px
                    refused.add(x)
                    if 0 <= x < vocab:
                        w[x] = 0
            if follow is None:
                break
            walk.append(follow)
        w = w if w.sum() > 0 else p
        u = float(uniforms[f])
        over = np.flatnonzero(np.cumsum(w) > (0 if u < 0 else u) * w.sum())
        mass = np.flatnonzero(w > 0)
        last = int(over[0]) if len(over) else int(mass[-1]) if len(mass) else 0
        counts.append(len(walk))
        path[f: f + len(walk)] = walk
        given[f: f + len(walk)] = [int(tokens[f + j]) for j in walk[1:]] + [last]
    return np.array(counts, np.int32), path, given
