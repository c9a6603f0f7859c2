"""Pages of 8-bit K/V for the tests, by their definition in 64 bits on the CPU: codes, scales, appends and moves, block by block."""
from __future__ import annotations

import dataclasses
from typing import Optional

import numpy as np
import torch

from draftutil import Step

LEAST = 2.0 ** -126


def e4m3_values() -> np.ndarray:
    """What the 256 codes stand for: sign, 4 bits of exponent (bias 7), 3 behind the point; 0x7F and 0xFF are none."""
    c = np.arange(256)
    e, f = c >> 3 & 15, c & 7
    x = np.where(e == 0, f / 8 * 2.0 ** -6, (1 + f / 8) * 2.0 ** (e - 7.0))
    x[c & 127 == 127] = np.nan
    return np.where(c & 128, -x, x)


VALUES = e4m3_values()


def encode(x: np.ndarray) -> np.ndarray:
    """Codes of x, |x| <= 464: to nearest, ties to the even code.  What is no number: 0x7F."""
    size = np.abs(np.nan_to_num(x, nan=0.0))
    up = VALUES[:127]
    hi = np.minimum(np.searchsorted(up, size), 126)
    lo = np.maximum(hi - 1, 0)
    near = np.where(size - up[lo] < up[hi] - size, lo, np.where(size - up[lo] > up[hi] - size, hi, np.where(lo % 2 == 0, lo, hi)))
    return np.where(np.isnan(x), 127, near | np.where(np.signbit(x), 128, 0)).astype(np.uint8)


def least_scale(most: float) -> float:
    s = LEAST
    if most > 0:
        m, e = np.frexp(most)                      # most = m * 2^e, m from [0.5, 1); 448 = 0.875 * 2^9
        s = max(LEAST, 2.0 ** float(e - 9 + (m > 0.875)))
    return s


@dataclasses.dataclass
class Records:
    """Codes (N, 2, Hkv, P, D) uint8 and scales (N, 2, Hkv) float64 of one layer."""
    codes: np.ndarray
    scales: np.ndarray

    @property
    def sizes(self):
        _, _, hkv, page, dim = self.codes.shape
        return page, hkv, dim

    def copy(self) -> "Records":
        return Records(self.codes.copy(), self.scales.copy())

    def values(self) -> np.ndarray:
        return VALUES[self.codes] * self.scales[..., None, None]

    def tensor(self) -> torch.Tensor:
        """(N, page_bytes) uint8, padding included."""
        n = self.codes.shape[0]
        flat, scales = self.codes.reshape(n, -1), self.scales.astype(np.float32).reshape(n, -1).view(np.uint8)
        size = -(-(flat.shape[1] + scales.shape[1]) // 128) * 128
        out = np.full((n, size), 0xA5, np.uint8)
        out[:, : flat.shape[1]] = flat
        out[:, flat.shape[1]: flat.shape[1] + scales.shape[1]] = scales
        return torch.from_numpy(out)

    @classmethod
    def of_tensor(cls, t: torch.Tensor, page: int, hkv: int, dim: int) -> "Records":
        raw, n, size = np.ascontiguousarray(t.cpu().numpy()), t.shape[0], 2 * hkv * page * dim
        scales = np.ascontiguousarray(raw[:, size: size + 8 * hkv]).view(np.float32)
        return cls(raw[:, :size].reshape(n, 2, hkv, page, dim).copy(), scales.reshape(n, 2, hkv).astype(np.float64))


def quantise(values: np.ndarray) -> Records:
    """Records of (N, 2, P, Hkv, D) values."""
    x = values.astype(np.float64).transpose(0, 1, 3, 2, 4)
    most = np.abs(x).max((3, 4))
    scales = np.vectorize(least_scale)(most)
    return Records(encode(x / scales[..., None, None]), scales)


def as_quantised(step: Step, spread: float = 1.0, seed: int = 0):
    """(records, the step over the values that they stand for); spread: pages' sizes lie over so many powers of two."""
    pages = step.pages.double().numpy()
    rng = np.random.default_rng(seed)
    if spread > 1:
        pages = pages * 2.0 ** rng.uniform(-spread / 2, spread / 2, (pages.shape[0], 2, 1, pages.shape[3], 1))
    records = quantise(pages)
    return records, dataclasses.replace(step, pages=torch.from_numpy(records.values().transpose(0, 1, 3, 2, 4).copy()))


def append(records: Records, step: Step, k: np.ndarray, v: np.ndarray, most: float) -> Records:
    """k, v (rows, Hkv, D) in 64 bits, k as it goes in; most: what magnitudes are cut to."""
    out, page = records.copy(), step.page
    for b in range(len(step.kv)):
        lo, hi, table, length = step.request(b)
        prior = int(step.kv[b])
        for p in range(prior // page, -(-length // page) if hi > lo else 0):
            begin, end, at = max(prior, p * page), min(length, (p + 1) * page), table[p]
            rows = slice(lo + begin - prior, lo + end - prior)
            for h in range(step.hkv):
                x = np.stack([k[rows, h], v[rows, h]])                          # (2, n, D)
                fine = np.isfinite(x).all((0, 2))
                x = np.clip(np.where(fine[None, :, None], x, 0), -most, most)
                for i in range(2):
                    s = least_scale(np.abs(x[i]).max(initial=0))
                    kept = begin - p * page
                    if kept:
                        s = max(s, records.scales[at, i, h])
                        again = VALUES[records.codes[at, i, h, :kept]] * (records.scales[at, i, h] / s)
                        out.codes[at, i, h, :kept] = encode(again)
                    code = encode(x[i] / s)
                    code[~fine] = 127 if i == 0 else 0
                    out.codes[at, i, h, kept: kept + end - begin] = code
                    out.scales[at, i, h] = s
    return out


def move(records: Records, step: Step, path: np.ndarray, counts: np.ndarray) -> Records:
    out, page = records.copy(), step.page
    values = records.values()
    for b in range(len(step.kv)):
        lo, hi, table, length = step.request(b)
        prior = int(step.kv[b])
        goes = {}
        if 2 <= counts[b] <= 64:
            walk = path[lo: lo + int(counts[b])]
            goes = {j: int(walk[j]) for j in range(1, min(len(walk), hi - lo)) if j < walk[j] < hi - lo and walk[j] > walk[j - 1]}
        for p in sorted({(prior + j) // page for j in goes}):
            at = table[p]
            here = {j: i for j, i in goes.items() if (prior + j) // page == p}
            x = np.stack([values[table[(prior + i) // page], :, :, (prior + i) % page] for i in here.values()])
            count = min(page, length - p * page)
            for i in range(2):
                for h in range(step.hkv):
                    most, s = np.nanmax(np.abs(x[:, i, h]), initial=0), records.scales[at, i, h]
                    if most > 0 and least_scale(most) > s:
                        s = least_scale(most)
                        out.codes[at, i, h, :count] = encode(values[at, i, h, :count] / s)
                        out.scales[at, i, h] = s
                    for n, j in enumerate(here):
                        out.codes[at, i, h, (prior + j) % page] = encode(x[n, i, h] / s)
    return out


def same(got: Records, want: Records) -> None:
    """The same codes (codes of no number and of zeros of either sign count as one) and scales."""
    a, b = got.codes, want.codes
    odd = (a != b) & ~((a & 127 == 127) & (b & 127 == 127)) & ~((a & 127 == 0) & (b & 127 == 0))
    assert not odd.any(), (np.argwhere(odd)[:3], int(odd.sum()), a[odd][:3], b[odd][:3])
    assert np.array_equal(got.scales, want.scales), np.argwhere(got.scales != want.scales)[:3]


def rows(seed: int, step: Step, dtype: torch.dtype, size: float = 1.0, heads: Optional[int] = None) -> torch.Tensor:
    gen = torch.Generator().manual_seed(seed)
    shape = (int(step.qo_indptr[-1]), step.hkv if heads is None else heads, step.dim)
    return (size * torch.randn(shape, generator=gen)).to(dtype)


def near(got: torch.Tensor, want: np.ndarray, bound: np.ndarray) -> None:
    """Every element within its own bound (one of 0 asks for the value itself)."""
    got = got.double().cpu().numpy()
    assert np.isfinite(got).all()
    over = np.abs(got - want) - bound
    assert over.max(initial=0) <= 0, (np.unravel_index(over.argmax(), over.shape), over.max())
