"""The 4-bit paged KV cache in 64 bits, written from its definition (numpy, one row at a time): the
quantiser, the record layout, and the attention of a batch's newest tokens.  Out-of-range entries of the
page table, lengths and cu_seqlens mean absent tokens, as include/nsa_sel.h says."""
from __future__ import annotations

from typing import List, Optional, Tuple

import numpy as np

PAGE = 64
LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def scale_value(byte: np.ndarray) -> np.ndarray:
    """Value of a scale byte: 5 exponent bits (bias 15), 3 mantissa bits; exponent 31 is infinity or NaN."""
    byte = np.asarray(byte, np.int64)
    e, m = byte >> 3, byte & 7
    v = np.where(e == 0, m * 2.0 ** -17, (8 + m) * 2.0 ** (e - 18.0))
    return np.where(e == 31, np.where(m == 0, np.inf, np.nan), v)


_SCALES = scale_value(np.arange(0xE3))  # the finite scales that writing uses, ascending to 10240


def _nearest_even(x: np.ndarray, grid: np.ndarray) -> np.ndarray:
    """Index of the entry of an ascending grid that is nearest to x >= 0, the even index in ties."""
    hi = np.clip(np.searchsorted(grid, x), 1, len(grid) - 1)
    lo = hi - 1
    up = (grid[hi] - x < x - grid[lo]) | ((grid[hi] - x == x - grid[lo]) & (hi % 2 == 0))
    return np.where(up, hi, lo)


def quantise(x: np.ndarray) -> Tuple[np.ndarray, np.ndarray]:
    """fp64 [..., d] -> (code 0..15 [..., d], scale byte [..., d / 16])."""
    g = np.asarray(x, np.float64).reshape(*x.shape[:-1], -1, 16)
    fine = np.isfinite(g).all(-1)
    g = np.where(fine[..., None], g, 0.0)
    byte = _nearest_even(np.abs(g).max(-1) / 6.0, _SCALES)
    s = _SCALES[byte][..., None]
    code = _nearest_even(np.abs(g) / np.where(s > 0, s, 1.0), LEVELS)
    code = np.where(s > 0, code + 8 * (np.signbit(g) & (code > 0)), 0)
    return code.reshape(x.shape), np.where(fine, byte, 255)


def values(code: np.ndarray, byte: np.ndarray) -> np.ndarray:
    v = LEVELS[code & 7] * np.where(code & 8, -1.0, 1.0)
    with np.errstate(invalid="ignore"):
        return (v.reshape(*byte.shape, 16) * scale_value(byte)[..., None]).reshape(code.shape)


def split(records: np.ndarray, d_qk: int, d_v: int) -> List[np.ndarray]:
    """K codes, K scales, V codes, V scales [..., 64, per token] of records uint8 [..., 36 (d_qk + d_v)]."""
    ends = np.cumsum([PAGE * d_qk // 2, PAGE * d_qk // 16, PAGE * d_v // 2])
    return [p.reshape(*p.shape[:-1], PAGE, -1) for p in np.split(records, ends, -1)]


def decode(records: np.ndarray, d_qk: int, d_v: int) -> Tuple[np.ndarray, np.ndarray]:
    """fp64 K and V [..., 64, d] of records."""
    kc, ks, vc, vs = split(records, d_qk, d_v)
    nib = lambda c: np.stack((c & 15, c >> 4), -1).reshape(*c.shape[:-1], -1)  # noqa: E731
    return values(nib(kc), ks), values(nib(vc), vs)


def place(row: int, pages: np.ndarray, lens: np.ndarray, cu: Optional[np.ndarray], num_pages: int):
    """(sequence, position, page or -1) of a row; sequence -1 for a row of none."""
    seq = row if cu is None else -1
    if cu is not None:
        at = np.nonzero(cu[:-1] <= row)[0]
        if at.size and row < cu[at[-1] + 1]:
            seq = int(at[-1])
    if seq < 0 or seq >= len(lens):
        return -1, -1, -1
    pos = max(int(lens[seq]), 0) - (1 if cu is None else int(cu[seq + 1]) - row)
    return seq, pos, page_of(pages, seq, pos, num_pages)


def page_of(pages: np.ndarray, seq: int, pos: int, num_pages: int) -> int:
    if pos < 0 or pos // PAGE >= pages.shape[1]:
        return -1
    p = int(pages[seq, pos // PAGE])
    return p if 0 <= p < num_pages else -1


def attend(q, cache, pages, lens, sel=None, l_prime=64, window=0, cu=None, scale=0.0):
    """(O, LSE, |O|, A, n, vmax): fp64 attention of the rows q [N, Hq, d_qk] over cache uint8 [P, Hkv, record], and for
    error bounds the mean of |v| under the weights, the largest sum |q k| scale, the keys and the largest |v| of each row."""
    q = np.asarray(q, np.float64)
    n_rows, hq, d_qk = q.shape
    hkv = cache.shape[1]
    d_v, g = cache.shape[2] // 36 - d_qk, hq // hkv
    scale = scale if scale > 0 else d_qk ** -0.5
    o, absolute = np.zeros((2, n_rows, hq, d_v))
    lse = np.full((n_rows, hq), -np.inf)
    size, count, vmax = np.zeros((3, n_rows, hq))
    for r in range(n_rows):
        seq, pos, _ = place(r, pages, lens, cu, cache.shape[0])
        if seq < 0 or pos < 0:
            continue
        for h in range(hkv):
            keys = np.arange(max(0, pos + 1 - window) if window > 0 else 0, min(pos + 1, pages.shape[1] * PAGE))
            if sel is not None:
                keys = keys[np.isin(keys // l_prime, sel[r, h][sel[r, h] >= 0])]
            ids = np.array([page_of(pages, seq, int(x) * PAGE, cache.shape[0]) for x in np.unique(keys // PAGE)], np.int64)
            subs = np.unique(keys // PAGE)[ids >= 0]
            ids = ids[ids >= 0]
            keys = keys[np.isin(keys // PAGE, subs)]
            if not keys.size:
                continue
            k, v = decode(cache[ids, h], d_qk, d_v)
            at = np.searchsorted(subs, keys // PAGE) * PAGE + keys % PAGE
            k, v = k.reshape(-1, d_qk)[at], v.reshape(-1, d_v)[at]
            heads = slice(h * g, (h + 1) * g)
            z = q[r, heads] @ k.T * scale
            m = z.max(-1, keepdims=True)
            p = np.exp(z - m)
            total = p.sum(-1, keepdims=True)
            o[r, heads], absolute[r, heads] = p @ v / total, p @ np.abs(v) / total
            lse[r, heads] = (m + np.log(total))[:, 0]
            size[r, heads] = (np.abs(q[r, heads]) @ np.abs(k).T).max(-1) * scale
            count[r, heads], vmax[r, heads] = len(keys), np.abs(v).max()
    return o, lse, absolute, size, count, vmax
