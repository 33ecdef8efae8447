"""What a decode step needs before attention, from the definitions: pages and packing one sequence after the other, block
selection with exact whole-number scores, rotary positions with angles reduced in fractions (numpy, Python)."""
from __future__ import annotations

from fractions import Fraction
from typing import List, Optional, Sequence, Tuple

import numpy as np
import torch

from . import cache as oc

PAGE = 64
PI = Fraction("3.14159265358979323846264338327950288419716939937510582097494459230781640629")


# ------------------------------------------------------------------ pages
def reserve(pages, held, rows, pool, n_free: int, n_rows: Optional[int] = None):
    """(pages, pool, lens, cu or None, positions, slots, held, n_free) after a call; the inputs stay as they are."""
    pages, pool = np.array(pages, np.int32), np.array(pool, np.int32)
    n, width = pages.shape
    most = min(width * PAGE, 2**31 - 1)
    have = [min(max(int(h), 0), most) for h in held]
    free = [int(x) for x in pool[:min(max(n_free, 0), len(pool))]]
    count = lambda t: -(-t // PAGE)  # noqa: E731
    after = list(have)
    for s in range(n):  # what is given back
        if rows[s] < 0:
            after[s] = max(0, have[s] + int(rows[s]))
            free += [int(x) for x in pages[s, count(after[s]):count(have[s])]]
    free = free[:len(pool)]
    pool[:len(free)] = free
    grants, wanted, lens = [], 0, [0] * n
    for s in range(n):
        want = have[s] + int(rows[s])
        if rows[s] <= 0 or want > most:
            continue
        need = count(want) - count(have[s])
        wanted += need
        if need == 0 or wanted <= len(free):
            grants.append((s, need))
            after[s] = lens[s] = want
    left = len(free) - sum(need for _, need in grants)
    at = left
    for s, need in grants:
        pages[s, count(have[s]):count(have[s]) + need] = free[at:at + need]
        at += need
    asked = [max(0, int(r)) for r in rows]
    cu = None
    if n_rows is None:
        where = [(s, lens[s] - 1) for s in range(n)]
    else:
        cu = np.minimum(np.concatenate(([0], np.cumsum(np.array(asked, np.int64)))), 2**31 - 1)
        where = [(-1, -1)] * n_rows
        for s in range(n):
            for r in range(cu[s], min(cu[s + 1], n_rows)):
                where[r] = (s, lens[s] - (cu[s + 1] - r) if lens[s] else -1)
    pos = [p for _, p in where]
    slots = [int(pages[s, p // PAGE]) * PAGE + p % PAGE if p >= 0 and pages[s, p // PAGE] >= 0 else -1 for s, p in where]
    return pages, pool, np.array(lens), cu, np.array(pos), np.array(slots, np.int64), np.array(after), left


# ------------------------------------------------------------------ selection
def completed(tokens: int, block: int, stride: int) -> int:
    return (tokens - block) // stride + 1 if tokens >= block else 0


def _whole(x: np.ndarray) -> np.ndarray:
    """Finite floats as Python integers, in units of 2^-200."""
    out = np.empty(x.shape, object)
    for i, v in np.ndenumerate(x):
        n, d = float(v).as_integer_ratio()
        out[i] = (n << 200) // d if d <= 1 << 200 else 0
    return out


def select(q, cache, pages, lens, n_sel, l_prime=64, block=32, stride=16, cu=None) -> np.ndarray:
    """int32 [N, Hkv, n_sel] of rows q [N, Hq, d_qk] over the compressed cache uint8 [P, Hkv, record], exact."""
    q = np.asarray(q, np.float64)
    n_rows, hq, d_qk = q.shape
    hkv = cache.shape[1]
    d_v = cache.shape[2] // 36 - d_qk
    out = np.full((n_rows, hkv, n_sel), -1, np.int32)
    for r in range(n_rows):
        seq, pos, _ = oc.place(r, pages, lens, cu, cache.shape[0])
        tokens = pos + 1
        if seq < 0 or pos < 0 or tokens > min(2**24, pages.shape[1] * PAGE * stride + block - 1):
            continue
        n, blocks = completed(tokens, block, stride), -(-tokens // l_prime)
        where = np.minimum(np.floor(torch.linspace(0, tokens - 1, n, dtype=torch.float32).numpy() / l_prime).astype(np.int64), blocks - 1)
        for h in range(hkv):
            heads = q[r, h * (hq // hkv):(h + 1) * (hq // hkv)]
            score, bad = [0] * blocks, [not np.isfinite(heads).all()] * blocks
            if n and not bad[0]:
                qs = _whole(heads).sum(0)
                ids = np.array([oc.page_of(pages, seq, i * PAGE, cache.shape[0]) for i in range(-(-n // PAGE))])
                k, _ = oc.decode(cache[np.maximum(ids, 0), h], d_qk, d_v)
                k = np.where((ids >= 0)[:, None, None], k, 0.0).reshape(-1, d_qk)[:n]
                for i in range(n):
                    if not np.isfinite(k[i]).all():
                        bad[where[i]] = True
                        continue
                    # (a key's values are multiples of 2^-18)
                    score[where[i]] += int((qs * (k[i] * 2.0**18).astype(np.int64).astype(object)).sum())
            order = sorted(range(blocks), key=lambda b: (bad[b], 0 if bad[b] else -score[b], b))[:n_sel]
            out[r, h, :len(order)] = order
    return out


# ------------------------------------------------------------------ rotary positions
def angles(positions: np.ndarray, inv_freq: Sequence[float], axis: Sequence[int]) -> np.ndarray:
    """Angles in [0, 2 pi) of positions [axes, ...] for each pair [..., pairs], fp64, off by less than 2^-50."""
    positions = np.asarray(positions)
    out = np.zeros(positions.shape[1:] + (len(axis),))
    for i, (f, a) in enumerate(zip(inv_freq, axis)):
        turn = Fraction(float(f)) / (2 * PI)
        for at in np.ndindex(*positions.shape[1:]):
            out[at + (i,)] = float(2 * PI * ((int(positions[(a,) + at]) * turn) % 1))
    return out


def rotary(x: np.ndarray, angle: np.ndarray, offset: int, interleaved: bool, inverse: bool = False) -> Tuple[np.ndarray, np.ndarray]:
    """x fp64 [..., H, d] turned by angle [..., pairs], and |a| + |b| of the pair that a value is of (0 for the others)."""
    pairs = angle.shape[-1]
    x = np.asarray(x, np.float64)
    out, size = x.copy(), np.zeros(x.shape)
    first = offset + (2 * np.arange(pairs) if interleaved else np.arange(pairs))
    second = first + (1 if interleaved else pairs)
    c, s = np.cos(angle)[..., None, :], np.sin(angle)[..., None, :] * (-1 if inverse else 1)
    a, b = x[..., first], x[..., second]
    out[..., first], out[..., second] = a * c - b * s, b * c + a * s
    size[..., first] = size[..., second] = np.abs(a) + np.abs(b)
    return out, size


def plan_frequencies(dim: int, base: float) -> List[float]:
    return [float(base) ** (-2 * i / dim) for i in range(dim // 2)]
