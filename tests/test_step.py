"""Pages, block selection and rotary positions of a decode step without a GPU: the index arithmetic that the kernels share
(compiled for the host and fed broken tables), the oracle, the plans, the checks of arguments."""
import ctypes
import math
import os
import subprocess
from fractions import Fraction

import numpy as np
import pytest
import torch

from nsa_hopper_b200 import capi, nsa, ops
from oracle import step as oracle

CSRC = os.path.join(capi.PKG_DIR, "csrc")
BIG = 2**31 - 1
FLAGS = ["g++", "-std=c++17", "-O1", "-ffp-contract=off", "-shared", "-fPIC", "-fsanitize=undefined", "-fno-sanitize-recover=all",
         f"-I{CSRC}"]

# What the kernel does, one thread after the other: sums over the sequences, then every page and row by itself.
RESERVE = r"""
#include <stdlib.h>
#include <vector>
#include "nsa_reserve_index.h"
using namespace nsa::reserve;
static uint32_t saturated(uint32_t a, uint32_t b) { return a + b < 0x7FFFFFFFu ? a + b : 0x7FFFFFFFu; }
extern "C" int reserve(int32_t* pages, const int32_t* held, const int32_t* rows, int32_t* pool, int32_t n_free, int n, int width,
                       int pool_size, int n_rows, int packed, int32_t* held_out, int32_t* lens, int32_t* cu_out, int32_t* pos_out,
                       int64_t* slot_out) {
  std::vector<uint32_t> need(n + 1), give(n + 1), cu(n + 1);
  std::vector<int32_t> from(n);
  for (int s = 0; s < n; ++s) {
    const Change c = change_of(held[s], rows[s], width);
    need[s + 1] = need[s] + c.need(), give[s + 1] = give[s] + c.give(), cu[s + 1] = saturated(cu[s], rows[s] > 0 ? rows[s] : 0);
  }
  const int32_t free = clamp_free(n_free, pool_size);
  const uint32_t sum = free + give[n];
  const int32_t top = sum < (uint32_t)pool_size ? sum : pool_size;
  uint32_t taken = 0;
  for (int s = 0; s < n; ++s) {
    const Change c = change_of(held[s], rows[s], width);
    const bool ok = granted(c, need[s + 1], top);
    if (need[s + 1] <= (uint32_t)top) taken = need[s + 1];
    from[s] = c.before_pages < c.after_pages ? c.before_pages : c.after_pages;
    lens[s] = ok ? c.after : 0;
    held_out[s] = rows[s] > 0 && !ok ? c.held : c.after;
  }
  Plan p;
  p.pages = pages, p.pool = pool, p.need = need.data(), p.give = give.data(), p.cu = cu.data(), p.from = from.data(), p.lens = lens;
  p.page_row = width, p.n_seqs = n, p.width = width, p.free = free, p.first = top - (int32_t)taken;
  // (rows first: in the kernel they are found while pages move)
  for (int r = 0; r < n_rows; ++r) {
    const int s = packed ? ((uint32_t)r < cu[n] ? range_of(cu.data(), n, r) : -1) : r;
    const int32_t pos = s >= 0 && lens[s] > 0 ? packed ? lens[s] - (int32_t)(cu[s + 1] - r) : lens[s] - 1 : -1;
    pos_out[r] = pos;
    slot_out[r] = pos < 0 ? -1 : slot_of(page_after(p, s, pos / kPage), pos);
  }
  std::vector<int32_t> back;
  for (uint32_t j = 0; j < give[n] && free + (int64_t)j < pool_size; ++j) back.push_back(given_page(p, j));
  std::vector<int32_t> got;
  for (uint32_t j = 0; j < taken; ++j) got.push_back(taken_page(p, j));
  for (uint32_t j = 0; j < taken; ++j) {
    const int s = range_of(need.data(), n, j);
    pages[(int64_t)s * width + from[s] + (int32_t)(j - need[s])] = got[j];
  }
  for (size_t j = 0; j < back.size(); ++j) pool[free + j] = back[j];
  for (int s = 0; s <= n; ++s) cu_out[s] = cu[s];
  return p.first;
}
"""

SELECT = r"""
#include "nsa_cache_select_index.h"
using namespace nsa::cache_select;
extern "C" {
int32_t keys(int32_t tokens, int32_t block, int32_t stride) { return completed(tokens, block, stride); }
int32_t most(int32_t width, int32_t block, int32_t stride) { return most_tokens(width, block, stride); }
// blocks of all keys, by float32 positions and by one rounding; the first key of every block and of one more
void places(int32_t tokens, int32_t block, int32_t stride, int32_t shift, int32_t* slow, int32_t* fast, int32_t* first) {
  const Places p = places_of(tokens, block, stride, shift);
  const int32_t blocks = blocks_of(tokens, shift);
  for (int i = 0; i < p.n; ++i) {
    const int32_t b = (int32_t)nsa::linspace_f32(i, tokens, p.n) >> shift;
    slow[i] = b < blocks ? b : blocks - 1;
    fast[i] = p.n == 1 ? 0 : block_of(p, i);
  }
  for (int b = 0; b <= blocks; ++b) first[b] = first_key(p, b);
}
int32_t tokens(const int32_t* lens, const int32_t* cu, int n_seqs, int row, int32_t most) {
  const nsa::cache::Batch b = {nullptr, lens, cu, 0, n_seqs, 0, 0, 0};
  return tokens_of(b, nsa::cache::sequence_of(b, row), row, most);
}
}
"""


def _build(tmp_path_factory, name, text):
    d = tmp_path_factory.mktemp(name)
    (d / "shim.cpp").write_text(text)
    subprocess.run([*FLAGS, "-o", str(d / "shim.so"), str(d / "shim.cpp")], check=True)
    return ctypes.CDLL(str(d / "shim.so"))


@pytest.fixture(scope="module")
def reserve_lib(tmp_path_factory):
    return _build(tmp_path_factory, "reserve", RESERVE)


@pytest.fixture(scope="module")
def select_lib(tmp_path_factory):
    return _build(tmp_path_factory, "select", SELECT)


def _ptr(a):
    return a.ctypes.data_as(ctypes.c_void_p)


def _reserve(lib, pages, held, rows, pool, n_free, n_rows):
    n, width = pages.shape
    pages, pool = pages.copy(), pool.copy()
    count = n if n_rows is None else n_rows
    held_out, lens, cu = np.zeros(n, np.int32), np.zeros(n, np.int32), np.zeros(n + 1, np.int32)
    pos, slots = np.zeros(count, np.int32), np.zeros(count, np.int64)
    left = lib.reserve(_ptr(pages), _ptr(held), _ptr(rows), _ptr(pool), n_free, n, width, len(pool), count, n_rows is not None,
                       _ptr(held_out), _ptr(lens), _ptr(cu), _ptr(pos), _ptr(slots))
    return pages, pool, lens, None if n_rows is None else cu, pos, slots, held_out, left


def _same(got, want):
    for name, g, w in zip(("pages", "pool", "lens", "cu", "positions", "slots", "held", "n_free"), got, want):
        assert (g is None) == (w is None) and (g is None or np.array_equal(g, w)), (name, g, w)


def random_batch(rng, n, width, broken=False):
    """Tables as a scheduler has them: each page in one row or in the pool."""
    held = rng.integers(0, width * 64 + 1, n).astype(np.int32)
    rows = np.where(rng.random(n) < 0.3, -rng.integers(0, width * 64 + 1, n), rng.integers(0, 200, n)).astype(np.int32)
    rows = np.where(rng.random(n) < 0.2, 0, np.where(rng.random(n) < 0.1, -held, rows)).astype(np.int32)
    used = int((-(-held // 64)).sum())
    n_free = int(rng.integers(0, 2 * n + 2))
    ids = rng.permutation(used + n_free + 9).astype(np.int32)
    pool = ids[:used + n_free + int(rng.integers(0, 3))].copy()
    pages = rng.integers(-5, 5, (n, width)).astype(np.int32)
    at = n_free
    for s in range(n):
        k = -(-int(held[s]) // 64)
        pages[s, :k] = pool[at:at + k]
        at += k
    if broken:
        wild = np.array([-2**31, -1, 0, 1, 63, 64, 65, width * 64, width * 64 + 1, BIG], np.int64)
        held = np.where(rng.random(n) < 0.5, rng.choice(wild, n), held).astype(np.int32)
        rows = np.where(rng.random(n) < 0.5, rng.choice(wild, n), rows).astype(np.int32)
        pages = np.where(rng.random(pages.shape) < 0.3, rng.choice(wild, pages.shape), pages).astype(np.int32)
        n_free = int(rng.choice([-2**31, -1, 0, 1, n_free, len(pool), len(pool) + 1, BIG]))
        pool = pool[:int(rng.integers(0, len(pool) + 1))]
    return pages, held, rows, pool, n_free


@pytest.mark.parametrize("broken", [False, True])
def test_reserve_moves_pages_as_defined(reserve_lib, broken):
    rng = np.random.default_rng(3)
    for case in range(400):
        n, width = int(rng.integers(1, 12)), int(rng.integers(0 if broken else 1, 9))
        pages, held, rows, pool, n_free = random_batch(rng, n, width, broken)
        total = int(np.maximum(rows.astype(np.int64), 0).sum())
        n_rows = None if case % 3 == 0 else min(total, 3000) + int(rng.integers(-3, 4)) if case % 3 == 1 else total % 3000
        n_rows = None if n_rows is None else max(0, n_rows)
        _same(_reserve(reserve_lib, pages, held, rows, pool, n_free, n_rows),
              oracle.reserve(pages, held, rows, pool, n_free, n_rows))


def test_reserve_loses_no_page(reserve_lib):
    """Call after call, every page is in one row of the table or in the pool."""
    rng = np.random.default_rng(5)
    n, width, count = 9, 6, 40
    pages, held, pool, n_free = np.full((n, width), -1, np.int32), np.zeros(n, np.int32), rng.permutation(count).astype(np.int32), count
    refused = 0
    for _ in range(300):
        rows = np.where(rng.random(n) < 0.25, -rng.integers(0, 400, n), rng.integers(0, 90, n)).astype(np.int32)
        pages, pool, lens, _, _, _, held, n_free = _reserve(reserve_lib, pages, held, rows, pool, n_free, None)
        refused += int(((rows > 0) & (lens == 0)).sum())
        have = [int(x) for s in range(n) for x in pages[s, :-(-int(held[s]) // 64)]]
        assert sorted(have + [int(x) for x in pool[:n_free]]) == list(range(count))
    assert refused > 50


def test_compressed_keys_lie_in_the_blocks_of_a_prompt(select_lib):
    rng = np.random.default_rng(7)
    sizes = list(range(1, 300)) + [2**k + d for k in range(9, 17) for d in (-1, 0, 1, 17)] + [int(x) for x in rng.integers(300, 200000, 30)]
    for t in sizes:
        for block, stride, shift in ((32, 16, 6), (1, 1, 8), (64, 64, 7), (7, 3, 6), (16, 5, 6)):
            n = select_lib.keys(t, block, stride)
            assert n == oracle.completed(t, block, stride)
            blocks = -(-t // 2**shift)
            slow, fast, first = np.zeros(n, np.int32), np.zeros(n, np.int32), np.zeros(blocks + 1, np.int32)
            select_lib.places(t, block, stride, shift, _ptr(slow), _ptr(fast), _ptr(first))
            want = np.minimum(np.floor(torch.linspace(0, t - 1, n, dtype=torch.float32).numpy() / 2**shift), blocks - 1)
            assert np.array_equal(slow, want) and np.array_equal(fast, want), (t, block, stride, shift)
            assert first[0] == 0 and first[blocks] == n and np.array_equal(np.searchsorted(want, np.arange(blocks)), first[:blocks])
            assert n == 0 or np.bincount(fast, minlength=blocks).max() <= 2**shift // stride + 2


def test_compressed_keys_of_the_longest_sequences(select_lib):
    """2^24 tokens, where float32 just holds the positions: every key is in one block, none behind the last."""
    for t in (2**24, 2**24 - 1, 2**24 - 33):
        for block, stride, shift in ((32, 16, 6), (5, 7, 8)):
            n, blocks = select_lib.keys(t, block, stride), -(-t // 2**shift)
            slow, fast, first = np.zeros(n, np.int32), np.zeros(n, np.int32), np.zeros(blocks + 1, np.int32)
            select_lib.places(t, block, stride, shift, _ptr(slow), _ptr(fast), _ptr(first))
            assert np.array_equal(slow, fast) and (np.diff(fast) >= 0).all() and fast[-1] < blocks
            assert np.array_equal(np.searchsorted(fast, np.arange(blocks + 1)), first)
    assert select_lib.most(2**31 - 1, 2**31 - 1, 2**31 - 1) == 2**24
    assert [select_lib.most(w, 32, 16) for w in (0, 1, 2)] == [31, 1055, 2079]


def test_tokens_of_rows(select_lib):
    lens, cu = np.array([5, 0, 100, -3, BIG], np.int32), np.array([0, 2, 3, 7, 8, 9], np.int32)
    got = [select_lib.tokens(_ptr(lens), _ptr(cu), 5, r, 99) for r in range(11)]
    assert got == [4, 5, 0, 97, 98, 99, 0, 0, 0, 0, 0]
    assert [select_lib.tokens(_ptr(lens), None, 5, r, 2**24) for r in range(5)] == [5, 0, 100, 0, 0]


# ------------------------------------------------------------------ the query as whole numbers
def test_bytes_and_codes_are_exact():
    """Signed bytes of a sum below 2^46 (any, not only small ones), and codes doubled and shifted by 12."""
    rng = np.random.default_rng(11)
    for x in [0, 1, -1, 127, 128, -128, -129, 2**46, -2**46, 2**46 - 1] + [int(v) for v in rng.integers(-2**46, 2**46, 200)]:
        rest, digits = x, []
        for _ in range(6):
            byte = (rest + 128) % 256 - 128
            digits.append(byte)
            rest = (rest - byte) >> 8
        assert rest == 0 and sum(d << 8 * i for i, d in enumerate(digits)) == x
    # a group's sum: three bytes' sums of 16 codes up to 12 in size stay in 31 bits
    assert 128 * 12 * 16 * (2**16 + 2**8 + 1) < 2**31


# ------------------------------------------------------------------ rotary plans
@pytest.mark.parametrize("dim,base", [(128, 10000.0), (64, 1e6), (72, 5e5), (2, 10.0)])
def test_plan_turns(dim, base):
    plan = ops.rotary_plan(dim, base=base)
    for i, t in enumerate(plan.turns.tolist()):
        want = Fraction(float(base) ** (-i / (dim // 2))) / (2 * oracle.PI) * 2**64
        assert abs((t - want + 2**63) % 2**64 - 2**63) <= Fraction(1, 2)
    assert plan.axes == 1 and plan.axis.tolist() == [0] * (dim // 2) and plan.d == dim and plan.offset == 0


def test_plan_axes():
    plan = ops.rotary_plan(192, rotary_dim=64, offset=128, sections=(8, 0, 24), interleaved=True)
    assert plan.axes == 3 and plan.axis.tolist() == [0] * 8 + [2] * 24 and plan.interleaved and plan.offset == 128
    mixed = ops.rotary_plan(8, axis=[0, 1, 2, 1], inv_freq=[1.0, -2.0, 0.5, 1e9])
    assert mixed.axes == 3 and mixed.axis.tolist() == [0, 1, 2, 1] and mixed.turns[1] < 0
    assert mixed.turns[0] == -(mixed.turns[1] // 2) or abs(mixed.turns[0] * 2 + mixed.turns[1]) <= 1


@pytest.mark.parametrize("args", [
    dict(d=0), dict(d=258), dict(d=8, rotary_dim=3), dict(d=8, rotary_dim=0), dict(d=8, rotary_dim=8, offset=2), dict(d=7),
    dict(d=8, offset=-2, rotary_dim=4), dict(d=8, base=0.0), dict(d=8, base=-1.0), dict(d=8, base=math.nan), dict(d=8, sections=(2, 3)), dict(d=8, sections=(5, -1)),
    dict(d=8, sections=(1, 1, 1, 1, 0)), dict(d=8, sections=(4,), axis=[0] * 4), dict(d=8, axis=[0, 1]), dict(d=8, axis=[0, 0, 0, 4]),
    dict(d=8, axis=[0, 0, 0, -1]), dict(d=8, inv_freq=[1.0]), dict(d=8, inv_freq=[1.0, math.inf, 1.0, 1.0]),
    dict(d=8, inv_freq=[1.0, math.nan, 1.0, 1.0])])
def test_plan_refusals(args):
    with pytest.raises(ValueError):
        ops.rotary_plan(**args)


def test_oracle_turns_back():
    rng = np.random.default_rng(2)
    x, pos = rng.standard_normal((3, 2, 10)), np.array([[0, -7, 2**31 - 1], [5, 2**30, -2**31]])
    angle = oracle.angles(pos, oracle.plan_frequencies(6, 100.0), [0, 1, 1])
    for inter in (False, True):
        y, size = oracle.rotary(x, angle, 3, inter)
        back, _ = oracle.rotary(y, angle, 3, inter, inverse=True)
        assert np.abs(back - x).max() < 1e-14 and (y[..., :3] == x[..., :3]).all() and (y[..., 9:] == x[..., 9:]).all()
        assert (size[..., 3:9] > 0).all() and (size[..., 9:] == 0).all()


# ------------------------------------------------------------------ refusals of the C ABI, before any device call
P = 1 << 20  # a pointer that is never used


def _code(fn, desc):
    return getattr(capi.load(), fn)(ctypes.byref(desc), None)


def _reserve_desc(**kw):
    base = dict(pages=P, held=P, rows=P, pool=P, n_free=P, held_out=P, n_free_out=P, lens=P, cu_seqlens=P, positions=P, slots=P,
                n_seqs=4, width=8, pool_size=32, n_rows=9)
    return capi.make_cache_reserve_desc(**{**base, **kw})


@pytest.mark.parametrize("kw,code", [
    (dict(n_seqs=-1), -1), (dict(width=-1), -1), (dict(pool_size=-1), -1), (dict(n_rows=-1), -1), (dict(cu_seqlens=None), -1),
    (dict(n_seqs=8193), -2), (dict(n_seqs=8192, width=1 << 18), -2), (dict(pages_stride=7), -1), (dict(n_free=None), -1), (dict(n_free_out=None), -1),
    (dict(pool=None), -1), (dict(held=None), -1), (dict(rows=None), -1), (dict(held_out=None), -1), (dict(lens=None), -1),
    (dict(pages=None), -1), (dict(held=P + 2), -1), (dict(cu_seqlens=P + 1), -1), (dict(positions=P + 4), -1), (dict(slots=P + 8), -1)])
def test_reserve_refusals(kw, code):
    assert _code("nsa_cache_reserve", _reserve_desc(**kw)) == code and capi.last_error()


def _select_desc(batch=None, **kw):
    b = capi.make_cache_batch(**{**dict(cache=P, pages=P, lens=P, num_pages=8, n_seqs=3, width=4, n_rows=3, heads_kv=2, d_qk=128,
                                        d_v=128), **(batch or {})})
    return capi.make_cache_select_desc(**{**dict(batch=b, q=P, sel=P, workspace=P, heads_q=8, n_sel=16, block_size=64, cmp_block=32,
                                                 cmp_stride=16, q_dtype=capi.DTYPE_BF16), **kw})


@pytest.mark.parametrize("batch,kw,code", [
    (dict(d_qk=96), {}, -2), (dict(n_rows=4), {}, -1), (dict(heads_kv=0), {}, -1), (dict(pages_stride=3), {}, -1), ({}, dict(heads_q=7), -1),
    ({}, dict(heads_q=0), -1), ({}, dict(heads_q=514), -2), ({}, dict(q_dtype=1), -1), ({}, dict(n_sel=0), -1), ({}, dict(n_sel=1025), -2),
    ({}, dict(block_size=96), -2), ({}, dict(cmp_block=0), -1), ({}, dict(cmp_stride=0), -1), ({}, dict(q=None), -1), ({}, dict(sel=None), -1),
    ({}, dict(q=P + 8), -1), ({}, dict(q_row_stride=4), -1), ({}, dict(q_head_stride=12), -1), ({}, dict(sel=P + 2), -1),
    ({}, dict(workspace=None), -1), ({}, dict(workspace=P + 8), -1),
    (dict(heads_kv=16384, width=2**31 - 1, n_rows=1, n_seqs=1, d_qk=64, d_v=64), dict(heads_q=16384, cmp_stride=1), -2)])
def test_select_refusals(batch, kw, code):
    assert _code("nsa_cache_select", _select_desc(batch, **kw)) == code and capi.last_error()


def test_select_workspace():
    # T up to 64 * 4 * 16 + 31 = 4127 tokens, 65 blocks of 64, 8 bytes each
    assert capi.cache_select_workspace_bytes(_select_desc()) == 3 * 2 * 65 * 8
    assert capi.cache_select_workspace_bytes(_select_desc(block_size=256)) == 3 * 2 * 17 * 8
    assert capi.cache_select_workspace_bytes(_select_desc(dict(width=2**31 - 1))) == 3 * 2 * 2**18 * 8
    assert capi.cache_select_workspace_bytes(_select_desc(dict(n_rows=0, n_seqs=0))) == 16
    with pytest.raises(capi.NsaSelError):
        capi.cache_select_workspace_bytes(_select_desc(n_sel=0))


def _rotary_desc(t=None, **kw):
    turns, axis = (ctypes.c_uint64 * 128)(), (ctypes.c_uint8 * 128)(0, 1)
    d = capi.make_rotary_desc(**{**dict(positions=P, turns=ctypes.addressof(turns), axis=ctypes.addressof(axis), batch=1, tokens=5,
                                        d=64, offset=0, pairs=32, axes=2, dtype=0), **kw})
    for i, values in enumerate(t if t is not None else [dict(x=P, y=P, heads=4), {}]):
        for key, value in values.items():
            setattr(d.t[i], key, value)
    return d, turns, axis


@pytest.mark.parametrize("t,kw,code", [
    (None, dict(batch=-1), -1), (None, dict(tokens=-1), -1), (None, dict(dtype=5), -1), (None, dict(pairs=0), -1), (None, dict(pairs=33), -1),
    (None, dict(offset=-1), -1), (None, dict(offset=2), -1), (None, dict(d=258, pairs=129), -2), (None, dict(axes=0), -2), (None, dict(axes=5), -2),
    (None, dict(turns=None), -1), (None, dict(axes=1), -1), (None, dict(positions=None), -1), (None, dict(positions=P + 2), -1),
    ([dict(x=P, heads=4), {}], {}, -1), ([dict(x=P + 1, y=P, heads=4), {}], {}, -1), ([dict(x=P, y=P + 2, heads=4), {}], dict(dtype=1), -1),
    ([dict(x=P, y=P, heads=-1), {}], {}, -1), ([dict(heads=1), {}], {}, -1), ([dict(x=P, y=P, heads=65536), {}], {}, -2),
    (None, dict(batch=1 << 16, tokens=1 << 16), -2), (None, dict(pairs=2**31 - 1, offset=2**31 - 1), -1)])
def test_rotary_refusals(t, kw, code):
    d, *keep = _rotary_desc(t, **kw)
    assert _code("nsa_rotary", d) == code and capi.last_error()


def test_nothing_to_turn_is_no_call():
    for kw in (dict(tokens=0, positions=None), dict(batch=0)):
        d, *keep = _rotary_desc(**kw)
        assert _code("nsa_rotary", d) == capi.NSA_OK
    d, *keep = _rotary_desc([{}, {}])
    assert _code("nsa_rotary", d) == capi.NSA_OK
    assert _code("nsa_cache_select", _select_desc(dict(n_rows=0, n_seqs=0))) == capi.NSA_OK


def test_struct_layout_matches_header(tmp_path):
    mirrors = {"nsa_cache_reserve_desc": capi.NsaCacheReserveDesc, "nsa_cache_select_desc": capi.NsaCacheSelectDesc,
               "nsa_rotary_tensor": capi.NsaRotaryTensor, "nsa_rotary_desc": capi.NsaRotaryDesc}
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{capi.HEADER_PATH}"', "int main(void) {"]
    want = []
    for name, cls in mirrors.items():
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        want.append(ctypes.sizeof(cls))
        for f, _ in cls._fields_:
            lines.append(f'printf("%zu\\n", offsetof({name}, {f}));')
            want.append(getattr(cls, f).offset)
    (tmp_path / "layout.c").write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-o", str(tmp_path / "layout"), str(tmp_path / "layout.c")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout
    assert [int(x) for x in out.split()] == want


# ------------------------------------------------------------------ the torch ops refuse before any device call
def test_torch_ops_refuse_host_tensors():
    i32 = dict(dtype=torch.int32)
    pages, held = torch.zeros(3, 2, **i32), torch.ones(3, **i32)
    with pytest.raises(RuntimeError, match="pages must be an int32 CUDA tensor"):
        ops.cache_reserve(pages, held, held, held, held[:1])
    cache = ops.cache_alloc(4, 2, 128, 128, device="cpu")
    with pytest.raises(RuntimeError, match="cache must be a CUDA tensor"):
        ops.cache_select(torch.zeros(3, 8, 128, dtype=torch.bfloat16), cache, pages, held, 16)
    with pytest.raises(RuntimeError, match="must be bfloat16 or float16"):
        ops.cache_select(torch.zeros(3, 8, 128), cache, pages, held, 16)
    with pytest.raises(RuntimeError, match="Q must be a CUDA tensor"):
        ops.rotary(torch.zeros(3, 8, 128), None, held, ops.rotary_plan(128))


def test_decode_needs_compressed_keys_to_select():
    q, i32 = torch.zeros(2, 4, 64, dtype=torch.bfloat16), dict(dtype=torch.int32)
    cache = ops.cache_alloc(2, 1, 64, 64, device="cpu")
    with pytest.raises(ValueError, match="cmp_cache"):
        nsa.nsa_decode(q, cache, torch.zeros(2, 1, **i32), torch.ones(2, **i32))
