"""The 4-bit paged KV cache without a GPU: the index arithmetic that the kernels share (compiled for the
host and fed broken tables), the plan, the checks of arguments, the number format."""
import ctypes
import os
import subprocess

import numpy as np
import pytest
import torch

from nsa_hopper_b200 import capi, nsa, ops
from oracle import cache as oc

CSRC = os.path.join(capi.PKG_DIR, "csrc")

SHIM = r"""
#include "nsa_cache_index.h"
using namespace nsa::cache;
extern "C" {
static Batch make(const int32_t* pages, const int32_t* lens, const int32_t* cu, int n_seqs, int width, int num_pages, int n_rows) {
  return {pages, lens, cu, width, n_seqs, width, num_pages, n_rows};
}
void locate(const int32_t* pages, const int32_t* lens, const int32_t* cu, int n_seqs, int width, int num_pages, int n_rows,
            int32_t* out) {
  const Batch b = make(pages, lens, cu, n_seqs, width, num_pages, n_rows);
  for (int r = 0; r < n_rows; ++r) {
    const int seq = sequence_of(b, r), pos = seq < 0 ? -1 : position_of(b, seq, r);
    out[4 * r] = seq, out[4 * r + 1] = pos;
    out[4 * r + 2] = pos < 0 ? -1 : page_of(b, seq, pos / kPage);
    out[4 * r + 3] = keys_up_to(b, pos);
  }
}
int selected(int entry, int part, int per, int first, int end) { return selected_sub(entry, part, per, first, end); }
int running(int j, int first, int end) { return running_sub(j, first, end); }
int slots(int first, int end) { return running_slots(first, end); }
int first(int pos, int window) { return first_key(pos, window); }
void split(uint32_t rows, uint32_t total, uint32_t longest, uint32_t warps, uint32_t* out) {
  const Split s = split_line(rows, total, longest, warps);
  out[0] = s.team, out[1] = s.share, out[2] = s.cut, out[3] = may_cut(rows, longest, warps), out[4] = cluster_of(rows, longest, warps);
}
int record(int dqk, int dv) { return record_bytes(dqk, dv); }
}
"""


@pytest.fixture(scope="module")
def index(tmp_path_factory):
    d = tmp_path_factory.mktemp("index")
    (d / "shim.cpp").write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                    f"-I{CSRC}", "-o", str(d / "shim.so"), str(d / "shim.cpp")], check=True)
    return ctypes.CDLL(str(d / "shim.so"))


def _locate(lib, pages, lens, cu, num_pages, n_rows):
    out = np.zeros((n_rows, 4), np.int32)
    ptr = lambda a: None if a is None else a.ctypes.data_as(ctypes.c_void_p)  # noqa: E731
    lib.locate(ptr(pages), ptr(lens), ptr(cu), len(lens), pages.shape[1], num_pages, n_rows, ptr(out))
    return out


BIG = 2**31 - 1


@pytest.mark.parametrize("cu", [
    None,
    [0, 1, 1, 4, 9],                 # an empty sequence, rows behind the last
    [0, 0, 0, 0, 0],                 # no rows at all
    [2, 3, 5, 6, 11],                # rows before the first
    [0, 7, 3, 5, 12],                # not in order
    [0, BIG, BIG, BIG, BIG],         # behind every row
    [-5, -3, 0, 2, 3],               # negative
    [12, 9, 5, 2, 0],                # backwards
])
@pytest.mark.parametrize("lens", [[0, 1, 64, 130], [-7, 63, 65, BIG], [256, 257, 10**9, 128]])
def test_rows_land_inside_the_cache_or_nowhere(index, cu, lens):
    width, num_pages, n_rows = 4, 6, 4 if cu is None else 12
    pages = np.array([[0, 5, 6, -1], [3, -2**31, BIG, 2], [1, 4, 0, 2], [5, 5, -1, 7]], np.int32)
    lens, cu = np.array(lens, np.int32), None if cu is None else np.array(cu, np.int32)
    got = _locate(index, pages, lens, cu, num_pages, n_rows)
    for r, (seq, pos, page, keys) in enumerate(got.tolist()):
        assert -1 <= seq < 4 and -1 <= page < num_pages and 0 <= keys <= width * 64
        if seq >= 0:
            assert cu is None or cu[seq] <= r < cu[seq + 1]
            assert page == (-1 if pos < 0 or pos >= width * 64 or not 0 <= pages[seq, pos // 64] < num_pages
                            else pages[seq, pos // 64])
            assert keys == min(max(pos + 1, 0), width * 64)
        if cu is None or (np.diff(cu) >= 0).all():
            assert (seq, pos if seq >= 0 else -1, page) == oc.place(r, pages, lens, cu, num_pages)


def test_sub_blocks(index):
    # selection: nothing behind the visible keys or before the window, no overflow for any entry
    for entry in (-2**31, -1, 0, 1, 2, 3, 7, 2**24, BIG):
        for per in (1, 2, 4):
            for part in range(per):
                for first, end in ((0, 0), (0, 1), (0, 64), (0, 65), (100, 300), (255, 256), (0, BIG // 64 * 64)):
                    sub = index.selected(entry, part, per, first, end)
                    want = entry * per + part
                    ok = entry >= 0 and want * 64 < end and (want + 1) * 64 > first
                    assert sub == (want if ok else -1), (entry, per, part, first, end)
    for first, end in ((0, 0), (0, 1), (63, 64), (63, 65), (64, 65), (100, 300), (0, 640)):
        n = index.slots(first, end)
        subs = [index.running(j, first, end) for j in range(n + 2)]
        want = [s for s in range(11) if s * 64 < end and (s + 1) * 64 > first] if end > first else []
        assert n == max(1, len(want)) and subs == want + [-1] * (n + 2 - len(want))
    assert [index.first(p, w) for p, w in ((5, 0), (5, 1), (5, 6), (5, 7), (5, BIG), (BIG - 1, 3))] == [0, 5, 0, 0, 0, BIG - 3]


def test_sub_blocks_of_the_longest_sequences(index):
    """Positions up to 2^31 - 2: the last sub-block ends at 2^31, which no int holds."""
    top = 2**31 - 1  # keys
    for per in (1, 2, 4):
        for first in (0, top - 1, top - 64, top - 100):
            for entry in range((top - 1) // (64 * per) - 1, (top - 1) // (64 * per) + 2):
                for part in range(per):
                    sub = entry * per + part
                    want = sub if sub * 64 < top and (sub + 1) * 64 > first else -1
                    assert index.selected(entry, part, per, first, top) == want, (per, first, entry, part)
    for first in (0, top - 64):
        assert index.running((top - 1) // 64 - first // 64, first, top) == 2**25 - 1
        assert index.running((top - 1) // 64 - first // 64 + 1, first, top) == -1


def test_shares_cover_the_line(index):
    rng = np.random.default_rng(0)
    warps = 148 * 8
    for i in range(4000):
        rows = int(np.exp(rng.uniform(0, np.log(5000))))
        longest = int(np.exp(rng.uniform(0, np.log(min(40000, (2**31 - 1) // rows)))))
        total = rows * longest if i % 2 else int(rng.integers(rows + longest - 1, rows * longest + 1))
        out = (ctypes.c_uint32 * 5)()
        index.split(rows, total, longest, warps, out)
        team, share, cut, may, cluster = out
        assert cluster in (1, 2, 4, 8)
        if cluster > 1:
            assert rows * cluster <= 148 and cluster * 4 <= longest <= 5 * 8 * cluster
        assert team in (1, 2, 4, 8) and share >= 1
        teams = warps // team
        if cut:
            assert may and share * teams >= total
        else:
            assert share * teams >= rows
        # a shorter longest row of the same rows is never cut where the host has said that none is
        if not may:
            for shorter in (x for x in {1, 2, 3, 5, longest // 2, longest - 1} if 0 < x < longest):
                index.split(rows, min(total, rows * shorter), shorter, warps, out)
                assert not out[2]
        # a warp never gets more slots than it would with whole rows of its own
        slots = -(-share // team) if cut else share * -(-longest // team)
        assert slots <= -(-rows // warps) * longest


def test_record_bytes():
    for dqk, dv, want in ((64, 64, 4608), (128, 128, 9216), (192, 128, 11520), (128, 64, 6912)):
        assert capi.cache_record_bytes(dqk, dv) == want
    assert capi.cache_record_bytes(96, 96) == -1
    assert capi.cache_record_bytes(64, 128) == -1


# ------------------------------------------------------------------ number format
def test_format_by_definition():
    s = oc._SCALES
    assert s[0] == 0 and s[1] == 2.0**-17 and s[8] == 2.0**-14 and s[-1] == 10240 and (np.diff(s) > 0).all()
    assert (s.astype(np.float16) == s).all() and ((6 * s).astype(np.float16) == 6 * s).all()
    every = (oc.LEVELS[:, None] * s).astype(np.float32)
    assert (torch.from_numpy(every).to(torch.bfloat16).float().numpy() == every).all()
    assert (every.astype(np.float16).astype(np.float32) == every).all()
    x = np.zeros((1, 16))
    x[0, :9] = [6, 0.25, 0.75, 1.25, -1.75, 2.5, 3.5, 5, -0.2]  # scale 1; ties go to the even code
    code, byte = oc.quantise(x)
    assert oc.scale_value(byte)[0, 0] == 1
    assert (oc.values(code, byte)[0, :9] == [6, 0, 1, 1, -2, 2, 4, 4, 0]).all()
    x[0, 3] = np.nan
    assert np.isnan(oc.values(*oc.quantise(x))).all()
    assert (oc.values(*oc.quantise(np.full((1, 16), 1e30))) == 61440).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_quantising_without_divisions_is_exact(dtype):
    """The kernel's arithmetic, restated in numpy's fp32, against the definition: every finite value of the type as a
    group's largest, and every value below each scale's saturation, with the approximate reciprocal off either way."""
    every = torch.arange(0x7F80 if dtype == torch.bfloat16 else 0x7C00, dtype=torch.int16).view(dtype).float().numpy()
    raw = ((every * np.float32(0.16666667)).view(np.uint32) + np.uint32(0x40)) & np.uint32(0xFFFFFF80)
    big = raw.view(np.float32) >= np.float32(2.0**-14)
    normal = np.minimum(((raw + np.uint32(0x7FFFF) + ((raw >> 20) & 1)) >> 20).astype(np.int64) - 896, 226)
    byte = np.where(big, normal, np.rint(np.where(big, 0, raw.view(np.float32)).astype(np.float64) * 2.0**17).astype(np.int64))
    want = oc._nearest_even(every.astype(np.float64) / 6.0, oc._SCALES)
    np.testing.assert_array_equal(byte, want)
    for b in range(1, 0xE3):
        s = oc._SCALES[b]
        x = every[(every <= 6.8 * s) & (every >= 0.2 * s)].astype(np.float64)
        want = oc._nearest_even(x / s, oc.LEVELS)
        for off in (-1, 0, 1):  # 2^-22: the reciprocal's error and the input's
            inv = float(np.float32((1 / s) * (1 + off * 2.0**-22)))
            y = ((x * inv + 192).astype(np.float32) - np.float32(192)).astype(np.float64)
            np.testing.assert_array_equal(oc._nearest_even(np.maximum(y, 0), oc.LEVELS), want)


# ------------------------------------------------------------------ plan and refusals of the C ABI
def _batch(**kw):
    base = dict(cache=256, pages=256, lens=256, num_pages=1000, n_seqs=8, width=64, n_rows=8, heads_kv=4, d_qk=128, d_v=128)
    base.update(kw)
    return capi.make_cache_batch(**base)


def _attend(batch=None, **kw):
    base = dict(q=256, o=256, heads_q=64, q_dtype=capi.DTYPE_BF16, o_dtype=capi.DTYPE_BF16)
    base.update(kw)
    return capi.make_cache_attend_desc(batch=_batch(**(batch or {})), **base)


def test_plan_shares_out_the_work():
    p = capi.cache_attend_plan(_attend(sel=256, n_sel=16, block_size=64))     # 32 rows, a cluster of 4 blocks for each
    assert (p["slots"], p["team"], p["cluster"], p["share"], p["grid"], p["merge"], p["workspace_bytes"]) == (16, 8, 4, 1, 128, 0, 16)
    p = capi.cache_attend_plan(_attend(dict(n_rows=32, n_seqs=32), sel=256, n_sel=16, block_size=64))
    assert (p["team"], p["cluster"], p["share"], p["grid"]) == (8, 1, 1, 128)  # 128 rows, a block for each
    assert p["smem_bytes"] <= 232448
    p = capi.cache_attend_plan(_attend(dict(n_rows=256, n_seqs=256), sel=256, n_sel=16, block_size=64))
    assert (p["team"], p["share"], p["grid"], p["merge"]) == (1, 1, 148, 0)    # a warp for each row
    p = capi.cache_attend_plan(_attend())                                      # every key, 64 pages
    assert (p["slots"], p["cluster"], p["grid"], p["merge"]) == (64, 4, 128, 0)
    p = capi.cache_attend_plan(_attend(dict(width=1500)))
    assert p["slots"] == 0 and p["share"] == 0 and p["merge"] >= 1 and p["workspace_bytes"] > 16
    p = capi.cache_attend_plan(_attend(dict(n_rows=30, n_seqs=30, width=16)))  # short rows are not cut
    assert p["slots"] == 16 and p["merge"] == 0 and p["cluster"] == 1
    p = capi.cache_attend_plan(_attend(dict(n_rows=4096, n_seqs=4096)))        # too many rows for it
    assert p["slots"] == 64
    p = capi.cache_attend_plan(_attend(window=1))
    assert p["slots"] == 1 and p["team"] == 1
    p = capi.cache_attend_plan(_attend(window=66, heads_q=4 * 17))
    assert p["slots"] == 3 and p["tiles"] == 2 and p["team"] == 4
    p = capi.cache_attend_plan(_attend(dict(n_rows=1, n_seqs=1, width=2048)))
    assert p["merge"] == 8                                                     # one row over many blocks
    for d in ((64, 64), (192, 128), (128, 64)):
        assert capi.cache_attend_plan(_attend(dict(d_qk=d[0], d_v=d[1])))["smem_bytes"] <= 232448
    p = capi.cache_attend_plan(_attend(dict(n_rows=0, n_seqs=0)))
    assert p["grid"] == 0 and p["workspace_bytes"] == 16


BAD = [
    (dict(d_qk=96), {}, capi.NSA_ERR_UNSUPPORTED),
    (dict(heads_kv=0), {}, capi.NSA_ERR_INVALID_ARG),
    (dict(n_rows=7), {}, capi.NSA_ERR_INVALID_ARG),               # no cu_seqlens: one row a sequence
    (dict(cache=0), {}, capi.NSA_ERR_INVALID_ARG),
    (dict(cache=264), {}, capi.NSA_ERR_INVALID_ARG),
    (dict(pages=0), {}, capi.NSA_ERR_INVALID_ARG),
    (dict(lens=258), {}, capi.NSA_ERR_INVALID_ARG),
    (dict(page_stride=4 * 9216 - 16), {}, capi.NSA_ERR_INVALID_ARG),
    (dict(page_stride=4 * 9216 + 8), {}, capi.NSA_ERR_INVALID_ARG),
    (dict(pages_stride=63), {}, capi.NSA_ERR_INVALID_ARG),
    (dict(n_rows=2**28, n_seqs=2**28), {}, capi.NSA_ERR_UNSUPPORTED),
]
BAD_ATTEND = BAD + [
    ({}, dict(heads_q=63), capi.NSA_ERR_INVALID_ARG),
    ({}, dict(q=0), capi.NSA_ERR_INVALID_ARG),
    ({}, dict(q=264), capi.NSA_ERR_INVALID_ARG),
    ({}, dict(q_row_stride=12), capi.NSA_ERR_INVALID_ARG),
    ({}, dict(o=0), capi.NSA_ERR_INVALID_ARG),
    ({}, dict(q_dtype=capi.DTYPE_F32), capi.NSA_ERR_INVALID_ARG),
    ({}, dict(o_dtype=capi.DTYPE_F16), capi.NSA_ERR_INVALID_ARG),
    ({}, dict(o_accumulate=1), capi.NSA_ERR_INVALID_ARG),
    ({}, dict(window=-1), capi.NSA_ERR_INVALID_ARG),
    ({}, dict(sel=256, n_sel=0, block_size=64), capi.NSA_ERR_INVALID_ARG),
    ({}, dict(sel=256, n_sel=16, block_size=96), capi.NSA_ERR_UNSUPPORTED),
    ({}, dict(sel=256, n_sel=1025, block_size=64), capi.NSA_ERR_UNSUPPORTED),
    (dict(n_rows=2**20, n_seqs=2**20, width=2**10), {}, capi.NSA_ERR_UNSUPPORTED),  # 2^32 slots
]


@pytest.mark.parametrize("batch,kw,code", BAD_ATTEND)
def test_attend_refusals(batch, kw, code):
    with pytest.raises(capi.NsaSelError) as e:
        capi.cache_attend_plan(_attend(batch, **kw))
    assert e.value.code == code and capi.last_error() != ""
    assert capi.load().nsa_cache_attend(ctypes.byref(_attend(batch, **kw)), None) == code


@pytest.mark.parametrize("batch,kw,code", BAD + [
    ({}, dict(k=0), capi.NSA_ERR_INVALID_ARG),
    ({}, dict(v=264), capi.NSA_ERR_INVALID_ARG),
    ({}, dict(strides=(512, 128, 513, 128)), capi.NSA_ERR_INVALID_ARG),
    ({}, dict(dtype=capi.DTYPE_F32), capi.NSA_ERR_INVALID_ARG),
])
def test_write_and_read_refusals(batch, kw, code):
    a = dict(k=256, v=256, strides=(512, 128, 512, 128), dtype=capi.DTYPE_BF16)
    a.update(kw)
    b = _batch(**batch)
    lib = capi.load()
    ptr = ctypes.c_void_p
    assert lib.nsa_cache_write(ctypes.byref(b), ptr(a["k"]), ptr(a["v"]), *a["strides"], a["dtype"], None) == code
    if "strides" not in kw and "dtype" not in kw:
        assert lib.nsa_cache_read(ctypes.byref(b), ptr(a["k"]), ptr(a["v"]), a["dtype"], None) == code
    assert lib.nsa_cache_read(ctypes.byref(_batch()), ptr(256), ptr(256), 7, None) == capi.NSA_ERR_INVALID_ARG
    assert lib.nsa_cache_read(ctypes.byref(_batch()), ptr(256), ptr(272), 0, None) == capi.NSA_ERR_INVALID_ARG


def test_struct_layout_matches_header(tmp_path):
    mirrors = {"nsa_cache_batch": capi.NsaCacheBatch, "nsa_cache_attend_desc": capi.NsaCacheAttendDesc,
               "nsa_cache_attend_plan_info": capi.NsaCacheAttendPlanInfo}
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{capi.HEADER_PATH}"', "int main(void) {"]
    want = []
    for name, cls in mirrors.items():
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        want.append(ctypes.sizeof(cls))
        for f, _ in cls._fields_:
            lines.append(f'printf("%zu\\n", offsetof({name}, {f}));')
            want.append(getattr(cls, f).offset)
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-o", str(tmp_path / "layout"), str(src)], check=True)
    out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout
    assert [int(x) for x in out.split()] == want


# ------------------------------------------------------------------ the torch ops refuse before any device call
def test_torch_ops_refuse_host_tensors():
    cache = ops.cache_alloc(4, 2, 128, 128, device="cpu")
    assert cache.shape == (4, 2, 9216) and cache.dtype == torch.uint8
    pages, lens = torch.zeros(3, 2, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    k = torch.zeros(3, 2, 128, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="cache must be a CUDA tensor"):
        ops.cache_write(cache, k, k, pages, lens)
    with pytest.raises(RuntimeError, match="cache must be a CUDA tensor"):
        ops.cache_read(cache, 128, pages, lens)
    with pytest.raises(RuntimeError, match="cache must be a CUDA tensor"):
        ops.cache_attend(torch.zeros(3, 8, 128, dtype=torch.bfloat16), cache, pages, lens)
    with pytest.raises(RuntimeError, match="must be bfloat16 or float16"):
        ops.cache_write(cache, k.float(), k.float(), pages, lens)
    with pytest.raises(RuntimeError, match="one dtype"):
        ops.cache_write(cache, k, k.half(), pages, lens)
    with pytest.raises(RuntimeError, match="dtype must be"):
        ops.cache_read(cache, 128, pages, lens, dtype=torch.float64)
    with pytest.raises(ValueError, match="n_tokens"):
        ops.cache_read(cache, 128, pages, lens, cu_seqlens=lens)
    with pytest.raises(RuntimeError, match="not one of"):
        ops.cache_alloc(4, 2, 96, 96, device="cpu")


# ------------------------------------------------------------------ compressed keys as tokens come
class _Model:
    """cache_write and cache_read on fp32 places [pages, Hkv, 64, d_qk + d_v], row by row through the oracle's `place`."""

    @staticmethod
    def write(cache, K, V, pages, lens, cu_seqlens=None):
        cu = None if cu_seqlens is None else cu_seqlens.numpy()
        for r in range(K.shape[0]):
            _, pos, page = oc.place(r, pages.numpy(), lens.numpy(), cu, cache.shape[0])
            if page >= 0:
                cache[page, :, pos % 64, :2] = torch.cat((K[r], V[r]), -1).float()

    @staticmethod
    def read(cache, d_qk, pages, lens, cu_seqlens, n_tokens, dtype):
        out = torch.zeros(cache.shape[1], n_tokens, 2)
        for r in range(n_tokens):
            _, pos, page = oc.place(r, pages.numpy(), lens.numpy(), cu_seqlens.numpy(), cache.shape[0])
            if page >= 0:
                out[:, r] = cache[page, :, pos % 64, :2]
        return out[None, ..., :1], out[None, ..., 1:]


@pytest.mark.parametrize("block,stride", [(32, 16), (8, 8), (4, 6), (1, 1), (16, 5)])
@pytest.mark.parametrize("chunk", [1, 10**9])
def test_every_completed_key_is_compressed(monkeypatch, block, stride, chunk):
    """Prompts, steps of one token and of several: every key that cache_compress counts is the mean of its tokens, all other
    places keep what they held."""
    monkeypatch.setattr(ops, "cache_write", _Model.write)
    monkeypatch.setattr(ops, "cache_read", _Model.read)
    monkeypatch.setattr(nsa, "COMPRESS_VALUES", chunk)
    rng = np.random.default_rng(block * 100 + stride)
    S, W, P = 4, 4, 20
    i32 = dict(dtype=torch.int32)
    pages = torch.from_numpy(rng.permutation(P)[:S * W].reshape(S, W)).int()
    cmp_pages = torch.from_numpy(rng.permutation(P)[:S * W].reshape(S, W)).int()
    cache, cmp_cache = torch.zeros(P, 1, 64, 36), torch.full((P, 1, 64, 36), -1000.0)  # (36: as wide as d = 1 in records)
    tokens = torch.from_numpy(rng.integers(-8, 9, (S, W * 64, 2))).float()             # (sums of them are exact)
    lens = torch.zeros(S, **i32)
    while int(lens.min()) < W * 64 - 40:
        if rng.random() < 0.3:   # one token each, no cu_seqlens
            new, cu, n = np.ones(S, int), None, None
        else:                    # several, or a prompt; rows of no sequence behind them
            new = np.minimum(rng.choice([0, 1, 3, 17, 40]) * rng.integers(0, 2, S), W * 64 - lens.numpy())
            cu, n = torch.tensor([0, *np.cumsum(new)], **i32), int(new.sum()) + int(rng.integers(0, 3))
        old, lens = lens, (lens + torch.from_numpy(new).int()).clamp(max=W * 64)
        rows = [tokens[s, int(old[s]):int(lens[s])] for s in range(S)] if cu is not None else \
            [tokens[s, int(lens[s]) - 1:int(lens[s])] for s in range(S)]
        flat = torch.cat(rows + [torch.full((0 if n is None else n - int(cu[-1]), 2), 77.0)])[:, None]
        ops.cache_write(cache, flat[..., :1], flat[..., 1:], pages, lens, cu)
        count = nsa.cache_compress(cache, 1, pages, lens, cmp_cache, cmp_pages, block, stride, cu, n)
        assert count.dtype == torch.int32
        want = torch.full_like(cmp_cache, -1000.0)
        for s in range(S):
            m = max(0, (int(lens[s]) - block) // stride + 1)
            assert int(count[s]) == m
            for i in range(min(m, W * 64)):
                want[cmp_pages[s, i // 64], 0, i % 64, :2] = tokens[s, i * stride:i * stride + block].mean(0).bfloat16().float()
        assert torch.equal(cmp_cache, want)


def test_compress_takes_broken_batches(monkeypatch):
    """More rows than tokens, rows before the first sequence, cu_seqlens behind the call's rows or out of order, negative and
    huge lengths: what a call writes is the mean of tokens that its rows complete."""
    monkeypatch.setattr(ops, "cache_write", _Model.write)
    monkeypatch.setattr(ops, "cache_read", _Model.read)
    i32 = dict(dtype=torch.int32)
    pages = torch.tensor([[0, 1], [2, 3], [-1, 99]], **i32)
    cache = torch.arange(4.0).view(4, 1, 1, 1) * 64 + torch.arange(64.0).view(1, 1, 64, 1) + torch.zeros(4, 1, 64, 36)
    for lens, cu, n in (([40, 128, 70], [0, 60, 61, 70], 80), ([40, 50, 60], [5, 9, 30, 31], 33), ([40, BIG, -5], [0, 40, 60, 90], 50),
                        ([33, 128, 64], [30, 3, 60, 10], 40), ([BIG, BIG, BIG], [0, BIG, BIG, BIG], 20),
                        ([48, 64, 0], [-7, 9, 40, 40], 40)):
        cmp_cache = torch.full((4, 1, 64, 36), -1000.0)
        lens, cu = torch.tensor(lens, **i32), torch.tensor(cu, **i32)
        count = nsa.cache_compress(cache, 1, pages, lens, cmp_cache, pages, 8, 4, cu, n)
        assert count.tolist() == [(x - 8) // 4 + 1 if x >= 8 else 0 for x in lens.tolist()]
        for p in range(4):
            for t in range(64):
                i, got = p % 2 * 64 + t, cmp_cache[p, 0, t, 0]
                if got != -1000:  # key i of sequence p // 2, of tokens 4 i to 4 i + 7
                    keys = [cache[pages[p // 2, x // 64], 0, x % 64, 0] if x < 128 else torch.tensor(0.0) for x in range(4 * i, 4 * i + 8)]
                    assert got == torch.stack(keys).mean().bfloat16()
        if (np.diff(cu.numpy()) >= 0).all():  # every key that a row completes is there
            for r in range(n):
                seq, pos, page = oc.place(r, pages.numpy(), lens.numpy(), cu.numpy(), 4)
                if page >= 0 and pos >= 7 and (pos - 7) % 4 == 0:
                    i = (pos - 7) // 4
                    assert cmp_cache[pages[seq, i // 64], 0, i % 64, 0] != -1000
    assert nsa.cache_compress(cache, 1, pages[:0], lens[:0], cmp_cache, pages[:0], 8, 4, torch.tensor([3], **i32), 9).shape == (0,)
    for kw in (dict(cu_seqlens=cu), dict(cu_seqlens=cu, n_tokens=-1), dict(cmp_stride=0), dict(cmp_block=0)):
        with pytest.raises(ValueError):
            nsa.cache_compress(cache, 1, pages, lens, cmp_cache, pages, **kw)


def test_decode_refuses_what_has_no_branch():
    """A window of 0 is no window to cache_attend (every key), but the window branch of 0 keys has none."""
    q, i32 = torch.zeros(2, 4, 64, dtype=torch.bfloat16), dict(dtype=torch.int32)
    cache, pages, lens = ops.cache_alloc(2, 1, 64, 64, device="cpu"), torch.zeros(2, 1, **i32), torch.ones(2, **i32)
    sel = torch.zeros(2, 1, 1, **i32)
    for kw in (dict(window=0), dict(window=-3), dict(cmp_cache=cache), dict(cmp_cache=cache, cmp_pages=pages)):
        with pytest.raises(ValueError, match="window|cmp_pages"):
            nsa.nsa_decode(q, cache, pages, lens, sel, **kw)


# ------------------------------------------------------------------ the search that a warp does
SHIM_32 = r"""
#include "nsa_cache_index.h"
using namespace nsa::cache;
extern "C" void both(const int32_t* cu, int n_seqs, const int32_t* rows, int n, int32_t* out) {
  const Batch b = {nullptr, nullptr, cu, 0, n_seqs, 0, 0, 0};
  for (int i = 0; i < n; ++i) {
    out[2 * i] = sequence_of(b, rows[i]);
    out[2 * i + 1] = sequence_by_32(b, rows[i], [&](int lo, int step, int hi) {
      uint32_t bits = 0;
      for (int lane = 0; lane < 32; ++lane) bits |= (uint32_t)(lane * step < hi - lo && cu[lo + lane * step] <= rows[i]) << lane;
      return bits;
    });
  }
}
"""


def test_a_thread_and_a_warp_find_a_rows_sequence(tmp_path):
    """The same in any cu_seqlens that is in order; out of order, one whose range holds the row, or none."""
    (tmp_path / "both.cpp").write_text(SHIM_32)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-fPIC", "-shared", f"-I{CSRC}",
                    "-o", str(tmp_path / "both.so"), str(tmp_path / "both.cpp")], check=True)
    lib = ctypes.CDLL(str(tmp_path / "both.so"))
    rng = np.random.default_rng(1)
    ptr = lambda a: a.ctypes.data_as(ctypes.c_void_p)  # noqa: E731
    for i in range(600):
        S = int(rng.choice([0, 1, 2, 31, 32, 33, 40, 64, 65, 1000, 1024, 1025, 3000]))
        if i % 3 == 0:
            cu = np.concatenate(([rng.integers(0, 3)], rng.integers(0, 4, S))).cumsum()
        elif i % 3 == 1:
            cu = rng.integers(-5, S + 5, S + 1)                        # in no order
        else:
            cu = np.arange(S + 1) * 2
            at = rng.integers(0, S + 1, 3)
            cu[at] = rng.choice([-2**31, BIG, 0, S], 3)                # a few entries broken
        cu = cu.astype(np.int32)
        rows = np.concatenate((rng.integers(0, 2 * S + 4, 40), [0, BIG])).astype(np.int32)
        out = np.zeros((len(rows), 2), np.int32)
        lib.both(ptr(cu), S, ptr(rows), len(rows), ptr(out))
        for r, found in zip(rows.tolist(), out.tolist()):
            for s in found:
                assert -1 <= s < S and (s < 0 or cu[s] <= r < cu[s + 1])
                if i % 3 == 0:
                    at = np.nonzero(cu[:-1] <= r)[0]
                    assert s == (at[-1] if at.size and r < cu[at[-1] + 1] else -1)
