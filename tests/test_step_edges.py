"""Edges of a decode step's preparation without a GPU: the largest calls' index arithmetic and the whole numbers of the exact
scores, compiled for the host; sizes of workspaces."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

from nsa_hopper_b200 import capi

CSRC = os.path.join(capi.PKG_DIR, "csrc")
BIG = 2**31 - 1
FLAGS = ["g++", "-std=c++17", "-O1", "-ffp-contract=off", "-shared", "-fPIC", "-fsanitize=undefined", "-fno-sanitize-recover=all",
         f"-I{CSRC}"]


def _build(tmp_path_factory, name, text):
    d = tmp_path_factory.mktemp(name)
    (d / "shim.cpp").write_text(text)
    subprocess.run([*FLAGS, "-o", str(d / "shim.so"), str(d / "shim.cpp")], check=True)
    return ctypes.CDLL(str(d / "shim.so"))


# ------------------------------------------------------------------ rotary positions
ROTARY = r"""
#include "nsa_rotary_index.h"
using namespace nsa::rotary;
extern "C" {
// Tokens of a block, and whose angles it makes.
int32_t block(uint32_t at, int32_t tokens_block, int32_t total, int32_t* tokens, int32_t* angles) {
  const int32_t first = first_token(at, tokens_block);
  int32_t n = 0;
  for (int32_t i = 0; i < 256; ++i)
    if (has_token(first, i, tokens_block, total)) tokens[n++] = first + i;
  for (int32_t i = 0; i < tokens_block; ++i) angles[i] = token_or_last(first, i, total);
  return n;
}
}
"""


@pytest.fixture(scope="module")
def rotary_lib(tmp_path_factory):
    return _build(tmp_path_factory, "rotary", ROTARY)


@pytest.mark.parametrize("total", [1, 255, 1000, 2**31 - 257, BIG])
def test_rotary_blocks_end_with_the_last_token(rotary_lib, total):
    """As many tokens as a call may have (2^31 - 1) among blocks of 1 to 256: the last block's end may pass 2^31 - 1."""
    passed = 0
    for each in range(1, 257):
        last = -(-total // each) - 1
        for at in {0, last // 2, max(last - 1, 0), last}:
            tokens, angles = np.zeros(256, np.int32), np.zeros(each, np.int32)
            n = rotary_lib.block(at, each, total, tokens.ctypes.data_as(ctypes.c_void_p), angles.ctypes.data_as(ctypes.c_void_p))
            want = range(at * each, min((at + 1) * each, total))
            assert tokens[:n].tolist() == list(want)
            assert angles.tolist() == [min(at * each + i, total - 1) for i in range(each)]
        passed += (last + 1) * each > BIG + 1
    assert (passed > 100) == (total == BIG)


# ------------------------------------------------------------------ block selection
def _select_desc(**batch):
    b = capi.make_cache_batch(**{**dict(cache=1 << 20, pages=1 << 20, lens=1 << 20, num_pages=8, n_seqs=3, width=4, n_rows=3, heads_kv=2,
                                        d_qk=128, d_v=128), **batch})
    return capi.make_cache_select_desc(batch=b, q=1 << 20, sel=1 << 20, heads_q=b.heads_kv, n_sel=16, block_size=64, cmp_block=32,
                                       cmp_stride=16, q_dtype=capi.DTYPE_BF16)


def test_select_workspace_is_that_of_a_launch():
    """65 blocks of 64 in a table of 4 pages; rows of a launch are 1024 at most, and fewer where units of a row are many."""
    for rows, counted in ((1, 1), (1023, 1023), (1024, 1024), (1025, 1024), (100000, 1024)):
        assert capi.cache_select_workspace_bytes(_select_desc(n_rows=rows, n_seqs=rows)) == counted * 2 * 65 * 8
    # 2^18 blocks, a unit for 16 of them, 2048 heads: 2^25 units a row, 63 rows below 2^31
    wide = dict(width=2**31 - 1, heads_kv=2048)
    assert capi.cache_select_workspace_bytes(_select_desc(n_rows=500, n_seqs=500, **wide)) == 63 * 2048 * 2**18 * 8
    assert capi.cache_select_workspace_bytes(_select_desc(n_rows=5, n_seqs=5, **wide)) == 5 * 2048 * 2**18 * 8


SELECT = r"""
#include <string.h>
#include "nsa_cache_select_index.h"
using namespace nsa::cache_select;
extern "C" {
uint32_t decode(uint32_t codes) { return decode4(codes); }
uint32_t scale(uint32_t byte) { return scale_high(byte); }
void bytes(int64_t x, int8_t* out) { for (int i = 0; i < 6; ++i) out[i] = next_byte(x); }
// The sum of 16 products, from the query's bytes and codes in words of eight: what the kernel's threads do.
int64_t group(const int64_t* q, const uint32_t* words) {
  uint32_t limb[6][4], codes[4], up = 0, lo = 0;
  for (int d = 0; d < 16; ++d) {
    int64_t x = q[d];
    for (int l = 0; l < 6; ++l) reinterpret_cast<int8_t*>(limb[l])[d] = next_byte(x);
  }
  for (int i = 0; i < 4; ++i) codes[i] = decode4(words[i / 2] >> i % 2 * 16);
  for (int l = 5; l >= 3; --l) up = add_group(up, codes, limb[l]);
  for (int l = 2; l >= 0; --l) lo = add_group(lo, codes, limb[l]);
  up += too_many(limb[3], limb[4], limb[5]), lo += too_many(limb[0], limb[1], limb[2]);
  return (int64_t)(int32_t)up * 16777216 + (int32_t)lo;
}
}
"""
DOUBLED = [0, 1, 2, 3, 4, 6, 8, 12, 0, -1, -2, -3, -4, -6, -8, -12]


@pytest.fixture(scope="module")
def select_lib(tmp_path_factory):
    lib = _build(tmp_path_factory, "select", SELECT)
    lib.decode.restype = lib.scale.restype = ctypes.c_uint32
    lib.group.restype = ctypes.c_int64
    return lib


def test_codes_become_whole_numbers(select_lib):
    for word in range(1 << 16):
        got = select_lib.decode(ctypes.c_uint32(word))
        assert all((got >> 8 * i & 255) - 12 == DOUBLED[word >> 4 * i & 15] for i in range(4))
        if word % 251 == 0:  # (what stands above four codes is not looked at)
            assert select_lib.decode(ctypes.c_uint32(word | 0xABCD0000)) == got


def test_scale_bytes_become_fp64(select_lib):
    """Every byte of a normal number: the fp16 of which it is the upper part, in the upper half of an fp64."""
    for byte in range(8, 256):
        want = np.float64(np.array([byte << 7], np.uint16).view(np.float16)[0])
        got = np.array([select_lib.scale(byte) << 32], np.uint64).view(np.float64)[0]
        assert got == want or not (np.isfinite(want) or np.isfinite(got)), byte


def test_signed_bytes_of_sums(select_lib):
    rng = np.random.default_rng(11)
    for x in [0, 1, -1, 127, 128, -128, -129, 2**46, -2**46, 2**46 - 1] + [int(v) for v in rng.integers(-2**46, 2**46, 500)]:
        out = np.zeros(6, np.int8)
        select_lib.bytes(ctypes.c_int64(x), out.ctypes.data_as(ctypes.c_void_p))
        assert sum(int(b) << 8 * i for i, b in enumerate(out)) == x


def test_sums_of_a_group_are_exact(select_lib):
    """Queries up to 2^46 in size (the bytes' largest sums among them) times all codes; 256 sequences of codes each."""
    rng = np.random.default_rng(12)
    worst = sum(127 << 8 * i for i in range(5)) + (63 << 40)  # (every byte as large as it gets below 2^46)
    queries = [np.full(16, s * x, np.int64) for x in (2**46, 2**46 - 1, worst, 1, 0) for s in (1, -1)]
    queries += [np.where(rng.random(16) < 0.5, worst, -worst), *rng.integers(-2**46, 2**46, (20, 16)), *rng.integers(-300, 300, (5, 16))]
    for q in queries:
        q = np.ascontiguousarray(q, np.int64)
        words = rng.integers(0, 2**32, (256, 2), dtype=np.uint32)
        words[:4] = [[0x77777777] * 2, [0xFFFFFFFF] * 2, [0, 0], [0x89ABCDEF, 0x76543210]]
        for w in words:
            codes = [DOUBLED[int(w[i // 8]) >> 4 * (i % 8) & 15] for i in range(16)]
            got = select_lib.group(q.ctypes.data_as(ctypes.c_void_p), w.ctypes.data_as(ctypes.c_void_p))
            assert got == sum(int(a) * b for a, b in zip(q, codes))
