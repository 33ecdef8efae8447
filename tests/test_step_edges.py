"""Edges of a decode step's preparation without a GPU: the largest calls' index arithmetic, compiled for the host."""
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
