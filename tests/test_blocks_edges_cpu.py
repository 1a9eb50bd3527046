"""Bucket attention without a GPU: offsets that the kernels look up against the extent of their bias table."""
import ctypes
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "grad-tts_amd", "csrc")

# Every 32 x 32 block that a wave of 32 consecutive positions pmin .. pmax visits, over the kernels' tiles: `last` keys
# end the visit (causal: the wave's last position + 1), a tile of `kt` keys is entered if the wave's first block of it
# begins before that, and then all of the wave's `nb` blocks in it are scored, `step` keys apart. Returns how many blocks
# read the table outside its extent; rule 0 is the kernels' own, rule 1 one that asks for dmin >= dsat alone.
SOURCE = r"""
#include "battn_index.h"
extern "C" long outside(int dsat, int causal, int kt, int nb, int step, int span, int rule, int* blocks) {
  using namespace gt;
  const int lo = -dsat - EXT, hi = lo + ext_entries(dsat, causal) - 1;
  long bad = 0;
  *blocks = 0;
  for (int pmin = -130; pmin < 2 * dsat + 200; ++pmin) {
    const int pmax = pmin + span - 1, klen = 2 * dsat + 300, last = causal ? (pmax + 1 < klen ? pmax + 1 : klen) : klen;
    for (int t = 0; t < last; t += kt)
      for (int ws = 0; ws < step / 32; ++ws) {
        if (t + 32 * ws >= last) continue;
        for (int n = 0; n < nb; ++n) {
          const int kk = t + 32 * ws + step * n, dmin = kk - pmax, dmax = kk + 31 - pmin;
          ++*blocks;
          if (rule ? dmax <= -dsat || dmin >= dsat : one_bias(dmin, dmax, dsat, causal)) continue;
          bad += dmin < lo || dmax > hi;
        }
      }
  }
  return bad;
}
"""


@pytest.fixture(scope="module")
def outside(tmp_path_factory):
    d = tmp_path_factory.mktemp("index")
    (d / "index.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O2", "-shared", "-fPIC", "-I", CSRC, str(d / "index.cpp"), "-o", str(d / "index.so")],
                   check=True)
    lib = ctypes.CDLL(str(d / "index.so"))
    lib.outside.restype = ctypes.c_long

    def call(*args):
        blocks = ctypes.c_int()
        bad = lib.outside(*args, ctypes.byref(blocks))
        assert blocks.value > 500
        return bad

    return call


# keys a tile, a wave's blocks in it and their distance, positions a wave: tiles shared by 128 and 64 rows, 16-bit and
# fp32; packed rows of 1, 4 and 32 heads
FORMS = [(64, 2, 32, 32), (32, 1, 32, 32), (64, 1, 64, 32), (128, 1, 128, 32), (128, 1, 128, 8), (128, 1, 128, 1)]


@pytest.mark.parametrize("causal", [0, 1])
@pytest.mark.parametrize("dsat", [1, 2, 31, 32, 33, 62, 63, 64, 95, 113, 1000])
@pytest.mark.parametrize("form", FORMS, ids=str)
def test_blocks_read_the_bias_table_inside_its_extent(outside, form, dsat, causal):
    kt, nb, step, span = form
    assert outside(dsat, causal, kt, nb, step, span, 0) == 0


def test_blocks_ahead_of_every_query_would_leave_the_causal_table(outside):
    """The second block of a 64-key tile, where positions do not start on a tile: without the rule for dmin > 0 it
    reads past the table's end."""
    assert outside(113, 1, 64, 2, 32, 32, 1) > 0
    assert outside(113, 0, 64, 2, 32, 32, 1) == 0
