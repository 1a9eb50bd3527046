"""Transformer-block operators without a GPU: offsets that the attention kernels look up against the extent of their bias
table, second derivatives."""
import ctypes
import os
import subprocess

import pytest
import torch

from gradtts_amd import _lib
from gradtts_amd.attention import bucket_attention
from gradtts_amd.norm import residual_norm

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


def test_second_derivatives_are_refused():
    """Gradients of a graph that is kept are values as any others; what differentiates them raises."""
    q, k, t = (torch.empty(s, device="meta", requires_grad=True) for s in ((2, 5, 4, 64), (2, 7, 2, 64), (32, 4)))
    x, w, g = (torch.empty(s, device="meta", requires_grad=True) for s in ((2, 3, 64), (64,), (2, 64)))
    out = bucket_attention(q, k, k, t)
    norm = residual_norm(x, x * 2, w, w, gate=g)
    for outs, leaves, name in ((out, [q, k, t], "bucket_attention"), (norm[0] + norm[1], [x, w, g], "residual_norm")):
        grads = torch.autograd.grad(outs.sum(), leaves, create_graph=True)
        assert [d.shape for d in grads] == [p.shape for p in leaves] and all(d.requires_grad for d in grads)
        for d in grads:
            with pytest.raises(NotImplementedError, match=f"{name} has no second derivatives"):
                torch.autograd.grad(d.sum(), leaves, allow_unused=True, retain_graph=True)
        plain = torch.autograd.grad(outs.sum(), leaves)
        assert not any(d.requires_grad for d in plain)


def test_bucket_encoder_trains_on_long_texts():
    """The window form's training pass ends at 4096 tokens, where its row of scores fills its memory; the bucket form's
    keeps no such row: it takes longer ones, in memory that grows with their length alone."""
    L = _lib.lib()
    sizes = (61, 80, 192, 768, 256, 2, 2, 3)
    for create, last, ends in ((L.gt_text_encoder_create, (4,), True), (L.gt_text_encoder_create_buckets, (32, 128), False)):
        h = ctypes.c_void_p()
        assert create(*sizes, *last, ctypes.byref(h)) == _lib.GT_OK
        try:
            at, past, far = (L.gt_text_encoder_train_workspace_bytes(h, 1, t) for t in (4096, 4097, 16384))
            assert at > 0 and (past == far == 0 if ends else at < past and far < 4.1 * at)
        finally:
            L.gt_text_encoder_destroy(h)
