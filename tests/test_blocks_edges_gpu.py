"""Bucket attention on the MI355X where one key, one half of a sum or one unseen place decides: against the 64-bit form
within the bounds that oracle/blocks.py counts. Many heads repeat two, so that the forms of many rows are reached while
the 64-bit form is computed for two heads."""
import pytest
import torch

from conftest import gpu_available
from oracle import blocks
from test_blocks_gpu import DT, attend, close, inputs

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not gpu_available():
        pytest.skip("no HIP device")


def check_two(name, args, dout, heads, **kw):
    """args, dout: two heads, each with keys of its own; the call has `heads` of them, the two in turn. Checks the first
    and the last two; returns what was compared."""
    want, bound = blocks.attention(*args, dout, **kw)
    n = heads // 2
    got = attend(*(t.repeat(1, 1, n, 1) for t in args[:3]), args[3].repeat(1, n), dout.repeat(1, 1, n, 1), **kw)
    for part, sl in (("first", slice(0, 2)), ("last", slice(heads - 2, heads))):
        for k in want:
            close(f"{name} {part} {k}", got[k][:, sl] if k == "dtable" else got[k][:, :, sl], want[k], bound[k])


# heads, queries: tiles of 128 rows, of 64, packed rows
ROWS = [(512, 130), (64, 130), (2, 40)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("heads, Tq", ROWS)
@pytest.mark.parametrize("gap", [9.0, 12.0, 14.0])
def test_first_key_outweighs_thousands(dtype, heads, Tq, gap):
    """The first key's score lies `gap` above some 2000 others', its value is zero: what the row gives is the others',
    whose probabilities are e^-gap of the first."""
    Tk, D = 2000, 32
    q, k, v, table, dout = inputs(31, DT[dtype], 1, Tq, Tk, 2, 2, D, 4)
    q, k, v, table = 0.3 * q, 0.3 * k, 1 + 0.2 * v, 0.1 * table
    q[..., 0], k[..., 0] = 1, 0
    k[:, 0], v[:, 0] = 0, 0
    k[:, 0, :, 0] = gap * D ** 0.5
    check_two(f"{dtype} gap {gap}", (q, k, v, table), dout, heads, max_distance=3)
