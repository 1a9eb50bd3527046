"""Bucket attention on the MI355X where one key, one half of a sum or one unseen place decides: against the 64-bit form
within the bounds that oracle/blocks.py counts. Many heads repeat two, so that the forms of many rows are reached while
the 64-bit form is computed for two heads."""
import pytest
import torch

from conftest import gpu_available
from gradtts_amd.attention import bucket_attention
from gradtts_amd.norm import residual_norm
from oracle import blocks
from test_blocks_gpu import DT, attend, close, inputs, norm_inputs, norm_step

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not gpu_available():
        pytest.skip("no HIP device")


def check_two(name, args, dout, heads, extra=0.0, **kw):
    """args, dout: two heads, each with keys of its own; the call has `heads` of them, the two in turn. Checks the first
    and the last two; returns what was compared."""
    want, bound = blocks.attention(*args, dout, **kw)
    n = heads // 2
    got = attend(*(t.repeat(1, 1, n, 1) for t in args[:3]), args[3].repeat(1, n), dout.repeat(1, 1, n, 1), **kw)
    for part, sl in (("first", slice(0, 2)), ("last", slice(heads - 2, heads))):
        for k in want:
            close(f"{name} {part} {k}", got[k][:, sl] if k == "dtable" else got[k][:, :, sl], want[k], bound[k] + extra)


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


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("heads, Tq", ROWS)
@pytest.mark.parametrize("pair", [(100, 104), (100, 132), (36, 67)])
def test_two_parts_of_a_sum_pass_the_range_together(dtype, heads, Tq, pair):
    """Two keys some 2^127.7 above the first ones: either one's term is a finite float32, their sum is none. They fall to
    the two halves of a wave, or to two waves. Values of 1 / 4 and less keep the sums over them finite."""
    Tk, D = 200, 64
    q, k, v, table, dout = inputs(32, DT[dtype], 1, Tq, Tk, 2, 2, D, 4)
    q, k, v, table = 0 * q, 0.1 * k, 0.06 * v, 0 * table
    q[..., 0], k[..., 0] = 1, 0
    for j in pair:
        k[:, j, :, 0] = 708   # 708 / 8 nats = 127.68 powers of two
    assert 127 < float(k[0, pair[0], 0, 0]) / D ** 0.5 * 1.4426950408889634 < 128 and float(v.abs().max()) < 0.5
    # the other keys' probabilities, 2^-128, lie below fp32's least normal number and count as zeros, 2^-126 each: times a
    # factor dP - delta below 2^7 (64 products of at most 5 and 0.5), keys and values below 2^10, and summed over at most
    # 130 x 200 < 2^15 pairs: below 2^-94 in any gradient
    check_two(f"{dtype} pair {pair}", (q, k, v, table), dout, heads, 2.0 ** -94, max_distance=3)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("heads", [512, 64, 2])
@pytest.mark.parametrize("start", [1, 2, 31, 33, 63])
def test_causal_chunk_that_starts_between_tiles(dtype, heads, start):
    """The next 140 tokens of a sequence, `start` of which are in the cache already."""
    *args, dout = inputs(33, DT[dtype], 1, 140, 140 + start, 2, 2, 40, 32)
    check_two(f"{dtype} start {start}", args, dout, heads, causal=True, q_start=[start])


def test_gradients_of_a_kept_graph():
    """create_graph changes no value; differentiating what it gives raises, eager and compiled code go on working."""
    q, k, v, table, dout = inputs(34, torch.bfloat16, 2, 40, 40, 4, 2, 64, 32)
    want = attend(q, k, v, table, dout)
    leaves = [t.cuda().requires_grad_() for t in (q, k, v, table)]
    out = bucket_attention(*leaves)
    got = torch.autograd.grad(out, leaves, dout.cuda(), create_graph=True)
    assert all(torch.equal(g, want[n]) for n, g in zip(("dq", "dk", "dv", "dtable"), got))
    with pytest.raises(NotImplementedError, match="second derivatives"):
        sum(g.float().square().sum() for g in got).backward()
    args, dout, dh = norm_inputs(35, torch.float32, 2, 30, 96, True, "batch")
    want = norm_step(args, dout, dh)
    dev = {n: t.cuda().requires_grad_() for n, t in args.items()}
    got = torch.autograd.grad(residual_norm(**dev), list(dev.values()), [dout.cuda(), dh.cuda()], create_graph=True)
    assert all(torch.equal(g, want["d" + n]) for n, g in zip(dev, got))
    with pytest.raises(NotImplementedError, match="second derivatives"):
        torch.autograd.grad(got[0].square().sum(), dev["x"])


# B, Tq, Tk, heads, keys the last query sees: packed rows, with key ranges of their own, tiles of 64 and 128 rows; the
# last query inside a 32-key block
CACHES = [(2, 1, 200, 2, 70), (1, 1, 3000, 2, 1500), (2, 3, 1400, 4, 1301), (1, 130, 400, 64, 201), (1, 130, 300, 512, 139),
          (1, 130, 300, 512, 21)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("case", CACHES, ids=str)
def test_a_cache_is_not_read_behind_the_last_query(dtype, case):
    """A causal step over a cache whose unwritten part holds NaN and infinities, without lengths: bit for bit what the
    written part alone gives; the unwritten keys' gradients are zeros."""
    B, Tq, Tk, H, n = case
    q, k, v, table, dout = inputs(36, DT[dtype], B, Tq, Tk, H, H, 40, 32)
    start = torch.tensor([n - Tq] * B)   # below zero: the first rows see no key
    want = attend(q, k, v, table, dout, causal=True, q_start=start.tolist(), lengths=[n] * B)
    k[:, n:], v[:, n::2], v[:, n + 1::2] = float("nan"), float("inf"), float("nan")
    got = attend(q, k, v, table, dout, causal=True, q_start=start.tolist())
    for name in want:
        assert torch.equal(got[name], want[name]), name
    assert not bool(got["dk"][:, n:].any()) and not bool(got["dv"][:, n:].any())


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("heads, Tq, Tk", [(512, 130, 130), (64, 130, 130), (2, 40, 40), (1, 5, 1500)])
def test_rows_before_the_first_key_beside_infinite_values(dtype, heads, Tq, Tk):
    """Rows that see no key are zeros whatever the keys' values are."""
    q, k, v, table, _ = inputs(37, DT[dtype], 1, Tq, Tk, heads, heads, 40, 32)
    v[:, 0] = float("inf")
    out = attend(q, k, v, table, causal=True, q_start=[-3])["out"]
    assert not bool(out[:, :3].any()) and bool((out[:, 3] == float("inf")).all())


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B, T", [(8, 190), (40, 140), (4, 60)])
def test_an_entry_alone_and_in_a_batch(dtype, B, T):
    """The forms are chosen by the number of rows, so an entry's digits may depend on its batch: both stay within the
    same bounds, and each call repeats bit for bit."""
    q, k, v, table, dout = inputs(38, DT[dtype], B, T, T, 16, 8, 40, 32)
    last = [t[-1:].contiguous() for t in (q, k, v)]
    want, bound = blocks.attention(*last, table, dout[-1:], causal=True)
    del want["dtable"]   # a sum over the batch
    batch, again = (attend(q, k, v, table, dout, causal=True) for _ in range(2))
    alone = attend(*last, table, dout[-1:], causal=True)
    assert all(torch.equal(batch[n], again[n]) for n in batch)
    for n in want:
        close(f"{dtype} in a batch {n}", batch[n][-1:], want[n], bound[n])
        close(f"{dtype} alone {n}", alone[n], want[n], bound[n])
