"""Transformer-block operators (gradtts_amd.attention.bucket_attention, gradtts_amd.norm.residual_norm) on the MI355X
against their plain 64-bit forms, elementwise within the bounds that oracle/blocks.py counts."""
import pytest
import torch

from conftest import gpu_available
from gradtts_amd.attention import bucket_attention
from gradtts_amd.norm import residual_norm
from oracle import blocks

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not gpu_available():
        pytest.skip("no HIP device")


def close(name, got, want, bound):
    got = got.detach().cpu().double()
    assert got.shape == want.shape
    off = (got - want).abs()
    bad = ~(off <= bound)
    worst = float((off / bound.clamp(min=1e-300))[bound > 0].max()) if bool((bound > 0).any()) else 0.0
    print(f"{name}: {worst:.3f} of the bound")
    assert not bool(bad.any()), f"{name}: {int(bad.sum())} of {bad.numel()} outside, worst {worst:.2f} of the bound"


def inputs(seed, dt, B, Tq, Tk, Hq, Hkv, D, nb):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).to(dt)
    return r(B, Tq, Hq, D), r(B, Tk, Hkv, D), r(B, Tk, Hkv, D), r(nb, Hq), r(B, Tq, Hq, D)


def attend(q, k, v, table, dout=None, **kw):
    leaves = [t.cuda().requires_grad_() for t in (q, k, v, table)]
    kw = {n: torch.tensor(x).cuda() if isinstance(x, list) else x for n, x in kw.items()}
    out = bucket_attention(*leaves, **kw)
    res = {"out": out}
    if dout is not None:
        res |= dict(zip(("dq", "dk", "dv", "dtable"), torch.autograd.grad(out, leaves, dout.cuda())))
    return res


CASES = [
    # B, Tq, Tk, Hq, Hkv, D, causal, n_buckets, max_distance, lengths, q_lengths, q_start
    (1, 1, 1, 1, 1, 1, False, 4, 2, None, None, None),
    (2, 1, 1, 2, 1, 96, True, 32, 128, None, None, None),
    (2, 33, 33, 2, 2, 96, False, 32, 128, [33, 20], [33, 20], None),
    (2, 64, 64, 4, 2, 64, True, 32, 128, None, None, None),
    (1, 130, 130, 2, 1, 100, True, 2, 2, None, None, None),
    (3, 129, 129, 2, 2, 40, False, 64, 256, [129, 1, 64], [129, 1, 64], None),
    (2, 300, 300, 3, 1, 128, True, 32, 128, [300, 77], [300, 77], None),
    (1, 260, 260, 2, 2, 33, False, 6, 40, None, None, None),
    (2, 5, 200, 4, 2, 64, True, 32, 128, [200, 64], None, [195, 59]),
    (2, 70, 31, 2, 2, 80, False, 32, 1000, [31, 0], None, [0, 3]),
    (1, 40, 700, 2, 1, 128, False, 16, 64, None, [39], [500]),
    (2, 40, 60, 2, 2, 64, True, 32, 128, None, None, [-20, 100]),
    (1, 64, 64, 2, 2, 64, True, 32, 128, None, None, [-64]),
    (1, 600, 600, 1, 1, 32, True, 128, 1024, None, None, None),
    (4, 1, 333, 8, 2, 128, True, 32, 128, [333, 1, 32, 257], None, [332, 0, 31, 256]),
    (1, 3, 2100, 4, 1, 72, False, 32, 128, None, None, [1000]),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_attention_and_gradients(case, dtype):
    B, Tq, Tk, Hq, Hkv, D, causal, nb, md, ln, ql, qs = CASES[case]
    q, k, v, table, dout = inputs(case, DT[dtype], B, Tq, Tk, Hq, Hkv, D, nb)
    kw = dict(lengths=ln, q_lengths=ql, q_start=qs, causal=causal, max_distance=md)
    want, bound = blocks.attention(q, k, v, table, dout, **kw)
    got = attend(q, k, v, table, dout, **kw)
    for n in want:
        close(f"{dtype} case {case} {n}", got[n], want[n], bound[n])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_one_visible_key_has_exactly_no_score_gradient(dtype):
    q, k, v, table, dout = inputs(5, DT[dtype], 3, 1, 1, 4, 2, 96, 32)
    got = attend(q, k, v, table, dout, causal=True)
    assert torch.equal(got["out"].cpu(), v.repeat_interleave(2, 2))
    for n in ("dq", "dk", "dtable"):
        assert not bool(got[n].any())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_padding_is_not_read(dtype):
    """NaN and infinities behind the lengths change nothing, bit for bit, and padded gradients are zero."""
    q, k, v, table, dout = inputs(6, DT[dtype], 2, 100, 100, 2, 1, 64, 32)
    kw = dict(lengths=[100, 37], q_lengths=[100, 37])
    a = attend(q, k, v, table, dout, **kw)
    for t, bad in ((q, float("nan")), (k, float("inf")), (v, float("nan")), (dout, float("-inf"))):
        t[1, 37:] = bad
    b = attend(q, k, v, table, dout, **kw)
    for n in a:
        assert torch.equal(a[n], b[n]), n
    for n in ("out", "dq", "dk", "dv"):
        assert not bool(b[n][1, 37:].any())


def test_large_and_infinite_scores():
    """Scores far apart (one key takes a row), a bias of the type's lowest value, and of -inf: a bucket shut off."""
    q, k, v, table, dout = inputs(7, torch.float32, 1, 70, 70, 2, 2, 64, 32)
    q = q * 30
    table[3] = torch.finfo(torch.float32).min
    want, _ = blocks.attention(q, k, v, table)
    got = attend(q, k, v, table)["out"].cpu().double()
    assert bool(torch.isfinite(got).all())
    # scores of about 30 x 8: 2^-24 x (D + 18) x 240 relative in P, twice, over values of about 1
    assert float((got - want["out"]).abs().max()) < 2 * (64 + 18) * 2.0 ** -24 * 30 * 64 ** 0.5 * 4 * 5
    table[3] = float("-inf")
    again = attend(q, k, v, table)["out"].cpu().double()
    assert torch.equal(again, got)


def test_strided_inputs_and_wrapped_views():
    """q, k, v as slices of one projection, expanded heads and transposed storage give the contiguous result."""
    torch.manual_seed(0)
    B, T, H, D = 2, 90, 4, 64
    for dt in (torch.float32, torch.bfloat16):
        qkv = torch.randn(B, T, 3, H, D, device="cuda", dtype=dt)
        table = torch.randn(32, H, device="cuda", dtype=dt)
        want = bucket_attention(*(qkv[:, :, i].contiguous() for i in range(3)), table)
        assert torch.equal(bucket_attention(qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2], table), want)
        assert torch.equal(bucket_attention(*(qkv[:, :, i].permute(0, 2, 3, 1).contiguous().permute(0, 3, 1, 2)
                                              for i in range(3)), table.t().contiguous().t()), want)
        odd = torch.zeros(B, T, 3 * H * D + 1, device="cuda", dtype=dt)
        odd[..., 1:] = qkv.reshape(B, T, -1)
        view = odd[..., 1:].unflatten(-1, (3, H, D))
        assert torch.equal(bucket_attention(view[:, :, 0], view[:, :, 1], view[:, :, 2], table), want)
        one = qkv[:, :, 1, :1]
        assert torch.equal(bucket_attention(qkv[:, :, 0], one.expand(B, T, H, D), one.expand(B, T, H, D), table),
                           bucket_attention(qkv[:, :, 0], one, one, table))


def test_gradient_against_differences():
    q, k, v, table, dout = inputs(9, torch.float32, 1, 40, 40, 2, 1, 32, 8)
    got = attend(q, k, v, table, dout, causal=True, max_distance=16)

    def f(**kw):
        args = {"q": q, "k": k, "v": v, "table": table, **kw}
        return float((blocks.attention(**args, causal=True, max_distance=16)[0]["out"] * dout.double()).sum())

    for n, t in (("q", q), ("k", k), ("v", v), ("table", table)):
        d = torch.randn(t.shape, generator=torch.Generator().manual_seed(3), dtype=torch.float64)
        h = 1e-4
        num = (f(**{n: t.double() + h * d}) - f(**{n: t.double() - h * d})) / (2 * h)
        ana = float((got["d" + n].cpu().double() * d).sum())
        # the difference quotient is off by h^2 times the third derivative, the gradient by its bound
        assert abs(num - ana) < 1e-4 * max(1.0, abs(num)), n


def test_attention_repeats_bit_for_bit_and_is_batch_invariant():
    q, k, v, table, dout = inputs(11, torch.bfloat16, 3, 333, 333, 4, 2, 80, 32)
    a, b = (attend(q, k, v, table, dout) for _ in range(2))
    for n in a:
        assert torch.equal(a[n], b[n])


def test_empty_tensors():
    for B, Tq, Tk in ((0, 4, 4), (2, 0, 5), (2, 5, 0)):
        q, k, v, table, dout = inputs(1, torch.float32, B, Tq, Tk, 2, 2, 64, 32)
        got = attend(q, k, v, table, dout)
        for n in got:
            assert not bool(got[n].any())


NORM_CASES = [
    # B, T, C, kind, bias, gate, lengths
    (1, 1, 1, "rms", False, None, None), (2, 3, 8, "layer", True, "channel", None), (8, 1, 192, "layer", True, "channel", None),
    (3, 50, 192, "layer", True, "batch", [50, 1, 0]), (2, 37, 1003, "rms", False, "batch", [37, 11]),
    (2, 9, 520, "layer", False, None, None), (1, 300, 256, "rms", True, "channel", None), (3, 5, 1024, "layer", True, "batch", None),
    (2, 7, 2047, "layer", True, "channel", [7, 3]), (1, 6, 4096, "rms", False, "channel", None), (2, 4, 8192, "layer", True, "batch", None),
    (1, 3, 5001, "layer", True, None, None),
]


def norm_inputs(seed, dt, B, T, C, bias, gate):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    return dict(x=r(B, T, C).to(dt), y=(r(B, T, C) * 3 + 0.5).to(dt), post_weight=1 + 0.3 * r(C), pre_weight=1 + 0.3 * r(C),
                post_bias=r(C) if bias else None, pre_bias=r(C) if bias else None,
                gate=None if gate is None else r(C) if gate == "channel" else r(B, C)), r(B, T, C).to(dt), r(B, T, C).to(dt)


def norm_step(args, dout=None, dh=None, **kw):
    dev = {n: t.cuda().requires_grad_() if t is not None else None for n, t in args.items()}
    kw = {n: torch.tensor(x).cuda() if isinstance(x, list) else x for n, x in kw.items()}
    out, h = residual_norm(**dev, **kw)
    res = {"out": out, "h": h}
    if dout is not None:
        names = [n for n, t in dev.items() if t is not None]
        res |= {"d" + n: t for n, t in zip(names, torch.autograd.grad([out, h], [dev[n] for n in names], [dout.cuda(), dh.cuda()]))}
    return res


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("case", range(len(NORM_CASES)))
def test_residual_norm_and_gradients(case, dtype):
    B, T, C, kind, bias, gate, lengths = NORM_CASES[case]
    args, dout, dh = norm_inputs(case, DT[dtype], B, T, C, bias, gate)
    kw = dict(scale=0.7, kind=kind, lengths=lengths)
    want, bound = blocks.residual_norm(**args, **kw, dout=dout, dh=dh)
    got = norm_step(args, dout, dh, **kw)
    assert set(got) == set(want)
    for n in want:
        close(f"{dtype} case {case} {n}", got[n], want[n], bound[n])


def test_residual_norm_padding_is_not_read_and_repeats():
    args, dout, dh = norm_inputs(3, torch.bfloat16, 2, 40, 200, True, "batch")
    kw = dict(lengths=[40, 13])
    a = norm_step(args, dout, dh, **kw)
    for t in (args["x"], args["y"], dout, dh):
        t[1, 13:] = float("nan")
    b = norm_step(args, dout, dh, **kw)
    for n in a:
        assert torch.equal(a[n], b[n]), n
    for n in ("out", "h", "dx", "dy"):
        assert not bool(b[n][1, 13:].any())


def test_residual_norm_strides_one_output_and_empty():
    args, dout, dh = norm_inputs(4, torch.float32, 2, 30, 96, True, "channel")
    want = norm_step(args, dout, dh)
    odd = {n: (torch.stack([t, t], -1)[..., 0] if t is not None else None) for n, t in args.items()}
    got = norm_step(odd, dout.transpose(1, 2).contiguous().transpose(1, 2), dh)
    for n in want:
        assert torch.equal(want[n], got[n]), n
    # only h used: the other gradient is zero
    dev = {n: t.cuda().requires_grad_() for n, t in args.items()}
    _, h = residual_norm(**dev)
    only = torch.autograd.grad(h, [dev["x"], dev["y"]], dh.cuda())
    ref = norm_step(args, torch.zeros_like(dout), dh)
    assert torch.equal(only[0], ref["dx"]) and torch.equal(only[1], ref["dy"])
    for shape in ((0, 3), (3, 0)):
        args, dout, dh = norm_inputs(4, torch.float32, *shape, 96, True, "batch")
        got = norm_step(args, dout, dh)
        for n in got:
            assert not bool(got[n].any())
