"""Transformer-block operators without a GPU: bucket borders in whole numbers, the C ABI's argument checks (made before
any HIP call), the op schemas' Meta kernels and refusals, and the oracle against torch's autograd."""
import ctypes
import math

import pytest
import torch

from gradtts_amd import _lib
from gradtts_amd.attention import bucket_attention, relative_bucket
from gradtts_amd.norm import residual_norm
from oracle import blocks


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("nb, md", [(4, 3), (32, 128), (64, 256), (16, 64), (6, 40), (128, 1024), (32, 1000), (20, 500), (2, 2), (32, 17)])
def test_buckets_equal_the_whole_number_borders(nb, md, causal):
    if nb == 2 and not causal:
        pytest.skip("two buckets leave none for single distances")
    got = [relative_bucket(o, nb, causal, md) for o in range(-1100, 1101)]
    assert got == [blocks.bucket(o, nb, causal, md) for o in range(-1100, 1101)]
    assert relative_bucket(-2 ** 40, nb, causal, md) == (nb if causal else nb // 2) - 1
    assert relative_bucket(2 ** 40, nb, causal, md) == (0 if causal else nb - 1)


def test_bucket_ranges_are_refused():
    for args in [(1, True, 128), (2, False, 128), (7, False, 128), (130, True, 1024), (32, True, 16), (32, False, 8), (32, True, 1025)]:
        with pytest.raises(ValueError):
            relative_bucket(0, *args)


def attention_args(**kw):
    a = _lib.BucketAttention(dtype=_lib.GT_ELEM_F32, causal=0, n_buckets=32, max_distance=128, scale=0.125, B=2, Tq=4, Tk=4,
                             Hq=4, Hkv=2, D=64, q=16, k=16, v=16, table=16)
    for n, x in kw.items():
        setattr(a, n, x)
    return a


@pytest.mark.parametrize("kw, msg", [
    (dict(dtype=3), b"dtype"), (dict(Hq=3), b"multiple"), (dict(Hkv=0), b"multiple"), (dict(D=129), b"head size"),
    (dict(D=0), b"head size"), (dict(B=-1), b"2^28"), (dict(Tk=2 ** 28 + 1), b"2^28"), (dict(scale=0.0), b"scale"),
    (dict(scale=float("nan")), b"scale"), (dict(scale=-1.0), b"scale"), (dict(n_buckets=3), b"n_buckets"),
    (dict(max_distance=8), b"max_distance"), (dict(max_distance=2000), b"max_distance"), (dict(q=None), b"null"),
    (dict(table=None), b"null")])
def test_attention_arguments_are_checked_before_any_hip_call(kw, msg):
    L = _lib.lib()
    a = attention_args(**kw)
    p = ctypes.c_void_p(16)
    assert L.gt_bucket_attention_forward(ctypes.byref(a), p, p, p, 1 << 40, None) == _lib.GT_ERR_ARG
    assert msg in L.gt_last_error()
    g = _lib.BucketAttentionGrads(dout=16, dq=16, dk=16, dv=16, dtable=16)
    assert L.gt_bucket_attention_backward(ctypes.byref(a), p, p, ctypes.byref(g), p, 1 << 40, None) == _lib.GT_ERR_ARG
    assert msg in L.gt_last_error()


def test_attention_nulls_and_workspace():
    L = _lib.lib()
    p = ctypes.c_void_p(16)
    a = attention_args()
    ok = dict(dout=16, dq=16, dk=16, dv=16, dtable=16)
    assert L.gt_bucket_attention_forward(None, p, p, p, 0, None) == _lib.GT_ERR_ARG
    assert L.gt_bucket_attention_forward(ctypes.byref(a), None, p, p, 1 << 40, None) == _lib.GT_ERR_ARG
    for n in ok:
        g = _lib.BucketAttentionGrads(**{**ok, n: None})
        assert L.gt_bucket_attention_backward(ctypes.byref(a), p, p, ctypes.byref(g), p, 1 << 40, None) == _lib.GT_ERR_ARG
    g = _lib.BucketAttentionGrads(**ok)
    need = L.gt_bucket_attention_backward_workspace_bytes(ctypes.byref(a))
    assert need > 0
    assert L.gt_bucket_attention_backward(ctypes.byref(a), p, p, ctypes.byref(g), p, need - 1, None) == _lib.GT_ERR_WORKSPACE
    assert L.gt_bucket_attention_backward_workspace_bytes(None) == 0
    # nothing to do: no tensor needed, no HIP call made
    e = attention_args(B=0, q=None, k=None, v=None)
    assert L.gt_bucket_attention_forward(ctypes.byref(e), None, None, None, 0, None) == _lib.GT_OK


def norm_args(**kw):
    a = _lib.ResidualNorm(dtype=_lib.GT_ELEM_BF16, rms=0, gate_per_batch=0, scale=1.0, eps=1e-5, B=2, T=3, C=64, x=16, y=16,
                          gate=16, post_weight=16, post_bias=16, pre_weight=16, pre_bias=16)
    for n, x in kw.items():
        setattr(a, n, x)
    return a


@pytest.mark.parametrize("kw, msg", [
    (dict(dtype=-1), b"dtype"), (dict(C=0), b"8192"), (dict(C=8193), b"8192"), (dict(T=-1), b"2^28"), (dict(eps=-1.0), b"eps"),
    (dict(eps=float("inf")), b"eps"), (dict(scale=float("nan")), b"finite"), (dict(x=None), b"null"),
    (dict(pre_weight=None), b"null"), (dict(gate=None, gate_per_batch=1), b"gate")])
def test_norm_arguments_are_checked_before_any_hip_call(kw, msg):
    L = _lib.lib()
    p = ctypes.c_void_p(16)
    a = norm_args(**kw)
    assert L.gt_residual_norm_forward(ctypes.byref(a), p, p, p, None) == _lib.GT_ERR_ARG
    assert msg in L.gt_last_error()
    g = _lib.ResidualNormGrads(*[16] * 9)
    assert L.gt_residual_norm_backward(ctypes.byref(a), p, ctypes.byref(g), p, 1 << 40, None) == _lib.GT_ERR_ARG


def test_norm_gradients_of_absent_parameters_and_workspace():
    L = _lib.lib()
    p = ctypes.c_void_p(16)
    g = _lib.ResidualNormGrads(*[16] * 9)
    for n in ("gate", "post_bias", "pre_bias"):
        a = norm_args(**{n: None})
        assert L.gt_residual_norm_backward(ctypes.byref(a), p, ctypes.byref(g), p, 1 << 40, None) == _lib.GT_ERR_ARG
        assert b"absent" in L.gt_last_error()
    a = norm_args()
    need = L.gt_residual_norm_backward_workspace_bytes(ctypes.byref(a))
    assert L.gt_residual_norm_backward(ctypes.byref(a), p, ctypes.byref(g), p, need - 1, None) == _lib.GT_ERR_WORKSPACE


def meta(*shape, dtype=torch.float32):
    return torch.empty(*shape, device="meta", dtype=dtype)


def test_ops_on_meta_tensors_and_their_refusals():
    q, k, t = meta(2, 5, 4, 64), meta(2, 7, 2, 64), meta(32, 4)
    assert bucket_attention(q, k, k, t).shape == q.shape
    n = torch.zeros(2, dtype=torch.int64, device="meta")
    assert bucket_attention(q, k, k, t, lengths=n, q_start=n).shape == q.shape
    bad = [(q[0], k, k, t, {}), (q, k, k[:, :6], t, {}), (q, k[:1], k[:1], t, {}), (q, meta(2, 7, 3, 64), meta(2, 7, 3, 64), t, {}),
           (q, k, k, meta(32, 2), {}), (q, k, k, t.half(), {}), (q.double(), k.double(), k.double(), t.double(), {}),
           (q, k, k, t, dict(lengths=n.float())), (q, k, k, t, dict(lengths=torch.zeros(3, dtype=torch.int64, device="meta"))),
           (q, k, k, t, dict(q_start=torch.zeros(2, 1, dtype=torch.int64, device="meta")))]
    for *args, kw in bad:
        with pytest.raises(RuntimeError, match="gradtts"):
            bucket_attention(*args, **kw)
    x, w = meta(2, 3, 64, dtype=torch.bfloat16), meta(64)
    out, h = residual_norm(x, x, w, w, gate=meta(2, 64))
    assert out.shape == h.shape == x.shape and h.dtype == torch.bfloat16
    for args, kw in [((x, x[:, :2], w, w), {}), ((x, x.float(), w, w), {}), ((x, x, w.bfloat16(), w), {}), ((x, x, w, meta(63)), {}),
                     ((x, x, w, w), dict(gate=meta(3, 64))), ((x, x, w, w), dict(post_bias=meta(2, 64))), ((x[0], x[0], w, w), {}),
                     ((x, x, w, w), dict(lengths=meta(2)))]:
        with pytest.raises(RuntimeError, match="gradtts"):
            residual_norm(*args, **kw)
    with pytest.raises(ValueError, match="kind"):
        residual_norm(x, x, w, w, kind="batch")


def test_no_cpu_path():
    x = torch.zeros(1, 2, 2, 64)
    with pytest.raises(RuntimeError, match="HIP"):
        bucket_attention(x, x, x, torch.zeros(32, 2))
    y = torch.zeros(1, 2, 8)
    with pytest.raises(RuntimeError, match="HIP"):
        residual_norm(y, y, torch.ones(8), torch.ones(8))


def test_oracle_attention_gradients_are_autograds():
    g = torch.Generator().manual_seed(0)
    q, k, v, table, dout = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((2, 9, 4, 8), (2, 11, 2, 8), (2, 11, 2, 8), (6, 4), (2, 9, 4, 8)))
    kw = dict(lengths=[11, 6], q_start=[2, 0], causal=True, max_distance=7)
    val, _ = blocks.attention(q.float(), k.float(), v.float(), table.float(), dout.float(), **kw)
    leaves = [t.float().double().requires_grad_() for t in (q, k, v, table)]
    qq, kk, vv, tt = leaves
    out = torch.zeros(2, 9, 4, 8, dtype=torch.float64)
    rows = []
    for b in range(2):
        for h in range(4):
            n = kw["lengths"][b]
            idx = torch.tensor([[blocks.bucket(j - kw["q_start"][b] - i, 6, True, 7) for j in range(n)] for i in range(9)])
            see = torch.tensor([[j <= kw["q_start"][b] + i for j in range(n)] for i in range(9)])
            s = (qq[b, :, h] @ kk[b, :n, h // 2].T / math.sqrt(8) + tt[:, h][idx]).masked_fill(~see, -math.inf)
            rows.append(torch.softmax(s, -1) @ vv[b, :n, h // 2])
    out = torch.stack(rows).reshape(2, 4, 9, 8).transpose(1, 2)
    grads = torch.autograd.grad(out, leaves, dout.float().double())
    for n, t in zip(("out", "dq", "dk", "dv", "dtable"), (out, *grads)):
        assert torch.allclose(val[n], t, atol=1e-12), n


@pytest.mark.parametrize("kind, bias, gate", [("layer", True, "batch"), ("rms", False, "channel"), ("layer", False, None), ("rms", True, "batch")])
def test_oracle_norm_gradients_are_autograds(kind, bias, gate):
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float32)
    args = dict(x=r(2, 5, 12), y=r(2, 5, 12), post_weight=r(12), pre_weight=r(12), post_bias=r(12) if bias else None,
                pre_bias=r(12) if bias else None, gate=None if gate is None else r(2, 12) if gate == "batch" else r(12))
    dout, dh = r(2, 5, 12), r(2, 5, 12)
    val, _ = blocks.residual_norm(**args, scale=0.6, kind=kind, dout=dout, dh=dh)
    a = {n: t.double().requires_grad_() if t is not None else None for n, t in args.items()}

    def norm(t, w, b):
        if kind == "layer":
            t = t - t.mean(-1, keepdim=True)
        t = t / torch.sqrt(t.square().mean(-1, keepdim=True) + 1e-5) * w
        return t if b is None else t + b

    gg = 1.0 if a["gate"] is None else a["gate"][:, None] if gate == "batch" else a["gate"]
    out = a["x"] + 0.6 * gg * norm(a["y"], a["post_weight"], a["post_bias"])
    h = norm(out, a["pre_weight"], a["pre_bias"])
    names = [n for n, t in a.items() if t is not None]
    grads = dict(zip(names, torch.autograd.grad([out, h], [a[n] for n in names], [dout.double(), dh.double()])))
    assert torch.allclose(val["out"], out, atol=1e-12) and torch.allclose(val["h"], h, atol=1e-12)
    for n in names:
        assert torch.allclose(val["d" + n], grads[n], atol=1e-11), n
