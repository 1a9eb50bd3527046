"""The transformer-block operators as programs use them, on the MI355X: every kernel form, overflow and shut-off
buckets, long caches, streams, captured graphs, compiled functions, decoding over a cache, a block with gradients.
Elementwise bounds are oracle/blocks.py's; where a test has its own, its reason stands beside it."""
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


def check(name, args, dout, **kw):
    want, bound = blocks.attention(*args, dout, **kw)
    got = attend(*args, dout, **kw)
    for n in want:
        close(f"{name} {n}", got[n], want[n], bound[n])
    return got


# B, Tq, Tk, Hq, Hkv, D, causal, n_buckets, max_distance, lengths, q_lengths, q_start: tiles of 128, 64 and 32 rows,
# alone and in pairs, head sizes between the padded ones, rows that are on the 16-byte grid and not
FORMS = [
    (16, 140, 140, 32, 16, 40, False, 32, 64, None, None, None),
    (16, 260, 260, 16, 16, 72, True, 16, 64, None, None, None),
    (12, 260, 260, 32, 8, 101, True, 4, 3, [260] * 11 + [131], None, None),
    (4, 130, 130, 16, 16, 24, True, 32, 128, None, None, None),
    (4, 190, 190, 16, 4, 72, True, 32, 128, [190, 65, 64, 1], [190, 65, 64, 1], None),
    (4, 130, 150, 16, 8, 104, False, 32, 128, None, None, [20, 0, 0, -30]),
    (4, 130, 130, 16, 16, 33, True, 32, 128, None, None, None),
    (6, 190, 190, 16, 16, 72, True, 32, 128, [190, 65, 64, 1, 0, 129], None, None),
    (7, 150, 150, 16, 8, 24, True, 32, 128, None, [150, 1, 64, 65, 0, 128, 150], None),
    (6, 140, 140, 16, 16, 109, True, 32, 128, None, None, None),
    (6, 400, 400, 16, 4, 40, True, 32, 128, None, None, None),
    (1, 1, 5000, 8, 2, 128, True, 32, 128, None, None, [4999]),
    (3, 2, 1500, 4, 2, 64, True, 32, 128, [1500, 3, 0], None, [1498, 1, 0]),
    (2, 7, 1300, 6, 1, 50, False, 32, 128, [1300, 700], None, [300, 0]),
    (3, 3, 1500, 4, 2, 64, False, 32, 128, [1500, 900, 1], [2, 0, 3], [100, 0, -5]),
    (1, 33, 2000, 2, 2, 96, True, 32, 128, [1999], [32], [1960]),
    (2, 1, 600, 32, 1, 64, True, 128, 1024, [600, 40], None, [599, 39]),
    (1, 3, 90, 80, 1, 16, True, 32, 128, None, None, [87]),
    (1, 40, 50, 2, 1, 128, False, 128, 1024, None, None, None),
    (1, 40, 1100, 1, 1, 128, True, 128, 1024, None, None, [1060]),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("form", range(len(FORMS)))
def test_every_form(form, dtype):
    B, Tq, Tk, Hq, Hkv, D, causal, nb, md, ln, ql, qs = FORMS[form]
    *args, dout = inputs(100 + form, DT[dtype], B, Tq, Tk, Hq, Hkv, D, nb)
    check(f"{dtype} form {form}", args, dout, lengths=ln, q_lengths=ql, q_start=qs, causal=causal, max_distance=md)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,Tq,Tk,causal", [(1, 60, 300, False), (4, 200, 200, True), (1, 1, 2500, False),
                                            (16, 130, 300, False)])
def test_later_keys_far_above_the_first(dtype, B, Tq, Tk, causal):
    """Scores that rise by hundreds along the keys: sums against the first keys' maximum overflow and are redone."""
    H = 16 if B > 1 else 2
    q, k, v, table, dout = inputs(8, DT[dtype], B, Tq, Tk, H, H, 64, 32)
    q, k = q.abs() + 1, (0.5 * k.float().abs() * torch.linspace(-3, 30, Tk)[None, :, None, None]).to(k.dtype)
    want, bound = blocks.attention(q, k, v, table, dout, causal=causal)
    got = attend(q, k, v, table, dout, causal=causal)
    # probabilities, and their products, below fp32's least normal number are zeros: 2^-126 a term, at most 2500 x 16
    # terms with factors (values, keys, queries, sums of 64 of their products) below 2^11 each: under 2^-126 + 16 + 2 x 11
    for n in want:
        close(f"{dtype} rising {B} {Tq} {Tk} {n}", got[n], want[n], bound[n] + 2.0 ** -88)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,T", [(1, 75), (4, 150), (16, 200)])
@pytest.mark.parametrize("low", [float("-inf"), -2.0 ** 18])
def test_shut_buckets_equal_the_causal_mask(dtype, B, T, low):
    """With every bucket of later keys shut, both directions' form sees what the causal form of half the buckets sees."""
    if dtype == "f16" and low > -float("inf"):
        pytest.skip("-2^18 is -inf in float16")
    H = 16 if B > 1 else 2
    q, k, v, table, dout = inputs(12, DT[dtype], B, T, T, H, H, 48, 16)
    want, bound = blocks.attention(q, k, v, table, dout, causal=True, max_distance=40)
    got = attend(q, k, v, torch.cat([table, torch.full_like(table, low)]), dout, causal=False, max_distance=40)
    assert not bool(got["dtable"][16:].any())
    got["dtable"] = got["dtable"][:16]
    for n in want:
        close(f"{dtype} shut {T} {n}", got[n], want[n], bound[n])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,T", [(1, 40), (16, 300)])
def test_rows_without_an_open_bucket(dtype, B, T):
    """A causal row whose only key is shut off gives zeros and no gradient; so does a table that is shut throughout."""
    H = 16 if B > 1 else 2
    q, k, v, table, dout = inputs(13, DT[dtype], B, T, T, H, H, 64, 8)
    table[0] = float("-inf")
    got = attend(q, k, v, table, dout, causal=True)
    assert not bool(got["out"][:, 0].any()) and not bool(got["dq"][:, 0].any()) and not bool(got["dtable"][0].any())
    assert not bool(got["dv"][:, -1].any()) and not bool(got["dk"][:, -1].any())   # the last key: its own row's only
    assert all(bool(torch.isfinite(t).all()) for t in got.values())
    table[:] = float("-inf")
    got = attend(q, k, v, table, dout, causal=True)
    assert not any(bool(t.any()) for t in got.values())


def test_nan_stays_in_its_rows():
    """A NaN query makes its row NaN and no other; a NaN key every row that sees it."""
    q, k, v, table, _ = inputs(14, torch.bfloat16, 1, 100, 100, 2, 2, 64, 32)
    want, bound = blocks.attention(q, k, v, table, causal=True)
    q[0, 50, 1, 3] = float("nan")
    out = attend(q, k, v, table, causal=True)["out"].detach().cpu()
    assert bool(out[0, 50, 1].isnan().all())
    out[0, 50, 1] = want["out"][0, 50, 1].bfloat16()
    close("beside a NaN query", out, want["out"], bound["out"] + 2.0 ** -8 * want["out"].abs())
    q[0, 50, 1, 3] = 0
    want, bound = blocks.attention(q, k, v, table, causal=True)
    k[0, 70, 0] = float("nan")
    out = attend(q, k, v, table, causal=True)["out"].detach().cpu()
    close("before a NaN key", out[:, :70], want["out"][:, :70], bound["out"][:, :70])
    close("the other head", out[:, :, 1], want["out"][:, :, 1], bound["out"][:, :, 1])
    assert bool(out[0, 70:, 0].isnan().all())


def test_cache_past_two_to_the_31_elements():
    """One decoding step over 2^18 + 999 positions of 64 heads of 128 channels: 4.3 GB a tensor."""
    T, H, D = (1 << 18) + 999, 64, 128
    assert T * H * D > 1 << 31
    torch.manual_seed(0)
    k, v = (torch.empty(1, T, H, D, device="cuda", dtype=torch.bfloat16).normal_() for _ in range(2))
    k[0, -300:] *= 1.5   # the weight lies past the 2^31st element too
    q, table = torch.randn(1, 1, H, D, device="cuda").bfloat16(), torch.randn(4, H, device="cuda").bfloat16()
    start = torch.tensor([T - 1], device="cuda")
    out = bucket_attention(q, k, v, table, q_start=start, causal=True, max_distance=3)
    for h in (0, 63):
        one = [t[:, :, h:h + 1].cpu() for t in (q, k, v)]
        want, bound = blocks.attention(*one, table[:, h:h + 1].cpu(), causal=True, max_distance=3, q_start=[T - 1])
        close(f"long cache head {h}", out[:, :, h:h + 1], want["out"], bound["out"])


def test_shared_leaves_and_broadcast_inputs():
    """q, k and v the same leaf: its gradient is the three's sum. An expanded key: the sum over what it stands for."""
    x, _, _, table, dout = inputs(15, torch.float32, 2, 50, 50, 2, 2, 64, 32)
    sep = attend(x, x, x, table, dout, causal=True)
    leaf = x.cuda().requires_grad_()
    g, = torch.autograd.grad(bucket_attention(leaf, leaf, leaf, table.cuda(), causal=True), leaf, dout.cuda())
    parts = sep["dq"] + sep["dk"] + sep["dv"]
    assert float((g - parts).abs().max()) <= 4 * 2.0 ** -24 * float(parts.abs().max())   # the sum's order alone
    one = x[:, :, :1].cuda().requires_grad_()
    g, = torch.autograd.grad(bucket_attention(x.cuda(), one.expand(2, 50, 2, 64), x.cuda(), table.cuda()), one, dout.cuda())
    ref = attend(x, x[:, :, :1].expand(2, 50, 2, 64).contiguous(), x, table, dout)["dk"].sum(2, keepdim=True)
    assert float((g - ref).abs().max()) <= 2.0 ** -24 * float(ref.abs().max())


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_gradients_through_rows_off_the_grid(dtype):
    """Inputs and an output gradient whose rows start between 16-byte steps give what aligned ones give."""
    q, k, v, table, dout = inputs(16, DT[dtype], 2, 90, 90, 4, 2, 64, 32)
    want = attend(q, k, v, table, dout, causal=True)

    def off(t):
        wide = torch.zeros(*t.shape[:2], t[0, 0].numel() + 1, dtype=t.dtype, device="cuda")
        wide[..., 1:] = t.flatten(2).cuda()
        return wide[..., 1:].unflatten(-1, t.shape[2:])

    leaves = [off(t).requires_grad_() for t in (q, k, v)] + [table.cuda().requires_grad_()]
    out = bucket_attention(*leaves, causal=True)
    got = torch.autograd.grad(out, leaves, off(dout))
    assert torch.equal(out, want["out"])
    for n, g in zip(("dq", "dk", "dv", "dtable"), got):
        assert torch.equal(g, want[n]), n


def step_fn(dev, kw, leaves, g):
    out = bucket_attention(*dev, **kw)
    return [out] + list(torch.autograd.grad(out, leaves, g))


def norm_fn(args, kw, leaves, g):
    out, h = residual_norm(**args, **kw)
    return [out, h] + list(torch.autograd.grad([out, h], leaves, g))


def programs():
    """(name, static inputs, function of them): forward and backward of both operators, forms with workspaces."""
    res = []
    for name, (B, Tq, Tk, H, kv, D) in (("split", (1, 2, 3000, 4, 2, 64)), ("rows", (4, 150, 150, 16, 4, 72))):
        q, k, v, table, dout = inputs(17, torch.bfloat16, B, Tq, Tk, H, kv, D, 32)
        st = [t.cuda() for t in (q, k, v, table)]
        lens = torch.full((B,), Tk - 5, device="cuda")
        res.append((name, st + [dout.cuda(), lens], lambda a: step_fn(
            a[:4], dict(lengths=a[5], causal=False), a[:4], a[4])))
    args, dout, dh = norm_inputs(18, torch.float32, 3, 70, 192, True, "batch")
    names = list(args)
    res.append(("norm", [t.cuda() for t in args.values()] + [dout.cuda(), dh.cuda()],
                lambda a: norm_fn(dict(zip(names, a)), dict(lengths=torch.arange(3, device="cuda") + 40), a[:-2], a[-2:])))
    return res


def test_two_streams_at_once():
    for (name, a, fn), seed in zip(programs(), (1, 2, 3)):
        torch.manual_seed(seed)
        for t in a:
            if t.is_floating_point():
                t.requires_grad_()
        b = [(torch.randn_like(t) if t.is_floating_point() else t - 20).detach() for t in a]
        for t in b:
            if t.is_floating_point():
                t.requires_grad_()
        want = [fn(a), fn(b)]
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        torch.cuda.synchronize()
        for _ in range(3):
            got = [None, None]
            for i, x in enumerate((a, b)):
                with torch.cuda.stream(streams[i]):
                    got[i] = fn(x)
            torch.cuda.synchronize()
            for g, w in zip(got, want):
                assert all(torch.equal(x, y) for x, y in zip(g, w)), name


def test_captured_graphs_with_gradients_replay():
    """Forward and backward of each program in a graph of its own; replays in turn, on new inputs, with eager work and
    synchronizations between them, give the eager result each time."""
    made = []
    for name, a, fn in programs():
        for t in a:
            if t.is_floating_point():
                t.requires_grad_()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            fn(a)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = fn(a)
        made.append((name, a, fn, graph, out))
    for round in range(3):
        want = []
        for name, a, fn, graph, out in made:
            with torch.no_grad():
                for i, t in enumerate(a):
                    if t.is_floating_point():
                        t.copy_(torch.randn(t.shape, generator=torch.Generator().manual_seed(31 * round + i)))
                    else:
                        t -= 3
            want.append([t.detach().clone() for t in fn(a)])
        if round == 1:
            torch.cuda.synchronize()
        for _, _, _, graph, _ in made:
            graph.replay()
        for (name, _, _, _, out), w in zip(made, want):
            assert all(torch.equal(x, y) for x, y in zip(out, w)), (name, round)


def test_capture_with_gradients_beside_a_living_eager_graph_is_refused():
    q, k, v, table, dout = (t.cuda() for t in inputs(19, torch.float32, 1, 20, 20, 2, 2, 64, 32))
    q.requires_grad_()
    alive = bucket_attention(q, k, v, table)
    with pytest.raises(RuntimeError, match="eager autograd graph"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            bucket_attention(q, k, v, table)
    args = {n: t.cuda() for n, t in norm_inputs(20, torch.float32, 1, 9, 64, True, "channel")[0].items()}
    args["pre_weight"].requires_grad_()
    kept = residual_norm(**args)
    with pytest.raises(RuntimeError, match="eager autograd graph"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            residual_norm(**args)
    w = torch.randn(64, 64, device="cuda", requires_grad=True)
    through = bucket_attention(q.detach() @ w, k, v, table)
    with pytest.raises(RuntimeError, match="eager autograd graph"):   # the leaf behind an input that is none
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            bucket_attention((q.detach().reshape(-1, 64) * w[0]).view(q.shape), k, v, table)
    through.sum().backward()
    del through
    alive.sum().backward()
    (kept[0].sum() + kept[1].sum()).backward()
    assert bool(torch.isfinite(q.grad).all()) and bool(torch.isfinite(args["pre_weight"].grad).all())
    del alive, kept
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):                       # and works once they are gone
        out = bucket_attention(q, k, v, table)
        g, = torch.autograd.grad(out, q, dout)
    graph.replay()
    ref = attend(q.detach(), k, v, table, dout)
    assert torch.equal(out, ref["out"]) and torch.equal(g, ref["dq"])


def test_compiled_functions_give_the_eager_result():
    q, k, v, table, dout = inputs(21, torch.bfloat16, 2, 40, 40, 4, 2, 64, 32)
    leaves = [t.cuda().requires_grad_() for t in (q, k, v, table)]
    args, _, dh = norm_inputs(22, torch.bfloat16, 2, 40, 256, True, None)
    dev = {n: t.cuda().requires_grad_() for n, t in args.items() if t is not None and n != "y"}

    def block(q, k, v, table, dev):
        return residual_norm(y=bucket_attention(q, k, v, table, causal=True).flatten(2), **dev)[1]

    res = []
    for fn in (block, torch.compile(block, backend="aot_eager", fullgraph=True)):
        h = fn(*leaves, dev)
        res.append([h] + list(torch.autograd.grad(h, leaves + list(dev.values()), dh.cuda())))
    assert all(torch.equal(a, b) for a, b in zip(*res))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_decoding_over_a_cache_is_the_full_pass(dtype):
    """A prompt of each length, then one token at a time into a longer cache: each step's row within the full pass's
    bound, the residual step's rows equal to it bit for bit."""
    B, T, Hq, Hkv, D, cap = 2, 150, 8, 2, 64, 400
    q, k, v, table, _ = inputs(23, DT[dtype], B, T, T, Hq, Hkv, D, 32)
    want, bound = blocks.attention(q, k, v, table, causal=True)
    args, _, _ = norm_inputs(24, DT[dtype], B, T, Hq * D, True, "channel")
    dev = {n: t.cuda() for n, t in args.items()}
    full = residual_norm(**dev)
    caches = [torch.full((B, cap, Hkv, D), float("nan"), dtype=DT[dtype], device="cuda") for _ in range(2)]
    prompt = torch.tensor([140, 97])
    for cache, t in zip(caches, (k, v)):
        for b in range(B):
            cache[b, :prompt[b]] = t[b, :prompt[b]].cuda()
    qp = q[:, :140].cuda()
    out = bucket_attention(qp, *caches, table.cuda(), lengths=prompt.cuda(), q_lengths=prompt.cuda(), causal=True)
    for b in range(B):
        n = int(prompt[b])
        close(f"{dtype} prompt {b}", out[b, :n], want["out"][b, :n], bound["out"][b, :n])
        assert not bool(out[b, n:].any())
    for step in range(10):
        at = prompt + step
        rows = torch.arange(B)
        for cache, t in zip(caches, (k, v)):
            cache[rows.cuda(), at.cuda()] = t[rows, at].cuda()
        out = bucket_attention(q[rows, at][:, None].cuda(), *caches, table.cuda(), lengths=(at + 1).cuda(), q_start=at.cuda(),
                               causal=True)
        close(f"{dtype} step {step}", out[:, 0], want["out"][rows, at], bound["out"][rows, at])
        one = residual_norm(**{n: (t[rows, at][:, None] if t.dim() == 3 else t) for n, t in dev.items()})
        assert torch.equal(one[0][:, 0], full[0][rows, at]) and torch.equal(one[1][:, 0], full[1][rows, at])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_two_layers_with_gradients(dtype):
    """Projections, attention, output projection and residual step, twice, in the type; every gradient against the same
    program in 64 bits. A layer rounds its tensors some 12 times in each direction, so four passes about 48 times, by
    2^-24 or 2^-9 (half a step, mean square a third) of a tensor's norm each; they add as squares, and a product of
    unit-variance weights keeps norms: sqrt(48) u, with a factor of 4 for the norms' and softmax's amplification; in fp32
    a product of 192 terms rounds its sum some sqrt(192) / 2 times besides, in norm: a factor of 8."""
    dt, B, T, H, kv, D, C = DT[dtype], 2, 70, 4, 2, 48, 192
    g = torch.Generator().manual_seed(25)
    r = lambda *s: torch.randn(*s, generator=g)
    lens = [70, 44]
    p = {"x": r(B, T, C)}
    for l in range(2):
        p |= {f"wq{l}": r(C, H * D) * C ** -0.5, f"wk{l}": r(C, 2 * kv * D) * C ** -0.5, f"wo{l}": r(H * D, C) * C ** -0.5,
              f"table{l}": r(32, H)}
        p = {n: t.to(dt) for n, t in p.items()}
    norms = {f"{n}{l}": 1 + 0.2 * r(C) if "weight" in n else 0.2 * r(C) for l in range(2)
             for n in ("post_weight", "post_bias", "pre_weight", "pre_bias")}
    up = r(2, B, T, C).to(dt)
    live = (torch.arange(T)[None] < torch.tensor(lens)[:, None])[..., None]
    near = {o: blocks.bucket(o, 32, True, 128) for o in range(-T, T)}
    idx = torch.tensor([[near[j - i] for j in range(T)] for i in range(T)])

    def plain_attention(q, k, v, table):
        k, v = (t.repeat_interleave(H // kv, 2) for t in (k, v))
        s = torch.matmul(q.transpose(1, 2), k.permute(0, 2, 3, 1)) * D ** -0.5 + table[idx].permute(2, 0, 1)
        j = torch.arange(T)
        s = s.masked_fill(~((j[None] <= j[:, None]) & live[:, None, None, :, 0]), -1e300)
        return torch.matmul(torch.softmax(s, -1), v.transpose(1, 2)).transpose(1, 2) * live[..., None]

    def plain_step(x, y, w1, b1, w2, b2):
        norm = lambda t, w, b: torch.nn.functional.layer_norm(t, (C,), w, b, 1e-5)
        out = (x + norm(y, w1, b1)) * live
        return out, norm(out, w2, b2) * live

    def run(p, norms, own):
        x = h = p["x"]
        for l in range(2):
            q = (h.reshape(-1, C) @ p[f"wq{l}"]).view(B, T, H, D)
            k, v = (h.reshape(-1, C) @ p[f"wk{l}"]).view(B, T, 2, kv, D).unbind(2)
            n = [norms[f"{n}{l}"] for n in ("post_weight", "post_bias", "pre_weight", "pre_bias")]
            if own:
                at = torch.tensor(lens, device="cuda")
                y = bucket_attention(q, k, v, p[f"table{l}"], lengths=at, q_lengths=at, causal=True)
                y = (y.reshape(-1, H * D) @ p[f"wo{l}"]).view(B, T, C)
                x, h = residual_norm(x, y, n[0], n[2], n[1], n[3], lengths=at)
            else:
                y = (plain_attention(q, k, v, p[f"table{l}"]).reshape(-1, H * D) @ p[f"wo{l}"]).view(B, T, C)
                x, h = plain_step(x, y, *n)
        return x, h

    sides = []
    for own in (True, False):
        to = (lambda t: t.cuda().requires_grad_()) if own else (lambda t: t.double().requires_grad_())
        a, b = ({n: to(t) for n, t in d.items()} for d in (p, norms))
        x, h = run(a, b, own)
        u = up.cuda() if own else up.double()
        grads = torch.autograd.grad([x, h], list(a.values()) + list(b.values()), [u[0], u[1]])
        sides.append([t.detach().cpu().double() for t in (x, h, *grads)])
    names = ["x", "h"] + ["d" + n for n in list(p) + list(norms)]
    tol = 4 * 48 ** 0.5 * (2.0 ** -24 if dtype == "f32" else 2.0 ** -9) * (8 if dtype == "f32" else 1)
    for n, got, want in zip(names, *sides):
        err = float((got - want).norm() / want.norm())
        print(f"{dtype} {n}: {err:.2e} of {tol:.2e}")
        assert err <= tol, (n, err)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,T,C,kind,gate", [(3, 1500, 64, "layer", "batch"), (90, 21, 192, "rms", "batch"),
                                             (2, 700, 520, "layer", "channel"), (1, 260, 2056, "rms", None),
                                             (5, 130, 4100, "layer", "batch")])
def test_residual_norm_over_many_rows(dtype, B, T, C, kind, gate):
    """Rows in several chunks and parameter sums in several ranges, ragged lengths."""
    args, dout, dh = norm_inputs(B + T, DT[dtype], B, T, C, True, gate)
    kw = dict(scale=-1.25, kind=kind, lengths=[(37 * b * b + T) % (T + 1) for b in range(B)])
    want, bound = blocks.residual_norm(**args, **kw, dout=dout, dh=dh)
    got = norm_step(args, dout, dh, **kw)
    for n in want:
        close(f"{dtype} {B} {T} {C} {n}", got[n], want[n], bound[n])


def test_residual_norm_of_constant_and_extreme_rows():
    """A row without variance: u = 0 exactly, the norm gives its bias. Values near float16's largest stay finite."""
    C = 256
    w, b = torch.full((C,), 1.5, device="cuda"), torch.linspace(-1, 1, C, device="cuda")
    x = torch.zeros(1, 4, C, device="cuda")
    y = torch.full((1, 4, C), 3.0, device="cuda")
    out, h = residual_norm(x, y, w, w, b, b)
    assert torch.equal(out[0, 0], b)
    big = torch.full((1, 4, C), 60000.0, device="cuda", dtype=torch.float16)
    big[..., ::2] = -60000.0
    out, h = residual_norm(torch.zeros_like(big), big, w, w)
    want = torch.where(torch.arange(C, device="cuda") % 2 == 0, -1.5, 1.5)
    # u = 1 up to (C + 8) 2^-24, then half a step of float16
    assert float((out[0, 0].float() - want).abs().max()) <= 1.5 * (264 * 2.0 ** -24 + 2.0 ** -11)
