"""Plain 64-bit forms of the transformer-block operators (gradtts_amd.attention, gradtts_amd.norm), with bounds on what
rounding may do to an implementation that keeps its sums in 32 bits.

Every quantity is written out from its formula; the gradients are explicit, not autograd's. The bounds count roundings:
half a step, u = finfo(type).eps / 2, for each value the operators round to the tensors' type, and 2^-24 a term for the
32-bit sums, propagated to first order through the formulas with absolute values.
"""
import math

import torch

U32 = 2.0 ** -24


def bucket(offset, n_buckets, causal, max_distance):
    """Bucket of one offset in whole numbers: the far bucket exact + k starts at the least distance d with
    (d / exact)^far >= (max_distance / exact)^k."""
    n = n_buckets if causal else n_buckets // 2
    exact = n // 2
    far = n - exact
    d = max(-offset, 0) if causal else abs(offset)
    b = d
    if d >= exact:
        k = 0
        while k < far - 1 and d ** far * exact ** (k + 1) >= max_distance ** (k + 1) * exact ** far:
            k += 1
        b = exact + k
    return b + (n if not causal and offset > 0 else 0)


def attention(q, k, v, table, dout=None, lengths=None, q_lengths=None, q_start=None, causal=False, max_distance=128,
              scale=None):
    """q [B, Tq, Hq, D], k, v [B, Tk, Hkv, D], table [n_buckets, Hq] of the operator's type (CPU). Returns (values,
    bounds): out, and with dout also dq, dk, dv, dtable, in float64."""
    dt = q.dtype
    u = torch.finfo(dt).eps / 2
    low = dt != torch.float32                       # P and dS enter their products rounded to the type
    tiny = 2.0 ** -25 if dt == torch.float16 else 0.0   # half the least step of float16
    B, Tq, Hq, D = q.shape
    Tk, Hkv = k.shape[1], k.shape[2]
    G = Hq // Hkv
    sc = D ** -0.5 if scale is None else scale
    nb = table.shape[0]
    val = {"out": torch.zeros(B, Tq, Hq, D, dtype=torch.float64)}
    if dout is not None:
        val |= {"dq": torch.zeros(B, Tq, Hq, D, dtype=torch.float64), "dk": torch.zeros(B, Tk, Hkv, D, dtype=torch.float64),
                "dv": torch.zeros(B, Tk, Hkv, D, dtype=torch.float64), "dtable": torch.zeros(nb, Hq, dtype=torch.float64)}
    err = {n: torch.zeros_like(t) for n, t in val.items()}
    for b in range(B):
        n = Tk if lengths is None else max(0, min(Tk, int(lengths[b])))
        nq = Tq if q_lengths is None else max(0, min(Tq, int(q_lengths[b])))
        start = 0 if q_start is None else int(q_start[b])
        if n == 0 or nq == 0:
            continue
        offs = {o: bucket(o, nb, causal, max_distance) for o in range(-(start + nq - 1), n - start)}
        idx = torch.tensor([[offs[j - start - i] for j in range(n)] for i in range(nq)])
        seen = torch.tensor([[not causal or j <= start + i for j in range(n)] for i in range(nq)])
        for h in range(Hq):
            qh, kh, vh = q[b, :nq, h].double(), k[b, :n, h // G].double(), v[b, :n, h // G].double()
            bias = table[:, h].double()[idx]
            s = (qh @ kh.T * sc + bias).masked_fill(~seen, -math.inf)
            m = s.amax(-1, keepdim=True)
            e = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
            z = e.sum(-1, keepdim=True)
            p = e / torch.where(z == 0, torch.ones_like(z), z)
            # score: D products and sums, the bias, the exponent's product, sum and rounded result, all 32-bit
            es = U32 * ((D + 2) * (qh.abs() @ kh.abs().T) * sc + 8 * bias.abs() + 8 * s.masked_fill(~seen, 0).abs() +
                        8 * torch.where(m == -math.inf, torch.zeros_like(m), m).abs())
            rel = 2 * (es + es.amax(-1, keepdim=True)) + (n + 16) * U32      # P's relative error
            ep = p * (rel + (u if low else 0.0)) + (tiny if low else 0.0) / torch.where(z == 0, torch.ones_like(z), z)
            o = p @ vh
            eo = ep @ vh.abs() + (n + 2) * U32 * (p @ vh.abs())
            val["out"][b, :nq, h] = o
            err["out"][b, :nq, h] = eo + u * (o.abs() + eo) + tiny
            if dout is None:
                continue
            g = dout[b, :nq, h].double()
            dp = g @ vh.T
            delta = (g * o).sum(-1, keepdim=True)
            ds = p * (dp - delta)
            edp = (D + 2) * U32 * (g.abs() @ vh.abs().T)
            edelta = (g.abs() * (eo + u * o.abs() + tiny)).sum(-1, keepdim=True) + (D + 2) * U32 * (g * o).abs().sum(-1, keepdim=True)
            eds32 = p * (edp + edelta) + p * rel * (dp - delta).abs() + 4 * U32 * ds.abs()
            eds = eds32 + (u * ds.abs() + tiny if low else 0.0)
            seen_f = seen.double()
            eds32, eds = eds32 * seen_f, eds * seen_f
            hk = h // G
            val["dq"][b, :nq, h] = ds @ kh * sc
            err["dq"][b, :nq, h] = (eds @ kh.abs() + (n + 2) * U32 * (ds.abs() @ kh.abs())) * sc
            val["dk"][b, :n, hk] += ds.T @ qh * sc
            err["dk"][b, :n, hk] += (eds.T @ qh.abs() + (G * nq + 2) * U32 * (ds.abs().T @ qh.abs())) * sc
            val["dv"][b, :n, hk] += p.T @ g
            err["dv"][b, :n, hk] += ep.T @ g.abs() + (G * nq + 2) * U32 * (p.T @ g.abs())
            one = torch.nn.functional.one_hot(idx.reshape(-1), nb).double()
            val["dtable"][:, h] += one.T @ ds.reshape(-1)
            err["dtable"][:, h] += one.T @ (eds32 + (n + nq) * B * U32 * ds.abs()).reshape(-1)
    for n in ("dq", "dk", "dv", "dtable"):
        if n in err:
            err[n] = err[n] + u * (val[n].abs() + err[n]) + tiny
    return val, err


def residual_norm(x, y, post_weight, pre_weight, post_bias=None, pre_bias=None, gate=None, scale=1.0, eps=1e-5,
                  kind="layer", lengths=None, dout=None, dh=None):
    """Returns (values, bounds): out, h, and with dout and dh also the gradients of the arguments that are there."""
    u = torch.finfo(x.dtype).eps / 2
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 0.0
    B, T, C = x.shape
    layer = kind == "layer"
    zero = torch.zeros(C, dtype=torch.float64)
    w1, w2 = post_weight.double(), pre_weight.double()
    b1, b2 = (zero if t is None else t.double() for t in (post_bias, pre_bias))
    g = torch.ones(C, dtype=torch.float64) if gate is None else gate.double()
    gs = scale * (g[:, None] if g.dim() == 2 else g)
    rows = torch.ones(B, T, 1, dtype=torch.bool)
    if lengths is not None:
        rows = (torch.arange(T)[None] < torch.as_tensor(lengths).clamp(0, T)[:, None])[:, :, None]
    x64, y64 = (torch.where(rows, t.double(), torch.ones(1, dtype=torch.float64)) for t in (x, y))

    def unit(t, et):
        """unit row, 1 / std, and the bound of the unit row's error for input error et"""
        mu = t.mean(-1, keepdim=True) if layer else torch.zeros_like(t[..., :1])
        d = t - mu
        r = (d.square().mean(-1, keepdim=True) + eps).rsqrt()
        ed = et + (et.mean(-1, keepdim=True) + (C + 4) * U32 * t.abs().mean(-1, keepdim=True) if layer else 0.0) + U32 * d.abs()
        erel = r.square() * (d.abs() * ed).mean(-1, keepdim=True) + (C + 8) * U32   # of r
        return d * r, r, r * ed + (d * r).abs() * erel, erel

    def unit_back(un, r, du, eun, edu, erel):
        c = (du * un).mean(-1, keepdim=True)
        a = du.mean(-1, keepdim=True) if layer else 0.0
        ec = (edu * un.abs() + du.abs() * eun).mean(-1, keepdim=True) + (C + 4) * U32 * (du * un).abs().mean(-1, keepdim=True)
        ea = (edu.mean(-1, keepdim=True) + (C + 4) * U32 * du.abs().mean(-1, keepdim=True)) if layer else 0.0
        out = r * (du - a - un * c)
        e = r * (edu + ea + eun * c.abs() + un.abs() * ec) + out.abs() * erel
        return out, e + 6 * U32 * r * (du.abs() + (a.abs() if layer else 0.0) + (un * c).abs())

    u1, r1, e1, er1 = unit(y64, torch.zeros_like(y64))
    n1 = u1 * w1 + b1
    en1 = e1 * w1.abs() + 4 * U32 * ((u1 * w1).abs() + b1.abs())
    out = x64 + gs * n1
    eout = gs.abs() * en1 + 4 * U32 * (x64.abs() + (gs * n1).abs())
    u2, r2, e2, er2 = unit(out, eout)
    h = u2 * w2 + b2
    eh = e2 * w2.abs() + 4 * U32 * ((u2 * w2).abs() + b2.abs())
    mask = rows.double()
    val = {"out": out * mask, "h": h * mask}
    err = {"out": (eout + u * (out.abs() + eout) + tiny) * mask, "h": (eh + u * (h.abs() + eh) + tiny) * mask}
    if dout is None:
        return val, err
    do, dh64 = (torch.where(rows, t.double(), torch.zeros(1, dtype=torch.float64)) for t in (dout, dh))
    du2 = dh64 * w2
    back2, eb2 = unit_back(u2, r2, du2, e2, U32 * du2.abs(), er2)
    d = (do + back2) * mask
    ed = (eb2 + 2 * U32 * (do.abs() + back2.abs())) * mask
    du1 = d * gs * w1
    dy, edy = unit_back(u1, r1, du1, e1, (ed + 4 * U32 * d.abs()) * (gs * w1).abs(), er1)
    n = B * T + 8
    val |= {"dx": d, "dy": dy * mask}
    err |= {"dx": (ed + u * (d.abs() + ed) + tiny), "dy": (edy + u * (dy.abs() + edy) + tiny) * mask}

    def cols(name, v, e, batch=False):
        val[name] = v.sum(1) if batch else v.sum((0, 1))
        err[name] = (e + n * U32 * v.abs()).sum(1) if batch else (e + n * U32 * v.abs()).sum((0, 1))

    cols("dpost_weight", gs * d * u1, gs.abs() * (ed * u1.abs() + d.abs() * e1))
    cols("dpre_weight", dh64 * u2, dh64.abs() * e2)
    if post_bias is not None:
        cols("dpost_bias", gs * d, gs.abs() * ed)
    if pre_bias is not None:
        cols("dpre_bias", dh64, torch.zeros_like(dh64))
    if gate is not None:
        # formed from the sums of d u1 and d, so their roundings count apart
        cols("dgate", scale * d * n1, abs(scale) * (ed * ((u1 * w1).abs() + b1.abs()) + d.abs() * en1 +
                                                    n * U32 * d.abs() * ((u1 * w1).abs() + b1.abs())), gate.dim() == 2)
    return val, err


def bucket_text_encoder(p, tokens, x_lengths, n_layers, n_heads, max_distance, drop=None):
    """The text encoder's bucket form in the parameters' type, by autograd's operations: prenet, projections and
    duration predictor as oracle.text_encoder, layers h = N_in(x); x += N_post(block(h)), h = N_pre(x). drop: None, or
    oracle.text_encoder.Dropouts (its masks fall on the blocks' outputs and the FFN's hidden channels)."""
    from .text_encoder import conv, ln
    D = (lambda site, v, q: drop.chan(site, v, q)) if drop is not None else (lambda site, v, q: v)
    pe, pp = (drop.p, drop.pp) if drop is not None else (0.0, 0.0)
    C = p["emb.weight"].shape[1]
    x = (p["emb.weight"][tokens] * math.sqrt(C)).transpose(1, -1)
    T = x.shape[2]
    live = torch.arange(T)[None] < x_lengths[:, None]
    m = live.unsqueeze(1).to(x.dtype)
    x_org = x
    for i in range(3):
        x = conv(p, f"prenet.conv_layers.{i}", x * m)
        x = D(1 + i, torch.relu(ln(p, f"prenet.norm_layers.{i}", x)), pp)
    x = (x_org + conv(p, "prenet.proj", x)) * m
    nb = p["encoder.attn_layers.0.table"].shape[0]
    near = {o: bucket(o, nb, False, max_distance) for o in range(-T, T + 1)}
    idx = torch.tensor([[near[j - i] for j in range(T)] for i in range(T)])
    shut = torch.where(live[:, None, None, :], 0.0, -1e30).to(x.dtype)   # a row without keys is masked afterwards
    h = ln(p, "encoder.norm_in", x) * m
    heads = lambda t: t.reshape(len(t), n_heads, C // n_heads, T).transpose(2, 3)
    for l in range(n_layers):
        a, f, site = f"encoder.attn_layers.{l}.", f"encoder.ffn_layers.{l}.", 16 + 8 * l
        q, k, v = (heads(conv(p, a + n, h)) for n in ("conv_q", "conv_k", "conv_v"))
        s = torch.matmul(q, k.transpose(2, 3)) * (C // n_heads) ** -0.5 + p[a + "table"][idx].permute(2, 0, 1)[None]
        y = torch.matmul(torch.softmax(s + shut, -1), v).transpose(2, 3).reshape(x.shape) * m
        y = D(site + 1, conv(p, a + "conv_o", y), pe)
        x = (x + ln(p, f"encoder.norm_post_1.{l}", y)) * m
        h = ln(p, f"encoder.norm_pre_1.{l}", x) * m
        y = D(site + 2, torch.relu(conv(p, f + "conv_1", h)), pe)
        y = D(site + 3, conv(p, f + "conv_2", y * m) * m, pe)
        x = (x + ln(p, f"encoder.norm_post_2.{l}", y)) * m
        h = ln(p, f"encoder.norm_pre_2.{l}", x) * m
    mu = conv(p, "proj_m", h) * m
    h = h.detach()
    d = D(8, ln(p, "proj_w.norm_1", torch.relu(conv(p, "proj_w.conv_1", h * m))), pe)
    d = D(9, ln(p, "proj_w.norm_2", torch.relu(conv(p, "proj_w.conv_2", d * m))), pe)
    return mu, conv(p, "proj_w.proj", d * m) * m, m
