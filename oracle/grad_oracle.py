"""Gradients of the layer's entry points in 64 bits, with bounds for a kernel that sums in fp32.  TEST INFRASTRUCTURE ONLY:
nothing in the product package imports this module.  Plain torch on whatever device the inputs are on.

Every function returns the gradient and, elementwise, how far an fp32 computation of the same definition may be from it
(the rounding of the result itself to bf16 not counted: ``half_step``)."""
import torch

BLOCK, FP8_MAX = 128, 448.0
X_FLOOR, GRAD_FLOOR = 1e-12, 1e-30
U = 2.0 ** -24          # half a step of fp32


def half_step(dtype):
    """Largest rounding error of ``dtype``, relative to the value."""
    return torch.finfo(dtype).eps / 2


def dequant_weights(q, s):
    """e4m3 [..., R, C] with scales [..., ceil(R/128), ceil(C/128)] -> fp64."""
    R, C = q.shape[-2:]
    return q.double() * s.double().repeat_interleave(BLOCK, -2)[..., :R, :].repeat_interleave(BLOCK, -1)[..., :C]


def quant_rows(v, floor):
    """Rows through e4m3 (per 128 columns).  ``v``: bf16 inputs (exact) or fp64 intermediates.  Returns (values as fp64,
    one step of e4m3 at each value times the scale, how far each scaled value is from the nearest rounding border
    relative to itself)."""
    R, C = v.shape
    pad = (-C) % BLOCK
    b = torch.nn.functional.pad(v.double(), (0, pad)).view(R, -1, BLOCK)
    top = b.abs().amax(-1, keepdim=True).float().clamp_min(floor)
    largest = torch.full_like(top, FP8_MAX)
    s = (top / largest).double()
    scaled32 = (b.float() * (largest / top)).clamp(-FP8_MAX, FP8_MAX)
    q = scaled32.to(torch.float8_e4m3fn).double()
    a = scaled32.double().abs()
    step = torch.exp2(torch.floor(torch.log2(a.clamp_min(2.0 ** -6))) - 3)    # e4m3: 3 bits, normal down to 2^-6
    border = torch.round(a / step - 0.5) + 0.5                                 # nearest half-odd multiple
    away = (a - border * step).abs()
    cut = lambda t: t.reshape(R, -1)[:, :C]  # noqa: E731
    return cut(q * s), cut(step * s), cut(away * s)


def route_backward(dw, logits, ids, score, renorm, scale, logit_bias=None, dw_bound=None):
    """``dw_bound``: how far dw itself may be from what is given here; the result's bound then covers that too."""
    T, E = logits.shape
    l = logits.double() + (logit_bias.double() if logit_bias is not None else 0.0)
    p = torch.softmax(l, -1) if score == "softmax" else torch.sigmoid(l)
    on = (ids >= 0) & (ids < E)
    safe = ids.clamp(0, E - 1).long()
    pj = p.gather(1, safe) * on
    d = dw.double() * on
    S = pj.sum(-1, keepdim=True)
    dp = scale * (d - (d * pj).sum(-1, keepdim=True) / S) / S if renorm else scale * d
    dp = dp * on
    dense = torch.zeros_like(l).scatter_add_(1, safe, dp)
    slope = p if score == "softmax" else p * (1 - p)
    mean = (dp * pj).sum(-1, keepdim=True) if score == "softmax" and not renorm else 0.0
    out = slope * (dense - mean)

    def reach(e):  # the same sums over the sizes of what goes into them
        size = scale * (e + (e * pj).sum(-1, keepdim=True) / S) / S if renorm else scale * e
        size = size * on
        spread = (size * pj).sum(-1, keepdim=True) if score == "softmax" and not renorm else 0.0
        return slope * (torch.zeros_like(l).scatter_add_(1, safe, size) + spread)

    big = reach(d.abs())
    # a few operations with k-fold and E-fold sums; expf is good to 2 steps and its argument l - m to one step of |l|
    k = ids.shape[1]
    bound = big * U * (2 * k + 40 + 4 * l[torch.isfinite(l)].abs().max() + E / 16)
    return out, bound if dw_bound is None else bound + reach(dw_bound.double() * on)


def combine_backward(dout, y, w, ids=None, E=0):
    d = dout.double()
    on = torch.ones_like(w, dtype=torch.bool) if ids is None else (ids >= 0) & (ids < E)
    yy = torch.where(on[..., None], y.double(), torch.zeros((), dtype=torch.float64, device=y.device))
    dy = torch.where(on[..., None], w.double()[..., None] * d[:, None], torch.zeros_like(yy))
    dw = (d[:, None] * yy).sum(-1)
    return dy, dy.abs() * U, dw, (d[:, None] * yy).abs().sum(-1) * U * 100   # sums 32 deep in a thread, then 5 + 8 additions, pieces


def product_bound(a, b, depth):
    """|a| @ |b| times what `depth` fp32 additions that may truncate (tensor cores do) can lose."""
    return (a.abs() @ b.abs()) * (2 * U * (depth + 8))


def router_backward(dlogits, x, wr):
    dl, xx, w = dlogits.double(), x.double(), wr.double()
    E = dl.shape[1]
    Ep = (E + 63) // 64 * 64
    lost = 2.0 ** -17                                                        # of dlogits, taken as two bf16 numbers
    dx, dwr = dl @ w, dl.t() @ xx
    bx = product_bound(dl, w, 2 * Ep) + (dl.abs() @ w.abs()) * lost
    bw = product_bound(dl.t(), xx, min(dl.shape[0], 2048) + 64) + (dl.abs().t() @ xx.abs()) * lost
    return dx, bx, dwr, bw


def linear_backward(dy, x, w, scale):
    q, _, _ = quant_rows(dy, GRAD_FLOOR)
    W = dequant_weights(w, scale)
    nk = (dy.shape[1] + 127) // 128
    d, xx = dy.double(), x.double()
    return (q @ W, product_bound(q, W, nk + 8), d.t() @ xx, product_bound(d.t(), xx, min(dy.shape[0], 2048) + 64))


def experts_backward(dout, x, wg, wu, wd, sg, su, sd, ids, topk_w=None, add=None):
    """dict of (value, bound) for dx, dw, dwg, dwu, dwd; dout [T,H] with topk_w or [T,k,H]."""
    T, k = ids.shape
    H, (E, I, _) = x.shape[1], wg.shape
    dev, f8 = x.device, dict(dtype=torch.float64, device=x.device)
    per_slot = dout.dim() == 3
    dx, bx, dw, bw = torch.zeros(T, H, **f8), torch.zeros(T, H, **f8), torch.zeros(T, k, **f8), torch.zeros(T, k, **f8)
    G = [torch.zeros(E, I, H, **f8) for _ in range(3)]
    B = [torch.zeros(E, I, H, **f8) for _ in range(3)]
    xq, _, _ = quant_rows(x, X_FLOOR)
    dq, _, _ = quant_rows(dout.reshape(-1, H), GRAD_FLOOR)
    op = half_step(torch.bfloat16)   # weight gradients take dg, du, w h in bf16
    for e in range(E):
        t, j = (ids == e).nonzero(as_tuple=True)
        if t.numel() == 0:
            continue
        Wg, Wu, Wd = dequant_weights(wg[e], sg[e]), dequant_weights(wu[e], su[e]), dequant_weights(wd[e], sd[e])
        a, d0 = xq[t], dq[t * k + j] if per_slot else dq[t]
        g, u, d = a @ Wg.t(), a @ Wu.t(), d0 @ Wd.t()
        nk = H // 128 + 8
        eg, eu, ed = product_bound(a, Wg.t(), nk), product_bound(a, Wu.t(), nk), product_bound(d0, Wd.t(), nk)
        s = torch.sigmoid(g)
        act, slope = g * s, s * (1 + g * (1 - s))
        es, ea = 0.25 * eg + s * 8 * U * (1 + g.abs()), 1.1 * eg + act.abs() * 8 * U * (1 + g.abs())
        h = act * u
        eh = ea * u.abs() + act.abs() * eu + h.abs() * 4 * U
        w = topk_w.double()[t, j][:, None] if not per_slot else torch.ones(t.numel(), 1, **f8)
        dw[t, j] = (h * d).sum(-1)
        bw[t, j] = (eh * d.abs() + h.abs() * ed).sum(-1) + (h * d).abs().sum(-1) * U * (64 + I / 32)
        dg, du = w * d * u * slope, w * d * act
        wa = w.abs()
        edg = wa * (ed * (u * slope).abs() + d.abs() * eu * slope.abs() + (d * u).abs() * (0.5 * eg + es * 0.01)) + dg.abs() * 16 * U * (1 + g.abs()) \
            + wa * (d * u).abs() * s * 8 * U * (1 + g.abs())
        edu = wa * (ed * act.abs() + d.abs() * ea) + du.abs() * 8 * U
        val, bound = torch.zeros(t.numel(), H, **f8), torch.zeros(t.numel(), H, **f8)
        for v, ev, W in ((dg, edg, Wg), (du, edu, Wu)):
            q, step, away = quant_rows(v, GRAD_FLOOR)
            # a value this near to a border may be rounded to the other side; the group's scale moves with its largest value
            top = ev.view(-1, I // 128, 128).amax(-1, keepdim=True) / v.abs().view(-1, I // 128, 128).amax(-1, keepdim=True).clamp_min(1e-300)
            rel = top.expand(-1, -1, 128).reshape(v.shape) + 4 * U
            eq = torch.where(away <= ev + v.abs() * rel, step, torch.zeros_like(step)) + q.abs() * rel
            val += q @ W
            bound += product_bound(q, W, 2 * I // 128 + 16) + eq @ W.abs()
        bound += (val.abs() + bound) * op      # a slot's row may be rounded to bf16 before the sum
        dx.index_add_(0, t, val)
        bx.index_add_(0, t, bound)
        rows = (dout.reshape(-1, H)[t * k + j] if per_slot else dout[t]).double()
        for i, (v, ev, r) in enumerate(((dg, edg, x[t].double()), (du, edu, x[t].double()), (w * h, wa * eh, rows))):
            G[i][e] = v.t() @ r
            B[i][e] = product_bound(v.t(), r, min(t.numel(), 2048) + 64) + ((v.abs() + ev) * op + ev).t() @ r.abs()
    if add is not None:
        dx = dx + add.double()
    bx = bx + dx.abs() * U * (k + 4)
    return {"dx": (dx, bx), "dw": (dw, bw), "dwg": (G[0], B[0]), "dwu": (G[1], B[1]), "dwd": (G[2], B[2])}
