"""The gradients of the routed FP8 layer: what a program that trains through it calls, and with which sizes.

Each operator is the gradient of a forward entry point of the same name:

  route     ops.route_backward           of the routing weights, with respect to the logits
  router    ops.router_logits_backward   of the router's product, with respect to the tokens and the router's weights
  combine   ops.combine_backward         of the weighted combine, with respect to the experts' rows and the routing weights
  experts   ops.experts_backward         of the FP8 experts, with respect to the tokens, the routing weights and (`wgrad`)
                                         the experts' weights
  linear    ops.linear_w8_backward       of the FP8 linear layer, with respect to its input and its weights

Activations and gradients enter an FP8 product quantised to e4m3, per row and 128 columns (scale = largest magnitude /
448); that quantisation is part of the operators' definition, and gradients pass it unchanged.  Shapes are those of
perf/cases.py: a small layer, the Mixtral-8x7B, DeepSeek-V3 and Qwen3-30B-A3B layers, random weights in e4m3 with a scale
for each block of 128 x 128."""
import math

import torch

own = False  # False: the plain forms; True: the framework's operators
DEV = "cuda:0"

SHAPES = {
    "small": dict(H=1024, I=512, E=8, k=2),
    "mixtral": dict(H=4096, I=14336, E=8, k=2),
    "deepseek": dict(H=7168, I=2048, E=256, k=8),
    "qwen": dict(H=2048, I=768, E=128, k=8),
}
BLOCK, FP8_MAX = 128, 448.0
X_FLOOR, GRAD_FLOOR = 1e-12, 1e-30  # smallest magnitude that a scale is made for: activations, gradients


def _experts(name, shape, tokens, wgrad, rows="combined", scales="fp32"):
    return {"name": name, "op": "experts", "shape": shape, "tokens": tokens, "wgrad": wgrad, "rows": rows, "scales": scales}


def listed():
    return [
        # the smallest routing gradient: one micro-batch of the small layer, latency is all there is
        {"name": "route_16", "op": "route", "tokens": 16, "E": 8, "k": 2, "score": "softmax", "renorm": True},
        # a training batch over 256 fine experts, sigmoid scores
        {"name": "route_8192", "op": "route", "tokens": 8192, "E": 256, "k": 8, "score": "sigmoid", "renorm": True},
        # the small layer's router
        {"name": "router_16", "op": "router", "tokens": 16, "H": 1024, "E": 8},
        # a router of 256 experts on a training batch of odd length
        {"name": "router_2047", "op": "router", "tokens": 2047, "H": 7168, "E": 256},
        # the small layer's combine
        {"name": "combine_16", "op": "combine", "tokens": 16, "H": 1024, "k": 2, "weights": "fp32"},
        # eight experts' rows for each token of a training batch
        {"name": "combine_2048", "op": "combine", "tokens": 2048, "H": 7168, "k": 8, "weights": "fp32"},
        # a projection's gradient on a handful of tokens: the weights are streamed
        {"name": "linear_16", "op": "linear", "tokens": 16, "K": 4096, "N": 6144},
        # a projection on a chunk of odd length
        {"name": "linear_1001", "op": "linear", "tokens": 1001, "K": 4096, "N": 6144},
        # all gradients of the small layer's experts
        _experts("experts_small_16", "small", 16, True),
        # fine-grained experts with heavy-tailed loads, ragged batch, all gradients
        _experts("experts_qwen_777", "qwen", 777, True),
        # a training batch over large experts, all gradients: the tensor cores' case
        _experts("experts_mixtral_4096", "mixtral", 4096, True),
        # fine-tuning what lies below frozen experts: no weight gradients
        _experts("experts_deepseek_2048", "deepseek", 2048, False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        c = _draw(rng)
        if all({**c, "name": d["name"]} != d for d in listed()):  # another case than the listed ones
            return c


def _draw(rng):
    op = rng.choice(["route", "router", "combine", "linear", "linear", "experts", "experts", "experts"])
    if op == "route":
        E = rng.choice([8, 64, 128, 256, rng.randint(2, 300)])
        k = rng.randint(1, min(E, 10))
        return {"op": op, "tokens": _log_int(rng, 1, 16384), "E": E, "k": k, "score": rng.choice(["softmax", "sigmoid"]),
                "renorm": k > 1 and rng.random() < 0.6}  # (one renormalised weight is constant: its gradient is zero)
    if op == "router":
        return {"op": op, "tokens": _log_int(rng, 1, 8192), "H": rng.choice([1024, 2048, 4096, 7168, 8 * rng.randint(16, 900)]),
                "E": rng.choice([8, 128, 256, rng.randint(2, 300)])}
    if op == "combine":
        return {"op": op, "tokens": _log_int(rng, 1, 4096), "H": rng.choice([1024, 2048, 4096, 7168, 8 * rng.randint(16, 900)]),
                "k": rng.randint(1, 8), "weights": rng.choice(["fp32", "bf16"])}
    if op == "linear":
        return {"op": op, "tokens": _log_int(rng, 1, 4096), "K": 128 * rng.randint(8, 56), "N": 64 * rng.randint(16, 128)}
    shape = rng.choice(["small", "mixtral", "deepseek", "qwen", "qwen"])
    most = {"small": 4096, "mixtral": 4096, "deepseek": 2048, "qwen": 8192}[shape]
    c = _experts("", shape, _log_int(rng, 1, most), shape != "deepseek" and rng.random() < 0.6,
                 rng.choice(["combined", "combined", "per_slot"]), rng.choice(["fp32", "bf16"]))
    c.pop("name")
    return c


# ---- inputs ------------------------------------------------------------------------------------------------------
def _grad(g, *size):
    """A loss's gradient: rows of different magnitude."""
    rows = torch.randn(size[0], *[1] * (len(size) - 1), generator=g, device=DEV).exp()
    return (torch.randn(*size, generator=g, device=DEV) * rows * 1e-3)


def _fp8_weights(g, E, R, C, dtype):
    """What quantising N(0, 0.02) by blocks gives: e4m3 values that fill the range, scales that vary a little."""
    q = torch.empty(E, R, C, dtype=torch.float8_e4m3fn, device=DEV)
    step = max(1, (1 << 28) // (R * C))
    for e in range(0, E, step):
        q[e:e + step] = torch.randn(min(step, E - e), R, C, generator=g, device=DEV).mul_(107.0).clamp_(-FP8_MAX, FP8_MAX)
    s = (0.9 + 0.2 * torch.rand(E, (R + BLOCK - 1) // BLOCK, (C + BLOCK - 1) // BLOCK, generator=g, device=DEV)) * (0.02 / 107.0)
    return q, s.to(torch.bfloat16 if dtype == "bf16" else torch.float32)


def _routing(g, T, E, k, skewed):
    """Distinct experts of each token, and normalised weights; `skewed`: heavy-tailed loads."""
    logits = torch.randn(T, E, generator=g, device=DEV)
    if skewed:
        rank = torch.randperm(E, generator=g, device=DEV) + 1
        logits -= 3.0 * 1.2 * rank.log()
    w, ids = logits.softmax(-1).topk(k, dim=-1)
    return ids.to(torch.int32), (w / w.sum(-1, keepdim=True)).contiguous()


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(seed)
    T = c["tokens"]
    s = {"case": c}
    normal = lambda *size: torch.randn(*size, generator=g, device=DEV).to(torch.bfloat16)  # noqa: E731
    if c["op"] == "route":
        s["logits"] = torch.randn(T, c["E"], generator=g, device=DEV)
        s["ids"] = s["logits"].topk(c["k"], dim=-1)[1].to(torch.int32)
        s["dw"] = _grad(g, T, c["k"])
    elif c["op"] == "router":
        s["x"], s["wr"] = normal(T, c["H"]), (torch.randn(c["E"], c["H"], generator=g, device=DEV) * 0.02).to(torch.bfloat16)
        s["dlogits"] = _grad(g, T, c["E"])
    elif c["op"] == "combine":
        s["dout"], s["y"] = _grad(g, T, c["H"]).to(torch.bfloat16), normal(T, c["k"], c["H"])
        s["w"] = torch.rand(T, c["k"], generator=g, device=DEV).to(torch.bfloat16 if c["weights"] == "bf16" else torch.float32)
    elif c["op"] == "linear":
        s["dy"], s["x"] = _grad(g, T, c["N"]).to(torch.bfloat16), normal(T, c["K"])
        q, scale = _fp8_weights(g, 1, c["N"], c["K"], "fp32")
        s["w"], s["scale"] = q[0], scale[0]
    else:
        z = SHAPES[c["shape"]]
        s["x"] = normal(T, z["H"])
        s["dout"] = _grad(g, *((T, z["H"]) if c["rows"] == "combined" else (T, z["k"], z["H"]))).to(torch.bfloat16)
        s["ids"], s["topk_w"] = _routing(g, T, z["E"], z["k"], c["shape"] == "qwen")
        parts = [_fp8_weights(g, z["E"], z["I"], z["H"], c["scales"]) for _ in range(3)]
        s["weights"], s["scales"] = [p[0] for p in parts], [p[1] for p in parts]
    return s


# ---- one pass ----------------------------------------------------------------------------------------------------
def run(state):
    return _run_own(state) if own else _PLAIN[state["case"]["op"]](state)


def _run_own(s):
    from torch_tpu_b200 import ops

    c = s["case"]
    if c["op"] == "route":
        return ops.route_backward(s["dw"], s["logits"], s["ids"], c["score"], c["renorm"], _scale(c))
    if c["op"] == "router":
        return ops.router_logits_backward(s["dlogits"], s["x"], s["wr"])
    if c["op"] == "combine":
        return ops.combine_backward(s["dout"], s["y"], s["w"])
    if c["op"] == "linear":
        return ops.linear_w8_backward(s["dy"], s["x"], s["w"], s["scale"])
    grads = [torch.empty_like(w, dtype=torch.bfloat16) for w in s["weights"]] if c["wgrad"] else None
    dx, dw = ops.experts_backward(s["dout"], s["x"], *s["weights"], *s["scales"], s["ids"],
                                  s["topk_w"] if c["rows"] == "combined" else None, weight_grads=grads)
    return {"dx": dx, "dw": dw, "weights": grads}


def _scale(c):
    return 2.5 if c["score"] == "sigmoid" else 1.0


def _quantised(x, floor):
    """Rows through e4m3 with a scale for each 128 columns, as fp32 values."""
    R, C = x.shape
    b = torch.nn.functional.pad(x.float(), (0, -C % BLOCK)).view(R, -1, BLOCK)
    amax = b.abs().amax(-1, keepdim=True).clamp_min(floor)
    top = torch.full_like(amax, FP8_MAX)  # (a division by a Python number would multiply by its rounded inverse)
    q = (b * (top / amax)).clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn).float()
    return (q * (amax / top)).reshape(R, -1)[:, :C]


def _dequantised(w, s):
    R, C = w.shape
    return w.float() * s.float().repeat_interleave(BLOCK, 0)[:R].repeat_interleave(BLOCK, 1)[:, :C]


def _plain_route(s):
    c, ids, dw = s["case"], s["ids"].long(), s["dw"]
    score = s["logits"].softmax(-1) if c["score"] == "softmax" else s["logits"].sigmoid()
    p = score.gather(1, ids)
    if c["renorm"]:
        S = p.sum(-1, keepdim=True)
        ds = _scale(c) * (dw - (dw * p).sum(-1, keepdim=True) / S) / S
    else:
        ds = _scale(c) * dw
    dense = torch.zeros_like(score).scatter_add_(1, ids, ds)
    if c["score"] == "softmax":
        return score * (dense - (ds * p).sum(-1, keepdim=True))
    return dense * score * (1 - score)


def _plain_router(s):
    return (s["dlogits"] @ s["wr"].float()).to(torch.bfloat16), s["dlogits"].t() @ s["x"].float()


def _plain_combine(s):
    dout = s["dout"].float()[:, None, :]
    return (s["w"].float()[..., None] * dout).to(torch.bfloat16), (dout * s["y"].float()).sum(-1)


def _plain_linear(s):
    dx = _quantised(s["dy"], GRAD_FLOOR) @ _dequantised(s["w"], s["scale"])
    return dx.to(torch.bfloat16), s["dy"].float().t() @ s["x"].float()


def _plain_experts(s):
    c, ids, x, dout = s["case"], s["ids"], s["x"], s["dout"]
    (T, k), H = ids.shape, x.shape[1]
    E, I, _ = s["weights"][0].shape
    combined = c["rows"] == "combined"
    grads = [torch.zeros(E, I, H, dtype=torch.bfloat16, device=x.device) for _ in range(3)] if c["wgrad"] else None
    slots = torch.zeros(T * k, H, device=x.device)
    dw = torch.zeros(T * k, device=x.device) if combined else None
    flat = ids.reshape(-1)
    order = flat.argsort(stable=True)
    ends = torch.bincount(flat, minlength=E).cumsum(0).tolist()
    for e in range(E):  # every expert has rows of its own, and another number of them
        pairs = order[ends[e - 1] if e else 0:ends[e]]
        if not len(pairs):
            continue
        wg, wu, wd = (_dequantised(w[e], sc[e]) for w, sc in zip(s["weights"], s["scales"]))
        xe = x[pairs // k]
        de = dout[pairs // k] if combined else dout.view(T * k, H)[pairs]
        xq, dq = _quantised(xe, X_FLOOR), _quantised(de, GRAD_FLOOR)
        gate, up, dh = xq @ wg.t(), xq @ wu.t(), dq @ wd.t()
        sg = gate.sigmoid()
        act = gate * sg
        h = act * up
        if combined:
            weight = s["topk_w"].view(-1)[pairs][:, None]
            dw[pairs] = (h * dh).sum(-1)
            dh, h = weight * dh, weight * h
        dgate, dup = dh * up * (sg + act * (1 - sg)), dh * act
        slots[pairs] = _quantised(dgate, GRAD_FLOOR) @ wg + _quantised(dup, GRAD_FLOOR) @ wu
        if grads:
            for out, a, b in zip(grads, (dgate, dup, h), (xe, xe, de)):
                out[e] = a.t() @ b.float()
    return {"dx": slots.view(T, k, H).sum(1).to(torch.bfloat16), "dw": dw.view(T, k) if combined else None, "weights": grads}


_PLAIN = {"route": _plain_route, "router": _plain_router, "combine": _plain_combine, "linear": _plain_linear,
          "experts": _plain_experts}


# ---- what a pass cannot do without -------------------------------------------------------------------------------
def work(case):
    c, T = case, case["tokens"]
    if c["op"] == "route":
        E, k = c["E"], c["k"]
        read = T * E * 4 if c["score"] == "softmax" and not c["renorm"] else T * k * 4  # else the selected logits alone matter
        return {"bytes": read + T * E * 4 + T * k * 8, "flops": 8 * T * E}
    if c["op"] == "router":
        E, H = c["E"], c["H"]
        return {"bytes": T * E * 4 + E * H * 2 + 2 * T * H * 2 + E * H * 4, "flops": 4 * T * E * H}
    if c["op"] == "combine":
        k, H = c["k"], c["H"]
        return {"bytes": T * H * 2 + 2 * T * k * H * 2 + T * k * 8, "flops": 3 * T * k * H}
    if c["op"] == "linear":
        K, N = c["K"], c["N"]
        return {"bytes": T * N * 2 + 2 * T * K * 2 + N * K + N * K * 4, "flops": 4 * T * N * K}
    z = SHAPES[c["shape"]]
    P, HI = T * z["k"], z["H"] * z["I"]
    rows = T * z["H"] * 2 * (2 + (1 if c["rows"] == "combined" else z["k"]))
    grads = 3 * z["E"] * HI * 2 if c["wgrad"] else 0
    return {"bytes": 3 * min(z["E"], P) * HI + rows + grads + P * 12, "flops": (16 if c["wgrad"] else 10) * P * HI}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------
def _through_e4m3(v, floor):
    """The same quantisation of a 64-bit (or an input's) row: the scale and its inverse are fp32 numbers by definition."""
    rows, cols = v.shape
    out = torch.zeros(rows, cols, dtype=torch.float64, device=v.device)
    for b in range(0, cols, BLOCK):
        part = v[:, b:b + BLOCK]
        top = part.abs().amax(1, keepdim=True).float().clamp_min(floor)
        largest = torch.full_like(top, FP8_MAX)
        scaled = (part.float() * (largest / top)).clamp(-FP8_MAX, FP8_MAX)
        out[:, b:b + BLOCK] = scaled.to(torch.float8_e4m3fn).double() * (top / largest).double()
    return out


def _weights64(q, s):
    out = q.double()
    for i in range(s.shape[0]):
        out[i * BLOCK:(i + 1) * BLOCK] *= s[i].double().repeat_interleave(BLOCK)[:q.shape[1]]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["op"] == "route":
        l, dw = s["logits"].double(), s["dw"].double()
        l.requires_grad_(True)
        score = (l - l.detach().amax(1, keepdim=True)).exp() if c["score"] == "softmax" else 1 / (1 + (-l).exp())
        if c["score"] == "softmax":
            score = score / score.sum(1, keepdim=True)
        w = score.gather(1, s["ids"].long())
        if c["renorm"]:
            w = w / w.sum(1, keepdim=True)
        return torch.autograd.grad((w * _scale(c) * dw).sum(), l)[0]
    if c["op"] == "router":
        return s["dlogits"].double() @ s["wr"].double(), s["dlogits"].double().t() @ s["x"].double()
    if c["op"] == "combine":
        d = s["dout"].double()
        return (torch.einsum("tk,th->tkh", s["w"].double(), d), torch.einsum("th,tkh->tk", d, s["y"].double()))
    if c["op"] == "linear":
        return (_through_e4m3(s["dy"], GRAD_FLOOR) @ _weights64(s["w"], s["scale"]), s["dy"].double().t() @ s["x"].double())
    ids, x, dout = s["ids"].long(), s["x"], s["dout"]
    T, k = ids.shape
    combined = c["rows"] == "combined"
    dx = torch.zeros(T, x.shape[1], dtype=torch.float64, device=x.device)
    dw = torch.zeros(T, k, dtype=torch.float64, device=x.device)
    xq = _through_e4m3(x, X_FLOOR)
    dq = _through_e4m3(dout.reshape(-1, x.shape[1]), GRAD_FLOOR).view(dout.shape)
    grads = [torch.zeros(w.shape, dtype=torch.float64, device=x.device) for w in s["weights"]] if c["wgrad"] else None
    for e in range(s["weights"][0].shape[0]):
        t, j = (ids == e).nonzero(as_tuple=True)
        if t.numel() == 0:
            continue
        wg, wu, wd = (_weights64(q[e], sc[e]) for q, sc in zip(s["weights"], s["scales"]))
        gate, up = xq[t] @ wg.t(), xq[t] @ wu.t()
        gate.requires_grad_(True)
        up.requires_grad_(True)
        h = gate / (1 + (-gate).exp()) * up
        d = (dq[t] if combined else dq[t, j]) @ wd.t()
        weight = s["topk_w"].double()[t, j][:, None] if combined else torch.ones_like(d[:, :1])
        dgate, dup = torch.autograd.grad((h * weight * d).sum(), (gate, up))
        h = h.detach()
        dw[t, j] = (h * d).sum(1)
        dx.index_add_(0, t, _through_e4m3(dgate, GRAD_FLOOR) @ wg + _through_e4m3(dup, GRAD_FLOOR) @ wu)
        if grads:
            rows = (dout[t] if combined else dout[t, j]).double()
            grads[0][e], grads[1][e], grads[2][e] = dgate.t() @ x[t].double(), dup.t() @ x[t].double(), (h * weight).t() @ rows
    return {"dx": dx, "dw": dw if combined else None, "weights": grads}
