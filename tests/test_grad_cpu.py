"""Gradients without a GPU: the 64-bit definitions (oracle/grad_oracle.py) against differences of the forward definitions, the
entry points' refusals, workspace sizes."""
import ctypes
import os

import pytest
import torch

from oracle import grad_oracle as G


@pytest.fixture(scope="module")
def m():
    import torch_tpu_b200
    if not os.path.exists(torch_tpu_b200.lib.LIB_PATH):
        from importlib import import_module
        import_module("torch_tpu_b200.build").build_all()
    return torch_tpu_b200


# ---- the definitions against differences ---------------------------------------------------------------------------------
def scores(logits, score):
    return torch.softmax(logits, -1) if score == "softmax" else torch.sigmoid(logits)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
def test_route_definition(score, renorm):
    g = torch.Generator().manual_seed(1)
    T, E, k, h = 3, 9, 4, 1e-4
    logits, dw = torch.randn(T, E, generator=g, dtype=torch.float64), torch.randn(T, k, generator=g, dtype=torch.float64)
    ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)]).to(torch.int32)

    def loss(l):
        w = scores(l, score).gather(1, ids.long())
        w = w / w.sum(-1, keepdim=True) if renorm else w
        return (2.5 * w * dw).sum()

    num = torch.zeros_like(logits)
    for t in range(T):
        for e in range(E):
            d = torch.zeros_like(logits)
            d[t, e] = h
            num[t, e] = (loss(logits + d) - loss(logits - d)) / (2 * h)
    got, _ = G.route_backward(dw, logits, ids, score, renorm, 2.5)
    assert (got - num).abs().max() < 1e-6        # h^2 / 6 times third derivatives of order 10


def exact_rows(g, R, C, lo, hi):
    """Rows that e4m3 quantisation leaves as they are: one 448 (times a power of two) in each group of 128, other values e4m3."""
    v = torch.randn(R, C, generator=g).mul(40).clamp(-448, 448).to(torch.float8_e4m3fn).double()
    v.view(R, -1, 128)[:, :, 0] = 448.0
    return v * torch.exp2(torch.randint(lo, hi, (R, 1), generator=g).double())


def problem(T, H, I, E, k):
    g = torch.Generator().manual_seed(T + I)
    x, dout = exact_rows(g, T, H, -8, -6).bfloat16(), exact_rows(g, T, H, -9, -6).bfloat16()
    w = [(torch.randn(E, I, H, generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn) for _ in range(3)]
    s = [(torch.rand(E, I // 128, H // 128, generator=g) + 0.5) * 2e-4 for _ in range(3)]
    ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)]).to(torch.int32)
    return x, dout, w, s, ids, torch.rand(T, k, generator=g) + 0.1


def forward64(x, W, ids, topk_w):
    """out[t] = sum_j w[t,j] (silu(x Wg^T) * x Wu^T) Wd, in 64 bits and without quantisation; W: three fp64 [E,I,H]."""
    out = torch.zeros_like(x)
    for t in range(x.shape[0]):
        for j in range(ids.shape[1]):
            e = int(ids[t, j])
            g, u = W[0][e] @ x[t], W[1][e] @ x[t]
            out[t] += topk_w[t, j] * ((g * torch.sigmoid(g) * u) @ W[2][e])
    return out


def test_experts_definition_against_differences():
    """Where x and dout are what their quantisation gives, the weights' and the routing weights' gradients are those of the
    unquantised function."""
    T, H, I, E, k = 4, 128, 128, 3, 2
    x, dout, w, s, ids, tw = problem(T, H, I, E, k)
    W = [G.dequant_weights(a, b) for a, b in zip(w, s)]
    q, _, _ = G.quant_rows(x, G.X_FLOOR)
    assert torch.equal(q, x.double())
    got = G.experts_backward(dout, x, *w, *s, ids, tw)
    X, D, TW = x.double(), dout.double(), tw.double()
    loss = lambda ww=W, tt=TW: (forward64(X, ww, ids, tt) * D).sum()  # noqa: E731
    h = 1e-5
    for t in range(T):
        for j in range(k):
            d = torch.zeros_like(TW)
            d[t, j] = h
            num = (loss(tt=TW + d) - loss(tt=TW - d)) / (2 * h)
            assert abs(got["dw"][0][t, j] - num) <= 1e-6 * got["dw"][0].abs().max()
    g = torch.Generator().manual_seed(5)
    for i, name in enumerate(("dwg", "dwu", "dwd")):
        for _ in range(3):  # along random directions
            d = torch.randn(E, I, H, generator=g, dtype=torch.float64) * W[i].abs().mean()
            step = lambda c: [W[n] + c * d if n == i else W[n] for n in range(3)]  # noqa: E731
            num = (loss(ww=step(h)) - loss(ww=step(-h))) / (2 * h)
            assert abs((got[name][0] * d).sum() - num) <= 1e-6 * (got[name][0].abs() * d.abs()).sum()


def test_experts_dx_definition_against_differences():
    """dx passes through the quantisation of dgate and dup: off the unquantised gradient by half a step of e4m3 of each."""
    T, H, I, E, k = 3, 128, 256, 2, 1
    x, dout, w, s, ids, tw = problem(T, H, I, E, k)
    W = [G.dequant_weights(a, b) for a, b in zip(w, s)]
    got = G.experts_backward(dout, x, *w, *s, ids, tw)["dx"][0]
    X, D = x.double().requires_grad_(True), dout.double()
    exact, = torch.autograd.grad((forward64(X, W, ids, tw.double()) * D).sum(), X)
    bound = torch.zeros_like(exact)
    half = G.half_step(torch.float8_e4m3fn)
    for t in range(T):
        e = int(ids[t, 0])
        g, u, d = W[0][e] @ x[t].double(), W[1][e] @ x[t].double(), W[2][e] @ D[t] * tw[t, 0].double()
        sg = torch.sigmoid(g)
        for v, M in ((d * u * sg * (1 + g * (1 - sg)), W[0][e]), (d * g * sg, W[1][e])):
            small = v.abs().view(-1, 128).amax(-1, keepdim=True).expand(-1, 128).reshape(-1) / 448 * 2.0 ** -10  # half a subnormal step
            bound[t] += torch.maximum(v.abs() * half, small) @ M.abs()
    assert ((got - exact).abs() <= bound * (1 + 1e-9)).all()
    assert (got - exact).abs().max() > 0


def test_quantisation_definition():
    """Zero rows, half a group, values below the floor."""
    v = torch.zeros(3, 192, dtype=torch.float64)
    v[1] = torch.linspace(-3, 3, 192)
    v[2] = 1e-33
    q, step, away = G.quant_rows(v, G.GRAD_FLOOR)
    assert not q[0].any() and q.shape == (3, 192)
    assert (q[1] - v[1]).abs().max() <= 3 * 2.0 ** -4
    assert (q[2] <= 1e-32).all()


# ---- refusals ---------------------------------------------------------------------------------------------------------------
def test_host_side_rejections(m):
    L, l = m.lib, m.lib.lib()
    null, one, odd = None, 4096, 4104
    r = l.b200moe_route_backward
    assert r(one, one, null, one, one, 0, 0, 8, 2, 0, 1, 1.0, null) == L.OK                 # empty batch
    assert r(null, null, null, null, null, 0, 0, 8, 2, 0, 1, 1.0, null) == L.OK
    assert r(null, one, null, one, one, 0, 4, 8, 2, 0, 1, 1.0, null) == L.EINVAL
    assert r(one, one, null, one, one, 0, 4, 8, 2, 7, 1, 1.0, null) == L.EINVAL             # unknown score
    assert r(one, one, null, one, one, L.F16, 4, 8, 2, 0, 1, 1.0, null) == L.EINVAL
    assert r(one, one, null, one, one, 0, -1, 8, 2, 0, 1, 1.0, null) == L.EINVAL
    for E, k in ((2048, 2), (64, 33), (4, 5)):
        assert r(one, one, null, one, one, 0, 4, E, k, 0, 1, 1.0, null) == L.ESHAPE
    c = l.b200moe_combine_backward
    assert c(null, null, null, null, null, 0, null, 0, 0, 2, 128, null) == L.OK
    assert c(null, null, one, one, one, 0, null, 0, 4, 2, 128, null) == L.EINVAL            # nothing asked for
    assert c(one, one, one, null, one, 0, null, 0, 4, 2, 128, null) == L.EINVAL             # dw without y
    assert c(one, null, one, one, null, 0, null, 0, 4, 2, 128, null) == L.EINVAL            # dy without w
    assert c(one, one, one, one, one, 0, one, 0, 4, 2, 128, null) == L.EINVAL               # ids without E
    assert c(one, one, one, one, one, 9, null, 0, 4, 2, 128, null) == L.EINVAL
    assert c(one, one, one, one, one, 0, null, 0, 4, 2, 12, null) == L.ESHAPE
    assert c(one, one, one, one, one, 0, null, 0, 4, 33, 128, null) == L.ESHAPE
    assert c(odd, one, one, one, one, 0, null, 0, 4, 2, 128, null) == L.EALIGN
    w = l.b200moe_router_logits_backward
    args = lambda **k: [k.get(n, d) for n, d in (("dx", one), ("add", 0), ("dwr", one), ("dt", 0), ("acc", 0), ("dl", one), ("x", one),  # noqa: E731
                                                 ("wr", one), ("T", 4), ("H", 128), ("E", 8), ("ws", one), ("n", 1 << 30), ("st", null), ("s", null))]
    assert w(*args(T=0, dwr=null)) == L.OK and w(*args(T=0, dx=null, dwr=null, dl=null, x=null, wr=null, add=1, ws=null, n=0)) == L.OK
    for bad in (dict(dx=null, dwr=null), dict(dx=null, add=1), dict(add=2), dict(dt=2), dict(dt=1, acc=1), dict(acc=2), dict(dl=null), dict(x=null),
                dict(wr=null), dict(E=0), dict(H=-8)):
        assert w(*args(**bad)) == L.EINVAL, bad
    assert w(*args(H=100)) == L.ESHAPE and w(*args(E=1025)) == L.ESHAPE and w(*args(T=1 << 24)) == L.ESHAPE
    for p in ("dx", "wr", "dwr", "x"):
        assert w(*args(**{p: odd})) == L.EALIGN
    n = l.b200moe_linear_w8_backward
    args = lambda **k: [k.get(a, d) for a, d in (("dx", one), ("dw", one), ("dt", 0), ("acc", 0), ("dy", one), ("x", one), ("w", one),  # noqa: E731
                                                 ("sc", one), ("sdt", 0), ("M", 4), ("K", 128), ("N", 64), ("ws", one), ("n", 1 << 30), ("st", null),
                                                 ("s", null))]
    assert n(*args(M=0, dw=null)) == L.OK and n(*args(M=0, dx=null, dw=null, dy=null, x=null, w=null, sc=null, ws=null, n=0)) == L.OK
    for bad in (dict(dx=null, dw=null), dict(dt=2), dict(dt=1, acc=1), dict(dy=null), dict(x=null), dict(w=null), dict(sc=null), dict(sdt=2), dict(K=0)):
        assert n(*args(**bad)) == L.EINVAL, bad
    assert n(*args(K=100)) == L.ESHAPE and n(*args(N=100)) == L.ESHAPE and n(*args(M=1 << 24)) == L.ESHAPE
    for p in ("dx", "w", "dw", "x", "dy"):
        assert n(*args(**{p: odd})) == L.EALIGN


def test_experts_rejections(m):
    L, l, ops = m.lib, m.lib.lib(), m.ops
    names = ["dx", "dw", "dwg", "dwu", "dwd", "dout", "x", "wg", "wu", "wd", "sg", "su", "sd", "ids", "w", "add"]
    base = dict(T=4, H=256, I=128, E=4, k=2)

    def call(ptr=None, **kw):
        d = dict(base, per_slot=0, scale_dtype=0, w_dtype=0, weight_grads=1, grad_dtype=0, accumulate=0)
        d.update(kw)
        p = dict({n: 4096 for n in names}, add=None)
        p.update(ptr or {})
        return l.b200moe_experts_backward(*[p[n] for n in names], ctypes.byref(L.ExpertsBackwardDesc(**d)), 4096, 1 << 40, None, None)

    for bad in (dict(T=-1), dict(k=0), dict(per_slot=2), dict(scale_dtype=2), dict(w_dtype=2), dict(weight_grads=3), dict(grad_dtype=2),
                dict(grad_dtype=1, accumulate=1), dict(per_slot=1)):      # (per_slot: topk_w and dw must be NULL)
        assert call(**bad) == L.EINVAL, bad
    for bad in (dict(H=100), dict(I=64), dict(E=1025), dict(T=1 << 23), dict(T=1 << 40, k=1 << 40)):
        assert call(**bad) == L.ESHAPE, bad
    for n in ("dwg", "dout", "x", "wu", "sd", "ids", "w"):
        assert call({n: None}) == L.EINVAL, n
    assert call({"dx": None, "add": 4096}) == L.EINVAL
    assert call({"dx": None, "dw": None}, weight_grads=0) == L.EINVAL
    assert call({n: None for n in names}, weight_grads=0, T=0) == L.OK      # an empty batch needs no pointers
    for n in ("dx", "dwd", "dout", "x", "wg", "add"):
        assert call({n: 4104}) == L.EALIGN, n
    if not torch.cuda.is_available():
        assert call() == L.EDRIVER            # nothing to run on: no other path
    assert l.b200moe_experts_backward_workspace_bytes(None) == 0
    assert ops.experts_backward_workspace_bytes(ops.make_backward_desc(4, 100, 128, 4, 2)) == 0


def test_workspace_bytes(m):
    """Never smaller for more tokens; what the weight gradients add is what they need."""
    l, ops = m.lib.lib(), m.ops
    for kw in (dict(H=512, I=256, E=64, k=6), dict(H=4096, I=14336, E=8, k=2), dict(H=256, I=128, E=1, k=1)):
        for grads in (False, True):
            prev = 0
            for T in (0, 1, 2, 63, 64, 85, 86, 128, 255, 256, 257, 600, 4096):
                n = ops.experts_backward_workspace_bytes(ops.make_backward_desc(T, weight_grads=grads, **kw))
                assert n >= max(prev, 1), (kw, T)
                prev = n
    a, b = (ops.experts_backward_workspace_bytes(ops.make_backward_desc(512, 1024, 512, 8, 2, weight_grads=g)) for g in (False, True))
    assert b - a == 1024 * 2 * (2 * 1024 + 3 * 512) + 256        # the rows in bf16, and the order of the experts
    for f, kw in ((l.b200moe_router_logits_backward_workspace_bytes, (7168, 256)), (l.b200moe_router_logits_backward_workspace_bytes, (1024, 8))):
        sizes = [f(T, *kw) for T in (0, 1, 64, 65, 129, 1000, 2047, 2048, 8192)]
        assert sizes == sorted(sizes) and sizes[0] > 0
    sizes = [l.b200moe_linear_w8_backward_workspace_bytes(M, 1024, 576, 1) for M in (0, 1, 33, 128, 129, 4096)]
    assert sizes == sorted(sizes) and sizes[0] > 0
    assert l.b200moe_linear_w8_backward_workspace_bytes(4, 100, 64, 0) == 0
    assert l.b200moe_router_logits_backward_workspace_bytes(4, 100, 8) == 0


def test_python_refusals_need_no_gpu(m):
    """Tensors that are not on a GPU are refused by name, before anything else is tried."""
    ops = m.ops
    f, b, i = torch.zeros(4, 8), torch.zeros(4, 128, dtype=torch.bfloat16), torch.zeros(4, 2, dtype=torch.int32)
    e4 = torch.zeros(2, 128, 128).to(torch.float8_e4m3fn)
    s = torch.zeros(2, 1, 1)
    with pytest.raises(ValueError, match="logits"):
        ops.route_backward(torch.zeros(4, 2), f, i)
    with pytest.raises(ValueError, match="dlogits"):
        ops.router_logits_backward(f, b, torch.zeros(8, 128, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="x or wr"):
        ops.router_logits_backward(f)
    with pytest.raises(ValueError, match="y must be"):
        ops.combine_backward(b, torch.zeros(4, 2, 128, dtype=torch.bfloat16), torch.zeros(4, 2))
    with pytest.raises(ValueError, match="dimensions"):
        ops.combine_backward(b, b, torch.zeros(4, 2))
    with pytest.raises(ValueError, match="dy"):
        ops.linear_w8_backward(b, b)
    with pytest.raises(ValueError, match="x must be"):
        ops.experts_backward(b, b, e4, e4, e4, s, s, s, i, torch.zeros(4, 2))
