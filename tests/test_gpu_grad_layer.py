"""FusedMoE.backward: the gradients of a whole layer (routing, router, experts, shared expert) as a training loop calls them, and
the same calls on other streams, beside each other and replayed from a graph."""
import pytest
import torch

from oracle import grad_oracle as G
from tests.test_gpu_grad import DEV, fp8_weights, gen, randn, rounded, within

pytestmark = pytest.mark.gpu


def make_layer(T, H, I, E, k, shared=0, score="softmax", groups=1, topk_groups=1, renorm=True, scale=1.0, seed=0, max_tokens=None,
               scale_dtype=torch.float32, with_bias=False):
    from torch_tpu_b200.layer import FusedMoE, MoEConfig
    g = gen(seed + T + E)
    cfg = MoEConfig(H, I, E, k, score, groups, topk_groups, renorm, scale, shared)
    parts = [fp8_weights(g, E, I, H, scale_dtype) for _ in range(3)]
    sh = None
    if shared:
        sp = [fp8_weights(g, 1, shared, H, scale_dtype) for _ in range(3)]
        sh = (*[q for q, _ in sp], *[s for _, s in sp])
    wr = randn(g, E, H, scale=0.05)
    bias = randn(g, E, scale=0.01, dtype=torch.float32) if with_bias else None
    layer = FusedMoE(cfg, wr, *[q for q, _ in parts], *[s for _, s in parts], bias=bias, shared=sh,
                     logit_bias=randn(g, E, scale=0.1, dtype=torch.float32) if with_bias else None, max_tokens=max_tokens or T)
    return layer, randn(g, T, H), randn(g, T, H, scale=1e-2), g


def grads_of(layer, dtype=torch.float32, fill=float("nan")):
    full = lambda w: torch.full(w.shape, fill, dtype=dtype, device=DEV)  # noqa: E731
    return dict(router_grad=full(layer.router_w), weight_grads=[full(w) for w in layer.w[:3]],
                shared_grads=[full(w) for w in layer.shared[:3]] if layer.shared else None)


CONFIGS = {
    "softmax": dict(T=40, H=256, I=256, E=8, k=2, with_bias=True),
    "dense softmax": dict(T=300, H=384, I=128, E=16, k=3, renorm=False, scale=1.5),
    "groups and shared": dict(T=33, H=256, I=128, E=32, k=4, shared=384, score="sigmoid", groups=8, topk_groups=4, scale=2.5,
                              with_bias=True, scale_dtype=torch.bfloat16),
    "one token": dict(T=1, H=128, I=128, E=4, k=2, shared=128),
    "larger": dict(T=700, H=512, I=256, E=24, k=4, shared=256, score="sigmoid", scale=2.0),
}


@pytest.mark.parametrize("name", CONFIGS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layer_backward(name, dtype):
    c = CONFIGS[name]
    layer, x, dout, _ = make_layer(**c)
    out = layer.forward(x).clone()
    got = layer.backward(x, dout, **grads_of(layer, dtype))
    assert int(layer.status.item()) == 0 and torch.equal(out, layer.forward(x))
    ids, w, logits = layer.ids[:c["T"]], layer.topk_w[:c["T"]], layer.logits[:c["T"]]
    e = G.experts_backward(dout, x, *layer.w, ids, w)
    dl, bl = G.route_backward(e["dw"][0], logits, ids, layer.cfg.score_func, layer.cfg.renorm, layer.cfg.routed_scale, layer.logit_bias,
                              dw_bound=e["dw"][1])
    within(got.dlogits, dl, bl, "dlogits")
    rx, bx, rw, bw = G.router_backward(dl, x, layer.router_w)
    bx, bw = bx + bl @ layer.router_w.double().abs(), bw + bl.t() @ x.double().abs()
    low = (lambda v, b: rounded(v, b, torch.bfloat16)) if dtype == torch.bfloat16 else (lambda v, b: b)
    within(got.router, rw, low(rw, bw), "router")
    for n, t in zip(("dwg", "dwu", "dwd"), got.experts):
        within(t, e[n][0], low(*e[n]), n)
    dx, bound, half = e["dx"][0], e["dx"][1], G.half_step(torch.bfloat16)
    if layer.shared:
        one = torch.zeros(c["T"], 1, dtype=torch.int32, device=DEV)
        s = G.experts_backward(dout, x, *layer.shared, one, torch.ones(c["T"], 1, device=DEV))
        for n, t in zip(("dwg", "dwu", "dwd"), got.shared):
            within(t, s[n][0], low(*s[n]), "shared " + n)
        bound = bound + s["dx"][1] + (s["dx"][0].abs() + s["dx"][1]) * half     # the shared expert's dx is rounded before the sum
        dx = dx + s["dx"][0]
    bound = bound + (dx.abs() + bound) * half + bx + (rx.abs() + bx) * half     # so is the experts', and the router's
    within(got.dx, dx + rx, rounded(dx + rx, bound, torch.bfloat16), "dx")


def test_layer_backward_accumulates_and_leaves_out():
    layer, x, dout, g = make_layer(**CONFIGS["larger"])
    first = layer.backward(x, dout, **grads_of(layer))
    dx = first.dx.clone()
    acc = grads_of(layer, fill=0.25)
    layer.backward(x, dout, accumulate=True, **acc)
    pairs = [(acc["router_grad"], first.router), *zip(acc["weight_grads"], first.experts), *zip(acc["shared_grads"], first.shared)]
    for a, b in pairs:
        assert torch.equal(a, b + 0.25)
    mine = torch.empty_like(x)
    only = layer.backward(x, dout, dx=mine)
    assert only.dx.data_ptr() == mine.data_ptr() and torch.equal(mine, dx)
    assert only.router is None and only.experts is None and only.shared is None


def test_layer_backward_refuses():
    from torch_tpu_b200 import lib as L
    layer, x, dout, _ = make_layer(T=8, H=128, I=128, E=4, k=2)
    with pytest.raises(ValueError, match="max_tokens"):
        layer.backward(x.repeat(2, 1), dout.repeat(2, 1))
    with pytest.raises(ValueError, match="shared"):
        layer.backward(x, dout, shared_grads=grads_of(layer)["weight_grads"])
    with pytest.raises(ValueError, match="accumulate"):
        layer.backward(x, dout, weight_grads=grads_of(layer, torch.bfloat16)["weight_grads"], accumulate=True)
    with pytest.raises(ValueError, match="dout"):
        layer.backward(x, dout[:4])
    layer.act_mode = L.ACT_W8A16
    with pytest.raises(ValueError, match="W8A8"):
        layer.backward(x, dout)


def test_layer_backward_refuses_dx_over_its_inputs():
    layer, x, dout, _ = make_layer(T=8, H=128, I=128, E=4, k=2, shared=128)
    with pytest.raises(ValueError, match="shares memory with x"):
        layer.backward(x, dout, dx=x)
    with pytest.raises(ValueError, match="shares memory with dout"):
        layer.backward(x, dout, dx=dout)
    got = layer.backward(x, dout)
    with pytest.raises(ValueError, match="shares memory with dout"):     # the returned view is the next call's dx
        layer.backward(x, got.dx)
    layer.backward(x, got.dx.clone())


@pytest.mark.parametrize("bad", ["router type", "router shape", "shared type", "shared count"])
def test_refused_call_adds_nothing(bad):
    """accumulate with one unfit buffer: the others keep what they hold."""
    layer, x, dout, _ = make_layer(T=8, H=128, I=128, E=4, k=2, shared=128)
    kw = grads_of(layer, fill=1.0)
    if bad == "router type":
        kw["router_grad"] = kw["router_grad"].bfloat16()
    elif bad == "router shape":
        kw["router_grad"] = kw["router_grad"][:3]
    elif bad == "shared type":
        kw["shared_grads"][2] = kw["shared_grads"][2].bfloat16()
    else:
        kw["shared_grads"] = kw["shared_grads"][:2]
    with pytest.raises(ValueError):
        layer.backward(x, dout, accumulate=True, **kw)
    torch.cuda.synchronize()
    assert all(bool((t == 1).all()) for t in (kw["router_grad"], *kw["weight_grads"], *kw["shared_grads"]))


def test_first_call_inside_a_capture_is_refused():
    layer, x, dout, _ = make_layer(T=8, H=128, I=128, E=4, k=2, shared=128)
    warm, _, _, _ = make_layer(T=8, H=128, I=128, E=4, k=2, shared=128)
    want = warm.backward(x, dout)                                        # (kernel attributes are set; `layer` has no buffers yet)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x.add_(0)
        with pytest.raises(RuntimeError, match="before the capture"):
            layer.backward(x, dout)
    assert not layer._bwd
    got = layer.backward(x, dout)                                        # same weights: the same generator
    assert torch.equal(got.dx, want.dx) and torch.equal(got.dlogits, want.dlogits)


def test_layer_backward_smaller_batches_and_empty():
    """One layer, one workspace, batches of any size up to max_tokens, in any order."""
    layer, x, dout, _ = make_layer(T=600, H=256, I=256, E=8, k=2, shared=128)
    for T in (600, 1, 37, 0, 256, 600):
        kw = grads_of(layer)
        got = layer.backward(x[:T], dout[:T], **kw)
        assert got.dx.shape == (T, 256)
        if T == 0:
            assert not got.router.any() and not any(t.any() for t in (*got.experts, *got.shared))
            continue
        e = G.experts_backward(dout[:T], x[:T], *layer.w, layer.ids[:T], layer.topk_w[:T])
        for n, t in zip(("dwg", "dwu", "dwd"), got.experts):
            within(t, *e[n], n)


def test_layer_backward_replayed_from_a_graph():
    layer, x, dout, g = make_layer(T=300, H=256, I=128, E=8, k=2, shared=128, score="sigmoid")
    kw = grads_of(layer)
    sx, sd = x.clone(), dout.clone()
    layer.backward(sx, sd, **kw)           # first call: allocations and kernel attributes
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = layer.backward(sx, sd, **kw)
    for seed in (1, 2):
        h = gen(seed)
        x2, d2 = randn(h, 300, 256), randn(h, 300, 256, scale=1e-2)
        want = layer.backward(x2, d2, **grads_of(layer))
        keep = [t.clone() for t in (want.dx, want.dlogits, want.router, *want.experts, *want.shared)]
        sx.copy_(x2), sd.copy_(d2)
        for t in (kw["router_grad"], *kw["weight_grads"], *kw["shared_grads"]):
            t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((res.dx, res.dlogits, res.router, *res.experts, *res.shared), keep):
            assert torch.equal(a, b)
    assert int(layer.status.item()) == 0


def test_graph_outlives_a_larger_workspace():
    """A graph captured without weight gradients is replayed after a call that needed a larger workspace."""
    layer, x, dout, _ = make_layer(T=260, H=256, I=256, E=8, k=2)
    layer.backward(x, dout)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = layer.backward(x, dout)
    graph.replay()
    want = res.dx.clone()
    small = layer._bwd["workspace"]
    layer.backward(x, dout, **grads_of(layer))
    assert layer._bwd["workspace"].numel() > small.numel()
    del small
    torch.cuda.empty_cache()
    fresh = [torch.full((1 << 20,), 255, dtype=torch.uint8, device=DEV) for _ in range(64)]   # takes what was given back
    res.dx.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(res.dx, want) and all(bool((t == 255).all()) for t in fresh)


def test_small_batch_replayed_from_a_graph():
    """dx of few pairs: a K range that is split, its partial sums cleared and added inside the graph."""
    layer, x, dout, _ = make_layer(T=12, H=512, I=1024, E=4, k=2)
    sx, sd = x.clone(), dout.clone()
    layer.backward(sx, sd)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = layer.backward(sx, sd)
    for seed in (1, 2, 3):
        h = gen(seed)
        sx.copy_(randn(h, 12, 512)), sd.copy_(randn(h, 12, 512, scale=1e-2))
        graph.replay()
        torch.cuda.synchronize()
        e = G.experts_backward(sd, sx, *layer.w, layer.ids[:12], layer.topk_w[:12])
        dl, bl = G.route_backward(e["dw"][0], layer.logits[:12], layer.ids[:12], "softmax", True, 1.0, dw_bound=e["dw"][1])
        within(res.dlogits, dl, bl, "dlogits")
        rx, bx, _, _ = G.router_backward(dl, sx, layer.router_w)
        half = G.half_step(torch.bfloat16)
        bound = e["dx"][1] + (e["dx"][0].abs() + e["dx"][1]) * half + bx + bl @ layer.router_w.double().abs() + (rx.abs() + bx) * half
        within(res.dx, e["dx"][0] + rx, rounded(e["dx"][0] + rx, bound, torch.bfloat16), "dx")


def test_two_calls_at_once_on_two_streams():
    """Calls on different streams with workspaces of their own."""
    import torch_tpu_b200
    ops = torch_tpu_b200.ops
    a = make_layer(T=500, H=256, I=256, E=8, k=2, seed=1)
    b = make_layer(T=400, H=256, I=128, E=6, k=3, seed=2)
    want = [[t.clone() for t in (r.dx, r.dlogits, r.router, *r.experts)] for r in (l.backward(x, d, **{**grads_of(l)}) for l, x, d, _ in (a, b))]
    g = gen(9)
    dy, xx = randn(g, 777, 512), randn(g, 777, 256)
    w, s = fp8_weights(g, 1, 512, 256)
    lin = [t.clone() for t in ops.linear_w8_backward(dy, xx, w[0], s[0])]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(4):
        got = []
        for st, (l, x, d, _) in zip(streams, (a, b)):
            with torch.cuda.stream(st):
                got.append(l.backward(x, d, **grads_of(l)))
        with torch.cuda.stream(streams[2]):
            lg = ops.linear_w8_backward(dy, xx, w[0], s[0])
        torch.cuda.synchronize()
        for r, k in zip(got, want):
            for t, u in zip((r.dx, r.dlogits, r.router, *r.experts), k):
                assert torch.equal(t, u)
        assert torch.equal(lg[0], lin[0]) and torch.equal(lg[1], lin[1])
