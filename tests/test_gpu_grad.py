"""Gradients of the layer's entry points (ops.*_backward) against the same definitions in 64 bits, elementwise, within bounds
that follow from the number formats and the number of additions (oracle/grad_oracle.py)."""
import pytest
import torch

from oracle import grad_oracle as G

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    import torch_tpu_b200
    return torch_tpu_b200.ops


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *size, scale=1.0, dtype=torch.bfloat16):
    return (torch.randn(*size, generator=g, device=DEV) * scale).to(dtype)


def fp8_weights(g, E, R, C, scale_dtype=torch.float32):
    q = (torch.randn(E, R, C, generator=g, device=DEV) * 107.0).clamp(-448, 448).to(torch.float8_e4m3fn)
    s = (0.5 + torch.rand(E, (R + 127) // 128, (C + 127) // 128, generator=g, device=DEV)) * (0.1 / 107.0)
    return q, s.to(scale_dtype)


def within(got, want, bound, what):
    got = got.double()
    if got.numel() == 0:
        assert got.shape == want.shape
        return
    assert torch.isfinite(got).all(), what
    off = (got - want).abs() - bound
    worst = off.argmax()
    assert off.max() <= 0, (what, tuple(got.shape), int(worst), float(got.flatten()[worst]), float(want.flatten()[worst]),
                            float(bound.flatten()[worst]))


def rounded(want, bound, dtype):
    """The bound of a result that is rounded to ``dtype`` once more."""
    return bound + (want.abs() + bound) * G.half_step(dtype)


def status_word():
    return torch.zeros(1, dtype=torch.int32, device=DEV)


# ---- routing ---------------------------------------------------------------------------------------------------------
ROUTE = [(1, 1, 1), (1, 8, 2), (5, 7, 3), (33, 128, 8), (130, 256, 8), (17, 300, 10), (3, 1024, 32), (64, 64, 1)]


@pytest.mark.parametrize("T,E,k", ROUTE)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
def test_route_backward(ops, T, E, k, score, renorm):
    g = gen(T * 1000 + E + k)
    logits = randn(g, T, E, scale=2.0, dtype=torch.float32)
    lb = randn(g, E, scale=0.5, dtype=torch.float32)
    bias = randn(g, E, scale=0.1, dtype=torch.float32)
    for use_bias, dt in ((False, torch.float32), (True, torch.bfloat16)):
        b = lb if use_bias else None
        ids, w = ops.route(logits, k, score, bias=bias, renorm=renorm, scale=2.5, logit_bias=b)
        dw = randn(g, T, k, dtype=dt)
        got = ops.route_backward(dw, logits, ids, score, renorm, 2.5, logit_bias=b)
        want, bound = G.route_backward(dw, logits, ids, score, renorm, 2.5, b)
        within(got, want, bound, "dlogits")


def test_route_backward_against_differences(ops):
    """The forward call, in steps of the logits: (w(l + h) - w(l - h)) / 2h, selection held by a large bias."""
    T, E, k, h = 4, 16, 3, 2.0 ** -6
    for score in ("softmax", "sigmoid"):
        for renorm in (True, False):
            g = gen(3)
            logits, dw = randn(g, T, E, dtype=torch.float32), randn(g, T, k, dtype=torch.float32)
            bias = torch.zeros(E, device=DEV)
            bias[[2, 7, 11]] = torch.tensor([300.0, 200.0, 100.0], device=DEV)
            ids, _ = ops.route(logits, k, score, bias=bias, renorm=renorm, scale=1.5)
            got = ops.route_backward(dw, logits, ids, score, renorm, 1.5)
            num = torch.zeros(T, E, dtype=torch.float64, device=DEV)
            for e in range(E):
                step = torch.zeros(T, E, device=DEV)
                step[:, e] = h
                hi = ops.route(logits + step, k, score, bias=bias, renorm=renorm, scale=1.5)
                lo = ops.route(logits - step, k, score, bias=bias, renorm=renorm, scale=1.5)
                assert torch.equal(hi[0], ids) and torch.equal(lo[0], ids)
                num[:, e] = ((hi[1].double() - lo[1].double()) * dw.double()).sum(-1) / (2 * h)
            # third derivatives of these scores are below 1: h^2 / 6 times sum |dw| * 1.5 (4 where weights are divided by
            # their sum); differences of fp32 weights carry 2^-22 / 2h
            size = dw.abs().sum(-1, keepdim=True).double() * 1.5
            within(got, num, size * (4 * h * h / 6 + 2.0 ** -22 / h), "differences")


def test_route_backward_dropped_and_repeated_slots(ops):
    g = gen(5)
    T, E, k = 6, 12, 4
    logits, dw = randn(g, T, E, dtype=torch.float32), randn(g, T, k, dtype=torch.float32)
    ids = torch.tensor([[0, 1, 2, 3], [-1, 5, 12, 7], [4, 4, 4, 4], [-1, -1, -1, -1], [11, 0, 11, 2], [9, 99, 8, -7]],
                       dtype=torch.int32, device=DEV)
    for score in ("softmax", "sigmoid"):
        for renorm in (True, False):
            got = ops.route_backward(dw, logits, ids, score, renorm, 1.0)
            want, bound = G.route_backward(dw, logits, ids, score, renorm, 1.0)
            if renorm:
                want[3], bound[3] = 0, 0     # a token without a slot has no weights, and no gradient
                want, bound = torch.nan_to_num(want), torch.nan_to_num(bound)
            within(got, want, bound, (score, renorm))


def test_route_backward_masked_logits_and_in_place(ops):
    g = gen(6)
    T, E, k = 9, 64, 6
    logits, dw = randn(g, T, E, dtype=torch.float32), randn(g, T, k, dtype=torch.float32)
    logits[:, 10:40] = -float("inf")            # experts that are switched off
    logits[0, :10] = torch.finfo(torch.float32).min
    for renorm in (True, False):
        ids, _ = ops.route(logits, k, "softmax", renorm=renorm)
        want = ops.route_backward(dw, logits, ids, "softmax", renorm)
        assert torch.isfinite(want).all() and not want[:, 10:40].any()
        buf = logits.clone()
        got = ops.route_backward(dw, buf, ids, "softmax", renorm, dlogits=buf)
        assert got.data_ptr() == buf.data_ptr() and torch.equal(got, want)


# ---- combine ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("T,k,H", [(1, 1, 8), (3, 2, 1024), (17, 8, 2056), (5, 32, 264), (2, 3, 8192), (2, 2, 16648), (300, 4, 128)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_combine_backward(ops, T, k, H, dtype):
    g = gen(T + k + H)
    dout, y = randn(g, T, H), randn(g, T, k, H)
    w = torch.rand(T, k, generator=g, device=DEV).to(dtype)
    dy, dw = ops.combine_backward(dout, y, w)
    wy, by, ww, bw = G.combine_backward(dout, y, w)
    within(dy, wy, rounded(wy, by, torch.bfloat16), "dy")
    within(dw, ww, bw, "dw")
    again = ops.combine_backward(dout, y.clone(), w)
    assert torch.equal(dy, again[0]) and torch.equal(dw, again[1])


def test_combine_backward_masked_and_in_place(ops):
    g = gen(8)
    T, k, H, E = 7, 3, 520, 5
    dout, y, w = randn(g, T, H), randn(g, T, k, H), torch.rand(T, k, generator=g, device=DEV)
    ids = torch.randint(-2, E + 2, (T, k), generator=g, device=DEV, dtype=torch.int32)
    ids[0] = -1
    on = (ids >= 0) & (ids < E)
    y[~on] = float("nan")                    # rows that nobody wrote
    w[~on] = float("inf")
    dy, dw = ops.combine_backward(dout, y, w, ids=ids, num_experts=E)
    wy, by, ww, bw = G.combine_backward(dout, y, w, ids, E)
    within(dy, wy, rounded(wy, by, torch.bfloat16), "dy")
    within(dw, ww, bw, "dw")
    assert not dy[~on].any() and not dw[~on].any()
    buf = y.clone()
    got = ops.combine_backward(dout, buf, w, ids=ids, num_experts=E, dy=buf)
    assert got[0].data_ptr() == buf.data_ptr() and torch.equal(got[0], dy) and torch.equal(got[1], dw)


# ---- router product --------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("T,H,E", [(1, 8, 1), (1, 1024, 8), (16, 1000, 8), (65, 264, 64), (130, 128, 65), (257, 2048, 128), (300, 520, 300),
                                   (63, 256, 1024), (1500, 776, 8), (4500, 264, 16), (700, 7168, 256), (64, 136, 128), (65, 136, 128)])
def test_router_logits_backward(ops, T, H, E):
    g = gen(T + H + E)
    dl, x, wr = randn(g, T, E, dtype=torch.float32), randn(g, T, H), randn(g, E, H, scale=0.1)
    st = status_word()
    dx, dwr = ops.router_logits_backward(dl, x, wr, status=st)
    wx, bx, ww, bw = G.router_backward(dl, x, wr)
    within(dx, wx, rounded(wx, bx, torch.bfloat16), "dx")
    within(dwr, ww, bw, "dwr")
    # each alone, in bf16, added to what is there
    assert torch.equal(ops.router_logits_backward(dl, None, wr)[0], dx)
    only = ops.router_logits_backward(dl, x, None, dwr=torch.empty(E, H, dtype=torch.bfloat16, device=DEV))
    assert only[0] is None
    within(only[1], ww, rounded(ww, bw, torch.bfloat16), "dwr bf16")
    base = randn(g, E, H, dtype=torch.float32)
    acc = ops.router_logits_backward(dl, x, None, dwr=base.clone(), accumulate=True)[1]
    assert torch.equal(acc, base + dwr)
    into = randn(g, T, H)
    got = ops.router_logits_backward(dl, None, wr, dx=into.clone(), add_dx=True)[0]
    want = into.double() + wx
    within(got, want, rounded(want, bx + (wx.abs() + bx) * G.half_step(torch.bfloat16), torch.bfloat16), "added to dx")
    assert int(st.item()) == 0


# ---- linear layer ----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("M,K,N", [(1, 128, 64), (1, 1024, 512), (5, 256, 192), (64, 384, 128), (65, 128, 320), (129, 640, 256),
                                   (300, 512, 1088), (2500, 128, 128), (4200, 256, 64)])
@pytest.mark.parametrize("scale_dtype", [torch.float32, torch.bfloat16])
def test_linear_w8_backward(ops, M, K, N, scale_dtype):
    g = gen(M + K + N)
    dy, x = randn(g, M, N, scale=1e-3), randn(g, M, K)
    w, s = fp8_weights(g, 1, N, K, scale_dtype)
    w, s = w[0], s[0]
    st = status_word()
    dx, dw = ops.linear_w8_backward(dy, x, w, s, status=st)
    wx, bx, ww, bw = G.linear_backward(dy, x, w, s)
    within(dx, wx, rounded(wx, bx, torch.bfloat16), "dx")
    within(dw, ww, bw, "dw")
    assert torch.equal(ops.linear_w8_backward(dy, None, w, s)[0], dx)
    assert torch.equal(ops.linear_w8_backward(dy, x)[1], dw)
    low = ops.linear_w8_backward(dy, x, dw=torch.empty(N, K, dtype=torch.bfloat16, device=DEV))[1]
    within(low, ww, rounded(ww, bw, torch.bfloat16), "dw bf16")
    base = randn(g, N, K, scale=1e-2, dtype=torch.float32)
    acc = ops.linear_w8_backward(dy, x, dw=base.clone(), accumulate=True)[1]
    within(acc, base.double() + ww, bw + (base.double().abs() + ww.abs() + bw) * 4 * G.U, "accumulated")
    assert int(st.item()) == 0


def test_linear_w8_backward_of_many_rows(ops):
    """bf16 weight gradients of more rows than one accumulator takes."""
    g = gen(12)
    M, K, N = 40000, 256, 192
    dy, x = randn(g, M, N).abs(), randn(g, M, K).abs()        # terms of one sign: the sum's error does not average out
    low = ops.linear_w8_backward(dy, x, dw=torch.empty(N, K, dtype=torch.bfloat16, device=DEV))[1]
    want = dy.double().t() @ x.double()
    within(low, want, rounded(want, G.product_bound(dy.double().t(), x.double(), 512 + M // 512), torch.bfloat16), "dw bf16")


def test_linear_w8_backward_of_small_gradients(ops):
    """Rows that are tiny throughout keep their bits: the scale's floor is for gradients."""
    g = gen(11)
    M, K, N = 40, 256, 256
    dy, x = randn(g, M, N), randn(g, M, K)
    dy[:20] *= 2.0 ** -60
    dy[3] = 0
    w, s = fp8_weights(g, 1, N, K)
    dx, dw = ops.linear_w8_backward(dy, x, w[0], s[0])
    wx, bx, ww, bw = G.linear_backward(dy, x, w[0], s[0])
    within(dx, wx, rounded(wx, bx, torch.bfloat16), "dx")
    within(dw, ww, bw, "dw")
    assert not dx[3].any() and dx[0].any()


# ---- experts ---------------------------------------------------------------------------------------------------------
def problem(T, H, I, E, k, seed=0, scale_dtype=torch.float32, per_slot=False, ids=None, w_dtype=torch.float32):
    g = gen(seed + T + H + I + E + k)
    parts = [fp8_weights(g, E, I, H, scale_dtype) for _ in range(3)]
    p = dict(x=randn(g, T, H), dout=randn(g, *((T, k, H) if per_slot else (T, H)), scale=1e-2), w=[q for q, _ in parts], s=[s for _, s in parts])
    if ids is None:
        ids = torch.stack([torch.randperm(E, generator=g, device=DEV)[:k] for _ in range(T)]) if T else torch.zeros(0, k, device=DEV)
    p["ids"] = ids.to(torch.int32).to(DEV)
    w = torch.rand(T, k, generator=g, device=DEV) + 0.1
    p["topk_w"] = None if per_slot else (w / w.sum(-1, keepdim=True)).to(w_dtype)
    return p


def run_experts(ops, p, grad_dtype=None, **kw):
    grads = [torch.full(w.shape, float("nan"), dtype=grad_dtype, device=DEV) for w in p["w"]] if grad_dtype else None
    st = status_word()
    dx, dw = ops.experts_backward(p["dout"], p["x"], *p["w"], *p["s"], p["ids"], p["topk_w"], weight_grads=grads, status=st, **kw)
    return dx, dw, grads, int(st.item())


def check_experts(ops, p, grad_dtype, bad=False, add=None):
    dx, dw, grads, st = run_experts(ops, p, grad_dtype, add=add)
    assert st == (1 if bad else 0)
    want = G.experts_backward(p["dout"], p["x"], *p["w"], *p["s"], p["ids"], p["topk_w"], add)
    within(dx, want["dx"][0], rounded(*want["dx"], torch.bfloat16), "dx")
    if p["topk_w"] is not None:
        within(dw, *want["dw"], "dw")
    else:
        assert dw is None
    if grads:
        for n, t in zip(("dwg", "dwu", "dwd"), grads):
            v, b = want[n]
            within(t, v, rounded(v, b, torch.bfloat16) if grad_dtype == torch.bfloat16 else b, n)
    return dx, dw, grads


@pytest.mark.parametrize("T,H,I,E,k", [(1, 128, 128, 1, 1), (1, 256, 384, 8, 2), (16, 1024, 512, 8, 2), (37, 640, 128, 5, 3), (130, 128, 256, 4, 2),
                                       (300, 384, 256, 6, 3), (700, 256, 128, 64, 4), (64, 256, 128, 200, 8),
                                       (1, 512, 2048, 4, 2), (30, 256, 1024, 8, 2), (33, 384, 1024, 3, 2)])
@pytest.mark.parametrize("grad_dtype", [None, torch.bfloat16, torch.float32])
def test_experts_backward(ops, T, H, I, E, k, grad_dtype):
    check_experts(ops, problem(T, H, I, E, k), grad_dtype)


@pytest.mark.parametrize("T,k", [(5, 2), (300, 3)])
def test_experts_backward_per_slot_bf16_scales_and_weights(ops, T, k):
    check_experts(ops, problem(T, 256, 256, 6, k, per_slot=True, scale_dtype=torch.bfloat16), torch.float32)
    check_experts(ops, problem(T, 256, 256, 6, k, w_dtype=torch.bfloat16, scale_dtype=torch.bfloat16), torch.bfloat16)


@pytest.mark.parametrize("H,I,per_slot,scale_dtype", [(1024, 1024, False, torch.float32), (1152, 1152, False, torch.bfloat16),
                                                      (1024, 1152, True, torch.float32), (2176, 896, False, torch.float32)])
def test_experts_backward_many_rows(ops, H, I, per_slot, scale_dtype):
    check_experts(ops, problem(1800, H, I, 4, 2, per_slot=per_slot, scale_dtype=scale_dtype), torch.bfloat16)


@pytest.mark.parametrize("counts", [(2560, 0, 1, 100), (256, 257, 2047, 256), (0, 0, 2816, 0), (1, 128, 129, 2558)])
def test_experts_backward_many_rows_uneven(ops, counts):
    """Experts that end before, at and behind the border of a second tile; dropped pairs behind them."""
    T = 2816
    ids = torch.full((T,), -1)
    flat = torch.repeat_interleave(torch.arange(4), torch.tensor(counts))
    ids[:len(flat)] = flat
    ids = ids[torch.randperm(T, generator=torch.Generator().manual_seed(1))].view(T, 1)
    p = problem(T, 1280, 1280, 4, 1, ids=ids)
    dropped = len(flat) < T
    first = check_experts(ops, p, torch.float32, bad=dropped)
    again = run_experts(ops, p, torch.float32)
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    assert all(torch.equal(a, b) for a, b in zip(first[2], again[2]))


def test_experts_backward_uneven_loads(ops):
    """All rows on one expert, experts without rows, a tail of one row behind whole tiles."""
    T, k, E = 257, 2, 9
    ids = torch.stack([torch.full((T,), 4), torch.where(torch.arange(T) < 129, 7, 1)], 1)
    p = problem(T, 256, 128, E, k, ids=ids)
    _, _, grads = check_experts(ops, p, torch.float32)
    for t in grads:
        for e in (0, 2, 3, 5, 6, 8):
            assert not t[e].any()
    check_experts(ops, problem(70, 128, 128, 3, 2, ids=torch.full((70, 2), 2)), torch.bfloat16)  # the same expert twice


@pytest.mark.parametrize("T,I", [(20, 1024), (20, 128), (400, 128)])
def test_experts_backward_dropped_pairs(ops, T, I):
    g = torch.Generator().manual_seed(T)
    ids = torch.randint(-1, 8, (T, 3), generator=g)          # -1, 6 and 7 are nobody's
    ids[3] = -1
    p = problem(T, 256, I, 6, 3, ids=ids)
    dx, dw, grads, st = run_experts(ops, p, torch.float32)
    assert st == 1
    on = (p["ids"] >= 0) & (p["ids"] < 6)
    assert not dw[~on].any() and not dx[3].any()
    check_experts(ops, p, torch.float32, bad=True)
    for ids in (torch.full((T, 3), -1), torch.full((T, 3), 1 << 30)):  # no pair at all
        p["ids"] = ids.to(torch.int32).to(DEV)
        dx, dw, grads, st = run_experts(ops, p, torch.bfloat16)
        assert st == 1 and not dx.any() and not dw.any() and not any(t.any() for t in grads)


@pytest.mark.parametrize("T", [9, 300])
def test_experts_backward_add_and_accumulate(ops, T):
    p = problem(T, 384, 128, 5, 2)
    g = gen(77)
    add = randn(g, T, 384, scale=1e-2)
    dx, dw, grads = check_experts(ops, p, torch.float32, add=add)
    buf = add.clone()                                         # add may be dx's own buffer
    again = ops.experts_backward(p["dout"], p["x"], *p["w"], *p["s"], p["ids"], p["topk_w"], add=buf, dx=buf)[0]
    want = G.experts_backward(p["dout"], p["x"], *p["w"], *p["s"], p["ids"], p["topk_w"], add)["dx"]
    within(again, want[0], rounded(*want, torch.bfloat16), "dx in place")
    base = [randn(g, *t.shape, scale=1e-2, dtype=torch.float32) for t in grads]
    acc = [t.clone() for t in base]
    ops.experts_backward(p["dout"], p["x"], *p["w"], *p["s"], p["ids"], p["topk_w"], weight_grads=acc, accumulate=True)
    for a, b, t in zip(acc, base, grads):
        assert torch.equal(a, b + t)                          # one fp32 addition to each element


@pytest.mark.parametrize("T,I", [(1, 1024), (20, 1024), (100, 512), (500, 256)])
def test_experts_backward_repeats_and_leaves_nothing_behind(ops, T, I):
    """Equal calls give equal bits; a workspace full of NaN changes nothing."""
    import torch_tpu_b200
    p = problem(T, 256, I, 16, 2)
    d = ops.make_backward_desc(T, 256, I, 16, 2, weight_grads=True, grad_dtype=torch.bfloat16)
    ws = torch.full((ops.experts_backward_workspace_bytes(d) + 256,), 255, dtype=torch.uint8, device=DEV)
    first = run_experts(ops, p, torch.bfloat16, workspace=ws)
    for _ in range(3):
        got = run_experts(ops, p, torch.bfloat16, workspace=ws)
        assert torch.equal(got[0], first[0]) and torch.equal(got[1], first[1])
        assert all(torch.equal(a, b) for a, b in zip(got[2], first[2]))
    assert torch_tpu_b200.lib.lib() is not None


def test_empty_batches(ops):
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype, device=DEV)  # noqa: E731
    assert ops.route_backward(z(0, 2, dtype=torch.float32), z(0, 8, dtype=torch.float32), z(0, 2, dtype=torch.int32)).shape == (0, 8)
    dx, dwr = ops.router_logits_backward(z(0, 8, dtype=torch.float32), z(0, 128), z(8, 128), dwr=torch.full((8, 128), 7.0, device=DEV))
    assert dx.shape == (0, 128) and not dwr.any()
    dy, dw = ops.combine_backward(z(0, 128), z(0, 2, 128), z(0, 2, dtype=torch.float32))
    assert dy.shape == (0, 2, 128) and dw.shape == (0, 2)
    w, s = fp8_weights(gen(1), 1, 128, 256)
    dx, dw = ops.linear_w8_backward(z(0, 128), z(0, 256), w[0], s[0], dw=torch.full((128, 256), 7.0, device=DEV))
    assert dx.shape == (0, 256) and not dw.any()
    p = problem(0, 256, 128, 4, 2)
    dx, dw, grads, st = run_experts(ops, p, torch.float32)
    assert dx.shape == (0, 256) and dw.shape == (0, 2) and not any(t.any() for t in grads) and st == 0
    keep = torch.full((4, 128, 256), 3.0, device=DEV)
    ops.experts_backward(p["dout"], p["x"], *p["w"], *p["s"], p["ids"], p["topk_w"], weight_grads=[keep, keep.clone(), keep.clone()],
                         accumulate=True)
    assert bool((keep == 3.0).all())


# ---- refusals with tensors on a GPU -----------------------------------------------------------------------------------
def test_refusals(ops):
    p = problem(8, 256, 128, 4, 2)
    call = lambda q, **kw: ops.experts_backward(q["dout"], q["x"], *q["w"], *q["s"], q["ids"], q["topk_w"], **kw)  # noqa: E731
    g32 = [torch.empty(w.shape, device=DEV) for w in p["w"]]
    for match, q, kw in (
        ("must have shape", {**p, "x": p["x"][:4]}, {}),
        ("ids", {**p, "ids": p["ids"].long()}, {}),
        ("contiguous", {**p, "x": p["x"].t().contiguous().t()}, {}),
        ("wu", {**p, "w": [p["w"][0], p["w"][1][:2].contiguous(), p["w"][2]]}, {}),
        ("wg", {**p, "w": [w.to(torch.bfloat16) for w in p["w"]]}, {}),              # bf16-weight experts
        ("su", {**p, "s": [p["s"][0], p["s"][1].bfloat16(), p["s"][2]]}, {}),
        ("topk_w", {**p, "topk_w": None}, {}),
        ("topk_w", {**p, "topk_w": p["topk_w"].double()}, {}),
        ("topk_w and dw", {**p, "dout": p["dout"][:, None].repeat(1, 2, 1)}, {}),
        ("weight_grads", p, dict(weight_grads=g32[:2])),
        ("one dtype", p, dict(weight_grads=[g32[0], g32[1].bfloat16(), g32[2]])),
        ("accumulate", p, dict(weight_grads=[t.bfloat16() for t in g32], accumulate=True)),
        ("dwd", p, dict(weight_grads=[g32[0], g32[1], None])),
        ("add", p, dict(add=torch.zeros(8, 256, device=DEV))),
        ("dx", p, dict(dx=torch.zeros(8, 128, dtype=torch.bfloat16, device=DEV))),
        ("workspace", p, dict(workspace=torch.zeros(1 << 20, dtype=torch.uint8))),
        ("status", p, dict(status=torch.zeros(1, dtype=torch.int32))),
    ):
        with pytest.raises(ValueError, match=match):
            call(q, **kw)
    with pytest.raises(RuntimeError, match="workspace"):
        call(p, workspace=torch.zeros(4096, dtype=torch.uint8, device=DEV))
    odd = torch.zeros(8 * 256 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(8, 256)      # not 16-byte aligned
    with pytest.raises(RuntimeError, match="aligned"):
        call({**p, "x": odd})
    g = gen(1)
    with pytest.raises(ValueError, match="unsupported sizes"):
        ops.linear_w8_backward(randn(g, 4, 128), randn(g, 4, 100))
    with pytest.raises(ValueError, match="unsupported sizes"):
        ops.router_logits_backward(randn(g, 4, 8, dtype=torch.float32), randn(g, 4, 100))
    with pytest.raises(ValueError, match="add_dx"):
        ops.router_logits_backward(randn(g, 4, 8, dtype=torch.float32), None, randn(g, 8, 128), add_dx=True)
    with pytest.raises(ValueError, match="scale"):
        ops.linear_w8_backward(randn(g, 4, 128), None, fp8_weights(g, 1, 128, 128)[0][0])
    with pytest.raises(RuntimeError, match="unsupported size"):
        ops.combine_backward(randn(g, 4, 12), randn(g, 4, 2, 12), torch.ones(4, 2, device=DEV))
    with pytest.raises(RuntimeError, match="unsupported size"):
        ops.route_backward(torch.ones(2, 33, device=DEV), torch.zeros(2, 64, device=DEV), torch.zeros(2, 33, dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError, match="score_func"):
        ops.route_backward(torch.ones(2, 2, device=DEV), torch.zeros(2, 64, device=DEV), torch.zeros(2, 2, dtype=torch.int32, device=DEV), "tanh")


def test_non_finite_rows_stay_their_own(ops):
    """A token whose row is not finite spoils what depends on it, and nothing else."""
    T, E = 200, 6
    p = problem(T, 256, 128, E, 2)
    clean = run_experts(ops, p, torch.float32)
    bad = 77
    p["dout"][bad, 5] = float("nan")
    p["x"][bad, 9] = float("inf")
    dx, dw, grads, st = run_experts(ops, p, torch.float32)
    keep = torch.arange(T, device=DEV) != bad
    assert torch.isfinite(dx[keep]).all() and torch.isfinite(dw[keep]).all()
    assert torch.equal(dw[keep], clean[1][keep])
    assert not torch.isfinite(dx[bad]).all() and not torch.isfinite(dw[bad]).any()
    mine = p["ids"][bad].long()
    others = [e for e in range(E) if e not in mine.tolist()]
    for t, c in zip(grads, clean[2]):
        assert torch.equal(t[others], c[others]) and not torch.isfinite(t[mine]).all()
