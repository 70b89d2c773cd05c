"""Gated feed-forward block: CPU path against the formula and differences, GPU kernels
(csrc/gated.hip) against 64-bit products with derived elementwise bounds."""
import math

import pytest
import torch

from mxtrain import ops

# bf16 half step; what fp32 products and activations leave, of the sum of magnitudes: a chain of K
# additions errs below K 2^-24, and v_exp / v_rcp below 2^-21, for every K tested
U, F32 = 2.0 ** -8, 2.0 ** -11


def _act(name, a):
    if name == "silu":
        s = torch.sigmoid(a)
        return a * s, s * (1 + a * (1 - s))
    z = math.sqrt(2 / math.pi) * (a + 0.044715 * a ** 3)
    s = torch.sigmoid(2 * z)
    return a * s, s + a * s * (1 - s) * 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * a * a)


def _oracle(act, x, w1, b1, w2, b2, dy=None):
    """{name: (value, bound)} in 64 bits.

    |pre err| <= F32 (|x||W1| + |b1|) =: ep (kept in fp32 for h; + U |pre| where backward uses it).
    h = act(a) b: slopes of act are below 1.13 and |act(a)| <= |a|, so
      |h err| <= 1.13 ep_a |b| + |act(a)| ep_b + U |h|.
    y: + one product of the erring h, one rounding.  Backward differentiates at the rounded pre:
      slopes of act' are below 1 (0.5 silu, 0.8 gelu), so with r = ep + U |pre|
      |da err| <= eh' |b act'| + |dh| (|act'| r_b + |b| r_a) + U |da|,  eh' = F32 |dy||W2|
      |db err| <= eh' |act| + |dh| 1.13 r_a + U |db|."""
    X, W1, W2 = x.double(), w1.double(), w2.double()
    f = W1.shape[0] // 2
    pre, mag = X @ W1.t(), X.abs() @ W1.abs().t()
    if b1 is not None:
        pre, mag = pre + b1.double(), mag + b1.double().abs()
    a, b = pre[:, :f], pre[:, f:]
    ya, da = _act(act, a)
    ep = F32 * mag
    h = ya * b
    eh = 1.13 * ep[:, :f] * b.abs() + ya.abs() * ep[:, f:] + ep[:, :f] * ep[:, f:] + (U + F32) * h.abs()
    y = h @ W2.t()
    ey = (eh + F32 * h.abs()) @ W2.abs().t()
    if b2 is not None:
        y = y + b2.double()
        ey = ey + F32 * b2.double().abs()
    res = {"y": (y, ey + U * (y.abs() + ey))}
    if dy is None:
        return res
    D = dy.double()
    dh, edh = D @ W2, F32 * (D.abs() @ W2.abs())
    r = ep + U * (pre.abs() + ep)
    ra, rb = r[:, :f], r[:, f:]
    g = dh * b * da
    eg = edh * (b * da).abs() + (dh.abs() + edh) * (1.13 * rb + (b.abs() + rb) * ra) + (U + F32) * g.abs()
    u = dh * ya
    eu = edh * ya.abs() + (dh.abs() + edh) * 1.13 * ra + (U + F32) * u.abs()
    dp, edp = torch.cat([g, u], 1), torch.cat([eg, eu], 1)

    def prod(p, ep_, q, eq=None):
        val = p @ q
        err = ep_ @ q.abs() + F32 * (p.abs() @ q.abs())
        if eq is not None:
            err = err + p.abs() @ eq
        return val, err + U * (val.abs() + err)
    res["dx"] = prod(dp, edp, W1)
    res["dw1"] = prod(dp.t(), edp.t(), X)
    res["dw2"] = prod(D.t(), torch.zeros_like(D.t()), h, eh)
    one = torch.ones(1, X.shape[0], dtype=torch.float64, device=x.device)
    if b1 is not None:
        v, e = prod(one, torch.zeros_like(one), dp, edp)
        res["db1"] = (v[0], e[0])
    if b2 is not None:
        v, e = prod(one, torch.zeros_like(one), D)
        res["db2"] = (v[0], e[0])
    return res


def _within(got, want, name):
    val, bound = want
    err = (got.double() - val).abs()
    bad = ~(err <= bound + 1e-30)
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} outside, worst {float((err / (bound + 1e-30)).max()):.2f} bounds"


def _make(T, H, F, Ho, bias, seed=0, dtype=torch.bfloat16, device="cpu"):
    gen = torch.Generator().manual_seed(seed)

    def r(*s, std=1.0):
        return (torch.randn(*s, generator=gen, dtype=torch.float64) * std).to(dtype).to(device)
    return (r(T, H), r(2 * F, H, std=H ** -0.5), r(2 * F, std=0.2) if bias else None, r(Ho, F, std=F ** -0.5),
            r(Ho, std=0.2) if bias else None, r(T, Ho))


# ------------------------------------------------------------------ CPU
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("bias", [True, False])
def test_cpu_formula_and_differences(act, bias):
    x, w1, b1, w2, b2, dy = _make(5, 3, 4, 2, bias, dtype=torch.float64)
    y, pre, h = ops.gated_mlp_fwd(x, w1, b1, w2, b2, act)
    want = _oracle(act, x, w1, b1, w2, b2, dy)
    got = dict(zip(("dx", "dw1", "db1", "dw2", "db2"), ops.gated_mlp_bwd(dy, x, pre, h, w1, b1, w2, b2, act)), y=y)
    for name, (val, _) in want.items():
        torch.testing.assert_close(got[name], val, rtol=1e-12, atol=1e-12)
    leaves = [t.requires_grad_(True) for t in (x, w1, b1, w2, b2) if t is not None]
    it = lambda ts: (ts[0], ts[1], ts[2] if bias else None, ts[3 if bias else 2], ts[4] if bias else None)
    assert torch.autograd.gradcheck(lambda *ts: ops.gated_mlp(*it(ts), act), leaves)


def test_cpu_accumulate_shapes_and_no_tokens():
    x, w1, b1, w2, b2, dy = _make(6, 3, 4, 2, True, dtype=torch.float64)
    y = ops.gated_mlp(x.view(2, 3, 3), w1, b1, w2, b2)
    assert y.shape == (2, 3, 2)
    _, pre, h = ops.gated_mlp_fwd(x, w1, b1, w2, b2)
    ref = ops.gated_mlp_bwd(dy, x, pre, h, w1, b1, w2, b2)
    bufs = [torch.ones_like(t) for t in ref[1:]]
    ops.gated_mlp_bwd(dy, x, pre, h, w1, b1, w2, b2, dw1=bufs[0], db1=bufs[1], dw2=bufs[2], db2=bufs[3], accumulate=True)
    for a, b in zip(bufs, ref[1:]):
        torch.testing.assert_close(a, b + 1)
    y, pre, h = ops.gated_mlp_fwd(x[:0], w1, b1, w2, b2)
    dx, *grads = ops.gated_mlp_bwd(dy[:0], x[:0], pre, h, w1, b1, w2, b2)
    assert y.shape == (0, 2) and dx.shape == (0, 3) and all((g == 0).all() for g in grads)


@pytest.mark.parametrize("case", ["act", "x3d", "w1", "w2", "b1", "dtype", "saved", "accumulate", "bias"])
def test_cpu_refusals(case):
    x, w1, b1, w2, b2, dy = _make(5, 3, 4, 2, True, dtype=torch.float32)
    y, pre, h = ops.gated_mlp_fwd(x, w1, b1, w2, b2)
    calls = {
        "act": (lambda: ops.gated_mlp_fwd(x, w1, b1, w2, b2, "relu"), ValueError),
        "x3d": (lambda: ops.gated_mlp_fwd(x[None], w1, b1, w2, b2), ValueError),
        "w1": (lambda: ops.gated_mlp_fwd(x, w1[:6], b1, w2, b2), ValueError),
        "w2": (lambda: ops.gated_mlp_fwd(x, w1, b1, w2[:, :3], b2), ValueError),
        "b1": (lambda: ops.gated_mlp_fwd(x, w1, b1[:4], w2, b2), ValueError),
        "dtype": (lambda: ops.gated_mlp_fwd(x, w1.double(), b1, w2, b2), TypeError),
        "saved": (lambda: ops.gated_mlp_bwd(dy, x, None, h, w1, b1, w2, b2), ValueError),
        "accumulate": (lambda: ops.gated_mlp_bwd(dy, x, pre, h, w1, b1, w2, b2, accumulate=True), ValueError),
        "bias": (lambda: ops.gated_mlp_bwd(dy, x, pre, h, w1, None, w2, b2, db1=b1), ValueError),
    }
    call, err = calls[case]
    with pytest.raises(err):
        call()


# ------------------------------------------------------------------ GPU
gpu = pytest.mark.gpu
DEV = "cuda"


@gpu
@pytest.mark.parametrize("act,bias", [("silu", True), ("gelu", False)])
@pytest.mark.parametrize("T,H,F,Ho", [
    (1, 64, 64, 64), (1, 1024, 344, 1024), (2, 72, 136, 40), (7, 8, 8, 8), (16, 256, 512, 256), (17, 264, 200, 264),
    (33, 128, 392, 128), (64, 512, 1376, 512), (65, 320, 128, 72), (127, 1000, 264, 1000), (128, 128, 128, 128),
    (129, 136, 72, 136), (300, 512, 1360, 512), (1003, 768, 2048, 768), (513, 2048, 640, 256)])
def test_gpu_forward_backward(T, H, F, Ho, act, bias):
    x, w1, b1, w2, b2, dy = _make(T, H, F, Ho, bias, seed=T + H, device=DEV)
    y, pre, h = ops.gated_mlp_fwd(x, w1, b1, w2, b2, act)
    got = dict(zip(("dx", "dw1", "db1", "dw2", "db2"), ops.gated_mlp_bwd(dy, x, pre, h, w1, b1, w2, b2, act)), y=y)
    for name, want in _oracle(act, x, w1, b1, w2, b2, dy).items():
        _within(got[name], want, name)
    only = ops.gated_mlp_fwd(x, w1, b1, w2, b2, act, save=False)
    assert torch.equal(only[0], y) and only[1] is None and only[2] is None


@gpu
def test_gpu_strided_rows_and_accumulate():
    T, H, F, Ho = 200, 128, 192, 64
    x, w1, b1, w2, b2, dy = _make(T, H, F, Ho, True, seed=2, device=DEV)
    wide = lambda t: torch.cat([torch.full_like(t[:, :8], float("nan")), t, torch.full_like(t[:, :16], float("nan"))], 1)[:, 8:8 + t.shape[1]]
    y, pre, h = ops.gated_mlp_fwd(x, w1, b1, w2, b2)
    ys, pres, hs = ops.gated_mlp_fwd(wide(x), wide(w1), b1, wide(w2), b2)
    assert torch.equal(y, ys) and torch.equal(pre, pres) and torch.equal(h, hs)
    ref = ops.gated_mlp_bwd(dy, x, pre, h, w1, b1, w2, b2)
    got = ops.gated_mlp_bwd(wide(dy), wide(x), pre, h, wide(w1), b1, wide(w2), b2)
    for a, b in zip(ref, got):
        assert torch.equal(a, b)
    bufs = [torch.randn_like(t) for t in ref[1:]]
    before = [t.double() for t in bufs]
    ops.gated_mlp_bwd(dy, x, pre, h, w1, b1, w2, b2, dw1=bufs[0], db1=bufs[1], dw2=bufs[2], db2=bufs[3], accumulate=True)
    want = _oracle("silu", x, w1, b1, w2, b2, dy)
    for name, t, b in zip(("dw1", "db1", "dw2", "db2"), bufs, before):
        val, bound = want[name]
        _within(t, (val + b, bound + U * (val + b).abs()), name)


@gpu
def test_gpu_non_finite_rows_stay_in_theirs():
    """A token with NaN spoils its own row of y and dx alone."""
    T, H, F = 150, 72, 136
    x, w1, b1, w2, b2, dy = _make(T, H, F, H, True, seed=4, device=DEV)
    want = _oracle("silu", x, w1, b1, w2, b2, dy)
    x[70], dy[20] = float("nan"), float("inf")
    y, pre, h = ops.gated_mlp_fwd(x, w1, b1, w2, b2)
    dx = ops.gated_mlp_bwd(dy, x, pre, h, w1, b1, w2, b2, need_dw=False)[0]
    ok = torch.ones(T, dtype=torch.bool, device=DEV)
    ok[70] = False
    _within(y[ok], tuple(t[ok] for t in want["y"]), "y")
    assert torch.isnan(y[70]).all()
    ok[20] = False
    _within(dx[ok], tuple(t[ok] for t in want["dx"]), "dx")


@gpu
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gpu_saturated_gates(act):
    """Gates far in both tails: act' is 0 or 1 there, nothing overflows."""
    vals = torch.tensor([-3e38, -1e20, -1e4, -200.0, -60.0, 0.0, 60.0, 200.0, 1e4, 1e18])
    T, F = len(vals), 8
    x = torch.zeros(T, 8)
    x[:, 0] = vals
    w1 = torch.zeros(16, 8)
    w1[:8, 0] = 1.0
    b1 = torch.cat([torch.zeros(8), torch.full((8,), 2.0 ** -10)])
    w2 = torch.eye(8)
    args = [t.to(torch.bfloat16).to(DEV) for t in (x, w1, b1, w2)]
    y, pre, h = ops.gated_mlp_fwd(*args, None, act)
    gate = args[0][:, 0].double().cpu()
    torch.testing.assert_close(y[:, 0].double().cpu(), gate.clamp_min(0) * 2.0 ** -10, rtol=2 * U, atol=1e-20)
    dy = torch.full((T, 8), 1.0, dtype=torch.bfloat16, device=DEV)
    dx = ops.gated_mlp_bwd(dy, args[0], pre, h, args[1], args[2], args[3], None, act, need_dw=False)[0]
    slope = (gate > 0).double() + 0.5 * (gate == 0).double()
    torch.testing.assert_close(dx[:, 0].double().cpu(), 8 * slope * 2.0 ** -10, rtol=2 * U, atol=1e-20)


@gpu
def test_gpu_refusals():
    x, w1, b1, w2, b2, dy = _make(5, 16, 16, 16, True, device=DEV)
    bad = [
        (lambda: ops.gated_mlp_fwd(x.float(), w1.float(), b1.float(), w2.float(), b2.float()), TypeError),
        (lambda: ops.gated_mlp_fwd(x[:, :12], w1[:, :12], b1, w2, b2), ValueError),      # not a multiple of 8
        (lambda: ops.gated_mlp_fwd(x.t().contiguous().t(), w1, b1, w2, b2), ValueError),  # column stride
        (lambda: ops.gated_mlp_fwd(x[:1].expand(5, 16), w1, b1, w2, b2), ValueError),
        (lambda: ops.gated_mlp_fwd(x, w1.cpu(), b1, w2, b2), ValueError),
    ]
    for call, err in bad:
        with pytest.raises(err):
            call()


@gpu
def test_gpu_autograd():
    T, H, F = 30, 64, 72
    x, w1, b1, w2, b2, dy = _make(T, H, F, H, True, seed=6, device=DEV)
    leaves = [t.t().contiguous().t().requires_grad_(True) if t.dim() == 2 else t.requires_grad_(True) for t in (x, w1, b1, w2, b2)]
    y = ops.gated_mlp(leaves[0].view(3, 10, H), *leaves[1:], "gelu")
    g = torch.autograd.grad(y, leaves, dy.view(3, 10, H).transpose(0, 1).contiguous().transpose(0, 1))
    want = _oracle("gelu", *[t.detach() for t in (x, w1, b1, w2, b2)], dy)
    for name, t in zip(("y", "dx", "dw1", "db1", "dw2", "db2"), (y.detach().reshape(T, H), *g)):
        _within(t, want[name], name)
    x2 = x.detach().requires_grad_(True)      # frozen parameters
    (dx,) = torch.autograd.grad(ops.gated_mlp(x2, w1.detach(), None, w2.detach(), None).sum(), x2)
    assert torch.isfinite(dx).all()


@gpu
def test_gpu_captured_and_replayed():
    T, H, F = 70, 64, 136
    x, w1, b1, w2, b2, dy = _make(T, H, F, H, True, seed=7, device=DEV)

    def go():
        y, pre, h = ops.gated_mlp_fwd(x, w1, b1, w2, b2)
        return (y, *ops.gated_mlp_bwd(dy, x, pre, h, w1, b1, w2, b2))
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        go()
    torch.cuda.current_stream().wait_stream(st)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = go()
    for seed in (1, 2, 3):
        nx, *_, ndy = _make(T, H, F, H, True, seed=seed, device=DEV)
        x.copy_(nx)
        dy.copy_(ndy)
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip([t.clone() for t in outs], go()):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("tile", range(4))
@pytest.mark.parametrize("T,H,F,Ho", [(65, 8, 40, 264), (200, 264, 136, 72), (1003, 768, 520, 768)])
def test_paired_weight_gradients_equal_single_ones(monkeypatch, T, H, F, Ho, tile, accumulate):
    """Both weight gradients in one launch: the bits of two launches with the same tile."""
    import mxtrain.ops.gated as gated
    gen = torch.Generator().manual_seed(T + tile)
    r = lambda *s: torch.randn(*s, generator=gen).to(torch.bfloat16).cuda()
    x, w1, w2, dy = r(T, H), r(2 * F, H), r(Ho, F), r(T, Ho)
    pre, h = r(T, 2 * F), r(T, F)
    start = r(2 * F, H), r(Ho, F)
    monkeypatch.setattr(gated, "_plan", lambda *a: (tile, 1, 0.0))

    def go(pair):
        monkeypatch.setattr(gated, "_plan_pair", lambda *a: pair)
        wide = torch.full((2 * F, H + 16), 3.0, dtype=torch.bfloat16, device="cuda")
        wide[:, :H] = start[0]
        dw1, dw2 = wide[:, :H], start[1].clone()
        gated.gated_mlp_bwd(dy, x, pre, h, w1, None, w2, None, dw1=dw1, dw2=dw2, accumulate=accumulate)
        assert (wide[:, H:] == 3.0).all()
        return dw1, dw2
    for a, b in zip(go(tile), go(None)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_gradient_buffers_over_operands_are_refused(device):
    T, H, F = 16, 8, 8
    x, w1, b1, w2, b2, dy = _make(T, H, F, 16, True, device=device)
    y, pre, h = ops.gated_mlp_fwd(x, w1, b1, w2, b2)
    for grads in ({"dw1": x}, {"dw2": dy}, {"dw1": h}, {"db1": torch.empty_like(b1)} | {"db2": None}):
        if "db1" in grads:
            grads = {"db1": grads["db1"], "db2": grads["db1"]}       # (2 F = Ho)
        with pytest.raises(ValueError):
            ops.gated_mlp_bwd(dy, x, pre, h, w1, b1, w2, b2, **grads)


@gpu
@pytest.mark.parametrize("T", [16, 17, 38, 39, 64])
def test_gpu_few_tokens_of_wide_features(T):
    """Around the most tokens of the weight-streaming form, where that depends on the product's size."""
    H, F = 2048, 4096
    x, w1, b1, w2, b2, _ = _make(T, H, F, H, True, seed=T, device=DEV)
    y, pre, h = ops.gated_mlp_fwd(x, w1, b1, w2, b2)
    _within(y, _oracle("silu", x, w1, b1, w2, b2)["y"], "y")
    assert torch.equal(ops.gated_mlp_fwd(x, w1, b1, w2, b2, save=False)[0], y)


@gpu
@pytest.mark.parametrize("tile", range(5))
@pytest.mark.parametrize("T,H,F,Ho", [(70, 72, 136, 40), (333, 264, 200, 392), (1003, 768, 520, 256)])
def test_gpu_every_tile(monkeypatch, T, H, F, Ho, tile):
    """Any tile may be chosen for a shape: all of them, where they are taken, give the block's results."""
    import mxtrain.ops.gated as gated
    plan = gated._plan
    monkeypatch.setattr(gated, "_plan", lambda kind, *a: plan(kind, *a) if kind == "dw" else (tile, 1, 0.0))
    x, w1, b1, w2, b2, dy = _make(T, H, F, Ho, True, seed=T, device=DEV)
    y, pre, h = ops.gated_mlp_fwd(x, w1, b1, w2, b2, "gelu")
    got = dict(zip(("dx", "dw1", "db1", "dw2", "db2"), ops.gated_mlp_bwd(dy, x, pre, h, w1, b1, w2, b2, "gelu")), y=y)
    for name, want in _oracle("gelu", x, w1, b1, w2, b2, dy).items():
        _within(got[name], want, name)


@gpu
def test_gpu_tile_table_matches_the_kernels():
    import mxtrain.ops.gated as gated
    from mxtrain.ops import _lib
    for tile, row in enumerate(gated._TILES):
        assert (_lib.query("mx_gated_tile", tile, 0), _lib.query("mx_gated_tile", tile, 1)) == row[:2]
    assert _lib.query("mx_gated_tile", len(gated._TILES), 0) == -1


def test_a_plan_is_returned_though_another_thread_clears_the_table(monkeypatch, kernel_library):
    import mxtrain.ops.gated as gated
    monkeypatch.setattr(gated, "_PLANS", {})
    first = gated._plan_pair(1003, 768, 2048, 768), gated._plan("gate", 1003, 4096, 768)

    class Cleared(dict):           # whatever is looked up is gone before it is looked up again
        def __contains__(self, key):
            found = super().__contains__(key)
            self.clear()
            return found

        def __setitem__(self, key, value):
            super().__setitem__(key, value)
            self.clear()
    for kept in ({}, dict(gated._PLANS)):
        monkeypatch.setattr(gated, "_PLANS", Cleared(kept))
        assert (gated._plan_pair(1003, 768, 2048, 768), gated._plan("gate", 1003, 4096, 768)) == first


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_gradient_buffers_partly_over_operands_are_refused(device):
    """By one row or one value as much as from their start; side by side in one buffer they are taken."""
    T, H, F = 24, 16, 8
    x, w1, b1, w2, b2, dy = _make(T, H, F, H, True, device=device)
    y, pre, h = ops.gated_mlp_fwd(x, w1, b1, w2, b2)
    e = lambda *s: torch.zeros(*s, dtype=x.dtype, device=device)

    def bwd(x=x, dy=dy, pre=pre, h=h, **kw):
        return ops.gated_mlp_bwd(dy, x, pre, h, w1, b1, w2, b2, **kw)
    want = bwd()
    both = e(T + 15, H)                                    # x: rows 15 .. 38; dw1: rows 0 .. 15
    both[15:] = x
    mixed = e(2 * F * H + H * F)
    flat = e(T * 2 * F + 2 * F)
    flat[8:8 + T * 2 * F] = pre.reshape(-1)
    for call in (lambda: bwd(x=both[15:], dw1=both[:2 * F]),
                 lambda: bwd(pre=flat[8:8 + T * 2 * F].view(T, 2 * F), db1=flat[:2 * F]),
                 lambda: bwd(pre=flat[8:8 + T * 2 * F].view(T, 2 * F), db2=flat[T * 2 * F:T * 2 * F + H]),
                 lambda: bwd(dw1=mixed[:2 * F * H].view(2 * F, H), dw2=mixed[2 * F * H - 8:-8].view(H, F)),
                 lambda: bwd(dw2=mixed[8:8 + H * F].view(H, F), db2=mixed[H * F:H * F + H])):
        with pytest.raises(ValueError):
            call()
    wide = e(T, 2 * H + 8)                                 # columns of one buffer: x, and behind it dw1
    wide[:, :H] = x
    apart = bwd(x=wide[:, :H], dw1=wide[:2 * F, H:2 * H], dw2=mixed[:H * F].view(H, F), db1=mixed[H * F:H * F + 2 * F])
    for a, b in zip(apart, want):
        assert torch.equal(a, b)
    assert torch.equal(wide[:, :H], x)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_gradients_in_place_of_the_weights(device):
    """The weights are read before their gradients are written."""
    x, w1, b1, w2, b2, dy = _make(40, 16, 24, 8, True, device=device)
    y, pre, h = ops.gated_mlp_fwd(x, w1, b1, w2, b2)
    want = ops.gated_mlp_bwd(dy, x, pre, h, w1, b1, w2, b2)
    a, c = w1.clone(), w2.clone()
    for p, q in zip(ops.gated_mlp_bwd(dy, x, pre, h, a, b1, c, b2, dw1=a, dw2=c), want):
        assert torch.equal(p, q)
