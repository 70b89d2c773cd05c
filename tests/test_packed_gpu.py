"""Packed attention kernels (csrc/packed.hip) against the 64-bit oracle and its derived bounds."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from mxtrain import ops  # noqa: E402
from packed_oracle import attention, within  # noqa: E402

DEV = "cuda"


def _cu(lens):
    return torch.tensor([0] + list(lens)).cumsum(0)


def _inputs(T, Hq, Hkv, D, seed=0, gap=0):
    """q, k, v as column ranges of one buffer (row stride wider than the heads by ``gap``)."""
    gen = torch.Generator().manual_seed(seed)
    buf = torch.randn(T, (Hq + 2 * Hkv) * D + gap, generator=gen).to(torch.bfloat16).to(DEV)
    do = torch.randn(T, Hq * D, generator=gen).to(torch.bfloat16).to(DEV)
    q, k, v = buf[:, :Hq * D], buf[:, Hq * D:(Hq + Hkv) * D], buf[:, (Hq + Hkv) * D:(Hq + 2 * Hkv) * D]
    return q, k, v, do


LENS = [
    ([1], 0), ([1, 1, 1], 1), ([0, 5, 0], 0), ([31, 32, 33], 0), ([127, 1, 129], 3), ([128, 128], 0),
    ([64, 2, 190, 0, 77], 51), ([300], 129), ([3] * 100, 0), ([513, 200], 0), ([0, 0], 4),
]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("heads", [(2, 2), (8, 2), (3, 1)])
@pytest.mark.parametrize("lens,pad", LENS)
def test_forward_backward(lens, pad, heads, D):
    Hq, Hkv = heads
    T = sum(lens) + pad
    q, k, v, do = _inputs(T, Hq, Hkv, D, seed=T, gap=8)
    s = ops.pack_sequences(_cu(lens), T, device=DEV)
    o, lse = ops.packed_attn_fwd(q, k, v, s, Hq, Hkv, D)
    dq, dk, dv = ops.packed_attn_bwd(do, q, k, v, o, lse, s, Hq, Hkv, D)
    want = attention(q, k, v, lens, Hq, Hkv, D, D ** -0.5, do)
    for name, t in (("o", o), ("lse", lse), ("dq", dq), ("dk", dk), ("dv", dv)):
        within(t, want[name], name)


@pytest.mark.parametrize("D,lens,heads", [(64, [2500, 1, 700, 895], (4, 2)), (128, [1500, 2600], (2, 1))])
def test_longer_sequences(D, lens, heads):
    Hq, Hkv = heads
    T = sum(lens) + 77
    q, k, v, do = _inputs(T, Hq, Hkv, D, seed=5)
    s = ops.pack_sequences(_cu(lens), T, device=DEV)
    o, lse = ops.packed_attn_fwd(q, k, v, s, Hq, Hkv, D, scale=0.3)
    grads = ops.packed_attn_bwd(do, q, k, v, o, lse, s, Hq, Hkv, D, scale=0.3)
    want = attention(q, k, v, lens, Hq, Hkv, D, 0.3, do)
    for name, t in zip(("o", "dq", "dk", "dv"), (o, *grads)):
        within(t, want[name], name)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_row_table_matches_cpu(dtype):
    lens = [0, 3, 0, 0, 260, 1, 77, 0]
    cu = _cu(lens).to(dtype)
    for given in (cu, cu.to(DEV)):
        a, b = ops.pack_sequences(given, 400, device=DEV), ops.pack_sequences(cu, 400)
        for f in ("start", "end", "positions"):
            assert torch.equal(getattr(a, f).cpu(), getattr(b, f)), f
        assert int(a.meta[0]) == int(b.meta[0])


def test_malformed_table_on_the_gpu_stays_in_range():
    cu = torch.tensor([5, -3, 900, 40, 1 << 40], device=DEV)
    s = ops.pack_sequences(cu, 200)
    t = torch.arange(200, device=DEV)
    assert ((s.start >= 0) & (s.start <= t)).all() and ((s.end > t) & (s.end <= 200)).all()
    assert int(s.meta[0]) == 200


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_non_finite_values_stay_in_their_sequence(D, bad):
    """Sequences 0, 2 and the rows behind the end hold non-finite values; sequence 1 and 3 must
    get exactly what they get beside finite neighbours."""
    lens, pad, H = [40, 50, 70, 30], 20, 2
    T = sum(lens) + pad
    q, k, v, do = _inputs(T, H, H, D, seed=3)
    s = ops.pack_sequences(_cu(lens), T, device=DEV)
    clean = ops.packed_attn_fwd(q, k, v, s, H, H, D)
    cleang = ops.packed_attn_bwd(do, q, k, v, *clean, s, H, H, D)
    want = attention(q, k, v, lens, H, H, D, D ** -0.5, do)
    for t in (q, k, v, do):
        t[10:20] = bad
        t[100:110] = bad
        t[190:] = bad
    o, lse = ops.packed_attn_fwd(q, k, v, s, H, H, D)
    grads = ops.packed_attn_bwd(do, q, k, v, o, lse, s, H, H, D)
    for name, t in zip(("o", "dq", "dk", "dv"), (o, *grads)):
        for rows in (slice(40, 90), slice(160, 190)):
            within(t[rows], tuple(x[rows] for x in want[name]), name)
        assert (t[190:] == 0).all(), name


@pytest.mark.parametrize("D", [64, 128])
def test_later_rows_do_not_reach_earlier_ones(D):
    """A NaN row inside a sequence: the rows before it see none of it; the rows from it on do."""
    T, H, at = 200, 2, 75
    q, k, v, do = _inputs(T, H, H, D, seed=4)
    s = ops.pack_sequences(_cu([T]), T, device=DEV)
    want = attention(q, k, v, [T], H, H, D, D ** -0.5)
    v[at] = float("nan")
    o, _ = ops.packed_attn_fwd(q, k, v, s, H, H, D)
    within(o[:at], tuple(x[:at] for x in want["o"]), "o")
    assert torch.isnan(o[at:]).all()
    q, k, v, do = _inputs(T, H, H, D, seed=4)
    o, lse = ops.packed_attn_fwd(q, k, v, s, H, H, D)
    want = attention(q, k, v, [T], H, H, D, D ** -0.5, do)
    do[at] = float("nan")      # row `at` touches the keys up to it alone
    dq, dk, dv = ops.packed_attn_bwd(do, q, k, v, o, lse, s, H, H, D)
    for name, t in (("dk", dk), ("dv", dv)):
        within(t[at + 1:], tuple(x[at + 1:] for x in want[name]), name)
        assert torch.isnan(t[:at + 1]).all()
    keep = torch.arange(T, device=DEV) != at
    within(dq[keep], tuple(x[keep] for x in want["dq"]), "dq")


def test_extreme_scores():
    """Rows whose scores span far more than the range of exp; the largest must win exactly."""
    T, H, D = 150, 2, 64
    q, k, v, _ = _inputs(T, H, H, D, seed=8)
    q.mul_(64.0)
    k.mul_(64.0)
    s = ops.pack_sequences(_cu([T]), T, device=DEV)
    o, _ = ops.packed_attn_fwd(q, k, v, s, H, H, D)
    assert torch.isfinite(o).all()
    top = torch.stack([(q[:, h * D:(h + 1) * D].double() @ k[:, h * D:(h + 1) * D].double().t())
                       .masked_fill(torch.ones(T, T, dtype=torch.bool, device=DEV).triu(1), -1e300).argmax(1)
                       for h in range(H)])
    for h in range(H):
        sc = (q[:, h * D:(h + 1) * D].double() @ k[:, h * D:(h + 1) * D].double().t()) * D ** -0.5
        sc = sc.masked_fill(torch.ones(T, T, dtype=torch.bool, device=DEV).triu(1), -1e300)
        two = sc.topk(2, 1).values if T > 1 else sc
        clear = two[:, 0] - two[:, 1] > 40.0       # every other weight is below 2^-57
        got = o[:, h * D:(h + 1) * D]
        assert torch.equal(got[clear], v[top[h][clear], h * D:(h + 1) * D])


def test_buffers_and_rows_behind():
    lens, pad, Hq, Hkv, D = [100, 33], 60, 4, 2, 64
    T = sum(lens) + pad
    q, k, v, do = _inputs(T, Hq, Hkv, D, seed=6)
    s = ops.pack_sequences(_cu(lens), T, device=DEV)
    o, lse = ops.packed_attn_fwd(q, k, v, s, Hq, Hkv, D)
    assert (o[133:] == 0).all() and torch.isinf(lse[:, 133:]).all()
    buf = torch.full((T, Hq * D + 64), 3.0, dtype=torch.bfloat16, device=DEV)
    out, _ = ops.packed_attn_fwd(q, k, v, s, Hq, Hkv, D, out=buf[:, 64:])
    assert torch.equal(out[:133], o[:133]) and (buf[133:] == 3.0).all() and (buf[:, :64] == 3.0).all()
    ref = ops.packed_attn_bwd(do, q, k, v, o, lse, s, Hq, Hkv, D)
    pack = torch.full((T, (Hq + 2 * Hkv) * D), 3.0, dtype=torch.bfloat16, device=DEV)
    views = pack[:, :Hq * D], pack[:, Hq * D:(Hq + Hkv) * D], pack[:, (Hq + Hkv) * D:]
    ops.packed_attn_bwd(do, q, k, v, o, lse, s, Hq, Hkv, D, dq=views[0], dk=views[1], dv=views[2])
    for a, b in zip(views, ref):
        assert torch.equal(a[:133], b[:133]) and (b[133:] == 0).all()
    assert (pack[133:] == 3.0).all()


def test_refusals():
    s = ops.pack_sequences(_cu([8]), 8, device=DEV)
    q = torch.randn(8, 128, device=DEV, dtype=torch.bfloat16)
    big = torch.randn(8, 136, device=DEV, dtype=torch.bfloat16)
    for args, err in (((q.half(), q.half(), q.half(), s, 2, 2, 64), TypeError),
                      ((q, q, q, s, 4, 4, 32), ValueError),                         # head dimension
                      ((big[:, 1:129], q, q, s, 2, 2, 64), ValueError),             # alignment
                      ((q[:1].expand(8, 128), q, q, s, 2, 2, 64), ValueError),      # rows that overlap
                      ((q, q.cpu(), q, s, 2, 2, 64), ValueError)):
        with pytest.raises(err):
            ops.packed_attn_fwd(*args)
    o, lse = ops.packed_attn_fwd(q, q, q, s, 2, 2, 64)
    with pytest.raises(ValueError):
        ops.packed_attn_bwd(o, q, q, q, o, lse, s, 2, 2, 64, dq=torch.empty_like(q))
    with pytest.raises(ValueError):
        ops.packed_attn_bwd(o, q, q, q, o, lse, s, 2, 2, 64, dq=q, dk=torch.empty_like(q), dv=torch.empty_like(q))


def test_autograd_takes_any_strides():
    T, H, D = 70, 2, 64
    s = ops.pack_sequences(_cu([30, 40]), T, device=DEV)
    x = [torch.randn(H * D, T, device=DEV).to(torch.bfloat16).t().requires_grad_(True) for _ in range(3)]
    o = ops.packed_attention(*x, s, H, H, D)
    g = torch.autograd.grad(o, x, torch.ones(1, 1, device=DEV, dtype=torch.bfloat16).expand(T, H * D))
    want = attention(*[t.detach() for t in x], [30, 40], H, H, D, D ** -0.5,
                     torch.ones(T, H * D, device=DEV))
    for name, t in zip(("o", "dq", "dk", "dv"), (o.detach(), *g)):
        within(t, want[name], name)


def test_two_runs_are_equal_and_streams():
    lens, Hq, Hkv, D = [400, 123, 300], 8, 2, 128
    T = sum(lens)
    q, k, v, do = _inputs(T, Hq, Hkv, D, seed=9)
    s = ops.pack_sequences(_cu(lens), T, device=DEV)

    def go():
        o, lse = ops.packed_attn_fwd(q, k, v, s, Hq, Hkv, D)
        return (o, *ops.packed_attn_bwd(do, q, k, v, o, lse, s, Hq, Hkv, D))
    a = go()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = go()
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip(a, b):
        assert torch.equal(x, y)


def test_captured_step_replays_on_new_batches():
    """Table, forward and backward captured once; replays see new lengths and new values."""
    Hq, Hkv, D, T = 4, 2, 64, 300
    batches = [([100, 150, 0], 1), ([10, 5, 280], 2), ([299, 0, 1], 3), ([0, 0, 0], 4)]
    cu = torch.zeros(4, dtype=torch.int64, device=DEV)
    buf = torch.zeros(T, (Hq + 2 * Hkv) * D, dtype=torch.bfloat16, device=DEV)
    do = torch.zeros(T, Hq * D, dtype=torch.bfloat16, device=DEV)
    q, k, v = buf[:, :Hq * D], buf[:, Hq * D:(Hq + Hkv) * D], buf[:, (Hq + Hkv) * D:]

    def go():
        s = ops.pack_sequences(cu, T)
        o, lse = ops.packed_attn_fwd(q, k, v, s, Hq, Hkv, D)
        return (o, *ops.packed_attn_bwd(do, q, k, v, o, lse, s, Hq, Hkv, D))

    def load(lens, seed):
        cu.copy_(_cu(lens))
        gen = torch.Generator().manual_seed(seed)
        buf.copy_(torch.randn(buf.shape, generator=gen))
        do.copy_(torch.randn(do.shape, generator=gen))
    load(*batches[0])
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        go()
    torch.cuda.current_stream().wait_stream(st)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = go()
    for b in batches[1:] + batches[:1]:
        load(*b)
        g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        for x, y in zip(got, go()):
            assert torch.equal(x, y)


@pytest.mark.parametrize("D", [64, 128])
def test_non_finite_values_beside_split_key_blocks(D):
    """Few key heads and long sequences: key blocks split over workgroups, with NaN next door."""
    lens, Hq, Hkv = [1300, 900], 4, 1
    T = sum(lens) + 10
    q, k, v, do = _inputs(T, Hq, Hkv, D, seed=21)
    s = ops.pack_sequences(_cu(lens), T, device=DEV)
    want = attention(q, k, v, lens, Hq, Hkv, D, D ** -0.5, do)
    for t in (q, k, v, do):
        t[1290:1300] = float("nan")
        t[2200:] = float("inf")
    o, lse = ops.packed_attn_fwd(q, k, v, s, Hq, Hkv, D)
    grads = ops.packed_attn_bwd(do, q, k, v, o, lse, s, Hq, Hkv, D)
    for name, t in zip(("o", "dq", "dk", "dv"), (o, *grads)):
        within(t[1300:2200], tuple(x[1300:2200] for x in want[name]), name)
        assert (t[2200:] == 0).all(), name
    within(o[:1290], tuple(x[:1290] for x in want["o"]), "o")
    assert torch.isnan(o[1290:1300]).all() and torch.isnan(grads[1][:1300]).all()


@pytest.mark.parametrize("lens,pad,heads", [([1500, 1, 30, 1200, 700], 351, (16, 4)), ([900, 3000], 0, (16, 2)),
                                            ([1000], 0, (64, 1)), ([5] * 400 + [1800], 7, (24, 8)),
                                            ([256, 256, 512, 255, 1], 9000, (8, 4))])
def test_shared_key_heads_over_even_shares(lens, pad, heads):
    """Grouped heads of 128 with enough work that the key blocks are cut into even shares."""
    (Hq, Hkv), D = heads, 128
    T = sum(lens) + pad
    nv = T - pad
    assert T * Hq >= 60000
    q, k, v, do = _inputs(T, Hq, Hkv, D, seed=31)
    s = ops.pack_sequences(_cu(lens), T, device=DEV)
    want = attention(q, k, v, lens, Hq, Hkv, D, D ** -0.5, do)
    q[nv:], k[nv:], v[nv:], do[nv:] = (float("nan"),) * 4
    o, lse = ops.packed_attn_fwd(q, k, v, s, Hq, Hkv, D)
    grads = ops.packed_attn_bwd(do, q, k, v, o, lse, s, Hq, Hkv, D)
    for name, t in zip(("dq", "dk", "dv"), grads):
        within(t[:nv], tuple(x[:nv] for x in want[name]), name)
        assert (t[nv:] == 0).all(), name
    mine = [torch.full_like(t, 3.0) for t in grads]
    ops.packed_attn_bwd(do, q, k, v, o, lse, s, Hq, Hkv, D, dq=mine[0], dk=mine[1], dv=mine[2])
    for name, a, b in zip(("dq", "dk", "dv"), mine, grads):
        assert torch.equal(a[:nv], b[:nv]) and (a[nv:] == 3.0).all(), name


def test_non_finite_values_beside_even_shares():
    lens, Hq, Hkv, D = [1900, 2300], 16, 4, 128
    T = sum(lens) + 10
    q, k, v, do = _inputs(T, Hq, Hkv, D, seed=32)
    s = ops.pack_sequences(_cu(lens), T, device=DEV)
    want = attention(q, k, v, lens, Hq, Hkv, D, D ** -0.5, do)
    for t in (q, k, v, do):
        t[1890:1900] = float("nan")
    o, lse = ops.packed_attn_fwd(q, k, v, s, Hq, Hkv, D)
    grads = ops.packed_attn_bwd(do, q, k, v, o, lse, s, Hq, Hkv, D)
    for name, t in zip(("o", "dq", "dk", "dv"), (o, *grads)):
        within(t[1900:4200], tuple(x[1900:4200] for x in want[name]), name)
    within(o[:1890], tuple(x[:1890] for x in want["o"]), "o")
    assert torch.isnan(grads[1][:1900]).all()


def test_shares_of_an_empty_and_a_changed_batch_in_a_graph():
    Hq, Hkv, D, T = 16, 4, 128, 3900
    cu = torch.zeros(4, dtype=torch.int64, device=DEV)
    q, k, v, do = _inputs(T, Hq, Hkv, D, seed=33)

    def go():
        s = ops.pack_sequences(cu, T)
        o, lse = ops.packed_attn_fwd(q, k, v, s, Hq, Hkv, D)
        return (o, *ops.packed_attn_bwd(do, q, k, v, o, lse, s, Hq, Hkv, D))
    cu.copy_(_cu([3000, 0, 900]))
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        go()
    torch.cuda.current_stream().wait_stream(st)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = go()
    for lens in ([0, 0, 0], [3900, 0, 0], [17, 2000, 1], [3000, 0, 900]):
        cu.copy_(_cu(lens))
        g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        for x, y in zip(got, go()):
            assert torch.equal(x, y)


def test_results_over_operands_are_refused():
    T, H, D = 40, 2, 64
    s = ops.pack_sequences(_cu([T]), T, device=DEV)
    buf = torch.randn(T, 8 * H * D, device=DEV).to(torch.bfloat16)
    q, k, v, do, a, b, c, e = buf.split(H * D, 1)
    o, lse = ops.packed_attn_fwd(q, k, v, s, H, H, D, out=a)       # other columns of the operands' buffer
    for bad in (q, k, v, buf[:, 64:64 + H * D]):
        with pytest.raises(ValueError):
            ops.packed_attn_fwd(q, k, v, s, H, H, D, out=bad)
    want = ops.packed_attn_bwd(do, q, k, v, o, lse, s, H, H, D)
    got = ops.packed_attn_bwd(do, q, k, v, o, lse, s, H, H, D, dq=b, dk=c, dv=e)
    for x, y in zip(want, got):
        assert torch.equal(x, y)
    for bad in ((b, c, c), (b, b, c), (o, b, c), (b, c, do), (b, k, c)):
        with pytest.raises(ValueError):
            ops.packed_attn_bwd(do, q, k, v, o, lse, s, H, H, D, dq=bad[0], dk=bad[1], dv=bad[2])


@pytest.mark.parametrize("lens,pad,Hq,Hkv", [([1200, 900], 31, 32, 32), ([40] * 50, 0, 32, 4), ([2048], 0, 17, 17),
                                             ([1, 2047], 1, 16, 16)])
def test_many_blocks_of_narrow_heads(lens, pad, Hq, Hkv):
    """More query blocks than CUs (whole 128-row blocks), and just as many (halved ones)."""
    D, T = 64, sum(lens) + pad
    nv = T - pad
    q, k, v, do = _inputs(T, Hq, Hkv, D, seed=41)
    s = ops.pack_sequences(_cu(lens), T, device=DEV)
    want = attention(q, k, v, lens, Hq, Hkv, D, D ** -0.5, do)
    for t in (q, k, v, do):
        t[nv:] = float("inf")
    o, lse = ops.packed_attn_fwd(q, k, v, s, Hq, Hkv, D)
    for name, t in zip(("o", "dq", "dk", "dv"), (o, *ops.packed_attn_bwd(do, q, k, v, o, lse, s, Hq, Hkv, D))):
        within(t[:nv], tuple(x[:nv] for x in want[name]), name)
        assert (t[nv:] == 0).all(), name


@pytest.mark.parametrize("bad", [float("nan"), float("-inf")])
@pytest.mark.parametrize("D,H,lens", [(64, 32, [700, 800]), (64, 4, [700, 800]), (128, 4, [700, 800])])
def test_non_finite_values_in_either_form(D, H, lens, bad):
    T = sum(lens)
    q, k, v, do = _inputs(T, H, H, D, seed=42)
    s = ops.pack_sequences(_cu(lens), T, device=DEV)
    want = attention(q, k, v, lens, H, H, D, D ** -0.5, do)
    for t in (q, k, v, do):
        t[690:700] = bad
    o, lse = ops.packed_attn_fwd(q, k, v, s, H, H, D)
    grads = ops.packed_attn_bwd(do, q, k, v, o, lse, s, H, H, D)
    for name, t in zip(("o", "dq", "dk", "dv"), (o, *grads)):
        within(t[700:], tuple(x[700:] for x in want[name]), name)
    within(o[:690], tuple(x[:690] for x in want["o"]), "o")
    within(grads[0][:690], tuple(x[:690] for x in want["dq"]), "dq")


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens", [[700], [1541], [641, 5]])
def test_one_key_head_of_one_document(lens, D):
    """Key blocks cut into the most splits, where a whole number of items does not divide among them."""
    Hq, Hkv, T = 8, 1, sum(lens)
    q, k, v, do = _inputs(T, Hq, Hkv, D, seed=51)
    s = ops.pack_sequences(_cu(lens), T, device=DEV)
    o, lse = ops.packed_attn_fwd(q, k, v, s, Hq, Hkv, D)
    want = attention(q, k, v, lens, Hq, Hkv, D, D ** -0.5, do)
    for name, t in zip(("o", "dq", "dk", "dv"), (o, *ops.packed_attn_bwd(do, q, k, v, o, lse, s, Hq, Hkv, D))):
        within(t, want[name], name)


@pytest.mark.parametrize("D,heads,lens", [(64, (2, 2), [100, 90]), (64, (4, 1), [1300, 900]), (128, (2, 2), [100, 90]),
                                          (128, (4, 1), [1300, 900]), (128, (16, 4), [1900, 2300])])
@pytest.mark.parametrize("inside", [False, True])
def test_large_finite_values_of_masked_pairs(D, heads, lens, inside):
    """dout of the first rows and V of the last ones are so large that their products, which no row may see,
    pass the fp32 range: on both sides of a border, and inside a document, where no earlier row sees a later
    key."""
    (Hq, Hkv), T = heads, sum(lens)
    q, k, v, do = _inputs(T, Hq, Hkv, D, seed=61)
    at = lens[0]
    do[:at] *= 1e20
    v[at:] *= 1e20
    lens = [T] if inside else lens
    s = ops.pack_sequences(_cu(lens), T, device=DEV)
    want = attention(q, k, v, lens, Hq, Hkv, D, D ** -0.5, do)
    o, lse = ops.packed_attn_fwd(q, k, v, s, Hq, Hkv, D)
    grads = ops.packed_attn_bwd(do, q, k, v, o, lse, s, Hq, Hkv, D)
    for name, t in zip(("o", "dq", "dk", "dv"), (o, *grads)):
        within(t, want[name], name)


def _mixed(T, longest, seed):
    gen, out = torch.Generator().manual_seed(seed), []
    while sum(out) < T:
        out.append(min(int(torch.randint(1, longest, (1,), generator=gen)), T - sum(out)))
    return out


@pytest.mark.parametrize("T,longest", [(1000, 300), (262144, 900), (262401, 60000), (600001, 3000)])
def test_dispatch_lists(T, longest):
    """Every block once (by work up to 2048 blocks), and the query tiles before each 256-key block."""
    s = ops.pack_sequences(_cu(_mixed(T, longest, T)), T, device=DEV)
    start, end, order = s.start.cpu().long(), s.end.cpu().long(), s.order.cpu().long()
    at = 0
    for which, B in (("query", 128), ("key", 128), ("key", 256)):
        nb = -(-T // B)
        first, last = torch.arange(nb) * B, (torch.arange(nb) * B + B).clamp_max(T)
        work = last - start[first] if which == "query" else end[last - 1] - first
        mine = order[at:at + nb]
        assert torch.equal(mine.sort().values, torch.arange(nb))
        if nb <= 2048:
            assert (work[mine].diff() <= 0).all()
        at += nb
    before = s.order[at + at % 2:].view(torch.int64).cpu()
    assert torch.equal(before[:nb + 1], torch.cat([torch.zeros(1, dtype=torch.int64), ((work + 63) // 64).cumsum(0)]))


@pytest.mark.parametrize("T,heads,D,longest", [(262500, (2, 2), 64, 900), (17000, (8, 4), 128, 2000), (40000, (16, 2), 128, 3000)])
def test_many_blocks(T, heads, D, longest):
    """Blocks in sequence order, and shares that begin past the 64th key block of a head."""
    Hq, Hkv = heads
    lens = _mixed(T, longest, T)
    q, k, v, do = _inputs(T, Hq, Hkv, D, seed=71)
    s = ops.pack_sequences(_cu(lens), T, device=DEV)
    o, lse = ops.packed_attn_fwd(q, k, v, s, Hq, Hkv, D)
    want = attention(q, k, v, lens, Hq, Hkv, D, D ** -0.5, do)
    for name, t in zip(("o", "dq", "dk", "dv"), (o, *ops.packed_attn_bwd(do, q, k, v, o, lse, s, Hq, Hkv, D))):
        within(t, want[name], name)
