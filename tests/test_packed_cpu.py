"""Packed attention on the CPU path: the row table, refusals, the formula and its gradients."""
import pytest
import torch

from mxtrain import ops
from packed_oracle import attention, within


def _cu(lens):
    return torch.tensor([0] + list(lens)).cumsum(0)


def test_row_table():
    s = ops.pack_sequences(_cu([3, 0, 0, 1, 4]), 10)
    assert s.start.tolist() == [0, 0, 0, 3, 4, 4, 4, 4, 8, 9]
    assert s.end.tolist() == [3, 3, 3, 4, 8, 8, 8, 8, 8, 9]
    assert s.positions.tolist() == [0, 1, 2, 0, 0, 1, 2, 3, 0, 0]
    assert int(s.meta[0]) == 8


def test_row_table_of_empty_sequences():
    s = ops.pack_sequences(_cu([0, 0]).int(), 3)
    assert int(s.meta[0]) == 0 and s.positions.tolist() == [0, 0, 0]


@pytest.mark.parametrize("cu,total,err", [
    (torch.tensor([0.0, 3.0]), 3, TypeError),
    (torch.tensor([[0, 3]]), 3, ValueError),
    (torch.tensor([0]), 3, ValueError),
    (torch.tensor([1, 3]), 3, ValueError),
    (torch.tensor([0, 3, 2]), 3, ValueError),
    (torch.tensor([0, 4]), 3, ValueError),
    (torch.tensor([0, 3]), 0, ValueError),
])
def test_row_table_refusals(cu, total, err):
    with pytest.raises(err):
        ops.pack_sequences(cu, total)


def test_attention_refusals():
    s = ops.pack_sequences(_cu([5, 3]), 8)
    q, k = torch.randn(8, 4 * 16), torch.randn(8, 2 * 16)
    for args, kw, err in (
            ((q, k, k, s, 4, 3, 16), {}, ValueError),            # heads do not group
            ((q[:7], k, k, s, 4, 2, 16), {}, ValueError),        # rows
            ((q, k[:, :16], k, s, 4, 2, 16), {}, ValueError),    # width
            ((q, k.double(), k, s, 4, 2, 16), {}, TypeError),    # types differ
            ((q, k, k, s, 4, 2, 16, -1.0), {}, ValueError),      # scale
            ((q, k, k, s, 4, 2, 16, float("nan")), {}, ValueError),
            ((q, k, k, [0, 5, 8], 4, 2, 16), {}, TypeError),
            ((q, k, k, s, 4, 2, 16), {"out": torch.empty(8, 16)}, ValueError)):
        with pytest.raises(err):
            ops.packed_attn_fwd(*args, **kw)
    o, lse = ops.packed_attn_fwd(q, k, k, s, 4, 2, 16)
    with pytest.raises(ValueError):
        ops.packed_attn_bwd(o, q, k, k, o, lse[:, :4], s, 4, 2, 16)


@pytest.mark.parametrize("lens,pad", [([1], 0), ([5, 0, 9, 1], 3), ([0], 2)])
def test_reference_matches_oracle(lens, pad):
    torch.manual_seed(1)
    T, Hq, Hkv, D = sum(lens) + pad, 4, 2, 16
    q, k, v, do = (torch.randn(T, h * D, dtype=torch.float64) for h in (Hq, Hkv, Hkv, Hq))
    s = ops.pack_sequences(_cu(lens), T)
    o, lse = ops.packed_attn_fwd(q, k, v, s, Hq, Hkv, D)
    dq, dk, dv = ops.packed_attn_bwd(do, q, k, v, o, lse, s, Hq, Hkv, D)
    want = attention(q, k, v, lens, Hq, Hkv, D, D ** -0.5, do)
    for name, t in (("o", o), ("dq", dq), ("dk", dk), ("dv", dv)):
        torch.testing.assert_close(t, want[name][0], rtol=1e-12, atol=1e-12)   # float64 on both sides
        assert (t[sum(lens):] == 0).all()


def test_gradients_against_differences():
    torch.manual_seed(2)
    s = ops.pack_sequences(_cu([4, 1, 3]), 9)
    q, k, v = (torch.randn(9, h * 8, dtype=torch.float64, requires_grad=True) for h in (4, 2, 2))
    assert torch.autograd.gradcheck(lambda a, b, c: ops.packed_attention(a, b, c, s, 4, 2, 8), (q, k, v))


def test_buffers_keep_the_rows_behind():
    s = ops.pack_sequences(_cu([2, 3]), 8)
    q = torch.randn(8, 16)
    out = torch.full((8, 16), 7.0)
    ops.packed_attn_fwd(q, q, q, s, 1, 1, 16, out=out)
    assert (out[5:] == 7.0).all() and not (out[:5] == 7.0).any()


def test_overlap_of_strided_matrices():
    from mxtrain.ops import _lib
    buf = torch.zeros(10, 96, dtype=torch.bfloat16)
    m = lambda t: (t.data_ptr(), t.stride(0), t.shape[1])
    owned = torch.zeros(40, 32, dtype=torch.int64)      # a plain count of who touches what

    def touch(t):
        owned.zero_()
        own = owned.view(-1)[:960].view(10, 96)
        r0, c0 = divmod((t.data_ptr() - buf.data_ptr()) // 2, 96)
        own[r0:r0 + t.shape[0], c0:c0 + t.shape[1]] = 1
        return own.clone()
    views = [buf[a:a + 6, c:c + w] for a in (0, 3, 4) for c, w in ((0, 32), (32, 32), (64, 32), (16, 40), (0, 96))]
    for x in views:
        for y in views:
            assert _lib.overlap(6, m(x), m(y)) >= bool((touch(x) & touch(y)).any())
    a, b = buf[:, :32], buf[:, 32:]
    assert not _lib.overlap(10, m(a), m(b)) and not _lib.overlap(10, m(b), m(a))
    assert _lib.overlap(10, m(a), m(a)) and _lib.overlap(10, m(a), (a.data_ptr() + 64, 200, 8))
    assert not _lib.overlap(10, m(buf), m(torch.zeros(10, 96, dtype=torch.bfloat16)))


@pytest.mark.parametrize("D,kb", [(64, 128), (128, 256)])
@pytest.mark.parametrize("heads", [(8, 1), (4, 1), (16, 4), (32, 8), (20, 5), (12, 12), (16, 16)])
def test_no_split_of_a_key_block_is_empty(heads, D, kb, kernel_library):
    """Every split of a key block begins at one of its (query head, query tile) items: one that did not
    would fetch the rows and statistics of a query head that is not there.  (Lengths of one document, and
    the first of two, up to where blocks are no longer split.)"""
    from mxtrain.ops import _lib
    Hq, Hkv = heads
    split = set()
    for T in (*range(1, 2200, 7), *range(640, 1605, 64), *range(2200, 20000, 411)):
        for n in {T, max(1, T // 3)}:
            ends = [n if k < n else T for k in range(0, T, kb)]
            per_block = [-(-(max(e, min(k + kb, T)) - k) // 64) for e, k in zip(ends, range(0, T, kb))]
            tiles = sum(per_block)
            for q in set(per_block):
                items = q * (Hq // Hkv)
                nsp = _lib.query("mx_packed_block_splits", T, Hq, Hkv, D, tiles, items)
                if nsp == 0:       # (cut into even shares)
                    continue
                assert 1 <= nsp <= 16
                per = -(-items // nsp)
                assert (nsp - 1) * per < items, (T, n, items, nsp)
                split.add(nsp)
    assert split


def test_more_sequences_than_the_table_counts_are_refused():
    for n in ((1 << 30) + 2, (1 << 32) + 3):
        with pytest.raises(ValueError, match="2\\^30"):
            ops.pack_sequences(torch.empty(n, dtype=torch.int64, device="meta"), 8)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_non_finite_values_reach_only_the_rows_that_see_them(bad):
    torch.manual_seed(3)
    lens, pad, Hq, Hkv, D = [7, 1, 9, 6], 3, 4, 2, 8
    T = sum(lens) + pad
    s = ops.pack_sequences(_cu(lens), T)
    q, k, v, do = (torch.randn(T, h * D, dtype=torch.float64) for h in (Hq, Hkv, Hkv, Hq))
    want = attention(q, k, v, lens, Hq, Hkv, D, D ** -0.5, do)

    def go(at, *which):
        x = [t.clone() for t in (q, k, v, do)]
        for i in which:
            x[i][at] = bad
        o, lse = ops.packed_attn_fwd(*x[:3], s, Hq, Hkv, D)
        return dict(zip(("o", "lse", "dq", "dk", "dv"),
                        (o, lse, *ops.packed_attn_bwd(x[3], *x[:3], o, lse, s, Hq, Hkv, D))))

    def same(t, name, rows):
        ref = want[name][0]
        if name == "lse":
            t, ref = t.double().t(), ref.float().double().t()
        torch.testing.assert_close(t[rows], ref[rows], rtol=1e-6 if name == "lse" else 1e-12, atol=1e-12)
    got = go([3, 20, 24, 25], 0, 1, 2, 3)         # in the first and the last sequence and behind them
    for name in got:
        same(got[name], name, slice(7, 17))
    same(got["o"], "o", slice(0, 3))              # (rows before the bad ones)
    same(got["dq"], "dq", slice(0, 3))
    for name in ("dk", "dv"):
        assert torch.isnan(got[name][:7]).all()   # (every key is seen by a row that sees the bad ones)
        assert (got[name][23:] == 0).all()
    assert torch.isnan(got["o"][3:7]).all() and (got["o"][23:] == 0).all()
    got = go([12], 3)                             # a row of dout: its own dq, and dk, dv of the keys it sees
    for name, rows in (("dq", 12), ("dk", slice(8, 13)), ("dv", slice(8, 13))):
        assert not torch.isfinite(got[name][rows]).any()
    for name, rows in (("dq", slice(13, 17)), ("dq", slice(8, 12)), ("dk", slice(13, 17)), ("dv", slice(13, 17))):
        same(got[name], name, rows)


def test_large_finite_values_of_masked_pairs_on_the_cpu():
    torch.manual_seed(4)
    s, T = ops.pack_sequences(_cu([5, 6]), 11), 11
    q, k, v, do = (torch.randn(T, 8) for _ in range(4))
    do[:5] *= 1e20
    v[5:] *= 1e20
    o, lse = ops.packed_attn_fwd(q, k, v, s, 1, 1, 8)
    for name, t in zip(("dq", "dk", "dv"), ops.packed_attn_bwd(do, q, k, v, o, lse, s, 1, 1, 8)):
        within(t, attention(q, k, v, [5, 6], 1, 1, 8, 8 ** -0.5, do)[name], name)


def test_gradients_over_the_statistics_are_refused(monkeypatch):
    from mxtrain.ops import _lib
    T, H, D = 8, 2, 64
    s = ops.pack_sequences(_cu([5, 3]), T)
    q, k, v, do, o, dk, dv = (torch.randn(T, H * D).bfloat16() for _ in range(7))
    mem = torch.zeros(T * H * D, dtype=torch.bfloat16)
    lse = mem.view(torch.float32)[-H * T:].view(H, T)
    monkeypatch.setattr(_lib, "use_hip", lambda t: True)
    with pytest.raises(ValueError, match="must not lie over"):
        ops.packed_attn_bwd(do, q, k, v, o, lse, s, H, H, D, dq=mem.view(T, H * D), dk=dk, dv=dv)


def test_scales_beyond_the_kernels_range_are_refused(monkeypatch):
    """They hold the scale, and lse divided by it, in fp32."""
    from mxtrain.ops import _lib
    T, H, D = 8, 2, 64
    s = ops.pack_sequences(_cu([5, 3]), T)
    q = torch.randn(T, H * D).bfloat16()
    o, lse = ops.packed_attn_fwd(q, q, q, s, H, H, D, 1e-39)          # (taken on the CPU)
    monkeypatch.setattr(_lib, "use_hip", lambda t: True)
    for scale in (1e-50, 1e-39, 1e31, 1e300):
        with pytest.raises(ValueError, match="scale"):
            ops.packed_attn_fwd(q, q, q, s, H, H, D, scale)
        with pytest.raises(ValueError, match="scale"):
            ops.packed_attn_bwd(q, q, q, q, o, lse, s, H, H, D, scale)
