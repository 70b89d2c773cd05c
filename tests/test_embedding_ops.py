"""Scaled embedding and its sorted-token gradient: CPU path against the formula and differences,
GPU kernels (csrc/embedding.hip) against 64-bit sums."""
import pytest
import torch

from mxtrain import ops

U = 2.0 ** -8      # bf16 half step


def _oracle_bwd(keys, dout, rows, scale, start=0):
    """(value, bound): sums in 64 bits.  The kernels add 32 rows at a time in fp32, then the sums of
    these: an fp32 chain of at most 32 + T / 32 additions (and the scale), half a step of 2^-24 each
    of the sum of magnitudes; then one bf16 rounding."""
    F = (32 + keys.numel() / 32 + 4) * 2.0 ** -24
    loc = keys.reshape(-1).cpu() - start
    ok = (loc >= 0) & (loc < rows)
    d = dout.double().cpu()[ok]
    val = torch.zeros(rows, dout.shape[1], dtype=torch.float64).index_add_(0, loc[ok], d) * scale
    mag = torch.zeros_like(val).index_add_(0, loc[ok], d.abs()) * abs(scale)
    return val, F * mag + U * val.abs()


def _within(got, val, bound):
    err = (got.double().cpu() - val).abs()
    bad = ~(err <= bound + 1e-30)
    assert not bad.any(), f"{int(bad.sum())} outside, worst {float(err[bad].max()):.3e}"


# ------------------------------------------------------------------ CPU
def test_cpu_formula():
    torch.manual_seed(0)
    ids, pos = torch.tensor([[3, 0, 9], [3, 5, -1]]), torch.tensor([[0, 1, 2], [0, 7, 1]])
    wte, wpe = torch.randn(6, 4, dtype=torch.float64), torch.randn(3, 4, dtype=torch.float64)
    out = ops.embedding(ids, wte, 2.5, pos, wpe)
    assert out.shape == (2, 3, 4)
    zero = torch.zeros(4, dtype=torch.float64)
    for i in range(2):
        for j in range(3):
            a, p = int(ids[i, j]), int(pos[i, j])
            want = (2.5 * wte[a] if 0 <= a < 6 else zero) + (wpe[p] if p < 3 else zero)
            torch.testing.assert_close(out[i, j], want)


def test_cpu_gradients_against_differences():
    ids, pos = torch.tensor([1, 3, 3, 8, 0]), torch.tensor([0, 1, 0, 1, 5])
    wte = torch.randn(5, 3, dtype=torch.float64, requires_grad=True)
    wpe = torch.randn(2, 3, dtype=torch.float64, requires_grad=True)
    assert torch.autograd.gradcheck(lambda a, b: ops.embedding(ids, a, -1.5, pos, b), (wte, wpe))


def test_cpu_accumulate_and_empty():
    out = torch.ones(4, 2)
    ops.embedding_bwd(torch.tensor([2, 2]), torch.tensor([[1.0, 2.0], [3.0, 4.0]]), 4, 0.5, out=out, accumulate=True)
    assert out.tolist() == [[1, 1], [1, 1], [3, 4], [1, 1]]
    none = torch.empty(0, dtype=torch.int64)
    assert ops.embedding_fwd(none, torch.randn(3, 2)).shape == (0, 2)
    assert (ops.embedding_bwd(none, torch.empty(0, 2), 3) == 0).all()


@pytest.mark.parametrize("call,err", [
    (lambda i, w: ops.embedding_fwd(i.int(), w), TypeError),
    (lambda i, w: ops.embedding_fwd(i, w[0]), ValueError),
    (lambda i, w: ops.embedding_fwd(i, w, positions=i), ValueError),
    (lambda i, w: ops.embedding_fwd(i, w, 1.0, i[:2], w), ValueError),
    (lambda i, w: ops.embedding_fwd(i, w, 1.0, i, w[:, :2]), ValueError),
    (lambda i, w: ops.embedding_fwd(i, w, float("inf")), ValueError),
    (lambda i, w: ops.embedding_bwd(i, w[:2], 4), ValueError),
    (lambda i, w: ops.embedding_bwd(i, w[:3], 0), ValueError),
    (lambda i, w: ops.embedding_bwd(i, w[:3], 4, accumulate=True), ValueError),
    (lambda i, w: ops.embedding_bwd(i, w[:3], 4, out=w), ValueError),
    (lambda i, w: ops.embedding_bwd(i, w[:3], 6, out=w.double()), ValueError),
])
def test_cpu_refusals(call, err):
    with pytest.raises(err):
        call(torch.tensor([0, 1, 2]), torch.randn(6, 4))


# ------------------------------------------------------------------ GPU
gpu = pytest.mark.gpu
DEV = "cuda"


def _ids(kind, T, V, gen):
    if kind == "one":
        return torch.full((T,), V // 2)
    if kind == "range":
        return torch.arange(T) % V
    if kind == "outside":
        return torch.randint(-V, 2 * V, (T,), generator=gen)
    if kind == "rank":      # frequencies that fall with the rank, as in text
        return (torch.exp(torch.rand(T, generator=gen, dtype=torch.float64) * torch.log(torch.tensor(float(V)))).long() - 1)
    return torch.randint(0, V, (T,), generator=gen)


@gpu
@pytest.mark.parametrize("kind", ["any", "one", "range", "outside", "rank"])
@pytest.mark.parametrize("T,V,H", [(1, 1, 8), (31, 7, 64), (33, 500, 512), (64, 40, 520), (1000, 300, 1024),
                                   (2048, 50304, 264), (5000, 70001, 72), (4097, 2, 2048)])
def test_gpu_forward_backward(kind, T, V, H):
    gen = torch.Generator().manual_seed(T)
    ids = _ids(kind, T, V, gen)
    wte = torch.randn(V, H, generator=gen).to(torch.bfloat16)
    dout = torch.randn(T, H, generator=gen).to(torch.bfloat16)
    out = ops.embedding_fwd(ids.to(DEV), wte.to(DEV), 3.25)
    assert torch.equal(out.cpu(), ops.embedding_fwd(ids, wte, 3.25))      # one fp32 product, one rounding
    g = ops.embedding_bwd(ids.to(DEV), dout.to(DEV), V, 3.25)
    _within(g, *_oracle_bwd(ids, dout, V, 3.25))
    again = ops.embedding_bwd(ids.to(DEV), dout.to(DEV), V, 3.25)
    assert torch.equal(g, again)


@gpu
@pytest.mark.parametrize("T,V", [(70000, 300000), (600000, 1500000)])
def test_gpu_many_tokens_and_rows(T, V):
    """More than one sort block share, three digit passes."""
    gen = torch.Generator().manual_seed(V)
    ids = torch.randint(0, V, (T,), generator=gen)
    ids[: T // 3] = 12345
    dout = torch.randn(T, 8, generator=gen).to(torch.bfloat16)
    got = ops.embedding_bwd(ids.to(DEV), dout.to(DEV), V)
    val, bound = _oracle_bwd(ids, dout, V, 1.0)
    _within(got, val, bound)


@gpu
def test_gpu_positions_shard_accumulate():
    T, V, Pn, H = 700, 1000, 64, 128
    gen = torch.Generator().manual_seed(3)
    ids, pos = torch.randint(0, V, (T,), generator=gen), torch.randint(0, Pn + 5, (T,), generator=gen)
    wte, wpe = (torch.randn(n, H, generator=gen).to(torch.bfloat16) for n in (400, Pn))
    dout = torch.randn(T, H + 8, generator=gen).to(torch.bfloat16)
    out = ops.embedding_fwd(ids.to(DEV), wte.to(DEV), 8.0, pos.to(DEV), wpe.to(DEV), vocab_start=300)
    assert torch.equal(out.cpu(), ops.embedding_fwd(ids, wte, 8.0, pos, wpe, vocab_start=300))
    base = torch.randn(400, H, generator=gen).to(torch.bfloat16)
    acc = base.to(DEV)
    ops.embedding_bwd(ids.to(DEV), dout.to(DEV)[:, 8:], 400, 8.0, out=acc, accumulate=True, vocab_start=300)
    val, bound = _oracle_bwd(ids, dout[:, 8:], 400, 8.0, 300)
    val = val + base.double()
    _within(acc, val, bound + U * val.abs())
    untouched = torch.ones(400, dtype=torch.bool)
    loc = ids - 300
    untouched[loc[(loc >= 0) & (loc < 400)]] = False
    assert torch.equal(acc.cpu()[untouched], base[untouched])


@gpu
def test_gpu_non_finite_rows_stay_in_theirs():
    ids = torch.tensor([5, 9, 5, 1, 9, 1] * 40)
    dout = torch.ones(240, 64)
    dout[ids == 9] = float("nan")
    g = ops.embedding_bwd(ids.to(DEV), dout.to(torch.bfloat16).to(DEV), 12).cpu().float()
    assert torch.isnan(g[9]).all() and (g[5] == 80).all() and (g[1] == 80).all()
    assert (g[[0, 2, 3, 4, 6, 7, 8, 10, 11]] == 0).all()


@gpu
def test_gpu_refusals():
    ids = torch.tensor([0, 1], device=DEV)
    w = torch.randn(4, 16, device=DEV, dtype=torch.bfloat16)
    for call, err in ((lambda: ops.embedding_fwd(ids, w.float()), TypeError),
                      (lambda: ops.embedding_fwd(ids, w[:, :12].contiguous()), ValueError),
                      (lambda: ops.embedding_fwd(ids, w[:, :8]), ValueError),
                      (lambda: ops.embedding_fwd(ids.cpu(), w), ValueError),
                      (lambda: ops.embedding_bwd(ids, w[:2].float(), 4), TypeError),
                      (lambda: ops.embedding_bwd(ids, w[:2], 8, out=torch.empty(8, 32, device=DEV, dtype=torch.bfloat16)[:, :16]), ValueError)):
        with pytest.raises(err):
            call()


@gpu
def test_gpu_autograd_expanded_gradient():
    ids = torch.tensor([[1, 2], [1, 0]], device=DEV)
    w = torch.randn(3, 16, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    ops.embedding(ids, w, 2.0).sum().backward()
    assert w.grad.float()[:, 0].tolist() == [2.0, 4.0, 2.0]


@gpu
def test_gpu_captured_and_replayed():
    T, V, H = 3000, 900, 256
    ids = torch.zeros(T, dtype=torch.int64, device=DEV)
    dout = torch.zeros(T, H, dtype=torch.bfloat16, device=DEV)
    w = torch.randn(V, H, device=DEV).to(torch.bfloat16)

    def go():
        return ops.embedding_fwd(ids, w, 2.0), ops.embedding_bwd(ids, dout, V, 2.0)

    def load(seed):
        gen = torch.Generator().manual_seed(seed)
        ids.copy_(torch.randint(0, V, (T,), generator=gen))
        dout.copy_(torch.randn(T, H, generator=gen))
    load(0)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        go()
    torch.cuda.current_stream().wait_stream(st)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = go()
    for seed in (1, 2, 0):
        load(seed)
        g.replay()
        torch.cuda.synchronize()
        for x, y in zip([t.clone() for t in outs], go()):
            assert torch.equal(x, y)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["any", "one", "range", "outside"])
@pytest.mark.parametrize("T", [4095, 8191, 8192, 8193])
def test_gpu_both_ways_to_sort_keep_token_order(T, kind):
    """Around the most tokens that are placed by counting; the sums are those of token order."""
    gen = torch.Generator().manual_seed(T)
    V, H = 900, 16
    ids = _ids(kind, T, V, gen).to("cuda")
    dout = torch.randn(T, H, generator=gen).to(torch.bfloat16).to("cuda")
    val, bound = _oracle_bwd(ids, dout, V, 0.75)
    first = ops.embedding_bwd(ids, dout, V, 0.75)
    _within(first, val, bound)
    assert torch.equal(first, ops.embedding_bwd(ids, dout, V, 0.75))


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_gradient_over_its_input_is_refused(device):
    ids = torch.tensor([0, 1, 0, 3], device=device)
    d = torch.ones(4, 8, dtype=torch.bfloat16, device=device)
    with pytest.raises(ValueError):
        ops.embedding_bwd(ids, d, 4, out=d)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_gradient_partly_over_its_input_is_refused(device):
    ids = torch.tensor([0, 1, 0, 3, 2, 2], device=device)
    buf = torch.ones(12, 8, dtype=torch.bfloat16, device=device)
    for out, dout in ((buf[:4], buf[3:9]), (buf[5:9], buf[:6]), (buf[:8], buf[1:7])):
        with pytest.raises(ValueError):
            ops.embedding_bwd(ids, dout, out.shape[0], out=out)
    want = ops.embedding_bwd(ids, buf[6:], 4)
    assert torch.equal(ops.embedding_bwd(ids, buf[6:], 4, out=buf[2:6]), want)


def test_shared_memory_against_a_count_of_who_touches_what():
    import random

    from mxtrain.ops import _lib
    rng, buf = random.Random(1), torch.zeros(400)

    def view():
        if rng.random() < 0.2:
            return buf[rng.randint(0, 200):][:rng.randint(1, 60)]
        ld = rng.choice((0, 8, 16, 24))
        return torch.as_strided(buf, (rng.randint(1, 6), rng.randint(1, max(ld, 8))), (ld, 1), rng.randint(0, 200))

    def cells(t):
        at = torch.zeros(400)
        torch.as_strided(at, t.shape, t.stride(), t.storage_offset()).fill_(1)
        return at
    refused = shared = 0
    for _ in range(2000):
        a, b = view(), view()
        both = bool((cells(a) * cells(b)).any())
        got = _lib.lies_over((a,), (b,))
        assert got == _lib.lies_over((a, b), ()) and got == _lib.lies_over((b,), (a,)) and (got or not both)
        refused, shared = refused + got, shared + both
    assert refused < 1.1 * shared + 50          # (ranges that only interleave are refused too)


def test_sizes_that_the_kernels_do_not_count_are_refused(monkeypatch):
    """Counts go through 32 bits: one that does not fit is named, not cut.  (No memory behind these tensors.)"""
    from mxtrain.ops import _lib
    monkeypatch.setattr(_lib, "use_hip", lambda t: True)
    e = lambda *s, dtype=torch.bfloat16: torch.empty(*s, dtype=dtype, device="meta")
    ids = lambda n: e(n, dtype=torch.int64)
    for call in (lambda: ops.embedding_fwd(ids((1 << 30) + 1), e(4, 8)),
                 lambda: ops.embedding_fwd(ids((1 << 32) + 4), e(4, 8)),
                 lambda: ops.embedding_fwd(ids(4), e((1 << 32) + 4, 8)),
                 lambda: ops.embedding_fwd(ids(4), e(4, 8), 1.0, ids(4), e((1 << 32) + 4, 8)),
                 lambda: ops.embedding_fwd(ids(4), e(4, (1 << 32) + 8))):
        with pytest.raises(ValueError, match="at most"):
            call()


@gpu
def test_gpu_lookup_of_more_tokens_than_threads_of_a_launch():
    """A wave a token: 2^26 tokens are 2^32 threads, more than one launch has."""
    T, V, H = (1 << 26) + 5, 1000, 8
    ids = torch.arange(T, device=DEV) * 7 % (V + 3)
    wte = torch.randn(V, H, device=DEV).to(torch.bfloat16)
    out = ops.embedding_fwd(ids, wte, 2.0)
    want = torch.cat([wte * 2.0, torch.zeros(3, H, dtype=torch.bfloat16, device=DEV)])
    for a, b in zip(out.split(1 << 23), ids.split(1 << 23)):
        assert torch.equal(a, want[b])


def test_gradient_sizes_that_the_kernels_do_not_count_are_refused(monkeypatch, kernel_library):
    from mxtrain.ops import _lib
    monkeypatch.setattr(_lib, "use_hip", lambda t: True)
    e = lambda *s, dtype=torch.bfloat16: torch.empty(*s, dtype=dtype, device="meta")
    ids = lambda n: e(n, dtype=torch.int64)
    for T, H, rows in (((1 << 30) + 1, 8, 4), ((1 << 32) + 4, 8, 4), (4, (1 << 32) + 8, 4),
                       (1 << 30, 8, (1 << 30) - 1)):      # (together more threads than a launch has)
        with pytest.raises(ValueError, match="more than the kernels take"):
            ops.embedding_bwd(ids(T), e(T, H), rows)


@gpu
def test_gpu_gradient_of_rows_far_apart():
    """A row stride beyond 32 bits (two rows of a buffer of 8 GiB)."""
    H, ld = 8, (1 << 32) + 8
    buf = torch.empty(ld + H, dtype=torch.bfloat16, device=DEV)
    dout = torch.as_strided(buf, (2, H), (ld, 1))
    dout.copy_(torch.tensor([[1.0], [2.0]]).expand(2, H))
    buf[H:2 * H] = 7.0
    got = ops.embedding_bwd(torch.tensor([3, 3], device=DEV), dout, 4)
    assert (got[:3] == 0).all() and (got[3] == 3.0).all()


def _in_order(keys, dout, rows, scale, order):
    """The gradient's fp32 sums, addition by addition: tokens in ``order`` (by key), 32 of them at a time,
    then the sums of a key that runs over several in order; one rounding at the end."""
    keys, d = keys[order].tolist(), dout.float()[order]
    table = torch.zeros(rows, dout.shape[1])
    t = 0
    while t < len(keys):
        end = t
        while end < len(keys) and keys[end] == keys[t]:
            end += 1
        total, e = None, t
        while e < end:
            stop = min(end, (e // 32 + 1) * 32)
            acc = torch.zeros(dout.shape[1])
            for i in range(e, stop):
                acc = acc + d[i]
            total, e = acc if total is None else total + acc, stop
        if 0 <= keys[t] < rows:
            table[keys[t]] = total * scale
        t = end
    return table.to(torch.bfloat16)


@pytest.mark.parametrize("kind", ["any", "one", "rank"])
@pytest.mark.parametrize("T,V", [(100, 7), (8192, 900), (8193, 900), (9000, 40)])
@pytest.mark.parametrize("device", [pytest.param("cuda", marks=pytest.mark.gpu), "cpu"])
def test_sums_are_those_of_token_order(device, T, V, kind):
    """Bit for bit, on values whose fp32 sum depends on the order of its terms: of a key's tokens the first is
    large, the third takes it away again, the second is lost beside it and the fourth is not, and so on.  (CPU:
    that it does.)"""
    gen = torch.Generator().manual_seed(T + V)
    H = 8
    keys = _ids(kind, T, V, gen)
    stable = torch.argsort(keys, stable=True)
    _, count = torch.unique_consecutive(keys[stable], return_counts=True)
    turn = torch.cat([torch.arange(int(n)) for n in count]) % 4
    large = 2.0 ** torch.randint(26, 30, (T, H), generator=gen)
    large[2:] = torch.where((turn[2:] == 2)[:, None], -large[:-2], large[2:])
    dout = torch.empty(T, H)
    pair = torch.zeros(T, dtype=torch.bool)          # (a first without its third stays small)
    pair[2:] = turn[2:] == 2
    pair[:-2] |= turn[2:] == 2
    dout[stable] = torch.where(pair[:, None], large, torch.rand(T, H, generator=gen) + 0.5)
    dout = dout.to(torch.bfloat16)
    want = _in_order(keys, dout, V, 0.75, stable)
    if device == "cpu":
        back = T - 1 - torch.argsort(keys.flip(0), stable=True)       # equal keys from the last to the first
        assert torch.equal(keys[back], keys[stable]) and not torch.equal(_in_order(keys, dout, V, 0.75, back), want)
        return
    got = ops.embedding_bwd(keys.to(DEV), dout.to(DEV), V, 0.75).cpu()
    assert torch.equal(got, want)
