"""A packed decoder layer -- scaled embedding with restarting positions, RMSNorm, packed attention
with grouped heads, gated feed-forward block, loss -- built from the public ops, forward and
backward, as a training step runs them."""
import pytest
import torch

from mxtrain import ops

HQ, HKV, D, F, V, P = 4, 2, 64, 704, 501, 300
H = HQ * D


def _params(dtype, device):
    gen = torch.Generator().manual_seed(11)

    def r(*s, std):
        return (torch.randn(*s, generator=gen, dtype=torch.float64) * std).to(torch.bfloat16).to(dtype).to(device).requires_grad_(True)
    return {"wte": r(V, H, std=0.05), "wpe": r(P, H, std=0.05), "g1": r(H, std=1.0), "g2": r(H, std=1.0),
            "q": r(HQ * D, H, std=H ** -0.5), "k": r(HKV * D, H, std=H ** -0.5), "v": r(HKV * D, H, std=H ** -0.5),
            "o": r(H, HQ * D, std=H ** -0.5), "w1": r(2 * F, H, std=H ** -0.5), "b1": r(2 * F, std=0.1),
            "w2": r(H, F, std=F ** -0.5), "b2": r(H, std=0.1)}


def _layer(p, ids, cu, total):
    s = ops.pack_sequences(cu, total, device=ids.device)
    h = ops.embedding(ids, p["wte"], 8.0, s.positions, p["wpe"])
    a = ops.rms_norm(h, p["g1"]) if ids.is_cuda else _rms(h, p["g1"])
    q, k, v = (torch.mm(a, p[n].t()) for n in ("q", "k", "v"))
    h = h + torch.mm(ops.packed_attention(q, k, v, s, HQ, HKV, D), p["o"].t())
    m = ops.rms_norm(h, p["g2"]) if ids.is_cuda else _rms(h, p["g2"])
    return h + ops.gated_mlp(m, p["w1"], p["b1"], p["w2"], p["b2"])


def _rms(x, g, eps=1e-6):
    return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps) * g


def _batch(lens, pad):
    gen = torch.Generator().manual_seed(5)
    T = sum(lens) + pad
    ids = torch.randint(0, V, (T,), generator=gen)
    return ids, torch.tensor([0] + lens).cumsum(0), T, torch.randn(T, H, generator=gen).to(torch.bfloat16)


def _step(p, ids, cu, T, g):
    out = _layer(p, ids, cu, T)
    return out, dict(zip(p, torch.autograd.grad(out, list(p.values()), g)))


def test_cpu_documents_match_one_by_one():
    """The packed layer equals the layer run on each document alone (float64)."""
    lens = [7, 1, 20, 0, 12]
    ids, cu, T, g = _batch(lens, 0)
    p = _params(torch.float64, "cpu")
    out, grads = _step(p, ids, cu, T, g.double())
    total = {n: torch.zeros_like(t) for n, t in p.items()}
    for a, b in zip(cu[:-1].tolist(), cu[1:].tolist()):
        if a == b:
            continue
        o, gr = _step(p, ids[a:b], torch.tensor([0, b - a]), b - a, g[a:b].double())
        torch.testing.assert_close(out[a:b], o, rtol=1e-9, atol=1e-10)
        for n in total:
            total[n] += gr[n]
    for n in total:
        torch.testing.assert_close(grads[n], total[n], rtol=1e-8, atol=1e-9)


@pytest.mark.gpu
def test_gpu_layer_matches_float64():
    """Relative error (2-norm) of the output and every gradient.  About 12 roundings to bf16 lie on
    the way to an output and 24 to a gradient, each at most half a step (2^-8) of what it rounds;
    the layer's maps neither amplify nor cancel more than the residual stream they feed."""
    ids, cu, T, g = _batch([150, 1, 300, 0, 33, 90], 26)
    p64, p = _params(torch.float64, "cpu"), _params(torch.bfloat16, "cuda")
    g[574:] = 0          # no loss on the rows behind the last document
    want, wg = _step(p64, ids, cu, T, g.double())
    out, grads = _step(p, ids.cuda(), cu, T, g.cuda())
    err = lambda a, b: float((a.double().cpu() - b).norm() / b.norm())
    assert err(out[:574], want[:574]) < 12 * 2.0 ** -8
    for n in wg:
        assert err(grads[n], wg[n]) < 24 * 2.0 ** -8, (n, err(grads[n], wg[n]))


@pytest.mark.gpu
def test_gpu_documents_do_not_see_each_other():
    """Replacing one document leaves every other document's output bit for bit as it was."""
    lens = [100, 64, 200, 50]
    ids, cu, T, _ = _batch(lens, 0)
    p = {n: t.detach() for n, t in _params(torch.bfloat16, "cuda").items()}
    a = _layer(p, ids.cuda(), cu, T)
    ids[100:164] = (ids[100:164] + 17) % V
    b = _layer(p, ids.cuda(), cu, T)
    assert torch.equal(a[:100], b[:100]) and torch.equal(a[164:], b[164:])
    assert not torch.equal(a[100:164], b[100:164])


@pytest.mark.gpu
def test_gpu_captured_training_step():
    """The whole step, row table included, in a graph: replays with new documents match eager ones."""
    p = _params(torch.bfloat16, "cuda")
    T = 300
    ids = torch.zeros(T, dtype=torch.int64, device="cuda")
    cu = torch.zeros(4, dtype=torch.int64, device="cuda")
    g = torch.zeros(T, H, dtype=torch.bfloat16, device="cuda")

    def load(lens):
        i, c, _, gr = _batch(lens, T - sum(lens))
        ids.copy_(i)
        cu.copy_(c)
        g.copy_(gr)
        g[sum(lens):] = 0
    load([100, 120, 60])
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        _step(p, ids, cu, T, g)
    torch.cuda.current_stream().wait_stream(st)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, grads = _step(p, ids, cu, T, g)
    for lens in ([1, 2, 290], [300, 0, 0], [50, 100, 150]):
        load(lens)
        graph.replay()
        torch.cuda.synchronize()
        got, gg = out.detach().clone(), {n: t.clone() for n, t in grads.items()}
        want, wg = _step(p, ids, cu, T, g)
        n = sum(lens)
        assert torch.equal(got[:n], want.detach()[:n])
        for k in wg:
            assert torch.equal(gg[k], wg[k]), k
