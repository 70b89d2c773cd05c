"""64-bit oracle of the packed attention, with the elementwise error bounds its bf16 form must meet.

Bounds: the kernels hold scores, sums and statistics in fp32 and round to bf16 (half a step:
U = 2^-8 relative) P before P V and P^T dO, dS before dS K and dS^T Q, and each result once.
With F for what fp32 leaves (exponents, sums: below 2^-12 of the sum of magnitudes for the sizes
tested), and the stored o entering delta = do . o with o's own error:
  |o - o*|   <= (U + F) sum p |v| + U |o|
  |dv - dv*| <= (U + F) sum p |do| + U |dv|
  |ds - ds*| <= (U + F) |ds| + p (err_delta + F sum |do| |v|),  err_delta = sum |do| err_o
  |dq - dq*| <= scale sum err_ds |k| + U |dq|,   |dk - dk*| <= scale sum err_ds |q| + U |dk|
"""
import torch

U = 2.0 ** -8
F = 2.0 ** -12


def attention(q, k, v, lens, Hq, Hkv, D, scale, dout=None):
    """{name: (value, bound)} in float64 for o, lse (base 2) and, with dout, dq, dk, dv.  Only
    the rows and keys of each sequence are read."""
    T, g, dev = q.shape[0], Hq // Hkv, q.device
    z = lambda h: [torch.zeros(T, h * D, dtype=torch.float64, device=dev) for _ in range(2)]
    res = {"o": z(Hq), "lse": [torch.full((Hq, T), float("inf"), dtype=torch.float64, device=dev),
                               torch.zeros(Hq, T, dtype=torch.float64, device=dev)]}
    if dout is not None:
        res.update(dq=z(Hq), dk=z(Hkv), dv=z(Hkv))
    t0 = 0
    for n in lens:
        rows = slice(t0, t0 + n)
        t0 += n
        if n == 0:
            continue
        seen = torch.ones(n, n, dtype=torch.bool, device=dev).tril_()
        for h in range(Hq):
            hk = h // g
            qc, kc = slice(h * D, (h + 1) * D), slice(hk * D, (hk + 1) * D)
            Q, K, V = q[rows, qc].double(), k[rows, kc].double(), v[rows, kc].double()
            s = (Q @ K.t() * scale).masked_fill(~seen, float("-inf"))
            lse = torch.logsumexp(s, 1)
            p = torch.exp(s - lse[:, None])
            o = p @ V
            eo = (U + F) * (p @ V.abs()) + U * o.abs()
            res["o"][0][rows, qc], res["o"][1][rows, qc] = o, eo
            res["lse"][0][h, rows] = lse * 1.4426950408889634
            res["lse"][1][h, rows] = F * (1.0 + lse.abs())
            if dout is None:
                continue
            dO = dout[rows, qc].double()
            dp = dO @ V.t()
            delta = (dO * o).sum(1, keepdim=True)
            ds = p * (dp - delta)
            eds = (U + F) * ds.abs() + p * ((dO.abs() * eo).sum(1, keepdim=True) + F * (dO.abs() @ V.abs().t()))
            dq, dk, dv = scale * ds @ K, scale * ds.t() @ Q, p.t() @ dO
            res["dq"][0][rows, qc], res["dq"][1][rows, qc] = dq, scale * eds @ K.abs() + U * dq.abs()
            res["dk"][0][rows, kc] += dk
            res["dk"][1][rows, kc] += scale * eds.t() @ Q.abs()
            res["dv"][0][rows, kc] += dv
            res["dv"][1][rows, kc] += (U + F) * (p.t() @ dO.abs())
    for name in ("dk", "dv"):
        if name in res:
            res[name][1] += U * res[name][0].abs()
    return {name: tuple(t) for name, t in res.items()}


def within(got, want, name):
    """Every element of ``got`` within its bound (plus the smallest bf16 step) of the oracle."""
    val, bound = (t.to(got.device) for t in want)
    got = got.double()
    same = (got == val) | (torch.isnan(got) & torch.isnan(val))
    off = (got - val).abs() - bound - 1e-30
    bad = ~same & ~(off <= 0)
    assert not bad.any(), (f"{name}: {int(bad.sum())} of {bad.numel()} outside their bound, worst "
                           f"{float((got - val).abs()[bad].max()):.3e} (bound {float(bound[bad].max()):.3e})")
