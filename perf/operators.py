"""Workloads of the packed-batch training operators: packed causal attention, the gated
feed-forward block, and the scaled embedding with its sorted-token gradient.

A packed batch holds documents of different lengths laid end to end in one token axis;
``listed()`` names fixed cases, ``draw(rng)`` more of the same ranges.  ``run(state)`` makes one
pass: in plain torch operations (``own`` false) or through ``mxtrain.ops`` (``own`` true).
"""
from __future__ import annotations

import math
import random

import torch

own = False


# ------------------------------------------------------------------ cases
def _attn(name, tokens, mean_doc, hq, hkv, d, train, pad=0, docs_seed=1):
    return {"name": name, "op": "attention", "tokens": tokens, "mean_doc": mean_doc, "hq": hq, "hkv": hkv, "d": d,
            "train": train, "pad": pad, "docs_seed": docs_seed}


def _mlp(name, tokens, hidden, ffn, act, bias, train):
    return {"name": name, "op": "mlp", "tokens": tokens, "hidden": hidden, "ffn": ffn, "act": act, "bias": bias,
            "train": train}


def _embed(name, tokens, hidden, vocab, scale, max_pos, mean_doc, train, docs_seed=1):
    return {"name": name, "op": "embedding", "tokens": tokens, "hidden": hidden, "vocab": vocab, "scale": scale,
            "max_pos": max_pos, "mean_doc": mean_doc, "train": train, "docs_seed": docs_seed}


def listed():
    return [
        # a handful of short prompts scored in one evaluation call: latency counts
        _attn("attn_eval_short", 203, 40, 16, 16, 64, False, pad=3),
        # one GPT-2 345M micro-batch (4 x 1024 tokens) of packed documents
        _attn("attn_train_docs", 4096, 300, 16, 16, 64, True),
        # grouped heads, an odd token count and a padded end (a batch padded to a fixed size)
        _attn("attn_train_grouped", 8001, 900, 32, 8, 128, True, pad=129),
        # one long document at the GPT-3 6.7B head layout
        _attn("attn_train_long", 16384, 0, 32, 32, 128, True),
        # a single token through the GPT-2 345M block (--swiglu width), inference
        _mlp("mlp_eval_token", 1, 1024, 2688, "silu", True, False),
        # an odd number of tokens, GeLU gate, no biases
        _mlp("mlp_train_ragged", 1003, 768, 2048, "gelu", False, True),
        # one GPT-2 345M micro-batch
        _mlp("mlp_train_345m", 4096, 1024, 2688, "silu", True, True),
        # one GPT-3 6.7B micro-batch (2 x 2048 tokens)
        _mlp("mlp_train_6b7", 4096, 4096, 10880, "silu", True, True),
        # lookup alone for a short evaluation batch
        _embed("embed_eval", 1000, 1024, 50304, 1.0, 1024, 100, False),
        # GPT-2 345M micro-batch with learned positions that restart at each document
        _embed("embed_train_345m", 4096, 1024, 50304, 1.0, 1024, 300, True),
        # a long packed batch, scaled embedding, no position table
        _embed("embed_train_wide", 32768, 4096, 50304, 64.0, 0, 700, True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("attention", "mlp", "embedding"))
    if kind == "attention":
        tokens = _log_int(rng, 1, 16384)
        hq, hkv = rng.choice(((16, 16), (12, 12), (16, 4), (32, 8), (8, 1), (20, 5), (32, 32)))
        # (at most a few hundred documents: the plain form loops over them)
        c = _attn("", tokens, _log_int(rng, max(1, tokens // 128), 4096), hq, hkv, rng.choice((64, 128)), rng.random() < 0.7,
                  pad=rng.choice((0, 0, rng.randint(0, tokens // 2))), docs_seed=rng.randint(1, 1 << 20))
    elif kind == "mlp":
        tokens = _log_int(rng, 1, 4096)
        step = rng.choice((8, 64, 128))
        hidden = _log_int(rng, 256, 4096) // step * step
        ffn = _log_int(rng, 256, 10880) // step * step
        c = _mlp("", tokens, hidden, ffn, rng.choice(("silu", "gelu")), rng.random() < 0.6,
                 tokens > 1 and rng.random() < 0.7)
    else:
        c = _embed("", _log_int(rng, 1, 32768), _log_int(rng, 64, 4096) // 8 * 8, _log_int(rng, 100, 50304),
                   rng.choice((1.0, 8.0, 45.25, 64.0)), rng.choice((0, 1024, 2048)), _log_int(rng, 1, 4096),
                   rng.random() < 0.7, docs_seed=rng.randint(1, 1 << 20))
    del c["name"]
    return c


def _lengths(tokens, mean_doc, docs_seed, longest):
    """Document lengths that fill ``tokens`` exactly (exponential around ``mean_doc``; 0 = one document)."""
    if mean_doc <= 0:
        return [tokens] if tokens else []
    rng = random.Random(docs_seed)
    out, left = [], tokens
    while left > 0:
        n = min(left, longest, max(1, int(rng.expovariate(1.0 / mean_doc) + 0.5)))
        out.append(n)
        left -= n
    return out


def _attn_lengths(case):
    return _lengths(case["tokens"] - case["pad"], case["mean_doc"], case["docs_seed"], case["tokens"])


def _positions(case):
    lens = _lengths(case["tokens"], case["mean_doc"], case["docs_seed"], case["max_pos"])
    return torch.cat([torch.arange(n) for n in lens])


# ------------------------------------------------------------------ inputs
def _randn(gen, *shape, std=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32) * std).to(torch.bfloat16)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    st = {"case": case}
    T = case["tokens"]
    if case["op"] == "attention":
        hq, hkv, d = case["hq"], case["hkv"], case["d"]
        st["lens"] = lens = _attn_lengths(case)
        # q, k, v are column ranges of the packed projection output, read in place
        qkv = _randn(gen, T, (hq + 2 * hkv) * d)
        st["q"], st["k"], st["v"] = qkv[:, :hq * d], qkv[:, hq * d:(hq + hkv) * d], qkv[:, (hq + hkv) * d:]
        st["dout"] = _randn(gen, T, hq * d) if case["train"] else None
        if own:
            from mxtrain import ops
            cu = torch.tensor([0] + lens, dtype=torch.int64).cumsum(0)
            st["seqs"] = ops.pack_sequences(cu, T, device="cuda")
    elif case["op"] == "mlp":
        h, f = case["hidden"], case["ffn"]
        st["x"] = _randn(gen, T, h)
        st["w1"] = _randn(gen, 2 * f, h, std=h ** -0.5)
        st["w2"] = _randn(gen, h, f, std=f ** -0.5)
        st["b1"] = _randn(gen, 2 * f, std=0.1) if case["bias"] else None
        st["b2"] = _randn(gen, h, std=0.1) if case["bias"] else None
        st["dy"] = _randn(gen, T, h) if case["train"] else None
    else:
        V, h = case["vocab"], case["hidden"]
        # token frequencies fall with the rank, as in text (log-uniform ranks)
        u = torch.rand(T, generator=gen, device="cuda", dtype=torch.float64)
        st["ids"] = (torch.exp(u * math.log(V)).long() - 1).clamp_(0, V - 1)
        st["wte"] = _randn(gen, V, h, std=0.02)
        st["pos"] = st["wpe"] = None
        if case["max_pos"]:
            st["pos"] = _positions(case).cuda()
            st["wpe"] = _randn(gen, case["max_pos"], h, std=0.02)
        st["dout"] = _randn(gen, T, h) if case["train"] else None
    return st


# ------------------------------------------------------------------ one pass
def run(state):
    op = state["case"]["op"]
    if op == "attention":
        return _run_attention(state)
    if op == "mlp":
        return _run_mlp(state)
    return _run_embedding(state)


def _run_attention(st):
    c = st["case"]
    q, k, v, dout = st["q"], st["k"], st["v"], st["dout"]
    hq, hkv, d = c["hq"], c["hkv"], c["d"]
    if own:
        from mxtrain import ops
        o, lse = ops.packed_attn_fwd(q, k, v, st["seqs"], hq, hkv, d)
        if dout is None:
            return {"o": o}
        dq, dk, dv = ops.packed_attn_bwd(dout, q, k, v, o, lse, st["seqs"], hq, hkv, d)
        return {"o": o, "dq": dq, "dk": dk, "dv": dv}
    T, g, scale = c["tokens"], hq // hkv, d ** -0.5
    out = {"o": torch.zeros(T, hq * d, dtype=q.dtype, device=q.device)}
    if dout is not None:
        out["dq"] = torch.zeros(T, hq * d, dtype=q.dtype, device=q.device)
        out["dk"] = torch.zeros(T, hkv * d, dtype=q.dtype, device=q.device)
        out["dv"] = torch.zeros(T, hkv * d, dtype=q.dtype, device=q.device)
    t0 = 0
    for n in st["lens"]:
        rows = slice(t0, t0 + n)
        t0 += n
        above = torch.ones(n, n, dtype=torch.bool, device=q.device).triu_(1)
        step = hkv if n <= 2048 else 1      # key heads at a time: bounds the score matrix
        for j in range(0, hkv, step):
            qc, kc = slice(j * g * d, (j + step) * g * d), slice(j * d, (j + step) * d)
            qs = q[rows, qc].float().view(n, step, g, d).permute(1, 2, 0, 3)        # [step, g, n, d]
            ks = k[rows, kc].float().view(n, step, 1, d).permute(1, 2, 0, 3)
            vs = v[rows, kc].float().view(n, step, 1, d).permute(1, 2, 0, 3)
            s = torch.matmul(qs, ks.transpose(-1, -2)).mul_(scale).masked_fill_(above, float("-inf"))
            p = torch.exp(s.sub_(s.amax(-1, keepdim=True)))
            del s
            p /= p.sum(-1, keepdim=True)
            o = torch.matmul(p, vs)
            out["o"][rows, qc] = o.permute(2, 0, 1, 3).reshape(n, -1).to(q.dtype)
            if dout is None:
                continue
            do = dout[rows, qc].float().view(n, step, g, d).permute(1, 2, 0, 3)
            dv = torch.matmul(p.transpose(-1, -2), do).sum(1)
            ds = torch.matmul(do, vs.transpose(-1, -2)).sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
            del p
            dq = torch.matmul(ds, ks)
            dk = torch.matmul(ds.transpose(-1, -2), qs).sum(1)
            out["dq"][rows, qc] = dq.permute(2, 0, 1, 3).reshape(n, -1).to(q.dtype)
            out["dk"][rows, kc] = dk.permute(1, 0, 2).reshape(n, -1).to(q.dtype)
            out["dv"][rows, kc] = dv.permute(1, 0, 2).reshape(n, -1).to(q.dtype)
    return out


def _run_mlp(st):
    c = st["case"]
    x, w1, b1, w2, b2, dy = st["x"], st["w1"], st["b1"], st["w2"], st["b2"], st["dy"]
    if own:
        from mxtrain import ops
        y, pre, h = ops.gated_mlp_fwd(x, w1, b1, w2, b2, act=c["act"], save=dy is not None)
        if dy is None:
            return {"y": y}
        dx, dw1, db1, dw2, db2 = ops.gated_mlp_bwd(dy, x, pre, h, w1, b1, w2, b2, act=c["act"])
        out = {"y": y, "dx": dx, "dw1": dw1, "dw2": dw2}
        if b1 is not None:
            out["db1"], out["db2"] = db1, db2
        return out
    f, dt = c["ffn"], x.dtype
    xf, w1f, w2f = x.float(), w1.float(), w2.float()
    pre = torch.matmul(xf, w1f.t())
    if b1 is not None:
        pre += b1.float()
    a, b = pre[:, :f], pre[:, f:]
    if c["act"] == "silu":
        sg = 1.0 / (1.0 + torch.exp(-a))
        ga, dga = a * sg, None if dy is None else sg * (1.0 + a * (1.0 - sg))
    else:
        k0, k1 = math.sqrt(2.0 / math.pi), 0.044715
        th = torch.tanh(k0 * (a + k1 * a * a * a))
        ga = 0.5 * a * (1.0 + th)
        dga = None if dy is None else 0.5 * (1.0 + th) + 0.5 * a * (1.0 - th * th) * k0 * (1.0 + 3.0 * k1 * a * a)
    h = ga * b
    y = torch.matmul(h, w2f.t())
    if b2 is not None:
        y += b2.float()
    if dy is None:
        return {"y": y.to(dt)}
    dyf = dy.float()
    dh = torch.matmul(dyf, w2f)
    dpre = torch.cat([dh * b * dga, dh * ga], 1)
    out = {"y": y.to(dt), "dx": torch.matmul(dpre, w1f).to(dt), "dw1": torch.matmul(dpre.t(), xf).to(dt),
           "dw2": torch.matmul(dyf.t(), h).to(dt)}
    if b1 is not None:
        out["db1"], out["db2"] = dpre.sum(0).to(dt), dyf.sum(0).to(dt)
    return out


def _run_embedding(st):
    c = st["case"]
    ids, wte, pos, wpe, dout = st["ids"], st["wte"], st["pos"], st["wpe"], st["dout"]
    if own:
        from mxtrain import ops
        out = {"out": ops.embedding_fwd(ids, wte, c["scale"], pos, wpe)}
        if dout is not None:
            out["dwte"] = ops.embedding_bwd(ids, dout, wte.shape[0], c["scale"])
            if wpe is not None:
                out["dwpe"] = ops.embedding_bwd(pos, dout, wpe.shape[0])
        return out
    e = wte[ids].float() * c["scale"]
    if wpe is not None:
        e += wpe[pos].float()
    out = {"out": e.to(wte.dtype)}
    if dout is not None:
        df = dout.float()
        acc = torch.zeros(wte.shape, dtype=torch.float32, device=wte.device)
        out["dwte"] = acc.index_add_(0, ids, df).mul_(c["scale"]).to(wte.dtype)
        if wpe is not None:
            acc = torch.zeros(wpe.shape, dtype=torch.float32, device=wte.device)
            out["dwpe"] = acc.index_add_(0, pos, df).to(wpe.dtype)
    return out


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    T, train = case["tokens"], case["train"]
    if case["op"] == "attention":
        hq, hkv, d = case["hq"], case["hkv"], case["d"]
        lens = _attn_lengths(case)
        rows, pairs = sum(lens), sum(n * (n + 1) // 2 for n in lens)
        flops = (14 if train else 4) * d * hq * pairs
        # q, k, v in, o out; training: dout in, dq, dk, dv out
        width = (2 * hq + 2 * hkv) * d + ((2 * hq + 2 * hkv) * d if train else 0)
        return {"bytes": 2 * rows * width, "flops": flops}
    if case["op"] == "mlp":
        h, f = case["hidden"], case["ffn"]
        weights = 3 * h * f + ((2 * f + h) if case["bias"] else 0)
        return {"bytes": 2 * (weights * (2 if train else 1) + T * h * (4 if train else 2)),
                "flops": (18 if train else 6) * T * h * f}
    h, V, P = case["hidden"], case["vocab"], case["max_pos"]
    # table rows touched: the expected distinct ids of T draws, and the positions of the longest document
    logs = [math.log(i + 1) for i in range(V + 1)]
    rows = sum(-math.expm1(T * math.log1p(-min((logs[i + 1] - logs[i]) / math.log(V), 1.0 - 1e-12)))
               for i in range(V - 1))
    if P:
        rows += max(_lengths(T, case["mean_doc"], case["docs_seed"], P))
    n = 2 * h * (int(rows) + T) + 8 * T * (2 if P else 1)
    if train:
        n += 2 * h * (T + V + P)
    return {"bytes": n, "flops": (2 + (2 if train else 0)) * T * h}


# ------------------------------------------------------------------ from the definitions, in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(case, st)
    if case["op"] == "mlp":
        return _exact_mlp(case, st)
    return _exact_embedding(case, st)


def _exact_attention(case, st):
    hq, hkv, d, T = case["hq"], case["hkv"], case["d"], case["tokens"]
    group = hq // hkv
    q, k, v = (st[n].double().view(T, -1, d) for n in ("q", "k", "v"))
    do = st["dout"].double().view(T, hq, d) if case["train"] else None
    res = {"o": torch.zeros_like(q)}
    if do is not None:
        res.update(dq=torch.zeros_like(q), dk=torch.zeros_like(k), dv=torch.zeros_like(v))
    bounds = [0]
    for n in st["lens"]:
        bounds.append(bounds[-1] + n)
    for lo, hi in zip(bounds[:-1], bounds[1:]):
        seen = torch.arange(hi - lo, device=q.device)
        seen = seen[None, :] <= seen[:, None]
        for head in range(hq):
            leaves = [q[lo:hi, head], k[lo:hi, head // group], v[lo:hi, head // group]]
            leaves = [t.clone().requires_grad_(do is not None) for t in leaves]
            score = leaves[0] @ leaves[1].mT / math.sqrt(d)
            prob = torch.softmax(torch.where(seen, score, -math.inf), dim=1)
            ctx = prob @ leaves[2]
            res["o"][lo:hi, head] = ctx.detach()
            if do is not None:
                gq, gk, gv = torch.autograd.grad(ctx, leaves, do[lo:hi, head])
                res["dq"][lo:hi, head] = gq
                res["dk"][lo:hi, head // group] += gk
                res["dv"][lo:hi, head // group] += gv
            del score, prob, ctx
    return {name: t.reshape(T, -1) for name, t in res.items()}


def _exact_mlp(case, st):
    names = [n for n in ("x", "w1", "w2", "b1", "b2") if st[n] is not None]
    leaf = {n: st[n].double().requires_grad_(case["train"]) for n in names}
    gate, up = (leaf["x"] @ part.mT for part in leaf["w1"].chunk(2))
    if case["bias"]:
        bg, bu = leaf["b1"].chunk(2)
        gate, up = gate + bg, up + bu
    if case["act"] == "silu":
        hid = gate * torch.sigmoid(gate) * up
    else:
        hid = gate * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (gate + 0.044715 * gate ** 3)) * up
    y = hid @ leaf["w2"].mT
    if case["bias"]:
        y = y + leaf["b2"]
    if not case["train"]:
        return {"y": y}
    grads = torch.autograd.grad(y, [leaf[n] for n in names], st["dy"].double())
    got = {"d" + n: g for n, g in zip(names, grads)}
    return {"y": y.detach(), **{n: got[n] for n in ("dx", "dw1", "dw2", "db1", "db2") if n in got}}


def _exact_embedding(case, st):
    ids, pos, dout = st["ids"], st["pos"], st["dout"]
    e = st["wte"].double().index_select(0, ids) * case["scale"]
    if pos is not None:
        e = e + st["wpe"].double().index_select(0, pos)
    res = {"out": e}
    if dout is None:
        return res

    def rows_summed(keys, n):
        # rows in the order of their keys; the sum of a run is a difference of prefix sums,
        # taken a column block at a time (64 bits: the prefixes stay far below 2^53 steps)
        order = torch.argsort(keys)
        ends = torch.searchsorted(keys[order], torch.arange(n + 1, device=keys.device))
        cols = []
        for c0 in range(0, dout.shape[1], 256):
            run_sum = dout[order, c0:c0 + 256].double().cumsum(0)
            run_sum = torch.cat([run_sum.new_zeros(1, run_sum.shape[1]), run_sum])
            cols.append(run_sum[ends[1:]] - run_sum[ends[:-1]])
        return torch.cat(cols, 1)

    res["dwte"] = rows_summed(ids, case["vocab"]) * case["scale"]
    if pos is not None:
        res["dwpe"] = rows_summed(pos, case["max_pos"])
    return res
