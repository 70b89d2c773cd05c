"""Gated feed-forward block (``csrc/gated.hip``) + reference:

    pre = x W1^T + b1 = [a | b],  h = act(a) * b,  y = h W2^T + b2        act "silu" or "gelu" (tanh)

The two projections, the activation and the product are one kernel; backward recomputes nothing
but the activation: it needs the ``pre`` and ``h`` that forward saves.  W1 is [2F, H] with the gate
half first (the layout of ``bias_swiglu_fwd`` and the GPT model's fc1), W2 [Ho, F].

On the GPU: bfloat16, feature counts that are multiples of 8, up to 1048560 tokens; rows may be
strided.  Products accumulate in fp32; ``pre``, ``h`` and every result are rounded once to bf16.
"""
from __future__ import annotations

import math

import torch

from . import _lib
from .norm import colsum, colsum_finalize, colsum_partials_buffer

ACTS = {"silu": 0, "gelu": 1}
MAX_TOKENS = 16 * 65535     # grid rows of the column-sum kernel


def _acc(t):   # at least float32
    return t.double() if t.dtype == torch.float64 else t.float()


def _act(name, a):
    if name == "silu":
        s = torch.sigmoid(a)
        return a * s, s * (1.0 + a * (1.0 - s))
    k0, k1 = math.sqrt(2.0 / math.pi), 0.044715
    t = torch.tanh(k0 * (a + k1 * a * a * a))
    return 0.5 * a * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * a * (1.0 - t * t) * k0 * (1.0 + 3.0 * k1 * a * a)


# ------------------------------------------------------------------ checks
def _ld(t):
    """Row stride (a single row has none: its width)."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _readable(t):
    return t.stride(1) == 1 and _ld(t) % 8 == 0 and t.shape[1] <= _ld(t) <= 1 << 21 and t.data_ptr() % 16 == 0


def _check(name, act, x, w1, b1, w2, b2, **more):
    """``more``: tensor -> expected shape.  Returns (T, H, F, Ho, hip)."""
    if act not in ACTS:
        raise ValueError(f"{name}: act must be one of {sorted(ACTS)}, got {act!r}")
    if x.dim() != 2 or w1.dim() != 2 or w2.dim() != 2:
        raise ValueError(f"{name}: x, w1 and w2 must be 2-D")
    T, H = x.shape
    Ho, F = w2.shape
    if H == 0 or F == 0 or Ho == 0:
        raise ValueError(f"{name}: features must not be empty")
    shapes = {"x": (x, (T, H)), "w1": (w1, (2 * F, H)), "w2": (w2, (Ho, F)), "b1": (b1, (2 * F,)), "b2": (b2, (Ho,))}
    shapes.update({k: (t, s(T, H, F, Ho)) for k, (t, s) in more.items()})
    hip = _lib.use_hip(x)
    if hip:
        if H % 8 or F % 8 or Ho % 8 or max(H, 2 * F, Ho) > 1 << 20:
            raise ValueError(f"{name}: the GPU kernels take features that are multiples of 8 (at most 2^20), got "
                             f"{H}, {F}, {Ho}")
        if T > MAX_TOKENS:
            raise ValueError(f"{name}: at most {MAX_TOKENS} tokens, got {T}")
    for key, (t, shape) in shapes.items():
        if t is None:
            continue
        if tuple(t.shape) != shape:
            raise ValueError(f"{name}: {key} must be {list(shape)}, got {list(t.shape)}")
        if t.device != x.device:
            raise ValueError(f"{name}: {key} is on {t.device}, x on {x.device}")
        if t.dtype != x.dtype:
            raise TypeError(f"{name}: {key} is {t.dtype}, x is {x.dtype}")
        if not hip:
            continue
        if t.dtype != torch.bfloat16:
            raise TypeError(f"{name}: the GPU kernels take bfloat16, {key} is {t.dtype}")
        flat = key in ("pre", "h", "b1", "b2", "db1", "db2")
        if t.numel() and (t.data_ptr() % 16 or (not t.is_contiguous() if flat else not _readable(t))):
            raise ValueError(f"{name}: {key} must be 16-byte aligned and " + (
                "contiguous" if flat else "have unit column stride and a row stride that is a multiple of 8"))
    return T, H, F, Ho, hip


def _mats(act, x, w1, b1, w2, b2):
    """Sizes, (address, row stride) of x, w1, w2 and the bias addresses of a valid GPU call, or None:
    a CPU call, no tokens, or a call whose fault :func:`_check` names."""
    if act not in ACTS or not _lib.use_hip(x) or x.dim() != 2 or w2.dim() != 2:
        return None
    (T, H), (Ho, F) = x.shape, w2.shape
    if (H | F | Ho) % 8 or not 0 < T <= MAX_TOKENS or max(H, 2 * F, Ho) > 1 << 20 or not H or not F or not Ho:
        return None
    dev = x.get_device()
    mats = [_lib.rows_of(t, r, c, dev, 1 << 21) for t, r, c in ((x, T, H), (w1, 2 * F, H), (w2, Ho, F))]
    if None in mats:
        return None
    for b, n in ((b1, 2 * F), (b2, Ho)):
        p = None
        if b is not None:
            p = b.data_ptr()
            if b.dtype is not torch.bfloat16 or b.shape != (n,) or b.get_device() != dev or not b.is_contiguous() \
                    or p % 16:
                return None
        mats.append(p)
    return (T, H, F, Ho), *mats


# ------------------------------------------------------------------ tiles
# Per tile of csrc/gated.hip: rows, columns, workgroups per CU; us per 64-deep step, the same of a
# workgroup alone on its CU; us per round of workgroups (one on every slot of the 256 CUs) beside the
# steps, more of it where the epilogue reads and writes as much as the gate gradient's, and once.
# Fitted to one MI355X over 4096 x 4096 x 10880 (steps), 4096 x 1024 x 2688 (rounds) and, the small
# tile, 1003 x 768 x 2048 and 300 x 512 x 1376.  Of 85 picks (five products of three of these and of
# 14 other shapes of 73 .. 3808 tokens) 71 were the fastest and 76 within 5 % of it; the worst took 17 % longer
# (453 x 504 x 1960 "down", two splits for four).
_TILES = ((128, 128, 2, 1.14, 0.97, 5.0, 3.5, 0.0), (256, 256, 1, 1.72, 1.72, 5.0, 30.0, 0.0),
          (128, 128, 1, 0.62, 0.62, 4.0, 4.2, 0.0),
          (256, 128, 1, 0.985, 0.985, 5.0, 7.5, 0.0), (64, 128, 2, 0.57, 0.45, 2.5, 3.6, 6.0))
_DW_TILES = 4          # (the last one does not take operands whose rows are the contraction)
_PLANS = {}


def _estimate(tile, wgs, steps, kind=""):
    """us of ``wgs`` workgroups of ``steps`` 64-deep steps each."""
    _, _, per, step, alone, fix, more, once = _TILES[tile]
    if wgs <= 256:
        step, once = alone, once / 4
    return -(-wgs // (256 * per)) * (steps * step + fix + (more if kind == "dgate" else 0.0)) + once


def _count(tile, M, N):
    bm, bn = _TILES[tile][:2]
    return -(-M // bm) * -(-N // bn)


def _plan(kind, M, N, K):
    """(tile, splits, us) of one product, M x N over K (N: columns of both halves for "gate"): the
    least estimated time.  Big tiles move the fewest operand bytes per product, so they win where
    they fill whole rounds (4096 x 4096 x 10880 "down": 298 us with 256 x 256 tiles, 387 with 128 x
    128); few tiles leave CUs idle, so smaller ones with a deeper ring win (1003 x 768 x 2048 "gate":
    12.6 us against 24.9), and a long K is split once the tiles cover less than half of the chip
    (its "dx": 21.2 us in 4 splits, 40 us in one).  Tiles of 64 rows, two workgroups a CU, run one's
    epilogue beside the other's loop, which the gate gradient gains from most (4096 x 1024 x 2688: 51
    us, 55 with 128 x 128, 62 with 256 x 256; 700 x 2048 x 5504: 30 and 42), and short batches (700 x
    2048 x 5504 "gate": 49 and 58).  Each product by itself, again and again; in a pass of the block they
    find less in the caches (gate gradient of 4096 x 1024 x 2688: 56)."""
    key = (kind, M, N, K)
    best = _PLANS.get(key)
    if best is None:
        if kind in ("gate", "down") and _lib.query("mx_gated_few", M, K, N // 2 if kind == "gate" else N):
            best = (0, 1, 0.0)       # (not looked at)
        steps = -(-K // 64)
        for tile in range(0 if best else _DW_TILES if kind == "dw" else len(_TILES)):
            tiles = _count(tile, M, N)
            for splits in ((1, 2, 4, 8) if kind in ("down", "dx", "dw") else (1,)):
                if splits > 1 and (tiles * splits > 256 or steps < 8 * splits):
                    break
                est = _estimate(tile, tiles * splits, -(-steps // splits), kind)
                if splits > 1:                   # partials written and read, one more launch
                    est += 4.0 + splits * M * N * 8 / 4e6
                if best is None or est < best[2]:
                    best = (tile, splits, est)
        _keep(key, best)
    return best


def _plan_pair(T, H, F, Ho):
    """The tile of both weight gradients in one launch, or None where two are faster: together they
    leave one round of workgroups unfilled, not two (4096 x 1024 x 2688: 65 us, apart 98; 4096 x 4096 x
    10880: 905 and 977; 2048 x 2048 x 5504 fills its rounds: 155 and 157; as in :func:`_plan`, by
    themselves: in a pass of the block 72 and 990)."""
    key = ("pair", T, H, F, Ho)
    plan = _PLANS.get(key)      # (one look: another thread may clear the table at any time)
    if plan is None:
        best, cost = None, _plan("dw", 2 * F, H, T)[2] + _plan("dw", Ho, F, T)[2] + 2.0
        for tile in range(_DW_TILES):
            est = _estimate(tile, _count(tile, 2 * F, H) + _count(tile, Ho, F), -(-T // 64))
            if est < cost:
                best, cost = tile, est
        plan = (best, cost)
        _keep(key, plan)
    return plan[0]


def _keep(key, plan):
    if len(_PLANS) > 4096:
        _PLANS.clear()
    _PLANS[key] = plan


def _split_ws(splits, M, N, device):
    return torch.empty(splits * M * N, dtype=torch.float32, device=device) if splits > 1 else None


# ------------------------------------------------------------------ forward / backward
def gated_mlp_fwd(x, w1, b1, w2, b2, act: str = "silu", save: bool = True):
    """x [T, H] -> (y [T, Ho], pre [T, 2F], h [T, F]); without ``save`` the last two are None.
    Biases may be None."""
    m = _mats(act, x, w1, b1, w2, b2)
    if m is None:
        T, H, F, Ho, hip = _check("gated_mlp_fwd", act, x, w1, b1, w2, b2)
        if hip and T:
            raise ValueError("gated_mlp_fwd: unsupported arguments")
        pre = _acc(x) @ _acc(w1).t()
        if b1 is not None:
            pre = pre + _acc(b1)
        h = _act(act, pre[:, :F])[0] * pre[:, F:]
        y = h @ _acc(w2).t()
        if b2 is not None:
            y = y + _acc(b2)
        y = y.to(x.dtype)
        return (y, pre.to(x.dtype), h.to(x.dtype)) if save else (y, None, None)
    (T, H, F, Ho), (x_, ldx), (w1_, ld1), (w2_, ld2), b1_, b2_ = m
    with _lib.on_device(x):
        y = torch.empty(T, Ho, dtype=x.dtype, device=x.device)
        h = torch.empty(T, F, dtype=x.dtype, device=x.device)
        pre = torch.empty(T, 2 * F, dtype=x.dtype, device=x.device) if save else None
        tile, splits, _ = _plan("down", T, Ho, F)
        part = _split_ws(splits, T, Ho, x.device)
        _lib.call("mx_gated_fwd", x_, ldx, w1_, ld1, b1_, _lib.ptr(pre), h.data_ptr(), w2_, ld2, b2_, y.data_ptr(), T,
                  H, F, Ho, ACTS[act], _plan("gate", T, 2 * F, H)[0], tile, splits, _lib.ptr(part), _lib.stream())
    return (y, pre, h) if save else (y, None, None)


def gated_mlp_bwd(dy, x, pre, h, w1, b1, w2, b2, act: str = "silu", dw1=None, db1=None, dw2=None, db2=None,
                  accumulate: bool = False, need_dx: bool = True, need_dw: bool = True):
    """(dx, dw1, db1, dw2, db2) from the saved ``pre`` and ``h``.  Given gradient buffers are
    written, or added to with ``accumulate`` (then all of them must be given); bias gradients are
    None where the bias is.  ``need_dx`` / ``need_dw``: skip dx / the parameter gradients."""
    name = "gated_mlp_bwd"
    if pre is None or h is None:
        raise ValueError(f"{name}: forward must have been called with save=True")
    if (b1 is None and db1 is not None) or (b2 is None and db2 is not None):
        raise ValueError(f"{name}: a bias gradient without its bias")
    if accumulate and need_dw and (dw1 is None or dw2 is None or (b1 is not None and db1 is None)
                                   or (b2 is not None and db2 is None)):
        raise ValueError(f"{name}: accumulate needs the gradient buffers")
    T, H, F, Ho, hip = _check(
        name, act, x, w1, b1, w2, b2, dy=(dy, lambda T, H, F, O: (T, O)), pre=(pre, lambda T, H, F, O: (T, 2 * F)),
        h=(h, lambda T, H, F, O: (T, F)), dw1=(dw1, lambda T, H, F, O: (2 * F, H)),
        db1=(db1, lambda T, H, F, O: (2 * F,)), dw2=(dw2, lambda T, H, F, O: (O, F)),
        db2=(db2, lambda T, H, F, O: (O,)))
    if need_dw:
        out = [t for t in (dw1, db1, dw2, db2) if t is not None]
        if T and out and _lib.lies_over(out, (dy, x, pre, h)):
            raise ValueError(f"{name}: gradient buffers must not lie over each other, nor over dy, x, pre or h")
        new = torch.zeros if T == 0 else torch.empty
        given = {k: t is not None for k, t in (("dw1", dw1), ("db1", db1), ("dw2", dw2), ("db2", db2))}
        dw1 = dw1 if given["dw1"] else new(2 * F, H, dtype=x.dtype, device=x.device)
        dw2 = dw2 if given["dw2"] else new(Ho, F, dtype=x.dtype, device=x.device)
        if b1 is not None and db1 is None:
            db1 = new(2 * F, dtype=x.dtype, device=x.device)
        if b2 is not None and db2 is None:
            db2 = new(Ho, dtype=x.dtype, device=x.device)
        if T == 0 and not accumulate:
            for k, t in (("dw1", dw1), ("db1", db1), ("dw2", dw2), ("db2", db2)):
                if given[k]:
                    t.zero_()
    else:
        dw1 = db1 = dw2 = db2 = None
    if T == 0:
        return (torch.empty_like(x) if need_dx else None), dw1, db1, dw2, db2
    if not hip:
        a, b = _acc(pre[:, :F]), _acc(pre[:, F:])
        ya, da = _act(act, a)
        dh = _acc(dy) @ _acc(w2)
        dpre = torch.cat([dh * b * da, dh * ya], 1)
        dx = (dpre @ _acc(w1)).to(x.dtype) if need_dx else None     # (before a gradient is written over w1)
        if need_dw:
            for buf, val in ((dw1, dpre.t() @ _acc(x)), (db1, dpre.sum(0)), (dw2, _acc(dy).t() @ _acc(h)),
                             (db2, _acc(dy).sum(0))):
                if buf is not None:
                    buf.copy_(_acc(buf) + val if accumulate else val)
        return dx, dw1, db1, dw2, db2
    with _lib.on_device(x):
        s = _lib.stream()
        dpre = torch.empty(T, 2 * F, dtype=x.dtype, device=x.device)
        part = buf = None
        tile = _plan("dgate", T, F, Ho)[0]
        bm = _lib.query("mx_gated_tile", tile, 0)
        nparts = (T + bm - 1) // bm * _lib.query("mx_gated_tile", tile, 2)
        if db1 is not None:
            part, buf = colsum_partials_buffer(nparts, 2 * F, x.device)
        _lib.call("mx_gated_dgate", _lib.ptr(dy), _ld(dy), _lib.ptr(w2), _ld(w2), _lib.ptr(pre), _lib.ptr(dpre),
                  _lib.ptr(part), T, Ho, F, ACTS[act], tile, s)
        dx = None
        if need_dx:
            dx = torch.empty(T, H, dtype=x.dtype, device=x.device)
            tile, splits, _ = _plan("dx", T, H, 2 * F)
            ws = _split_ws(splits, T, H, x.device)
            _lib.call("mx_gated_dx", _lib.ptr(dpre), _lib.ptr(w1), _ld(w1), _lib.ptr(dx), T, H, 2 * F, tile, splits,
                      _lib.ptr(ws), s)
        if need_dw:
            pair = _plan_pair(T, H, F, Ho)
            if pair is not None:
                _lib.call("mx_gated_dw_pair", _lib.ptr(dpre), 2 * F, _lib.ptr(x), _ld(x), _lib.ptr(dw1), _ld(dw1),
                          2 * F, H, _lib.ptr(dy), _ld(dy), _lib.ptr(h), F, _lib.ptr(dw2), _ld(dw2), Ho, F, T,
                          int(accumulate), pair, s)
            for a, b, out in ((dpre, x, dw1), (dy, h, dw2)) if pair is None else ():
                (m, n) = out.shape
                tile, splits, _ = _plan("dw", m, n, T)
                ws = _split_ws(splits, m, n, x.device)
                _lib.call("mx_gated_dw", _lib.ptr(a), _ld(a), _lib.ptr(b), _ld(b), _lib.ptr(out), _ld(out), T, m, n,
                          int(accumulate), tile, splits, _lib.ptr(ws), s)
            if db1 is not None:
                colsum_finalize(buf, nparts, 2 * F, db1, accumulate)
            if db2 is not None:
                colsum(dy if dy.is_contiguous() else dy.contiguous(), db2, accumulate)
    return dx, dw1, db1, dw2, db2


class GatedMLPFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w1, b1, w2, b2, act):
        shape = x.shape
        x, w1, w2 = (_rows(t) for t in (x.reshape(-1, shape[-1]), w1, w2))
        b1, b2 = (None if b is None else _flat(b) for b in (b1, b2))
        train = any(ctx.needs_input_grad)
        y, pre, h = gated_mlp_fwd(x, w1, b1, w2, b2, act, save=train)
        if train:
            ctx.save_for_backward(x, pre, h, w1, w2, *[b for b in (b1, b2) if b is not None])
        ctx.meta = (shape, act, b1 is not None, b2 is not None)
        return y.view(*shape[:-1], y.shape[1])

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        shape, act, has1, has2 = ctx.meta
        x, pre, h, w1, w2, *b = ctx.saved_tensors
        b1 = b[0] if has1 else None
        b2 = b[-1] if has2 else None
        need = ctx.needs_input_grad
        dx, dw1, db1, dw2, db2 = gated_mlp_bwd(_rows(dy.reshape(-1, dy.shape[-1])), x, pre, h, w1, b1, w2, b2, act,
                                               need_dx=need[0], need_dw=any(need[1:5]))
        return dx.view(shape) if dx is not None else None, dw1, db1, dw2, db2, None


def _rows(t):
    """``t`` itself when the kernels read it in place, else a contiguous copy."""
    return t if not t.is_cuda or not t.numel() or _readable(t) else t.clone(memory_format=torch.contiguous_format)


def _flat(t):
    return t if not t.is_cuda or (t.is_contiguous() and t.data_ptr() % 16 == 0) else \
        t.clone(memory_format=torch.contiguous_format)


def gated_mlp(x, w1, b1, w2, b2, act: str = "silu"):
    """Differentiable gated feed-forward block: x [..., H] -> [..., Ho] (first derivatives only)."""
    return GatedMLPFn.apply(x, w1, b1, w2, b2, act)
