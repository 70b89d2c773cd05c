"""Packed causal attention (``csrc/packed.hip``) + reference: sequences of different lengths laid
end to end on one token axis, grouped heads, no attention across a border.

:func:`pack_sequences` builds the row table of a batch from its cumulative lengths -- once per
batch, shared by every layer and by forward and backward.  Tensors are token-major 2-D views
[T, H * D] with any row stride (the packed QKV projection output is read in place), as in
``ops/attention.py``; ``lse`` is the base-2 log-sum-exp [Hq, T] the backward needs.

Rows behind the last sequence (a batch padded to a fixed size, so a captured step keeps its
shapes) never matter, whatever they hold: in tensors the op allocates they are zero, in buffers the
caller passes they are left as they were.  A value that is not finite reaches only the rows that see it.

On the GPU: bfloat16, head dimensions 64 and 128, a scale of 2^-100 .. 2^100.  Scores, softmax statistics and sums are fp32; P and dS are rounded once to bf16 as operands of
the matrix products, and delta = do . o is taken from the bf16 ``o`` that forward returned.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _lib

LOG2E = 1.4426950408889634
SCALES = 2.0 ** -100, 2.0 ** 100     # of the GPU kernels: lse / (scale log2 e) stays in the fp32 range


class PackedSequences:
    """Row table of one packed batch: ``cu_seqlens`` [n + 1] and, for each of ``total`` rows,
    the bounds of its sequence (``start``, ``end``, int32) and its position in it
    (``positions``, int64: RoPE's ``pos_ids``, the rows of a learned position table)."""

    __slots__ = ("cu_seqlens", "total", "start", "end", "meta", "positions", "order", "ptrs")

    def __init__(self, cu_seqlens, total, start, end, meta, positions, order=None):
        self.cu_seqlens, self.total, self.order = cu_seqlens, total, order
        self.start, self.end, self.meta, self.positions = start, end, meta, positions
        # kernel arguments (this object owns the tensors)
        self.ptrs = (start.data_ptr(), end.data_ptr(), meta.data_ptr(), _lib.ptr(order))

    @property
    def device(self):
        return self.start.device


def pack_sequences(cu_seqlens: torch.Tensor, total: int, device=None) -> PackedSequences:
    """``cu_seqlens``: [n + 1] int32 / int64 cumulative lengths, first 0, non-decreasing, last
    <= ``total`` (the rows of the batch; the rows behind the last sequence belong to none).
    A sequence may have length zero.  A CPU tensor is checked; a tensor on the GPU is not (that
    would wait for the device): its values are clamped into range by the kernel, so a table
    that breaks the contract gives wrong sequences, not an access out of range."""
    if cu_seqlens.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"pack_sequences: cu_seqlens must be int32 or int64, got {cu_seqlens.dtype}")
    if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 2:
        raise ValueError("pack_sequences: cu_seqlens must be a 1-D tensor of at least two entries")
    if cu_seqlens.numel() > 1 << 30:      # (counted in 32 bits)
        raise ValueError(f"pack_sequences: at most 2^30 entries of cu_seqlens, got {cu_seqlens.numel()}")
    total = int(total)
    if not 0 < total <= 1 << 30:
        raise ValueError(f"pack_sequences: total must be in 1 .. 2^30, got {total}")
    if not cu_seqlens.is_cuda:
        c = cu_seqlens.tolist()
        if c[0] != 0 or c[-1] > total or any(b < a for a, b in zip(c, c[1:])):
            raise ValueError(f"pack_sequences: cu_seqlens must start at 0, not decrease and end at most at {total}")
    dev = torch.device(device) if device is not None else cu_seqlens.device
    cu = cu_seqlens.to(dev).contiguous()
    n = cu.numel() - 1
    if not _lib.use_hip(cu):
        t = torch.arange(total, device=dev)
        nv = int(cu[-1])
        i = (torch.searchsorted(cu.to(torch.int64), t, right=True) - 1).clamp_(0, n - 1)
        real = t < nv
        start = torch.where(real, cu.to(torch.int64)[i], t)
        end = torch.where(real, cu.to(torch.int64)[i + 1], t)
        meta = torch.tensor([nv, 0, 0, 0], dtype=torch.int32, device=dev)
        return PackedSequences(cu, total, start.int(), end.int(), meta, t - start)
    with _lib.on_device(cu):
        tab = torch.empty(2 * total + 4 + _lib.query64("mx_packed_order_len", total), dtype=torch.int32,
                          device=cu.device)
        pos = torch.empty(total, dtype=torch.int64, device=cu.device)
        start, end, meta, order = tab.split((total, total, 4, tab.numel() - 2 * total - 4))
        _lib.call("mx_packed_plan", _lib.ptr(cu), int(cu.dtype == torch.int64), n, total, _lib.ptr(start),
                  _lib.ptr(end), _lib.ptr(meta), _lib.ptr(pos), _lib.ptr(order), _lib.stream())
    return PackedSequences(cu, total, start, end, meta, pos, order)


# ------------------------------------------------------------------ checks
def _check(name, seqs, Hq, Hkv, D, scale, **mats):
    if not isinstance(seqs, PackedSequences):
        raise TypeError(f"{name}: seqs must come from pack_sequences()")
    if Hq <= 0 or Hkv <= 0 or Hq % Hkv:
        raise ValueError(f"{name}: Hq ({Hq}) must be a positive multiple of Hkv ({Hkv})")
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not (scale > 0.0 and math.isfinite(scale)):
        raise ValueError(f"{name}: scale must be positive and finite, got {scale}")
    q = mats["q"]
    hip = _lib.use_hip(q)
    if hip and not SCALES[0] <= scale <= SCALES[1]:
        raise ValueError(f"{name}: the GPU kernels take a scale of 2^-100 .. 2^100, got {scale}")
    if hip and D not in (64, 128):
        raise ValueError(f"{name}: the GPU kernels take a head dimension of 64 or 128, got {D}")
    for key, t in mats.items():
        if t is None:
            continue
        width = (Hkv if key in ("k", "v", "dk", "dv") else Hq) * D
        if t.dim() != 2 or t.shape[0] != seqs.total or t.shape[1] != width:
            raise ValueError(f"{name}: {key} must be [{seqs.total}, {width}], got {list(t.shape)}")
        if t.device != seqs.device:
            raise ValueError(f"{name}: {key} is on {t.device}, the sequences on {seqs.device}")
        if t.dtype != q.dtype:
            raise TypeError(f"{name}: {key} is {t.dtype}, q is {q.dtype}")
        if hip:
            if t.dtype != torch.bfloat16:
                raise TypeError(f"{name}: the GPU kernels take bfloat16, {key} is {t.dtype}")
            if not _readable(t) or _ld(t) > 1 << 22:
                raise ValueError(f"{name}: {key} needs unit column stride, rows that do not overlap, a row stride "
                                 f"that is a multiple of 8 (at most 2^22) and 16-byte alignment; strides "
                                 f"{list(t.stride())}, address % 16 = {t.data_ptr() % 16}")
    return scale, hip


def _ld(t):
    """Row stride (a single row has none: its width)."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _readable(t):
    """Rows the kernels read (and write) in place."""
    return (t.dim() == 2 and t.stride(1) == 1 and _ld(t) % 8 == 0 and _ld(t) >= t.shape[1]
            and t.data_ptr() % 16 == 0)


def _mats(seqs, Hq, Hkv, D, scale, q, *mats):
    """[(address, row stride)] of a valid GPU call's matrices (None for those not given), or None: a
    CPU call, or one whose fault :func:`_check` names."""
    if (type(seqs) is not PackedSequences or not _lib.use_hip(q) or (D != 64 and D != 128) or Hkv <= 0 or Hq <= 0
            or Hq % Hkv or not (scale is None or SCALES[0] <= scale <= SCALES[1])):
        return None
    dev, T, out = seqs.start.get_device(), seqs.total, []
    for t, heads in mats:
        m = None
        if t is not None:
            m = _lib.rows_of(t, T, heads * D, dev, 1 << 22)
            if m is None:
                return None
        out.append(m)
    return out


# ------------------------------------------------------------------ reference (CPU)
def _ref_mask(seqs):
    t = torch.arange(seqs.total, device=seqs.device)
    real = (t < seqs.meta[0])[:, None]
    return real & (t[None, :] <= t[:, None]) & (t[None, :] >= seqs.start[:, None])


def _acc(t):   # at least float32
    return t.double() if t.dtype == torch.float64 else t.float()


def _ref_parts(seqs, *mats):
    """(rows, keys) ranges that are taken by themselves so that a value that is not finite reaches only the
    rows that see it (0 * NaN is NaN inside a product): each row of a sequence that holds one, any other
    sequence whole; None: everything is finite."""
    nv = int(seqs.meta[0])
    bad = torch.zeros(nv, dtype=torch.bool, device=seqs.device)
    for t in mats:
        bad |= ~torch.isfinite(t.detach()[:nv]).all(1)
    if not bad.any():
        return None
    parts, a, ends = [], 0, seqs.end.tolist()
    while a < nv:
        b = ends[a]
        parts += [((i, i + 1), (a, i + 1)) for i in range(a, b)] if bad[a:b].any() else [((a, b), (a, b))]
        a = b
    return parts


def _ref_fwd(q, k, v, seqs, Hq, Hkv, D, scale, dout=None):
    T = seqs.total
    real = torch.arange(T, device=q.device) < seqs.meta[0]

    def heads(t, h):   # [h, T, D]; the rows behind the last sequence are never read
        return torch.where(real[:, None], _acc(t), torch.zeros((), dtype=_acc(t).dtype)).reshape(T, h, D).transpose(0, 1)
    g = Hq // Hkv
    qf, kf, vf = heads(q, Hq), heads(k, Hkv).repeat_interleave(g, 0), heads(v, Hkv).repeat_interleave(g, 0)

    def attend(qf, kf, vf, m):
        s = (torch.matmul(qf, kf.transpose(1, 2)) * scale).masked_fill(~m, float("-inf"))
        lse = torch.logsumexp(s, -1)
        p = torch.where(m, torch.exp(s - lse[..., None]), torch.zeros((), dtype=s.dtype))
        return torch.matmul(p, vf), lse
    m, parts = _ref_mask(seqs), _ref_parts(seqs, q, k, v, *(() if dout is None else (dout,)))
    if parts is None:
        o, lse = attend(qf, kf, vf, m)
    else:
        got = [attend(qf[:, a:b], kf[:, c:d], vf[:, c:d], m[a:b, c:d]) for (a, b), (c, d) in parts]
        rest = T - parts[-1][0][1]
        o = torch.cat([x for x, _ in got] + [qf.new_zeros(Hq, rest, D)], 1)
        lse = torch.cat([x for _, x in got] + [qf.new_zeros(Hq, rest)], 1)
    o = o.transpose(0, 1).reshape(T, Hq * D)
    lse = torch.where(real, lse * LOG2E, torch.full_like(lse, float("inf")))
    return o, lse


def _emit(val, buf, seqs):
    """``val`` rounded to the result: a new tensor (zero behind the last sequence), or into the
    caller's buffer, whose rows there stay as they are."""
    if buf is None:
        return val
    nv = int(seqs.meta[0])
    buf[:nv] = val[:nv].to(buf.dtype)
    return buf


def _apart(name, T, outs, ins):
    """Results that lie over an operand, or over each other, would be read after they are written."""
    for i, a in enumerate(outs):
        if any(_lib.overlap(T, a, b) for b in ins + outs[:i]):
            raise ValueError(f"{name}: results must not lie over the operands or over each other")


# ------------------------------------------------------------------ forward / backward
def packed_attn_fwd(q, k, v, seqs: PackedSequences, Hq: int, Hkv: int, D: int, scale: Optional[float] = None,
                    out=None):
    """Causal attention within each sequence: q [T, Hq*D], k / v [T, Hkv*D] -> (o [T, Hq*D],
    lse [Hq, T]).  Query head h reads key head h // (Hq // Hkv).  ``out``: a buffer for o."""
    m = _mats(seqs, Hq, Hkv, D, scale, q, (q, Hq), (k, Hkv), (v, Hkv), (out, Hq))
    if m is None:
        scale, hip = _check("packed_attn_fwd", seqs, Hq, Hkv, D, scale, q=q, k=k, v=v, out=out)
        if not hip:
            o, lse = _ref_fwd(q, k, v, seqs, Hq, Hkv, D, scale)
            return _emit(o.to(q.dtype), out, seqs), lse.float()
        raise ValueError("packed_attn_fwd: unsupported arguments")
    T = seqs.total
    (q_, ldq), (k_, ldk), (v_, ldv), o_ = m
    if out is not None:
        _apart("packed_attn_fwd", T, [(*o_, Hq * D)], [(q_, ldq, Hq * D), (k_, ldk, Hkv * D), (v_, ldv, Hkv * D)])
    with _lib.on_device(q):
        o = out if out is not None else torch.empty(T, Hq * D, dtype=q.dtype, device=q.device)
        lse = torch.empty(Hq, T, dtype=torch.float32, device=q.device)
        _lib.call("mx_packed_attn_fwd", q_, k_, v_, ldq, ldk, ldv, o.data_ptr(), o_[1] if o_ else Hq * D,
                  lse.data_ptr(), *seqs.ptrs, T, Hq, Hkv, D, D ** -0.5 if scale is None else scale, int(out is None),
                  _lib.stream())
    return o, lse


def packed_attn_bwd(dout, q, k, v, o, lse, seqs: PackedSequences, Hq: int, Hkv: int, D: int,
                    scale: Optional[float] = None, dq=None, dk=None, dv=None):
    """(dq, dk, dv) of :func:`packed_attn_fwd`; given views (e.g. column ranges of one packed
    dqkv) are written in place.  Deterministic: no atomics."""
    m = _mats(seqs, Hq, Hkv, D, scale, q, (q, Hq), (k, Hkv), (v, Hkv), (o, Hq), (dout, Hq), (dq, Hq), (dk, Hkv),
              (dv, Hkv))
    if m is None:
        scale, hip = _check("packed_attn_bwd", seqs, Hq, Hkv, D, scale, q=q, k=k, v=v, dout=dout, o=o, dq=dq, dk=dk,
                            dv=dv)
        if hip:
            raise ValueError("packed_attn_bwd: unsupported arguments")
    if lse.shape != (Hq, seqs.total) or lse.dtype is not torch.float32 or not lse.is_contiguous() \
            or lse.device != q.device:
        raise ValueError(f"packed_attn_bwd: lse must be the float32 [{Hq}, {seqs.total}] tensor packed_attn_fwd returned")
    if m is None:
        with torch.enable_grad():
            leaves = [_acc(t.detach()).clone().requires_grad_(True) for t in (q, k, v)]
            of, _ = _ref_fwd(*leaves, seqs, Hq, Hkv, D, scale, dout)
            nv = int(seqs.meta[0])
            grads = torch.autograd.grad(of[:nv], leaves, _acc(dout)[:nv])
        return tuple(_emit(g.to(q.dtype), buf, seqs) for g, buf in zip(grads, (dq, dk, dv)))
    T, given = seqs.total, dq is not None
    if (dk is not None) != given or (dv is not None) != given:
        raise ValueError("packed_attn_bwd: give all of dq, dk, dv or none")
    (q_, ldq), (k_, ldk), (v_, ldv), (o_, ldo), (do_, lddo), *grads = m
    if given:
        wide, narrow = Hq * D, Hkv * D
        _apart("packed_attn_bwd", T, [(*g, w) for g, w in zip(grads, (wide, narrow, narrow))],
               [(q_, ldq, wide), (k_, ldk, narrow), (v_, ldv, narrow), (o_, ldo, wide), (do_, lddo, wide),
                (lse.data_ptr(), 2 * Hq, 2 * Hq)])     # (lse: as many bytes as [T, 2 Hq] of bf16)
    with _lib.on_device(q):
        if not given:
            dq = torch.empty(T, Hq * D, dtype=q.dtype, device=q.device)
            dk = torch.empty(T, Hkv * D, dtype=q.dtype, device=q.device)
            dv = torch.empty(T, Hkv * D, dtype=q.dtype, device=q.device)
            grads = (dq.data_ptr(), Hq * D), (dk.data_ptr(), Hkv * D), (dv.data_ptr(), Hkv * D)
        stats = torch.empty(2, Hq, T, dtype=torch.float32, device=q.device)
        nf = _lib.query64("mx_packed_attn_bwd_floats", T, Hq, Hkv, D)
        part = torch.empty(nf, dtype=torch.float32, device=q.device) if nf else None
        (dq_, lddq), (dk_, lddk), (dv_, lddv) = grads
        _lib.call("mx_packed_attn_bwd", q_, k_, v_, ldq, ldk, ldv, o_, ldo, do_, lddo, lse.data_ptr(),
                  stats.data_ptr(), dq_, lddq, dk_, dv_, lddk, lddv, *seqs.ptrs, T, Hq, Hkv, D,
                  D ** -0.5 if scale is None else scale, int(not given), _lib.ptr(part), nf, _lib.stream())
    return dq, dk, dv


class PackedAttnFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, seqs, Hq, Hkv, D, scale):
        q, k, v = (_rows(t) for t in (q, k, v))
        o, lse = packed_attn_fwd(q, k, v, seqs, Hq, Hkv, D, scale)
        ctx.save_for_backward(q, k, v, o, lse)
        ctx.meta = (seqs, Hq, Hkv, D, scale)
        return o

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, do):
        q, k, v, o, lse = ctx.saved_tensors
        seqs, Hq, Hkv, D, scale = ctx.meta
        dq, dk, dv = packed_attn_bwd(_rows(do), q, k, v, o, lse, seqs, Hq, Hkv, D, scale)
        return dq, dk, dv, None, None, None, None, None


def _rows(t):
    """``t`` itself when the kernels can read it in place, else a contiguous copy (an expanded
    or transposed tensor, an unaligned view)."""
    return t if not t.is_cuda or _readable(t) else t.clone(memory_format=torch.contiguous_format)


def packed_attention(q, k, v, seqs: PackedSequences, Hq: int, Hkv: int, D: int, scale: Optional[float] = None):
    """Differentiable packed causal attention (see :func:`packed_attn_fwd`).  First derivatives
    only."""
    return PackedAttnFn.apply(q, k, v, seqs, Hq, Hkv, D, scale)
