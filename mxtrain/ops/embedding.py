"""Scaled embedding lookup and its gradient by sorted tokens (``csrc/embedding.hip``) + reference.

``out[t] = scale * wte[ids[t]] (+ wpe[positions[t]])``: the lookup of a packed batch, where the
positions restart with each sequence (``ops.pack_sequences(...).positions``), next to
``embed_fwd`` / ``embed_bwd`` (ops/fused.py) for fixed [B, S] batches.  An id outside
[vocab_start, vocab_start + V) (another vocabulary shard's) or a position outside the table adds
nothing, forward and backward.

On the GPU: bfloat16, rows of a multiple of 8 values, at most 2^30 tokens, rows and columns.
"""
from __future__ import annotations

import math

import torch

from . import _lib

MAX_COUNT = 1 << 30     # tokens, rows and columns (the kernels count them in 32 bits)


def _acc(t):   # at least float32
    return t.double() if t.dtype == torch.float64 else t.float()


def _check_keys(name, what, keys, n=None):
    if keys.dtype != torch.int64:
        raise TypeError(f"{name}: {what} must be int64, got {keys.dtype}")
    if n is not None and keys.numel() != n:
        raise ValueError(f"{name}: {what} has {keys.numel()} entries, expected {n}")


def _check_table(name, what, t, device, cols=None):
    if t.dim() != 2 or t.shape[0] == 0 or t.shape[1] == 0 or (cols is not None and t.shape[1] != cols):
        raise ValueError(f"{name}: {what} must be a 2-D table" + (f" of {cols} columns" if cols else "")
                         + f", got {list(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name}: {what} is on {t.device}, expected {device}")


def _check_hip(name, what, t, H):
    if t.dtype != torch.bfloat16:
        raise TypeError(f"{name}: the GPU kernels take bfloat16, {what} is {t.dtype}")
    if H % 8:
        raise ValueError(f"{name}: the GPU kernels take rows of a multiple of 8 values, got {H}")
    if not t.is_contiguous() or t.data_ptr() % 16:
        raise ValueError(f"{name}: {what} must be contiguous and 16-byte aligned")


def _check_scale(name, scale):
    scale = float(scale)
    if not math.isfinite(scale):
        raise ValueError(f"{name}: scale must be finite, got {scale}")
    return scale


def _local(keys, start, n):
    loc = keys.reshape(-1) - start
    return loc, (loc >= 0) & (loc < n)


def embedding_fwd(ids, wte, scale: float = 1.0, positions=None, wpe=None, vocab_start: int = 0):
    """ids (int64, any shape of T entries), wte [V, H], positions (int64, T entries) and wpe
    [P, H] together or not at all -> [T, H], computed in fp32 and rounded once."""
    name = "embedding_fwd"
    _check_keys(name, "ids", ids)
    scale = _check_scale(name, scale)
    dev = ids.device
    _check_table(name, "wte", wte, dev)
    V, H = wte.shape
    T = ids.numel()
    if (positions is None) != (wpe is None):
        raise ValueError(f"{name}: give positions and wpe together or not at all")
    if wpe is not None:
        _check_keys(name, "positions", positions, T)
        _check_table(name, "wpe", wpe, dev, H)
        if positions.device != dev or wpe.dtype != wte.dtype:
            raise ValueError(f"{name}: positions / wpe must be on {dev}, wpe of type {wte.dtype}")
    if T == 0:
        return torch.empty(0, H, dtype=wte.dtype, device=dev)
    if not _lib.use_hip(wte):
        loc, ok = _local(ids, vocab_start, V)
        zero = torch.zeros((), dtype=_acc(wte).dtype, device=dev)
        out = torch.where(ok[:, None], _acc(wte)[loc.clamp(0, V - 1)] * scale, zero)
        if wpe is not None:
            loc, ok = _local(positions, 0, wpe.shape[0])
            out = out + torch.where(ok[:, None], _acc(wpe)[loc.clamp(0, wpe.shape[0] - 1)], zero)
        return out.to(wte.dtype)
    if max(T, V, H) > MAX_COUNT or (wpe is not None and wpe.shape[0] > MAX_COUNT):
        raise ValueError(f"{name}: the GPU kernels take at most 2^30 tokens, rows and columns, got {T}, {V} "
                         f"(positions: {0 if wpe is None else wpe.shape[0]}), {H}")
    _check_hip(name, "wte", wte, H)
    if wpe is not None:
        _check_hip(name, "wpe", wpe, H)
    ids = ids.contiguous()
    pos = positions.contiguous() if positions is not None else None
    with _lib.on_device(wte):
        out = torch.empty(T, H, dtype=wte.dtype, device=dev)
        _lib.call("mx_embedding_fwd", _lib.ptr(ids), _lib.ptr(wte), vocab_start, V, scale, _lib.ptr(pos),
                  _lib.ptr(wpe), wpe.shape[0] if wpe is not None else 0, _lib.ptr(out), T, H, _lib.stream())
    return out


def embedding_bwd(keys, dout, rows: int, scale: float = 1.0, out=None, accumulate: bool = False,
                  vocab_start: int = 0):
    """Gradient of a table of ``rows`` rows: out[v] = scale * sum of dout[t] over keys[t] == v,
    every row written (zeros where no token points), or added to ``out`` with ``accumulate``
    (only the rows with tokens are touched).  Sums are fp32 in token order: deterministic."""
    name = "embedding_bwd"
    _check_keys(name, "keys", keys)
    scale = _check_scale(name, scale)
    T, rows = keys.numel(), int(rows)
    if dout.dim() != 2 or dout.shape[0] != T or dout.shape[1] == 0:
        raise ValueError(f"{name}: dout must be [{T}, H], got {list(dout.shape)}")
    if not 0 < rows < 1 << 30:
        raise ValueError(f"{name}: rows must be in 1 .. 2^30 - 1, got {rows}")
    H, dev = dout.shape[1], dout.device
    if keys.device != dev:
        raise ValueError(f"{name}: keys are on {keys.device}, dout on {dev}")
    if accumulate and out is None:
        raise ValueError(f"{name}: accumulate needs out")
    if out is not None:
        _check_table(name, "out", out, dev, H)
        if T and _lib.lies_over((out,), (dout,)):
            raise ValueError(f"{name}: out must not lie over dout")
        if out.shape[0] != rows or out.dtype != dout.dtype:
            raise ValueError(f"{name}: out must be [{rows}, {H}] of type {dout.dtype}")
    hip = _lib.use_hip(dout)
    if hip and out is not None:
        _check_hip(name, "out", out, H)
    if out is None:
        out = torch.empty(rows, H, dtype=dout.dtype, device=dev)
    if T == 0:
        return out if accumulate else out.zero_()
    if not hip:
        loc, ok = _local(keys, vocab_start, rows)
        acc = torch.zeros(rows, H, dtype=_acc(dout).dtype, device=dev).index_add_(0, loc[ok], _acc(dout)[ok]) * scale
        return out.copy_(_acc(out) + acc if accumulate else acc)
    words = _lib.query64("mx_embedding_bwd_words", T, rows, H) if max(T, H) <= MAX_COUNT else -1
    if words < 0:
        raise ValueError(f"{name}: {T} tokens of {H} columns, {rows} rows are more than the kernels take")
    if dout.stride(1) != 1 or (T > 1 and (not H <= dout.stride(0) <= MAX_COUNT or dout.stride(0) % 8)) \
            or dout.data_ptr() % 16:
        dout = dout.clone(memory_format=torch.contiguous_format)
    _check_hip(name, "dout", dout[:1], H)
    keys = keys.contiguous()
    ld = dout.stride(0) if T > 1 else H
    with _lib.on_device(dout):
        ws = torch.empty(words, dtype=torch.int32, device=dev)
        _lib.call("mx_embedding_bwd", _lib.ptr(keys), vocab_start, _lib.ptr(dout), ld, _lib.ptr(out), T, rows, H,
                  scale, int(accumulate), _lib.ptr(ws), words, _lib.stream())
    return out


class EmbeddingFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, wte, scale, positions, wpe, vocab_start):
        ctx.save_for_backward(ids, positions if positions is not None else ids)
        ctx.meta = (wte.shape[0], wpe.shape[0] if wpe is not None else 0, scale, vocab_start)
        return embedding_fwd(ids, wte, scale, positions, wpe, vocab_start).view(*ids.shape, wte.shape[1])

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        ids, pos = ctx.saved_tensors
        V, P, scale, vocab_start = ctx.meta
        d = dout.reshape(-1, dout.shape[-1])
        dwte = embedding_bwd(ids, d, V, scale, vocab_start=vocab_start) if ctx.needs_input_grad[1] else None
        dwpe = embedding_bwd(pos, d, P) if P and ctx.needs_input_grad[4] else None
        return None, dwte, None, None, dwpe, None


def embedding(ids, wte, scale: float = 1.0, positions=None, wpe=None, vocab_start: int = 0):
    """Differentiable scaled lookup: ids [...] -> [..., H] (see :func:`embedding_fwd`)."""
    return EmbeddingFn.apply(ids, wte, scale, positions, wpe, vocab_start)
