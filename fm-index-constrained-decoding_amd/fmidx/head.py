"""The scores product of a document-constrained model: hidden states times the
output embedding, with bias, soft cap, residual and the constraint's mask in its
epilogue (fm_head_scores).

Replaces the model's last ``hidden @ weight.T`` followed by a processor's
``scores + mask`` in a serving loop that keeps the allowed bits on the device:

    bits = index.decode_step(next_tokens, lo, hi, bits, V, 10, packed=True)
    scores = head_scores(hidden, lm_head.weight, constraint=Constraint(allowed=bits),
                         out_dtype=torch.float32)

Under a hard mask the constraint is known before the product, so only weight
rows that some sequence of the batch may still take are read.
"""
from __future__ import annotations

import ctypes
import functools
import math
from ctypes import c_double, c_int32, c_int64, c_uint64, c_void_p
from typing import Optional

import torch

from ._lib import check, lib
from .constraint import Constraint
from .losses import _on, _ptr, _stream
from .processors import _DTYPE_CODE


class _HeadArgs(ctypes.Structure):
    """fm_head_args (include/fmidx.h)."""
    _fields_ = [("d_hidden", c_void_p), ("d_weight", c_void_p), ("d_bias", c_void_p), ("d_residual", c_void_p),
                ("d_out", c_void_p), ("ld_hidden", c_uint64), ("ld_weight", c_uint64), ("ld_residual", c_uint64),
                ("ld_out", c_uint64), ("B", c_uint64), ("V", c_uint64), ("d", c_uint64), ("d_bits", c_void_p),
                ("ld_bits", c_uint64), ("d_unigram_bits", c_void_p), ("d_rows", c_void_p), ("eos", c_int64),
                ("softcap", c_double), ("dtype", c_int32), ("out_dtype", c_int32), ("d_ws", c_void_p),
                ("ws_bytes", c_uint64)]


assert ctypes.sizeof(_HeadArgs) == 168


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(n: int, vocab: int) -> int:
    need = c_uint64()
    check(lib().fm_head_workspace(n, vocab, ctypes.byref(need)), "head_workspace")
    return need.value


def _rows_of(t, cols: int):
    """t as 2-D rows of unit stride, and their pitch."""
    if t.dim() != 2:
        t = t.reshape(-1, cols)
    if cols > 1 and t.stride(1) != 1 or t.shape[0] > 1 and t.stride(0) < cols:
        t = t.contiguous()
    return t, (t.stride(0) if t.shape[0] > 1 else cols)


def head_scores(hidden, weight, *, bias=None, softcap: float = 0.0, residual=None,
                constraint: Optional[Constraint] = None, out_dtype: Optional[torch.dtype] = None, out=None):
    """scores [..., V] = f(hidden @ weight.T + bias) + residual + mask, with
    f(x) = softcap * tanh(x / softcap) (0: none); -inf where the constraint
    forbids the token.  Accumulated in f32 and rounded once.

    hidden      bf16 / f16 [..., d] on the GPU
    weight      [V, d], hidden's dtype (an nn.Linear's)
    bias        [V], hidden's dtype
    residual    [..., V] in out_dtype, e.g. another head's scores
    constraint  fmidx.constraint.Constraint over hidden.shape[:-1] rows, or None
    out_dtype   hidden's dtype (default) or float32
    out         where to write: [..., V] in out_dtype, rows of unit stride; may be residual
                itself, and must not overlap the inputs otherwise

    The serving form: no gradient (call it under no_grad, or with tensors that
    need none).  Runs on hidden's device and its current stream, never
    synchronises, and can be captured into a HIP graph."""
    what = "head_scores"
    for name, t in (("hidden", hidden), ("weight", weight)):
        if not isinstance(t, torch.Tensor) or t.dtype not in (torch.bfloat16, torch.float16):
            raise TypeError(f"{what}: {name} must be a bfloat16 or float16 tensor")
    for name, t in (("bias", bias), ("residual", residual), ("out", out)):
        if t is not None and not isinstance(t, torch.Tensor):
            raise TypeError(f"{what}: {name} must be a tensor")
    if weight.dtype != hidden.dtype or bias is not None and bias.dtype != hidden.dtype:
        raise TypeError(f"{what}: weight and bias must be {hidden.dtype} like hidden")
    out_dtype = hidden.dtype if out_dtype is None else out_dtype
    if out_dtype not in (hidden.dtype, torch.float32):
        raise TypeError(f"{what}: out_dtype must be {hidden.dtype} or float32, not {out_dtype}")
    for name, t in (("residual", residual), ("out", out)):
        if t is not None and t.dtype != out_dtype:
            raise TypeError(f"{what}: {name} must be {out_dtype}")
    if weight.dim() != 2 or hidden.dim() < 1 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"{what}: hidden {tuple(hidden.shape)}, weight {tuple(weight.shape)}")
    vocab, d = weight.shape
    shape = hidden.shape[:-1] + (vocab,)
    n = math.prod(shape[:-1])
    if bias is not None and bias.shape != (vocab,):
        raise ValueError(f"{what}: bias {tuple(bias.shape)} for {vocab} tokens")
    for name, t in (("residual", residual), ("out", out)):
        if t is not None and t.shape != shape:
            raise ValueError(f"{what}: {name} {tuple(t.shape)}, expected {tuple(shape)}")
    if not hidden.is_cuda or any(t is not None and t.device != hidden.device for t in (weight, bias, residual, out)):
        raise ValueError(f"{what}: every tensor must be on hidden's GPU (hidden is on {hidden.device})")
    if not isinstance(softcap, (int, float)) or not math.isfinite(softcap) or softcap < 0:
        raise ValueError(f"{what}: softcap must be 0 or positive, not {softcap!r}")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (hidden, weight, bias, residual, out)):
        raise ValueError(f"{what} has no gradient: call it under torch.no_grad()")
    dev = hidden.device
    if constraint is not None and not isinstance(constraint, Constraint):
        raise TypeError(f"{what}: constraint must be a fmidx.constraint.Constraint")
    con = constraint.checked(n, vocab, dev) if constraint is not None else Constraint()
    given = out is not None
    with _on(dev):
        if not given:
            out = torch.empty(shape, dtype=out_dtype, device=dev)
        if n == 0 or vocab == 0:
            return out
        try:
            o = out if out.dim() == 2 else out.view(n, vocab)       # the caller's own rows, never a copy
        except RuntimeError as e:
            raise ValueError(f"{what}: out {tuple(out.shape)} of strides {out.stride()} is no [{n}, {vocab}] view") from e
        if o.stride(1) != 1 and vocab > 1 or n > 1 and o.stride(0) < vocab:
            raise ValueError(f"{what}: out needs rows of unit stride that do not overlap")
        h, ldh = _rows_of(hidden, d) if d else (hidden, 0)
        w, ldw = _rows_of(weight, d) if d else (weight, 0)
        r, ldr = _rows_of(residual, vocab) if residual is not None else (None, 0)
        b = bias.contiguous() if bias is not None else None
        need = _workspace_bytes(n, vocab) if constraint is not None else 0
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        a = _HeadArgs(_ptr(h), _ptr(w), _ptr(b), _ptr(r), _ptr(o), ldh, ldw, ldr,
                      o.stride(0) if n > 1 else vocab, n, vocab, d, _ptr(con.allowed),
                      con.allowed.stride(0) if con.allowed is not None else 0, _ptr(con.unigrams), _ptr(con.rows),
                      con.eos, float(softcap), _DTYPE_CODE[hidden.dtype], _DTYPE_CODE[out_dtype], _ptr(ws), need)
        check(lib().fm_head_scores(ctypes.byref(a), _stream(dev)), what)
        if given:                 # a backward pass that still needs what out held raises
            torch._C._increment_version((out,))
    return out


__all__ = ["head_scores"]
