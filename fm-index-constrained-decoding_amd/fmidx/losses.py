"""Training on constrained scores: log-probabilities of chosen tokens under the
document constraint, and the policy and preference losses on them, each with
its gradient (fm_token_logprobs, fm_policy_loss, fm_preference_loss).

A model that samples behind a document-constrained processor draws from the
masked distribution, so the log-probabilities a loss compares have to be that
distribution's: ``scores + mask`` in the scores' own type -- what the processor
returns -- normalised over the tokens the mask leaves in.

    con = prefix_constraint(index, answers, vocab)          # fmidx.constraint
    old = token_logprobs(scores, answers, constraint=con)   # when sampling
    loss, logp = policy_loss(scores, answers, old, advantages, constraint=con)
    loss.backward()

Common arguments

scores       f32 / bf16 / f16 [..., V] on the GPU.  2-D and 3-D tensors are read
             in place through their strides when V is contiguous (a slice
             ``logits[:, :-1]``, a padded row pitch, any alignment); anything
             else is copied first
tokens       integers, scores.shape[:-1].  A token outside [0, V) (the padding's
             -100) leaves its position out: log-probability 0, no gradient
constraint   fmidx.constraint.Constraint over scores.shape[:-1] rows, or None
temperature  scores are divided by it, after the mask

A token that the constraint forbids -- any token, when a row's mask leaves
nothing -- has log-probability -inf; such a position adds nothing to a loss and
gets a gradient of zeros, and so do positions of weight 0.  Scores of forbidden
tokens are never used, NaN and infinities included, and their gradient is 0.
+inf or NaN among the tokens that count makes their position's results NaN, and
with them the loss, unless its weight is 0.
Only ``scores`` is differentiated, once; sums are in fixed order, so results
repeat bit for bit.  Calls run on the scores' device and its current stream,
allocate through torch and never synchronise, so they can be captured into a
HIP graph -- with leaves that no eager graph still holds, as torch asks of any
captured backward pass.
"""
from __future__ import annotations

import contextlib
import ctypes
import functools
import math
from ctypes import c_double, c_int32, c_int64, c_uint64, c_void_p
from typing import NamedTuple, Optional

import torch

from ._lib import check, lib
from .constraint import Constraint
from .processors import _DTYPE_CODE


class _ScoreRows(ctypes.Structure):
    """fm_score_rows (include/fmidx.h)."""
    _fields_ = [("d_scores", c_void_p), ("ld_scores", c_uint64), ("ld_outer", c_uint64), ("inner", c_uint64),
                ("N", c_uint64), ("V", c_uint64), ("d_tokens", c_void_p), ("d_bits", c_void_p),
                ("ld_bits", c_uint64), ("d_unigram_bits", c_void_p), ("d_rows", c_void_p), ("eos", c_int64),
                ("temperature", c_double), ("dtype", c_int32), ("reserved", c_int32)]


class _PolicyArgs(ctypes.Structure):
    """fm_policy_args (include/fmidx.h)."""
    _fields_ = [("d_old_logp", c_void_p), ("d_ref_logp", c_void_p), ("d_advantages", c_void_p),
                ("d_weights", c_void_p), ("clip_low", c_double), ("clip_high", c_double), ("kl_coef", c_double),
                ("d_loss", c_void_p), ("d_logp", c_void_p), ("d_stats", c_void_p), ("d_coef", c_void_p),
                ("d_grad", c_void_p), ("ld_grad", c_uint64), ("d_ws", c_void_p), ("ws_bytes", c_uint64)]


class _PreferenceArgs(ctypes.Structure):
    """fm_preference_args (include/fmidx.h)."""
    _fields_ = [("d_cu", c_void_p), ("d_ref_logp", c_void_p), ("d_weights", c_void_p), ("pairs", c_uint64),
                ("beta", c_double), ("label_smoothing", c_double), ("margin", c_double), ("d_loss", c_void_p),
                ("d_seq_logp", c_void_p), ("d_stats", c_void_p), ("d_coef", c_void_p), ("d_ws", c_void_p),
                ("ws_bytes", c_uint64)]


assert ctypes.sizeof(_ScoreRows) == 112 and ctypes.sizeof(_PolicyArgs) == 120 and \
    ctypes.sizeof(_PreferenceArgs) == 104


class PolicyLoss(NamedTuple):
    loss: torch.Tensor           # f32 scalar
    logprobs: torch.Tensor       # f32 tokens.shape, detached


class PreferenceLoss(NamedTuple):
    loss: torch.Tensor           # f32 scalar
    logprobs: torch.Tensor       # f32 [2 * pairs], the sequences' weighted sums, detached


_HERE = contextlib.nullcontext()


def _on(device):
    return _HERE if torch._C._cuda_getDevice() == device.index else torch.cuda.device(device)


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(n: int, vocab: int, pairs: int) -> int:
    need = c_uint64()
    check(lib().fm_score_workspace(n, vocab, pairs, ctypes.byref(need)), "score_workspace")
    return need.value


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _stream(device) -> c_void_p:
    return c_void_p(torch._C._cuda_getCurrentRawStream(device.index))


def _capture(device) -> int:
    """The number of the capture that records the device's current stream, or 0."""
    if not torch._C._cuda_isCurrentStreamCapturing():
        return 0
    n = c_uint64()
    check(lib().fm_stream_capture(_stream(device), ctypes.byref(n)), "stream_capture")
    return n.value


def _rows(scores, tokens, allowed, unigrams, rows, eos: int, temperature: float) -> _ScoreRows:
    n, vocab = tokens.numel(), scores.shape[-1]
    inner, ld_outer, ld = max(1, n), 0, vocab
    if scores.dim() == 2:
        ld = scores.stride(0)
    elif scores.dim() == 3 and scores.shape[1] > 0:
        inner, ld_outer, ld = scores.shape[1], scores.stride(0), scores.stride(1)
    return _ScoreRows(_ptr(scores), ld, ld_outer, inner, n, vocab, _ptr(tokens), _ptr(allowed),
                      allowed.stride(0) if allowed is not None else 0, _ptr(unigrams), _ptr(rows), eos, temperature,
                      _DTYPE_CODE[scores.dtype], 0)


class _Call:
    """One call's checked arguments: what the kernels read, and the struct that
    says where."""

    def __init__(self, scores, tokens, constraint, temperature, what: str):
        if not isinstance(scores, torch.Tensor) or not isinstance(tokens, torch.Tensor):
            raise TypeError(f"{what}: scores and tokens must be tensors")
        if scores.dtype not in _DTYPE_CODE:
            raise TypeError(f"{what}: unsupported scores dtype {scores.dtype}")
        if tokens.dtype.is_floating_point or tokens.dtype.is_complex or tokens.dtype == torch.bool:
            raise TypeError(f"{what}: tokens must be integers, not {tokens.dtype}")
        if scores.dim() < 1 or tokens.shape != scores.shape[:-1]:
            raise ValueError(f"{what}: tokens {tuple(tokens.shape)} for scores {tuple(scores.shape)}")
        if scores.shape[-1] == 0:
            raise ValueError(f"{what}: scores of no tokens")
        if not scores.is_cuda or tokens.device != scores.device:
            raise ValueError(f"{what}: scores and tokens must be on one GPU (scores {scores.device}, "
                             f"tokens {tokens.device})")
        if not (isinstance(temperature, (int, float)) and math.isfinite(temperature) and temperature > 0):
            raise ValueError(f"{what}: temperature must be positive and finite, not {temperature!r}")
        self.device = scores.device
        self.vocab = scores.shape[-1]
        self.n = tokens.numel()
        if scores.dim() not in (2, 3) or scores.stride(-1) != 1:
            scores = scores.contiguous()
        self.scores = scores
        self.tokens = tokens.to(torch.int64).contiguous()
        if constraint is not None and not isinstance(constraint, Constraint):
            raise TypeError(f"{what}: constraint must be a fmidx.constraint.Constraint")
        self.con = constraint.checked(self.n, self.vocab, self.device) if constraint is not None else Constraint()
        c = self.con
        self.temperature, self.eos = float(temperature), c.eos
        self.args = _rows(self.scores, self.tokens, c.allowed, c.unigrams, c.rows, c.eos, self.temperature)

    def floats(self, x, name: str, what: str, shape):
        """x as contiguous f32 on the scores' device (a constant of the loss)."""
        if not isinstance(x, torch.Tensor) or x.dtype.is_complex:
            raise TypeError(f"{what}: {name} must be a real tensor")
        if x.shape != shape:
            raise ValueError(f"{what}: {name} {tuple(x.shape)}, expected {tuple(shape)}")
        if x.device != self.device:
            raise ValueError(f"{what}: {name} is on {x.device}, the scores on {self.device}")
        if x.dtype is torch.float32 and x.is_contiguous():
            return x
        return x.detach().to(torch.float32).contiguous()

    def scratch(self, pairs: int = 0):
        """One buffer for the call's small results: the rows' statistics (2 N
        floats) and coefficients (N), which the gradient reads, then the
        workspace.  Returns it, the addresses of the three, and the workspace's size."""
        ws = _workspace_bytes(self.n, self.vocab, pairs)
        head = (12 * self.n + 15) // 16 * 16
        buf = torch.empty(head + ws, dtype=torch.uint8, device=self.device)
        p = buf.data_ptr()
        return buf, p, p + 8 * self.n, p + head, ws

    def keep(self, ctx, shape, *more):
        """Everything the gradient reads goes through save_for_backward, so an
        in-place change before backward(), by torch or by this package's calls, is
        an error, not a wrong gradient."""
        c = self.con
        ctx.save_for_backward(self.scores, self.tokens, c.allowed, c.unigrams, c.rows, *more)
        ctx.eos, ctx.temperature, ctx.shape = self.eos, self.temperature, shape
        ctx.set_materialize_grads(False)      # else a zero tensor is filled for the detached output

    @staticmethod
    def grad(ctx, coef, scale, made=None):
        """The scores' gradient (shape ctx.shape, contiguous).  coef: per row,
        or None for those kept in the scratch buffer; made: the gradient already
        if the scale turns out to be 1."""
        scores, tokens, allowed, unigrams, rows, buf = ctx.saved_tensors
        stats = buf.data_ptr()
        # laid out anew: saved-tensor hooks may hand back copies
        a = _rows(scores, tokens, allowed, unigrams, rows, ctx.eos, ctx.temperature)
        out = torch.empty(ctx.shape, dtype=scores.dtype, device=scores.device) if made is None else made
        if out.numel():
            with _on(out.device):
                check(lib().fm_token_logprobs_grad(ctypes.byref(a), stats,
                                                   stats + 8 * a.N if coef is None else _ptr(coef), _ptr(scale),
                                                   0 if made is None else 1, _ptr(out), a.V, _stream(out.device)), "token_logprobs_grad")
        return out


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, scores, tokens, constraint, temperature):
        call = _Call(scores, tokens, constraint, temperature, "token_logprobs")
        with _on(call.device):
            logp = torch.empty(tokens.shape, dtype=torch.float32, device=call.device)
            buf, stats, _, ws, ws_bytes = call.scratch()
            check(lib().fm_token_logprobs(ctypes.byref(call.args), _ptr(logp), stats, ws, ws_bytes,
                                          _stream(call.device)), "token_logprobs")
        call.keep(ctx, scores.shape, buf)
        return logp

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        if g is None:
            return None, None, None, None
        return _Call.grad(ctx, g.to(torch.float32).contiguous(), None), None, None, None


class _PolicyLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, scores, tokens, old, adv, weights, ref, lo, hi, kl, constraint, temperature, grad):
        what = "policy_loss"
        call = _Call(scores, tokens, constraint, temperature, what)
        old = call.floats(old, "old_logprobs", what, tokens.shape)
        adv = call.floats(adv, "advantages", what, tokens.shape)
        weights = None if weights is None else call.floats(weights, "weights", what, tokens.shape)
        ref = None if ref is None else call.floats(ref, "ref_logprobs", what, tokens.shape)
        with _on(call.device):
            loss = torch.empty((), dtype=torch.float32, device=call.device)
            logp = torch.empty(tokens.shape, dtype=torch.float32, device=call.device)
            buf, stats, coef, ws, ws_bytes = call.scratch()
            made = torch.empty(scores.shape, dtype=scores.dtype, device=call.device) if grad else None
            p = _PolicyArgs(_ptr(old), _ptr(ref), _ptr(adv), _ptr(weights), lo, hi, kl, _ptr(loss), _ptr(logp),
                            stats, coef, _ptr(made), call.vocab, ws, ws_bytes)
            check(lib().fm_policy_loss(ctypes.byref(call.args), ctypes.byref(p), _stream(call.device)), what)
            # a backward pass replayed apart from this call cannot take what only this call writes
            ctx.capture = _capture(call.device) if grad else 0
        call.keep(ctx, scores.shape, buf)
        ctx.made = made
        ctx.mark_non_differentiable(logp)
        return loss, logp

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g, _):
        if g is None:
            return (None,) * 12
        made, ctx.made = ctx.made, None       # handed out once: a second backward makes its own
        with _on(g.device):
            if ctx.capture != _capture(g.device):
                made = None
        return (_Call.grad(ctx, None, g.to(torch.float32), made),) + (None,) * 11


class _PreferenceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, scores, tokens, cu, ref, weights, beta, smoothing, margin, constraint, temperature):
        what = "preference_loss"
        call = _Call(scores, tokens, constraint, temperature, what)
        if not isinstance(cu, torch.Tensor) or cu.dtype not in (torch.int64, torch.int32):
            raise TypeError(f"{what}: cu_seqlens must be an int64 tensor")
        if cu.dim() != 1 or cu.numel() % 2 == 0 or cu.device != call.device:
            raise ValueError(f"{what}: cu_seqlens must hold 2 * pairs + 1 bounds on {call.device}")
        pairs = cu.numel() // 2
        cu = cu.to(torch.int64).contiguous()
        ref = None if ref is None else call.floats(ref, "ref_logprobs", what, torch.Size((2 * pairs,)))
        weights = None if weights is None else call.floats(weights, "weights", what, tokens.shape)
        with _on(call.device):
            loss = torch.empty((), dtype=torch.float32, device=call.device)
            seq = torch.empty(2 * pairs, dtype=torch.float32, device=call.device)
            buf, stats, coef, ws, ws_bytes = call.scratch(pairs)
            p = _PreferenceArgs(_ptr(cu), _ptr(ref), _ptr(weights), pairs, beta, smoothing, margin, _ptr(loss),
                                _ptr(seq), stats, coef, ws, ws_bytes)
            check(lib().fm_preference_loss(ctypes.byref(call.args), ctypes.byref(p), _stream(call.device)), what)
        call.keep(ctx, scores.shape, buf)
        ctx.mark_non_differentiable(seq)
        return loss, seq

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g, _):
        if g is None:
            return (None,) * 10
        return (_Call.grad(ctx, None, g.to(torch.float32)),) + (None,) * 9


def _number(x, name: str, what: str) -> float:
    if not isinstance(x, (int, float)) or not math.isfinite(x):
        raise ValueError(f"{what}: {name} must be a finite number, not {x!r}")
    return float(x)


def token_logprobs(scores, tokens, *, constraint: Optional[Constraint] = None, temperature: float = 1.0):
    """log p(token | the constraint's tokens) of every position, f32 in tokens'
    shape, differentiable by scores."""
    return _TokenLogprobs.apply(scores, tokens, constraint, temperature)


def policy_loss(scores, tokens, old_logprobs, advantages, *, weights=None, ref_logprobs=None, clip_low: float = 0.2,
                clip_high: float = 0.2, kl_coef: float = 0.0, constraint: Optional[Constraint] = None,
                temperature: float = 1.0) -> PolicyLoss:
    """The clipped policy loss with a KL term:

        sum w (-min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_coef (e^d - d - 1)),
        r = exp(logp - old_logprobs), d = ref_logprobs - logp.

    old_logprobs, advantages, weights, ref_logprobs: tensors in tokens' shape,
    constants of the loss.  weights: None weighs every position 1 / tokens.numel();
    for a mean over the live positions give mask / mask.sum().  Where the two
    terms of the minimum are equal the gradient is the unclipped one's.

    With gradients enabled the scores' gradient is made in the same pass over
    them and kept (scores.numel() elements of their type) until backward(),
    which returns it as it is when the loss's own gradient is 1, and makes it
    anew, from the scores, for any other -- and where only one of the two passes
    is captured into a graph, or each into a graph of its own."""
    what = "policy_loss"
    lo, hi = _number(clip_low, "clip_low", what), _number(clip_high, "clip_high", what)
    if not 0 <= lo <= 1 or hi < 0:
        raise ValueError(f"{what}: clip_low must lie in [0, 1] and clip_high must not be negative")
    kl = _number(kl_coef, "kl_coef", what)
    if kl != 0 and ref_logprobs is None:
        raise ValueError(f"{what}: kl_coef needs ref_logprobs")
    return PolicyLoss(*_PolicyLoss.apply(scores, tokens, old_logprobs, advantages, weights, ref_logprobs, lo, hi, kl,
                                         constraint, temperature,
                                         torch.is_grad_enabled() and getattr(scores, "requires_grad", False)))


def preference_loss(scores, tokens, cu_seqlens, *, ref_logprobs=None, weights=None, beta: float = 0.1,
                    label_smoothing: float = 0.0, margin: float = 0.0, constraint: Optional[Constraint] = None,
                    temperature: float = 1.0) -> PreferenceLoss:
    """The preference loss on paired log ratios, over packed sequences.

    Positions (flattened) cu_seqlens[q] .. cu_seqlens[q + 1] are sequence q, its
    log-probability S_q the weighted sum of theirs; sequences 2 i and 2 i + 1
    are pair i's preferred and other answer:

        D_i = beta ((S_2i - ref_2i) - (S_2i+1 - ref_2i+1)) - margin
        loss = mean_i (1 - label_smoothing) softplus(-D_i) + label_smoothing softplus(D_i)

    cu_seqlens    int64 [2 * pairs + 1] on the GPU, non-decreasing (clamped to the
                  positions there are); positions of no sequence get no gradient
    ref_logprobs  [2 * pairs]: the reference model's sums, or None for 0
    weights       in tokens' shape or None for 1: 0 leaves prompts out, 1 / length
                  gives per-token means"""
    what = "preference_loss"
    ls = _number(label_smoothing, "label_smoothing", what)
    if not 0 <= ls <= 1:
        raise ValueError(f"{what}: label_smoothing must lie in [0, 1]")
    return PreferenceLoss(*_PreferenceLoss.apply(scores, tokens, cu_seqlens, ref_logprobs, weights,
                                                 _number(beta, "beta", what), ls, _number(margin, "margin", what),
                                                 constraint, temperature))


__all__ = ["token_logprobs", "policy_loss", "preference_loss", "PolicyLoss", "PreferenceLoss"]
