"""Which tokens each row of scores may take, as the operators on constrained
scores read it (``fmidx.losses``, ``fmidx.head``): the packed allowed-token bits
that ``FMIndex.allowed_mask(packed=True)`` and ``decode_step(packed=True)``
write, and the per-row mask values of ``fm_row_params`` that the processors
build (document_constrained_generation_causal_qwen.py:151-214).
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from .processors import FLAG_BITS, FLAG_EOS, FLAG_SPECIAL, FLAG_UNIGRAM, ROW_DTYPE


@dataclass(frozen=True)
class Constraint:
    """Rows of mask values, added to scores as fm_apply_boosts adds them.

    allowed   int32 [..., >= ceil(V / 32)]: the allowed-token bits of each row
    rows      uint8 [..., 32]: the rows' fm_row_params (``row_params``); None:
              a hard mask, 0 for the allowed tokens and -inf for the rest
    unigrams  int32 [>= ceil(V / 32)]: the corpus's tokens, for rows with FLAG_UNIGRAM
    eos       the token that rows with FLAG_EOS give v_eos

    A token whose mask value is -inf is out: its score is never used."""

    allowed: Optional[torch.Tensor] = None
    rows: Optional[torch.Tensor] = None
    unigrams: Optional[torch.Tensor] = None
    eos: int = -1

    def checked(self, n: int, vocab: int, device) -> "Constraint":
        """The same constraint as [n, words] / [n, 32] tensors with contiguous
        rows, or ValueError / TypeError."""
        words = (vocab + 31) // 32
        if self.allowed is None and self.rows is None:
            raise ValueError("Constraint: allowed bits or row records are needed")
        allowed, rows, uni = self.allowed, self.rows, self.unigrams
        for name, t, dt in (("allowed", allowed, torch.int32), ("rows", rows, torch.uint8),
                            ("unigrams", uni, torch.int32)):
            if t is None:
                continue
            if not isinstance(t, torch.Tensor) or t.dtype != dt:
                raise TypeError(f"Constraint.{name} must be a {dt} tensor")
            if t.device != device:
                raise ValueError(f"Constraint.{name} is on {t.device}, the scores on {device}")
        if allowed is not None:
            if allowed.dim() < 1 or allowed.shape[-1] < words or allowed.numel() != n * allowed.shape[-1]:
                raise ValueError(f"Constraint.allowed: {tuple(allowed.shape)} for {n} rows of at least {words} words")
            if allowed.dim() != 2:
                allowed = allowed.reshape(n, allowed.shape[-1])
            if n and (allowed.stride(1) != 1 or allowed.stride(0) < words):
                allowed = allowed.contiguous()
        if rows is not None:
            if rows.dim() < 1 or rows.shape[-1] != ROW_DTYPE.itemsize or rows.numel() != n * ROW_DTYPE.itemsize:
                raise ValueError(f"Constraint.rows: {tuple(rows.shape)} for {n} records of {ROW_DTYPE.itemsize} bytes")
            if rows.dim() != 2:
                rows = rows.reshape(n, ROW_DTYPE.itemsize)
            rows = rows.contiguous()
            if rows.data_ptr() % 8:
                rows = rows.clone()
        if uni is not None:
            if uni.dim() != 1 or uni.shape[0] < words:
                raise ValueError(f"Constraint.unigrams: {tuple(uni.shape)}, at least {words} words needed")
            uni = uni.contiguous()
        return Constraint(allowed, rows, uni, int(self.eos))


def row_params(n: int, *, base=0.0, v_dist=0.0, v_uni=0.0, v_eos=0.0, flags=FLAG_BITS, special=-1,
               device="cuda") -> torch.Tensor:
    """n fm_row_params as uint8 [n, 32]; each field a number or a tensor of n.
    Values are added in the scores' type: give them rounded to it, as the
    processors do."""
    def col(x, dtype):
        t = torch.as_tensor(x, device=device).to(dtype)
        return t.expand(n) if t.dim() == 0 else t.reshape(n)

    rec = torch.zeros((n, ROW_DTYPE.itemsize // 4), dtype=torch.int32, device=device)
    for i, x in enumerate((base, v_dist, v_uni, v_eos)):
        rec[:, i] = col(x, torch.float32).contiguous().view(torch.int32)
    rec[:, 4] = col(flags, torch.int32)
    rec[:, 6:8] = col(special, torch.int64).contiguous().view(torch.int32).reshape(n, 2)
    return rec.view(torch.uint8)


def prefix_constraint(index, tokens: torch.Tensor, vocab: int, shift: int = 10, lo=None, hi=None) -> Constraint:
    """The hard constraint at every position of given answers: position l of
    sequence b may take the tokens that follow tokens[b, :l] in the corpus (all
    of the corpus's tokens at l = 0).  One fused decode step per position over
    the batch (``FMIndex.decode_step``, packed), the state kept on the device.

    tokens    int64 [B, L] on the index's device; from a sequence's first
              token < 0 (padding) on, its positions are empty rows
    lo, hi    int64 [B]: the ranges the answers start from (``get_range_batch``
              of a forced prefix); None: the whole corpus
    Returns Constraint(allowed=int32 [B, L, ceil(vocab / 32)])."""
    if not isinstance(tokens, torch.Tensor):
        raise TypeError("prefix_constraint: tokens must be a tensor")
    if tokens.dim() != 2 or tokens.dtype != torch.int64:
        raise ValueError("prefix_constraint: tokens must be int64 [B, L]")
    if getattr(index, "sharded", False):
        raise ValueError("prefix_constraint: a doc-range shard knows only its own documents; OR the shards' bits")
    if vocab < 1:
        raise ValueError("prefix_constraint: vocab must be positive")
    for name, r in (("lo", lo), ("hi", hi)):
        if r is not None and not isinstance(r, torch.Tensor):
            raise TypeError(f"prefix_constraint: {name} must be a tensor")
        if r is not None and (r.dtype != torch.int64 or r.shape != tokens.shape[:1] or r.device != tokens.device):
            raise ValueError(f"prefix_constraint: {name} must be int64 [{tokens.shape[0]}] on {tokens.device}")
    if (lo is None) != (hi is None):
        raise ValueError("prefix_constraint: lo and hi go together")
    dev = torch.device("cuda", index.device)
    if tokens.device != dev:
        raise ValueError(f"prefix_constraint: tokens are on {tokens.device}, the index on {dev}")
    B, L = tokens.shape
    bits = torch.empty((B, L, (vocab + 31) // 32), dtype=torch.int32, device=dev)
    if B == 0 or L == 0:
        return Constraint(allowed=bits)
    with torch.cuda.device(dev):
        lo = torch.zeros(B, dtype=torch.int64, device=dev) if lo is None else lo.clone()
        hi = torch.full((B,), index.size(), dtype=torch.int64, device=dev) if hi is None else hi.clone()
        step = torch.empty((B, bits.shape[2]), dtype=torch.int32, device=dev)
        # a token that is no symbol of the corpus empties the range for good
        cols = tokens.masked_fill(tokens < 0, vocab).t().contiguous()
        bits[:, 0] = index.allowed_mask(lo, hi, vocab, shift, out=step, packed=True)
        for i in range(1, L):
            index.decode_step(cols[i - 1], lo, hi, step, vocab, shift, packed=True)
            bits[:, i] = step
        # a padded position itself is an empty row
        ended = (tokens < 0).cumsum(1) > 0
        bits.masked_fill_(ended.unsqueeze(2), 0)
    return Constraint(allowed=bits)


__all__ = ["Constraint", "row_params", "prefix_constraint", "FLAG_BITS", "FLAG_UNIGRAM", "FLAG_EOS", "FLAG_SPECIAL"]
