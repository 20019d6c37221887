"""Beam search over recurrent states: the selection of the next beams and the moving of states to where their beams went.

What a beam carries in a recurrent model is its state (there is no cache of keys and values).  Rows of a state tensor are
(request, beam); ``parents`` (requests, beams) names for every beam the beam of its request that it goes on from.  One token
of a search over ``decode_step`` or ``decay_attention_step`` is

    out = decay_attention_step(state, log_decay, value, key, query, parents=parents)   # moves the states on its way
    scores, tokens, parents = beam_select(logits_of(out), scores, finished=finished)

and ``reorder_states`` moves whatever else is kept per beam.  No counterpart in the reference, which has no decoding loop.
There is no CPU path: CPU tensors raise.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from .gla import _DT, _stream


def beam_select(logits, scores, num_select: Optional[int] = None, finished=None,
                pad_token: int = 0) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The ``num_select`` (default: the number of beams) best continuations of each request.

    ``logits`` (N, K, V) float32 or bfloat16, ``scores`` (N, K): log-probabilities of the beams so far, finite or ``-inf``.
    Continuations rank by ``scores + log_softmax(logits)``, formed in 64 bits from float32 scores and sums of float32
    exponentials, the lowest (beam, token) first among equal ones.  Returns the totals (N, M) in float32, tokens (N, M) int64 and parents (N, M) int32, best first.

    ``-inf`` or NaN masks a token; a beam without any token left, or with a score of ``-inf`` or NaN, offers totals of
    ``-inf``.  ``finished`` (N, K) bool: such a beam goes on with ``pad_token`` alone, at its score.  K and M are at most
    32.  Not differentiable."""
    m = logits.shape[1] if num_select is None and logits.dim() == 3 else num_select
    if logits.is_cuda and m is not None:
        r = _lib.native().beam_select(logits, scores, int(m), finished, int(pad_token))
        if r is not None:
            return r
    if not logits.is_cuda:
        raise RuntimeError("gla_jax_b200 operators need CUDA tensors; there is no CPU fallback")
    if logits.dim() != 3 or tuple(scores.shape) != tuple(logits.shape[:2]) or 0 in logits.shape[1:]:
        raise ValueError(f"beam_select: logits must be (N, K, V) and scores (N, K), got {tuple(logits.shape)}, {tuple(scores.shape)}")
    N, K, V = logits.shape
    if logits.dtype not in _DT or not scores.is_floating_point():
        raise TypeError(f"beam_select: logits must be float32 or bfloat16 and scores floating, got {logits.dtype}, {scores.dtype}")
    if K > 32 or not 1 <= m <= min(32, K * V):
        raise ValueError(f"beam_select: at most 32 beams, and num_select from 1 to 32 and to the {K * V} continuations there are; got "
                         f"{K} beams, num_select {m}")
    if not 0 <= pad_token < V:
        raise ValueError(f"beam_select: pad_token must be one of the {V} tokens, got {pad_token}")
    if finished is not None and (tuple(finished.shape) != (N, K) or finished.dtype != torch.bool):
        raise ValueError(f"beam_select: finished must be a bool tensor ({N}, {K})")
    _stream(logits.device)
    raise ValueError(f"beam_select: all arrays must be on {logits.device}")


def reorder_states(states, parents) -> None:
    """Move rows of ``states`` to where ``parents`` (N, K) says, IN PLACE: row ``n K + j`` becomes what row
    ``n K + parents[n, j]`` was.

    ``states``: a tensor or a list of tensors (N K, ...), contiguous, of any type, that do not overlap.  All of them move
    in one launch; rows that stay where they are are neither read nor written.  Up to 32 beams.  Entries of ``parents``
    outside [0, K) are held inside and reported by ``check_device``."""
    states = [states] if torch.is_tensor(states) else list(states)
    if torch.is_tensor(parents) and parents.is_cuda and _lib.native().reorder_states(states, parents):
        return
    if not parents.is_cuda or any(not s.is_cuda for s in states):
        raise RuntimeError("gla_jax_b200 operators need CUDA tensors; there is no CPU fallback")
    if parents.dim() != 2 or parents.shape[1] == 0:
        raise ValueError(f"reorder_states: parents must be (requests, beams), got {tuple(parents.shape)}")
    if parents.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"reorder_states: parents must be int32 or int64, got {parents.dtype}")
    _stream(parents.device)
    for s in states:
        if s.dim() < 1 or s.shape[0] != parents.numel() or not s.is_contiguous() or s.device != parents.device:
            raise ValueError(f"reorder_states: states must be contiguous, on {parents.device}, with {parents.numel()} rows; got "
                             f"{tuple(s.shape)} on {s.device}")
        if s.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("reorder_states works in place and is not differentiable: a state requires a gradient")
    raise ValueError("reorder_states: the states overlap in memory")


__all__ = ["beam_select", "reorder_states"]
