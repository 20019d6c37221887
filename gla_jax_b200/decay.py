"""Linear attention with one decay per head: ``S_t = exp(g_t) S_{t-1} + k_t (x) v_t``, ``o_t = q_t S_t`` with ``g`` a number
per token and head, the sibling of ``chunk_gla`` (a decay per key feature) with the same argument order.

    chunk_decay_attention(hidden_init, log_decay, value, key, query)                     prompts and training
    chunk_decay_attention_packed(hidden_init, log_decay, value, key, query, cu_seqlens)  the same, sequences end to end
    decay_attention_step(state, log_decay, value, key, query)                            one token

The decay being a scalar per head, any length is taken as it is (there is no chunk size to choose), keys and values may have
different head sizes, and keys and queries may be shared by several value heads.  No counterpart in the reference, whose
operators have a gate per key feature (gla.py:26-47).  There is no CPU path: CPU tensors raise.
"""
from __future__ import annotations

from typing import Tuple

import torch

from . import _lib
from .gla import _DT, _refuse_parents, _stream


def _refused(what, hidden, log_decay, value, key, query, packed):
    """The native host path did not take these arguments: raise the error that says why."""
    if not value.is_cuda:
        raise RuntimeError("gla_jax_b200 operators need CUDA tensors; there is no CPU fallback")
    dims = (3,) if packed else (3, 4)
    if value.dim() not in dims or key.dim() != value.dim():
        raise ValueError(f"{what}: value must be {'(T,H,Dv)' if packed else '(T,H,Dv) or (B,T,H,Dv)'} and key, query (..,T,Hk,Dk), got "
                         f"{tuple(value.shape)}, {tuple(key.shape)}")
    if key.shape != query.shape or key.shape[:-2] != value.shape[:-2]:
        raise ValueError(f"{what}: key and query must have one shape and value's tokens ({tuple(key.shape)}, {tuple(query.shape)}, "
                         f"{tuple(value.shape)})")
    H, Hk = value.shape[-2], key.shape[-2]
    if min(*key.shape[-2:], *value.shape[-2:]) < 1 or H % Hk or (value.dim() == 4 and value.shape[0] < 1):
        raise ValueError(f"{what}: the number of value heads ({H}) must be a multiple of that of key heads ({Hk}), and no size may be 0")
    if tuple(log_decay.shape) not in ((H,), tuple(value.shape[:-1])):
        raise ValueError(f"{what}: log_decay must be {tuple(value.shape[:-1])} or ({H},), got {tuple(log_decay.shape)}")
    if value.dtype not in _DT:
        raise TypeError(f"unsupported dtype {value.dtype}: float32 and bfloat16 are implemented")
    if key.dtype != value.dtype or query.dtype != value.dtype or hidden.dtype not in (value.dtype, torch.float32):
        raise TypeError(f"{what}: value, key and query must share one dtype, which hidden must have too, or float32")
    if not packed:
        want = (*value.shape[:-3], H, key.shape[-1], value.shape[-1])
        if tuple(hidden.shape) != want:
            raise ValueError(f"{what}: hidden must be {want}, got {tuple(hidden.shape)}")
    _stream(value.device)
    raise ValueError(f"{what}: all arrays must be real and on {value.device}")


def chunk_decay_attention(hidden_init, log_decay, value, key, query) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(hidden_final, out)`` of linear attention with a decay per head, in chunks; differentiable in every argument.

    ``value`` (B, T, H, Dv), ``key`` and ``query`` (B, T, Hk, Dk) with ``H`` a multiple of ``Hk`` (value head ``h`` uses key
    head ``h // (H // Hk)``), ``hidden_init`` (B, H, Dk, Dv); without the batch axis everywhere, one sequence.
    ``log_decay`` (B, T, H), or (H,) for decays that do not depend on the token, is converted to float32; ``-inf`` resets the
    state.  Head sizes are multiples of 8 up to 256, ``T`` is any, ``H`` up to 16383.  float32 or bfloat16 (products of a query
    and a key below 2^62, as of a value and its cotangent); ``hidden_init`` (and with it
    ``hidden_final``) may be float32 beside bfloat16 arrays, for a state that ``decay_attention_step`` goes on with."""
    r = _lib.native().chunk_decay(hidden_init, log_decay, value, key, query, None)
    return r if r is not None else _refused("chunk_decay_attention", hidden_init, log_decay, value, key, query, False)


def chunk_decay_attention_packed(hidden_init, log_decay, value, key, query, cu_seqlens) -> Tuple[torch.Tensor, torch.Tensor]:
    """``chunk_decay_attention`` for sequences of any length (0 included) packed end to end on one time axis.

    ``value`` (T, H, Dv), ``key`` and ``query`` (T, Hk, Dk), ``log_decay`` (T, H) or (H,), ``hidden_init``
    (nseq, H, Dk, Dv); ``cu_seqlens`` holds the ``nseq + 1`` token offsets.  As a list or CPU tensor they are checked: they
    rise from 0 to T.  A CUDA tensor is used as it is, without a round trip to the host: offsets that fall or leave [0, T] are
    held inside and reported by ``check_device``; the last may be less than T, and the rows behind it are zeros in ``out`` and
    in the gradients."""
    cu = cu_seqlens if torch.is_tensor(cu_seqlens) else torch.tensor(cu_seqlens, dtype=torch.int64)
    what, T = "chunk_decay_attention_packed", value.shape[0] if value.dim() else 0
    if cu.dim() != 1 or cu.numel() < 2 or cu.is_floating_point() or cu.is_complex():
        raise ValueError(f"{what}: cu_seqlens must hold nseq + 1 whole numbers on one axis, nseq at least 1")
    if not cu.is_cuda:
        if int(cu[0]) != 0 or int(cu[-1]) != T or bool((cu[1:] < cu[:-1]).any()):
            raise ValueError(f"{what}: cu_seqlens must rise from 0 to {T}")
        if value.is_cuda:
            cu = cu.to(torch.int32).to(value.device)
    elif cu.dtype != torch.int32:
        # (what 32 bits do not hold leaves [0, T] on the same side)
        cu = (cu.clamp(-1, 2 ** 31 - 1) if cu.dtype == torch.int64 else cu).to(torch.int32)
    r = _lib.native().chunk_decay(hidden_init, log_decay, value, key, query, cu) if value.is_cuda else None
    if r is not None:
        return r
    if value.is_cuda and value.dim() == 3 and key.dim() == 3:
        if cu.device != value.device:
            raise ValueError(f"{what}: cu_seqlens must be on {value.device} or the CPU, got {cu.device}")
        want = (cu.numel() - 1, value.shape[-2], key.shape[-1], value.shape[-1])
        if tuple(hidden_init.shape) != want:
            raise ValueError(f"{what}: hidden_init must be (nseq, H, Dk, Dv) = {want}, got {tuple(hidden_init.shape)}")
    return _refused(what, hidden_init, log_decay, value, key, query, True)


def decay_attention_step(state, log_decay, value, key, query, out_dtype=None, parents=None):
    """One token of the recurrence for a batch of requests, as ``decode_step`` for a decay per head.

    ``state`` (B, H, Dk, Dv) float32 is updated IN PLACE; ``value`` (B, H, Dv), ``key`` and ``query`` (B, Hk, Dk),
    ``log_decay`` (B, H); returns ``out`` (B, H, Dv) in ``out_dtype`` (default: value's dtype).  Not differentiable.

    ``parents`` (requests, beams), with ``B = requests * beams``: every row goes on from the state of the row of its
    request that ``parents`` names (see ``reorder_states``), in the same pass; up to 32 beams."""
    out = _lib.native().decay_step(state, log_decay, value, key, query, out_dtype, parents)
    if out is not None:
        return out
    what = "decay_attention_step"
    if not value.is_cuda or not state.is_cuda:
        raise RuntimeError(f"{what} needs CUDA tensors on one device; there is no CPU fallback")
    if state.dtype != torch.float32 or not state.is_contiguous() or state.dim() != 4:
        raise TypeError(f"{what}: state must be a contiguous float32 (B, H, Dk, Dv) tensor")
    B, H, Dk, Dv = state.shape
    if tuple(value.shape) != (B, H, Dv) or key.dim() != 3 or key.shape != query.shape or key.shape[0] != B or key.shape[2] != Dk \
            or key.shape[1] < 1 or H % key.shape[1] or tuple(log_decay.shape) != (B, H):
        raise ValueError(f"{what}: expected state (B, H, Dk, Dv), log_decay (B, H), value (B, H, Dv) and key, query (B, Hk, Dk), "
                         "H a multiple of Hk")
    if key.dtype != value.dtype or query.dtype != value.dtype or value.dtype not in _DT or (out_dtype or value.dtype) not in _DT:
        raise TypeError(f"{what}: value, key, query must share a dtype, float32 or bfloat16")
    _refuse_parents(what, parents, state)
    _stream(value.device)
    raise ValueError(f"{what}: all arrays must be real and on {state.device}")


__all__ = ["chunk_decay_attention", "chunk_decay_attention_packed", "decay_attention_step"]
