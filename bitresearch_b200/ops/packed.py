"""Attention inside the sequences of a packed batch, and the spans that it goes by.

A packed batch is ``N`` rows (tokens) of any number of sequences one behind the other. ``start[i]`` and
``end[i]`` (int32 ``[N]``) are the first row of row ``i``'s sequence and the row past its last one; a row of no
sequence (padding) has the empty span ``[i, i)``. The spans come from the sequences' offsets or from token ids in
which each document starts with BOS, are made once per batch, and serve the forward and backward of every layer.

Row ``i`` sees the rows ``j`` of its sequence with ``i - window < j <= i`` (``window=0``: all up to ``i``).
What a row does not see (other sequences, later rows, rows outside its window, padding rows) does not reach its results,
values that are no numbers included, nor do queries that do not see a key reach that key's gradients (a value that is no
number because of what its row does see may be infinite or NaN, whichever comes first); rows of no
sequence are left as they were in every output (zero in one that the call makes).
Spans must be those of sequences that follow one another; any other contents give wrong values but read and
write no row outside the tensors.

Calls run on the current stream of the tensors' device, in a captured graph too (once any kernel of this package
has run on that device), allocate only the outputs and the
backward's scratch when they are not given, and give the same bits for the same inputs. Wrong arguments raise ``ValueError``, outputs that
share memory with another argument ``RuntimeError``.
As with the other tensor-core kernels, results count only while the device status word is zero (``check_status``): once it
holds an error, attention calls leave their outputs as they were.
"""
from __future__ import annotations

import math

import torch

from ._ext import ext


def bounds_from_offsets(offsets: torch.Tensor, rows: int, start: torch.Tensor | None = None,
                        end: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``(start, end)`` of ``rows`` rows from ``offsets`` (int32 ``[sequences + 1]``, not decreasing): sequence
    ``s`` holds the rows ``offsets[s]`` to ``offsets[s + 1] - 1``. Empty sequences are allowed. Offsets that
    decrease or leave ``[0, rows]`` are reported through the device status word (``check_status``)."""
    return ext().bounds_from_offsets(offsets, rows, start, end)


def bounds_from_ids(ids: torch.Tensor, bos: int, start: torch.Tensor | None = None,
                    end: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``(start, end)`` of the ``B * T`` rows of ``ids`` (int32 ``[B, T]``): a sequence starts at every ``bos`` and
    at the first token of each of the ``B`` rows of ids. Fewer than 2^30 tokens."""
    return ext().bounds_from_ids(ids, bos, start, end)


def attention_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, start: torch.Tensor, end: torch.Tensor,
                  window: int = 0, scale: float | None = None, out: torch.Tensor | None = None,
                  lse: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``out[i, h] = sum_j softmax_j(scale q[i, h].k[j, g]) v[j, g]`` over the rows that ``i`` sees, ``g`` the kv
    head of ``h``, and ``lse`` (fp32 ``[H, N]``), the natural log of the softmax's denominator.

    ``q`` is ``[N, H, D]``, ``k`` and ``v`` ``[N, KV, D]`` with ``H`` a multiple of ``KV``, ``D`` 64 or 128, bf16
    or fp16; views with row and head strides of multiples of 8 elements are taken as they are (a fused QKV
    buffer, head-major storage). ``scale`` defaults to ``1 / sqrt(D)``."""
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale
    return ext().packed_attn_fwd(q, k, v, start, end, window, scale, out, lse)


def bwd_scratch(rows: int, heads: int) -> int:
    """Entries of the fp32 scratch of :func:`attention_bwd`, for both types and any number of kv heads."""
    return 5 * heads * ((rows + 127) // 128 * 128)  # a row's lse and delta; in fp16 also its factors' three bounds


def attention_bwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor, lse: torch.Tensor,
                  dout: torch.Tensor, start: torch.Tensor, end: torch.Tensor, window: int = 0,
                  scale: float | None = None, dq: torch.Tensor | None = None, dk: torch.Tensor | None = None,
                  dv: torch.Tensor | None = None,
                  scratch: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(dq, dk, dv)`` of :func:`attention_fwd` for the gradient ``dout`` of ``out``, with the ``out`` and ``lse``
    that it returned. Gradients of a kv head are summed over its query heads. ``scratch`` is fp32 memory of
    :func:`bwd_scratch` entries that no other call uses at the same time."""
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale
    return ext().packed_attn_bwd(q, k, v, out, lse, dout, start, end, window, scale, dq, dk, dv, scratch)
