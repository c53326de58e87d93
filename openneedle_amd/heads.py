"""Norms and rotation of the heads of q and k for a batch of tokens, on the device.

The reference does this for one token inside its step (needle2/csrc/engine.cpp:994-1004), with angles in 32 bits from the
host; here the angles are formed in 64 bits on the device, for any positions.
"""
from __future__ import annotations

import numpy as np

from . import _ffi
from ._ffi import addr, check
from .device import stream_ptr


def rotary_frequencies(theta: float, rotary: int) -> np.ndarray:
    """Angle per position of dimensions ``j`` and ``j + rotary / 2``: fp64 ``theta ** (-2 j / rotary)``."""
    return float(theta) ** (-np.arange(rotary // 2, dtype=np.float64) * 2.0 / max(rotary, 1))


def rotate_heads(d_q, d_k, heads: int, kvheads: int, head_dim: int, tokens: int, d_positions=None, d_freq=None,
                 rotary: int = 0, d_q_gain=None, d_k_gain=None, eps: float = 1e-6, q_stride: int = 0, k_stride: int = 0,
                 d_q_out=None, d_k_out=None, q_out_stride: int = 0, k_out_stride: int = 0, stream=None) -> None:
    """Every head of q (device fp32 ``[tokens][heads][head_dim]``) and of k (``kvheads`` heads) normed over its values and
    times ``1 + gain`` (``d_q_gain``, ``d_k_gain``: device fp32 ``[head_dim]``; None: not normed), then its dimensions
    ``j`` and ``j + rotary / 2`` turned by ``d_positions[token] * d_freq[j]`` (device int32 and fp64). A stride is the
    floats from one token's row to the next (0: rows without gaps), so q and k may lie in the rows of one projection.
    Outputs default to the inputs' own places. ``heads`` or ``kvheads`` 0: no q or k. A token at a negative position is
    left out. Capturable."""
    qs, ks = q_stride or heads * head_dim, k_stride or kvheads * head_dim
    qo, qos = (d_q, qs) if d_q_out is None else (d_q_out, q_out_stride or heads * head_dim)
    ko, kos = (d_k, ks) if d_k_out is None else (d_k_out, k_out_stride or kvheads * head_dim)
    check(_ffi.lib().needle2_gpu_heads(addr(d_q), int(qs), addr(qo), int(qos), int(heads), addr(d_k), int(ks), addr(ko),
                                       int(kos), int(kvheads), int(head_dim), int(tokens), addr(d_positions),
                                       addr(d_q_gain), addr(d_k_gain), float(eps), addr(d_freq), int(rotary),
                                       stream_ptr(stream)), "heads")
