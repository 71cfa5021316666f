"""Rotary embedding by positions with several axes.

``rope_axes_qk`` stands beside ``rope_qk`` (attention.py): that one applies a
model's bf16 cos / sin with the rounding steps of its torch ops; this one takes
the positions themselves -- one axis, or time, height and width for image and
video tokens -- and computes in fp32, rounding once.  Positions are not cache
indices: after an eviction they go on counting (``AoHKVCache.tokens_seen``).
"""
from __future__ import annotations

import torch

from . import _lib

_DTYPES = {torch.bfloat16: _lib.BF16, torch.float32: _lib.F32}
_POSITIONS_64 = {torch.int64: 1, torch.int32: 0}


_known_sections: dict[tuple, tuple] = {}


def _sections(sections: tuple):
    """(the sections padded to the 8 of the call's arguments, how many, their sum)."""
    values = tuple(int(s) for s in sections)
    if not 1 <= len(values) <= 8:
        raise ValueError(f"1 to 8 sections, got {len(values)}")
    if max(map(abs, values)) > 1 << 20:
        raise ValueError(f"bad sections {values}")
    found = values + (0,) * (8 - len(values)), len(values), sum(values)
    # only plain numbers are kept: a tensor is looked up by its identity, and its value may change
    if len(_known_sections) < 64 and all(type(s) is int for s in sections):
        _known_sections[sections] = found
    return found


def rope_axes_qk(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, sections, *,
                 interleaved: bool = False, q_norm_weight: torch.Tensor | None = None,
                 k_norm_weight: torch.Tensor | None = None, eps: float = 1e-6,
                 scaling: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """Optional per-head RMSNorm and the rotation of q and k by their positions.

    q (B, C, Hq, D), k (B, C, G, D): bf16 or f32, any strides with D contiguous
    (views of a fused projection need no copy), D even and at most 256.
    positions (A, B, C): int64 or int32, one position per axis.  inv_freq (half,)
    float32: the model's rotary frequencies; dimensions i and i + half turn by
    positions[axis(i)] * inv_freq[i], those from 2 * half on stay.
    ``sections``: A counts that sum to half.  The frequencies take their axes
    section by section, or, with ``interleaved``, in turn: frequency i takes axis
    a = i mod A while i < A * sections[a], else axis 0.
    Norm weights (D,): both of q's type, or of another, then taken in fp32.
    ``scaling`` multiplies cos and sin.  Returns contiguous (q, k).
    """
    # a call's Python is most of the time that a single token takes: each property is read once
    shape, k_shape, qs, ks = q.shape, k.shape, q.stride(), k.stride()
    if len(shape) != 4 or len(k_shape) != 4:
        raise ValueError("q must be (B, C, Hq, D) and k (B, C, G, D)")
    B, n, Hq, D = shape
    G = k_shape[2]
    if k_shape[0] != B or k_shape[1] != n or k_shape[3] != D:
        raise ValueError(f"q {tuple(shape)} and k {tuple(k_shape)} must agree in all but their heads")
    dt, dev = q.dtype, q.device
    code = _DTYPES.get(dt)
    if code is None:
        raise ValueError(f"dtype must be torch.bfloat16 or torch.float32, got {dt}")
    if not q.is_cuda or k.dtype != dt or k.device != dev:
        raise ValueError("q and k must be CUDA tensors of one dtype on one device")
    if qs[3] != 1 or ks[3] != 1:
        raise ValueError("the head dimension of q and k must be contiguous")
    if type(sections) is not tuple:
        sections = tuple(sections)
    secs, A, half = _known_sections.get(sections) or _sections(sections)
    if positions.shape != (A, B, n):
        raise ValueError(f"positions must have shape (axes, B, C) = {(A, B, n)}, got {tuple(positions.shape)}")
    wide = _POSITIONS_64.get(positions.dtype)
    if wide is None or positions.device != dev:
        raise ValueError("positions must be int64 or int32 on q's device")
    if inv_freq.dtype != torch.float32 or inv_freq.device != dev or inv_freq.shape != (half,) \
            or not inv_freq.is_contiguous():
        raise ValueError(f"inv_freq must be a contiguous float32 tensor of sum(sections) = {half} on q's device")
    qw, kw, norm_f32 = 0, 0, False
    if q_norm_weight is not None or k_norm_weight is not None:
        if q_norm_weight is None or k_norm_weight is None:
            raise ValueError("give both norm weights or neither")
        for w in (q_norm_weight, k_norm_weight):
            if w.shape != (D,) or w.device != dev:
                raise ValueError(f"norm weights must be ({D},) on q's device")
        # of q's type as they are, of any other in fp32: none is rounded to bf16; held here until the launch
        norm_f32 = q_norm_weight.dtype != dt or k_norm_weight.dtype != dt
        if norm_f32:
            q_norm_weight, k_norm_weight = q_norm_weight.float(), k_norm_weight.float()
        q_norm_weight, k_norm_weight = q_norm_weight.contiguous(), k_norm_weight.contiguous()
        qw, kw = q_norm_weight.data_ptr(), k_norm_weight.data_ptr()
    q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
    if B == 0 or n == 0:
        return q_out, k_out
    if D == 0 or Hq == 0 or G == 0:
        raise ValueError("q and k must have heads and dimensions")
    _lib.launch(dev, _lib.lib().aoh_rope_axes_qk, "aoh_rope_axes_qk", _lib.pack_rope_axes(
        q.data_ptr(), k.data_ptr(), positions.data_ptr(), inv_freq.data_ptr(), qw, kw, q_out.data_ptr(), k_out.data_ptr(),
        qs[0], qs[1], qs[2], ks[0], ks[1], ks[2], *positions.stride(), *secs, A, bool(interleaved), code, wide, B, n, Hq,
        G, D, eps, scaling, norm_f32))
    return q_out, k_out
