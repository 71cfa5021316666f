"""Rotary embedding by positions with several axes.

``rope_axes_qk`` stands beside ``rope_qk`` (attention.py): that one applies a
model's bf16 cos / sin with the rounding steps of its torch ops; this one takes
the positions themselves -- one axis, or time, height and width for image and
video tokens -- and computes in fp32, rounding once.  Positions are not cache
indices: after an eviction they go on counting (``AoHKVCache.tokens_seen``).
"""
from __future__ import annotations

import functools

import torch

from . import _lib
from .cache import _dtype_code

@functools.lru_cache(maxsize=64)
def _sections(sections: tuple[int, ...]):
    if not 1 <= len(sections) <= 8:
        raise ValueError(f"1 to 8 sections, got {len(sections)}")
    if max(map(abs, sections)) > 1 << 20:
        raise ValueError(f"bad sections {sections}")
    return sections + (0,) * (8 - len(sections)), len(sections), sum(sections)


def _ptr(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.data_ptr()


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
    ``scaling`` multiplies cos and sin.  Returns contiguous (q, k).
    """
    if q.dim() != 4 or k.dim() != 4:
        raise ValueError("q must be (B, C, Hq, D) and k (B, C, G, D)")
    B, n, Hq, D = q.shape
    G = k.shape[2]
    qs, ks = q.stride(), k.stride()
    if k.shape[0] != B or k.shape[1] != n or k.shape[3] != D:
        raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} must agree in all but their heads")
    dt, dev = q.dtype, q.device
    code = _dtype_code(dt)
    if not q.is_cuda or k.dtype != dt or k.device != dev:
        raise ValueError("q and k must be CUDA tensors of one dtype on one device")
    if qs[3] != 1 or ks[3] != 1:
        raise ValueError("the head dimension of q and k must be contiguous")
    secs, A, half = _sections(tuple(int(s) for s in sections))
    if positions.shape != (A, B, n):
        raise ValueError(f"positions must have shape (axes, B, C) = {(A, B, n)}, got {tuple(positions.shape)}")
    if positions.dtype not in (torch.int64, torch.int32) or positions.device != dev:
        raise ValueError("positions must be int64 or int32 on q's device")
    if inv_freq.dtype != torch.float32 or inv_freq.device != dev or inv_freq.shape != (half,) \
            or not inv_freq.is_contiguous():
        raise ValueError(f"inv_freq must be a contiguous float32 tensor of sum(sections) = {half} on q's device")
    if (q_norm_weight is None) != (k_norm_weight is None):
        raise ValueError("give both norm weights or neither")
    ws = [None, None]
    if q_norm_weight is not None:
        for i, w in enumerate((q_norm_weight, k_norm_weight)):
            if w.shape != (D,) or w.device != dev:
                raise ValueError(f"norm weights must be ({D},) on q's device")
            ws[i] = w.to(dt).contiguous()
    q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
    if B == 0 or n == 0:
        return q_out, k_out
    if D == 0 or Hq == 0 or G == 0:
        raise ValueError("q and k must have heads and dimensions")
    args = _lib.pack_rope_axes(
        q.data_ptr(), k.data_ptr(), positions.data_ptr(), inv_freq.data_ptr(), _ptr(ws[0]), _ptr(ws[1]),
        q_out.data_ptr(), k_out.data_ptr(), *qs[:3], *ks[:3], *positions.stride(), *secs, A, bool(interleaved), code,
        positions.dtype == torch.int64, B, n, Hq, G, D, eps, scaling, 0)
    _lib.launch(dev, _lib.lib().aoh_rope_axes_qk, "aoh_rope_axes_qk", args)
    return q_out, k_out
