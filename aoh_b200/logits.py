"""Logits on their way to the next token: penalties for repeated tokens, biases
and grammar masks.  ``ModelDecodeGraph`` (hf.py) runs them within its captured
step."""
from __future__ import annotations

import torch

from . import _lib


class TokenHistory:
    """Which tokens the prompt and the output of each sequence hold.

    ``counts`` (rows, vocab) int32: occurrences in the output, bit 31: in the
    prompt; ``seen`` (rows, ceil(vocab / 32)) int32: a bit per token of either.
    Updates are stream-ordered, need no host read and can be captured."""

    def __init__(self, rows: int, vocab: int, device=None):
        if not 0 <= rows < 1 << 31 or not 1 <= vocab < 1 << 31:
            raise ValueError("rows must be non-negative and vocab positive, both of 32 bits")
        self.device = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        self.rows, self.vocab = int(rows), int(vocab)
        self.counts = torch.zeros((self.rows, self.vocab), dtype=torch.int32, device=self.device)
        self.seen = torch.zeros((self.rows, -(-self.vocab // 32)), dtype=torch.int32, device=self.device)
        self.device = self.counts.device

    def reset(self, row: int | None = None) -> None:
        """Forget one row (a new sequence takes its place), or all."""
        at = slice(None) if row is None else row
        self.counts[at] = 0
        self.seen[at] = 0

    def add_prompt(self, ids: torch.Tensor, lengths: torch.Tensor | None = None) -> None:
        """Mark the prompts' tokens: ids (rows, n) int64 or int32, of which row r
        has lengths[r] (int32); ids outside [0, vocab), as padding, are left out."""
        self._add(ids, lengths, True)

    def append(self, ids: torch.Tensor, lengths: torch.Tensor | None = None) -> None:
        """Count the tokens put out: ids (rows,) or (rows, n), as in add_prompt."""
        self._add(ids.unsqueeze(1) if ids.dim() == 1 else ids, lengths, False)

    def _add(self, ids, lengths, prompt) -> None:
        if ids.dim() != 2 or ids.shape[0] != self.rows or ids.dtype not in (torch.int64, torch.int32) \
                or ids.device != self.device:
            raise ValueError(f"ids must be int64 or int32 ({self.rows}, n) on {self.device}, "
                             f"got {ids.dtype} {tuple(ids.shape)} on {ids.device}")
        if lengths is not None and (lengths.dtype != torch.int32 or tuple(lengths.shape) != (self.rows,)
                                    or lengths.device != self.device or not lengths.is_contiguous()):
            raise ValueError(f"lengths must be contiguous int32 ({self.rows},) on {self.device}")
        if ids.shape[1] >= 1 << 31:
            raise ValueError(f"{ids.shape[1]} ids of a row are more than 32 bits count")
        if ids.numel() == 0:
            return
        if ids.shape[1] > 1 and ids.stride(1) != 1:
            ids = ids.contiguous()
        _lib.launch(self.device, _lib.lib().aoh_history_add, "aoh_history_add", self.counts.data_ptr(),
                    self.seen.data_ptr(), self.rows, self.vocab, ids.data_ptr(), ids.dtype == torch.int64, ids.stride(0),
                    ids.shape[1], None if lengths is None else lengths.data_ptr(), prompt)


_DTYPES = {torch.bfloat16: _lib.BF16, torch.float32: _lib.F32}


def _row_tensor(x, name: str, rows: int, device) -> int:
    if x.dtype != torch.float32 or x.shape != (rows,) or x.device != device or not x.is_contiguous():
        raise ValueError(f"{name} must be a number or a contiguous float32 tensor ({rows},) on {device}")
    return x.data_ptr()


def penalize_logits(logits: torch.Tensor, history: TokenHistory | None = None, *, repetition=None, presence=None,
                    frequency=None, bias: tuple[torch.Tensor, torch.Tensor] | None = None,
                    allowed: torch.Tensor | None = None, allowed_rows: torch.Tensor | None = None,
                    out: torch.Tensor | None = None, greedy: bool = False):
    """Penalties, biases and a grammar's mask on logits (N, V), bf16 or f32.

    In this order, in fp32: tokens of the prompt or output are divided by
    ``repetition`` (multiplied where not positive); ``frequency`` times its count
    and ``presence`` are taken from a token of the output; ``bias`` = (ids (N, K)
    int32, values (N, K) float32, K <= 4096) is added, ids outside [0, V)
    (padding) left out and repeated ids added up; tokens whose bit of ``allowed`` is 0 become -inf.
    repetition (> 0), presence, frequency: numbers or float32 (N,); they need
    ``history``.  allowed (M, ceil(V / 32)) int32, bit t % 32 of word t // 32 for
    token t; row n has allowed[n], or allowed[allowed_rows[n]] (int32 (N,); an
    index outside [0, M) means no mask).
    out: float32 (default: a new tensor) or bf16 (N, V), or the logits themselves;
    it must not overlap them otherwise.  With ``greedy`` returns (out, ids (N,)
    int64): the largest fp32 result, the lowest id of equal ones, NaN above every
    number, 0 where nothing is allowed."""
    # a call's Python is most of the time that a single row takes: each property is read once
    shape, strides, dev = logits.shape, logits.stride(), logits.device
    if len(shape) != 2 or not logits.is_cuda:
        raise ValueError("logits must be a CUDA tensor (N, V)")
    N, V = shape
    code = _DTYPES.get(logits.dtype)
    if code is None:
        raise ValueError(f"logits must be torch.bfloat16 or torch.float32, got {logits.dtype}")
    if V < 1 or (V > 1 and strides[1] != 1):
        raise ValueError("the vocabulary of logits must be contiguous and not empty")
    # pointers, 0 where there is none, and the numbers that stand for a missing one
    counts = seen = rep = pres = freq = 0
    rep_s, pres_s, freq_s = 1.0, 0.0, 0.0
    if history is None:
        if repetition is not None or presence is not None or frequency is not None:
            raise ValueError("penalties need a history")
    else:
        if history.rows != N or history.vocab != V or history.device != dev:
            raise ValueError(f"history of ({history.rows}, {history.vocab}) on {history.device} for logits {(N, V)} "
                             f"on {dev}")
        counts, seen = history.counts.data_ptr(), history.seen.data_ptr()
        if repetition is not None:
            if isinstance(repetition, torch.Tensor):
                rep = _row_tensor(repetition, "repetition", N, dev)
            elif repetition > 0:
                rep_s = float(repetition)
            else:
                raise ValueError("repetition must be positive")
        if presence is not None:
            if isinstance(presence, torch.Tensor):
                pres = _row_tensor(presence, "presence", N, dev)
            else:
                pres_s = float(presence)
        if frequency is not None:
            if isinstance(frequency, torch.Tensor):
                freq = _row_tensor(frequency, "frequency", N, dev)
            else:
                freq_s = float(frequency)
    ids = values = K = 0
    if bias is not None:
        i, v = bias
        K = i.shape[1] if i.dim() == 2 else -1
        if i.dtype != torch.int32 or v.dtype != torch.float32 or i.shape != (N, K) or v.shape != (N, K) \
                or i.device != dev or v.device != dev or not i.is_contiguous() or not v.is_contiguous():
            raise ValueError(f"bias must be contiguous int32 ids and float32 values of one shape ({N}, K) on {dev}")
        ids, values = i.data_ptr(), v.data_ptr()
    mask = rows = M = 0
    if allowed is not None:
        words = -(-V // 32)
        if allowed.dtype != torch.int32 or allowed.dim() != 2 or allowed.shape[1] != words or allowed.device != dev \
                or not allowed.is_contiguous():
            raise ValueError(f"allowed must be contiguous int32 (rows, {words}) on {dev}")
        mask, M = allowed.data_ptr(), allowed.shape[0]
        if allowed_rows is None and M != N:
            raise ValueError(f"{M} mask rows for {N} rows of logits need allowed_rows")
    if allowed_rows is not None:
        if allowed is None or allowed_rows.dtype != torch.int32 or allowed_rows.shape != (N,) \
                or allowed_rows.device != dev or not allowed_rows.is_contiguous():
            raise ValueError(f"allowed_rows must be contiguous int32 ({N},) on {dev}, with allowed")
        rows = allowed_rows.data_ptr()
    if out is None:
        out = logits.new_empty(shape, dtype=torch.float32)
        out_stride, out_code = V, _lib.F32
    else:
        out_stride, out_code = out.stride(0) if out.dim() == 2 else 0, _DTYPES.get(out.dtype)
        if out.shape != shape or out.device != dev or (V > 1 and out.stride(1) != 1) or (N > 1 and out_stride < V):
            raise ValueError(f"out must be ({N}, {V}) on {dev}, its vocabulary contiguous and its rows apart")
        if out_code is None:
            raise ValueError(f"out must be torch.bfloat16 or torch.float32, got {out.dtype}")
    best = logits.new_empty(N, dtype=torch.int64) if greedy else None
    if N:
        _lib.launch(dev, _lib.lib().aoh_logits_penalize, "aoh_logits_penalize", _lib.pack_logits(
            logits.data_ptr(), out.data_ptr(), best.data_ptr() if greedy else 0, counts, seen, rep, pres, freq, ids,
            values, mask, rows, strides[0], out_stride, N, V, code, out_code, K, M, rep_s, pres_s, freq_s, 0))
    return (out, best) if greedy else out
