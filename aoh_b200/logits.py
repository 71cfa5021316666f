"""Logits on their way to the next token: penalties for repeated tokens, biases
and grammar masks.  ``ModelDecodeGraph`` (hf.py) runs them within its captured
step."""
from __future__ import annotations

import torch

from . import _lib
from .cache import _dtype_code


class TokenHistory:
    """Which tokens the prompt and the output of each sequence hold.

    ``counts`` (rows, vocab) int32: occurrences in the output, bit 31: in the
    prompt; ``seen`` (rows, ceil(vocab / 32)) int32: a bit per token of either.
    Updates are stream-ordered, need no host read and can be captured."""

    def __init__(self, rows: int, vocab: int, device=None):
        if rows < 0 or vocab < 1:
            raise ValueError("rows must be non-negative and vocab positive")
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
        if ids.numel() == 0:
            return
        if ids.shape[1] > 1 and ids.stride(1) != 1:
            ids = ids.contiguous()
        _lib.launch(self.device, _lib.lib().aoh_history_add, "aoh_history_add", self.counts.data_ptr(),
                    self.seen.data_ptr(), self.rows, self.vocab, ids.data_ptr(), ids.dtype == torch.int64, ids.stride(0),
                    ids.shape[1], None if lengths is None else lengths.data_ptr(), prompt)


def _ptr(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.data_ptr()


def _per_row(x, name: str, rows: int, device, neutral: float):
    """(pointer or 0, scalar) of a penalty given as a number, a (rows,) tensor or None."""
    if x is None:
        return 0, neutral
    if isinstance(x, torch.Tensor):
        if x.dtype != torch.float32 or x.shape != (rows,) or x.device != device or not x.is_contiguous():
            raise ValueError(f"{name} must be a number or a contiguous float32 tensor ({rows},) on {device}")
        return x.data_ptr(), neutral
    return 0, float(x)


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
    if logits.dim() != 2 or not logits.is_cuda:
        raise ValueError("logits must be a CUDA tensor (N, V)")
    N, V = logits.shape
    dev = logits.device
    code = _dtype_code(logits.dtype)
    if V < 1 or (V > 1 and logits.stride(1) != 1):
        raise ValueError("the vocabulary of logits must be contiguous and not empty")
    if history is None:
        if repetition is not None or presence is not None or frequency is not None:
            raise ValueError("penalties need a history")
    elif history.rows != N or history.vocab != V or history.device != dev:
        raise ValueError(f"history of ({history.rows}, {history.vocab}) on {history.device} for logits {(N, V)} on {dev}")
    if repetition is not None and not isinstance(repetition, torch.Tensor) and not repetition > 0:
        raise ValueError("repetition must be positive")
    rep, rep_s = _per_row(repetition, "repetition", N, dev, 1.0)
    pres, pres_s = _per_row(presence, "presence", N, dev, 0.0)
    freq, freq_s = _per_row(frequency, "frequency", N, dev, 0.0)
    ids = values = None
    K = 0
    if bias is not None:
        ids, values = bias
        K = ids.shape[1] if ids.dim() == 2 else -1
        if ids.dtype != torch.int32 or values.dtype != torch.float32 or ids.shape != (N, K) \
                or values.shape != (N, K) or ids.device != dev or values.device != dev \
                or not ids.is_contiguous() or not values.is_contiguous():
            raise ValueError(f"bias must be contiguous int32 ids and float32 values of one shape ({N}, K) on {dev}")
    M = 0
    if allowed is not None:
        if allowed.dtype != torch.int32 or allowed.dim() != 2 or allowed.shape[1] != -(-V // 32) \
                or allowed.device != dev or not allowed.is_contiguous():
            raise ValueError(f"allowed must be contiguous int32 (rows, {-(-V // 32)}) on {dev}")
        M = allowed.shape[0]
        if allowed_rows is None and M != N:
            raise ValueError(f"{M} mask rows for {N} rows of logits need allowed_rows")
    if allowed_rows is not None and (allowed is None or allowed_rows.dtype != torch.int32
                                     or allowed_rows.shape != (N,) or allowed_rows.device != dev
                                     or not allowed_rows.is_contiguous()):
        raise ValueError(f"allowed_rows must be contiguous int32 ({N},) on {dev}, with allowed")
    if out is None:
        out = logits.new_empty((N, V), dtype=torch.float32)
    elif out.shape != (N, V) or out.device != dev or (V > 1 and out.stride(1) != 1) \
            or (N > 1 and out.stride(0) < V):
        raise ValueError(f"out must be ({N}, {V}) on {dev}, its vocabulary contiguous and its rows apart")
    out_code = _dtype_code(out.dtype)
    best = logits.new_empty((N,), dtype=torch.int64) if greedy else None
    if N:
        args = _lib.pack_logits(
            logits.data_ptr(), out.data_ptr(), _ptr(best), _ptr(history and history.counts),
            _ptr(history and history.seen), rep, pres, freq, _ptr(ids), _ptr(values), _ptr(allowed), _ptr(allowed_rows),
            logits.stride(0), out.stride(0), N, V, code, out_code, K, M, rep_s, pres_s, freq_s, 0)
        _lib.launch(dev, _lib.lib().aoh_logits_penalize, "aoh_logits_penalize", args)
    return (out, best) if greedy else out
