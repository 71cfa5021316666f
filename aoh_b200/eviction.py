"""Eviction by accumulated attention weight.

The reference's retrieval heads keep every token; these operators bound them.
``key_weights`` sums the attention that each cached key of a layer's retrieval
heads received, ``select_keys`` picks the keys to keep by it, and ``evict``
copies their rows -- and the streaming heads' sink and window -- into another,
shorter cache, in which decoding goes on.  ``KeyWeights`` holds the sums of a
whole cache:

    sums = KeyWeights(cache)
    for layer in range(L):                      # a prefill chunk or a decode step
        past = cache.kv_seq_len
        out = aoh_attention(cache, layer, q, k, v)
        sums.add(layer, q, past_len=past)
    small = AoHKVCache(labels, num_q_heads, max_context=8192 + 1024, ...)
    sums = sums.evict(8192, into=small)         # small.tokens_seen goes on counting

A kept key's RoPE position stays what it was: after an eviction, rotate new
tokens by ``tokens_seen``, not by ``kv_seq_len``.
"""
from __future__ import annotations

import torch

from . import _lib
from .attention import _check_q
from .cache import AoHKVCache


def key_weights(cache: AoHKVCache, layer_idx: int, q: torch.Tensor, *, past_len: int | None = None,
                out: torch.Tensor | None = None, accumulate: bool = False) -> torch.Tensor:
    """The attention weight that each key received from the queries ``q``.

    q (B, C, Hq, D): the post-RoPE queries of the tokens at positions past_len..
    past_len + C - 1, whose keys the cache holds already (call it after
    :func:`aoh_attention` of the layer).  ``past_len`` defaults to
    ``cache.kv_seq_len``, which moves after the last layer only.  Returns (B,
    n_ret, T = past_len + C) float32: for each of the layer's retrieval heads in
    ascending order the softmax probabilities of its group's heads, summed over
    heads and queries.  ``out``: a float32 tensor (B, n_ret, >= T) whose rows are
    contiguous and evenly spaced (a slice of a larger buffer); its first T columns
    are written, or with ``accumulate`` added to.  A cache in device-length mode
    takes single tokens and ``out`` of max_context columns or more.
    q and the keys are finite: a NaN among them may make weights of its retrieval
    head NaN or be left out of the sums.
    """
    if not 0 <= layer_idx < cache.num_layers:
        raise ValueError(f"layer_idx {layer_idx} out of range")
    # a call's Python is most of the time that a single token takes: each property is read once
    shape, dev, B, R = q.shape, q.device, cache.batch, cache.n_ret[layer_idx]
    if len(shape) != 4:
        raise ValueError("q must be (B, C, Hq, D)")
    n = shape[1]
    _check_q(cache, q, n)
    if cache.device_length:
        if n != 1 or past_len is not None or out is None:
            raise ValueError("a cache in device-length mode takes single tokens (q_len 1), no past_len, and an out")
        past, total = _lib.PAST_LEN_DEVICE, cache.max_context
    else:
        past = cache.kv_seq_len if past_len is None else int(past_len)
        if past < 0:
            raise ValueError("past_len must be non-negative")
        total = past + n
        if total >= 1 << 31:
            raise ValueError(f"{total} keys are more than 32 bits count")
    if out is None:
        if accumulate:
            raise ValueError("accumulate needs an out to add to")
        out, stride = q.new_empty((B, R, total), dtype=torch.float32), total
    elif (out.dim() != 3 or out.shape[0] != B or out.shape[1] != R or out.shape[2] < total
          or out.dtype != torch.float32 or out.device != dev):
        raise ValueError(f"out must be float32 (batch, n_ret, >= keys) = {(B, R, total)} on {cache.device}, "
                         f"got {out.dtype} {tuple(out.shape)}")
    elif R > 0:
        stride = out.stride(1) if R > 1 else out.stride(0) if B > 1 else out.shape[2]
        if out.stride(2) != 1 or stride < total or (B > 1 and out.stride(0) != R * stride):
            raise ValueError("out's rows must be contiguous and evenly spaced over (batch, n_ret)")
    if R == 0 or n == 0:
        if not accumulate:
            out[:, :, :total].zero_()
        return out
    L = cache._L
    nbytes = L.aoh_key_weights_workspace_bytes(cache._h, layer_idx, past, n)
    ws = q.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    _lib.launch(dev, L.aoh_key_weights, "aoh_key_weights", cache._h, layer_idx, past, n, q.data_ptr(),
                out.data_ptr(), stride, bool(accumulate), ws.data_ptr() if nbytes else None, nbytes)
    return out


def select_keys(weights: torch.Tensor, keep: int, *, sink: int = 0, recent: int = 0
                ) -> tuple[torch.Tensor, torch.Tensor]:
    """The keys to keep by their weights.

    weights (..., n) float32, n contiguous.  Keeps, per row, the first ``sink``
    and the last ``recent`` keys and the largest weights between them, ``keep``
    keys in all; the lower position first among equal weights, NaN like -inf.
    Returns (positions (..., keep) int32, ascending, and their weights)."""
    if weights.dim() < 1 or weights.dtype != torch.float32 or not weights.is_cuda:
        raise ValueError("weights must be a float32 CUDA tensor (..., n)")
    n = weights.shape[-1]
    keep, sink, recent = int(keep), int(sink), int(recent)
    if not 0 <= keep <= n:
        raise ValueError(f"keep {keep} of {n} keys")
    if sink < 0 or recent < 0 or sink + recent > keep:
        raise ValueError(f"sink {sink} and recent {recent} must be non-negative and fit keep {keep}")
    lead = weights.shape[:-1]
    kept = weights.new_empty((*lead, keep), dtype=torch.int32)
    kept_w = weights.new_empty((*lead, keep))
    if kept.numel() == 0:
        return kept, kept_w
    # rows evenly spaced: a view, or a copy where they are not
    w = weights if weights.dim() == 2 else weights.reshape(-1, n)
    rows = w.shape[0]
    if rows >> 31 or n >> 31:
        raise ValueError(f"weights {tuple(weights.shape)}: rows and keys must fit 32 bits")
    stride, one = w.stride()
    if n > 1 and one != 1:
        raise ValueError("the last dimension of weights must be contiguous")
    _lib.launch(weights.device, _lib.lib().aoh_select_keys, "aoh_select_keys", w.data_ptr(), stride, rows, n, keep,
                sink, recent, kept.data_ptr(), kept_w.data_ptr())
    return kept, kept_w


def evict(cache: AoHKVCache, kept: torch.Tensor, into: AoHKVCache) -> AoHKVCache:
    """Copy the rows that stay of every layer into another cache.

    kept (R, keep) int32, rows contiguous: the positions to keep of each
    retrieval unit, in (layer, sequence, KV head) order, R = batch * sum(n_ret).
    Position kept[r, i] becomes position i; streaming heads keep their sink and
    their latest rows.  ``into``: a different cache with the same labels, batch,
    windows and dtype and room for keep tokens; what it held is given up.  It then
    holds keep tokens (``kv_seq_len``) of ``tokens_seen`` seen.  With streaming
    heads, keep must reach sink + recent (or kv_seq_len)."""
    if into is cache:
        raise ValueError("into must be another cache")
    if cache.device_length or into.device_length:
        raise ValueError("a cache in device-length mode cannot be evicted")
    R, shape, dev = cache.batch * sum(cache.n_ret), kept.shape, cache.device
    if len(shape) != 2 or shape[0] != R or kept.dtype != torch.int32 or kept.device != dev:
        raise ValueError(f"kept must be int32 ({R}, keep) on {dev}, got {kept.dtype} {tuple(shape)}")
    keep, (stride, one) = shape[1], kept.stride()
    if keep > 1 and one != 1:
        raise ValueError("the rows of kept must be contiguous")
    if into.device != dev:
        raise ValueError(f"the caches are on {dev} and {into.device}")
    total = cache._kv_seq_len
    if keep > total:
        raise ValueError(f"keep {keep} of {total} tokens")
    if keep > into.max_context:
        raise ValueError(f"keep {keep} exceeds the destination's max_context {into.max_context}")
    into.reserve(keep)
    _lib.launch(dev, cache._L.aoh_kv_evict, "aoh_kv_evict", cache._h, into._h, total, kept.data_ptr(), stride, keep)
    if into._sums:
        into._forget(0)
    into._kv_seq_len = keep
    into.evicted = total + cache.evicted - keep
    return into


class KeyWeights:
    """The attention weight of every cached key of every retrieval unit.

    ``rows`` (R, max_context) float32, zero at the start, R = batch *
    sum(n_ret) rows in (layer, sequence, KV head) order; column j belongs to the
    key at cache position j.  The sums follow the cache: they start at zero again from
    the position that its ``kv_seq_len`` is set back to (0: a new sequence), and
    everywhere when another cache is evicted into it."""

    def __init__(self, cache: AoHKVCache):
        self.cache = cache
        self.rows = torch.zeros((cache.batch * sum(cache.n_ret), cache.max_context), dtype=torch.float32,
                                device=cache.device)
        cache._track(self)
        self._first = [cache.batch * sum(cache.n_ret[:i]) for i in range(cache.num_layers + 1)]

    def layer(self, layer_idx: int) -> torch.Tensor:
        """(batch, n_ret, max_context) of one layer, a view."""
        lo, hi = self._first[layer_idx], self._first[layer_idx + 1]
        return self.rows[lo:hi].view(self.cache.batch, self.cache.n_ret[layer_idx], self.rows.shape[1])

    def add(self, layer_idx: int, q: torch.Tensor, past_len: int | None = None) -> None:
        """Add what the queries q gave (see :func:`key_weights`)."""
        key_weights(self.cache, layer_idx, q, past_len=past_len, out=self.layer(layer_idx), accumulate=True)

    def evict(self, keep: int, into: AoHKVCache, *, sink: int | None = None, recent: int | None = None) -> "KeyWeights":
        """Keep ``keep`` keys of every retrieval unit -- the first ``sink`` and the
        last ``recent`` (default: the cache's window) among them -- and copy them
        into ``into``.  Returns its KeyWeights, with the kept keys' sums."""
        c = self.cache
        sink, recent = c.sink_size if sink is None else sink, c.recent_size if recent is None else recent
        if keep == c.kv_seq_len:  # all of them, however short the sequence is
            sink, recent = keep, 0
        kept, weights = select_keys(self.rows[:, :c.kv_seq_len], keep, sink=sink, recent=recent)
        evict(c, kept, into)
        new = KeyWeights(into)
        new.rows[:, :keep] = weights
        return new
