"""Refusals of the operators' C entry points and Python functions that need no
GPU: every one is reported before any CUDA call."""
import ctypes as C
import re
import struct
from pathlib import Path

import numpy as np
import pytest
import torch

import aoh_b200
from aoh_b200 import _lib
from tests.test_capi_host import _cfg, _create

ROOT = Path(__file__).resolve().parents[1]
PTR = 4096  # stands for a device pointer that no refused call touches


def _fields(struct_name):
    """(name, format, count) of a C structure of the header, in order."""
    txt = (ROOT / "include" / "aoh.h").read_text()
    end = txt.index("} %s;" % struct_name)
    body = re.sub(r"/\*.*?\*/", "", txt[txt.rindex("typedef struct {", 0, end) + 16:end], flags=re.S)
    out = []
    for line in body.split(";"):
        m = re.match(r"\s*(const )?(\w+)\s*(\*?)\s*(\w+)(?:\[(\w+)\])?\s*$", line)
        if m:
            kind = "Q" if m[3] else {"int64_t": "q", "int32_t": "i", "float": "f"}[m[2]]
            n = {None: 1, "AOH_ROPE_MAX_AXES": 8}.get(m[5]) or int(m[5])
            out.append((m[4], kind, n))
    return out


@pytest.mark.parametrize("name,pack", [("aoh_rope_axes_args", _lib.pack_rope_axes), ("aoh_logits_args", _lib.pack_logits)])
def test_packed_arguments_follow_the_header(name, pack):
    fields = _fields(name)
    assert len(fields) > 15
    fmt = "@" + "".join(f"{n}{k}" for _, k, n in fields)
    assert struct.calcsize(fmt) == struct.calcsize(pack.__self__.format) and struct.calcsize(fmt) % 8 == 0
    values = list(range(1, 1 + sum(n for _, _, n in fields)))
    assert struct.pack(fmt, *values) == pack(*values)


def _rope(**over):
    args = dict(q=PTR, k=PTR, positions=PTR, inv_freq=PTR, qw=0, kw=0, q_out=2 * PTR, k_out=2 * PTR, qs=(64, 64, 64),
                ks=(64, 64, 64), ps=(0, 0, 1), sections=(32, 0, 0, 0, 0, 0, 0, 0), n_axes=1, interleaved=0,
                dtype=_lib.BF16, wide=1, batch=0, q_len=1, hq=1, g=1, d=64, eps=1e-6, scaling=1.0)
    args.update(over)
    flat = []
    for v in args.values():
        flat += v if isinstance(v, tuple) else (v,)
    return _lib.lib().aoh_rope_axes_qk(_lib.pack_rope_axes(*flat, 0), None)


def test_rope_axes_refusals():
    assert _rope() == _lib.OK  # no tokens: nothing to do
    sec = lambda *s: s + (0,) * (8 - len(s))  # noqa: E731
    for over, want in [
        (dict(q=0), _lib.INVALID), (dict(inv_freq=0), _lib.INVALID), (dict(k_out=0), _lib.INVALID),
        (dict(dtype=7), _lib.UNSUPPORTED), (dict(batch=-1), _lib.INVALID), (dict(hq=0), _lib.INVALID),
        (dict(d=0), _lib.UNSUPPORTED), (dict(d=63), _lib.UNSUPPORTED), (dict(d=258), _lib.UNSUPPORTED),
        (dict(n_axes=0), _lib.UNSUPPORTED), (dict(n_axes=9), _lib.UNSUPPORTED), (dict(qw=PTR), _lib.INVALID),
        (dict(q_out=PTR), _lib.INVALID), (dict(sections=sec(33)), _lib.INVALID), (dict(sections=sec(0)), _lib.INVALID),
        (dict(sections=sec(33, -1), n_axes=2), _lib.INVALID),
        (dict(sections=sec(2, 30), n_axes=2, interleaved=1), _lib.INVALID),  # axis 1 has 16 of 32 turns at most
    ]:
        assert _rope(**over) == want, over
    assert _rope(sections=sec(16, 16), n_axes=2, interleaved=1) == _lib.OK
    assert _lib.lib().aoh_rope_axes_qk(None, None) == _lib.INVALID


def _logits(**over):
    args = dict(logits=PTR, out=2 * PTR, greedy=0, counts=0, seen=0, rep=0, pres=0, freq=0, ids=0, bias=0, allowed=0,
                rows_map=0, stride=100, out_stride=100, rows=0, vocab=100, dtype=_lib.F32, out_dtype=_lib.F32, n_bias=0,
                n_allowed=0, rep_s=1.0, pres_s=0.0, freq_s=0.0)
    args.update(over)
    return _lib.lib().aoh_logits_penalize(_lib.pack_logits(*args.values(), 0), None)


def test_logits_refusals():
    assert _logits() == _lib.OK and _logits(logits=0, out=0) == _lib.OK  # no rows
    for over, want in [
        (dict(rows=-1), _lib.INVALID), (dict(vocab=0), _lib.INVALID), (dict(rows=1, logits=0), _lib.INVALID),
        (dict(dtype=9), _lib.UNSUPPORTED), (dict(out_dtype=9), _lib.UNSUPPORTED), (dict(counts=PTR), _lib.INVALID),
        (dict(n_bias=3), _lib.INVALID), (dict(n_bias=-1), _lib.INVALID),
        (dict(n_bias=4097, ids=PTR, bias=PTR), _lib.UNSUPPORTED), (dict(rows=2, allowed=PTR, n_allowed=1), _lib.INVALID),
        (dict(vocab=(1 << 21) + 1), _lib.UNSUPPORTED), (dict(rows=2, out=PTR, out_stride=120), _lib.INVALID),
        (dict(rows=1, out=PTR, out_dtype=_lib.BF16), _lib.INVALID), (dict(rows=1 << 30), _lib.UNSUPPORTED),
    ]:
        assert _logits(**over) == want, over
    L = _lib.lib()
    assert L.aoh_logits_penalize(None, None) == _lib.INVALID
    add = L.aoh_history_add
    assert add(None, None, 0, 10, None, 1, 0, 5, None, 0, None) == _lib.OK
    assert add(None, None, 2, 10, None, 1, 0, 5, None, 0, None) == _lib.INVALID
    assert add(PTR, PTR, -1, 10, PTR, 1, 0, 5, None, 0, None) == _lib.INVALID
    assert add(PTR, PTR, 2, 0, PTR, 1, 0, 5, None, 0, None) == _lib.INVALID
    assert add(PTR, PTR, 65536, 10, PTR, 1, 0, 5, None, 0, None) == _lib.UNSUPPORTED


def test_select_refusals():
    sel = _lib.lib().aoh_select_keys
    assert sel(PTR, 10, 0, 10, 5, 0, 0, PTR, None, None) == _lib.OK
    assert sel(None, 10, 3, 10, 0, 0, 0, None, None, None) == _lib.OK
    for rows, n, keep, sink, recent in [(1, 10, 11, 0, 0), (1, 10, -1, 0, 0), (1, 10, 5, 3, 3), (-1, 10, 5, 0, 0),
                                        (1, 10, 5, -1, 0), (1, 10, 5, 0, -1), (1, -1, 0, 0, 0)]:
        assert sel(PTR, 10, rows, n, keep, sink, recent, PTR, None, None) == _lib.INVALID, (rows, n, keep, sink, recent)
    assert sel(None, 10, 1, 10, 5, 0, 0, PTR, None, None) == _lib.INVALID
    assert sel(PTR, 10, 1 << 28, 10, 5, 0, 0, PTR, None, None) == _lib.UNSUPPORTED


def _make(labels, **kw):
    cfg, keep = _cfg(labels, **kw)
    rc, h = _create(cfg)
    assert rc == 0
    return h, keep


def test_key_weights_and_evict_refusals():
    L = _lib.lib()
    h, _k = _make([[1, 0], [0, 0]])
    assert L.aoh_key_weights(None, 0, 0, 1, PTR, PTR, 100, 0, PTR, 1 << 20, None) == _lib.INVALID
    assert L.aoh_key_weights(h, 0, 0, 1, PTR, PTR, 100, 0, PTR, 1 << 20, None) == _lib.STATE  # not bound
    # workspaces: none for what cannot run, more for more queries
    ws = lambda *a: L.aoh_key_weights_workspace_bytes(h, *a)  # noqa: E731
    assert ws(0, 0, 0) == ws(5, 0, 1) == ws(-1, 0, 1) == ws(0, 1024, 1) == ws(0, -2, 1) == 0
    assert 0 < ws(0, 500, 1) and ws(0, 0, 1) <= ws(0, _lib.PAST_LEN_DEVICE, 1) and ws(0, 500, 300) > 0
    assert L.aoh_key_weights_workspace_bytes(None, 0, 0, 1) == 0
    assert L.aoh_kv_evict(h, None, 10, PTR, 5, 5, None) == _lib.INVALID
    assert L.aoh_kv_evict(h, h, 10, PTR, 5, 5, None) == _lib.INVALID
    for kw in (dict(sink=64), dict(recent=128), dict(batch=2), dict(dtype=_lib.F32),
               dict(owned=[[[1, 1]], [[0, 1]]])):
        o, _ko = _make([[1, 0], [0, 0]], **kw)
        assert L.aoh_kv_evict(h, o, 500, PTR, 400, 400, None) == _lib.INVALID and b"differ" in L.aoh_last_error(), kw
        L.aoh_kv_destroy(o)
    o, _ko = _make([[1, 1], [0, 0]])
    assert L.aoh_kv_evict(h, o, 500, PTR, 400, 400, None) == _lib.INVALID
    L.aoh_kv_destroy(o)
    o, _ko = _make([[1, 0], [0, 0]], max_ctx=512)
    ev = lambda past, keep, ptr=PTR: L.aoh_kv_evict(h, o, past, ptr, keep, keep, None)  # noqa: E731
    assert ev(500, 501) == _lib.INVALID and ev(500, -1) == _lib.INVALID and ev(-1, -1) == _lib.INVALID
    assert ev(500, 383) == _lib.INVALID and b"sink" in L.aoh_last_error()  # 128 + 256 do not fit
    assert ev(500, 400, None) == _lib.INVALID
    assert ev(500, 400) == _lib.STATE and ev(100, 100) == _lib.STATE  # not bound
    L.aoh_kv_destroy(o)
    L.aoh_kv_destroy(h)


def test_python_functions_refuse_host_tensors():
    q, k = torch.zeros(1, 2, 4, 64), torch.zeros(1, 2, 2, 64)
    with pytest.raises(ValueError):
        aoh_b200.rope_axes_qk(q, k, torch.zeros(1, 1, 2, dtype=torch.int64), torch.ones(32), (32,))
    with pytest.raises(ValueError):
        aoh_b200.rope_axes_qk(q, k[0], torch.zeros(1, 1, 2, dtype=torch.int64), torch.ones(32), (32,))
    with pytest.raises(ValueError):
        aoh_b200.select_keys(torch.zeros(3, 5), 2)
    with pytest.raises(ValueError):
        aoh_b200.penalize_logits(torch.zeros(3, 5))
    with pytest.raises(ValueError):
        aoh_b200.TokenHistory(1, 0, device="cpu")


def test_tables_hold_the_retrieval_rows():
    """The table buffer grew by the retrieval rows (16 bytes a unit) and their index (4)."""
    h, _k = _make([[1, 0, 1]], hq=3, max_ctx=64, sink=16, recent=16)
    pool, tab = C.c_int64(), C.c_int64()
    assert _lib.lib().aoh_kv_buffer_sizes(h, C.byref(pool), C.byref(tab)) == 0
    entries = 2 * 4 + 2  # pages of two retrieval units and of one streaming unit
    assert tab.value == 4 * (4 + -(-entries // 4) * 4 + 4 + 5 * 3)
    _lib.lib().aoh_kv_destroy(h)
