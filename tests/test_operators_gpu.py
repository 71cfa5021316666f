"""rope_axes_qk, key_weights, select_keys, evict, TokenHistory and
penalize_logits against plain implementations in 64 bits (the logits' steps, and
everything that is copied or counted, bit for bit)."""
import math

import numpy as np
import pytest
import torch

import aoh_b200
from aoh_b200 import (AoHKVCache, KeyWeights, TokenHistory, aoh_attention, evict, key_weights, penalize_logits,
                      rope_axes_qk, select_keys)

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=F32):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


# -- rope_axes_qk ----------------------------------------------------------------
def rope_exact(x, pos, inv, sections, interleaved, w, eps, scaling):
    """(y, bound of its fp32 error) in 64 bits."""
    A, half, D = len(sections), sum(sections), x.shape[-1]
    x = x.double().cpu()
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double().cpu()
    axis = []
    for i in range(half):
        if interleaved:
            axis.append(i % A if i < A * sections[i % A] else 0)
        else:
            axis.append(int(np.searchsorted(np.cumsum(sections), i, side="right")))
    angle = torch.stack([pos[a].double().cpu() * float(inv[i]) for i, a in enumerate(axis)], -1)[:, :, None]
    c, s = angle.cos() * scaling, angle.sin() * scaling
    a, b = x[..., :half], x[..., half:2 * half]
    y = torch.cat((a * c - b * s, b * c + a * s, x[..., 2 * half:]), -1)
    # sine and cosine: 2 ulp of sincospif and the rounding of its argument (2.1e-7), three roundings of the
    # rotation; the norm's mean of squares: 22 additions, halved by the root, and 4 roundings: 1.1e-6.  Below 2^-18.
    mag = (a.abs() + b.abs()) * max(1.0, abs(scaling))
    return y, torch.cat((mag, mag, x[..., 2 * half:].abs()), -1) * 2.0 ** -18


def check_rope(x, got, *args):
    want, err = rope_exact(x, *args)
    assert got.dtype == x.dtype and got.is_contiguous()
    # one rounding of the stored value: half a step of the type
    bound = err + want.abs() * (torch.finfo(x.dtype).eps / 2)
    assert ((got.double().cpu() - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,C,Hq,G,D,sections,interleaved,norm", [
    (1, 1, 1, 1, 2, (1,), False, False),
    (1, 1, 32, 8, 128, (16, 24, 24), False, False),
    (2, 5, 7, 1, 128, (64,), False, True),
    (3, 33, 12, 4, 80, (12, 10, 10), True, True),
    (1, 130, 28, 4, 128, (24, 20, 20), True, False),
    (2, 9, 3, 3, 96, (20, 0, 3), False, True),
    (1, 7, 2, 1, 256, (100, 28), False, True),
    (1, 7, 2, 2, 256, (3,), False, True),
    (1, 3, 5, 1, 70, (17, 3), False, True),
    (4, 300, 16, 2, 64, (8, 8, 8, 8), True, False),
])
def test_rope_axes(dtype, B, C, Hq, G, D, sections, interleaved, norm):
    g = gen(B * 1000 + C + D)
    A, half = len(sections), sum(sections)
    q, k = randn(g, B, C, Hq, D, dtype=dtype), randn(g, B, C, G, D, dtype=dtype)
    pos = torch.randint(0, 1_000_000, (A, B, C), generator=g, device="cuda")
    inv = 1e4 ** (-torch.arange(half, device="cuda", dtype=F32) / half)
    w = (1 + 0.1 * randn(g, D)).to(dtype) if norm else None
    wk = (1 + 0.1 * randn(g, D)).to(dtype) if norm else None
    for positions in (pos, pos.int()):
        qo, ko = rope_axes_qk(q, k, positions, inv, sections, interleaved=interleaved, q_norm_weight=w,
                              k_norm_weight=wk, eps=1e-5, scaling=1.25)
        check_rope(q, qo, pos, inv, sections, interleaved, w, 1e-5, 1.25)
        check_rope(k, ko, pos, inv, sections, interleaved, wk, 1e-5, 1.25)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shift", [0, 1])
def test_rope_axes_takes_views(dtype, shift):
    """q and k as views of one fused projection, at any alignment; expanded positions."""
    g = gen(5)
    B, C, Hq, G, D = 2, 19, 6, 2, 64
    fused = randn(g, B, C, (Hq + 2 * G) * D + 5 + shift, dtype=dtype)
    q = fused[..., shift:shift + Hq * D].view(B, C, Hq, D)
    k = fused[..., shift + Hq * D:shift + (Hq + G) * D].view(B, C, G, D)
    pos = torch.arange(C, device="cuda").expand(3, B, C)
    inv = 1e4 ** (-torch.arange(32, device="cuda", dtype=F32) / 32)
    qo, ko = rope_axes_qk(q, k, pos, inv, (16, 8, 8))
    check_rope(q, qo, pos, inv, (16, 8, 8), False, None, 0, 1.0)
    check_rope(k, ko, pos, inv, (16, 8, 8), False, None, 0, 1.0)
    # heads before tokens
    qt = q.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(rope_axes_qk(qt, k, pos, inv, (16, 8, 8))[0], qo)


def test_rope_axes_far_and_negative_positions():
    g = gen(6)
    q, k = randn(g, 1, 4, 2, 64), randn(g, 1, 4, 1, 64)
    pos = torch.tensor([[[-3, 2 ** 31 + 5, 2 ** 40 + 1, 10 ** 9 + 7]]], device="cuda")
    inv = 1e4 ** (-torch.arange(32, device="cuda", dtype=F32) / 32)
    qo, _ = rope_axes_qk(q, k, pos, inv, (32,))
    # at 2^40 the fp64 angle and its reduction round to 2^40 * 3 * 2^-53 = 4e-4 radians
    want, err = rope_exact(q, pos, inv, (32,), False, None, 0, 1.0)
    far = (pos[0, 0].double().abs() * 3 * 2.0 ** -53).cpu()[None, :, None, None] * (err * 2 ** 18)
    assert ((qo.double().cpu() - want).abs() <= err + far + want.abs() * 2.0 ** -24).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rope_axes_rows_more_than_32_bits_apart(dtype):
    """Sequences whose rows lie more than 2^31 elements apart, as views of one buffer."""
    apart, Hq, G, D = 2 ** 31 + 64, 3, 1, 64
    buf = torch.empty(apart + 4096, device="cuda", dtype=dtype)
    q, k = buf.as_strided((2, 2, Hq, D), (apart, 512, D, 1)), buf.as_strided((2, 2, G, D), (apart, 512, D, 1), 256)
    q.copy_(randn(gen(1), 2, 2, Hq, D, dtype=dtype))
    k.copy_(randn(gen(2), 2, 2, G, D, dtype=dtype))
    pos = torch.tensor([[[3, 4], [70_000, 70_001]]], device="cuda")
    inv = 1e4 ** (-torch.arange(32, device="cuda", dtype=F32) / 32)
    got = rope_axes_qk(q, k, pos, inv, (32,))
    want = rope_axes_qk(q.contiguous(), k.contiguous(), pos, inv, (32,))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_rope_axes_agrees_with_rope_qk():
    """One axis of ordinary positions is the framework's other rotation, up to the roundings that one makes."""
    g = gen(7)
    q, k = randn(g, 2, 40, 8, 128, dtype=BF16), randn(g, 2, 40, 2, 128, dtype=BF16)
    pos = torch.arange(40, device="cuda").expand(1, 2, 40)
    inv = 1e4 ** (-torch.arange(64, device="cuda", dtype=F32) / 64)
    ang = (pos[0][..., None].float() * inv).repeat(1, 1, 2)
    qa, ka = rope_axes_qk(q, k, pos, inv, (64,))
    qb, kb = aoh_b200.rope_qk(q, k, ang.cos().to(BF16).contiguous(), ang.sin().to(BF16).contiguous())
    # rope_qk rounds cos, sin, both products and the sum to bf16: 5 half steps of values up to |u| + |v|
    bound = lambda x: (x.abs().float() + x.abs().float().roll(64, -1)) * (5 * 2.0 ** -8 + 2.0 ** -8)  # noqa: E731
    assert ((qa.float() - qb.float()).abs() <= bound(q)).all() and ((ka.float() - kb.float()).abs() <= bound(k)).all()


def test_rope_axes_empty():
    q, k = torch.empty(2, 0, 4, 64, device="cuda", dtype=BF16), torch.empty(2, 0, 2, 64, device="cuda", dtype=BF16)
    pos = torch.empty(1, 2, 0, device="cuda", dtype=torch.int64)
    qo, ko = rope_axes_qk(q, k, pos, torch.ones(32, device="cuda"), (32,))
    assert qo.shape == q.shape and ko.shape == k.shape


# -- key_weights -------------------------------------------------------------------
def filled(labels, Hq, B, T, dtype, seed, sink=128, recent=256, max_context=None, owned=None):
    """(cache holding T random tokens, k, v (L, B, T, G, D))."""
    L, G = np.asarray(labels).shape
    g = gen(seed)
    cache = AoHKVCache(labels, Hq, batch=B, sink_size=sink, recent_size=recent, max_context=max_context or T,
                       dtype=dtype, owned=owned)
    k, v = randn(g, L, B, T, G, 128, dtype=dtype), randn(g, L, B, T, G, 128, dtype=dtype)
    for layer in range(L):
        cache.append_layer(layer, k[layer], v[layer])
    cache.kv_seq_len = T
    return cache, k, v


def weights_exact(q, k, heads, past):
    """(weights, bound of their relative error) in 64 bits; q (B, C, Hq, D), k (B, T, G, D)."""
    B, C, Hq, D = q.shape
    G, T = k.shape[2], k.shape[1]
    grp = Hq // G
    out = torch.zeros(B, len(heads), T, dtype=torch.float64)
    most = 0.0
    late = torch.arange(T, device="cuda") > past + torch.arange(C, device="cuda")[:, None]
    for b in range(B):
        for r, g in enumerate(heads):
            kk = k[b, :, g].double()
            for h in range(g * grp, (g + 1) * grp):
                qq = q[b, :, h].double()
                s = (qq @ kk.T / math.sqrt(D)).masked_fill(late, -math.inf)
                out[b, r] += torch.softmax(s, 1).sum(0).cpu()
                most = max(most, float((qq.abs() @ kk.abs().T).max()) / math.sqrt(D))
    # a score's error: 128 products added in fp32, its scaling; the exponential sees it in the weight and in
    # the sum; the sums over the keys and over the rows add a rounding an addition
    tol = 2 * 130 * 2.0 ** -24 * most + (T + C * grp + 16) * 2.0 ** -24
    return out, tol


def check_weights(got, q, k, heads, past):
    want, tol = weights_exact(q, k, heads, past)
    assert got.dtype == F32 and tuple(got.shape) == tuple(want.shape)
    # a weight below 2^-100 may come out as zero
    assert ((got.double().cpu() - want).abs() <= tol * want + 2.0 ** -100).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("labels,Hq,B,C,past", [
    ([[1]], 1, 1, 1, 0),                 # one key
    ([[1]], 4, 1, 1, 1),
    ([[0, 1]], 14, 2, 1, 127),           # group of 7, two sequences
    ([[1, 0, 1, 1]], 8, 1, 1, 2049),
    ([[1, 1]], 2, 1, 5, 0),              # no cached keys: causal among themselves
    ([[1, 0]], 10, 1, 17, 31),           # group of 5
    ([[0, 1, 0]], 21, 3, 40, 201),
    ([[1, 0]], 64, 1, 3, 90),            # group of 32
    ([[1]], 160, 1, 2, 90),              # group of 160
    ([[1, 1]], 8, 1, 130, 1000),
    ([[1, 0]], 8, 2, 257, 0),
])
def test_key_weights(dtype, labels, Hq, B, C, past):
    T = past + C
    cache, k, _ = filled(labels, Hq, B, T, dtype, T + Hq)
    cache.kv_seq_len = past
    q = randn(gen(3), B, C, Hq, 128, dtype=dtype) * 1.5
    heads = [g for g, x in enumerate(labels[0]) if x]
    got = key_weights(cache, 0, q)
    check_weights(got, q, k[0], heads, past)
    # added into a slice of a larger buffer; what lies behind stays
    big = torch.full((B, len(heads), T + 5), 2.0, device="cuda")
    assert key_weights(cache, 0, q, past_len=past, out=big, accumulate=True) is big
    assert torch.equal(big[..., :T], got + 2) and (big[..., T:] == 2).all()
    key_weights(cache, 0, q, out=big)
    assert torch.equal(big[..., :T], got) and (big[..., T:] == 2).all()
    assert cache.device_status() == 0


@pytest.mark.parametrize("C", [1, 3, 32, 700])
def test_key_weights_long(C):
    """Long enough for every key range and tile path; second layer of a cache."""
    labels = [[1, 0, 0, 0], [0, 1, 0, 1]]
    past, Hq = 20_000 + C % 7, 16
    cache, k, _ = filled(labels, Hq, 1, past + C, BF16, C)
    q = randn(gen(C), 1, C, Hq, 128, dtype=BF16) * 2
    got = key_weights(cache, 1, q, past_len=past)
    check_weights(got, q, k[1], [1, 3], past)
    assert torch.equal(key_weights(cache, 1, q, past_len=past), got)  # a fixed order of sums


@pytest.mark.parametrize("G,grp,C,past", [
    (1, 8, 600, 6_000),    # 4800 rows over 6600 keys: a second block of 1024 rows
    (8, 1, 20, 100_003),   # 8 units of 20 rows over many keys: blocks of 16 rows
])
def test_key_weights_f32_in_blocks_of_rows(G, grp, C, past):
    """More scores than one block of query rows has room for; added to what is there."""
    cache, k, _ = filled([[1] * G], G * grp, 1, past + C, F32, C)
    q = randn(gen(C), 1, C, G * grp, 128, dtype=F32)
    got = key_weights(cache, 0, q, past_len=past)
    check_weights(got, q, k[0], range(G), past)
    twice = got.clone()
    key_weights(cache, 0, q, past_len=past, out=twice, accumulate=True)
    # an addition to another start rounds once a block in another place
    assert ((twice - 2 * got).abs() <= 4 * 2.0 ** -24 * twice).all()


@pytest.mark.parametrize("C,T", [(1, 8192), (1, 8193), (2, 8191), (2, 255), (5, 4096), (5, 4097), (5, 8192), (5, 8193), (6, 4096), (7, 511)])
@pytest.mark.parametrize("labels", [[1, 1], [1, 0]])
def test_key_weights_where_the_kernels_change(labels, C, T):
    """Groups of 6: 6 to 42 query rows, around the lengths that one launch takes; the other sequence is not
    stored here."""
    owned = np.array([[[1, 1], [0, 0]]])
    cache, k, _ = filled([labels], 12, 2, T, BF16, T + C, owned=owned)
    q = randn(gen(C), 2, C, 12, 128, dtype=BF16) * 1.5
    heads = [g for g, x in enumerate(labels) if x]
    out = torch.full((2, len(heads), T + 3), 1.0, device="cuda")
    key_weights(cache, 0, q, past_len=T - C, out=out)
    check_weights(out[:1, :, :T], q[:1], k[0][:1], heads, T - C)
    assert (out[1, :, :T] == 0).all() and (out[..., T:] == 1).all()
    again = key_weights(cache, 0, q, past_len=T - C)
    assert torch.equal(again, out[..., :T])


def test_key_weights_large_scores():
    """Scores far apart: one key takes nearly everything; no overflow."""
    cache, k, _ = filled([[1]], 4, 1, 900, BF16, 1)
    q = (k[0][:, 400:401].expand(1, 1, 1, 128) * 20).expand(1, 1, 4, 128).contiguous()
    got = key_weights(cache, 0, q, past_len=899)
    check_weights(got, q, k[0], [0], 899)
    assert got[0, 0, 400] > 3.99


def test_key_weights_ignores_what_the_cache_does_not_hold_yet():
    """NaN in the slots behind the last key (a page's tail) reaches no weight."""
    cache, k, _ = filled([[1, 0]], 8, 1, 203, BF16, 2, max_context=256)
    pg, sl = cache.locate(0, 0, 0, 202)
    want = key_weights(cache, 0, randn(gen(1), 1, 7, 8, 128, dtype=BF16), past_len=196)
    cache.kv_seq_len = 208
    bad = torch.full((1, 5, 2, 128), float("nan"), device="cuda", dtype=BF16)
    cache.kv_seq_len = 203
    cache.append_layer(0, bad, bad)
    got = key_weights(cache, 0, randn(gen(1), 1, 7, 8, 128, dtype=BF16), past_len=196)
    assert torch.equal(got, want) and torch.isfinite(got).all()


@pytest.mark.parametrize("dtype,C", [(BF16, 60), (BF16, 140), (F32, 7), (F32, 60)])
def test_key_weights_of_chunks_ignore_what_is_not_held_yet(dtype, C):
    """The same for the kernels that take more query rows, and for fp32."""
    T = 331  # 11 slots of the last page in use
    cache, k, _ = filled([[1, 0]], 8, 1, T, dtype, C, max_context=384)
    q = randn(gen(1), 1, C, 8, 128, dtype=dtype)
    want = key_weights(cache, 0, q, past_len=T - C)
    check_weights(want, q, k[0], [0], T - C)
    bad = torch.full((1, 5, 2, 128), float("nan"), device="cuda", dtype=dtype)
    cache.append_layer(0, bad, bad)
    assert torch.equal(key_weights(cache, 0, q, past_len=T - C), want)


def test_key_weights_of_units_stored_elsewhere_are_zero():
    owned = np.array([[[1, 0], [0, 1]]])
    cache, k, _ = filled([[1, 1]], 4, 2, 50, BF16, 4, owned=owned)
    q = randn(gen(1), 2, 1, 4, 128, dtype=BF16)
    got = key_weights(cache, 0, q, past_len=49)
    want, tol = weights_exact(q, k[0], [0, 1], 49)
    assert (got[0, 1] == 0).all() and (got[1, 0] == 0).all()
    for b, r in ((0, 0), (1, 1)):
        assert ((got[b, r].double().cpu() - want[b, r]).abs() <= tol * want[b, r] + 2.0 ** -100).all()


def test_key_weights_without_retrieval_heads():
    cache, _, _ = filled([[0, 0]], 4, 1, 40, BF16, 4)
    assert key_weights(cache, 0, randn(gen(1), 1, 1, 4, 128, dtype=BF16), past_len=39).shape == (1, 0, 40)


# -- select_keys -------------------------------------------------------------------
def select_plain(w, keep, sink, recent):
    w = w.cpu().numpy().astype(np.float64)
    n = w.shape[-1]
    flat = np.where(np.isnan(w), -np.inf, w).reshape(-1, n)
    out = np.empty((flat.shape[0], keep), np.int64)
    for r, row in enumerate(flat):
        mid = np.arange(sink, n - recent)
        best = mid[np.argsort(-row[sink:n - recent], kind="stable")[:keep - sink - recent]]
        out[r] = np.sort(np.concatenate((np.arange(sink), best, np.arange(n - recent, n))))
    return out.reshape(*w.shape[:-1], keep)


def check_select(w, keep, sink, recent):
    kept, kw = select_keys(w, keep, sink=sink, recent=recent)
    want = select_plain(w, keep, sink, recent)
    assert kept.dtype == torch.int32 and np.array_equal(kept.cpu().numpy(), want)
    want_w = torch.gather(w, -1, kept.long())
    assert torch.equal(kw.view(torch.int32), want_w.view(torch.int32))


@pytest.mark.parametrize("rows,n,keep,sink,recent", [
    (1, 1, 1, 0, 0), (1, 1, 0, 0, 0), (3, 7, 7, 0, 0), (3, 7, 3, 1, 2), (2, 33, 32, 0, 32), (5, 100, 60, 60, 0),
    (4, 4095, 1000, 128, 256), (4, 4096, 1, 0, 0), (2, 4097, 4096, 3, 5), (3, 20_001, 777, 16, 0),
    (2, 70_000, 8192, 128, 256), (1, 500_000, 100_003, 4, 250),  # the last: more than shared memory holds
])
@pytest.mark.parametrize("kind", ["distinct", "ties", "equal", "odd"])
def test_select_keys(rows, n, keep, sink, recent, kind):
    g = gen(n + keep)
    w = torch.rand((rows, n), generator=g, device="cuda")
    if kind == "ties":
        w = (w * 6).floor() / 6
    elif kind == "equal":
        w = torch.full_like(w, 0.25)
    elif kind == "odd":
        w = torch.where(w < 0.5, -w, w)
        special = torch.tensor([math.nan, math.inf, -math.inf, 0.0, -0.0, 1e-40, -1e-40, -math.nan], device="cuda")
        pick = torch.randint(0, 24, (rows, n), generator=g, device="cuda")
        w = torch.where(pick < 8, special[pick.clamp(max=7)], w)
    check_select(w, keep, sink, recent)


def test_select_keys_strided_rows():
    big = torch.rand((3, 2, 1000), generator=gen(1), device="cuda")
    check_select(big[:, :, :777], 100, 4, 30)
    check_select(big[:, 1, 3:700], 100, 0, 0)
    check_select(big[1, 1], 10, 0, 0)
    check_select(big[:1].expand(3, 2, 1000), 10, 0, 0)
    assert select_keys(big[:0], 10)[0].shape == (0, 2, 10)


# -- evict -------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("labels,B,T,keep,sink,recent", [
    ([[1]], 1, 1, 1, 0, 0),
    ([[1]], 1, 300, 17, 0, 0),
    ([[1, 0], [0, 1]], 2, 700, 384, 128, 256),
    ([[1, 0], [1, 1], [0, 0]], 1, 1000, 401, 20, 40),     # ring of 48 turned by an odd number
    ([[0, 1]], 2, 333, 333, 20, 40),                      # everything stays
    ([[0, 1]], 1, 90, 30, 5, 0),                          # no window
    ([[1, 0]], 1, 12, 12, 20, 40),                        # shorter than the sink
    ([[0]], 1, 500, 100, 16, 33),                         # streaming heads alone
])
def test_evict_copies_rows(dtype, labels, B, T, keep, sink, recent):
    L, G = np.asarray(labels).shape
    cache, k, v = filled(labels, G, B, T, dtype, T, sink, recent)
    into = AoHKVCache(labels, G, batch=B, sink_size=sink, recent_size=recent, max_context=keep + 40, dtype=dtype)
    into.pool.view(torch.uint8).fill_(0x11)  # rows behind the kept ones stay as they were
    before = into.pool.clone()
    R = B * sum(cache.n_ret)
    g = gen(keep)
    kept = torch.stack([torch.randperm(T, generator=g, device="cuda")[:keep].sort().values for _ in range(R)] or
                       [torch.empty(keep, device="cuda")])[:R].to(torch.int32)
    assert evict(cache, kept, into) is into
    assert (into.kv_seq_len, into.evicted, into.tokens_seen) == (keep, T - keep, T)
    assert cache.kv_seq_len == T
    ring = -(-recent // 16) * 16
    r = 0
    for layer in range(L):
        for b in range(B):
            for h in range(G):
                if labels[layer][h]:
                    new, old = range(keep), kept[r].tolist()
                    r += 1
                else:
                    s = min(sink, keep)
                    held = max(0, min(ring, keep - sink))
                    new = [*range(s), *range(keep - held, keep)]
                    old = [*range(s), *range(T - held, T)]
                gk, gv = into.read_rows(layer, b, h, new)
                assert torch.equal(gk, k[layer, b, old, h]) and torch.equal(gv, v[layer, b, old, h])
    changed = (into.pool != before).view(into.num_pages, -1).any(1).sum().item()
    assert changed <= sum(-(-keep // 16) if x else -(-sink // 16) + ring // 16 for row in labels for x in row) * B
    if any(x for row in labels for x in row) and keep % 16:
        u = next((l, h) for l in range(L) for h in range(G) if labels[l][h])
        into.kv_seq_len = keep + 1
        gk, gv = into.read_rows(u[0], 0, u[1], [keep])
        assert (gk.view(torch.uint8) == 0x11).all() and (gv.view(torch.uint8) == 0x11).all()
    assert into.device_status() == 0 and cache.device_status() == 0


def test_evict_partitioned_cache():
    labels, owned = [[1, 0], [1, 1]], np.array([[[1, 0]], [[0, 1]]])
    cache, k, v = filled(labels, 2, 1, 200, BF16, 3, 16, 32, owned=owned)
    into = AoHKVCache(labels, 2, sink_size=16, recent_size=32, max_context=100, owned=owned)
    kept = torch.arange(100, 200, device="cuda", dtype=torch.int32).repeat(3, 1)
    evict(cache, kept, into)
    for layer, h in ((0, 0), (1, 1)):
        gk, gv = into.read_rows(layer, 0, h, range(100))
        assert torch.equal(gk, k[layer, 0, 100:, h]) and torch.equal(gv, v[layer, 0, 100:, h])
    assert into.device_status() == 0


def test_evict_reports_positions_outside_the_cache():
    cache, k, _ = filled([[1]], 1, 1, 64, BF16, 3, 0, 0)
    into = AoHKVCache([[1]], 1, sink_size=0, recent_size=0, max_context=32)
    kept = torch.arange(32, device="cuda", dtype=torch.int32)[None].clone()
    kept[0, 3], kept[0, 9] = 64, -1
    evict(cache, kept, into)
    assert into.device_status() == 1 and into.device_status() == 0
    gk, _ = into.read_rows(0, 0, 0, [2, 4])
    assert torch.equal(gk, k[0, 0, [2, 4], 0])


# -- history and logits ----------------------------------------------------------------
def penalize_plain(x, counts, in_prompt, rep, pres, freq, bias, allowed):
    """The documented steps, each rounded to fp32."""
    x = x.float().cpu().numpy().copy()
    f = np.float32
    N, V = x.shape
    if counts is not None:
        seen = (counts > 0) | in_prompt
        with np.errstate(all="ignore"):
            pen = np.where(x > 0, (x / rep[:, None]).astype(f), (x * rep[:, None]).astype(f))
            x = np.where(seen, pen, x)
            x = np.where(seen, (x - (freq[:, None] * counts.astype(f)).astype(f)).astype(f), x)
            x = np.where(counts > 0, (x - pres[:, None]).astype(f), x)
    if bias is not None:
        ids, val = (t.cpu().numpy() for t in bias)
        for n in range(N):
            total = {}
            for i, b in zip(ids[n], val[n]):
                if 0 <= i < V:
                    total[i] = f(total[i] + b) if i in total else b
            for i, b in total.items():
                x[n, i] = f(x[n, i] + b)
    if allowed is not None:
        bits = np.unpackbits(allowed.view(np.uint8), axis=1, bitorder="little")[:, :V].astype(bool)
        x = np.where(bits, x, f(-np.inf))
    return x


def greedy_plain(x):
    return np.array([int(np.argmax(np.isnan(r))) if np.isnan(r).any() else int(np.argmax(r)) for r in x])


def same_bits(a, b):
    return np.array_equal(a.view(np.int32), b.view(np.int32)) or (
        np.array_equal(np.isnan(a), np.isnan(b)) and np.array_equal(a[~np.isnan(a)], b[~np.isnan(b)]))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("N,V,K", [(1, 1, 0), (1, 31, 1), (2, 64, 5), (3, 4096, 0), (5, 4097, 300), (2, 32_003, 7),
                                   (1, 128_256, 16), (3, 50_000, 2000),
                                   # more rows, fewer CTAs each: slices of several rounds, aligned rows and not
                                   (40, 70_000, 9), (80, 40_001, 0), (2, 400_000, 4096)])
def test_penalize_logits(dtype, N, V, K):
    g = gen(N * V + K)
    x = randn(g, N, V, dtype=dtype) * 3
    if V > 100:
        x[:, ::97] = 0
        x[0, 5], x[0, 6], x[-1, 7] = math.inf, -math.inf, -0.0
    prompt = torch.randint(0, V, (N, 40), generator=g, device="cuda")
    output = torch.randint(0, max(1, V // 3), (N, 60), generator=g, device="cuda").int()
    lengths = torch.randint(0, 61, (N,), generator=g, device="cuda", dtype=torch.int32)
    prompt[:, 3], prompt[:, 4], output[:, 5] = -1, V, 2 ** 31 - 1  # padding and what is no token
    h = TokenHistory(N, V)
    h.add_prompt(prompt)
    h.append(output, lengths)
    h.append(prompt[:, 0])
    counts, in_prompt = np.zeros((N, V), np.int64), np.zeros((N, V), bool)
    for n in range(N):
        for t in prompt[n].tolist():
            if 0 <= t < V:
                in_prompt[n, t] = True
        for t in output[n, :int(lengths[n])].tolist() + prompt[n, :1].tolist():
            if 0 <= t < V:
                counts[n, t] += 1
    words = h.counts.cpu().numpy().view(np.uint32)
    assert np.array_equal(words & 0x7FFFFFFF, counts) and np.array_equal(words >> 31 == 1, in_prompt)
    rep = 1 + torch.rand(N, generator=g, device="cuda")
    pres, freq = torch.rand(N, generator=g, device="cuda") - 0.3, torch.rand(N, generator=g, device="cuda")
    bias = None
    if K:
        ids = torch.randint(0, V, (N, K), generator=g, device="cuda", dtype=torch.int32)
        ids[:, K // 2] = -1
        ids[:, -1] = ids[:, 0]  # listed twice
        if K > 2:
            ids[:, K // 3] = ids[:, 0]
        bias = (ids, 5 * randn(g, N, K))
    allowed = torch.randint(-2 ** 31, 2 ** 31, (N, -(-V // 32)), generator=g, device="cuda").to(torch.int32)
    allowed[-1] = 0  # nothing
    num = lambda t: t.cpu().numpy()  # noqa: E731
    for a in (None, allowed):
        want = penalize_plain(x, counts, in_prompt, num(rep), num(pres), num(freq), bias,
                              None if a is None else num(a))
        got, ids = penalize_logits(x, h, repetition=rep, presence=pres, frequency=freq, bias=bias, allowed=a,
                                   greedy=True)
        assert same_bits(num(got), want)
        assert np.array_equal(num(ids), greedy_plain(want))
        # in place, and rounded to bf16
        y = x.clone()
        assert penalize_logits(y, h, repetition=rep, presence=pres, frequency=freq, bias=bias, allowed=a, out=y) is y
        assert torch.equal(y.float().nan_to_num(7), torch.from_numpy(want).cuda().to(dtype).float().nan_to_num(7))
        z = torch.empty((N, V), dtype=BF16, device="cuda")
        penalize_logits(x, h, repetition=rep, presence=pres, frequency=freq, bias=bias, allowed=a, out=z)
        assert torch.equal(z.float().nan_to_num(7), torch.from_numpy(want).cuda().to(BF16).float().nan_to_num(7))
    # numbers in the place of tensors
    want = penalize_plain(x, counts, in_prompt, np.full(N, 1.5, np.float32), np.full(N, 0.25, np.float32),
                          np.full(N, 0.5, np.float32), None, None)
    got = penalize_logits(x, h, repetition=1.5, presence=0.25, frequency=0.5)
    assert same_bits(num(got), want)
    h.reset()
    assert same_bits(num(penalize_logits(x, h, repetition=1.5, presence=0.25, frequency=0.5)), num(x.float()))


def test_penalize_logits_rows_and_strides():
    g = gen(8)
    N, V = 4, 1000
    x = randn(g, N, 3, V + 24, dtype=BF16)[:, 1, 3:V + 3]  # the last position of a larger tensor, misaligned
    allowed = torch.randint(-2 ** 31, 2 ** 31, (2, -(-V // 32)), generator=g, device="cuda").to(torch.int32)
    rows = torch.tensor([1, -1, 2, 0], dtype=torch.int32, device="cuda")  # -1 and 2: no mask
    full = torch.full((4, allowed.shape[1]), -1, dtype=torch.int32, device="cuda")
    full[0], full[3] = allowed[1], allowed[0]
    want = penalize_plain(x, None, None, None, None, None, None, full.cpu().numpy())
    out = torch.full((N, V + 8), 9.0, device="cuda")
    got, ids = penalize_logits(x, allowed=allowed, allowed_rows=rows, out=out[:, :V], greedy=True)
    assert same_bits(got.cpu().numpy(), want) and (out[:, V:] == 9).all()
    assert np.array_equal(ids.cpu().numpy(), greedy_plain(want))
    assert penalize_logits(x[:0]).shape == (0, V)


@pytest.mark.parametrize("N,V,V_of_ids", [(75, 1 << 21, 1 << 21), (75, 1 << 21, 64), (2, 700, 3), (20, 5_001, 5_001)])
def test_biases_as_many_as_a_row_may_have(N, V, V_of_ids):
    """4096 biases of a row -- of few tokens, or of the largest vocabulary -- added up in their order."""
    g = gen(V_of_ids + N)
    x = torch.zeros((N, V), device="cuda", dtype=BF16)
    ids = torch.randint(0, V_of_ids, (N, 4096), generator=g, device="cuda").int()
    ids[:, 1000:1003] = -1
    values = randn(g, N, 4096)
    got, best = penalize_logits(x, bias=(ids, values), greedy=True)
    for n in {0, N // 2, N - 1}:
        want = np.zeros(V, np.float32)
        for i, v in zip(ids[n].tolist(), values[n].cpu().numpy()):
            if i >= 0:
                want[i] += v  # from 0 instead of from the first: the same sum
        assert same_bits(got[n].cpu().numpy() + np.float32(0), want)
        assert best[n] == int(np.argmax(want))
    assert int((got != 0).sum()) <= N * 4096


def test_greedy_ties_nan_and_empty_rows():
    V = 40_000
    x = torch.zeros((5, V), device="cuda")
    x[0, 123] = x[0, 30_000] = 4.0
    x[1] = -0.0
    x[1, 39_999] = 0.0
    x[2, 17], x[2, 20_000] = math.inf, math.nan
    x[3] = -math.inf
    x[4, 39_000], x[4, 38_999] = 2.0, 1.0
    allowed = torch.full((5, V // 32), -1, dtype=torch.int32, device="cuda")
    allowed[4, 39_000 // 32] = 0
    allowed[4, 38_999 // 32] = 0
    _, ids = penalize_logits(x, allowed=allowed, greedy=True)
    assert ids.tolist() == [123, 0, 20_000, 0, 0]
    allowed[2, 20_000 // 32] = 0  # a masked NaN counts no more
    out, ids = penalize_logits(x, allowed=allowed, greedy=True)
    assert ids[2] == 17 and torch.isinf(out[2, 20_000])


# -- together, on streams and in graphs --------------------------------------------------
def test_prefill_evict_decode():
    """A prompt is prefilled, scored and cut, then decoded over the kept keys,
    rotated by tokens seen: every step against plain attention over the same keys."""
    labels = np.array([[1, 0, 1], [0, 1, 1]])
    L, G, Hq, T, keep, sink, recent = 2, 3, 12, 600, 300, 16, 64
    g = gen(11)
    inv = 1e4 ** (-torch.arange(64, device="cuda", dtype=F32) / 64)
    cache = AoHKVCache(labels, Hq, sink_size=sink, recent_size=recent, max_context=T)
    small = AoHKVCache(labels, Hq, sink_size=sink, recent_size=recent, max_context=keep + 8)
    sums = KeyWeights(cache)
    keys = [[[] for _ in range(G)] for _ in range(L)]  # what plain attention holds, per head: (k, v)
    weights = [torch.zeros(len(np.flatnonzero(labels[i])), 0, dtype=torch.float64) for i in range(L)]
    for c in (256, 344):
        past = cache.kv_seq_len
        pos = torch.arange(past, past + c, device="cuda").expand(3, 1, c)
        for i in range(L):
            q, k, v = (randn(g, 1, c, h, 128, dtype=BF16) for h in (Hq, G, G))
            q, k = rope_axes_qk(q, k, pos, inv, (24, 20, 20))
            aoh_attention(cache, i, q, k, v)
            sums.add(i, q, past_len=past)
            for h in range(G):
                keys[i][h].append((k[0, :, h].double(), v[0, :, h].double()))
            kk = torch.stack([torch.cat([a for a, _ in keys[i][h]]) for h in range(G)], 1)[None]
            w, tol = weights_exact(q, kk, list(np.flatnonzero(labels[i])), past)
            weights[i] = torch.nn.functional.pad(weights[i], (0, c)) + w[0]
            got = sums.layer(i)[0, :, :past + c].double().cpu()
            assert ((got - weights[i]).abs() <= 2 * tol * weights[i] + 2.0 ** -100).all()
    kept, _ = select_keys(sums.rows[:, :T], keep, sink=sink, recent=recent)
    new = sums.evict(keep, small)
    assert torch.equal(new.rows[:, :keep], torch.gather(sums.rows, 1, kept.long())) and (new.rows[:, keep:] == 0).all()
    assert (small.kv_seq_len, small.tokens_seen) == (keep, T)
    held, r = {}, 0
    for i in range(L):
        for h in range(G):
            k, v = (torch.cat([t[j] for t in keys[i][h]]) for j in (0, 1))
            at = kept[r].long() if labels[i][h] else torch.cat((torch.arange(sink), torch.arange(T - recent, T))).cuda()
            r += int(labels[i][h])
            held[i, h] = [k[at], v[at]]
    for step in range(3):
        past = small.kv_seq_len
        pos = torch.full((3, 1, 1), small.tokens_seen, device="cuda")
        assert small.tokens_seen == T + step
        for i in range(L):
            q, k, v = (randn(g, 1, 1, h, 128, dtype=BF16) for h in (Hq, G, G))
            q, k = rope_axes_qk(q, k, pos, inv, (24, 20, 20))
            out = aoh_attention(small, i, q, k, v)
            new.add(i, q, past_len=past)
            for h in range(G):
                kk, vv = (torch.cat((held[i, h][j], t[0, :, h].double())) for j, t in ((0, k), (1, v)))
                qq = q[0, 0, h * 4:(h + 1) * 4].double()
                p = torch.softmax(qq @ kk.T / math.sqrt(128), -1)
                assert ((out[0, 0, h * 4:(h + 1) * 4].double() - p @ vv).abs() <= 2e-2).all()
                if not labels[i][h]:  # the window moves on
                    kk, vv = (torch.cat((t[:sink], t[sink + 1:])) for t in (kk, vv))
                held[i, h] = [kk, vv]
    # the kept sums and the three steps' weights: 4 heads a step
    total = new.rows[:, :small.kv_seq_len].double().sum(1)
    was = torch.gather(sums.rows, 1, kept.long()).double().sum(1)
    assert ((total - was - 12).abs() <= 1e-3).all()
    assert small.device_status() == 0 and cache.device_status() == 0


def test_key_weights_object():
    """Rows by layer and sequence, sums moved by an eviction, sequences shorter than the window."""
    labels = [[1, 0, 1], [0, 0, 0], [0, 1, 0]]
    cache, k, _ = filled(labels, 6, 2, 60, BF16, 14, 16, 48, max_context=70)
    sums = KeyWeights(cache)
    assert sums.rows.shape == (6, 70)
    q = [randn(gen(i), 2, 2, 6, 128, dtype=BF16) for i in range(3)]
    for _ in range(2):
        for layer in range(3):
            sums.add(layer, q[layer], past_len=58)
    for layer, heads in ((0, [0, 2]), (2, [1])):
        want, tol = weights_exact(q[layer], k[layer], heads, 58)
        got = sums.layer(layer)[:, :, :60].double().cpu()
        assert got.shape == want.shape and ((got - 2 * want).abs() <= 2 * tol * want + 2.0 ** -100).all()
    assert (sums.rows[:, 60:] == 0).all()
    # 60 tokens are fewer than the sink and the window: all of them stay
    into = AoHKVCache(labels, 6, batch=2, sink_size=16, recent_size=48, max_context=80)
    moved = sums.evict(60, into)
    assert torch.equal(moved.rows[:, :60], sums.rows[:, :60]) and moved.cache is into and into.tokens_seen == 60
    with pytest.raises(ValueError):
        sums.evict(50, into)  # some would have to go, and the window does not fit
    with pytest.raises(ValueError):
        sums.evict(61, into)


def test_operators_on_a_side_stream_and_in_a_graph():
    g = gen(12)
    labels = [[1, 0, 1]]
    cache, k, v = filled(labels, 6, 1, 500, BF16, 12, 16, 32, max_context=512)
    into = AoHKVCache(labels, 6, sink_size=16, recent_size=32, max_context=128, reserve_all=True)
    q0, k0 = randn(g, 1, 2, 6, 128, dtype=BF16), randn(g, 1, 2, 3, 128, dtype=BF16)
    pos = torch.arange(498, 500, device="cuda").expand(1, 1, 2)
    inv = 1e4 ** (-torch.arange(64, device="cuda", dtype=F32) / 64)
    x = randn(g, 3, 5000, dtype=BF16)
    h = TokenHistory(3, 5000)
    tok = torch.tensor([1, 2, 3], device="cuda")

    def step():
        q, kk = rope_axes_qk(q0, k0, pos, inv, (64,))
        w = key_weights(cache, 0, q, past_len=498)
        kept, kw = select_keys(w.view(2, -1), 100, sink=16, recent=32)
        evict(cache, kept, into)
        h.append(tok)
        y, ids = penalize_logits(x, h, frequency=0.5, greedy=True)
        return q, kk, w, kept, kw, y, ids, into.pool

    h.reset()
    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        h.reset()
        into.pool.zero_()
        torch.cuda._sleep(20_000_000)  # work enqueued on another stream would run ahead of the reset
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    # two graphs, replayed in turn and beside one another on two streams
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            w = key_weights(cache, 0, q0, past_len=498)
            kept, kw = select_keys(w.view(2, -1), 100, sink=16, recent=32)
            y, ids = penalize_logits(x, frequency=None, greedy=True)
        graphs.append((gr, (w, kept, kw, y, ids)))
    w = key_weights(cache, 0, q0, past_len=498)
    eager = (w, *select_keys(w.view(2, -1), 100, sink=16, recent=32), *penalize_logits(x, greedy=True))
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    for _ in range(20):
        graphs[0][0].replay()
        with torch.cuda.stream(other):
            graphs[1][0].replay()
    torch.cuda.synchronize()
    for _, outs in graphs:
        assert all(torch.equal(a, b) for a, b in zip(eager, outs))


def test_operators_wait_for_copies_from_the_host():
    """A kernel, a long copy from pinned memory, an operator on what arrives, a copy back."""
    g = gen(9)
    host = [torch.randn((64, 128_256), generator=torch.Generator().manual_seed(i)).pin_memory() for i in range(3)]
    x, out = torch.empty((64, 128_256), device="cuda"), torch.empty((64, 128_256), device="cuda")
    back = torch.empty((64, 128_256)).pin_memory()
    q0, k0 = randn(g, 1, 64, 8, 128), randn(g, 1, 64, 8, 128)
    pos, inv = torch.arange(64, device="cuda").expand(1, 1, 64), torch.ones(64, device="cuda")
    for i in range(9):
        rope_axes_qk(q0, k0, pos, inv, (64,))
        x.copy_(host[i % 3], non_blocking=True)
        _, ids = penalize_logits(x, out=out, greedy=True)
        back.copy_(out, non_blocking=True)
        x.fill_(9.0)
        torch.cuda.synchronize()
        assert torch.equal(back, host[i % 3]) and torch.equal(ids.cpu(), host[i % 3].argmax(1))


def test_captured_behind_copies_and_joined_streams():
    """In a captured graph: the first node, behind a copy, behind a fill, and where two streams meet."""
    g = gen(5)
    cache, k, _ = filled([[1, 1]], 8, 1, 600, BF16, 5)
    q0, k0 = randn(g, 1, 1, 8, 128, dtype=BF16), randn(g, 1, 1, 2, 128, dtype=BF16)
    pos, inv = torch.full((1, 1, 1), 599, device="cuda"), 1e4 ** (-torch.arange(64, device="cuda", dtype=F32) / 64)
    x, buf = randn(g, 2, 9_000), torch.empty(2, 9_000, device="cuda")

    def steps(side):
        main = torch.cuda.current_stream()
        q, kk = rope_axes_qk(q0, k0, pos, inv, (64,))
        buf.copy_(x)
        y, ids = penalize_logits(buf, greedy=True)
        w = key_weights(cache, 0, q, past_len=599)
        side.wait_stream(main)
        with torch.cuda.stream(side):
            w2 = key_weights(cache, 0, q, past_len=599)
            kept2, _ = select_keys(w2.view(2, 600), 50)
        w.zero_()
        key_weights(cache, 0, q, past_len=599, out=w, accumulate=True)
        main.wait_stream(side)
        kept, kw = select_keys(w.view(2, 600), 50)
        return q, kk, y, ids, w, w2, kept2, kept, kw

    want = [t.clone() for t in steps(torch.cuda.Stream())]
    torch.cuda.synchronize()
    gr, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(gr):
        got = steps(side)
    for _ in range(3):
        for t in got:
            t.zero_()
        gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("dtype,C,T", [(BF16, 1, 30_000), (BF16, 4, 2_000), (BF16, 64, 9_000), (BF16, 700, 5_000),
                                       (F32, 30, 3_000)])
def test_each_operator_waits_for_the_one_before(dtype, C, T):
    """The operators one behind the other, each fed by the last one, give what they give one at a time."""
    g = gen(T)
    labels, Hq, keep = [[1, 0, 1, 1]], 16, 400
    cache, k, _ = filled(labels, Hq, 1, T, dtype, C, 16, 32)
    into = AoHKVCache(labels, Hq, sink_size=16, recent_size=32, max_context=512, dtype=dtype, reserve_all=True)
    q0, k0 = randn(g, 1, C, Hq, 128, dtype=dtype), randn(g, 1, C, 4, 128, dtype=dtype)
    pos = torch.arange(T - C, T, device="cuda").expand(1, 1, C)
    inv = 1e4 ** (-torch.arange(64, device="cuda", dtype=F32) / 64)
    x = randn(g, 40, 60_000, dtype=dtype)

    def steps(after):
        out = []
        h = TokenHistory(40, 60_000)
        q = rope_axes_qk(q0, k0, pos, inv, (64,))[0]
        after()
        q = rope_axes_qk(q, k0, pos, inv, (64,))[0]
        after()
        w = key_weights(cache, 0, q, past_len=T - C)
        after()
        key_weights(cache, 0, q, past_len=T - C, out=w, accumulate=True)
        after()
        kept, kw = select_keys(w.view(3, T), keep, sink=16, recent=32)
        after()
        evict(cache, kept, into)
        after()
        w2 = key_weights(into, 0, q[:, :1].contiguous(), past_len=keep - 1)
        after()
        y, ids = penalize_logits(x, greedy=True)
        for _ in range(3):
            after()
            h.append(ids)
            after()
            y, ids = penalize_logits(y, h, frequency=3.0, presence=2.0, out=y, greedy=True)
            out.append(ids)
        return [q, w, kept, kw, w2, y, *out]

    want = steps(torch.cuda.synchronize)
    for _ in range(5):
        into.pool.zero_()
        got = steps(lambda: None)
        assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("dtype,C,T", [
    (BF16, 1, 20_000), (BF16, 2, 700),      # few query rows: two launches, one
    (BF16, 40, 3_000), (BF16, 300, 3_000),  # the tensor cores: query rows resident, keys resident
    (F32, 9, 1_000),
])
def test_key_weights_in_two_graphs_and_eager_at_once(dtype, C, T):
    """Each call has its own workspace: graphs replayed beside one another and beside an eager call."""
    cache, k, _ = filled([[1, 1]], 8, 1, T, dtype, C)
    qs = [randn(gen(i), 1, C, 8, 128, dtype=dtype) for i in range(3)]
    want = [key_weights(cache, 0, q, past_len=T - C) for q in qs]
    graphs = []
    for q in qs[:2]:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            w = key_weights(cache, 0, q, past_len=T - C)
            key_weights(cache, 0, q, past_len=T - C, out=w, accumulate=True)
        graphs.append((gr, w))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(10):
        for (gr, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
        eager = key_weights(cache, 0, qs[2], past_len=T - C)
    torch.cuda.synchronize()
    assert torch.equal(eager, want[2])
    for (_, w), x in zip(graphs, want):
        # added to what one call gave: blocks of rows or ranges may be added one by one
        assert ((w - 2 * x).abs() <= 4 * 2.0 ** -24 * w).all()


def test_key_weights_with_the_devices_length():
    """A captured single-token call reads the length that the graph advances."""
    from aoh_b200 import _lib

    cache, k, _ = filled([[1, 0]], 8, 2, 300, BF16, 13, max_context=320)
    cache.reserve(320)
    q = randn(gen(2), 2, 1, 8, 128, dtype=BF16)
    out = torch.zeros((2, 1, 320), device="cuda")
    key_weights(cache, 0, q, past_len=280)  # set up before the capture
    lib = _lib.lib()
    st = lambda: _lib.stream_handle()  # noqa: E731
    _lib.check(lib.aoh_kv_set_length(cache._h, 280, st()))
    cache.device_length = True
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        key_weights(cache, 0, q, out=out, accumulate=True)
        _lib.check(lib.aoh_kv_advance(cache._h, 1, st()))
    cache.device_length = False
    _lib.check(lib.aoh_kv_set_length(cache._h, 280, st()))
    want = torch.zeros_like(out)
    for past in range(280, 284):
        gr.replay()
        want[..., :past + 1] += key_weights(cache, 0, q, past_len=past)
    # the split into key ranges may differ from the plan for the full length: fp32 sums in another order
    assert torch.allclose(out, want, rtol=1e-4, atol=0) and (out[..., 284:] == 0).all()


def test_key_weights_f32_with_the_devices_length():
    from aoh_b200 import _lib

    cache, k, _ = filled([[1, 0]], 8, 2, 150, F32, 13, max_context=160)
    cache.reserve(160)
    q = randn(gen(2), 2, 1, 8, 128, dtype=F32)
    out = torch.full((2, 1, 170), 3.0, device="cuda")
    _lib.check(_lib.lib().aoh_kv_set_length(cache._h, 140, _lib.stream_handle()))
    cache.device_length = True
    key_weights(cache, 0, q, out=out)
    cache.device_length = False
    check_weights(out[..., :141], q, k[0][:, :141], [0], 140)
    assert (out[..., 141:] == 3).all()


# -- refusals -------------------------------------------------------------------------
def test_refusals():
    q, k = torch.zeros(1, 2, 4, 64, device="cuda"), torch.zeros(1, 2, 2, 64, device="cuda")
    pos, inv = torch.zeros(1, 1, 2, dtype=torch.int64, device="cuda"), torch.ones(32, device="cuda")
    ok = dict(q=q, k=k, positions=pos, inv_freq=inv, sections=(32,))
    rope_axes_qk(**ok)
    for bad in (dict(q=q[0]), dict(q=q.cpu()), dict(q=q.half()), dict(k=k.bfloat16()), dict(k=k[:, :1]),
                dict(q=q.transpose(2, 3)), dict(positions=pos.float()), dict(positions=pos[0]), dict(sections=(16, 16)),
                dict(sections=(31,)), dict(inv_freq=inv.double()), dict(inv_freq=torch.ones(64, device="cuda")[::2]),
                dict(q_norm_weight=torch.ones(64, device="cuda")), dict(sections=(40, -8), positions=pos.expand(2, 1, 2)),
                dict(sections=(16, 16), positions=pos.expand(2, 1, 2), interleaved=True, k=k[..., :63], q=q[..., :63]),
                dict(sections=(2, 30), positions=pos.expand(2, 1, 2), interleaved=True)):
        with pytest.raises((ValueError, NotImplementedError)):
            rope_axes_qk(**{**ok, **bad})
    cache, _, _ = filled([[1, 0]], 4, 1, 100, BF16, 1, 16, 32)
    qq = torch.zeros(1, 2, 4, 128, device="cuda", dtype=BF16)
    with pytest.raises(ValueError):
        key_weights(cache, 1, qq, past_len=98)
    with pytest.raises(ValueError):
        key_weights(cache, 0, qq.float(), past_len=98)
    with pytest.raises(torch.OutOfMemoryError):
        key_weights(cache, 0, qq)  # the tokens are not cached
    for out in (torch.zeros(1, 1, 99, device="cuda"), torch.zeros(1, 2, 100, device="cuda"),
                torch.zeros(1, 1, 100, device="cuda", dtype=torch.float64), torch.zeros(1, 1, 200, device="cuda")[..., ::2]):
        with pytest.raises(ValueError):
            key_weights(cache, 0, qq, past_len=98, out=out)
    with pytest.raises(ValueError):
        key_weights(cache, 0, qq, past_len=98, accumulate=True)
    with pytest.raises(ValueError):
        key_weights(cache, 0, qq, past_len=-1)
    w = torch.zeros(2, 10, device="cuda")
    for args in (dict(keep=11), dict(keep=-1), dict(keep=5, sink=3, recent=3), dict(keep=5, sink=-1)):
        with pytest.raises(ValueError):
            select_keys(w, **args)
    with pytest.raises(ValueError):
        select_keys(w.double(), 3)
    with pytest.raises(ValueError):
        select_keys(w.cpu(), 3)
    kept = torch.zeros(1, 60, device="cuda", dtype=torch.int32)
    make = lambda **a: AoHKVCache(**{**dict(labels=[[1, 0]], num_q_heads=4, sink_size=16, recent_size=32,  # noqa: E731
                                            max_context=100), **a})
    for into, kk in ((cache, kept), (make(recent_size=48), kept), (make(labels=[[0, 1]]), kept),
                     (make(dtype=F32), kept), (make(max_context=59), kept), (make(), kept.long()), (make(), kept[0]),
                     (make(), kept[:, :40]), (make(), kept.expand(2, 60))):
        with pytest.raises(ValueError):
            evict(cache, kk, into)
    x = torch.zeros(2, 64, device="cuda")
    h = TokenHistory(2, 64)
    i2 = torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    for args in (dict(logits=x[0]), dict(logits=x.cpu()), dict(logits=x.half()), dict(logits=x.t()),
                 dict(history=None, repetition=1.5), dict(logits=x[:, :32]), dict(repetition=0.0),
                 dict(repetition=torch.ones(3, device="cuda")), dict(presence=torch.ones(2, device="cuda").double()),
                 dict(bias=(i2.long(), i2.float())), dict(bias=(i2, i2.float()[:, :2])), dict(allowed=i2),
                 dict(allowed=i2[:1, :2].contiguous()), dict(allowed_rows=i2[:, 0]), dict(out=x[:1]),
                 dict(out=x.half()), dict(out=torch.zeros(64, device="cuda").expand(2, 64)),
                 dict(out=torch.zeros(64, 2, device="cuda").t())):
        with pytest.raises(ValueError):
            penalize_logits(**{**dict(logits=x, history=h), **args})
    for ids in (torch.zeros(3, 1, dtype=torch.int64, device="cuda"), torch.zeros(2, 1, device="cuda"),
                torch.zeros(2, 1, dtype=torch.int64)):
        with pytest.raises(ValueError):
            h.append(ids)
    with pytest.raises(ValueError):
        TokenHistory(2, 0)
