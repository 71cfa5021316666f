"""Edges of the operators around a decode step."""
import math

import numpy as np
import pytest
import torch

from aoh_b200 import (AoHKVCache, KeyWeights, TokenHistory, _lib, evict, key_weights, penalize_logits, rope_axes_qk,
                      select_keys)
from tests.test_operators_gpu import check_rope, check_select, check_weights, filled, gen, randn

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


# -- clusters ---------------------------------------------------------------------
@pytest.mark.parametrize("N,V", [(5, 8_192), (9, 16_384), (16, 30_008), (16, 65_536), (27, 131_072), (70, 131_072),
                                 (90, 131_072), (24, 32_771)])
def test_greedy_token_of_every_cta_of_a_cluster(N, V):
    """The largest logit in each CTA's part of the vocabulary in turn (64 tokens a turn, up to 16 CTAs)."""
    x = randn(gen(V), N, V, dtype=BF16).clamp(max=3)
    at = [(64 * r + 7 * r % 64) % V for r in range(N)]
    at[-1] = V - 1
    for r, t in enumerate(at):
        x[r, t] = 4
    outs = [penalize_logits(x, greedy=True) for _ in range(20)]  # one behind the other
    for out, ids in outs:
        assert ids.tolist() == at and torch.equal(out, x.float())


@pytest.mark.parametrize("rows,n", [(1, 9_000), (3, 16_384), (2, 20_000), (1, 40_000), (2, 70_001), (2, 300_000)])
def test_select_keys_in_clusters_one_behind_the_other(rows, n):
    """Clusters of 2 to 8, parts in registers and in memory."""
    w = (torch.rand((rows, n), generator=gen(n), device="cuda") * 50).floor()
    check_select(w, n // 3, 4, 9)
    outs = [select_keys(w, n // 3, sink=4, recent=9) for _ in range(20)]
    assert all(torch.equal(a, b) for o in outs for a, b in zip(o, outs[0]))


def test_select_keys_of_the_longest_row():
    """2^31 - 1 keys, as many as 32 bits count: parts of 2^28 keys."""
    n = 2 ** 31 - 1
    at = [3, 2 ** 28 - 1, 2 ** 28, 2 ** 30 + 17, 2 ** 31 - 9]
    w = torch.zeros(1, n, device="cuda")
    w[0, at] = torch.tensor([1.0, 5.0, 2.0, 3.0, 4.0], device="cuda")
    kept, kw = select_keys(w, 9, sink=1, recent=1)
    want = sorted([0, 1, 2, *at, n - 1])
    assert kept[0].tolist() == want and torch.equal(kw, w[:, want])


def test_sizes_that_32_bits_do_not_count_are_refused():
    """Cut to 32 bits they would be other sizes."""
    w = torch.empty(2 ** 32 + 40, device="cuda", dtype=torch.float32)  # 17 GB, never read
    with pytest.raises(ValueError):
        select_keys(w, 10)
    with pytest.raises(ValueError):
        select_keys(w[:, None], 1)
    history = TokenHistory(1, 8)
    with pytest.raises(ValueError):
        history.append(w.view(torch.int32)[None])
    cache, _, _ = filled([[1]], 1, 1, 20, BF16, 1, 0, 0)
    with pytest.raises(ValueError):
        key_weights(cache, 0, torch.zeros(1, 1, 1, 128, device="cuda", dtype=BF16), past_len=2 ** 32 + 19,
                    out=w[None, None])


# -- key weights ------------------------------------------------------------------
@pytest.mark.parametrize("C,grp,T", [(32, 7, 90_000), (40, 3, 70_001), (5, 8, 120_003)])
def test_key_weights_of_resident_rows_over_many_tiles(C, grp, T):
    """One and two tiles of query rows, ranges of many key tiles: every stage of the ring is used several times."""
    cache, k, _ = filled([[1, 1, 0]], 3 * grp, 1, T, BF16, C)
    q = randn(gen(C), 1, C, 3 * grp, 128, dtype=BF16)
    outs = [key_weights(cache, 0, q, past_len=T - C) for _ in range(4)]
    check_weights(outs[0], q, k[0], [0, 1], T - C)
    assert all(torch.equal(x, outs[0]) for x in outs) and cache.device_status() == 0


def test_the_sums_exp2_polynomial():
    """Against 2^x in 64 bits: 1.55e-7 of the fit and five roundings of at most 2^-24 each, of which the fit's factors
    f <= 1/2 leave one and a half: below 2.5e-7; at the clamped end next to nothing."""
    xs = np.concatenate([np.linspace(-126, 8, 2_000_001), np.arange(-126, 9), np.arange(-126, 8) + 0.5,
                         [-126.5, -1000, -np.inf]]).astype(np.float32)
    x = torch.from_numpy(xs).cuda()
    out = torch.empty_like(x)
    _lib.check(_lib.lib().aoh_diag_exp2_poly_f32(x.data_ptr(), out.data_ptr(), x.numel(), _lib.stream_handle()))
    got, want = out.cpu().numpy().astype(np.float64), np.exp2(xs.astype(np.float64))
    m = xs >= -125
    assert (np.abs(got[m] - want[m]) <= 2.5e-7 * want[m]).all()
    assert (got[~m] >= 0).all() and (np.abs(got[~m] - want[~m]) <= 2.0 ** -125).all()


@pytest.mark.parametrize("C,row", [(c, r) for c in (3, 40, 200, 300, 700)
                                   for r in (0, 1, 14, 15, 31, 39, 46, 47, 143, 270, 655) if r < c])
def test_key_weights_of_exact_scores(C, row):
    """Scores without an error of their own: what is left is the softmax's.  One query row spreads its weight over
    1024 keys, the others give theirs to one key; every product has one term that is not zero.

    Bound, in steps of 2^-24 of an exponent's error times ln 2: the scale's constant, 3 x 12; the exponent's own
    rounding, 32 (|x| < 64), in the weight and in the sum's terms; -lse's rounding 16 (below 32) and its logarithm's
    8; the sum's additions, 8 a key tile of a thread, at most 9 tiles, and 16 of the merges, 88 / ln 2, and an
    exponential's 2.5e-7 (4.2 steps) in both, 12: (2 * (36 + 32) + 24 + 127 + 12) = 299 steps = 1.24e-5.  The one
    key's weight: its maximum of 98 and -lse rounded, 64 steps each, and the additions: fewer."""
    T, keys = 1024 + C, 1024
    cache = AoHKVCache([[1]], 1, sink_size=0, recent_size=0, max_context=T)
    k = torch.zeros(1, T, 1, 128, device="cuda", dtype=BF16)
    k[0, :keys, 0, 5] = (12 * torch.rand(keys, generator=gen(row), device="cuda") - 6).to(BF16)
    k[0, 7, 0] = 0
    k[0, 7, 0, 9] = 24  # takes the other rows' weight
    k[0, keys:, 0, 5] = -100  # out of reach of the row
    cache.append_layer(0, k, k)
    q = torch.zeros(1, C, 1, 128, device="cuda", dtype=BF16)
    q[0, :, 0, 9] = 32
    q[0, row, 0] = 0
    q[0, row, 0, 5] = 8
    got = key_weights(cache, 0, q, past_len=keys)[0, 0].double().cpu()
    x = 8 * k[0, :keys + row + 1, 0, 5].double().cpu() / math.sqrt(128)
    want = torch.zeros(T, dtype=torch.float64)
    want[:keys + row + 1] = torch.softmax(x, 0)
    want[7] += C - 1
    assert ((got - want).abs() <= 1.24e-5 * want + 2.0 ** -80).all()


# -- caches used again --------------------------------------------------------------
def test_a_cache_used_again_starts_from_nothing(cuda_device):
    """After an eviction and for the next prompt: positions and sums are those of a fresh cache."""
    from aoh_b200.hf import patch_aoh_model
    from tests.test_hf_gpu import _tiny
    from tests.test_operators_hf_gpu import LABELS, _prompt, _run

    model = _tiny("llama")
    make_cache, _, _ = patch_aoh_model(model, LABELS, 16, 48)
    first, second = _prompt(250, seed=1), _prompt(180, seed=2)
    fresh = make_cache(max_context=300)
    fresh.track_weights()
    want = _run(model, fresh, second, [0, 100, 179, 180])
    used = make_cache(max_context=300)
    used.track_weights()
    _run(model, used, first, [0, 250])
    moved = used.evict(120, max_context=300)
    assert moved.get_seq_length() == 250
    for cache, restart in ((used, lambda c: setattr(c, "kv_seq_len", 0)), (moved, lambda c: c.reset())):
        restart(cache)
        assert cache.get_seq_length() == cache.paged.tokens_seen == cache.paged.evicted == 0
        got = _run(model, cache, second, [0, 100, 179, 180])
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert torch.equal(cache.key_weights.rows, fresh.key_weights.rows)
        assert cache.get_seq_length() == 180 and cache.paged.device_status() == 0


def test_sums_forget_dropped_tokens():
    """Tokens taken back and decoded otherwise: their keys' sums are those of the new tokens alone."""
    cache, k, _ = filled([[1, 0, 1]], 6, 1, 200, BF16, 1, max_context=256)
    sums, other = KeyWeights(cache), KeyWeights(cache)
    q = randn(gen(1), 1, 200, 6, 128, dtype=BF16)
    sums.add(0, q, past_len=0)
    kept = sums.rows[:, :150].clone()
    cache.kv_seq_len = 150
    assert torch.equal(sums.rows[:, :150], kept) and (sums.rows[:, 150:] == 0).all() and (other.rows == 0).all()
    again = randn(gen(2), 1, 50, 3, 128, dtype=BF16)
    cache.append_layer(0, again, again)
    sums.add(0, q[:, 150:])
    new = key_weights(cache, 0, q[:, 150:])
    cache.kv_seq_len = 200
    assert torch.equal(sums.rows[:, 150:200], new[0, :, 150:])
    cache.reset()
    assert (sums.rows == 0).all()


def test_evicting_into_a_cache_that_is_tracked():
    """What the destination held is given up, its sums too."""
    cache, _, _ = filled([[1, 0]], 4, 1, 120, BF16, 1, 16, 32)
    into, _, _ = filled([[1, 0]], 4, 1, 200, BF16, 2, 16, 32)
    old = KeyWeights(into)
    old.add(0, randn(gen(1), 1, 200, 4, 128, dtype=BF16), past_len=0)
    assert (old.rows > 0).all()
    evict(cache, torch.arange(60, device="cuda", dtype=torch.int32)[None], into)
    assert (old.rows == 0).all() and (into.kv_seq_len, into.evicted) == (60, 60)


# -- rotary positions ----------------------------------------------------------------
@pytest.mark.parametrize("D,sections", [(128, (64,)), (80, (12, 10, 10)), (256, (100, 28)), (70, (17, 3))])
@pytest.mark.parametrize("dtype,wq,wk", [(BF16, F32, F32), (BF16, F32, BF16), (F32, BF16, F32),
                                         (BF16, torch.float16, F32), (BF16, torch.float16, torch.float16)])
def test_norm_weights_of_another_type_are_not_rounded(dtype, wq, wk, D, sections):
    """fp32 weights beside bf16 rows: rounded once, in the result."""
    g = gen(D)
    q, k = randn(g, 2, 37, 6, D, dtype=dtype), randn(g, 2, 37, 2, D, dtype=dtype)
    pos = torch.randint(0, 100_000, (len(sections), 2, 37), generator=g, device="cuda")
    inv = 1e4 ** (-torch.arange(sum(sections), device="cuda", dtype=F32) / sum(sections))
    w = [(1 + 0.1 * randn(g, D + 1)).to(t) for t in (wq, wk)]
    for shift in (0, 1):  # weights aligned and not
        a, b = (x[shift:shift + D] for x in w)
        qo, ko = rope_axes_qk(q, k, pos, inv, sections, q_norm_weight=a, k_norm_weight=b)
        check_rope(q, qo, pos, inv, sections, False, a, 1e-6, 1.0)
        check_rope(k, ko, pos, inv, sections, False, b, 1e-6, 1.0)


def test_sections_given_as_tensors_that_change():
    """A call takes the sections' values of its own time."""
    q, k = randn(gen(1), 1, 9, 2, 64), randn(gen(2), 1, 9, 1, 64)
    pos = torch.randint(0, 1000, (2, 1, 9), generator=gen(3), device="cuda")
    inv = 1e4 ** (-torch.arange(32, device="cuda", dtype=F32) / 32)
    sections = (torch.tensor(20), torch.tensor(12))
    for a in (20, 5, 20):
        sections[0].fill_(a)
        sections[1].fill_(32 - a)
        got, _ = rope_axes_qk(q, k, pos, inv, sections)
        check_rope(q, got, pos, inv, (a, 32 - a), False, None, 0, 1.0)


def test_a_captured_step_follows_the_cache(cuda_device):
    """One captured step for two prompts, and with eager steps between its own."""
    from aoh_b200.hf import ModelDecodeGraph, patch_aoh_model
    from tests.test_hf_gpu import _tiny
    from tests.test_operators_hf_gpu import LABELS, _prompt, _run

    model = _tiny("llama")
    make_cache, _, _ = patch_aoh_model(model, LABELS, 16, 48)
    first, second = _prompt(120, seed=1), _prompt(260, seed=2)
    eager, cache = make_cache(max_context=512), make_cache(max_context=512)
    cache.track_weights()
    eager.track_weights()
    _run(model, cache, first, [0, 110])
    g = ModelDecodeGraph(model, cache, max_steps=16)
    for t in range(110, 114):
        g.step(first[:, t])
    cache.reset()
    for c in (cache, eager):
        _run(model, c, second, [0, 200])
    for t in range(200, 212):
        want = _run(model, eager, second, [t, t + 1])[0]
        got = (_run(model, cache, second, [t, t + 1])[0] if t % 4 == 3 else g.step(second[:, t])).float()
        assert (got - want).abs().max() <= 0.05 * want.abs().max()
    assert cache.get_seq_length() == 212 and cache.paged.device_status() == 0
    for layer in range(2):
        for head in range(2):
            rows = range(212) if LABELS[layer][head] else range(164, 212)
            for x, y in zip(*(c.paged.read_rows(layer, 0, head, rows) for c in (cache, eager))):
                assert torch.equal(x, y)
    # sums in key ranges planned for max_context: fp32 in another order, of values up to 4 * 212
    assert ((cache.key_weights.rows - eager.key_weights.rows).abs() <= 4 * 212 * 2.0 ** -18).all()


def test_a_captured_step_refuses_weights_that_it_does_not_add_to(cuda_device):
    """Tracked from a later time on, the sums would lack the captured steps."""
    from aoh_b200.hf import ModelDecodeGraph, patch_aoh_model
    from tests.test_hf_gpu import _tiny
    from tests.test_operators_hf_gpu import LABELS, _prompt, _run

    model = _tiny("llama")
    make_cache, _, _ = patch_aoh_model(model, LABELS, 16, 48)
    cache, ids = make_cache(max_context=128), _prompt(70)
    _run(model, cache, ids, [0, 64])
    g = ModelDecodeGraph(model, cache, max_steps=8)
    g.step(ids[:, 64])
    cache.track_weights()
    with pytest.raises(RuntimeError):
        g.step(ids[:, 65])
    assert cache.get_seq_length() == 65
    g = ModelDecodeGraph(model, cache, max_steps=8)
    g.step(ids[:, 65])
    # the step's query gave its keys 1 for each of a group's 4 heads: 66 weights' roundings
    assert ((cache.key_weights.rows.double().sum(1) - 4).abs() <= 4 * 70 * 2.0 ** -24 + 4e-5).all()


FIRST_CALLS = """
import torch
from aoh_b200 import AoHKVCache, key_weights, penalize_logits, rope_axes_qk, select_keys, evict
def make(n, dt=torch.bfloat16):
    return AoHKVCache([[1, 0]], 8, sink_size=16, recent_size=32, max_context=n, dtype=dt, reserve_all=True)
def fill(c, n):
    k = torch.randn((1, n, 2, 128), generator=torch.Generator("cuda").manual_seed(1), device="cuda").to(c.dtype)
    c.append_layer(0, k, k)
    c.kv_seq_len = n
    return c
big, into = fill(make(20_000), 20_000), make(512)
f32 = fill(make(300, torch.float32), 300)
q = {c: torch.randn((1, c, 8, 128), device="cuda").bfloat16() for c in (1, 5, 40, 300)}
k = torch.randn((1, 300, 2, 128), device="cuda").bfloat16()
pos, inv = torch.arange(300, device="cuda").expand(1, 1, 300), torch.ones(64, device="cuda")
x = torch.randn((3, 128_256), device="cuda")
def calls():
    out = [*rope_axes_qk(q[300], k, pos, inv, (64,))]
    out.append(key_weights(big, 0, q[1], past_len=3999))
    out += [key_weights(big, 0, q[c], past_len=20_000 - c) for c in (1, 5, 40, 300)]
    out.append(key_weights(f32, 0, q[5].float(), past_len=295))
    kept, w = select_keys(out[3].view(1, -1), 400, sink=16, recent=32)
    evict(big, kept, into)
    return out + [kept, w, into.pool, *penalize_logits(x, greedy=True), *penalize_logits(x[:, 1:], greedy=True)]
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    captured = calls()
g.replay()
torch.cuda.synchronize()
captured = [t.clone() for t in captured]
assert all(torch.equal(a, b) for a, b in zip(captured, calls()))
print("alike")
"""


def test_the_first_calls_of_a_process_may_be_captured(cuda_device):
    """No operator needs an eager call before: kernels are prepared within a capture as well."""
    import subprocess
    import sys
    from pathlib import Path

    r = subprocess.run([sys.executable, "-c", FIRST_CALLS], capture_output=True, text=True, timeout=300,
                       cwd=Path(__file__).resolve().parents[1])
    assert r.returncode == 0 and "alike" in r.stdout, r.stderr[-2000:]
