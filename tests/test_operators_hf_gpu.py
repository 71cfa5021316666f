"""Key weights, eviction and logits controls through the patched HF models."""
import numpy as np
import pytest
import torch

from tests.test_hf_gpu import _tiny

pytestmark = pytest.mark.gpu

LABELS = np.array([[1, 0], [0, 1]], dtype=np.float64)


def _prompt(n, B=1, seed=5):
    return torch.randint(0, 128, (B, n), generator=torch.Generator().manual_seed(seed)).cuda()


def _run(model, cache, ids, cuts):
    out = []
    with torch.no_grad():
        for a, b in zip(cuts, cuts[1:]):
            out.append(model(input_ids=ids[:, a:b], past_key_values=cache, use_cache=True).logits.float())
    return out


def test_keeping_every_key_changes_nothing(cuda_device):
    """Evicting down to all keys is a move to another cache: the same logits, bit for bit."""
    from aoh_b200.hf import patch_aoh_model

    model = _tiny("llama")
    make_cache, _, _ = patch_aoh_model(model, LABELS, 16, 48)
    ids = _prompt(300)
    plain, tracked = make_cache(max_context=512), make_cache(max_context=512)
    tracked.track_weights()
    a = _run(model, plain, ids, [0, 160, 290])
    b = _run(model, tracked, ids, [0, 160, 290])
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    # each query of each of a group's 4 heads gives its keys 1
    got = tracked.key_weights.rows[:, :290].double().sum(1)
    assert ((got - 4 * 290).abs() <= 4 * 290 * 1e-4).all()
    moved = tracked.evict(290, max_context=400)
    assert moved.get_seq_length() == 290 and moved.paged.kv_seq_len == 290 and moved.paged.evicted == 0
    assert torch.equal(moved.key_weights.rows[:, :290], tracked.key_weights.rows[:, :290])
    steps = list(range(290, 301))
    for x, y in zip(_run(model, plain, ids, steps), _run(model, moved, ids, steps)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("kind", ["llama", "qwen3"])
def test_decoding_goes_on_after_an_eviction(cuda_device, kind):
    """Positions count the tokens seen; a captured decode step agrees with eager ones."""
    from aoh_b200.hf import ModelDecodeGraph, patch_aoh_model

    model = _tiny(kind)
    make_cache, _, _ = patch_aoh_model(model, LABELS, 16, 48)
    ids = _prompt(300)
    small = []
    for _ in range(2):
        cache = make_cache(max_context=512)
        cache.track_weights()
        _run(model, cache, ids, [0, 160, 290])
        small.append(cache.evict(100, max_context=128))
        assert small[-1].get_seq_length() == 290 and small[-1].paged.kv_seq_len == 100
    before = small[1].key_weights.rows.clone()
    assert torch.equal(before, small[0].key_weights.rows)
    g = ModelDecodeGraph(model, small[1], max_steps=16)
    assert torch.equal(small[1].key_weights.rows, before)  # the dry run left nothing
    for t in range(290, 300):
        want = _run(model, small[0], ids, [t, t + 1])[0]
        got = g.step(ids[:, t]).float()
        assert (got - want).abs().max() <= 0.05 * want.abs().max()
    assert small[0].get_seq_length() == small[1].get_seq_length() == 300
    for layer in range(2):  # the same rows were appended at the same places
        h = int(np.flatnonzero(LABELS[layer])[0])
        for x, y in zip(*(c.paged.read_rows(layer, 0, h, range(100, 110)) for c in small)):
            assert torch.equal(x, y)
    got = small[1].key_weights.rows - before
    want = small[0].key_weights.rows - before
    # the same sums, but in key ranges planned for max_context: fp32 in another order, of values up to 4 * 300
    assert ((got - want).abs() <= 4 * 300 * 2.0 ** -18).all()
    assert ((got.double().sum(1) - 40).abs() <= 40 * 1e-3).all()
    for c in small:
        assert c.paged.device_status() == 0


def test_controls_in_the_captured_step(cuda_device):
    """A decode loop that stays on the GPU: penalties by the history, a mask
    rewritten between steps, the greedy token fed back."""
    from aoh_b200 import TokenHistory, penalize_logits
    from aoh_b200.hf import ModelDecodeGraph, patch_aoh_model

    model = _tiny("llama")
    make_cache, _, _ = patch_aoh_model(model, LABELS, 16, 48)
    B, V = 2, 128
    ids = _prompt(200, B)
    caches = [make_cache(batch=B, max_context=256) for _ in range(2)]
    logits = [_run(model, c, ids, [0, 200])[0][:, -1] for c in caches]
    h = [TokenHistory(B, V) for _ in range(2)]
    for x in h:
        x.add_prompt(ids)
    allowed = torch.full((B, V // 32), -1, dtype=torch.int32, device="cuda")
    pen = dict(repetition=1.3, frequency=torch.tensor([0.5, 0.0], device="cuda"), allowed=allowed)
    g = ModelDecodeGraph(model, caches[1], max_steps=12, history=h[1], controls=pen)
    assert torch.equal(h[0].counts, h[1].counts)  # the set-up counted nothing
    _, tok = penalize_logits(logits[0], h[0], greedy=True, **pen)
    nxt = tok.clone()
    seen = [tok.tolist()]
    for step in range(8):
        allowed.fill_(-1)
        allowed[0, step % 4] = 0
        h[0].append(tok)
        raw = _run(model, caches[0], torch.cat([ids, tok[:, None]], 1), [200, 201])[0][:, -1]
        want, tok = penalize_logits(raw.bfloat16(), h[0], greedy=True, **pen)
        got = g.step(nxt)
        assert got.shape == (B, 1, V) and torch.equal(h[0].counts, h[1].counts) and torch.equal(h[0].seen, h[1].seen)
        assert torch.equal(torch.isinf(got[:, 0]), torch.isinf(want)) and torch.isinf(got[0, 0, 32 * (step % 4)])
        ok = torch.isfinite(want)
        assert (got[:, 0][ok] - want[ok]).abs().max() <= 0.05 * want[ok].abs().max()
        assert torch.equal(got[:, 0].argmax(1), g.next_ids)
        nxt = tok  # the eager loop's choice, so that both stay on one path
        seen.append(tok.tolist())
    assert caches[0].get_seq_length() == caches[1].get_seq_length() == 208


def test_evict_needs_weights(cuda_device):
    from aoh_b200.hf import patch_aoh_model

    make_cache, _, _ = patch_aoh_model(_tiny("llama"), LABELS, 16, 48)
    with pytest.raises(RuntimeError):
        make_cache(max_context=64).evict(32)
