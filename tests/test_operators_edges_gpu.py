"""Edges of the operators around a decode step."""
import pytest
import torch

from aoh_b200 import key_weights, penalize_logits, select_keys
from tests.test_operators_gpu import check_select, check_weights, filled, gen, randn

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


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


# -- key weights ------------------------------------------------------------------
@pytest.mark.parametrize("C,grp,T", [(32, 7, 90_000), (40, 3, 70_001), (5, 8, 120_003)])
def test_key_weights_of_resident_rows_over_many_tiles(C, grp, T):
    """One and two tiles of query rows, ranges of many key tiles: every stage of the ring is used several times."""
    cache, k, _ = filled([[1, 1, 0]], 3 * grp, 1, T, BF16, C)
    q = randn(gen(C), 1, C, 3 * grp, 128, dtype=BF16)
    outs = [key_weights(cache, 0, q, past_len=T - C) for _ in range(4)]
    check_weights(outs[0], q, k[0], [0, 1], T - C)
    assert all(torch.equal(x, outs[0]) for x in outs) and cache.device_status() == 0
