"""Host rules of sessions that share pages and verify drafts (CPU): the uniforms of a verified step, arguments that are
refused."""
import numpy as np
import pytest
import torch

from mesh_b200 import ops
from mesh_b200.engine import serving
from mesh_b200.oracle.tensor_ops import deterministic_sample_threshold


def _draw(weights, u):
    c = np.cumsum(weights)
    return int(np.nonzero(c > u * c[-1])[0][0])


@pytest.mark.parametrize("kv_len", [0, 11, 4096])
@pytest.mark.parametrize("drafted_by", ["prefill or decode", "a verified step"])
def test_verified_tokens_follow_the_target_when_drafts_have_the_sessions_seed(kv_len, drafted_by):
    """One draft over three tokens, drawn with the number this framework's own sampler uses at that position for the same
    seed; accepting and drawing as the verification does. Over 60000 seeds each frequency's standard deviation is
    sqrt(1/3 2/3 / 60000) = 0.0019; five of them bound every token."""
    n = 60000
    p, q = np.full(3, 1 / 3), np.array([0.8, 0.1, 0.1])
    count = np.zeros(3)
    for seed in range(n):
        if drafted_by == "prefill or decode":
            u = deterministic_sample_threshold(seed ^ (kv_len + 1))
        else:  # a step without drafts in the draft model's engine
            u = serving._verify_thresholds(seed, kv_len, 0)[1]
        x = _draw(q, u)
        (accept,), draw = serving._verify_thresholds(seed, kv_len, 1)
        count[x if accept * q[x] < p[x] else _draw(np.maximum(p - q, 0), draw)] += 1
    assert np.abs(count / n - p).max() <= 5 * np.sqrt(1 / 3 * 2 / 3 / n), count / n


def test_thresholds_of_a_session_are_all_different():
    """Every uniform that one seed gives: those of ordinary steps, of accepting, and of drawing behind drafts."""
    seen = set()
    for kv_len in range(300):
        accept, draw = serving._verify_thresholds(77, kv_len, 1)
        seen |= {serving._verify_thresholds(77, kv_len, 0)[1], accept[0], draw}
    assert len(seen) >= 898  # 24-bit numbers: 900 of them coincide 0.02 times on average
    # a draft's own number does not depend on how many stand before it
    assert serving._verify_thresholds(77, 40, 5)[0][3] == serving._verify_thresholds(77, 43, 1)[0][0]
    # without drafts the token is decode_step's
    assert serving._verify_thresholds(77, 40, 0) == ([], deterministic_sample_threshold(77 ^ 41))


@pytest.mark.parametrize("scale", [0.0, -0.1, float("nan"), float("inf"), 1e-40])
def test_attention_over_shared_prefixes_refuses_a_scale_that_is_not_positive(scale):
    plan = ops.PrefixGroups(2, 4, 2, 64, device="cpu")
    q, cache = torch.zeros(2, 256, dtype=torch.bfloat16), torch.zeros(3, 2, 16, 64, dtype=torch.bfloat16)
    table, lens = torch.ones(2, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="scale"):
        ops.attn_shared_prefix(q, cache, cache, table, lens, plan, torch.empty_like(q), scale)
