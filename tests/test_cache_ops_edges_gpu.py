"""Edges of the operators around a shared paged cache, on the GPU: what their range holds
besides what engines call them with."""

import pytest
import torch

pytestmark = pytest.mark.gpu

from cache_ops_util import (
    NAN, assert_attended, assert_stored, prefix_call, prefix_inputs, prefix_oracle,
    store_inputs, store_oracle)
from parallax_amd import ops
from test_head_norm_store import call

STORE = ops.qk_norm_rope_and_cache
ATTEND = ops.shared_prefix_attention_decode
ODD = [(0, 300), (1, 233), (0, 201), (-1, 170), (0, 0), (1, 5), (7, 9), (0, 200),
       (1, 640), (-3, 1), (0, 1000), (1, 130), (0, 199)]
INF = float("inf")


@pytest.mark.parametrize("T", [5, 600])
@pytest.mark.parametrize("D,rot,head_gap", [
    (64, 64, 0), (64, 32, 1), (66, 34, 0), (112, 24, 0), (24, 0, 0)])
def test_store_without_pages(T, D, rot, head_gap):
    """A cache of no pages takes no row, and the queries come back all the same."""
    s = store_inputs(T, 4, 2, D, rot, 16, seed=D, head_gap=head_gap, blocks=0,
                     slots=torch.arange(T))
    torch.full((T, 4, D), NAN, dtype=torch.bfloat16, device="cuda")  # what `out` finds
    assert_stored(call(STORE, s, "cuda"), *store_oracle(s, True))


CAPS = [1e3, 1e5, 1e8, 1e30, 3e38, 1e300]


@pytest.mark.parametrize("softcap", CAPS)
@pytest.mark.parametrize("D,fp8", [(64, False), (64, True), (128, False), (128, True)])
def test_large_caps(softcap, D, fp8):
    """Caps far above the scores leave them as they are."""
    s = prefix_inputs(8, 2, D, 32, ODD, [200, 129], fp8, seed=D)
    for scale in (None, -0.3):
        got = prefix_call(ATTEND, s, "cuda", softcap=softcap, scale=scale)
        assert_attended(got, prefix_oracle(s, softcap=softcap, scale=scale))


@pytest.mark.parametrize("softcap", [1e-300, 1e-20, 1e-3, 0.5, 3.0, 8.0, 20.0])
def test_caps_about_the_scores(softcap):
    """Scores on both sides of where a cap begins to bend them, and caps that leave
    nothing of them."""
    s = prefix_inputs(8, 2, 64, 32, ODD, [200, 129], seed=3)
    got = prefix_call(ATTEND, s, "cuda", softcap=softcap)
    assert_attended(got, prefix_oracle(s, softcap=softcap))
