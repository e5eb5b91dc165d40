"""Edges of the operators around a shared paged cache, and of the engine options that use
them, on the CPU."""

import pytest
import torch

from cache_ops_util import (
    assert_attended, prefix_call, prefix_inputs, prefix_oracle, store_inputs, store_views)
from parallax_amd import ops
from test_head_norm_store import call
from test_shared_prefix import ROWS, arguments
from test_shared_prefix_engine import PROMPTS, SPS, _cfg, _engine, _generate

EXT = pytest.mark.skipif(not ops.has_extension(), reason="extension not built")
STORE = ops.qk_norm_rope_and_cache
ATTEND = ops.shared_prefix_attention_decode


@pytest.mark.parametrize("softcap", [1e-300, 1e-20, 3.0, 1e5, 1e30, 3e38, 1e300])
def test_caps(softcap):
    s = prefix_inputs(4, 2, 64, 16, ROWS, [20, 32])
    got = prefix_call(ATTEND, s, "cpu", softcap=softcap)
    assert_attended(got, prefix_oracle(s, softcap=softcap), weights=0.0)
