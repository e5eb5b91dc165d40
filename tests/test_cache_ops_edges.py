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


@pytest.mark.parametrize("name", ["q_norm", "k_norm"])
def test_hooks_of_head_norms_run(name):
    """A hook on a head's norm sees its rows and may change them, fused or not."""
    cfg = _cfg(qk_norm=True)
    outs, calls = [], []
    for fused in (False, True):
        eng = _engine(cfg, fused_head_norms=fused)
        for layer in eng.model.layers:
            getattr(layer.self_attn, name).register_forward_hook(
                lambda m, x, y: calls.append(fused) or -2 * y)
        outs.append(_generate(eng))
    assert outs[0] == outs[1] and calls.count(True) == calls.count(False) > 0


def test_other_head_norms_run():
    """A module in a norm's place, and norms of two epsilons, are called."""
    from parallax_amd.models.llama import RMSNorm

    class Shifted(RMSNorm):
        def forward(self, x):
            return super().forward(x) + 1

    def shift(attn):
        old = attn.k_norm
        attn.k_norm = Shifted(attn.head_dim, old.eps)
        attn.k_norm.weight = old.weight

    def loosen(attn):
        attn.k_norm.eps = 3.0

    cfg = _cfg(qk_norm=True)
    plain = _generate(_engine(cfg))
    for change in (shift, loosen):
        outs = []
        for fused in (False, True):
            eng = _engine(cfg, fused_head_norms=fused)
            for layer in eng.model.layers:
                change(layer.self_attn)
            outs.append(_generate(eng))
        assert outs[0] == outs[1] != plain


def test_scales_of_a_bf16_cache():
    """Scales are those of fp8 caches; a bf16 one holds its values as they are."""
    s = prefix_inputs(4, 2, 64, 16, ROWS, [20, 32])
    want = prefix_call(ATTEND, s, "cpu")
    assert torch.equal(prefix_call(ATTEND, {**s, "scales": (0.5, 0.25)}, "cpu"), want)
    s = store_inputs(9, 4, 2, 64, 64, 16)
    for got, want in zip(call(STORE, s, change=dict(k_scale=0.5, v_scale=0.25)),
                         call(STORE, s)):
        assert torch.equal(got, want)


def test_no_pages():
    """A cache of no pages: zeros, as on the GPU."""
    s = prefix_inputs(4, 2, 64, 16, ROWS, [20, 32])
    s["kc"], s["vc"] = s["kc"][:0], s["vc"][:0]
    assert (prefix_call(ATTEND, s, "cpu") == 0).all()


@EXT
def test_too_many_heads_refused():
    s = store_inputs(1, 1, 1, 2, 2, 16)
    q = torch.zeros(1, (1 << 20) - 1, 2, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="2\\^20 heads"):
        call(ops._require_ext("test").qk_norm_rope_and_cache, s, change=dict(q=q))


def test_wide_integers():
    """Lengths, groups, pages and positions of 64 bits are what they say, not what is
    left of them in 32."""
    s = prefix_inputs(4, 2, 64, 16, [(0, 48), (0, 48), (1, 48), (2, 48)], [20, 30])
    s["tables"] = s["tables"][:, :3].contiguous()
    s["kc"], s["vc"] = (x.float().nan_to_num().bfloat16() for x in (s["kc"], s["vc"]))
    want = prefix_call(ATTEND, s, "cpu")
    wide = {**s, **{n: s[n].long() for n in ("lens", "group", "tables", "prefix")}}
    wide["lens"][1] += 1 << 32
    wide["group"][3] += (1 << 32) - 2       # not group 0
    assert torch.equal(prefix_call(ATTEND, wide, "cpu"), want)
    wide["tables"][0, 1] = 1 << 32          # the last page, not the first
    s["tables"][0, 1] = s["kc"].shape[0] - 1
    assert torch.equal(prefix_call(ATTEND, wide, "cpu"), prefix_call(ATTEND, s, "cpu"))
    s = store_inputs(6, 4, 2, 64, 64, 16)
    s["pos"] = s["pos"].long()
    s["pos"][2] += 1 << 32
    q, kc, vc = call(STORE, s)
    assert q[2].isnan().all() and not q[:2].isnan().any() and not q[3:].isnan().any()


@EXT
@pytest.mark.parametrize("change", [
    dict(scale=1e39), dict(k_scale=1e39), dict(v_scale=1e39), dict(k_scale=1e-46),
    dict(v_scale=1e-46), dict(k_scale=float("nan")), dict(softcap=float("nan")),
])
def test_beyond_fp32_refused(change):
    """What fp32 cannot hold."""
    s = prefix_inputs(4, 2, 64, 16, [(0, 40), (0, 21), (-1, 17)], [20])
    with pytest.raises(RuntimeError) as e:
        ops._require_ext("test").shared_prefix_attention_decode(*arguments(s, change))
    assert "must be on GPU" not in str(e.value)


@EXT
@pytest.mark.parametrize("change", [
    dict(k_scale=1e39), dict(v_scale=1e39), dict(k_scale=1e-46), dict(v_scale=1e-46),
    dict(k_scale=1e-40), dict(eps=float("inf")), dict(eps=1e39), dict(eps=float("nan")),
])
def test_store_beyond_fp32_refused(change):
    s = store_inputs(5, 4, 2, 64, 64, 16)
    with pytest.raises(RuntimeError) as e:
        call(ops._require_ext("test").qk_norm_rope_and_cache, s, change=change)
    assert "must be on GPU" not in str(e.value)


@EXT
@pytest.mark.parametrize("native", [False, True])
@pytest.mark.parametrize("name", ["k_cache", "v_cache", "sinks"])
def test_no_gradient_of_what_is_read(name, native):
    s = prefix_inputs(4, 2, 64, 16, [(0, 40), (0, 21), (-1, 17)], [20])
    fn = (ops._require_ext("test") if native else ops).shared_prefix_attention_decode
    leaf = dict(k_cache=s["kc"], v_cache=s["vc"], sinks=torch.zeros(4))[name]
    change = {name: leaf.clone().requires_grad_()}
    with pytest.raises(RuntimeError, match="no gradient"):
        fn(*arguments(s, change))
    with torch.no_grad():
        if not native:
            fn(*arguments(s, change))


@EXT
@pytest.mark.parametrize("native", [False, True])
@pytest.mark.parametrize("name", ["k_cache", "v_cache", "cos_sin"])
def test_store_no_gradient_of_caches_and_table(name, native):
    s = store_inputs(5, 4, 2, 64, 64, 16)
    _, _, _, a = store_views(s, "cpu")
    leaf = dict(k_cache=a["kc"], v_cache=a["vc"], cos_sin=a["table"])[name]
    fn = ops._require_ext("test").qk_norm_rope_and_cache if native else STORE
    with pytest.raises(RuntimeError, match="no gradient"):
        call(fn, s, change={name: leaf.clone().requires_grad_()})


def test_sinks_that_take_all():
    s = prefix_inputs(4, 2, 64, 16, ROWS, [20, 32])
    inf = float("inf")
    got = prefix_call(ATTEND, s, "cpu", sinks=torch.tensor([inf, 0.0, -inf, 3e38]))
    want, size = prefix_oracle(s, sinks=torch.tensor([1e30, 0.0, -inf, 1e30]))
    assert_attended(got, (want, size), weights=0.0)
    assert (got[:, [0, 3]] == 0).all()
