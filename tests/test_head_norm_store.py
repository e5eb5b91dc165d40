"""Head norms, rotation and append in one pass: the CPU form against 64 bits, and what
the operator refuses."""

import pytest
import torch

from cache_ops_util import assert_stored, store_inputs, store_oracle, store_views
from parallax_amd import ops

EXT = pytest.mark.skipif(not ops.has_extension(), reason="extension not built")


def call(fn, s, device="cpu", neox=True, change=None):
    q, k, v, a = store_views(s, device)
    args = dict(q=q, k=k, v=v, q_weight=a["qw"], k_weight=a["kw"], eps=s["eps"],
                k_cache=a["kc"], v_cache=a["vc"], positions=a["pos"],
                cos_sin=a["table"], slot_mapping=a["slots"], is_neox=neox,
                k_scale=s["scales"][0], v_scale=s["scales"][1])
    args.update(change or {})
    return (fn(*args.values()), args["k_cache"], args["v_cache"])


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("neox", [False, True])
@pytest.mark.parametrize("T,Hq,Hk,D,rot", [
    (1, 4, 2, 64, 64), (9, 3, 1, 10, 6), (5, 2, 2, 128, 32), (4, 4, 4, 7, 0),
])
def test_cpu_form(T, Hq, Hk, D, rot, neox, fp8):
    s = store_inputs(T, Hq, Hk, D, rot, 4, fp8, seed=T, head_gap=3, row_gap=1)
    if T > 2:
        s["slots"][1], s["slots"][2] = -1, 10 ** 6
    assert_stored(call(ops.qk_norm_rope_and_cache, s, neox=neox), *store_oracle(s, neox))


def test_cpu_form_no_rows():
    s = store_inputs(0, 4, 2, 64, 64, 16)
    out, kc, vc = call(ops.qk_norm_rope_and_cache, s)
    assert out.shape == (0, 4, 64) and torch.equal(kc, s["kc"])


def bad_calls():
    x = torch.randn
    b = torch.bfloat16
    return {
        "fp32 q": dict(q=x(5, 4, 64)),
        "fp16 v": dict(v=x(5, 2, 64).half()),
        "rows of k": dict(k=x(4, 2, 64).to(b)),
        "heads of v": dict(v=x(5, 4, 64).to(b)),
        "strided values": dict(q=x(5, 4, 128).to(b)[..., ::2]),
        "a flat q": dict(q=x(5, 256).to(b)),
        "short weight": dict(q_weight=x(32).to(b)),
        "fp32 weight": dict(k_weight=x(64)),
        "strided weight": dict(k_weight=x(128).to(b)[::2]),
        "fp16 cache": dict(k_cache=x(5, 2, 16, 64).half(), v_cache=x(5, 2, 64, 16).half()),
        "caches of two types": dict(v_cache=x(5, 2, 64, 16).to(torch.float8_e4m3fn)),
        "v not transposed": dict(v_cache=x(5, 2, 16, 64).to(b)),
        "heads of the cache": dict(k_cache=x(5, 3, 16, 64).to(b)),
        "strided cache": dict(k_cache=x(5, 2, 16, 128).to(b)[..., :64]),
        "positions of another length": dict(positions=torch.zeros(4, dtype=torch.int32)),
        "slots of another length": dict(slot_mapping=torch.zeros(6, dtype=torch.int64)),
        "odd rotation": dict(cos_sin=x(200, 63)),
        "rotation past the head": dict(cos_sin=x(200, 66)),
        "bf16 table": dict(cos_sin=x(200, 64).to(b)),
        "no positions": dict(cos_sin=x(0, 64)),
        "negative eps": dict(eps=-1e-5),
        "scale of 0": dict(k_scale=0.0),
        "infinite scale": dict(v_scale=float("inf")),
    }


@EXT
@pytest.mark.parametrize("name", bad_calls())
def test_refused(name):
    """Before the device is looked at: CPU tensors show it."""
    torch.manual_seed(0)
    s = store_inputs(5, 4, 2, 64, 64, 16)
    fn = ops._require_ext("test").qk_norm_rope_and_cache
    with pytest.raises(RuntimeError) as e:
        call(fn, s, change=bad_calls()[name])
    assert "must be on GPU" not in str(e.value)


@EXT
def test_refused_on_cpu_last():
    s = store_inputs(5, 4, 2, 64, 64, 16)
    with pytest.raises(RuntimeError, match="must be on GPU"):
        call(ops._require_ext("test").qk_norm_rope_and_cache, s)


@EXT
@pytest.mark.parametrize("native", [False, True])
@pytest.mark.parametrize("name", ["q", "k", "v", "q_weight", "k_weight"])
def test_no_gradient(name, native):
    s = store_inputs(5, 4, 2, 64, 64, 16)
    q, k, v, a = store_views(s, "cpu")
    leaf = dict(q=q, k=k, v=v, q_weight=a["qw"], k_weight=a["kw"])[name]
    fn = ops._require_ext("test").qk_norm_rope_and_cache if native \
        else ops.qk_norm_rope_and_cache
    with pytest.raises(RuntimeError, match="no gradient"):
        call(fn, s, change={name: leaf.clone().requires_grad_()})
