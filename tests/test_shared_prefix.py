"""Decode over shared prefixes: the CPU form against 64 bits, and what the operator
refuses."""

import pytest
import torch

from cache_ops_util import assert_attended, prefix_call, prefix_inputs, prefix_oracle
from parallax_amd import ops

EXT = pytest.mark.skipif(not ops.has_extension(), reason="extension not built")
ROWS = [(0, 40), (1, 33), (0, 21), (-1, 17), (0, 0), (1, 5), (7, 9), (0, 20), (1, 64)]


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("kw", [
    {}, dict(sliding_window=25), dict(sliding_window=1), dict(softcap=3.0),
    dict(sinks=torch.tensor([0.5, -1.0, 4.0, 0.0])), dict(scale=-0.2), dict(scale=0.0),
])
def test_cpu_form(kw, fp8):
    s = prefix_inputs(4, 2, 64, 16, ROWS, [20, 32], fp8)
    got = prefix_call(ops.shared_prefix_attention_decode, s, "cpu", **kw)
    assert_attended(got, prefix_oracle(s, **kw), weights=0.0)


def test_cpu_form_is_decode():
    """Where rows hold their own copies of the prefix, plain decode attention."""
    s = prefix_inputs(4, 2, 64, 16, [(-1, 40), (-1, 21), (-1, 64)], [])
    got = prefix_call(ops.shared_prefix_attention_decode, s, "cpu")
    want = ops.paged_attention_decode(
        s["q"].view(3, 4, 64), s["kc"].float().nan_to_num().bfloat16(),
        s["vc"].float().nan_to_num().bfloat16(), s["tables"], s["lens"], 0.125)
    assert (got.float() - want.float()).abs().max() < 0.02


def test_lengths_past_the_table():
    """A row that claims more tokens than its table has pages for ends with the table;
    a prefix past that has no rows."""
    s = prefix_inputs(4, 2, 64, 16, [(0, 48), (0, 48), (1, 48)], [20, 60])
    s["tables"] = s["tables"][:, :3].contiguous()
    want = prefix_oracle(s)
    s["lens"] = torch.tensor([48, 49, 2 ** 31 - 1], dtype=torch.int32)
    assert_attended(prefix_call(ops.shared_prefix_attention_decode, s, "cpu"), want,
                    weights=0.0)


def bad_calls():
    x, i = torch.randn, torch.int32
    b = torch.bfloat16
    return {
        "fp32 q": dict(q=x(3, 4, 64)),
        "flat q": dict(q=x(3, 256).to(b)),
        "heads apart": dict(q=x(3, 4, 72).to(b)[..., :64]),
        "width": dict(q=x(3, 4, 32).to(b)),
        "heads that do not divide": dict(q=x(3, 5, 64).to(b)),
        "too many heads a head": dict(q=x(3, 34, 64).to(b)),
        "fp16 caches": dict(k_cache=x(5, 2, 16, 64).half(), v_cache=x(5, 2, 64, 16).half()),
        "v not transposed": dict(v_cache=x(5, 2, 16, 64).to(b)),
        "two types": dict(v_cache=x(5, 2, 64, 16).to(torch.float8_e4m3fn)),
        "page of 8": dict(k_cache=x(5, 2, 8, 64).to(b), v_cache=x(5, 2, 64, 8).to(b)),
        "tables of other rows": dict(block_tables=torch.zeros(2, 3, dtype=i)),
        "flat tables": dict(block_tables=torch.zeros(3, dtype=i)),
        "strided tables": dict(block_tables=torch.zeros(3, 6, dtype=i)[:, ::2]),
        "lengths of other rows": dict(seq_lens=torch.zeros(4, dtype=i)),
        "groups of other rows": dict(prefix_group=torch.zeros(2, dtype=i)),
        "prefixes in two dimensions": dict(prefix_lens=torch.zeros(1, 1, dtype=i)),
        "infinite scale": dict(scale=float("inf")),
        "negative softcap": dict(softcap=-1.0),
        "too few sinks": dict(sinks=torch.zeros(3)),
        "scale of 0": dict(k_scale=0.0),
        "negative v_scale": dict(v_scale=-1.0),
    }


def arguments(s, change=None):
    B, Hq, D = s["shape"]
    args = dict(q=s["q"].view(B, Hq, D), k_cache=s["kc"], v_cache=s["vc"],
                block_tables=s["tables"], seq_lens=s["lens"], prefix_group=s["group"],
                prefix_lens=s["prefix"], scale=0.125, sliding_window=-1, softcap=0.0,
                sinks=None, k_scale=1.0, v_scale=1.0)
    args.update(change or {})
    return args.values()


@EXT
@pytest.mark.parametrize("name", bad_calls())
def test_refused(name):
    s = prefix_inputs(4, 2, 64, 16, [(0, 40), (0, 21), (-1, 17)], [20])
    with pytest.raises(RuntimeError) as e:
        ops._require_ext("test").shared_prefix_attention_decode(
            *arguments(s, bad_calls()[name]))
    assert "must be on GPU" not in str(e.value)


@EXT
def test_refused_on_cpu_last():
    s = prefix_inputs(4, 2, 64, 16, [(0, 40), (0, 21), (-1, 17)], [20])
    with pytest.raises(RuntimeError, match="must be on GPU"):
        ops._require_ext("test").shared_prefix_attention_decode(*arguments(s))


@EXT
def test_too_many_rows():
    n = 4097
    i = torch.int32
    with pytest.raises(RuntimeError, match="4096"):
        ops._require_ext("test").shared_prefix_attention_decode(
            *arguments(prefix_inputs(4, 2, 64, 16, [(0, 40)], [20]), dict(
                q=torch.zeros(n, 4, 64).bfloat16(), seq_lens=torch.zeros(n, dtype=i),
                block_tables=torch.zeros(n, 1, dtype=i),
                prefix_group=torch.zeros(n, dtype=i))))
    with pytest.raises(RuntimeError, match="256 groups"):
        ops._require_ext("test").shared_prefix_attention_decode(
            *arguments(prefix_inputs(4, 2, 64, 16, [(0, 40)], [20]), dict(
                prefix_lens=torch.zeros(257, dtype=i))))


@EXT
@pytest.mark.parametrize("native", [False, True])
def test_no_gradient(native):
    s = prefix_inputs(4, 2, 64, 16, [(0, 40), (0, 21), (-1, 17)], [20])
    fn = (ops._require_ext("test") if native else ops).shared_prefix_attention_decode
    with pytest.raises(RuntimeError, match="no gradient"):
        fn(*arguments(s, dict(q=s["q"].view(3, 4, 64).clone().requires_grad_())))
