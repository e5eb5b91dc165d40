"""Engines that read shared prefixes once and norm heads on the way into the cache, on the
GPU, against the fp32 engine on the CPU fed the same tokens: prompts of a common head,
steps replayed and not, rows that leave, a second batch over other groups."""

import gc

import pytest
import torch

from parallax_amd import ops
from parallax_amd.models.config import ModelConfig
from parallax_amd.parallel.comm import CommContext
from parallax_amd.server.engine import Engine, EngineArgs
from parallax_amd.server.graph_runner import SHARED
from parallax_amd.server.sampling_params import SamplingParams

pytestmark = pytest.mark.gpu

SIZES = {
    "vocab_size": 512, "hidden_size": 256, "num_hidden_layers": 2,
    "num_attention_heads": 8, "num_key_value_heads": 2, "head_dim": 64,
    "intermediate_size": 256, "max_position_embeddings": 2048, "eos_token_id": None,
}
FAMILIES = {
    "llama": {"architectures": ["LlamaForCausalLM"], "model_type": "llama"},
    "wide": {"architectures": ["LlamaForCausalLM"], "model_type": "llama",
             "head_dim": 128},
    "windows": {"architectures": ["LlamaForCausalLM"], "model_type": "llama",
                "sliding_window": 48,
                "layer_types": ["sliding_attention", "full_attention"]},
    "qwen3": {"architectures": ["Qwen3ForCausalLM"], "model_type": "qwen3"},
}
HEADS = [[(7 * i + 3 + 50 * g) % 500 for i in range(150 + 60 * g)] for g in range(2)]


@pytest.fixture(autouse=True)
def engines_end_with_their_test():
    # graphs captured in inference mode leave torch's generator state such that none can
    # be captured outside of it while they live, and an engine lives on in cycles
    yield
    gc.collect()


def _prompts(groups):
    return [HEADS[g][:] + [(31 * i + j) % 500 for j in range(1 + 5 * i)] if g >= 0
            else [(13 * i + 5 * j) % 500 for j in range(40)]
            for i, g in enumerate(groups)]


def _logits(family, monkeypatch, gpu, **kw):
    """What every step's sampler sees of two batches, each fed the same tokens."""
    cfg = ModelConfig.from_hf_config(SIZES | FAMILIES[family])
    comm = None if gpu else CommContext(
        world_size=1, rank=0, pp_size=1, tp_size=1, pp_rank=0, tp_rank=0,
        device=torch.device("cpu"))
    torch.manual_seed(0)
    eng = Engine(cfg, EngineArgs(**{**dict(
        block_size=16, num_kv_blocks=512, max_batch_size=8, max_model_len=1024,
        dtype=torch.bfloat16 if gpu else torch.float32), **kw}), comm=comm,
        random_weights=True)
    if eng.shared_prefixes is not None:
        eng.shared_prefixes.least_tokens = 1
    seen = []

    def forced(logits, *a, **kw):
        seen.append(logits.detach().float().cpu())
        rows = torch.arange(logits.shape[0], device=logits.device)
        return (37 * rows + 11 * len(seen)) % 500

    with monkeypatch.context() as m:
        m.setattr(ops, "sample_tokens", forced)
        for h in HEADS:
            eng.generate([h], [SamplingParams(temperature=0.0, max_new_tokens=1)])
        for groups in ((0, 1, 0, -1, 0), (1, 1, -1, 0, 1, 0, 0)):
            eng.generate(_prompts(groups), [
                SamplingParams(temperature=0.0, max_new_tokens=4 + 3 * (i % 3),
                               ignore_eos=True) for i in range(len(groups))])
    return seen, eng


def _apart(a, b):
    assert len(a) == len(b) and all(x.shape == y.shape for x, y in zip(a, b))
    return max(((x - y).norm() / y.norm()).item() for x, y in zip(a, b))


@pytest.mark.parametrize("family,fused,graphs,kv", [
    ("llama", False, True, "auto"),
    ("llama", False, False, "auto"),
    ("llama", False, True, "fp8"),
    ("wide", False, True, "auto"),
    ("windows", False, True, "auto"),
    ("qwen3", False, True, "auto"),
    ("qwen3", True, True, "auto"),
    ("qwen3", True, False, "fp8"),
])
def test_against_the_fp32_engine(family, fused, graphs, kv, monkeypatch):
    ref, _ = _logits(family, monkeypatch, gpu=False)
    calls = []
    inner = ops.shared_prefix_attention_decode
    with monkeypatch.context() as m:
        m.setattr(ops, "shared_prefix_attention_decode",
                  lambda *a, **kw: calls.append(1) or inner(*a, **kw))
        if fused:
            m.delattr(ops, "rope_and_cache")
            m.delattr(ops, "rope_cache_attention_decode")
        got, eng = _logits(family, monkeypatch, gpu=True, fused_head_norms=fused,
                           shared_prefix_attention=True, enable_graphs=graphs,
                           kv_cache_dtype=kv)
    assert calls and (not graphs or any(c == SHARED for _, c in eng.graph_runner._graphs))
    assert _apart(got, ref) < 0.10


def test_the_heads_matter(monkeypatch):
    """Without its head a prompt's logits are further away than that."""
    ref, _ = _logits("llama", monkeypatch, gpu=False)
    with monkeypatch.context() as m:
        m.setitem(globals(), "HEADS", [[(11 * i + 9) % 500 for i in range(len(h))]
                                       for h in HEADS])
        other, _ = _logits("llama", monkeypatch, gpu=False)
    assert _apart(other, ref) > 0.3


def test_all_graphs_ahead():
    cfg = ModelConfig.from_hf_config(SIZES | FAMILIES["llama"])
    eng = Engine(cfg, EngineArgs(block_size=16, num_kv_blocks=64, max_batch_size=4,
                                 max_model_len=1024, shared_prefix_attention=True),
                 random_weights=True)
    with torch.inference_mode():
        eng.graph_runner.capture_all()
    assert {b for b, c in eng.graph_runner._graphs if c == SHARED} == {2, 4}


@pytest.mark.parametrize("kw,cfg", [
    (dict(block_size=8), {}), (dict(dtype=torch.float16), {}), ({}, dict(head_dim=32)),
    ({}, dict(num_attention_heads=34, num_key_value_heads=2)),
])
def test_refusals(kw, cfg):
    cfg = ModelConfig.from_hf_config(SIZES | FAMILIES["llama"] | cfg)
    with pytest.raises(ValueError, match="shared_prefix_attention needs bfloat16"):
        Engine(cfg, EngineArgs(num_kv_blocks=64, shared_prefix_attention=True, **kw),
               random_weights=True)
