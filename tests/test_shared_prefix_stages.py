"""Pipeline stages that hold different layers, with the engine options around a shared
cache, as processes on the CPU: a stage without a layer for an option goes on, and a
refusal reaches all of them."""

import os
import socket

import pytest
import torch
import torch.multiprocessing as mp

from parallax_amd.models.config import ModelConfig

PROMPTS = [list(range(1, 30)) + [100 + i, 50, 60 + i] for i in range(3)]


def _cfg(layer_types, **kw):
    return ModelConfig(**{**dict(
        architecture="LlamaForCausalLM", vocab_size=211, hidden_size=64, num_layers=4,
        num_heads=4, num_kv_heads=2, head_dim=16, intermediate_size=128,
        max_position_embeddings=512, eos_token_ids=[], rope_theta=10000.0,
        sliding_window=12, layer_types=layer_types), **kw})


def _weights(eng):
    g = torch.Generator().manual_seed(1)
    every = {}
    for i in range(eng.cfg.num_layers):
        for name, size in (("q", 64), ("k", 32), ("v", 32)):
            every[f"model.layers.{i}.self_attn.{name}_proj.weight"] = (size, 64)
        every[f"model.layers.{i}.self_attn.o_proj.weight"] = (64, 64)
        every[f"model.layers.{i}.mlp.gate_proj.weight"] = (128, 64)
        every[f"model.layers.{i}.mlp.up_proj.weight"] = (128, 64)
        every[f"model.layers.{i}.mlp.down_proj.weight"] = (64, 128)
        for name in ("input", "post_attention"):
            every[f"model.layers.{i}.{name}_layernorm.weight"] = None
    every["model.embed_tokens.weight"] = every["lm_head.weight"] = (211, 64)
    every["model.norm.weight"] = None
    for name, shape in every.items():
        eng.model.load_hf_weight(
            name, torch.ones(64) if shape is None
            else 0.15 * torch.randn(shape, generator=g))


def _engine(cfg, comm, **kw):
    from parallax_amd.server.engine import Engine, EngineArgs

    eng = Engine(cfg, EngineArgs(block_size=4, num_kv_blocks=256, dtype=torch.float32,
                                 **kw), comm=comm, random_weights=True)
    if eng.shared_prefixes is not None:
        eng.shared_prefixes.least_tokens = 1
    return eng


def _generate(eng):
    from parallax_amd.server.sampling_params import SamplingParams

    _weights(eng)
    eng.generate([PROMPTS[0][:29]], [SamplingParams(temperature=0.0, max_new_tokens=1)])
    return list(eng.generate(PROMPTS, [SamplingParams(
        temperature=0.0, max_new_tokens=8, ignore_eos=True)] * len(PROMPTS)).values())


def _stage(rank, world, port, work, out):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank),
                      WORLD_SIZE=str(world))
    import torch.distributed as dist

    from parallax_amd.parallel.comm import init_distributed

    torch.set_num_threads(2)
    comm = init_distributed(pp_size=world, tp_size=1, backend="gloo",
                            device=torch.device("cpu"), timeout_s=60)
    torch.save(work(rank, comm), f"{out}.{rank}")
    dist.barrier()
    dist.destroy_process_group()


def _two_stages(work, tmp_path):
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    out = str(tmp_path / "out")
    mp.spawn(_stage, args=(2, port, work, out), nprocs=2, join=True)
    return [torch.load(f"{out}.{r}") for r in range(2)]


def _windows_first(rank, comm):
    from parallax_amd import ops

    calls = []
    inner = ops.shared_prefix_attention_decode
    ops.shared_prefix_attention_decode = lambda *a, **kw: calls.append(1) or inner(*a, **kw)
    try:
        eng = _engine(_cfg(["sliding_attention"] * 2 + ["full_attention"] * 2), comm,
                      shared_prefix_attention=True)
        return _generate(eng), eng.shared_prefixes is not None, len(calls)
    finally:
        ops.shared_prefix_attention_decode = inner


def test_a_stage_of_windows(tmp_path):
    """The first stage's layers all have windows: it goes on without, the other shares."""
    from parallax_amd.parallel.comm import CommContext

    alone = CommContext(world_size=1, rank=0, pp_size=1, tp_size=1, pp_rank=0, tp_rank=0,
                        device=torch.device("cpu"))
    want, shares, calls = _windows_first(0, alone)
    assert shares and calls
    first, second = _two_stages(_windows_first, tmp_path)
    assert first[0] == want
    assert first[1:] == (False, 0) and second[1] and second[2]


def _refusals(rank, comm):
    """What each option says where rank 1, or no rank, has layers for it."""
    from parallax_amd.server.engine import Engine

    own = Engine._attentions
    said = []
    for lacking in ((0,), (0, 1)):
        Engine._attentions = lambda self: [] if rank in lacking else own(self)
        for option in ("shared_prefix_attention", "fused_head_norms"):
            try:
                _engine(_cfg(None, qk_norm=True, sliding_window=-1), comm,
                        **{option: True})
                said.append(None)
            except ValueError as e:
                said.append(str(e))
    Engine._attentions = own
    return said


def test_refusals_reach_all(tmp_path):
    first, second = _two_stages(_refusals, tmp_path)
    assert first == second
    assert [bool(x) for x in first] == [True, False, True, True]
    assert "layers without it" in first[0] and "no norms of single heads" in first[3]
