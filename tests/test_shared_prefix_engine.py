"""Engines that read shared prefixes once and norm heads on the way into the cache: which
rows of a batch are grouped, that the same tokens come out, what is refused, on the CPU."""

import itertools
import random

import pytest
import torch

from parallax_amd import ops
from parallax_amd.cli import add_engine_args, engine_args_from_cli
from parallax_amd.models.config import ModelConfig
from parallax_amd.parallel.comm import CommContext
from parallax_amd.server.engine import Engine, EngineArgs
from parallax_amd.server.kv_cache import KVCacheSpec
from parallax_amd.server.sampling_params import SamplingParams
from parallax_amd.server.shared_prefix import SharedPrefixes, find_shared_prefixes

BS = 4


def _best(tables, seq_lens):
    """Most tokens' reads saved by any grouping, by trying all (few rows)."""
    def head(rows):
        n = min(min(len(tables[r]), seq_lens[r] // BS) for r in rows)
        k = 0
        while k < n and len({tables[r][k] for r in rows}) == 1:
            k += 1
        return k * BS

    def partitions(rows):
        if not rows:
            yield []
            return
        first, rest = rows[0], rows[1:]
        for n in range(len(rest) + 1):
            for others in itertools.combinations(rest, n):
                left = [r for r in rest if r not in others]
                for p in partitions(left):
                    yield [(first, *others)] + p

    return max(sum(head(g) * (len(g) - 1) for g in p)
               for p in partitions(list(range(len(tables)))))


def _saved(tables, seq_lens, groups, lens):
    total = 0
    for g, tokens in enumerate(lens):
        rows = [i for i, x in enumerate(groups) if x == g]
        assert len(rows) > 1 and tokens > 0 and tokens % BS == 0
        n = tokens // BS
        assert len({tuple(tables[r][:n]) for r in rows}) == 1
        assert all(len(tables[r]) >= n and seq_lens[r] >= tokens for r in rows)
        total += tokens * (len(rows) - 1)
    return total


def test_nothing_to_share():
    assert find_shared_prefixes([], [], BS) == ([], [])
    assert find_shared_prefixes([[1, 2]], [8], BS) == ([-1], [])
    assert find_shared_prefixes([[1, 2], [3, 2]], [8, 8], BS) == ([-1, -1], [])
    assert find_shared_prefixes([[], []], [0, 0], BS) == ([-1, -1], [])


def test_whole_pages_within_every_length():
    tables = [[1, 2, 3, 4], [1, 2, 3, 5], [9]]
    assert find_shared_prefixes(tables, [16, 14, 3], BS) == ([0, 0, -1], [12])
    assert find_shared_prefixes(tables, [16, 11, 3], BS) == ([0, 0, -1], [8])
    # one table that begins another, and one table twice
    assert find_shared_prefixes([[1, 2], [1, 2, 3]], [8, 9], BS) == ([0, 0], [8])
    assert find_shared_prefixes([[1, 2], [1, 2]], [8, 8], BS) == ([0, 0], [8])


def test_deeper_groups_where_they_save_more():
    # a short head of all, long ones of two pairs: 2 pages x 3 against 10 + 10
    a, b = list(range(10, 20)), list(range(20, 30))
    tables = [[1, 2] + a[2:] + [50], [1, 2] + a[2:] + [51],
              [1, 2] + b[2:] + [52], [1, 2] + b[2:] + [53]]
    groups, lens = find_shared_prefixes(tables, [44] * 4, BS)
    assert groups[0] == groups[1] != groups[2] == groups[3] and lens == [40, 40]
    # and the head of all where the branches are short
    tables = [list(range(8)) + [30 + i // 2, 50 + i] for i in range(4)]
    assert find_shared_prefixes(tables, [40] * 4, BS) == ([0] * 4, [32])


@pytest.mark.parametrize("seed", range(40))
def test_saves_the_most(seed):
    rnd = random.Random(seed)
    heads = [[rnd.randrange(3) + 10 * d for d in range(6)] for _ in range(3)]
    tables, lens = [], []
    for i in range(rnd.randint(2, 6)):
        t = list(rnd.choice(heads)[:rnd.randint(0, 6)])
        t += [1000 + 100 * i + k for k in range(rnd.randint(1, 3))]
        tables.append(t)
        lens.append(rnd.randint(1, len(t) * BS))
    groups, shared = find_shared_prefixes(tables, lens, BS)
    assert _saved(tables, lens, groups, shared) == _best(tables, lens)


def test_the_groups_that_save_most_are_kept():
    tables = [[10 * g + d for d in range(g + 1)] + [1000 + 2 * g + r]
              for g in range(5) for r in range(2)]
    groups, lens = find_shared_prefixes(tables, [100] * 10, BS, max_groups=2)
    assert lens == [5 * BS, 4 * BS] and groups == [-1] * 6 + [1, 1, 0, 0]


def test_found_again_only_for_other_rows():
    spec = KVCacheSpec(1, 2, 64, BS)
    token = 2 * 2 * 64 * 2
    s = SharedPrefixes(spec, least_bytes=8 * token)
    a, b = [1, 2, 3], [1, 2, 4]
    found = s.find([a, b], [9, 9])
    assert found == ([0, 0], [8])
    a.append(7)
    assert s.find([a, b], [13, 10]) is found
    assert s.find([a, list(b)], [13, 10]) is not found
    assert s.find([a, b], [13, 10]) is found      # two batches in turn
    assert s.find([b, a], [10, 13]) == found
    c = [1, 2, 5]
    for _ in range(20):
        s.find([list(a), c], [13, 9])
    assert len(s._batches) == s.BATCHES
    again = s.find([a, b], [13, 10])
    assert again is not found and again == found
    assert SharedPrefixes(spec, least_bytes=8 * token + 1).find([a, b], [13, 9]) is None
    assert SharedPrefixes(spec, least_bytes=0).find([a, [9]], [13, 3]) is None


def _cfg(**kw):
    return ModelConfig(**{**dict(
        architecture="LlamaForCausalLM", vocab_size=211, hidden_size=64, num_layers=2,
        num_heads=4, num_kv_heads=2, head_dim=16, intermediate_size=128,
        max_position_embeddings=512, eos_token_ids=[], rope_theta=10000.0), **kw})


def _engine(cfg, **kw):
    comm = CommContext(world_size=1, rank=0, pp_size=1, tp_size=1, pp_rank=0, tp_rank=0,
                       device=torch.device("cpu"))
    torch.manual_seed(0)
    eng = Engine(cfg, EngineArgs(**{**dict(block_size=BS, num_kv_blocks=256,
                                           dtype=torch.float32), **kw}),
                 comm=comm, random_weights=True)
    if eng.shared_prefixes is not None:
        eng.shared_prefixes.least_tokens = 1
    return eng


HEAD = list(range(1, 30))
PROMPTS = [HEAD + [100 + i, 50, 60 + i] for i in range(3)] + [[7, 8, 9]]
SPS = [SamplingParams(temperature=0.0, max_new_tokens=n, ignore_eos=True)
       for n in (6, 9, 12, 12)]


def _generate(eng):
    eng.generate([HEAD], [SamplingParams(temperature=0.0, max_new_tokens=1)])
    return list(eng.generate(PROMPTS, SPS).values())


@pytest.mark.parametrize("kind", ["plain", "windows", "norms"])
def test_same_tokens(kind, monkeypatch):
    cfg = _cfg(**{"plain": {}, "norms": dict(qk_norm=True),
                  "windows": dict(sliding_window=12, layer_types=[
                      "sliding_attention", "full_attention"])}[kind])
    plain = _generate(_engine(cfg))
    calls = []
    inner = ops.shared_prefix_attention_decode

    def counted(*a, **kw):
        calls.append((a[5].tolist(), a[6].tolist()))
        return inner(*a, **kw)

    monkeypatch.setattr(ops, "shared_prefix_attention_decode", counted)
    eng = _engine(cfg, shared_prefix_attention=True)
    assert _generate(eng) == plain
    shared = len(HEAD) // BS * BS
    assert ([0, 0, 0, -1], [shared]) in calls and ([0, 0, -1], [shared]) in calls
    # too little saved: not used
    calls.clear()
    eng = _engine(cfg, shared_prefix_attention=True)
    eng.shared_prefixes.least_tokens = 1000
    assert _generate(eng) == plain and not calls


@pytest.mark.parametrize("shared", [False, True])
def test_fused_head_norms_same_tokens(shared, monkeypatch):
    cfg = _cfg(qk_norm=True)
    plain = _generate(_engine(cfg))
    for name in ("rope_and_cache", "rope_cache_attention_decode"):
        monkeypatch.delattr(ops, name)
    eng = _engine(cfg, fused_head_norms=True, shared_prefix_attention=shared)
    assert _generate(eng) == plain


def test_refusals():
    with pytest.raises(ValueError, match="no norms of single heads"):
        _engine(_cfg(), fused_head_norms=True)
    with pytest.raises(ValueError, match="no norms of single heads"):
        _engine(_cfg(qk_norm=True, qk_norm_full=True), fused_head_norms=True)
    with pytest.raises(ValueError, match="all layers have windows"):
        _engine(_cfg(sliding_window=8, layer_types=["sliding_attention"] * 2),
                shared_prefix_attention=True)
    with pytest.raises(ValueError, match="needs the prefix cache"):
        _engine(_cfg(), shared_prefix_attention=True, enable_prefix_cache=False)


def test_command_line():
    import argparse

    p = argparse.ArgumentParser()
    add_engine_args(p)
    args = engine_args_from_cli(p.parse_args([]))
    assert not args.fused_head_norms and not args.shared_prefix_attention
    args = engine_args_from_cli(p.parse_args(
        ["--fused-head-norms", "--shared-prefix-attention"]))
    assert args.fused_head_norms and args.shared_prefix_attention
