"""Decode over shared prefixes, on the GPU against 64 bits."""

import random

import pytest
import torch

pytestmark = pytest.mark.gpu

from cache_ops_util import (
    assert_attended, assert_stored, prefix_call, prefix_inputs, prefix_oracle,
    store_oracle)
from parallax_amd import ops

OP = ops.shared_prefix_attention_decode
ODD = [(0, 300), (1, 233), (0, 201), (-1, 170), (0, 0), (1, 5), (7, 9), (0, 200),
       (1, 640), (-3, 1), (0, 1000), (1, 130), (0, 199)]


def check(s, **kw):
    got = prefix_call(OP, s, "cuda", **kw)
    if kw.get("sinks") is not None:
        kw = dict(kw, sinks=kw["sinks"].cpu())
    assert_attended(got, prefix_oracle(s, **kw))
    return got


def shared(B, prefix, most, seed=0):
    """B rows of a group, of 1 to `most` tokens of their own."""
    r = random.Random(seed)
    return [(0, prefix + r.randint(1, most)) for _ in range(B)]


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("BS", [16, 32, 64])
@pytest.mark.parametrize("Hq,Hk", [(4, 2), (7, 1), (16, 1), (3, 3), (24, 8)])
def test_groups(Hq, Hk, BS, D, fp8):
    """Rows of two groups among each other, rows of none, shorter than their prefix,
    empty ones, prefixes that end inside pages and tiles."""
    check(prefix_inputs(Hq, Hk, D, BS, ODD, [200, 129], fp8, seed=BS + Hq))


@pytest.mark.parametrize("prefix", [1, 15, 16, 31, 32, 33, 63, 64, 65, 127, 128, 129, 513])
@pytest.mark.parametrize("rows", [1, 2, 9])
def test_prefix_lengths(rows, prefix):
    r = [(0, prefix + (i * 7 if i % 3 else 0)) for i in range(rows)]
    check(prefix_inputs(8, 2, 64, 16, r, [prefix], seed=prefix))


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("window", [1, 2, 31, 64, 100, 129, 250, 10 ** 12])
def test_windows(window, fp8):
    """Windows that leave nothing, an end or all of a prefix, for each row its own."""
    check(prefix_inputs(8, 2, 128, 32, ODD, [200, 129], fp8, seed=window % 97),
          sliding_window=window)


@pytest.mark.parametrize("kw", [
    dict(softcap=2.0), dict(scale=-0.11), dict(scale=0.0), dict(softcap=30.0, scale=-0.3),
    dict(softcap=5.0, sliding_window=150),
])
@pytest.mark.parametrize("D", [64, 128])
def test_scores(kw, D):
    check(prefix_inputs(8, 2, D, 32, ODD, [200, 129], seed=D), **kw)


@pytest.mark.parametrize("size", [0.0, 3.0, 40.0, -1e4])
def test_sinks(size):
    sinks = torch.linspace(-1, 1, 8).cuda() * size + (size if size < 0 else 0)
    check(prefix_inputs(8, 2, 64, 16, ODD, [200, 129]), sinks=sinks)
    check(prefix_inputs(8, 2, 64, 16, ODD, [200, 129]), sinks=sinks, sliding_window=40)


def test_infinite_sinks():
    """A head whose sink takes all, one whose sink takes nothing."""
    s = prefix_inputs(4, 2, 64, 16, ODD, [200, 129])
    sinks = torch.tensor([float("-inf"), 0.0, float("-inf"), 1.0]).cuda()
    check(s, sinks=sinks)


@pytest.mark.parametrize("rows,prefix,most,Hq,Hk,D,fp8", [
    (40, 1000, 50, 32, 8, 128, False),
    (70, 333, 200, 16, 2, 64, True),
    (130, 520, 33, 8, 1, 128, False),
    (33, 4000, 3000, 8, 2, 128, True),
    (3, 9000, 20, 4, 1, 64, False),
    (300, 65, 10, 16, 1, 64, False),
])
def test_batches(rows, prefix, most, Hq, Hk, D, fp8):
    check(prefix_inputs(Hq, Hk, D, 32, shared(rows, prefix, most), [prefix], fp8,
                        seed=rows))


def test_many_groups():
    r = random.Random(4)
    prefix = [r.choice([1, 16, 40, 64, 65, 200]) for _ in range(150)]
    rows = [(g, prefix[g] + r.randint(0, 30)) for g in range(150) for _ in range(2)]
    r.shuffle(rows)
    check(prefix_inputs(4, 1, 64, 16, rows, prefix))


@pytest.mark.parametrize("rows", [0, 1])
def test_no_groups(rows):
    got = prefix_call(OP, prefix_inputs(4, 2, 64, 16, [(0, 20)] * rows, []), "cuda")
    assert got.shape == (rows, 4, 64)


def test_most_rows():
    rows = shared(4096, 20, 12)
    check(prefix_inputs(2, 1, 64, 16, rows, [20] + [7] * 255))


def test_empty_batch_of_rows():
    got = check(prefix_inputs(4, 2, 64, 16, [(0, 0), (-1, 0), (1, 0)], [5, 0]))
    assert (got == 0).all()


def test_strided_queries():
    check(prefix_inputs(8, 2, 64, 16, ODD, [200, 129], q_gap=264))
    check(prefix_inputs(8, 2, 64, 16, ODD, [200, 129], q_gap=1))  # rows at odd addresses


def test_alignment():
    s = prefix_inputs(8, 2, 64, 16, ODD, [200, 129])
    want = prefix_call(OP, s, "cuda")

    def odd(q, kc, vc, *a, **kw):
        def at(x):
            y = torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")[1:].view(x.shape)
            return y.copy_(x)
        return OP(at(q), at(kc), at(vc), *a, **kw)

    assert torch.equal(prefix_call(odd, s, "cuda"), want)


def test_sharp():
    """Scores of some hundreds: one key takes all."""
    check(prefix_inputs(8, 2, 64, 16, ODD, [200, 129], sharp=16.0))


def test_pages_outside_the_cache():
    """Entries that are no pages are read as the cache's nearest one."""
    s = prefix_inputs(8, 2, 64, 16, [(0, 300), (0, 330), (-1, 50)], [280], spare=0)
    bad = {**s, "tables": s["tables"].clone()}
    pages = s["kc"].shape[0]
    s["kc"], s["vc"] = (x.float().nan_to_num().bfloat16() for x in (s["kc"], s["vc"]))
    bad["kc"], bad["vc"] = s["kc"], s["vc"]
    for (b, i), page in {(0, 2): -7, (0, 17): 1 << 30, (1, 20): pages, (2, 0): -1}.items():
        bad["tables"][b, i] = page
        s["tables"][b, i] = min(max(page, 0), pages - 1)
    assert torch.equal(prefix_call(OP, bad, "cuda"), prefix_call(OP, s, "cuda"))


def test_same_twice():
    s = prefix_inputs(16, 2, 128, 32, shared(90, 700, 900), [700])
    assert torch.equal(prefix_call(OP, s, "cuda"), prefix_call(OP, s, "cuda"))


def test_far_pages():
    """A cache of over 2^32 values, whose last pages hold the sequences."""
    s = prefix_inputs(16, 8, 128, 64, [(0, 300), (0, 330), (-1, 50)], [280], fp8=True)
    want = prefix_oracle(s)
    n = s["kc"].shape[0]
    blocks = (1 << 32) // (8 * 64 * 128) + 2 + n
    kc = torch.empty(blocks, 8, 64, 128, dtype=s["kc"].dtype, device="cuda")
    vc = torch.empty(blocks, 8, 128, 64, dtype=s["kc"].dtype, device="cuda")
    kc[-n:], vc[-n:] = s["kc"].cuda(), s["vc"].cuda()

    def far(q, _, __, tables, *a, **kw):
        return OP(q, kc, vc, tables + (blocks - n), *a, **kw)

    assert_attended(prefix_call(far, s, "cuda"), want)


@torch.inference_mode()  # engines capture in it: outside, none could behind them
def test_captured():
    """Two captured calls follow lengths, groups and tables, also between eager ones."""
    B = 24
    sets = [prefix_inputs(8, 2, 64, 16, rows, prefix, seed=i, spare=spare)
            for i, (rows, prefix, spare) in enumerate([
                (shared(B, 500, 40), [500, 0], 0),
                ([(i % 2, 300 + 13 * i) for i in range(B)], [100, 290], 0),
                ([(-1, i) for i in range(B)], [9, 9], 0)])]
    pages = max(s["kc"].shape[0] for s in sets)
    wide = max(s["tables"].shape[1] for s in sets)

    def put(s, to):
        for x, y in zip((s["q"].view(B, 8, 64), s["kc"], s["vc"], s["tables"], s["lens"],
                         s["group"], s["prefix"]), to):
            y[tuple(slice(0, n) for n in x.shape)] = x.to(y.device)

    def buffers():
        i = dict(dtype=torch.int32, device="cuda")
        b = dict(dtype=torch.bfloat16, device="cuda")
        return [torch.zeros(B, 8, 64, **b), torch.zeros(pages, 2, 16, 64, **b),
                torch.zeros(pages, 2, 64, 16, **b), torch.zeros(B, wide, **i),
                torch.zeros(B, **i), torch.zeros(B, **i), torch.zeros(2, **i)]

    two, graphs, outs, pool = [buffers(), buffers()], [], [], None
    side = torch.cuda.Stream()
    for k in range(2):
        put(sets[2], two[k])
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            OP(*two[k], 0.125)
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[k], pool=pool):
            outs.append(OP(*two[k], 0.125))
        pool = graphs[0].pool()
    for turn in range(4):
        for k in range(2):
            s = sets[(turn + k) % 3]
            put(s, two[k])
            graphs[k].replay()
            got = outs[k].clone()
            assert torch.equal(got, OP(*two[k], 0.125))
            assert_attended(got, prefix_oracle(s))


def test_other_stream():
    s = prefix_inputs(8, 2, 64, 16, ODD, [200, 129])
    want = prefix_call(OP, s, "cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = prefix_call(OP, s, "cuda")
    side.synchronize()
    assert torch.equal(got, want)


def test_steps_together():
    """Decode steps as a layer makes them: norms, rotation and append of every row's
    token, then attention over the shared prefix, the rows growing."""
    Hq, Hk, D, BS, P = 8, 2, 64, 16, 50
    rows = [(0, P + 1 + i * 5) for i in range(6)] + [(-1, 14), (-1, 31)]
    B = len(rows)
    s = prefix_inputs(Hq, Hk, D, BS, rows, [P], spare=0)
    # room for three more tokens in every row
    grown = prefix_inputs(Hq, Hk, D, BS, [(g, n + 3) for g, n in rows], [P], seed=1)
    kc, vc = grown["kc"].cuda(), grown["vc"].cuda()
    g = torch.Generator().manual_seed(0)
    table = torch.randn(200, D, generator=g)
    qw, kw = ((1 + 0.3 * torch.randn(D, generator=g)).bfloat16() for _ in range(2))
    for step in range(3):
        lens = torch.tensor([n + step + 1 for _, n in rows], dtype=torch.int32)
        pos = lens - 1
        slots = torch.tensor([int(grown["tables"][b, p // BS]) * BS + p % BS
                              for b, p in enumerate(pos.tolist())])
        full = torch.randn(B, (Hq + 2 * Hk) * D, generator=g).bfloat16()
        before = (kc.cpu(), vc.cpu())
        heads = full.cuda().view(B, -1, D)
        q, k, v = heads.split([Hq, Hk, Hk], 1)
        out = ops.qk_norm_rope_and_cache(
            q, k, v, qw.cuda(), kw.cuda(), 1e-5, kc, vc, pos.cuda(), table.cuda(),
            slots.cuda())
        want, err = store_oracle(dict(
            full=full, T=B, Hq=Hq, Hk=Hk, D=D, W=D, qw=qw, kw=kw, eps=1e-5,
            kc=before[0], vc=before[1], pos=pos, table=table, slots=slots,
            scales=(1.0, 1.0)), True)
        assert_stored((out, kc, vc), want, err)
        now = {**grown, "q": out.cpu().view(B, -1), "kc": kc.cpu(), "vc": vc.cpu(),
               "lens": lens}
        assert_attended(prefix_call(OP, now, "cuda"), prefix_oracle(now))


def test_lengths_past_the_table():
    s = prefix_inputs(4, 2, 64, 16, [(0, 48), (0, 48), (1, 48)], [20, 60])
    s["tables"] = s["tables"][:, :3].contiguous()
    want = prefix_oracle(s)
    s["lens"] = torch.tensor([48, 49, 2 ** 31 - 1], dtype=torch.int32)
    assert_attended(prefix_call(OP, s, "cuda"), want)


@pytest.mark.parametrize("Hk,D,groups,prefix", [
    (32, 64, 40, 150),    # 24 workgroups a head, 40 tiles of items
    (64, 128, 20, 500),   # 8 and 20
    (300, 64, 3, 70),     # 2 and 3
    (400, 128, 1, 200),   # 2, of which one takes suffixes
    (1, 64, 256, 130),    # all groups that there can be
])
def test_tiles_and_workgroups(Hk, D, groups, prefix):
    """More tiles of items than workgroups: runs that go from one group to the next."""
    r = random.Random(Hk)
    lens = [prefix + r.randint(-60, 60) for _ in range(groups)]
    rows = [(g, lens[g] + r.randint(0, 40)) for g in range(groups) for _ in range(3)]
    r.shuffle(rows)
    check(prefix_inputs(Hk, Hk, D, 16, rows, lens, seed=Hk))


def test_only_prefixes():
    """No row has a token of its own."""
    check(prefix_inputs(8, 2, 128, 16, [(0, 700)] * 20 + [(1, 64)] * 3, [700, 64]))
    check(prefix_inputs(64, 64, 128, 16, [(g, 100) for g in range(20)] * 2, [100] * 20))


@pytest.mark.parametrize("seed", range(24))
def test_any(seed):
    """Rows, groups, heads, pages, windows as they come."""
    r = random.Random(100 + seed)
    Hk, D, BS = r.choice([1, 2, 3, 8]), r.choice([64, 128]), r.choice([16, 32, 64])
    Hq = Hk * r.choice([1, 2, 5, 7, 8, 16])
    prefix = [r.choice([0, 1, 17, 64, 100, 400, 1500]) for _ in range(r.randint(0, 12))]
    rows = []
    for _ in range(r.choice([1, 3, 17, 64, 150])):
        g = r.randint(-1, len(prefix))
        P = prefix[g] if 0 <= g < len(prefix) else 0
        rows.append((g, max(0, r.choice([P, P, P, 0]) + r.choice([-1, 0, 1, 30, 200]))))
    kw = {}
    if r.random() < 0.4:
        kw["sliding_window"] = r.choice([1, 30, 64, 200, 1000])
    if r.random() < 0.3:
        kw["softcap"] = r.choice([1.0, 20.0])
    if r.random() < 0.3:
        kw["sinks"] = torch.randn(Hq, generator=torch.Generator().manual_seed(seed)).cuda()
    check(prefix_inputs(Hq, Hk, D, BS, rows, prefix, fp8=r.random() < 0.5, seed=seed,
                        q_gap=r.choice([0, 8])), **kw)


@torch.inference_mode()  # engines capture in it: outside, none could behind them
def test_two_at_once():
    """Calls on two streams and graphs replayed on both, each with results of its own."""
    a = prefix_inputs(8, 2, 64, 16, ODD, [200, 129])
    b = prefix_inputs(16, 2, 128, 32, shared(30, 900, 100), [900], fp8=True)
    want = [prefix_call(OP, s, "cuda") for s in (a, b)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    args, graphs, outs = [], [], []
    for s in (a, b):
        B, Hq, D = s["shape"]
        args.append([s["q"].cuda().view(B, Hq, D)] + [s[n].cuda() for n in (
            "kc", "vc", "tables", "lens", "group", "prefix")] + [D ** -0.5, -1, 0.0, None,
                                                                 *s["scales"]])
    torch.cuda.synchronize()
    for x in args:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(OP(*x))
        graphs.append(g)
    for _ in range(20):
        eager = []
        for s, g, x in zip(streams, graphs, args):
            with torch.cuda.stream(s):
                g.replay()
                eager.append(OP(*x))
        torch.cuda.synchronize()
        for w, o, e in zip(want, outs, eager):
            assert torch.equal(o, w) and torch.equal(e, w)
