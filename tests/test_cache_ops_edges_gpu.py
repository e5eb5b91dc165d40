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


CAPS = [64.0, 64.1, 1e3, 1e5, 1e8, 1e30, 3e38, 1e300]


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


def assert_same_numbers(got, oracle):
    """Infinities and NaN where the oracle has them, and what is left as ever. -> how
    many values and rows have some."""
    want, size = oracle
    x = got.cpu().double()
    assert torch.equal(x.isnan(), want.isnan())
    assert torch.equal(x.isinf(), want.isinf())
    assert torch.equal(x[x.isinf()], want[want.isinf()])
    none = ~torch.isfinite(want)
    assert_attended(x.masked_fill(none, 0.0),
                    (want.masked_fill(none, 0.0), size.masked_fill(none, 0.0)))
    return int(none.sum()), int(none.any(-1).any(-1).sum())


def put_value(s, row, token, head, d, value):
    BS = s["kc"].shape[2]
    page = int(s["tables"][row, token // BS])
    s["vc"][page, head, d, token % BS] = value


@pytest.mark.parametrize("value", [NAN, INF])
@pytest.mark.parametrize("D", [64, 128])
def test_values_that_are_no_numbers(D, value):
    """Of a prefix and of a row's own tokens, in rows of many parts and of one: one value
    a head is none, the others are as ever."""
    rows = [(0, 3000 + 70 * i) for i in range(5)] + [(-1, 5000), (-1, 33), (0, 3000)]
    s = prefix_inputs(8, 2, D, 32, rows, [3000], seed=D)
    put_value(s, 0, 17, 0, 5, value)
    put_value(s, 2, 3100, 1, 9, value)
    put_value(s, 5, 4000, 0, 30, value)
    put_value(s, 6, 32, 1, 31, value)
    got = prefix_call(ATTEND, s, "cuda")
    values, _ = assert_same_numbers(got, prefix_oracle(s))
    # head 0 of the six rows of the group, head 1 of row 2, one each of rows 5 and 6: four
    # query heads a head
    assert values == 4 * (6 + 1 + 1 + 1)


@pytest.mark.parametrize("value", [NAN, INF, -INF])
@pytest.mark.parametrize("Hq,Hk,D,BS,fp8", [
    (8, 1, 64, 16, False), (8, 2, 128, 32, False), (3, 3, 128, 64, False),
    (16, 1, 128, 32, True), (6, 2, 64, 64, True),
])
def test_windows_over_no_numbers(Hq, Hk, D, BS, fp8, value):
    """A shared token that one row's window hides and another's does not: only the rows
    that see it get its NaN or infinity."""
    rows = [(0, 300 + 3 * i) for i in range(33)] + [(0, 900), (-1, 170), (0, 320)]
    s = prefix_inputs(Hq, Hk, D, BS, rows, [250], fp8, seed=D + BS)
    put = [(152, 0, 5), (200, Hk - 1, D - 1), (201, Hk - 1, 0), (231, 0, 33),
           (249, 0, 40)]
    for token, head, d in put:
        put_value(s, 0, token, head, d, value)
    want = prefix_oracle(s, sliding_window=150)
    got = prefix_call(ATTEND, s, "cuda", sliding_window=150)
    values, seen_by = assert_same_numbers(got, want)
    assert 0 < values and 30 < seen_by < len(rows)


def test_scales_of_a_bf16_cache():
    """Scales are those of fp8 caches; a bf16 one holds its values as they are."""
    s = prefix_inputs(8, 2, 64, 16, ODD, [200, 129])
    want = prefix_call(ATTEND, s, "cuda")
    assert torch.equal(prefix_call(ATTEND, {**s, "scales": (0.5, 0.25)}, "cuda"), want)
    s = store_inputs(40, 4, 2, 64, 64, 16)
    for got, want in zip(call(STORE, s, "cuda", change=dict(k_scale=0.5, v_scale=0.25)),
                         call(STORE, s, "cuda")):
        assert torch.equal(got, want)


@pytest.mark.parametrize("T,D,rot", [(1 << 25, 1, 0), (1 << 26, 16, 16)])
def test_more_rows_than_a_launch_has(T, D, rot):
    """Of one head: more than 2^26 waves of the form for any sizes, more than 2^24
    workgroups of the other. The same as in portions."""
    g = torch.Generator(device="cuda").manual_seed(0)
    b = torch.bfloat16
    q, k, v = (torch.randn(T, 1, D, generator=g, device="cuda", dtype=b) for _ in range(3))
    qw, kw = (1 + torch.randn(2, D, generator=g, device="cuda")).to(b)
    table = torch.randn(50, rot, generator=g, device="cuda")
    pos = torch.randint(0, 50, (T,), generator=g, device="cuda", dtype=torch.int32)
    slots = torch.randperm(T // 64, generator=g, device="cuda")[:, None] * 64 + torch.arange(
        64, device="cuda")
    slots = slots.view(-1)

    def caches():
        return (torch.zeros(T // 16, 1, 16, D, dtype=b, device="cuda"),
                torch.zeros(T // 16, 1, D, 16, dtype=b, device="cuda"))

    kc, vc = caches()
    out = STORE(q, k, v, qw, kw, 1e-5, kc, vc, pos, table, slots)
    kc2, vc2 = caches()
    n = 1 << 22
    for a in range(0, T, n):
        at = slice(a, a + n)
        part = STORE(q[at], k[at], v[at], qw, kw, 1e-5, kc2, vc2, pos[at], table, slots[at])
        assert torch.equal(out[at], part)
    assert torch.equal(kc, kc2) and torch.equal(vc, vc2) and bool((vc != 0).any())


def test_wide_integers():
    """Lengths, groups, pages and positions of 64 bits are what they say, not what is
    left of them in 32."""
    s = prefix_inputs(4, 2, 64, 16, [(0, 48), (0, 48), (1, 48), (2, 48)], [20, 30])
    s["tables"] = s["tables"][:, :3].contiguous()
    s["kc"], s["vc"] = (x.float().nan_to_num().bfloat16() for x in (s["kc"], s["vc"]))
    want = prefix_call(ATTEND, s, "cuda")
    wide = {**s, **{n: s[n].long() for n in ("lens", "group", "tables", "prefix")}}
    wide["lens"][1] += 1 << 32
    wide["group"][3] += (1 << 32) - 2       # not group 0
    assert torch.equal(prefix_call(ATTEND, wide, "cuda"), want)
    wide["tables"][0, 1] = 1 << 32          # the last page, not the first
    s["tables"][0, 1] = s["kc"].shape[0] - 1
    assert torch.equal(prefix_call(ATTEND, wide, "cuda"),
                       prefix_call(ATTEND, s, "cuda"))
    s = store_inputs(6, 4, 2, 64, 64, 16)
    pos = s["pos"].long()
    pos[2] += 1 << 32
    q, kc, vc = call(STORE, s, "cuda", change=dict(positions=pos.cuda()))
    assert q[2].isnan().all() and not q[:2].isnan().any() and not q[3:].isnan().any()


@pytest.mark.parametrize("sink", [90.0, 1e4, 3e38, INF])
def test_sinks_that_take_all(sink):
    """Of a row that one wave finishes, of rows that are joined: nothing is left."""
    s = prefix_inputs(4, 2, 64, 16, ODD, [200, 129])
    sinks = torch.tensor([sink, 0.0, -INF, sink])
    for kw in (dict(), dict(sliding_window=40)):
        got = prefix_call(ATTEND, s, "cuda", sinks=sinks.cuda(), **kw)
        # the oracle's softmax of an infinite sink is no number
        want = prefix_oracle(s, sinks=sinks.clamp(max=1e30), **kw)
        # below 2^-126 bf16 goes in steps of 2^-133: beside what a weight is off by, a
        # rounding is off by up to 2^-134, which no share of the value covers
        x = got.cpu().double()
        assert_attended(x - (x - want[0]).clamp(-(2.0 ** -134), 2.0 ** -134), want)
        assert (got[:, [0, 3]].abs() < 1e-30).all()


@pytest.mark.parametrize("kw", [dict(), dict(softcap=30.0), dict(scale=-0.1)])
@pytest.mark.parametrize("Hq,Hk,D,fp8", [
    (8, 1, 128, False), (8, 2, 128, True), (2, 2, 64, False), (16, 1, 64, True)])
def test_long_windows_over_no_numbers(Hq, Hk, D, fp8, kw):
    """Windows that begin in other tiles for other waves, tiles that all see whole behind
    them, two groups of which one has no such values, none that any row sees."""
    rows = [(i % 2, 3000 + 20 * i) for i in range(60)]
    s = prefix_inputs(Hq, Hk, D, 32, rows, [3000, 1500], fp8, seed=D)
    for token in (300, 500, 2000):
        put_value(s, 0, token, Hk - 1, 7, NAN)
    put_value(s, 0, 90, 0, 9, NAN)  # hidden from all
    got = prefix_call(ATTEND, s, "cuda", sliding_window=2900, **kw)
    values, seen_by = assert_same_numbers(got, prefix_oracle(s, sliding_window=2900, **kw))
    assert values == seen_by * (Hq // Hk) and seen_by == 30


def test_sinks_that_are_no_numbers():
    """Their heads are none, of rows of one part and of many, the others as ever."""
    s = prefix_inputs(4, 2, 64, 16, ODD, [200, 129])
    sinks = torch.tensor([NAN, 0.5, NAN, -2.0])
    got = prefix_call(ATTEND, s, "cuda", sinks=sinks.cuda())
    want, size = prefix_oracle(s, sinks=sinks.nan_to_num())
    some = s["lens"] > 0
    assert got[some][:, [0, 2]].isnan().all() and (got[~some] == 0).all()
    assert_attended(got[:, [1, 3]], (want[:, [1, 3]], size[:, [1, 3]]))


@pytest.mark.parametrize("softcap", [1e-20, 30.0, 1e10])
def test_large_scales(softcap):
    """Scores of 0, and others that a scale takes past any cap."""
    s = prefix_inputs(4, 2, 64, 16, ODD, [200, 129])
    s["q"][::2] = 0
    got = prefix_call(ATTEND, s, "cuda", scale=1e25, softcap=softcap)
    assert_attended(got, prefix_oracle(s, scale=1e25, softcap=softcap))
