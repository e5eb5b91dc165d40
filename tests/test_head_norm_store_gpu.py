"""Head norms, rotation and append in one pass, on the GPU against 64 bits."""

import pytest
import torch

pytestmark = pytest.mark.gpu

from cache_ops_util import FP8, NAN, assert_stored, store_inputs, store_oracle
from parallax_amd import ops
from test_head_norm_store import call

OP = ops.qk_norm_rope_and_cache


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("neox", [False, True])
@pytest.mark.parametrize("T,Hq,Hk,D,rot,BS", [
    (1, 32, 8, 128, 128, 32),
    (3, 14, 2, 64, 64, 16),
    (67, 64, 8, 64, 32, 64),
    (130, 16, 2, 256, 64, 64),
    (33, 6, 6, 96, 48, 16),
    (20, 5, 1, 80, 80, 32),
    (9, 3, 3, 512, 512, 16),
    (7, 2, 1, 16, 16, 16),
    (5, 3, 2, 112, 24, 4),     # pairs that do not come in eights
    (17, 2, 1, 66, 34, 5),
    (4, 4, 2, 7, 6, 1),
    (6, 2, 2, 1024, 1024, 16),
    (11, 4, 2, 128, 0, 16),    # nothing rotated
])
def test_sizes(T, Hq, Hk, D, rot, BS, neox, fp8):
    s = store_inputs(T, Hq, Hk, D, rot, BS, fp8, seed=T + D)
    if T > 2:
        s["slots"][1], s["slots"][2] = -1, s["kc"].shape[0] * BS
    assert_stored(call(OP, s, "cuda", neox), *store_oracle(s, neox))


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("starts,lengths", [
    ([0], [1500]), ([5], [1403]), ([31, 2, 64, 7], [700, 1, 9, 450]),
    ([1] * 130, list(range(1, 18)) * 7 + [9] * 11),
])
@pytest.mark.parametrize("BS", [16, 64, 12])
def test_portions(starts, lengths, BS, fp8):
    """Prompt portions behind contexts of any length, in shuffled pages."""
    g = torch.Generator().manual_seed(3)
    blocks = sum((s % BS + n + BS - 1) // BS for s, n in zip(starts, lengths)) + 2
    ids = torch.randperm(blocks, generator=g)
    slots, at = [], 0
    for s, n in zip(starts, lengths):
        i = s % BS + torch.arange(n)
        slots.append(ids[at + i // BS] * BS + i % BS)
        at += int(i[-1]) // BS + 1
    slots = torch.cat(slots)
    slots[::97] = -1
    s = store_inputs(len(slots), 4, 2, 64, 32, BS, fp8, slots=slots, blocks=blocks)
    assert_stored(call(OP, s, "cuda"), *store_oracle(s, True))


@pytest.mark.parametrize("head_gap,row_gap", [(8, 0), (1, 0), (0, 3), (64, 8), (0, 8)])
@pytest.mark.parametrize("T", [40, 1100])
def test_strides(head_gap, row_gap, T):
    s = store_inputs(T, 4, 2, 64, 64, 16, seed=T, head_gap=head_gap, row_gap=row_gap)
    assert_stored(call(OP, s, "cuda"), *store_oracle(s, True))


def test_alignment():
    """Tensors that begin at odd offsets."""
    s = store_inputs(30, 4, 2, 64, 64, 16)
    want = store_oracle(s, True)
    for name in ("qw", "kw", "table", "kc", "vc"):
        x = s[name].cuda()
        at = torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")[1:].view(x.shape)
        at.view(torch.uint8).copy_(x.view(torch.uint8))
        key = dict(qw="q_weight", kw="k_weight", table="cos_sin", kc="k_cache",
                   vc="v_cache")[name]
        assert_stored(call(OP, s, "cuda", change={key: at}), *want)


def test_same_as_apart():
    """Beside the norms and rope_and_cache() apart, whose values between are rounded."""
    s = store_inputs(50, 8, 2, 128, 128, 32)
    (q, kc, vc) = call(OP, s, "cuda")

    def apart(q, k, v, qw, kw, eps, kc, vc, pos, table, slots, neox, ks, vs):
        q, k = ops.rmsnorm(q.contiguous(), qw, eps), ops.rmsnorm(k.contiguous(), kw, eps)
        ops.rope_and_cache(q, k, v.contiguous(), kc, vc, pos, table, slots, neox)
        return q

    q2, kc2, vc2 = call(apart, s, "cuda")
    assert torch.equal(vc, vc2)
    # table values of up to 4: two roundings of 2^-8 and what is turned
    assert ((q - q2).abs() <= (q.abs() + 8 * q.abs().amax(-1, keepdim=True)) * 2 ** -7).all()


def test_numbers_that_are_none():
    """NaN and infinity stay with their head, positions outside the table make NaN."""
    s = store_inputs(6, 4, 2, 64, 32, 16)
    W = s["W"]
    s["full"][0, 5] = NAN
    s["full"][1, W + 3] = float("inf")
    s["full"][2, :W] = 0
    q, kc, vc = call(OP, s, "cuda")
    assert q[0, 0].isnan().all() and q[1, 1].isnan().any()
    assert not q[0, 1:].isnan().any() and not q[2:].isnan().any()
    assert (q[2, 0] == 0).all() and not kc.isnan().any() and not vc.isnan().any()
    s = store_inputs(6, 4, 2, 64, 32, 16)
    s["pos"][1], s["pos"][3] = -1, 200
    q, kc, vc = call(OP, s, "cuda")
    want, err = store_oracle({**s, "pos": s["pos"].clamp(0, 199)}, True)
    for t in (1, 3):
        want[0][t, :, :32] = NAN
        b, o = int(s["slots"][t]) // 16, int(s["slots"][t]) % 16
        want[1][b, :, o, :32] = NAN
    assert_stored((q, kc, vc), want, err)


def test_far_slots():
    """A cache of over 2^32 values, whose last pages take the rows."""
    D, Hk, BS = 256, 8, 64
    blocks = (1 << 32) // (Hk * BS * D) + 3
    s = store_inputs(70, 8, Hk, D, D, BS, blocks=4, slots=torch.arange(70) + 4 * BS - 70)
    kc = torch.empty(blocks, Hk, BS, D, dtype=FP8, device="cuda")
    vc = torch.empty(blocks, Hk, D, BS, dtype=FP8, device="cuda")
    tail_k, tail_v = s["kc"].to(FP8), s["vc"].to(FP8)
    kc[-4:], vc[-4:] = tail_k.cuda(), tail_v.cuda()
    s.update(kc=tail_k, vc=tail_v)
    far = (s["slots"] + (blocks - 4) * BS).cuda()
    q, kc, vc = call(OP, s, "cuda", change=dict(k_cache=kc, v_cache=vc, slot_mapping=far))
    assert_stored((q, kc[-4:], vc[-4:]), *store_oracle(s, True))


@pytest.mark.parametrize("T", [8, 1200])
@torch.inference_mode()  # engines capture in it: outside, none could behind them
def test_captured(T):
    """A captured call follows its inputs, on a stream of its own."""
    s = store_inputs(T, 8, 2, 128, 64, 32, True, slots=torch.arange(T))
    args = {}

    def keep(*a):
        args["a"] = a
        return OP(*a)

    call(keep, s, "cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        OP(*args["a"])
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = OP(*args["a"])
    torch.cuda.current_stream().wait_stream(side)
    q, kc, vc, pos, slots = (args["a"][i] for i in (0, 6, 7, 8, 10))
    for seed in range(3):
        new = store_inputs(T, 8, 2, 128, 64, 32, True, seed=seed)
        q.copy_(call(lambda q, *_: q, new, "cuda")[0])
        pos.copy_(new["pos"])
        slots.copy_(torch.roll(slots, 7))
        graph.replay()
        got = (out.clone(), kc.clone(), vc.clone())
        kc.zero_(), vc.zero_()
        want = OP(*args["a"])
        torch.cuda.synchronize()
        assert torch.equal(got[0], want)
        at = slots.long()
        assert torch.equal(got[1].float()[at // 32, :, at % 32],
                           kc.float()[at // 32, :, at % 32])
        assert torch.equal(got[2].float()[at // 32, :, :, at % 32],
                           vc.float()[at // 32, :, :, at % 32])
