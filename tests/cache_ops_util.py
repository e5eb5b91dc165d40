"""Inputs and 64-bit results of the operators around a shared paged cache. Everything
is made on the CPU; what an operator must not read holds NaN."""

import math

import torch

FP8 = torch.float8_e4m3fn
NAN = float("nan")


# -- head norms, rotation, append --------------------------------------------------------


def store_inputs(T, Hq, Hk, D, rot, BS, fp8=False, seed=0, head_gap=0, row_gap=0,
                 slots=None, blocks=None, positions=200):
    """q, k and v as rows of a fused projection: heads head_gap values apart, rows
    row_gap values longer than their heads."""
    g = torch.Generator().manual_seed(seed)
    W = D + head_gap
    rows = torch.randn(T, (Hq + 2 * Hk) * W + row_gap, generator=g) * torch.exp(
        torch.randn(T, 1, generator=g))
    heads = rows[:, :(Hq + 2 * Hk) * W].view(T, Hq + 2 * Hk, W)[..., :D].bfloat16()
    full = torch.full((T, (Hq + 2 * Hk) * W + row_gap), NAN).bfloat16()
    full[:, :(Hq + 2 * Hk) * W].view(T, Hq + 2 * Hk, W)[..., :D] = heads
    if blocks is None:
        blocks = (T + BS - 1) // BS + 3
    if slots is None:
        slots = torch.randperm(blocks * BS, generator=g)[:T]
    scales = (0.037, 0.11) if fp8 else (1.0, 1.0)
    old = [torch.randn(s, generator=g) for s in
           ((blocks, Hk, BS, D), (blocks, Hk, D, BS))]
    kc, vc = (x.to(FP8 if fp8 else torch.bfloat16) for x in old)
    return dict(
        full=full, T=T, Hq=Hq, Hk=Hk, D=D, W=W,
        qw=(1 + 0.3 * torch.randn(D, generator=g)).bfloat16(),
        kw=(1 + 0.3 * torch.randn(D, generator=g)).bfloat16(), eps=1e-5, kc=kc, vc=vc,
        pos=torch.randint(0, positions, (T,), generator=g, dtype=torch.int32),
        table=torch.randn(positions, rot, generator=g), slots=slots, scales=scales)


def store_views(s, device):
    """The operator's arguments on a device, with the strides of the fused rows."""
    full = s["full"].to(device)
    heads = full[:, :(s["Hq"] + 2 * s["Hk"]) * s["W"]].view(
        s["T"], s["Hq"] + 2 * s["Hk"], s["W"])[..., :s["D"]]
    q, k, v = heads.split([s["Hq"], s["Hk"], s["Hk"]], 1)
    to = {n: s[n].to(device) for n in ("qw", "kw", "kc", "vc", "pos", "table", "slots")}
    return q, k, v, to


def store_oracle(s, neox):
    """(q, k_cache, v_cache) in 64 bits, before their rounding, and how far fp32
    arithmetic may take the normed and rotated values from them."""
    q, k, v, to = store_views(s, "cpu")
    D, rot = s["D"], to["table"].shape[1]
    cs = to["table"].double()[to["pos"].long()][:, None]
    i = torch.arange(rot // 2)
    one, two = (i, i + rot // 2) if neox else (2 * i, 2 * i + 1)

    def turn(x, w):
        y = x.double()
        y = y / ((y * y).mean(-1, keepdim=True) + s["eps"]).sqrt() * w.double()
        z, size = y.clone(), y.abs().clone()
        a, b, c, t = y[..., one], y[..., two], cs[..., :rot // 2], cs[..., rot // 2:]
        z[..., one], z[..., two] = a * c - b * t, b * c + a * t
        size[..., one] = (a * c).abs() + (b * t).abs()
        size[..., two] = (b * c).abs() + (a * t).abs()
        # a sum of D squares is off by D 2^-24 of itself at most, its root by half of
        # that; eight more operations of half a step each
        return z, size * (D / 2 + 8) * 2.0 ** -24

    zq, eq = turn(q, to["qw"])
    zk, ek = turn(k, to["kw"])
    kc, vc = to["kc"].double(), to["vc"].double()
    kerr, verr = torch.zeros_like(kc), torch.zeros_like(vc)
    BS = kc.shape[2]
    fp8 = s["kc"].dtype == FP8
    for t, slot in enumerate(to["slots"].tolist()):
        if 0 <= slot < kc.shape[0] * BS:
            b, o = slot // BS, slot % BS
            kc[b, :, o], kerr[b, :, o] = zk[t] / s["scales"][0], ek[t] / s["scales"][0]
            vc[b, :, :, o] = v[t].double() / s["scales"][1]
            # times the inverse scale: two roundings
            verr[b, :, :, o] = vc[b, :, :, o].abs() * 2.0 ** -23
    if fp8:
        kc, vc = kc.clamp(-448, 448), vc.clamp(-448, 448)
        kerr += kc.abs() * 2.0 ** -23
    return (zq, kc, vc), (eq, kerr, verr)


def assert_stored(got, want, err):
    for x, y, e in zip(got, want, err):
        half = 2.0 ** -4 if x.dtype == FP8 else 2.0 ** -8
        least = 2.0 ** -10 if x.dtype == FP8 else 0.0  # half of e4m3's least step
        x = x.cpu().float().double()
        assert torch.equal(x.isnan(), y.isnan())
        # what fp32 is off by may move the value that is rounded
        bound = (y.abs() + e) * half + least + e
        off = torch.where(y.isnan() | (x == y), 0.0, (x - y).abs() - bound)
        assert (off <= 0).all(), (off.max(), x.flatten()[off.argmax()],
                                  y.flatten()[off.argmax()])


# -- decode over shared prefixes ---------------------------------------------------------


def prefix_inputs(Hq, Hk, D, BS, rows, prefix, fp8=False, seed=0, q_gap=0, spare=2,
                  sharp=1.0):
    """rows: (group, length) each; prefix: the groups' lengths. Every row has pages of
    its own for all of its tokens; only those that the operator reads hold numbers, and
    table entries past a row's end are no pages at all."""
    g = torch.Generator().manual_seed(seed)
    B = len(rows)
    need = [(max(n, 0) + BS - 1) // BS for _, n in rows]
    ids = torch.randperm(sum(need) + spare, generator=g).to(torch.int32)
    tables = torch.full((B, max(need + [1]) + 1), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        tables[b, :n] = ids[at:at + n]
        at += n
    NB = len(ids)
    k = torch.full((NB, Hk, BS, D), NAN)
    v = torch.full((NB, Hk, D, BS), NAN)
    seen = set()
    for b, (gr, n) in enumerate(rows):
        P = prefix[gr] if 0 <= gr < len(prefix) and 0 < prefix[gr] <= n else 0
        lo = P if P and gr in seen else 0
        if P:
            seen.add(gr)
        for t0 in range(lo // BS * BS, n, BS):
            a, e = max(lo, t0) - t0, min(n, t0 + BS) - t0
            page = int(tables[b, t0 // BS])
            k[page, :, a:e] = sharp * torch.randn(Hk, e - a, D, generator=g)
            v[page, :, :, a:e] = torch.randn(Hk, D, e - a, generator=g) + 0.3
    scales = (0.043, 0.027) if fp8 else (1.0, 1.0)
    if fp8:
        k, v = (k / scales[0]).clamp(-448, 448), (v / scales[1]).clamp(-448, 448)
    q = torch.randn(B, Hq * D + q_gap, generator=g).bfloat16()
    dtype = FP8 if fp8 else torch.bfloat16
    i32 = torch.int32
    return dict(
        q=q, shape=(B, Hq, D), kc=k.to(dtype), vc=v.to(dtype), tables=tables,
        lens=torch.tensor([n for _, n in rows], dtype=i32),
        group=torch.tensor([gr for gr, _ in rows], dtype=i32),
        prefix=torch.tensor(prefix, dtype=i32), scales=scales)


def prefix_call(fn, s, device, scale=None, **kw):
    B, Hq, D = s["shape"]
    q = s["q"].to(device)[:, :Hq * D].view(B, Hq, D) if B else s["q"].new_empty(
        B, Hq, D).to(device)
    a = [s[n].to(device) for n in ("kc", "vc", "tables", "lens", "group", "prefix")]
    return fn(q, *a, D ** -0.5 if scale is None else scale, k_scale=s["scales"][0],
              v_scale=s["scales"][1], **kw)


def prefix_oracle(s, scale=None, sliding_window=-1, softcap=0.0, sinks=None):
    """(result in 64 bits, the same weights over |v|)"""
    B, Hq, D = s["shape"]
    scale = D ** -0.5 if scale is None else scale
    Hk, BS = s["kc"].shape[1:3]
    out = torch.zeros(2, B, Hq, D, dtype=torch.float64)
    first = {}
    for b in range(B):
        L, g = int(s["lens"][b]), int(s["group"][b])
        P = int(s["prefix"][g]) if 0 <= g < len(s["prefix"]) else 0
        P = P if 0 < P <= L else 0
        if L <= 0:
            continue
        if P:
            first.setdefault(g, b)
        lo = max(0, L - sliding_window) if sliding_window > 0 else 0
        ks, vs = [], []
        for t0 in range(lo // BS * BS, L, BS):
            cut = min(max(P - t0, 0), BS) if P else 0  # of this page's tokens: shared
            for row, a, e in ((first.get(g, b), 0, cut), (b, cut, BS)):
                a, e = max(a, lo - t0), min(e, L - t0)
                if a < e:
                    page = int(s["tables"][row, t0 // BS])
                    ks.append(s["kc"][page][:, a:e].float().double())
                    vs.append(s["vc"][page][..., a:e].float().double())
        k = torch.cat(ks, 1) * s["scales"][0]
        v = torch.cat(vs, 2) * s["scales"][1]
        x = s["q"][b, :Hq * D].double().view(Hk, Hq // Hk, D)
        z = (x @ k.transpose(1, 2)).reshape(Hq, -1) * scale
        if softcap > 0:
            z = softcap * torch.tanh(z / softcap)
        if sinks is not None:
            z = torch.cat([z, sinks.double().cpu()[:, None]], 1)
        p = torch.softmax(z, 1)
        if sinks is not None:
            p = p[:, :-1]
        p = p.view(Hk, Hq // Hk, -1)
        for i, x in enumerate((v, v.abs())):
            out[i, b] = (p @ x.transpose(1, 2)).reshape(Hq, D)
    return out


def assert_attended(got, oracle, weights=2.0 ** -8):
    """weights: half a step of the type in which a kernel's weights meet the values.
    Beside it, fp32 scores are off by 128 2^-24 of sums of magnitudes up to 64 here:
    2^-11 of a weight; and the result is rounded."""
    want, size = oracle
    x = got.cpu().double()
    assert torch.isfinite(x).all()
    bound = size * (weights + 2.0 ** -11)
    bound = bound + (want.abs() + bound) * 2.0 ** -8
    off = (x - want).abs() - bound
    assert (off <= 0).all(), (float(off.max()), x.flatten()[off.argmax()],
                              want.flatten()[off.argmax()])
