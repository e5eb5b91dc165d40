"""Two operators of a decode step or a prompt portion, and what they are measured by.

``store``: the RMS norm of every query and key head, the rotation, and the append of
keys and values to the paged cache. ``prefix``: decode attention of a batch whose
sequences share prefixes, such as a system prompt or a document that many requests ask
about. Head layouts are those of the repository's dense stacks and of its families with
head norms; caches are paged, K by rows and V transposed, in bf16 or in fp8 with a
scale; pages are shuffled and lengths ragged, as continuous batching leaves them.
"""

import math

import torch

own = False

DEV = "cuda"
FP8 = torch.float8_e4m3fn
FP8_MAX = 448.0
EPS = 1e-6
# query heads, key/value heads, head width
HEADS = {
    "14/2x64": (14, 2, 64),
    "64/8x64": (64, 8, 64),
    "32/8x128": (32, 8, 128),
    "32/4x128": (32, 4, 128),
    "64/8x128": (64, 8, 128),
    "16/2x256": (16, 2, 256),
}


def _store(name, heads, tokens, batch, rot, neox, fp8, page):
    return {"name": name, "op": "store", "heads": heads, "tokens": tokens,
            "batch": batch, "rot": rot, "neox": neox, "fp8": fp8, "page": page}


def _prefix(name, heads, batch, groups, prefix, suffix, fp8, page, alone=0, window=-1,
            softcap=0.0, sinks=False):
    return {"name": name, "op": "prefix", "heads": heads, "batch": batch,
            "groups": groups, "prefix": prefix, "suffix": suffix, "fp8": fp8,
            "page": page, "alone": alone, "window": window, "softcap": softcap,
            "sinks": sinks}


def listed():
    return [
        # a decode step of one request
        _store("store_one", "32/8x128", 1, 1, 128, True, False, 32),
        # a decode step of a full batch into an fp8 cache
        _store("store_batch_fp8", "64/8x128", 200, 200, 128, True, True, 32),
        # portions of three prompts, interleaved pairs on half of the head
        _store("store_interleaved", "32/4x128", 1111, 3, 64, False, False, 16),
        # wide heads of which a quarter is rotated, an odd number of tokens
        _store("store_wide_fp8", "16/2x256", 5003, 2, 64, True, True, 64),
        # a whole budget of prompt tokens
        _store("store_prompt", "32/8x128", 8192, 4, 128, True, False, 32),
        # few requests with one short system prompt
        _prefix("prefix_few", "14/2x64", 4, 1, 700, 60, False, 16),
        # chats behind a system prompt
        _prefix("prefix_chat", "32/8x128", 48, 1, 2001, 1000, False, 32),
        # questions about one long document
        _prefix("prefix_document", "32/8x128", 8, 1, 100000, 500, False, 32),
        # several system prompts, rows that share nothing, a sink in every head
        _prefix("prefix_groups", "64/8x64", 100, 5, 5000, 900, False, 64, alone=7,
                sinks=True),
        # many short answers behind a prompt of examples
        _prefix("prefix_batch", "32/8x128", 256, 1, 8000, 600, False, 32),
        # a long context in fp8 and long answers
        _prefix("prefix_long_fp8", "64/8x128", 64, 1, 60000, 4000, True, 32),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    page = rng.choice([16, 32, 64])
    fp8 = rng.random() < 0.4
    if rng.random() < 0.45:
        heads = rng.choice(sorted(HEADS))
        dim = HEADS[heads][2]
        tokens = _log(rng, 1, 8000)
        batch = tokens if rng.random() < 0.4 and tokens <= 256 else min(
            tokens, rng.randint(1, 6))
        c = _store("", heads, tokens, batch, rng.choice([dim, dim // 2, dim // 4]),
                   rng.random() < 0.6, fp8, page)
    else:
        heads = rng.choice([h for h in sorted(HEADS) if HEADS[h][2] <= 128])
        batch = _log(rng, 2, 256)
        groups = rng.choice([1, 1, 1, rng.randint(1, max(1, min(8, batch // 2)))])
        kv = HEADS[heads][1] * HEADS[heads][2] * batch
        most = (1 << 31) // kv  # tokens a row that the longest plain pass allows
        prefix = _log(rng, 64, max(128, min(80000, int(most * 0.7))))
        suffix = _log(rng, 1, max(2, min(4000, int(most * 0.3))))
        c = _prefix("", heads, batch, groups, prefix, suffix, fp8, page,
                    alone=rng.choice([0, 0, min(batch // 4, 9)]),
                    window=rng.choice([-1, -1, -1, rng.randint(1, prefix + suffix)]),
                    softcap=rng.choice([0.0, 0.0, 0.0, 30.0]),
                    sinks=rng.random() < 0.3)
    del c["name"]
    return c


def _scales(case):
    return (0.043, 0.027) if case["fp8"] else (1.0, 1.0)


def _cache(gen, pages, hk, page, dim, fp8, scales):
    """Normed keys and values of a filled cache."""
    out = []
    for shape, s in (((pages, hk, page, dim), scales[0]),
                     ((pages, hk, dim, page), scales[1])):
        x = torch.randn(shape, generator=gen, device=DEV, dtype=torch.bfloat16)
        out.append((x.float() / s).clamp(-FP8_MAX, FP8_MAX).to(FP8) if fp8 else x)
    return out


def _split(total, parts, rng):
    """`total` tokens in `parts` ragged portions of one token at least."""
    cuts = torch.randperm(total - 1, generator=rng)[:parts - 1].sort().values + 1
    ends = [0] + cuts.tolist() + [total]
    return [b - a for a, b in zip(ends, ends[1:])]


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rng = torch.Generator().manual_seed(seed)
    if case["op"] == "store":
        return _prepare_store(case, gen, rng)
    return _prepare_prefix(case, gen, rng)


def _prepare_store(case, gen, rng):
    hq, hk, dim = HEADS[case["heads"]]
    T, B, page, rot = case["tokens"], case["batch"], case["page"], case["rot"]
    # rows of the fused projection, which every pass finds as it left them
    rows = torch.randn(T, (hq + 2 * hk) * dim, generator=gen, device=DEV,
                       dtype=torch.bfloat16)
    q, k, v = (x.view(T, -1, dim) for x in rows.split([hq * dim, hk * dim, hk * dim], 1))
    weights = [(1 + 0.2 * torch.randn(dim, generator=gen, device=DEV)).bfloat16()
               for _ in range(2)]
    most = 40000
    inv = 10000.0 ** (-torch.arange(0, rot, 2, device=DEV, dtype=torch.float64) / rot)
    angle = torch.arange(most, device=DEV, dtype=torch.float64)[:, None] * inv
    table = torch.cat([angle.cos(), angle.sin()], -1).float()
    # each portion goes behind a context of its own, into pages of its own; a
    # batch that a graph pads has rows without a slot
    portions = _split(T, B, rng)
    starts = torch.randint(0, most - T, (B,), generator=rng).tolist()
    counts = [(s % page + n + page - 1) // page for s, n in zip(starts, portions)]
    ids = torch.randperm(T // page + 2 * B, generator=rng)
    pos, slots, at = [], [], 0
    for s, n, c in zip(starts, portions, counts):
        i = torch.arange(n)
        pos.append(s + i)
        slots.append(ids[at + (s % page + i) // page] * page + (s + i) % page)
        at += c
    slots = torch.cat(slots)
    if B == T and T > 8:
        slots[T - T // 8:] = -1
    scales = _scales(case)
    kc, vc = _cache(gen, len(ids), hk, page, dim, case["fp8"], scales)
    return {"case": case, "q": q, "k": k, "v": v, "qw": weights[0], "kw": weights[1],
            "kc": kc, "vc": vc, "pos": torch.cat(pos).to(torch.int32).to(DEV),
            "table": table, "slots": slots.to(DEV), "scales": scales}


def _lengths(case, rng):
    """Each row's group (-1: none), the groups' prefixes, the rows' lengths."""
    B, N, alone = case["batch"], case["groups"], case["alone"]
    group = torch.cat([torch.arange(B - alone) % N, torch.full((alone,), -1)])
    group = group[torch.randperm(B, generator=rng)]
    prefix = [case["prefix"]] + torch.randint(
        max(1, case["prefix"] // 8), case["prefix"] + 1, (N - 1,),
        generator=rng).tolist()
    suffix = torch.randint(1, case["suffix"] + 1, (B,), generator=rng)
    own_prefix = torch.tensor(prefix + [0])[group]
    return group, prefix, own_prefix + suffix


def _prepare_prefix(case, gen, rng):
    hq, hk, dim = HEADS[case["heads"]]
    B, page = case["batch"], case["page"]
    group, prefix, lens = _lengths(case, rng)
    shared = [p // page for p in prefix] + [0]  # whole pages only can be shared
    firsts = [0]
    for n in shared:
        firsts.append(firsts[-1] + n)
    need = [(n + page - 1) // page for n in lens.tolist()]
    total = firsts[-1] + sum(n - shared[g] for n, g in zip(need, group.tolist()))
    ids = torch.randperm(total, generator=rng).to(torch.int32)
    tables = torch.zeros(B, max(need), dtype=torch.int32)
    at = firsts[-1]
    for b, (n, g) in enumerate(zip(need, group.tolist())):
        s = shared[g]
        tables[b, :s] = ids[firsts[g]:firsts[g] + s]
        tables[b, s:n] = ids[at:at + n - s]
        at += n - s
    scales = _scales(case)
    kc, vc = _cache(gen, total, hk, page, dim, case["fp8"], scales)
    # rows of a prefix that share its whole pages share its last tokens too
    for g, p in enumerate(prefix):
        rows = (group == g).nonzero().view(-1).tolist()
        if p % page and len(rows) > 1:
            to = tables[rows[1:], p // page].long().to(DEV)
            src = int(tables[rows[0], p // page])
            for c, bytes_of in ((kc, lambda c: c.view(torch.uint8)[:, :, :p % page]),
                                (vc, lambda c: c.view(torch.uint8)[
                                    ..., :p % page * c.element_size()])):
                part = bytes_of(c)
                part[to] = part[src].clone()
    q = 2 * torch.randn(B, hq, dim, generator=gen, device=DEV)
    sinks = torch.randn(hq, generator=gen, device=DEV) if case["sinks"] else None
    return {"case": case, "q": q.bfloat16(), "kc": kc, "vc": vc,
            "tables": tables.to(DEV), "lens": lens.to(torch.int32).to(DEV),
            "group": group.to(torch.int32).to(DEV),
            "prefix": torch.tensor(prefix, dtype=torch.int32, device=DEV),
            "sinks": sinks, "scale": dim ** -0.5, "scales": scales}


def run(state):
    return run_store(state) if state["case"]["op"] == "store" else run_prefix(state)


def run_store(s):
    if own:
        from parallax_amd import ops
        q = ops.qk_norm_rope_and_cache(
            s["q"], s["k"], s["v"], s["qw"], s["kw"], EPS, s["kc"], s["vc"], s["pos"],
            s["table"], s["slots"], is_neox=s["case"]["neox"], k_scale=s["scales"][0],
            v_scale=s["scales"][1])
    else:
        q = plain_store(s)
    return {"q": q, "k_cache": s["kc"], "v_cache": s["vc"]}


def plain_store(s):
    neox = s["case"]["neox"]
    table = s["table"][s["pos"].long()][:, None]
    rot = table.shape[-1]
    c, t = table[..., :rot // 2], table[..., rot // 2:]

    def turned(x, w):
        x = x.float()
        y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
        a, b = (y[..., :rot // 2], y[..., rot // 2:rot]) if neox else (
            y[..., 0:rot:2], y[..., 1:rot:2])
        z = (a * c - b * t, b * c + a * t)
        z = torch.cat(z, -1) if neox else torch.stack(z, -1).flatten(-2)
        return torch.cat([z, y[..., rot:]], -1)

    def held(x, cache, scale):  # as the cache's bytes
        if cache.dtype == FP8:
            return (x / scale).clamp(-FP8_MAX, FP8_MAX).to(FP8).view(torch.uint8)
        return x.to(cache.dtype).view(torch.int16)

    kc, vc = s["kc"], s["vc"]
    page = kc.shape[2]
    stored = s["slots"] >= 0
    slots = s["slots"][stored]
    k = held(turned(s["k"], s["kw"])[stored], kc, s["scales"][0])
    v = held(s["v"].float()[stored], vc, s["scales"][1])
    kc.view(k.dtype)[slots // page, :, slots % page] = k
    vc.view(v.dtype)[slots // page, :, :, slots % page] = v
    return turned(s["q"], s["qw"]).to(s["q"].dtype)


def run_prefix(s):
    if own:
        from parallax_amd import ops
        c = s["case"]
        return ops.shared_prefix_attention_decode(
            s["q"], s["kc"], s["vc"], s["tables"], s["lens"], s["group"], s["prefix"],
            s["scale"], sliding_window=c["window"], softcap=c["softcap"],
            sinks=s["sinks"], k_scale=s["scales"][0], v_scale=s["scales"][1])
    return plain_prefix(s)


def plain_prefix(s):
    """Every row over its own pages, all rows at once."""
    case, q, kc, vc = s["case"], s["q"], s["kc"], s["vc"]
    B, hq, dim = q.shape
    hk = kc.shape[1]
    tables = s["tables"].long()
    bits = torch.uint8 if case["fp8"] else torch.int16
    k = kc.view(bits)[tables].view(kc.dtype).transpose(1, 2).float()
    k = k.reshape(B * hk, -1, dim) * s["scales"][0]
    x = q.float().reshape(B * hk, hq // hk, dim) * s["scale"]
    z = torch.bmm(k, x.transpose(1, 2).contiguous()).transpose(1, 2)
    del k
    z = z.reshape(B, hq, -1)
    if case["softcap"] > 0:
        z = case["softcap"] * torch.tanh(z / case["softcap"])
    at = torch.arange(z.shape[-1], device=DEV)[None, None]
    lens = s["lens"].long()[:, None, None]
    seen = at < lens
    if case["window"] > 0:
        seen = seen & (at >= lens - case["window"])
    z = z.masked_fill(~seen, -math.inf)
    top = z.amax(-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(z - top)
    total = p.sum(-1, keepdim=True)
    if s["sinks"] is not None:
        total = total + torch.exp(s["sinks"].float()[None, :, None] - top)
    v = vc.view(bits)[tables].view(vc.dtype).permute(0, 2, 1, 4, 3).float()
    v = v.reshape(B * hk, -1, dim)
    o = torch.bmm(p.reshape(B * hk, hq // hk, -1), v).reshape(B, hq, dim)
    return (o * s["scales"][1] / total.clamp(min=1e-30)).to(q.dtype)


def exact(case, seed):
    s = prepare(case, seed)
    return exact_store(s) if case["op"] == "store" else exact_prefix(s)


def exact_store(s):
    rot = s["table"].shape[1]
    half = rot // 2
    i = torch.arange(half, device=DEV)
    one, two = (i, i + half) if s["case"]["neox"] else (2 * i, 2 * i + 1)
    angle = s["table"].double()[s["pos"].long()].unsqueeze(1)

    def of(x, w):
        x = x.double()
        out = x / torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS)
        out = out * w.double()
        turned = out.clone()
        turned[..., one] = out[..., one] * angle[..., :half] - out[..., two] * angle[
            ..., half:]
        turned[..., two] = out[..., two] * angle[..., :half] + out[..., one] * angle[
            ..., half:]
        return turned

    page = s["kc"].shape[2]
    slots = s["slots"].cpu()
    rows = (slots >= 0).nonzero().view(-1)
    block, place = (slots[rows] // page).to(DEV), (slots[rows] % page).to(DEV)
    rows = rows.to(DEV)
    k, v = of(s["k"], s["kw"]) / s["scales"][0], s["v"].double() / s["scales"][1]
    if s["case"]["fp8"]:
        k, v = k.clamp(-FP8_MAX, FP8_MAX), v.clamp(-FP8_MAX, FP8_MAX)
    kc, vc = s["kc"].float().double(), s["vc"].float().double()
    kc[block, :, place] = k[rows]
    vc[block, :, :, place] = v[rows]
    return {"q": of(s["q"], s["qw"]), "k_cache": kc, "v_cache": vc}


def exact_prefix(s):
    case = s["case"]
    B, hq, dim = s["q"].shape
    hk, page = s["kc"].shape[1:3]
    out = torch.zeros(B, hq, dim, dtype=torch.float64, device=DEV)
    for b, n in enumerate(s["lens"].tolist()):
        lo = max(0, n - case["window"]) if case["window"] > 0 else 0
        ids = s["tables"][b, lo // page:(n + page - 1) // page].long()
        k = s["kc"].view(torch.uint8)[ids].view(s["kc"].dtype)
        v = s["vc"].view(torch.uint8)[ids].view(s["vc"].dtype)
        skip, count = lo % page, n - lo
        k = k.double().movedim(1, 0).reshape(hk, -1, dim)[:, skip:skip + count]
        v = v.double().movedim(1, 0).transpose(2, 3).reshape(hk, -1, dim)[
            :, skip:skip + count]
        x = s["q"][b].double().view(hk, hq // hk, dim)
        z = torch.matmul(x, k.transpose(1, 2).contiguous()) * (
            s["scale"] * s["scales"][0])
        if case["softcap"] > 0:
            z = torch.tanh(z / case["softcap"]) * case["softcap"]
        top = z.max(-1, keepdim=True).values
        if s["sinks"] is not None:
            sink = s["sinks"].double().view(hk, hq // hk, 1)
            top = torch.maximum(top, sink)
        p = torch.exp(z - top)
        total = p.sum(-1, keepdim=True)
        if s["sinks"] is not None:
            total = total + torch.exp(sink - top)
        out[b] = (torch.matmul(p / total, v) * s["scales"][1]).view(hq, dim)
    return out


def work(case):
    hq, hk, dim = HEADS[case["heads"]]
    size = 1 if case["fp8"] else 2
    if case["op"] == "store":
        T = case["tokens"]
        values = T * (2 * hq + 2 * hk) * dim * 2 + T * 2 * hk * dim * size
        return {"bytes": values + T * (case["rot"] * 4 + 12) + 4 * dim,
                "flops": T * (hq + hk) * dim * 8}
    # the lengths of seed 0, which other seeds' are like
    group, prefix, lens = _lengths(case, torch.Generator().manual_seed(0))
    w = case["window"]
    lo = (lens - w).clamp(min=0) if w > 0 else torch.zeros_like(lens)
    own_prefix = torch.tensor(prefix + [0])[group]
    tokens = int((lens - torch.maximum(lo, own_prefix)).sum())
    for g, p in enumerate(prefix):
        if (group == g).any():
            tokens += max(0, p - int(lo[group == g].min()))
    return {"bytes": tokens * hk * dim * 2 * size + 4 * case["batch"] * hq * dim,
            "flops": 4 * hq * dim * int((lens - lo).sum())}
