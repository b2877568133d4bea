"""Rotary positions, a paged key-value cache, attention over it and eviction from it, as cases that can be timed and compared.

Four kinds of case:

  rope     ``capi.rope``: rotary positions of fp32 heads, half or interleaved pairs, all of a head or its first part.
  append   ``capi.rope_append``: the fused projection's output (queries, keys and values of every token, fp32) is rotated,
           the queries go to a buffer of their own, the keys and values into the pages of the cache in its type.
  attend   ``capi.paged_attention_q8_1``: one new token of every sequence against the pages of that sequence; ``weights``
           accumulates what every cached token was given, for eviction.
  evict    ``capi.kv_evict``: of every sequence and key-value head the tokens with the largest accumulated weight, the
           first and the last ones stay, in their order, in other pages or (``in_place``) at the front of their own.

Head counts are those of the decoders that the benchmark and the tests know (32 heads of 128 on a hidden size of 4096, 64 on
8192), with shared key-value heads, and ragged ones.  Without ``own`` the same is computed with elementary operations in 32 bits
(angles in 64).
"""
import math
import random

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
SIZE = {"f16": 2, "bf16": 2, "e4m3": 1}
BASE = 10000.0
ORIGINAL = 4096  # positions that a scaled table was trained on
FACTOR = 16.0


def listed():
    return [
        # one token of one sequence enters the cache, far behind its start: the smallest call, all latency
        _append("append_m1", 1, 1, 32, 32, 128, 128, False, 16, "f16", 900, "none"),
        # a decode step of 48 sequences, shared heads, positions stretched
        _append("append_m48_gqa", 48, 48, 32, 8, 128, 128, False, 32, "bf16", 700, "yarn"),
        # a prefill chunk of three prompts, odd length, interleaved pairs in half of the head
        _append("append_chunk_4097", 4097, 3, 32, 8, 128, 64, True, 16, "f16", 100, "linear"),
        # rotary positions by themselves, ragged: heads of 80, a quarter of them rotated
        _rope("rope_2049x25x80", 2049, 25, 80, 20, True, 200000, "none"),
        # the queries of a long prefill chunk
        _rope("rope_8192x64x128", 8192, 64, 128, 128, False, 131072, "wavelength"),
        # one sequence of a few hundred tokens: all latency
        _attend("attend_m1_l700", 1, 32, 8, 128, 700, 16, "f16", 0, False, "slots"),
        # a batch of ragged sequences, every query head with its own keys
        _attend("attend_m16_mha", 16, 32, 32, 128, 2500, 16, "f16", 0, False, "heads"),
        # one very long sequence
        _attend("attend_m1_l131071", 1, 64, 8, 128, 131071, 64, "bf16", 0, False, "slots"),
        # a serving batch on an 8-bit cache
        _attend("attend_m64_e4m3", 64, 32, 8, 128, 5000, 32, "e4m3", 0, False, "slots"),
        # the same step with the weights that eviction goes by
        _attend("attend_m8_weights", 8, 32, 8, 128, 6001, 16, "f16", 0, True, "slots"),
        # a decode batch goes back under its budget, a page or two over it
        _evict("evict_m4_in_place", 4, 8, 128, 1100, 1024, 256, 4, 16, "f16", True),
        # a long prompt is cut down after its prefill
        _evict("evict_l100003", 1, 8, 128, 100003, 16000, 512, 4, 64, "bf16", False),
    ]


def _append(name, rows, seqs, q_heads, kv_heads, dim, rotary, interleaved, page, dtype, length, scaling):
    return {"name": name, "op": "append", "rows": rows, "seqs": seqs, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim,
            "rotary": rotary, "interleaved": interleaved, "page": page, "dtype": dtype, "length": length, "scaling": scaling,
            "layout": "slots"}


def _rope(name, rows, heads, dim, rotary, interleaved, far, scaling):
    return {"name": name, "op": "rope", "rows": rows, "heads": heads, "dim": dim, "rotary": rotary, "interleaved": interleaved,
            "far": far, "scaling": scaling}


def _attend(name, rows, q_heads, kv_heads, dim, length, page, dtype, window, weights, layout):
    return {"name": name, "op": "attend", "rows": rows, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "length": length,
            "page": page, "dtype": dtype, "window": window, "weights": weights, "layout": layout}


def _evict(name, rows, kv_heads, dim, length, keep, recent, sinks, page, dtype, in_place):
    return {"name": name, "op": "evict", "rows": rows, "kv_heads": kv_heads, "dim": dim, "length": length, "keep": keep,
            "recent": recent, "sinks": sinks, "page": page, "dtype": dtype, "in_place": in_place, "layout": "slots"}


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], even over the logarithm."""
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["append", "append", "rope", "attend", "attend", "attend", "attend", "evict", "evict"])
    dim = rng.choice([64, 80, 96, 128, 128, 256])
    rotary = rng.choice([dim, dim, dim // 2, 16])
    interleaved, scaling = rng.random() < 0.4, rng.choice(["none", "linear", "yarn", "wavelength", "ntk"])
    kv_heads, group = rng.choice([1, 2, 4, 5, 8, 32]), rng.choice([1, 2, 3, 4, 7, 8, 16])
    q_heads = min(128, kv_heads * group) // kv_heads * kv_heads
    page, layout = rng.choice([1, 16, 16, 24, 32, 64, 128]), rng.choice(["slots", "heads"])
    if op == "rope":
        heads = _spread(rng, 1, 64)
        rows = min(_spread(rng, 1, 16384), (8192 * 64 * 128) // (heads * dim))
        c = _rope("", max(1, rows), heads, dim, rotary, interleaved, _spread(rng, 128, 1 << 20), scaling)
    elif op == "append":
        rows = min(_spread(rng, 1, 8192), (4097 * 48 * 128) // ((q_heads + 2 * kv_heads) * dim))
        rows = max(1, rows)
        seqs = rows if rng.random() < 0.5 and rows <= 256 else rng.randint(1, min(rows, 7))
        length = max(1, min(_spread(rng, 1, 2000), (1 << 27) // (seqs * kv_heads * dim)))
        c = _append("", rows, seqs, q_heads, kv_heads, dim, rotary, interleaved, page, rng.choice(["f16", "bf16"]), length, scaling)
        c["layout"] = layout
    elif op == "attend":
        rows = _spread(rng, 1, 96)
        dtype = rng.choice(["f16", "f16", "bf16", "bf16", "e4m3"])
        length = max(1, min(_spread(rng, 1, 100000), (131071 * 8 * 128) // (rows * kv_heads * dim)))
        window = rng.choice([0, 0, 0, _spread(rng, 1, 4096)])
        c = _attend("", rows, q_heads, kv_heads, dim, length, page, dtype, window, rng.random() < 0.3, layout)
    else:
        rows = _spread(rng, 1, 24)
        length = max(8, min(_spread(rng, 16, 100000), (1 << 27) // (rows * kv_heads * dim)))
        keep = max(2, min(length, _spread(rng, 2, 16000)))
        recent = rng.randint(0, keep // 2)
        c = _evict("", rows, kv_heads, dim, length, keep, recent, rng.randint(0, min(8, keep - recent)), page,
                   rng.choice(["f16", "bf16"]), rng.random() < 0.4)
        c["layout"] = layout
    c.pop("name", None)
    return c


# ---- inputs ----------------------------------------------------------------------------------------------------
def _lengths(case):
    """Tokens that every sequence has in the cache: the first as many as the case says, the others fewer, by the case alone."""
    n = case["seqs"] if case["op"] == "append" else case["rows"]
    rng = random.Random(1000003 * n + case["length"])
    return [case["length"]] + [rng.randint(max(1, case["length"] // 4), case["length"]) for _ in range(n - 1)]


def _device():
    return torch.device("cuda", torch.cuda.current_device())


def _scaled(base, rotary, scaling):
    """Radians per position of every pair, and the factor of sine and cosine."""
    i = torch.arange(rotary // 2, dtype=torch.float64)
    if scaling == "ntk":
        base = base * FACTOR ** (rotary / max(rotary - 2, 1))
    inv = base ** (-2.0 * i / rotary)
    if scaling == "linear":
        return inv / FACTOR, 1.0
    if scaling == "yarn":
        def turns_at(turns):
            return rotary * math.log(ORIGINAL / (turns * 2 * math.pi)) / (2 * math.log(base))

        low, high = max(math.floor(turns_at(32.0)), 0), min(math.ceil(turns_at(1.0)), rotary - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        return inv / FACTOR * ramp + inv * (1 - ramp), 0.1 * math.log(FACTOR) + 1.0
    if scaling == "wavelength":
        share = ((ORIGINAL * inv / (2 * math.pi) - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return (1 - share) * inv / FACTOR + share * inv, 1.0
    return inv, 1.0


def _pool(gen, case, pages):
    """Keys and values [pages, slot, head, dim] as they lie in memory after some serving: stale values everywhere."""
    shape = (pages, case["page"], case["kv_heads"], case["dim"])
    if case["layout"] == "heads":
        shape = (shape[0], shape[2], shape[1], shape[3])
    got = []
    for _ in range(2):
        if case["dtype"] == "e4m3":
            t = torch.randn(shape, generator=gen, device=gen.device, dtype=torch.float16).mul_(16.0).to(DTYPES["e4m3"])
        else:
            t = torch.randn(shape, generator=gen, device=gen.device, dtype=DTYPES[case["dtype"]])
        got.append(t.transpose(1, 2) if case["layout"] == "heads" else t)
    return got


def _tables(gen, case, lengths, tables):
    """Page tables over distinct pages of one pool, in random order; entries behind a sequence's last page are -1."""
    need = [-(-n // case["page"]) for n in lengths]
    wide, total = max(need), tables * sum(need)
    order = torch.randperm(total + 3, generator=gen, device=gen.device).to(torch.int32)
    got, at = [], 0
    for _ in range(tables):
        pages = torch.arange(wide, device=gen.device)[None, :]
        n = torch.tensor(need, device=gen.device)[:, None]
        first = torch.cumsum(n, 0) - n
        got.append(torch.where(pages < n, order[(at + first + pages).clamp(max=total)], -1).to(torch.int32).contiguous())
        at += sum(need)
    return got, total + 3


def prepare(case, seed):
    gen = torch.Generator(device=_device())
    gen.manual_seed(seed)
    dev, op = gen.device, case["op"]
    s = {"case": case}
    if op in ("rope", "append"):
        s["inv"], s["mscale"] = _scaled(BASE, case["rotary"], case["scaling"])
        s["inv"] = s["inv"].to(dev)
        if own:
            from jjjetson_ops_b200 import capi

            s["table"], s["mscale"] = capi.rope_table(case["rotary"], BASE, case["scaling"], FACTOR, ORIGINAL, device=dev)
    if op == "rope":
        s["x"] = torch.randn((case["rows"], case["heads"], case["dim"]), generator=gen, device=dev)
        s["positions"] = torch.randint(0, case["far"], (case["rows"],), generator=gen, device=dev, dtype=torch.int32)
        s["out"] = torch.empty_like(s["x"])
        return s
    lengths = _lengths(case)
    if op == "append":
        rows, seqs = case["rows"], case["seqs"]
        t = torch.arange(rows, device=dev)
        s["seqs"] = (t * seqs // rows).to(torch.int32)
        first = -((-torch.arange(seqs, device=dev) * rows) // seqs)  # the first row of every sequence
        held = torch.tensor(lengths, device=dev)  # tokens that are in the cache before
        s["index"] = (t - first[s["seqs"].long()] + held[s["seqs"].long()]).to(torch.int32)
        s["positions"] = s["index"]
        counts = torch.bincount(s["seqs"].long(), minlength=seqs)
        (s["pages"],), pool = _tables(gen, case, (held + counts).tolist(), 1)
        s["k"], s["v"] = _pool(gen, case, pool)
        s["qkv"] = torch.randn((rows, (case["q_heads"] + 2 * case["kv_heads"]) * case["dim"]), generator=gen, device=dev)
        s["q"] = torch.empty((rows, case["q_heads"], case["dim"]), device=dev)
        return s
    s["scale"] = 1.0 / 16.0 if case["dtype"] == "e4m3" else 1.0
    s["lens"] = torch.tensor(lengths, device=dev, dtype=torch.int32)
    s["S"] = case["length"]
    if op == "attend":
        (s["pages"],), pool = _tables(gen, case, lengths, 1)
        s["k"], s["v"] = _pool(gen, case, pool)
        s["q"] = torch.randn((case["rows"], case["q_heads"], case["dim"]), generator=gen, device=dev).mul_(1.5)
        s["out"] = torch.empty_like(s["q"])
        s["weights"] = None
        if case["weights"]:
            s["weights"] = torch.rand((case["rows"], case["kv_heads"], s["S"]), generator=gen, device=dev)
        if own:
            from jjjetson_ops_b200 import capi

            s["ws"] = capi.paged_attention_workspace(s["q"], s["k"], s["pages"], weights=case["weights"])
        return s
    tables, pool = _tables(gen, case, lengths, 1 if case["in_place"] else 2)
    s["pages"], s["new_pages"] = tables[0], tables[-1]
    s["k"], s["v"] = _pool(gen, case, pool)
    # weights as decode steps leave them: a few tokens carry most, many have next to nothing, some exactly nothing
    w = torch.rand((case["rows"], case["kv_heads"], s["S"]), generator=gen, device=dev)
    s["weights"] = torch.where(w < 0.02, 0.0, (w * 16).floor() / 16 + w.pow(24) * 8)
    s["new_weights"] = s["weights"] if case["in_place"] else torch.empty_like(s["weights"])
    s["new_lens"] = torch.empty_like(s["lens"])
    s["kept"] = torch.empty((case["rows"], case["kv_heads"], case["keep"]), device=dev, dtype=torch.int32)
    return s


# ---- one pass ---------------------------------------------------------------------------------------------------
def run(state):
    return {"rope": _run_rope, "append": _run_append, "attend": _run_attend, "evict": _run_evict}[state["case"]["op"]](state)


def _rotate(x, positions, inv, mscale, rotary, interleaved):
    angle = positions.to(torch.float64)[:, None, None] * inv
    cos, sin = (angle.cos() * mscale).to(torch.float32), (angle.sin() * mscale).to(torch.float32)
    part = x[..., :rotary]
    if interleaved:
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = part[..., : rotary // 2], part[..., rotary // 2 :]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, x[..., rotary:]), -1)


def _run_rope(s):
    c = s["case"]
    if own:
        from jjjetson_ops_b200 import capi

        return capi.rope(s["x"], s["positions"], s["table"], interleaved=c["interleaved"], mscale=s["mscale"], out=s["out"])
    return _rotate(s["x"], s["positions"], s["inv"], s["mscale"], c["rotary"], c["interleaved"])


def _run_append(s):
    c = s["case"]
    if own:
        from jjjetson_ops_b200 import capi

        capi.rope_append(s["qkv"], s["positions"], s["table"], s["k"], s["v"], s["pages"], s["index"], seqs=s["seqs"],
                         q_out=s["q"], interleaved=c["interleaved"], mscale=s["mscale"])
        return s["q"], s["k"], s["v"]
    x = s["qkv"].view(c["rows"], c["q_heads"] + 2 * c["kv_heads"], c["dim"])
    hq, hk = c["q_heads"], c["kv_heads"]
    turned = _rotate(x[:, : hq + hk], s["positions"], s["inv"], s["mscale"], c["rotary"], c["interleaved"])
    index = s["index"].long()
    page, slot = s["pages"][s["seqs"].long(), index // c["page"]].long(), index % c["page"]
    s["k"][page, slot] = turned[:, hq:].to(s["k"].dtype)
    s["v"][page, slot] = x[:, hq + hk :].to(s["v"].dtype)
    return turned[:, :hq], s["k"], s["v"]


def _run_attend(s):
    c = s["case"]
    if own:
        from jjjetson_ops_b200 import capi

        capi.paged_attention_q8_1(s["q"], s["k"], s["v"], s["pages"], s["lens"], window=c["window"], k_scale=s["scale"],
                                  v_scale=s["scale"], out=s["out"], want_q8=False, weights=s["weights"], ws=s["ws"])
        return s["out"], s["weights"]
    B, hk, g, d, S = c["rows"], c["kv_heads"], c["q_heads"] // c["kv_heads"], c["dim"], s["S"]
    at = torch.arange(S, device=s["q"].device)
    page, slot = s["pages"][:, at // c["page"]].clamp(min=0).long(), at % c["page"]
    lens = s["lens"].long()[:, None]
    there = (at < lens) & ((at >= lens - c["window"]) if c["window"] else (at >= 0))
    there = there[:, None, None, :]
    k, v = (t[page, slot].to(torch.float32).mul_(s["scale"]).permute(0, 2, 1, 3) for t in (s["k"], s["v"]))
    logits = torch.matmul(s["q"].view(B, hk, g, d), k.transpose(-1, -2)) * (1.0 / math.sqrt(d))
    logits = logits.masked_fill(~there, -math.inf)
    p = torch.exp(logits - logits.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    out = torch.matmul(p, v).view(B, hk * g, d)
    if s["weights"] is not None:
        s["weights"] += p.sum(2)
    return out, s["weights"]


def _run_evict(s):
    c = s["case"]
    if own:
        from jjjetson_ops_b200 import capi

        capi.kv_evict(s["weights"], s["lens"], s["k"], s["v"], s["pages"], c["keep"], recent=c["recent"], sinks=c["sinks"],
                      new_page_table=None if c["in_place"] else s["new_pages"], new_weights=s["new_weights"],
                      new_lens=s["new_lens"], kept=s["kept"])
        return s["k"], s["v"], s["new_weights"], s["new_lens"], s["kept"]
    S, keep = s["S"], c["keep"]
    at, n = torch.arange(S, device=s["lens"].device), s["lens"].long()[:, None, None]
    key = torch.where((at < c["sinks"]) | (at >= n - c["recent"]), math.inf, s["weights"])
    key = torch.where(at < n, key, -math.inf)
    best = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :keep]
    kept = torch.sort(torch.where(best < n, best, S), dim=-1).values  # in their order, S where there are fewer
    full = kept < S
    source = torch.where(full, kept, 0)
    heads = torch.arange(c["kv_heads"], device=at.device)[None, :, None]
    row, head, to = torch.where(full)
    seq = torch.arange(c["rows"], device=at.device)[:, None, None]
    page, slot = s["pages"][seq, source // c["page"]].long(), source % c["page"]
    new_page, new_slot = s["new_pages"][row, to // c["page"]].long(), to % c["page"]
    for t in (s["k"], s["v"]):
        t[new_page, new_slot, head] = t[page, slot, heads][full]
    w = torch.where(full, s["weights"].gather(-1, source), 0.0)
    s["new_weights"].zero_()
    s["new_weights"][..., :keep] = w
    s["new_lens"].copy_(s["lens"].clamp(max=keep))
    s["kept"].copy_(torch.where(full, kept, -1))
    return s["k"], s["v"], s["new_weights"], s["new_lens"], s["kept"]


# ---- what a pass cannot do without --------------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "rope":
        n = case["rows"] * case["heads"]
        return {"bytes": 8 * n * case["dim"] + 4 * case["rows"] + 4 * case["rotary"], "flops": 3 * n * case["rotary"]}
    size = SIZE[case["dtype"]] * case["dim"] * case["kv_heads"]  # of one token's keys
    if op == "append":
        rows, hq, hk = case["rows"], case["q_heads"], case["kv_heads"]
        moved = 4 * (hq + 2 * hk) * case["dim"] + 4 * hq * case["dim"] + 2 * size + 16
        return {"bytes": rows * moved + 4 * case["rotary"], "flops": 3 * rows * (hq + hk) * case["rotary"]}
    lengths = _lengths(case)
    if op == "attend":
        seen = sum(min(n, case["window"] or n) for n in lengths)
        moved = 2 * size * seen + 8 * case["rows"] * case["q_heads"] * case["dim"] + 4 * sum(-(-n // case["page"]) for n in lengths)
        moved += 8 * case["kv_heads"] * seen if case["weights"] else 0
        return {"bytes": moved, "flops": 4 * seen * case["q_heads"] * case["dim"]}
    kept = sum(min(n, case["keep"]) for n in lengths)
    moving = sum(min(n, case["keep"]) - case["sinks"] for n in lengths if n > case["keep"]) if case["in_place"] else kept
    moved = 4 * size * max(moving, 0) + 4 * case["kv_heads"] * (sum(lengths) + case["rows"] * (case["length"] + case["keep"]))
    return {"bytes": moved, "flops": 0}


# ---- the definition, in 64 bits -------------------------------------------------------------------------------------
def _frequencies(case):
    """One pair after the other."""
    r, base, how = case["rotary"], BASE, case["scaling"]
    if how == "ntk":
        base *= math.pow(FACTOR, r / max(r - 2, 1))
    found = []
    for i in range(r // 2):
        f = math.pow(base, -2.0 * i / r)
        if how == "linear":
            f /= FACTOR
        elif how == "yarn":
            low = max(math.floor(r * math.log(ORIGINAL / (64 * math.pi)) / (2 * math.log(base))), 0)
            high = min(math.ceil(r * math.log(ORIGINAL / (2 * math.pi)) / (2 * math.log(base))), r - 1)
            t = min(max((i - low) / max(high - low, 0.001), 0.0), 1.0)
            f = t * f / FACTOR + (1 - t) * f
        elif how == "wavelength":
            wave = 2 * math.pi / f
            if wave > ORIGINAL:
                f /= FACTOR
            elif wave > ORIGINAL / 4:
                t = (ORIGINAL / wave - 1) / 3
                f = (1 - t) * f / FACTOR + t * f
        found.append(f)
    return found, (0.1 * math.log(FACTOR) + 1.0 if how == "yarn" else 1.0)


def _turned(x, positions, case):
    """Every pair as a complex number, turned by its angle."""
    f, m = _frequencies(case)
    f = torch.tensor(f, dtype=torch.float64, device=x.device)
    turn = torch.polar(torch.full_like(f, m).expand(len(positions), -1).contiguous(), positions.double()[:, None] * f[None, :])
    y, r = x.double().clone(), case["rotary"]
    first, second = (slice(0, r, 2), slice(1, r, 2)) if case["interleaved"] else (slice(0, r // 2), slice(r // 2, r))
    z = torch.complex(y[..., first], y[..., second]) * turn[:, None, :]
    y[..., first], y[..., second] = z.real, z.imag
    return y


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "rope":
        return _turned(s["x"], s["positions"], case)
    if op == "append":
        hq, hk, p = case["q_heads"], case["kv_heads"], case["page"]
        x = s["qkv"].view(case["rows"], hq + 2 * hk, case["dim"])
        y = _turned(x[:, : hq + hk], s["positions"], case)
        k, v = s["k"].double(), s["v"].double()
        index = s["index"].long()
        at = s["pages"].long()[s["seqs"].long(), torch.div(index, p, rounding_mode="floor")] * p + index.remainder(p)
        flat = lambda t: t.reshape(-1, hk, case["dim"])  # noqa: E731
        k = flat(k).index_copy(0, at, y[:, hq:]).view(k.shape)
        v = flat(v).index_copy(0, at, x[:, hq + hk :].double()).view(v.shape)
        return y[:, :hq], k, v
    lengths = s["lens"].tolist()
    hk, p = case["kv_heads"], case["page"]
    if op == "attend":
        g, out = case["q_heads"] // hk, torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
        w = s["weights"].double() if case["weights"] else None
        for b, n in enumerate(lengths):
            lo = max(0, n - case["window"]) if case["window"] else 0
            pages = s["pages"][b, : -(-n // p)].long()
            for h in range(hk):
                k, v = (t[pages, :, h].reshape(-1, case["dim"])[lo:n].double() * s["scale"] for t in (s["k"], s["v"]))
                q = s["q"][b, h * g : (h + 1) * g].double()
                share = torch.softmax(q @ k.T / math.sqrt(case["dim"]), -1)
                out[b, h * g : (h + 1) * g] = share @ v
                if w is not None:
                    w[b, h, lo:n] += share.sum(0)
        return out, w
    k, v = s["k"].double(), s["v"].double()
    new = torch.zeros(s["weights"].shape, dtype=torch.float64, device=s["lens"].device)
    weights = s["weights"].cpu().tolist()
    for b, n in enumerate(lengths):
        for h in range(hk):
            stays = set(range(min(case["sinks"], n))) | set(range(max(0, n - case["recent"]), n))
            rest = sorted((i for i in range(n) if i not in stays), key=lambda i: (-weights[b][h][i], i))
            chosen = sorted(list(stays) + rest[: max(0, min(n, case["keep"]) - len(stays))])
            i = torch.tensor(chosen, device=new.device)
            j = torch.arange(len(chosen), device=new.device)
            old, to = s["pages"][b].long()[i // p], s["new_pages"][b].long()[j // p]
            k[to, j % p, h], v[to, j % p, h] = s["k"][old, i % p, h].double(), s["v"][old, i % p, h].double()
            new[b, h, : len(chosen)] = s["weights"][b, h, i].double()
    return k, v, new, None, None
