"""Cases for the operators around a decode step on the paged head-mixed cache.

* ``rope``: q and k rotated by positions with several axes (text, image and video tokens).
* ``weights``: the attention weight that each cached key received, summed over queries and over a group's heads.
* ``evict``: the keys to keep, by that weight, and the cache's rows copied into a smaller cache.
* ``logits``: penalties for repeated tokens, biases and grammar masks on logits, and the greedy token.

A case runs either in a plain form of elementary torch operations in 32 bits (``own`` false)
or through ``aoh_b200`` (``own`` true), on the same inputs.
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
PAGE = 16  # tokens of one cache page
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# -- the cases ------------------------------------------------------------------
def _rope(name, B, C, Hq, G, D, sections, dtype="bf16", interleaved=False, norm=False, start=0, rot=0):
    return {"name": name, "op": "rope", "B": B, "C": C, "Hq": Hq, "G": G, "D": D, "sections": sections,
            "dtype": dtype, "interleaved": interleaved, "norm": norm, "start": start, "rot": rot or D}


def _weights(name, B, C, past, Hq, G, n_ret, dtype="bf16"):
    return {"name": name, "op": "weights", "B": B, "C": C, "past": past, "Hq": Hq, "G": G, "n_ret": n_ret,
            "dtype": dtype}


def _evict(name, L, B, T, keep, G, n_ret, sink, recent, dtype="bf16"):
    return {"name": name, "op": "evict", "L": L, "B": B, "T": T, "keep": keep, "G": G, "n_ret": n_ret,
            "sink": sink, "recent": recent, "dtype": dtype}


def _logits(name, N, V, prompt, output, K, mask, dtype="bf16"):
    return {"name": name, "op": "logits", "N": N, "V": V, "prompt": prompt, "output": output, "K": K,
            "mask": mask, "dtype": dtype}


def listed():
    return [
        # one decoded token of a batch of eight, far into a long video: the smallest call, all latency
        _rope("rope token", 8, 1, 32, 8, 128, "16,24,24", start=250_000),
        # a prompt chunk of image patches, Qwen2.5-7B heads, views of one fused projection
        _rope("rope chunk", 1, 4096, 28, 4, 128, "16,24,24"),
        # a ragged float32 batch: interleaved axes, QK-norm, head size 80 of which 64 rotate
        _rope("rope f32 ragged", 3, 1021, 12, 4, 80, "12,10,10", "f32", True, True, 70_001, 64),
        # one token's weights over a 128K cache, 2 of 8 KV heads retrieval (Llama-3.1-8B heads)
        _weights("weights token", 1, 1, 131_071, 32, 8, 2),
        # the prompt's last 32 queries over 32K keys, group of 7: how a prompt is scored before eviction
        _weights("weights window", 1, 32, 32_745, 28, 4, 4),
        # a 4096-token prefill chunk, every query counted
        _weights("weights chunk", 1, 4096, 12_288, 32, 8, 4),
        # a float32 cache, batch of two, odd lengths
        _weights("weights f32", 2, 33, 1_990, 8, 4, 3, "f32"),
        # a short decode-time eviction of one layer
        _evict("evict short", 1, 2, 1_283, 768, 8, 4, 128, 256),
        # eight layers of a 64K prompt cut to 8K rows a head
        _evict("evict prompt", 8, 1, 65_536, 8_192, 8, 4, 128, 256),
        # one sequence's logits, no grammar
        _logits("logits one", 1, 128_256, 900, 300, 16, False),
        # a batch under a grammar, long histories
        _logits("logits batch", 64, 128_256, 4_000, 2_000, 64, True),
        # float32 logits with an odd vocabulary
        _logits("logits f32 odd", 37, 32_003, 500, 100, 300, True, "f32"),
    ]


def _log_int(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(("rope", "weights", "weights", "evict", "logits"))
    dtype = rng.choice(("bf16", "bf16", "bf16", "f32"))
    if op == "rope":
        D = rng.choice((64, 80, 96, 128, 128, 128, 256))
        half = rng.choice((D, D, D // 2)) // 2
        a = rng.randrange(1, half // 2)
        b = rng.randrange(0, (half - a) // 2 + 1)
        sections = rng.choice(([half], [half - a, a], [half - a - b, a, b]))
        A = len(sections)
        # interleaved axes fit while every axis but the first stays within its share of the frequencies
        inter = rng.random() < 0.4 and all(A * s <= half for s in sections[1:])
        G = rng.choice((1, 2, 4, 8))
        B = _log_int(rng, 1, 16)
        return _drop(_rope("", B, _log_int(rng, 1, max(1, 4096 // B)), G * rng.choice((1, 2, 4, 5, 7)), G, D,
                           ",".join(map(str, sections)), dtype, inter, rng.random() < 0.5,
                           rng.choice((0, _log_int(rng, 1, 1_000_000))), 2 * half))
    if op == "weights":
        G = rng.choice((1, 2, 4, 8))
        n_ret = rng.randrange(1, min(G, 4) + 1)
        grp = rng.choice((1, 2, 4, 5, 7, 8))
        B = rng.choice((1, 1, 1, 2, 3))
        if dtype == "f32":
            C = rng.choice((1, _log_int(rng, 2, 128)))
            return _drop(_weights("", B, C, _log_int(rng, 1, 4_000), G * grp, G, n_ret, dtype))
        rows = B * n_ret * grp
        C = rng.choice((1, _log_int(rng, 2, min(4_096, math.isqrt(2 ** 29 // rows)))))
        most = 131_071 // B if C == 1 else min(65_536, 2 ** 29 // (C * rows))
        return _drop(_weights("", B, C, rng.choice((0, _log_int(rng, 1, max(2, most)))), G * grp, G, n_ret, dtype))
    if op == "evict":
        G = rng.choice((1, 2, 4, 8))
        n_ret = rng.randrange(1, G + 1)
        L, B = rng.choice((1, 2, 5)), rng.choice((1, 2))
        sink, recent = rng.choice(((128, 256), (0, 0), (5, 37), (16, 0)))
        T = _log_int(rng, max(64, sink + recent + 2), 262_144 // (L * B * G) + 1_024)
        return _drop(_evict("", L, B, T, rng.randrange(max(1, sink + recent), T), G, n_ret, sink, recent, dtype))
    N = _log_int(rng, 1, 64)
    V = _log_int(rng, 1_000, 131_072)
    return _drop(_logits("", N, V, _log_int(rng, 1, 4_000), _log_int(rng, 1, 2_000), rng.choice((0, 3, 64, 301)),
                         rng.random() < 0.6, dtype))


def _drop(case):
    del case["name"]
    return case


# -- inputs ---------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _randn(gen, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32).to(dtype)


def _labels(L, G, n_ret):
    """n_ret retrieval heads spread over the G KV heads, moved by one from layer to layer."""
    heads = [[0] * G for _ in range(L)]
    for layer in range(L):
        for i in range(n_ret):
            heads[layer][(i * G // n_ret + layer) % G] = 1
    return heads


def _retrieval(labels):
    """(layer, KV head) of every retrieval head, layer by layer."""
    return [(layer, g) for layer, row in enumerate(labels) for g, x in enumerate(row) if x]


def _make_rope(c, seed):
    g = _gen(seed)
    B, C, Hq, G, D = c["B"], c["C"], c["Hq"], c["G"], c["D"]
    dt = DTYPES[c["dtype"]]
    sections = [int(s) for s in c["sections"].split(",")]
    qkv = _randn(g, B, C, (Hq + 2 * G) * D, dtype=dt)
    i = torch.arange(C, device=DEVICE).expand(B, C)
    shift = torch.randint(0, 50, (B, 1), generator=g, device=DEVICE)
    # frames of 24 x 32 patches: time moves every 768 tokens, rows and columns within a frame
    axes = [c["start"] + shift + i // 768, c["start"] + shift + (i % 768) // 32, c["start"] + shift + i % 32]
    axes = axes[:len(sections)] if len(sections) > 1 else [c["start"] + shift + i]
    half = c["rot"] // 2
    inv = 1e6 ** (-torch.arange(half, device=DEVICE, dtype=torch.float64) / half)
    s = {"q": qkv[..., :Hq * D].view(B, C, Hq, D), "k": qkv[..., Hq * D:(Hq + G) * D].view(B, C, G, D),
         "positions": torch.stack(axes).contiguous(), "inv_freq": inv.float(), "sections": sections, "qw": None, "kw": None}
    if c["norm"]:
        s["qw"] = (1 + 0.1 * _randn(g, D)).to(dt)
        s["kw"] = (1 + 0.1 * _randn(g, D)).to(dt)
    return s


def _make_weights(c, seed):
    g = _gen(seed)
    B, C, G, D = c["B"], c["C"], c["G"], 128
    T, dt = c["past"] + c["C"], DTYPES[c["dtype"]]
    k = _randn(g, B, T, G, D)
    k[:, :4] += 0.5  # the first keys draw weight from every query
    q = (1.5 * _randn(g, B, C, c["Hq"], D) + 0.2).to(dt)
    return {"q": q, "k": k.to(dt), "labels": _labels(1, G, c["n_ret"])}


def _make_evict(c, seed):
    g = _gen(seed)
    L, B, T, G = c["L"], c["B"], c["T"], c["G"]
    dt = DTYPES[c["dtype"]]
    labels = _labels(L, G, c["n_ret"])
    R = B * L * c["n_ret"]
    # most keys get next to nothing, some exactly nothing, many the same amount
    w = torch.rand((R, T), generator=g, device=DEVICE).log().neg().pow(3)
    w = torch.where(w < 0.05, torch.zeros_like(w), (w * 512).round() / 512)
    k = torch.randn((L, B, T, G, 128), generator=g, device=DEVICE, dtype=dt)
    v = torch.randn((L, B, T, G, 128), generator=g, device=DEVICE, dtype=dt)
    return {"weights": w, "k": k, "v": v, "labels": labels}


def _make_logits(c, seed):
    g = _gen(seed)
    N, V = c["N"], c["V"]
    dt = DTYPES[c["dtype"]]

    def ids(n):  # token frequencies fall like 1 / rank
        u = torch.rand((N, n), generator=g, device=DEVICE)
        return (torch.exp(u * math.log(V)) - 1).long().clamp(0, V - 1)

    s = {"logits": (3 * _randn(g, N, V)).to(dt), "prompt": ids(c["prompt"]), "output": ids(c["output"]),
         "repetition": 1 + 0.3 * torch.rand(N, generator=g, device=DEVICE),
         "presence": torch.rand(N, generator=g, device=DEVICE),
         "frequency": 0.5 * torch.rand(N, generator=g, device=DEVICE),
         "bias_ids": None, "bias": None, "allowed": None}
    if c["K"]:
        s["bias_ids"] = ids(c["K"]).to(torch.int32)
        s["bias_ids"][:, -1] = -1  # a shorter list is padded with -1
        s["bias"] = 4 * _randn(g, N, c["K"])
    if c["mask"]:
        words = (V + 31) // 32
        bits = torch.randint(-2 ** 31, 2 ** 31, (2, N, words), generator=g, device=DEVICE)
        s["allowed"] = (bits[0] & bits[1]).to(torch.int32)
        if N > 1:
            s["allowed"][N // 2] = 0  # a row that allows nothing
            s["allowed"][0] = -1      # and one that allows everything
    return s


def prepare(case, seed):
    make = {"rope": _make_rope, "weights": _make_weights, "evict": _make_evict, "logits": _make_logits}[case["op"]]
    s = {"case": case, **make(case, seed)}
    if own:
        _hold(case, s)
    elif case["op"] == "logits":
        one = torch.ones((), dtype=torch.int32, device=DEVICE)
        zero = torch.zeros((case["N"], case["V"]), dtype=torch.int32, device=DEVICE)
        s["counts"] = zero.scatter_add(1, s.pop("output"), one.expand(case["N"], case["output"]))
        s["in_prompt"] = zero.scatter_add(1, s.pop("prompt"), one.expand(case["N"], case["prompt"])) > 0
    return s


def _hold(c, s):
    """The caches and histories that a user's program has filled before the call."""
    import aoh_b200

    if c["op"] == "weights":
        T = c["past"] + c["C"]
        k = s.pop("k")
        cache = aoh_b200.AoHKVCache(s["labels"], c["Hq"], batch=c["B"], max_context=T, dtype=k.dtype, reserve_all=True)
        cache.append_layer(0, k, k)
        cache.kv_seq_len = c["past"]  # the chunk's rows are stored, the length moves after the last layer
        s["cache"] = cache
    elif c["op"] == "evict":
        k, v = s.pop("k"), s.pop("v")
        make = lambda n: aoh_b200.AoHKVCache(  # noqa: E731
            s["labels"], c["G"], batch=c["B"], sink_size=c["sink"], recent_size=c["recent"], max_context=n,
            dtype=k.dtype, reserve_all=True)
        s["cache"], s["into"] = make(c["T"]), make(c["keep"])
        for layer in range(c["L"]):
            s["cache"].append_layer(layer, k[layer], v[layer])
        s["cache"].kv_seq_len = c["T"]
    elif c["op"] == "logits":
        s["history"] = aoh_b200.TokenHistory(c["N"], c["V"], device=DEVICE)
        s["history"].add_prompt(s.pop("prompt"))
        s["history"].append(s.pop("output"))


# -- one pass -------------------------------------------------------------------
def run(state):
    c = state["case"]
    if own:
        return _own(c, state)
    return {"rope": _plain_rope, "weights": _plain_weights, "evict": _plain_evict, "logits": _plain_logits}[c["op"]](c, state)


def _own(c, s):
    import aoh_b200

    if c["op"] == "rope":
        q, k = aoh_b200.rope_axes_qk(s["q"], s["k"], s["positions"], s["inv_freq"], s["sections"],
                                     interleaved=c["interleaved"], q_norm_weight=s["qw"], k_norm_weight=s["kw"])
        return {"q": q, "k": k}
    if c["op"] == "weights":
        return {"weights": aoh_b200.key_weights(s["cache"], 0, s["q"])}
    if c["op"] == "evict":
        kept, kept_weights = aoh_b200.select_keys(s["weights"], c["keep"], sink=c["sink"], recent=c["recent"])
        aoh_b200.evict(s["cache"], kept, s["into"])
        return {"kept": kept, "weights": kept_weights, "pool": s["into"].pool_view()}
    bias = None if s["bias_ids"] is None else (s["bias_ids"], s["bias"])
    logits, ids = aoh_b200.penalize_logits(
        s["logits"], s["history"], repetition=s["repetition"], presence=s["presence"], frequency=s["frequency"],
        bias=bias, allowed=s["allowed"], greedy=True)
    return {"logits": logits, "ids": ids}


def _axis_of(c, sections):
    """The position axis of each frequency."""
    half, A = c["rot"] // 2, len(sections)
    if c["interleaved"]:
        return [i % A if i < A * sections[i % A] else 0 for i in range(half)]
    return [a for a, n in enumerate(sections) for _ in range(n)]


def _plain_rope(c, s):
    half = c["rot"] // 2
    axis = torch.tensor(_axis_of(c, s["sections"]), device=DEVICE)
    # far positions: the product needs more bits than a float has
    angle = s["positions"][axis].permute(1, 2, 0).double() * s["inv_freq"].double()
    cos, sin = angle.cos().float()[:, :, None], angle.sin().float()[:, :, None]

    def turn(x, w):
        x = x.float()
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.float()
        a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
        return torch.cat((a * cos - b * sin, b * cos + a * sin, rest), -1).to(s["q"].dtype)

    return {"q": turn(s["q"], s["qw"]), "k": turn(s["k"], s["kw"])}


def _plain_weights(c, s):
    B, C, G, past = c["B"], c["C"], c["G"], c["past"]
    T, grp = past + C, c["Hq"] // G
    heads = torch.tensor([g for _, g in _retrieval(s["labels"])], device=DEVICE)
    k = s["k"].float().index_select(2, heads).permute(0, 2, 1, 3)  # (B, n_ret, T, D)
    q = s["q"].float().view(B, C, G, grp, 128).index_select(2, heads).permute(0, 2, 3, 1, 4)
    x = torch.matmul(q.reshape(B, len(heads), grp * C, 128), k.transpose(2, 3)).mul_(1 / math.sqrt(128))
    x = x.view(B, len(heads), grp, C, T)
    late = torch.arange(T, device=DEVICE) > past + torch.arange(C, device=DEVICE)[:, None]
    x.masked_fill_(late, -math.inf)
    x = x.sub_(x.amax(-1, keepdim=True)).exp_()
    x = x.div_(x.sum(-1, keepdim=True))
    return {"weights": x.sum((2, 3))}


def _plain_evict(c, s):
    L, B, T, G, keep, sink, recent = (c[n] for n in ("L", "B", "T", "G", "keep", "sink", "recent"))
    w = s["weights"]
    R = w.shape[0]
    middle = w[:, sink:T - recent].sort(dim=-1, descending=True, stable=True).indices[:, :keep - sink - recent] + sink
    first = torch.arange(sink, device=DEVICE).expand(R, sink)
    last = torch.arange(T - recent, T, device=DEVICE).expand(R, recent)
    kept = torch.cat((first, middle, last), 1).sort(-1).values
    # rows of the units in the order (layer, sequence, KV head)
    retrieval = torch.tensor(s["labels"], device=DEVICE, dtype=torch.bool)[:, None].expand(L, B, G)
    layer, b, g = (i[:, None] for i in retrieval.nonzero(as_tuple=True))
    ret = torch.stack((s["k"][layer, b, kept, g], s["v"][layer, b, kept, g]), 2)
    layer, b, g = (i[:, None] for i in (~retrieval).nonzero(as_tuple=True))
    ring = -(-recent // PAGE) * PAGE
    held = min(ring, keep - sink)  # rows behind the sink that a streaming head still holds
    behind = torch.arange(keep - held, keep, device=DEVICE)
    from_ = torch.cat((torch.arange(sink, device=DEVICE), behind + T - keep))[None]
    strm = torch.stack((s["k"][layer, b, from_, g], s["v"][layer, b, from_, g]), 2)
    sink_rows = _pages(strm[:, :sink])
    ring_rows = strm.new_zeros((strm.shape[0], ring, 2, 128))
    ring_rows[:, (behind - sink) % max(1, ring)] = strm[:, sink:]
    # pages in the order they are granted: the streaming heads' first, then the retrieval heads'
    streaming = torch.cat((sink_rows, _pages(ring_rows)), 1).flatten(0, 1)
    pool = torch.cat((streaming, _pages(ret).flatten(0, 1)), 0)
    return {"kept": kept.to(torch.int32), "weights": w.gather(1, kept), "pool": pool}


def _pages(x):
    """Rows (units, n, 2, 128) as pages (units, pages, 2, 16, 128) in the cache's stored layout."""
    units, n = x.shape[:2]
    pages = -(-n // PAGE)
    x = torch.cat((x, x.new_zeros((units, pages * PAGE - n, 2, 128))), 1)
    if x.dtype == torch.float32:
        return x.view(units, pages, PAGE, 2, 128).transpose(2, 3)
    # bf16: [64-dim half][K | V][slot][8 chunks of 16 bytes], chunk c of a slot stored at c ^ (slot & 7)
    x = x.view(units, pages, PAGE, 2, 2, 8, 8).permute(0, 1, 4, 3, 2, 5, 6)
    chunk = torch.arange(8, device=DEVICE)[None] ^ (torch.arange(PAGE, device=DEVICE)[:, None] & 7)
    x = torch.gather(x, 5, chunk[None, None, None, None, :, :, None].expand(units, pages, 2, 2, PAGE, 8, 8))
    return x.reshape(units, pages, 2, PAGE, 128)


def _plain_logits(c, s):
    x = s["logits"].float()
    n = s["counts"]
    col = lambda t: s[t][:, None]  # noqa: E731
    x = torch.where((n > 0) | s["in_prompt"], torch.where(x > 0, x / col("repetition"), x * col("repetition")), x)
    x = x - col("frequency") * n.float()
    x = x - col("presence") * (n > 0).float()
    if s["bias_ids"] is not None:
        # one column more takes what the padding adds
        at = torch.where(s["bias_ids"] < 0, c["V"], s["bias_ids"]).long()
        x = x + x.new_zeros((c["N"], c["V"] + 1)).scatter_add(1, at, s["bias"])[:, :-1]
    if s["allowed"] is not None:
        bits = s["allowed"][:, :, None] >> torch.arange(32, device=DEVICE, dtype=torch.int32) & 1
        x = x.masked_fill(bits.flatten(1)[:, :c["V"]] == 0, -math.inf)
    # the lowest index of the largest value
    at = torch.arange(c["V"], device=DEVICE).expand_as(x)
    return {"logits": x, "ids": torch.where(x == x.amax(1, keepdim=True), at, c["V"]).amin(1)}


# -- what a pass cannot do without ------------------------------------------------
def work(case):
    c, es = case, 2 if case["dtype"] == "bf16" else 4
    if c["op"] == "rope":
        n = c["B"] * c["C"] * (c["Hq"] + c["G"]) * c["D"]
        return {"bytes": 2 * n * es + 8 * c["B"] * c["C"] * len(c["sections"].split(",")) + 2 * c["rot"],
                "flops": (10 if c["norm"] else 6) * n}
    if c["op"] == "weights":
        B, C, past, grp = c["B"], c["C"], c["past"], c["Hq"] // c["G"]
        pairs = B * c["n_ret"] * grp * (C * past + C * (C + 1) // 2)
        return {"bytes": B * c["n_ret"] * ((past + C) * (128 * es + 4) + C * grp * 128 * es), "flops": pairs * (2 * 128 + 4)}
    if c["op"] == "evict":
        ring = -(-c["recent"] // PAGE) * PAGE
        rows = c["L"] * c["B"] * (c["n_ret"] * c["keep"] + (c["G"] - c["n_ret"]) * (c["sink"] + min(ring, c["keep"] - c["sink"])))
        R = c["L"] * c["B"] * c["n_ret"]
        return {"bytes": 2 * rows * 256 * es + R * (4 * c["T"] + 8 * c["keep"]), "flops": R * c["T"]}
    N, V = c["N"], c["V"]
    return {"bytes": N * (V * (es + 4) + V / 8 * (2 if c["mask"] else 1) + 8 * c["K"] + 20), "flops": 2 * N * V}


# -- the definitions in 64 bits ---------------------------------------------------
def exact(case, seed):
    make = {"rope": _make_rope, "weights": _make_weights, "evict": _make_evict, "logits": _make_logits}[case["op"]]
    s = make(case, seed)
    return {"rope": _exact_rope, "weights": _exact_weights, "evict": _exact_evict, "logits": _exact_logits}[case["op"]](case, s)


def _exact_rope(c, s):
    half, sections = c["rot"] // 2, s["sections"]
    pos = s["positions"].double()
    angle = torch.empty(c["B"], c["C"], 1, half, dtype=torch.float64, device=DEVICE)
    for i in range(half):
        if c["interleaved"]:
            a = i % len(sections)
            a = a if i // len(sections) < sections[a] else 0
        else:
            a = next(j for j in range(len(sections)) if i < sum(sections[:j + 1]))
        angle[:, :, 0, i] = pos[a] * float(s["inv_freq"][i])
    turn = torch.polar(torch.ones_like(angle), angle)
    out = {}
    for name, w in (("q", s["qw"]), ("k", s["kw"])):
        x = s[name].double()
        if w is not None:
            x = x / ((x ** 2).sum(-1, keepdim=True) / c["D"] + 1e-6).sqrt() * w.double()
        y = torch.complex(x[..., :half], x[..., half:2 * half]) * turn
        x[..., :half], x[..., half:2 * half] = y.real, y.imag
        out[name] = x
    return out


def _exact_weights(c, s):
    B, C, past, grp = c["B"], c["C"], c["past"], c["Hq"] // c["G"]
    heads = [g for g, x in enumerate(s["labels"][0]) if x]
    out = torch.zeros(B, len(heads), past + C, dtype=torch.float64, device=DEVICE)
    for b in range(B):
        for r, g in enumerate(heads):
            k = s["k"][b, :, g].double()
            for h in range(g * grp, (g + 1) * grp):
                for lo in range(0, C, 1024):
                    n = min(1024, C - lo)
                    x = s["q"][b, lo:lo + n, h].double() @ k.T / 128 ** 0.5
                    x = x + torch.full_like(x, -math.inf).triu(past + lo + 1)
                    out[b, r] += torch.softmax(x, 1).sum(0)
    return {"weights": out}


def _exact_evict(c, s):
    if c["T"] * c["L"] > 20_000:
        return None  # the rows are copies: the smaller cases say as much
    L, B, T, keep, sink, recent = (c[n] for n in ("L", "B", "T", "keep", "sink", "recent"))
    w = s["weights"].cpu().numpy()
    k, v = s["k"].double().cpu().numpy(), s["v"].double().cpu().numpy()
    sp, rp = -(-sink // PAGE), -(-recent // PAGE)
    kp, pages, kept_w, streaming, retrieval = -(-keep // PAGE), [], [], [], []
    r = 0
    for layer in range(L):
        for b in range(B):
            for g in range(c["G"]):
                if s["labels"][layer][g]:
                    row = w[r]
                    r += 1
                    best = sorted(range(sink, T - recent), key=lambda j: (-row[j], j))[:keep - sink - recent]
                    kept = sorted([*range(sink), *best, *range(T - recent, T)])
                    kept_w.append([float(row[j]) for j in kept])
                    retrieval.append((layer, b, g, kp, {n: j for n, j in enumerate(kept)}))
                else:
                    place = {n: n for n in range(sink)}
                    for n in range(max(sink, keep - rp * PAGE), keep):
                        place[sp * PAGE + (n - sink) % (rp * PAGE)] = n + T - keep
                    streaming.append((layer, b, g, sp + rp, place))
    for layer, b, g, n_pages, place in streaming + retrieval:
        page = torch.zeros(n_pages, 2, PAGE, 128, dtype=torch.float64)
        to, of = torch.tensor(list(place), dtype=torch.long), list(place.values())
        if of:
            for kv, x in ((0, k), (1, v)):
                page[to // PAGE, kv, to % PAGE] = torch.from_numpy(x[layer, b, of, g])
        if c["dtype"] == "bf16":
            flat = torch.zeros(n_pages, 4096, dtype=torch.float64)
            for slot in range(PAGE):
                for chunk in range(16):
                    for kv in range(2):
                        at = chunk // 8 * 2048 + kv * 1024 + slot * 64 + (chunk % 8 ^ slot % 8) * 8
                        flat[:, at:at + 8] = page[:, kv, slot, chunk * 8:chunk * 8 + 8]
            page = flat.view(n_pages, 2, PAGE, 128)
        pages.append(page)
    return {"kept": None, "weights": torch.tensor(kept_w, dtype=torch.float64), "pool": torch.cat(pages)}


def _exact_logits(c, s):
    V = c["V"]
    x = s["logits"].double().cpu()
    for n in range(c["N"]):
        count = torch.bincount(s["output"][n].cpu(), minlength=V).double()
        seen = (count + torch.bincount(s["prompt"][n].cpu(), minlength=V).double()) > 0
        rep, freq, pres = (float(s[t][n]) for t in ("repetition", "frequency", "presence"))
        row = x[n]
        row[seen & (row > 0)] /= rep
        row[seen & (s["logits"][n].cpu() <= 0)] *= rep
        row -= freq * count + pres * (count > 0).double()
        if s["bias_ids"] is not None:
            for i, v in zip(s["bias_ids"][n].tolist(), s["bias"][n].tolist()):
                if i >= 0:
                    row[i] += v
        if s["allowed"] is not None:
            words = s["allowed"][n].cpu().long() & 0xFFFFFFFF
            ids = torch.arange(V)
            row[(words[ids // 32] >> (ids % 32)) & 1 == 0] = -math.inf
    return {"logits": x, "ids": None}
