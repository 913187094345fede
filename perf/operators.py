"""Measured calls of the operators that carry a step from request lengths to attention.

Three operators that run one after the other when a batch of prompts, or the next token of many
requests, goes through a layer over the paged cache:

  step    block tables, slot mapping and positions of a step, built on the GPU from the requests'
          lengths (``PagedBlockPool.build_step``)
  rope    rotary positions with several axes (time, height, width), fused with the q / k / v prologue
          and the append of k and v into their slots (``PagedBlockPool.mrope_append``)
  prompt  causal attention over whole prompts of different lengths, packed, with grouped heads, read
          from the projections and not from the cache (``PagedBlockPool.prompt_attention``)

``own`` selects between the plain form of each (elementary torch operations in 32 bits) and the
framework's calls.
"""
import math
import os
import random
import sys

import torch

own = False

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def framework():
    """The package of this tree."""
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "glacier.serve_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import glacier_kv

    return glacier_kv


# ---- cases ------------------------------------------------------------------------------------

def listed():
    return [
        # the next prompt of a quiet server: one short request, where the call's latency counts
        {"name": "prompt: one short", "op": "prompt", "seqs": 1, "median": 97, "longest": 97, "mix": 0, "heads": 28, "heads_kv": 4,
         "dim": 128, "dtype": "bf16", "fused": False, "sinks": False, "lse": False},
        # a prefill step of a busy server: requests of many lengths, one token among them, with the
        # softmax statistics that a merge with a cached prefix needs
        {"name": "prompt: busy batch", "op": "prompt", "seqs": 24, "median": 500, "longest": 6000, "mix": 1, "heads": 28, "heads_kv": 4,
         "dim": 128, "dtype": "bf16", "fused": True, "sinks": False, "lse": True},
        # one long document
        {"name": "prompt: long document", "op": "prompt", "seqs": 1, "median": 16384, "longest": 16384, "mix": 0, "heads": 28,
         "heads_kv": 4, "dim": 128, "dtype": "bf16", "fused": False, "sinks": False, "lse": False},
        # small heads in half precision, with a sink per head
        {"name": "prompt: small heads", "op": "prompt", "seqs": 9, "median": 1100, "longest": 4000, "mix": 2, "heads": 16, "heads_kv": 4,
         "dim": 64, "dtype": "f16", "fused": True, "sinks": True, "lse": False},
        # the engine's own precision: 32 bits throughout
        {"name": "prompt: 32 bits", "op": "prompt", "seqs": 6, "median": 400, "longest": 1500, "mix": 3, "heads": 32, "heads_kv": 8,
         "dim": 128, "dtype": "f32", "fused": False, "sinks": False, "lse": True},
        # one new token for each of 64 requests: q goes on in 32 bits to the paged decode
        {"name": "rope: decode step", "op": "rope", "tokens": 64, "heads": 28, "heads_kv": 4, "dim": 128, "rope_dim": 128, "dtype": "bf16",
         "out": "f32", "cache": "bf16", "norm": False, "bias": True, "interleaved": False, "style": 0, "farthest": 32768, "keep": False},
        # prompts with images: q and the rotated k go on to the prompt attention, k and v to the cache
        {"name": "rope: image prompts", "op": "rope", "tokens": 8192, "heads": 28, "heads_kv": 4, "dim": 128, "rope_dim": 128, "dtype": "bf16",
         "out": "bf16", "cache": "bf16", "norm": False, "bias": True, "interleaved": False, "style": 0, "farthest": 131072, "keep": True},
        # video prompts with normed heads into an 8-bit cache, from 32-bit projections, half of each head rotated
        {"name": "rope: video into 8 bits", "op": "rope", "tokens": 2049, "heads": 32, "heads_kv": 8, "dim": 128, "rope_dim": 64,
         "dtype": "f32", "out": "f32", "cache": "fp8", "norm": True, "bias": False, "interleaved": True, "style": 0, "farthest": 1000000,
         "keep": False},
        # the next token of 64 requests
        {"name": "step: 64 decodes", "op": "step", "requests": 64, "median": 1500, "longest": 8192, "new": 1, "mix": 4, "block": 16},
        # the next token of 1024 requests, some of them long
        {"name": "step: 1024 decodes", "op": "step", "requests": 1024, "median": 1500, "longest": 32768, "new": 1, "mix": 5, "block": 16},
        # a prefill step: 40 requests with prompts (or further chunks) of many lengths
        {"name": "step: 40 prompts", "op": "step", "requests": 40, "median": 700, "longest": 8192, "new": 4000, "mix": 6, "block": 16},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["prompt", "prompt", "rope", "step"])
    if op == "prompt":
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        heads_kv = rng.choice([1, 2, 4, 8])
        group = rng.choice([1, 4, 7, 8]) if heads_kv <= 4 else rng.choice([1, 4])
        seqs = _log(rng, 1, 40)
        longest = min(_log(rng, 1, 1500 if dtype == "f32" else 12000), int(math.sqrt(2e8 / seqs)))
        return {"op": op, "seqs": seqs, "median": max(1, int(longest * rng.uniform(0.1, 0.8))), "longest": longest, "mix": rng.randrange(1 << 20),
                "heads": heads_kv * group, "heads_kv": heads_kv, "dim": rng.choice([64, 128, 128]), "dtype": dtype,
                "fused": rng.random() < 0.5, "sinks": rng.random() < 0.3, "lse": rng.random() < 0.5}
    if op == "rope":
        heads_kv = rng.choice([1, 2, 4, 8])
        dim = rng.choice([64, 128, 128, 256])
        dtype = rng.choice(["bf16", "f16", "f32"])
        return {"op": op, "tokens": _log(rng, 1, 8192), "heads": heads_kv * rng.choice([1, 4, 7]), "heads_kv": heads_kv, "dim": dim,
                "rope_dim": rng.choice([dim, dim, dim // 2]), "dtype": dtype, "out": rng.choice([dtype, "f32"]),
                "cache": rng.choice(["bf16", "f16", "f32", "fp8"]), "norm": rng.random() < 0.5, "bias": rng.random() < 0.5,
                "interleaved": rng.random() < 0.5, "style": rng.randrange(2), "farthest": _log(rng, 10000, 1000000), "keep": rng.random() < 0.5}
    return {"op": op, "requests": _log(rng, 1, 1024), "median": _log(rng, 50, 1500), "longest": _log(rng, 1600, 32768), "new": rng.choice([1, 1, 8, 300]),
            "mix": rng.randrange(1 << 20), "block": rng.choice([8, 16, 32])}


def lengths(n, median, longest, mix, spread=1.0):
    """n lengths around `median` (lognormal), within [1, longest], the same for the same numbers; where there are several, one of them is 1 and one `longest`."""
    r = random.Random(mix * 1000003 + n)
    got = [min(longest, max(1, int(median * math.exp(spread * r.gauss(0, 1))))) for _ in range(n)]
    if n > 1:
        got[n // 3] = 1
    got[n - 1 if n < 3 else (2 * n) // 3] = longest
    return got


def request_lengths(case):
    """(tokens stored, tokens added) of each request of a step: every seventh has nothing stored yet; in a prefill step every fifth only decodes."""
    n = case["requests"]
    ctx = lengths(n, case["median"], case["longest"], case["mix"])
    ctx = [0 if i % 7 == 3 else c for i, c in enumerate(ctx)]
    if case["new"] == 1:
        return ctx, [1] * n
    new = lengths(n, max(1, case["new"] // 4), case["new"], case["mix"] + 1)
    return ctx, [1 if i % 5 == 4 else x for i, x in enumerate(new)]


def axes_of(case):
    """The position axis of each rotary frequency: three sections of the frequencies (time, height, width), one after the other or interleaved."""
    half = case["rope_dim"] // 2
    side = half * 3 // 8
    sections = [half - 2 * side, side, side]
    if case["interleaved"]:
        axis = [0] * half
        for a in (1, 2):
            for i in range(a, min(half, 3 * sections[a]), 3):
                axis[i] = a
        return sections, axis
    return sections, [0] * sections[0] + [1] * side + [2] * side


def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2, "fp8": 1}
    if case["op"] == "prompt":
        lens = lengths(case["seqs"], case["median"], case["longest"], case["mix"])
        t, d, e = sum(lens), case["dim"], size[case["dtype"]]
        pairs = sum(n * (n + 1) // 2 for n in lens)
        nbytes = t * d * (2 * case["heads"] + 2 * case["heads_kv"]) * e + (t * case["heads"] * 4 if case["lse"] else 0)
        return {"bytes": nbytes + 4 * (len(lens) + 1), "flops": 4 * d * case["heads"] * pairs}
    if case["op"] == "rope":
        t, d, h, hk = case["tokens"], case["dim"], case["heads"], case["heads_kv"]
        e, o, c = size[case["dtype"]], size[case["out"]], size[case["cache"]]
        nbytes = t * d * (h * (e + o) + 2 * hk * (e + c) + (2 * hk * o if case["keep"] else 0)) + t * (3 * 4 + 8)
        return {"bytes": nbytes, "flops": t * (h + hk) * d * (3 + (4 if case["norm"] else 0))}
    ctx, new = request_lengths(case)
    b = case["block"]
    pages = sum((c + x + b - 1) // b - (c + b - 1) // b for c, x in zip(ctx, new))
    return {"bytes": len(ctx) * 24 + sum(new) * 12 + pages * 8, "flops": 0}


# ---- inputs -----------------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return {"prompt": prepare_prompt, "rope": prepare_rope, "step": prepare_step}[case["op"]](case, g)


def projections(t, case, g):
    """q, k and v of t tokens: separate tensors, or the three parts of one fused projection."""
    h, hk, d, dtype = case["heads"], case["heads_kv"], case["dim"], DT[case["dtype"]]
    if case.get("fused", True):
        qkv = torch.randn(t, (h + 2 * hk) * d, device="cuda", generator=g).to(dtype)
        return qkv[:, :h * d].view(t, h, d), qkv[:, h * d:(h + hk) * d].view(t, hk, d), qkv[:, (h + hk) * d:].view(t, hk, d)
    return tuple(torch.randn(t, n, d, device="cuda", generator=g).to(dtype) for n in (h, hk, hk))


def prepare_prompt(case, g):
    lens = lengths(case["seqs"], case["median"], case["longest"], case["mix"])
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    q, k, v = projections(cu[-1], case, g)
    s = {"case": case, "cu": cu, "q": q, "k": k, "v": v, "scale": 1.0 / math.sqrt(case["dim"]),
         "sinks": torch.randn(case["heads"], device="cuda", generator=g) if case["sinks"] else None}
    if own:
        G = framework()

        s["pool"] = G.PagedBlockPool(1, 1, case["heads_kv"], case["dim"], 16, dtype="bf16")
        s["cu_seqlens"] = torch.tensor(cu, dtype=torch.int32, device="cuda")
        s["out"] = torch.empty(cu[-1], case["heads"], case["dim"], dtype=q.dtype, device="cuda")
        s["lse"] = torch.empty(cu[-1], case["heads"], device="cuda") if case["lse"] else None
    return s


def prepare_rope(case, g):
    t, h, hk, d = case["tokens"], case["heads"], case["heads_kv"], case["dim"]
    q, k, v = projections(t, case, g)
    sections, axis = axes_of(case)
    half = case["rope_dim"] // 2
    # time runs on; a picture's height and width start from its time
    time = torch.randint(0, case["farthest"], (t,), device="cuda", generator=g, dtype=torch.int32)
    side = torch.randint(0, 64, (2, t), device="cuda", generator=g, dtype=torch.int32)
    blocks = (t + 15) // 16 + 3
    order = torch.randperm(blocks, device="cuda", generator=g)
    at = torch.arange(t, device="cuda")
    s = {"case": case, "q": q, "k": k, "v": v, "positions": torch.cat([time[None], time[None] + side]).contiguous(),
         "inv_freq": [float(torch.tensor(10000.0 ** (-i / half), dtype=torch.float32)) for i in range(half)], "axis": axis,
         "slots": order[at // 16] * 16 + at % 16, "eps": 1e-6,
         "bias": [torch.randn(n * d, device="cuda", generator=g) * 0.1 for n in (h, hk, hk)] if case["bias"] else [None] * 3,
         "norm": [1 + 0.1 * torch.randn(d, device="cuda", generator=g) for _ in range(2)] if case["norm"] else [None] * 2}
    s["scales"] = [0.02 + 0.01 * torch.rand(hk, device="cuda", generator=g) for _ in range(2)] if case["cache"] == "fp8" else None
    if own:
        G = framework()

        s["pool"] = pool = G.PagedBlockPool(blocks, 1, hk, d, 16, dtype=case["cache"])
        if s["scales"]:
            pool.set_kv_scales(*(x.cpu().numpy() for x in s["scales"]))
        pool.upload_step([[0]], [1], s["slots"].cpu().numpy())
        s["rope"] = G.MultiAxisRope(sections, case["rope_dim"], interleaved=case["interleaved"], style=case["style"], inv_freq=s["inv_freq"])
        keys, values = pool.key_view(), pool.value_view()
        s["cache"] = [x.view(torch.float8_e4m3fn) if case["cache"] == "fp8" else x for x in (keys, values)]
        o = DT[case["out"]]
        s["q_out"] = torch.empty(t, h, d, dtype=o, device="cuda")
        s["k_out"], s["v_out"] = (torch.empty(t, hk, d, dtype=o, device="cuda") if case["keep"] else None for _ in range(2))
    else:
        kind = torch.float8_e4m3fn if case["cache"] == "fp8" else DT[case["cache"]]
        s["cache"] = [torch.zeros(blocks, 1, hk, 16, d, device="cuda").to(kind) for _ in range(2)]
        s["axis_index"] = torch.tensor(axis, device="cuda")
        s["freq"] = torch.tensor(s["inv_freq"], device="cuda", dtype=torch.float64)
    return s


def prepare_step(case, g):
    ctx, new = request_lengths(case)
    n, b = len(ctx), case["block"]
    old = [(c + b - 1) // b for c in ctx]
    opened = [(c + x + b - 1) // b - o for c, x, o in zip(ctx, new, old)]
    width = max(o + p for o, p in zip(old, opened)) + 1
    total = sum(old) + sum(opened)
    ids = torch.randperm(total + 5, device="cuda", generator=g, dtype=torch.int32)
    page = torch.arange(width, device="cuda")
    have = torch.tensor(old, device="cuda")[:, None] > page[None]
    tables = torch.full((n, width), -1, dtype=torch.int32, device="cuda")
    tables[have] = ids[:sum(old)]
    s = {"case": case, "tables": tables, "ctx": torch.tensor(ctx, dtype=torch.int32, device="cuda"),
         "new": torch.tensor(new, dtype=torch.int32, device="cuda"), "new_blocks": ids[sum(old):total].contiguous(), "tokens": sum(new)}
    if own:
        G = framework()

        s["pool"] = pool = G.PagedBlockPool(total + 5, 1, 1, 64, b, dtype="bf16")
        pool.reserve_step(n, width, sum(new), 1)
        pool.set_static_step()
        s["io"] = G.StepBuffers(tables, s["ctx"], s["new"], s["new_blocks"], max_tokens=sum(new))
    return s


# ---- one pass ---------------------------------------------------------------------------------

def run(s):
    op = s["case"]["op"]
    if op == "prompt":
        if own:
            s["pool"].prompt_attention(s["q"], s["k"], s["v"], s["cu_seqlens"], s["out"], s["scale"], sinks=s["sinks"], lse=s["lse"])
            return [s["out"], s["lse"]]
        return plain_prompt(s)
    if op == "rope":
        if own:
            s["pool"].mrope_append(0, s["q"], s["k"], s["v"], s["positions"], s["rope"], s["q_out"], k_out=s["k_out"], v_out=s["v_out"],
                                   q_bias=s["bias"][0], k_bias=s["bias"][1], v_bias=s["bias"][2], q_norm=s["norm"][0], k_norm=s["norm"][1],
                                   eps=s["eps"])
            return [s["q_out"], s["k_out"], s["v_out"], s["cache"]]
        return plain_rope(s)
    if own:
        s["pool"].build_step(s["io"])
        io = s["io"]
        return [io.block_tables, io.ctx_out, io.cu_new, io.slots, io.positions, io.counts]
    return plain_step(s)


def plain_prompt(s):
    """softmax(scale * q k^T [, sink]) v of each prompt. Query positions go 1024 at a time, with the keys they see: the scores of a long prompt would not fit the card."""
    case = s["case"]
    h, hk, d = case["heads"], case["heads_kv"], case["dim"]
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    out, lse = torch.empty_like(q), torch.empty(q.shape[0], h, device=q.device)
    for begin, end in zip(s["cu"], s["cu"][1:]):
        kt, vt = k[begin:end].permute(1, 2, 0)[:, None], v[begin:end].transpose(0, 1)[:, None]
        for i in range(begin, end, 1024):
            j = min(end, i + 1024)
            n = j - begin
            x = (q[i:j] * s["scale"]).view(j - i, hk, h // hk, d).permute(1, 2, 0, 3) @ kt[..., :n]
            x.masked_fill_(torch.ones(j - i, n, dtype=torch.bool, device=q.device).triu(i - begin + 1), -math.inf)
            top = x.amax(-1, keepdim=True)
            if s["sinks"] is not None:
                sink = s["sinks"].view(hk, h // hk, 1, 1)
                top = torch.maximum(top, sink)
            x.sub_(top).exp_()
            total = x.sum(-1, keepdim=True)
            if s["sinks"] is not None:
                total = total + (sink - top).exp()
            out[i:j] = ((x @ vt[:, :, :n]) / total).permute(2, 0, 1, 3).reshape(j - i, h, d)
            lse[i:j] = (top + total.log()).permute(2, 0, 1, 3).reshape(j - i, h)
    return [out.to(s["q"].dtype), lse if case["lse"] else None]


def plain_rope(s):
    case = s["case"]
    r = case["rope_dim"]
    angle = s["positions"][s["axis_index"]].t().double() * s["freq"]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turned(x, bias, weight):
        x = x.float()
        if bias is not None:
            x = x + bias.view(x.shape[1:])
        if weight is not None:
            x = x * (x.square().mean(-1, keepdim=True) + s["eps"]).rsqrt() * weight
        y = x.clone()
        a, b = (slice(0, r // 2), slice(r // 2, r)) if case["style"] == 0 else (slice(0, r, 2), slice(1, r, 2))
        y[..., a] = x[..., a] * cos - x[..., b] * sin
        y[..., b] = x[..., b] * cos + x[..., a] * sin
        return y

    q, k = turned(s["q"], s["bias"][0], s["norm"][0]), turned(s["k"], s["bias"][1], s["norm"][1])
    v = s["v"].float()
    if s["bias"][2] is not None:
        v = v + s["bias"][2].view(v.shape[1:])
    block, place = s["slots"] // 16, s["slots"] % 16
    for i, x in enumerate((k, v)):
        to = s["cache"][i]
        if s["scales"]:
            x = (x / s["scales"][i][:, None]).clamp(-448, 448)
            to.view(torch.uint8)[block, 0, :, place] = x.to(to.dtype).view(torch.uint8)
        else:
            to[block, 0, :, place] = x.to(to.dtype)
    o = DT[case["out"]]
    return [q.to(o), k.to(o) if case["keep"] else None, v.to(o) if case["keep"] else None, s["cache"]]


def plain_step(s):
    b, ctx, new, tables = s["case"]["block"], s["ctx"].long(), s["new"].long(), s["tables"]
    n = ctx.numel()
    cu = torch.cat([new.new_zeros(1), new.cumsum(0)])
    old = (ctx + b - 1) // b
    opened = (ctx + new + b - 1) // b - old
    first = opened.cumsum(0) - opened
    page = torch.arange(tables.shape[1], device=tables.device)[None] - old[:, None]
    fresh = (page >= 0) & (page < opened[:, None])
    at = (first[:, None] + page).clamp(0, max(0, s["new_blocks"].numel() - 1))
    if s["new_blocks"].numel():
        tables.copy_(torch.where(fresh, s["new_blocks"][at], tables))
    request = torch.repeat_interleave(torch.arange(n, device=tables.device), new, output_size=s["tokens"])
    position = torch.arange(s["tokens"], device=tables.device) - cu[request] + ctx[request]
    slot = tables[request, position // b].long() * b + position % b
    counts = torch.stack([cu[-1], opened.sum()]).int()
    return [tables, (ctx + new).int(), cu.int(), slot, position.int(), counts]


# ---- the definition in 64 bits ----------------------------------------------------------------

def exact(case, seed):
    if case["op"] == "step":
        return None
    s = prepare(case, seed)
    return exact_prompt(s) if case["op"] == "prompt" else exact_rope(s)


def exact_prompt(s):
    case = s["case"]
    group = case["heads"] // case["heads_kv"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(out.shape[:2], dtype=torch.float64, device="cuda")
    for b in range(len(s["cu"]) - 1):
        rows = range(s["cu"][b], s["cu"][b + 1], 2048)
        for h in range(case["heads"]):
            key = s["k"][s["cu"][b]:s["cu"][b + 1], h // group].double()
            value = s["v"][s["cu"][b]:s["cu"][b + 1], h // group].double()
            for i in rows:
                j = min(i + 2048, s["cu"][b + 1])
                seen = torch.arange(i, j, device="cuda")[:, None] >= torch.arange(s["cu"][b], s["cu"][b + 1], device="cuda")[None]
                score = torch.where(seen, s["scale"] * torch.einsum("id,jd->ij", s["q"][i:j, h].double(), key), -math.inf)
                norm = torch.logsumexp(score, 1)
                if s["sinks"] is not None:
                    norm = torch.logaddexp(norm, s["sinks"][h].double())
                lse[i:j, h] = norm
                out[i:j, h] = torch.exp(score - norm[:, None]) @ value
    return [out, lse if case["lse"] else None]


def exact_rope(s):
    case = s["case"]
    half = case["rope_dim"] // 2
    done = []
    for i, name in enumerate(("q", "k", "v")):
        x = s[name].double()
        if s["bias"][i] is not None:
            x = x + s["bias"][i].double().view(1, x.shape[1], x.shape[2])
        if name != "v":
            if s["norm"][i] is not None:
                x = s["norm"][i].double() * x / torch.sqrt((x ** 2).mean(-1, keepdim=True) + s["eps"])
            first = [j if case["style"] == 0 else 2 * j for j in range(half)]
            second = [j + half if case["style"] == 0 else 2 * j + 1 for j in range(half)]
            theta = torch.stack([s["positions"][s["axis"][j]].double() * s["inv_freq"][j] for j in range(half)], 1)
            z = torch.complex(x[..., first], x[..., second]) * torch.polar(torch.ones_like(theta), theta)[:, None]
            x = x.clone()
            x[..., first], x[..., second] = z.real, z.imag
        done.append(x)
    cache = []
    for i in (0, 1):
        to = torch.zeros(s["cache"][i].shape, dtype=torch.float64, device="cuda")
        x = done[i + 1] / s["scales"][i].double()[None, :, None] if s["scales"] else done[i + 1]
        to[s["slots"] // 16, 0, :, s["slots"] % 16] = x.clamp(-448, 448) if s["scales"] else x
        cache.append(to)
    return [done[0], done[1] if case["keep"] else None, done[2] if case["keep"] else None, cache]
