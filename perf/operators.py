"""Cases that measure the decode-serving operators: the 8-bit KV cache, attention over a prefix that a
batch shares, and token sampling.

Each case names one operator (`op`) and its sizes.  `prepare` makes what a serving program holds before the
call, `run` makes one pass, either through the library (`own`) or in plain 32-bit torch, and `exact` gives
the same outputs from the definitions in 64 bits.

Definitions.

Cache.  A row is the head_dim values of one (sequence, kv head, position) of K or of V.  "f16" keeps it
rounded.  The 8-bit formats keep one f32 scale and one byte per value.  With a = max|x| over the row:
  "i8":   scale = a / 127,  byte = 128 + rint(x * (127 / a)),  value = (byte - 128) * scale
  "e4m3": scale = a / 448,  byte = e4m3(x * (448 / a)),        value = e4m3^-1(byte) * scale
A row whose a is under 2^-100 is kept as zeros.

Attention.  T new tokens of each sequence, whose K and V are already the last T of the sequence's own_len
cached positions.  Token t sees all `prefix` positions of a cache that every sequence shares and the own
positions 0 .. own_len - T + t:  out = sum_j p_j v_j,  p = softmax(scale * q . k_j), and 0 where it sees none.

Sampling.  Per row, with m = max(logits) and e_i = exp((l_i - m) / temperature), the tokens ranked by logit
(ties: the lower index first).  Kept are the first top_k of the ranking, of those the shortest leading part
whose mass reaches top_p of theirs, and of those the ones with e_i >= min_p (the first is always kept).
Masses are whole numbers, w_i = rint(e_i * 2^31), so that no order of summation matters.  The token is the
first kept index whose running mass over the kept indices, in index order, exceeds floor(u * mass(kept)); its
probability is w / mass(kept).  Temperature 0 takes the largest logit.
"""
import math
import os
import sys

import torch

own = False

SPAN = 1 << 31  # fixed-point one of the sampling weights
TINY = 2.0 ** -100

_backend = None


def _library():
    """The binding and one backend on torch's default stream (handle 1 is CUDA's name for it)."""
    global _backend
    pkg = os.path.join(os.getcwd(), "universal-ai-inference_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import uaii_moe as um
    if _backend is None:
        _backend = um.Backend(0, stream=1)
    return um, _backend


# ---------------------------------------------------------------- cases


def listed():
    return [
        # one decode step of 32 sequences near 4096 positions: K and V straight out of the fused q/k/v
        # projection into the int8 cache, and the written rows back as attention will see them
        dict(name="cache_step_i8", op="cache", fmt="i8", dtype="f32", batch=32, tokens=1, kv_heads=8, q_heads=32,
             head_dim=128, at=4095, read_from=4095, read=1, out="f32", ragged=0),
        # the first 4096 tokens of four prompts of unequal length written to an e4m3 cache and read back in f16
        dict(name="cache_prompt_e4m3", op="cache", fmt="e4m3", dtype="f16", batch=4, tokens=4096, kv_heads=8,
             q_heads=0, head_dim=128, at=0, read_from=0, read=4096, out="f16", ragged=1),
        # a chunk appended to a long int8 cache, then the whole context read back for a full-precision pass
        dict(name="cache_context_i8", op="cache", fmt="i8", dtype="f32", batch=16, tokens=129, kv_heads=4,
             q_heads=32, head_dim=64, at=8000, read_from=0, read=8129, out="f16", ragged=0),
        # one sequence, one token, a short f16 cache: latency
        dict(name="attend_one_f16", op="attend", fmt="f16", dtype="f32", batch=1, tokens=1, heads=32, kv_heads=8,
             head_dim=128, prefix=0, own=777, spread=0),
        # a decode step of 32 sequences around 4096 positions on the int8 cache, nothing shared: the cache's bytes
        dict(name="attend_batch_i8", op="attend", fmt="i8", dtype="f32", batch=32, tokens=1, heads=32, kv_heads=8,
             head_dim=128, prefix=0, own=4096, spread=64),
        # 64 conversations behind one 8192-token system prompt
        dict(name="attend_shared_i8", op="attend", fmt="i8", dtype="f16", batch=64, tokens=1, heads=32, kv_heads=8,
             head_dim=128, prefix=8192, own=512, spread=500),
        # four drafted tokens of 24 sequences, seven query heads per kv head, head_dim 64, an odd prefix
        dict(name="attend_draft_e4m3", op="attend", fmt="e4m3", dtype="f32", batch=24, tokens=4, heads=28, kv_heads=4,
             head_dim=64, prefix=4101, own=300, spread=290),
        # 128 samples of one long document: the prefix is arithmetic, not memory
        dict(name="attend_document_i8", op="attend", fmt="i8", dtype="f16", batch=128, tokens=1, heads=32, kv_heads=8,
             head_dim=128, prefix=32801, own=256, spread=255),
        # one sequence's next token: latency
        dict(name="sample_one", op="sample", dtype="f32", batch=1, vocab=32000, temperature=0.8, top_k=40, top_p=0.95,
             min_p=0.05, mixed=0),
        # a decode step's 32 sequences, each with its own settings (greedy ones among them)
        dict(name="sample_batch", op="sample", dtype="f32", batch=32, vocab=32000, temperature=1.0, top_k=50,
             top_p=0.9, min_p=0.02, mixed=1),
        # a large batch over a large vocabulary with f16 logits and a nucleus alone
        dict(name="sample_wide_f16", op="sample", dtype="f16", batch=256, vocab=151936, temperature=0.9, top_k=0,
             top_p=0.92, min_p=0.0, mixed=0),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, uniform in its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        cost = max(w["bytes"], w["flops"] / 250)
        most[c["op"]] = max(most.get(c["op"], 0), cost)
    op = rng.choice(["cache", "attend", "attend", "sample"])
    while True:
        if op == "cache":
            tokens = _spread(rng, 1, 4096)
            at = rng.choice([0, _spread(rng, 1, 8000)])
            start = rng.choice([0, at, max(0, at - 3)])
            c = dict(op=op, fmt=rng.choice(["i8", "e4m3", "f16"]), dtype=rng.choice(["f32", "f16"]),
                     batch=_spread(rng, 1, 64), tokens=tokens, kv_heads=rng.choice([1, 2, 4, 8]),
                     q_heads=rng.choice([0, 8, 32]), head_dim=rng.choice([64, 128]), at=at, read_from=start,
                     read=at + tokens - start, out=rng.choice(["f32", "f16"]), ragged=rng.choice([0, 1]))
        elif op == "attend":
            kv = rng.choice([1, 2, 4, 8])
            mine = _spread(rng, 16, 4096)
            c = dict(op=op, fmt=rng.choice(["i8", "e4m3", "f16"]), dtype=rng.choice(["f32", "f16"]),
                     batch=_spread(rng, 1, 128), tokens=rng.choice([1, 1, 1, 2, 4, 5, 16]),
                     heads=kv * rng.choice([1, 2, 3, 4, 6, 7, 8]), kv_heads=kv, head_dim=rng.choice([64, 128, 128]),
                     prefix=rng.choice([0, _spread(rng, 1, 33000), _spread(rng, 1, 33000)]), own=mine,
                     spread=rng.randrange(0, mine))
        else:
            c = dict(op=op, dtype=rng.choice(["f32", "f16"]), batch=_spread(rng, 1, 256),
                     vocab=_spread(rng, 1000, 152000), temperature=round(rng.uniform(0.5, 1.5), 2),
                     top_k=rng.choice([0, _spread(rng, 1, 1000)]), top_p=rng.choice([1.0, round(rng.uniform(0.3, 0.99), 2)]),
                     min_p=rng.choice([0.0, round(rng.uniform(0.001, 0.2), 3)]), mixed=rng.choice([0, 1]))
        w = work(c)
        if max(w["bytes"], w["flops"] / 250) <= most[op]:
            return c


def _row_bytes(c):
    return 2 * c["head_dim"] if c["fmt"] == "f16" else c["head_dim"] + 4


def _counts(c):
    """New tokens of each sequence of a cache case."""
    b, t = c["batch"], c["tokens"]
    return [max(1, t - (i * 997) % max(1, t // 2)) if c["ragged"] else t for i in range(b)]


def _lens(c):
    """Own positions of each sequence of an attention case."""
    return [max(1, c["own"] - (i * 389) % (c["spread"] + 1)) for i in range(c["batch"])]


def work(case):
    c = case
    size = {"f32": 4, "f16": 2}[c["dtype"]]
    if c["op"] == "cache":
        new = 2 * c["kv_heads"] * sum(_counts(c))
        seen = 2 * c["kv_heads"] * c["batch"] * c["read"]
        out = {"f32": 4, "f16": 2}[c["out"]]
        return {"bytes": new * (c["head_dim"] * size + _row_bytes(c)) + seen * (_row_bytes(c) + c["head_dim"] * out),
                "flops": 2 * c["head_dim"] * (new + seen)}
    if c["op"] == "attend":
        lens = _lens(c)
        rows = c["batch"] * c["tokens"] * c["heads"]
        pairs = rows * c["prefix"] + c["heads"] * sum(max(0, n - c["tokens"] + t + 1) for n in lens
                                                      for t in range(c["tokens"]))
        return {"bytes": 2 * rows * c["head_dim"] * size + 2 * c["kv_heads"] * _row_bytes(c) * (c["prefix"] + sum(lens)),
                "flops": 4 * pairs * c["head_dim"]}
    return {"bytes": c["batch"] * (c["vocab"] * size + 32), "flops": 4 * c["batch"] * c["vocab"]}


# ---------------------------------------------------------------- inputs


def _dtype(name):
    return {"f32": torch.float32, "f16": torch.float16}[name]


def _encode(x, fmt):
    """Rows of f32 values -> (bytes or halves, scale or None)."""
    if fmt == "f16":
        return x.to(torch.float16), None
    a = x.abs().amax(-1, keepdim=True)
    top = torch.full_like(a, 127.0 if fmt == "i8" else 448.0)
    fine = a >= TINY
    scale = torch.where(fine, a / top, torch.zeros_like(a))
    y = x * torch.where(fine, top / a, torch.zeros_like(a))
    code = (torch.round(y) + 128).to(torch.uint8) if fmt == "i8" else y.to(torch.float8_e4m3fn).view(torch.uint8)
    return code, scale.squeeze(-1)


def _decode(code, scale, fmt):
    """(bytes or halves, scale) -> f32 values."""
    if fmt == "f16":
        return code.float()
    v = code.float() - 128 if fmt == "i8" else code.view(torch.float8_e4m3fn).float()
    return v * scale.unsqueeze(-1)


def _kv(gen, fmt, b, h, s, d):
    """A filled cache: K with a few strong channels, as keys have, and V; bytes and scales."""
    channel = torch.exp(0.5 * torch.randn((1, h, 1, d), generator=gen, device="cuda"))
    cache = {}
    for name in ("k", "v"):
        x = torch.randn((b, h, s, d), generator=gen, device="cuda")
        if name == "k":
            x *= channel
        cache[name], cache[name + "_scale"] = _encode(x, fmt)
    return cache


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)
    state = {"case": c}
    if c["op"] == "cache":
        b, t, h, d = c["batch"], c["tokens"], c["kv_heads"], c["head_dim"]
        size = c["at"] + t + 3
        state["cache"] = _kv(gen, c["fmt"], b, h, size, d)
        wide = (c["q_heads"] + 2 * h) * d  # q | k | v of one projection; without q heads K and V alone
        qkv = torch.randn((b, t, wide), generator=gen, device="cuda").to(_dtype(c["dtype"]))
        split = c["q_heads"] * d
        state["k"] = qkv[..., split:split + h * d].unflatten(-1, (h, d))
        state["v"] = qkv[..., split + h * d:].unflatten(-1, (h, d))
        state["pos"] = torch.tensor([c["at"] + (i % 3 if c["ragged"] else 0) for i in range(b)], dtype=torch.int32,
                                    device="cuda")
        state["count"] = torch.tensor(_counts(c), dtype=torch.int32, device="cuda")
        for name in ("k_out", "v_out"):
            state[name] = torch.empty((b, h, c["read"], d), dtype=_dtype(c["out"]), device="cuda")
    elif c["op"] == "attend":
        b, t, hq, h, d = c["batch"], c["tokens"], c["heads"], c["kv_heads"], c["head_dim"]
        state["cache"] = _kv(gen, c["fmt"], b, h, c["own"] + 5, d)
        if c["prefix"]:
            state["prefix"] = _kv(gen, c["fmt"], 1, h, c["prefix"] + 2, d)
        state["lens"] = torch.tensor(_lens(c), dtype=torch.int32, device="cuda")
        state["q"] = torch.randn((b, t, hq, d), generator=gen, device="cuda").to(_dtype(c["dtype"]))
        state["out"] = torch.empty((b, t, hq, d), dtype=_dtype(c["dtype"]), device="cuda")
    else:
        b, v = c["batch"], c["vocab"]
        x = 3.0 * torch.randn((b, v), generator=gen, device="cuda")
        banned = torch.rand((b, v), generator=gen, device="cuda") < 0.01  # tokens a grammar forbids
        state["logits"] = x.masked_fill(banned, float("-inf")).to(_dtype(c["dtype"]))
        f = lambda v: torch.full((b,), float(v), device="cuda")  # noqa: E731
        state["temperature"], state["top_p"], state["min_p"] = f(c["temperature"]), f(c["top_p"]), f(c["min_p"])
        state["top_k"] = torch.full((b,), c["top_k"], dtype=torch.int32, device="cuda")
        if c["mixed"]:  # sequences of several callers: greedy ones, and ones without each of the cuts
            i = torch.arange(b, device="cuda")
            state["temperature"][i % 5 == 4] = 0.0
            state["top_k"][i % 4 == 1] = 0
            state["top_p"][i % 3 == 2] = 1.0
            state["min_p"][i % 2 == 1] = 0.0
        state["u"] = torch.rand((b,), generator=gen, device="cuda")
        state["tokens"] = torch.empty((b,), dtype=torch.int32, device="cuda")
        state["kept"] = torch.empty((b,), dtype=torch.int32, device="cuda")
        state["probs"] = torch.empty((b,), device="cuda")
    return state


# ---------------------------------------------------------------- one pass


def run(state):
    return (_run_own if own else _run_plain)(state)


def _handle(um, state, name):
    """The library's description of a cache, made once as a serving program does."""
    key = "handle_" + name
    if key not in state:
        x = state[name]
        fmt = {"f16": um.F16, "i8": um.KV_I8, "e4m3": um.KV_E4M3}[state["case"]["fmt"]]
        state[key] = um.kv_cache(fmt, x["k"], x["v"], x["k_scale"], x["v_scale"])
    return state[key]


def _run_own(state):
    um, be = _library()
    c = state["case"]
    if c["op"] == "cache":
        cache = _handle(um, state, "cache")
        be.kv_append(cache, state["k"], state["v"], state["pos"], state["count"])
        be.kv_read(cache, c["read_from"], c["read"], state["k_out"], state["v_out"])
        return {"k": state["k_out"], "v": state["v_out"], **_scales(state)}
    if c["op"] == "attend":
        prefix = _handle(um, state, "prefix") if c["prefix"] else None
        be.prefix_attention(state["q"], _handle(um, state, "cache"), state["lens"], state["out"], prefix=prefix,
                            prefix_len=c["prefix"])
        return state["out"]
    be.sample(state["logits"], state["temperature"], state["top_k"], state["top_p"], state["min_p"], state["u"],
              state["tokens"], state["probs"], state["kept"])
    return {"tokens": state["tokens"], "probs": state["probs"], "kept": state["kept"]}


def _scales(state):
    x = state["cache"]
    return {} if x["k_scale"] is None else {"k_scale": x["k_scale"], "v_scale": x["v_scale"]}


def _run_plain(state):
    return {"cache": _plain_cache, "attend": _plain_attend, "sample": _plain_sample}[state["case"]["op"]](state)


def _plain_write(state, name):
    x, b = state["cache"], state["case"]["batch"]
    code, scale = _encode(state[name].float(), state["case"]["fmt"])
    t = torch.arange(state["case"]["tokens"], device="cuda")
    seq, tok = torch.nonzero(t < state["count"][:, None], as_tuple=True)
    at = state["pos"].long()[seq] + tok
    x[name][seq, :, at] = code[seq, tok]
    if scale is not None:
        x[name + "_scale"][seq, :, at] = scale[seq, tok]


def _plain_read(state, name):
    c, x = state["case"], state["cache"]
    part = slice(c["read_from"], c["read_from"] + c["read"])
    scale = x[name + "_scale"]
    return _decode(x[name][:, :, part], None if scale is None else scale[:, :, part], c["fmt"]).to(_dtype(c["out"]))


def _plain_cache(state):
    _plain_write(state, "k")
    _plain_write(state, "v")
    return {"k": _plain_read(state, "k"), "v": _plain_read(state, "v"), **_scales(state)}


def _plain_attend(state):
    c = state["case"]
    b, t, hq, h, d = c["batch"], c["tokens"], c["heads"], c["kv_heads"], c["head_dim"]
    values = lambda x, n: _decode(x[n], x[n + "_scale"], c["fmt"])  # noqa: E731
    q = state["q"].float().view(b, t, h, hq // h, d) * (1.0 / math.sqrt(d))
    k, v = values(state["cache"], "k"), values(state["cache"], "v")
    s = torch.einsum("bthgd,bhjd->bthgj", q, k)
    last = state["lens"][:, None] - t + torch.arange(t, device="cuda")
    seen = torch.arange(k.shape[2], device="cuda") <= last[..., None]
    s = s.masked_fill(~seen[:, :, None, None, :], float("-inf"))
    if c["prefix"]:
        pk, pv = values(state["prefix"], "k")[0, :, :c["prefix"]], values(state["prefix"], "v")[0, :, :c["prefix"]]
        s = torch.cat([torch.einsum("bthgd,hjd->bthgj", q, pk), s], -1)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == float("-inf"), torch.zeros_like(m), m))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    out = torch.einsum("bthgj,bhjd->bthgd", p[..., c["prefix"]:], v)
    if c["prefix"]:
        out = out + torch.einsum("bthgj,hjd->bthgd", p[..., :c["prefix"]], pv)
    return out.reshape(b, t, hq, d).to(_dtype(c["dtype"]))


def _plain_sample(state):
    x = state["logits"].float()
    n = x.shape[1]
    top = x.amax(1, keepdim=True)
    greedy = state["temperature"] == 0
    heat = torch.where(greedy, torch.ones_like(state["temperature"]), state["temperature"])[:, None]
    e = torch.exp((x - top) / heat)
    w = torch.round(e * SPAN).to(torch.int64)
    _, order = torch.sort(x, dim=1, descending=True, stable=True)
    rank = torch.arange(n, device="cuda")
    limit = torch.where(state["top_k"] > 0, state["top_k"], torch.full_like(state["top_k"], n))
    limit = torch.where(greedy, torch.ones_like(limit), limit)[:, None]
    ranked = torch.where(rank < limit, w.gather(1, order), torch.zeros_like(w))
    mass = ranked.cumsum(1)
    reach = torch.ceil(state["top_p"].double()[:, None] * mass[:, -1:].double())
    nucleus = ((mass - ranked).double() < reach) | (state["top_p"][:, None] >= 1)
    keep = (rank < limit) & nucleus & (e.gather(1, order) >= state["min_p"][:, None]) | (rank == 0)
    kept = torch.zeros_like(keep).scatter_(1, order, keep)
    run_mass = torch.where(kept, w, torch.zeros_like(w)).cumsum(1)
    total = run_mass[:, -1:]
    goal = torch.minimum(torch.floor(state["u"].double()[:, None] * total.double()).to(torch.int64), total - 1)
    token = (run_mass <= goal).sum(1, keepdim=True)
    p = w.gather(1, token).double() / total.double()
    return {"tokens": token[:, 0].to(torch.int32), "probs": p[:, 0].float(), "kept": kept.sum(1).to(torch.int32)}


# ---------------------------------------------------------------- the same in 64 bits


def _exact_values(x, name, fmt):
    if fmt == "f16":
        return x[name].double()
    code = x[name].double() - 128.0 if fmt == "i8" else x[name].view(torch.float8_e4m3fn).float().double()
    return code * x[name + "_scale"].double()[..., None]


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "cache":
        return _exact_cache(case, state)
    return _exact_attend(case, state) if case["op"] == "attend" else _exact_sample(case, state)


def _exact_cache(c, state):
    """The scale of a written row in 64 bits, and each value's nearest multiple of it (e4m3: nearest e4m3 value)."""
    got = {}
    for name in ("k", "v"):
        values = _exact_values(state["cache"], name, c["fmt"])
        scales = None if c["fmt"] == "f16" else state["cache"][name + "_scale"].double()
        for i, (at, n) in enumerate(zip(state["pos"].tolist(), state["count"].tolist())):
            rows = state[name][i, :n].double().transpose(0, 1)
            if c["fmt"] == "f16":
                values[i, :, at:at + n] = rows.half().double()
                continue
            largest = rows.abs().max(-1).values
            unit = largest / (127.0 if c["fmt"] == "i8" else 448.0)
            y = rows / unit[..., None]
            if c["fmt"] == "i8":
                y = torch.round(y)
            else:  # the spacing of the value's binade (3 mantissa bits), the same below 2^-6
                step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
                y = torch.round(y / step) * step
            values[i, :, at:at + n] = y * unit[..., None]
            scales[i, :, at:at + n] = unit
        got[name] = values[:, :, c["read_from"]:c["read_from"] + c["read"]].contiguous()
        if scales is not None:
            got[name + "_scale"] = scales
    return got


def _exact_attend(c, state):
    b, t, hq, h, d = c["batch"], c["tokens"], c["heads"], c["kv_heads"], c["head_dim"]
    g = hq // h
    out = torch.zeros((b, t, hq, d), dtype=torch.float64, device="cuda")
    if c["prefix"]:
        pk, pv = (_exact_values(state["prefix"], n, c["fmt"])[0, :, :c["prefix"]] for n in ("k", "v"))
    for i, n in enumerate(state["lens"].tolist()):
        k, v = (_exact_values({m: (x if x is None else x[i, :, :n]) for m, x in state["cache"].items()}, w, c["fmt"])
                for w in ("k", "v"))
        if c["prefix"]:
            k, v = torch.cat([pk, k], 1), torch.cat([pv, v], 1)
        for j in range(t):
            see = c["prefix"] + max(0, n - t + j + 1)
            if see:
                q = state["q"][i, j].double().view(h, g, d)
                p = torch.softmax(q @ k[:, :see].transpose(1, 2) / math.sqrt(d), -1)
                out[i, j] = (p @ v[:, :see]).reshape(hq, d)
    return out


def _exact_sample(c, state):
    """Row by row from the definition; the tokens and counts are whole numbers, held to equality elsewhere."""
    probs = torch.empty((c["batch"],), dtype=torch.float64)
    setting = [state[n].tolist() for n in ("temperature", "top_k", "top_p", "min_p", "u")]
    for i, (heat, k, p, least, u) in enumerate(zip(*setting)):
        if heat == 0:
            probs[i] = 1.0
            continue
        x = state["logits"][i].double()
        e = torch.exp((x - x.max()) / heat)
        w = torch.round(e * SPAN)
        order = torch.argsort(-x, stable=True)
        if k > 0:
            order = order[:k]
        if p < 1:
            before = torch.cumsum(w[order], 0) - w[order]
            order = order[before < math.ceil(p * float(w[order].sum()))]
        strong = order[e[order] >= least]
        order = strong if len(strong) else order[:1]
        index = torch.sort(order).values
        mass = torch.cumsum(w[index], 0)
        goal = min(math.floor(u * float(mass[-1])), float(mass[-1]) - 1)
        probs[i] = float(w[index][int((mass <= goal).sum())] / mass[-1])
    return {"tokens": None, "probs": probs, "kept": None}
