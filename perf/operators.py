"""The workload of the serving operators around the paged KV cache, for timing and comparison.

Three operators are called one after the other for every layer of a served batch:

* ``qk_norm_rope``: RMSNorm of every query and key head and the rotation of its position, in one
  pass (for a packed prefill that keeps no cache);
* ``rope_paged_kv_append``: the same on the way into the paged cache: keys are normalised, rotated
  and stored (as they are, or as e4m3 codes) in their slots, values are stored beside them, and the
  rotated queries come back;
* ``paged_prefill_attention``: causal attention of each request's chunk of new tokens (one token
  when it decodes, a few when drafts are checked, thousands when it prefills) over its paged cache.

With ``own`` false, ``run`` computes them with elementary torch operations in 32 bits; with ``own``
true it calls this repository's operators.  ``exact`` follows the definitions in 64 bits.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6
E4M3_MAX = 448.0


# ------------------------------------------------------------------------------------------ cases
def _norm_rope(name, tokens, heads, kv_heads, dim, rotary, dtype="bf16", norm=True, interleaved=False):
    return {"op": "norm_rope", "name": name, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "rotary": rotary, "dtype": dtype, "norm": norm, "interleaved": interleaved}


def _append(name, tokens, heads, kv_heads, dim, rotary, block, blocks, dtype="bf16", e4m3=False, norm=False,
            interleaved=False, padded=0):
    return {"op": "append", "name": name, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "rotary": rotary, "block": block, "blocks": blocks, "dtype": dtype, "e4m3": e4m3, "norm": norm,
            "interleaved": interleaved, "padded": padded}


def _attend(name, requests, chunk, context, heads, kv_heads, dim, block, dtype="bf16", e4m3=False, lse=False,
            shape="even", mix=0):
    """``shape`` says how the requests' lengths go: "even" (all of ``chunk`` new tokens on ``context`` tokens in the
    cache, the new ones included), "ragged" (contexts from a sixteenth up to ``context``, chunks up to ``chunk``), or
    "mixed" (every fourth request brings a ragged chunk, the others decode one token)."""
    return {"op": "attend", "name": name, "requests": requests, "chunk": chunk, "context": context, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "block": block, "dtype": dtype, "e4m3": e4m3, "lse": lse, "shape": shape,
            "mix": mix}


def listed():
    return [
        # one decode step of a small batch before a dense attention: latency counts
        _norm_rope("norm_rope_step", 8, 32, 8, 128, 128),
        # the queries and keys of a long packed prefill
        _norm_rope("norm_rope_prefill", 8192, 32, 8, 128, 128),
        # heads of which half is rotated, neighbouring elements paired, no norm, odd counts
        _norm_rope("norm_rope_partial", 1021, 9, 3, 80, 40, dtype="fp16", norm=False, interleaved=True),
        # one decode step of 64 sequences into the e4m3 cache
        _append("append_step_e4m3", 64, 32, 8, 128, 128, 16, 4096, e4m3=True),
        # a chunk of 4096 prompt tokens, normalised, into a bf16 cache
        _append("append_chunk_bf16", 4096, 32, 8, 128, 128, 16, 1024, norm=True),
        # a padded batch, pages of 20 tokens, half of each head rotated
        _append("append_padded_fp16", 1003, 12, 4, 64, 32, 20, 200, dtype="fp16", interleaved=True, padded=37),
        # two requests that check four drafted tokens each on a short cache: latency counts
        _attend("attend_draft", 2, 4, 1000, 32, 8, 128, 16, lse=True),
        # one decode step of 64 sequences of 512 to 8192 tokens over the e4m3 cache
        _attend("attend_step_e4m3", 64, 1, 8192, 32, 8, 128, 16, e4m3=True, shape="ragged"),
        # a batch that decodes and prefills at once
        _attend("attend_mixed", 16, 400, 4100, 32, 8, 128, 16, shape="mixed"),
        # the last chunk of a long prompt
        _attend("attend_chunk_bf16", 1, 2048, 16384, 32, 8, 128, 16),
        # chunks of four prompts over the e4m3 cache
        _attend("attend_chunk_e4m3", 4, 512, 4096, 32, 8, 128, 16, e4m3=True),
        # float32 throughout, pages of 12 tokens, contexts shorter than their chunk
        _attend("attend_fp32", 5, 130, 700, 6, 2, 64, 12, dtype="fp32", lse=True, shape="ragged", mix=3),
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], even over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def _drop_name(case):
    return {k: v for k, v in case.items() if k != "name"}


def draw(rng):
    op = rng.choice(("norm_rope", "append", "attend", "attend"))
    kv_heads = rng.choice((1, 2, 3, 4, 8))
    heads = kv_heads * rng.choice((1, 2, 3, 4, 5, 7, 8))
    dim = rng.choice((64, 80, 96, 128, 128))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    if op != "attend":
        rotary = rng.choice((dim, dim, dim // 2))
        most = 8192 * 40 * 128 // ((heads + 2 * kv_heads) * dim)
        tokens = _spread(rng, 1, min(9000, most))
        norm, interleaved = rng.random() < 0.5, rng.random() < 0.3
        if op == "norm_rope":
            return _drop_name(_norm_rope("", tokens, heads, kv_heads, dim, rotary, dtype, norm, interleaved))
        block = rng.choice((8, 12, 16, 20, 32, 64, 128))
        padded = rng.choice((0, tokens // 9))
        blocks = tokens // block + _spread(rng, 1, 400)
        return _drop_name(_append("", tokens, heads, kv_heads, dim, rotary, block, blocks, dtype, rng.random() < 0.5, norm,
                                  interleaved, padded))
    block = rng.choice((8, 12, 16, 16, 20, 32, 64, 128))
    context = _spread(rng, 1, 8192 if dtype != "fp32" else 2048)
    requests = _spread(rng, 1, 64)
    most = (1 << 28) // (heads * context * requests)          # padded scores of the plain form
    chunk = _spread(rng, 1, max(1, min(1500 if dtype != "fp32" else 300, context, most)))
    return _drop_name(_attend("", requests, chunk, context, heads, kv_heads, dim, block, dtype, rng.random() < 0.5,
                              rng.random() < 0.3, rng.choice(("even", "ragged", "ragged", "mixed")),
                              rng.randrange(1 << 20)))


def _lengths(case):
    """(new tokens, tokens in the cache with them) of every request: the case's own, whatever the seed."""
    rng = random.Random(case["mix"])
    chunks, contexts = [], []
    for i in range(case["requests"]):
        if case["shape"] == "even":
            chunk, context = case["chunk"], case["context"]
        else:
            context = _spread(rng, max(1, case["context"] // 16), case["context"])
            chunk = _spread(rng, max(1, case["chunk"] // 16), case["chunk"])
            if case["shape"] == "mixed" and i % 4:
                chunk = 1
        chunks.append(chunk)
        contexts.append(context)
    return chunks, contexts


def work(case):
    size = DTYPES[case["dtype"]].itemsize
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "attend":
        chunks, contexts = _lengths(case)
        held = 1 if case["e4m3"] else size
        pairs = sum(max(0, c - n + i + 1) for n, c in zip(chunks, contexts) for i in range(n))
        pages = sum(-(-c // case["block"]) for c in contexts)
        return {"bytes": 2 * sum(chunks) * hq * d * size + 2 * sum(contexts) * hk * d * held + 4 * pages
                + 8 * case["requests"] + (4 * sum(chunks) * hq if case["lse"] else 0), "flops": 4 * pairs * hq * d}
    t, r = case["tokens"], case["rotary"]
    flops = t * (hq + hk) * (3 * r + (4 * d if case["norm"] else 0))
    weights = 2 * d * size if case["norm"] else 0
    if case["op"] == "norm_rope":
        return {"bytes": t * (2 * (hq + hk) * d * size + 4 * r + 8) + weights, "flops": flops}
    live, held = t - case["padded"], 1 if case["e4m3"] else size
    return {"bytes": t * (2 * hq * d * size + 16) + t * 4 * r + live * 2 * hk * d * (size + held) + weights
            + (8 * hk if case["e4m3"] else 0), "flops": flops}


# ------------------------------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _table(positions, rotary):
    """cos and sin of every position, [positions, rotary]: the angles in 64 bits, rounded once."""
    inverse = 10000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device="cuda") / rotary)
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * inverse
    return torch.cat((angle.cos(), angle.sin()), 1).float()


def _scales(g, n):
    return torch.rand((n,), generator=g, device="cuda") * 0.01 + 0.005


def _cache(g, shape, dtype, scale):
    """Values that a cache holds; with ``scale``, as e4m3 codes."""
    x = torch.randn(shape, generator=g, device="cuda")
    if scale is None:
        return x.to(dtype)
    return (x / scale[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)


def prepare(case, seed):
    g = _generator(seed)
    dtype, hq, hk, d = DTYPES[case["dtype"]], case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "attend":
        chunks, contexts = _lengths(case)
        pages = [-(-c // case["block"]) for c in contexts]
        total = sum(pages) + 3
        free = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
        table = torch.zeros((len(pages), max(pages)), dtype=torch.int32, device="cuda")
        at = 0
        for i, n in enumerate(pages):
            table[i, :n] = free[at:at + n]
            at += n
        starts = [0]
        for n in chunks:
            starts.append(starts[-1] + n)
        ks, vs = (_scales(g, hk), _scales(g, hk)) if case["e4m3"] else (None, None)
        shape = (total, case["block"], hk, d)
        return {"case": case, "q": _normal(g, (starts[-1], hq, d), dtype), "k_cache": _cache(g, shape, dtype, ks),
                "v_cache": _cache(g, shape, dtype, vs), "k_scale": ks, "v_scale": vs, "table": table,
                "starts": torch.tensor(starts, dtype=torch.int32, device="cuda"),
                "lens": torch.tensor(contexts, dtype=torch.int32, device="cuda"), "scale": d ** -0.5,
                "longest": max(chunks), "context": max(contexts)}
    t = case["tokens"]
    fused = _normal(g, (t, (hq + 2 * hk) * d), dtype)          # one projection's output: q, k and v are views of it
    state = {"case": case, "q": fused[:, :hq * d].view(t, hq, d), "k": fused[:, hq * d:(hq + hk) * d].view(t, hk, d),
             "v": fused[:, (hq + hk) * d:].view(t, hk, d), "cos_sin": _table(16384, case["rotary"]),
             "positions": torch.randint(0, 16384, (t,), generator=g, device="cuda"),
             "q_weight": _normal(g, (d,), dtype, 0.1) + 1 if case["norm"] else None,
             "k_weight": _normal(g, (d,), dtype, 0.1) + 1 if case["norm"] else None}
    if case["op"] == "append":
        ks, vs = (_scales(g, hk), _scales(g, hk)) if case["e4m3"] else (None, None)
        shape = (case["blocks"], case["block"], hk, d)
        slots = torch.randperm(case["blocks"] * case["block"], generator=g, device="cuda")[:t]
        if case["padded"]:
            slots[-case["padded"]:] = -1
        state.update({"k_cache": _cache(g, shape, dtype, ks), "v_cache": _cache(g, shape, dtype, vs), "k_scale": ks,
                      "v_scale": vs, "slots": slots})
    return state


# ------------------------------------------------------------------------------------------ the plain forms
def _plain_norm_rope(x, weight, cos_sin, positions, interleaved):
    """One head's RMSNorm (where it has a weight) and rotation, in 32 bits and not rounded."""
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
    half = cos_sin.shape[1] // 2
    rows = cos_sin[positions][:, None, :]
    cos, sin = rows[..., :half], rows[..., half:]
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, x[..., 2 * half:]), -1)


def _plain_store(cache, slots, x, scale):
    if scale is not None:
        x = (x / scale[:, None]).clamp(-E4M3_MAX, E4M3_MAX)
    live = slots >= 0
    tokens = torch.arange(slots.shape[0], device=slots.device)
    tokens = torch.where(live, tokens, live.int().argmax())     # a token without a slot repeats the first one's store
    rows = cache.view(-1, *cache.shape[2:])
    if scale is not None:                                       # codes move as bytes
        rows.view(torch.uint8)[slots[tokens]] = x.to(cache.dtype).view(torch.uint8)[tokens]
    else:
        rows[slots[tokens]] = x.to(cache.dtype)[tokens]


def _plain_attend(s):
    """All requests at once, padded to the longest chunk and the longest context."""
    q, starts, lens = s["q"], s["starts"].long(), s["lens"].long()
    hk, d = s["k_cache"].shape[2:]
    block, group = s["k_cache"].shape[1], q.shape[1] // hk
    batch, most, context = lens.shape[0], s["longest"], s["context"]
    row = torch.arange(most, device=q.device)
    key = torch.arange(context, device=q.device)
    count = starts[1:] - starts[:-1]
    rows = torch.minimum(starts[:-1, None] + row, starts[-1] - 1)
    slots = s["table"].long()[:, key // block] * block + key % block

    def gathered(cache, scale):
        flat = cache.view(-1, hk, d)
        x = flat.view(torch.uint8)[slots].view(torch.float8_e4m3fn).float() if scale is not None else flat[slots].float()
        return (x * scale[:, None] if scale is not None else x).permute(0, 2, 1, 3)            # [batch, hk, context, d]

    k, v = gathered(s["k_cache"], s["k_scale"]), gathered(s["v_cache"], s["v_scale"])
    x = q[rows].float().view(batch, most, hk, group, d).permute(0, 2, 3, 1, 4).reshape(batch, hk, group * most, d)
    scores = (x @ k.transpose(2, 3) * s["scale"]).view(batch, hk, group, most, context)
    seen = key <= (lens - count)[:, None, None] + row[:, None]                                 # [batch, most, context]
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p.view(batch, hk, group * most, context) @ v).view(batch, hk, group, most, d)
    out = torch.where(total > 0, out / total, 0.0)
    place = starts[:-1, None] + row
    place = torch.where(row < count[:, None], place, q.shape[0]).flatten()                     # what pads goes behind the last row
    packed = torch.zeros((q.shape[0] + 1, *q.shape[1:]), device=q.device)
    packed[place] = out.permute(0, 3, 1, 2, 4).reshape(batch * most, hk * group, d)
    packed = packed[:-1].to(q.dtype)
    if not s["case"]["lse"]:
        return packed
    lse = torch.zeros((q.shape[0] + 1, q.shape[1]), device=q.device)
    lse[place] = (top + total.log()).squeeze(-1).permute(0, 3, 1, 2).reshape(batch * most, hk * group)
    return packed, lse[:-1]


def run(state):
    s, case = state, state["case"]
    if own:
        from kernelverse_b200 import ops

        if case["op"] == "attend":
            return ops.paged_prefill_attention(s["q"], s["k_cache"], s["v_cache"], s["starts"], s["lens"], s["table"],
                                               s["scale"], k_scale=s["k_scale"], v_scale=s["v_scale"],
                                               max_seq_len=s["context"], return_lse=case["lse"])
        if case["op"] == "norm_rope":
            return ops.qk_norm_rope(s["q"], s["k"], s["positions"], s["cos_sin"], s["q_weight"], s["k_weight"], EPS,
                                    interleaved=case["interleaved"])
        q = ops.rope_paged_kv_append(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"], s["positions"],
                                     s["cos_sin"], k_scale=s["k_scale"], v_scale=s["v_scale"], q_weight=s["q_weight"],
                                     k_weight=s["k_weight"], eps=EPS, interleaved=case["interleaved"])
        return q, s["k_cache"], s["v_cache"]
    if case["op"] == "attend":
        return _plain_attend(s)
    dtype = s["q"].dtype
    q = _plain_norm_rope(s["q"], s["q_weight"], s["cos_sin"], s["positions"], case["interleaved"]).to(dtype)
    k = _plain_norm_rope(s["k"], s["k_weight"], s["cos_sin"], s["positions"], case["interleaved"])
    if case["op"] == "norm_rope":
        return q, k.to(dtype)
    _plain_store(s["k_cache"], s["slots"], k, s["k_scale"])
    _plain_store(s["v_cache"], s["slots"], s["v"].float(), s["v_scale"])
    return q, s["k_cache"], s["v_cache"]


# ------------------------------------------------------------------------------------------ from the definitions, in 64 bits
def _exact_heads(x, weight, s):
    """y_i = x_i w_i / sqrt(mean x^2 + eps); the pair (i, j) of angle a becomes (y_i cos a - y_j sin a, y_i sin a + y_j cos a)."""
    y = x.double()
    if weight is not None:
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + EPS) * weight.double()
    out = y.clone()
    half = s["case"]["rotary"] // 2
    rows = s["cos_sin"].double().index_select(0, s["positions"])
    for n in range(half):
        i, j = (2 * n, 2 * n + 1) if s["case"]["interleaved"] else (n, n + half)
        c, z = rows[:, n, None], rows[:, half + n, None]
        out[..., i] = y[..., i] * c - y[..., j] * z
        out[..., j] = y[..., i] * z + y[..., j] * c
    return out


def _exact_cache(cache, slots, x, scale):
    held = cache.double()
    flat = held.view(-1, *cache.shape[2:])
    live = slots >= 0
    x = x.double() if scale is None else (x.double() / scale.double()[:, None]).clamp(-E4M3_MAX, E4M3_MAX)
    flat[slots[live]] = x[live]
    return held


def _exact_attend(s):
    case = s["case"]
    chunks, contexts = _lengths(case)
    group, block = case["heads"] // case["kv_heads"], case["block"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    at = 0
    for b, (n, c) in enumerate(zip(chunks, contexts)):
        pages = s["table"][b, :-(-c // block)].long()
        for h in range(case["kv_heads"]):
            k = s["k_cache"].view(torch.uint8).view(*s["k_cache"].shape[:3], -1)[pages, :, h].view(s["k_cache"].dtype)
            v = s["v_cache"].view(torch.uint8).view(*s["v_cache"].shape[:3], -1)[pages, :, h].view(s["v_cache"].dtype)
            k, v = k.reshape(-1, case["dim"])[:c].double(), v.reshape(-1, case["dim"])[:c].double()
            if case["e4m3"]:
                k, v = k * s["k_scale"][h].double(), v * s["v_scale"][h].double()
            first = max(0, n - c)                               # rows before it stand at negative positions: nothing to see
            for x in range(h * group, (h + 1) * group):
                z = s["q"][at + first:at + n, x].double() @ k.T * s["scale"]
                hidden = torch.ones(z.shape, dtype=torch.bool, device="cuda").triu(c - n + first + 1)
                z = z.masked_fill(hidden, -math.inf)
                lse[at + first:at + n, x] = torch.logsumexp(z, -1)
                out[at + first:at + n, x] = torch.exp(z - lse[at + first:at + n, x, None]) @ v
        at += n
    return (out, lse) if case["lse"] else out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attend":
        return _exact_attend(s)
    q, k = _exact_heads(s["q"], s["q_weight"], s), _exact_heads(s["k"], s["k_weight"], s)
    if case["op"] == "norm_rope":
        return q, k
    return (q, _exact_cache(s["k_cache"], s["slots"], k, s["k_scale"]),
            _exact_cache(s["v_cache"], s["slots"], s["v"], s["v_scale"]))
