"""Rotary positions joined to the cache write, and attention over a paged cache of latent vectors.

A latent cache holds one row a token, shared by every head: a latent vector of ``latent`` elements
and a rotated key part of ``rope`` elements behind it. Four operators around it and around the
caches of keys and values:

* ``rotate``: a step's queries and keys are rotated by their positions and the keys and values
  written into a paged cache;
* ``latent_store``: a step's latents and rotated key parts are written into a latent cache, and the
  queries' rotary parts rotated with them;
* ``absorbed``: attention on the rows as they are stored, score ``q . row``, output the weighted sum
  of the latents (the keys' and values' matrices are absorbed by the projections around it);
* ``chunks``: attention on keys and values expanded from the latents, ``k = keys[h] @ latent`` beside
  the shared rotary part, ``v = values[h] @ latent``, for chunks of new tokens.

``own`` False computes all of them in elementary torch operations; True calls the framework.
"""

from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


# --- cases ------------------------------------------------------------------------------------------


def _case(name, kind, dtype, heads, block, requests, shortest, longest, rows_least=1, rows_most=1, *, padding=0,
          mix=1, **more):
    """``requests`` contexts of ``shortest`` to ``longest`` positions, each with ``rows_least`` to
    ``rows_most`` new rows, the last ``padding`` of them empty; ``more`` as the kind asks for."""
    return {"name": name, "kind": kind, "dtype": dtype, "heads": heads, "block": block, "requests": requests,
            "shortest": shortest, "longest": longest, "rows_least": rows_least, "rows_most": rows_most,
            "padding": padding, "mix": mix, **more}


def _dense(kv_heads, head_dim, layout="nhd"):
    return {"kv_heads": kv_heads, "head_dim": head_dim, "layout": layout}


def _turning(rotary_dim, base, interleaved=False, scaling="none", factor=1.0, original=0):
    return {"rotary_dim": rotary_dim, "base": base, "interleaved": interleaved, "scaling": scaling, "factor": factor,
            "original": original}


def listed():
    return [
        # A small model's decode step at a handful of users: one token each, every launch counts.
        _case("rotate_decode_small", "rotate", "fp16", 9, 16, 4, 128, 1000, **_dense(3, 64), **_turning(64, 10000.0)),
        # Continuous batching at a full batch of a large model with positions scaled for long contexts.
        _case("rotate_decode_batch", "rotate", "bf16", 64, 32, 256, 16, 16384, padding=6, mix=2, **_dense(8, 128),
              **_turning(128, 500000.0, False, "bands", 8.0, 8192)),
        # Uneven prefill chunks far into long contexts, half of each head rotated, pairs side by side.
        _case("rotate_chunks", "rotate", "bf16", 32, 16, 8, 9000, 30000, 400, 2000, mix=3, **_dense(8, 128),
              **_turning(64, 10000.0, True, "linear", 4.0, 0)),
        # Decode of a full batch over a latent cache, the heads of one of eight tensor-parallel ranks.
        _case("latent_store_batch", "latent_store", "bf16", 16, 64, 256, 16, 16384, padding=6, mix=4, latent=512, rope=64,
              **_turning(64, 10000.0, True, "yarn", 40.0, 4096)),
        # Prefill chunks of uneven size into a latent cache, all heads on one card.
        _case("latent_store_chunks", "latent_store", "bf16", 128, 16, 4, 2000, 6000, 500, 2000, mix=5, latent=512, rope=64,
              **_turning(64, 10000.0, True, "yarn", 40.0, 4096)),
        # Decode at a handful of users: latency.
        _case("absorbed_decode_small", "absorbed", "bf16", 16, 16, 4, 128, 1000, latent=512, rope=64),
        # Decode of a full batch of equal contexts, one of eight tensor-parallel ranks.
        _case("absorbed_decode_batch", "absorbed", "bf16", 16, 64, 64, 4096, 4096, latent=512, rope=64),
        # Continuous batching with all heads on one card: contexts from 16 to 16K, some slots of the batch empty.
        _case("absorbed_decode_ragged", "absorbed", "bf16", 128, 32, 64, 16, 16384, padding=3, mix=5, latent=512, rope=64),
        # Speculative decoding: windows of 4 draft tokens over 4K contexts.
        _case("absorbed_verify", "absorbed", "fp16", 32, 16, 32, 4096, 4096, 4, 4, latent=512, rope=64),
        # One user's short prompt.
        _case("chunks_prompt_small", "chunks", "bf16", 16, 16, 1, 300, 300, 300, 300, latent=512, rope=64, nope=128, value=128),
        # Chunked prefill: 512-row chunks at the end of 4K contexts.
        _case("chunks_long", "chunks", "bf16", 16, 64, 4, 4096, 4096, 512, 512, latent=512, rope=64, nope=128, value=128),
        # Uneven chunks and whole prompts over blocks of an odd size.
        _case("chunks_ragged", "chunks", "bf16", 32, 24, 4, 900, 6000, 300, 2500, mix=6, latent=512, rope=64, nope=128, value=128),
    ]


def _between(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("rotate", "latent_store", "absorbed", "absorbed", "chunks"))
    mix = rng.randrange(1, 1000)
    dtype, block = rng.choice(("fp16", "bf16")), rng.choice((1, 7, 16, 24, 32, 64, 128))
    form = rng.choice(("decode", "verify", "chunks"))
    scaling = rng.choice(("none", "linear", "bands", "yarn"))
    turning = dict(base=rng.choice((10000.0, 500000.0, 1234.5)), interleaved=rng.choice((True, False)), scaling=scaling,
                   factor=1.0 if scaling == "none" else rng.choice((2.0, 8.0, 40.0)),
                   original=0 if scaling in ("none", "linear") else rng.choice((2048, 4096, 8192)))
    most = {"decode": 1, "verify": 8, "chunks": 600}[form]
    if kind == "rotate":
        kv_heads, head_dim = rng.choice((1, 2, 3, 8)), rng.choice((64, 80, 96, 128, 256))
        longest = _between(rng, max(32, most), 20000)
        # at most about what the largest listed case of the kind holds
        requests = max(1, min(_between(rng, 1, 256), (96 << 20) // (longest * kv_heads * head_dim)))
        requests = min(requests, 8) if form == "chunks" else requests
        case = _case("", kind, rng.choice(("fp16", "bf16", "fp32")), kv_heads * rng.choice((1, 2, 3, 4, 8)), block, requests,
                     _between(rng, most, longest), longest, min(most, rng.choice((1, 2, 40))), most,
                     padding=rng.randrange(0, 1 + requests // 4), mix=mix,
                     **_dense(kv_heads, head_dim, rng.choice(("nhd", "hnd"))),
                     rotary_dim=rng.choice((head_dim, head_dim // 2, 32)), **turning)
    else:
        heads, latent = rng.choice((1, 4, 8, 16, 20, 32, 64, 128)), rng.choice((512, 512, 256))
        longest = _between(rng, max(32, most), {"latent_store": 16384, "absorbed": 8192, "chunks": 4096}[kind])
        tokens = {"latent_store": 1 << 20, "absorbed": 1 << 18, "chunks": 1 << 14}[kind]
        requests = max(1, min(_between(rng, 1, 128), tokens // longest))
        if kind == "chunks":
            most, form, dtype = 600, "chunks", "bf16"
            heads, longest = min(heads, 32), max(longest, 600)
        elif kind == "absorbed":
            if form == "chunks":
                most, heads, longest = 64, min(heads, 32), min(longest, 4096)
            requests = max(1, min(requests, (1 << 24) // (longest * heads * most)))
        if form == "chunks":
            requests = min(requests, 4)
        case = _case("", kind, dtype, heads, block, requests, _between(rng, most, longest), longest,
                     min(most, rng.choice((1, 2, 40))), most, padding=rng.randrange(0, 1 + requests // 4), mix=mix,
                     latent=latent, rope=64)
        if kind == "latent_store":
            case.update(rotary_dim=64, **turning)
        if kind == "chunks":
            case.update(nope=128, value=128)
    case.pop("name")
    return case


def _generator(seed, device="cpu"):
    return torch.Generator(device=device).manual_seed(seed)


def _log_uniform(count, low, high, g):
    x = torch.rand(count, generator=g, dtype=torch.float64)
    return torch.exp(math.log(low) + x * (math.log(high) - math.log(low))).round().long().clamp(low, high)


def _requests(case):
    """Lengths and row counts of the case's requests (they do not change with the inputs' seed)."""
    g = _generator(9000 + case["mix"])
    n, pad = case["requests"], case["padding"]
    lengths = _log_uniform(n, case["shortest"], case["longest"], g)
    rows = _log_uniform(n, case["rows_least"], case["rows_most"], g).minimum(lengths)
    if pad:
        lengths[n - pad:] = 0
        rows[n - pad:] = 1
    return lengths, rows


def _blocks(lengths, block):
    return (lengths + block - 1) // block


def work(case):
    lengths, rows = _requests(case)
    n, live, size = int(rows.sum()), lengths > 0, 4 if case["dtype"] == "fp32" else 2
    stored = int(rows[live].sum())
    if case["kind"] == "rotate":
        width = case["kv_heads"] * case["head_dim"]
        return {"bytes": 2 * size * (n * case["heads"] * case["head_dim"] + 2 * stored * width) + 12 * n, "flops": 0}
    width = case["latent"] + case["rope"]
    if case["kind"] == "latent_store":
        return {"bytes": 2 * size * (n * case["heads"] * case["rope"] + stored * width) + 12 * n, "flops": 0}
    positions, blocks = int(lengths.sum()), int(_blocks(lengths, case["block"]).sum())
    pairs = int((rows * lengths - rows * (rows - 1) // 2)[live].sum()) * case["heads"]
    cache = size * positions * width + 4 * blocks + 4 * len(lengths)
    if case["kind"] == "absorbed":
        return {"bytes": cache + size * n * case["heads"] * (width + case["latent"]), "flops": 2 * pairs * (width + case["latent"])}
    inner = case["nope"] + case["value"]
    return {"bytes": cache + size * case["heads"] * (n * (inner + case["rope"]) + inner * case["latent"]),
            "flops": 2 * (pairs * (inner + case["rope"]) + positions * case["heads"] * inner * case["latent"])}


# --- inputs -----------------------------------------------------------------------------------------


def _table(lengths, block, g):
    """Every request's blocks, shuffled over a pool whose block 0 is padding; and the pool's size."""
    counts = _blocks(lengths, block)
    table = torch.zeros(len(lengths), max(1, int(counts.max())), dtype=torch.int32)
    mask = torch.arange(table.shape[1])[None, :] < counts[:, None]
    total = int(counts.sum())
    table[mask] = (1 + torch.randperm(total, generator=g)).int()
    return table, total + 1


def _rows(lengths, rows, table, block):
    """Each row's request, place within it, position and slot (0: a padding request's)."""
    request = torch.repeat_interleave(torch.arange(len(rows)), rows)
    within = torch.arange(int(rows.sum())) - (torch.cumsum(rows, 0) - rows)[request]
    live = lengths[request] > 0
    position = torch.where(live, (lengths - rows)[request] + within, 0)
    slot = table[request, position // block].long() * block + position % block
    return request, within, position, torch.where(live, slot, 0)


def _frequencies(case):
    """Radians per position of each pair, in 64 bits, and what cosines and sines are multiplied by."""
    pairs, factor, original = case["rotary_dim"] // 2, case["factor"], case["original"]
    index = torch.arange(pairs, dtype=torch.float64)
    plain = case["base"] ** (-2 * index / case["rotary_dim"])
    if case["scaling"] == "linear":
        return plain / factor, 1.0
    if case["scaling"] == "bands":
        # wavelengths under original / 4 stay, over original / 1 stretch by the factor, between both blend
        share = ((original * plain / (2 * math.pi) - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return plain * (share + (1 - share) / factor), 1.0
    if case["scaling"] == "yarn":
        # pairs that turn over 32 times within `original` positions stay, under 1 stretch, a ramp over the pairs between
        def pair_of(turns):
            return case["rotary_dim"] * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(case["base"]))

        low, high = max(0, math.floor(pair_of(32))), min(case["rotary_dim"] - 1, math.ceil(pair_of(1)))
        stretch = ((index - low) / max(high - low, 0.001)).clamp(0, 1)
        return plain * (1 - stretch + stretch / factor), 0.1 * math.log(factor) + 1.0
    return plain, 1.0


def _values(shape, g):
    """Rows as layers make them: a few loud channels."""
    channels = torch.where(torch.rand(shape[-1], generator=g, device="cuda") < 0.03, 4.0, 1.0)
    return torch.randn(*shape, generator=g, device="cuda") * channels


def prepare(case, seed):
    host, g = _generator(seed), _generator(seed, "cuda")
    lengths, rows = _requests(case)
    block, kind, dtype, heads = case["block"], case["kind"], _DTYPES[case["dtype"]], case["heads"]
    table, pool = _table(lengths, block, host)
    request, within, position, slots = _rows(lengths, rows, table, block)
    n = len(slots)
    state = {"case": case, "request": request.cuda(), "within": within.cuda(), "position": position.cuda(),
             "slots": slots.cuda(), "lengths": lengths.int().cuda(), "rows": rows.int().cuda(), "table": table.cuda()}
    if kind in ("rotate", "latent_store"):
        frequencies, state["magnitude"] = _frequencies(case)
        state["frequencies"] = frequencies.cuda()
    if kind == "rotate":
        kv_heads, head_dim = case["kv_heads"], case["head_dim"]
        # q, k and v are the parts of one projection's output, as a layer has them
        both = _values((n, (heads + 2 * kv_heads) * head_dim), g).to(dtype)
        q, k, v = both.split((heads * head_dim, kv_heads * head_dim, kv_heads * head_dim), dim=1)
        state.update(q=q.unflatten(1, (heads, head_dim)), k=k.unflatten(1, (kv_heads, head_dim)),
                     v=v.unflatten(1, (kv_heads, head_dim)), q_out=torch.empty(n, heads, head_dim, dtype=dtype, device="cuda"))
        shape = (pool, block, kv_heads, head_dim) if case["layout"] == "nhd" else (pool, kv_heads, block, head_dim)
        state["k_cache"], state["v_cache"] = (torch.randn(shape, generator=g, device="cuda", dtype=dtype) for _ in range(2))
    else:
        latent, rope = case["latent"], case["rope"]
        cache = _values((pool, block, latent + rope), g).to(dtype)
        if kind == "latent_store":
            # the latent and the key's rotary part come out of one projection, the query's parts out of another
            down = _values((n, latent + rope), g).to(dtype)
            state["latent"], state["k_rope"] = down[:, :latent], down[:, latent:]
            state["q"] = torch.randn(n, heads, 128 + rope, generator=g, device="cuda").to(dtype)[:, :, 128:]
            state["q_out"] = torch.zeros(n, heads, latent + rope, dtype=dtype, device="cuda")[:, :, latent:]
        else:
            # slots that no token holds (padding block, tails of blocks) are NaN: nothing may read them
            held = torch.zeros(pool, dtype=torch.int64)
            start = torch.arange(table.shape[1])[None, :] * block
            held[table[table > 0].long()] = (lengths[:, None] - start)[table > 0].clamp(0, block)
            cache[(torch.arange(block)[None, :] >= held[:, None]).cuda()] = math.nan
            if kind == "absorbed":
                q = torch.randn(n, heads, latent + rope, generator=g, device="cuda")
                q[:, :, :latent] *= math.sqrt(128 / latent)  # 128 elements by a matrix that keeps lengths
                state["q"], state["scale"] = q.to(dtype), (128 + rope) ** -0.5
                state["out"] = torch.empty(n, heads, latent, dtype=dtype, device="cuda")
            else:
                nope, value = case["nope"], case["value"]
                state["q"] = torch.randn(n, heads, nope + rope, generator=g, device="cuda").to(dtype)
                state["keys"], state["values"] = (
                    (torch.randn(heads, width, latent, generator=g, device="cuda") * latent ** -0.5).to(dtype)
                    for width in (nope, value))
                state["scale"] = (nope + rope) ** -0.5
                state["out"] = torch.empty(n, heads, value, dtype=dtype, device="cuda")
        state["cache"] = cache
    if own:
        from ayaka_amd.backend import load_backend
        from ayaka_amd.enums import DType, ForwardMode, KVLayoutKind
        from ayaka_amd.kvcache import RAW_CODEC, KVBuffers, LatentBuffers, LatentWeights
        from ayaka_amd.rotary import BandScaling, LinearScaling, YarnScaling, rotary

        label = {"fp16": DType.FP16, "bf16": DType.BF16, "fp32": DType.FP32}[case["dtype"]]
        state["ops"] = load_backend(["hip"], device="cuda", dtype=label)
        decode = bool((rows == 1).all())
        state["meta"] = state["ops"].attention.plan(ForwardMode.DECODE if decode else ForwardMode.MIXED, state["rows"],
                                                    state["lengths"], state["table"], block)
        if kind in ("rotate", "latent_store"):
            scaling = {"none": lambda: None, "linear": lambda: LinearScaling(case["factor"]),
                       "bands": lambda: BandScaling(case["factor"], case["original"]),
                       "yarn": lambda: YarnScaling(case["factor"], case["original"])}[case["scaling"]]()
            state["rotary"] = rotary(case["rotary_dim"], base=case["base"], interleaved=case["interleaved"],
                                     scaling=scaling, device="cuda")
        if kind == "rotate":
            layout = KVLayoutKind.NHD if case["layout"] == "nhd" else KVLayoutKind.HND
            state["buffers"] = KVBuffers(state["k_cache"], state["v_cache"], layout, RAW_CODEC)
        else:
            state["buffers"] = LatentBuffers(state["cache"], case["latent"])
        if kind == "chunks":
            state["weights"] = LatentWeights(state["keys"], state["values"])
    return state


# --- one pass ---------------------------------------------------------------------------------------


def run(state):
    kind = state["case"]["kind"]
    if kind == "rotate":
        if own:
            state["ops"].kvcache.store_rotated(state["q"], state["k"], state["v"], state["buffers"], state["meta"],
                                               state["rotary"], q_out=state["q_out"])
        else:
            _rotate(state)
        return {"q": state["q_out"], "k": state["k_cache"], "v": state["v_cache"]}
    if kind == "latent_store":
        if own:
            state["ops"].kvcache.store_latent(state["latent"], state["k_rope"], state["buffers"], state["meta"],
                                              rotary=state["rotary"], q=state["q"], q_out=state["q_out"])
        else:
            _latent_store(state)
        return {"q": state["q_out"], "cache": state["cache"]}
    if not own:
        return _absorbed(state) if kind == "absorbed" else _chunks(state)
    if kind == "absorbed":
        state["ops"].attention.attend_latent(state["q"], state["buffers"], state["meta"], state["out"], scale=state["scale"])
    else:
        state["ops"].attention.attend_latent_chunks(state["q"], state["weights"], state["buffers"], state["meta"], state["out"],
                                                    scale=state["scale"])
    return state["out"]


def _turned(x, state):
    """Rows [N, heads, width] with their first ``rotary_dim`` elements rotated, in 32 bits."""
    case = state["case"]
    size = case["rotary_dim"]
    angle = state["position"].double()[:, None] * state["frequencies"][None, :]  # 64 bits: positions reach far
    cos, sin = ((f(angle) * state["magnitude"]).float()[:, None, :] for f in (torch.cos, torch.sin))
    x = x.float()
    if case["interleaved"]:
        a, b = x[..., 0:size:2], x[..., 1:size:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = x[..., : size // 2], x[..., size // 2:size]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned, x[..., size:]), dim=-1)


def _rotate(state):
    block, slots = state["case"]["block"], state["slots"]
    state["q_out"].copy_(_turned(state["q"], state))
    live = slots >= block  # a padding request's rows are not stored
    at, offset = slots[live] // block, slots[live] % block
    for name, rows in (("k_cache", _turned(state["k"], state).to(state["k"].dtype)), ("v_cache", state["v"])):
        cache = state[name].transpose(1, 2) if state["case"]["layout"] == "hnd" else state[name]
        cache[at, offset] = rows[live]


def _latent_store(state):
    block, slots = state["case"]["block"], state["slots"]
    state["q_out"].copy_(_turned(state["q"], state))
    key = _turned(state["k_rope"][:, None], state)[:, 0].to(state["latent"].dtype)
    live = slots >= block
    state["cache"][slots[live] // block, slots[live] % block] = torch.cat((state["latent"], key), dim=-1)[live]


def _gathered(state):
    """The requests' cached rows side by side, [requests, positions, latent + rope] in 32 bits, zeros
    behind each one's length; and which (row of the request, position) pairs are visible."""
    case, lengths, table = state["case"], state["lengths"].long(), state["table"].long()
    longest = min(case["longest"], table.shape[1] * case["block"])
    position = torch.arange(longest, device="cuda")
    held = position[None, :] < lengths[:, None]
    x = state["cache"][table].flatten(1, 2)[:, :longest].float()
    x = torch.where(held[:, :, None], x, 0.0)
    sees = torch.full((len(lengths), max(1, case["rows_most"])), -1, device="cuda", dtype=torch.long)
    sees[state["request"], state["within"]] = state["position"]
    return x, held[:, None, :] & (position[None, None, :] <= sees[:, :, None])


def _padded(state, x):
    """Rows [N, heads, width] as [requests, rows, heads, width] in 32 bits."""
    out = torch.zeros(len(state["lengths"]), max(1, state["case"]["rows_most"]), *x.shape[1:], device="cuda")
    out[state["request"], state["within"]] = x.float()
    return out


def _weights(scores):
    largest = scores.amax(-1, keepdim=True)
    scores = torch.exp(scores - torch.where(largest == -math.inf, 0.0, largest))
    total = scores.sum(-1, keepdim=True)
    return scores / torch.where(total > 0, total, 1.0)


def _absorbed(state):
    x, visible = _gathered(state)
    q = _padded(state, state["q"])  # [requests, rows, heads, width]
    requests, most, heads, width = q.shape
    scores = torch.matmul(q.view(requests, most * heads, width), x.transpose(1, 2).contiguous()) * state["scale"]
    scores = scores.view(requests, most, heads, -1).masked_fill(~visible[:, :, None, :], -math.inf)
    p = _weights(scores).view(requests, most * heads, -1)
    out = torch.matmul(p, x[..., : state["case"]["latent"]].contiguous()).view(requests, most, heads, -1)
    return out[state["request"], state["within"]].to(state["q"].dtype)


def _chunks(state):
    case = state["case"]
    x, visible = _gathered(state)
    latent, heads = x[..., : case["latent"]], case["heads"]
    k, v = (torch.matmul(latent, state[name].float().flatten(0, 1).T).unflatten(-1, (heads, -1)) for name in ("keys", "values"))
    k = torch.cat((k, x[:, :, None, case["latent"]:].expand(-1, -1, heads, -1)), dim=-1)
    q = _padded(state, state["q"]).transpose(1, 2).contiguous()  # [requests, heads, rows, width]
    scores = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()) * state["scale"]
    p = _weights(scores.masked_fill(~visible[:, None], -math.inf))
    out = torch.matmul(p, v.transpose(1, 2).contiguous()).transpose(1, 2)
    return out[state["request"], state["within"]].to(state["q"].dtype)


# --- the definitions in 64 bits -----------------------------------------------------------------------


def _exactly_turned(x, state):
    """Each pair of elements as a complex number times e^(i angle)."""
    case = state["case"]
    size, x = case["rotary_dim"], x.double()
    first = torch.arange(size // 2, device="cuda") * (2 if case["interleaved"] else 1)
    second = first + (1 if case["interleaved"] else size // 2)
    turn = torch.polar(torch.full_like(state["frequencies"], state["magnitude"])[None, :].expand(len(x), -1).contiguous(),
                       state["position"].double()[:, None] * state["frequencies"][None, :])
    pair = torch.complex(x[..., first], x[..., second]) * turn[:, None, :]
    out = x.clone()
    out[..., first], out[..., second] = pair.real, pair.imag
    return out


def exact(case, seed):
    state = prepare(case, seed)
    lengths, rows = _requests(case)
    block, size, last = case["block"], case["heads"], 0
    if case["kind"] == "rotate":
        caches = [state[name].double() for name in ("k_cache", "v_cache")]
        new = (_exactly_turned(state["k"], state), state["v"].double())
    elif case["kind"] == "latent_store":
        caches = [state["cache"].double()]
        new = (torch.cat((state["latent"].double(), _exactly_turned(state["k_rope"][:, None], state)[:, 0]), dim=-1),)
    else:
        out = torch.zeros(state["out"].shape, dtype=torch.float64, device="cuda")
    for b, (length, count) in enumerate(zip(lengths.tolist(), rows.tolist())):
        first, last = last, last + count
        if length == 0:
            continue
        positions = torch.arange(length, device="cuda")
        blocks, offsets = state["table"][b].long()[positions // block], positions % block
        if case["kind"] in ("rotate", "latent_store"):
            for cache, x in zip(caches, new):
                flat = cache.transpose(1, 2) if case.get("layout") == "hnd" else cache
                flat[blocks[length - count:], offsets[length - count:]] = x[first:last]
            continue
        row = state["cache"][blocks, offsets].double()
        hidden = positions[None, :] > (length - count + torch.arange(count, device="cuda"))[:, None]
        latent, key = row[:, : case["latent"]], row[:, case["latent"]:]
        for h in range(size):
            q = state["q"][first:last, h].double()
            if case["kind"] == "absorbed":
                score, value = q @ row.T.contiguous(), latent
            else:
                score = (q[:, : case["nope"]] @ state["keys"][h].double()) @ latent.T.contiguous()
                score = score + q[:, case["nope"]:] @ key.T.contiguous()
                value = latent @ state["values"][h].double().T.contiguous()
            weight = torch.softmax((score * state["scale"]).masked_fill(hidden, -math.inf), dim=-1)
            out[first:last, h] = weight @ value
    if case["kind"] == "rotate":
        return {"q": _exactly_turned(state["q"], state), "k": caches[0], "v": caches[1]}
    if case["kind"] == "latent_store":
        return {"q": _exactly_turned(state["q"], state), "cache": caches[0]}
    return out
