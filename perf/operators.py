"""The cases on which the cache operators are measured, with the operators' plain forms.

Four operators that serve one path, several action samples (or several token sequences) drawn behind one shared prefix:

* ``axes``       sine / cosine tables of rotary positions with several axes (time, height, width);
* ``write``      rotation of queries and keys, and the keys / values quantised to e4m3 (one fp32 scale per token and head)
                 as they are written into a cache;
* ``read``       the quantised cache read back as bf16;
* ``attention``  attention of a batch whose members share prefixes: each prefix is read once for all its members, then
                 each member's own keys; over a bf16 or a quantised cache.

``run`` computes a case in elementary torch operations, or through the package's own entry points where ``own`` is true.
"""

import math

import numpy as np
import torch

own = False

#: the magnitudes that a quantised cache holds: rows whose largest is below TINY are stored as zero, from HUGE on as NaN
TINY, HUGE = 2.0 ** -50, 2.0 ** 40
E4M3_MAX = 448.0


# ---- the cases -----------------------------------------------------------------------------------------


def listed():
    return [
        # positions of one observation's prefix: two cameras of 16 x 16 patches and 48 text tokens, head dimension 256
        {"name": "axes_prefix", "op": "axes", "batch": 1, "tokens": 560, "dim": 256, "axes": 3, "own_spectrum": False, "far": 4096},
        # positions of long videos, another table for every sequence, head dimension 128
        {"name": "axes_video", "op": "axes", "batch": 8, "tokens": 16384, "dim": 128, "axes": 3, "own_spectrum": False, "far": 262144},
        # the action expert's ten tokens of eight samples, written at every flow step
        {"name": "write_chunk", "op": "write", "batch": 8, "tokens": 10, "heads": 8, "kv_heads": 1, "dim": 256, "capacity": 10, "ragged": False},
        # one token of each of 64 sequences, each at its own position
        {"name": "write_token", "op": "write", "batch": 64, "tokens": 1, "heads": 32, "kv_heads": 8, "dim": 128, "capacity": 512, "ragged": True},
        # prompts of different lengths in one padded batch
        {"name": "write_prompts", "op": "write", "batch": 16, "tokens": 1000, "heads": 32, "kv_heads": 8, "dim": 128, "capacity": 1024, "ragged": True},
        # the prefixes of 32 observations with 2 or 3 cameras' worth of tokens, read back for another consumer
        {"name": "read_prefix", "op": "read", "batch": 32, "kv_heads": 1, "dim": 256, "capacity": 712, "ragged": True},
        # a long cache read back whole
        {"name": "read_long", "op": "read", "batch": 8, "kv_heads": 8, "dim": 128, "capacity": 8192, "ragged": False},
        # four action samples of one observation, one flow step of a control loop: latency
        {"name": "attention_chunk", "op": "attention", "groups": 1, "members": 4, "heads": 8, "kv_heads": 1, "dim": 256, "tokens": 10,
         "prefix": 560, "suffix": 10, "fp8": False, "causal": False, "ragged": False},
        # a rollout step: 32 observations of different lengths, eight samples each, over a quantised cache
        {"name": "attention_rollout", "op": "attention", "groups": 32, "members": 8, "heads": 8, "kv_heads": 1, "dim": 256, "tokens": 10,
         "prefix": 712, "suffix": 10, "fp8": True, "causal": False, "ragged": True},
        # token by token behind one long shared context, each sequence with its own tail
        {"name": "attention_long", "op": "attention", "groups": 1, "members": 64, "heads": 32, "kv_heads": 8, "dim": 128, "tokens": 1,
         "prefix": 32768, "suffix": 512, "fp8": True, "causal": True, "ragged": True},
        # several contexts of unequal popularity, four drafted tokens each
        {"name": "attention_groups", "op": "attention", "groups": 8, "members": 5, "heads": 16, "kv_heads": 2, "dim": 128, "tokens": 4,
         "prefix": 4097, "suffix": 300, "fp8": False, "causal": True, "ragged": True},
        # fifty-step action chunks over long video prefixes: bound by the products
        {"name": "attention_video", "op": "attention", "groups": 4, "members": 16, "heads": 8, "kv_heads": 1, "dim": 256, "tokens": 50,
         "prefix": 8192, "suffix": 50, "fp8": False, "causal": False, "ragged": False},
    ]


def _log(rng, low, high):
    """A whole number of [low, high], even over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["axes", "write", "read", "attention", "attention"])
    if op == "axes":
        dim = rng.choice([64, 128, 256])
        batch = _log(rng, 1, 32)
        return {"op": op, "batch": batch, "tokens": _log(rng, 1, max(1, 16777216 // (batch * dim))), "dim": dim, "axes": rng.choice([1, 2, 3]),
                "own_spectrum": rng.random() < 0.5, "far": _log(rng, 16, 262144)}
    dim = rng.choice([128, 256])
    heads, kv_heads = rng.choice([(8, 1), (32, 8), (16, 2), (8, 8), (28, 4), (6, 2), (1, 1)])
    if op == "write":
        batch = _log(rng, 1, 64)
        tokens = _log(rng, 1, max(1, 16000 * 48 * 128 // (batch * (heads + 2 * kv_heads) * dim)))
        return {"op": op, "batch": batch, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "capacity": tokens + rng.choice([0, 1, 24, 333]), "ragged": rng.random() < 0.6}
    if op == "read":
        batch = _log(rng, 1, 64)
        return {"op": op, "batch": batch, "kv_heads": kv_heads, "dim": dim, "capacity": _log(rng, 1, max(1, 67108864 // (batch * kv_heads * dim))),
                "ragged": rng.random() < 0.6}
    groups, members = _log(rng, 1, 32), _log(rng, 1, 64)
    tokens = _log(rng, 1, 50)
    suffix = max(tokens, _log(rng, 1, 512))
    # at most what the largest listed case costs, in products (5e10 multiply-adds) and in bytes of the queries, own keys and prefixes
    while groups * members * dim * max(kv_heads * suffix, heads * tokens) > 33554432 and groups * members > 1:
        groups, members = (groups, (members + 1) // 2) if members > 1 else (groups // 2, members)
    rows = groups * members * heads * tokens
    longest = min(32768, 50000000000 // (rows * dim), 33554432 // (groups * kv_heads * dim))
    return {"op": op, "groups": groups, "members": members, "heads": heads, "kv_heads": kv_heads, "dim": dim, "tokens": tokens,
            "prefix": _log(rng, 1, max(1, longest)), "suffix": suffix, "fp8": rng.random() < 0.5, "causal": rng.random() < 0.5,
            "ragged": rng.random() < 0.6}


# ---- lengths: set by the case alone, so that its work is known -------------------------------------------


def _spread(count, high, low=0):
    """`count` whole numbers of [low, high], scattered, the first of them `high`."""
    return [high - (i * 7919) % (high - low + 1) for i in range(count)]


def _sections(case):
    half, axes = case["dim"] // 2, case["axes"]
    first = half if axes == 1 else half // 2 if axes == 2 else half // 4
    rest = (half - first) // max(1, axes - 1)
    return [first] + [rest] * (axes - 2) + ([half - first - rest * (axes - 2)] if axes > 1 else [])


def _write_plan(case):
    """(offset of every sequence, its number of real tokens)"""
    count, tokens, room = case["batch"], case["tokens"], case["capacity"] - case["tokens"]
    if not case["ragged"]:
        return [0] * count, [tokens] * count
    return _spread(count, room), _spread(count, tokens, tokens // 2 if tokens > 1 else 1)


def _read_lengths(case):
    return _spread(case["batch"], case["capacity"], case["capacity"] // 2) if case["ragged"] else [case["capacity"]] * case["batch"]


def _attention_plan(case):
    """(bounds of the groups' members, prefix lengths, own lengths)"""
    groups, members = case["groups"], case["members"]
    if not case["ragged"]:
        return [g * members for g in range(groups + 1)], [case["prefix"]] * groups, [case["suffix"]] * (groups * members)
    counts = [members + (members // 2 if g % 2 else -(members // 2)) for g in range(groups - groups % 2)] + [members] * (groups % 2)
    bounds = [0]
    for count in counts:
        bounds.append(bounds[-1] + count)
    return bounds, _spread(groups, case["prefix"], case["prefix"] // 2), _spread(bounds[-1], case["suffix"], case["tokens"])


# ---- inputs --------------------------------------------------------------------------------------------


def _quantised(x):
    """bf16 rows -> (e4m3 codes, one fp32 scale for each row)"""
    scale = x.float().abs().amax(-1) / E4M3_MAX
    return (x.float() / scale.unsqueeze(-1)).to(torch.float8_e4m3fn), scale


def _rows(generator, *shape):
    """Keys or values: rows of unequal size, a few strong channels."""
    x = torch.randn(shape, device="cuda", generator=generator)
    size = torch.exp(0.4 * torch.randn((*shape[:-1], 1), device="cuda", generator=generator))
    channel = torch.ones(shape[-1], device="cuda")
    channel[:: 37] = 3.0
    return (x * size * channel).to(torch.bfloat16)


def prepare(case, seed):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    whole = lambda values: torch.tensor(values, device="cuda", dtype=torch.int32)
    state = {"case": case}
    if case["op"] == "axes":
        # a time that runs to `far`, rows and columns of image patches
        shape = (case["batch"], case["tokens"])
        reach = [case["far"], 64, 64]
        state["positions"] = torch.stack([torch.randint(0, reach[a], shape, device="cuda", generator=generator) for a in range(case["axes"])])
        state["sections"] = tuple(_sections(case))
        return state
    dim = case["dim"]
    if case["op"] == "write":
        batch, tokens, heads, kv_heads, capacity = (case[k] for k in ("batch", "tokens", "heads", "kv_heads", "capacity"))
        offsets, lengths = _write_plan(case)
        state["qkv"] = _rows(generator, batch, tokens, heads + 2 * kv_heads, dim)
        angle = torch.rand((tokens, dim // 2), device="cuda", generator=generator) * 6.0
        state["sine"], state["cosine"] = angle.sin(), angle.cos()
        state["q_out"] = torch.zeros((batch, heads, tokens, dim), device="cuda", dtype=torch.bfloat16)
        for name in ("k", "v"):          # what earlier calls have left in the cache
            codes, scales = _quantised(_rows(generator, 1, kv_heads, capacity, dim))
            state[name + "_codes"] = codes.view(torch.uint8).repeat(batch, 1, 1, 1).view(torch.float8_e4m3fn)
            state[name + "_scales"] = scales.repeat(batch, 1, 1)
        state["offsets"], state["lengths"] = whole(offsets), whole(lengths)
        real = [(b, t, offsets[b] + t) for b in range(batch) for t in range(lengths[b])]
        state["real"] = tuple(torch.tensor(column, device="cuda") for column in zip(*real))
        return state
    if case["op"] == "read":
        shape = (case["batch"], case["kv_heads"], case["capacity"], dim)
        lengths = _read_lengths(case)
        for name in ("k", "v"):
            state[name + "_codes"], state[name + "_scales"] = _quantised(_rows(generator, *shape))
            state[name + "_out"] = torch.zeros(shape, device="cuda", dtype=torch.bfloat16)
        state["lengths"] = whole(lengths)
        return state
    groups, heads, kv_heads, tokens = (case[k] for k in ("groups", "heads", "kv_heads", "tokens"))
    bounds, prefix_lengths, suffix_lengths = _attention_plan(case)
    batch = bounds[-1]
    state["q"] = (1.5 * torch.randn((batch, heads, tokens, dim), device="cuda", generator=generator)).to(torch.bfloat16)
    for part, count, length in (("prefix", groups, case["prefix"]), ("suffix", batch, case["suffix"])):
        for name in ("k", "v"):
            rows = _rows(generator, count, kv_heads, length, dim)
            if case["fp8"]:
                state[f"{part}_{name}"], state[f"{part}_{name}_scales"] = _quantised(rows)
            else:
                state[f"{part}_{name}"] = rows
    state["bounds"], state["prefix_lengths"], state["suffix_lengths"] = whole(bounds), whole(prefix_lengths), whole(suffix_lengths)
    most = max(b - a for a, b in zip(bounds, bounds[1:]))
    # plain form: member `slot` of group `group` for each batch element, and the batch element at each place of the padded groups
    group = [g for g in range(groups) for _ in range(bounds[g], bounds[g + 1])]
    state["group"] = torch.tensor(group, device="cuda")
    state["slot"] = torch.tensor([b - bounds[g] for b, g in enumerate(group)], device="cuda")
    state["padded"] = torch.tensor([[min(bounds[g] + m, batch - 1) for m in range(most)] for g in range(groups)], device="cuda")
    return state


# ---- one pass ------------------------------------------------------------------------------------------


def _axes(state):
    case, half, sections = state["case"], state["case"]["dim"] // 2, state["sections"]
    counts = torch.tensor(sections, device="cuda")
    axis = torch.repeat_interleave(torch.arange(len(sections), device="cuda"), counts, output_size=half)
    index = torch.arange(half, device="cuda", dtype=torch.float64)
    if case["own_spectrum"]:
        exponent = (index - (torch.cumsum(counts, 0) - counts)[axis]) / counts[axis]
    else:
        exponent = index / half
    frequency = torch.pow(torch.tensor(10000.0, device="cuda", dtype=torch.float64), -exponent)
    angle = state["positions"][axis].movedim(0, -1).double() * frequency
    return {"sine": angle.sin().float(), "cosine": angle.cos().float()}


def _rotated(x, sine, cosine):
    """x [B, T, heads, D], factors [T, 1, D/2]"""
    first, second = x.chunk(2, dim=-1)
    return torch.cat((first * cosine - second * sine, second * cosine + first * sine), dim=-1)


def _encoded(x):
    """fp32 rows -> (e4m3 codes, fp32 scales) as a cache holds them"""
    largest = x.abs().amax(-1)
    scale = torch.where(largest < TINY, 0.0, torch.where(largest < HUGE, largest / E4M3_MAX, math.nan))
    codes = (x / scale.unsqueeze(-1)).clamp(-E4M3_MAX, E4M3_MAX)
    return torch.where(scale.unsqueeze(-1) == 0, 0.0, codes).to(torch.float8_e4m3fn), scale


def _write(state):
    case = state["case"]
    heads, kv_heads = case["heads"], case["kv_heads"]
    x = state["qkv"].float()
    sine, cosine = state["sine"].unsqueeze(1), state["cosine"].unsqueeze(1)
    b, t, position = state["real"]
    q = _rotated(x[:, :, :heads], sine, cosine).to(torch.bfloat16)
    state["q_out"][b, :, t] = q[b, t]
    for name, rows in (("k", _rotated(x[:, :, heads: heads + kv_heads], sine, cosine)), ("v", x[:, :, heads + kv_heads:])):
        codes, scales = _encoded(rows)
        state[name + "_codes"].view(torch.uint8)[b, :, position] = codes.view(torch.uint8)[b, t]
        state[name + "_scales"][b, :, position] = scales[b, t]
    return {name: state[name] for name in ("q_out", "k_codes", "k_scales", "v_codes", "v_scales")}


def _read(state):
    inside = torch.arange(state["case"]["capacity"], device="cuda") < state["lengths"].unsqueeze(1)      # [B, capacity]
    result = {}
    for name in ("k", "v"):
        values = (state[name + "_codes"].float() * state[name + "_scales"].unsqueeze(-1)).to(torch.bfloat16)
        result[name] = torch.where(inside[:, None, :, None], values, state[name + "_out"])
    return result


def _stored(state, name):
    values = state[name].float()
    return values * state[name + "_scales"].unsqueeze(-1) if state["case"]["fp8"] else values


def _part(scores, visible, values):
    """Softmax statistics and the unnormalised output over one part of the keys."""
    scores = torch.where(visible, scores, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min(-1e30)
    weights = torch.exp(scores - top)
    return top, weights.sum(-1, keepdim=True), weights @ values


def _attention(state):
    case = state["case"]
    groups, heads, kv_heads, tokens, dim = (case[k] for k in ("groups", "heads", "kv_heads", "tokens", "dim"))
    share = heads // kv_heads
    batch = state["q"].shape[0]
    q = state["q"].float().view(batch, kv_heads, share * tokens, dim) / math.sqrt(dim)
    # the prefix part: all members of a group against its one prefix
    most = state["padded"].shape[1]
    together = q[state["padded"]].permute(0, 2, 1, 3, 4).reshape(groups, kv_heads, most * share * tokens, dim)
    seen = torch.arange(case["prefix"], device="cuda") < state["prefix_lengths"][:, None, None, None]
    part = _part(together @ _stored(state, "prefix_k").transpose(-1, -2), seen, _stored(state, "prefix_v"))
    back = lambda x: x.view(groups, kv_heads, most, share * tokens, -1).transpose(1, 2)[state["group"], state["slot"]]
    top, total, output = (back(x) for x in part)
    # each member's own keys
    limit = state["suffix_lengths"][:, None].expand(batch, tokens)
    if case["causal"]:
        limit = (limit - tokens + 1 + torch.arange(tokens, device="cuda")).clamp_min(0)
    limit = limit.repeat(1, share)[:, None, :, None]
    seen = torch.arange(case["suffix"], device="cuda") < limit
    own_top, own_total, own_output = _part(q @ _stored(state, "suffix_k").transpose(-1, -2), seen, _stored(state, "suffix_v"))
    both = torch.maximum(top, own_top)
    a, b = torch.exp(top - both), torch.exp(own_top - both)
    total = a * total + b * own_total
    result = torch.where(total > 0, (a * output + b * own_output) / total, 0.0)
    return result.view(batch, heads, tokens, dim).to(torch.bfloat16)


def _own(state):
    from embodiinfer_b200 import kernels as K
    from embodiinfer_b200.kv_cache import QuantizedKVCache

    case = state["case"]
    cache = lambda prefix, k="_codes", s="_scales": QuantizedKVCache(state[f"{prefix}k{k}"], state[f"{prefix}k{s}"], state[f"{prefix}v{k}"], state[f"{prefix}v{s}"])
    if case["op"] == "axes":
        sine, cosine = K.rope_axes(state["positions"], state["sections"], theta=10000.0, own_spectrum=case["own_spectrum"])
        return {"sine": sine, "cosine": cosine}
    if case["op"] == "write":
        heads, kv_heads = case["heads"], case["kv_heads"]
        rows = state["qkv"].transpose(1, 2)          # [B, heads, T, D], a view
        K.kv_cache_write(rows[:, heads: heads + kv_heads], rows[:, heads + kv_heads:], cache(""), q=rows[:, :heads], q_out=state["q_out"],
                         sine=state["sine"], cosine=state["cosine"], offsets=state["offsets"], lengths=state["lengths"])
        return {name: state[name] for name in ("q_out", "k_codes", "k_scales", "v_codes", "v_scales")}
    if case["op"] == "read":
        K.kv_cache_read(cache(""), state["k_out"], state["v_out"], lengths=state["lengths"])
        return {"k": state["k_out"], "v": state["v_out"]}
    if case["fp8"]:
        prefix, suffix = cache("prefix_", "", "_scales"), cache("suffix_", "", "_scales")
    else:
        prefix, suffix = (state["prefix_k"], state["prefix_v"]), (state["suffix_k"], state["suffix_v"])
    return K.prefix_attention(state["q"], prefix, suffix, members=state["bounds"], prefix_lengths=state["prefix_lengths"],
                              own_lengths=state["suffix_lengths"], causal=case["causal"])


def run(state):
    if own:
        return _own(state)
    return {"axes": _axes, "write": _write, "read": _read, "attention": _attention}[state["case"]["op"]](state)


# ---- what a pass cannot do without ---------------------------------------------------------------------


def work(case):
    if case["op"] == "axes":
        count = case["batch"] * case["tokens"]
        return {"bytes": count * (8 * case["axes"] + 4 * case["dim"]), "flops": count * case["dim"]}
    dim, kv_heads = case["dim"], case["kv_heads"]
    if case["op"] == "write":
        heads, tokens = case["heads"], sum(_write_plan(case)[1])
        per_token = (heads + 2 * kv_heads) * dim * 2 + heads * dim * 2 + 2 * kv_heads * (dim + 4)
        return {"bytes": tokens * per_token + case["tokens"] * dim * 4, "flops": tokens * dim * (3 * heads + 6 * kv_heads)}
    if case["op"] == "read":
        rows = sum(_read_lengths(case)) * kv_heads * 2
        return {"bytes": rows * (dim + 4 + 2 * dim), "flops": rows * dim}
    bounds, prefix_lengths, suffix_lengths = _attention_plan(case)
    heads, tokens = case["heads"], case["tokens"]
    per_row = dim + 4 if case["fp8"] else 2 * dim
    size = 2 * kv_heads * per_row * (sum(prefix_lengths) + sum(suffix_lengths)) + 2 * 2 * bounds[-1] * heads * tokens * dim
    pairs = sum((bounds[g + 1] - bounds[g]) * prefix_lengths[g] * tokens for g in range(case["groups"]))
    for length in suffix_lengths:
        pairs += sum(max(0, length - tokens + t + 1) for t in range(tokens)) if case["causal"] else length * tokens
    return {"bytes": size, "flops": 4 * dim * heads * pairs}


# ---- the operators' definitions in 64 bits ---------------------------------------------------------------


def _exact_axes(case, state):
    positions = state["positions"].cpu().numpy().astype(np.float64)
    half, start = case["dim"] // 2, 0
    angles = np.empty((case["batch"], case["tokens"], half))
    for axis, count in enumerate(state["sections"]):
        for j in range(count):
            power = j / count if case["own_spectrum"] else (start + j) / half
            angles[:, :, start + j] = positions[axis] * 10000.0 ** -power
        start += count
    return {"sine": np.sin(angles), "cosine": np.cos(angles)}


def _exact_write(case, state):
    heads, kv_heads, half = case["heads"], case["kv_heads"], case["dim"] // 2
    x = state["qkv"].double()
    turn = torch.complex(state["cosine"].double(), state["sine"].double()).unsqueeze(1)
    z = torch.complex(x[:, :, : heads + kv_heads, :half].contiguous(), x[:, :, : heads + kv_heads, half:].contiguous()) * turn
    turned = torch.cat((z.real, z.imag), dim=-1)
    result = {"q_out": state["q_out"].double()}
    offsets, lengths = _write_plan(case)
    for b in range(case["batch"]):
        result["q_out"][b, :, : lengths[b]] = turned[b, : lengths[b], :heads].transpose(0, 1)
    for name, rows in (("k", turned[:, :, heads:]), ("v", x[:, :, heads + kv_heads:])):
        codes, scales = state[name + "_codes"].float().double(), state[name + "_scales"].double()
        for b in range(case["batch"]):
            fresh = rows[b, : lengths[b]].transpose(0, 1)
            size = fresh.abs().amax(-1) / E4M3_MAX
            codes[b, :, offsets[b]: offsets[b] + lengths[b]] = fresh / size.unsqueeze(-1)
            scales[b, :, offsets[b]: offsets[b] + lengths[b]] = size
        result[name + "_codes"], result[name + "_scales"] = codes, scales
    return result


def _exact_read(case, state):
    result = {}
    for name in ("k", "v"):
        result[name] = torch.zeros(state[name + "_out"].shape, device="cuda", dtype=torch.float64)
        for b, length in enumerate(_read_lengths(case)):
            scale = state[name + "_scales"][b, :, :length, None].double()
            result[name][b, :, :length] = state[name + "_codes"][b, :, :length].float().double() * scale
    return result


def _exact_attention(case, state):
    heads, kv_heads, tokens, dim = (case[k] for k in ("heads", "kv_heads", "tokens", "dim"))
    bounds, prefix_lengths, suffix_lengths = _attention_plan(case)

    def stored(name, index, length):
        values = state[name][index, :, :length].float().double()
        return values * state[name + "_scales"][index, :, :length, None].double() if case["fp8"] else values

    result = torch.zeros(state["q"].shape, device="cuda", dtype=torch.float64)
    for g in range(case["groups"]):
        shared = [stored("prefix_" + name, g, prefix_lengths[g]).repeat_interleave(heads // kv_heads, 0) for name in ("k", "v")]
        for b in range(bounds[g], bounds[g + 1]):
            length = suffix_lengths[b]
            mine = [stored("suffix_" + name, b, length).repeat_interleave(heads // kv_heads, 0) for name in ("k", "v")]
            keys, values = (torch.cat(pair, 1) for pair in zip(shared, mine))
            scores = torch.einsum("htd,hsd->hts", state["q"][b].double(), keys) * dim ** -0.5
            if case["causal"]:
                last = prefix_lengths[g] + length - tokens + torch.arange(tokens, device="cuda")
                scores.masked_fill_(torch.arange(keys.shape[1], device="cuda") > last[:, None], -math.inf)
            result[b] = torch.softmax(scores, -1) @ values
    return result


def exact(case, seed):
    state = prepare(case, seed)
    return {"axes": _exact_axes, "write": _exact_write, "read": _exact_read, "attention": _exact_attention}[case["op"]](case, state)
