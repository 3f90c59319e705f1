"""Attention over shared prefixes against a plain implementation in 64 bits."""

from __future__ import annotations

import math

import pytest
import torch

from embodiinfer_b200 import _native as N
from embodiinfer_b200 import kernels as K
from embodiinfer_b200.kv_cache import QuantizedKVCache

pytestmark = pytest.mark.gpu


def values_of(part):
    """The cache's keys and values in 64 bits."""
    if isinstance(part, QuantizedKVCache):
        return tuple(codes.view(torch.float8_e4m3fn).float().double() * scales.double()[..., None]
                     for codes, scales in ((part.k_codes, part.k_scales), (part.v_codes, part.v_scales)))
    return tuple(t.double() for t in part)


def reference(q, prefix, own, bounds, prefix_lengths, own_lengths, causal, scale):
    """(output, bound of the kernel's error), both [B, H, T, D] in 64 bits.

    The bound, with A = sum p |v| (p the probabilities) and one rounding off by at most half a step:
      output to bf16                   2^-8 |out|
      probabilities                    2^-8 A (bf16 cache) or 2^-11 A + (keys) 2^-25 max|v| (f16 weights of at most 1 beside a largest
                                       one of at least 1, subnormal below 2^-14)
      scores, 2 e A: fp32 sums of D products, e = 2 D 2^-24 sum |q k| scale, + the argument and the result of the base-2
                                       exponential, 2^-22 (|score| + 1); quantised: q's second half below 2^-17 of the row's largest value
      sums over the keys in fp32       2 (keys) 2^-24 A
    """
    batch, heads, queries, dim = q.shape
    quantised = isinstance(prefix, QuantizedKVCache)
    shared_k, shared_v = values_of(prefix)
    own_k, own_v = values_of(own) if own is not None else (None, None)
    share = heads // shared_k.shape[1]
    out, bound = torch.zeros((2, *q.shape), device=q.device, dtype=torch.float64)
    for g in range(shared_k.shape[0]):
        for b in range(bounds[g], bounds[g + 1]):
            keys, values, count = shared_k[g, :, :prefix_lengths[g]], shared_v[g, :, :prefix_lengths[g]], prefix_lengths[g]
            if own is not None:
                keys, values = torch.cat((keys, own_k[b, :, :own_lengths[b]]), 1), torch.cat((values, own_v[b, :, :own_lengths[b]]), 1)
                count += own_lengths[b]
            if count == 0:
                continue
            keys, values = keys.repeat_interleave(share, 0), values.repeat_interleave(share, 0)
            rows = q[b].double()
            scores = scale * rows @ keys.transpose(-1, -2)
            seen = torch.full((queries,), count, device=q.device)
            if causal:
                seen = seen - queries + 1 + torch.arange(queries, device=q.device)
                seen = seen.clamp_min(prefix_lengths[g])
            masked = torch.arange(count, device=q.device) >= seen[:, None]
            scores = scores.masked_fill(masked, -math.inf)
            p = torch.softmax(scores, -1).nan_to_num(0.0) if (seen == 0).any() else torch.softmax(scores, -1)
            out[b] = p @ values
            # bound
            size = scale * rows.abs() @ keys.abs().transpose(-1, -2)
            e = (2 * dim * 2.0 ** -24 * size + 2.0 ** -22 * (size + 1)).masked_fill(masked, 0.0)
            if quantised:
                e = e + 2.0 ** -17 * scale * rows.abs().amax(-1, keepdim=True) * keys.abs().sum(-1)[:, None]
            weighted = p @ values.abs()
            e_bound = (2 * e.masked_fill(masked, 0.0).amax(-1, keepdim=True)) * weighted
            rounding = 2.0 ** -11 * weighted + count * 2.0 ** -25 * values.abs().amax() if quantised else 2.0 ** -8 * weighted
            bound[b] = 2.0 ** -8 * out[b].abs() + (1 + 2.0 ** -6) * (rounding + e_bound + 2 * count * 2.0 ** -24 * weighted)
    return out, bound


def make_cache(generator, count, kv_heads, capacity, dim, quantised, device, stale=None):
    """Random keys and values; rows behind `stale[i]` hold NaN."""
    parts = []
    for _ in range(2):
        rows = torch.randn((count, kv_heads, capacity, dim), device=device, generator=generator)
        rows = (rows * torch.exp(0.5 * torch.randn((count, kv_heads, capacity, 1), device=device, generator=generator))).to(torch.bfloat16)
        if not quantised:
            if stale is not None:
                for i, length in enumerate(stale):
                    rows[i, :, length:] = math.nan
            parts.append(rows)
            continue
        scale = rows.float().abs().amax(-1) / 448.0
        codes = (rows.float() / scale[..., None]).to(torch.float8_e4m3fn)
        if stale is not None:
            for i, length in enumerate(stale):
                codes.view(torch.uint8)[i, :, length:], scale[i, :, length:] = 0x7f, math.nan
        parts += [codes, scale]
    return QuantizedKVCache(*parts) if quantised else tuple(parts)


def whole(values, device):
    return torch.tensor(values, device=device, dtype=torch.int32)


def check(got, want, bound):
    assert not got.isnan().any()
    excess = (got.double() - want).abs() - bound
    assert (excess <= 0).all(), f"{int((excess > 0).sum())} of {excess.numel()} values off by up to {float(excess.max()):.3g} more than their bound"


def run_case(device, bounds, heads, kv_heads, queries, dim, prefix, own, causal, quantised, prefix_lengths=None, own_lengths=None, uniform=False, seed=0):
    generator = torch.Generator(device=device).manual_seed(1000 * queries + prefix + seed)
    batch, groups = bounds[-1], len(bounds) - 1
    q = (1.5 * torch.randn((batch, heads, queries, dim), device=device, generator=generator)).to(torch.bfloat16)
    shared = make_cache(generator, groups, kv_heads, prefix, dim, quantised, device, prefix_lengths)
    mine = make_cache(generator, batch, kv_heads, own, dim, quantised, device, own_lengths) if own is not None else None
    got = K.prefix_attention(q, shared, mine, members=None if uniform else whole(bounds, device),
                             prefix_lengths=None if prefix_lengths is None else whole(prefix_lengths, device),
                             own_lengths=None if own_lengths is None else whole(own_lengths, device), causal=causal)
    K.check_status(device)
    want, bound = reference(q, shared, mine, bounds, prefix_lengths or [prefix] * groups, own_lengths or [own or 0] * batch, causal, dim ** -0.5)
    check(got, want, bound)
    return got


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("bounds,heads,kv_heads,queries,prefix,own,causal", [
    ([0, 1], 1, 1, 1, 1, None, False),                   # one row, one key
    ([0, 1], 8, 1, 1, 63, 1, True),
    ([0, 1], 8, 1, 10, 64, 10, False),
    ([0, 4], 8, 1, 10, 560, 10, False),                  # one observation, four action samples
    ([0, 2, 4, 6], 8, 1, 10, 65, 10, True),
    ([0, 3], 8, 8, 1, 130, 70, True),                    # a key/value head per query head: a row of every member in a tile
    ([0, 5], 28, 4, 3, 200, 64, True),
    ([0, 1], 2, 1, 200, 129, 200, True),                 # a prompt behind a prefix: several row tiles of one member
    ([0, 130], 1, 1, 1, 70, 3, False),                   # 130 members of one row each
    ([0, 40], 16, 2, 4, 300, 20, True),
])
def test_matches_the_reference(device, bounds, heads, kv_heads, queries, dim, prefix, own, causal, quantised):
    run_case(device, bounds, heads, kv_heads, queries, dim, prefix, own, causal, quantised, uniform=True)


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("bounds,heads,kv_heads,queries,dim,prefix_lengths,own_lengths,causal", [
    ([0, 3, 3, 4], 8, 1, 10, 256, [100, 7, 0], [10, 3, 0, 1], False),                         # an empty group, an empty prefix
    ([0, 1, 2, 3], 8, 1, 4, 256, [0, 0, 65], [0, 2, 0], True),                                # rows that see no key
    ([0, 2, 7, 8], 8, 2, 1, 128, [640, 64, 1], [1, 64, 65, 0, 128, 5, 127, 20], False),
    ([0, 9, 10, 45], 4, 4, 2, 128, [33, 500, 128], [(11 * b) % 40 for b in range(45)], True),
    ([0, 1, 2], 8, 1, 50, 256, [712, 360], [50, 49], True)])
def test_lengths_and_unequal_groups(device, bounds, heads, kv_heads, queries, dim, prefix_lengths, own_lengths, causal, quantised):
    """Rows behind the lengths hold NaN."""
    run_case(device, bounds, heads, kv_heads, queries, dim, max(prefix_lengths) + 9, max(own_lengths) + 1, causal, quantised, prefix_lengths, own_lengths)


def test_many_groups(device):
    """More groups than a warp has lanes, some of them empty."""
    counts = [(3 * g) % 4 for g in range(75)]
    bounds = [sum(counts[:g]) for g in range(76)]
    run_case(device, bounds, 4, 1, 3, 128, 90, 5, False, True, [(7 * g) % 91 for g in range(75)], [b % 6 for b in range(bounds[-1])])


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("dim", [128, 256])
def test_cut_and_uncut_launches_agree(device, monkeypatch, dim, quantised):
    """A long prefix and few rows: with the workspace the keys are cut across the SMs, without it one CTA walks them all."""
    cut = run_case(device, [0, 2, 3], 8, 2, 5, dim, 2500, 100, True, quantised, [2500, 1900], [100, 64, 7])
    monkeypatch.setattr(N.load(), "b2_prefix_attention_workspace_bytes", lambda desc: 0)
    uncut = run_case(device, [0, 2, 3], 8, 2, 5, dim, 2500, 100, True, quantised, [2500, 1900], [100, 64, 7])
    assert not torch.equal(cut, uncut)          # another order of the sums: both within their bounds


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 1, 256), (16, 2, 128)])
def test_the_last_wave_is_cut(device, monkeypatch, heads, kv_heads, dim, quantised):
    """Some more row tiles than SMs, fewer than the bound that the launch is sized by: the ones behind the first wave are cut."""
    counts = [12 if g % 2 else 4 for g in range(32 // kv_heads)]
    bounds = [sum(counts[:g]) for g in range(len(counts) + 1)]
    lengths = [2000 - (137 * g) % 900 for g in range(len(counts))], [10 - b % 9 for b in range(bounds[-1])]
    cut = run_case(device, bounds, heads, kv_heads, 10, dim, 2000, 10, False, quantised, *lengths)
    monkeypatch.setattr(N.load(), "b2_prefix_attention_workspace_bytes", lambda desc: 0)
    uncut = run_case(device, bounds, heads, kv_heads, 10, dim, 2000, 10, False, quantised, *lengths)
    assert (cut == uncut).flatten(1).all(1).sum() >= bounds[-1] // 2 and not torch.equal(cut, uncut)          # most are in the whole wave


def test_uniform_groups_in_several_waves(device):
    """No bounds given, more row tiles than SMs: the row tiles are taken in the order of their prefixes' lengths."""
    bounds = [10 * g for g in range(25)]
    run_case(device, bounds, 8, 1, 10, 256, 130, 10, True, True, [(59 * g) % 131 for g in range(24)], [b % 11 for b in range(240)], uniform=True)


def test_without_a_prefix(device):
    generator = torch.Generator(device=device).manual_seed(5)
    q = torch.randn((3, 8, 4, 128), device=device, generator=generator).to(torch.bfloat16)
    own = make_cache(generator, 3, 2, 40, 128, False, device)
    empty = tuple(t[:1, :, :0].contiguous() for t in own)
    got = K.prefix_attention(q, empty, own, causal=True)
    check(got, *reference(q, empty, own, [0, 3], [0], [40] * 3, True, 128 ** -0.5))
    nothing = K.prefix_attention(q, empty)
    assert not nothing.any()
    assert K.prefix_attention(q[:0], empty, tuple(t[:0] for t in own), members=whole([0, 0], device)).shape == (0, 8, 4, 128)


def test_strided_queries_scale_and_output(device):
    generator = torch.Generator(device=device).manual_seed(6)
    packed = torch.randn((2, 6, 12 * 128 + 8), device=device, generator=generator).to(torch.bfloat16)
    q = packed[:, :, : 12 * 128].unflatten(-1, (12, 128)).transpose(1, 2)[:, :8]          # token before head, rows longer than used
    shared, own = make_cache(generator, 1, 4, 77, 128, True, device), make_cache(generator, 2, 4, 6, 128, True, device)
    out = torch.empty((2, 8, 6, 128), device=device, dtype=torch.bfloat16)
    assert K.prefix_attention(q, shared, own, scale=0.3, out=out) is out
    check(out, *reference(q, shared, own, [0, 2], [77], [6, 6], False, 0.3))


@pytest.mark.parametrize("quantised", [False, True])
def test_not_finite_values_stay_with_the_rows_that_see_them(device, quantised):
    """Member 1 of three in one row tile has a key, a value or a query that is not finite."""
    generator = torch.Generator(device=device).manual_seed(7)
    q = torch.randn((3, 8, 4, 128), device=device, generator=generator).to(torch.bfloat16)
    shared = make_cache(generator, 1, 1, 30, 128, quantised, device)
    for what in ("key", "value", "query", "late value"):
        own = make_cache(generator, 3, 1, 20, 128, quantised, device)
        changed = q.clone()
        clean_own = tuple(t.clone() for t in own)
        want = K.prefix_attention(changed, shared, QuantizedKVCache(*clean_own) if quantised else clean_own, causal=True)
        position = 19 if what == "late value" else 5
        if what == "query":
            changed[1, 2, 3, 100] = math.inf
        elif quantised:
            own[1 if what == "key" else 3][1, 0, position] = math.nan
        else:
            own[0 if what == "key" else 1][1, 0, position, 17] = math.inf if what != "key" else math.nan
        got = K.prefix_attention(changed, shared, own, causal=True)
        touched = torch.zeros((3, 8, 4), device=device, dtype=torch.bool)
        if what == "query":
            touched[1, 2, 3] = True
        else:
            touched[1, :, max(0, position - 16):] = True          # causal: query t sees 17 + t own keys
        assert got[touched].isnan().all() if what != "query" or quantised else got[touched].isnan().any()
        assert torch.equal(got[~touched], want[~touched])


def test_extreme_scores(device):
    """One key far above the rest, far below them, and scores that move by hundreds from tile to tile."""
    generator = torch.Generator(device=device).manual_seed(8)
    for quantised in (False, True):
        q = torch.randn((2, 4, 2, 128), device=device, generator=generator).to(torch.bfloat16)
        rows = torch.randn((1, 1, 400, 128), device=device, generator=generator) * torch.linspace(0.1, 30.0, 400, device=device)[:, None]
        rows[0, 0, 210] *= 20.0
        keys, values = rows.to(torch.bfloat16), (rows.flip(2) * 1e-3).to(torch.bfloat16)
        shared = (keys, values)
        if quantised:
            shared = QuantizedKVCache.allocate(1, 1, 400, 128, device)
            K.kv_cache_write(keys, values, shared)
        got = K.prefix_attention(q, shared)
        check(got, *reference(q, shared, None, [0, 2], [400], [0, 0], False, 128 ** -0.5))


def test_quantised_rows_of_zeros_and_of_unequal_size(device):
    """Value rows of zeros count in the sum; value scales that differ by 2^40 keep the precision of every row."""
    generator = torch.Generator(device=device).manual_seed(9)
    keys = torch.randn((1, 1, 150, 256), device=device, generator=generator)
    values = torch.randn((1, 1, 150, 256), device=device, generator=generator)
    values[0, 0, ::3] = 0.0
    values[0, 0, 1::3] *= 2.0 ** -40
    keys[0, 0, 100:] = 0.0
    cache = QuantizedKVCache.allocate(1, 1, 150, 256, device)
    K.kv_cache_write(keys.to(torch.bfloat16), values.to(torch.bfloat16), cache)
    q = torch.randn((1, 8, 3, 256), device=device, generator=generator).to(torch.bfloat16)
    got = K.prefix_attention(q, cache)
    check(got, *reference(q, cache, None, [0, 1], [150], [0], False, 1 / 16))
    # rows that see nothing but the small values keep them
    small = K.prefix_attention(q, cache, prefix_lengths=whole([2], device))
    want, bound = reference(q, cache, None, [0, 1], [2], [0], False, 1 / 16)
    check(small, want, bound)
    assert want.abs().max() < 2.0 ** -36 and small.abs().max() > 0


def test_capture_replay_streams_and_repetition(device):
    """Two graphs replayed at the same time on two streams, beside eager calls on a third: each has its own scratch."""
    generator = torch.Generator(device=device).manual_seed(10)
    cases = []
    for seed in range(2):
        q = torch.randn((2, 8, 10, 256), device=device, generator=generator).to(torch.bfloat16)
        shared, own = make_cache(generator, 1, 1, 1500, 256, seed == 1, device), make_cache(generator, 2, 1, 10, 256, seed == 1, device)
        cases.append((q, shared, own))
    want = [K.prefix_attention(*case) for case in cases]
    graphs, outs = [], []
    for case in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(K.prefix_attention(*case))
        graphs.append(graph)
    streams = [torch.cuda.Stream(device) for _ in range(3)]
    torch.cuda.synchronize()
    eager = []
    for _ in range(20):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        with torch.cuda.stream(streams[2]):
            eager.append(K.prefix_attention(*cases[0]))
    torch.cuda.synchronize()
    K.check_status(device)
    for got, expected in zip(outs, want):
        assert torch.equal(got, expected)
    assert all(torch.equal(got, want[0]) for got in eager)
    del graphs


@pytest.mark.parametrize("quantised", [False, True])
def test_a_replay_follows_the_device_data(device, quantised):
    """Bounds and lengths are read when the launch runs: a captured call of few row tiles, and so its cut, follows them."""
    generator = torch.Generator(device=device).manual_seed(12)
    batch, groups, prefix, own = 9, 3, 900, 70
    q = (1.5 * torch.randn((batch, 8, 3, 128), device=device, generator=generator)).to(torch.bfloat16)
    shared, mine = make_cache(generator, groups, 2, prefix, 128, quantised, device), make_cache(generator, batch, 2, own, 128, quantised, device)
    bounds, prefix_lengths, own_lengths = whole([0, 3, 6, 9], device), whole([prefix] * groups, device), whole([own] * batch, device)
    run = lambda: K.prefix_attention(q, shared, mine, members=bounds, prefix_lengths=prefix_lengths, own_lengths=own_lengths, causal=True)
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for new in (([0, 3, 6, 9], [900, 900, 900], [70] * 9), ([0, 9, 9, 9], [5, 900, 0], [1, 70, 0, 3, 64, 65, 2, 69, 7]),
                ([0, 0, 1, 9], [900, 63, 640], [0] * 9), ([0, 1, 8, 9], [0, 1, 128], [0, 9, 9, 9, 0, 0, 1, 2, 0])):
        for tensor, values in zip((bounds, prefix_lengths, own_lengths), new):
            tensor.copy_(whole(values, device))
        got.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        K.check_status(device)
        check(got, *reference(q, shared, mine, *new, True, 128 ** -0.5))
    del graph


def test_keys_behind_four_gigabytes(device):
    """The last group's rows start beyond 2^32 bytes; only what the lengths cover is ever written or read."""
    if torch.cuda.mem_get_info(device)[0] < 40 << 30:
        pytest.skip("needs 40 GB of device memory")
    generator = torch.Generator(device=device).manual_seed(11)
    groups, capacity, lengths = 3, 4_500_000, [5, 0, 150]
    shared = tuple(torch.empty((groups, 1, capacity, 256), device=device, dtype=torch.bfloat16) for _ in range(2))
    small = make_cache(generator, groups, 1, 150, 256, False, device)
    for large, rows in zip(shared, small):
        large[:, :, :150] = rows
    q = torch.randn((3, 8, 1, 256), device=device, generator=generator).to(torch.bfloat16)
    got = K.prefix_attention(q, shared, prefix_lengths=whole(lengths, device))
    check(got, *reference(q, small, None, [0, 1, 2, 3], lengths, [0] * 3, False, 1 / 16))


def test_refuses(device):
    q = torch.zeros((4, 8, 2, 128), device=device, dtype=torch.bfloat16)
    shared = tuple(torch.zeros((2, 2, 16, 128), device=device, dtype=torch.bfloat16) for _ in range(2))
    own = tuple(torch.zeros((4, 2, 4, 128), device=device, dtype=torch.bfloat16) for _ in range(2))
    quantised = QuantizedKVCache.allocate(4, 2, 4, 128, device)
    for bad in (lambda: K.prefix_attention(q.float(), shared), lambda: K.prefix_attention(q, None, own), lambda: K.prefix_attention(q, shared, quantised),
                lambda: K.prefix_attention(q, shared, tuple(t[:3] for t in own)), lambda: K.prefix_attention(q[..., :64], shared),
                lambda: K.prefix_attention(q[:3], shared), lambda: K.prefix_attention(q[:, :7], shared),
                lambda: K.prefix_attention(q, (shared[0], shared[1][:, :, :8])), lambda: K.prefix_attention(q, tuple(t.transpose(1, 2) for t in shared)),
                lambda: K.prefix_attention(q, shared, members=whole([0, 4], device)), lambda: K.prefix_attention(q, shared, prefix_lengths=whole([1], device)),
                lambda: K.prefix_attention(q, shared, own, own_lengths=torch.zeros(4, device=device)),
                lambda: K.prefix_attention(q, shared, out=torch.empty((4, 8, 2, 128), device=device)), lambda: K.prefix_attention(q.cpu(), shared)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="error -1"):
        K.prefix_attention(q, shared, scale=-1.0)


def test_out_of_order_members_stay_in_bounds(device):
    """Group bounds that the documentation forbids: no access leaves the batch, members of no group keep their output."""
    generator = torch.Generator(device=device).manual_seed(12)
    q = torch.randn((4, 8, 2, 128), device=device, generator=generator).to(torch.bfloat16)
    shared = make_cache(generator, 2, 2, 16, 128, False, device)
    out = torch.full_like(q, 7.0)
    K.prefix_attention(q, shared, members=whole([3, -5, 900], device), out=out)          # groups [3, 0) and [0, 4) after clamping
    K.check_status(device)
    want, bound = reference(q, tuple(t[1:] for t in shared), None, [0, 4], [16], [0] * 4, False, 128 ** -0.5)
    check(out, want, bound)
