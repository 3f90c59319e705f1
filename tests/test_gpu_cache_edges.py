"""Edges of the cache operators: magnitudes, values that are not finite, layouts and positions at the end of what is allowed."""

from __future__ import annotations

import math
from decimal import Decimal, localcontext

import pytest
import torch

from embodiinfer_b200 import kernels as K
from embodiinfer_b200.kv_cache import QuantizedKVCache
from tests.test_gpu_prefix_attention import check, make_cache, reference, whole

pytestmark = pytest.mark.gpu


def written(keys, values):
    """The quantised cache of fp32 keys and values [n, kv_heads, capacity, D]."""
    cache = QuantizedKVCache.allocate(*keys.shape, keys.device)
    K.kv_cache_write(keys.to(torch.bfloat16), values.to(torch.bfloat16), cache)
    return cache


def no_keys(part):
    """A prefix cache of `part`'s kind and shape without keys."""
    empty = tuple(t[:1, :, :0].contiguous() for t in part)
    return QuantizedKVCache(*empty) if isinstance(part, QuantizedKVCache) else empty


# ---- attention: magnitudes --------------------------------------------------------------------------------


@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("exponents", [(38, -49), (-49, 38), (38, -20, -49)])
def test_members_of_one_row_tile_with_values_from_both_ends_of_the_range(device, dim, exponents):
    """A member's values keep their precision whatever its neighbours' are.  Beside the reference's bound a value is off by the roundings
    of its scale and of the product to f16, half a step (2^-11) each."""
    generator = torch.Generator(device=device).manual_seed(20)
    members, keys = len(exponents), 40
    size = torch.tensor([2.0 ** e for e in exponents], device=device).view(-1, 1, 1, 1)
    sign = torch.randint(0, 2, (members, 1, keys, dim), device=device, generator=generator) * 2.0 - 1.0
    values = sign * (1.0 + torch.rand((members, 1, keys, dim), device=device, generator=generator)) * size
    own = written(torch.randn((members, 1, keys, dim), device=device, generator=generator), values)
    q = torch.randn((members, 8, 4, dim), device=device, generator=generator).to(torch.bfloat16)
    got = K.prefix_attention(q, no_keys(own), own)
    want, bound = reference(q, no_keys(own), own, [0, members], [0], [keys] * members, False, dim ** -0.5)
    check(got, want, bound + 2 * 2.0 ** -11 * values.to(torch.bfloat16).double().abs().amax((1, 2, 3), keepdim=True))


@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("exponents", [(38, -49), (-49, 38)])
def test_small_values_behind_large_ones_of_no_weight(device, dim, exponents):
    """Two key tiles; the scores of the one with large values are lower by 800, a weight of 2^-1154."""
    generator = torch.Generator(device=device).manual_seed(21)
    keys = torch.zeros((1, 1, 128, dim), device=device)
    values = 1.0 + torch.rand((1, 1, 128, dim), device=device, generator=generator)
    for tile, exponent in enumerate(exponents):
        values[:, :, 64 * tile: 64 * tile + 64] *= 2.0 ** exponent
        keys[:, :, 64 * tile: 64 * tile + 64, 0] = 400.0 if exponent < 0 else -400.0
    cache = written(keys, values)
    q = torch.ones((1, 8, 1, dim), device=device, dtype=torch.bfloat16)
    got = K.prefix_attention(q, cache, scale=1.0)
    seen = 64 * exponents.index(min(exponents))
    want = (cache.v_codes.float().double() * cache.v_scales.double()[..., None])[0, 0, seen: seen + 64].mean(0)
    # all weights are 1: the result's rounding, the scale's and the product's to f16; sums of 64 positive fp32 numbers
    assert ((got.double() - want).abs() <= (2.0 ** -8 + 2 * 2.0 ** -11 + 2.0 ** -15) * want).all()


@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("query,key,scale", [(126, -48, -78), (-124, 39, 85)])
def test_queries_from_both_ends_of_the_range(device, dim, query, key, scale):
    """Query rows whose largest values are at 2^query, behind quantised keys that bring the scores back to order 1.  The query is held
    down to 2^-17 of its row's largest value, or of 2^-119 (2^-12 of 2^-124): the reference's bound with that in place of 2^-17."""
    generator = torch.Generator(device=device).manual_seed(23)
    draw = lambda *shape: 2.0 * torch.rand(shape, device=device, generator=generator) - 1.0
    q = (draw(2, 8, 3, dim) * 2.0 ** (query + 1)).to(torch.bfloat16)
    q[..., 0] = 1.5 * 2.0 ** query
    cache = written(draw(1, 1, 100, dim) * 2.0 ** key, draw(1, 1, 100, dim))
    factor = 0.25 * 2.0 ** scale
    got = K.prefix_attention(q, cache, scale=factor)
    want, bound = reference(q, cache, None, [0, 2], [100], [0, 0], False, factor)
    if query < -119:
        keys, values = (codes.float().double() * scales.double()[..., None] for codes, scales in ((cache.k_codes, cache.k_scales), (cache.v_codes, cache.v_scales)))
        lost = 2.0 ** -12 * factor * float(q.double().abs().amax() * keys.abs().sum(-1).amax())
        bound = bound + 2 * lost * float(values.abs().amax())
    check(got, want, bound)


@pytest.mark.parametrize("dim", [128, 256])
def test_a_long_tail_of_small_weights(device, dim):
    """One key of value 0 and weight 1, 2^19 of value 1 and weight e^-8 to e^-20, a part of the result from 0.99 to 0.001.  Beside the result's
    rounding: weights in f16 off by 2^-11 of themselves and 2^-32 of the largest, the exponential by 2^-22 (20 + 1), the
    weights' sum in fp32 over 2^13 tiles by 2^-24 of itself each, and the accumulator, which takes 16 keys at a time: 2^15 additions, each off
    by at most a step (the tensor core's rounding is not specified), 2^-23 of a sum that grows evenly, half of the last one on average:
    2^15 2^-23 / 2.  Rows for every SM, so that one CTA walks all keys."""
    count, rows = 1 << 19, 128 * torch.cuda.get_device_properties(device).multi_processor_count
    codes = lambda: torch.zeros((1, 1, count, dim), device=device, dtype=torch.uint8)
    k, v, scales = codes(), codes(), torch.ones((1, 1, count), device=device)
    k[0, 0, 1:, 0], v[0, 0, 1:] = 0xb8, 0x38          # -1 and 1
    q = torch.zeros((1, rows, 1, dim), device=device, dtype=torch.bfloat16)
    q[..., 0] = torch.linspace(8.0, 20.0, rows, device=device).to(torch.bfloat16)[:, None]
    got = K.prefix_attention(q, QuantizedKVCache(k, scales, v, scales), scale=1.0)
    tail = (count - 1) * torch.exp(-q[..., :1].double())
    want = (tail / (1.0 + tail)).expand_as(got)
    bound = (2.0 ** -8 + 2.0 ** -11 + 2.0 ** -22 * 21 + 2.0 ** 13 * 2.0 ** -24 + 2.0 ** 15 * 2.0 ** -23 / 2) * want + count * 2.0 ** -32 / (1.0 + tail)
    check(got, want, bound)


# ---- attention: values that are not finite ----------------------------------------------------------------


@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("which", ["k_codes", "v_codes"])
@pytest.mark.parametrize("code", [0x7f, 0xff])
def test_codes_that_are_nan_under_a_finite_scale(device, dim, which, code):
    """An own key's reach the rows that see it, a prefix key's all rows (a value's: its column, in whole and partial key tiles alike);
    those behind a length reach none."""
    generator = torch.Generator(device=device).manual_seed(22)
    q = torch.randn((3, 8, 4, dim), device=device, generator=generator).to(torch.bfloat16)
    own = make_cache(generator, 3, 1, 20, dim, True, device)

    def with_code(cache, b, position):
        changed = cache._replace(**{which: getattr(cache, which).clone()})
        getattr(changed, which).view(torch.uint8)[b, 0, position, 17] = code
        return changed

    for length in (30, 64, 100):
        shared = make_cache(generator, 1, 1, 128, dim, True, device, [length])
        shared.k_scales.nan_to_num_(1.0), shared.v_scales.nan_to_num_(1.0)          # behind the length: NaN codes, finite scales
        run = lambda prefix, mine: K.prefix_attention(q, prefix, mine, causal=True, prefix_lengths=whole([length], device))
        want = run(shared, own)
        assert not want.isnan().any()
        for position in (5, 19):
            got = run(shared, with_code(own, 1, position))
            touched = torch.zeros((3, 8, 4), device=device, dtype=torch.bool)
            touched[1, :, max(0, position - 16):] = True          # causal: query t sees 17 + t own keys
            assert got[touched].isnan().all() and torch.equal(got[~touched], want[~touched])
        for position in (3, length - 1):
            got = run(with_code(shared, 0, position), own)
            if which == "k_codes":
                assert got.isnan().all()
            else:
                others = torch.arange(dim, device=device) != 17
                assert got[..., 17].isnan().all() and torch.equal(got[..., others], want[..., others])


def test_codes_that_are_nan_in_cut_launches_and_many_members(device):
    """One row tile of 128 members, and keys cut across SMs: only the rows of the member with the NaN are touched."""
    generator = torch.Generator(device=device).manual_seed(25)
    for members, heads, own_keys, position in ((128, 1, 70, 69), (3, 8, 3000, 2500)):
        q = torch.randn((members, heads, 1, 128), device=device, generator=generator).to(torch.bfloat16)
        own = make_cache(generator, members, 1, own_keys, 128, True, device)
        want = K.prefix_attention(q, no_keys(own), own)
        changed = own._replace(v_codes=own.v_codes.clone())
        changed.v_codes.view(torch.uint8)[1, 0, position, 100] = 0x7f
        got = K.prefix_attention(q, no_keys(own), changed)
        assert got[1].isnan().all() and torch.equal(got[[0, *range(2, members)]], want[[0, *range(2, members)]])
        seen = K.prefix_attention(q, no_keys(own), changed, own_lengths=whole([position] * members, device))
        assert torch.equal(seen, K.prefix_attention(q, no_keys(own), own, own_lengths=whole([position] * members, device)))


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("own_keys", [9, 2000])          # 2000: cut across SMs
def test_a_query_that_is_not_finite_and_sees_no_key(device, dim, quantised, own_keys):
    """Members of one row tile: the one without keys is zero, whatever its queries hold."""
    generator = torch.Generator(device=device).manual_seed(24)
    q = torch.randn((3, 8, 2, dim), device=device, generator=generator).to(torch.bfloat16)
    want_q = q.clone()
    q[1, 3, 0, 7], q[1, 4, 1, 7] = math.nan, math.inf
    own = make_cache(generator, 3, 1, own_keys, dim, quantised, device)
    lengths = whole([own_keys, 0, 3], device)
    got, want = (K.prefix_attention(queries, no_keys(own), own, own_lengths=lengths) for queries in (q, want_q))
    assert not got[1].any() and not got.isnan().any() and torch.equal(got, want)
    causal = K.prefix_attention(q, no_keys(own), own, own_lengths=whole([own_keys, 1, 3], device), causal=True)          # query 0 sees nothing
    assert not causal[1, :, 0].any() and not causal[[0, 2]].isnan().any()
    assert causal[1, 4, 1].isnan().all() or not quantised          # bf16: its one score is an infinity of either sign


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("own_keys", [20, 2500])          # 2500: cut across SMs
def test_scores_of_minus_infinity(device, dim, quantised, own_keys):
    """A key whose score is -inf has no weight; a row that sees no other is NaN, one that sees no key at all zero."""
    generator = torch.Generator(device=device).manual_seed(26)
    q = torch.rand((4, 8, 2, dim), device=device, generator=generator).add(0.5).to(torch.bfloat16)
    own = make_cache(generator, 4, 1, own_keys, dim, quantised, device)
    def sink(b, keys):          # all channels negative and one, or the scale, infinite: -inf for these queries
        if quantised:
            own.k_codes.view(torch.uint8)[b, 0, keys] = 0xb8
            own.k_scales[b, 0, keys] = math.inf
        else:
            own[0][b, 0, keys] = -1.0
            own[0][b, 0, keys, 5] = -math.inf
    sink(0, own_keys - 1), sink(1, slice(None)), sink(2, slice(None))
    run = lambda *lengths: K.prefix_attention(q, no_keys(own), own, own_lengths=whole(lengths, device))
    got = run(own_keys, own_keys, 0, own_keys)
    assert torch.equal(got[[0, 3]], run(own_keys - 1, own_keys, 0, own_keys)[[0, 3]])          # (the same key tiles)
    assert not got[[0, 3]].isnan().any()
    assert got[1].isnan().all() and not got[2].any()
    assert run(own_keys, 1, 1, own_keys)[1:3].isnan().all()


@pytest.mark.parametrize("dim", [128, 256])
def test_value_scales_that_no_write_leaves(device, dim):
    """2^32 and more count as not finite; 2^31 is a scale like any other."""
    generator = torch.Generator(device=device).manual_seed(27)
    q = torch.randn((3, 8, 4, dim), device=device, generator=generator).to(torch.bfloat16)
    own = make_cache(generator, 3, 1, 20, dim, True, device)
    own.v_codes.view(torch.uint8)[1, 0, 5, ::2] = 0
    want = K.prefix_attention(q, no_keys(own), own)
    for exponent in (31, 32, 70, 127):
        changed = own._replace(v_scales=own.v_scales.clone())
        changed.v_scales[1, 0, 5] = 2.0 ** exponent
        got = K.prefix_attention(q, no_keys(own), changed)
        if exponent < 32:
            check(got, *reference(q, no_keys(own), changed, [0, 3], [0], [20] * 3, False, dim ** -0.5))
        else:
            assert got[1].isnan().all() and torch.equal(got[[0, 2]], want[[0, 2]])


# ---- layouts ----------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dim", [128, 256])
def test_any_stride_along_an_extent_of_one(device, dim):
    """One token per sequence as a view whose token stride is 1, and one sequence whose batch stride is odd."""
    generator = torch.Generator(device=device).manual_seed(28)
    draw = lambda *shape: torch.randn(shape, device=device, generator=generator).to(torch.bfloat16)
    view = lambda x: x.unsqueeze(-1).transpose(2, 3)          # [B, heads, D] -> [B, heads, 1, D]
    k, v, q = draw(3, 2, dim), draw(3, 2, dim), draw(3, 8, dim)
    assert view(k).stride(2) == 1
    got, want = (QuantizedKVCache.allocate(3, 2, 4, dim, device) for _ in range(2))
    got_q, want_q = (torch.empty((3, 8, 1, dim), device=device, dtype=torch.bfloat16) for _ in range(2))
    K.kv_cache_write(view(k), view(v), got, q=view(q), q_out=got_q)
    K.kv_cache_write(k[:, :, None].contiguous(), v[:, :, None].contiguous(), want, q=q[:, :, None].contiguous(), q_out=want_q)
    assert torch.equal(got_q, want_q) and all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, want))
    assert torch.equal(K.prefix_attention(view(q), got), K.prefix_attention(want_q, got))
    outs = [view(torch.empty((3, 2, dim), device=device, dtype=torch.bfloat16)) for _ in range(2)]
    wants = [torch.empty((3, 2, 1, dim), device=device, dtype=torch.bfloat16) for _ in range(2)]
    for a, b in zip(K.kv_cache_read(got, *outs), K.kv_cache_read(got, *wants)):
        assert torch.equal(a, b)
    one = torch.empty(2 * dim, device=device, dtype=torch.bfloat16).as_strided((1, 2, 1, dim), (3, dim, 5, 1))
    K.kv_cache_read(QuantizedKVCache(*(t[:1].contiguous() for t in got)), one, wants[1][:1])
    assert torch.equal(one, wants[0][:1])


def test_no_keys_at_all_and_members_of_no_group(device):
    q = torch.randn((5, 8, 2, 128), device=device).to(torch.bfloat16)
    empty = tuple(torch.empty((2, 1, 0, 128), device=device, dtype=torch.bfloat16) for _ in range(2))
    out = torch.full_like(q, 7.0)
    assert K.prefix_attention(q, empty, members=whole([1, 2, 4], device), out=out) is out
    assert not out[1:4].any() and (out[[0, 4]] == 7.0).all()
    assert not K.prefix_attention(q, tuple(t[:1] for t in empty), out=out).any()


# ---- rotary tables ----------------------------------------------------------------------------------------

PI = Decimal("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899")
# The series, for the fraction r of a turn in [-1/8, 1/8]: r rounded to fp32 2 pi 2^-28; what the series leave out, (pi/4)^11 / 11!; of the
# sine's sum the last step (near 2 pi, times 1/8), its constant and the step before (near 41, times 1/64 and 1/8) 2^-25 + 2^-25 + 2 * 2^-28;
# the product 2^-25.  The cosine's are smaller.
SERIES = 2 * math.pi * 2.0 ** -28 + (math.pi / 4) ** 11 / 39916800 + 3 * 2.0 ** -25 + 2 * 2.0 ** -28


@pytest.mark.parametrize("sections,theta,own_spectrum", [((64,), 500000.0, False), ((6,), 10000.0, True), ((5, 2), 10000.0, True)])
def test_tables_of_far_positions(device, sections, theta, own_spectrum):
    """Against angles reduced in 70 decimal digits.  A frequency f is known to some 2^-53 of itself -- theta's logarithm and its division and
    product 3 log2(theta) 2^-53 ln 2, the exponential 2^-52, the constant and its product 2^-53 each, three steps of 2^-52 (with the ratio's
    own 3 times that) to the last of four columns -- and to 2^-65 turns; the position multiplies both."""
    positions = [0, 1, -1, 262143, 2 ** 31 - 1, -2 ** 31, 2 ** 36 + 12345, -(2 ** 33), (1 << 40) + 3]
    sine, cosine = K.rope_axes(torch.tensor([positions] * len(sections), device=device), sections, theta=theta, own_spectrum=own_spectrum)
    sine, cosine = sine.cpu().double(), cosine.cpu().double()
    relative = (3 * math.log2(theta) * math.log(2) + 2 + 2 + 3 * 2 * 4) * 2.0 ** -53
    column = 0
    for count in sections:
        for j in range(count):
            with localcontext() as context:
                context.prec = 70
                power = Decimal(j) / count if own_spectrum else Decimal(column) / sum(sections)
                frequency = (-power * Decimal(theta).ln()).exp()
                for t, position in enumerate(positions):
                    turns = position * frequency / (2 * PI)
                    angle = float(2 * PI * (turns - turns.to_integral_value()))
                    bound = SERIES + abs(position) * (float(frequency) * relative + 2 * math.pi * 2.0 ** -65)
                    assert abs(float(sine[t, column]) - math.sin(angle)) <= bound, (column, position)
                    assert abs(float(cosine[t, column]) - math.cos(angle)) <= bound, (column, position)
            column += 1
