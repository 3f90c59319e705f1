"""Edges of the cache operators: magnitudes, values that are not finite, layouts and positions at the end of what is allowed."""

from __future__ import annotations

import pytest
import torch

from embodiinfer_b200 import kernels as K
from embodiinfer_b200.kv_cache import QuantizedKVCache
from tests.test_gpu_prefix_attention import check, reference

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
