"""Rotary tables with several axes and the quantised cache's write and read against plain torch."""

from __future__ import annotations

import math

import pytest
import torch

from embodiinfer_b200 import kernels as K
from embodiinfer_b200.kv_cache import QuantizedKVCache

pytestmark = pytest.mark.gpu

TINY, HUGE = 2.0 ** -50, 2.0 ** 40


# ---- rotary tables -------------------------------------------------------------------------------------

# The fraction of a turn is rounded to fp32 (half a step of values below 1: 2^-25, as an angle pi 2^-25 = 9.4e-8), sincospif is
# documented to 2 steps of its result (at most 2 * 2^-24 = 1.2e-7), and 64-bit angles of positions below 2^20 move by less than 1e-9.
TABLE_TOLERANCE = math.pi * 2.0 ** -25 + 2.0 * 2.0 ** -24 + 1e-9


def expected_tables(positions, sections, theta, own_spectrum):
    half, start, angles = sum(sections), 0, []
    for axis, count in enumerate(sections):
        for j in range(count):
            power = j / count if own_spectrum else (start + j) / half
            angles.append(positions[axis].double() * theta ** -power)
        start += count
    angle = torch.stack(angles, -1)
    return angle.sin(), angle.cos()


@pytest.mark.parametrize("sections,shape,own_spectrum,dtype", [
    ((128,), (560,), False, torch.int64), ((16, 24, 24), (3, 77), False, torch.int64), ((16, 24, 24), (2, 33), True, torch.int32),
    ((32, 48, 48), (1, 1), False, torch.int32), ((3, 5, 2, 1), (19,), True, torch.int64), ((18, 18), (256,), True, torch.int64),
    ((300, 212), (5,), False, torch.int64), ((1,), (4,), False, torch.int32), ((5, 300), (7,), False, torch.int64), ((64,), (20011,), False, torch.int64)])
def test_rope_axes(device, sections, shape, own_spectrum, dtype):
    generator = torch.Generator(device=device).manual_seed(sum(sections))
    positions = torch.randint(-70, 1 << 20, (len(sections), *shape), device=device, generator=generator).to(dtype)
    sine, cosine = K.rope_axes(positions, sections, theta=10000.0, own_spectrum=own_spectrum)
    assert sine.shape == cosine.shape == (*shape, sum(sections)) and sine.dtype == torch.float32
    for got, want in zip((sine, cosine), expected_tables(positions, sections, 10000.0, own_spectrum)):
        assert (got.double() - want).abs().max() <= TABLE_TOLERANCE


def test_rope_axes_into_given_tables_and_far_positions(device):
    positions = torch.tensor([[0, 1, (1 << 40) + 3, -(1 << 33)]], device=device)
    storage = torch.full((2, 4 * 6 + 1), 7.0, device=device)
    sine, cosine = (storage[i, 1:].view(4, 6) for i in range(2))          # 4 bytes behind a 16-byte boundary
    K.rope_axes(positions, (6,), sine, cosine, theta=500000.0)
    want = expected_tables(positions[:, :2], (6,), 500000.0, False)
    assert (sine[:2].double() - want[0]).abs().max() <= TABLE_TOLERANCE and (cosine[:2].double() - want[1]).abs().max() <= TABLE_TOLERANCE
    assert (sine.double() ** 2 + cosine.double() ** 2 - 1).abs().max() < 1e-6 and (storage[:, 0] == 7.0).all()
    assert K.rope_axes(positions[:, :0].contiguous(), (6,))[0].shape == (0, 6)


def test_rope_axes_refuses(device):
    positions = torch.zeros((2, 8), device=device, dtype=torch.int64)
    for bad in (lambda: K.rope_axes(positions.float(), (4, 4)), lambda: K.rope_axes(positions, (8,)), lambda: K.rope_axes(positions, (8, 0)),
                lambda: K.rope_axes(positions.t(), (4,) * 8), lambda: K.rope_axes(positions, (4, 4), torch.empty((8, 8), device=device)),
                lambda: K.rope_axes(positions, (4, 4), *(torch.empty((8, 7), device=device) for _ in range(2)))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="error -1"):
        K.rope_axes(positions, (4, 4), theta=0.0)


# ---- the cache's write -----------------------------------------------------------------------------------


def rotate(x, sine, cosine):
    """x [B, heads, T, D] fp32; factors [T, D/2] or [B, T, D/2]"""
    if sine.ndim == 3:
        sine, cosine = sine[:, None], cosine[:, None]
    first, second = x.chunk(2, dim=-1)
    return torch.cat((first * cosine - second * sine, second * cosine + first * sine), dim=-1)


def quantise(x):
    """The format's definition in fp32 torch operations: (code bytes, scales)."""
    largest = x.abs().amax(-1)
    quotient = largest / torch.full_like(largest, 448.0)          # by a Python number torch multiplies with the rounded reciprocal on CUDA
    scale = torch.where(largest < TINY, 0.0, torch.where(largest < HUGE, quotient, math.nan))
    codes = torch.where(scale[..., None] == 0, 0.0, (x / scale[..., None]).clamp(-448.0, 448.0)).to(torch.float8_e4m3fn)
    return codes.view(torch.uint8), scale


def filled_cache(batch, kv_heads, capacity, head_dim, device):
    cache = QuantizedKVCache.allocate(batch, kv_heads, capacity, head_dim, device)
    for part in cache:
        part.view(torch.uint8).fill_(0x35) if part.element_size() == 1 else part.fill_(0.25)
    return cache


def expected_cache(cache, k, v, offsets, lengths):
    parts = [part.view(torch.uint8).clone() if part.element_size() == 1 else part.clone() for part in cache]
    for which, rows in enumerate((k, v)):
        codes, scales = quantise(rows)
        for b in range(rows.shape[0]):
            for t in range(min(rows.shape[2], lengths[b])):
                position = offsets[b] + t
                if 0 <= position < cache.k_codes.shape[2]:
                    parts[2 * which][b, :, position], parts[2 * which + 1][b, :, position] = codes[b, :, t], scales[b, :, t]
    return parts


def assert_same_cache(cache, expected):
    for got, want in zip(cache, expected):
        got = got.view(torch.uint8) if got.element_size() == 1 else got
        if got.dtype == torch.uint8:
            nan = (want & 0x7f) == 0x7f
            assert torch.equal((got & 0x7f) == 0x7f, nan) and torch.equal(got[~nan], want[~nan])
        else:
            assert torch.equal(got.nan_to_num(-1.0), want.nan_to_num(-1.0))


def packed_rows(generator, batch, tokens, heads, kv_heads, head_dim, device, extra=0):
    """Views [B, heads, T, D] of q, k and v of one packed projection whose rows may be longer than what is used."""
    width = (heads + 2 * kv_heads) * head_dim
    rows = torch.randn((batch, tokens, width + extra), device=device, generator=generator) * torch.exp(torch.randn((batch, tokens, 1), device=device, generator=generator))
    rows = rows.to(torch.bfloat16)[:, :, :width].unflatten(-1, (heads + 2 * kv_heads, head_dim)).transpose(1, 2)
    return rows[:, :heads], rows[:, heads: heads + kv_heads], rows[:, heads + kv_heads:]


@pytest.mark.parametrize("batch,tokens,heads,kv_heads,head_dim,per_batch,extra", [
    (1, 1, 8, 1, 256, False, 0), (3, 10, 8, 1, 256, True, 0), (2, 7, 4, 2, 128, False, 64), (5, 3, 28, 4, 128, True, 0), (1, 33, 1, 1, 128, False, 8),
    (2, 301, 8, 1, 256, False, 0), (4, 257, 32, 8, 128, True, 0)])          # the last two: several rows per thread
def test_write_is_bit_exact(device, batch, tokens, heads, kv_heads, head_dim, per_batch, extra):
    generator = torch.Generator(device=device).manual_seed(tokens)
    q, k, v = packed_rows(generator, batch, tokens, heads, kv_heads, head_dim, device, extra)
    angle = 6.0 * torch.rand((batch, tokens, head_dim // 2) if per_batch else (tokens, head_dim // 2), device=device, generator=generator)
    sine, cosine = angle.sin(), angle.cos()
    offsets = [(3 * b) % 5 for b in range(batch)]
    lengths = [max(0, tokens - 2 * b) for b in range(batch)]
    cache = filled_cache(batch, kv_heads, tokens + 3, head_dim, device)          # the larger offsets leave the cache
    turned_k = rotate(k.float(), sine, cosine)
    expected = expected_cache(cache, turned_k, v.float(), offsets, lengths)
    q_out = torch.full((batch, heads, tokens, head_dim), 5.0, device=device, dtype=torch.bfloat16)
    q_expected = rotate(q.float(), sine, cosine).to(torch.bfloat16)
    for b in range(batch):
        q_expected[b, :, lengths[b]:] = 5.0
    whole = lambda values: torch.tensor(values, device=device, dtype=torch.int32)
    K.kv_cache_write(k, v, cache, q=q, q_out=q_out, sine=sine, cosine=cosine, offsets=whole(offsets), lengths=whole(lengths))
    assert torch.equal(q_out, q_expected)
    assert_same_cache(cache, expected)


def test_write_defaults_and_no_rotation(device):
    generator = torch.Generator(device=device).manual_seed(2)
    k, v = (torch.randn((3, 2, 9, 256), device=device, generator=generator).to(torch.bfloat16) for _ in range(2))
    cache = filled_cache(3, 2, 12, 256, device)
    expected = expected_cache(cache, k.float(), v.float(), [0] * 3, [9] * 3)
    K.kv_cache_write(k, v, cache)
    assert_same_cache(cache, expected)
    K.kv_cache_write(k[:, :, :0], v[:, :, :0], cache)          # nothing to write
    assert_same_cache(cache, expected)


def test_write_passes_over_positions_outside_the_cache(device):
    rows = torch.ones((4, 1, 3, 128), device=device, dtype=torch.bfloat16)
    cache = filled_cache(4, 1, 4, 128, device)
    offsets, lengths = [-2, 3, 2 ** 31 - 1, -2 ** 31], [3, 3, 3, 2 ** 31 - 1]
    expected = expected_cache(cache, rows.float(), rows.float(), offsets, lengths)
    whole = lambda values: torch.tensor(values, device=device, dtype=torch.int32)
    K.kv_cache_write(rows, rows, cache, offsets=whole(offsets), lengths=whole(lengths))
    assert_same_cache(cache, expected)
    K.kv_cache_write(rows, rows, cache, lengths=whole([0, -5, 0, 0]))
    assert_same_cache(cache, expected)


@pytest.mark.parametrize("head_dim", [128, 256])
def test_write_of_unusual_rows(device, head_dim):
    rows = torch.randn((1, 1, 9, head_dim), device=device, generator=torch.Generator(device=device).manual_seed(1))
    rows[0, 0, 0] = 0.0
    rows[0, 0, 1, 3] = math.inf
    rows[0, 0, 2, head_dim - 1] = math.nan
    rows[0, 0, 3] *= 2.0 ** -100
    rows[0, 0, 4] = 0.0
    rows[0, 0, 4, 5] = TINY
    rows[0, 0, 5] *= 2.0 ** 36
    rows[0, 0, 6] *= 2.0 ** -45
    rows[0, 0, 7, 0] = -0.0
    rows[0, 0, 8] = 0.0
    rows[0, 0, 8, 7] = HUGE
    rows = rows.to(torch.bfloat16)
    cache = filled_cache(1, 1, 9, head_dim, device)
    expected = expected_cache(cache, rows.float(), rows.float(), [0], [9])
    K.kv_cache_write(rows, rows, cache)
    assert_same_cache(cache, expected)
    k, v = (torch.empty_like(rows) for _ in range(2))
    K.kv_cache_read(cache, k, v)
    finite = [0, 3, 4, 5, 6, 7]
    assert k[0, 0, [1, 2, 8]].isnan().all() and not k[0, 0, finite].isnan().any() and not k[0, 0, 0].any() and not k[0, 0, 3].any()
    # half a step of e4m3, 2^-4 of a value, or of its smallest normal numbers; then the bf16 result
    source, got = rows[0, 0, finite].float(), k[0, 0, finite].float()
    largest = source.abs().amax(-1, keepdim=True)
    bound = torch.maximum(source.abs() * 2.0 ** -4, largest / 448.0 * 2.0 ** -10) * (1 + 2.0 ** -6) + largest * 2.0 ** -8
    bound[1] = TINY
    assert ((got - source).abs() <= bound).all()


# ---- the cache's read ------------------------------------------------------------------------------------


@pytest.mark.parametrize("batch,kv_heads,capacity,tokens,head_dim", [(1, 1, 1, 1, 256), (3, 2, 40, 17, 128), (2, 1, 712, 712, 256), (4, 8, 700, 650, 128)])
def test_read(device, batch, kv_heads, capacity, tokens, head_dim):
    generator = torch.Generator(device=device).manual_seed(capacity)
    codes = [torch.randint(0, 256, (batch, kv_heads, capacity, head_dim), device=device, dtype=torch.uint8, generator=generator) for _ in range(2)]
    scales = [torch.rand((batch, kv_heads, capacity), device=device, generator=generator) for _ in range(2)]
    cache = QuantizedKVCache(codes[0], scales[0], codes[1].view(torch.float8_e4m3fn), scales[1])
    offsets, lengths = [(5 * b) % 7 - 1 for b in range(batch)], [max(1, tokens - 3 * b) for b in range(batch)]
    whole = lambda values: torch.tensor(values, device=device, dtype=torch.int32)
    # outputs as the projection's layout has them: token before head
    k, v = (torch.full((batch, tokens, kv_heads, head_dim), 3.0, device=device, dtype=torch.bfloat16).transpose(1, 2) for _ in range(2))
    expected = []
    for code, scale in zip(codes, scales):
        values = (code.view(torch.float8_e4m3fn).float() * scale[..., None]).to(torch.bfloat16)
        want = torch.full((batch, kv_heads, tokens, head_dim), 3.0, device=device, dtype=torch.bfloat16)
        for b in range(batch):
            for t in range(lengths[b]):
                if 0 <= offsets[b] + t < capacity:
                    want[b, :, t] = values[b, :, offsets[b] + t]
        expected.append(want)
    K.kv_cache_read(cache, k, v, offsets=whole(offsets), lengths=whole(lengths))
    for got, want in zip((k, v), expected):
        assert torch.equal(got.nan_to_num(99.0), want.nan_to_num(99.0))


def test_cache_operators_refuse(device):
    cache = QuantizedKVCache.allocate(2, 1, 8, 128, device)
    rows = torch.zeros((2, 1, 4, 128), device=device, dtype=torch.bfloat16)
    factors = torch.zeros((4, 64), device=device)
    for bad in (lambda: K.kv_cache_write(rows.float(), rows.float(), cache), lambda: K.kv_cache_write(rows, rows[:, :, :3], cache),
                lambda: K.kv_cache_write(rows[:1], rows[:1], cache), lambda: K.kv_cache_write(rows, rows, cache, q=rows),
                lambda: K.kv_cache_write(rows, rows, cache, sine=factors), lambda: K.kv_cache_write(rows, rows, cache, sine=factors[:3], cosine=factors[:3]),
                lambda: K.kv_cache_write(rows, rows, cache, offsets=torch.zeros(2, device=device, dtype=torch.int64)),
                lambda: K.kv_cache_write(rows, rows, cache, lengths=torch.zeros(3, device=device, dtype=torch.int32)),
                lambda: K.kv_cache_write(rows, rows, cache._replace(k_scales=cache.k_scales.half())),
                lambda: K.kv_cache_write(rows, rows, cache._replace(v_codes=cache.v_codes[:, :, :4])),
                lambda: K.kv_cache_read(cache, rows, rows[..., :64]), lambda: K.kv_cache_read(cache, rows.cpu(), rows)):
        with pytest.raises(ValueError):
            bad()
    shifted = torch.zeros(2 * 4 * 128 + 4, device=device, dtype=torch.bfloat16)[4:].view(2, 1, 4, 128)
    with pytest.raises(RuntimeError, match="error -1"):
        K.kv_cache_write(shifted, rows, cache)
    small = QuantizedKVCache.allocate(2, 1, 8, 64, device)
    with pytest.raises(RuntimeError, match="error -2"):
        K.kv_cache_write(rows[..., :64], rows[..., :64], small)


def test_codes_behind_four_gigabytes(device):
    """The last sequence's codes start beyond 2^32 bytes."""
    batch, capacity = 3, 9_000_000
    if torch.cuda.mem_get_info(device)[0] < 30 << 30:
        pytest.skip("needs 30 GB of device memory")
    empty = lambda: torch.empty((batch, 1, capacity, 256), device=device, dtype=torch.uint8)
    scales = lambda: torch.empty((batch, 1, capacity), device=device)
    cache = QuantizedKVCache(empty(), scales(), empty(), scales())
    rows = torch.randn((batch, 1, 5, 256), device=device, generator=torch.Generator(device=device).manual_seed(4)).to(torch.bfloat16)
    offsets = torch.full((batch,), capacity - 5, device=device, dtype=torch.int32)
    K.kv_cache_write(rows, rows, cache, offsets=offsets)
    codes, scale = quantise(rows.float())
    assert torch.equal(cache.k_codes[:, :, -5:], codes) and torch.equal(cache.v_scales[:, :, -5:], scale)
    out = torch.empty_like(rows)
    K.kv_cache_read(cache, out, torch.empty_like(rows), offsets=offsets)
    assert torch.equal(out, (codes.view(torch.float8_e4m3fn).float() * scale[..., None]).to(torch.bfloat16))
