"""Refusals of the cache operators at the C ABI and in the Python wrappers.  No kernel is launched here."""

from __future__ import annotations

import ctypes
import re
from pathlib import Path

import pytest
import torch

from embodiinfer_b200 import _native as N
from embodiinfer_b200 import kernels as K
from embodiinfer_b200.kv_cache import QuantizedKVCache

HEADER = Path(__file__).resolve().parent.parent / "include" / "embodiinfer_b200.h"
FAKE = 4096      # aligned, never dereferenced: the checks come before any launch


@pytest.mark.parametrize("name,mirror", [("b2_kv_cache_desc", N.KVCacheDesc), ("b2_prefix_attention_desc", N.PrefixAttentionDesc)])
def test_descriptor_layouts_match_the_header(name, mirror):
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), HEADER.read_text(), flags=re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    fields = [field for line in re.findall(r"(?:const\s+)?(?:int32_t|int64_t|float|void\*)\s+([^;]+);", body) for field in line.split(",")]
    assert [field.strip().removesuffix("[3]") for field in fields] == [field for field, _ in mirror._fields_]


def test_constants_match_the_header():
    text = HEADER.read_text()
    assert int(re.search(r"#define B2_ROPE_OWN_SPECTRUM (\d+)", text).group(1)) == N.ROPE_OWN_SPECTRUM
    assert int(re.search(r"#define B2_ATTENTION_CAUSAL (\d+)", text).group(1)) == N.ATTENTION_CAUSAL


def _cache_desc(**changes):
    fields = dict(k=FAKE, v=FAKE, k_codes=FAKE, k_scales=FAKE, v_codes=FAKE, v_scales=FAKE, k_stride=(128, 128, 128), v_stride=(128, 128, 128),
                  batch=2, tokens=3, kv_heads=1, head_dim=128, capacity=8)
    return N.KVCacheDesc(**{**fields, **changes})


@pytest.mark.parametrize("changes,code", [
    (dict(k=None), N.E_INVALID), (dict(v_scales=None), N.E_INVALID), (dict(batch=0), N.E_INVALID), (dict(tokens=0), N.E_INVALID),
    (dict(capacity=0), N.E_INVALID), (dict(kv_heads=-1), N.E_INVALID), (dict(head_dim=64), N.E_UNSUPPORTED), (dict(head_dim=192), N.E_UNSUPPORTED),
    (dict(k=FAKE + 8), N.E_INVALID), (dict(k_codes=FAKE + 8), N.E_INVALID), (dict(k_scales=FAKE + 2), N.E_INVALID),
    (dict(offsets=FAKE + 1), N.E_INVALID), (dict(k_stride=(128, 128, 4)), N.E_INVALID), (dict(v_stride=(128, -128, 128)), N.E_INVALID),
    (dict(batch=1 << 20, tokens=1 << 11), N.E_TOO_LARGE), (dict(kv_heads=(1 << 31) - 1), N.E_TOO_LARGE)])
def test_cache_write_and_read_refuse(changes, code):
    library = N.load()
    assert library.b2_kv_cache_write(ctypes.byref(_cache_desc(**changes)), None) == code
    assert library.b2_kv_cache_read(ctypes.byref(_cache_desc(**changes)), None) == code


def test_cache_write_refuses_half_given_operands():
    library = N.load()
    assert library.b2_kv_cache_write(None, None) == N.E_INVALID
    for changes in (dict(q=FAKE, heads=8), dict(q_out=FAKE, heads=8), dict(sine=FAKE), dict(cosine=FAKE), dict(q=FAKE, q_out=FAKE, heads=0),
                    dict(q=FAKE, q_out=FAKE, heads=8, q_stride=(8, 8, 1)), dict(sine=FAKE, cosine=FAKE, factor_batch_stride=2),
                    dict(sine=FAKE, cosine=FAKE + 4)):
        assert library.b2_kv_cache_write(ctypes.byref(_cache_desc(**changes)), None) == N.E_INVALID, changes
    for changes in (dict(q=FAKE, q_out=FAKE, heads=8), dict(sine=FAKE, cosine=FAKE), dict(batch=2, k_stride=(0, 2048, 256)),
                    dict(tokens=2, v_stride=(4096, 2048, 64))):          # rows written over one another
        assert library.b2_kv_cache_read(ctypes.byref(_cache_desc(**changes)), None) == N.E_INVALID, changes


def _attention_desc(**changes):
    fields = dict(q=FAKE, out=FAKE, prefix_k=FAKE, prefix_v=FAKE, own_k=FAKE, own_v=FAKE, q_stride=(2048, 256, 256), scale=0.0625, batch=4, groups=2,
                  heads=8, kv_heads=1, queries=10, head_dim=256, prefix_capacity=560, own_capacity=10, cache_bits=16)
    return N.PrefixAttentionDesc(**{**fields, **changes})


@pytest.mark.parametrize("changes,code", [
    (dict(q=None), N.E_INVALID), (dict(out=None), N.E_INVALID), (dict(prefix_k=None), N.E_INVALID), (dict(own_v=None), N.E_INVALID),
    (dict(batch=0), N.E_INVALID), (dict(groups=0), N.E_INVALID), (dict(queries=0), N.E_INVALID), (dict(kv_heads=3), N.E_INVALID),
    (dict(groups=3), N.E_INVALID), (dict(prefix_capacity=0, own_capacity=0), N.E_INVALID), (dict(own_capacity=-1), N.E_INVALID),
    (dict(flags=2), N.E_INVALID), (dict(scale=0.0), N.E_INVALID), (dict(scale=float("nan")), N.E_INVALID), (dict(scale=float("inf")), N.E_INVALID),
    (dict(head_dim=64), N.E_UNSUPPORTED), (dict(cache_bits=4), N.E_UNSUPPORTED), (dict(cache_bits=8), N.E_INVALID),
    (dict(q=FAKE + 8), N.E_INVALID), (dict(prefix_v=FAKE + 4), N.E_INVALID), (dict(members=FAKE + 2), N.E_INVALID),
    (dict(workspace=FAKE + 16), N.E_INVALID), (dict(q_stride=(2048, 256, 4)), N.E_INVALID),
    (dict(prefix_capacity=(1 << 30)), N.E_TOO_LARGE), (dict(own_capacity=(1 << 29)), N.E_TOO_LARGE), (dict(queries=1 << 26), N.E_TOO_LARGE)])
def test_prefix_attention_refuses(changes, code):
    assert N.load().b2_prefix_attention(ctypes.byref(_attention_desc(**changes)), None) == code


def test_prefix_attention_workspace():
    size = N.load().b2_prefix_attention_workspace_bytes
    assert size(None) == 0 and size(ctypes.byref(_attention_desc(head_dim=64))) == 0
    few = size(ctypes.byref(_attention_desc(prefix_capacity=32768)))            # two groups of 2 x 80 rows, four row tiles; 512 key tiles
    part = 128 * (256 * 4 + 2 * 4 + 4)                                          # of one CTA: fp32 rows, their statistics, half of the row offsets
    assert few >= 32 + 8 * part and (few - 32) % part == 0
    assert size(ctypes.byref(_attention_desc(batch=4096, groups=2))) == 0       # row tiles for many waves: nothing to cut


@pytest.mark.parametrize("arguments,code", [
    ((None, 8, (4, 4), 2, 10, 16, 1e4, 0, FAKE, FAKE), N.E_INVALID), ((FAKE, 2, (4, 4), 2, 10, 16, 1e4, 0, FAKE, FAKE), N.E_INVALID),
    ((FAKE, 8, (4, 4), 2, 0, 16, 1e4, 0, FAKE, FAKE), N.E_INVALID), ((FAKE, 8, (4, 3), 2, 10, 16, 1e4, 0, FAKE, FAKE), N.E_INVALID),
    ((FAKE, 8, (8, 0), 2, 10, 16, 1e4, 0, FAKE, FAKE), N.E_INVALID), ((FAKE, 8, (4, 4), 2, 10, 16, -1.0, 0, FAKE, FAKE), N.E_INVALID),
    ((FAKE, 8, (4, 4), 2, 10, 16, float("nan"), 0, FAKE, FAKE), N.E_INVALID), ((FAKE, 8, (4, 4), 2, 10, 16, 1e4, 2, FAKE, FAKE), N.E_INVALID),
    ((FAKE + 4, 8, (4, 4), 2, 10, 16, 1e4, 0, FAKE, FAKE), N.E_INVALID), ((FAKE, 8, (4, 4), 2, 10, 16, 1e4, 0, FAKE + 2, FAKE), N.E_INVALID),
    ((FAKE, 8, (4, 4), 5, 10, 16, 1e4, 0, FAKE, FAKE), N.E_UNSUPPORTED), ((FAKE, 8, (4, 4), 2, 10, 17, 1e4, 0, FAKE, FAKE), N.E_UNSUPPORTED),
    ((FAKE, 8, (1024, 4), 2, 10, 2056, 1e4, 0, FAKE, FAKE), N.E_UNSUPPORTED)])
def test_rope_axes_refuses(arguments, code):
    positions, width, sections, *rest = arguments
    assert N.load().b2_rope_axes(positions, width, (ctypes.c_int32 * 8)(*sections), *rest, None) == code


def test_wrappers_refuse_cpu_tensors():
    cache = QuantizedKVCache.allocate(2, 1, 16, 128, "cpu")
    rows = torch.zeros((2, 1, 4, 128), dtype=torch.bfloat16)
    for call in (lambda: K.kv_cache_write(rows, rows, cache), lambda: K.kv_cache_read(cache, rows, rows.clone()),
                 lambda: K.prefix_attention(rows, cache), lambda: K.rope_axes(torch.zeros((3, 4), dtype=torch.int64), (32, 16, 16))):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_allocated_cache_is_empty():
    cache = QuantizedKVCache.allocate(2, 3, 5, 256, "cpu")
    assert cache.k_codes.shape == cache.v_codes.shape == (2, 3, 5, 256) and cache.k_scales.shape == (2, 3, 5)
    assert cache.k_codes.dtype == torch.float8_e4m3fn and not cache.k_codes.view(torch.uint8).any() and not cache.v_scales.any()
