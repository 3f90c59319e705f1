"""Edges of the cache operators' checks, at the C ABI and in the wrappers.  No kernel is launched here."""

from __future__ import annotations

import ctypes
from types import SimpleNamespace

import pytest
import torch

from embodiinfer_b200 import _native as N
from embodiinfer_b200.pi05_shaped import ACTION_DIM, ACTION_HORIZON, Pi05ShapedPolicy
from tests.test_kv_cache import FAKE, _cache_desc

MOST = (1 << 31) - 1


@pytest.mark.parametrize("changes", [dict(batch=1, tokens=MOST, k_stride=(3, 128, 128), v_stride=(1 << 50, 128, 128)),
                                     dict(batch=1 << 20, tokens=1 << 11, k_stride=(768, 5, 128)), dict(batch=MOST, tokens=1, v_stride=(256, 128, 1))])
def test_strides_count_only_where_there_are_steps(changes):
    """A stride along an extent of 1 is not looked at: these calls are refused for their size alone, which is looked at behind the strides.
    Along an extent of 2 the same strides are refused."""
    grown = {**changes, **{name: max(2, changes.get(name, 0)) for name in ("batch", "tokens")}, "kv_heads": 2}
    for call in (N.load().b2_kv_cache_write, N.load().b2_kv_cache_read):
        assert call(ctypes.byref(_cache_desc(**changes)), None) == N.E_TOO_LARGE
        assert call(ctypes.byref(_cache_desc(**grown)), None) == N.E_INVALID


@pytest.mark.parametrize("k_stride,v_stride,extents", [
    ((128, 128, 128), (768, 384, 128), (2, 2, 3)), ((768, 384, 128), (256, 384, 128), (2, 2, 3)),          # steps that fall on other rows
    ((768, 128, 128), (768, 384, 128), (2, 2, 3)), ((0, 0, 0), (0, 0, 0), (2, 1, 1)), ((384, 256, 128), (384, 256, 128), (1, 2, 3))])
def test_read_refuses_rows_on_one_another(k_stride, v_stride, extents):
    batch, kv_heads, tokens = extents
    fields = dict(batch=batch, kv_heads=kv_heads, tokens=tokens, v=2 * FAKE)
    assert N.load().b2_kv_cache_read(ctypes.byref(_cache_desc(k_stride=k_stride, v_stride=v_stride, **fields)), None) == N.E_INVALID


def test_read_refuses_one_tensor_for_both():
    assert N.load().b2_kv_cache_read(ctypes.byref(_cache_desc(k_stride=(384, 384, 128), v_stride=(384, 384, 128), v=FAKE)), None) == N.E_INVALID


@pytest.mark.parametrize("options", [dict(), dict(shared_prefix=True), dict(quantised_cache=True)])
def test_samples_refuse_noise_of_other_observations(options):
    """Noise for four observations behind the cache of two would hand every prefix to other observations' samples."""
    policy = SimpleNamespace(expert=[None], device_=torch.device("cpu"))          # refused before anything of it is used
    cache = [tuple(torch.zeros((2, 1, 12, 256), dtype=torch.bfloat16) for _ in range(2))]
    for shape in ((4, 3, ACTION_HORIZON, ACTION_DIM), (1, 3, ACTION_HORIZON, ACTION_DIM), (2, 3, ACTION_DIM, ACTION_HORIZON)):
        with pytest.raises(ValueError, match="noise"):
            Pi05ShapedPolicy.denoise_samples(policy, cache, 12, torch.zeros(shape), **options)
    observations = dict(images=torch.zeros((2, 1)), tokens=torch.zeros((2, 1)))
    with pytest.raises(ValueError, match="noise"):
        Pi05ShapedPolicy.sample(policy, observations, 3, torch.zeros((2, 4, ACTION_HORIZON, ACTION_DIM)), **options)
