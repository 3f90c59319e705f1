"""Samples of an observation over copies of its prefix: the copies' memory, and when a call makes them."""

from __future__ import annotations

import pytest
import torch

from embodiinfer_b200.pi05_shaped import ACTION_DIM, ACTION_HORIZON, GEMMA_300M, Pi05ShapedPolicy

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def policy(device):
    return Pi05ShapedPolicy("fp8", device=device, layer_scale=0.01, vocabulary=4096)


def random_call(policy, observations, samples, prefix, seed):
    """(cache, prefix length, noise)"""
    generator = torch.Generator(device=policy.device_).manual_seed(seed)
    draw = lambda *shape: torch.randn(shape, device=policy.device_, generator=generator)
    cache = [tuple(draw(observations, GEMMA_300M.kv_heads, prefix, GEMMA_300M.head_dim).to(torch.bfloat16) for _ in range(2)) for _ in policy.expert]
    return cache, prefix, draw(observations, samples, ACTION_HORIZON, ACTION_DIM)


@torch.no_grad()
def test_one_copy_of_the_prefix_per_sample(policy):
    """A call's peak is its buffers [prefix | own] and what 240 rows of activations need (below 64 MB), not another copy;
    and it gives what copies made by the caller give."""
    cache, length, noise = random_call(policy, 2, 12, 6000, 1)
    run = lambda: policy.denoise_samples(cache, length, noise, shared_prefix=False)
    run()
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = run()
    torch.cuda.synchronize()
    buffers = sum(24 * part.shape[1] * (length + ACTION_HORIZON) * part.shape[3] * 2 for pair in cache[: len(policy.expert)] for part in pair)
    assert buffers > 128 << 20 and torch.cuda.max_memory_allocated() - before < buffers + (64 << 20)
    repeated = [tuple(part.repeat_interleave(12, 0) for part in pair) for pair in cache]
    assert torch.equal(got, policy.denoise(repeated, length, noise.flatten(0, 1)).view(noise.shape))


@torch.no_grad()
@pytest.mark.parametrize("observations,samples,prefix,shared", [(3, 16, 560, True), (3, 14, 560, False), (9, 8, 136, False), (1, 4, 6200, True)])
def test_the_default_goes_by_the_rows_that_copies_would_hold(policy, observations, samples, prefix, shared):
    cache, length, noise = random_call(policy, observations, samples, prefix, 2)
    got = policy.denoise_samples(cache, length, noise)
    assert torch.equal(got, policy.denoise_samples(cache, length, noise, shared_prefix=shared))
    assert not torch.equal(got, policy.denoise_samples(cache, length, noise, shared_prefix=not shared))
