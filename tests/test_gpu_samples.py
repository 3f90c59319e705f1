"""Several action samples behind one prefix: the cache operators as one path runs them, and the policy that calls them."""

from __future__ import annotations

import pytest
import torch

from embodiinfer_b200 import kernels as K
from embodiinfer_b200.kv_cache import QuantizedKVCache
from embodiinfer_b200.pi05_shaped import ACTION_DIM, ACTION_HORIZON, Pi05ShapedPolicy, synthetic_observations
from tests.test_gpu_prefix_attention import check, reference, whole

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kv_heads,dim,steps", [(8, 1, 256, 3), (8, 2, 128, 70)])
def test_tables_write_attention_and_read_together(device, heads, kv_heads, dim, steps):
    """Prompts of unequal length written into prefix caches, then token after token of every member behind them: tables at each
    member's own positions, the write at its own offset, the attention over everything written so far.  The reference attends in
    64 bits over what the caches hold; what they hold is checked against the write's own tests' definition by reading it back."""
    generator = torch.Generator(device=device).manual_seed(7 + dim)
    bounds, prompt_lengths = [0, 2, 5], [37, 64]
    groups, batch, capacity = 2, 5, max(prompt_lengths)
    sections = (dim // 8, 3 * dim // 16, 3 * dim // 16)
    draw = lambda *shape: torch.randn(shape, device=device, generator=generator).to(torch.bfloat16)
    prefix = QuantizedKVCache.allocate(groups, kv_heads, capacity, dim, device)
    own = QuantizedKVCache.allocate(batch, kv_heads, steps + 2, dim, device)
    width = heads + 2 * kv_heads

    positions = torch.stack([torch.arange(capacity, device=device), *torch.randint(0, 16, (2, capacity), device=device, generator=generator)])
    sine, cosine = K.rope_axes(positions, sections)
    prompt = draw(groups, capacity, width, dim).transpose(1, 2)
    K.kv_cache_write(prompt[:, heads: heads + kv_heads], prompt[:, heads + kv_heads:], prefix, sine=sine, cosine=cosine, lengths=whole(prompt_lengths, device))

    start = torch.tensor([0, 1, 2, 0, 1], device=device, dtype=torch.int32)          # rows that another call has written before
    earlier = draw(batch, 2, width, dim).transpose(1, 2)
    K.kv_cache_write(earlier[:, heads: heads + kv_heads], earlier[:, heads + kv_heads:], own, lengths=start)
    written = []
    for step in range(steps):
        offsets = start + step
        at = offsets.long() + torch.tensor(prompt_lengths, device=device).repeat_interleave(torch.tensor([2, 3], device=device))
        sine, cosine = K.rope_axes(torch.stack([at, at % 5, at % 3]).unsqueeze(-1), sections)          # [batch, 1, dim / 2]
        rows = draw(batch, 1, width, dim).transpose(1, 2)
        q = torch.empty((batch, heads, 1, dim), device=device, dtype=torch.bfloat16)
        K.kv_cache_write(rows[:, heads: heads + kv_heads], rows[:, heads + kv_heads:], own, q=rows[:, :heads], q_out=q, sine=sine, cosine=cosine,
                         offsets=offsets)
        first, second = rows[:, :heads + kv_heads].float().chunk(2, -1)
        s, c = sine[:, None], cosine[:, None]
        rotated = torch.cat((first * c - second * s, second * c + first * s), -1)
        assert torch.equal(q, rotated[:, :heads].to(torch.bfloat16))
        written.append((offsets, rotated[:, heads:], rows[:, heads + kv_heads:].float()))
        if step in (0, 1, steps - 1):
            lengths = (offsets + 1).tolist()
            got = K.prefix_attention(q, prefix, own, members=whole(bounds, device), prefix_lengths=whole(prompt_lengths, device), own_lengths=whole(lengths, device),
                                     causal=True)
            K.check_status(device)
            check(got, *reference(q, prefix, own, bounds, prompt_lengths, lengths, True, dim ** -0.5))
    k, v = (torch.full((batch, kv_heads, steps, dim), 7.0, device=device, dtype=torch.bfloat16) for _ in range(2))
    K.kv_cache_read(own, k, v, offsets=start)
    for step, (_, keys, values) in enumerate(written):
        for got, want in ((k, keys), (v, values)):
            # e4m3 rounds a value to 2^-4 of itself or, below 2^-6 of 448ths of the largest, by 2^-10 of those; bf16 to 2^-8
            largest = want.abs().amax(-1, keepdim=True)
            bound = want.abs() * (2.0 ** -4 + 2.0 ** -8 + 2.0 ** -11) + largest / 448.0 * 2.0 ** -10 * 1.01
            assert ((got[:, :, step: step + 1].float() - want).abs() <= bound).all()


def test_samples_share_the_prefix(device):
    """One layer per tower.  Samples over one prefix per observation against the same denoise with a copy per sample: the attention
    kernels round differently, and ten Euler steps through requantising layers amplify that (2e-2, as between the Linear routes)."""
    policy = Pi05ShapedPolicy("fp8", device=device, layer_scale=0.01, vocabulary=4096)
    observations = synthetic_observations(3, vocabulary=4096)
    for calibrated in (False, True):
        if calibrated:
            policy.calibrate_fused_mlp(observations)
        actions = policy.sample(observations, 4, shared_prefix=True)
        assert actions.shape == (3, 4, ACTION_HORIZON, ACTION_DIM) and torch.isfinite(actions).all()
        assert torch.equal(actions, policy.sample(observations, 4, shared_prefix=True)), "sampling must be deterministic"
        cache, length = policy.encode_prefix(observations["images"], observations["tokens"])
        repeated = [tuple(part.repeat_interleave(4, 0) for part in pair) for pair in cache]
        noise = policy.noise(12)
        with torch.no_grad():
            expected = policy.denoise(repeated, length, noise).view(actions.shape)
        assert torch.equal(policy.sample(observations, 4), expected)          # few chunks: a copy each
        assert float((actions - expected).norm() / expected.norm()) < 2e-2
        # the quantised cache rounds keys and values to 2^-4 of themselves
        quantised = policy.sample(observations, 4, quantised_cache=True)
        error = float((quantised - actions).norm() / actions.norm())
        assert 0.0 < error < 2.0 ** -4
        assert not torch.equal(actions[:, 0], actions[:, 1])
    many = policy.sample(observations, 24)
    assert torch.equal(many, policy.sample(observations, 24, shared_prefix=True)) and not torch.equal(many, policy.sample(observations, 24, shared_prefix=False))
    assert policy.sample(observations, 0).shape == (3, 0, ACTION_HORIZON, ACTION_DIM)
    K.check_status(device)


def test_samples_in_a_graph(device):
    policy = Pi05ShapedPolicy("fp8", device=device, layer_scale=0.01, vocabulary=4096)
    observations = synthetic_observations(2, vocabulary=4096)
    policy.calibrate_fused_mlp(observations)
    with torch.no_grad():
        cache, length = policy.encode_prefix(observations["images"], observations["tokens"])
        noise = policy.noise(6).view(2, 3, ACTION_HORIZON, ACTION_DIM)
        for options in (dict(), dict(shared_prefix=True), dict(quantised_cache=True)):
            run = lambda: policy.denoise_samples(cache, length, noise, **options)
            eager = run()
            stream = torch.cuda.Stream()
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                run()
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                captured = run()
            for _ in range(2):
                captured.zero_()
                graph.replay()
                torch.cuda.synchronize()
                assert torch.equal(captured, eager)
    K.check_status(device)
