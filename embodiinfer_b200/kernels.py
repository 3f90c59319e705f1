"""Tensor-level wrappers over the C ABI: raw pointers, the caller's current stream, no allocation.

These are the calls the plan objects (``embodiinfer_b200.backend``) and the registry kernels
(``embodiinfer_b200.layers.linear``) are built from.  Every function launches on
``torch.cuda.current_stream(device)`` like the reference's ctypes wrappers
(embodiinfer/backend/cuda/quantization.py:139-166) and raises ``RuntimeError`` on a non-zero status.
"""

from __future__ import annotations

import ctypes
import struct

import torch

from . import _native as N
from .kv_cache import QuantizedKVCache


def _stream(device: torch.device) -> int:
    # the handle alone: building the Stream object around it takes some 2 us
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device() if device.index is None else device.index)


def _ptr(tensor: torch.Tensor | None) -> int | None:
    return None if tensor is None else tensor.data_ptr()


def _require_cuda(*tensors: torch.Tensor | None) -> torch.device:
    indices = {tensor.get_device() for tensor in tensors if tensor is not None}          # -1: not on a GPU
    if len(indices) != 1 or -1 in indices:
        if -1 in indices:
            raise ValueError("embodiinfer_b200 kernels require CUDA tensors; there is no CPU fallback")
        raise ValueError("all operands must live on one CUDA device" if indices else "no tensor operands")
    for tensor in tensors:
        if tensor is not None:
            return tensor.device


def _launch(function, device: torch.device, *arguments) -> int:
    """``function(*arguments, stream)`` with ``device`` current; its context is entered only where it is not (that costs more than
    the launch)."""
    if device.index == torch.cuda.current_device():
        return function(*arguments, torch._C._cuda_getCurrentRawStream(device.index))
    with torch.cuda.device(device):
        return function(*arguments, _stream(device))


def gelu_table_range(table: torch.Tensor) -> tuple[int, int]:
    """Magnitude-code range of a GELU table that the fused epilogue must keep in shared memory
    (``b2_gelu_table_range``); ``(0, 0)`` when the table has no closed-form tails.  Copies the table
    to the host: call it once per table, outside graph capture."""
    host = table.detach().to("cpu").contiguous().view(torch.uint16)
    if host.numel() != 65536:
        raise ValueError("a GELU table has 65536 entries")
    lo, hi = ctypes.c_int32(0), ctypes.c_int32(0)
    status = N.load().b2_gelu_table_range(host.data_ptr(), ctypes.byref(lo), ctypes.byref(hi))
    if status == N.E_UNSUPPORTED:
        return (0, 0)
    N.check(status, "b2_gelu_table_range")
    return (lo.value, hi.value)


def new_scale_scratch(device: torch.device) -> torch.Tensor:
    """Zeroed scratch for :func:`tensor_scale`; allocate once per plan, outside graph capture."""
    return torch.zeros(N.SCALE_SCRATCH_BYTES // 4, device=device, dtype=torch.int32)


def tensor_scale(x: torch.Tensor, bound: float, flags: int, scratch: torch.Tensor, scale: torch.Tensor) -> None:
    """``scale <- amax(|x|) / bound`` (device fp32), see ``b2_tensor_scale``."""
    device = _require_cuda(x, scratch, scale)
    if x.dtype != torch.bfloat16 or not x.is_contiguous():
        raise ValueError("tensor_scale requires a contiguous bf16 tensor")
    with torch.cuda.device(device):
        status = N.load().b2_tensor_scale(
            x.data_ptr(), x.numel(), float(bound), int(flags), scratch.data_ptr(), scale.data_ptr(), _stream(device)
        )
    N.check(status, "b2_tensor_scale")


def tensor_scale_static(x: torch.Tensor, bound: float, flags: int, scale: torch.Tensor) -> None:
    """``tensor_scale`` for callers that may not allocate or pass scratch memory: the scratch is a static
    array inside the library (``b2_tensor_scale_static``).  At most ``STATIC_SCALE_MAX_COUNT`` elements;
    calls that overlap on one GPU race on the shared array; make the first call on a device outside
    any stream capture."""
    device = _require_cuda(x, scale)
    if x.dtype != torch.bfloat16 or not x.is_contiguous():
        raise ValueError("tensor_scale_static requires a contiguous bf16 tensor")
    with torch.cuda.device(device):
        status = N.load().b2_tensor_scale_static(
            x.data_ptr(), x.numel(), float(bound), int(flags), scale.data_ptr(), _stream(device)
        )
    N.check(status, "b2_tensor_scale_static")


def fp8_quantize(x: torch.Tensor, out: torch.Tensor, scale: torch.Tensor, flags: int) -> None:
    """bf16 -> e4m3 at ``*scale``, see ``b2_fp8_quantize``."""
    device = _require_cuda(x, out, scale)
    if x.dtype != torch.bfloat16 or not x.is_contiguous() or not out.is_contiguous() or out.numel() != x.numel():
        raise ValueError("fp8_quantize requires contiguous bf16 input and a same-sized 1-byte output")
    with torch.cuda.device(device):
        status = N.load().b2_fp8_quantize(
            x.data_ptr(), out.data_ptr(), scale.data_ptr(), x.numel(), int(flags), _stream(device)
        )
    N.check(status, "b2_fp8_quantize")


def nvfp4_quantize(
    x: torch.Tensor,
    out: torch.Tensor,
    scales: torch.Tensor | None,
    blocked: torch.Tensor | None,
    global_scale: torch.Tensor,
    flags: int,
) -> None:
    """bf16 [R, K] -> packed e2m1 + e4m3 block scales, see ``b2_nvfp4_quantize``."""
    device = _require_cuda(x, out, scales, blocked, global_scale)
    if x.dtype != torch.bfloat16 or x.ndim != 2 or not x.is_contiguous():
        raise ValueError("nvfp4_quantize requires a contiguous bf16 matrix")
    rows, columns = x.shape
    with torch.cuda.device(device):
        status = N.load().b2_nvfp4_quantize(
            x.data_ptr(),
            out.data_ptr(),
            _ptr(scales),
            _ptr(blocked),
            global_scale.data_ptr(),
            rows,
            columns,
            int(flags),
            _stream(device),
        )
    N.check(status, "b2_nvfp4_quantize")


def geglu(
    gate: torch.Tensor,
    up: torch.Tensor | None,
    out: torch.Tensor,
    *,
    bits: int,
    table: torch.Tensor,
    rows: int,
    columns: int,
    row_stride: int,
    scale: torch.Tensor | None = None,
    scales: torch.Tensor | None = None,
    blocked: torch.Tensor | None = None,
    flags: int = 0,
) -> None:
    """GELU(gate) * up with the reference's two bf16 roundings, see ``b2_geglu``."""
    device = _require_cuda(gate, up, out, table, scale, scales, blocked)
    with torch.cuda.device(device):
        status = N.load().b2_geglu(
            gate.data_ptr(),
            _ptr(up),
            out.data_ptr(),
            _ptr(scales),
            _ptr(blocked),
            _ptr(scale),
            rows,
            columns,
            row_stride,
            bits,
            table.data_ptr(),
            int(flags),
            _stream(device),
        )
    N.check(status, "b2_geglu")


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor | None = None, *, status: torch.Tensor | None = None,
              codes: torch.Tensor | None = None, multiplier: float | None = None, blocked: torch.Tensor | None = None,
              scales: torch.Tensor | None = None, global_scale: float | None = None) -> torch.Tensor:
    """Unmasked multi-query attention, ``softmax(q k^T / sqrt(D)) v``: q [B, H, T, 256], k / v [B, 1, S, 256], all
    contiguous bf16; returns [B, H, T, 256] (``b2_attention``; the reference's ``SDPAAttention``).  With ``codes`` (a
    contiguous 1-byte [B*T, H*256] tensor) and ``multiplier`` the output is written as the e4m3 rows of the output
    projection instead (``b2_attention_fp8``) and ``codes`` is returned.  With ``codes`` ([B*T, H*128] bytes), ``blocked``
    (the tiled block scales, padding zeroed), ``global_scale`` and optionally ``scales`` (row-major [B*T, H*16]) it is
    written as the projection's NVFP4 rows (``b2_attention_nvfp4``)."""
    _require_cuda(q, k, v)
    if q.dim() != 4 or k.shape != v.shape or k.dim() != 4 or k.shape[1] != 1 or k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3]:
        raise ValueError("attention requires q [B, H, T, D] and k, v [B, 1, S, D]")
    if any(t.dtype != torch.bfloat16 or not t.is_contiguous() for t in (q, k, v)):
        raise ValueError("attention requires contiguous bf16 tensors")
    batch, heads, queries, head_dim = q.shape
    if status is None:
        status = status_word(q.device)
    if codes is not None and blocked is not None:
        rows, blocks = batch * queries, heads * head_dim // 16
        if global_scale is None or codes.element_size() != 1 or not codes.is_contiguous() or codes.numel() * 2 != q.numel() or \
                codes.device != q.device or blocked.element_size() != 1 or not blocked.is_contiguous() or blocked.device != q.device or \
                blocked.numel() < (rows + 127) // 128 * ((blocks + 3) // 4) * 512:
            raise ValueError("NVFP4 attention output needs contiguous codes [B*T, H*D/2], tiled block scales and a global scale")
        if scales is not None and (scales.element_size() != 1 or not scales.is_contiguous() or scales.numel() != rows * blocks or
                                   scales.device != q.device):
            raise ValueError("row-major block scales must be a contiguous 1-byte [B*T, H*D/16] tensor")
        with torch.cuda.device(q.device):
            code = N.load().b2_attention_nvfp4(q.data_ptr(), k.data_ptr(), v.data_ptr(), codes.data_ptr(),
                                               None if scales is None else scales.data_ptr(), blocked.data_ptr(), float(global_scale),
                                               batch, heads, queries, k.shape[2], head_dim, status.data_ptr(), _stream(q.device))
        N.check(code, "b2_attention_nvfp4")
        return codes
    if codes is not None:
        if multiplier is None or codes.element_size() != 1 or not codes.is_contiguous() or codes.numel() != q.numel() or codes.device != q.device:
            raise ValueError("encoded attention output must be a contiguous 1-byte [B*T, H*D] tensor with a multiplier")
        with torch.cuda.device(q.device):
            code = N.load().b2_attention_fp8(q.data_ptr(), k.data_ptr(), v.data_ptr(), codes.data_ptr(), float(multiplier), batch, heads,
                                             queries, k.shape[2], head_dim, status.data_ptr(), _stream(q.device))
        N.check(code, "b2_attention_fp8")
        return codes
    if out is None:
        out = torch.empty_like(q)
    elif out.shape != q.shape or out.dtype != torch.bfloat16 or not out.is_contiguous():
        raise ValueError("attention output must be a contiguous bf16 tensor of the queries' shape")
    with torch.cuda.device(q.device):
        code = N.load().b2_attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), batch, heads, queries, k.shape[2],
                                     head_dim, status.data_ptr(), _stream(q.device))
    N.check(code, "b2_attention")
    return out


def _rope_desc(sine: torch.Tensor, cosine: torch.Tensor, q_out: torch.Tensor, k_out: torch.Tensor, v_out: torch.Tensor, *,
               batch: int, tokens: int, heads: int, kv_heads: int, head_dim: int, kv_offset: int = 0) -> "N.RopeDesc":
    """The ``b2_rope_desc`` of these arguments (checked like :func:`rope_split`'s)."""
    _require_cuda(sine, cosine, q_out, k_out, v_out)
    for factor in (sine, cosine):
        if factor.dtype != torch.float32 or not factor.is_contiguous() or factor.shape[-2:] != (tokens, head_dim // 2):
            raise ValueError("rope requires contiguous fp32 factors [tokens, head_dim/2] (optionally with a batch dimension)")
    if q_out.shape != (batch, heads, tokens, head_dim) or not q_out.is_contiguous() or q_out.dtype != torch.bfloat16:
        raise ValueError("q_out must be a contiguous bf16 [batch, heads, tokens, head_dim] tensor")
    for cache in (k_out, v_out):
        if cache.ndim != 4 or cache.shape[0] != batch or cache.shape[1] != kv_heads or cache.shape[3] != head_dim or \
                not cache.is_contiguous() or cache.dtype != torch.bfloat16 or cache.shape != k_out.shape:
            raise ValueError("key/value buffers must be contiguous bf16 [batch, kv_heads, capacity, head_dim] tensors")
    return N.RopeDesc(sine=sine.data_ptr(), cosine=cosine.data_ptr(), q_out=q_out.data_ptr(), k_out=k_out.data_ptr(),
                      v_out=v_out.data_ptr(), factor_batch_stride=tokens * (head_dim // 2) if sine.ndim == 3 else 0,
                      batch=batch, tokens=tokens, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                      kv_capacity=k_out.shape[2], kv_offset=kv_offset)


def rope_split(qkv: torch.Tensor, sine: torch.Tensor, cosine: torch.Tensor, q_out: torch.Tensor, k_out: torch.Tensor,
               v_out: torch.Tensor, *, batch: int, tokens: int, heads: int, kv_heads: int, head_dim: int, kv_offset: int = 0) -> None:
    """Split a packed QKV projection, rotate queries and keys, write ``q_out`` [B, heads, T, D] and the
    keys / values into ``k_out`` / ``v_out`` [B, kv_heads, S, D] at ``kv_offset``; see ``b2_rope_split``.
    ``sine`` / ``cosine``: fp32 [T, D/2] or [B, T, D/2]."""
    device = _require_cuda(qkv, sine, cosine, q_out, k_out, v_out)
    width = (heads + 2 * kv_heads) * head_dim
    if qkv.dtype != torch.bfloat16 or not qkv.is_contiguous() or qkv.numel() != batch * tokens * width:
        raise ValueError("rope_split requires a contiguous bf16 [batch*tokens, (heads + 2*kv_heads)*head_dim] projection")
    for factor in (sine, cosine):
        if factor.dtype != torch.float32 or not factor.is_contiguous() or factor.shape[-2:] != (tokens, head_dim // 2):
            raise ValueError("rope_split requires contiguous fp32 factors [tokens, head_dim/2] (optionally with a batch dimension)")
    if q_out.shape != (batch, heads, tokens, head_dim) or not q_out.is_contiguous() or q_out.dtype != torch.bfloat16:
        raise ValueError("q_out must be a contiguous bf16 [batch, heads, tokens, head_dim] tensor")
    for cache in (k_out, v_out):
        if cache.ndim != 4 or cache.shape[0] != batch or cache.shape[1] != kv_heads or cache.shape[3] != head_dim or \
                not cache.is_contiguous() or cache.dtype != torch.bfloat16:
            raise ValueError("key/value buffers must be contiguous bf16 [batch, kv_heads, capacity, head_dim] tensors")
    stride = tokens * (head_dim // 2) if sine.ndim == 3 else 0
    with torch.cuda.device(device):
        status = N.load().b2_rope_split(qkv.data_ptr(), sine.data_ptr(), cosine.data_ptr(), q_out.data_ptr(), k_out.data_ptr(),
                                        v_out.data_ptr(), batch, tokens, heads, kv_heads, head_dim, stride, k_out.shape[2],
                                        kv_offset, _stream(device))
    N.check(status, "b2_rope_split")


def rope_axes(positions: torch.Tensor, sections: tuple[int, ...], sine: torch.Tensor | None = None, cosine: torch.Tensor | None = None, *,
              theta: float = 10000.0, own_spectrum: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """Sine / cosine tables of rotary positions with several axes, see ``b2_rope_axes``: ``positions`` int32 or int64
    [axes, ..., T] (contiguous), ``sections`` the number of frequencies of each axis (their sum is head_dim / 2).  Returns
    fp32 (sine, cosine) [..., T, head_dim / 2], the factors of :func:`rope_split` and :func:`kv_cache_write`."""
    device = _require_cuda(positions, sine, cosine)
    if positions.dtype not in (torch.int32, torch.int64) or positions.ndim < 2 or not positions.is_contiguous():
        raise ValueError("rope_axes requires contiguous int32 or int64 positions [axes, ..., tokens]")
    shape = positions.shape
    axes, half = shape[0], 0
    for section in sections:
        if type(section) is not int or not 0 < section < 1 << 30:
            axes = -1
            break
        half += section
    if len(sections) != axes:
        raise ValueError("rope_axes requires one positive section for each axis")
    shape = (*shape[1:], half)
    if sine is None and cosine is None:
        sine = positions.new_empty(shape, dtype=torch.float32)
        cosine = torch.empty_like(sine)
    else:
        for table in (sine, cosine):
            if table is None or table.dtype != torch.float32 or table.shape != shape or not table.is_contiguous():
                raise ValueError("rope_axes requires contiguous fp32 tables [..., tokens, head_dim/2], both or neither")
    tokens = positions.numel() // axes if axes else 0
    if tokens == 0:
        return sine, cosine
    status = _launch(N.load().b2_rope_axes, device, positions.data_ptr(), positions.element_size(), struct.pack(f"{axes}i", *sections), axes,
                     tokens, 2 * half, float(theta), N.ROPE_OWN_SPECTRUM if own_spectrum else 0, sine.data_ptr(), cosine.data_ptr())
    N.check(status, "b2_rope_axes")
    return sine, cosine


# The descriptors of the calls that a decoding step makes for every token, packed: filling the ctypes structures takes longer than
# launching the kernel.
_CACHE_DESC = struct.Struct("12P10q6i0q")
_ATTENTION_DESC = struct.Struct("15P4qf10i0q")
assert _CACHE_DESC.size == ctypes.sizeof(N.KVCacheDesc) and _ATTENTION_DESC.size == ctypes.sizeof(N.PrefixAttentionDesc)


def _address(tensor: torch.Tensor | None) -> int:
    return 0 if tensor is None else tensor.data_ptr()


def _check_cache(cache: QuantizedKVCache, what: str) -> tuple[int, int, int, int]:
    """The (batch, kv_heads, capacity, head_dim) of a quantised cache."""
    k_codes, k_scales, v_codes, v_scales = cache
    shape = k_codes.shape
    rows = shape[:3]
    if len(shape) != 4 or v_codes.shape != shape or k_scales.shape != rows or v_scales.shape != rows:
        raise ValueError(f"{what} requires codes [batch, kv_heads, capacity, head_dim] and scales [batch, kv_heads, capacity]")
    if not (k_codes.element_size() == 1 == v_codes.element_size() and k_scales.dtype is torch.float32 is v_scales.dtype and k_codes.is_contiguous()
            and v_codes.is_contiguous() and k_scales.is_contiguous() and v_scales.is_contiguous()):
        raise ValueError(f"{what} requires contiguous one-byte codes and contiguous fp32 scales")
    return shape


def _check_whole(values: torch.Tensor, count: int, what: str) -> None:
    if values.dtype is not torch.int32 or values.shape != (count,) or not values.is_contiguous():
        raise ValueError(f"{what} must be a contiguous int32 tensor of {count} values")


def _check_cache_rows(k: torch.Tensor, v: torch.Tensor, cache: QuantizedKVCache, offsets, lengths, what: str) -> tuple:
    """Everything that a write and a read have in common: (batch, kv_heads, capacity, head_dim, tokens, the strides of k and v)."""
    batch, kv_heads, capacity, head_dim = _check_cache(cache, what)
    shape = k.shape
    if v.shape != shape or len(shape) != 4 or shape[0] != batch or shape[1] != kv_heads or shape[3] != head_dim:
        raise ValueError(f"{what} requires keys and values [batch, kv_heads, tokens, head_dim] that fit the cache")
    k_stride, v_stride = k.stride(), v.stride()
    if not (k.dtype is torch.bfloat16 is v.dtype and k_stride[3] == 1 == v_stride[3]):
        raise ValueError(f"{what} requires bf16 keys and values whose last dimension is contiguous")
    if offsets is not None:
        _check_whole(offsets, batch, "offsets")
    if lengths is not None:
        _check_whole(lengths, batch, "lengths")
    return batch, kv_heads, capacity, head_dim, shape[2], (*k_stride[:3], *v_stride[:3])


def kv_cache_write(k: torch.Tensor, v: torch.Tensor, cache: QuantizedKVCache, *, q: torch.Tensor | None = None,
                   q_out: torch.Tensor | None = None, sine: torch.Tensor | None = None, cosine: torch.Tensor | None = None,
                   offsets: torch.Tensor | None = None, lengths: torch.Tensor | None = None) -> None:
    """Quantise keys and values [B, kv_heads, T, D] into ``cache`` at positions ``offsets[b] + t`` for ``t < lengths[b]``
    (int32 [B]; default 0 and T); with ``sine`` / ``cosine`` (fp32 [T, D/2] or [B, T, D/2]) keys are rotated first, and the
    rotated ``q`` [B, H, T, D] goes to ``q_out`` (contiguous).  k, v and q may be views of one packed projection.  See
    ``b2_kv_cache_write``; padded tokens and positions outside the cache are passed over."""
    device = _require_cuda(k, v, *cache, q, q_out, sine, cosine, offsets, lengths)
    batch, kv_heads, capacity, head_dim, tokens, strides = _check_cache_rows(k, v, cache, offsets, lengths, "kv_cache_write")
    if (q is None) != (q_out is None) or (sine is None) != (cosine is None):
        raise ValueError("kv_cache_write takes q with q_out, and sine with cosine")
    heads, q_stride, factor_stride = 0, (0, 0, 0), 0
    if q is not None:
        shape, q_stride = q.shape, q.stride()
        if q.dtype is not torch.bfloat16 or len(shape) != 4 or shape[0] != batch or shape[2] != tokens or shape[3] != head_dim or q_stride[3] != 1:
            raise ValueError("q must be bf16 [batch, heads, tokens, head_dim] with a contiguous last dimension")
        if q_out.dtype is not torch.bfloat16 or q_out.shape != shape or not q_out.is_contiguous():
            raise ValueError("q_out must be a contiguous bf16 tensor of q's shape")
        heads, q_stride = shape[1], q_stride[:3]
    if sine is not None:
        shape, half = sine.shape, head_dim // 2
        if not (sine.dtype is torch.float32 is cosine.dtype and cosine.shape == shape and sine.is_contiguous() and cosine.is_contiguous()
                and (shape == (tokens, half) or shape == (batch, tokens, half))):
            raise ValueError("kv_cache_write requires contiguous fp32 factors [tokens, head_dim/2] or [batch, tokens, head_dim/2]")
        factor_stride = tokens * half if len(shape) == 3 else 0
    if not (batch and kv_heads and tokens and head_dim and capacity):
        return
    k_codes, k_scales, v_codes, v_scales = cache
    desc = _CACHE_DESC.pack(_address(q), _address(q_out), k.data_ptr(), v.data_ptr(), _address(sine), _address(cosine), k_codes.data_ptr(),
                            k_scales.data_ptr(), v_codes.data_ptr(), v_scales.data_ptr(), _address(offsets), _address(lengths), *q_stride,
                            *strides, factor_stride, batch, tokens, heads, kv_heads, head_dim, capacity)
    N.check(_launch(N.load().b2_kv_cache_write, device, desc), "b2_kv_cache_write")


def kv_cache_read(cache: QuantizedKVCache, k_out: torch.Tensor, v_out: torch.Tensor, *, offsets: torch.Tensor | None = None,
                  lengths: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Positions ``offsets[b] + t`` of ``cache`` as bf16 into row ``t`` of ``k_out`` / ``v_out`` [B, kv_heads, T, D], for
    ``t < lengths[b]`` (defaults 0 and T); the other rows are left as they are.  See ``b2_kv_cache_read``."""
    device = _require_cuda(*cache, k_out, v_out, offsets, lengths)
    batch, kv_heads, capacity, head_dim, tokens, strides = _check_cache_rows(k_out, v_out, cache, offsets, lengths, "kv_cache_read")
    if batch and kv_heads and tokens and head_dim and capacity:
        k_codes, k_scales, v_codes, v_scales = cache
        desc = _CACHE_DESC.pack(0, 0, k_out.data_ptr(), v_out.data_ptr(), 0, 0, k_codes.data_ptr(), k_scales.data_ptr(), v_codes.data_ptr(),
                                v_scales.data_ptr(), _address(offsets), _address(lengths), 0, 0, 0, *strides, 0, batch, tokens, 0, kv_heads,
                                head_dim, capacity)
        N.check(_launch(N.load().b2_kv_cache_read, device, desc), "b2_kv_cache_read")
    return k_out, v_out


def _cache_part(part, count: int, width: int, what: str) -> tuple[int, int, int, int, tuple]:
    """(bits, batch, kv_heads, capacity, the four pointers k, v, k_scales, v_scales) of a prefix or own cache."""
    if isinstance(part, QuantizedKVCache):
        batch, kv_heads, capacity, head_dim = _check_cache(part, "prefix_attention")
        k, k_scales, v, v_scales = part
        bits, pointers = 8, (k.data_ptr(), v.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr())
    else:
        k, v = part
        shape = k.shape
        if not (len(shape) == 4 and v.shape == shape and k.dtype is torch.bfloat16 is v.dtype and k.is_contiguous() and v.is_contiguous()):
            raise ValueError("prefix_attention requires contiguous bf16 keys and values [n, kv_heads, capacity, head_dim], or quantised caches")
        batch, kv_heads, capacity, head_dim = shape
        bits, pointers = 16, (k.data_ptr(), v.data_ptr(), 0, 0)
    if batch != count and count >= 0 or head_dim != width:
        raise ValueError(f"prefix_attention: the {what} cache does not fit the queries")
    return bits, batch, kv_heads, capacity, pointers if capacity else (0, 0, 0, 0)


def _attend(library, q: torch.Tensor, pointers: tuple, sizes: tuple, stream: int) -> int:
    desc = _ATTENTION_DESC.pack(*pointers, 0, 0, *sizes)
    size = library.b2_prefix_attention_workspace_bytes(desc)
    if size:          # scratch of this call alone (also inside a captured graph: it is the graph's own)
        workspace = q.new_empty(size, dtype=torch.uint8)
        desc = _ATTENTION_DESC.pack(*pointers, workspace.data_ptr(), size, *sizes)
    return library.b2_prefix_attention(desc, stream)


def prefix_attention(q: torch.Tensor, prefix, own=None, *, members: torch.Tensor | None = None, prefix_lengths: torch.Tensor | None = None,
                     own_lengths: torch.Tensor | None = None, causal: bool = False, scale: float | None = None,
                     out: torch.Tensor | None = None, status: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of a batch whose members share prefixes: ``q`` bf16 [B, H, T, D]; ``prefix`` holds one key/value cache for each
    of G groups and ``own`` (or None) one for each batch element -- a pair (k, v) of bf16 tensors [G or B, kv_heads, capacity, D]
    or a :class:`QuantizedKVCache`, both of one kind.  ``members`` int32 [G + 1]: group g is the batch elements
    [members[g], members[g + 1]); default B / G each.  ``prefix_lengths`` int32 [G], ``own_lengths`` int32 [B]: default the
    capacities.  ``causal``: query t sees all but the last T - 1 - t own keys.  ``scale`` defaults to 1 / sqrt(D).  Returns bf16
    [B, H, T, D]; rows that see no key are zero, batch elements outside every group are left as ``out`` had them.  See
    ``b2_prefix_attention``."""
    if prefix is None:
        raise ValueError("prefix_attention requires a prefix cache (its capacity may be 0)")
    device = _require_cuda(q, *prefix, *(own or ()), members, prefix_lengths, own_lengths, out, status)
    shape, q_stride = q.shape, q.stride()
    if len(shape) != 4 or q.dtype is not torch.bfloat16 or q_stride[3] != 1:
        raise ValueError("prefix_attention requires bf16 queries [batch, heads, tokens, head_dim] with a contiguous last dimension")
    batch, heads, queries, head_dim = shape
    bits, groups, kv_heads, prefix_capacity, prefix_pointers = _cache_part(prefix, -1, head_dim, "prefix")
    own_capacity, own_pointers = 0, (0, 0, 0, 0)
    if own is not None:
        own_bits, _, own_kv_heads, own_capacity, own_pointers = _cache_part(own, batch, head_dim, "own")
        if own_bits != bits or own_kv_heads != kv_heads:
            raise ValueError("prefix_attention requires prefix and own caches of one kind with equal kv_heads")
    for values, count, name in ((members, groups + 1, "members"), (prefix_lengths, groups, "prefix_lengths"), (own_lengths, batch, "own_lengths")):
        if values is not None:
            _check_whole(values, count, name)
    if kv_heads == 0 or heads % kv_heads or groups == 0 or (members is None and batch % groups):
        raise ValueError("prefix_attention requires heads divisible by kv_heads, and a batch divisible by the groups unless members is given")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.shape != shape or out.dtype is not torch.bfloat16 or not out.is_contiguous():
        raise ValueError("attention output must be a contiguous bf16 tensor of the queries' shape")
    if not (batch and heads and queries and head_dim):
        return out
    if prefix_capacity == 0 and own_capacity == 0:          # nothing to see: zeros, for what the groups hold
        if members is None:
            return out.zero_()
        index = torch.arange(batch, device=device)
        return out.masked_fill_(((index >= members[0]) & (index < members[-1])).view(batch, 1, 1, 1), 0.0)
    if status is None:
        status = status_word(device)
    pointers = (q.data_ptr(), out.data_ptr(), *prefix_pointers, *own_pointers, _address(members), _address(prefix_lengths),
                _address(own_lengths), status.data_ptr())
    sizes = (*q_stride[:3], head_dim ** -0.5 if scale is None else scale, N.ATTENTION_CAUSAL if causal else 0, batch, groups, heads,
             kv_heads, queries, head_dim, prefix_capacity, own_capacity, bits)
    N.check(_launch(_attend, device, N.load(), q, pointers, sizes), "b2_prefix_attention")
    return out


def norm_quant(inputs: torch.Tensor, output: torch.Tensor, *, bits: int, tokens: int, scale: torch.Tensor | None = None,
               modulation: torch.Tensor | None = None, update: torch.Tensor | None = None,
               update_gate: torch.Tensor | None = None, mean: torch.Tensor | None = None,
               global_scale: torch.Tensor | None = None, residual: torch.Tensor | None = None,
               scales: torch.Tensor | None = None, blocked: torch.Tensor | None = None, gate: torch.Tensor | None = None,
               inverse: torch.Tensor | None = None, flags: int = 0) -> None:
    """Residual update + RMSNorm (offset scale or adaptive modulation) + bf16 rounding + encoder over the
    contiguous bf16 rows of ``inputs`` [..., columns]; see ``b2_norm_quant`` for every argument."""
    present = [t for t in (inputs, output, scale, modulation, update, update_gate, mean, global_scale, residual, scales,
                           blocked, gate, inverse) if t is not None]
    device = _require_cuda(*present)
    if inputs.dtype != torch.bfloat16 or not inputs.is_contiguous():
        raise ValueError("norm_quant requires contiguous bf16 rows")
    for other in (update, residual):
        if other is not None and (other.shape != inputs.shape or other.dtype != torch.bfloat16 or not other.is_contiguous()):
            raise ValueError("update and residual must match the input's shape, dtype and layout")
    for affine in (scale, modulation, mean, inverse):
        if affine is not None and (affine.dtype != torch.float32 or not affine.is_contiguous()):
            raise ValueError("scale, modulation, mean and inverse must be contiguous fp32 tensors")
    columns = inputs.shape[-1]
    rows = inputs.numel() // columns
    desc = N.NormDesc(
        input=inputs.data_ptr(), update=_ptr(update), update_gate=_ptr(update_gate), scale=_ptr(scale),
        modulation=_ptr(modulation), mean=_ptr(mean), global_scale=_ptr(global_scale), residual=_ptr(residual),
        output=output.data_ptr(), scales=_ptr(scales), blocked=_ptr(blocked), gate=_ptr(gate), inverse=_ptr(inverse),
        rows=rows, columns=columns, tokens=tokens, bits=bits, flags=int(flags))
    with torch.cuda.device(device):
        status = N.load().b2_norm_quant(ctypes.byref(desc), _stream(device))
    N.check(status, "b2_norm_quant")


def layer_norm_quant(inputs: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor, output: torch.Tensor, *, bits: int,
                     scale_value: float = 1.0, update: torch.Tensor | None = None, residual: torch.Tensor | None = None,
                     scales: torch.Tensor | None = None, blocked: torch.Tensor | None = None,
                     statistics: torch.Tensor | None = None) -> None:
    """Residual update + LayerNorm + bf16 rounding + encoder over the contiguous bf16 rows of ``inputs``
    [..., columns]; ``scale_value`` is the e4m3 multiplier (bits 8) or the NVFP4 global scale (bits 4); see
    ``b2_layer_norm_quant``."""
    device = _require_cuda(inputs, weight, bias, output, update, residual, scales, blocked, statistics)
    if inputs.dtype != torch.bfloat16 or not inputs.is_contiguous():
        raise ValueError("layer_norm_quant requires contiguous bf16 rows")
    columns = inputs.shape[-1]
    for affine in (weight, bias):
        if affine.dtype != torch.bfloat16 or affine.shape != (columns,) or not affine.is_contiguous():
            raise ValueError("weight and bias must be contiguous bf16 [columns] tensors")
    for other in (update, residual):
        if other is not None and (other.shape != inputs.shape or other.dtype != torch.bfloat16 or not other.is_contiguous()):
            raise ValueError("update and residual must match the input's shape, dtype and layout")
    with torch.cuda.device(device):
        status = N.load().b2_layer_norm_quant(inputs.data_ptr(), _ptr(update), weight.data_ptr(), bias.data_ptr(), _ptr(residual),
                                              output.data_ptr(), _ptr(scales), _ptr(blocked), _ptr(statistics), float(scale_value),
                                              inputs.numel() // columns, columns, bits, _stream(device))
    N.check(status, "b2_layer_norm_quant")


def bhsd_quant(attended: torch.Tensor, output: torch.Tensor, *, bits: int, scale_value: float = 1.0,
               scales: torch.Tensor | None = None, blocked: torch.Tensor | None = None) -> None:
    """Attention output [B, H, S, D] (any strides with D contiguous) -> encoded rows [B*S, H*D]; ``scale_value`` is
    the e4m3 multiplier (bits 8) or the NVFP4 global scale (bits 4); see ``b2_bhsd_quant``."""
    device = _require_cuda(attended, output, scales, blocked)
    if attended.dtype != torch.bfloat16 or attended.ndim != 4 or attended.stride(3) != 1:
        raise ValueError("bhsd_quant requires a bf16 [B, H, S, D] tensor whose last dimension is contiguous")
    batch, heads, tokens, head_dim = attended.shape
    with torch.cuda.device(device):
        status = N.load().b2_bhsd_quant(attended.data_ptr(), output.data_ptr(), _ptr(scales), _ptr(blocked), float(scale_value),
                                        attended.stride(0), attended.stride(1), attended.stride(2), batch, heads, tokens,
                                        head_dim, bits, _stream(device))
    N.check(status, "b2_bhsd_quant")


def normalize_frames(frames: torch.Tensor, images: torch.Tensor) -> None:
    """``(frames / 255) * 2 - 1`` into fp32 ``images`` [cameras, 3, H, W]; ``frames`` is contiguous uint8
    [cameras, H, W, 3] (same checks and errors as the reference's ``normalize_frames``)."""
    if frames.dtype != torch.uint8 or frames.ndim != 4 or frames.shape[3] != 3 or not frames.is_contiguous():
        raise ValueError("frames must be contiguous uint8 [cameras, height, width, 3]")
    if images.dtype != torch.float32 or images.ndim != 4 or tuple(images.shape[:2]) != (frames.shape[0], 3) or \
            not images.is_contiguous():
        raise ValueError("images must be contiguous float32 [cameras, 3, height, width]")
    if frames.device.type != "cuda" or images.device != frames.device:
        raise ValueError("frames and images must share a CUDA device")
    if tuple(images.shape[2:]) != tuple(frames.shape[1:3]):
        raise ValueError("images must have the frame height and width")
    with torch.cuda.device(frames.device):
        status = N.load().b2_normalize_frames(frames.data_ptr(), images.data_ptr(), frames.shape[0],
                                              frames.shape[1] * frames.shape[2], _stream(frames.device))
    N.check(status, "b2_normalize_frames")


def frames_to_patches(frames: torch.Tensor, patches: torch.Tensor, patch: int) -> None:
    """uint8 frames [cameras, H, W, 3] -> bf16 patch rows [cameras * (H/patch) * (W/patch), 3*patch*patch] holding
    ``bf16((x / 255) * 2 - 1)`` in (channel, y, x) order; see ``b2_frames_to_patches``."""
    device = _require_cuda(frames, patches)
    if frames.dtype != torch.uint8 or frames.ndim != 4 or frames.shape[3] != 3 or not frames.is_contiguous():
        raise ValueError("frames must be contiguous uint8 [cameras, height, width, 3]")
    cameras, height, width, _ = frames.shape
    expected = (cameras * (height // patch) * (width // patch), 3 * patch * patch)
    if patches.dtype != torch.bfloat16 or tuple(patches.shape) != expected or not patches.is_contiguous():
        raise ValueError("patches must be contiguous bf16 [cameras * grid_h * grid_w, 3 * patch * patch]")
    with torch.cuda.device(device):
        status = N.load().b2_frames_to_patches(frames.data_ptr(), patches.data_ptr(), cameras, height, width, patch,
                                               _stream(device))
    N.check(status, "b2_frames_to_patches")


# ---- the status word of the bounded waits -------------------------------------------------------------
# Every wait inside the tensor-core kernels is bounded; a wait that runs out leaves a code in the launch's status
# word and the kernel drains with a wrong result instead of hanging.  The plan objects and the registry kernels
# pass ONE word per device to every launch (a launch only ever writes a non-zero code into a zero word), and the
# host reads it where it synchronises anyway: at the end of a rollout step, when a workspace scope is released.
STATUS_NAMES = {0x101: "the TMA producer waited for a free stage", 0x102: "the MMA issuer waited for a filled stage",
                0x103: "the MMA issuer waited for a drained accumulator", 0x104: "the epilogue waited for a finished accumulator",
                0x105: "the producer waited for its copies in flight", 0x106: "a CTA waited for the other K ranges of its tile",
                0x107: "a CTA waited for the partial sums of its cluster",
                0x108: "a CTA waited for the partial attention rows of its cluster"}
_status_words: dict[int, torch.Tensor] = {}


def status_word(device: torch.device) -> torch.Tensor:
    """The device's status word (int32, zero unless a bounded wait expired since the last check).  Created on first
    use: touch it once before capturing a CUDA graph, as with every plan buffer."""
    index = device.index if device.index is not None else torch.cuda.current_device()
    word = _status_words.get(index)
    if word is None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("Warm tensor-core launches before graph capture")
        word = _status_words[index] = torch.zeros(1, device=torch.device("cuda", index), dtype=torch.int32)
    return word


def check_status(device: torch.device) -> None:
    """Read the device's status word (this synchronises with the device) and raise ``RuntimeError`` naming the wait
    that expired; the word is cleared so that later launches are judged on their own."""
    index = device.index if device.index is not None else torch.cuda.current_device()
    word = _status_words.get(index)
    if word is None:
        return
    code = int(word.item())
    if code != 0:
        word.zero_()
        what = STATUS_NAMES.get(code, "an unknown wait")
        raise RuntimeError(f"a tensor-core launch on cuda:{index} gave up a bounded wait (status {code:#x}: {what} for longer than "
                           "its limit); its result and those of the launches after it are invalid")


_WORKSPACE_BYTES = 32 << 20
_workspaces: dict[tuple[int, int], torch.Tensor] = {}


def linear_workspace(device: torch.device) -> torch.Tensor:
    """Zeroed split-K scratch for launches on the current stream of ``device`` (one per device and stream,
    created on first use: warm a shape up before capturing it, as with every plan buffer).  Launches that
    follow one another on a stream can share it: each leaves its ticket words zero again."""
    key = (device.index if device.index is not None else torch.cuda.current_device(), _stream(device))
    workspace = _workspaces.get(key)
    if workspace is None:
        workspace = _workspaces[key] = torch.zeros(_WORKSPACE_BYTES, device=device, dtype=torch.uint8)
    return workspace


def linear(
    *,
    kind: int,
    epilogue: int,
    out_format: int,
    tokens: int,
    features: int,
    width: int,
    act: torch.Tensor,
    act_scale: torch.Tensor,
    weight: torch.Tensor,
    weight_scale: torch.Tensor,
    out: torch.Tensor,
    act_scales: torch.Tensor | None = None,
    weight_scales: torch.Tensor | None = None,
    weight_scale_up: torch.Tensor | None = None,
    bias: torch.Tensor | None = None,
    residual: torch.Tensor | None = None,
    gelu_table: torch.Tensor | None = None,
    out_scale: torch.Tensor | None = None,
    out_scales: torch.Tensor | None = None,
    out_blocked: torch.Tensor | None = None,
    status: torch.Tensor | None = None,
    flags: int = 0,
    feature_tile: int = 0,
    gelu_range: tuple[int, int] = (0, 0),
    workspace: torch.Tensor | None | bool = None,
    rope: dict | None = None,
) -> None:
    """One fused tensor-core launch, see ``b2_linear``.  ``status``: the word an expired bounded wait is reported in
    (default: the device's word, read by :func:`check_status`).  ``workspace``: zeroed split-K scratch, e.g.
    :func:`linear_workspace`; without one (the default) K is never split.  The fix-up through the L2 costs
    more than the shorter K loop saves at every shape of the pi0.5 stacks measured so far (560x2048x16384:
    35 vs 28 us; 10x2560x1024: 12.5 vs 5.6 us), so the plans do not pass one."""
    device = _require_cuda(
        act, act_scale, weight, weight_scale, out, act_scales, weight_scales, weight_scale_up, bias, residual, gelu_table, out_scale,
        out_scales, out_blocked, status,
    )
    if status is None:
        status = status_word(device)
    desc = N.LinearDesc(
        kind=kind,
        epilogue=epilogue,
        out_format=out_format,
        flags=flags,
        tokens=tokens,
        features=features,
        width=width,
        feature_tile=feature_tile,
        gelu_lo=gelu_range[0],
        gelu_hi=gelu_range[1],
        act=act.data_ptr(),
        act_scales=_ptr(act_scales),
        act_scale=act_scale.data_ptr(),
        weight=weight.data_ptr(),
        weight_scales=_ptr(weight_scales),
        weight_scale=weight_scale.data_ptr(),
        weight_scale_up=_ptr(weight_scale_up),
        bias=_ptr(bias),
        residual=_ptr(residual),
        gelu_table=_ptr(gelu_table),
        out_scale=_ptr(out_scale),
        out=out.data_ptr(),
        out_scales=_ptr(out_scales),
        out_blocked=_ptr(out_blocked),
        status=_ptr(status),
    )
    if isinstance(workspace, torch.Tensor):
        desc.workspace, desc.workspace_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    preparation = None
    if rope is not None:
        # the attention preparation as this projection's epilogue (``b2_linear_desc.rope``); `out` is not written
        preparation = _rope_desc(**rope)
        desc.rope = ctypes.addressof(preparation)
    with torch.cuda.device(device):
        code = N.load().b2_linear(ctypes.byref(desc), _stream(device))
    N.check(code, "b2_linear")
