// The quantised key/value cache: rows of head_dim e4m3 codes with one fp32 scale for each (token, head), written behind
// the QKV projection and read back as bf16.
//
//   write   x' = rotation of the row (keys; queries go to q_out as bf16), or the row itself (values, no tables given)
//           scale = max|x'| / 448,  code = e4m3(x' / scale)
//           scale = 0 and codes 0 when max|x'| < 2^-50; scale = NaN when max|x'| >= 2^40 or a value of the row is not finite,
//           so that the whole row reads back as NaN.  Between the two lie 90 binades, which is what lets the attention kernel
//           carry 1 / scale and weights that contain the scale in fp32 without losing either end.
//   read    bf16(code * scale)
//
// The rotation is b2_rope_split's: fp32 factors, separate multiplies and add / subtract.  Keys are quantised from the fp32
// rotation: one rounding, not two.  The scale is held in fp32 and is not rounded to a power of two: that costs 4 bytes per row
// of 128 or 256 and keeps all of the codes' range.
//
// Both kernels move bytes: 16-byte loads, a row dealt to head_dim / 16 lanes (a lane holds 8 values of the first half and the
// 8 values they rotate with), the row maximum by shuffles inside those lanes, no shared memory.
// Measured (B200): 16 prompts of 500 to 1000 tokens, 32 query and 8 key/value heads of 128, written in 58 us (285 MB, 4.9 TB/s).  Neither
// memory (46 % of DRAM's rate over the launch) nor issue (61 % of the slots: the rotation's separate roundings, row maxima, exact division)
// is full: 20 warps per SM, 8 cycles from one instruction of a warp to its next.  More of them cost more than they give (80 registers: four
// rows per thread share their factors; two rows per thread 68 us, 64 registers 66).  8 x 8 x 8192 rows of 128 read in 63 us (406 MB,
// 6.5 TB/s: copy speed; with two 16-byte stores for each 32 bytes 72).  The few tokens of a decoding step take 2.8 us either way.
#include "common.cuh"

namespace b2 {

namespace {

constexpr int CACHE_THREADS = 256;
constexpr float CACHE_TINY = 8.8817841970012523e-16f, CACHE_HUGE = 1099511627776.0f;      // 2^-50, 2^40

struct CacheArgs {
    const __nv_bfloat16* q;      // write: queries, or nullptr
    __nv_bfloat16* q_out;        // write: [batch, heads, tokens, head_dim]
    __nv_bfloat16* rows[2];      // keys, values [batch, kv_heads, tokens, head_dim]: read by write, written by read
    const float* sine;           // or nullptr: no rotation
    const float* cosine;
    uint8_t* codes[2];           // [batch, kv_heads, capacity, head_dim]
    float* scales[2];            // [batch, kv_heads, capacity]
    const int32_t* offsets;      // [batch] or nullptr: 0
    const int32_t* lengths;      // [batch] or nullptr: tokens
    int64_t q_stride[3], stride[2][3];      // elements: batch, head, token
    int64_t factor_batch_stride;
    int batch, tokens, heads, kv_heads, capacity, slots;
    bool wide;                   // read: every output row starts on 32 bytes
};

// Cache position of token t of sequence b, or -1: beyond the sequence's length or outside the cache.
__device__ __forceinline__ int64_t cache_position(const CacheArgs& args, int b, int t) {
    const int length = args.lengths == nullptr ? args.tokens : __ldg(args.lengths + b);
    const int64_t position = int64_t(t) + (args.offsets == nullptr ? 0 : __ldg(args.offsets + b));
    return t < length && position >= 0 && position < args.capacity ? position : -1;
}

// HEADS rows of one token per thread: they share the rotation factors, and their loads are in flight together.
template <int D, int HEADS>
__global__ void __launch_bounds__(CACHE_THREADS) kv_cache_write_kernel(const __grid_constant__ CacheArgs args) {
    pdl_launch_dependents();
    pdl_wait();
    constexpr int LANES = D / 16, HALF = D / 2;
    const uint32_t item = blockIdx.x * uint32_t(CACHE_THREADS / LANES) + threadIdx.x / LANES;
    const int lane = threadIdx.x % LANES;
    const uint32_t token = item / uint32_t(args.slots);
    const int slot = int(item - token * uint32_t(args.slots));
    const int b = int(token / uint32_t(args.tokens));
    const int t = int(token - uint32_t(b) * uint32_t(args.tokens));
    // every lane stays for the shuffles; a row that is not there is a row of zeros that is not stored
    const bool present = b < args.batch && t < (args.lengths == nullptr ? args.tokens : __ldg(args.lengths + (b < args.batch ? b : 0)));
    const int64_t position = present ? cache_position(args, b, t) : -1;
    const int all_heads = args.heads + 2 * args.kv_heads;

    uint4 first[HEADS], second[HEADS];
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
        const int head = slot + i * args.slots;
        first[i] = second[i] = make_uint4(0, 0, 0, 0);
        if (!present || head >= all_heads) continue;
        const __nv_bfloat16* source;
        if (head < args.heads) {
            source = args.q + b * args.q_stride[0] + head * args.q_stride[1] + t * args.q_stride[2];
        } else {
            const int which = head >= args.heads + args.kv_heads;
            const int kv_head = head - args.heads - which * args.kv_heads;
            source = args.rows[which] + b * args.stride[which][0] + kv_head * args.stride[which][1] + t * args.stride[which][2];
        }
        first[i] = ld_nc_u4(reinterpret_cast<const uint4*>(source + lane * 8));
        second[i] = ld_nc_u4(reinterpret_cast<const uint4*>(source + HALF + lane * 8));
    }
    float s[8], c[8];
    if (args.sine != nullptr && present) {
        const int64_t base = b * args.factor_batch_stride + int64_t(t) * HALF + lane * 8;
        const float4* sp = reinterpret_cast<const float4*>(args.sine + base);
        const float4* cp = reinterpret_cast<const float4*>(args.cosine + base);
        const float4 s0 = __ldg(sp), s1 = __ldg(sp + 1), c0 = __ldg(cp), c1 = __ldg(cp + 1);
        s[0] = s0.x; s[1] = s0.y; s[2] = s0.z; s[3] = s0.w; s[4] = s1.x; s[5] = s1.y; s[6] = s1.z; s[7] = s1.w;
        c[0] = c0.x; c[1] = c0.y; c[2] = c0.z; c[3] = c0.w; c[4] = c1.x; c[5] = c1.y; c[6] = c1.z; c[7] = c1.w;
    }
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
        const int head = slot + i * args.slots;
        const bool exists = present && head < all_heads;
        const bool is_query = head < args.heads;
        const int which = head >= args.heads + args.kv_heads;
        float x[8], y[8];
        unpack_bf16x8(first[i], x);
        unpack_bf16x8(second[i], y);
        if (args.sine != nullptr && exists && which == 0) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {          // (the packed multiply and add would be contracted to one rounding)
                const float low = __fsub_rn(__fmul_rn(x[j], c[j]), __fmul_rn(y[j], s[j]));
                const float high = __fadd_rn(__fmul_rn(y[j], c[j]), __fmul_rn(x[j], s[j]));
                x[j] = low;
                y[j] = high;
            }
        }
        if (exists && is_query) {
            __nv_bfloat16* out = args.q_out + ((int64_t(b) * args.heads + head) * args.tokens + t) * D + lane * 8;
            *reinterpret_cast<uint4*>(out) = make_uint4(float2_to_bf16x2(make_float2(x[0], x[1])), float2_to_bf16x2(make_float2(x[2], x[3])),
                                                        float2_to_bf16x2(make_float2(x[4], x[5])), float2_to_bf16x2(make_float2(x[6], x[7])));
            *reinterpret_cast<uint4*>(out + HALF) = make_uint4(float2_to_bf16x2(make_float2(y[0], y[1])), float2_to_bf16x2(make_float2(y[2], y[3])),
                                                               float2_to_bf16x2(make_float2(y[4], y[5])), float2_to_bf16x2(make_float2(y[6], y[7])));
        }
        if (!__any_sync(0xffffffffu, exists && !is_query)) continue;      // a warp of queries only
        // the largest magnitude as bits: infinities and NaN order above every number
        uint32_t largest = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            largest = max(largest, __float_as_uint(x[j]) & 0x7fffffffu);
            largest = max(largest, __float_as_uint(y[j]) & 0x7fffffffu);
        }
#pragma unroll
        for (int step = LANES / 2; step > 0; step >>= 1) largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, step));
        if (!exists || is_query || position < 0) continue;
        const float amax = __uint_as_float(largest);
        float scale = __fdiv_rn(amax, 448.0f);
        if (amax < CACHE_TINY) scale = 0.0f;
        if (!(amax < CACHE_HUGE)) scale = __uint_as_float(0x7fc00000u);
        uint32_t codes[4] = {0u, 0u, 0u, 0u};
        if (scale != 0.0f) {
            const ExactDivider divide(scale);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float2 a = make_float2(x[2 * j], x[2 * j + 1]), d = make_float2(y[2 * j], y[2 * j + 1]);
                if (divide.fast) {
                    a = divide.unchecked2(a);
                    d = divide.unchecked2(d);
                } else {
                    a = make_float2(__fdiv_rn(a.x, scale), __fdiv_rn(a.y, scale));
                    d = make_float2(__fdiv_rn(d.x, scale), __fdiv_rn(d.y, scale));
                }
                codes[j >> 1] |= uint32_t(__nv_cvt_float2_to_fp8x2(a, __NV_SATFINITE, __NV_E4M3)) << (16 * (j & 1));
                codes[2 + (j >> 1)] |= uint32_t(__nv_cvt_float2_to_fp8x2(d, __NV_SATFINITE, __NV_E4M3)) << (16 * (j & 1));
            }
        }
        const int kv_head = head - args.heads - which * args.kv_heads;
        const int64_t row = (int64_t(b) * args.kv_heads + kv_head) * args.capacity + position;
        uint8_t* out = args.codes[which] + row * D + lane * 8;
        *reinterpret_cast<uint2*>(out) = make_uint2(codes[0], codes[1]);
        *reinterpret_cast<uint2*>(out + HALF) = make_uint2(codes[2], codes[3]);
        if (lane == 0) args.scales[which][row] = scale;
    }
}

// Two e4m3 codes -> two bf16 values of code * scale.
__device__ __forceinline__ uint32_t decode_pair(uint32_t codes, float scale) {
    const __half2 pair = __half2(__nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(codes & 0xffffu), __NV_E4M3));
    const float2 values = __half22float2(pair);
    return float2_to_bf16x2(make_float2(__fmul_rn(values.x, scale), __fmul_rn(values.y, scale)));
}

// ROWS rows per thread, a block's rows apart, all loads first; blockIdx.y: keys, values.
template <int D, int ROWS>
__global__ void __launch_bounds__(CACHE_THREADS) kv_cache_read_kernel(const __grid_constant__ CacheArgs args) {
    pdl_launch_dependents();
    pdl_wait();
    constexpr int LANES = D / 16, BLOCK_ROWS = CACHE_THREADS / LANES;
    const int which = int(blockIdx.y), lane = threadIdx.x % LANES;
    const uint32_t total = uint32_t(args.batch) * uint32_t(args.kv_heads) * uint32_t(args.tokens);
    uint4 codes[ROWS];
    float scale[ROWS];
    __nv_bfloat16* out[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const uint32_t row = (blockIdx.x * uint32_t(ROWS) + uint32_t(i)) * uint32_t(BLOCK_ROWS) + threadIdx.x / LANES;
        out[i] = nullptr;
        if (row >= total) continue;
        const uint32_t line = row / uint32_t(args.tokens);
        const int t = int(row - line * uint32_t(args.tokens));
        const int b = int(line / uint32_t(args.kv_heads)), head = int(line - uint32_t(b) * uint32_t(args.kv_heads));
        const int64_t position = cache_position(args, b, t);
        if (position < 0) continue;
        const int64_t source = int64_t(line) * args.capacity + position;
        codes[i] = ld_nc_u4(reinterpret_cast<const uint4*>(args.codes[which] + source * D + lane * 16));
        scale[i] = __ldg(args.scales[which] + source);
        out[i] = args.rows[which] + b * args.stride[which][0] + head * args.stride[which][1] + t * args.stride[which][2] + lane * 16;
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        if (out[i] == nullptr) continue;
        const uint32_t words[4] = {codes[i].x, codes[i].y, codes[i].z, codes[i].w};
        uint32_t values[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            values[2 * j] = decode_pair(words[j], scale[i]);
            values[2 * j + 1] = decode_pair(words[j] >> 16, scale[i]);
        }
        if (args.wide) {
            st_u8(out[i], values);
        } else {
            reinterpret_cast<uint4*>(out[i])[0] = make_uint4(values[0], values[1], values[2], values[3]);
            reinterpret_cast<uint4*>(out[i])[1] = make_uint4(values[4], values[5], values[6], values[7]);
        }
    }
}

CacheArgs cache_args(const b2_kv_cache_desc* d) {
    CacheArgs args{};
    args.q = static_cast<const __nv_bfloat16*>(d->q);
    args.q_out = static_cast<__nv_bfloat16*>(d->q_out);
    args.rows[0] = static_cast<__nv_bfloat16*>(d->k);
    args.rows[1] = static_cast<__nv_bfloat16*>(d->v);
    args.sine = static_cast<const float*>(d->sine);
    args.cosine = static_cast<const float*>(d->cosine);
    args.codes[0] = static_cast<uint8_t*>(d->k_codes);
    args.codes[1] = static_cast<uint8_t*>(d->v_codes);
    args.scales[0] = static_cast<float*>(d->k_scales);
    args.scales[1] = static_cast<float*>(d->v_scales);
    args.offsets = static_cast<const int32_t*>(d->offsets);
    args.lengths = static_cast<const int32_t*>(d->lengths);
    for (int i = 0; i < 3; ++i) {
        args.q_stride[i] = d->q_stride[i];
        args.stride[0][i] = d->k_stride[i];
        args.stride[1][i] = d->v_stride[i];
    }
    args.factor_batch_stride = d->factor_batch_stride;
    args.batch = d->batch;
    args.tokens = d->tokens;
    args.heads = d->q == nullptr ? 0 : d->heads;
    args.kv_heads = d->kv_heads;
    args.capacity = d->capacity;
    return args;
}

}  // namespace

int launch_kv_cache_write(const b2_kv_cache_desc* desc, cudaStream_t stream) {
    CacheArgs args = cache_args(desc);
    const int all_heads = args.heads + 2 * args.kv_heads;
    const int64_t lanes = desc->head_dim / 16, tokens = int64_t(args.batch) * args.tokens;
    // Four rows of a token per thread once that still leaves two blocks for every SM; single rows below that, where the
    // time is the latency of one load.
    const bool several = tokens * ((all_heads + 3) / 4) * lanes >= int64_t(sm_count()) * 2 * CACHE_THREADS;
    args.slots = several ? (all_heads + 3) / 4 : all_heads;
    const int64_t items = tokens * args.slots;
    const dim3 grid(unsigned((items * lanes + CACHE_THREADS - 1) / CACHE_THREADS)), block(CACHE_THREADS);
    if (desc->head_dim == 256)
        return several ? launch_kernel(kv_cache_write_kernel<256, 4>, grid, block, size_t(0), stream, args)
                       : launch_kernel(kv_cache_write_kernel<256, 1>, grid, block, size_t(0), stream, args);
    return several ? launch_kernel(kv_cache_write_kernel<128, 4>, grid, block, size_t(0), stream, args)
                   : launch_kernel(kv_cache_write_kernel<128, 1>, grid, block, size_t(0), stream, args);
}

int launch_kv_cache_read(const b2_kv_cache_desc* desc, cudaStream_t stream) {
    CacheArgs args = cache_args(desc);
    args.wide = ((reinterpret_cast<uintptr_t>(desc->k) | reinterpret_cast<uintptr_t>(desc->v)) & 31u) == 0;
    const int32_t extents[3] = {desc->batch, desc->kv_heads, desc->tokens};
    for (int i = 0; i < 3; ++i) args.wide = args.wide && (extents[i] == 1 || (desc->k_stride[i] | desc->v_stride[i]) % 16 == 0);
    const int64_t rows = int64_t(args.batch) * args.kv_heads * args.tokens;
    const int64_t block_rows = CACHE_THREADS / (desc->head_dim / 16);
    // as in the write: four rows per thread once the launch fills the device with them
    const bool several = rows >= block_rows * 4 * sm_count();
    const int64_t per_block = block_rows * (several ? 4 : 1);
    const dim3 grid(unsigned((rows + per_block - 1) / per_block), 2), block(CACHE_THREADS);
    if (desc->head_dim == 256)
        return several ? launch_kernel(kv_cache_read_kernel<256, 4>, grid, block, size_t(0), stream, args)
                       : launch_kernel(kv_cache_read_kernel<256, 1>, grid, block, size_t(0), stream, args);
    return several ? launch_kernel(kv_cache_read_kernel<128, 4>, grid, block, size_t(0), stream, args)
                   : launch_kernel(kv_cache_read_kernel<128, 1>, grid, block, size_t(0), stream, args);
}

}  // namespace b2
