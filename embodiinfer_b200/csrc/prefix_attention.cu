// Attention for a batch whose members share prefixes, each prefix computed once for all its members, over a bf16 cache or the
// quantised one (kv_cache.cu):
//
//   keys of member b of group g = prefix[g, :plen[g]] followed by own[b, :visible(b, t)]
//   out[b, h, t] = softmax(scale q[b, h, t] K^T) V,  0 where a row sees no key
//
// A group's members, the query heads of one key/value head and the queries are one matrix of rows (row = member, head, query):
// a CTA takes 128 of them and walks the prefix in tiles of 64 keys -- every key tile is loaded once for all 128 rows -- and then
// the own keys of the members its rows belong to, where the rows of the other members are masked.  The own part so spends tensor
// instructions on masked rows; it stays below the time of loading those keys, which nobody else needs.
//   warp 0        TMA producer: key and value tiles through rings
//   warp 1        tensor-memory owner and MMA issuer: S = Q K^T (128 x 64) and O += P V (128 x D), fp32 accumulators in tensor memory
//   warps 2-9     two softmax groups of 128 threads, one thread per row, for the even and the odd key tiles: scores, reference and
//                 sum, probabilities, output
//   warps 10..    what the value tile still needs before the tensor core may read it (see below)
// What bounds such a loop is shared memory: 128 bytes per cycle have to take the tiles from TMA and give them to the tensor core,
// and with Q and P there as well (128 rows of 32 bytes again for every 64 keys) they cost more than K and V themselves.  So Q lives
// in tensor memory as the first product's "A" operand, and P as the second one's:
// S of the even and odd tiles 2 x 64 columns, O D columns, Q and P the rest (D = 256: a quarter of Q stays in shared memory).
// The two softmax groups work a tile apart and pass one float per row: the running reference, which a group needs from the
// other only after it has the maximum of its own tile.  Every wait is bounded and reports through the status word.
//
// bf16 cache.  K and V are read as they lie in memory.  What the tensor core must not see is taken out of the value tile in
// shared memory, because a probability of zero times an infinity or a NaN is not zero: rows behind the end of a segment are set to
// zero, and so are values of own keys that are not finite (other members' rows, and earlier queries, pass over them with
// probability zero); the rows that do see such a key get NaN from their sum.
//
// Quantised cache (e4m3 codes, one fp32 scale per row: ks for keys, vs for values).
//   Scores.  The codes go to the tensor core as they are (kind::f8f6f4).  Q is split into two e4m3 operands, q 2^e = hi + lo with
//   2^e bringing the row's largest value into [128, 256): a bf16 value has 8 significant bits, hi takes 4 and lo the rest,
//   exactly, down to 2^-18 of the row's largest value.  Two products at twice the bf16 rate cost what one bf16 product
//   would, and no key is ever converted.  ks multiplies the score.
//   Output.  The four value warps turn the codes into f16 (exact: the code's bits shifted into place are the value times
//   2^-8).  vs cannot be divided out afterwards, so it joins the probability:
//       w = 2^(s + log2 vs - M),   O = sum w v,   L = sum w / vs,   out = O / L
//   with M the running reference of s + log2 vs: the weights that meet the values are at most 2^8, whatever the spread of the
//   scales, and f16 with its 11 bits is enough (bf16 probabilities would double the error of the result; two e4m3 halves, which
//   would spare the conversion of V, have no room for a long tail of weights 2^-15 below the largest).
//   A row whose scale is 0 holds zeros; it takes part in L alone, with a vs below every scale that the cache's write leaves
//   (2^-59 to 2^32), so that it never sets M.
//
// Few CTAs: the key tiles of a row tile are cut across `splits` CTAs, which leave O, M and L in fp32 in the workspace; a second
// launch joins them in split order (no atomics: the result does not depend on timing).
#include "gemm_epilogue.cuh"

#include <cuda.h>
#include <cuda_fp16.h>

namespace b2 {

namespace {

constexpr int PA_ROWS = 128;                     // query rows per CTA
constexpr int PA_KEYS = 64;                      // keys per tile
constexpr int PA_SOFTMAX_WARP = 2, PA_VALUE_WARP = 10;      // first softmax warp (of 8), first value warp
constexpr int PA_SCALE_STAGES = 4;
constexpr int PA_SCALE_FLOATS = 3 * PA_KEYS;     // ks, log2 vs, 1 / vs of a key tile
constexpr float PA_ZERO_ROW_SCALE = 8.6736173798840355e-19f;      // 2^-60
constexpr int PA_MAX_SEGMENTS = PA_ROWS + 1;     // the prefix and at most one member per row

template <int D, bool FP8>
struct PaShape {
    static constexpr int ELEMENT = FP8 ? 1 : 2;
    static constexpr int ROW_BYTES = D * ELEMENT;                           // of a cached row
    static constexpr int KV_ATOMS = ROW_BYTES / 128;                        // 128-byte column groups of a cached tile
    static constexpr uint32_t KV_ATOM_BYTES = PA_KEYS * 128;
    static constexpr uint32_t KV_BYTES = KV_ATOMS * KV_ATOM_BYTES;
    static constexpr int STAGES = D == 256 ? (FP8 ? 4 : 3) : (FP8 ? 8 : 6); // of the K and the V ring each
    static constexpr int VALUE_STAGES = FP8 ? 2 : 0;                        // converted value tiles
    static constexpr uint32_t VALUE_BYTES = PA_KEYS * D * 2;
    static constexpr int VALUE_WARPS = FP8 ? 4 : 2;
    static constexpr int WARPS = PA_VALUE_WARP + VALUE_WARPS + (FP8 ? 1 : 0);   // + the scale warp
    static constexpr int THREADS = WARPS * 32;
    // Q: atoms of 32 columns (64 bf16 or 128 e4m3 values of a row).  With D = 256 there is room for three of the four, and for one P;
    // the last atom of Q lies in shared memory.
    static constexpr int Q_ATOMS = D / 64, Q_TMEM_ATOMS = Q_ATOMS < 3 ? Q_ATOMS : 3, P_BUFFERS = D == 256 ? 1 : 2;
    static constexpr uint32_t TMEM_S = 0, TMEM_O = 2 * PA_KEYS, TMEM_Q = TMEM_O + D, TMEM_P = TMEM_Q + Q_TMEM_ATOMS * 32;
    static_assert(TMEM_P + P_BUFFERS * 32 <= TMEM_COLUMNS, "tensor memory");
    static constexpr uint32_t OFF_K = 0;
    static constexpr uint32_t OFF_V = OFF_K + STAGES * KV_BYTES;
    static constexpr uint32_t OFF_VALUES = OFF_V + STAGES * KV_BYTES;
    static constexpr uint32_t OFF_Q = OFF_VALUES + VALUE_STAGES * VALUE_BYTES;
    static constexpr uint32_t OFF_SCALES = OFF_Q + (Q_ATOMS - Q_TMEM_ATOMS) * PA_ROWS * 128;
    static constexpr uint32_t OFF_ROWS = OFF_SCALES + (FP8 ? PA_SCALE_STAGES * PA_SCALE_FLOATS * 4 : 0);      // float [2][128], twice
    static constexpr uint32_t OFF_SEGMENTS = OFF_ROWS + 4 * PA_ROWS * 4;
    static constexpr uint32_t OFF_BARS = OFF_SEGMENTS + (PA_MAX_SEGMENTS + 3) * 8;
    static constexpr int SHARED_BYTES = 1024 + int(OFF_BARS) + 768;
};

struct PaArgs {
    const __nv_bfloat16* q;
    __nv_bfloat16* out;               // [batch, heads, queries, D]
    const float* prefix_scales[2];    // keys, values [groups, kv_heads, prefix_capacity]
    const float* own_scales[2];       // [batch, kv_heads, own_capacity]
    const int32_t* members;           // [groups + 1] or nullptr: batch / groups each
    const int32_t* prefix_lengths;    // or nullptr: the capacity
    const int32_t* own_lengths;
    float* partial;                   // splits > 1: O [work][splits][128][D], then (M, L) [work][splits][128][2]
    int64_t* row_offsets;             // splits > 1: element offset of each row's output, -1 for rows that do not exist [work][128]
    unsigned int* status;
    int64_t q_stride[3];
    float scale_log2;
    int batch, groups, heads, kv_heads, queries, prefix_capacity, own_capacity;
    int rows_per_member, tiles, splits, causal;
};

// What a CTA works on, in shared memory: written by warp 0 before the block barrier.
struct PaWork {
    int group, first_member, member_count, row0, rows, segments, first_segment_member, key_tiles;
};

__device__ __forceinline__ int clamp_length(int value, int capacity) { return value < 0 ? 0 : (value > capacity ? capacity : value); }

__device__ __forceinline__ uint32_t pa_idesc_16bit(uint32_t m, uint32_t n, bool bf16, bool b_mn_major) {
    return (1u << 4) | (uint32_t(bf16) << 7) | (uint32_t(bf16) << 10) | (uint32_t(b_mn_major) << 16) | ((n >> 3) << 17) | ((m >> 4) << 24);
}

__device__ __forceinline__ uint64_t pa_desc_mn(uint32_t mn_group_bytes) {
    return (static_cast<uint64_t>(mn_group_bytes >> 4) << 16) | (static_cast<uint64_t>(1024 >> 4) << 32) | (static_cast<uint64_t>(1) << 46) |
           (static_cast<uint64_t>(2) << 61);
}

// D[tmem] (+)= A[tmem] B[smem]: A's row is the tensor-memory lane, 32-bit columns hold 2 (16-bit) or 4 (8-bit) consecutive K values.
template <bool EIGHT_BIT>
__device__ __forceinline__ void pa_mma(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    if (EIGHT_BIT)
        asm volatile(
            "{\n\t"
            ".reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], [%1], %2, %3, p;\n\t"
            "}\n"
            ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t"
            ".reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
            "}\n"
            ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
            : "memory");
}

// The same with A in shared memory.
template <bool EIGHT_BIT>
__device__ __forceinline__ void pa_mma_shared(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    if (EIGHT_BIT) {
        mma_f8f6f4(d_tmem, a_desc, b_desc, idesc, accumulate);
        return;
    }
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t"
        "}\n"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

__device__ __forceinline__ void pa_tmem_store(uint32_t address, const uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
        ::"r"(address), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
          "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]),
          "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]),
          "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
        : "memory");
}

__device__ __forceinline__ void pa_tmem_store16(uint32_t address, const uint32_t* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(address), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
          "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}

__device__ __forceinline__ void pa_tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float pa_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void sts_u4(uint32_t address, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(address), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

__device__ __forceinline__ uint4 lds_u4(uint32_t address) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(address) : "memory");
    return v;
}

__device__ __forceinline__ float4 lds_f4(uint32_t address) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(address) : "memory");
    return v;
}

__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ uint32_t float2_to_half2_bits(float a, float b) {
    const __half2 pair = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&pair);
}

// Two e4m3 codes in the low half of `codes` -> two f16 holding the values times 2^-8: sign to the top bit, the other seven
// bits under the f16 exponent's top bit (subnormal codes are subnormal halves).
__device__ __forceinline__ uint32_t codes_to_halves(uint32_t codes, uint32_t selector) {
    const uint32_t spread = __byte_perm(codes, 0u, selector);          // code 0 in byte 1, code 1 in byte 3
    return (spread & 0x80008000u) | ((spread & 0x7f007f00u) >> 1);
}

// Whether one of the two bf16 values of a word is an infinity or a NaN.
__device__ __forceinline__ bool has_not_finite(uint32_t word) {
    return (word & 0x7f80u) == 0x7f80u || (word & 0x7f800000u) == 0x7f800000u;
}

// Walks the key tiles of a CTA: the prefix (segment 0), then the own keys of its members.
struct PaCursor {
    const int* first_tile;      // [segments + 1], shared memory
    int segment, offset;        // offset: key tile inside the segment
    __device__ __forceinline__ PaCursor(const int* first, int segments, int tile) : first_tile(first), segment(0), offset(0) {
        int low = 0, high = segments;      // the last segment that starts at or before `tile`; empty ones are passed over
        while (high - low > 1) {
            const int middle = (low + high) >> 1;
            if (first[middle] <= tile) low = middle;
            else high = middle;
        }
        segment = low;
        offset = tile - first[low];
    }
    __device__ __forceinline__ void seek(int tile) {          // forward to `tile`, which exists
        while (first_tile[segment + 1] <= tile) ++segment;
        offset = tile - first_tile[segment];
    }
};

template <int D, bool FP8>
__global__ void __launch_bounds__(PaShape<D, FP8>::THREADS, 1)
prefix_attention_kernel(const __grid_constant__ CUtensorMap prefix_k_map, const __grid_constant__ CUtensorMap prefix_v_map,
                        const __grid_constant__ CUtensorMap own_k_map, const __grid_constant__ CUtensorMap own_v_map,
                        const __grid_constant__ PaArgs args) {
    using Shape = PaShape<D, FP8>;
    pdl_launch_dependents();
    extern __shared__ uint8_t shared_raw[];
    const uint32_t base = (smem_u32(shared_raw) + 1023u) & ~1023u;
    uint8_t* const generic = shared_raw + (base - smem_u32(shared_raw));
    const uint32_t k_smem = base + Shape::OFF_K, v_smem = base + Shape::OFF_V, values_smem = base + Shape::OFF_VALUES;
    const uint32_t q_smem = base + Shape::OFF_Q, scales_smem = base + Shape::OFF_SCALES;
    float* const row_reference = reinterpret_cast<float*>(generic + Shape::OFF_ROWS);           // [2][128]: of the latest even and odd tile
    float* const row_exchange = row_reference + 2 * PA_ROWS;                                    // [2][128]: row maxima of Q, then the sums
    int* const segment_first = reinterpret_cast<int*>(generic + Shape::OFF_SEGMENTS);
    int* const segment_length = segment_first + PA_MAX_SEGMENTS + 3;
    const uint32_t bars = base + Shape::OFF_BARS;
    constexpr int STAGES = Shape::STAGES;
    static_assert(STAGES <= 8, "barrier arrays");
    const uint32_t k_full = bars, k_empty = bars + 64, v_full = bars + 128, v_empty = bars + 192;        // [STAGES] each
    const uint32_t value_full = bars + 256, value_empty = bars + 320;      // converted tiles [2]; bf16: value_full [STAGES] = the tile may be read
    const uint32_t s_full = bars + 384, s_free = bars + 400, p_ready = bars + 416, o_done = bars + 432;      // [2]: even and odd tiles
    const uint32_t scale_full = bars + 448, scale_empty = bars + 480;      // [PA_SCALE_STAGES]
    const uint32_t reference_ready = bars + 512;                           // [4 quarters][2]
    const uint32_t all_done = bars + 576, q_ready = bars + 584, tmem_slot = bars + 592;
    PaWork* const work = reinterpret_cast<PaWork*>(generic + Shape::OFF_BARS + 608);
    unsigned long long* const bad_keys = reinterpret_cast<unsigned long long*>(generic + Shape::OFF_BARS + 640);      // bf16: [STAGES]

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // row tile fastest: CTAs that run together share the key tiles of their group in the L2
    const int tile = int(blockIdx.x) % args.tiles;
    const int kv_head = (int(blockIdx.x) / args.tiles) % args.kv_heads;
    const int split = int(blockIdx.x) / (args.tiles * args.kv_heads);

    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES; ++i) {
            mbar_init(k_full + 8 * i, 1);
            mbar_init(k_empty + 8 * i, 1);
            mbar_init(v_full + 8 * i, 1);
            mbar_init(v_empty + 8 * i, FP8 ? Shape::VALUE_WARPS : 1);
        }
        for (int i = 0; i < (FP8 ? 2 : STAGES); ++i) {
            mbar_init(value_full + 8 * i, Shape::VALUE_WARPS);
            mbar_init(value_empty + 8 * i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(s_full + 8 * i, 1);
            mbar_init(s_free + 8 * i, 4);
            mbar_init(p_ready + 8 * i, 4);
            mbar_init(o_done + 8 * i, 1);
        }
        for (int i = 0; i < PA_SCALE_STAGES; ++i) {
            mbar_init(scale_full + 8 * i, 1);
            mbar_init(scale_empty + 8 * i, 4);
        }
        for (int i = 0; i < 8; ++i) mbar_init(reference_ready + 8 * i, 1);
        mbar_init(all_done, 1);
        mbar_init(q_ready, 8);
        fence_barrier_init();
        tma_prefetch_descriptor(&prefix_k_map);
        tma_prefetch_descriptor(&prefix_v_map);
        tma_prefetch_descriptor(&own_k_map);
        tma_prefetch_descriptor(&own_v_map);
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, TMEM_COLUMNS);
        tmem_relinquish();
    }
    pdl_wait();
    if (warp == 0) {
        // ---- which rows, which keys
        int group = -1, first = 0, count = 0, group_tile = 0;
        if (args.members == nullptr) {
            count = args.batch / args.groups;
            const int per_group = (count * args.rows_per_member + PA_ROWS - 1) / PA_ROWS;
            group = tile / per_group;
            group_tile = tile - group * per_group;
            first = group * count;
        } else {
            int before = 0;
            for (int g0 = 0; g0 < args.groups && group < 0; g0 += 32) {
                const int g = g0 + lane;
                int a = 0, n = 0;
                if (g < args.groups) {
                    a = clamp_length(__ldg(args.members + g), args.batch);
                    n = clamp_length(__ldg(args.members + g + 1), args.batch) - a;
                    n = n < 0 ? 0 : n;
                }
                const int mine = (n * args.rows_per_member + PA_ROWS - 1) / PA_ROWS;
                int sum = mine;
#pragma unroll
                for (int step = 1; step < 32; step <<= 1) {
                    const int other = __shfl_up_sync(0xffffffffu, sum, step);
                    if (lane >= step) sum += other;
                }
                const unsigned hit = __ballot_sync(0xffffffffu, mine > 0 && tile >= before + sum - mine && tile < before + sum);
                if (hit != 0u) {
                    const int source = __ffs(int(hit)) - 1;
                    group = g0 + source;
                    first = __shfl_sync(0xffffffffu, a, source);
                    count = __shfl_sync(0xffffffffu, n, source);
                    group_tile = tile - before - __shfl_sync(0xffffffffu, sum - mine, source);
                }
                before += __shfl_sync(0xffffffffu, sum, 31);
            }
        }
        const int row0 = group_tile * PA_ROWS;
        int rows = group < 0 ? 0 : count * args.rows_per_member - row0;
        rows = rows < 0 ? 0 : (rows > PA_ROWS ? PA_ROWS : rows);
        const int first_own = row0 / args.rows_per_member;                      // first member with rows in this tile
        const int segments = rows == 0 ? 1 : (row0 + rows - 1) / args.rows_per_member - first_own + 2;
        int total = 0;
        for (int s0 = 0; s0 < segments; s0 += 32) {
            const int s = s0 + lane;
            int length = 0;
            if (rows > 0 && s < segments) {
                if (s == 0) {
                    length = args.prefix_lengths == nullptr ? args.prefix_capacity : clamp_length(__ldg(args.prefix_lengths + group), args.prefix_capacity);
                } else {
                    length = args.own_lengths == nullptr ? args.own_capacity
                                                         : clamp_length(__ldg(args.own_lengths + first + first_own + s - 1), args.own_capacity);
                }
            }
            const int mine = (length + PA_KEYS - 1) / PA_KEYS;
            int sum = mine;
#pragma unroll
            for (int step = 1; step < 32; step <<= 1) {
                const int other = __shfl_up_sync(0xffffffffu, sum, step);
                if (lane >= step) sum += other;
            }
            if (s < segments) {
                segment_first[s] = total + sum - mine;
                segment_length[s] = length;
            }
            total += __shfl_sync(0xffffffffu, sum, 31);
        }
        if (lane == 0) {
            segment_first[segments] = total;
            *work = PaWork{group, first, count, row0, rows, segments, first_own, total};
        }
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    uint32_t tmem_base;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem_base) : "r"(tmem_slot) : "memory");
    const PaWork w = *work;
    const int start_tile = int(int64_t(w.key_tiles) * split / args.splits);
    const int num_tiles = int(int64_t(w.key_tiles) * (split + 1) / args.splits) - start_tile;

    bool failed = false;
    if (warp == 0) {
        // ------------------------------------------------------------- TMA producer
        if (num_tiles > 0) {
            PaCursor cursor(segment_first, w.segments, start_tile);
            for (int j = 0; j < num_tiles; ++j) {
                cursor.seek(start_tile + j);
                const int b = j % STAGES;
                const uint32_t parity = uint32_t(j / STAGES) & 1u;
                const bool prefix = cursor.segment == 0;
                const CUtensorMap* k_map = prefix ? &prefix_k_map : &own_k_map;
                const CUtensorMap* v_map = prefix ? &prefix_v_map : &own_v_map;
                const int sequence = prefix ? w.group : w.first_member + w.first_segment_member + cursor.segment - 1;
                const int row = (sequence * args.kv_heads + kv_head) * (prefix ? args.prefix_capacity : args.own_capacity) + cursor.offset * PA_KEYS;
                mbar_wait(k_empty + 8 * b, parity ^ 1u, failed, args.status, STATUS_WAIT_PRODUCER);
                __syncwarp();
                if (elect_one()) {
                    mbar_expect_tx(k_full + 8 * b, Shape::KV_BYTES);
                    for (int a = 0; a < Shape::KV_ATOMS; ++a)
                        tma_load_2d(k_smem + b * Shape::KV_BYTES + a * Shape::KV_ATOM_BYTES, k_map, k_full + 8 * b, a * 128, row);
                }
                __syncwarp();
                mbar_wait(v_empty + 8 * b, parity ^ 1u, failed, args.status, STATUS_WAIT_PRODUCER);
                __syncwarp();
                if (elect_one()) {
                    mbar_expect_tx(v_full + 8 * b, Shape::KV_BYTES);
                    for (int a = 0; a < Shape::KV_ATOMS; ++a)
                        tma_load_2d(v_smem + b * Shape::KV_BYTES + a * Shape::KV_ATOM_BYTES, v_map, v_full + 8 * b, a * 128, row);
                }
                __syncwarp();
            }
            // every copy has landed before this CTA may leave (on the normal path the readers have long seen them)
            bool drain_failed = false;
            for (int b = 0; b < STAGES && b < num_tiles; ++b) {
                const int last = ((num_tiles - 1 - b) / STAGES) * STAGES + b;
                mbar_wait(k_full + 8 * b, uint32_t(last / STAGES) & 1u, drain_failed, args.status, STATUS_WAIT_DRAIN);
                mbar_wait(v_full + 8 * b, uint32_t(last / STAGES) & 1u, drain_failed, args.status, STATUS_WAIT_DRAIN);
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------- MMA issuer
        const uint32_t idesc_scores = FP8 ? idesc_f8(PA_ROWS, PA_KEYS) : pa_idesc_16bit(PA_ROWS, PA_KEYS, true, false);
        const uint32_t idesc_output = pa_idesc_16bit(PA_ROWS, D, !FP8, true);
        const uint64_t k_major = smem_desc_sw128(0), mn_major = pa_desc_mn(Shape::KV_ATOM_BYTES);
        const uint32_t k_low = uint32_t(k_major), k_high = uint32_t(k_major >> 32);
        const uint32_t mn_low = uint32_t(mn_major), mn_high = uint32_t(mn_major >> 32);
        auto field = [](uint32_t address) { return (address & 0x3FFFFu) >> 4; };
        if (num_tiles > 0) mbar_wait(q_ready, 0u, failed, args.status, STATUS_WAIT_MMA_FULL);
        tc_fence_after_sync();
        auto scores = [&](int j) {          // S[j & 1] = Q K_j^T
            const int b = j % STAGES, d = j & 1;
            mbar_wait(k_full + 8 * b, uint32_t(j / STAGES) & 1u, failed, args.status, STATUS_WAIT_MMA_FULL);
            mbar_wait(s_free + 8 * d, (uint32_t(j >> 1) & 1u) ^ 1u, failed, args.status, STATUS_WAIT_MMA_TMEM);
            tc_fence_after_sync();
            __syncwarp();
            if (elect_one()) {
                const uint32_t d_tmem = tmem_base + Shape::TMEM_S + uint32_t(d) * PA_KEYS;
                const uint32_t k_base = k_low + field(k_smem + b * Shape::KV_BYTES);
                // 32 bytes along K per instruction: 8 columns of Q.  Quantised: first all of hi, then all of lo.
#pragma unroll
                for (int a = 0; a < Shape::Q_ATOMS; ++a)
#pragma unroll
                    for (int s = 0; s < 4; ++s) {
                        const uint64_t k_desc = desc_from_words(k_base + (a % Shape::KV_ATOMS) * (Shape::KV_ATOM_BYTES >> 4) + 2 * s, k_high);
                        if (a < Shape::Q_TMEM_ATOMS) pa_mma<FP8>(d_tmem, tmem_base + Shape::TMEM_Q + uint32_t((a * 4 + s) * 8), k_desc, idesc_scores, (a | s) != 0);
                        else pa_mma_shared<FP8>(d_tmem, desc_from_words(k_low + field(q_smem) + 2 * s, k_high), k_desc, idesc_scores, 1u);
                    }
                tc_commit(k_empty + 8 * b);
                tc_commit(s_full + 8 * d);
            }
            __syncwarp();
        };
        auto output = [&](int j) {          // O += P V_j
            const int b = FP8 ? (j & 1) : j % STAGES, d = j & 1;
            const uint32_t parity = uint32_t(FP8 ? j >> 1 : j / STAGES) & 1u;
            mbar_wait(value_full + 8 * b, parity, failed, args.status, STATUS_WAIT_MMA_FULL);
            mbar_wait(p_ready + 8 * d, uint32_t(j >> 1) & 1u, failed, args.status, STATUS_WAIT_MMA_TMEM);
            // One output at a time: who has seen the output of tile j - 2 done can tell by its parity whether that of j - 1 is.  The
            // scores issued in between keep the tensor core busy.
            if (j > 0) mbar_wait(o_done + 8 * (d ^ 1), uint32_t((j - 1) >> 1) & 1u, failed, args.status, STATUS_WAIT_MMA_TMEM);
            tc_fence_after_sync();
            __syncwarp();
            if (elect_one()) {
                const uint32_t p_tmem = tmem_base + Shape::TMEM_P + uint32_t(d % Shape::P_BUFFERS) * 32;
                const uint32_t v_base = mn_low + field(FP8 ? values_smem + b * Shape::VALUE_BYTES : v_smem + b * Shape::KV_BYTES);
#pragma unroll
                for (int s = 0; s < PA_KEYS / 16; ++s)          // 16 keys per instruction: 8 columns of P, 16 rows (2048 bytes) of V
                    pa_mma<false>(tmem_base + Shape::TMEM_O, p_tmem + 8 * s, desc_from_words(v_base + s * (2048 >> 4), mn_high), idesc_output, (j | s) != 0);
                tc_commit((FP8 ? value_empty : v_empty) + 8 * b);
                tc_commit(o_done + 8 * d);
            }
            __syncwarp();
        };
        if (num_tiles > 0) scores(0);
        if (num_tiles > 1) scores(1);
        for (int j = 0; j < num_tiles; ++j) {
            if (j + 2 < num_tiles) scores(j + 2);          // as soon as its group has the scores of tile j in registers
            output(j);
        }
        if (num_tiles > 0 && elect_one()) tc_commit(all_done);
        __syncwarp();
    } else if (warp < PA_VALUE_WARP) {
        // ------------------------------------------------------------- one thread per query row and tile parity
        const int quarter = warp & 3, row = quarter * 32 + lane;          // row of the tile = tensor-memory lane
        const int parity_group = (warp - PA_SOFTMAX_WARP) >> 2;           // 0: even tiles, 1: odd tiles
        const uint32_t lane_address = tmem_base + (uint32_t(quarter * 32) << 16);
        const bool exists = row < w.rows;
        int my_segment = -1, hidden = 0;          // the segment of this row's own keys; causal: how many of them lie behind the query
        int64_t out_offset = -1;
        const __nv_bfloat16* query_row = args.q;
        if (exists) {
            const int member = (w.row0 + row) / args.rows_per_member, inside = w.row0 + row - member * args.rows_per_member;
            const int head_in_group = inside / args.queries, query = inside - head_in_group * args.queries;
            const int head = kv_head * (args.heads / args.kv_heads) + head_in_group;
            my_segment = member - w.first_segment_member + 1;
            hidden = args.causal ? args.queries - 1 - query : 0;
            out_offset = ((int64_t(w.first_member + member) * args.heads + head) * args.queries + query) * D;
            query_row += int64_t(w.first_member + member) * args.q_stride[0] + head * args.q_stride[1] + query * args.q_stride[2];
        }
        // ---- the queries into tensor memory: each group brings one half of the columns
        float factor = args.scale_log2;
        if (num_tiles > 0) {
            constexpr int WORDS = D / 4;          // 32-bit words of half a bf16 row
            uint32_t words[WORDS];
            const uint4* source = reinterpret_cast<const uint4*>(query_row + parity_group * (D / 2));
#pragma unroll
            for (int i = 0; i < WORDS / 4; ++i) {
                const uint4 v = exists ? source[i] : make_uint4(0, 0, 0, 0);
                words[4 * i] = v.x; words[4 * i + 1] = v.y; words[4 * i + 2] = v.z; words[4 * i + 3] = v.w;
            }
            // atom `a` of Q: 32 words of this row
            auto store_atom = [&](int a, const uint32_t* atom) {
                if (a < Shape::Q_TMEM_ATOMS) {
                    pa_tmem_store(lane_address + Shape::TMEM_Q + uint32_t(a) * 32, *reinterpret_cast<const uint32_t(*)[32]>(atom));
                    return;
                }
                const uint32_t line = q_smem + uint32_t(row >> 3) * 1024u + uint32_t(row & 7) * 128u;
#pragma unroll
                for (int c = 0; c < 8; ++c) sts_u4(line + uint32_t((c ^ (row & 7)) * 16), atom[4 * c], atom[4 * c + 1], atom[4 * c + 2], atom[4 * c + 3]);
                fence_async_shared();
            };
            if (!FP8) {
#pragma unroll
                for (int i = 0; i < WORDS / 32; ++i) store_atom(parity_group * (WORDS / 32) + i, words + 32 * i);
            } else {
                uint32_t largest = 0;      // bf16 magnitude bits: NaN and infinities order above numbers
#pragma unroll
                for (int i = 0; i < WORDS; ++i) largest = max(largest, max(words[i] & 0x7fffu, (words[i] >> 16) & 0x7fffu));
                row_exchange[parity_group * PA_ROWS + row] = __uint_as_float(largest);
                asm volatile("bar.sync 1, 256;" ::: "memory");
                largest = max(largest, __float_as_uint(row_exchange[(parity_group ^ 1) * PA_ROWS + row]));
                // 2^e that brings the largest magnitude into [128, 256), kept a normal number
                int exponent = int(largest >> 7) - 127;
                exponent = exponent < -110 ? -110 : (exponent > 120 ? 120 : exponent);
                const float up = largest == 0u ? 1.0f : __uint_as_float(uint32_t(127 + 7 - exponent) << 23);
                const float down = largest == 0u ? 1.0f : __uint_as_float(uint32_t(127 - 7 + exponent) << 23);
                // a row with an infinity or a NaN: every score is NaN
                factor = largest >= 0x7f80u ? __uint_as_float(0x7fc00000u) : args.scale_log2 * down;
                uint32_t high[WORDS / 2], low[WORDS / 2];
#pragma unroll
                for (int i = 0; i < WORDS; ++i) {
                    const float2 value = bf16x2_to_float2(words[i]);
                    const float2 scaled = make_float2(value.x * up, value.y * up);
                    const uint32_t h = __nv_cvt_float2_to_fp8x2(scaled, __NV_SATFINITE, __NV_E4M3);
                    const float2 back = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(h), __NV_E4M3)));
                    const uint32_t l = __nv_cvt_float2_to_fp8x2(make_float2(scaled.x - back.x, scaled.y - back.y), __NV_SATFINITE, __NV_E4M3);
                    high[i >> 1] = (i & 1) ? high[i >> 1] | (h << 16) : h;
                    low[i >> 1] = (i & 1) ? low[i >> 1] | (l << 16) : l;
                }
                if (D == 256) {          // the half row is one atom of hi and one of lo
                    store_atom(parity_group, high);
                    store_atom(2 + parity_group, low);
                } else {
                    pa_tmem_store16(lane_address + Shape::TMEM_Q + parity_group * 16, high);
                    pa_tmem_store16(lane_address + Shape::TMEM_Q + 32 + parity_group * 16, low);
                }
            }
            pa_tmem_store_wait();
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_ready);
        }
        float reference = -INFINITY, running_sum = 0.0f;          // of this group's tiles so far: the sum in units of 2^reference
        PaCursor cursor(segment_first, w.segments, start_tile);
        for (int j = parity_group; j < num_tiles; j += 2) {
            cursor.seek(start_tile + j);
            const uint32_t s_tmem = lane_address + Shape::TMEM_S + uint32_t(parity_group) * PA_KEYS;
            // keys of this tile that this row sees: the first `valid`
            int valid = 0;
            if (exists) {
                if (cursor.segment == 0) valid = segment_length[0] - cursor.offset * PA_KEYS;
                else if (cursor.segment == my_segment) valid = segment_length[cursor.segment] - hidden - cursor.offset * PA_KEYS;
            }
            const bool whole = __all_sync(0xffffffffu, valid >= PA_KEYS), none = __all_sync(0xffffffffu, valid <= 0);
            mbar_wait(s_full + 8 * parity_group, uint32_t(j >> 1) & 1u, failed, args.status, STATUS_WAIT_EPILOGUE);
            tc_fence_after_sync();
            uint32_t raw[2][32];
            const int stage = j % PA_SCALE_STAGES;
            const uint32_t tile_scales = scales_smem + uint32_t(stage) * PA_SCALE_FLOATS * 4;
            if (!none) {
                tmem_load_32x32(s_tmem, raw[0]);
                tmem_load_32x32(s_tmem + 32, raw[1]);
            }
            if (FP8) mbar_wait(scale_full + 8 * stage, uint32_t(j / PA_SCALE_STAGES) & 1u, failed, args.status, STATUS_WAIT_EPILOGUE);
            float tile_max = -INFINITY;
            if (!none) tmem_load_wait();
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(s_free + 8 * parity_group);
            if (!none) {
                if (FP8) {      // score in units of log2, + log2 vs
                    const float2 factor2 = make_float2(factor, factor);
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float4 ks = lds_f4(tile_scales + i * 16), lv = lds_f4(tile_scales + PA_KEYS * 4 + i * 16);
                        uint32_t* r = &raw[i >> 3][(i & 7) * 4];
                        const float2 a = __ffma2_rn(__fmul2_rn(make_float2(__uint_as_float(r[0]), __uint_as_float(r[1])), make_float2(ks.x, ks.y)), factor2, make_float2(lv.x, lv.y));
                        const float2 c = __ffma2_rn(__fmul2_rn(make_float2(__uint_as_float(r[2]), __uint_as_float(r[3])), make_float2(ks.z, ks.w)), factor2, make_float2(lv.z, lv.w));
                        r[0] = __float_as_uint(a.x); r[1] = __float_as_uint(a.y); r[2] = __float_as_uint(c.x); r[3] = __float_as_uint(c.y);
                    }
                }
                if (!whole) {
#pragma unroll
                    for (int i = 0; i < 64; ++i)
                        if (i >= valid) raw[i >> 5][i & 31] = __float_as_uint(-INFINITY);
                }
                float partial_max[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    partial_max[i & 3] = fmaxf(fmaxf(partial_max[i & 3], __uint_as_float(raw[0][i])), __uint_as_float(raw[1][i]));
                tile_max = fmaxf(fmaxf(partial_max[0], partial_max[1]), fmaxf(partial_max[2], partial_max[3]));
                if (!FP8) tile_max *= factor;
            }
            // The reference of the tile before comes from the other group.  It follows the maximum lazily: it moves only when the
            // maximum has grown by more than 2^8 since it was set, so weights stay below 2^8 and the accumulator is rescaled a few
            // times per row.  A row that has seen no key yet has none; 0 stands in, its weights are 0.
            float previous = -INFINITY;
            if (j > 0) {
                const int other = parity_group ^ 1;
                mbar_wait(reference_ready + 16 * quarter + 8 * other, uint32_t((j - 1) >> 1) & 1u, failed, args.status, STATUS_WAIT_EPILOGUE);
                previous = *static_cast<volatile float*>(row_reference + other * PA_ROWS + row);
            }
            const float now = tile_max > previous + 8.0f ? tile_max : previous;
            *static_cast<volatile float*>(row_reference + parity_group * PA_ROWS + row) = now;
            __syncwarp();
            if (lane == 0) mbar_arrive(reference_ready + 16 * quarter + 8 * parity_group);
            const float correction = now == previous ? 1.0f : pa_exp2(previous - now);
            if (now != reference) running_sum *= pa_exp2(reference - now);
            reference = now;
            uint32_t packed[32];
            if (none) {
#pragma unroll
                for (int i = 0; i < 32; ++i) packed[i] = 0u;
            } else {
                const float shift = now == -INFINITY ? 0.0f : -now;
                const float2 shift2 = make_float2(shift, shift);
                float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
                if (FP8) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float4 inverse = lds_f4(tile_scales + 2 * PA_KEYS * 4 + i * 16);
                        const uint32_t* r = &raw[i >> 3][(i & 7) * 4];
                        const float2 a = __fadd2_rn(make_float2(__uint_as_float(r[0]), __uint_as_float(r[1])), shift2);
                        const float2 c = __fadd2_rn(make_float2(__uint_as_float(r[2]), __uint_as_float(r[3])), shift2);
                        const float2 p = make_float2(pa_exp2(a.x), pa_exp2(a.y)), q = make_float2(pa_exp2(c.x), pa_exp2(c.y));
                        sum[0] = __ffma2_rn(p, make_float2(inverse.x, inverse.y), sum[0]);
                        sum[1] = __ffma2_rn(q, make_float2(inverse.z, inverse.w), sum[1]);
                        packed[2 * i] = float2_to_half2_bits(p.x, p.y);
                        packed[2 * i + 1] = float2_to_half2_bits(q.x, q.y);
                    }
                } else {
                    const float2 factor2 = make_float2(factor, factor);
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const float2 a = __ffma2_rn(make_float2(__uint_as_float(raw[i >> 4][2 * (i & 15)]), __uint_as_float(raw[i >> 4][2 * (i & 15) + 1])), factor2, shift2);
                        const float2 p = make_float2(pa_exp2(a.x), pa_exp2(a.y));
                        packed[i] = float2_to_bf16x2(p);
                        sum[i & 1] = __fadd2_rn(sum[i & 1], p);
                    }
                    if (cursor.segment > 0) {
                        mbar_wait(value_full + 8 * (j % STAGES), uint32_t(j / STAGES) & 1u, failed, args.status, STATUS_WAIT_EPILOGUE);
                        const unsigned long long seen = valid >= PA_KEYS ? ~0ull : valid <= 0 ? 0ull : (1ull << valid) - 1ull;
                        if ((*static_cast<volatile unsigned long long*>(bad_keys + j % STAGES) & seen) != 0ull) sum[0].x = __uint_as_float(0x7fc00000u);
                    }
                }
                running_sum += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
            }
            if (FP8) {
                __syncwarp();
                if (lane == 0) mbar_arrive(scale_empty + 8 * stage);
            }
            // the P that lies where this one goes has been read: that of the tile before, or of this group's last
            if (j >= Shape::P_BUFFERS) {
                const int last = j - Shape::P_BUFFERS;
                mbar_wait(o_done + 8 * (last & 1), uint32_t(last >> 1) & 1u, failed, args.status, STATUS_WAIT_EPILOGUE);
                tc_fence_after_sync();
            }
            pa_tmem_store(lane_address + Shape::TMEM_P + uint32_t(parity_group % Shape::P_BUFFERS) * 32, packed);      // 64 keys in 32 columns
            if (j > 0 && __any_sync(0xffffffffu, correction != 1.0f)) {
                // O holds the tiles before this one in units of the reference before: wait for the last of them
                if (Shape::P_BUFFERS > 1) mbar_wait(o_done + 8 * (parity_group ^ 1), uint32_t((j - 1) >> 1) & 1u, failed, args.status, STATUS_WAIT_EPILOGUE);
                tc_fence_after_sync();
#pragma unroll 1
                for (int chunk = 0; chunk < D / 32; ++chunk) {
                    uint32_t o[32];
                    tmem_load_32x32(lane_address + Shape::TMEM_O + chunk * 32, o);
                    tmem_load_wait();
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * correction);
                    pa_tmem_store(lane_address + Shape::TMEM_O + chunk * 32, o);
                }
            }
            pa_tmem_store_wait();
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_ready + 8 * parity_group);
        }
        // ---- the two groups' sums; the later reference is the one O is held in
        if (num_tiles > 0) {
            mbar_wait(all_done, 0u, failed, args.status, STATUS_WAIT_EPILOGUE);
            tc_fence_after_sync();
        }
        row_reference[parity_group * PA_ROWS + row] = reference;      // what the last tile of this group left there, or -inf
        row_exchange[parity_group * PA_ROWS + row] = running_sum;
        asm volatile("bar.sync 1, 256;" ::: "memory");
        {
            const float other_reference = row_reference[(parity_group ^ 1) * PA_ROWS + row], other_sum = row_exchange[(parity_group ^ 1) * PA_ROWS + row];
            const float last = fmaxf(reference, other_reference);
            if (other_reference != last) running_sum += other_sum * pa_exp2(other_reference - last);
            else if (reference != last) running_sum = running_sum * pa_exp2(reference - last) + other_sum;
            else running_sum += other_sum;
            reference = last;
        }
        // the codes reached the tensor core as values times 2^-8
        constexpr float UNIT = FP8 ? 256.0f : 1.0f;
        const int work_index = kv_head * args.tiles + tile;
        const int first_column = parity_group * (D / 2);          // each group stores half of the columns
        if (args.splits > 1) {
            const int64_t partial_row = (int64_t(work_index) * args.splits + split) * PA_ROWS + row;
            const int64_t total_rows = int64_t(args.tiles) * args.kv_heads * args.splits * PA_ROWS;
            if (parity_group == 0) {
                if (split == 0) args.row_offsets[int64_t(work_index) * PA_ROWS + row] = out_offset;
                if (exists) *reinterpret_cast<float2*>(args.partial + total_rows * D + partial_row * 2) = make_float2(reference, running_sum);
            }
            if (num_tiles > 0) {
                float* destination = args.partial + partial_row * D + first_column;
#pragma unroll 1
                for (int chunk = 0; chunk < D / 128; ++chunk) {
                    uint32_t o[2][32];
                    tmem_load_32x32(lane_address + Shape::TMEM_O + first_column + chunk * 64, o[0]);
                    tmem_load_32x32(lane_address + Shape::TMEM_O + first_column + chunk * 64 + 32, o[1]);
                    tmem_load_wait();
                    if (exists) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            uint32_t eight[8];
#pragma unroll
                            for (int v = 0; v < 8; ++v) eight[v] = __float_as_uint(__uint_as_float(o[i >> 2][(i & 3) * 8 + v]) * UNIT);
                            st_u8(destination + chunk * 64 + i * 8, eight);
                        }
                    }
                }
            }
        } else {
            // sum 0: the row sees no key
            const bool empty = running_sum == 0.0f;
            const float inverse = UNIT / running_sum;
#pragma unroll 1
            for (int chunk = 0; chunk < D / 128; ++chunk) {
                uint32_t o[2][32];
                if (num_tiles > 0) {
                    tmem_load_32x32(lane_address + Shape::TMEM_O + first_column + chunk * 64, o[0]);
                    tmem_load_32x32(lane_address + Shape::TMEM_O + first_column + chunk * 64 + 32, o[1]);
                    tmem_load_wait();
                }
                if (exists) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t words[8];
#pragma unroll
                        for (int v = 0; v < 8; ++v) {
                            const float a = __uint_as_float(o[i >> 1][(i & 1) * 16 + 2 * v]) * inverse;
                            const float c = __uint_as_float(o[i >> 1][(i & 1) * 16 + 2 * v + 1]) * inverse;
                            words[v] = empty ? 0u : float2_to_bf16x2(make_float2(a, c));
                        }
                        __nv_bfloat16* destination = args.out + out_offset + first_column + chunk * 64 + i * 16;
                        *reinterpret_cast<uint4*>(destination) = make_uint4(words[0], words[1], words[2], words[3]);
                        *reinterpret_cast<uint4*>(destination + 8) = make_uint4(words[4], words[5], words[6], words[7]);
                    }
                }
            }
        }
    } else if (!FP8) {
        // ------------------------------------------------------------- bf16: values the tensor core must not see
        if (num_tiles > 0) {
            constexpr int CHUNKS = Shape::KV_ATOMS * 8;          // 16-byte chunks of a row
            const int thread = (warp - PA_VALUE_WARP) * 32 + lane;
            PaCursor cursor(segment_first, w.segments, start_tile);
            for (int j = 0; j < num_tiles; ++j) {
                cursor.seek(start_tile + j);
                const int b = j % STAGES;
                mbar_wait(v_full + 8 * b, uint32_t(j / STAGES) & 1u, failed, args.status, STATUS_WAIT_PRODUCER);
                int valid = segment_length[cursor.segment] - cursor.offset * PA_KEYS;
                valid = valid < PA_KEYS ? valid : PA_KEYS;
                const uint32_t stage = v_smem + b * Shape::KV_BYTES;
                for (int i = valid * CHUNKS + thread; i < PA_KEYS * CHUNKS; i += 32 * Shape::VALUE_WARPS)
                    sts_u4(stage + uint32_t((i & (CHUNKS - 1)) >> 3) * Shape::KV_ATOM_BYTES + uint32_t(i / CHUNKS) * 128u + uint32_t(i & 7) * 16u, 0u, 0u, 0u, 0u);
                if (cursor.segment > 0) {
                    if (thread == 0) bad_keys[b] = 0ull;
                    asm volatile("bar.sync 2, %0;" ::"n"(32 * Shape::VALUE_WARPS) : "memory");
#pragma unroll 4
                    for (int i = thread; i < valid * CHUNKS; i += 32 * Shape::VALUE_WARPS) {
                        const int key = i / CHUNKS;
                        const uint32_t address = stage + uint32_t((i & (CHUNKS - 1)) >> 3) * Shape::KV_ATOM_BYTES + uint32_t(key) * 128u + uint32_t(i & 7) * 16u;
                        const uint4 v = lds_u4(address);
                        if (has_not_finite(v.x) || has_not_finite(v.y) || has_not_finite(v.z) || has_not_finite(v.w)) {
                            sts_u4(address, 0u, 0u, 0u, 0u);
                            atomicOr(bad_keys + b, 1ull << key);
                        }
                    }
                }
                fence_async_shared();
                __syncwarp();
                if (lane == 0) mbar_arrive(value_full + 8 * b);
            }
        }
    } else if (warp < PA_VALUE_WARP + Shape::VALUE_WARPS) {
        // ------------------------------------------------------------- codes of the value tile -> f16 operand
        // 16 codes of a key per thread and step: chunk `piece` of its row (stored at piece ^ (key % 8) inside its 128-byte group)
        // becomes two 16-byte chunks of the 64-column group they belong to.
        constexpr int PIECES = D / 16;
        const int thread = (warp - PA_VALUE_WARP) * 32 + lane;
        for (int j = 0; j < num_tiles; ++j) {
            const int b = j % STAGES, c = j & 1;
            mbar_wait(v_full + 8 * b, uint32_t(j / STAGES) & 1u, failed, args.status, STATUS_WAIT_PRODUCER);
            mbar_wait(value_empty + 8 * c, (uint32_t(j >> 1) & 1u) ^ 1u, failed, args.status, STATUS_WAIT_PRODUCER);
#pragma unroll 4
            for (int i = thread; i < PA_KEYS * PIECES; i += 32 * Shape::VALUE_WARPS) {
                const uint32_t key = uint32_t(i) / PIECES, piece = uint32_t(i) % PIECES, swizzle = key & 7u;
                const uint4 codes = lds_u4(v_smem + b * Shape::KV_BYTES + (piece >> 3) * Shape::KV_ATOM_BYTES + key * 128u + (((piece & 7u) ^ swizzle) << 4));
                const uint32_t group = values_smem + c * Shape::VALUE_BYTES + (piece >> 2) * Shape::KV_ATOM_BYTES + key * 128u;
                const uint32_t first = (piece & 3u) * 2u;
                const uint32_t a0 = codes_to_halves(codes.x, 0x1404), a1 = codes_to_halves(codes.x, 0x3424);
                const uint32_t a2 = codes_to_halves(codes.y, 0x1404), a3 = codes_to_halves(codes.y, 0x3424);
                const uint32_t b0 = codes_to_halves(codes.z, 0x1404), b1 = codes_to_halves(codes.z, 0x3424);
                const uint32_t b2 = codes_to_halves(codes.w, 0x1404), b3 = codes_to_halves(codes.w, 0x3424);
                sts_u4(group + ((first ^ swizzle) << 4), a0, a1, a2, a3);
                sts_u4(group + (((first + 1u) ^ swizzle) << 4), b0, b1, b2, b3);
            }
            fence_async_shared();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(v_empty + 8 * b);
                mbar_arrive(value_full + 8 * c);
            }
        }
    } else if (num_tiles > 0) {
        // ------------------------------------------------------------- scales of the key tile, loaded a tile ahead
        PaCursor cursor(segment_first, w.segments, start_tile);
        float ks[2], vs[2];
        auto load = [&](int j) {
            cursor.seek(start_tile + j);
            const bool prefix = cursor.segment == 0;
            const int sequence = prefix ? w.group : w.first_member + w.first_segment_member + cursor.segment - 1;
            const int64_t first = (int64_t(sequence) * args.kv_heads + kv_head) * (prefix ? args.prefix_capacity : args.own_capacity) + cursor.offset * PA_KEYS;
            const int valid = segment_length[cursor.segment] - cursor.offset * PA_KEYS;
            const float* key_scales = (prefix ? args.prefix_scales[0] : args.own_scales[0]) + first;
            const float* value_scales = (prefix ? args.prefix_scales[1] : args.own_scales[1]) + first;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const bool inside = lane + 32 * i < valid;
                ks[i] = inside ? __ldg(key_scales + lane + 32 * i) : 0.0f;
                vs[i] = inside ? __ldg(value_scales + lane + 32 * i) : 0.0f;
            }
        };
        load(0);
        for (int j = 0; j < num_tiles; ++j) {
            const int stage = j % PA_SCALE_STAGES;
            const float key_scale[2] = {ks[0], ks[1]}, value_scale[2] = {vs[0], vs[1]};
            if (j + 1 < num_tiles) load(j + 1);
            mbar_wait(scale_empty + 8 * stage, (uint32_t(j / PA_SCALE_STAGES) & 1u) ^ 1u, failed, args.status, STATUS_WAIT_PRODUCER);
            float* out = reinterpret_cast<float*>(generic + Shape::OFF_SCALES) + stage * PA_SCALE_FLOATS;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float value = value_scale[i] == 0.0f ? PA_ZERO_ROW_SCALE : value_scale[i];
                out[lane + 32 * i] = key_scale[i];
                out[PA_KEYS + lane + 32 * i] = log2f(value);
                out[2 * PA_KEYS + lane + 32 * i] = value == value ? 1.0f / value : 0.0f;      // NaN reaches the rows that see it by its logarithm
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(scale_full + 8 * stage);
        }
    }

    tc_fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc(tmem_base, TMEM_COLUMNS);
    }
}

// out = sum_s 2^(M_s - M) O_s / sum_s 2^(M_s - M) L_s in split order; one row per D / 8 lanes.
template <int D>
__global__ void __launch_bounds__(256) prefix_attention_join_kernel(const float* __restrict__ partial, const int64_t* __restrict__ row_offsets,
                                                                    __nv_bfloat16* __restrict__ out, int64_t rows, int splits) {
    pdl_launch_dependents();
    pdl_wait();
    constexpr int LANES = D / 8;
    const int64_t index = (int64_t(blockIdx.x) * 256 + threadIdx.x) / LANES;
    const int lane = threadIdx.x % LANES;
    if (index >= rows) return;
    const int64_t offset = row_offsets[index];
    if (offset < 0) return;
    const int64_t work = index / PA_ROWS, row = index - work * PA_ROWS;
    const float* statistics = partial + rows * splits * D;
    float top = -INFINITY;
    for (int s = 0; s < splits; ++s) top = fmaxf(top, statistics[((work * splits + s) * PA_ROWS + row) * 2]);
    const float reference = top == -INFINITY ? 0.0f : top;
    float total = 0.0f, sum[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int s = 0; s < splits; ++s) {
        const int64_t at = (work * splits + s) * PA_ROWS + row;
        const float2 entry = *reinterpret_cast<const float2*>(statistics + at * 2);
        const float weight = pa_exp2(entry.x - reference);
        if (entry.y == 0.0f) continue;      // no visible key in this split: O may not even have been written
        total = __fmaf_rn(weight, entry.y, total);
        const float4 a = *reinterpret_cast<const float4*>(partial + at * D + lane * 8), b = *reinterpret_cast<const float4*>(partial + at * D + lane * 8 + 4);
        const float values[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[i] = __fmaf_rn(weight, values[i], sum[i]);
    }
    const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
    *reinterpret_cast<uint4*>(out + offset + lane * 8) =
        make_uint4(float2_to_bf16x2(make_float2(sum[0] * inverse, sum[1] * inverse)), float2_to_bf16x2(make_float2(sum[2] * inverse, sum[3] * inverse)),
                   float2_to_bf16x2(make_float2(sum[4] * inverse, sum[5] * inverse)), float2_to_bf16x2(make_float2(sum[6] * inverse, sum[7] * inverse)));
}

struct PaPlan {
    int tiles = 0, splits = 1;
    int64_t bytes = 0;          // of workspace
};

PaPlan pa_plan(const b2_prefix_attention_desc* d) {
    PaPlan plan;
    const int64_t per_member = int64_t(d->heads / d->kv_heads) * d->queries;
    const int64_t per_group = d->batch / d->groups;
    // unequal groups (their bounds are device data): one partly filled tile per group more than the rows fill
    const int64_t tiles = d->members == nullptr ? d->groups * ((per_group * per_member + PA_ROWS - 1) / PA_ROWS)
                                                : d->batch * per_member / PA_ROWS + (d->groups < d->batch ? d->groups : d->batch);
    plan.tiles = int(tiles);
    // key tiles of a row tile: the prefix, and the own keys of the members that 128 rows can belong to
    int64_t sharing = (PA_ROWS + per_member - 2) / per_member + 1;
    if (d->members == nullptr && sharing > per_group) sharing = per_group;
    if (sharing > d->batch) sharing = d->batch;
    const int64_t key_tiles = (int64_t(d->prefix_capacity) + PA_KEYS - 1) / PA_KEYS + sharing * ((int64_t(d->own_capacity) + PA_KEYS - 1) / PA_KEYS);
    const int64_t work = tiles * d->kv_heads;
    const int64_t sms = sm_count();
    int64_t best = 0;
    for (int64_t splits = 1; splits <= 64 && splits <= key_tiles; ++splits) {
        // In units of a key tile's time: waves of CTAs times (set-up + tiles), and the join's second launch and traffic.
        const int64_t waves = (work * splits + sms - 1) / sms;
        const int64_t cost = waves * (4 + (key_tiles + splits - 1) / splits) * 64 + (splits > 1 ? 5 * 64 + work * splits * 64 / 100 : 0);
        if (best == 0 || cost < best) {
            best = cost;
            plan.splits = int(splits);
        }
    }
    if (plan.splits > 1) plan.bytes = work * PA_ROWS * (int64_t(plan.splits) * (d->head_dim + 2) * 4 + 8);
    return plan;
}

template <int D, bool FP8>
int pa_launch(const b2_prefix_attention_desc* d, const PaPlan& plan, PaArgs& args, cudaStream_t stream) {
    using Shape = PaShape<D, FP8>;
    static_assert(Shape::SHARED_BYTES <= 232448, "shared memory of a CTA");
    static bool configured[64] = {false};
    int device = 0;
    cudaGetDevice(&device);
    if (device < 0 || device >= 64 || !configured[device]) {
        const cudaError_t error = cudaFuncSetAttribute(prefix_attention_kernel<D, FP8>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::SHARED_BYTES);
        if (error != cudaSuccess) return int(error);
        if (device >= 0 && device < 64) configured[device] = true;
    }
    // a part that is not there is never read; its map describes the other part
    const bool has_prefix = d->prefix_capacity > 0, has_own = d->own_capacity > 0;
    const int64_t prefix_rows = int64_t(d->groups) * d->kv_heads * d->prefix_capacity, own_rows = int64_t(d->batch) * d->kv_heads * d->own_capacity;
    CUtensorMap prefix_k, prefix_v, own_k, own_v;
    if (has_prefix && (!make_operand_map(&prefix_k, d->prefix_k, prefix_rows, Shape::ROW_BYTES, PA_KEYS) ||
                       !make_operand_map(&prefix_v, d->prefix_v, prefix_rows, Shape::ROW_BYTES, PA_KEYS)))
        return B2_E_DRIVER;
    if (has_own && (!make_operand_map(&own_k, d->own_k, own_rows, Shape::ROW_BYTES, PA_KEYS) ||
                    !make_operand_map(&own_v, d->own_v, own_rows, Shape::ROW_BYTES, PA_KEYS)))
        return B2_E_DRIVER;
    if (!has_prefix) prefix_k = own_k, prefix_v = own_v;
    if (!has_own) own_k = prefix_k, own_v = prefix_v;
    const int64_t work = int64_t(plan.tiles) * d->kv_heads;
    const int status = launch_kernel(prefix_attention_kernel<D, FP8>, dim3(unsigned(work * plan.splits)), dim3(Shape::THREADS),
                                     size_t(Shape::SHARED_BYTES), stream, prefix_k, prefix_v, own_k, own_v, args);
    if (status != B2_OK || plan.splits == 1) return status;
    const int64_t rows = work * PA_ROWS;
    return launch_kernel(prefix_attention_join_kernel<D>, dim3(unsigned((rows * (D / 8) + 255) / 256)), dim3(256), size_t(0), stream,
                         static_cast<const float*>(args.partial), static_cast<const int64_t*>(args.row_offsets), args.out, rows, plan.splits);
}

}  // namespace

int64_t prefix_attention_workspace(const b2_prefix_attention_desc* desc) { return pa_plan(desc).bytes; }

int launch_prefix_attention(const b2_prefix_attention_desc* desc, cudaStream_t stream) {
    PaPlan plan = pa_plan(desc);
    if (plan.bytes > 0 && (desc->workspace == nullptr || desc->workspace_bytes < plan.bytes)) plan.splits = 1;
    if (int64_t(plan.tiles) * desc->kv_heads * plan.splits * PA_ROWS >= (int64_t(1) << 31)) return B2_E_TOO_LARGE;
    PaArgs args{};
    args.q = static_cast<const __nv_bfloat16*>(desc->q);
    args.out = static_cast<__nv_bfloat16*>(desc->out);
    args.prefix_scales[0] = static_cast<const float*>(desc->prefix_k_scales);
    args.prefix_scales[1] = static_cast<const float*>(desc->prefix_v_scales);
    args.own_scales[0] = static_cast<const float*>(desc->own_k_scales);
    args.own_scales[1] = static_cast<const float*>(desc->own_v_scales);
    args.members = static_cast<const int32_t*>(desc->members);
    args.prefix_lengths = static_cast<const int32_t*>(desc->prefix_lengths);
    args.own_lengths = static_cast<const int32_t*>(desc->own_lengths);
    if (plan.splits > 1) {
        const int64_t rows = int64_t(plan.tiles) * desc->kv_heads * PA_ROWS;
        args.row_offsets = static_cast<int64_t*>(desc->workspace);
        args.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(desc->workspace) + rows * 8);
    }
    args.status = static_cast<unsigned int*>(desc->status);
    for (int i = 0; i < 3; ++i) args.q_stride[i] = desc->q_stride[i];
    args.scale_log2 = desc->scale * 1.4426950408889634f;
    args.batch = desc->batch;
    args.groups = desc->groups;
    args.heads = desc->heads;
    args.kv_heads = desc->kv_heads;
    args.queries = desc->queries;
    args.prefix_capacity = desc->prefix_capacity;
    args.own_capacity = desc->own_capacity;
    args.rows_per_member = desc->heads / desc->kv_heads * desc->queries;
    args.tiles = plan.tiles;
    args.splits = plan.splits;
    args.causal = (desc->flags & B2_ATTENTION_CAUSAL) != 0;
    if (desc->head_dim == 256)
        return desc->cache_bits == 8 ? pa_launch<256, true>(desc, plan, args, stream) : pa_launch<256, false>(desc, plan, args, stream);
    return desc->cache_bits == 8 ? pa_launch<128, true>(desc, plan, args, stream) : pa_launch<128, false>(desc, plan, args, stream);
}

}  // namespace b2
