// Attention for a batch whose members share prefixes, each prefix computed once for all its members, over a bf16 cache or the
// quantised one (kv_cache.cu):
//
//   keys of member b of group g = prefix[g, :plen[g]] followed by own[b, :visible(b, t)]
//   out[b, h, t] = softmax(scale q[b, h, t] K^T) V,  0 where a row sees no key
//
// A group's members, the query heads of one key/value head and the queries are one matrix of rows (row = member, head, query):
// a CTA takes 128 of them and walks the prefix in tiles of 64 keys -- every key tile is loaded once for all 128 rows -- and then
// the own keys of the members its rows belong to, where the rows of the other members are masked.  An own key tile so costs as much as a
// prefix tile, whatever part of the 128 rows sees it: 2 of a row tile's 11 key tiles for ten-query chunks, 151 of 663 for single tokens behind
// 32768 keys with 4 rows and up to 512 own keys per member.
//   warps 0-7     two softmax groups of 128 threads, one thread per row, for the even and the odd key tiles: queries into tensor memory,
//                 scores, reference and sum, probabilities, output
//   warp 8        which rows and keys; TMA producer: key and value tiles through rings
//   warps 9, 10   issuers of S = Q K^T (128 x 64) and of O += P V (128 x D), fp32 accumulators in tensor memory
//   warp 11       the scales of a quantised cache
//   warps 12-15   what the value tile still needs before the tensor core may read it (see below)
// Shared memory has 128 bytes per cycle to take the tiles from TMA and give them to the tensor core; with Q and P there as well (128
// rows of 32 bytes again for every 64 keys) they would cost more than K and V themselves.  So Q lives in tensor memory as the first
// product's "A" operand, and P as the second one's.  D = 128: S of the even and odd tiles 2 x 64 columns, an accumulator for each
// group 2 x 128, Q 64, P 2 x 32: the groups meet at the end only.  D = 256: S 2 x 64, one accumulator 256, three quarters of Q 96 (the
// last one in shared memory), one P 32: the groups work a tile apart and pass one float per row, the running reference, which a group
// needs from the other only after it has the maximum of its own tile.  Every wait is bounded and reports through the status word.
//
// Measured (B200; a tile is 64 keys for 128 rows, whose products alone are 500 cycles at D = 128 and 1000 at D = 256):
//   fifty-query chunks of 64 members over 4 x 8192 bf16 keys, D = 256: 188 us (1150 TFLOP/s), 1430 cycles per tile
//   64 members, one query, 32768 quantised keys, D = 128: 79 us, 1350 cycles per tile; of an earlier 83 without its exponentials 74,
//   without its products 78, without the conversion of values 74: the chain of a softmax group -- scores out, maximum, exponentials, P in, each with
//   its latency and two warps per scheduler to hide it -- and not one unit is what bounds the loop
//   256 ten-query chunks over 32 x 712 quantised keys, D = 256: 42 us (in the groups' order 44): 176 row tiles of 12 key tiles on 148
//   SMs, 21 k of a CTA's 41 k cycles before and behind the loop (4.8 k look-up, 3.6 k splitting Q, 5 k output)
//   four ten-query chunks over 560 bf16 keys, D = 256: 13.6 us, 9 in this kernel for two tiles per CTA, the rest the join (b2_attention, one cluster
//   launch over a copy of the keys for each chunk: 8.0 us)
// The quantised D = 128 kernel spills 40 bytes per thread, the others 12.
//
// bf16 cache.  K and V are read as they lie in memory.  What the tensor core must not see is taken out of the value tile in
// shared memory, because a probability of zero times an infinity or a NaN is not zero: rows behind the end of a segment are set to
// zero, and so are values of own keys that are not finite (other members' rows, and earlier queries, pass over them with
// probability zero); the rows that do see such a key get NaN from their sum.
//
// Quantised cache (e4m3 codes, one fp32 scale per row: ks for keys, vs for values).
//   Scores.  The codes go to the tensor core as they are (kind::f8f6f4).  Q is split into two e4m3 operands, q 2^e = hi + lo with
//   2^e bringing the row's largest value into [128, 256): a bf16 value has 8 significant bits, hi takes 4 and lo the rest,
//   exactly, down to 2^-17 of the row's largest value (of 2^-119 in a row of smaller ones).  Two products at twice the bf16 rate cost what one
//   bf16 product would, and no key is ever converted.  ks multiplies the score.
//   Output.  The four value warps, two teams a tile apart, turn the codes into f16, exactly, and multiply by vs 2^-E: one rounding of 2^-11 for the scale and
//   one for the product, beside the 2^-8 of the result.  2^E is the unit of the accumulator, the same for all rows: it follows the
//   largest vs of a key tile when that leaves [2^-3, 2^6) units (2^-48 is the smallest), and the accumulator is rescaled then as it is for a
//   new reference.
//   A value is so off by at most 2^-10 of itself and, f16 ending at 2^-24 units, 2^-22 of the largest in its tile of 64 keys, whatever
//   other tiles hold.  P is f16 as well, down to 2^-31 of the reference's weight: with its 11 bits the result is as exact as its own rounding
//   allows (bf16 probabilities would add as much error again; two e4m3 halves, which would spare the conversion of V, have no room for a long
//   tail of weights 2^-15 below the largest).
//   A scale that is not finite zeroes its row of values and marks the key: rows that see it get NaN from their sum.  So do rows that see an
//   own key with a NaN among its codes: those codes are zeroed as they are converted, and the first such key of each member is kept to the end.
//
// Row tiles that do not fill the device -- all of a small call's, or those of the last, partial wave -- have their key tiles cut across
// several CTAs, which leave O, M and L in fp32 in the workspace; a second launch joins them in their order (no atomics: the result does
// not depend on timing).  The host bounds the row tiles and sizes the launch; how many there are, and so the cut, each CTA works out
// from the groups' bounds on the device.
#include "gemm_epilogue.cuh"

#include <cuda.h>
#include <cuda_fp16.h>

#include <climits>
#include <type_traits>

namespace b2 {

namespace {

constexpr int PA_ROWS = 128;                     // query rows per CTA
constexpr int PA_KEYS = 64;                      // keys per tile
constexpr int PA_LOAD_WARP = 8, PA_SCORES_WARP = 9, PA_OUTPUT_WARP = 10, PA_SCALE_WARP = 11, PA_VALUE_WARP = 12, PA_WARPS = 16;      // 0-7: softmax
// Registers per thread: 128 at launch (512 threads); the softmax warpgroups take what the others give up (168 / 88: 84 us for the 32768 keys).
constexpr int PA_SOFTMAX_REGISTERS = 184, PA_OTHER_REGISTERS = 72;
static_assert(256 * PA_SOFTMAX_REGISTERS + (PA_WARPS * 32 - 256) * PA_OTHER_REGISTERS <= PA_WARPS * 32 * 128, "registers of the launch");
constexpr uint32_t PA_PATIENCE = 1400000000u;     // cycles of a wait
constexpr int PA_SCALE_STAGES = 4, PA_RAW_STAGES = 8;      // of the quantised cache's scales: as the softmax reads them; as they come
// A key tile's scales as the roles read them: ks, vs in units as pairs of halves, then bits of keys whose vs is not finite (2 words), the
// unit, and the unit of the tile before less this one (exponents).
constexpr int PA_SCALE_FLOATS = 2 * PA_KEYS + 4;
// Weights and their sums are held 2^7 times as large where P is f16 (they stay below 2^15): its smallest number, 2^-24, is then 2^-31 of the
// reference's weight, and a tail of 2^19 keys with weights of 2^-25 each, a hundredth of the sum, is there.  bf16 has fp32's range.
template <bool FP8>
constexpr float PA_WEIGHT_BITS = FP8 ? 7.0f : 0.0f;
constexpr int PA_UNIT_LEAST = -48;               // the smallest unit of the values, as an exponent
constexpr uint32_t PA_SCALE_END = 0x4f800000u;   // 2^32: value scales from here on, which no write leaves, count as not finite; f16 could not hold them in any unit
constexpr int PA_MAX_SEGMENTS = PA_ROWS + 1;     // the prefix and at most one member per row

template <int D, bool FP8>
struct PaShape {
    static constexpr int ELEMENT = FP8 ? 1 : 2;
    static constexpr int ROW_BYTES = D * ELEMENT;                           // of a cached row
    static constexpr int KV_ATOMS = ROW_BYTES / 128;                        // 128-byte column groups of a cached tile
    static constexpr uint32_t KV_ATOM_BYTES = PA_KEYS * 128;
    static constexpr uint32_t KV_BYTES = KV_ATOMS * KV_ATOM_BYTES;
    static constexpr int STAGES = D == 256 ? (FP8 ? 4 : 3) : (FP8 ? 8 : 6); // of the K and the V ring each
    static constexpr int FREE_V_STAGES = FP8 ? STAGES : STAGES - int(PA_ROWS * D * 2 / KV_BYTES);      // of V: not under the queries as they come in
    static constexpr int VALUE_STAGES = FP8 ? 2 : 0;                        // converted value tiles
    static constexpr uint32_t VALUE_BYTES = PA_KEYS * D * 2;
    static constexpr int VALUE_WARPS = 4, VALUE_TEAM = FP8 ? 2 : 4;         // warps that prepare a value tile: quantised, two teams a tile apart
    static constexpr int THREADS = PA_WARPS * 32;
    // With D = 128 each softmax group has an accumulator of its own and never meets the other before the end; with D = 256 there is
    // room for one accumulator and one P, and for three of Q's four atoms (32 columns: 64 bf16 or 128 e4m3 values of a row): the last one
    // lies in shared memory.
    static constexpr bool SHARED = D == 256;
    static constexpr int Q_ATOMS = D / 64, Q_TMEM_ATOMS = Q_ATOMS < 3 ? Q_ATOMS : 3, P_BUFFERS = SHARED ? 1 : 2, O_BUFFERS = SHARED ? 1 : 2;
    static constexpr uint32_t TMEM_S = 0, TMEM_O = 2 * PA_KEYS, TMEM_Q = TMEM_O + O_BUFFERS * D, TMEM_P = TMEM_Q + Q_TMEM_ATOMS * 32;
    static_assert(TMEM_P + P_BUFFERS * 32 <= TMEM_COLUMNS, "tensor memory");
    static_assert(PA_ROWS * (D * 4 + 16) <= 2 * STAGES * KV_BYTES + VALUE_STAGES * VALUE_BYTES, "room of the output's rows");
    static constexpr uint32_t OFF_K = 0;
    static constexpr uint32_t OFF_V = OFF_K + STAGES * KV_BYTES;
    static constexpr uint32_t OFF_VALUES = OFF_V + STAGES * KV_BYTES;
    static constexpr uint32_t OFF_Q = OFF_VALUES + VALUE_STAGES * VALUE_BYTES;
    static constexpr uint32_t OFF_SCALES = OFF_Q + (Q_ATOMS - Q_TMEM_ATOMS) * PA_ROWS * 128;
    static constexpr uint32_t OFF_RAW_SCALES = OFF_SCALES + (FP8 ? PA_SCALE_STAGES * PA_SCALE_FLOATS * 4 : 0);
    static constexpr uint32_t OFF_ROWS = OFF_RAW_SCALES + (FP8 ? PA_RAW_STAGES * 2 * PA_KEYS * 4 : 0);      // float [2][128], twice
    static constexpr uint32_t OFF_ROW_OFFSETS = OFF_ROWS + 4 * PA_ROWS * 4;          // int64 [2][128]
    static constexpr uint32_t OFF_SEGMENTS = OFF_ROW_OFFSETS + 2 * PA_ROWS * 8;
    static constexpr uint32_t OFF_BARS = OFF_SEGMENTS + (PA_MAX_SEGMENTS + 3) * (FP8 ? 12 : 8);
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
    float* partial;                   // O [slots][128][D], then (M, L) [slots][128][2]
    int64_t* row_offsets;             // of the row tiles that are cut: element offset of each row's output, + 1 if it sees a key; -1 for rows that do not
                                      // exist [slots / 2][128]
    int32_t* cut;                     // [2], 8-byte aligned: how many row tiles are cut, and into how many parts each
    unsigned int* status;
    int64_t q_stride[3];
    float scale_log2;
    int batch, groups, heads, kv_heads, queries, prefix_capacity, own_capacity;
    int rows_per_member, sms, slots, max_splits, causal, share;      // share: query heads of a key/value head; slots: CTAs that may leave partial rows; 0 = nothing is cut
};

// What a CTA works on, in shared memory: written by warp 0 before the block barrier.
struct PaWork {
    int group, first_member, row0, rows, segments, first_segment_member, key_tiles;
    int kv_head, split, splits, place;      // place: among the row tiles that are cut, and in all of their parts (split * row tiles + it)
};

// a / b for a >= 0, b > 0.  Below 2^21 the fp32 quotient (2 steps of 2^-23 off at most) is within one of it and takes a quarter of an integer
// division's time; the look-up is a chain of them.
__device__ __forceinline__ int pa_divide(int a, int b) {
    if (a >= 1 << 21) return a / b;
    int q = int(__fdividef(float(a), float(b)));
    const int r = a - q * b;
    q += r < 0 ? -1 : r >= b ? 1 : 0;
    return q;
}

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

// Nothing that uses `v` is moved ahead of this place.
__device__ __forceinline__ void pa_tie(uint32_t (&v)[32]) {
    asm volatile(""
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]),
                   "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]), "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]),
                   "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31]));
}

// The loads issued so far have arrived, `v`'s among them.
__device__ __forceinline__ void pa_tmem_load_wait(uint32_t (&v)[32]) {
    tmem_load_wait();
    pa_tie(v);
}

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

template <int ID, int THREADS>
__device__ __forceinline__ void named_barrier() {
    __syncwarp();
    __barrier_sync_count(ID, THREADS);
}

__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ uint32_t float2_to_half2_bits(float a, float b) {
    const __half2 pair = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&pair);
}

// Two e4m3 codes in the low half of `codes` -> two f16 of the values times `scale`.
__device__ __forceinline__ uint32_t codes_to_halves(uint32_t codes, __half2 scale) {
    const __half2 value = __hmul2(__half2(__nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(codes), __NV_E4M3)), scale);
    return *reinterpret_cast<const uint32_t*>(&value);
}

// The bytes of `codes` that are e4m3 NaN (all magnitude bits set), as their top bits.
__device__ __forceinline__ uint32_t codes_not_a_number(uint32_t codes) { return ((codes & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// Whether one of the two bf16 values of a word is an infinity or a NaN.
__device__ __forceinline__ bool has_not_finite(uint32_t word) {
    return (word & 0x7f80u) == 0x7f80u || (word & 0x7f800000u) == 0x7f800000u;
}

// Bounded wait, as small as it can be made: the roles' loops have to share the instruction caches.  `patience` is its limit in cycles (0.7
// seconds or more); once a wait has run out it stays 0, every later wait of the thread gives up at once, and the role reports it when it ends.
__device__ __forceinline__ void pa_wait(uint32_t bar, uint32_t parity, uint32_t& patience) {
    if (mbar_try_wait(bar, parity)) return;
    const uint32_t start = uint32_t(clock());
    while (!mbar_try_wait(bar, parity))
        if (uint32_t(clock()) - start >= patience) {
            patience = 0;
            break;
        }
}

// Walks the key tiles of a CTA: the prefix (segment 0), then the own keys of its members.
struct PaCursor {
    const int* first_tile;      // [segments + 1], shared memory
    const int* length;          // [segments]
    int segment, start, end, keys_left;      // of the segment: its tiles and the keys from its tile `start` on
    __device__ __forceinline__ PaCursor(const int* first, const int* lengths, int tile) : first_tile(first), length(lengths), segment(-1), start(0), end(-1), keys_left(0) {
        seek(tile);
    }
    __device__ __forceinline__ void seek(int tile) {          // forward to `tile`; empty segments are passed over
        while (tile >= end) {
            ++segment;
            start = first_tile[segment];
            end = first_tile[segment + 1];
            keys_left = length[segment];
        }
    }
    __device__ __forceinline__ int first_key(int tile) const { return (tile - start) * PA_KEYS; }
    __device__ __forceinline__ int keys(int tile) const {          // of this tile: 1 to PA_KEYS
        const int left = keys_left - first_key(tile);
        return left < PA_KEYS ? left : PA_KEYS;
    }
};

// A place in a ring of slots and the parity of its current use.
template <int SLOTS>
struct PaRing {
    int slot = 0;
    uint32_t parity = 0;
    __device__ __forceinline__ void next() {
        if (++slot == SLOTS) {
            slot = 0;
            parity ^= 1u;
        }
    }
    __device__ __forceinline__ void next(int count) {
        for (int i = 0; i < count; ++i) next();
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
    // the queries come in where the values, or the last value tiles, will lie
    const uint32_t q_smem = base + Shape::OFF_Q, staging_smem = FP8 ? values_smem : v_smem + Shape::FREE_V_STAGES * Shape::KV_BYTES;
    int64_t* const row_query = reinterpret_cast<int64_t*>(generic + Shape::OFF_ROW_OFFSETS);          // [128]: element offset of a row's query, -1: no row
    int64_t* const row_output = row_query + PA_ROWS;                                                  // [128]: of its output
    float* const row_reference = reinterpret_cast<float*>(generic + Shape::OFF_ROWS);           // [2][128]: of the latest even and odd tile
    float* const row_exchange = row_reference + 2 * PA_ROWS;                                    // [2][128]: row maxima of Q, then the sums
    int* const group_unit = reinterpret_cast<int*>(generic + Shape::OFF_BARS + 728);          // [2]: last units of the accumulators, as exponents
    int* const segment_first = reinterpret_cast<int*>(generic + Shape::OFF_SEGMENTS);
    int* const segment_length = segment_first + PA_MAX_SEGMENTS + 3;
    int* const segment_nan = segment_length + PA_MAX_SEGMENTS + 3;          // quantised: first of its own keys here whose value has a code that is NaN
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
    unsigned long long* const bad_keys = reinterpret_cast<unsigned long long*>(generic + Shape::OFF_BARS + 664);      // bf16: [STAGES]
    static_assert(sizeof(PaWork) <= 664 - 608 && 664 + STAGES * 8 <= 728, "places behind the barriers");

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (warp == 0) {          // one lane per barrier (8 bytes each, in the order above); unused places of the arrays are barriers too
        for (int i = lane; i < 74; i += 32) {
            int count = 1;
            if (i >= 24 && i < 32 && FP8) count = Shape::VALUE_TEAM;                  // v_empty
            else if (i >= 32 && i < 40) count = Shape::VALUE_TEAM;                    // value_full
            else if (i >= 50 && i < 54) count = 4;                                    // s_free, p_ready
            else if (i >= 60 && i < 64) count = 4 + Shape::VALUE_TEAM;                // scale_empty
            else if (i == 73) count = 8;                                              // q_ready
            mbar_init(bars + 8 * i, count);
        }
        fence_barrier_init();
    }
    if (threadIdx.x == 32) {
        tma_prefetch_descriptor(&prefix_k_map);
        tma_prefetch_descriptor(&prefix_v_map);
        tma_prefetch_descriptor(&own_k_map);
        tma_prefetch_descriptor(&own_v_map);
    }
    if (warp == PA_SCORES_WARP) {
        tmem_alloc(tmem_slot, TMEM_COLUMNS);
        tmem_relinquish();
    }
    pdl_wait();
    if (warp == PA_LOAD_WARP) {
        // ---- which rows, which keys
        int group = -1, first = 0, count = 0, group_tile = 0;
        auto group_members = [&](int g, int& a) {
            a = clamp_length(__ldg(args.members + g), args.batch);
            const int n = clamp_length(__ldg(args.members + g + 1), args.batch) - a;
            return n < 0 ? 0 : n;
        };
        auto row_tiles = [&](int n) { return (n * args.rows_per_member + PA_ROWS - 1) / PA_ROWS; };
        auto inclusive_sum = [&](int sum) {
#pragma unroll
            for (int step = 1; step < 32; step <<= 1) {
                const int other = __shfl_up_sync(0xffffffffu, sum, step);
                if (lane >= step) sum += other;
            }
            return sum;
        };
        constexpr int MANY = 1 << 29;          // bounds that run backwards may add up to anything: enough for every CTA
        int total_tiles = 0;
        // More row tiles than SMs: the longest prefixes first, so that the last wave is made of short ones (as far as a warp sees all groups: up
        // to 32 of them; more are taken in their own order).
        const bool sorted = args.prefix_lengths != nullptr && args.groups <= 32 && int(gridDim.x) > args.sms;
        int group_at = lane;          // sorted: the group at this place
        if (sorted) {
            const int length = lane < args.groups ? clamp_length(__ldg(args.prefix_lengths + lane), args.prefix_capacity) : -1;
            int rank = 0;
#pragma unroll 8
            for (int other = 0; other < 32; ++other) {
                const int its = __shfl_sync(0xffffffffu, length, other);
                rank += its > length || (its == length && other < lane);
            }
            segment_first[rank] = lane;
            __syncwarp();
            group_at = segment_first[lane];
            __syncwarp();
        }
        int batch_first = 0, batch_count = 0, batch_sum = 0;          // of 32 groups, one per lane: the first 32, until they have to be passed
        auto load_groups = [&](int g0) {
            const int g = g0 + group_at;
            batch_first = batch_count = 0;
            if (g < args.groups) batch_count = group_members(g, batch_first);
            batch_sum = inclusive_sum(row_tiles(batch_count));
        };
        if (args.members == nullptr) {
            total_tiles = args.groups * row_tiles(args.batch / args.groups);
        } else {
            load_groups(0);
            total_tiles = __shfl_sync(0xffffffffu, batch_sum, 31);
            for (int g0 = 32; g0 < args.groups && total_tiles < MANY; g0 += 32) {
                int a;
                total_tiles += __reduce_add_sync(0xffffffffu, g0 + lane < args.groups ? row_tiles(group_members(g0 + lane, a)) : 0);
            }
        }
        // ---- which row tile and head, and which part of its keys: whole waves of them uncut, the rest cut into equal parts
        const int ctas = int(gridDim.x), block = int(blockIdx.x);
        const int items = int(min(int64_t(total_tiles) * args.kv_heads, int64_t(ctas)));
        const int uncut = items > args.sms ? pa_divide(items, args.sms) * args.sms : 0, rest = items - uncut;
        int splits = 1, split = 0, place = 0, item = block;
        if (rest > 0 && args.slots > 0) splits = max(1, min(args.max_splits, pa_divide(min(args.slots, ctas - uncut), rest)));
        if (block >= uncut) {
            place = block - uncut;
            split = rest > 0 ? pa_divide(place, rest) : splits;
            item = uncut + place - split * rest;
        }
        if (block == 0 && lane == 0 && args.slots > 0) {
            args.cut[0] = splits > 1 ? rest : 0;
            args.cut[1] = splits;
        }
        // row tile fastest: CTAs that run together share the key tiles of their group in the L2; sorted: all heads of a row tile in its turn
        const int slow = pa_divide(item, sorted ? args.kv_heads : max(total_tiles, 1)), fast = item - slow * (sorted ? args.kv_heads : max(total_tiles, 1));
        const int kv_head = sorted ? fast : slow, tile = sorted ? slow : fast;
        if (split >= splits) {
            group = -1;          // nothing left for this one
        } else if (args.members == nullptr) {
            count = args.batch / args.groups;
            group = pa_divide(tile, row_tiles(count));
            group_tile = tile - group * row_tiles(count);
            if (sorted) group = __shfl_sync(0xffffffffu, group_at, group);
            first = group * count;
        } else {
            int before = 0;
            for (int g0 = 0; g0 < args.groups && group < 0 && before < MANY; g0 += 32) {
                if (g0 > 0) load_groups(g0);
                const int mine = row_tiles(batch_count), start = before + batch_sum - mine;
                const unsigned hit = __ballot_sync(0xffffffffu, mine > 0 && tile >= start && tile < start + mine);
                if (hit != 0u) {
                    const int source = __ffs(int(hit)) - 1;
                    group = g0 + __shfl_sync(0xffffffffu, group_at, source);
                    first = __shfl_sync(0xffffffffu, batch_first, source);
                    count = __shfl_sync(0xffffffffu, batch_count, source);
                    group_tile = tile - __shfl_sync(0xffffffffu, start, source);
                }
                before += __shfl_sync(0xffffffffu, batch_sum, 31);
            }
        }
        const int row0 = group_tile * PA_ROWS;
        int rows = group < 0 ? 0 : count * args.rows_per_member - row0;
        rows = rows < 0 ? 0 : (rows > PA_ROWS ? PA_ROWS : rows);
        const int first_own = pa_divide(row0, args.rows_per_member);                      // first member with rows in this tile
        if (lane == 0) *work = PaWork{group, first, row0, rows, 0, first_own, 0, kv_head, split, rows > 0 && block >= uncut ? splits : 1, place};
        named_barrier<3, 288>();          // the softmax warps fetch the queries while the lengths come
        const int segments = rows == 0 ? 1 : pa_divide(row0 + rows - 1, args.rows_per_member) - first_own + 2;
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
                if (FP8) segment_nan[s] = INT_MAX;
            }
            total += __shfl_sync(0xffffffffu, sum, 31);
        }
        if (lane == 0) {
            segment_first[segments] = total;
            work->segments = segments;
            work->key_tiles = total;
        }
    }
    // ---- softmax warps: which query a thread has, and all rows of queries on their way
    bool exists = false;
    int my_segment = -1, hidden = 0;          // the segment of this row's own keys; causal: how many of them lie behind the query
    constexpr int PIECES = D / 8;             // 16-byte pieces of a row; in the staging area piece p lies at p ^ (row % 8)
    if (warp < 8) {
        named_barrier<3, 288>();
        const PaWork found = *work;
        const int row = int(threadIdx.x) & (PA_ROWS - 1);
        int64_t query_offset = -1, out_offset = -1;
        exists = row < found.rows;
        if (exists) {
            const int member = pa_divide(found.row0 + row, args.rows_per_member), inside = found.row0 + row - member * args.rows_per_member;
            const int head_in_group = pa_divide(inside, args.queries), query = inside - head_in_group * args.queries;
            const int head = found.kv_head * args.share + head_in_group;
            my_segment = member - found.first_segment_member + 1;
            hidden = args.causal ? args.queries - 1 - query : 0;
            out_offset = ((int64_t(found.first_member + member) * args.heads + head) * args.queries + query) * D;
            query_offset = int64_t(found.first_member + member) * args.q_stride[0] + head * args.q_stride[1] + query * args.q_stride[2];
        }
        if (threadIdx.x < PA_ROWS) {
            row_query[row] = query_offset;
            row_output[row] = out_offset;
        }
        named_barrier<1, 256>();
        constexpr int BATCH = 8;          // the copies would hold the next offset's load back
#pragma unroll 1
        for (int first = int(threadIdx.x); first < PA_ROWS * PIECES; first += BATCH * 256) {
            int64_t from[BATCH];
#pragma unroll
            for (int n = 0; n < BATCH; ++n) from[n] = row_query[(first + n * 256) / PIECES];
#pragma unroll
            for (int n = 0; n < BATCH; ++n) {
                const int i = first + n * 256, r = i / PIECES, piece = i % PIECES;
                const uint32_t to = staging_smem + uint32_t(r * D * 2 + ((piece ^ (r & 7)) << 4));
                const __nv_bfloat16* source = args.q + (from[n] < 0 ? 0 : from[n]) + piece * 8;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(source), "r"(from[n] < 0 ? 0 : 16) : "memory");
            }
        }
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    uint32_t tmem_base;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem_base) : "r"(tmem_slot) : "memory");
    const PaWork w = *work;
    const int kv_head = w.kv_head, start_tile = int(int64_t(w.key_tiles) * w.split / w.splits);
    const int num_tiles = int(int64_t(w.key_tiles) * (w.split + 1) / w.splits) - start_tile;

    uint32_t patience = PA_PATIENCE;
    if (warp < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(PA_SOFTMAX_REGISTERS));
        // ------------------------------------------------------------- one thread per query row and tile parity
        const int quarter = warp & 3, row = quarter * 32 + lane;          // row of the tile = tensor-memory lane
        const int parity_group = warp >> 2;           // 0: even tiles, 1: odd tiles
        const uint32_t lane_address = tmem_base + (uint32_t(quarter * 32) << 16);
        // ---- the queries into tensor memory: rows came to shared memory as they lie (16 bytes per thread), each thread takes one half of the
        // columns of its row
        float factor = args.scale_log2;
        asm volatile("cp.async.wait_all;" ::: "memory");
        if (num_tiles > 0) {
            constexpr int CHUNKS = D / 128;          // of 32 words (64 values) of half a bf16 row
            named_barrier<1, 256>();
            auto load = [&](int chunk, uint32_t (&words)[32]) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int piece = (parity_group * CHUNKS + chunk) * 8 + i;
                    const uint4 v = lds_u4(staging_smem + uint32_t(row * D * 2 + ((piece ^ (row & 7)) << 4)));
                    words[4 * i] = v.x; words[4 * i + 1] = v.y; words[4 * i + 2] = v.z; words[4 * i + 3] = v.w;
                }
            };
            const uint32_t line = q_smem + uint32_t(row >> 3) * 1024u + uint32_t(row & 7) * 128u;          // of the atom in shared memory
            auto store_line = [&](int c, const uint32_t* four) { sts_u4(line + uint32_t((c ^ (row & 7)) * 16), four[0], four[1], four[2], four[3]); };
            if (!FP8) {
#pragma unroll 1
                for (int chunk = 0; chunk < CHUNKS; ++chunk) {
                    uint32_t words[32];
                    load(chunk, words);
                    const int atom = parity_group * CHUNKS + chunk;
                    if (atom < Shape::Q_TMEM_ATOMS) {
                        pa_tmem_store(lane_address + Shape::TMEM_Q + uint32_t(atom) * 32, words);
                    } else {
#pragma unroll
                        for (int c = 0; c < 8; ++c) store_line(c, words + 4 * c);
                    }
                }
            } else {
                uint32_t largest = 0;      // bf16 magnitude bits: NaN and infinities order above numbers
#pragma unroll 1
                for (int chunk = 0; chunk < CHUNKS; ++chunk) {
                    uint32_t words[32];
                    load(chunk, words);
#pragma unroll
                    for (int i = 0; i < 32; ++i) largest = __vmaxu2(largest, words[i] & 0x7fff7fffu);
                }
                largest = max(largest & 0xffffu, largest >> 16);
                row_exchange[parity_group * PA_ROWS + row] = __uint_as_float(largest);
                named_barrier<1, 256>();
                largest = max(largest, __float_as_uint(row_exchange[(parity_group ^ 1) * PA_ROWS + row]));
                // 2^e that brings the largest magnitude into [128, 256); it and its reciprocal are normal numbers for every finite row from
                // 2^-119 on
                int exponent = int(largest >> 7) - 127;
                exponent = exponent < -119 ? -119 : (exponent > 127 ? 127 : exponent);
                const float up = largest == 0u ? 1.0f : __uint_as_float(uint32_t(127 + 7 - exponent) << 23);
                const float down = largest == 0u ? 1.0f : __uint_as_float(uint32_t(127 - 7 + exponent) << 23);
                // a row with an infinity or a NaN: every score is NaN
                factor = largest >= 0x7f80u ? __uint_as_float(0x7fc00000u) : args.scale_log2 * down;
                const __nv_bfloat162 up2 = __float2bfloat162_rn(up);
                // hi of this half is columns [HALF_COLUMNS * group, ..), lo the same behind all of hi
                constexpr uint32_t HALF_COLUMNS = D / 8;
#pragma unroll 1
                for (int chunk = 0; chunk < CHUNKS; ++chunk) {
                    uint32_t words[32], high[16], low[16];
                    load(chunk, words);
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        // of the 8 significant bits hi takes the upper 4 and lo the lower; below 2^-6, where e4m3 has fewer, lo takes all
                        const __nv_bfloat162 x = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&words[i]), up2);
                        const uint32_t small = __hlt2_mask(__habs2(x), __float2bfloat162_rn(0.015625f));
                        const uint32_t upper = *reinterpret_cast<const uint32_t*>(&x) & 0xfff0fff0u & ~small;
                        const __nv_bfloat162 rest = __hsub2(x, *reinterpret_cast<const __nv_bfloat162*>(&upper));
                        const uint32_t h = __nv_cvt_float2_to_fp8x2(bf16x2_to_float2(upper), __NV_SATFINITE, __NV_E4M3);
                        const uint32_t l = __nv_cvt_float2_to_fp8x2(bf16x2_to_float2(*reinterpret_cast<const uint32_t*>(&rest)), __NV_SATFINITE, __NV_E4M3);
                        high[i >> 1] = (i & 1) ? high[i >> 1] | (h << 16) : h;
                        low[i >> 1] = (i & 1) ? low[i >> 1] | (l << 16) : l;
                    }
                    const uint32_t column = uint32_t(parity_group) * HALF_COLUMNS + uint32_t(chunk) * 16;
                    pa_tmem_store16(lane_address + Shape::TMEM_Q + column, high);
                    if (2 * HALF_COLUMNS + column < Shape::Q_TMEM_ATOMS * 32) {
                        pa_tmem_store16(lane_address + Shape::TMEM_Q + 2 * HALF_COLUMNS + column, low);
                    } else {
#pragma unroll
                        for (int c = 0; c < 4; ++c) store_line(4 * chunk + c, low + 4 * c);
                    }
                }
            }
            fence_async_shared();          // the atom in shared memory; and the staging area is the copies' or the values' again
            pa_tmem_store_wait();
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_ready);
        }
        float reference = -INFINITY, running_sum = 0.0f;          // of this group's tiles so far: the sum in units of 2^reference
        int unit = 0;                                             // of the values in its accumulator, as an exponent
        const uint32_t s_tmem = lane_address + Shape::TMEM_S + uint32_t(parity_group) * PA_KEYS;
        const uint32_t p_tmem = lane_address + Shape::TMEM_P + uint32_t(parity_group % Shape::P_BUFFERS) * 32;
        const uint32_t o_tmem = lane_address + Shape::TMEM_O + uint32_t(parity_group % Shape::O_BUFFERS) * D;
        PaCursor cursor(segment_first, segment_length, parity_group < num_tiles ? start_tile + parity_group : -1);
        uint32_t phase = 0;                                       // of this group's barriers: (j / 2) % 2
        for (int j = parity_group; j < num_tiles; j += 2, phase ^= 1u) {
            cursor.seek(start_tile + j);
            // keys of this tile that this row sees: the first `valid`
            int valid = cursor.keys_left - cursor.first_key(start_tile + j);
            bool whole = valid >= PA_KEYS, none = false;
            if (cursor.segment > 0) {
                valid = cursor.segment == my_segment ? valid - hidden : 0;
                whole = __all_sync(0xffffffffu, valid >= PA_KEYS);
                none = __all_sync(0xffffffffu, valid <= 0);
            }
            const int stage = j % PA_SCALE_STAGES;
            const float4* tile_scales = reinterpret_cast<const float4*>(generic + Shape::OFF_SCALES) + stage * (PA_SCALE_FLOATS / 4);
            if (FP8) pa_wait(scale_full + 8 * stage, uint32_t(j / PA_SCALE_STAGES) & 1u, patience);
            pa_wait(s_full + 8 * parity_group, phase, patience);
            tc_fence_after_sync();
            uint32_t raw[2][32];
            float tile_max = -INFINITY;
            // D = 128: one half of the scores is scaled while the other one is on its way (80 us for the 32768 keys, both first 81.5; D = 256, where
            // the scores' place is waited for: 188.5 and 187 us for the fifty-query chunks)
            auto scaled = [&](int half) {
                if (FP8) {
#pragma unroll
                    for (int i = 8 * half; i < 8 * half + 8; ++i) {
                        const float4 ks = tile_scales[i];
                        uint32_t* r = &raw[half][(i & 7) * 4];
                        const float2 a = __fmul2_rn(make_float2(__uint_as_float(r[0]), __uint_as_float(r[1])), make_float2(ks.x, ks.y));
                        const float2 c = __fmul2_rn(make_float2(__uint_as_float(r[2]), __uint_as_float(r[3])), make_float2(ks.z, ks.w));
                        r[0] = __float_as_uint(a.x); r[1] = __float_as_uint(a.y); r[2] = __float_as_uint(c.x); r[3] = __float_as_uint(c.y);
                    }
                }
                if (!whole) {
#pragma unroll
                    for (int i = 32 * half; i < 32 * half + 32; ++i)
                        if (i >= valid) raw[half][i & 31] = __float_as_uint(-INFINITY);
                }
                float partial_max[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < 32; ++i) partial_max[i & 3] = fmaxf(partial_max[i & 3], __uint_as_float(raw[half][i]));
                return fmaxf(fmaxf(partial_max[0], partial_max[1]), fmaxf(partial_max[2], partial_max[3]));
            };
            if (!none) {
                tmem_load_32x32(s_tmem, raw[0]);
                if (Shape::SHARED) tmem_load_32x32(s_tmem + 32, raw[1]);
                pa_tmem_load_wait(raw[0]);
                if (Shape::SHARED) {
                    pa_tie(raw[1]);
                } else {
                    tmem_load_32x32(s_tmem + 32, raw[1]);
                    tile_max = scaled(0);
                    pa_tmem_load_wait(raw[1]);
                }
            }
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(s_free + 8 * parity_group);
            if (!none) {
                if (Shape::SHARED) tile_max = scaled(0);
                tile_max = fmaxf(tile_max, scaled(1)) * factor;
            }
            // The reference follows the maximum lazily: it moves only when the maximum has grown by more than 2^8 since it was set, so
            // weights stay within 2^8 of its and the accumulator is rescaled a few times per row.  A row that has seen no key yet has none; 0
            // stands in, its weights are 0.  With one accumulator the reference of the tile before comes from the other group.
            float previous = reference;
            if (Shape::SHARED && j > 0) {
                const int other = parity_group ^ 1;
                pa_wait(reference_ready + 16 * quarter + 8 * other, parity_group == 0 ? phase ^ 1u : phase, patience);
                previous = *static_cast<volatile float*>(row_reference + other * PA_ROWS + row);
            }
            const float now = tile_max > previous + 8.0f ? tile_max : previous;
            if (Shape::SHARED) {
                *static_cast<volatile float*>(row_reference + parity_group * PA_ROWS + row) = now;
                __syncwarp();
                if (lane == 0) mbar_arrive(reference_ready + 16 * quarter + 8 * parity_group);
            }
            // what O holds is in units of the reference before (a row without one has nothing but zeros there) and of the values' unit before
            float correction = now == previous || previous == -INFINITY ? 1.0f : pa_exp2(previous - now);
            running_sum *= Shape::SHARED ? (now == reference ? 1.0f : pa_exp2(reference - now)) : correction;
            reference = now;
            unsigned long long bad = 0ull;          // keys that give NaN to the rows that see them
            if (FP8) {
                const float4 entry = tile_scales[2 * PA_KEYS / 4];
                bad = __float_as_uint(entry.x) | (static_cast<unsigned long long>(__float_as_uint(entry.y)) << 32);
                const int tile_unit = __float_as_int(Shape::SHARED ? entry.w : entry.z);
                if (Shape::SHARED) {          // the change from the tile before
                    if (tile_unit != 0) correction *= exp2f(float(tile_unit));
                } else {
                    if (j >= 2 && tile_unit != unit) correction *= exp2f(float(unit - tile_unit));
                    unit = tile_unit;
                }
            }
            const uint32_t output_bar = o_done + 8 * (Shape::SHARED ? parity_group ^ 1 : parity_group);
            const uint32_t output_phase = Shape::SHARED && parity_group == 1 ? phase : phase ^ 1u;
            uint32_t packed[32];
            if (none) {
#pragma unroll
                for (int i = 0; i < 32; ++i) packed[i] = 0u;
            } else {
                const float shift = now == -INFINITY ? 0.0f : PA_WEIGHT_BITS<FP8> - now;
                const float2 shift2 = make_float2(shift, shift), factor2 = make_float2(factor, factor);
                float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    const float2 a = __ffma2_rn(make_float2(__uint_as_float(raw[i >> 4][2 * (i & 15)]), __uint_as_float(raw[i >> 4][2 * (i & 15) + 1])), factor2, shift2);
                    const float2 p = make_float2(pa_exp2(a.x), pa_exp2(a.y));
                    packed[i] = FP8 ? float2_to_half2_bits(p.x, p.y) : float2_to_bf16x2(p);
                    sum[i & 1] = __fadd2_rn(sum[i & 1], p);
                }
                running_sum += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                if (!FP8 && cursor.segment > 0) {
                    pa_wait(value_full + 8 * (j % STAGES), uint32_t(j / STAGES) & 1u, patience);
                    bad = *static_cast<volatile unsigned long long*>(bad_keys + j % STAGES);
                }
                if (bad != 0ull) {
                    const unsigned long long seen = valid >= PA_KEYS ? ~0ull : valid <= 0 ? 0ull : (1ull << valid) - 1ull;
                    if ((bad & seen) != 0ull) running_sum = __uint_as_float(0x7fc00000u);
                }
            }
            if (FP8) {
                __syncwarp();
                if (lane == 0) mbar_arrive(scale_empty + 8 * stage);
            }
            // the P that lies where this one goes has been read, and O holds everything before this tile: the product of the tile before, or
            // of this group's last, is done
            if (j >= Shape::P_BUFFERS) {
                pa_wait(output_bar, output_phase, patience);
                __syncwarp();
                tc_fence_after_sync();
                if (__any_sync(0xffffffffu, correction != 1.0f)) {
#pragma unroll 1
                    for (int chunk = 0; chunk < D / 32; ++chunk) {
                        uint32_t o[32];
                        tmem_load_32x32(o_tmem + chunk * 32, o);
                        pa_tmem_load_wait(o);
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * correction);
                        pa_tmem_store(o_tmem + chunk * 32, o);
                    }
                }
            }
            pa_tmem_store(p_tmem, packed);          // 64 keys in 32 columns
            pa_tmem_store_wait();
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_ready + 8 * parity_group);
        }
        // ---- the two groups' results.  One accumulator is in units of the later reference; two have one each.
        if (num_tiles > 0) {
            pa_wait(all_done, 0u, patience);
            __syncwarp();
            tc_fence_after_sync();
        }
        const bool sees = segment_length[0] > 0 || (my_segment > 0 && segment_length[my_segment] > hidden);          // a key, anywhere
        if (FP8) {          // what the value warps have found: their last arrivals
            for (int j = num_tiles > 2 ? num_tiles - 2 : 0; j < num_tiles; ++j) pa_wait(value_full + 8 * (j & 1), uint32_t(j >> 1) & 1u, patience);
            if (my_segment > 0 && num_tiles > 0 && segment_nan[my_segment] < segment_length[my_segment] - hidden) running_sum = __uint_as_float(0x7fc00000u);
            // a query that is not finite makes NaN of masked scores too: a row that sees no key is zero all the same
            if (!sees) running_sum = 0.0f;
        }
        row_reference[parity_group * PA_ROWS + row] = reference;      // what its last tile left there, or -inf
        row_exchange[parity_group * PA_ROWS + row] = running_sum;
        if (!Shape::SHARED && row == 0) group_unit[parity_group] = unit;
        named_barrier<1, 256>();
        const float last = fmaxf(row_reference[row], row_reference[PA_ROWS + row]);
        float weight[2];          // of the groups' sums, and of their accumulators
#pragma unroll
        for (int g = 0; g < 2; ++g) weight[g] = row_reference[g * PA_ROWS + row] == last ? 1.0f : pa_exp2(row_reference[g * PA_ROWS + row] - last);
        running_sum = weight[0] * row_exchange[row] + weight[1] * row_exchange[PA_ROWS + row];
        reference = last;
        if (FP8) {
            if (Shape::SHARED) weight[0] = exp2f(float(num_tiles > 0 ? group_unit[0] : 0));
            else weight[0] *= exp2f(float(group_unit[0])), weight[1] *= exp2f(float(group_unit[1]));
        } else if (Shape::SHARED) {
            weight[0] = 1.0f;
        }
        // 32 columns of the row (D = 256: 64) in units of the reference
        auto output_columns = [&](int column, auto& o) {
            tmem_load_32x32(lane_address + Shape::TMEM_O + column, o[0]);
            if constexpr (Shape::SHARED) {
                tmem_load_32x32(lane_address + Shape::TMEM_O + column + 32, o[1]);
                pa_tmem_load_wait(o[0]);
                pa_tie(o[1]);
#pragma unroll
                for (int i = 0; i < 64; ++i) o[i / 32][i % 32] = __float_as_uint(__uint_as_float(o[i / 32][i % 32]) * weight[0]);
            } else if (num_tiles > 1) {
                uint32_t other[32];
                tmem_load_32x32(lane_address + Shape::TMEM_O + D + column, other);
                pa_tmem_load_wait(o[0]);
                pa_tie(other);
#pragma unroll
                for (int i = 0; i < 32; ++i) o[0][i] = __float_as_uint(__uint_as_float(o[0][i]) * weight[0] + __uint_as_float(other[i]) * weight[1]);
            } else {
                pa_tmem_load_wait(o[0]);
#pragma unroll
                for (int i = 0; i < 32; ++i) o[0][i] = __float_as_uint(__uint_as_float(o[0][i]) * weight[0]);
            }
        };
        const int first_column = parity_group * (D / 2);          // each group stores half of the columns
        const bool stored = w.splits == 1;
        const int64_t first_partial = int64_t(w.place) * PA_ROWS;
        if (!stored && parity_group == 0) {
            if (w.split == 0) args.row_offsets[first_partial + row] = exists ? row_output[row] | int64_t(sees) : -1;
            if (exists) *reinterpret_cast<float2*>(args.partial + int64_t(args.slots) * PA_ROWS * D + (first_partial + row) * 2) = make_float2(reference, running_sum);
        }
        // Rows go out through shared memory (the rings are empty now), a bulk copy for each: a thread has a row of the accumulator, and its
        // own stores would touch a sector at a time.  16 bytes between rows spread them over the banks.
        // sum 0: the row sees no key, or (IEEE arithmetic: NaN) none whose score is above -inf
        if (stored && sees && running_sum == 0.0f) running_sum = __uint_as_float(0x7fc00000u);
        const float inverse = stored ? (running_sum == 0.0f ? 0.0f : 1.0f / running_sum) : 1.0f;
        const uint32_t row_bytes = stored ? D * 2 : D * 4, out_row = base + uint32_t(row) * (row_bytes + 16);
        constexpr int BATCH = Shape::SHARED ? 2 : 1;          // of 32 columns
#pragma unroll 1
        for (int column = first_column; column < first_column + D / 2; column += 32 * BATCH) {
            uint32_t o[BATCH][32];
            if (num_tiles > 0) {
                output_columns(column, o);
            } else {
#pragma unroll
                for (int i = 0; i < 32 * BATCH; ++i) o[i / 32][i % 32] = 0u;
            }
#pragma unroll
            for (int i = 0; i < 4 * BATCH; ++i) {
                uint32_t eight[8];
#pragma unroll
                for (int v = 0; v < 8; ++v) {
                    const uint32_t value = o[i / 4][(8 * i + v) % 32];
                    eight[v] = running_sum == 0.0f ? 0u : __float_as_uint(__uint_as_float(value) * inverse);
                }
                if (stored) {
                    uint32_t words[4];
#pragma unroll
                    for (int v = 0; v < 4; ++v) words[v] = float2_to_bf16x2(make_float2(__uint_as_float(eight[2 * v]), __uint_as_float(eight[2 * v + 1])));
                    sts_u4(out_row + (column + 8 * i) * 2, words[0], words[1], words[2], words[3]);
                } else {
                    sts_u4(out_row + (column + 8 * i) * 4, eight[0], eight[1], eight[2], eight[3]);
                    sts_u4(out_row + (column + 8 * i) * 4 + 16, eight[4], eight[5], eight[6], eight[7]);
                }
            }
        }
        // each thread sends what it has written: the other group's half of the row does not have to be waited for
        fence_async_shared();
        if (exists) {
            const uint32_t half_bytes = row_bytes / 2, from = out_row + uint32_t(parity_group) * half_bytes;
            const void* destination = stored ? static_cast<const void*>(args.out + row_output[row] + first_column)
                                             : static_cast<const void*>(args.partial + (first_partial + row) * D + first_column);
            asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(destination), "r"(from), "r"(half_bytes) : "memory");
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");          // the rows have been taken: the CTA may leave
        }
    } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PA_OTHER_REGISTERS));
    if (warp == PA_LOAD_WARP) {
        // ------------------------------------------------------------- TMA producer
        if (num_tiles > 0) {
            auto load = [&](const PaCursor& cursor, const CUtensorMap& prefix_map, const CUtensorMap& own_map, uint32_t smem, uint32_t full, int j) {
                const int b = j % STAGES;
                const bool prefix = cursor.segment == 0;
                const int sequence = prefix ? w.group : w.first_member + w.first_segment_member + cursor.segment - 1;
                const int row = (sequence * args.kv_heads + kv_head) * (prefix ? args.prefix_capacity : args.own_capacity) + cursor.first_key(start_tile + j);
                __syncwarp();
                if (elect_one()) {
                    mbar_expect_tx(full + 8 * b, Shape::KV_BYTES);
                    for (int a = 0; a < Shape::KV_ATOMS; ++a)
                        tma_load_2d(smem + b * Shape::KV_BYTES + a * Shape::KV_ATOM_BYTES, prefix ? &prefix_map : &own_map, full + 8 * b, a * 128, row);
                }
                __syncwarp();
            };
            // D = 256: keys go two tiles ahead of values, because the scores run ahead of the output and a value slot is free only behind
            // the output (fifty-query chunks over 8192 keys: 213 us, in step 219).  D = 128 has the slots to go in step (a 32768-key prefix:
            // 83 us, ahead 86).
            constexpr int AHEAD = Shape::SHARED ? 2 : 0;
            PaCursor key_cursor(segment_first, segment_length, start_tile), value_cursor(segment_first, segment_length, start_tile);
            for (int i = 0; i < num_tiles + AHEAD; ++i) {
                if (i < num_tiles) {
                    key_cursor.seek(start_tile + i);
                    pa_wait(k_empty + 8 * (i % STAGES), (uint32_t(i / STAGES) & 1u) ^ 1u, patience);
                    load(key_cursor, prefix_k_map, own_k_map, k_smem, k_full, i);
                }
                const int j = i - AHEAD;
                if (j >= 0) {
                    if (AHEAD > 0) value_cursor.seek(start_tile + j);
                    pa_wait(v_empty + 8 * (j % STAGES), (uint32_t(j / STAGES) & 1u) ^ 1u, patience);
                    if (j == Shape::FREE_V_STAGES && j < STAGES) pa_wait(q_ready, 0u, patience);          // the queries came through this place
                    load(AHEAD > 0 ? value_cursor : key_cursor, prefix_v_map, own_v_map, v_smem, v_full, j);
                }
            }
            // every copy has landed before this CTA may leave (on the normal path the readers have long seen them)
            for (int b = 0; b < STAGES && b < num_tiles; ++b) {
                const int last = ((num_tiles - 1 - b) / STAGES) * STAGES + b;
                pa_wait(k_full + 8 * b, uint32_t(last / STAGES) & 1u, patience);
                pa_wait(v_full + 8 * b, uint32_t(last / STAGES) & 1u, patience);
            }
        }
    } else if (warp == PA_SCORES_WARP) {
        // ------------------------------------------------------------- MMA issuer: S[j & 1] = Q K_j^T
        // Products into different accumulators are ordered by nothing but the barriers, so each kind has a warp that issues it: neither
        // waits behind the other's operands, and the tensor core finds the next product queued.
        const uint32_t idesc = FP8 ? idesc_f8(PA_ROWS, PA_KEYS) : pa_idesc_16bit(PA_ROWS, PA_KEYS, true, false);
        const uint64_t k_major = smem_desc_sw128(0);
        const uint32_t k_low = uint32_t(k_major), k_high = uint32_t(k_major >> 32);
        auto field = [](uint32_t address) { return (address & 0x3FFFFu) >> 4; };
        if (num_tiles > 0) pa_wait(q_ready, 0u, patience);
        PaRing<STAGES> ring;
        for (int j = 0; j < num_tiles; ++j) {
            const int d = j & 1;
            pa_wait(s_free + 8 * d, (uint32_t(j >> 1) & 1u) ^ 1u, patience);
            pa_wait(k_full + 8 * ring.slot, ring.parity, patience);
            tc_fence_after_sync();
            __syncwarp();
            if (elect_one()) {
                const uint32_t d_tmem = tmem_base + Shape::TMEM_S + uint32_t(d) * PA_KEYS;
                const uint32_t k_base = k_low + field(k_smem + ring.slot * Shape::KV_BYTES);
                // 32 bytes along K per instruction: 8 columns of Q.  Quantised: first all of hi, then all of lo.
#pragma unroll
                for (int a = 0; a < Shape::Q_ATOMS; ++a)
#pragma unroll
                    for (int s = 0; s < 4; ++s) {
                        const uint64_t k_desc = desc_from_words(k_base + (a % Shape::KV_ATOMS) * (Shape::KV_ATOM_BYTES >> 4) + 2 * s, k_high);
                        if (a < Shape::Q_TMEM_ATOMS) pa_mma<FP8>(d_tmem, tmem_base + Shape::TMEM_Q + uint32_t((a * 4 + s) * 8), k_desc, idesc, (a | s) != 0);
                        else pa_mma_shared<FP8>(d_tmem, desc_from_words(k_low + field(q_smem) + 2 * s, k_high), k_desc, idesc, 1u);
                    }
                tc_commit(s_full + 8 * d);
                tc_commit(k_empty + 8 * ring.slot);
            }
            __syncwarp();
            ring.next();
        }
    } else if (warp == PA_OUTPUT_WARP) {
        // ------------------------------------------------------------- MMA issuer: O += P V_j
        const uint32_t idesc = pa_idesc_16bit(PA_ROWS, D, !FP8, true);
        const uint64_t mn_major = pa_desc_mn(Shape::KV_ATOM_BYTES);
        const uint32_t mn_low = uint32_t(mn_major), mn_high = uint32_t(mn_major >> 32);
        auto field = [](uint32_t address) { return (address & 0x3FFFFu) >> 4; };
        PaRing<FP8 ? 2 : STAGES> ring;
        for (int j = 0; j < num_tiles; ++j) {
            const int d = j & 1;
            pa_wait(value_full + 8 * ring.slot, ring.parity, patience);
            pa_wait(p_ready + 8 * d, uint32_t(j >> 1) & 1u, patience);
            tc_fence_after_sync();
            __syncwarp();
            if (elect_one()) {
                const uint32_t p_tmem = tmem_base + Shape::TMEM_P + uint32_t(d % Shape::P_BUFFERS) * 32;
                const uint32_t v_base = mn_low + field(FP8 ? values_smem + ring.slot * Shape::VALUE_BYTES : v_smem + ring.slot * Shape::KV_BYTES);
#pragma unroll
                for (int s = 0; s < PA_KEYS / 16; ++s)          // 16 keys per instruction: 8 columns of P, 16 rows (2048 bytes) of V
                    pa_mma<false>(tmem_base + Shape::TMEM_O + uint32_t(d % Shape::O_BUFFERS) * D, p_tmem + 8 * s, desc_from_words(v_base + s * (2048 >> 4), mn_high), idesc,
                                  j >= Shape::O_BUFFERS || s > 0);
                tc_commit(o_done + 8 * d);
                tc_commit((FP8 ? value_empty : v_empty) + 8 * ring.slot);
                if (j == num_tiles - 1) tc_commit(all_done);
            }
            __syncwarp();
            ring.next();
        }
    } else if (warp >= PA_VALUE_WARP && !FP8) {
        // ------------------------------------------------------------- bf16: values the tensor core must not see
        if (num_tiles > 0) {
            constexpr int CHUNKS = Shape::KV_ATOMS * 8;          // 16-byte chunks of a row
            const int thread = (warp - PA_VALUE_WARP) * 32 + lane;
            PaCursor cursor(segment_first, segment_length, start_tile);
            for (int j = 0; j < num_tiles; ++j) {
                cursor.seek(start_tile + j);
                const int b = j % STAGES;
                pa_wait(v_full + 8 * b, uint32_t(j / STAGES) & 1u, patience);
                int valid = cursor.keys_left - cursor.first_key(start_tile + j);
                valid = valid < PA_KEYS ? valid : PA_KEYS;
                const uint32_t stage = v_smem + b * Shape::KV_BYTES;
                for (int i = valid * CHUNKS + thread; i < PA_KEYS * CHUNKS; i += 32 * Shape::VALUE_WARPS)
                    sts_u4(stage + uint32_t((i & (CHUNKS - 1)) >> 3) * Shape::KV_ATOM_BYTES + uint32_t(i / CHUNKS) * 128u + uint32_t(i & 7) * 16u, 0u, 0u, 0u, 0u);
                if (cursor.segment > 0) {
                    if (thread == 0) bad_keys[b] = 0ull;
                    named_barrier<2, 32 * Shape::VALUE_WARPS>();
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
    } else if (warp >= PA_VALUE_WARP) {
        // ------------------------------------------------------------- codes of the value tile -> f16 operand
        // 16 codes of a key per thread and step: chunk `piece` of its row (stored at piece ^ (key % 8) inside its 128-byte group)
        // becomes two 16-byte chunks of the 64-column group they belong to.  Odd groups store their two chunks in the other order: the
        // eight lanes of a store then meet all banks.
        constexpr int PIECES = D / 16, BATCH = 4;
        static_assert(PA_KEYS * PIECES % (BATCH * 32 * Shape::VALUE_TEAM) == 0, "whole batches");
        const int team = (warp - PA_VALUE_WARP) / Shape::VALUE_TEAM, thread = ((warp - PA_VALUE_WARP) % Shape::VALUE_TEAM) * 32 + lane;
        PaCursor cursor(segment_first, segment_length, team < num_tiles ? start_tile + team : -1);
        if (num_tiles > 0) pa_wait(q_ready, 0u, patience);          // the queries came through this place
        for (int j = team; j < num_tiles; j += 2) {
            const int c = team, stage = j % PA_SCALE_STAGES, slot = j % STAGES;
            const uint32_t* value_scales = reinterpret_cast<const uint32_t*>(generic + Shape::OFF_SCALES) + stage * PA_SCALE_FLOATS + PA_KEYS;
            cursor.seek(start_tile + j);
            // Prefix keys are seen by every row: a NaN among their codes may reach all.  A row with a NaN among own keys' codes is zero here,
            // because the tile's other members' rows, and earlier queries, pass over it with probability zero; where it lies is kept for the
            // rows that do see it.
            const bool own = cursor.segment > 0;
            const int valid = cursor.keys(start_tile + j), first_key = cursor.first_key(start_tile + j);
            const bool plain = !own && valid == PA_KEYS;
            pa_wait(scale_full + 8 * stage, uint32_t(j / PA_SCALE_STAGES) & 1u, patience);
            pa_wait(v_full + 8 * slot, uint32_t(j / STAGES) & 1u, patience);
            pa_wait(value_empty + 8 * c, (uint32_t(j >> 1) & 1u) ^ 1u, patience);
            auto convert = [&](auto tag) {
                constexpr bool PLAIN = decltype(tag)::value;
#pragma unroll 1
                for (int first = thread; first < PA_KEYS * PIECES; first += BATCH * 32 * Shape::VALUE_TEAM) {
                    if (!PLAIN && (first - thread) / PIECES >= valid) {          // behind the end, all of the batch: no code to look at
#pragma unroll
                        for (int n = 0; n < BATCH; ++n) {
                            const uint32_t i = first + n * 32 * Shape::VALUE_TEAM, key = i / PIECES, piece = i % PIECES, left = (piece & 3u) * 2u;
                            const uint32_t group = values_smem + c * Shape::VALUE_BYTES + (piece >> 2) * Shape::KV_ATOM_BYTES + key * 128u;
                            sts_u4(group + ((left ^ (key & 7u)) << 4), 0u, 0u, 0u, 0u);
                            sts_u4(group + (((left + 1u) ^ (key & 7u)) << 4), 0u, 0u, 0u, 0u);
                        }
                        continue;
                    }
                    uint4 codes[BATCH];
                    uint32_t scale_bits[BATCH];
#pragma unroll
                    for (int n = 0; n < BATCH; ++n) {          // all loads first: each of the stores would hold the next load back
                        const uint32_t i = first + n * 32 * Shape::VALUE_TEAM, key = i / PIECES, piece = i % PIECES;
                        codes[n] = lds_u4(v_smem + slot * Shape::KV_BYTES + (piece >> 3) * Shape::KV_ATOM_BYTES + key * 128u + (((piece & 7u) ^ (key & 7u)) << 4));
                        scale_bits[n] = value_scales[key];
                        if (!PLAIN) {
                            const uint32_t nan = codes_not_a_number(codes[n].x) | codes_not_a_number(codes[n].y) | codes_not_a_number(codes[n].z) | codes_not_a_number(codes[n].w);
                            const bool there = int(key) < valid, marked = there && own && nan != 0u;
                            if (marked) atomicMin(segment_nan + cursor.segment, first_key + int(key));
                            if (!there || marked) codes[n] = make_uint4(0u, 0u, 0u, 0u);
                        }
                    }
#pragma unroll
                    for (int n = 0; n < BATCH; ++n) {
                        const uint32_t i = first + n * 32 * Shape::VALUE_TEAM, key = i / PIECES, piece = i % PIECES, swizzle = key & 7u;
                        const __half2 scale = *reinterpret_cast<const __half2*>(&scale_bits[n]);
                        const uint32_t group = values_smem + c * Shape::VALUE_BYTES + (piece >> 2) * Shape::KV_ATOM_BYTES + key * 128u;
                        const uint32_t odd = (piece >> 2) & 1u, left = (piece & 3u) * 2u;
                        const uint32_t x = odd ? codes[n].z : codes[n].x, y = odd ? codes[n].w : codes[n].y;
                        const uint32_t z = odd ? codes[n].x : codes[n].z, w = odd ? codes[n].y : codes[n].w;
                        sts_u4(group + (((left + odd) ^ swizzle) << 4), codes_to_halves(x, scale), codes_to_halves(x >> 16, scale),
                               codes_to_halves(y, scale), codes_to_halves(y >> 16, scale));
                        sts_u4(group + (((left + 1u - odd) ^ swizzle) << 4), codes_to_halves(z, scale), codes_to_halves(z >> 16, scale),
                               codes_to_halves(w, scale), codes_to_halves(w >> 16, scale));
                    }
                }
            };
            if (plain) convert(std::true_type{});
            else convert(std::false_type{});
            fence_async_shared();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(v_empty + 8 * slot);
                mbar_arrive(value_full + 8 * c);
                mbar_arrive(scale_empty + 8 * stage);
            }
        }
    } else if (FP8 && warp == PA_SCALE_WARP) {
        // ------------------------------------------------------------- scales of the key tiles
        // Copied PA_RAW_STAGES - 1 tiles ahead, by the lane that converts them: a key tile's time is less than a load from memory takes.
        if (num_tiles > 0) {
            PaCursor cursor(segment_first, segment_length, start_tile);
            const uint32_t raw_scales = base + Shape::OFF_RAW_SCALES;
            int unit_exponent = 0;
            auto copy = [&](int j) {
                if (j < num_tiles) {
                    cursor.seek(start_tile + j);
                    const bool prefix = cursor.segment == 0;
                    const int sequence = prefix ? w.group : w.first_member + w.first_segment_member + cursor.segment - 1;
                    const int64_t first = (int64_t(sequence) * args.kv_heads + kv_head) * (prefix ? args.prefix_capacity : args.own_capacity) + cursor.first_key(start_tile + j);
                    const int valid = cursor.keys(start_tile + j);
#pragma unroll
                    for (int i = 0; i < PA_KEYS; i += 32) {
                        // keys behind the end are not read: 0 takes their place
                        const int bytes = lane + i < valid ? 4 : 0;
                        const int64_t at = first + (lane + i < valid ? lane + i : 0);
                        const uint32_t slot = raw_scales + uint32_t(((j % PA_RAW_STAGES) * 2 * PA_KEYS + lane + i) * 4);
                        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(slot), "l"((prefix ? args.prefix_scales[0] : args.own_scales[0]) + at), "r"(bytes) : "memory");
                        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(slot + PA_KEYS * 4), "l"((prefix ? args.prefix_scales[1] : args.own_scales[1]) + at), "r"(bytes) : "memory");
                    }
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
            };
#pragma unroll 1
            for (int j = 0; j < PA_RAW_STAGES - 1; ++j) copy(j);
#pragma unroll 1
            for (int j = 0; j < num_tiles; ++j) {
                copy(j + PA_RAW_STAGES - 1);
                asm volatile("cp.async.wait_group %0;" ::"n"(PA_RAW_STAGES - 1) : "memory");
                const int stage = j % PA_SCALE_STAGES;
                pa_wait(scale_empty + 8 * stage, (uint32_t(j / PA_SCALE_STAGES) & 1u) ^ 1u, patience);
                const volatile float* raw = reinterpret_cast<const volatile float*>(generic + Shape::OFF_RAW_SCALES) + (j % PA_RAW_STAGES) * 2 * PA_KEYS + lane;
                uint32_t* out = reinterpret_cast<uint32_t*>(generic + Shape::OFF_SCALES) + stage * PA_SCALE_FLOATS;
                float vs[2];
                uint32_t not_finite[2], largest = 0u;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    vs[i] = raw[PA_KEYS + 32 * i];
                    const uint32_t bits = __float_as_uint(vs[i]) & 0x7fffffffu;
                    not_finite[i] = __ballot_sync(0xffffffffu, bits >= PA_SCALE_END);
                    if (bits >= PA_SCALE_END) vs[i] = 0.0f;
                    else largest = max(largest, bits);
                }
                largest = __reduce_max_sync(0xffffffffu, largest);
                // the unit 2^E: kept unless the tile's largest scale is outside [2^-3, 2^6) of it (a tile of zeros fits any).  It may fall by any
                // step, by which the accumulator grows; the smallest unit keeps that in fp32's range: values below 2^40 with weights of at most
                // 2^15 are below 2^103 units, and 2^24 keys of them below 2^127.  Scales from 2^-59 on are still 2^-11 of the smallest unit,
                // normal numbers of f16.
                const int exponent = int(largest >> 23) - 127, relative = exponent - unit_exponent;
                int change = 0;
                if (largest != 0u && (j == 0 || relative > 5 || relative < -3)) {
                    const int next = exponent < PA_UNIT_LEAST ? PA_UNIT_LEAST : exponent;
                    if (j > 0) change = unit_exponent - next;
                    unit_exponent = next;
                }
                const float up = __uint_as_float(uint32_t(127 - unit_exponent) << 23);          // 2^-E
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    out[lane + 32 * i] = __float_as_uint(raw[32 * i]);
                    const __half2 pair = __float2half2_rn(vs[i] * up);
                    out[PA_KEYS + lane + 32 * i] = *reinterpret_cast<const uint32_t*>(&pair);
                }
                if (lane == 0) {
                    out[2 * PA_KEYS] = not_finite[0];
                    out[2 * PA_KEYS + 1] = not_finite[1];
                    out[2 * PA_KEYS + 2] = uint32_t(unit_exponent);
                    out[2 * PA_KEYS + 3] = uint32_t(change);
                    if (Shape::SHARED) group_unit[0] = unit_exponent;
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(scale_full + 8 * stage);
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
        }
    }
    }

    if (patience == 0 && args.status != nullptr)
        atomicCAS(args.status, 0u, warp < 8 ? STATUS_WAIT_EPILOGUE : warp == PA_SCORES_WARP || warp == PA_OUTPUT_WARP ? STATUS_WAIT_MMA_FULL : STATUS_WAIT_PRODUCER);
    tc_fence_before_sync();
    __syncthreads();
    if (warp == PA_SCORES_WARP) {
        tc_fence_after_sync();
        tmem_dealloc(tmem_base, TMEM_COLUMNS);
    }
}

// out = sum_s 2^(M_s - M) O_s / sum_s 2^(M_s - M) L_s; D / 8 lanes per row, each with 8 columns.  The time is latency: everything that does
// not need another load's result is on its way before that result is waited for.
template <int D>
__global__ void __launch_bounds__(256) prefix_attention_join_kernel(const __grid_constant__ PaArgs args) {
    pdl_launch_dependents();
    constexpr int LANES = D / 8, PER_LANE = 64 / LANES, BATCH = 8;
    const int64_t index = (int64_t(blockIdx.x) * 256 + threadIdx.x) / LANES;
    const int lane = threadIdx.x % LANES;
    pdl_wait();
    const int2 cut = *reinterpret_cast<const int2*>(args.cut);
    const int64_t offset_and_sees = args.row_offsets[index], offset = offset_and_sees & ~int64_t(1);          // inside the table, whatever the cut
    const int64_t rows = int64_t(cut.x) * PA_ROWS;
    const int splits = cut.y;
    if (rows == 0) return;
    const bool there = index < rows && offset_and_sees >= 0;          // lanes without a row stay for the shuffles, on a row that is there
    const int64_t row = index < rows ? index : 0;
    const float2* statistics = reinterpret_cast<const float2*>(args.partial + int64_t(args.slots) * PA_ROWS * D) + row;
    const float* partial = args.partial + row * D + lane * 8;
    float2 entry[PER_LANE];          // of parts lane, lane + LANES, ..
#pragma unroll
    for (int i = 0; i < PER_LANE; ++i) {
        const int s = lane + i * LANES;
        entry[i] = there && s < splits ? statistics[s * rows] : make_float2(-INFINITY, 0.0f);
    }
    float4 a[BATCH], b[BATCH];
    auto load = [&](int first) {
#pragma unroll
        for (int n = 0; n < BATCH; ++n) {
            a[n] = b[n] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (there && first + n < splits) {
                a[n] = *reinterpret_cast<const float4*>(partial + (first + n) * rows * D);
                b[n] = *reinterpret_cast<const float4*>(partial + (first + n) * rows * D + 4);
            }
        }
    };
    load(0);
    float top = entry[0].x, total = 0.0f;
#pragma unroll
    for (int i = 1; i < PER_LANE; ++i) top = fmaxf(top, entry[i].x);
#pragma unroll
    for (int step = LANES / 2; step > 0; step >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, step));
    const float reference = top == -INFINITY ? 0.0f : top;
    float weight[PER_LANE];
#pragma unroll
    for (int i = 0; i < PER_LANE; ++i) {
        weight[i] = entry[i].y == 0.0f ? 0.0f : pa_exp2(entry[i].x - reference);      // sum 0: no visible key in this part, O is 0
        total = __fmaf_rn(weight[i], entry[i].y, total);
    }
#pragma unroll
    for (int step = LANES / 2; step > 0; step >>= 1) total += __shfl_xor_sync(0xffffffffu, total, step);
    float sum[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
    for (int first = 0; first < splits; first += BATCH) {
        if (first > 0) load(first);
#pragma unroll
        for (int n = 0; n < BATCH; ++n) {
            const int s = first + n;
            float mine = weight[0];
#pragma unroll
            for (int i = 1; i < PER_LANE; ++i) mine = s / LANES == i ? weight[i] : mine;
            const float w = __shfl_sync(0xffffffffu, mine, s % LANES, LANES);
            const float values[8] = {a[n].x, a[n].y, a[n].z, a[n].w, b[n].x, b[n].y, b[n].z, b[n].w};
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[i] = __fmaf_rn(w, values[i], sum[i]);
        }
    }
    if (!there) return;
    const float inverse = total == 0.0f ? ((offset_and_sees & 1) != 0 ? __uint_as_float(0x7fc00000u) : 0.0f) : 1.0f / total;
    *reinterpret_cast<uint4*>(args.out + offset + lane * 8) =
        make_uint4(float2_to_bf16x2(make_float2(sum[0] * inverse, sum[1] * inverse)), float2_to_bf16x2(make_float2(sum[2] * inverse, sum[3] * inverse)),
                   float2_to_bf16x2(make_float2(sum[4] * inverse, sum[5] * inverse)), float2_to_bf16x2(make_float2(sum[6] * inverse, sum[7] * inverse)));
}

struct PaPlan {
    int64_t items = 0;          // row tiles times key/value heads, at most
    int64_t ctas = 0;
    int slots = 0, max_splits = 1;
    int64_t bytes = 0;          // of workspace: the cut, row offsets, partial rows and their statistics
};

PaPlan pa_plan(const b2_prefix_attention_desc* d) {
    PaPlan plan;
    const int64_t per_member = int64_t(d->heads / d->kv_heads) * d->queries;
    const int64_t per_group = d->batch / d->groups;
    // unequal groups (their bounds are device data): n rows have 1 + (n - 1) / 128 tiles, and as many groups as can be have rows
    const int64_t filled = d->groups < d->batch ? d->groups : d->batch;
    const int64_t tiles = d->members == nullptr ? d->groups * ((per_group * per_member + PA_ROWS - 1) / PA_ROWS)
                                                : filled + (d->batch * per_member - filled) / PA_ROWS;
    // key tiles of a row tile: the prefix, and the own keys of the members that 128 rows can belong to
    int64_t sharing = (PA_ROWS + per_member - 2) / per_member + 1;
    if (d->members == nullptr && sharing > per_group) sharing = per_group;
    if (sharing > d->batch) sharing = d->batch;
    const int64_t key_tiles = (int64_t(d->prefix_capacity) + PA_KEYS - 1) / PA_KEYS + sharing * ((int64_t(d->own_capacity) + PA_KEYS - 1) / PA_KEYS);
    plan.items = tiles * d->kv_heads;
    const int64_t sms = sm_count(), uncut = plan.items > sms ? plan.items / sms * sms : 0, rest = plan.items - uncut;
    // The cut of what is behind the last whole wave, in 1/32 of a key tile's time (0.6 to 0.9 us): waves of CTAs times (set-up + tiles) --
    // looking up the work, fetching the queries and leaving the output take as long as 12 tiles -- and the join's launch and traffic.  At most
    // four waves of parts: their fp32 rows are 64 or 128 KB each.
    int64_t best = 0, splits = 1;
    for (int64_t s = 1; rest > 0 && s <= 64 && s <= key_tiles && (s == 1 || rest * s <= 4 * sms); ++s) {
        const int64_t waves = (rest * s + sms - 1) / sms;
        const int64_t cost = waves * (12 + (key_tiles + s - 1) / s) * 32 + (s > 1 ? 5 * 32 + 3 * rest * s : 0);
        if (best == 0 || cost < best) {
            best = cost;
            splits = s;
        }
    }
    plan.ctas = plan.items;
    if (splits > 1) {
        // fewer row tiles than the bound are cut finer, to two key tiles at least
        plan.slots = int(rest * splits);
        plan.max_splits = int(splits > key_tiles / 2 ? splits : key_tiles / 2);
        if (plan.max_splits > 64) plan.max_splits = 64;
        plan.ctas = uncut + plan.slots;
        plan.bytes = 32 + int64_t(plan.slots) * PA_ROWS * (4 + (d->head_dim + 2) * 4);
    }
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
        // the softmax warps' registers come out of those that the launch has
        cudaFuncAttributes attributes{};
        const cudaError_t found = cudaFuncGetAttributes(&attributes, prefix_attention_kernel<D, FP8>);
        if (found != cudaSuccess) return int(found);
        if (attributes.numRegs * Shape::THREADS < 256 * PA_SOFTMAX_REGISTERS + (Shape::THREADS - 256) * PA_OTHER_REGISTERS) return B2_E_UNSUPPORTED;
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
    const int status = launch_kernel(prefix_attention_kernel<D, FP8>, dim3(unsigned(plan.ctas)), dim3(Shape::THREADS), size_t(Shape::SHARED_BYTES), stream,
                                     prefix_k, prefix_v, own_k, own_v, args);
    if (status != B2_OK || plan.slots == 0) return status;
    const int64_t rows = (plan.items < plan.slots / 2 ? plan.items : plan.slots / 2) * PA_ROWS;          // a row tile that is cut has two parts at least
    return launch_kernel(prefix_attention_join_kernel<D>, dim3(unsigned((rows * (D / 8) + 255) / 256)), dim3(256), size_t(0), stream, args);
}

}  // namespace

int64_t prefix_attention_workspace(const b2_prefix_attention_desc* desc) { return pa_plan(desc).bytes; }

int launch_prefix_attention(const b2_prefix_attention_desc* desc, cudaStream_t stream) {
    PaPlan plan = pa_plan(desc);
    if (plan.bytes > 0 && (desc->workspace == nullptr || desc->workspace_bytes < plan.bytes)) {
        plan.slots = 0;          // nothing is cut
        plan.ctas = plan.items;
    }
    if (plan.ctas * PA_ROWS >= (int64_t(1) << 31)) return B2_E_TOO_LARGE;
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
    if (plan.slots > 0) {
        uint8_t* const workspace = static_cast<uint8_t*>(desc->workspace);
        args.cut = reinterpret_cast<int32_t*>(workspace);
        args.row_offsets = reinterpret_cast<int64_t*>(workspace + 32);
        args.partial = reinterpret_cast<float*>(workspace + 32 + int64_t(plan.slots) * PA_ROWS * 4);
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
    args.share = desc->heads / desc->kv_heads;
    args.rows_per_member = args.share * desc->queries;
    args.sms = sm_count();
    args.slots = plan.slots;
    args.max_splits = plan.slots > 0 ? plan.max_splits : 1;
    args.causal = (desc->flags & B2_ATTENTION_CAUSAL) != 0;
    if (desc->head_dim == 256)
        return desc->cache_bits == 8 ? pa_launch<256, true>(desc, plan, args, stream) : pa_launch<256, false>(desc, plan, args, stream);
    return desc->cache_bits == 8 ? pa_launch<128, true>(desc, plan, args, stream) : pa_launch<128, false>(desc, plan, args, stream);
}

}  // namespace b2
