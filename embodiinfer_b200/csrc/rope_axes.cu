// Sine / cosine tables of rotary positions with several axes (time, height, width; one axis is the ordinary table).
//
//   frequency i belongs to axis a(i): the axes' sections follow one another over the head_dim / 2 frequencies
//   f_i = theta^(-i / half)            one spectrum shared by the axes, or
//   f_i = theta^(-j / section)         a spectrum of its own for each axis, j counted inside its section
//   sine[t, i] = sin(position[a(i), t] f_i), cosine likewise, fp32
//
// Angles are counted in turns and in whole numbers: a frequency is held as the fraction of f / 2 pi in 64 bits (2^64 = one turn), and
// position * fraction modulo 2^64 is the angle's fraction of a turn.  The product loses nothing, however far the position (a video's
// 2.6e5th frame at f = 1 has no fraction left in fp32); the error is the position times the frequency's own, which is formed in
// fp64 to a few 2^-53 of itself: at most some 2^-30 of a turn at position 2^20, 2^-10 at 2^40.  The top bits name the quadrant, the rest, in
// [-1/8, 1/8) turns, goes to fp32 (an error of 2^-28 turns, 2.3e-8) and into the Taylor series of sine (to the 9th power) and cosine
// (to the 10th), both at once on the packed fp32 pipe.
//
// Each thread keeps the frequencies of VECTOR neighbouring columns and walks down the tokens: one 16-byte store per table
// and token.  Measured (B200): 8 x 16384 positions, head dimension 128, 14.9 us (70 MB, 4.7 TB/s), bound by the stores: without the
// series it takes no less.  Stores that leave the L2 first (kept there 16.0 us); as many blocks as fit at once, for the frequencies are
// formed once per block (two waves of them 17.5 us); 40 registers 18.1, eight columns per thread 25; angles in fp64 and the library's
// sincospif 24.
#include "common.cuh"

namespace b2 {

namespace {

constexpr int AXES_THREADS = 256;

struct AxesArgs {
    const void* positions;
    float* sine;
    float* cosine;
    double log2_step[4], step[4];      // of an axis: frequencies are 2^-log2_step, `step`, apart
    int64_t tokens;
    int32_t section[4];
    int32_t axes, half, own_spectrum;
};

// Sine and cosine of `angle` / 2^64 turns.
__device__ __forceinline__ void sincos_turns(uint64_t angle, float& sine, float& cosine) {
    const uint32_t high = uint32_t(angle >> 32), quadrant = (high + 0x20000000u) >> 30;
    const float r = __fmaf_rn(float(uint32_t(angle)), 5.4210108624275222e-20f, float(int32_t(high - (quadrant << 30))) * 2.3283064365386963e-10f);
    const float z = r * r;
    // (2 pi)^n / n! with alternating signs: n = 9, 7, 5, 3, 1 and 10, 8, 6, 4, 2, 0
    const float2 z2 = make_float2(z, z);
    float2 sum = make_float2(42.058693944897634f, __fmaf_rn(z, -26.426256783374388f, 60.244641371876661f));
    sum = __ffma2_rn(sum, z2, make_float2(-76.705859753061360f, -85.456817206693727f));
    sum = __ffma2_rn(sum, z2, make_float2(81.605249276075040f, 64.939394022668292f));
    sum = __ffma2_rn(sum, z2, make_float2(-41.341702240399755f, -19.739208802178717f));
    sum = __ffma2_rn(sum, z2, make_float2(6.2831853071795865f, 1.0f));
    const float s = sum.x * r;
    const bool swapped = (quadrant & 1u) != 0;
    sine = __uint_as_float(__float_as_uint(swapped ? sum.y : s) ^ ((quadrant & 2u) << 30));
    cosine = __uint_as_float(__float_as_uint(swapped ? s : sum.y) ^ (((quadrant + 1u) & 2u) << 30));
}

template <typename Position, int VECTOR>
__global__ void __launch_bounds__(AXES_THREADS) rope_axes_kernel(const __grid_constant__ AxesArgs args, int columns_per_row, int rows_per_block,
                                                                 int64_t row_step) {
    pdl_launch_dependents();
    const int column = (blockIdx.y * columns_per_row + int(threadIdx.x) % columns_per_row) * VECTOR;
    const int row = int(threadIdx.x) / columns_per_row;
    if (row >= rows_per_block || column >= args.half) return;
    uint64_t frequency[VECTOR];          // turns of one position, as a fraction of 2^64
    const Position* source[VECTOR];
    double turns = 0.0;
#pragma unroll
    for (int v = 0; v < VECTOR; ++v) {
        const int i = column + v;
        int axis = 0, start = 0;
        while (axis + 1 < args.axes && i >= start + args.section[axis]) start += args.section[axis++];
        // neighbours are one ratio apart; an axis' own spectrum begins with 1
        const int power = args.own_spectrum ? i - start : i;
        if (v == 0) turns = exp2(-double(power) * args.log2_step[axis]) * 0.15915494309189535;      // 1 / (2 pi)
        else turns = power == 0 ? 0.15915494309189535 : turns * args.step[axis];
        frequency[v] = uint64_t(__double2ll_rn((turns - rint(turns)) * 18446744073709551616.0));
        source[v] = static_cast<const Position*>(args.positions) + int64_t(axis) * args.tokens;
    }
    bool one_axis = true;
#pragma unroll
    for (int v = 1; v < VECTOR; ++v) one_axis = one_axis && source[v] == source[0];
    pdl_wait();
    int64_t t = int64_t(blockIdx.x) * rows_per_block + row;
    Position position[VECTOR];
    auto load = [&](int64_t at) {
        position[0] = __ldg(source[0] + at);
        if (!one_axis) {
#pragma unroll
            for (int v = 1; v < VECTOR; ++v) position[v] = __ldg(source[v] + at);
        } else {
#pragma unroll
            for (int v = 1; v < VECTOR; ++v) position[v] = position[0];
        }
    };
    if (t < args.tokens) load(t);
    while (t < args.tokens) {
        uint64_t angle[VECTOR];
#pragma unroll
        for (int v = 0; v < VECTOR; ++v) angle[v] = uint64_t(int64_t(position[v])) * frequency[v];
        const int64_t out = t * args.half + column;
        t += row_step;
        if (t < args.tokens) load(t);          // the next row's, while this one is computed
        float s[VECTOR], c[VECTOR];
#pragma unroll
        for (int v = 0; v < VECTOR; ++v) sincos_turns(angle[v], s[v], c[v]);
        if (VECTOR == 4) {
            __stcs(reinterpret_cast<float4*>(args.sine + out), make_float4(s[0], s[1 % VECTOR], s[2 % VECTOR], s[3 % VECTOR]));
            __stcs(reinterpret_cast<float4*>(args.cosine + out), make_float4(c[0], c[1 % VECTOR], c[2 % VECTOR], c[3 % VECTOR]));
        } else {
            args.sine[out] = s[0];
            args.cosine[out] = c[0];
        }
    }
}

}  // namespace

int launch_rope_axes(const void* positions, int position_bytes, const int32_t* sections, int axes, int64_t tokens, int head_dim,
                     double theta, int own_spectrum, void* sine, void* cosine, cudaStream_t stream) {
    AxesArgs args{};
    args.positions = positions;
    args.sine = static_cast<float*>(sine);
    args.cosine = static_cast<float*>(cosine);
    args.tokens = tokens;
    for (int a = 0; a < axes; ++a) {
        args.section[a] = sections[a];
        args.log2_step[a] = log2(theta) / (own_spectrum ? sections[a] : head_dim / 2);
        args.step[a] = exp2(-args.log2_step[a]);
    }
    args.axes = axes;
    args.half = head_dim / 2;
    args.own_spectrum = own_spectrum;
    // 16-byte stores when every row of the tables starts on 16 bytes
    const uintptr_t outputs = reinterpret_cast<uintptr_t>(sine) | reinterpret_cast<uintptr_t>(cosine);
    const bool vectors = args.half % 4 == 0 && (outputs & 15u) == 0;
    const int columns = vectors ? args.half / 4 : args.half;
    const int columns_per_row = columns < AXES_THREADS ? columns : AXES_THREADS;
    const int rows_per_block = AXES_THREADS / columns_per_row;
    const unsigned planes = unsigned((columns + columns_per_row - 1) / columns_per_row);
    const int64_t wanted = (tokens + rows_per_block - 1) / rows_per_block, cap = int64_t(sm_count()) * 5;      // what the registers let run at once
    const int64_t blocks = wanted < cap ? wanted : cap;
    const dim3 grid(unsigned(blocks), planes), block(AXES_THREADS);
    const int64_t step = blocks * rows_per_block;
    if (position_bytes == 8)
        return vectors ? launch_kernel(rope_axes_kernel<int64_t, 4>, grid, block, size_t(0), stream, args, columns_per_row, rows_per_block, step)
                       : launch_kernel(rope_axes_kernel<int64_t, 1>, grid, block, size_t(0), stream, args, columns_per_row, rows_per_block, step);
    return vectors ? launch_kernel(rope_axes_kernel<int32_t, 4>, grid, block, size_t(0), stream, args, columns_per_row, rows_per_block, step)
                   : launch_kernel(rope_axes_kernel<int32_t, 1>, grid, block, size_t(0), stream, args, columns_per_row, rows_per_block, step);
}

}  // namespace b2
