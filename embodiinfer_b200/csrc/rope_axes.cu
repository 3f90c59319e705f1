// Sine / cosine tables of rotary positions with several axes (time, height, width; one axis is the ordinary table).
//
//   frequency i belongs to axis a(i): the axes' sections follow one another over the head_dim / 2 frequencies
//   f_i = theta^(-i / half)            one spectrum shared by the axes, or
//   f_i = theta^(-j / section)         a spectrum of its own for each axis, j counted inside its section
//   sine[t, i] = sin(position[a(i), t] f_i), cosine likewise, fp32
//
// Angles of far positions (a video's 2.6e5th frame at f = 1) have no fraction left in fp32, so the angle is counted in whole
// turns in 64 bits -- position * (f / 2 pi), of which only the fraction goes on to fp32 -- and sine and cosine are
// sincospif of twice the fraction: no range reduction by a rounded pi.  Rounding the fraction to fp32 moves the angle by at most
// pi 2^-25 (9e-8), about the rounding of the result.
//
// Each thread keeps the frequencies of VECTOR neighbouring columns and walks down the tokens: one 16-byte store per table
// and token, bound by those stores.
#include "common.cuh"

namespace b2 {

namespace {

constexpr int AXES_THREADS = 256;

struct AxesArgs {
    const void* positions;
    float* sine;
    float* cosine;
    double log2_theta;
    int64_t tokens;
    int32_t section[4];
    int32_t axes, half, own_spectrum;
};

template <typename Position, int VECTOR>
__global__ void __launch_bounds__(AXES_THREADS) rope_axes_kernel(const __grid_constant__ AxesArgs args, int columns_per_row, int rows_per_block,
                                                                 int64_t row_step) {
    pdl_launch_dependents();
    const int column = int(threadIdx.x) % columns_per_row;
    const int row = int(threadIdx.x) / columns_per_row;
    double turns[VECTOR];
    const Position* source[VECTOR];
#pragma unroll
    for (int v = 0; v < VECTOR; ++v) {
        const int i = (blockIdx.y * columns_per_row + column) * VECTOR + v;
        int axis = 0, start = 0;
        while (axis + 1 < args.axes && i >= start + args.section[axis]) start += args.section[axis++];
        const double power = args.own_spectrum ? double(i - start) / double(args.section[axis]) : double(i) / double(args.half);
        turns[v] = exp2(-power * args.log2_theta) * 0.15915494309189535;      // 1 / (2 pi)
        source[v] = static_cast<const Position*>(args.positions) + int64_t(axis) * args.tokens;
    }
    if (row >= rows_per_block || (blockIdx.y * columns_per_row + column) * VECTOR >= args.half) return;
    pdl_wait();
    for (int64_t t = int64_t(blockIdx.x) * rows_per_block + row; t < args.tokens; t += row_step) {
        float s[VECTOR], c[VECTOR];
        Position position[VECTOR];
        position[0] = __ldg(source[0] + t);
#pragma unroll
        for (int v = 1; v < VECTOR; ++v) position[v] = source[v] == source[0] ? position[0] : __ldg(source[v] + t);
#pragma unroll
        for (int v = 0; v < VECTOR; ++v) {
            const double u = double(position[v]) * turns[v];
            sincospif(2.0f * float(u - rint(u)), &s[v], &c[v]);
        }
        const int64_t out = t * args.half + int64_t(blockIdx.y * columns_per_row + column) * VECTOR;
        if (VECTOR == 4) {
            *reinterpret_cast<float4*>(args.sine + out) = make_float4(s[0], s[1 % VECTOR], s[2 % VECTOR], s[3 % VECTOR]);
            *reinterpret_cast<float4*>(args.cosine + out) = make_float4(c[0], c[1 % VECTOR], c[2 % VECTOR], c[3 % VECTOR]);
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
    args.log2_theta = log2(theta);
    args.tokens = tokens;
    for (int a = 0; a < axes; ++a) args.section[a] = sections[a];
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
    const int64_t wanted = (tokens + rows_per_block - 1) / rows_per_block, cap = int64_t(sm_count()) * 8;
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
