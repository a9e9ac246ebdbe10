// The passes around a dense product, each bound by memory: rows of bf16 that the tile kernel's 128-bit loads cannot take copied
// to ones they can, and deltaZ = deltaY * act'(Z) with its column sums (fp32 SiLU 4992 x 2496 28 us, 5.3 TB/s; GELU 12544 x 1024 36 us,
// 4.3 TB/s; bf16 SiLU 8192 x 4096 47 us, 4.3 TB/s).
// A bf16 call stores deltaZ in bf16, as the products' operand is on the matrix pipe: each element off by half a step, 2^-8 at most, so
// deltaX and deltaW are off by 0.0023 of their rms instead of the 0.0017 that their own rounding leaves. Two bf16 parts would keep the
// difference and double both products (410 of the 466 us of 8192 x 4096 -> 4096). The column sums are of the unrounded values.
#include "dense_common.hpp"

#include <algorithm>
#include <type_traits>

namespace alpha {

namespace {

// Eight consecutive elements of a row, c .. c+7 of `cols`, whatever their alignment. Not WHOLE: the row ends before the eighth, whose
// place the last element takes again. (No branch around a load: those would wait for each other, 115 x 833 of fp32 20 us.)
template <bool WHOLE, typename T>
__device__ __forceinline__ void load8(const T *row, int c, int cols, T (&v)[8])
{
    if constexpr (WHOLE) {
        __builtin_memcpy(v, row + c, 8 * sizeof(T));
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = row[c + e < cols ? c + e : cols - 1];
    }
}

// eight elements at an address aligned to 16 bytes
template <typename T>
__device__ __forceinline__ void store8(T *dst, const float (&v)[8])
{
    if constexpr (sizeof(T) == 2) {
        bf16x8 t;
#pragma unroll
        for (int e = 0; e < 8; e++) t[e] = (__bf16)v[e];
        *reinterpret_cast<bf16x8 *>(dst) = t;
    } else {
        quad_store(dst, floatx4{v[0], v[1], v[2], v[3]});
        quad_store(dst + 4, floatx4{v[4], v[5], v[6], v[7]});
    }
}

}  // namespace

template <typename T>
__global__ __launch_bounds__(256) void dense_pack_kernel(const T *__restrict__ src, long src_ld, long total, int cols, T *__restrict__ dst,
                                                         long ld, FastDiv d_chunks)
{
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long)gridDim.x * 256) {
        const long row = fdiv((uint32_t)i, d_chunks);
        const int c = (int)(i - row * d_chunks.d) * 8;
        T t[8];
        if (c + 8 <= cols) load8<true>(src + row * src_ld, c, cols, t);
        else load8<false>(src + row * src_ld, c, cols, t);
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = c + e < cols ? (float)t[e] : 0.f;
        store8(dst + row * ld + c, v);
    }
}

namespace {

template <typename T>
hipError_t launch_pack(hipStream_t s, const void *src, long src_ld, long total, int cols, void *dst, long ld)
{
    const dim3 grid((unsigned)std::min<long>((total + 255) / 256, 16384));
    const FastDiv d = make_fastdiv((uint32_t)(ld / 8));
    const T *p = static_cast<const T *>(src);
    hipLaunchKernelGGL((dense_pack_kernel<T>), grid, dim3(256), 0, s, p, src_ld, total, cols, static_cast<T *>(dst), ld, d);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_dense_pack(hipStream_t s, int f32, const void *src, long src_ld, long rows, int cols, void *dst, long ld)
{
    const long total = rows * (ld / 8);
    if (total <= 0) return hipSuccess;
    if (total >= (1l << 31)) return hipErrorInvalidValue;
    return f32 ? launch_pack<float>(s, src, src_ld, total, cols, dst, ld) : launch_pack<__bf16>(s, src, src_ld, total, cols, dst, ld);
}

constexpr int DELTA_ROWS = 4;

// A workgroup takes 256 columns (32 lanes of 8) of a run of rows, eight rows side by side - or, where that makes few workgroups, 64
// columns and 32 rows; its column sums go to sums[run], or, of a single run, where they are wanted. The lane at the end of a row
// takes the row's last eight elements and leaves out those that its neighbour has (115 x 833 of fp32: 20.5 us element by element,
// 7.0 so). LANES = 1: rows of less than eight.
// (A kernel per activation: with all of them behind a switch the code was 17 to 44 KB, and a small call the time of fetching it.)
template <typename T, bool GATED, int LANES, int ACT>
__global__ __launch_bounds__(256) void dense_delta_kernel(const DenseDelta d, long rows_per)
{
    constexpr int ROWS = LANES == 1 ? 1 : DELTA_ROWS;
    constexpr int SIDE = 256 / LANES, COLS = LANES * 8;       // rows side by side, columns
    __shared__ float part[GATED ? 2 : 1][SIDE][COLS + 1];
    const int lane = threadIdx.x % LANES, ry = threadIdx.x / LANES, c = (blockIdx.x * LANES + lane) * 8;
    const int at = LANES == 1 || c + 8 <= d.cols ? c : d.cols - 8, skip = c - at;      // columns at + skip .. at + 7 are the lane's
    const long r0 = (long)blockIdx.y * rows_per, r1 = r0 + rows_per < d.rows ? r0 + rows_per : d.rows;
    float sum[8], sum2[8];
#pragma unroll
    for (int e = 0; e < 8; e++) sum[e] = sum2[e] = 0.f;
    if (c < d.ld) {
        auto load = [&](const void *p, long ld, long row, T (&v)[8]) __attribute__((always_inline)) {
            const T *from = static_cast<const T *>(p) + row * ld + at;
            if constexpr (LANES == 1) {
#pragma unroll
                for (int e = 0; e < 8; e++) v[e] = from[e < d.cols ? e : d.cols - 1];
            } else {
                __builtin_memcpy(v, from, 8 * sizeof(T));
            }
        };
        auto store = [&](void *p, long row, const float (&v)[8]) __attribute__((always_inline)) {
            T *to = static_cast<T *>(p) + row * d.ld2;
            if (LANES > 1 && skip == 0) {
                store8(to + at, v);
                return;
            }
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (e >= skip && at + e < d.cols) dense_store(to + at + e, v[e]);
            for (int x = d.cols; x < d.ld; x++) dense_store(to + x, 0.f);              // pad columns
        };
        // ROWS rows of a lane at a time: their loads first, then the arithmetic
        for (long r = r0 + ry; r < r1; r += SIDE * ROWS) {
            T dy[ROWS][8], z[ROWS][8], u[ROWS][8];
#pragma unroll
            for (int y = 0; y < ROWS; y++) {
                const long row = r + SIDE * y < r1 ? r + SIDE * y : r;
                load(d.dY, d.ldY, row, dy[y]);
                if (GATED || ACT != ALPHA_DENSE_ACT_NONE) load(d.Z, d.ldZ, row, z[y]);
                if constexpr (GATED) load(d.U, d.ldU, row, u[y]);
            }
#pragma unroll
            for (int y = 0; y < ROWS; y++) {
                const long row = r + SIDE * y;
                if (row >= r1) break;
                float out[8], out2[8];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    out[e] = (float)dy[y][e];
                    if constexpr (GATED) {
                        out2[e] = out[e] * dense_act<T>(ACT, (float)z[y][e], d.slope);
                        out[e] *= (float)u[y][e] * dense_act_slope<T>(ACT, (float)z[y][e], d.slope);
                        sum2[e] += out2[e];
                    } else if (ACT != ALPHA_DENSE_ACT_NONE) {
                        out[e] *= dense_act_slope<T>(ACT, (float)z[y][e], d.slope);
                    }
                    sum[e] += out[e];
                }
                if (d.dst) store(d.dst, row, out);
                if constexpr (GATED)
                    if (d.dst2) store(d.dst2, row, out2);
            }
        }
    }
    if (!d.dB && !d.dB2) return;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        if (e < skip) continue;
        part[0][ry][lane * 8 + e - skip] = sum[e];
        if constexpr (GATED) part[1][ry][lane * 8 + e - skip] = sum2[e];
    }
    __syncthreads();
    const int col = blockIdx.x * COLS + threadIdx.x;
    if (threadIdx.x >= COLS || col >= d.cols) return;
#pragma unroll
    for (int w = 0; w < (GATED ? 2 : 1); w++) {
        float t = 0.f;
#pragma unroll
        for (int y = 0; y < SIDE; y++) t += part[w][y][threadIdx.x];
        if (gridDim.y > 1) {
            d.sums[((long)blockIdx.y * (GATED ? 2 : 1) + w) * d.cols + col] = t;
        } else if (void *dB = w ? d.dB2 : d.dB) {   // one run: the sums are final
            dense_store(static_cast<T *>(dB) + col, t);
        }
    }
}

// dB[col] = sum over the runs, in a fixed order: 16 lanes a column, each its share of the runs.
template <typename T>
__global__ __launch_bounds__(256) void dense_delta_sum_kernel(const float *__restrict__ sums, int runs, int cols, int which, int of, T *__restrict__ dB)
{
    __shared__ float part[16][17];
    const int cx = threadIdx.x & 15, ry = threadIdx.x >> 4, col = blockIdx.x * 16 + cx;
    float t = 0.f;
    if (col < cols)
#pragma unroll 4
        for (int r = ry; r < runs; r += 16) t += sums[((long)r * of + which) * cols + col];
    part[ry][cx] = t;
    __syncthreads();
    if (ry == 0 && col < cols) {
        t = 0.f;
#pragma unroll
        for (int y = 0; y < 16; y++) t += part[y][cx];
        dense_store(dB + col, t);
    }
}

namespace {

// Runs of rows: enough workgroups for the device, whole turns of 8 * DELTA_ROWS rows, at most 256 (a run costs a row of sums); up
// to four turns one run, whose sums need no second kernel.
long delta_rows_per(long rows, int cols)
{
    const long turn = 8 * DELTA_ROWS;
    if (rows <= 4 * turn) return std::max<long>(1, rows);
    const long blocks_x = (cols + 255) / 256, want = std::max<long>(1, 2048 / std::max<long>(1, blocks_x));
    const long runs = std::min<long>(256, std::max<long>(1, std::min(want, rows / turn))), per = (rows + runs - 1) / runs;
    return (per + turn - 1) / turn * turn;
}

template <typename T, bool GATED, int LANES>
void launch_delta_act(hipStream_t s, const DenseDelta &d, int runs, long rows_per)
{
    const dim3 grid((unsigned)((d.ld + 8 * LANES - 1) / (8 * LANES)), (unsigned)runs);
    auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, d, rows_per); };
    switch (d.act) {
    case ALPHA_DENSE_ACT_LEAKY_RELU: launch(dense_delta_kernel<T, GATED, LANES, ALPHA_DENSE_ACT_LEAKY_RELU>); break;
    case ALPHA_DENSE_ACT_GELU: launch(dense_delta_kernel<T, GATED, LANES, ALPHA_DENSE_ACT_GELU>); break;
    case ALPHA_DENSE_ACT_SILU: launch(dense_delta_kernel<T, GATED, LANES, ALPHA_DENSE_ACT_SILU>); break;
    case ALPHA_DENSE_ACT_SIGMOID: launch(dense_delta_kernel<T, GATED, LANES, ALPHA_DENSE_ACT_SIGMOID>); break;
    default: launch(dense_delta_kernel<T, GATED, LANES, ALPHA_DENSE_ACT_NONE>); break;
    }
}

template <typename T>
hipError_t launch_delta_typed(hipStream_t s, const DenseDelta &d, long rows_per, int runs)
{
    if (runs > 0) {
        const bool narrow = (d.ld + 255) / 256 * runs < 2l * device_cu_count();
        if (d.cols < 8) d.gated ? launch_delta_act<T, true, 1>(s, d, runs, rows_per) : launch_delta_act<T, false, 1>(s, d, runs, rows_per);
        else if (d.gated) narrow ? launch_delta_act<T, true, 8>(s, d, runs, rows_per) : launch_delta_act<T, true, 32>(s, d, runs, rows_per);
        else narrow ? launch_delta_act<T, false, 8>(s, d, runs, rows_per) : launch_delta_act<T, false, 32>(s, d, runs, rows_per);
    }
    if (runs == 1) return hipGetLastError();
    const dim3 cols((unsigned)((d.cols + 15) / 16));
    const int of = d.gated ? 2 : 1;
    if (d.dB) hipLaunchKernelGGL((dense_delta_sum_kernel<T>), cols, dim3(256), 0, s, d.sums, runs, d.cols, 0, of, static_cast<T *>(d.dB));
    if (d.dB2) hipLaunchKernelGGL((dense_delta_sum_kernel<T>), cols, dim3(256), 0, s, d.sums, runs, d.cols, 1, of, static_cast<T *>(d.dB2));
    return hipGetLastError();
}

}  // namespace

size_t dense_delta_sum_bytes(long rows, int cols, int gated)
{
    if (rows <= 0 || cols <= 0) return 0;
    const long per = delta_rows_per(rows, cols), runs = (rows + per - 1) / per;
    return runs > 1 ? (size_t)runs * cols * (gated ? 2 : 1) * 4 : 0;
}

hipError_t launch_dense_delta(hipStream_t s, const DenseDelta &given)
{
    DenseDelta d = given;
    if (d.cols <= 0) return hipSuccess;
    const long per = delta_rows_per(d.rows, d.cols), runs = d.rows > 0 ? (d.rows + per - 1) / per : 0;
    return d.f32 ? launch_delta_typed<float>(s, d, per, (int)runs) : launch_delta_typed<__bf16>(s, d, per, (int)runs);
}

}  // namespace alpha
