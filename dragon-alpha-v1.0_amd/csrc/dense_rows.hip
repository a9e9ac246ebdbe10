// The passes around a dense product, each bound by memory: rows of bf16 that the tile kernel's 128-bit loads cannot take copied
// to ones they can, and deltaZ = deltaY * act'(Z) with its column sums.
#include "dense_common.hpp"

#include <algorithm>

namespace alpha {

namespace {

// Eight consecutive elements of a row, c .. c+7 of `cols`; the rest zeros. VEC: rows begin at multiples of four elements (128-bit
// loads take an 8-byte address).
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T *row, int c, int cols, float (&v)[8])
{
    if (VEC && c + 8 <= cols) {
        if constexpr (sizeof(T) == 2) {
            bf16x8 t;
            __builtin_memcpy(&t, __builtin_assume_aligned(row + c, 8), 16);
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = (float)t[e];
        } else {
            const floatx4 lo = quad_load(row + c), hi = quad_load(row + c + 4);
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = lo[e], v[4 + e] = hi[e];
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = c + e < cols ? dense_load(row + c + e) : 0.f;
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

template <typename T, bool VEC>
__global__ __launch_bounds__(256) void dense_pack_kernel(const T *__restrict__ src, long src_ld, long total, int cols, T *__restrict__ dst,
                                                         long ld, FastDiv d_chunks)
{
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long)gridDim.x * 256) {
        const long row = fdiv((uint32_t)i, d_chunks);
        const int c = (int)(i - row * d_chunks.d) * 8;
        float v[8];
        load8<T, VEC>(src + row * src_ld, c, cols, v);
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
    if ((reinterpret_cast<uintptr_t>(src) & (4 * sizeof(T) - 1)) == 0 && (src_ld & 3) == 0)
        hipLaunchKernelGGL((dense_pack_kernel<T, true>), grid, dim3(256), 0, s, p, src_ld, total, cols, static_cast<T *>(dst), ld, d);
    else
        hipLaunchKernelGGL((dense_pack_kernel<T, false>), grid, dim3(256), 0, s, p, src_ld, total, cols, static_cast<T *>(dst), ld, d);
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

// A workgroup takes 256 columns (32 lanes of 8) of a run of rows, eight rows side by side; its column sums go to sums[run], or, of
// a single run, where they are wanted.
// (A kernel per activation: with all of them behind a switch the code was 17 to 44 KB, and a small call the time of fetching it.)
template <typename T, bool VEC, bool GATED, int ACT>
__global__ __launch_bounds__(256) void dense_delta_kernel(const DenseDelta d, long rows_per)
{
    constexpr int ROWS = sizeof(T) == 4 && ACT == ALPHA_DENSE_ACT_GELU ? 2 : DELTA_ROWS;   // (erf is long)
    __shared__ float part[GATED ? 2 : 1][8][257];
    const int lane = threadIdx.x & 31, ry = threadIdx.x >> 5, c = (blockIdx.x * 32 + lane) * 8;
    const long r0 = (long)blockIdx.y * rows_per, r1 = r0 + rows_per < d.rows ? r0 + rows_per : d.rows;
    float sum[8], sum2[8];
#pragma unroll
    for (int e = 0; e < 8; e++) sum[e] = sum2[e] = 0.f;
    if (c < d.ld) {
        // ROWS rows of a lane at a time: their loads first, then the arithmetic
        for (long r = r0 + ry; r < r1; r += 8 * ROWS) {
            float dy[ROWS][8], z[ROWS][8], u[ROWS][8];
#pragma unroll
            for (int y = 0; y < ROWS; y++) {
                const long row = r + 8 * y < r1 ? r + 8 * y : r;
                load8<T, VEC>(static_cast<const T *>(d.dY) + row * d.ldY, c, d.cols, dy[y]);
                if (GATED || ACT != ALPHA_DENSE_ACT_NONE) load8<T, VEC>(static_cast<const T *>(d.Z) + row * d.ldZ, c, d.cols, z[y]);
                if constexpr (GATED) load8<T, VEC>(static_cast<const T *>(d.U) + row * d.ldU, c, d.cols, u[y]);
            }
#pragma unroll
            for (int y = 0; y < ROWS; y++) {
                const long row = r + 8 * y;
                if (row >= r1) break;
                float out2[8];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    if (c + e >= d.cols) {   // pad columns: zeros, whatever act(0) is
                        dy[y][e] = out2[e] = 0.f;
                    } else if constexpr (GATED) {
                        out2[e] = dy[y][e] * dense_act<T>(ACT, z[y][e], d.slope);
                        dy[y][e] *= u[y][e] * dense_act_slope<T>(ACT, z[y][e], d.slope);
                    } else if (ACT != ALPHA_DENSE_ACT_NONE) {
                        dy[y][e] *= dense_act_slope<T>(ACT, z[y][e], d.slope);
                    }
                    sum[e] += dy[y][e];
                    if constexpr (GATED) sum2[e] += out2[e];
                }
                if (d.dst) store8(static_cast<T *>(d.dst) + row * d.ld2 + c, dy[y]);
                if constexpr (GATED)
                    if (d.dst2) store8(static_cast<T *>(d.dst2) + row * d.ld2 + c, out2);
            }
        }
    }
    if (!d.dB && !d.dB2) return;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        part[0][ry][lane * 8 + e] = sum[e];
        if constexpr (GATED) part[1][ry][lane * 8 + e] = sum2[e];
    }
    __syncthreads();
    const int col = blockIdx.x * 256 + threadIdx.x;
    if (col >= d.cols) return;
#pragma unroll
    for (int w = 0; w < (GATED ? 2 : 1); w++) {
        float t = 0.f;
#pragma unroll
        for (int y = 0; y < 8; y++) t += part[w][y][threadIdx.x];
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
// to two turns one run, whose sums need no second kernel.
long delta_rows_per(long rows, int cols)
{
    const long turn = 8 * DELTA_ROWS;
    if (rows <= 2 * turn) return std::max<long>(1, rows);
    const long blocks_x = (cols + 255) / 256, want = std::max<long>(1, 2048 / std::max<long>(1, blocks_x));
    const long runs = std::min<long>(256, std::max<long>(1, std::min(want, rows / turn))), per = (rows + runs - 1) / runs;
    return (per + turn - 1) / turn * turn;
}

template <typename T, bool VEC, bool GATED>
void launch_delta_act(hipStream_t s, const DenseDelta &d, dim3 grid, long rows_per)
{
    switch (d.act) {
    case ALPHA_DENSE_ACT_LEAKY_RELU: hipLaunchKernelGGL((dense_delta_kernel<T, VEC, GATED, ALPHA_DENSE_ACT_LEAKY_RELU>), grid, dim3(256), 0, s, d, rows_per); break;
    case ALPHA_DENSE_ACT_GELU: hipLaunchKernelGGL((dense_delta_kernel<T, VEC, GATED, ALPHA_DENSE_ACT_GELU>), grid, dim3(256), 0, s, d, rows_per); break;
    case ALPHA_DENSE_ACT_SILU: hipLaunchKernelGGL((dense_delta_kernel<T, VEC, GATED, ALPHA_DENSE_ACT_SILU>), grid, dim3(256), 0, s, d, rows_per); break;
    case ALPHA_DENSE_ACT_SIGMOID: hipLaunchKernelGGL((dense_delta_kernel<T, VEC, GATED, ALPHA_DENSE_ACT_SIGMOID>), grid, dim3(256), 0, s, d, rows_per); break;
    default: hipLaunchKernelGGL((dense_delta_kernel<T, VEC, GATED, ALPHA_DENSE_ACT_NONE>), grid, dim3(256), 0, s, d, rows_per); break;
    }
}

template <typename T>
hipError_t launch_delta_typed(hipStream_t s, const DenseDelta &d, bool vec, long rows_per, int runs)
{
    const dim3 grid((unsigned)((d.ld + 255) / 256), (unsigned)std::max(runs, 1));
    if (runs > 0) {
        if (d.gated) {
            if (vec) launch_delta_act<T, true, true>(s, d, grid, rows_per);
            else launch_delta_act<T, false, true>(s, d, grid, rows_per);
        } else {
            if (vec) launch_delta_act<T, true, false>(s, d, grid, rows_per);
            else launch_delta_act<T, false, false>(s, d, grid, rows_per);
        }
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
    auto fits = [&](const void *p, long ld) { return (reinterpret_cast<uintptr_t>(p) & (d.f32 ? 15 : 7)) == 0 && (ld & 3) == 0; };
    const bool vec = fits(d.dY, d.ldY) && fits(d.Z, d.ldZ) && fits(d.U, d.ldU);
    return d.f32 ? launch_delta_typed<float>(s, d, vec, per, (int)runs) : launch_delta_typed<__bf16>(s, d, vec, per, (int)runs);
}

}  // namespace alpha
