// Clipping by the global norm: one pass that sums the squares of all tensors, one short kernel for norm and factor, one
// pass that scales. A launch takes up to SLOTS tensors by value in its arguments (nothing of the host is read after the
// call returns, and a captured graph holds its own copy).
//
// Squares are summed in fp64: exact to the last bit of a long sum, and neither 1e-25 nor 1e+25 leaves the range. A
// workgroup takes a piece of one tensor; its partial sum goes to its own word, and the short kernel
// adds the words in a fixed order, so the norm's bits do not change from run to run.
#include "dense_common.hpp"

#include <algorithm>

namespace alpha {

struct GradTensors {
    static constexpr int SLOTS = 96;
    const void *src[SLOTS];
    void *dst[SLOTS];
    long length[SLOTS];
    int first_piece[SLOTS + 1];   // pieces of tensor i: first_piece[i] .. first_piece[i + 1] - 1 of the launch
    unsigned char f32[SLOTS];
    int count;
    int piece;                    // elements of a piece
};
constexpr int PIECE = 16384, MORE = 4;   // a piece, or MORE of them where there are many

namespace {

__device__ __forceinline__ int tensor_of(const GradTensors &t, int piece)
{
    int lo = 0, hi = t.count;   // first_piece[lo] <= piece < first_piece[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (t.first_piece[mid] <= piece) lo = mid;
        else hi = mid;
    }
    return lo;
}

template <typename T>
__device__ __forceinline__ double piece_squares(const T *p, int n)
{
    constexpr int V = 16 / sizeof(T);
    typedef T vec __attribute__((ext_vector_type(V)));
    double sum = 0.0;
    // up to the first 16-byte boundary, whole vectors, the rest
    int head = (int)(((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / sizeof(T));
    if (head > n) head = n;
    if ((int)threadIdx.x < head) {
        const double v = (float)p[threadIdx.x];
        sum += v * v;
    }
    const int vectors = (n - head) / V;
    const vec *q = reinterpret_cast<const vec *>(p + head);
#pragma unroll 8
    for (int i = threadIdx.x; i < vectors; i += 256) {
        const vec v = q[i];
#pragma unroll
        for (int e = 0; e < V; e++) {
            const double x = (float)v[e];
            sum += x * x;
        }
    }
    const int tail = head + vectors * V + threadIdx.x;
    if (tail < n) {
        const double v = (float)p[tail];
        sum += v * v;
    }
    return sum;
}

__device__ __forceinline__ double workgroup_sum(double v, double *lds)
{
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_down(v, d, 64);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    return lds[0] + lds[1] + lds[2] + lds[3];
}

template <typename T>
__device__ __forceinline__ void piece_scale(const T *p, T *out, int n, float c)
{
    constexpr int V = 16 / sizeof(T);
    typedef T vec __attribute__((ext_vector_type(V)));
    const uintptr_t a = reinterpret_cast<uintptr_t>(p), b = reinterpret_cast<uintptr_t>(out);
    if ((a & 15) != (b & 15)) {
        for (int i = threadIdx.x; i < n; i += 256) out[i] = (T)((float)p[i] * c);
        return;
    }
    int head = (int)(((16 - (a & 15)) & 15) / sizeof(T));
    if (head > n) head = n;
    if ((int)threadIdx.x < head) out[threadIdx.x] = (T)((float)p[threadIdx.x] * c);
    const int vectors = (n - head) / V;
    const vec *q = reinterpret_cast<const vec *>(p + head);
    vec *o = reinterpret_cast<vec *>(out + head);
#pragma unroll 4
    for (int i = threadIdx.x; i < vectors; i += 256) {
        vec v = q[i];
#pragma unroll
        for (int e = 0; e < V; e++) v[e] = (T)((float)v[e] * c);
        o[i] = v;
    }
    const int tail = head + vectors * V + threadIdx.x;
    if (tail < n) out[tail] = (T)((float)p[tail] * c);
}

}  // namespace

__global__ __launch_bounds__(256) void grad_squares_kernel(const GradTensors t, double *__restrict__ words)
{
    __shared__ double lds[4];
    const int i = tensor_of(t, blockIdx.x);
    const long at = (long)(blockIdx.x - t.first_piece[i]) * t.piece;
    const int n = (int)(t.length[i] - at < t.piece ? t.length[i] - at : t.piece);
    const double v = t.f32[i] ? piece_squares(static_cast<const float *>(t.src[i]) + at, n)
                              : piece_squares(static_cast<const __bf16 *>(t.src[i]) + at, n);
    const double sum = workgroup_sum(v, lds);
    if (threadIdx.x == 0) words[blockIdx.x] = sum;
}

__global__ __launch_bounds__(1024) void grad_norm_kernel(const double *__restrict__ words, long count, float max_norm, float eps, float *__restrict__ norm_c)
{
    __shared__ double lds[16];
    double v = 0.0;
#pragma unroll 4
    for (long i = threadIdx.x; i < count; i += 1024) v += words[i];
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_down(v, d, 64);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    if (threadIdx.x == 0) {
        v = 0.0;
        for (int i = 0; i < 16; i++) v += lds[i];
        const double norm = sqrt(v), c = (double)max_norm / (norm + (double)eps);
        norm_c[0] = (float)norm;
        norm_c[1] = c < 1.0 || c != c ? (float)c : 1.f;
    }
}

__global__ __launch_bounds__(256) void grad_scale_kernel(const GradTensors t, const float *__restrict__ norm_c)
{
    const int i = tensor_of(t, blockIdx.x);
    const float c = norm_c[1];
    if (c == 1.f && t.src[i] == t.dst[i]) return;
    const long at = (long)(blockIdx.x - t.first_piece[i]) * t.piece;
    const int n = (int)(t.length[i] - at < t.piece ? t.length[i] - at : t.piece);
    if (t.f32[i]) piece_scale(static_cast<const float *>(t.src[i]) + at, static_cast<float *>(t.dst[i]) + at, n, c);
    else piece_scale(static_cast<const __bf16 *>(t.src[i]) + at, static_cast<__bf16 *>(t.dst[i]) + at, n, c);
}

long grad_pieces(long length)   // at most
{
    return (length + PIECE - 1) / PIECE;
}

hipError_t launch_grad_clip(hipStream_t s, int count, const int *types, const int64_t *lengths, const void *const *src, void *const *dst,
                            float max_norm, float eps, float *norm_c, double *words)
{
    long done = 0, total = 0;
    for (int i = 0; i < count; i++) total += lengths[i];
    // up to 4096 pieces of the small size are 16 per compute unit; beyond, longer pieces save their beginnings and ends
    const int piece = total > 4096l * PIECE ? MORE * PIECE : PIECE;
    for (int pass = 0; pass < (dst ? 2 : 1); pass++) {
        int next = 0;
        long offset = 0;   // elements of tensor `next` already dealt with (a launch holds at most 2^30 pieces)
        while (true) {
            GradTensors t{};
            t.piece = piece;
            long pieces = 0;
            while (next < count && t.count < GradTensors::SLOTS && pieces < (1l << 30)) {
                const long rest = lengths[next] - offset;
                if (rest <= 0) {
                    next++;
                    offset = 0;
                    continue;
                }
                const long size = types[next] == ALPHA_DENSE_F32 ? 4 : 2;
                const long take = std::min<long>(rest, ((1l << 30) - pieces) * piece);
                t.src[t.count] = static_cast<const char *>(src[next]) + offset * size;
                t.dst[t.count] = dst ? static_cast<char *>(dst[next]) + offset * size : nullptr;
                t.length[t.count] = take;
                t.f32[t.count] = types[next] == ALPHA_DENSE_F32;
                t.first_piece[t.count] = (int)pieces;
                pieces += (take + piece - 1) / piece;
                t.count++;
                offset += take;
            }
            if (t.count == 0) break;
            t.first_piece[t.count] = (int)pieces;
            if (pass == 0) hipLaunchKernelGGL(grad_squares_kernel, dim3((unsigned)pieces), dim3(256), 0, s, t, words + done);
            else hipLaunchKernelGGL(grad_scale_kernel, dim3((unsigned)pieces), dim3(256), 0, s, t, norm_c);
            if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
            if (pass == 0) done += pieces;
        }
        if (pass == 0) {
            hipLaunchKernelGGL(grad_norm_kernel, dim3(1), dim3(1024), 0, s, words, done, max_norm, eps, norm_c);
            if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
        }
    }
    return hipSuccess;
}

}  // namespace alpha
