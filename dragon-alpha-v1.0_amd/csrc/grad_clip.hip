// Clipping by the global norm: one pass that sums the squares of all tensors, one short kernel for norm and factor, one
// pass that scales. Both passes are bound by memory; they take the tensors by value in the kernel's arguments (nothing of the
// host is read after the call returns, and a captured graph holds its own copy), up to 240 and 164 in a launch.
//
// Squares: a workgroup takes a piece of one tensor. The squares of a lane's 16 bytes are added in fp32 and go on in fp64, so a
// sum over billions keeps its last bits; where those 16 bytes' sum leaves [2^-90, 2^120] - squares of 1e-25 and 1e+25 do -
// they are taken again in fp64. A workgroup's sum goes to its own word, and the short kernel adds the words in a fixed order:
// the norm's bits do not change from run to run.
// Scaling goes through the pieces from the last to the first, so what the first pass read last is still in the last-level cache
// (256 MB).
// Measured: 162 tensors, 102 MB of fp32, squares / norm / scaling 19 / 4 / 36 us (5.4 and 5.7 TB/s);
// 48 tensors, 418 MB of bf16, 99 / 5 / 135 us (4.2 and 6.2 TB/s, the writes of the pass before still on their way to memory in the
// first).
#include "dense_common.hpp"

#include <algorithm>

namespace alpha {

namespace {

constexpr int PIECE = 16384;   // elements

struct GradSlot {
    const void *src;
    int first_piece;           // of the launch
    unsigned last;             // elements of its last piece, and the sign bit: fp32
};
struct GradSquares {
    static constexpr int SLOTS = 240;
    GradSlot slot[SLOTS];
    int count, pieces;
};
struct GradScale {
    static constexpr int SLOTS = 164;
    GradSlot slot[SLOTS];
    void *dst[SLOTS];
    int count, pieces;
};
static_assert(sizeof(GradSquares) <= 4000 && sizeof(GradScale) <= 4000, "kernel arguments");

// the tensor of a piece: first_piece[i] <= piece < first_piece[i + 1]
template <typename L>
__device__ __forceinline__ int tensor_of(const L &t, int piece)
{
    int lo = 0, hi = t.count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (t.slot[mid].first_piece <= piece) lo = mid;
        else hi = mid;
    }
    return lo;
}
template <typename L>
__device__ __forceinline__ int elements_of(const L &t, int i, int piece)
{
    const int end = i + 1 < t.count ? t.slot[i + 1].first_piece : t.pieces;
    return piece + 1 < end ? PIECE : (int)(t.slot[i].last & 0x7fffffffu);
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
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < V; e++) s = fmaf((float)v[e], (float)v[e], s);
        if (s >= 0x1p-90f && s <= 0x1p120f) {
            sum += (double)s;
        } else {
#pragma unroll
            for (int e = 0; e < V; e++) {
                const double x = (float)v[e];
                sum += x * x;
            }
        }
    }
    const int tail = head + vectors * V + threadIdx.x;
    if (tail < n) {
        const double v = (float)p[tail];
        sum += v * v;
    }
    return sum;
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
#pragma unroll 8
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

__global__ __launch_bounds__(256) void grad_squares_kernel(const GradSquares t, double *__restrict__ words)
{
    __shared__ double lds[4];
    const int piece = blockIdx.x, i = tensor_of(t, piece), n = elements_of(t, i, piece);
    const long at = (long)(piece - t.slot[i].first_piece) * PIECE;
    double v = t.slot[i].last >> 31 ? piece_squares(static_cast<const float *>(t.slot[i].src) + at, n)
                                    : piece_squares(static_cast<const __bf16 *>(t.slot[i].src) + at, n);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_down(v, d, 64);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    if (threadIdx.x == 0) words[piece] = lds[0] + lds[1] + lds[2] + lds[3];
}

__global__ __launch_bounds__(1024) void grad_norm_kernel(const double *__restrict__ words, long count, float max_norm, float eps, float *__restrict__ norm_c)
{
    __shared__ double lds[16];
    double v = 0.0;
#pragma unroll 8
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

__global__ __launch_bounds__(256) void grad_scale_kernel(const GradScale t, const float *__restrict__ norm_c)
{
    const int i = tensor_of(t, blockIdx.x), first = t.slot[i].first_piece, end = i + 1 < t.count ? t.slot[i + 1].first_piece : t.pieces;
    const int piece = first + end - 1 - (int)blockIdx.x, n = elements_of(t, i, piece);     // a tensor's last one first
    const float c = norm_c[1];
    if (c == 1.f && t.slot[i].src == t.dst[i]) return;
    const long at = (long)(piece - first) * PIECE;
    if (t.slot[i].last >> 31) piece_scale(static_cast<const float *>(t.slot[i].src) + at, static_cast<float *>(t.dst[i]) + at, n, c);
    else piece_scale(static_cast<const __bf16 *>(t.slot[i].src) + at, static_cast<__bf16 *>(t.dst[i]) + at, n, c);
}

long grad_pieces(long length) { return (length + PIECE - 1) / PIECE; }

namespace {

// Fills a launch with runs of whole pieces of tensors until it has no slot or 2^23 pieces; false when there is nothing left.
// `next`, `done`: the tensor and the pieces of it that are dealt with; `step` +1 or -1 (then the pieces from a tensor's end).
template <typename L>
bool fill(L &t, int count, const int *types, const int64_t *lengths, const void *const *src, void *const *dst, int &next, long &done, int step)
{
    t.count = t.pieces = 0;
    while (next >= 0 && next < count && t.count < L::SLOTS && t.pieces < (1 << 23)) {
        const long pieces = grad_pieces(lengths[next]), size = types[next] == ALPHA_DENSE_F32 ? 4 : 2;
        const long take = std::min<long>(pieces - done, (1l << 23) - t.pieces);
        if (take <= 0) {
            next += step;
            done = 0;
            continue;
        }
        const long first = step > 0 ? done : pieces - done - take;       // of the tensor's pieces
        const long rest = lengths[next] - (first + take - 1) * PIECE;    // elements from the last one's beginning on
        t.slot[t.count] = GradSlot{static_cast<const char *>(src[next]) + first * PIECE * size, t.pieces,
                                   (unsigned)std::min<long>(rest, PIECE) | (types[next] == ALPHA_DENSE_F32 ? 0x80000000u : 0u)};
        if constexpr (L::SLOTS == GradScale::SLOTS) t.dst[t.count] = static_cast<char *>(dst[next]) + first * PIECE * size;
        t.pieces += (int)take;
        t.count++;
        done += take;
    }
    return t.count > 0;
}

}  // namespace

hipError_t launch_grad_clip(hipStream_t s, int count, const int *types, const int64_t *lengths, const void *const *src, void *const *dst,
                            float max_norm, float eps, float *norm_c, double *words)
{
    long total = 0, done = 0;
    int next = 0;
    for (GradSquares t; fill(t, count, types, lengths, src, dst, next, done, 1); total += t.pieces) {
        hipLaunchKernelGGL(grad_squares_kernel, dim3((unsigned)t.pieces), dim3(256), 0, s, t, words + total);
        if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    hipLaunchKernelGGL(grad_norm_kernel, dim3(1), dim3(1024), 0, s, words, total, max_norm, eps, norm_c);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    if (dst == nullptr) return hipSuccess;
    next = count - 1;
    done = 0;
    for (GradScale t; fill(t, count, types, lengths, src, dst, next, done, -1);) {
        hipLaunchKernelGGL(grad_scale_kernel, dim3((unsigned)t.pieces), dim3(256), 0, s, t, norm_c);
        if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace alpha
