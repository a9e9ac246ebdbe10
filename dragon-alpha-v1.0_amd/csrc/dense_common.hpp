// Shared declarations of the dense operators (include/alpha_dense.h): activations, the epilogue of a product, the operand
// description of the tile kernel and the host-side launchers.
#pragma once
#include "../../include/alpha_dense.h"
#include "common.hpp"

namespace alpha {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef unsigned uintx4 __attribute__((ext_vector_type(4)));

// ---- activations ---------------------------------------------------------------------------------------------------
// exp(z) from the hardware's 2^x: z log2(e) as a rounded product and its remainder, the remainder applied to first order;
// within a few units of 2^-24, 2^x's own error among them.
static __device__ __forceinline__ float dense_exp(float z)
{
    const float t = z * 1.44269504f, r = fmaf(z, 1.44269504f, -t) + z * 1.925963e-8f;
    const float p = __builtin_amdgcn_exp2f(t);
    return fabsf(t) < 126.f ? fmaf(p, r * 0.69314718f, p) : p;   // (beyond: near 0 or infinity, and r may be no number)
}
// S(z) = 1 / (1 + exp(-z)); 1 / (1 + inf) = 0 from the hardware's reciprocal (2^-23).
static __device__ __forceinline__ float dense_sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + dense_exp(-z)); }
// S(z) (1 - S(z)) = S(z) S(-z) = e / (1 + e)^2 with e = exp(-|z|). (1 minus a rounded S has nothing left from z = 17 on.)
static __device__ __forceinline__ float dense_sigmoid_slope(float z)
{
    const float e = dense_exp(-fabsf(z)), r = __builtin_amdgcn_rcpf(1.f + e);
    return e * r * r;
}

// P(z) = (1 + erf(z / sqrt 2)) / 2 and its derivative D(z) = exp(-z^2 / 2) / sqrt(2 pi), from one exponential. The tail P(-a), a = |z|,
// is exp(-a^2 / 2) R(a) with a smooth R (half the scaled complementary error function), so it keeps its relative accuracy however small
// it is; 1 + erf(..) would cancel, off by 4 % at z = -5 and 0 from -5.6 on. R is a polynomial in t = 1 / (1 + p a), fitted by weighted
// least squares to the smallest relative error on 0 <= a <= 14, where exp(-a^2 / 2) leaves fp32: fp32 degree 9, 2.7e-7 with the roundings of
// its evaluation; bf16 (T) degree 7, 5.7e-7. fp32 takes a^2 with its remainder, as exp turns an absolute error into a relative one.
template <typename T>
static __device__ __forceinline__ float dense_normal(float z, float &density)
{
    const float a = fminf(fabsf(z), 20.f);                // (beyond, P(-a) is 0; a NaN passes through the caller's factor z)
    float e, q;
    if constexpr (sizeof(T) == 4) {
        const float s = a * a, rest = fmaf(a, a, -s), g = dense_exp(-0.5f * s);
        e = fmaf(g, -0.5f * rest, g);
        const float t = __builtin_amdgcn_rcpf(fmaf(0.46f, a, 1.f));
        q = fmaf(t, fmaf(t, fmaf(t, fmaf(t, 0.045149371f, -0.25367415f), 0.57395941f), -0.613239527f), 0.235497072f);
        q = fmaf(t, fmaf(t, fmaf(t, fmaf(t, fmaf(t, q, -0.0135250678f), 0.160627916f), 0.181561515f), 0.183647409f), -3.92358834e-06f);
    } else {
        e = __builtin_amdgcn_exp2f(-0.72134752f * a * a);
        const float t = __builtin_amdgcn_rcpf(fmaf(0.35f, a, 1.f));
        q = fmaf(t, fmaf(t, fmaf(t, 0.0489424318f, -0.202119246f), 0.240640774f), -0.0170233995f);
        q = fmaf(t, fmaf(t, fmaf(t, fmaf(t, q, 0.155961469f), 0.133355096f), 0.140270337f), -2.73155074e-05f);
    }
    density = 0.39894228f * e;
    const float tail = q * e;
    return z < 0.f ? tail : 1.f - tail;
}

template <typename T>
static __device__ __forceinline__ float dense_act(int act, float z, float k)
{
    float density;
    switch (act) {   // uniform
    case ALPHA_DENSE_ACT_LEAKY_RELU: return z > 0.f ? z : z * k;
    case ALPHA_DENSE_ACT_GELU: return z * dense_normal<T>(z, density);
    case ALPHA_DENSE_ACT_SILU: return z * dense_sigmoid(z);
    case ALPHA_DENSE_ACT_SIGMOID: return dense_sigmoid(z);
    default: return z;
    }
}

template <typename T>
static __device__ __forceinline__ float dense_act_slope(int act, float z, float k)
{
    switch (act) {
    case ALPHA_DENSE_ACT_LEAKY_RELU: return z > 0.f ? 1.f : k;
    case ALPHA_DENSE_ACT_GELU: {
        float density;
        const float p = dense_normal<T>(z, density);
        return fmaf(z, density, p);
    }
    case ALPHA_DENSE_ACT_SILU: {
        const float s = dense_sigmoid(z);
        return s * fmaf(z, 1.f - s, 1.f);
    }
    case ALPHA_DENSE_ACT_SIGMOID: return dense_sigmoid_slope(z);
    default: return 1.f;
    }
}

// ---- element types -------------------------------------------------------------------------------------------------
template <typename T> static __device__ __forceinline__ float dense_load(const T *p) { return (float)*p; }
template <typename T> static __device__ __forceinline__ void dense_store(T *p, float v) { *p = (T)v; }   // round to nearest even

// Four consecutive elements; VEC: the address is aligned to the whole group.
template <typename T> struct Quad;
template <> struct Quad<float> { typedef floatx4 type; };
template <> struct Quad<__bf16> { typedef bf16x4 type; };

template <typename T>
static __device__ __forceinline__ floatx4 quad_load(const T *p)
{
    const typename Quad<T>::type v = *reinterpret_cast<const typename Quad<T>::type *>(p);
    return floatx4{(float)v[0], (float)v[1], (float)v[2], (float)v[3]};
}
template <typename T>
static __device__ __forceinline__ void quad_store(T *p, floatx4 v)
{
    typename Quad<T>::type q;
    q[0] = (T)v[0]; q[1] = (T)v[1]; q[2] = (T)v[2]; q[3] = (T)v[3];
    *reinterpret_cast<typename Quad<T>::type *>(p) = q;
}

// COLS consecutive elements of a row from column c on, whatever their alignment. At the row's end (`cols` >= COLS) the last
// COLS are loaded instead, without a branch, and moved to their places by at_edge: zeros from `cols` on.
template <int COLS, typename T>
static __device__ __forceinline__ void load_columns(const T *row, int c, int cols, T (&v)[COLS])
{
    __builtin_memcpy(v, row + (c < cols - COLS ? c : cols - COLS), COLS * sizeof(T));
}
template <int COLS, typename T>
static __device__ __forceinline__ void at_edge(int c, int cols, T (&v)[COLS])
{
    const int by = c - (cols - COLS);
#pragma unroll
    for (int i = 0; i < COLS; i++) {
        const bool move = by > i;
#pragma unroll
        for (int e = 0; e < COLS; e++) v[e] = move ? (e + 1 < COLS ? v[e + 1] : (T)0.f) : v[e];
    }
}

// ---- the product's epilogue ----------------------------------------------------------------------------------------
// Plain:  z = acc + bias[n];  Z = z;  Y = act(z) + R     (two stacked products, row2 > 0: rows m < rows1 to Y, m >= row2 to Y2)
// Gated:  g = acc_g + bias[n], u = acc_u + bias2[n];  Z = g, Z2 = u;  Y = act(g) * u
struct DenseEpilogue {
    const void *bias, *bias2, *R;
    void *Z, *Z2, *Y, *Y2;
    long ldR, ldZ, ldZ2, ldY, ldY2;
    int act;
    float slope;
    int rows1, row2;
    int vec;      // groups of four columns are aligned (bases and strides): vector accesses
};

// C[m, n] = sum over sources and k of A(m, k) B(n, k). bf16 operands: rows of whole 16-byte chunks at 16-byte aligned
// addresses, zeros after a row's last element; fp32: any.
struct DenseOperand {
    const void *p[2];     // up to two sources
    long ld;              // element (row r, column c) at r * ld + c
};
struct DenseProduct {
    DenseOperand A, B;
    int sources;          // 2: the sum goes on over A.p[1], B.p[1]
    int gated;            // B.p[0], B.p[1] are the two filters of a gated pair
    int a_t, b_t;         // operand stored with k as its rows
    int M, N;             // N: of one filter where gated
    int K;
    int f32;
    DenseEpilogue ep;
    float *pieces;        // room for the pieces of cut reductions, `piece_bytes`
    size_t piece_bytes;
};
size_t dense_product_piece_bytes(int M, int N, int K, int f32, int sources, int gated);
constexpr double DENSE_LEAST_TILES_US = 6.5;                                                         // no estimate of that is less
double dense_product_us(int M, int N, int K, int f32, int sources, int gated);   // the plan's estimate
hipError_t launch_dense_product(hipStream_t s, const DenseProduct &p);

// Few rows, operands as they are (dense_few_rows.hip).
struct DenseFewRows {
    const void *X, *W, *W2;
    long ldX, ldW, ldW2;
    int f32, gated;
    int M, N, K;
    DenseEpilogue ep;
    float *pieces;        // room for the pieces of a cut reduction, `piece_bytes`
    size_t piece_bytes;
    int cuts, per;        // set by the launcher
};

// How a forward product is computed: by tiles, or straight from memory as few rows or as a short reduction.
enum DenseForm { DENSE_TILES_FORM, DENSE_FEW_ROWS, DENSE_SHORT };
DenseForm dense_forward_form(int f32, int gated, int M, int N, int K);
double dense_few_rows_us(int f32, int gated, int M, int N, int K);   // estimates
size_t dense_few_rows_piece_bytes(int f32, int gated, int M, int N, int K);
double dense_short_us(int f32, int gated, int M, int N, int K);
hipError_t launch_dense_short(hipStream_t s, const DenseFewRows &a);
hipError_t launch_dense_few_rows(hipStream_t s, const DenseFewRows &a);

// Small products of a backward (B with k as its rows), operands as they are (dense_small.hip).
size_t dense_small_piece_bytes(int f32, int M, int N, int K, int sources);
bool dense_small_preferred(int f32, int a_t, int M, int N, int K, int sources);
hipError_t launch_dense_small(hipStream_t s, const DenseProduct *px, const DenseProduct *pw);   // deltaX and deltaW, one may be null

// dst <- src[rows, cols]; row stride ld (multiple of 8), columns cols .. ld zero.
hipError_t launch_dense_pack(hipStream_t s, int f32, const void *src, long src_ld, long rows, int cols, void *dst, long ld);

// deltaZ (or deltaG and deltaU) in the operands' type and the column sums of the unrounded values.
struct DenseDelta {
    const void *dY, *Z, *U;
    long ldY, ldZ, ldU;
    int f32, act, gated;
    float slope;
    long rows;
    int cols;
    void *dst, *dst2;     // NULL: only the sums
    long ld;              // columns written (cols, then zeros): a multiple of 8
    long ld2;             // row stride of dst, dst2
    void *dB, *dB2;       // NULL: no sums
    float *sums;          // dense_delta_sum_bytes of scratch
};
size_t dense_delta_sum_bytes(long rows, int cols, int gated);
hipError_t launch_dense_delta(hipStream_t s, const DenseDelta &d);

// Clipping by the global norm (grad_clip.hip); `words`: the sum of grad_pieces over the tensors.
long grad_pieces(long length);
hipError_t launch_grad_clip(hipStream_t s, int count, const int *types, const int64_t *lengths, const void *const *src, void *const *dst,
                            float max_norm, float eps, float *norm_c, double *words);

}  // namespace alpha
