// The epilogues of the dense products, for a run of consecutive columns of one row that a lane holds.
#pragma once
#include "dense_common.hpp"

namespace alpha {

// R consecutive elements of a row, aligned to groups of four, or one element.
template <int R, typename T>
static __device__ __forceinline__ void run_load(const T *p, float (&v)[R])
{
    if constexpr (R == 1) v[0] = dense_load(p);
    else
#pragma unroll
    for (int i = 0; i < R; i += 4) {
        const floatx4 q = quad_load(p + i);
#pragma unroll
        for (int e = 0; e < 4; e++) v[i + e] = q[e];
    }
}
template <int R, typename T>
static __device__ __forceinline__ void run_store(T *p, const float (&v)[R])
{
    if constexpr (R == 1) {
        dense_store(p, v[0]);
    } else if constexpr (R == 8 && sizeof(T) == 2) {   // one 128-bit store (the hardware takes 8-byte alignment)
        bf16x8 q;
#pragma unroll
        for (int e = 0; e < 8; e++) q[e] = (T)v[e];
        __builtin_memcpy(__builtin_assume_aligned(p, 8), &q, 16);
    } else {
#pragma unroll
        for (int i = 0; i < R; i += 4) quad_store(p + i, floatx4{v[i], v[i + 1], v[i + 2], v[i + 3]});
    }
}
template <typename T, int R>
static __device__ __forceinline__ void run_act(int act, float (&v)[R], float k)
{
    switch (act) {   // one branch for the run
    case ALPHA_DENSE_ACT_LEAKY_RELU:
#pragma unroll
        for (int e = 0; e < R; e++) v[e] = dense_act<T>(ALPHA_DENSE_ACT_LEAKY_RELU, v[e], k);
        break;
    case ALPHA_DENSE_ACT_GELU:
#pragma unroll
        for (int e = 0; e < R; e++) v[e] = dense_act<T>(ALPHA_DENSE_ACT_GELU, v[e], k);
        break;
    case ALPHA_DENSE_ACT_SILU:
#pragma unroll
        for (int e = 0; e < R; e++) v[e] = dense_act<T>(ALPHA_DENSE_ACT_SILU, v[e], k);
        break;
    case ALPHA_DENSE_ACT_SIGMOID:
#pragma unroll
        for (int e = 0; e < R; e++) v[e] = dense_act<T>(ALPHA_DENSE_ACT_SIGMOID, v[e], k);
        break;
    default: break;
    }
}

// The epilogues of R consecutive columns n .. n+R-1 of row m, R a multiple of four and aligned to it, or one element. FULL: all
// of the epilogue; else only the store (the products of a backward).
template <typename T, int R, bool FULL>
static __device__ __forceinline__ void dense_finish(const DenseEpilogue &ep, float (&v)[R], long m, int n)
{
    const bool second = !FULL && ep.row2 > 0 && m >= ep.row2;
    if (!FULL && ep.row2 > 0 && !second && m >= ep.rows1) return;   // a row between two stacked products
    T *Y = static_cast<T *>(second ? ep.Y2 : ep.Y) + (second ? (m - ep.row2) * ep.ldY2 : m * ep.ldY) + n;
    if constexpr (FULL) {
        const T *bias = static_cast<const T *>(ep.bias), *res = static_cast<const T *>(ep.R);
        T *Z = static_cast<T *>(ep.Z);
        float t[R];
        if (bias) {
            run_load(bias + n, t);
#pragma unroll
            for (int e = 0; e < R; e++) v[e] += t[e];
        }
        if (Z) run_store(Z + m * ep.ldZ + n, v);
        run_act<T>(ep.act, v, ep.slope);
        if (res) {
            run_load(res + m * ep.ldR + n, t);
#pragma unroll
            for (int e = 0; e < R; e++) v[e] += t[e];
        }
    }
    run_store(Y, v);
}

template <typename T, int R>
static __device__ __forceinline__ void dense_finish_gated(const DenseEpilogue &ep, float (&g)[R], float (&u)[R], long m, int n)
{
    const T *bg = static_cast<const T *>(ep.bias), *bu = static_cast<const T *>(ep.bias2);
    T *G = static_cast<T *>(ep.Z), *U = static_cast<T *>(ep.Z2);
    float t[R];
    if (bg) {
        run_load(bg + n, t);
#pragma unroll
        for (int e = 0; e < R; e++) g[e] += t[e];
    }
    if (bu) {
        run_load(bu + n, t);
#pragma unroll
        for (int e = 0; e < R; e++) u[e] += t[e];
    }
    if (G) run_store(G + m * ep.ldZ + n, g);
    if (U) run_store(U + m * ep.ldZ2 + n, u);
    run_act<T>(ep.act, g, ep.slope);
#pragma unroll
    for (int e = 0; e < R; e++) g[e] *= u[e];
    run_store(static_cast<T *>(ep.Y) + m * ep.ldY + n, g);
}

}  // namespace alpha
