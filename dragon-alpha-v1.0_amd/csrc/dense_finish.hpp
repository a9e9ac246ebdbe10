// The epilogues of the dense products, for a run of consecutive columns of one row that a lane holds.
#pragma once
#include "dense_common.hpp"

namespace alpha {

// R consecutive elements of a row, aligned to groups of four.
template <int R, typename T>
static __device__ __forceinline__ void run_load(const T *p, float (&v)[R])
{
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
    if constexpr (R == 8 && sizeof(T) == 2) {   // one 128-bit store (the hardware takes 8-byte alignment)
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

// The epilogues of R consecutive columns n .. n+R-1 of row m (fewer at the right edge).
template <typename T, int R>
static __device__ __forceinline__ void dense_finish(const DenseEpilogue &ep, float (&v)[R], long m, int n, int N)
{
    const bool second = ep.row2 > 0 && m >= ep.row2;
    if (ep.row2 > 0 && !second && m >= ep.rows1) return;   // a row between two stacked products
    T *Y = static_cast<T *>(second ? ep.Y2 : ep.Y) + (second ? (m - ep.row2) * ep.ldY2 : m * ep.ldY) + n;
    const T *bias = static_cast<const T *>(ep.bias), *res = static_cast<const T *>(ep.R);
    T *Z = static_cast<T *>(ep.Z);
    const bool whole = R % 4 == 0 && ep.vec && n + R <= N;
    float t[R];
    if (bias) {
        if constexpr (R % 4 == 0)
            if (whole) run_load(bias + n, t);
        if (!whole) {
#pragma unroll
            for (int e = 0; e < R; e++) t[e] = n + e < N ? dense_load(bias + n + e) : 0.f;
        }
#pragma unroll
        for (int e = 0; e < R; e++) v[e] += t[e];
    }
    if (Z) {
        if constexpr (R % 4 == 0)
            if (whole) run_store(Z + m * ep.ldZ + n, v);
        if (!whole) {
#pragma unroll
            for (int e = 0; e < R; e++)
                if (n + e < N) dense_store(Z + m * ep.ldZ + n + e, v[e]);
        }
    }
    run_act<T>(ep.act, v, ep.slope);
    if (res) {
        if constexpr (R % 4 == 0)
            if (whole) run_load(res + m * ep.ldR + n, t);
        if (!whole) {
#pragma unroll
            for (int e = 0; e < R; e++) t[e] = n + e < N ? dense_load(res + m * ep.ldR + n + e) : 0.f;
        }
#pragma unroll
        for (int e = 0; e < R; e++) v[e] += t[e];
    }
    if constexpr (R % 4 == 0)
        if (whole) run_store(Y, v);
    if (!whole) {
#pragma unroll
        for (int e = 0; e < R; e++)
            if (n + e < N) dense_store(Y + e, v[e]);
    }
}

template <typename T, int R>
static __device__ __forceinline__ void dense_finish_gated(const DenseEpilogue &ep, float (&g)[R], float (&u)[R], long m, int n, int N)
{
    T *Y = static_cast<T *>(ep.Y) + m * ep.ldY + n;
    const bool whole = R % 4 == 0 && ep.vec && n + R <= N;
#pragma unroll
    for (int which = 0; which < 2; which++) {
        float(&v)[R] = which ? u : g;
        const T *bias = static_cast<const T *>(which ? ep.bias2 : ep.bias);
        T *Z = static_cast<T *>(which ? ep.Z2 : ep.Z) + m * (which ? ep.ldZ2 : ep.ldZ) + n;
        if (bias) {
            float t[R];
            if constexpr (R % 4 == 0)
                if (whole) run_load(bias + n, t);
            if (!whole) {
#pragma unroll
                for (int e = 0; e < R; e++) t[e] = n + e < N ? dense_load(bias + n + e) : 0.f;
            }
#pragma unroll
            for (int e = 0; e < R; e++) v[e] += t[e];
        }
        if (which ? ep.Z2 != nullptr : ep.Z != nullptr) {
            if constexpr (R % 4 == 0)
                if (whole) run_store(Z, v);
            if (!whole) {
#pragma unroll
                for (int e = 0; e < R; e++)
                    if (n + e < N) dense_store(Z + e, v[e]);
            }
        }
    }
    run_act<T>(ep.act, g, ep.slope);
#pragma unroll
    for (int e = 0; e < R; e++) g[e] *= u[e];
    if constexpr (R % 4 == 0)
        if (whole) run_store(Y, g);
    if (!whole) {
#pragma unroll
        for (int e = 0; e < R; e++)
            if (n + e < N) dense_store(Y + e, g[e]);
    }
}

}  // namespace alpha
