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

// The same for the `left` first of R elements at any address.
template <int R, typename T>
static __device__ __forceinline__ void edge_load(const T *p, int left, float (&v)[R])
{
#pragma unroll
    for (int e = 0; e < R; e++) v[e] = dense_load(p + (e < left ? e : left - 1));
}
template <int R, typename T>
static __device__ __forceinline__ void edge_store(T *p, int left, const float (&v)[R])
{
#pragma unroll
    for (int e = 0; e < R; e++)
        if (e < left) dense_store(p + e, v[e]);
}

// The epilogues of R consecutive columns n .. n+R-1 of row m. WHOLE: all of them exist and groups of four are aligned; else the
// `left` first. FULL: all of the epilogue; else only the store (the products of a backward). `ahead`: the residual's elements, where they
// have been loaded before.
template <typename T, int R, bool FULL, bool WHOLE>
static __device__ __forceinline__ void dense_finish(const DenseEpilogue &ep, float (&v)[R], long m, int n, int left = R, const T *ahead = nullptr)
{
    const bool second = !FULL && ep.row2 > 0 && m >= ep.row2;
    if (!FULL && ep.row2 > 0 && !second && m >= ep.rows1) return;   // a row between two stacked products
    T *Y = static_cast<T *>(second ? ep.Y2 : ep.Y) + (second ? (m - ep.row2) * ep.ldY2 : m * ep.ldY) + n;
    auto load = [&](const T *p, float (&t)[R]) {
        if constexpr (WHOLE) run_load(p, t);
        else edge_load(p, left, t);
    };
    auto store = [&](T *p, const float (&t)[R]) {
        if constexpr (WHOLE) run_store(p, t);
        else edge_store(p, left, t);
    };
    if constexpr (FULL) {
        const T *bias = static_cast<const T *>(ep.bias), *res = static_cast<const T *>(ep.R);
        T *Z = static_cast<T *>(ep.Z);
        float t[R], r[R];
        if (res) {
            if (ahead) {
#pragma unroll
                for (int e = 0; e < R; e++) r[e] = (float)ahead[e];
            } else {
                load(res + m * ep.ldR + n, r);
            }
        }
        if (bias) {
            load(bias + n, t);
#pragma unroll
            for (int e = 0; e < R; e++) v[e] += t[e];
        }
        if (Z) store(Z + m * ep.ldZ + n, v);
        run_act<T>(ep.act, v, ep.slope);
        if (res) {
#pragma unroll
            for (int e = 0; e < R; e++) v[e] += r[e];
        }
    }
    store(Y, v);
}

template <typename T, int R, bool WHOLE>
static __device__ __forceinline__ void dense_finish_gated(const DenseEpilogue &ep, float (&g)[R], float (&u)[R], long m, int n, int left = R)
{
    auto load = [&](const T *p, float (&t)[R]) {
        if constexpr (WHOLE) run_load(p, t);
        else edge_load(p, left, t);
    };
    auto store = [&](void *p, long ld, const float (&t)[R]) {
        T *const q = static_cast<T *>(p) + m * ld + n;
        if constexpr (WHOLE) run_store(q, t);
        else edge_store(q, left, t);
    };
    float t[R];
    if (ep.bias) {
        load(static_cast<const T *>(ep.bias) + n, t);
#pragma unroll
        for (int e = 0; e < R; e++) g[e] += t[e];
    }
    if (ep.bias2) {
        load(static_cast<const T *>(ep.bias2) + n, t);
#pragma unroll
        for (int e = 0; e < R; e++) u[e] += t[e];
    }
    if (ep.Z) store(ep.Z, ep.ldZ, g);
    if (ep.Z2) store(ep.Z2, ep.ldZ2, u);
    run_act<T>(ep.act, g, ep.slope);
#pragma unroll
    for (int e = 0; e < R; e++) g[e] *= u[e];
    store(ep.Y, ep.ldY, g);
}

}  // namespace alpha
