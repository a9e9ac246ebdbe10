// What the kernels that take X and W from memory straight into MFMA registers share: a lane holds 16 bytes of a row.
#pragma once
#include "dense_finish.hpp"

namespace alpha {

template <typename T> struct FewVec;
template <> struct FewVec<float> { typedef floatx4 type; };
template <> struct FewVec<__bf16> { typedef bf16x8 type; };

// 16 bytes of a row from element k on, whatever its alignment. ODD: bf16 that may begin in the middle of a word, which the memory
// pipe serves at a third of its rate (100 x 2001 x 500 28.0 -> 17.2 us); the words they lie in are loaded instead and shifted. (The
// half word beside them is dropped: it shares its word, and so its page, with an element that is asked for.)
template <bool ODD, typename T>
static __device__ __forceinline__ typename FewVec<T>::type few_load(const T *row, int k)
{
    typename FewVec<T>::type v;
    if constexpr (ODD) {
        const char *c = reinterpret_cast<const char *>(row + k);
        const unsigned odd = (unsigned)reinterpret_cast<uintptr_t>(c) & 2;
        c -= odd;
        uint32_t w[5];
        __builtin_memcpy(w, __builtin_assume_aligned(c, 4), 16);
        __builtin_memcpy(w + 4, __builtin_assume_aligned(c + 12 + 2 * odd, 4), 4);
#pragma unroll
        for (int i = 0; i < 4; i++) w[i] = __builtin_amdgcn_alignbit(w[i + 1], w[i], odd * 8);
        __builtin_memcpy(&v, w, 16);
    } else {
        __builtin_memcpy(&v, row + k, 16);
    }
    return v;
}
// What was loaded at end - V instead of at k > end - V, moved to its place: zeros from K on. Whole words first (end and k are even
// in bf16 unless ODD), then half of one, then the element behind K that end may include.
template <typename T, bool ODD>
static __device__ __forceinline__ typename FewVec<T>::type few_at_edge(typename FewVec<T>::type x, int k, int end, int K)
{
    constexpr int V = 16 / sizeof(T), PER_WORD = 4 / sizeof(T);
    const int by = k > end - V ? k - (end - V) : 0, words = by / PER_WORD;
    const bool one = words & 1, two = words & 2, none = words >= 4;
    uintx4 w = __builtin_bit_cast(uintx4, x);
    w = two ? uintx4{w[2], w[3], 0, 0} : w;
    w = one ? uintx4{w[1], w[2], w[3], 0} : w;
    if constexpr (ODD) {
        const int half = (by & 1) * 16;
        w = uintx4{__builtin_amdgcn_alignbit(w[1], w[0], half), __builtin_amdgcn_alignbit(w[2], w[1], half), __builtin_amdgcn_alignbit(w[3], w[2], half), w[3] >> half};
    }
    w = none ? uintx4{0, 0, 0, 0} : w;
    if constexpr (sizeof(T) == 2 && !ODD) {
#pragma unroll
        for (int i = 0; i < 4; i++) w[i] &= k + 2 * i + 1 == K ? 0xffffu : ~0u;
    }
    x = __builtin_bit_cast(typename FewVec<T>::type, w);
    return x;
}

static __device__ __forceinline__ floatx4 few_multiply(bf16x8 w, bf16x8 x, floatx4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, x, c, 0, 0, 0); }
static __device__ __forceinline__ floatx4 few_multiply(floatx4 w, floatx4 x, floatx4 c)
{
#pragma unroll
    for (int s = 0; s < 4; s++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(w[s], x[s], c, 0, 0, 0);
    return c;
}

// May a load of bf16 from these rows begin in the middle of a word?
static inline bool odd_rows(std::initializer_list<const void *> p, std::initializer_list<long> strides)
{
    for (const void *q : p)
        if (reinterpret_cast<uintptr_t>(q) & 3) return true;
    for (long x : strides)
        if (x & 1) return true;
    return false;
}

}  // namespace alpha
