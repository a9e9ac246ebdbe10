// What the dense tile kernels share: their arguments, the order of the tiles, the bank permutations of their LDS tiles, how
// a finished tile leaves, and the element that is computed once more.
#pragma once
#include "dense_finish.hpp"

#include <type_traits>

namespace alpha {

typedef short shortx4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char lds_char;

struct DenseTileArgs {
    const void *A[2], *B[2];   // bf16 or fp32
    long ldA, ldB;
    int M, N, K;
    int sources;       // 2: the sum goes on over A[1], B[1]
    int steps;         // sources for every 32 k
    int tiles_m, tiles_n;
    int whole;         // the first `whole` tiles are a workgroup's whole work; the others' reductions are cut
    int split, per;    // into `split` runs of `per` steps (an even number)
    DenseEpilogue ep;
    float *pieces;     // [split][tiles - whole][BM][BN], as the tile kernel has them
};

// The XCD-aware order of tiles. Workgroups go round the eight XCDs, so every eighth one shares an L2: an XCD gets a contiguous
// run of `count` places.
static __device__ __forceinline__ int xcd_place(int id, int count)
{
    const int each = count / 8, more = count % 8, xcd = id & 7;
    return xcd * each + (xcd < more ? xcd : more) + (id >> 3);
}
// Tile number -> tile row and column: panels of 8 tile rows, so that a run of tiles reuses both operands out of the L2.
static __device__ __forceinline__ void tile_at(int tile, int tiles_m, int tiles_n, int &tm, int &tn)
{
    const int panel = tile / (8 * tiles_n), first = panel * 8, deep = tiles_m - first < 8 ? tiles_m - first : 8, in = tile - panel * 8 * tiles_n;
    tm = first + in % deep;
    tn = in / deep;
}

// f(0), f(1), .. f(N - 1) with constants: unrolled whatever its size
template <int N, int I = 0, typename F>
static __device__ __forceinline__ void for_each(F &&f)
{
    if constexpr (I < N) {
        f(std::integral_constant<int, I>{});
        for_each<N, I + 1>(f);
    }
}

// Between LDS accesses of one wavefront's lanes: LDS serves a wavefront in order, the compiler must keep that order.
static __device__ __forceinline__ void wave_fence()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
}

// Which 16-byte chunk of a T tile's k row a chunk is kept at: number ^ this. The 32 lanes that one cycle of a transposing
// read serves touch eight k rows (0 .. 3 and 8 .. 11), whose 32-byte pieces so lie in eight different parts of the 256 bytes
// that a cycle delivers.
static __device__ __forceinline__ int t_permutation(int k) { return ((k & 3) | ((k >> 3) & 1) << 2) << 1; }
// The same for a straight tile, by g = row / 4. The 16 lanes that a cycle of a 128-bit read serves are rows 0-3 and 12-15
// of a fragment in one chunk and rows 4-11 in the chunk beside it (or the other way round); four rows are 256 bytes, so the
// four groups of rows must come to four different chunks: 0, 3, 2, 1 for g = 0 .. 3. Counted: no conflicts.
static __device__ __forceinline__ int s_permutation(int g) { return (g & 1) | ((g ^ (g >> 1)) & 1) << 1; }


// One fp32 element of C once more as a plain chain of fused multiply-adds: taken where the sum of the products of parts is NaN,
// which it also is where an operand is infinite (or within 2^-9 of the end of the range). Ends at the first NaN.
static __device__ __attribute__((noinline)) float dense_element(const void *A0, const void *A1, long a_row, long a_k, const void *B0, const void *B1,
                                                                long b_row, long b_k, int sources, int K)
{
    float acc = 0.f;
    for (int s = 0; s < sources; s++) {
        const float *a = static_cast<const float *>(s ? A1 : A0) + a_row, *b = static_cast<const float *>(s ? B1 : B0) + b_row;
        for (int k = 0; k < K; k++, a += a_k, b += b_k) {
            acc = fmaf(*a, *b, acc);
            if (acc != acc) return acc;
        }
    }
    return acc;
}

// A finished tile leaves two fragment rows (32 rows of C) at a time through the wavefront's part of LDS, so that a lane then has
// eight consecutive columns and a row goes out as one run: stored from the MFMA's registers as they are, 4096 x 4096 of bf16
// took 17 us to write, this way 10. acc[i][j][e]: row 16 i + lane % 16, column 16 j + 4 (lane / 16) + e of the wavefront's part
// of the tile. Every wavefront is done with the tiles in LDS.
template <typename T, bool AT, bool BT, bool GATED, int BM, int BN, int WM, int WN, int LDS>
static __device__ __forceinline__ void tile_out(const DenseTileArgs &a, const floatx4 (&acc)[BM / WM / 16][BN / WN / 16], char *smem, int lane, int wave, int wm,
                                                int wn, int m0, int n0, bool cut, int piece, int cut_tile, int cut_tiles)
{
    constexpr int TM = BM / WM, TN = BN / WN, MF = TM / 16;
    constexpr bool FULL = !BT;     // B with k as its rows: a backward's product
    constexpr bool AHEAD = FULL && !GATED && BM * BN >= 256 * 256;
    const int l16 = lane & 15, q = lane >> 4;
    constexpr int ROW = 68;                              // floats from row to row: 16 bytes past a multiple of the banks
    constexpr int LANES = GATED ? 4 : 8;                 // lanes of a row, eight columns each (gated: eight of each filter)
    constexpr int AT_ONCE = 64 / LANES, TURNS = 32 / AT_ONCE;
    static_assert(TN == 64, "a wavefront's rows are 64 columns");
    static_assert(WM * WN * 32 * ROW * 4 <= LDS, "the tiles' buffers hold the parts");
    float *const part = reinterpret_cast<float *>(smem) + wave * (32 * ROW);
    const int at = (lane % LANES) * 8, n = n0 + wn * (GATED ? 32 : 64) + at;
    // The turns over pairs of fragment rows are not unrolled (only their copies out of the registers are): a workgroup runs
    // this once, and what it costs is largely the fetching of its code.
    const bool vec = a.ep.vec;
    unsigned again = 0;   // fp32: runs with a NaN among them, computed once more below
#pragma unroll 1
    for (int i = 0; i < MF; i += 2) {
        for_each<MF / 2>([&](auto pair) __attribute__((always_inline)) {
            if (i == 2 * pair) {
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int j = 0; j < 4; j++) *reinterpret_cast<floatx4 *>(part + (h * 16 + l16) * ROW + j * 16 + q * 4) = acc[2 * pair + h][j];
            }
        });
        wave_fence();
        // One turn: AT_ONCE rows. AHEAD: a large tile's residual is loaded for all turns first, or each
        // would wait for its own (8192 x 1024 x 4096 of bf16 with a residual 104 -> 96 us).
        T ahead[AHEAD ? TURNS : 1][8];
        const bool use = AHEAD && vec && a.ep.R != nullptr && n + 8 <= a.N && !cut;
        if constexpr (AHEAD) {
            if (use) {
                for_each<TURNS>([&](auto t) __attribute__((always_inline)) {
                    long m = m0 + wm * TM + i * 16 + t * AT_ONCE + lane / LANES;
                    if (m >= a.M) m = a.M - 1;
                    __builtin_memcpy(ahead[t], static_cast<const T *>(a.ep.R) + m * a.ep.ldR + n, 8 * sizeof(T));
                });
            }
        }
        auto turn = [&](int y, const T *residual) __attribute__((always_inline)) {
            const int row = y + lane / LANES;
            const long m = m0 + wm * TM + i * 16 + row;
            const float *src = part + row * ROW + at;
            float v[8], u[8];
            run_load(src, v);
            if constexpr (GATED) run_load(src + 32, u);
            if (m >= a.M || n >= a.N) return;
            if (cut) {
                float *dst = a.pieces + (((long)piece * cut_tiles + cut_tile) * BM + (wm * TM + i * 16 + row)) * BN + wn * TN + at;
                run_store(dst, v);
                if constexpr (GATED) run_store(dst + 32, u);
                return;
            }
            if constexpr (__is_same(T, float)) {
                float sum = 0.f;
#pragma unroll
                for (int e = 0; e < 8; e++) sum += GATED ? v[e] + u[e] : v[e];
                if (sum != sum) {   // (also where infinities of both signs meet: no harm)
                    again |= 1u << (i / 2 * TURNS + y / AT_ONCE);
                    return;
                }
            }
            if (vec && n + 8 <= a.N) {
                if constexpr (GATED) dense_finish_gated<T, 8, true>(a.ep, v, u, m, n);
                else dense_finish<T, 8, FULL, true>(a.ep, v, m, n, 8, residual);
            } else {
                const int left = a.N - n < 8 ? a.N - n : 8;
                if constexpr (GATED) dense_finish_gated<T, 8, false>(a.ep, v, u, m, n, left);
                else dense_finish<T, 8, FULL, false>(a.ep, v, m, n, left);
            }
        };
        if (use) {
            for_each<AHEAD ? TURNS : 0>([&](auto t) __attribute__((always_inline)) { turn(t * AT_ONCE, ahead[t]); });
        } else {
#pragma unroll 1
            for (int y = 0; y < 32; y += AT_ONCE) turn(y, nullptr);
        }
        wave_fence();
    }
    if constexpr (__is_same(T, float)) {
        static_assert(MF / 2 * TURNS <= 32, "one bit per run");
#pragma unroll 1
        while (again) {
            const int bit = __ffs(again) - 1;
            again &= again - 1;
            const long m = m0 + wm * TM + bit / TURNS * 32 + bit % TURNS * AT_ONCE + lane / LANES;
#pragma unroll 1
            for (int e = 0; e < 8 && n + e < a.N; e++) {
                float x[1], z[1] = {0.f};
                x[0] = dense_element(a.A[0], a.A[1], AT ? m : m * a.ldA, AT ? a.ldA : 1, a.B[0], a.B[1], BT ? n + e : (n + e) * a.ldB,
                                     BT ? a.ldB : 1, GATED ? 1 : a.sources, a.K);
                if constexpr (GATED) {
                    z[0] = dense_element(a.A[0], a.A[0], m * a.ldA, 1, a.B[1], a.B[1], (n + e) * a.ldB, 1, 1, a.K);
                    dense_finish_gated<T, 1, false>(a.ep, x, z, m, n + e);
                } else {
                    dense_finish<T, 1, FULL, false>(a.ep, x, m, n + e);
                }
            }
        }
    }
}

}  // namespace alpha
