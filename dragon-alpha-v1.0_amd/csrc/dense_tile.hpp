// What the dense tile kernels share: their arguments, the order of the tiles, the bank permutations of their LDS tiles and how
// a finished tile leaves.
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

static __device__ __forceinline__ bool finite_sum(float v) { return fabsf(v) <= 3.40282347e38f; }

// fp32: 16 rows of C (from m0 on, 64 columns from n0 on, at `part` in LDS) whose sums are not all finite, once more as plain fp32
// products over the workgroup's reduction (cut tiles: its piece of it), on v_mfma_f32_16x16x4_f32 with operands straight from memory; what is
// finite stays the sum of the parts. 16 k a turn, the lane's being k + 4 (lane / 16) + s in the s-th MFMA. What lies beyond M, N or
// K is not read (the last row, column or k again), and what is beyond M or N not looked at. All wavefronts and pieces work side by
// side, none longer than its own part of the product: 12544 x 256 -> 1024 forward 62 us, with one infinity in X 76, all of X infinite
// 198; its backward 104, 251 and 357.
template <bool AT, bool BT, bool GATED>
static __device__ __forceinline__ void plain_rows(const DenseTileArgs &a, float *part, int row_floats, int lane, int m0, int n0, int k_first, int k_end)
{
    const int l16 = lane & 15, q = lane >> 4, m = m0 + l16;
    float *const mine = part + l16 * row_floats + q * 4;      // + 16 j: four columns of fragment j
    bool any = false;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const floatx4 v = *reinterpret_cast<const floatx4 *>(mine + 16 * j);
        const int n = n0 + 16 * (GATED ? j & 1 : j) + 4 * q;
#pragma unroll
        for (int e = 0; e < 4; e++) any |= m < a.M && n + e < a.N && !finite_sum(v[e]);
    }
    if (__ballot(any) == 0) return;     // uniform
    const long row = (m < a.M ? m : a.M - 1) * (AT ? 1 : a.ldA);
    long col[4];
    floatx4 c[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int n = n0 + 16 * (GATED ? j & 1 : j) + l16;
        col[j] = (n < a.N ? n : a.N - 1) * (BT ? 1 : a.ldB);
        c[j] = floatx4{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll 1
    for (int source = 0; source < (GATED ? 1 : a.sources); source++) {
        const float *A = static_cast<const float *>(source ? a.A[1] : a.A[0]) + row;
        const float *B0 = static_cast<const float *>(source ? a.B[1] : a.B[0]), *B1 = GATED ? static_cast<const float *>(a.B[1]) : B0;
        // four consecutive k of a row or column: 16 bytes, or four rows
        auto load = [&](auto whole, const float *p, long ld, int k, float (&v)[4]) __attribute__((always_inline)) {
            if (whole && ld == 1) {
                __builtin_memcpy(v, p + k, 16);
                return;
            }
#pragma unroll
            for (int s = 0; s < 4; s++) v[s] = p[(whole || k + s < k_end ? k + s : k_end - 1) * ld];
        };
        auto turn = [&](auto whole, int k) __attribute__((always_inline)) {
            float x[4], w[4][4];
            load(whole, A, AT ? a.ldA : 1, k, x);
#pragma unroll
            for (int j = 0; j < 4; j++) load(whole, (GATED && j >= 2 ? B1 : B0) + col[j], BT ? a.ldB : 1, k, w[j]);
#pragma unroll
            for (int s = 0; s < 4; s++) {
                const bool there = whole || k + s < k_end;
#pragma unroll
                for (int j = 0; j < 4; j++) c[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(there ? w[j][s] : 0.f, there ? x[s] : 0.f, c[j], 0, 0, 0);
            }
        };
        int k0 = k_first;
#pragma unroll 1
        for (; k0 + 16 <= k_end; k0 += 16) turn(std::true_type{}, k0 + 4 * q);
        if (k0 < k_end) turn(std::false_type{}, k0 + 4 * q);
    }
#pragma unroll
    for (int j = 0; j < 4; j++) {
        floatx4 *const to = reinterpret_cast<floatx4 *>(mine + 16 * j);
        floatx4 v = *to;
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = finite_sum(v[e]) ? v[e] : c[j][e];
        *to = v;
    }
}

// A finished tile leaves two fragment rows (32 rows of C) at a time through the wavefront's part of LDS, so that a lane then has
// eight consecutive columns and a row goes out as one run: stored from the MFMA's registers as they are, 4096 x 4096 of bf16
// took 17 us to write, this way 10. acc[i][j][e]: row 16 i + lane % 16, column 16 j + 4 (lane / 16) + e of the wavefront's part
// of the tile. Every wavefront is done with the tiles in LDS.
template <typename T, bool AT, bool BT, bool GATED, int BM, int BN, int WM, int WN, int LDS>
static __device__ __forceinline__ void tile_out(const DenseTileArgs &a, const floatx4 (&acc)[BM / WM / 16][BN / WN / 16], char *smem, int lane, int wave, int wm,
                                                int wn, int m0, int n0, bool cut, int piece, int cut_tile, int cut_tiles, int k_first = 0,
                                                int k_end = 0)
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
    // fp32: an operand that is infinite or NaN (or within 2^-9 of the end of the range) makes NaN of the products of its parts
    bool again = false;
    if constexpr (__is_same(T, float)) {
        float check = 0.f;     // NaN as soon as one of the sums is not finite
#pragma unroll
        for (int i = 0; i < MF; i++)
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int e = 0; e < 4; e++) check = fmaf(acc[i][j][e], 0.f, check);
        again = __ballot(check != check) != 0;
    }
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
        if constexpr (__is_same(T, float)) {
            if (again) {   // uniform; a lane reads and writes what it wrote itself
#pragma unroll 1
                for (int h = 0; h < 2; h++)
                    plain_rows<AT, BT, GATED>(a, part + h * 16 * ROW, ROW, lane, m0 + wm * TM + (i + h) * 16, n0 + wn * (GATED ? 32 : 64), k_first, k_end);
            }
        }
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
}

}  // namespace alpha
