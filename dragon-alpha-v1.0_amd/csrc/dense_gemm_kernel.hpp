// The dense product's tile kernel: C[m, n] = sum_k A(m, k) B(n, k), bf16 operands, fp32 sums, on v_mfma_f32_16x16x32_bf16.
//
// A workgroup computes BM x BN of C in steps of 64 k. A step's tiles go from memory straight into LDS (128-bit
// buffer loads with LDS as their target) two steps ahead into two buffers; a wavefront owns BM/WM x BN/WN of C in
// registers and reads its operand fragments one half step ahead of the MFMAs that use them, so the one barrier of a step
// falls between two runs of MFMAs whose operands are in registers already.
// Operands may be stored with k along their rows (row r: k = 0, 1, ..: "straight") or with k as the rows ("T"). Straight
// tiles are [rows][64 k] of 128-byte rows whose eight 16-byte chunks are permuted by the row (chunk ^ f(row)), so the 16
// rows that a fragment read touches lie in different banks; T tiles are [64 k][rows] and are read by the transposing LDS
// load, four k of 16 rows per instruction, their 32-byte pieces permuted by k.
// Rows beyond the operand read zeros (the buffer descriptor ends with the last row's last 16-byte chunk: rows are whole
// chunks long, zeros after their last element); k beyond K reads zeros too.
// The MFMA's rows are n and its columns m, so a lane holds runs of consecutive n of one m. Straight B: fragment nf of a
// 64-column group takes the columns 16 * (i / 4) + 4 * nf + i % 4 (i = 0..15), which makes a lane's run 16 long.
#pragma once
#include "dense_common.hpp"

namespace alpha {

typedef unsigned uintx4 __attribute__((ext_vector_type(4)));
typedef short shortx4 __attribute__((ext_vector_type(4)));

struct DenseTileArgs {
    const __bf16 *A[2], *B[2];
    long ldA, ldB, planeA, planeB;
    int M, N, K;
    int nk;            // steps of 64 k
    int combos;        // products per k step: parts (1 or 6) x sources
    int parts6;        // 6 for the three-part split, else 1
    int steps;         // nk * combos
    int split, per;    // the reduction is cut into `split` runs of `per` steps
    int tiles_m, tiles_n;
    DenseEpilogue ep;
    float *partial;    // [split][M][columns of C]
    int columns;       // N, or 2 N where gated (gate columns first)
};

// what leaves the kernel
enum DenseOut { DENSE_PLAIN, DENSE_GATED, DENSE_PARTIAL, DENSE_PARTIAL_GATED };

static __device__ __forceinline__ void load_to_lds(unsigned lds, unsigned voffset, uintx4 rsrc)
{
    // no register is written and nothing of the compiler's waits on it: the kernel's own s_waitcnt does (m0 is reserved to
    // single instructions' use on this target, so nothing of the compiler's lives in it across this)
    asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(voffset), "s"(rsrc) : "memory");
}

static __device__ __forceinline__ uintx4 make_rsrc(const void *p, long bytes)
{
    const uint64_t a = reinterpret_cast<uint64_t>(p);
    const long n = bytes < 0 ? 0 : (bytes > 0x7fffffffl ? 0x7fffffffl : bytes);
    return uintx4{(unsigned)a, (unsigned)(a >> 32) & 0xffffu, (unsigned)n, 0x00020000u};
}

// which parts the c-th of the six products multiplies: (l,h) (h,l) (m,m) (m,h) (h,m) (h,h), small ones first
static __device__ __forceinline__ int combo_part_a(int c) { return (0x052 >> (2 * c)) & 3; }
static __device__ __forceinline__ int combo_part_b(int c) { return (0x118 >> (2 * c)) & 3; }

// One element of C once more in plain fp32, from the parts: taken where the sum of the parts' products is NaN, which it
// also is where one operand is infinite and a part of the other zero. Ends at the first NaN.
static __device__ __attribute__((noinline)) float dense_element(const __bf16 *A0, const __bf16 *A1, long a_row, long a_k, long planeA,
                                                                const __bf16 *B0, const __bf16 *B1, long b_row, long b_k, long planeB,
                                                                int sources, int K)
{
    float acc = 0.f;
    for (int s = 0; s < sources; s++) {
        const __bf16 *a = (s ? A1 : A0) + a_row, *b = (s ? B1 : B0) + b_row;
        for (int k = 0; k < K; k++, a += a_k, b += b_k) {
            const float x = (float)a[0] + (float)a[planeA] + (float)a[2 * planeA];
            const float y = (float)b[0] + (float)b[planeB] + (float)b[2 * planeB];
            acc = fmaf(x, y, acc);
            if (acc != acc) return acc;
        }
    }
    return acc;
}

// The plain epilogue of four consecutive columns n .. n+3 of row m (fewer at the right edge).
template <typename T>
static __device__ __forceinline__ void dense_finish4(const DenseEpilogue &ep, floatx4 v, long m, int n, int N)
{
    const bool second = ep.row2 > 0 && m >= ep.row2;
    if (ep.row2 > 0 && !second && m >= ep.rows1) return;   // a row between two stacked products
    T *Y = static_cast<T *>(second ? ep.Y2 : ep.Y) + (second ? (m - ep.row2) * ep.ldY2 : m * ep.ldY) + n;
    const T *bias = static_cast<const T *>(ep.bias), *R = static_cast<const T *>(ep.R);
    T *Z = static_cast<T *>(ep.Z);
    if (ep.vec && n + 4 <= N) {
        if (bias) v += quad_load(bias + n);
        if (Z) quad_store(Z + m * ep.ldZ + n, v);
        if (ep.act != ALPHA_DENSE_ACT_NONE)
            v = floatx4{dense_act(ep.act, v[0], ep.slope), dense_act(ep.act, v[1], ep.slope), dense_act(ep.act, v[2], ep.slope), dense_act(ep.act, v[3], ep.slope)};
        if (R) v += quad_load(R + m * ep.ldR + n);
        quad_store(Y, v);
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (n + i < N) {
            float z = v[i];
            if (bias) z += dense_load(bias + n + i);
            if (Z) dense_store(Z + m * ep.ldZ + n + i, z);
            z = dense_act(ep.act, z, ep.slope);
            if (R) z += dense_load(R + m * ep.ldR + n + i);
            dense_store(Y + i, z);
        }
}

template <typename T>
static __device__ __forceinline__ void dense_finish4_gated(const DenseEpilogue &ep, floatx4 g, floatx4 u, long m, int n, int N)
{
    T *Y = static_cast<T *>(ep.Y) + m * ep.ldY + n;
    const T *bg = static_cast<const T *>(ep.bias), *bu = static_cast<const T *>(ep.bias2);
    T *G = static_cast<T *>(ep.Z), *U = static_cast<T *>(ep.Z2);
    if (ep.vec && n + 4 <= N) {
        if (bg) g += quad_load(bg + n);
        if (bu) u += quad_load(bu + n);
        if (G) quad_store(G + m * ep.ldZ + n, g);
        if (U) quad_store(U + m * ep.ldZ2 + n, u);
        quad_store(Y, floatx4{dense_act(ep.act, g[0], ep.slope), dense_act(ep.act, g[1], ep.slope), dense_act(ep.act, g[2], ep.slope),
                              dense_act(ep.act, g[3], ep.slope)} * u);
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (n + i < N) {
            const float gi = g[i] + (bg ? dense_load(bg + n + i) : 0.f), ui = u[i] + (bu ? dense_load(bu + n + i) : 0.f);
            if (G) dense_store(G + m * ep.ldZ + n + i, gi);
            if (U) dense_store(U + m * ep.ldZ2 + n + i, ui);
            dense_store(Y + i, dense_act(ep.act, gi, ep.slope) * ui);
        }
}

template <typename T, bool AT, bool BT, DenseOut OUT, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM * WN * 64, 1) void dense_tile_kernel(const DenseTileArgs a)
{
    constexpr int NT = WM * WN * 64, TM = BM / WM, TN = BN / WN, MF = TM / 16, NF = TN / 16;
    constexpr int LA = BM * 8 / NT, LB = BN * 8 / NT;       // 16-byte loads of a thread per step
    constexpr unsigned ABYTES = BM * 128, BBYTES = BN * 128, STAGE = ABYTES + BBYTES;
    constexpr bool GATED = OUT == DENSE_GATED || OUT == DENSE_PARTIAL_GATED;
    constexpr bool PERM = !BT;                              // a lane's columns in runs of 16
    static_assert(TM % 16 == 0 && TN % 64 == 0 && LA >= 1 && LB >= 1 && NT % 256 == 0, "tile shape");
    extern __shared__ char smem[];

    const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WN, wn = wave % WN;

    // The tile: workgroups go round the eight XCDs, so every eighth one shares an L2; an XCD gets a contiguous run of tiles,
    // ordered in panels of 8 tile rows so that the run reuses both operands out of that L2.
    const int tiles = a.tiles_m * a.tiles_n;
    int id = blockIdx.x, piece = 0;
    {
        const int total = tiles * a.split, each = total / 8, more = total % 8, xcd = id & 7, at = id >> 3;
        id = xcd * each + (xcd < more ? xcd : more) + at;
    }
    if (a.split > 1) {
        piece = id / tiles;
        id -= piece * tiles;
    }
    const int panel = id / (8 * a.tiles_n), first = panel * 8, deep = a.tiles_m - first < 8 ? a.tiles_m - first : 8;
    const int tm = first + (id - panel * 8 * a.tiles_n) % deep, tn = (id - panel * 8 * a.tiles_n) / deep;
    const int m0 = tm * BM, n0 = tn * (GATED ? BN / 2 : BN);

    // ---- where the loads of a step come from: a per-lane offset, the rest in the descriptor ----
    unsigned offA[LA], offB[LB];
    int kchunkA = 0, kchunkB = 0;      // straight: first k (within the step) of the lane's chunk
    if constexpr (AT) {
#pragma unroll
        for (int j = 0; j < LA; j++) {
            const int slot = j * NT + tid, row = slot / (BM / 8), c = (slot % (BM / 8)) ^ ((row & 3) << 1);
            offA[j] = (unsigned)((long)row * a.ldA * 2) + c * 16;
        }
    } else {
        kchunkA = ((lane & 7) ^ (lane >> 3)) * 8;
#pragma unroll
        for (int j = 0; j < LA; j++) offA[j] = (unsigned)((long)(j * (NT / 8) + (tid >> 3)) * a.ldA * 2) + kchunkA * 2;
    }
    if constexpr (BT) {
#pragma unroll
        for (int j = 0; j < LB; j++) {
            const int slot = j * NT + tid, row = slot / (BN / 8), c = (slot % (BN / 8)) ^ ((row & 3) << 1);
            offB[j] = (unsigned)((long)row * a.ldB * 2) + c * 16;
        }
    } else {
        // tile row r; its bank permutation uses bits 0, 1 and 4, the ones that differ within a fragment's 16 rows
        kchunkB = ((lane & 7) ^ (((lane >> 3) & 3) | (((wave >> 1) & 1) << 2))) * 8;
#pragma unroll
        for (int j = 0; j < LB; j++) {
            const int r = j * (NT / 8) + (tid >> 3);
            // gated: of every 16 tile rows the first 8 are the gate's filter, the last 8 the other's (one filter per wavefront's load)
            const int row = GATED ? (r >> 6) * 32 + ((r >> 4) & 3) * 8 + (r & 7) : r;
            offB[j] = (unsigned)((long)row * a.ldB * 2) + kchunkB * 2;
        }
    }

    // ---- the steps of this workgroup ----
    const int t0 = piece * a.per;
    int left = a.steps - t0;
    if (left > a.per) left = a.per;
    int kt = t0 / a.combos, combo = t0 % a.combos;    // of the next step to load

    const unsigned lds0 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char *)smem;
    auto load_step = [&](unsigned stage) {
        const int src = combo >= a.parts6 ? 1 : 0, c = combo - src * a.parts6;
        const int pa = a.parts6 == 6 ? combo_part_a(c) : 0, pb = a.parts6 == 6 ? combo_part_b(c) : 0;
        const int krem = kt < a.nk ? a.K - kt * 64 : 0;   // beyond the last step: nothing
        const __bf16 *pA = (src ? a.A[1] : a.A[0]) + pa * a.planeA;
        const __bf16 *pB = (GATED ? ((wave & 1) ? a.B[1] : a.B[0]) : (src ? a.B[1] : a.B[0])) + pb * a.planeB;
        long bytesA, bytesB;
        if constexpr (AT) {
            pA += (long)kt * 64 * a.ldA + m0;
            bytesA = krem > 0 ? ((long)(krem - 1) * a.ldA + ((a.M - m0 + 7) & ~7)) * 2 : 0;
        } else {
            const int rows = a.M - m0 < BM ? a.M - m0 : BM;
            pA += (long)m0 * a.ldA + kt * 64;
            bytesA = krem > 0 ? ((long)(rows - 1) * a.ldA + ((krem + 7) & ~7)) * 2 : 0;
        }
        if constexpr (BT) {
            pB += (long)kt * 64 * a.ldB + n0;
            bytesB = krem > 0 ? ((long)(krem - 1) * a.ldB + ((a.N - n0 + 7) & ~7)) * 2 : 0;
        } else {
            const int span = GATED ? BN / 2 : BN, rows = a.N - n0 < span ? a.N - n0 : span;
            pB += (long)n0 * a.ldB + kt * 64;
            bytesB = krem > 0 ? ((long)(rows - 1) * a.ldB + ((krem + 7) & ~7)) * 2 : 0;
        }
        const uintx4 rA = make_rsrc(pA, bytesA), rB = make_rsrc(pB, bytesB);
        const unsigned lds = __builtin_amdgcn_readfirstlane(lds0 + stage + wave * 1024);
        const bool inA = AT || kchunkA < krem, inB = BT || kchunkB < krem;   // a straight row goes on into the next one
#pragma unroll
        for (int j = 0; j < LA; j++) load_to_lds(lds + j * NT * 16, inA ? offA[j] : 0x80000000u, rA);
#pragma unroll
        for (int j = 0; j < LB; j++) load_to_lds(lds + ABYTES + j * NT * 16, inB ? offB[j] : 0x80000000u, rB);
        if (++combo == a.combos) {
            combo = 0;
            kt++;
        }
    };

    // ---- where the fragments are read ----
    typedef __attribute__((address_space(3))) char lds_char;
    unsigned rdA[AT ? 4 : 1], rdB[BT ? 4 : 1];
    if constexpr (AT) {
#pragma unroll
        for (int x = 0; x < 4; x++)
            rdA[x] = (q * 8 + (l16 >> 2)) * (BM * 2) + wm * (TM / 16) * 32 + ((x ^ (l16 >> 2)) * 32) + ((l16 & 3) >> 1) * 16 + (l16 & 1) * 8;
    } else {
        rdA[0] = (wm * TM + l16) * 128 + ((q ^ (l16 & 7)) * 16);
    }
    if constexpr (BT) {
#pragma unroll
        for (int x = 0; x < 4; x++)
            rdB[x] = ABYTES + (q * 8 + (l16 >> 2)) * (BN * 2) + wn * (TN / 16) * 32 + ((x ^ (l16 >> 2)) * 32) + ((l16 & 3) >> 1) * 16 + (l16 & 1) * 8;
    } else {
        rdB[0] = ABYTES + (wn * TN + (l16 >> 2) * 16 + (l16 & 3)) * 128 + ((q ^ (l16 & 7)) * 16);
    }
    auto read_a = [&](unsigned stage, int ks, bf16x8 (&f)[MF]) {
#pragma unroll
        for (int i = 0; i < MF; i++) {
            if constexpr (AT) {
                const unsigned at = stage + rdA[i & 3] + (i >> 2) * 128 + ks * 32 * (BM * 2);
                const shortx4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) shortx4 *)((lds_char *)smem + at));
                const shortx4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) shortx4 *)((lds_char *)smem + at + 4 * (BM * 2)));
                f[i] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
            } else {
                f[i] = *(const __attribute__((address_space(3))) bf16x8 *)((lds_char *)smem + stage + (rdA[0] ^ (ks * 64)) + i * 2048);
            }
        }
    };
    auto read_b = [&](unsigned stage, int ks, bf16x8 (&f)[NF]) {
#pragma unroll
        for (int i = 0; i < NF; i++) {
            if constexpr (BT) {
                const unsigned at = stage + rdB[i & 3] + (i >> 2) * 128 + ks * 32 * (BN * 2);
                const shortx4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) shortx4 *)((lds_char *)smem + at));
                const shortx4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) shortx4 *)((lds_char *)smem + at + 4 * (BN * 2)));
                f[i] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
            } else {
                f[i] = *(const __attribute__((address_space(3))) bf16x8 *)((lds_char *)smem + stage + (rdB[0] ^ (ks * 64)) + (i >> 2) * 8192 + (i & 3) * 512);
            }
        }
    };

    floatx4 acc[MF][NF];
#pragma unroll
    for (int i = 0; i < MF; i++)
#pragma unroll
        for (int j = 0; j < NF; j++) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
    auto multiply = [&](const bf16x8 (&fa)[MF], const bf16x8 (&fb)[NF]) {
#pragma unroll
        for (int i = 0; i < MF; i++)
#pragma unroll
            for (int j = 0; j < NF; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[j], fa[i], acc[i][j], 0, 0, 0);
    };

    bf16x8 a0[MF], b0[NF], a1[MF], b1[NF];
    load_step(0);
    load_step(STAGE);
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(LA + LB) : "memory");
    read_a(0, 0, a0);
    read_b(0, 0, b0);
    unsigned stage = 0;
    for (int t = 0; t < left; t++) {
        read_a(stage, 1, a1);
        read_b(stage, 1, b1);
        multiply(a0, b0);
        // all reads of this step's tiles are done and the next step's tiles have landed, for every wavefront
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        load_step(stage);
        stage ^= STAGE;
        read_a(stage, 0, a0);
        read_b(stage, 0, b0);
        multiply(a1, b1);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // no load may reach LDS after the workgroup has gone

    // ---- out ----
    // Column of fragment group g (64 columns), run j; gated: of the gate's fragment g + j and its partner g + j + 2.
    auto column = [&](int g, int j) {
        const int col = wn * TN + g * 16;
        return n0 + (GATED ? col / 2 + q * 8 + j * 4 : col + (PERM ? q * 16 + j * 4 : j * 16 + q * 4));
    };
    constexpr int RUNS = GATED ? 2 : 4;
    unsigned again = 0;   // fp32: runs with a NaN among them, computed once more below
#pragma unroll
    for (int i = 0; i < MF; i++) {
        const int m = m0 + wm * TM + i * 16 + l16;
        if (m >= a.M) continue;
#pragma unroll
        for (int g = 0; g < NF; g += 4) {
#pragma unroll
            for (int j = 0; j < RUNS; j++) {
                const int n = column(g, j);
                if (n >= a.N) continue;
                const floatx4 v = acc[i][g + j], u = acc[i][GATED ? g + j + 2 : g + j];
                if constexpr (OUT == DENSE_PARTIAL || OUT == DENSE_PARTIAL_GATED) {
                    float *dst = a.partial + ((long)piece * a.M + m) * a.columns + n;
                    if ((a.N & 3) == 0) {
                        *reinterpret_cast<floatx4 *>(dst) = v;
                        if constexpr (GATED) *reinterpret_cast<floatx4 *>(dst + a.N) = u;
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            if (n + e < a.N) {
                                dst[e] = v[e];
                                if constexpr (GATED) dst[a.N + e] = u[e];
                            }
                    }
                } else {
                    if constexpr (__is_same(T, float)) {
                        const float sum = (v[0] + v[1]) + (v[2] + v[3]) + (GATED ? (u[0] + u[1]) + (u[2] + u[3]) : 0.f);
                        if (sum != sum) {   // (also where infinities of both signs meet: no harm)
                            again |= 1u << (i * (NF / 4 * RUNS) + g / 4 * RUNS + j);
                            continue;
                        }
                    }
                    if constexpr (GATED) dense_finish4_gated<T>(a.ep, v, u, m, n, a.N);
                    else dense_finish4<T>(a.ep, v, m, n, a.N);
                }
            }
        }
    }
    if constexpr (__is_same(T, float) && (OUT == DENSE_PLAIN || OUT == DENSE_GATED)) {
        static_assert(MF * (NF / 4) * RUNS <= 32, "one bit per run");
        while (again) {
            const int bit = __ffs(again) - 1, i = bit / (NF / 4 * RUNS), g = bit / RUNS % (NF / 4) * 4, j = bit % RUNS;
            again &= again - 1;
            const long m = m0 + wm * TM + i * 16 + l16;
            const int n = column(g, j);
            floatx4 v{0.f, 0.f, 0.f, 0.f}, u = v;
            for (int e = 0; e < 4 && n + e < a.N; e++) {
                const float x = dense_element(a.A[0], a.A[1], AT ? m : m * a.ldA, AT ? a.ldA : 1, a.planeA, a.B[0], a.B[1],
                                              BT ? n + e : (n + e) * a.ldB, BT ? a.ldB : 1, a.planeB, GATED ? 1 : a.combos / a.parts6, a.K);
                const float y = GATED ? dense_element(a.A[0], a.A[0], m * a.ldA, 1, a.planeA, a.B[1], a.B[1], (n + e) * a.ldB, 1, a.planeB, 1, a.K) : 0.f;
                v[0] = e == 0 ? x : v[0], v[1] = e == 1 ? x : v[1], v[2] = e == 2 ? x : v[2], v[3] = e == 3 ? x : v[3];
                u[0] = e == 0 ? y : u[0], u[1] = e == 1 ? y : u[1], u[2] = e == 2 ? y : u[2], u[3] = e == 3 ? y : u[3];
            }
            if constexpr (GATED) dense_finish4_gated<T>(a.ep, v, u, m, n, a.N);
            else dense_finish4<T>(a.ep, v, m, n, a.N);
        }
    }
}

}  // namespace alpha
