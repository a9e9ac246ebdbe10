// The dense product's tile kernel: C[m, n] = sum_k A(m, k) B(n, k), bf16 operands, fp32 sums, on v_mfma_f32_16x16x32_bf16.
//
// A workgroup computes BM x BN of C in steps of 32 k. A step's tiles go from memory straight into LDS (128-bit buffer
// loads with LDS as their target) through a ring of STAGES buffers, that many steps ahead; a wavefront owns BM/WM x BN/WN of C in
// registers and reads the operand fragments of a step while it multiplies those of the step before, so the one barrier of
// a step falls between two runs of MFMAs whose operands are in registers already.
// Operands may be stored with k along their rows (row r: k = 0, 1, ..: "straight") or with k as the rows ("T"). Straight
// tiles are [rows][32 k] of 64-byte rows whose four 16-byte chunks are permuted by the row, so the 16 lanes that LDS serves
// in a cycle (eight rows, two chunks each) touch different banks; T tiles are [32 k][rows] and are read by the transposing
// LDS load, four k of 16 rows per instruction, their 32-byte pieces permuted by k.
// Rows beyond the operand read zeros (the buffer descriptor ends with the last row's last 16-byte chunk: rows are whole
// chunks long, zeros after their last element); k beyond K reads zeros too.
// The MFMA's rows are n and its columns m, so a lane holds four consecutive n of one m. A finished tile goes through LDS
// (each wavefront its own part) so that every lane then has eight consecutive columns and a row leaves as one run of 128
// bytes: stored from the registers as they are, 4096 x 4096 of bf16 took 17 us to write, this way 10.
// Gated: of every 64 tile columns 32 are of one filter and 32, the same ones, of the other.
#pragma once
#include "dense_finish.hpp"

#include <type_traits>

namespace alpha {

typedef unsigned uintx4 __attribute__((ext_vector_type(4)));
typedef short shortx4 __attribute__((ext_vector_type(4)));

struct DenseTileArgs {
    const __bf16 *A[2], *B[2];
    long ldA, ldB, planeA, planeB;
    int M, N, K;
    int combos;        // products per 32 k: parts (1 or 6) x sources
    int parts6;        // 6 for the three-part split, else 1
    int steps;         // combos for every 32 k
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

static __device__ __forceinline__ void load_to_lds(unsigned lds, unsigned voffset, uintx4 rsrc)
{
    // no register is written and nothing of the compiler's waits on it: the kernel's own s_waitcnt does (m0 is reserved to
    // single instructions' use on this target, so nothing of the compiler's lives in it across this)
    asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(voffset), "s"(rsrc) : "memory");
}

static __device__ __forceinline__ uintx4 make_rsrc(const void *p, unsigned bytes)   // bytes < 2^31: lanes that must read zeros ask for 2^31
{
    const uint64_t a = reinterpret_cast<uint64_t>(p);
    return uintx4{(unsigned)a, (unsigned)(a >> 32) & 0xffffu, bytes, 0x00020000u};
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

template <typename T, bool AT, bool BT, bool GATED, int BM, int BN, int WM, int WN, int STAGES>
__global__ __launch_bounds__(WM * WN * 64, 1) void dense_tile_kernel(const DenseTileArgs a)
{
    constexpr int NT = WM * WN * 64, TM = BM / WM, TN = BN / WN, MF = TM / 16, NF = TN / 16;
    constexpr int LA = BM * 4 / NT, LB = BN * 4 / NT;       // 16-byte loads of a thread per step
    constexpr unsigned ABYTES = BM * 64, BBYTES = BN * 64, STAGE = ABYTES + BBYTES, RING = STAGES * STAGE;
    static_assert(TM % 16 == 0 && TN % 64 == 0 && LA >= 1 && LB >= 1 && NT % 256 == 0, "tile shape");
    extern __shared__ char smem[];

    const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WN, wn = wave % WN;

    const int cut_tiles = a.tiles_m * a.tiles_n - a.whole;
    const bool cut = (int)blockIdx.x >= a.whole;
    int piece = 0, tile, tm, tn;
    if (cut) {   // piece by piece over all cut tiles: neighbours read the same k
        const int at = xcd_place((int)blockIdx.x - a.whole, cut_tiles * a.split);
        piece = at / cut_tiles;
        tile = a.whole + at % cut_tiles;
    } else {
        tile = xcd_place((int)blockIdx.x, a.whole);
    }
    tile_at(tile, a.tiles_m, a.tiles_n, tm, tn);
    const int m0 = tm * BM, n0 = tn * (GATED ? BN / 2 : BN);

    // ---- where the loads of a step come from: a per-lane offset, the rest in the descriptor ----
    unsigned offA[LA], offB[LB];
    int kchunkA = 0, kchunkB = 0;      // straight: first k (within the step) of the lane's chunk
    if constexpr (AT) {
#pragma unroll
        for (int j = 0; j < LA; j++) {
            const int slot = j * NT + tid, row = slot / (BM / 8), c = (slot % (BM / 8)) ^ t_permutation(row);
            offA[j] = (unsigned)((long)row * a.ldA * 2) + c * 16;
        }
    } else {
        kchunkA = ((lane & 3) ^ s_permutation(lane >> 4)) * 8;    // tile row .. + (lane >> 2)
#pragma unroll
        for (int j = 0; j < LA; j++) offA[j] = (unsigned)((long)(j * (NT / 4) + (tid >> 2)) * a.ldA * 2) + kchunkA * 2;
    }
    if constexpr (BT) {
#pragma unroll
        for (int j = 0; j < LB; j++) {
            const int slot = j * NT + tid, row = slot / (BN / 8), c = (slot % (BN / 8)) ^ t_permutation(row);
            offB[j] = (unsigned)((long)row * a.ldB * 2) + c * 16;
        }
    } else {
        kchunkB = ((lane & 3) ^ s_permutation(lane >> 4)) * 8;
#pragma unroll
        for (int j = 0; j < LB; j++) {
            const int r = j * (NT / 4) + (tid >> 2);
            const int row = GATED ? (r >> 6) * 32 + (r & 31) : r;   // gated: 32 rows of one filter, 32 of the other
            offB[j] = (unsigned)((long)row * a.ldB * 2) + kchunkB * 2;
        }
    }

    // ---- the steps of this workgroup ----
    const int t0 = piece * a.per;
    int left = a.steps - t0;
    if (cut && left > a.per) left = a.per;
    int combo = t0 % a.combos;                         // of the next step to load
    int krem = a.K - t0 / a.combos * 32;               // k from its first on; <= 0: nothing, zeros
    const long stepA = AT ? 32 * a.ldA : 32, stepB = BT ? 32 * a.ldB : 32;
    const long atA = AT ? (long)m0 : (long)m0 * a.ldA, atB = BT ? (long)n0 : (long)n0 * a.ldB;
    const __bf16 *pA = a.A[0] + atA + t0 / a.combos * stepA, *pB = a.B[0] + atB + t0 / a.combos * stepB;   // first source, first part
    const long toA1 = a.A[1] - a.A[0], toB1 = a.B[1] - a.B[0];
    // bytes from a tile's first element to its end: straight, its rows' last chunk; T, of one k row
    const int spanN = GATED ? BN / 2 : BN;
    const unsigned endA = AT ? (unsigned)((a.M - m0 + 7) & ~7) * 2 : (unsigned)(((long)((a.M - m0 < BM ? a.M - m0 : BM) - 1) * a.ldA + 32) * 2);
    const unsigned endB = BT ? (unsigned)((a.N - n0 + 7) & ~7) * 2 : (unsigned)(((long)((a.N - n0 < spanN ? a.N - n0 : spanN) - 1) * a.ldB + 32) * 2);

    const unsigned lds0 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char *)smem;
    uintx4 rA, rB;
    unsigned lds;
    bool inA, inB;
    const __bf16 *qA, *qB;
    // the descriptors of the next step's loads, in four parts that the main loop spreads between its MFMAs
    auto load_begin = [&](unsigned stage, int part) {
        if (part == 0) {
            qA = pA;
            qB = pB;
            if (a.combos > 1) {   // uniform
                const bool second = combo >= a.parts6;
                const int c = second ? combo - a.parts6 : combo;
                if (second) {
                    qA += toA1;
                    qB += toB1;
                }
                if (a.parts6 == 6) {
                    qA += combo_part_a(c) * a.planeA;
                    qB += combo_part_b(c) * a.planeB;
                }
            }
            if (GATED && (wave & 2)) qB += toB1;
        } else if (part == 1) {
            const int rows = krem < 32 ? krem : 32;
            rA = make_rsrc(qA, !AT ? endA : rows > 0 ? (unsigned)(rows - 1) * (unsigned)(a.ldA * 2) + endA : 0u);
            inA = AT || kchunkA < krem;   // a straight row goes on into the next one
        } else if (part == 2) {
            const int rows = krem < 32 ? krem : 32;
            rB = make_rsrc(qB, !BT ? endB : rows > 0 ? (unsigned)(rows - 1) * (unsigned)(a.ldB * 2) + endB : 0u);
            inB = BT || kchunkB < krem;
        } else {
            lds = __builtin_amdgcn_readfirstlane(lds0 + stage + wave * 1024);
            if (++combo == a.combos) {
                combo = 0;
                krem -= 32;
                pA += stepA;
                pB += stepB;
            }
        }
    };
    auto load_one = [&](int j) {
        if (j < LA) load_to_lds(lds + j * NT * 16, inA ? offA[j < LA ? j : 0] : 0x80000000u, rA);
        else load_to_lds(lds + ABYTES + (j - LA) * NT * 16, inB ? offB[j < LA ? 0 : j - LA] : 0x80000000u, rB);
    };

    // ---- where the fragments are read ----
    typedef __attribute__((address_space(3))) char lds_char;
    unsigned rdA[AT ? MF : 1], rdB[BT ? NF : 1];                 // (a T fragment's piece is permuted by the lane: an address each)
    const int tk = q * 8 + (l16 >> 2), t16 = (l16 & 3) >> 1;     // T: the lane's k row and 16-byte half of a piece
    const int chunk = (q ^ s_permutation(l16 >> 2)) * 16;
    if constexpr (AT) {
#pragma unroll
        for (int x = 0; x < MF; x++) rdA[x] = tk * (BM * 2) + (((wm * MF + x) * 2 + t16) ^ t_permutation(tk)) * 16 + (l16 & 1) * 8;
    } else {
        rdA[0] = (wm * TM + l16) * 64 + chunk;
    }
    if constexpr (BT) {
#pragma unroll
        for (int x = 0; x < NF; x++) rdB[x] = ABYTES + tk * (BN * 2) + (((wn * NF + x) * 2 + t16) ^ t_permutation(tk)) * 16 + (l16 & 1) * 8;
    } else {
        rdB[0] = ABYTES + (wn * TN + l16) * 64 + chunk;
    }
    auto read_t = [&](unsigned at, int row_bytes) {   // k .. k+3 and k+4 .. k+7 of the lane's row
        const shortx4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) shortx4 *)((lds_char *)smem + at));
        const shortx4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) shortx4 *)((lds_char *)smem + at + 4 * row_bytes));
        return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    auto read_a = [&](unsigned stage, int i) -> bf16x8 {
        if constexpr (AT) return read_t(stage + rdA[i], BM * 2);
        else return *(const __attribute__((address_space(3))) bf16x8 *)((lds_char *)smem + stage + rdA[0] + i * 1024);
    };
    auto read_b = [&](unsigned stage, int i) -> bf16x8 {
        if constexpr (BT) return read_t(stage + rdB[i], BN * 2);
        else return *(const __attribute__((address_space(3))) bf16x8 *)((lds_char *)smem + stage + rdB[0] + i * 1024);
    };

    floatx4 acc[MF][NF];
#pragma unroll
    for (int i = 0; i < MF; i++)
#pragma unroll
        for (int j = 0; j < NF; j++) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
    // The MFMAs of a step. Between them, one at a time, so that none keeps the next MFMA waiting: the reads of the next
    // step's fragments (B's first, since its first row needs all of them), the loads of the step STAGES ahead (into the
    // buffer of this step's tiles, which are in registers), and towards the end the scalar arithmetic of the next loads. So
    // nothing stands between the barrier and the MFMAs, and the wait before the next barrier finds the reads done.
    unsigned stage = 0;
    auto step = [&](const bf16x8 (&fa)[MF], const bf16x8 (&fb)[NF], bf16x8 (&na)[MF], bf16x8 (&nb)[NF]) {
        constexpr int READS = MF + NF, LOADS = LA + LB, ALL = MF * NF, EARLY = ALL * 3 / 4;
        // this step's fragments are in every wavefront's registers and the next step's tiles have landed, STAGES - 2 more on their way
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((STAGES - 2) * LOADS) : "memory");
        __builtin_amdgcn_sched_barrier(0);
        const unsigned next = stage + STAGE == RING ? 0 : stage + STAGE;
        for_each<ALL>([&](auto at) __attribute__((always_inline)) {
            constexpr int x = at;
            for_each<READS>([&](auto read) __attribute__((always_inline)) {
                constexpr int r = read;
                if constexpr (r * EARLY / READS == x) {
                    if constexpr (r < NF) nb[r] = read_b(next, r);
                    else na[r - NF] = read_a(next, r - NF);
                }
            });
            for_each<LOADS>([&](auto load) __attribute__((always_inline)) {
                constexpr int j = load;
                if constexpr ((2 * j + 1) * EARLY / (2 * LOADS) == x) load_one(j);
            });
            for_each<4>([&](auto c) __attribute__((always_inline)) {
                if constexpr (EARLY + c * (ALL - EARLY) / 4 == x) load_begin(next, c);
            });
            acc[x / NF][x % NF] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[x % NF], fa[x / NF], acc[x / NF][x % NF], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        });
        stage = next;
    };

    bf16x8 a0[MF], b0[NF], a1[MF], b1[NF];
#pragma unroll
    for (int r = 0; r < STAGES; r++) {
        for (int c = 0; c < 4; c++) load_begin(r * STAGE, c);
#pragma unroll
        for (int j = 0; j < LA + LB; j++) load_one(j);
    }
    for (int c = 0; c < 4; c++) load_begin(0, c);
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((STAGES - 1) * (LA + LB)) : "memory");
#pragma unroll
    for (int i = 0; i < NF; i++) b0[i] = read_b(0, i);
#pragma unroll
    for (int i = 0; i < MF; i++) a0[i] = read_a(0, i);
    for (int t = 0; t < left; t += 2) {   // (an odd number of steps ends with one of zeros: the loads beyond the last are none)
        step(a0, b0, a1, b1);
        step(a1, b1, a0, b0);
    }
    asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");   // every load into LDS has landed, every read of it is done

    // ---- out: two fragment rows (32 rows of C) at a time through the wavefront's part of LDS ----
    constexpr int ROW = 68;                              // floats from row to row: 16 bytes past a multiple of the banks
    constexpr int LANES = GATED ? 4 : 8;                 // lanes of a row, eight columns each (gated: eight of each filter)
    constexpr int AT_ONCE = 64 / LANES, TURNS = 32 / AT_ONCE;
    static_assert(TN == 64, "a wavefront's rows are 64 columns");
    static_assert(WM * WN * 32 * ROW * 4 <= (int)RING, "the ring holds the parts");
    float *const part = reinterpret_cast<float *>(smem) + wave * (32 * ROW);
    const int at = (lane % LANES) * 8, n = n0 + wn * (GATED ? 32 : 64) + at;
    unsigned again = 0;   // fp32: runs with a NaN among them, computed once more below
#pragma unroll
    for (int i = 0; i < MF; i += 2) {
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int j = 0; j < 4; j++) *reinterpret_cast<floatx4 *>(part + (h * 16 + l16) * ROW + j * 16 + q * 4) = acc[i + h][j];
        wave_fence();
#pragma unroll 1
        for (int y = 0; y < 32; y += AT_ONCE) {
            const int row = y + lane / LANES;
            const long m = m0 + wm * TM + i * 16 + row;
            float v[8], u[8];
            run_load(part + row * ROW + at, v);
            if constexpr (GATED) run_load(part + row * ROW + 32 + at, u);
            if (m >= a.M || n >= a.N) continue;
            if (cut) {
                float *dst = a.pieces + (((long)piece * cut_tiles + (tile - a.whole)) * BM + (wm * TM + i * 16 + row)) * BN + wn * TN + at;
                run_store(dst, v);
                if constexpr (GATED) run_store(dst + 32, u);
            } else {
                if constexpr (__is_same(T, float)) {
                    float sum = 0.f;
#pragma unroll
                    for (int e = 0; e < 8; e++) sum += GATED ? v[e] + u[e] : v[e];
                    if (sum != sum) {   // (also where infinities of both signs meet: no harm)
                        again |= 1u << (i / 2 * TURNS + y / AT_ONCE);
                        continue;
                    }
                }
                if constexpr (GATED) dense_finish_gated<T>(a.ep, v, u, m, n, a.N);
                else dense_finish<T>(a.ep, v, m, n, a.N);
            }
        }
        wave_fence();
    }
    if constexpr (__is_same(T, float)) {
        static_assert(MF / 2 * TURNS <= 32, "one bit per run");
        while (again) {
            const int bit = __ffs(again) - 1;
            again &= again - 1;
            const long m = m0 + wm * TM + bit / TURNS * 32 + bit % TURNS * AT_ONCE + lane / LANES;
            for (int e = 0; e < 8 && n + e < a.N; e++) {
                float v[1], u[1] = {0.f};
                v[0] = dense_element(a.A[0], a.A[1], AT ? m : m * a.ldA, AT ? a.ldA : 1, a.planeA, a.B[0], a.B[1], BT ? n + e : (n + e) * a.ldB,
                                     BT ? a.ldB : 1, a.planeB, GATED ? 1 : a.combos / a.parts6, a.K);
                if constexpr (GATED) {
                    u[0] = dense_element(a.A[0], a.A[0], m * a.ldA, 1, a.planeA, a.B[1], a.B[1], (n + e) * a.ldB, 1, a.planeB, 1, a.K);
                    dense_finish_gated<T>(a.ep, v, u, m, n + e, a.N);
                } else {
                    dense_finish<T>(a.ep, v, m, n + e, a.N);
                }
            }
        }
    }
}

}  // namespace alpha
