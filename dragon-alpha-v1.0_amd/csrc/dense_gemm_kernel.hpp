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
// Rows beyond the operand read zeros (the buffer descriptor ends with the last row's last 16-byte chunk of the step, dense_bounds.hpp:
// rows are whole chunks long, zeros after their last element); k beyond K reads zeros too.
// The MFMA's rows are n and its columns m, so a lane holds four consecutive n of one m. A finished tile goes through LDS
// (each wavefront its own part) so that every lane then has eight consecutive columns and a row leaves as one run of 128
// bytes: stored from the registers as they are, 4096 x 4096 of bf16 took 17 us to write, this way 10.
// Gated: of every 64 tile columns 32 are of one filter and 32, the same ones, of the other.
// Measured: 8192 x 4096 x 8192 391 us, 1405 TF; the matrix pipe is busy 66 % of the cycles, at 1.6 GHz: the card's power limit sets the
// clock (the same product of zeros runs at 1776 TF). With bias, SiLU and a residual (8192 x 8192 x 4096) 455 us
// (443 to 460 from card to card). 1 % of the LDS
// cycles are bank conflicts.
#pragma once
#include "dense_bounds.hpp"
#include "dense_tile.hpp"

namespace alpha {

static __device__ __forceinline__ void load_to_lds(unsigned lds, unsigned voffset, uintx4 rsrc)
{
    // no register is written and nothing of the compiler's waits on it: the kernel's own s_waitcnt does (m0 is reserved to
    // single instructions' use on this target, so nothing of the compiler's lives in it across this). A load into LDS may
    // read m0 one wait state after a scalar write of it at the earliest, which the compiler keeps for its own instructions only.
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(voffset), "s"(rsrc) : "memory");
}

static __device__ __forceinline__ uintx4 make_rsrc(const void *p, unsigned bytes)   // bytes < 2^31: lanes that must read zeros ask for 2^31
{
    const uint64_t a = reinterpret_cast<uint64_t>(p);
    return uintx4{(unsigned)a, (unsigned)(a >> 32) & 0xffffu, bytes, 0x00020000u};
}

template <bool AT, bool BT, bool GATED, int BM, int BN, int WM, int WN, int STAGES>
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
    int source = t0 % a.sources;                       // of the next step to load
    int krem = a.K - t0 / a.sources * 32;              // k from its first on; <= 0: nothing, zeros
    const long stepA = AT ? 32 * a.ldA : 32, stepB = BT ? 32 * a.ldB : 32;
    const long atA = AT ? (long)m0 : (long)m0 * a.ldA, atB = BT ? (long)n0 : (long)n0 * a.ldB;
    const __bf16 *const A0 = static_cast<const __bf16 *>(a.A[0]), *const B0 = static_cast<const __bf16 *>(a.B[0]);
    const __bf16 *pA = A0 + atA + t0 / a.sources * stepA, *pB = B0 + atB + t0 / a.sources * stepB;   // in the first source
    const long toA1 = static_cast<const __bf16 *>(a.A[1]) - A0, toB1 = static_cast<const __bf16 *>(a.B[1]) - B0;
    const int spanN = GATED ? BN / 2 : BN;
    const int rowsA = a.M - m0 < BM ? a.M - m0 : BM, rowsB = a.N - n0 < spanN ? a.N - n0 : spanN;

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
            if (source) {   // uniform
                qA += toA1;
                qB += toB1;
            }
            if (GATED && (wave & 2)) qB += toB1;
        } else if (part == 1) {
            rA = make_rsrc(qA, AT ? tile_end_t(a.M - m0, (unsigned)a.ldA, krem) : tile_end_straight(rowsA, (unsigned)a.ldA, krem));
            inA = AT || kchunkA < krem;   // a straight row goes on into the next one
        } else if (part == 2) {
            rB = make_rsrc(qB, BT ? tile_end_t(a.N - n0, (unsigned)a.ldB, krem) : tile_end_straight(rowsB, (unsigned)a.ldB, krem));
            inB = BT || kchunkB < krem;
        } else {
            lds = __builtin_amdgcn_readfirstlane(lds0 + stage + wave * 1024);
            if (++source == a.sources) {
                source = 0;
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

    tile_out<__bf16, AT, BT, GATED, BM, BN, WM, WN, RING>(a, acc, smem, lane, wave, wm, wn, m0, n0, cut, piece, tile - a.whole, cut_tiles);
}

}  // namespace alpha
