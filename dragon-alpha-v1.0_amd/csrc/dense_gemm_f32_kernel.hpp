// The dense product's tile kernel for fp32: C[m, n] = sum_k A(m, k) B(n, k) on the bf16 matrix pipe, sixteen times the rate of
// the fp32 one. x = h + m + l exactly, three bf16 of 8 significant bits each (rounded to nearest, signs of their own; |x| < 2^-110
// to within half of bf16's last subnormal, 2^-134, which the matrix pipe takes as they are); of the
// nine products of parts the six above 2^-24 of the whole are summed, small ones first, in fp32:
//     x y = h l' + m m' + h m' + l h' + m h' + h h'   (left out: m l', l m', l l', together below 2^-23 |x y|).
// 2.5 PF / 6 = 417 TF bound, 157 TF through v_mfma_f32_16x16x4_f32. Measured: 4096 x 1024 x 4096 with GELU and both outputs 185 us,
// 185 TF; the matrix pipe is busy 54 % of the cycles at 1.84 GHz, the rest is the splitting, which it waits for.
//
// A workgroup takes BM x BN of C in steps of 32 k. An element is split once per workgroup: loaded to registers (128-bit buffer
// loads, a step ahead), split, and written to LDS as three bf16 planes of the layout that dense_gemm_kernel.hpp describes, in
// two buffers. Operands are read in place, whatever their stride, alignment and storage. A step has three runs of MFMAs - by
// l', m' and h' of B, 16 + 32 + 48 per wavefront of 64 x 64, half of them of 32 x 64 -, and a run's fragments are read during the run
// before:
//     run 1: h l'              reads m', m        splits and writes the next step's elements, asks for those of the step after
//     run 2: m m', h m'        reads h', l          (the same, on to the barrier)
//     barrier: every read of this step's planes and every write of the next step's is done
//     run 3: l h', m h', h h'  reads the next step's l', h
// so the one barrier of a step (256 x 128: 192 MFMAs per SIMD) stands between MFMAs whose operands are in registers.
// An infinity or NaN makes NaN (h - h), and so does a value that rounds up beyond bf16's range; products of parts may overflow
// where the whole does not. What is not finite at the end is computed once more in plain fp32 (plain_rows).
#pragma once
#include "dense_tile.hpp"

namespace alpha {

// Four values as bf16, and what those leave of them. The halves are widened again as the integers they are: from the vector
// type the compiler rounds every value a second time to do it (34 instructions for three parts of four values instead of 22,
// and the matrix pipe waits for each of them).
static __device__ __forceinline__ uint2 round_off(floatx4 &x, bool rest)
{
    typedef float floatx2 __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const uint32_t lo = __builtin_bit_cast(uint32_t, __builtin_convertvector(floatx2{x[0], x[1]}, bf16x2));
    const uint32_t hi = __builtin_bit_cast(uint32_t, __builtin_convertvector(floatx2{x[2], x[3]}, bf16x2));
    if (rest) {
        x[0] -= __uint_as_float(lo << 16);
        x[1] -= __uint_as_float(lo & 0xffff0000u);
        x[2] -= __uint_as_float(hi << 16);
        x[3] -= __uint_as_float(hi & 0xffff0000u);
    }
    return uint2{lo, hi};
}

template <bool AT, bool BT, bool GATED, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM * WN * 64, 1) void dense_tile_f32_kernel(const DenseTileArgs a)
{
    constexpr int NT = WM * WN * 64, TM = BM / WM, TN = BN / WN, MF = TM / 16, NF = TN / 16;
    constexpr int LA = BM * 8 / NT, LB = BN * 8 / NT, LOADS = LA + LB;       // 16-byte loads of a thread per step
    constexpr unsigned APLANE = BM * 64, BPLANE = BN * 64, BUFFER = 3 * (APLANE + BPLANE);
    static_assert((MF == 4 || MF == 2) && NF == 4 && NT % 256 == 0, "a wavefront owns 64 or 32 x 64");
    constexpr int R = MF * NF;     // MFMAs of a product of two parts
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

    // ---- where a thread's loads come from (offset in the operand, from the tile's first element of the step) and go to ----
    unsigned off[LOADS], to[LOADS];
    int kfirst[LOADS];     // straight: the first of the four k
    for_each<LOADS>([&](auto index) __attribute__((always_inline)) {
        constexpr int j = index;
        constexpr bool T = j < LA ? AT : BT;
        constexpr int ROWS = j < LA ? BM : BN;
        const int at = (j < LA ? j : j - LA) * NT + tid;
        const long ld = j < LA ? a.ldA : a.ldB;
        const unsigned plane0 = j < LA ? 0u : 3 * APLANE;
        if constexpr (T) {
            const int k = at / (ROWS / 4), c = at % (ROWS / 4);
            off[j] = (unsigned)(k * ld * 4) + c * 16;
            to[j] = plane0 + k * (ROWS * 2) + ((c >> 1) ^ t_permutation(k)) * 16 + (c & 1) * 8;
            kfirst[j] = 0;
        } else {
            const int r = at >> 3, c = at & 7;
            const int row = GATED && j >= LA ? (r >> 6) * 32 + (r & 31) : r;   // gated: 32 tile rows of one filter, 32 of the other
            off[j] = (unsigned)(row * ld * 4) + c * 16;
            to[j] = plane0 + r * 64 + ((c >> 1) ^ s_permutation(r >> 2)) * 16 + (c & 1) * 8;
            kfirst[j] = c * 4;
        }
    });

    const int t0 = piece * a.per;
    int left = a.steps - t0;
    if (cut && left > a.per) left = a.per;
    int source = t0 % a.sources;                       // of the next step to load
    int krem = a.K - t0 / a.sources * 32;              // k from its first on; <= 0: nothing, zeros
    const long stepA = AT ? 32 * a.ldA : 32, stepB = BT ? 32 * a.ldB : 32;
    const float *const A0 = static_cast<const float *>(a.A[0]), *const B0 = static_cast<const float *>(a.B[0]);
    const float *pA = A0 + (AT ? (long)m0 : (long)m0 * a.ldA) + t0 / a.sources * stepA;
    const float *pB = B0 + (BT ? (long)n0 : (long)n0 * a.ldB) + t0 / a.sources * stepB;
    const long toA1 = static_cast<const float *>(a.A[1]) - A0, toB1 = static_cast<const float *>(a.B[1]) - B0;
    constexpr int SPAN = GATED ? BN / 2 : BN;
    const int rowsA = AT ? a.M - m0 : (a.M - m0 < BM ? a.M - m0 : BM), rowsB = BT ? a.N - n0 : (a.N - n0 < SPAN ? a.N - n0 : SPAN);

    // the next step's descriptors: they end with the operand's last element, so rows beyond it read zeros
    __amdgpu_buffer_rsrc_t rA, rB, rB1;
    int kleft = 0;
    auto begin = [&]() {
        const float *qA = source ? pA + toA1 : pA, *qB = source ? pB + toB1 : pB;
        kleft = krem < 32 ? krem : 32;
        const unsigned bytesA = kleft <= 0 ? 0u : (unsigned)((AT ? (kleft - 1) * a.ldA + rowsA : (rowsA - 1) * a.ldA + kleft) * 4);
        const unsigned bytesB = kleft <= 0 ? 0u : (unsigned)((BT ? (kleft - 1) * a.ldB + rowsB : (rowsB - 1) * a.ldB + kleft) * 4);
        rA = __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(qA), 0, bytesA, 0x00020000);
        rB = __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(qB), 0, bytesB, 0x00020000);
        if constexpr (GATED) rB1 = __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(qB + toB1), 0, bytesB, 0x00020000);
        if (++source == a.sources) {
            source = 0;
            krem -= 32;
            pA += stepA;
            pB += stepB;
        }
    };
    floatx4 raw[LOADS];
    auto load = [&](auto index) __attribute__((always_inline)) {
        constexpr int j = index;
        // gated: which filter a load's eight rows are of is one for the wavefront
        if constexpr (j < LA) {
            raw[j] = __builtin_bit_cast(floatx4, __builtin_amdgcn_raw_buffer_load_b128(rA, off[j], 0, 0));
        } else if (GATED && (((j - LA) * (NT / 8) + wave * 8) & 32)) {
            raw[j] = __builtin_bit_cast(floatx4, __builtin_amdgcn_raw_buffer_load_b128(rB1, off[j], 0, 0));
        } else {
            raw[j] = __builtin_bit_cast(floatx4, __builtin_amdgcn_raw_buffer_load_b128(rB, off[j], 0, 0));
        }
    };
    // a straight row goes on into the next one: what lies beyond K is cleared (kept: the k that were there when `raw` was asked for)
    auto clear_tail = [&](auto index, int kept) __attribute__((always_inline)) {
        constexpr int j = index;
        if constexpr (!(j < LA ? AT : BT)) {
            if (kept < 32) {   // uniform
#pragma unroll
                for (int e = 0; e < 4; e++) raw[j][e] = kfirst[j] + e < kept ? raw[j][e] : 0.f;
            }
        }
    };
    // split and write one load, in three turns
    auto split = [&](auto index, auto turn, unsigned buffer) __attribute__((always_inline)) {
        constexpr int j = index;
        typedef unsigned uintx2 __attribute__((ext_vector_type(2)));
        const uint2 part = round_off(raw[j], turn < 2);
        *(__attribute__((address_space(3))) uintx2 *)((lds_char *)smem + buffer + to[j] + turn * (j < LA ? APLANE : BPLANE)) = uintx2{part.x, part.y};
    };

    // ---- where the fragments are read ----
    unsigned rdA[AT ? MF : 1], rdB[BT ? NF : 1];
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
        for (int x = 0; x < NF; x++) rdB[x] = 3 * APLANE + tk * (BN * 2) + (((wn * NF + x) * 2 + t16) ^ t_permutation(tk)) * 16 + (l16 & 1) * 8;
    } else {
        rdB[0] = 3 * APLANE + (wn * TN + l16) * 64 + chunk;
    }
    auto read_t = [&](unsigned at, int row_bytes) {   // k .. k+3 and k+4 .. k+7 of the lane's row
        const shortx4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) shortx4 *)((lds_char *)smem + at));
        const shortx4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) shortx4 *)((lds_char *)smem + at + 4 * row_bytes));
        return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    auto read_a = [&](unsigned buffer, int part, int i) -> bf16x8 {
        if constexpr (AT) return read_t(buffer + part * APLANE + rdA[i], BM * 2);
        else return *(const __attribute__((address_space(3))) bf16x8 *)((lds_char *)smem + buffer + part * APLANE + rdA[0] + i * 1024);
    };
    auto read_b = [&](unsigned buffer, int part, int i) -> bf16x8 {
        if constexpr (BT) return read_t(buffer + part * BPLANE + rdB[i], BN * 2);
        else return *(const __attribute__((address_space(3))) bf16x8 *)((lds_char *)smem + buffer + part * BPLANE + rdB[0] + i * 1024);
    };

    floatx4 acc[MF][NF];
#pragma unroll
    for (int i = 0; i < MF; i++)
#pragma unroll
        for (int j = 0; j < NF; j++) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};

    unsigned buffer = 0;
    int kept = 0;          // kleft of the step that `raw` holds
    auto step = [&](const bf16x8 (&ah)[MF], const bf16x8 (&bl)[4], bf16x8 (&next_ah)[MF], bf16x8 (&next_bl)[4]) {
        const unsigned next = BUFFER - buffer;
        bf16x8 am[MF], bm[4], al[MF], bh[4];
        begin();
        // runs 1 and 2: 3 R MFMAs, 3 LOADS turns of splitting, 8 + 2 MF reads
        for_each<3 * R>([&](auto index) __attribute__((always_inline)) {
            constexpr int x = index;
            for_each<3 * LOADS>([&](auto turn) __attribute__((always_inline)) {
                constexpr int w = turn;
                if constexpr (w * R / LOADS == x) {
                    if constexpr (w % 3 == 0) clear_tail(std::integral_constant<int, w / 3>{}, kept);
                    split(std::integral_constant<int, w / 3>{}, std::integral_constant<int, w % 3>{}, next);
                    if constexpr (w % 3 == 2) load(std::integral_constant<int, w / 3>{});
                }
            });
            if constexpr (x < R) {
                constexpr int every = MF / 2, r = x / every;
                if constexpr (x % every == 0 && r < 4) bm[r] = read_b(buffer, 1, r);
                if constexpr (x % every == 0 && r >= 4 && r < 4 + MF) am[r - 4] = read_a(buffer, 1, r - 4);
            } else {
                constexpr int r = (x - R) / 2;
                if constexpr (x % 2 == 0 && r < 4) bh[r] = read_b(buffer, 0, r);
                if constexpr (x % 2 == 0 && r >= 4 && r < 4 + MF) al[r - 4] = read_a(buffer, 2, r - 4);
            }
            constexpr int i = x / 4 % MF, j = x % 4;
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x < R ? bl[j] : bm[j], x < R ? ah[i] : x < 2 * R ? am[i] : ah[i], acc[i][j], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        });
        kept = kleft;
        lds_barrier();
        __builtin_amdgcn_sched_barrier(0);
        for_each<3 * R>([&](auto index) __attribute__((always_inline)) {
            constexpr int x = index, r = x / 4;
            if constexpr (x % 4 == 0 && r < 4) next_bl[r] = read_b(next, 2, r);
            if constexpr (x % 4 == 0 && r >= 4 && r < 4 + MF) next_ah[r - 4] = read_a(next, 0, r - 4);
            constexpr int i = r % MF, j = x % 4;
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bh[j], x < R ? al[i] : x < 2 * R ? am[i] : ah[i], acc[i][j], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        });
        buffer = next;
    };

    // the first step's planes, the second step's elements on their way
    begin();
    kept = kleft;
    for_each<LOADS>(load);
    begin();
    for_each<LOADS>([&](auto j) __attribute__((always_inline)) {
        clear_tail(j, kept);
        for_each<3>([&](auto turn) __attribute__((always_inline)) { split(j, turn, 0u); });
        load(j);
    });
    kept = kleft;
    lds_barrier();
    bf16x8 ah0[MF], bl0[4], ah1[MF], bl1[4];
#pragma unroll
    for (int i = 0; i < 4; i++) bl0[i] = read_b(0, 2, i);
#pragma unroll
    for (int i = 0; i < MF; i++) ah0[i] = read_a(0, 0, i);
    for (int t = 0; t < left; t += 2) {   // (an odd number of steps ends with one of zeros)
        step(ah0, bl0, ah1, bl1);
        step(ah1, bl1, ah0, bl0);
    }
    lds_barrier();   // every read of the tiles is done
    const int k_first = t0 / a.sources * 32, k_end = k_first + left / a.sources * 32;
    tile_out<float, AT, BT, GATED, BM, BN, WM, WN, 2 * (int)BUFFER>(a, acc, smem, lane, wave, wm, wn, m0, n0, cut, piece, tile - a.whole, cut_tiles, k_first,
                                                                    k_end < a.K ? k_end : a.K);
}

}  // namespace alpha
