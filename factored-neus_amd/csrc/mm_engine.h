// Tiled matrix product D(i, j) = sum_k A(i, k) B(j, k) over 16-bit PLANES (linear_kernels.hip, muon_kernels.hip).
//
// A plane is a matrix of bf16 or fp16 values stored along k: row r at base + r * row_bytes, k padded with zeros to a multiple of 64 (so
// a row is a whole number of 128-byte lines and no load needs a mask along k).  An operand of more bits is several planes (its terms),
// and the contraction then runs over SEGMENTS, one per pair of terms: the pipeline does not drain between them.
//
// A workgroup owns a BM x BN tile of D; 64 values of k of both operands are one stage of an LDS ring, filled by LDS-DMA (no staging
// registers), read back as the 16-byte fragments of v_mfma_f32_32x32x16.  Rows of 128 bytes would put the 32 lanes of a fragment read on
// the same banks: the 16-byte chunk c of row r lies at slot c ^ (r & 7), applied to the DMA's global addresses (its LDS side is linear),
// and every group of 8 lanes reads 8 different slots.
// Rows beyond an operand's last are loaded as its last row again: their products end in elements of D nobody stores.
#pragma once
#include "fneus_types.h"

namespace fneus {

typedef __attribute__((address_space(3))) unsigned char mm_lds_t;

struct MmOperand {
    const unsigned char* plane[3];
    unsigned row_bytes;
};

template <int BM_, int BN_, int WGM, int WGN, int STAGES_>
struct MmCfg {
    static constexpr int BM = BM_, BN = BN_, WAVES = WGM * WGN, THREADS = 64 * WAVES, STAGES = STAGES_;
    static constexpr int WM = BM / WGM, WN = BN / WGN, MI = WM / 32, NJ = WN / 32, WAVES_N = WGN;
    static constexpr int STAGE_BYTES = (BM + BN) * 128, DPW = (BM + BN) / 8 / WAVES, LDS = STAGES * STAGE_BYTES;
    static_assert((BM / 8) % DPW == 0 && (BN / 8) % DPW == 0, "a wave fills rows of one operand");
};

template <int N>
FN_DEV void mm_wait_barrier() {      // all but the newest N of this wave's loads have landed, its LDS reads are done; then everyone's
    static_assert(N == 0 || N == 4 || N == 8 || N == 12 || N == 16 || N == 24, "add the count");
    if constexpr (N == 0) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    else if constexpr (N == 4) asm volatile("s_waitcnt vmcnt(4) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    else if constexpr (N == 8) asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    else if constexpr (N == 12) asm volatile("s_waitcnt vmcnt(12) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    else if constexpr (N == 16) asm volatile("s_waitcnt vmcnt(16) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    else asm volatile("s_waitcnt vmcnt(24) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// a wave-uniform address into scalar registers
FN_DEV const unsigned char* mm_uniform(const unsigned char* p) {
    const unsigned long v = (unsigned long)p;
    const unsigned lo = __builtin_amdgcn_readfirstlane((int)(unsigned)v), hi = __builtin_amdgcn_readfirstlane((int)(unsigned)(v >> 32));
    return (const unsigned char*)(((unsigned long)hi << 32) | lo);
}

template <class T> struct MmVec;
template <> struct MmVec<__bf16> {
    typedef bf16x8 type;
    static FN_DEV f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <> struct MmVec<_Float16> {
    typedef fn_f16x8 type;
    static FN_DEV f32x16 mfma(fn_f16x8 a, fn_f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};

// Segment tables, 4 bits a segment: the terms of A (bits 0, 1) and B (bits 2, 3).
constexpr unsigned kMmOne = 0x0u;                 // 1 segment
constexpr unsigned kMmThree = 0x140u;             // 3: (0, 0), (0, 1), (1, 0): two-term operands
constexpr unsigned kMmSix = 0x041528u;            // 6: (0, 2), (2, 0), (1, 1), (1, 0), (0, 1), (0, 0): three-term operands, smallest first

// acc[mi][nj], element e of a lane: row i = mi * 32 + (lane & 31), column j = nj * 32 + 8 (e >> 2) + 4 (lane >> 5) + (e & 3) of the
// wave's part of the tile (mm_i0, mm_j0): four consecutive columns in four consecutive registers.
template <class Cfg>
FN_DEV int mm_wave() { return __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)); }
template <class Cfg>
FN_DEV int mm_row() { return (mm_wave<Cfg>() / Cfg::WAVES_N) * Cfg::WM + (int)(threadIdx.x & 31); }
template <class Cfg>
FN_DEV int mm_col() { return (mm_wave<Cfg>() % Cfg::WAVES_N) * Cfg::WN + 4 * (int)((threadIdx.x >> 5) & 1); }

// it: steps of 64 along the concatenated segments, [it0, it1) of n_seg * k_tiles.  After segment 0 the sums are multiplied by `carry`
// (RESCALE: the later segments' terms are held at a larger scale).
template <class Cfg, class T, bool RESCALE>
FN_DEV void mm_run(unsigned char* smem, const MmOperand& A, const MmOperand& B, long i0, long ni, long j0, long nj, int k_tiles,
                   unsigned segs, int it0, int it1, float carry, f32x16 (&acc)[Cfg::MI][Cfg::NJ]) {
    typedef typename MmVec<T>::type V8;
    const int lane = threadIdx.x & 63, wave = mm_wave<Cfg>();
#pragma unroll
    for (int m = 0; m < Cfg::MI; ++m)
#pragma unroll
        for (int n = 0; n < Cfg::NJ; ++n)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[m][n][e] = 0.0f;
    // this wave's DMA: 8 rows an instruction, lane -> row lane >> 3, slot lane & 7 <- chunk slot ^ (row & 7)
    const int q0 = wave * Cfg::DPW;
    const bool is_b = q0 >= Cfg::BM / 8;
    const unsigned row_bytes = is_b ? B.row_bytes : A.row_bytes;
    const unsigned char *pl0 = is_b ? B.plane[0] : A.plane[0], *pl1 = is_b ? B.plane[1] : A.plane[1], *pl2 = is_b ? B.plane[2] : A.plane[2];
    const long first = is_b ? j0 : i0, count = is_b ? nj : ni;
    const int valid = (int)(count - first < 256 ? count - first : 256);        // >= 1
    const int row0 = (q0 - (is_b ? Cfg::BM / 8 : 0)) * 8 + (lane >> 3);
    unsigned off[Cfg::DPW];
#pragma unroll
    for (int d = 0; d < Cfg::DPW; ++d) {
        const int row = row0 + 8 * d;
        off[d] = (unsigned)(row < valid ? row : valid - 1) * row_bytes + ((unsigned)((lane & 7) ^ (lane >> 3)) << 4);
    }
    int is_seg = it0 / k_tiles, is_kt = it0 - is_seg * k_tiles;
    auto base_of = [&](int seg) {
        const unsigned c = (segs >> (4 * seg + (is_b ? 2 : 0))) & 3;
        return mm_uniform((c == 0 ? pl0 : (c == 1 ? pl1 : pl2)) + first * (long)row_bytes);
    };
    const unsigned char* base = base_of(is_seg);
    const unsigned lds_base = (unsigned)(uintptr_t)(mm_lds_t*)(smem + q0 * 1024);
    int is_stage = 0;
    auto issue = [&]() {
        const unsigned char* src = base + (long)is_kt * 128;
        const unsigned dst = lds_base + is_stage * Cfg::STAGE_BYTES;
#pragma unroll
        for (int d = 0; d < Cfg::DPW; ++d) {
            // (inline asm: the compiler counts a builtin LDS-DMA as a pending LDS write and would drain the ring in front of every LDS read;
            //  the waits are counted in mm_wait_barrier)
            unsigned keep;
            asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0"
                         : "=&s"(keep)
                         : "v"(off[d]), "s"(src), "s"(dst + d * 1024)
                         : "memory");
        }
        is_stage = is_stage + 1 == Cfg::STAGES ? 0 : is_stage + 1;
        if (++is_kt == k_tiles) {
            is_kt = 0;
            ++is_seg;
            base = base_of(is_seg < 6 ? is_seg : 0);
        }
    };
    constexpr int P = Cfg::STAGES - 1;
    for (int s = 0; s < P; ++s)
        if (it0 + s < it1) issue();
    const unsigned char* ra = smem + mm_row<Cfg>() * 128;
    const unsigned char* rb = smem + Cfg::BM * 128 + ((wave % Cfg::WAVES_N) * Cfg::WN + (lane & 31)) * 128;
    const int h = lane >> 5;
    int stage = 0, left0 = RESCALE ? k_tiles - it0 : 0;
#pragma unroll 1
    for (int it = it0; it < it1; ++it) {
        if (it1 - 1 - it >= P - 1) mm_wait_barrier<(P - 1) * Cfg::DPW>();
        else mm_wait_barrier<0>();
        if (it + P < it1) issue();
        const unsigned char *pa = ra + stage * Cfg::STAGE_BYTES, *pb = rb + stage * Cfg::STAGE_BYTES;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
            const unsigned x = (unsigned)((2 * ks + h) ^ (lane & 7)) << 4;
            V8 fa[Cfg::MI], fb[Cfg::NJ];
#pragma unroll
            for (int m = 0; m < Cfg::MI; ++m) fa[m] = *reinterpret_cast<const V8*>(pa + m * 4096 + x);
#pragma unroll
            for (int n = 0; n < Cfg::NJ; ++n) fb[n] = *reinterpret_cast<const V8*>(pb + n * 4096 + x);
#pragma unroll
            for (int m = 0; m < Cfg::MI; ++m)
#pragma unroll
                for (int n = 0; n < Cfg::NJ; ++n) acc[m][n] = MmVec<T>::mfma(fb[n], fa[m], acc[m][n]);
        }
        stage = stage + 1 == Cfg::STAGES ? 0 : stage + 1;
        if constexpr (RESCALE) {
            if (--left0 == 0) {
#pragma unroll
                for (int m = 0; m < Cfg::MI; ++m)
#pragma unroll
                    for (int n = 0; n < Cfg::NJ; ++n)
#pragma unroll
                        for (int e = 0; e < 16; ++e) acc[m][n][e] *= carry;
            }
        }
    }
}

// tile index -> (row, column) of tiles: workgroups of one XCD (launch index mod 8) take one contiguous stretch of the tiles, and a
// stretch runs down 8 rows of tiles before it moves to the next column: the operand rows of a stretch stay in that XCD's L2
FN_DEV void mm_tile(long wg, long tiles, int tiles_i, int tiles_j, int& ti, int& tj) {
    const long q = tiles >> 3, r = tiles & 7, xcd = wg & 7;
    const long t = xcd * q + (xcd < r ? xcd : r) + (wg >> 3);
    const long band = 8L * tiles_j;
    const int b = (int)(t / band), in = (int)(t - b * band);
    const int rows = tiles_i - 8 * b < 8 ? tiles_i - 8 * b : 8;
    tj = in / rows;
    ti = 8 * b + (in - tj * rows);
}

}  // namespace fneus
