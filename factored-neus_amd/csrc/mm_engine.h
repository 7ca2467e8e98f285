// Tiled matrix product D(i, j) = sum_k A(i, k) B(j, k) (linear_kernels.hip, muon_kernels.hip).
//
// Operands are bf16, fp16 or fp32 matrices in memory, stored along k ("rows": element (i, k) at i * row_bytes + k) or along i ("k-major":
// (i, k) at k * row_bytes + i), 16-byte aligned.  An operand of more terms than one is several planes (muon_kernels.hip), and the
// contraction then runs over SEGMENTS, one per pair of terms: the pipeline does not drain between them.  An fp32 operand is split into three
// bf16 terms behind LDS (linear_act.h).
//
// A workgroup owns a BM x BN tile of D; one stage of an LDS ring holds 128 bytes of k of every row of both operands (64 values of 16 bits,
// 32 of 32), filled by LDS-DMA (no staging registers).
//   rows:    a row is 128 bytes; its 16-byte chunk c lies at slot c ^ (row & 7), applied to the DMA's global addresses (its LDS side is
//            linear): the 8 lanes that read 16 bytes in one cycle hit 8 different slots.
//   k-major, 16 bits: a line is one k, BM values; chunk c of line k at slot c ^ ((k & 7) << 1); ds_read_b64_tr_b16 hands every lane four
//            consecutive k of its row (16 lanes read 4 lines x 32 bytes, which the swizzle puts on different banks).
//   k-major, 32 bits: the same lines, 4-byte reads, 32 consecutive values a half wave.
// Rows beyond an operand's last are loaded as its last row (k-major: its first chunk) again: their products end in elements of D nobody
// stores.  The last values of k, where they do not fill a stage, are brought by ordinary loads with zeros behind them.
#pragma once
#include <type_traits>
#include "linear_act.h"

namespace fneus {

typedef __attribute__((address_space(3))) unsigned char mm_lds_t;
typedef __attribute__((address_space(3))) bf16x4 mm_lds_bf16x4_t;

struct MmOperand {
    const unsigned char* plane[3];
    long row_bytes;
};

// GROUPS > 1: that many groups of waves share the k of every stage and their sums are added behind the last (a tile that is alone on its CU
// is done that much sooner)
template <int BM_, int BN_, int WGM, int WGN, int STAGES_, int GROUPS_ = 1>
struct MmCfg {
    static constexpr int BM = BM_, BN = BN_, GROUPS = GROUPS_, GROUP_WAVES = WGM * WGN, WAVES = GROUPS * GROUP_WAVES, THREADS = 64 * WAVES;
    static constexpr int STAGES = STAGES_, ROW = 128 * GROUPS;             // bytes of k of a row in a stage
    template <class T> static constexpr int kv() { return ROW / (int)sizeof(T); }        // values of k in a stage
    static constexpr int WM = BM / WGM, WN = BN / WGN, MI = WM / 32, NJ = WN / 32, WAVES_N = WGN;
    static constexpr int STAGE_BYTES = (BM + BN) * ROW, DPW = STAGE_BYTES / 1024 / WAVES, LDS = STAGES * STAGE_BYTES;
    static_assert((BM * ROW / 1024) % DPW == 0 && (BN * ROW / 1024) % DPW == 0, "a wave fills rows of one operand");
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

// Segment tables, 4 bits a segment: the terms of A (bits 0, 1) and B (bits 2, 3).
constexpr unsigned kMmOne = 0x0u;                 // 1 segment
constexpr unsigned kMmThree = 0x140u;             // 3: (0, 0), (0, 1), (1, 0): two-term operands

// acc[mi][nj], element e of a lane: row i = mi * 32 + (lane & 31), column j = nj * 32 + 8 (e >> 2) + 4 (lane >> 5) + (e & 3) of the
// wave's part of the tile: four consecutive columns in four consecutive registers.
FN_DEV int mm_wave() { return __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)); }
template <class Cfg>
FN_DEV int mm_wave_i() { return (mm_wave() % Cfg::GROUP_WAVES / Cfg::WAVES_N) * Cfg::WM; }
template <class Cfg>
FN_DEV int mm_wave_j() { return (mm_wave() % Cfg::WAVES_N) * Cfg::WN; }

// the places `load` and `finish` of mm_epilogue are called for, slot s of block 0
template <class Cfg>
FN_DEV long mm_quad_i(long i0, int s) { return i0 + mm_wave_i<Cfg>() + (s * 64 + (int)(threadIdx.x & 63)) / (Cfg::WN / 4); }
template <class Cfg>
FN_DEV long mm_quad_j(long j0) { return j0 + mm_wave_j<Cfg>() + 4 * ((int)(threadIdx.x & 63) % (Cfg::WN / 4)); }

// One operand's side of a stage: which bytes its DMA fetches, where a fragment lies.
template <class T, bool KM, int B, int ROW>
struct MmSide {
    static constexpr int E = sizeof(T), KV = ROW / E;            // values of k in a stage
    static constexpr int LINE = KM ? B * E : ROW, CHUNKS = LINE / 16, LINES = KM ? KV : B;      // LINES * LINE == B * ROW
    static FN_DEV int slot(int line, int c) {
        if constexpr (KM) return E == 2 ? c ^ (((line & 7) << 1) & (CHUNKS - 1)) : c;
        else return c ^ (line & 7);
    }
    // byte offset (from the tile's origin, at the stage's first k) of what DMA instruction q brings to this lane's 16 bytes of LDS
    static FN_DEV unsigned dma_offset(int q, int lane, int valid_rows, long row_bytes) {
        const int at = q * 64 + lane, line = at / CHUNKS, c = slot(line, at % CHUNKS);
        if constexpr (KM) return (unsigned)line * (unsigned)row_bytes + (unsigned)(c * (16 / E) < valid_rows ? c : 0) * 16u;
        else return (unsigned)(line < valid_rows ? line : valid_rows - 1) * (unsigned)row_bytes + (unsigned)c * 16u;
    }
    // a stage whose k ends after `left` values: ordinary loads, zeros behind
    static FN_DEV void fill_tail(unsigned char* lds, const unsigned char* src, int valid_rows, long row_bytes, int left, int thread, int threads) {
        for (int at = thread; at < B * ROW / 16; at += threads) {
            const int line = at / CHUNKS, c = at % CHUNKS;
            T v[16 / E];
#pragma unroll
            for (int e = 0; e < 16 / E; ++e) {
                const int i = KM ? c * (16 / E) + e : line, k = KM ? line : c * (16 / E) + e;
                v[e] = i < valid_rows && k < left ? reinterpret_cast<const T*>(src + (KM ? k : i) * row_bytes)[KM ? i : k] : (T)0.0f;
            }
            __builtin_memcpy(lds + line * LINE + slot(line, c) * 16, v, 16);
        }
    }
};

// Fragments of one wave's rows w0 .. of an operand; base: LDS address of the operand's part of a stage
template <class T, bool KM, int B, int ROW, int COUNT>
struct MmReader {
    typedef MmSide<T, KM, B, ROW> Side;
    unsigned at[(KM && sizeof(T) == 2) ? 2 * COUNT : COUNT];
    unsigned x7;
    FN_DEV void init(int w0, int lane) {
        const int r = lane & 31, h = lane >> 5;
        x7 = (unsigned)(lane & 7);
        if constexpr (!KM) {
#pragma unroll
            for (int m = 0; m < COUNT; ++m) at[m] = (unsigned)(w0 + 32 * m + r) * (unsigned)ROW;
        } else if constexpr (sizeof(T) == 2) {
            const int fh = (lane >> 4) & 1, q = (lane & 15) >> 2, p = lane & 3;
#pragma unroll
            for (int m = 0; m < COUNT; ++m)
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const int k = 8 * h + 4 * t + q, c = (w0 + 32 * m) / 8 + 2 * fh + (p >> 1);
                    at[2 * m + t] = (unsigned)(k * Side::LINE + Side::slot(k, c) * 16 + (p & 1) * 8);
                }
        } else {
#pragma unroll
            for (int m = 0; m < COUNT; ++m) at[m] = (unsigned)(8 * h * Side::LINE + (w0 + 32 * m + r) * 4);
        }
    }
    // k = 16 ks + 8 (lane >> 5) .. + 7
    FN_DEV void read(const unsigned char* base, int m, int ks, int h, LinFrag<T>& f) const {
        if constexpr (!KM && sizeof(T) == 2) {
            f.t = *reinterpret_cast<const decltype(f.t)*>(base + at[m] + (((unsigned)(2 * ks + h) ^ x7) << 4));
        } else if constexpr (!KM) {
            float v[8];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const f32x4 q = *reinterpret_cast<const f32x4*>(base + at[m] + (((unsigned)(4 * ks + 2 * h + u) ^ x7) << 4));
#pragma unroll
                for (int e = 0; e < 4; ++e) v[4 * u + e] = q[e];
            }
            lin_frag(v, f);
        } else if constexpr (sizeof(T) == 2) {
            bf16x8 v;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const bf16x4 q = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((mm_lds_bf16x4_t*)(base + at[2 * m + t] + ks * 16 * Side::LINE));
#pragma unroll
                for (int e = 0; e < 4; ++e) v[4 * t + e] = q[e];
            }
            f.t = __builtin_bit_cast(decltype(f.t), v);
        } else {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = *reinterpret_cast<const float*>(base + at[m] + (16 * ks + e) * Side::LINE);
            lin_frag(v, f);
        }
    }
};

// steps [it0, it1) of the concatenated segments, `k_tiles` full stages each; tail: values of k behind the last full stage (one segment
// only), taken when TAIL and `with_tail`.  Segment 0's sums are multiplied by `carry` (RESCALE: the later segments' terms are held at a
// larger scale).  ni - i0 and nj - j0 are positive.
template <class Cfg, class T, bool AKM, bool BKM, bool RESCALE, bool TAIL>
FN_DEV void mm_run(unsigned char* smem, const MmOperand& A, const MmOperand& B, long i0, long ni, long j0, long nj, int k_tiles, int tail,
                   unsigned segs, int it0, int it1, bool with_tail, float carry, f32x16 (&acc)[Cfg::MI][Cfg::NJ]) {
    typedef MmSide<T, AKM, Cfg::BM, Cfg::ROW> SideA;
    typedef MmSide<T, BKM, Cfg::BN, Cfg::ROW> SideB;
    constexpr int QA = Cfg::BM * Cfg::ROW / 1024;        // DMA instructions of A's part of a stage
    const int lane = threadIdx.x & 63, wave = mm_wave(), h = lane >> 5;
#pragma unroll
    for (int m = 0; m < Cfg::MI; ++m)
#pragma unroll
        for (int n = 0; n < Cfg::NJ; ++n)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[m][n][e] = 0.0f;
    const int va = (int)(ni - i0 < Cfg::BM ? ni - i0 : Cfg::BM), vb = (int)(nj - j0 < Cfg::BN ? nj - j0 : Cfg::BN);
    // this wave's DMA
    const int q0 = wave * Cfg::DPW;
    const bool is_b = q0 >= QA;
    unsigned off[Cfg::DPW];
#pragma unroll
    for (int d = 0; d < Cfg::DPW; ++d)
        off[d] = is_b ? SideB::dma_offset(q0 + d - QA, lane, vb, B.row_bytes) : SideA::dma_offset(q0 + d, lane, va, A.row_bytes);
    const long origin = is_b ? (BKM ? j0 * (long)sizeof(T) : j0 * B.row_bytes) : (AKM ? i0 * (long)sizeof(T) : i0 * A.row_bytes);
    const long step = is_b ? (BKM ? SideB::KV * B.row_bytes : Cfg::ROW) : (AKM ? SideA::KV * A.row_bytes : Cfg::ROW);
    const unsigned char *pl0 = is_b ? B.plane[0] : A.plane[0], *pl1 = is_b ? B.plane[1] : A.plane[1];
    int is_seg = it0 / (k_tiles > 0 ? k_tiles : 1), is_kt = it0 - is_seg * k_tiles;
    auto base_of = [&](int seg) {
        const unsigned c = (segs >> (4 * seg + (is_b ? 2 : 0))) & 3;
        return mm_uniform((c ? pl1 : pl0) + origin);
    };
    const unsigned char* base = base_of(is_seg);
    const unsigned lds_base = (unsigned)(uintptr_t)(mm_lds_t*)(smem + q0 * 1024);
    int is_stage = 0;
    auto issue = [&]() {
        const unsigned char* src = mm_uniform(base + (long)is_kt * step);
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
            base = base_of(is_seg < 7 ? is_seg : 0);
        }
    };
    constexpr int P = Cfg::STAGES - 1;
    for (int s = 0; s < P; ++s)
        if (it0 + s < it1) issue();
    MmReader<T, AKM, Cfg::BM, Cfg::ROW, Cfg::MI> ra;
    MmReader<T, BKM, Cfg::BN, Cfg::ROW, Cfg::NJ> rb;
    ra.init(mm_wave_i<Cfg>(), lane);
    rb.init(mm_wave_j<Cfg>(), lane);
    constexpr int KS = SideA::KV / 16 / Cfg::GROUPS;         // of this group
    const int ks0 = Cfg::GROUPS > 1 ? mm_wave() / Cfg::GROUP_WAVES * KS : 0;
    auto fetch = [&](const unsigned char* pa, int ks, LinFrag<T> (&fa)[Cfg::MI], LinFrag<T> (&fb)[Cfg::NJ]) {
        const unsigned char* pb = pa + Cfg::BM * Cfg::ROW;
#pragma unroll
        for (int m = 0; m < Cfg::MI; ++m) ra.read(pa, m, ks0 + ks, h, fa[m]);
#pragma unroll
        for (int n = 0; n < Cfg::NJ; ++n) rb.read(pb, n, ks0 + ks, h, fb[n]);
    };
    auto multiply = [&](const LinFrag<T> (&fa)[Cfg::MI], const LinFrag<T> (&fb)[Cfg::NJ]) {
#pragma unroll
        for (int m = 0; m < Cfg::MI; ++m)
#pragma unroll
            for (int n = 0; n < Cfg::NJ; ++n) acc[m][n] = lin_mfma32(fb[n], fa[m], acc[m][n]);
    };
    auto compute = [&](const unsigned char* pa) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            LinFrag<T> fa[Cfg::MI], fb[Cfg::NJ];
            fetch(pa, ks, fa, fb);
            multiply(fa, fb);
        }
    };
    int left0 = RESCALE ? k_tiles - it0 : 0;              // stages up to the end of segment 0 (<= 0: it lies behind)
    auto rescale = [&]() {
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
    };
    int stage = 0;
    auto wait = [&](int it) {               // stage `it` has landed, for everyone
        if (it1 - 1 - it >= P - 1) mm_wait_barrier<(P - 1) * Cfg::DPW>();
        else mm_wait_barrier<0>();
    };
    if constexpr (sizeof(T) == 2 && Cfg::MI * Cfg::NJ == 1) {
        // One accumulator a wave: its products are few and the reads' latency is what a stage takes, so a whole stage's fragments are on
        // their way under the products of the one before.
        LinFrag<T> fa[2][KS][Cfg::MI], fb[2][KS][Cfg::NJ];
        auto fetch_stage = [&](int set, const unsigned char* pa) {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) fetch(pa, ks, fa[set][ks], fb[set][ks]);
        };
        auto step = [&](int it, auto set_) {
            constexpr int set = decltype(set_)::value;
            stage = stage + 1 == Cfg::STAGES ? 0 : stage + 1;
            if (it + 1 < it1) {
                wait(it + 1);
                fetch_stage(set ^ 1, smem + stage * Cfg::STAGE_BYTES);
                if (it + 1 + P < it1) issue();
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) multiply(fa[set][ks], fb[set][ks]);
            __builtin_amdgcn_sched_barrier(0);
            rescale();
        };
        if (it0 < it1) {
            wait(it0);
            if (it0 + P < it1) issue();
            fetch_stage(0, smem);
#pragma unroll 1
            for (int it = it0; it < it1; it += 2) {
                step(it, std::integral_constant<int, 0>{});
                if (it + 1 < it1) step(it + 1, std::integral_constant<int, 1>{});
            }
        }
    } else if constexpr (sizeof(T) == 2) {
        // The fragments of the next 16 k are on their way from LDS while this one's are multiplied, across the stages too: the barrier that
        // frees a stage's buffer comes when its last fragments are in registers, in front of their products.
        if (it0 < it1) {
            LinFrag<T> fa[2][Cfg::MI], fb[2][Cfg::NJ];
            wait(it0);
            if (it0 + P < it1) issue();
            fetch(smem, 0, fa[0], fb[0]);
#pragma unroll 1
            for (int it = it0; it < it1; ++it) {
                const unsigned char* pa = smem + stage * Cfg::STAGE_BYTES;
                stage = stage + 1 == Cfg::STAGES ? 0 : stage + 1;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    if (ks + 1 < KS) {
                        fetch(pa, ks + 1, fa[(ks + 1) & 1], fb[(ks + 1) & 1]);
                    } else if (it + 1 < it1) {
                        wait(it + 1);
                        if (it + 1 + P < it1) issue();
                        fetch(smem + stage * Cfg::STAGE_BYTES, 0, fa[0], fb[0]);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                    multiply(fa[ks & 1], fb[ks & 1]);
                    __builtin_amdgcn_sched_barrier(0);
                }
                rescale();
            }
        }
        static_assert(KS % 2 == 0, "the two sets alternate");
    } else {
#pragma unroll 1
        for (int it = it0; it < it1; ++it) {
            wait(it);
            if (it + P < it1) issue();
            compute(smem + stage * Cfg::STAGE_BYTES);
            stage = stage + 1 == Cfg::STAGES ? 0 : stage + 1;
            rescale();
        }
    }
    if constexpr (RESCALE) {
        if (it1 < k_tiles) {                 // a part of segment 0 alone
#pragma unroll
            for (int m = 0; m < Cfg::MI; ++m)
#pragma unroll
                for (int n = 0; n < Cfg::NJ; ++n)
#pragma unroll
                    for (int e = 0; e < 16; ++e) acc[m][n][e] *= carry;
        }
    }
    if constexpr (TAIL) {
        if (with_tail && tail > 0) {
            mm_wait_barrier<0>();                        // (the ring is empty; everyone has read its last stage)
            const unsigned char* sa = A.plane[0] + (AKM ? i0 * (long)sizeof(T) + (long)k_tiles * SideA::KV * A.row_bytes : i0 * A.row_bytes + k_tiles * (long)Cfg::ROW);
            const unsigned char* sb = B.plane[0] + (BKM ? j0 * (long)sizeof(T) + (long)k_tiles * SideB::KV * B.row_bytes : j0 * B.row_bytes + k_tiles * (long)Cfg::ROW);
            SideA::fill_tail(smem, sa, va, A.row_bytes, tail, threadIdx.x, Cfg::THREADS);
            SideB::fill_tail(smem + Cfg::BM * Cfg::ROW, sb, vb, B.row_bytes, tail, threadIdx.x, Cfg::THREADS);
            mm_wait_barrier<0>();
            compute(smem);
        }
    }
    if constexpr (Cfg::GROUPS > 1) {          // the groups' sums, added in their order by the first
        constexpr int PART = Cfg::MI * Cfg::NJ * 16 * 64;
        static_assert((Cfg::GROUPS - 1) * Cfg::GROUP_WAVES * PART * 4 <= Cfg::LDS, "the sums fit the ring");
        float* sums = reinterpret_cast<float*>(smem) + (wave % Cfg::GROUP_WAVES) * PART + lane;
        const int group = wave / Cfg::GROUP_WAVES;
        __syncthreads();
#pragma unroll
        for (int m = 0; m < Cfg::MI; ++m)
#pragma unroll
            for (int n = 0; n < Cfg::NJ; ++n)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (group) sums[(group - 1) * Cfg::GROUP_WAVES * PART + ((m * Cfg::NJ + n) * 16 + e) * 64] = acc[m][n][e];
        __syncthreads();
        if (group) return;
#pragma unroll
        for (int g = 1; g < Cfg::GROUPS; ++g)
#pragma unroll
            for (int m = 0; m < Cfg::MI; ++m)
#pragma unroll
                for (int n = 0; n < Cfg::NJ; ++n)
#pragma unroll
                    for (int e = 0; e < 16; ++e) acc[m][n][e] += sums[(g - 1) * Cfg::GROUP_WAVES * PART + ((m * Cfg::NJ + n) * 16 + e) * 64];
    }
}

// The epilogue: the accumulators hold a column of 32 rows in a register, memory wants rows, so a wave's 32 rows at a time go through its
// part of LDS.  `load(i, j, slot)` fetches what the four outputs (i, j .. j + 3) need from memory -- all of a block's loads are in flight before
// the first is used -- and `finish(i, j, slot, v, cell)` ends them; slot numbers the quads of a block, j is the same in all of a lane's.
// `turn(ib, jb, rows)` runs once a block behind that.
// EARLY: the caller has made the loads in front of the product (one block a wave).  The first group's waves alone go in (mm_wave() <
// GROUP_WAVES), the others only meet the barrier.
template <class Cfg, bool EARLY = false, class Load, class Finish, class Turn>
FN_DEV void mm_epilogue(unsigned char* smem, long i0, long j0, float scale, f32x16 (&acc)[Cfg::MI][Cfg::NJ], Load load, Finish finish, Turn turn) {
    constexpr int STRIDE = Cfg::WN + 4, QUADS = Cfg::WN / 4, SLOTS = 32 * QUADS / 64;
    static_assert(Cfg::GROUP_WAVES * 32 * STRIDE * 4 <= Cfg::LDS, "the epilogue's rows fit the ring");
    static_assert(!EARLY || Cfg::MI == 1, "the early loads are the one block's");
    float* rows = reinterpret_cast<float*>(smem) + mm_wave() * 32 * STRIDE;
    const int lane = threadIdx.x & 63, c = 4 * (lane % QUADS);
    const long jb = j0 + mm_wave_j<Cfg>();
    __syncthreads();                                  // (everyone has read the last stage)
    if (Cfg::GROUPS > 1 && mm_wave() >= Cfg::GROUP_WAVES) return;
#pragma unroll
    for (int m = 0; m < Cfg::MI; ++m) {
        const long ib = i0 + mm_wave_i<Cfg>() + 32 * m;
#pragma unroll
        for (int s = 0; s < SLOTS; ++s)
            if constexpr (!EARLY) load(ib + (s * 64 + lane) / QUADS, jb + c, s);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int n = 0; n < Cfg::NJ; ++n)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                f32x4 q;
#pragma unroll
                for (int k = 0; k < 4; ++k) q[k] = acc[m][n][4 * g + k] * scale;
                *reinterpret_cast<f32x4*>(rows + (lane & 31) * STRIDE + 32 * n + 8 * g + 4 * (lane >> 5)) = q;
            }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) {
            const int r = (s * 64 + lane) / QUADS;
            float* cell = rows + r * STRIDE + c;
            const f32x4 q = *reinterpret_cast<const f32x4*>(cell);
            float v[4] = {q[0], q[1], q[2], q[3]};
            finish(ib + r, jb + c, s, v, cell);
        }
        turn(ib, jb, rows);
    }
}

// Launch index -> work item: the workgroups of one XCD (launch index mod 8) take one contiguous stretch of the items, so that what
// neighbours share stays in that XCD's L2.
FN_DEV long mm_spread(long wg, long total) {
    const long q = total >> 3, r = total & 7, xcd = wg & 7;
    return xcd * q + (xcd < r ? xcd : r) + (wg >> 3);
}
// tile index -> (row, column) of tiles: down 8 rows of tiles, then the next column
FN_DEV void mm_tile(long t, int tiles_i, int tiles_j, int& ti, int& tj) {
    const long band = 8L * tiles_j;
    const int b = (int)(t / band), in = (int)(t - b * band);
    const int rows = tiles_i - 8 * b < 8 ? tiles_i - 8 * b : 8;
    tj = in / rows;
    ti = 8 * b + (in - tj * rows);
}

}  // namespace fneus
