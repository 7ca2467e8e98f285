// Linear layer with bias, activation and residual in its epilogue, forward and backward, fp32 / bf16 / fp16:
//   z = x W^T + b,  y = act(z) + res;      delta = dy act'(z),  dx = delta W,  dW = delta^T x,  db = column sums of delta
// The three products are one form, D(i, j) = sum_k A(i, k) B(j, k), with either operand stored along k or along its rows.
// Three forms of it: one for up to 16 rows (bound by reading W), direct tiles (bound by latency), tiles through LDS (mm_engine.h: bound by the
// matrix rate the part sustains; an fp32 product is six bf16 ones).  MEASURED (MI355X, us): 1 x 4096 -> 4096 bf16 SiLU + residual 7.9 (4.3 TB/s of
// W); 512 x 512 -> 512 fp32 forward 9, backward 27; 65536 x 256 -> 256 fp32 softplus + residual forward 102, delta 46, dx 66 (0.78 PFLOP/s of
// MFMAs), dW 69 + 5 + 5; 8192 x 4096 -> 8192 bf16 dx 465 (1.18 PFLOP/s; the library's 8192^3: 1.34), dW 499, forward with GELU, residual and
// the stored pre-activation 625 (its epilogue has nothing to run beside at one workgroup a CU), delta 95.  Heads (up to 16 outputs) have a
// form of their own each way, bound by reading x: 18135 x 4308 -> 1 fp32 forward 68 (4.6 TB/s), backward 155 (6 TB/s with the caches' help).
// Roundings beside the outputs': 16-bit rows store z in their own type, and act' is taken at that z (as a module that keeps its pre-activation in the
// rows' type does: an fp32 z would double what the forward writes beside y); their products take delta rounded to the rows' type (one matrix
// product instead of the two that a second term of delta needs).  Against 64 bits that leaves dx and dW with 1.4 roundings of the type instead of one
// (relative, bf16 8192 x 4096 -> 8192: 2.4e-3 / 1.7e-3; fp16 1999 x 777 -> 1111: 3.0e-4 / 2.1e-4).  The bias gradient and the heads' form take delta
// unrounded.  fp32 rows have neither.
#include <type_traits>
#include "mm_engine.h"
#include "fneus_kernels.h"

namespace fneus {

enum { LIN_FWD = 0, LIN_DX = 1, LIN_DW = 2 };

// One product as the direct kernels see it.
struct LinProduct {
    const void *a, *b;       // the operands of D's rows and columns
    const void* az;          // backward: the pre-activations in a's layout (a := a act'(az)), or null
    long lda, ldz, ldb;
    const void *bias, *res;  // forward
    void *d, *z;             // D [rows_i][ldd]; forward: the pre-activation beside it, or null
    void* db;                // LIN_DW: sums of a over k, [rows_i], or null
    long ldres, ldd;
    long ni, nk;
    int nj, act;
    int tiles_j;
    long first_tile;
};

// 8 values of an operand for one lane, (i, k0 .. k0 + 7).  ROWS: stored along k (unaligned 16-byte loads), else element (i, k) at
// p[k ld + i] (the lanes of a half read consecutive values).  No branch around a load, whose result the compiler would wait for inside it:
// a row beyond the last is the last one again (its products end in elements nobody stores); MASKED, the last values of k: addresses are
// kept below kend and what lies beyond counts as zero.
template <class T, bool ROWS, bool MASKED>
FN_DEV void lin_load8(const T* __restrict__ p, long ld, long i, long ni, long k0, long kend, float (&v)[8]) {
    i = i < ni ? i : ni - 1;
    if constexpr (ROWS && !MASKED) {
        const T* q = p + i * ld + k0;
        constexpr int N = Chunk<T>::N;
#pragma unroll
        for (int c = 0; c < 8 / N; ++c) {
            const typename Chunk<T>::type u = *reinterpret_cast<const typename Chunk<T>::type*>(q + c * N);
#pragma unroll
            for (int k = 0; k < N; ++k) v[c * N + k] = (float)u[k];
        }
    } else {
        const T* q = ROWS ? p + i * ld : p + i;
        const long step = ROWS ? 1 : ld;
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = (float)q[(MASKED && k0 + k >= kend ? kend - 1 : k0 + k) * step];
        if constexpr (MASKED) {
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = k0 + k < kend ? v[k] : 0.0f;
        }
    }
}

// The direct kernel: a workgroup owns a 32 x 32 tile of D, its 8 waves split the contraction, operands go from memory to the matrix
// instructions without LDS, the partial tiles are added in wave order (LDS).  For products too small for the tiled kernel to fill the
// chip, where a launch's latency is what counts: one launch forward, one backward.
template <class T, int KIND>
FN_DEV void lin_direct_tile(const LinProduct& P, long tile, float (*red)[16][65], float (*red_db)[32]) {
    constexpr bool AROWS = KIND != LIN_DW, BROWS = KIND == LIN_FWD;      // (how a and b are stored)
    const long i0 = 32 * (tile / P.tiles_j);
    const int j0 = 32 * (int)(tile % P.tiles_j);
    const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const long part = ((P.nk + 7) / 8 + 15) / 16 * 16;
    const long kb = wave * part, ke = kb + part < P.nk ? kb + part : P.nk;
    const T *a = (const T*)P.a, *b = (const T*)P.b, *az = (const T*)P.az;
    f32x16 acc;
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e] = 0.0f;
    float asum = 0.0f;
    const bool scaled = KIND != LIN_FWD && az, multiply = KIND != LIN_DW || P.d;       // (no D: the bias gradient alone)
    auto round = [&](auto masked, auto unroll, long k) {
        constexpr bool M = decltype(masked)::value;
        constexpr int U = decltype(unroll)::value;
        float av[U][8], bv[U][8], zv[U][8];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long k0 = k + 16 * u + 8 * h;
            lin_load8<T, AROWS, M>(a, P.lda, i0 + r, P.ni, k0, ke, av[u]);
            if (multiply) lin_load8<T, BROWS, M>(b, P.ldb, j0 + r, P.nj, k0, ke, bv[u]);
            if (scaled) lin_load8<T, AROWS, M>(az, P.ldz, i0 + r, P.ni, k0, ke, zv[u]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (scaled) {
#pragma unroll
                for (int s = 0; s < 8; ++s) av[u][s] *= lin_dact(zv[u][s], P.act);
            }
            if constexpr (KIND == LIN_DW) {
#pragma unroll
                for (int s = 0; s < 8; ++s) asum += av[u][s];
            }
            if (multiply) {
                LinFrag<T> fa, fb;
                lin_frag(av[u], fa);
                lin_frag(bv[u], fb);
                acc = lin_mfma32(fb, fa, acc);           // accumulator rows = j, columns (lanes) = i
            }
        }
    };
    long k = kb;
    for (; k + 64 <= ke; k += 64) round(std::false_type{}, std::integral_constant<int, 4>{}, k);
    for (; k + 16 <= ke; k += 16) round(std::false_type{}, std::integral_constant<int, 1>{}, k);
    if (k < ke) round(std::true_type{}, std::integral_constant<int, 1>{}, k);
#pragma unroll
    for (int e = 0; e < 16; ++e) red[wave][e][lane] = acc[e];
    if constexpr (KIND == LIN_DW) {
        asum += xor32(asum);
        if (lane < 32) red_db[wave][lane] = asum;
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const int o = (int)threadIdx.x + 512 * q;
        const int jj = o & 31, ii = o >> 5;
        const int e = (jj & 3) + 4 * (jj >> 3), ln = ii + 32 * ((jj >> 2) & 1);
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < 8; ++w) v += red[w][e][ln];
        const long gi = i0 + ii;
        const int gj = j0 + jj;
        if (gi < P.ni && gj < P.nj) {
            if constexpr (KIND == LIN_FWD) {
                if (P.bias) v += (float)((const T*)P.bias)[gj];
                if (P.z) ((T*)P.z)[gi * P.ldd + gj] = (T)v;
                v = lin_act(v, P.act);
                if (P.res) v += (float)((const T*)P.res)[gi * P.ldres + gj];
            }
            if (KIND != LIN_DW || P.d) ((T*)P.d)[gi * P.ldd + gj] = (T)v;
        }
    }
    if constexpr (KIND == LIN_DW) {
        if (P.db && j0 == 0 && threadIdx.x < 32 && i0 + (long)threadIdx.x < P.ni) {
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < 8; ++w) s += red_db[w][threadIdx.x];
            ((T*)P.db)[i0 + threadIdx.x] = (T)s;
        }
    }
}

template <class T>
__global__ void __launch_bounds__(512) linear_direct_fwd_kernel(LinProduct p) {
    __shared__ float red[8][16][65];
    lin_direct_tile<T, LIN_FWD>(p, blockIdx.x, red, nullptr);
}

template <class T>
__global__ void __launch_bounds__(512) linear_direct_bwd_kernel(LinProduct dx, LinProduct dw) {
    __shared__ float red[8][16][65];
    __shared__ float red_db[8][32];
    if ((long)blockIdx.x < dw.first_tile) lin_direct_tile<T, LIN_DX>(dx, blockIdx.x, red, red_db);
    else lin_direct_tile<T, LIN_DW>(dw, (long)blockIdx.x - dw.first_tile, red, red_db);
}

// Up to 16 rows (tokens): reading W once is all there is.  A workgroup owns 16 outputs, its 8 waves split the contraction, a wave's
// load covers 64 consecutive bytes of each of its 16 weight rows and UNROLL of them are in flight.
// HEAD: the same with the operands' places exchanged, for up to 16 outputs: reading x once is all there is, a workgroup owns 16 rows (a = W, b = x).
template <class T, bool HEAD>
__global__ void __launch_bounds__(512) linear_row_kernel(LinProduct P) {
    __shared__ float red[8][16][17];
    const long j0 = 16 * wide_block();
    if (j0 >= P.nj) return;
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const long part = ((P.nk + 7) / 8 + 31) / 32 * 32;
    const long kb = wave * part, ke = kb + part < P.nk ? kb + part : P.nk;
    const T *a = (const T*)P.a, *b = (const T*)P.b;
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    auto round = [&](auto masked, auto unroll, long k) {
        constexpr bool M = decltype(masked)::value;
        constexpr int U = decltype(unroll)::value;
        float av[U][8], bv[U][8];
#pragma unroll
        for (int u = 0; u < U; ++u) lin_load8<T, true, M>(b, P.ldb, j0 + r, P.nj, k + 32 * u + 8 * g, ke, bv[u]);
#pragma unroll
        for (int u = 0; u < U; ++u) lin_load8<T, true, M>(a, P.lda, r, P.ni, k + 32 * u + 8 * g, ke, av[u]);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            LinFrag<T> fa, fb;
            lin_frag(av[u], fa);
            lin_frag(bv[u], fb);
            acc = lin_mfma16(fb, fa, acc);
        }
    };
    long k = kb;
    constexpr int DEEP = sizeof(T) == 2 ? 8 : 4;             // loads of W in flight a wave
    for (; k + 32 * DEEP <= ke; k += 32 * DEEP) round(std::false_type{}, std::integral_constant<int, DEEP>{}, k);
    for (; k + 32 <= ke; k += 32) round(std::false_type{}, std::integral_constant<int, 1>{}, k);
    if (k < ke) round(std::true_type{}, std::integral_constant<int, 1>{}, k);
#pragma unroll
    for (int e = 0; e < 4; ++e) red[wave][4 * g + e][r] = acc[e];        // row j = 4 g + e, column i = r
    __syncthreads();
    if (threadIdx.x < 256) {
        const int lo = threadIdx.x & 15, hi = threadIdx.x >> 4, jj = HEAD ? hi : lo, ii = HEAD ? lo : hi;
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < 8; ++w) v += red[w][jj][ii];
        if (ii < P.ni && j0 + jj < P.nj) {
            const long row = HEAD ? j0 + jj : ii;
            const int col = HEAD ? ii : (int)j0 + jj;
            if (P.bias) v += (float)((const T*)P.bias)[col];
            if (P.z) ((T*)P.z)[row * P.ldd + col] = (T)v;
            v = lin_act(v, P.act);
            if (P.res) v += (float)((const T*)P.res)[row * P.ldres + col];
            ((T*)P.d)[row * P.ldd + col] = (T)v;
        }
    }
}

// ---- the tiled form ------------------------------------------------------------------------------------------------------------
struct LinTiled {
    MmOperand a, b;
    const void *bias, *res;
    void *d, *z;
    float* partial;              // [splits][ni][nj]
    long ni, ldres, ldd;
    int nj, k_tiles, tail, act, splits, tiles_i, tiles_j, pad_;
};

enum { LIN_EPI_FWD = 0, LIN_EPI_STORE = 1, LIN_EPI_PART = 2 };

// bias, pre-activation, activation, residual of four consecutive outputs of row i
template <class T>
FN_DEV void lin_finish(const T* bias, const T* res, T* d, T* z, int act, int valid, float (&v)[4]) {
    float q[4];
    if (bias) {
        quad_load(bias, valid, q);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] += q[k];
    }
    if (z) quad_store(z, valid, v);
    if (act) {
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = lin_act(v[k], act);
    }
    if (res) {
        quad_load(res, valid, q);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] += q[k];
    }
    quad_store(d, valid, v);
}

// CLASS: the activation's (LIN_EPI_FWD)
template <class Cfg, class T, bool AKM, bool BKM, int EPI, int CLASS>
__global__ void __launch_bounds__(Cfg::THREADS, 2) linear_tiled_kernel(LinTiled P) {
    extern __shared__ __attribute__((aligned(16))) unsigned char mm_smem[];
    const long tiles = (long)P.tiles_i * P.tiles_j;
    const long wg = wide_block();
    if (wg >= tiles * P.splits) return;
    const long t = mm_spread(wg, tiles * P.splits);
    const int split = (int)(t / tiles);
    int ti, tj;
    mm_tile(t - split * tiles, P.tiles_i, P.tiles_j, ti, tj);
    const long i0 = (long)ti * Cfg::BM, j0 = (long)tj * Cfg::BN;
    const int it0 = (int)((long)P.k_tiles * split / P.splits), it1 = (int)((long)P.k_tiles * (split + 1) / P.splits);
    f32x16 acc[Cfg::MI][Cfg::NJ];
    mm_run<Cfg, T, AKM, BKM, false, true>(mm_smem, P.a, P.b, i0, P.ni, j0, P.nj, P.k_tiles, P.tail, kMmOne, it0, it1, split == P.splits - 1, 1.0f, acc);
    if constexpr (EPI == LIN_EPI_FWD) {
        constexpr int SLOTS = Cfg::WN / 8;
        float bias[4] = {0.0f, 0.0f, 0.0f, 0.0f}, res[SLOTS][4];
        {
            const long j = mm_quad_j<Cfg>(j0);
            if (P.bias && j < P.nj) quad_load((const T*)P.bias + j, (int)(P.nj - j), bias);
        }
        const float slope = P.act == 0 ? 1.0f : (P.act == 2 ? 0.2f : 0.0f);
        const bool times = P.act == 6;
        mm_epilogue<Cfg>(mm_smem, i0, j0, 1.0f, acc,
            [&](long i, long j, int s) {
                if (P.res && i < P.ni && j < P.nj) quad_load((const T*)P.res + i * P.ldres + j, (int)(P.nj - j), res[s]);
            },
            [&](long i, long j, int s, float (&v)[4], float*) {
                if (i >= P.ni || j >= P.nj) return;
                const int valid = (int)(P.nj - j);
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] += bias[k];
                if (P.z) quad_store((T*)P.z + i * P.ldd + j, valid, v);
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = lin_act_of<CLASS>(v[k], slope, times);
                if (P.res) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) v[k] += res[s][k];
                }
                quad_store((T*)P.d + i * P.ldd + j, valid, v);
            },
            [](long, long, float*) {});
    } else {
        mm_epilogue<Cfg>(mm_smem, i0, j0, 1.0f, acc, [](long, long, int) {},
            [&](long i, long j, int, float (&v)[4], float*) {
                if (i >= P.ni || j >= P.nj) return;
                const int valid = (int)(P.nj - j);
                if constexpr (EPI == LIN_EPI_STORE) quad_store<T>((T*)P.d + i * P.ldd + j, valid, v);
                else quad_store<float>(P.partial + ((long)split * P.ni + i) * P.nj + j, valid, v);
            },
            [](long, long, float*) {});
    }
}

// the partial products of a split contraction and the epilogue: GROUPS threads share the parts of four outputs, each adds its own in order,
// the groups are added in order
template <class T, bool FWD, int GROUPS>
__global__ void __launch_bounds__(256) linear_reduce_kernel(LinTiled P) {
    __shared__ float red[GROUPS > 1 ? GROUPS : 1][GROUPS > 1 ? 256 / GROUPS : 1][4];
    const int quads = (P.nj + 3) / 4;
    const int slot = threadIdx.x % (256 / GROUPS), group = threadIdx.x / (256 / GROUPS);
    const long at = (long)blockIdx.x * (256 / GROUPS) + slot;
    const bool live = at < P.ni * quads;
    const long i = live ? at / quads : 0;
    const int j = live ? 4 * (int)(at - i * quads) : 0, valid = P.nj - j;
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (live) {
        const float* p = P.partial + i * P.nj + j;
#pragma unroll 8
        for (int s = group; s < P.splits; s += GROUPS) {
            float q[4];
            quad_load<float>(p + (long)s * P.ni * P.nj, valid, q);
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] += q[k];
        }
    }
    if constexpr (GROUPS > 1) {
#pragma unroll
        for (int k = 0; k < 4; ++k) red[group][slot][k] = v[k];
        __syncthreads();
        if (group) return;
#pragma unroll
        for (int g = 1; g < GROUPS; ++g)
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] += red[g][slot][k];
    }
    if (!live) return;
    if constexpr (FWD)
        lin_finish<T>(P.bias ? (const T*)P.bias + j : nullptr, P.res ? (const T*)P.res + i * P.ldres + j : nullptr, (T*)P.d + i * P.ldd + j,
                      P.z ? (T*)P.z + i * P.ldd + j : nullptr, P.act, valid, v);
    else quad_store<T>((T*)P.d + i * P.ldd + j, valid, v);
}

// The gradients of a layer with up to 16 outputs (a head): one pass over x and dx, whose bytes are all there is.  A thread owns four columns: their
// weights and their sums of dW stay in fp32 registers, delta = dy act'(z) of kHeadRows rows lies in LDS (unrounded).  `lanes` threads share a
// row, the others of a workgroup take further rows; a workgroup leaves its part of dW and of the bias gradient, added in order by
// linear_reduce_kernel and linear_fold_kernel.  The last columns' thread takes the row's last four (what it shares with its neighbour is written
// twice, the same).
constexpr int kHeadRows = 64;
template <class T>
struct LinHead {
    const T *dy, *z, *x, *w;
    T* dx;
    float *part, *sums;                 // [parts][n_out][n_in], [parts][n_out]
    long lddy, ldx, rows, per;          // per: rows a part
    int n_in, n_out, act, lanes, strips, pad_;
};
template <class T, int N, bool DX, bool DW>
__global__ void __launch_bounds__(256) linear_head_bwd_kernel(LinHead<T> a) {
    __shared__ __attribute__((aligned(16))) float delta[kHeadRows][N];
    __shared__ f32x4 fold[256];
    typedef typename Quad<T>::type Q;
    const int strip = blockIdx.x % a.strips, part = blockIdx.x / a.strips;
    const int c = threadIdx.x & (a.lanes - 1), g = threadIdx.x / a.lanes, groups = 256 / a.lanes;
    const int at = (strip * a.lanes + c) * 4, col = at < a.n_in - 4 ? at : a.n_in - 4;
    const bool live = at < a.n_in;
    const long r0 = part * a.per, r1 = r0 + a.per < a.rows ? r0 + a.per : a.rows;
    float w[N][4], acc[N][4], db = 0.0f;
#pragma unroll
    for (int o = 0; o < N; ++o) {
        Q q = {};
        if constexpr (DX) q = *reinterpret_cast<const Q*>(a.w + (long)(o < a.n_out ? o : a.n_out - 1) * a.n_in + col);
#pragma unroll
        for (int k = 0; k < 4; ++k) w[o][k] = o < a.n_out ? (float)q[k] : 0.0f, acc[o][k] = 0.0f;
    }
    for (long rb = r0; rb < r1; rb += kHeadRows) {
        __syncthreads();
#pragma unroll
        for (int q = 0; q < kHeadRows * N / 256; ++q) {
            const int idx = (int)threadIdx.x + 256 * q, o = idx % N;
            const long row = rb + idx / N;
            const bool ok = row < r1 && o < a.n_out;
            const long ra = row < r1 ? row : r1 - 1;
            const int oa = o < a.n_out ? o : 0;
            float d = (float)a.dy[ra * a.lddy + oa];
            if (a.z) d *= lin_dact((float)a.z[ra * a.n_out + oa], a.act);
            d = ok ? d : 0.0f;
            delta[idx / N][o] = d;
            db += d;
        }
        __syncthreads();
        for (int s = g; s < kHeadRows; s += 4 * groups) {
            if (rb + s >= r1) break;
            Q x[4];
            if constexpr (DW) {
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const long row = rb + s + u * groups;
                    x[u] = *reinterpret_cast<const Q*>(a.x + (row < r1 ? row : r1 - 1) * a.ldx + col);
                }
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const long row = rb + s + u * groups;
                if (row < r1) {
                    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int o = 0; o < N; o += 4) {
                        const f32x4 d = *reinterpret_cast<const f32x4*>(&delta[s + u * groups][o]);
#pragma unroll
                        for (int p = 0; p < 4; ++p)
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                if constexpr (DX) v[k] += d[p] * w[o + p][k];
                                if constexpr (DW) acc[o + p][k] += d[p] * (float)x[u][k];
                            }
                    }
                    if constexpr (DX) {
                        Q q;
#pragma unroll
                        for (int k = 0; k < 4; ++k) q[k] = (T)v[k];
                        if (live) *reinterpret_cast<Q*>(a.dx + row * a.n_in + col) = q;
                    }
                }
            }
        }
    }
    if constexpr (DW) {
#pragma unroll
        for (int o = 0; o < N; ++o) {
            if (o < a.n_out) {
                f32x4 v = {acc[o][0], acc[o][1], acc[o][2], acc[o][3]};
                if (groups > 1) {
                    __syncthreads();
                    fold[threadIdx.x] = v;
                    __syncthreads();
                    for (int q = 1; q < groups && g == 0; ++q) v += fold[c + q * a.lanes];
                }
                if (g == 0 && live) *reinterpret_cast<f32x4_u*>(a.part + ((long)part * a.n_out + o) * a.n_in + col) = v;
            }
        }
    }
    if (a.sums && strip == 0) {
        float* red = reinterpret_cast<float*>(fold);
        __syncthreads();
        red[threadIdx.x] = db;                       // (of output threadIdx % N)
        __syncthreads();
        if ((int)threadIdx.x < a.n_out) {
            float v = 0.0f;
#pragma unroll 8
            for (int q = threadIdx.x; q < 256; q += N) v += red[q];
            a.sums[(long)part * a.n_out + threadIdx.x] = v;
        }
    }
}

// What a product needs ready, in one launch: matrices whose rows its 16-byte accesses do not fit, copied to rows that do (zeros behind), and
// delta = dy act'(z) (rounded to T for the products; rows of ldp, zeros behind) with the column sums of delta before that rounding, a
// partial row of sums for every `sum_parts`-th of the rows.
template <class T>
struct LinPad {
    const T* x;
    T* out;
    long ld, rows;
    int n, ldp, blocks, pad_;
};
template <class T>
struct LinDelta {
    const T *dy, *z;
    T* delta;
    float* sums;
    long lddy, rows;
    int n, ldp, act, strips, sum_parts, pad_;
};

template <class T>
FN_DEV void lin_pad_block(const LinPad<T>& p, int block) {
    constexpr int V = Chunk<T>::N;
    const int chunks = p.ldp / V;
    for (long at = (long)block * 256 + threadIdx.x; at < p.rows * chunks; at += (long)p.blocks * 256) {
        const long r = at / chunks;
        const int c = V * (int)(at - r * chunks);
        float v[V];
        load_chunk<T>(p.x + r * p.ld + c, p.n - c, v);
        store_chunk<T>(p.out + r * p.ldp + c, V, v);
    }
}

template <class T>
__global__ void __launch_bounds__(256) linear_prepare_kernel(LinDelta<T> d, LinPad<T> px, LinPad<T> pw) {
    constexpr int V = Chunk<T>::N;
    __shared__ float red[8][32 * V];
    const int first = d.strips * d.sum_parts;
    if ((int)blockIdx.x >= first) {
        const int at = (int)blockIdx.x - first;
        if (at < px.blocks) lin_pad_block(px, at);
        else lin_pad_block(pw, at - px.blocks);
        return;
    }
    // 32 chunks of columns, 8 rows at a time
    const int strip = blockIdx.x % d.strips, part = blockIdx.x / d.strips;
    const int c = threadIdx.x & 31, r = threadIdx.x >> 5;
    const int col = (strip * 32 + c) * V, left = d.n - col;
    const long r0 = d.rows * part / d.sum_parts, r1 = d.rows * (part + 1) / d.sum_parts;
    float s[V];
#pragma unroll
    for (int k = 0; k < V; ++k) s[k] = 0.0f;
    for (long row = r0 + r; row < r1; row += 8) {
        float v[V], q[V];
        load_chunk<T>(d.dy + row * d.lddy + col, left, v);
        if (d.act) {
            load_chunk<T>(d.z + row * d.n + col, left, q);
#pragma unroll
            for (int k = 0; k < V; ++k) v[k] *= lin_dact(q[k], d.act);
        }
#pragma unroll
        for (int k = 0; k < V; ++k) s[k] += v[k];
        if (d.delta && col < d.ldp) store_chunk<T>(d.delta + row * d.ldp + col, V, v);
    }
    if (!d.sums) return;
#pragma unroll
    for (int k = 0; k < V; ++k) red[r][c * V + k] = s[k];
    __syncthreads();
    for (int at = threadIdx.x; at < 32 * V; at += 256) {
        const int j = strip * 32 * V + at;
        float v = 0.0f;
#pragma unroll
        for (int q = 0; q < 8; ++q) v += red[q][at];
        if (j < d.n) d.sums[(long)part * d.n + j] = v;
    }
}

template <class T>
__global__ void __launch_bounds__(1024) linear_fold_kernel(const float* __restrict__ sums, int parts, int n, T* __restrict__ out) {
    __shared__ float red[128][9];
    const float s = fold_rows8(sums, parts, n, 8L * blockIdx.x, n, red);
    if (threadIdx.x < 8 && 8 * blockIdx.x + threadIdx.x < (unsigned)n) out[8 * blockIdx.x + threadIdx.x] = (T)s;
}

typedef MmCfg<64, 64, 2, 2, 4> LinSmall;          // 4 waves, 64 KiB of LDS, three stages in flight: two workgroups a CU
typedef MmCfg<64, 64, 2, 2, 4, 2> LinSmall8;      // 8 waves on each stage's k, 128 KiB: for a launch of no more than a workgroup a CU
typedef MmCfg<128, 128, 2, 2, 2> LinMid;          // 4 waves, 64 KiB: two workgroups a CU
typedef MmCfg<128, 128, 2, 2, 2, 2> LinMid8;      // 8 waves, 128 KiB: one
typedef MmCfg<256, 256, 2, 4, 2> LinBig;          // 8 waves, 128 KiB: one

// How a product runs: tile size and the parts of its contraction.  256-wide tiles where they occupy the chip; below, MEASURED (us a launch
// by the tile's width, 64 / 128): fp32 512^3 15 / 24, 4096 x 256 x 256 14 / 25, 2000 x 776 -> 1112 58 / 50, 256 x 4096 x 4096 105 / 65, 8192 x
// 512 x 512 48 / 41; bf16 1024^3 11 / 18, 2000 x 776 -> 1112 21 / 20, 2048^3 33 / 31, 65536 x 256 x 256 38 / 27: a narrow tile where the
// wide ones are few, but not where the contraction of fp32 (whose terms cost a narrow tile as much as its products) is long.
struct LinShape { int tile, splits; };            // tile: 64, 128, 256
template <class T>
static LinShape lin_shape(long ni, long nj, long nk) {
    const long t256 = ((ni + 255) / 256) * ((nj + 255) / 256), t128 = ((ni + 127) / 128) * ((nj + 127) / 128);
    const long t64 = ((ni + 63) / 64) * ((nj + 63) / 64), k_tiles = nk / (128 / (long)sizeof(T));
    LinShape s{128, 1};
    if (t256 >= 240 && ni > 64 && nj > 64) s.tile = 256;
    else if (ni <= 64 || nj <= 64) s.tile = 64;
    else if (sizeof(T) == 2 ? t128 < 144 : t128 <= 64 && nk <= 1024) s.tile = 64;
    const long t = s.tile == 64 ? t64 : (s.tile == 128 ? t128 : t256);
    if (t <= 128 && s.tile != 256) {    // split to a workgroup a CU, at least 8 stages of 64 (32) k each, 2^28 partial sums at most
        long want = 256 / t;
        const long room = (1L << 28) / (ni * nj), most = k_tiles / 8 < room ? k_tiles / 8 : room;
        if (want > most) want = most;
        if (want > 1) s.splits = (int)want;
    }
    return s;
}

// Everything a call launches and where its scratch lies.
struct LinPlan {
    bool tiled;
    bool pad_x, pad_w, delta, head;            // head: linear_head_bwd_kernel, `parts` parts of `per` rows
    int parts, lanes, strips;
    long per;
    int ldx, ldw, ldd, sum_parts;              // padded row lengths
    LinShape fwd, dx, dw;
    long off_x, off_w, off_delta, off_sums, off_part, total;
};

static long lin_up(long v, long to) { return (v + to - 1) / to * to; }

// whether the tiled kernel can take a matrix as it lies: whole 16-byte chunks, and 256 rows within the 32-bit offsets of its loads
template <class T>
static bool lin_aligned(const void* p, long ld, long n, bool k_major) {
    constexpr int V = 16 / (int)sizeof(T);
    return ((uintptr_t)p & 15) == 0 && ld % V == 0 && (!k_major || n % V == 0) && ld * (long)sizeof(T) <= 1L << 24;
}

// Which form: a direct tile is one launch for a direction and needs no scratch, the tiled kernel shares its operands.  MEASURED (us, forward /
// backward, direct against tiled): fp32 512^3 9 / 26 against 15 / 35, 2048 x 512 x 512 23 / 88 against 20 / 48, 4096 x 256 x 256 15 / 114
// against 14 / 35; bf16 512^3 6 / 19 against 8 / 20, 4096 x 256 x 256 10 / 72 against 7 / 25: up to 2^27 multiplications (forward, fp32: 2^28),
// and for the weight gradient, whose contraction the direct form does not split, up to 1024 rows.  Where the contraction is short its eight
// waves have nothing to split: at most 8192 tiles (65536 x 3 -> 256 fp32, 16384 of them, 60 against 36), and of a few rows' weight gradient at
// most 1024 (16 x 8192 -> 8192 fp32, 65536 of them, 683 against 86).
// Heads (up to 16 outputs) take linear_row_kernel<HEAD>: MEASURED (us, it against the tiled or direct form) fp32 18135 x 4308 -> 1 73 / 106, 23662 x 6183
// -> 2 141 / 459 (rows that had to be copied), 1444 x 4919 -> 12 19 / 44, 512 x 512 -> 3 5.0 / 7.3, 65536 x 512 -> 3 29 / 36; bf16 36042 x 909 -> 8 33 / 48;
// but 65536 x 256 -> 16 23 / 21, 65536 x 32 -> 4 11 / 9: not where many rows are short for its eight waves.
static bool lin_head(const FneusLinear& f) { return f.n_out <= 16 && (f.n_in > 256 || f.rows <= 8192); }

template <class T>
static bool lin_direct(const FneusLinear& f, bool backward) {
    if (!backward && (f.rows <= 16 || lin_head(f))) return true;
    const double work = (double)f.rows * f.n_in * f.n_out;
    const long ti = (f.rows + 31) / 32, tj = (f.n_in + 31) / 32, to = (f.n_out + 31) / 32;
    if (backward) return f.rows <= 1024 && work <= (double)(1L << 27) && (ti + to) * tj <= (f.rows > 16 ? 8192 : 1024);
    return work <= (double)(sizeof(T) == 4 ? 1L << 28 : 1L << 27) && ti * to <= 8192;
}

// Heads, backward: MEASURED (us, dx, dW and db, linear_head_bwd_kernel against the others) fp32 65536 x 256 -> 1 40 / 65, -> 16 43 / 66, 200000 x 96 -> 3
// 45 / 129, 23662 x 6183 -> 2 333 / 637, 2000 x 2000 -> 4 26 / 37; bf16 32 / 46, 43 / 50, 39 / 105, 201 / 336, 26 / 31; but 512 x 512 -> 3 16 / 16 (bf16 17 / 13),
// 200 x 4000 -> 6 26 / 15, 8000 x 2000 -> 16 70 / 61 (bf16 74 / 41): many rows, fewer where the outputs are few.
static bool lin_head_bwd(const FneusLinear& f) { return f.n_out <= 16 && f.n_in >= 16 && f.rows > (f.n_out <= 8 ? 1024 : 32768) && (f.dx || f.dweight); }

template <class T>
static LinPlan lin_plan(const FneusLinear& f, bool backward) {
    constexpr int V = 16 / (int)sizeof(T);
    LinPlan p;
    memset(&p, 0, sizeof p);
    long o = 0, part = 0;
    auto take = [&](long bytes) { const long at = o; o += lin_up(bytes, 256); return at; };
    if (backward && lin_head_bwd(f)) {
        // as many threads a row as it has quads (16 .. 256), 1024 workgroups, and no more parts than keep their sums a small part of x's bytes
        p.head = true;
        for (p.lanes = 16; p.lanes < 256 && p.lanes * 4 < f.n_in;) p.lanes *= 2;
        p.strips = (f.n_in + 4 * p.lanes - 1) / (4 * p.lanes);
        const long rows = f.n_out * 8 > kHeadRows && f.dweight ? 2 * kHeadRows : kHeadRows;
        long parts = (1024 + p.strips - 1) / p.strips, most = (f.rows + rows - 1) / rows;
        parts = parts < most ? parts : most;
        p.per = lin_up((f.rows + parts - 1) / parts, kHeadRows);
        p.parts = (int)((f.rows + p.per - 1) / p.per);
        if (f.dbias) p.off_sums = take((long)p.parts * f.n_out * 4);
        p.off_part = o;
        p.total = f.dweight ? o + (long)p.parts * f.n_out * f.n_in * 4 : o;
        return p;
    }
    p.tiled = !lin_direct<T>(f, backward);
    if (!p.tiled) return p;
    auto partial = [&](const LinShape& s, long ni, long nj) { if (s.splits > 1) { const long b = (long)s.splits * ni * nj * 4; part = b > part ? b : part; } };
    if (!backward) {
        p.pad_x = !lin_aligned<T>(f.x, f.ldx, f.n_in, false);
        p.pad_w = !lin_aligned<T>(f.weight, f.n_in, f.n_in, false);
        p.fwd = lin_shape<T>(f.rows, f.n_out, f.n_in);
        partial(p.fwd, f.rows, f.n_out);
    } else {
        p.pad_x = f.dweight && !lin_aligned<T>(f.x, f.ldx, f.n_in, true);
        p.pad_w = f.dx && !lin_aligned<T>(f.weight, f.n_in, f.n_in, true);
        p.delta = (f.dx || f.dweight) && (f.act != 0 || !lin_aligned<T>(f.dy, f.lddy, f.n_out, f.dweight != nullptr));
        p.dx = lin_shape<T>(f.rows, f.n_in, f.n_out);
        p.dw = lin_shape<T>(f.n_out, f.n_in, f.rows);
        if (f.dx) partial(p.dx, f.rows, f.n_in);
        if (f.dweight) partial(p.dw, f.n_out, f.n_in);
        if (p.delta) p.ldd = (int)lin_up(f.n_out, V), p.off_delta = take(f.rows * p.ldd * (long)sizeof(T));
        if (p.delta || f.dbias) {
            const long strips = (f.n_out + 32 * V - 1) / (32 * V);
            long parts = (1024 + strips - 1) / strips, most = (f.rows + 31) / 32;
            p.sum_parts = (int)(parts < most ? parts : most);
            if (f.dbias) p.off_sums = take((long)p.sum_parts * f.n_out * 4);
        }
    }
    if (p.pad_x) p.ldx = (int)lin_up(f.n_in, V), p.off_x = take(f.rows * p.ldx * (long)sizeof(T));
    if (p.pad_w) p.ldw = (int)lin_up(f.n_in, V), p.off_w = take((long)f.n_out * p.ldw * (long)sizeof(T));
    p.off_part = o;
    p.total = o + part;
    return p;
}

static MmOperand lin_operand(const void* p, long ld, int e) {
    MmOperand o;
    o.plane[0] = o.plane[1] = o.plane[2] = (const unsigned char*)p;
    o.row_bytes = ld * e;
    return o;
}

template <class Cfg, class T, bool AKM, bool BKM, int EPI, int CLASS>
static void lin_tiled_launch(const LinTiled& t, hipStream_t stream) {
    auto kernel = linear_tiled_kernel<Cfg, T, AKM, BKM, EPI, CLASS>;
    allow_big_lds(kernel);
    hipLaunchKernelGGL(kernel, wide_grid((long)t.tiles_i * t.tiles_j * t.splits), dim3(Cfg::THREADS), Cfg::LDS, stream, t);
}

template <class Cfg, class T, bool AKM, bool BKM, bool FWD>
static void lin_tiled_whole(const LinTiled& t, hipStream_t stream) {
    if constexpr (!FWD) {
        lin_tiled_launch<Cfg, T, AKM, BKM, LIN_EPI_STORE, 0>(t, stream);
    } else {
        switch (lin_class(t.act)) {
            case 0: lin_tiled_launch<Cfg, T, AKM, BKM, LIN_EPI_FWD, 0>(t, stream); break;
            case 3: lin_tiled_launch<Cfg, T, AKM, BKM, LIN_EPI_FWD, 3>(t, stream); break;
            case 4: lin_tiled_launch<Cfg, T, AKM, BKM, LIN_EPI_FWD, 4>(t, stream); break;
            default: lin_tiled_launch<Cfg, T, AKM, BKM, LIN_EPI_FWD, 5>(t, stream); break;
        }
    }
}

template <class Cfg, class T, bool AKM, bool BKM, bool FWD>
static void lin_tiled_with(LinTiled t, long nk, hipStream_t stream) {
    constexpr int kv = Cfg::template kv<T>();
    t.k_tiles = (int)(nk / kv), t.tail = (int)(nk % kv);
    if (t.splits > 1) lin_tiled_launch<Cfg, T, AKM, BKM, LIN_EPI_PART, 0>(t, stream);
    else lin_tiled_whole<Cfg, T, AKM, BKM, FWD>(t, stream);
}

template <class T, bool FWD>
static void lin_reduce(const LinTiled& t, hipStream_t stream) {
    const long quads = t.ni * ((t.nj + 3) / 4);
    if (t.splits >= 16) hipLaunchKernelGGL((linear_reduce_kernel<T, FWD, 8>), dim3((unsigned)((quads + 31) / 32)), dim3(256), 0, stream, t);
    else hipLaunchKernelGGL((linear_reduce_kernel<T, FWD, 1>), dim3((unsigned)((quads + 255) / 256)), dim3(256), 0, stream, t);
}

template <class T, bool AKM, bool BKM, bool FWD>
static void lin_tiled_product(LinTiled t, const LinShape& s, long nk, float* partial, hipStream_t stream) {
    const int b = s.tile;
    t.splits = s.splits, t.partial = partial;
    t.tiles_i = (int)((t.ni + b - 1) / b), t.tiles_j = (t.nj + b - 1) / b;
    const bool few = (long)t.tiles_i * t.tiles_j * t.splits <= 256;
    if (s.tile == 256) lin_tiled_with<LinBig, T, AKM, BKM, FWD>(t, nk, stream);
    else if (s.tile == 128 && !few) lin_tiled_with<LinMid, T, AKM, BKM, FWD>(t, nk, stream);
    else if (s.tile == 128) lin_tiled_with<LinMid8, T, AKM, BKM, FWD>(t, nk, stream);
    else if (!few) lin_tiled_with<LinSmall, T, AKM, BKM, FWD>(t, nk, stream);
    else lin_tiled_with<LinSmall8, T, AKM, BKM, FWD>(t, nk, stream);
    if (s.splits > 1) lin_reduce<T, FWD>(t, stream);
}

template <class T>
static LinPad<T> lin_pad(const void* x, long ld, long rows, int n, unsigned char* out, int ldp) {
    LinPad<T> p{};
    const long blocks = (rows * (ldp / Chunk<T>::N) + 255) / 256;
    p.x = (const T*)x, p.out = (T*)out, p.ld = ld, p.rows = rows, p.n = n, p.ldp = ldp, p.blocks = (int)(blocks < 2048 ? blocks : 2048);
    return p;
}

template <class T>
static void lin_prepare(const FneusLinear& f, const LinPlan& p, const LinDelta<T>& d, hipStream_t stream) {
    unsigned char* S = (unsigned char*)f.scratch;
    LinPad<T> px{}, pw{};
    if (p.pad_x) px = lin_pad<T>(f.x, f.ldx, f.rows, f.n_in, S + p.off_x, p.ldx);
    if (p.pad_w) pw = lin_pad<T>(f.weight, f.n_in, f.n_out, f.n_in, S + p.off_w, p.ldw);
    const unsigned blocks = (unsigned)(d.strips * d.sum_parts + px.blocks + pw.blocks);
    if (blocks) hipLaunchKernelGGL((linear_prepare_kernel<T>), dim3(blocks), dim3(256), 0, stream, d, px, pw);
}

template <class T>
static void lin_tiled_fwd(const FneusLinear& f, const LinPlan& p, hipStream_t stream) {
    unsigned char* S = (unsigned char*)f.scratch;
    lin_prepare<T>(f, p, LinDelta<T>{}, stream);
    LinTiled t{};
    t.a = p.pad_x ? lin_operand(S + p.off_x, p.ldx, sizeof(T)) : lin_operand(f.x, f.ldx, sizeof(T));
    t.b = p.pad_w ? lin_operand(S + p.off_w, p.ldw, sizeof(T)) : lin_operand(f.weight, f.n_in, sizeof(T));
    t.bias = f.bias, t.res = f.residual, t.ldres = f.ld_residual, t.d = f.y, t.z = f.z, t.ldd = f.n_out, t.ni = f.rows, t.nj = f.n_out, t.act = f.act;
    lin_tiled_product<T, false, false, true>(t, p.fwd, f.n_in, (float*)(S + p.off_part), stream);
}

template <class T>
static void lin_tiled_bwd(const FneusLinear& f, const LinPlan& p, hipStream_t stream) {
    unsigned char* S = (unsigned char*)f.scratch;
    float* part = (float*)(S + p.off_part);
    LinDelta<T> d{};
    if (p.delta || f.dbias) {
        d.dy = (const T*)f.dy, d.z = (const T*)f.z, d.delta = p.delta ? (T*)(S + p.off_delta) : nullptr, d.sums = f.dbias ? (float*)(S + p.off_sums) : nullptr;
        d.lddy = f.lddy, d.rows = f.rows, d.n = f.n_out, d.ldp = p.ldd, d.act = f.act, d.sum_parts = p.sum_parts;
        d.strips = (f.n_out + 32 * Chunk<T>::N - 1) / (32 * Chunk<T>::N);
    }
    lin_prepare<T>(f, p, d, stream);
    if (f.dbias)
        hipLaunchKernelGGL((linear_fold_kernel<T>), dim3((unsigned)((f.n_out + 7) / 8)), dim3(1024), 0, stream, d.sums, p.sum_parts, f.n_out, (T*)f.dbias);
    const MmOperand delta = p.delta ? lin_operand(S + p.off_delta, p.ldd, sizeof(T)) : lin_operand(f.dy, f.lddy, sizeof(T));
    if (f.dx) {
        LinTiled t{};
        t.a = delta, t.b = p.pad_w ? lin_operand(S + p.off_w, p.ldw, sizeof(T)) : lin_operand(f.weight, f.n_in, sizeof(T));
        t.d = f.dx, t.ldd = f.n_in, t.ni = f.rows, t.nj = f.n_in;
        lin_tiled_product<T, false, true, false>(t, p.dx, f.n_out, part, stream);
    }
    if (f.dweight) {
        LinTiled t{};
        t.a = delta, t.b = p.pad_x ? lin_operand(S + p.off_x, p.ldx, sizeof(T)) : lin_operand(f.x, f.ldx, sizeof(T));
        t.d = f.dweight, t.ldd = f.n_in, t.ni = f.n_out, t.nj = f.n_in;
        lin_tiled_product<T, true, true, false>(t, p.dw, f.rows, part, stream);
    }
}

template <class T, int N>
static void lin_head_launch(const LinHead<T>& h, int parts, bool dw, hipStream_t stream) {
    const dim3 grid((unsigned)(h.strips * parts));
    if (h.dx && dw) hipLaunchKernelGGL((linear_head_bwd_kernel<T, N, true, true>), grid, dim3(256), 0, stream, h);
    else if (h.dx) hipLaunchKernelGGL((linear_head_bwd_kernel<T, N, true, false>), grid, dim3(256), 0, stream, h);
    else hipLaunchKernelGGL((linear_head_bwd_kernel<T, N, false, true>), grid, dim3(256), 0, stream, h);
}

template <class T>
static void lin_head_run(const FneusLinear& f, const LinPlan& p, hipStream_t stream) {
    unsigned char* S = (unsigned char*)f.scratch;
    LinHead<T> h{};
    h.dy = (const T*)f.dy, h.z = f.act ? (const T*)f.z : nullptr, h.x = (const T*)f.x, h.w = (const T*)f.weight, h.dx = (T*)f.dx;
    h.part = (float*)(S + p.off_part), h.sums = f.dbias ? (float*)(S + p.off_sums) : nullptr;
    h.lddy = f.lddy, h.ldx = f.ldx, h.rows = f.rows, h.per = p.per;
    h.n_in = f.n_in, h.n_out = f.n_out, h.act = f.act, h.lanes = p.lanes, h.strips = p.strips;
    if (f.n_out <= 4) lin_head_launch<T, 4>(h, p.parts, f.dweight, stream);
    else if (f.n_out <= 8) lin_head_launch<T, 8>(h, p.parts, f.dweight, stream);
    else lin_head_launch<T, 16>(h, p.parts, f.dweight, stream);
    if (f.dweight) {
        LinTiled t{};
        t.d = f.dweight, t.ldd = f.n_in, t.ni = f.n_out, t.nj = f.n_in, t.splits = p.parts, t.partial = h.part;
        lin_reduce<T, false>(t, stream);
    }
    if (f.dbias) hipLaunchKernelGGL((linear_fold_kernel<T>), dim3((unsigned)((f.n_out + 7) / 8)), dim3(1024), 0, stream, h.sums, p.parts, f.n_out, (T*)f.dbias);
}

static int lin_refuse(const char* msg) {
    set_last_error(msg);
    return -2;
}

static int lin_check(const FneusLinear* f, bool backward) {
    if (!f) return lin_refuse("fneus_linear: a job must be given");
    if (f->rows < 0 || f->n_in <= 0 || f->n_out <= 0 || f->act < 0 || f->act >= kLinActs || f->dtype < 0 || f->dtype > 2)
        return lin_refuse("fneus_linear: rows >= 0, n_in and n_out > 0, act 0..6, dtype 0..2");
    if (f->rows > 0x7fffffffL || f->n_in > (1 << 22) || f->n_out > (1 << 22)) return lin_refuse("fneus_linear: at most 2^31 - 1 rows, 2^22 columns");
    if (!backward) {
        if (f->rows > 0 && (!f->x || !f->weight || !f->y)) return lin_refuse("fneus_linear_fwd: x, weight and y must be given");
        if (f->ldx < f->n_in || (f->residual && f->ld_residual < f->n_out)) return lin_refuse("fneus_linear_fwd: a row stride smaller than the row");
    } else {
        if (f->rows == 0) return lin_refuse("fneus_linear_bwd: no rows (the sums are empty: clear the gradients)");
        if (!f->dy || f->lddy < f->n_out || (f->act != 0 && !f->z)) return lin_refuse("fneus_linear_bwd: dy (and z for an activation) must be given");
        if ((f->dx && !f->weight) || (f->dweight && (!f->x || f->ldx < f->n_in))) return lin_refuse("fneus_linear_bwd: weight for dx, x for dweight");
        if (!f->dx && !f->dweight && !f->dbias) return lin_refuse("fneus_linear_bwd: no gradient asked for");
    }
    return 0;
}

static bool lin_scratch_ok(const FneusLinear& f, const LinPlan& p) {
    return p.total == 0 || (f.scratch && f.scratch_bytes >= p.total && ((uintptr_t)f.scratch & 15) == 0);
}

template <class T>
static int lin_fwd(const FneusLinear& f, hipStream_t stream) {
    const LinPlan plan = lin_plan<T>(f, false);
    if (plan.tiled) {
        if (!lin_scratch_ok(f, plan)) return lin_refuse("fneus_linear_fwd: scratch of fneus_linear_scratch_bytes bytes, 16-byte aligned, must be given");
        lin_tiled_fwd<T>(f, plan, stream);
        return launch_status();
    }
    LinProduct p{};
    p.a = f.x, p.lda = f.ldx, p.b = f.weight, p.ldb = f.n_in, p.bias = f.bias, p.res = f.residual, p.ldres = f.ld_residual;
    p.d = f.y, p.z = f.z, p.ldd = f.n_out, p.ni = f.rows, p.nj = f.n_out, p.nk = f.n_in, p.act = f.act;
    if (f.rows <= 16) {
        hipLaunchKernelGGL((linear_row_kernel<T, false>), dim3((unsigned)((f.n_out + 15) / 16)), dim3(512), 0, stream, p);
        return launch_status();
    }
    if (lin_head(f)) {
        p.a = f.weight, p.lda = f.n_in, p.b = f.x, p.ldb = f.ldx, p.ni = f.n_out, p.nj = (int)f.rows;
        hipLaunchKernelGGL((linear_row_kernel<T, true>), wide_grid((f.rows + 15) / 16), dim3(512), 0, stream, p);
        return launch_status();
    }
    p.tiles_j = (p.nj + 31) / 32;
    const long tiles = (p.ni + 31) / 32 * p.tiles_j;
    if (tiles > 0x7fffffffL) return lin_refuse("fneus_linear_fwd: more than 2^31 tiles: split the rows");
    hipLaunchKernelGGL((linear_direct_fwd_kernel<T>), dim3((unsigned)tiles), dim3(512), 0, stream, p);
    return launch_status();
}

template <class T>
static int lin_bwd(const FneusLinear& f, hipStream_t stream) {
    const LinPlan plan = lin_plan<T>(f, true);
    if (plan.tiled) {
        if (!lin_scratch_ok(f, plan)) return lin_refuse("fneus_linear_bwd: scratch of fneus_linear_scratch_bytes bytes, 16-byte aligned, must be given");
        lin_tiled_bwd<T>(f, plan, stream);
        return launch_status();
    }
    if (plan.head) {
        if (!lin_scratch_ok(f, plan)) return lin_refuse("fneus_linear_bwd: scratch of fneus_linear_scratch_bytes bytes, 16-byte aligned, must be given");
        lin_head_run<T>(f, plan, stream);
        return launch_status();
    }
    LinProduct dx{}, dw{};
    const void* z = f.act ? f.z : nullptr;
    dx.a = f.dy, dx.lda = f.lddy, dx.az = z, dx.ldz = f.n_out, dx.b = f.weight, dx.ldb = f.n_in, dx.d = f.dx, dx.ldd = f.n_in;
    dx.ni = f.rows, dx.nj = f.n_in, dx.nk = f.n_out, dx.act = f.act, dx.tiles_j = (dx.nj + 31) / 32;
    dw.a = f.dy, dw.lda = f.lddy, dw.az = z, dw.ldz = f.n_out, dw.b = f.x, dw.ldb = f.ldx, dw.d = f.dweight, dw.ldd = f.n_in;
    dw.db = f.dbias, dw.ni = f.n_out, dw.nj = f.n_in, dw.nk = f.rows, dw.act = f.act, dw.tiles_j = f.dweight ? (dw.nj + 31) / 32 : 1;
    dw.first_tile = f.dx ? (dx.ni + 31) / 32 * dx.tiles_j : 0;
    const long tiles = dw.first_tile + (f.dweight || f.dbias ? (dw.ni + 31) / 32 * dw.tiles_j : 0);
    if (tiles > 0x7fffffffL) return lin_refuse("fneus_linear_bwd: more than 2^31 tiles: split the rows");
    hipLaunchKernelGGL((linear_direct_bwd_kernel<T>), dim3((unsigned)tiles), dim3(512), 0, stream, dx, dw);
    return launch_status();
}

}  // namespace fneus

using namespace fneus;

extern "C" long fneus_linear_scratch_bytes(const FneusLinear* f, int backward) {
    if (!f || f->rows <= 0 || f->n_in <= 0 || f->n_out <= 0) return 0;
    if (f->dtype == DT_F32) return lin_plan<float>(*f, backward != 0).total;
    if (f->dtype == DT_BF16) return lin_plan<__bf16>(*f, backward != 0).total;
    return lin_plan<_Float16>(*f, backward != 0).total;
}

extern "C" int fneus_linear_fwd(const FneusLinear* f, fneus_stream_t stream) {
    fneus::clear_status();
    if (int rc = lin_check(f, false)) return rc;
    if (f->rows == 0) return 0;
    if (f->dtype == DT_F32) return lin_fwd<float>(*f, (hipStream_t)stream);
    if (f->dtype == DT_BF16) return lin_fwd<__bf16>(*f, (hipStream_t)stream);
    return lin_fwd<_Float16>(*f, (hipStream_t)stream);
}

extern "C" int fneus_linear_bwd(const FneusLinear* f, fneus_stream_t stream) {
    fneus::clear_status();
    if (int rc = lin_check(f, true)) return rc;
    if (f->dtype == DT_F32) return lin_bwd<float>(*f, (hipStream_t)stream);
    if (f->dtype == DT_BF16) return lin_bwd<__bf16>(*f, (hipStream_t)stream);
    return lin_bwd<_Float16>(*f, (hipStream_t)stream);
}
