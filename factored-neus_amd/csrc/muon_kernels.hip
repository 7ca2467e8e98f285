// The Muon update of weight matrices: momentum, orthogonalisation by Newton-Schulz products, step -- every matrix of a model in the same
// 2 + 3 * steps launches, or three (matrices whose shorter side is at most 64; both where a model has both).  For each matrix u, as X [m][n] with m <= n (the transpose where rows > cols):
//   X = u / max(|u|_F, eps);   steps times:  A = X X^T,  B = b A + c A A,  X <- a X + B X
// All three products run on the tiled engine (mm_engine.h): X X^T and A A on operands stored along k, B X with X k-major.
//
// Numbers: fp16 planes with fp32 sums.  Every entry of X, A and B is bounded (the polynomial keeps the singular values below about 1.2),
// entries as small as 1 / n matter, and fp16 loses digits below 2^-14, so a plane holds its matrix times a
// power of two that puts the bound just below fp16's largest value (2^14 for the usual coefficients).  prec 2: one plane, 11 bits -- the
// error that 16-bit gradients bring along, an eighth of what bf16 operands would add.  prec 3: a second plane holds what the first one's
// rounding left, times another 2^11, so that it is as normal as the first; products hi hi + hi lo + lo hi (22 bits: fp32's accuracy at
// half the matrix work of three bf16 terms).
//
// What bounds it (MI355X, us): one fp32 4096^2 matrix 4600, of which matrix products 3950 at 1.0 - 1.1 PFLOP/s of fp16 MFMAs (a bare stream
// of them: 1.6), the joins of the shared-out ones 550, the momentum and norm 56 (5 x 64 MiB: 6 TB/s); four bf16 4096 x 1024 544 (X X^T 41, A A 18, B X 48 a step); eight fp32
// 256^2 142 = 17 launches of 8 .. 10: 1.3 until the job is read, 2.7 until the first stage has arrived from the other XCDs' writes, 0.4 a stage.
#include <math.h>
#include "mm_engine.h"
#include "fneus_kernels.h"

namespace fneus {

constexpr int kMuonMaxJobs = 32;             // per launch (kernel-argument space); more take further rounds of launches
constexpr int kMuonChunks = 256;             // partial sums of a matrix's norm
constexpr float kLoScale = 2048.0f;          // the second plane's extra scale

struct MuonJob {
    void *grad, *momentum, *param, *out;
    int rows, cols;
    float adjust;
    int pad_;
    long off;                                // its scratch
};

struct MuonJobs {
    MuonJob j[kMuonMaxJobs];
    unsigned char* scratch;
    long n;
};

struct MuonNum {
    float a, b, c;                           // the polynomial
    int ex, ea, eb;                          // planes hold X 2^ex, A 2^ea, B 2^eb
    float eps, mu, omu, wd;
    int nesterov, zero_grad;
    const float* lr;
};

// Arguments of the launches behind the first.  Arguments lie in host memory: their first lines arrive with the launch, each later line costs
// a microsecond.  So the table of jobs travels once: the first launch leaves it at the start of the scratch.  `first`: the launch's first
// workgroup of each job (beyond the last job: none).
struct MuonArgs {
    MuonNum P;
    int cur, total;                          // total: workgroups
    unsigned char* scratch;
    int first[kMuonMaxJobs];
    // a symmetric product whose contractions are shared out evenly: `stages` a tile, parts of tiles at `parts`
    int stages, shares, narrow, pad_;        // narrow: X X^T alone, in 64-wide tiles
    float* parts;
};
constexpr long kMuonTable = kMuonMaxJobs * sizeof(MuonJob);

// where a matrix's buffers lie in its scratch: norm partials, X twice (a step reads one and writes the other), A, B.  Rows of X and
// columns of all are padded with zeros to multiples of 128: whole stages of the engine's ring
struct MuonLay {
    int m, n, mp;
    bool trans;
    unsigned ldx, lda;                       // bytes of a plane's row: X, and A and B
    long px, pa;                             // bytes of a plane
    long x[2], a, b, total;
};
__host__ __device__ inline MuonLay muon_lay(int rows, int cols, int planes) {
    MuonLay L;
    L.trans = rows > cols;
    L.m = L.trans ? cols : rows;
    L.n = L.trans ? rows : cols;
    L.mp = (L.m + 127) / 128 * 128;
    L.ldx = (unsigned)((L.n + 127) / 128) * 256u;
    L.lda = (unsigned)L.mp * 2u;
    L.px = (long)L.mp * L.ldx;
    L.pa = (long)L.m * L.lda;
    long o = kMuonChunks * 8;
    for (int k = 0; k < 2; ++k) L.x[k] = o, o += planes * L.px;
    L.a = o, o += planes * L.pa;
    L.b = o, o += planes * L.pa;
    L.total = (o + 255) / 256 * 256;
    return L;
}

FN_DEV int muon_find(const MuonArgs& a, int wg) {
    int q = 0;
#pragma unroll
    for (int k = 1; k < kMuonMaxJobs; ++k) q += a.first[k] <= wg ? 1 : 0;
    return q;
}
FN_DEV MuonJob muon_job(const MuonArgs& a, int q) {
    MuonJob J = reinterpret_cast<const MuonJob*>(a.scratch)[q];
    // (addresses read from memory are of no known space to the compiler: global, not flat, accesses)
    J.grad = (void*)(FN_GLOBAL char*)J.grad, J.momentum = (void*)(FN_GLOBAL char*)J.momentum;
    J.param = (void*)(FN_GLOBAL char*)J.param, J.out = (void*)(FN_GLOBAL char*)J.out;
    return J;
}

// u = (1 - mu) g + mu m', m' = mu m + (1 - mu) g as it is stored
template <class T>
FN_DEV float muon_u(float g, float m, const MuonNum& P) { return P.nesterov ? P.omu * g + P.mu * m : m; }

// launch 1: the momentum, and the partial sums of |u|^2 (fp64: no overflow, no underflow), kMuonChunks workgroups a matrix
template <class T, bool MOM>
__global__ void __launch_bounds__(256) muon_norm_kernel(MuonJobs js, MuonNum P) {
    const int q = blockIdx.x / kMuonChunks, c = blockIdx.x % kMuonChunks;
    const MuonJob& J = js.j[q];
    if (c == 0 && threadIdx.x == 0) reinterpret_cast<MuonJob*>(js.scratch)[q] = J;
    const long total = (long)J.rows * J.cols;
    const T* g = (const T*)J.grad;
    T* m = (T*)J.momentum;
    constexpr int V = Chunk<T>::N;
    double s = 0.0;
    for (long at = ((long)c * 256 + threadIdx.x) * V; at < total; at += (long)kMuonChunks * 256 * V) {
        const int valid = total - at < V ? (int)(total - at) : V;
        float gv[V], mv[V];
        load_chunk<T>(g + at, valid, gv);
        if constexpr (MOM) {
            load_chunk<T>(m + at, valid, mv);
#pragma unroll
            for (int k = 0; k < V; ++k) mv[k] = (float)(T)(P.mu * mv[k] + P.omu * gv[k]);
            store_chunk<T>(m + at, valid, mv);
#pragma unroll
            for (int k = 0; k < V; ++k) gv[k] = muon_u<T>(gv[k], mv[k], P);
        }
#pragma unroll
        for (int k = 0; k < V; ++k) s += (double)gv[k] * (double)gv[k];
    }
    __shared__ double red[4];
#pragma unroll
    for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) reinterpret_cast<double*>(js.scratch + J.off)[c] = red[0] + red[1] + red[2] + red[3];
}

// one value's planes: hi at p, lo behind it
template <int NP>
FN_DEV void muon_split(float v, _Float16& hi, _Float16& lo) {
    hi = (_Float16)v;
    if constexpr (NP == 2) lo = (_Float16)((v - (float)hi) * kLoScale);
}

// launch 2: X (with its zero padding) from 64 x 64 tiles of u
template <class T, bool MOM, int NP>
__global__ void __launch_bounds__(256) muon_init_kernel(MuonArgs args) {
    __shared__ float tile[64][65];
    __shared__ double red[4];
    const MuonNum& P = args.P;
    const int q = muon_find(args, blockIdx.x);
    const MuonJob J = muon_job(args, q);
    const MuonLay L = muon_lay(J.rows, J.cols, NP);
    unsigned char* S = args.scratch + J.off;
    double s = reinterpret_cast<const double*>(S)[threadIdx.x];       // kMuonChunks == 256 partials
#pragma unroll
    for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    const int tiles_c = (J.cols + 127) / 128 * 2;
    const int t = blockIdx.x - args.first[q], r0 = 64 * (t / tiles_c), c0 = 64 * (t % tiles_c);
    const int lc = threadIdx.x & 63, lr = threadIdx.x >> 6;
#pragma unroll 4
    for (int r = lr; r < 64; r += 4) {
        float u = 0.0f;
        if (r0 + r < J.rows && c0 + lc < J.cols) {
            const long at = (long)(r0 + r) * J.cols + c0 + lc;
            u = (float)((const T*)J.grad)[at];
            if constexpr (MOM) {
                u = muon_u<T>(u, (float)((const T*)J.momentum)[at], P);
                if (P.zero_grad) ((T*)J.grad)[at] = (T)0.0f;
            }
        }
        tile[r][lc] = u;
    }
    __syncthreads();
    const double norm = sqrt(red[0] + red[1] + red[2] + red[3]);
    const float scale = (float)(ldexp(1.0, P.ex) / (norm > (double)P.eps || norm != norm ? norm : (double)P.eps));
    _Float16* x = reinterpret_cast<_Float16*>(S + L.x[0]);
    const unsigned ld = L.ldx / 2;
#pragma unroll 4
    for (int r = lr; r < 64; r += 4) {               // (r, lc): row and column of X within the tile
        _Float16 hi, lo;
        muon_split<NP>((L.trans ? tile[lc][r] : tile[r][lc]) * scale, hi, lo);
        _Float16* o = x + (long)((L.trans ? c0 : r0) + r) * ld + (L.trans ? r0 : c0) + lc;
        o[0] = hi;
        if constexpr (NP == 2) o[L.px / 2] = lo;
        const int row = (L.trans ? c0 : r0) + r, col = (L.trans ? r0 : c0) + lc;
        if (row >= L.m || col >= L.n) {              // the padding of the other X: the steps write the matrix alone
            o += (L.x[1] - L.x[0]) / 2;
            o[0] = (_Float16)0.0f;
            if constexpr (NP == 2) o[L.px / 2] = (_Float16)0.0f;
        }
    }
    // the padding of A and B: columns m .. mp of row t, t + tiles, ...
    const int tiles = tiles_c * ((J.rows + 127) / 128 * 2);
    for (int row = t; row < L.m; row += tiles)
        for (int at = threadIdx.x; at < 2 * NP * (L.mp - L.m); at += 256) {
            const int which = at / (L.mp - L.m), col = L.m + at % (L.mp - L.m);
            *reinterpret_cast<_Float16*>(S + (which & 1 ? L.b : L.a) + (which >> 1) * L.pa + (long)row * L.lda + col * 2) = (_Float16)0.0f;
        }
}

template <int NP>
FN_DEV MmOperand muon_op(const unsigned char* base, long plane, long row_bytes) {
    MmOperand o;
    o.plane[0] = base;
    o.plane[1] = NP == 2 ? base + plane : base;
    o.plane[2] = base;
    o.row_bytes = row_bytes;
    return o;
}

template <int NP>
FN_DEV void muon_write4(unsigned char* p, long plane, const float (&v)[4], f16x4& hi, f16x4& lo) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        _Float16 a, b = (_Float16)0.0f;
        muon_split<NP>(v[k], a, b);
        hi[k] = a, lo[k] = b;
    }
    *reinterpret_cast<f16x4*>(p) = hi;
    if constexpr (NP == 2) *reinterpret_cast<f16x4*>(p + plane) = lo;
}

enum { MU_GRAM = 0, MU_POLY = 1, MU_STEP = 2, MU_LAST = 3 };

// The tiles on and above the diagonal of a symmetric product, numbered by columns
FN_DEV void muon_upper(int t, int& ti, int& tj) {
    tj = (int)((sqrtf(8.0f * (float)t + 1.0f) - 1.0f) * 0.5f);
    while ((tj + 1) * (tj + 2) / 2 <= t) ++tj;
    while (tj * (tj + 1) / 2 > t) --tj;
    ti = t - tj * (tj + 1) / 2;
}

// A symmetric product of few wide tiles (4096: 136 of 256 x 256 for 256 CUs, 528 of 128 x 128 for twice as many places) leaves half the chip
// idle in its last round.  There the stages of ALL its tiles, end to end, are shared out evenly to kMuonParts workgroups; each leaves the sums
// of its part of a tile (two at most) and the product kernel's JOIN form adds a tile's parts in their order.
constexpr int kMuonParts = 256;
template <class Cfg>
FN_DEV float* muon_part(const MuonArgs& a, int wg, int which) { return a.parts + ((long)wg * 2 + which) * (Cfg::BM * Cfg::BN) + threadIdx.x * 4; }
FN_DEV long muon_part_begin(const MuonArgs& a, long wg) { return wg * a.total * a.stages / a.shares; }

template <class Cfg>
FN_DEV void muon_join(const MuonArgs& a, int tile, f32x16 (&acc)[Cfg::MI][Cfg::NJ]) {
#pragma unroll
    for (int m = 0; m < Cfg::MI; ++m)
#pragma unroll
        for (int n = 0; n < Cfg::NJ; ++n)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[m][n][e] = 0.0f;
    const long lo = (long)tile * a.stages, hi = lo + a.stages, all = (long)a.total * a.stages;
    int w = (int)(lo * a.shares / all);
    while (w > 0 && muon_part_begin(a, w) > lo) --w;
    while (muon_part_begin(a, w + 1) <= lo) ++w;              // the part that holds the tile's first stage
    for (; w < a.shares && muon_part_begin(a, w) < hi; ++w) {
        const float* p = muon_part<Cfg>(a, w, muon_part_begin(a, w) < lo ? 1 : 0);
#pragma unroll
        for (int m = 0; m < Cfg::MI; ++m)
#pragma unroll
            for (int n = 0; n < Cfg::NJ; ++n)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const f32x4 q = *reinterpret_cast<const f32x4*>(p + ((m * Cfg::NJ + n) * 4 + g) * (Cfg::THREADS * 4));
#pragma unroll
                    for (int k = 0; k < 4; ++k) acc[m][n][4 * g + k] += q[k];
                }
    }
}

template <class Cfg, int NP, int KIND>
__global__ void __launch_bounds__(Cfg::THREADS, 2) muon_part_kernel(MuonArgs args) {
    extern __shared__ __attribute__((aligned(16))) unsigned char mm_smem[];
    const int wg = (int)mm_spread(blockIdx.x, args.shares);
    long at = muon_part_begin(args, wg);
    const long end = muon_part_begin(args, wg + 1);
#pragma unroll 1
    for (int which = 0; at < end; ++which) {
        const int tile = (int)(at / args.stages), it0 = (int)(at - (long)tile * args.stages);
        const int it1 = end - at < args.stages - it0 ? it0 + (int)(end - at) : args.stages;
        const int q = muon_find(args, tile);
        const MuonJob J = muon_job(args, q);
        const MuonLay L = muon_lay(J.rows, J.cols, NP);
        const unsigned char* S = args.scratch + J.off;
        int ti, tj;
        muon_upper(tile - args.first[q], ti, tj);
        const MmOperand A = KIND == MU_GRAM ? muon_op<NP>(S + L.x[args.cur], L.px, L.ldx) : muon_op<NP>(S + L.a, L.pa, L.lda);
        f32x16 acc[Cfg::MI][Cfg::NJ];
        __syncthreads();                                  // (everyone has read the last part's last stage)
        mm_run<Cfg, _Float16, false, false, NP == 2, false>(mm_smem, A, A, (long)ti * Cfg::BM, L.m, (long)tj * Cfg::BN, L.m,
                                                            args.stages / (NP == 2 ? 3 : 1), 0, NP == 2 ? kMmThree : kMmOne, it0, it1, false, kLoScale, acc);
        float* p = muon_part<Cfg>(args, wg, which);
#pragma unroll
        for (int m = 0; m < Cfg::MI; ++m)
#pragma unroll
            for (int n = 0; n < Cfg::NJ; ++n)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    f32x4 v;
#pragma unroll
                    for (int k = 0; k < 4; ++k) v[k] = acc[m][n][4 * g + k];
                    *reinterpret_cast<f32x4*>(p + ((m * Cfg::NJ + n) * 4 + g) * (Cfg::THREADS * 4)) = v;
                }
        at += it1 - it0;
    }
}

// GRAM: A = X X^T.  POLY: B = b A + c A A.  STEP: X' = a X + B X.  LAST: the same into `out` or the parameter.
// A and B are symmetric: the tiles below the diagonal are the mirror images the tiles above it write.  The epilogue goes through LDS, 32
// rows of a wave at a time, so that either orientation writes runs of a line.
// JOIN: the tile's sums come from the parts of muon_part_kernel.
template <class Cfg, int NP, int KIND, class T, bool MOM, bool JOIN>
__global__ void __launch_bounds__(Cfg::THREADS, 2) muon_product_kernel(MuonArgs args) {
    extern __shared__ __attribute__((aligned(16))) unsigned char mm_smem[];
    const MuonNum& P = args.P;
    const int cur = args.cur;
    const int wg = (int)mm_spread(blockIdx.x, args.total);      // (over all the matrices: a small one stays on one XCD)
    const int q = muon_find(args, wg);
    const MuonJob J = muon_job(args, q);
    const MuonLay L = muon_lay(J.rows, J.cols, NP);
    unsigned char* S = args.scratch + J.off;
    constexpr bool SYM = KIND <= MU_POLY;
    const int ni = L.m, nj = SYM ? L.m : L.n;
    const int tiles_i = (ni + Cfg::BM - 1) / Cfg::BM, tiles_j = (nj + Cfg::BN - 1) / Cfg::BN;
    int ti, tj;
    const int t = wg - args.first[q];
    if constexpr (SYM) muon_upper(t, ti, tj);
    else mm_tile(t, tiles_i, tiles_j, ti, tj);
    const long i0 = (long)ti * Cfg::BM, j0 = (long)tj * Cfg::BN;
    MmOperand A, B;
    if constexpr (KIND == MU_GRAM) A = B = muon_op<NP>(S + L.x[cur], L.px, L.ldx);
    else if constexpr (KIND == MU_POLY) A = B = muon_op<NP>(S + L.a, L.pa, L.lda);
    else A = muon_op<NP>(S + L.b, L.pa, L.lda), B = muon_op<NP>(S + L.x[cur], L.px, L.ldx);
    constexpr int STRIDE = Cfg::WN + 4, SLOTS = Cfg::WN / 8;
    // what the quads of a block add: b A (POLY), a X (STEP, LAST), and the parameters they end in
    f16x4 old_hi[SLOTS], old_lo[SLOTS];
    float par[SLOTS][4];
    const unsigned char* old = S + (KIND == MU_POLY ? L.a : L.x[cur]);
    const long ld_old = KIND == MU_POLY ? L.lda : L.ldx, pl_old = KIND == MU_POLY ? L.pa : L.px, width = ld_old / 2;
    constexpr bool EARLY = Cfg::MI == 1;
    auto load = [&](long i, long j, int s) {
            if constexpr (KIND != MU_GRAM) {
                old_hi[s] = old_lo[s] = f16x4{0, 0, 0, 0};
                if (i < ni && j < width) {
                    old_hi[s] = *reinterpret_cast<const f16x4*>(old + i * ld_old + j * 2);
                    if constexpr (NP == 2) old_lo[s] = *reinterpret_cast<const f16x4*>(old + pl_old + i * ld_old + j * 2);
                }
            }
            if constexpr (KIND == MU_LAST && MOM)
                if (!L.trans && i < ni && j < nj) quad_load((const T*)J.param + i * (long)J.cols + j, (int)(nj - j), par[s]);
        };
    if constexpr (EARLY) {
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) load(mm_quad_i<Cfg>(i0, s), mm_quad_j<Cfg>(j0), s);
    }
    const int k_tiles = (int)((KIND == MU_GRAM ? L.ldx : L.lda) / Cfg::ROW);
    f32x16 acc[Cfg::MI][Cfg::NJ];
    if constexpr (JOIN) muon_join<Cfg>(args, wg, acc);
    else
        mm_run<Cfg, _Float16, false, (KIND >= MU_STEP), NP == 2, false>(mm_smem, A, B, i0, ni, j0, nj, k_tiles, 0, NP == 2 ? kMmThree : kMmOne, 0,
                                                                        (NP == 2 ? 3 : 1) * k_tiles, false, kLoScale, acc);
    const float lo = NP == 2 ? 1.0f / kLoScale : 1.0f;
    // acc -> value: the product of the operands' scales (and the second plane's) is taken out, the result's put in
    float f;
    if constexpr (KIND == MU_GRAM) f = ldexpf(lo, P.ea - 2 * P.ex);
    else if constexpr (KIND == MU_POLY) f = P.c * ldexpf(lo, P.eb - 2 * P.ea);
    else f = ldexpf(lo, (KIND == MU_STEP ? P.ex : 0) - P.eb - P.ex);
    const float fb = KIND == MU_POLY ? ldexpf(P.b, P.eb - P.ea) : 0.0f;
    const float fa = KIND == MU_STEP ? P.a : ldexpf(P.a, -P.ex);
    const float lr = KIND == MU_LAST && MOM ? *P.lr : 0.0f;
    const float keep = 1.0f - lr * P.wd, step = lr * J.adjust;
    const bool turn = SYM ? ti != tj : (KIND == MU_LAST && L.trans);          // the second orientation is written too (SYM) or alone
    mm_epilogue<Cfg, EARLY>(mm_smem, i0, j0, f, acc, load,
        [&](long i, long j, int s, float (&v)[4], float* cell) {
            f16x4 hi, lo4;
            if constexpr (KIND != MU_GRAM) {
                const float w = KIND == MU_POLY ? fb : fa;
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] += w * ((float)old_hi[s][k] + (NP == 2 ? (float)old_lo[s][k] * (1.0f / kLoScale) : 0.0f));
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = i < ni && j + k < nj ? v[k] : 0.0f;
            if (turn) *reinterpret_cast<f32x4*>(cell) = f32x4{v[0], v[1], v[2], v[3]};
            if constexpr (SYM) {
                if (i < ni && j < L.mp) muon_write4<NP>(S + (KIND == MU_GRAM ? L.a : L.b) + i * L.lda + j * 2, L.pa, v, hi, lo4);
            } else if constexpr (KIND == MU_STEP) {
                if (i < L.mp && j < width) muon_write4<NP>(S + L.x[cur ^ 1] + i * L.ldx + j * 2, L.px, v, hi, lo4);
            } else if (!L.trans && i < ni && j < nj) {
                if constexpr (MOM) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) v[k] = par[s][k] * keep - step * v[k];
                }
                quad_store((T*)(MOM ? J.param : J.out) + i * (long)J.cols + j, (int)(nj - j), v);
            }
        },
        [&](long ib, long jb, float* rows) {
            if constexpr (KIND == MU_STEP) return;
            if (!turn) return;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            const int lane = threadIdx.x & 63;
            if constexpr (KIND == MU_LAST && MOM) {
#pragma unroll
                for (int s = 0; s < SLOTS; ++s) {
                    const long j = jb + s * 8 + lane / 8, i = ib + 4 * (lane % 8);
                    if (j < nj && i < ni) quad_load((const T*)J.param + j * (long)J.cols + i, (int)(ni - i), par[s]);
                }
            }
#pragma unroll
            for (int s = 0; s < SLOTS; ++s) {
                const int c = s * 8 + lane / 8, r = 4 * (lane % 8);
                const long i = ib + r, j = jb + c;
                if (j >= nj || i >= ni) continue;
                float v[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = rows[(r + k) * STRIDE + c];
                if constexpr (SYM) {          // (beyond row ni - 1 the rows hold zeros: the padding of row j)
                    f16x4 hi, lo4;
                    muon_write4<NP>(S + (KIND == MU_GRAM ? L.a : L.b) + j * L.lda + i * 2, L.pa, v, hi, lo4);
                } else {
                    if constexpr (MOM) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) v[k] = par[s][k] * keep - step * v[k];
                    }
                    quad_store((T*)(MOM ? J.param : J.out) + j * (long)J.cols + i, (int)(ni - i), v);
                }
            }
        });
}

// ---- matrices whose shorter side m is at most 64 ----------------------------------------------------------------------------------
// Every step multiplies X by a symmetric P = a I + b A + c A A from the left, so with A = X X^T known once the steps need no X:
//   Q <- P Q,  A <- P (P A);   behind the last  O = Q u / |u|_F,  |u|_F^2 = the trace of u u^T.
// Three launches instead of 2 + 3 steps: the momentum and parts of u u^T over stretches of the long axis, the steps on m x m matrices (a workgroup
// a matrix, in LDS), and Q u with the update.  In fp64, on its matrix instructions: a rounding of A grows by up to g' = d(l p(l)^2) / dl a step, 11.9
// at l = 0 for the usual coefficients, which fp32 has no room for (6e-8 x 11.9^4 = 1e-3); muon_scales() keeps 2^-53 x the growth below fp32's.
// Bound by the fp64 matrix instructions of one CU: 0.8 us a step at m <= 16, 2 at 32, 9 at 64; the rest of a call 10 - 20.
typedef double f64x4 __attribute__((ext_vector_type(4)));

constexpr int kFewSide = 64, kFewParts = 64, kFewRun = 64;      // kFewRun: positions along the long axis in LDS at a time

struct MuonFew { int m, n, M, parts; bool trans; long q, total; };
__host__ __device__ inline MuonFew muon_few_lay(int rows, int cols) {
    MuonFew L;
    L.trans = rows > cols;
    L.m = L.trans ? cols : rows;
    L.n = L.trans ? rows : cols;
    L.M = L.m <= 16 ? 16 : (L.m <= 32 ? 32 : 64);
    L.parts = (L.n + 127) / 128 < kFewParts ? (L.n + 127) / 128 : kFewParts;
    const long tiles = L.M / 16 * (L.M / 16 + 1) / 2;
    L.q = L.parts * tiles * 2048;                                // behind the parts of u u^T (the 16 x 16 tiles on and above the diagonal)
    L.total = (L.q + (long)L.M * L.M * 8 + 255) / 256 * 256;
    return L;
}
// runs of the long axis that part p takes
FN_DEV int muon_few_run(const MuonFew& L, int p) { return (int)((long)((L.n + kFewRun - 1) / kFewRun) * p / L.parts); }

// u at (i of the short axis, k of the stretch that starts at `at`) in LDS: i along memory's rows where the matrix is stored so (trans)
template <int M>
FN_DEV int few_at(bool trans, int i, int k) { return trans ? k * (M + 16) + i : i * (kFewRun + 4) + k; }
constexpr int kFewTile = kFewRun * (kFewSide + 16);

// UPDATE: the momentum is updated and stored; else it is taken as it is stored (and `zero_grad` clears the gradient)
template <int M, class T, bool MOM, bool UPDATE>
FN_DEV void few_load(const MuonJob& J, const MuonFew& L, const MuonNum& P, int at, float* tile, int threads) {
    constexpr int N = M * kFewRun / 256;
    float g[N], mo[N];
    long where[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
        const int x = e * threads + threadIdx.x;
        const int i = L.trans ? x % M : x / kFewRun, k = L.trans ? x / M : x % kFewRun;
        where[e] = i < L.m && at + k < L.n ? (L.trans ? (long)(at + k) * J.cols + i : (long)i * J.cols + at + k) : -1;
        const long w = where[e] < 0 ? 0 : where[e];
        g[e] = (float)((const T*)J.grad)[w];
        mo[e] = MOM ? (float)((const T*)J.momentum)[w] : 0.0f;
    }
#pragma unroll
    for (int e = 0; e < N; ++e) {
        const int x = e * threads + threadIdx.x;
        const int i = L.trans ? x % M : x / kFewRun, k = L.trans ? x / M : x % kFewRun;
        float u = g[e];
        if constexpr (MOM) {
            float m = mo[e];
            if constexpr (UPDATE) m = (float)(T)(P.mu * m + P.omu * g[e]);
            u = muon_u<T>(g[e], m, P);
            if (where[e] >= 0) {
                if constexpr (UPDATE) ((T*)J.momentum)[where[e]] = (T)m;
                else if (P.zero_grad) ((T*)J.grad)[where[e]] = (T)0.0f;
            }
        }
        tile[few_at<M>(L.trans, i, k)] = where[e] < 0 ? 0.0f : u;
    }
}

// the tiles of an M x M matrix on and above the diagonal, numbered by columns
FN_DEV constexpr int few_tj(int t) { return t < 1 ? 0 : (t < 3 ? 1 : (t < 6 ? 2 : 3)); }
FN_DEV constexpr int few_ti(int t) { return t - few_tj(t) * (few_tj(t) + 1) / 2; }

// launch 1: parts of u u^T.  Every wave takes a quarter of a stretch's positions for all tiles; the waves are added in order at the end.
template <int M, class T, bool MOM>
FN_DEV void few_gram(const MuonJob& J, const MuonFew& L, const MuonNum& P, int part, double* out, float* tile, f64x4* sums) {
    constexpr int B = M / 16, TILES = B * (B + 1) / 2;
    f64x4 acc[TILES];
#pragma unroll
    for (int t = 0; t < TILES; ++t) acc[t] = f64x4{0.0, 0.0, 0.0, 0.0};
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int end = muon_few_run(L, part + 1);
    for (int run = muon_few_run(L, part); run < end; ++run) {
        few_load<M, T, MOM, true>(J, L, P, run * kFewRun, tile, 256);
        __syncthreads();
#pragma unroll
        for (int s = 0; s < kFewRun / 16; ++s) {
            double f[B];
#pragma unroll
            for (int b = 0; b < B; ++b) f[b] = (double)tile[few_at<M>(L.trans, b * 16 + (lane & 15), wave * 16 + s * 4 + (lane >> 4))];
#pragma unroll
            for (int t = 0; t < TILES; ++t) acc[t] = __builtin_amdgcn_mfma_f64_16x16x4f64(f[few_ti(t)], f[few_tj(t)], acc[t], 0, 0, 0);
        }
        __syncthreads();
    }
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        if (wave == w) {
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
                if (w > 0) acc[t] = sums[t * 64 + lane] + acc[t];
                if (w < 3) sums[t * 64 + lane] = acc[t];
                else reinterpret_cast<f64x4*>(out)[((long)part * TILES + t) * 64 + lane] = acc[t];
            }
        }
        __syncthreads();
    }
}
template <class T, bool MOM>
__global__ void __launch_bounds__(256) muon_few_gram_kernel(MuonJobs js, MuonArgs args) {
    __shared__ float tile[kFewTile];
    __shared__ f64x4 sums[10 * 64];
    const int q = muon_find(args, blockIdx.x), part = blockIdx.x - args.first[q];
    const MuonJob J = js.j[q];
    if (part == 0 && threadIdx.x == 0) reinterpret_cast<MuonJob*>(js.scratch)[q] = J;
    const MuonFew L = muon_few_lay(J.rows, J.cols);
    double* out = reinterpret_cast<double*>(js.scratch + J.off);
    if (L.M == 16) few_gram<16, T, MOM>(J, L, args.P, part, out, tile, sums);
    else if (L.M == 32) few_gram<32, T, MOM>(J, L, args.P, part, out, tile, sums);
    else few_gram<64, T, MOM>(J, L, args.P, part, out, tile, sums);
}

// launch 2: the steps.  Element (k, i) of an M x M matrix in LDS; odd rows swapped by 16 columns: four rows of 16 on different banks
template <int M>
FN_DEV int few_mat(int k, int i) { return k * M + (i ^ ((k & 1) << 4 & (M - 1))); }
// tile t of U V, both symmetric
template <int M>
FN_DEV f64x4 few_product(const double* U, const double* V, int t) {
    const int lane = threadIdx.x & 63, i = few_ti(t) * 16 + (lane & 15), j = few_tj(t) * 16 + (lane & 15);
    f64x4 acc = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
    for (int s = 0; s < M / 4; ++s) {
        const int k = s * 4 + (lane >> 4);
        acc = __builtin_amdgcn_mfma_f64_16x16x4f64(U[few_mat<M>(k, i)], V[few_mat<M>(k, j)], acc, 0, 0, 0);
    }
    return acc;
}
// (a lane holds rows 4 r + lane / 16 of the tile, column lane % 16)
template <int M, class F>
FN_DEV void few_each(int t, f64x4 v, F&& f) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int r = 0; r < 4; ++r) f(few_ti(t) * 16 + 4 * r + (lane >> 4), few_tj(t) * 16 + (lane & 15), v[r]);
}
template <int M>
FN_DEV void few_put(double* D, int t, f64x4 v) {
    few_each<M>(t, v, [&](int i, int j, double x) {
        D[few_mat<M>(i, j)] = x;
        if (few_ti(t) != few_tj(t)) D[few_mat<M>(j, i)] = x;
    });
}
constexpr int kFewWaves = 8;
template <int M>
FN_DEV void few_steps(const MuonFew& L, const MuonNum& P, int steps, unsigned char* scratch, double* lds) {
    constexpr int B = M / 16, TILES = B * (B + 1) / 2, HELD = (TILES + kFewWaves - 1) / kFewWaves;
    double *A = lds, *S = lds + M * M, *W = lds + 2 * M * M, *Q = lds + 3 * M * M;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int other = (wave + kFewWaves - TILES % kFewWaves) % kFewWaves;      // the second product of a phase starts where the first one ends
    for (int t = wave; t < TILES; t += kFewWaves) {
        f64x4 v = {0.0, 0.0, 0.0, 0.0};
        const f64x4* parts = reinterpret_cast<const f64x4*>(scratch) + t * 64 + lane;
#pragma unroll 8
        for (int p = 0; p < L.parts; ++p) v += parts[(long)p * TILES * 64];
        few_put<M>(A, t, v);
    }
    __syncthreads();
    double trace = lane < M ? A[few_mat<M>(lane, lane)] : 0.0;
#pragma unroll
    for (int d = 32; d; d >>= 1) trace += __shfl_xor(trace, d, 64);
    const double root = sqrt(trace), norm = root > (double)P.eps || root != root ? root : (double)P.eps;
    double s = 1.0 / (norm * norm);                     // (the first step's A is not scaled yet)
    f64x4 held[HELD];
    for (int step = 0; step < steps; ++step) {
        const double b = (double)P.b * s, c = (double)P.c * s * s;
        for (int t = wave; t < TILES; t += kFewWaves) {
            const f64x4 v = few_product<M>(A, A, t);
            few_each<M>(t, v, [&](int i, int j, double x) {
                const double y = c * x + b * A[few_mat<M>(i, j)] + (i == j ? (double)P.a : 0.0);
                S[few_mat<M>(i, j)] = y;
                if (step == 0) Q[few_mat<M>(i, j)] = y;
                if (few_ti(t) != few_tj(t)) {
                    S[few_mat<M>(j, i)] = y;
                    if (step == 0) Q[few_mat<M>(j, i)] = y;
                }
            });
        }
        __syncthreads();
        if (step > 0) {
#pragma unroll
            for (int h = 0; h < HELD; ++h)
                if (wave + h * kFewWaves < TILES) held[h] = few_product<M>(S, Q, wave + h * kFewWaves);
        }
        const bool more = step + 1 < steps;
        if (more)
            for (int t = other; t < TILES; t += kFewWaves) few_put<M>(W, t, few_product<M>(S, A, t));
        __syncthreads();
        if (step > 0) {
#pragma unroll
            for (int h = 0; h < HELD; ++h)
                if (wave + h * kFewWaves < TILES) few_put<M>(Q, wave + h * kFewWaves, held[h]);
        }
        if (more)
            for (int t = wave; t < TILES; t += kFewWaves) few_put<M>(A, t, few_product<M>(S, W, t) * s);
        __syncthreads();
        s = 1.0;
    }
    double* out = reinterpret_cast<double*>(scratch + L.q);
    for (int e = threadIdx.x; e < M * M; e += 64 * kFewWaves) out[e] = Q[few_mat<M>(e / M, e % M)] / norm;
}
__global__ void __launch_bounds__(64 * kFewWaves) muon_few_steps_kernel(MuonArgs args, int steps) {
    extern __shared__ __attribute__((aligned(16))) unsigned char mm_smem[];
    double* lds = reinterpret_cast<double*>(mm_smem);
    const MuonJob J = muon_job(args, blockIdx.x);
    const MuonFew L = muon_few_lay(J.rows, J.cols);
    if (L.M == 16) few_steps<16>(L, args.P, steps, args.scratch + J.off, lds);
    else if (L.M == 32) few_steps<32>(L, args.P, steps, args.scratch + J.off, lds);
    else few_steps<64>(L, args.P, steps, args.scratch + J.off, lds);
}

// launch 3: O = Q u, a workgroup a run of the long axis, a wave 16 positions of it; the output's lanes run along memory's rows
template <int M, class T, bool MOM>
FN_DEV void few_apply(const MuonJob& J, const MuonFew& L, const MuonNum& P, int run, const double* q, float* tile, double* Q) {
    constexpr int B = M / 16;
    for (int e = threadIdx.x; e < M * M; e += 256) Q[few_mat<M>(e / M, e % M)] = q[e];
    few_load<M, T, MOM, false>(J, L, P, run * kFewRun, tile, 256);
    __syncthreads();
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    f64x4 acc[B];
#pragma unroll
    for (int b = 0; b < B; ++b) acc[b] = f64x4{0.0, 0.0, 0.0, 0.0};
#pragma unroll 4
    for (int s = 0; s < M / 4; ++s) {
        const int k = s * 4 + (lane >> 4);
        const double x = (double)tile[few_at<M>(L.trans, k, wave * 16 + (lane & 15))];
#pragma unroll
        for (int b = 0; b < B; ++b) {
            const double w = Q[few_mat<M>(k, b * 16 + (lane & 15))];
            acc[b] = L.trans ? __builtin_amdgcn_mfma_f64_16x16x4f64(x, w, acc[b], 0, 0, 0) : __builtin_amdgcn_mfma_f64_16x16x4f64(w, x, acc[b], 0, 0, 0);
        }
    }
    const float lr = MOM ? *P.lr : 0.0f, keep = 1.0f - lr * P.wd, step = lr * J.adjust;
#pragma unroll
    for (int b = 0; b < B; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = 4 * r + (lane >> 4), col = lane & 15;
            const int i = b * 16 + (L.trans ? col : row), k = run * kFewRun + wave * 16 + (L.trans ? row : col);
            if (i >= L.m || k >= L.n) continue;
            const long at = L.trans ? (long)k * J.cols + i : (long)i * J.cols + k;
            if constexpr (MOM) ((T*)J.param)[at] = (T)((float)((const T*)J.param)[at] * keep - step * (float)acc[b][r]);
            else ((T*)J.out)[at] = (T)(float)acc[b][r];
        }
}
template <class T, bool MOM>
__global__ void __launch_bounds__(256) muon_few_apply_kernel(MuonArgs args) {
    __shared__ float tile[kFewTile];
    __shared__ double Q[kFewSide * kFewSide];
    const int q = muon_find(args, blockIdx.x), run = blockIdx.x - args.first[q];
    const MuonJob J = muon_job(args, q);
    const MuonFew L = muon_few_lay(J.rows, J.cols);
    const double* w = reinterpret_cast<const double*>(args.scratch + J.off + L.q);
    if (L.M == 16) few_apply<16, T, MOM>(J, L, args.P, run, w, tile, Q);
    else if (L.M == 32) few_apply<32, T, MOM>(J, L, args.P, run, w, tile, Q);
    else few_apply<64, T, MOM>(J, L, args.P, run, w, tile, Q);
}

typedef MmCfg<64, 64, 2, 2, 4, 2> MuonSmall;       // 8 waves, two sharing each stage's 128 k; 128 KiB: three stages in flight
typedef MmCfg<128, 128, 2, 2, 2> MuonMid;          // 64 KiB, two
typedef MmCfg<128, 128, 2, 2, 2, 2> MuonMid8;      // 8 waves, 128 KiB: for no more than a workgroup a CU
typedef MmCfg<256, 256, 2, 4, 2> MuonBig;          // 128 KiB, one

static long muon_tiles(long m, long n, bool sym, int b) {
    const long ti = (m + b - 1) / b, tj = (n + b - 1) / b;
    return sym ? ti * (ti + 1) / 2 : ti * tj;
}

// whether a symmetric product is shared out evenly: one shape (every tile as long), enough 256-wide tiles and stages that the parts are worth
// their way through memory, and no more tiles than parts (a part then ends at most one tile).  MEASURED at 4096^2, prec 3 (us a product): 528
// tiles of 128 x 128 310, shared out 206 and 38 .. 72 to join
static bool muon_one_shape(const MuonJobs& js) {
    for (int q = 1; q < js.n; ++q)
        if (js.j[q].rows != js.j[0].rows || js.j[q].cols != js.j[0].cols) return false;
    return true;
}
static bool muon_shared(const MuonJobs& js, int planes) {
    if (!muon_one_shape(js)) return false;
    const long m = js.j[0].rows < js.j[0].cols ? js.j[0].rows : js.j[0].cols, tiles = muon_tiles(m, m, true, 256) * js.n;
    return tiles >= 96 && tiles <= kMuonParts && m >= 1024 * (3 - planes);
}
// The same with 64-wide tiles for X X^T of a few rows that are long: tiles and stages such that what the other CUs take over, at 0.4 us a stage, is
// worth the launch that joins.  MEASURED (us a call, shared out against not; in brackets the stages taken over): fp32 65 x 65536 505 / 3540
// [3036], 256 x 4096 247 / 358 [185], 2975 x 422 300 / 383 [128], 3 x (188 x 1436) 215 / 226 [67], 4 x (512 x 2048) 363 / 343 [42], 2 x (128 x 640)
// 156 / 147 [29]; bf16 256 x 4096 180 / 190 [62], 2975 x 422 221 / 216 [43]
typedef MmCfg<64, 64, 2, 2, 4> MuonPart;
static bool muon_gram_shared(const MuonJobs& js, int planes) {
    if (!muon_one_shape(js)) return false;
    const long m = js.j[0].rows < js.j[0].cols ? js.j[0].rows : js.j[0].cols, n = js.j[0].rows < js.j[0].cols ? js.j[0].cols : js.j[0].rows;
    const long tiles = muon_tiles(m, m, true, 64) * js.n, stages = (planes == 2 ? 3 : 1) * ((n + 127) / 128 * 2);
    return muon_tiles(m, m, true, 128) * js.n < 128 && tiles < kMuonParts && stages * (kMuonParts - tiles) >= 56L * kMuonParts;
}
static long muon_part_bytes(const MuonJobs& js, int planes) {
    return muon_shared(js, planes) ? (long)kMuonParts * 2 * MuonBig::BM * MuonBig::BN * 4
                                   : (muon_gram_shared(js, planes) ? (long)kMuonParts * 2 * MuonPart::BM * MuonPart::BN * 4 : 0);
}

template <class Cfg, int NP, int KIND, class T, bool MOM, bool JOIN = false>
static void muon_product_launch(const MuonJobs& js, MuonArgs& args, hipStream_t stream) {
    long tiles = 0;
    for (int q = 0; q < js.n; ++q) {
        const MuonJob& J = js.j[q];
        args.first[q] = (int)tiles;
        tiles += muon_tiles(J.rows < J.cols ? J.rows : J.cols, J.rows < J.cols ? J.cols : J.rows, KIND <= MU_POLY, Cfg::BM);
    }
    args.total = (int)tiles;
    if constexpr (JOIN) {
        const MuonLay L = muon_lay(js.j[0].rows, js.j[0].cols, NP);
        args.stages = (NP == 2 ? 3 : 1) * (int)((KIND == MU_GRAM ? L.ldx : L.lda) / Cfg::ROW);
        args.shares = (int)(tiles * args.stages / 4 < kMuonParts ? tiles * args.stages / 4 : kMuonParts);       // (four stages at least: none empty)
        auto part = muon_part_kernel<Cfg, NP, KIND>;
        allow_big_lds(part);
        hipLaunchKernelGGL(part, dim3((unsigned)args.shares), dim3(Cfg::THREADS), Cfg::LDS, stream, args);
    }
    auto kernel = muon_product_kernel<Cfg, NP, KIND, T, MOM, JOIN>;
    allow_big_lds(kernel);
    hipLaunchKernelGGL(kernel, dim3((unsigned)tiles), dim3(Cfg::THREADS), Cfg::LDS, stream, args);
}

// the largest tile that still occupies the chip (256: three quarters of the CUs, 128: half of them)
template <int NP, int KIND, class T, bool MOM>
static void muon_product(const MuonJobs& js, MuonArgs& args, hipStream_t stream) {
    long big = 0, mid = 0;
    for (int q = 0; q < js.n; ++q) {
        const MuonJob& J = js.j[q];
        const long m = J.rows < J.cols ? J.rows : J.cols, n = J.rows < J.cols ? J.cols : J.rows;
        big += muon_tiles(m, n, KIND <= MU_POLY, 256), mid += muon_tiles(m, n, KIND <= MU_POLY, 128);
    }
    if constexpr (KIND <= MU_POLY) {
        if (args.parts && !args.narrow) {
            muon_product_launch<MuonBig, NP, KIND, T, MOM, true>(js, args, stream);
            return;
        }
        if (KIND == MU_GRAM && args.parts) {
            muon_product_launch<MuonPart, NP, MU_GRAM, T, MOM, true>(js, args, stream);
            return;
        }
    }
    if (big >= 192) muon_product_launch<MuonBig, NP, KIND, T, MOM>(js, args, stream);
    else if (mid > 256) muon_product_launch<MuonMid, NP, KIND, T, MOM>(js, args, stream);
    else if (mid >= 128) muon_product_launch<MuonMid8, NP, KIND, T, MOM>(js, args, stream);
    else muon_product_launch<MuonSmall, NP, KIND, T, MOM>(js, args, stream);
}

template <int NP, class T, bool MOM>
static void muon_steps(const MuonJobs& js, MuonArgs& args, int steps, hipStream_t stream) {
    for (int s = 0; s < steps; ++s) {
        args.cur = s & 1;
        muon_product<NP, MU_GRAM, T, MOM>(js, args, stream);
        muon_product<NP, MU_POLY, T, MOM>(js, args, stream);
        if (s + 1 < steps) muon_product<NP, MU_STEP, T, MOM>(js, args, stream);
        else muon_product<NP, MU_LAST, T, MOM>(js, args, stream);
    }
}

// which form a matrix takes; `few`: whether the polynomial and the steps allow the one for short sides (muon_scales).  MEASURED (us a call, it
// against the tiled one): fp32 2 x (2038 x 3) 17 / 205, 8 x (32 x 256) 27 / 117, one 64 x 64 63 / 109, 40 of them 129 / 233, 64 x 8192 88 / 537,
// 32 x (64 x 4096) 166 / 566; bf16 73 / 97 for 8 x (64 x 256), 88 / 234 for 64 x 8192.  Sides beyond 64 do not fit the four matrices in LDS.
static bool muon_few(const FneusMuonJob& f, bool few) { return few && (f.rows < f.cols ? f.rows : f.cols) <= kFewSide; }

// the next round of launches: up to kMuonMaxJobs matrices of one form, from jobs[at] on; `off`: the scratch it takes
enum { MU_ALL = 0, MU_TILED = 1, MU_FEW = 2 };       // ALL: every matrix tiled
static int muon_round(const FneusMuonJob* jobs, int n_jobs, int& at, int form, int planes, MuonJobs& js, long& off) {
    js.n = 0;
    off = kMuonTable;
    for (; at < n_jobs && js.n < kMuonMaxJobs; ++at) {
        const FneusMuonJob& f = jobs[at];
        if (f.rows <= 0 || f.cols <= 0 || (form != MU_ALL && muon_few(f, true) != (form == MU_FEW))) continue;
        MuonJob& J = js.j[js.n++];
        J.grad = f.grad, J.momentum = f.momentum, J.param = f.param, J.out = f.out;
        J.rows = f.rows, J.cols = f.cols, J.adjust = f.adjust, J.pad_ = 0, J.off = off;
        off += form == MU_FEW ? muon_few_lay(f.rows, f.cols).total : muon_lay(f.rows, f.cols, planes).total;
    }
    return (int)js.n;
}

template <class T, bool MOM>
static void muon_few_run(MuonJobs& js, MuonArgs& args, int steps, hipStream_t stream) {
    long parts = 0, runs = 0, M = 16;
    MuonArgs apply = args;
    for (int q = 0; q < js.n; ++q) {
        const MuonFew L = muon_few_lay(js.j[q].rows, js.j[q].cols);
        args.first[q] = (int)parts, apply.first[q] = (int)runs;
        parts += L.parts, runs += (L.n + kFewRun - 1) / kFewRun;
        M = L.M > M ? L.M : M;
    }
    hipLaunchKernelGGL((muon_few_gram_kernel<T, MOM>), dim3((unsigned)parts), dim3(256), 0, stream, js, args);
    auto kernel = muon_few_steps_kernel;
    allow_big_lds(kernel);
    hipLaunchKernelGGL(kernel, dim3((unsigned)js.n), dim3(64 * kFewWaves), (unsigned)(4 * M * M * 8), stream, args, steps);
    hipLaunchKernelGGL((muon_few_apply_kernel<T, MOM>), dim3((unsigned)runs), dim3(256), 0, stream, apply);
}

template <class T, bool MOM, int NP>
static int muon_run(const FneusMuonJob* jobs, int n_jobs, const MuonNum& P, int steps, bool few, unsigned char* scratch, hipStream_t stream) {
    MuonJobs js;                                        // (a local: filled anew for every round)
    js.scratch = scratch;
    long off;
    MuonArgs args;
    args.P = P, args.cur = 0, args.scratch = scratch, args.stages = 0, args.shares = 0, args.narrow = 0, args.pad_ = 0, args.parts = nullptr, args.total = 0;
    for (int at = 0; few && muon_round(jobs, n_jobs, at, MU_FEW, NP, js, off) > 0;) {
        for (int q = 0; q < kMuonMaxJobs; ++q) args.first[q] = 0x7fffffff;
        muon_few_run<T, MOM>(js, args, steps, stream);
    }
    for (int at = 0; muon_round(jobs, n_jobs, at, few ? MU_TILED : MU_ALL, NP, js, off) > 0;) {
        for (int q = 0; q < kMuonMaxJobs; ++q) args.first[q] = 0x7fffffff;
        long tiles = 0;
        for (int q = 0; q < js.n; ++q) {
            args.first[q] = (int)tiles;
            tiles += (long)((js.j[q].rows + 127) / 128) * ((js.j[q].cols + 127) / 128) * 4;
        }
        args.parts = muon_part_bytes(js, NP) > 0 ? reinterpret_cast<float*>(scratch + off) : nullptr;
        args.narrow = !muon_shared(js, NP);
        hipLaunchKernelGGL((muon_norm_kernel<T, MOM>), dim3((unsigned)(js.n * kMuonChunks)), dim3(256), 0, stream, js, P);
        hipLaunchKernelGGL((muon_init_kernel<T, MOM, NP>), dim3((unsigned)tiles), dim3(256), 0, stream, args);
        muon_steps<NP, T, MOM>(js, args, steps, stream);
    }
    return launch_status();
}

static int muon_refuse(const char* msg) {
    set_last_error(msg);
    return -2;
}

// the largest power of two that keeps `bound` (with 2 % for rounding) within fp16, at most 2^14
static int muon_exponent(double bound) {
    int e = 14;
    while (e > -14 && ldexp(bound * 1.02, e) > 65504.0) --e;
    return e;
}

// bounds of the singular values over the steps (from [0, 1]: the Frobenius norm) give the planes' scales
// `few`: whether the form that keeps A = X X^T through the steps may run: an error of A grows by the slope of l p(l)^2 in every step but the last
static bool muon_scales(double a, double b, double c, int steps, MuonNum& P, bool& few) {
    double top = 1.0, x = 1.0, poly = 0.0, gain = 1.0, last = 1.0;
    if (!isfinite(a) || !isfinite(b) || !isfinite(c)) return false;
    for (int s = 0; s < steps; ++s) {
        double next = 0.0;
        gain *= last, last = 1.0;
        for (int k = 0; k <= 512; ++k) {
            const double v = top * k / 512.0, q = v * v;
            const double p = fabs(b * q + c * q * q), w = fabs(a * v + b * v * q + c * v * q * q);
            const double slope = fabs((a + b * q + c * q * q) * (a + 3.0 * b * q + 5.0 * c * q * q));
            last = slope > last ? slope : last;
            poly = p > poly ? p : poly;
            next = w > next ? w : next;
        }
        x = top > x ? top : x;
        top = next * 1.001 + 1e-6;
        if (!(top <= 16.0)) return false;
    }
    few = gain <= 1e7;                   // (x 2^-53 x 64: below fp32's half step)
    // (the last step's result is not kept in planes)
    P.ex = muon_exponent(x), P.ea = muon_exponent(x * x), P.eb = muon_exponent(poly > 1e-3 ? poly : 1e-3);
    return true;
}

static int muon_check(const FneusMuonJob* jobs, int n_jobs, int steps, int prec, int dtype, void* scratch, long bytes, bool mom) {
    if (n_jobs < 0 || (n_jobs > 0 && !jobs)) return muon_refuse("fneus_muon: jobs must be given");
    if (steps < 1 || steps > 64) return muon_refuse("fneus_muon: 1 to 64 steps");
    if ((prec != 2 && prec != 3) || dtype < 0 || dtype > 2) return muon_refuse("fneus_muon: prec 2 or 3, dtype 0..2");
    for (int q = 0; q < n_jobs; ++q) {
        const FneusMuonJob& f = jobs[q];
        if (f.rows <= 0 || f.cols <= 0 || f.rows > 65536 || f.cols > 65536) return muon_refuse("fneus_muon: a matrix needs 1 to 65536 rows and columns");
        if (!f.grad || (mom ? !f.momentum || !f.param : !f.out)) return muon_refuse("fneus_muon: grad, and momentum and param (or out), must be given");
    }
    if (n_jobs > 0 && (!scratch || bytes < fneus_muon_scratch_bytes(jobs, n_jobs, prec) || ((uintptr_t)scratch & 255)))
        return muon_refuse("fneus_muon: scratch of fneus_muon_scratch_bytes bytes, 256-byte aligned, must be given");
    return 0;
}

template <bool MOM>
static int muon_dispatch(const FneusMuonJob* jobs, int n, const MuonNum& P, int steps, bool few, int prec, int dtype, void* scratch, hipStream_t s) {
    unsigned char* w = (unsigned char*)scratch;
    if (dtype == DT_F32) return prec == 3 ? muon_run<float, MOM, 2>(jobs, n, P, steps, few, w, s) : muon_run<float, MOM, 1>(jobs, n, P, steps, few, w, s);
    if (dtype == DT_BF16) return prec == 3 ? muon_run<__bf16, MOM, 2>(jobs, n, P, steps, few, w, s) : muon_run<__bf16, MOM, 1>(jobs, n, P, steps, few, w, s);
    return prec == 3 ? muon_run<_Float16, MOM, 2>(jobs, n, P, steps, few, w, s) : muon_run<_Float16, MOM, 1>(jobs, n, P, steps, few, w, s);
}

}  // namespace fneus

using namespace fneus;

extern "C" long fneus_muon_scratch_bytes(const FneusMuonJob* jobs, int n_jobs, int prec) {
    long most = 0, off;
    if (!jobs) return 0;
    const int planes = prec == 3 ? 2 : 1;
    MuonJobs js;
    for (int form = MU_ALL; form <= MU_FEW; ++form)       // (a further round of launches uses the same memory: one stream)
        for (int at = 0; muon_round(jobs, n_jobs, at, form, planes, js, off) > 0;) {
            if (form != MU_FEW) off += muon_part_bytes(js, planes);
            most = off > most ? off : most;
        }
    return most;
}

extern "C" int fneus_newton_schulz(const FneusMuonJob* jobs, int n_jobs, double a, double b, double c, int steps, double eps, int prec,
                                   int dtype, void* scratch, long scratch_bytes, fneus_stream_t stream) {
    fneus::clear_status();
    if (int rc = muon_check(jobs, n_jobs, steps, prec, dtype, scratch, scratch_bytes, false)) return rc;
    MuonNum P{};
    bool few = false;
    P.a = (float)a, P.b = (float)b, P.c = (float)c, P.eps = (float)eps;
    if (!(P.eps >= 1e-30f) || !muon_scales(a, b, c, steps, P, few)) return muon_refuse("fneus_newton_schulz: eps >= 1e-30, a polynomial that keeps [0, 1] below 16 over the steps");
    if (n_jobs == 0) return 0;
    return muon_dispatch<false>(jobs, n_jobs, P, steps, few, prec, dtype, scratch, (hipStream_t)stream);
}

extern "C" int fneus_muon(const FneusMuonJob* jobs, int n_jobs, const float* lr, double mu, int nesterov, double weight_decay, double a,
                          double b, double c, int steps, double eps, int prec, int dtype, int zero_grad, void* scratch,
                          long scratch_bytes, fneus_stream_t stream) {
    fneus::clear_status();
    if (int rc = muon_check(jobs, n_jobs, steps, prec, dtype, scratch, scratch_bytes, true)) return rc;
    MuonNum P{};
    bool few = false;
    P.a = (float)a, P.b = (float)b, P.c = (float)c, P.eps = (float)eps;
    if (!lr || !(P.eps >= 1e-30f) || !muon_scales(a, b, c, steps, P, few)) return muon_refuse("fneus_muon: lr, eps >= 1e-30, a polynomial that keeps [0, 1] below 16 over the steps");
    P.mu = (float)mu, P.omu = (float)(1.0 - mu), P.wd = (float)weight_decay, P.nesterov = nesterov, P.zero_grad = zero_grad, P.lr = lr;
    if (n_jobs == 0) return 0;
    return muon_dispatch<true>(jobs, n_jobs, P, steps, few, prec, dtype, scratch, (hipStream_t)stream);
}
