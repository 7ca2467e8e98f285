// The Muon update of weight matrices: momentum, orthogonalisation by Newton-Schulz products, step -- every matrix of a model in the same
// 2 + 3 * steps launches.  For each matrix u, as X [m][n] with m <= n (the transpose where rows > cols):
//   X = u / max(|u|_F, eps);   steps times:  A = X X^T,  B = b A + c A A,  X <- a X + B X
// All three products run on the tiled engine (mm_engine.h): X X^T and A A on operands stored along k, B X with X k-major.
//
// Numbers: fp16 planes with fp32 sums.  Every entry of X, A and B is bounded (the polynomial keeps the singular values below about 1.2),
// entries as small as 1 / n matter, and the fp16 matrix instruction takes subnormal operands as zero, so a plane holds its matrix times a
// power of two that puts the bound just below fp16's largest value (2^14 for the usual coefficients).  prec 2: one plane, 11 bits -- the
// error that 16-bit gradients bring along, an eighth of what bf16 operands would add.  prec 3: a second plane holds what the first one's
// rounding left, times another 2^11, so that it is as normal as the first; products hi hi + hi lo + lo hi (22 bits: fp32's accuracy at
// half the matrix work of three bf16 terms).
//
// What bounds it (MI355X, us): one fp32 4096^2 matrix 4600, of which matrix products 4470 at 1.0 - 1.1 PFLOP/s of fp16 MFMAs (a bare stream
// of them: 1.6), the momentum and norm 56 (5 x 64 MiB: 6 TB/s); four bf16 4096 x 1024 531 (X X^T 41, A A 18, B X 48 a step); eight fp32
// 256^2 145 = 17 launches of 8 .. 10: 1.3 until the job is read, 2.7 until the first stage has arrived from the other XCDs' writes, 0.4 a stage.
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
    int stages, pad_;
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
FN_DEV long muon_part_begin(const MuonArgs& a, long wg) { return wg * a.total * a.stages / kMuonParts; }

template <class Cfg>
FN_DEV void muon_join(const MuonArgs& a, int tile, f32x16 (&acc)[Cfg::MI][Cfg::NJ]) {
#pragma unroll
    for (int m = 0; m < Cfg::MI; ++m)
#pragma unroll
        for (int n = 0; n < Cfg::NJ; ++n)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[m][n][e] = 0.0f;
    const long lo = (long)tile * a.stages, hi = lo + a.stages, all = (long)a.total * a.stages;
    int w = (int)(lo * kMuonParts / all);
    while (w > 0 && muon_part_begin(a, w) > lo) --w;
    while (muon_part_begin(a, w + 1) <= lo) ++w;              // the part that holds the tile's first stage
    for (; w < kMuonParts && muon_part_begin(a, w) < hi; ++w) {
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
    const int wg = (int)mm_spread(blockIdx.x, kMuonParts);
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
static bool muon_shared(int rows, int cols, int n_jobs, int planes) {
    const long m = rows < cols ? rows : cols, tiles = muon_tiles(m, m, true, 256) * n_jobs;
    return tiles >= 96 && tiles <= kMuonParts && m >= 1024 * (3 - planes);
}
static bool muon_one_shape(const FneusMuonJob* jobs, int n) {
    for (int q = 1; q < n; ++q)
        if (jobs[q].rows != jobs[0].rows || jobs[q].cols != jobs[0].cols) return false;
    return n > 0;
}
constexpr long kMuonPartBytes = (long)kMuonParts * 2 * MuonBig::BM * MuonBig::BN * 4;

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
        auto part = muon_part_kernel<Cfg, NP, KIND>;
        allow_big_lds(part);
        hipLaunchKernelGGL(part, dim3(kMuonParts), dim3(Cfg::THREADS), Cfg::LDS, stream, args);
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
        if (args.parts) {
            muon_product_launch<MuonBig, NP, KIND, T, MOM, true>(js, args, stream);
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

template <class T, bool MOM, int NP>
static int muon_run(const FneusMuonJob* jobs, int n_jobs, const MuonNum& P, int steps, unsigned char* scratch, hipStream_t stream) {
    for (int first = 0; first < n_jobs; first += kMuonMaxJobs) {
        MuonJobs js;
        js.n = n_jobs - first < kMuonMaxJobs ? n_jobs - first : kMuonMaxJobs;       // (a local: filled anew for every round)
        js.scratch = scratch;
        MuonArgs args;
        args.P = P, args.cur = 0, args.scratch = scratch;
        for (int q = 0; q < kMuonMaxJobs; ++q) args.first[q] = 0x7fffffff;
        long off = kMuonTable, tiles = 0;
        for (int q = 0; q < js.n; ++q) {
            const FneusMuonJob& f = jobs[first + q];
            MuonJob& J = js.j[q];
            J.grad = f.grad, J.momentum = f.momentum, J.param = f.param, J.out = f.out;
            J.rows = f.rows, J.cols = f.cols, J.adjust = f.adjust, J.off = off, args.first[q] = (int)tiles;
            off += muon_lay(f.rows, f.cols, NP).total;
            tiles += (long)((f.rows + 127) / 128) * ((f.cols + 127) / 128) * 4;
        }
        args.stages = 0, args.parts = nullptr;
        if (muon_one_shape(jobs + first, js.n) && muon_shared(js.j[0].rows, js.j[0].cols, js.n, NP)) args.parts = reinterpret_cast<float*>(scratch + off);
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
static bool muon_scales(double a, double b, double c, int steps, MuonNum& P) {
    double top = 1.0, x = 1.0, poly = 0.0;
    if (!isfinite(a) || !isfinite(b) || !isfinite(c)) return false;
    for (int s = 0; s < steps; ++s) {
        double next = 0.0;
        for (int k = 0; k <= 512; ++k) {
            const double v = top * k / 512.0, q = v * v;
            const double p = fabs(b * q + c * q * q), w = fabs(a * v + b * v * q + c * v * q * q);
            poly = p > poly ? p : poly;
            next = w > next ? w : next;
        }
        x = top > x ? top : x;
        top = next * 1.001 + 1e-6;
        if (!(top <= 16.0)) return false;
    }
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
static int muon_dispatch(const FneusMuonJob* jobs, int n, const MuonNum& P, int steps, int prec, int dtype, void* scratch, hipStream_t s) {
    unsigned char* w = (unsigned char*)scratch;
    if (dtype == DT_F32) return prec == 3 ? muon_run<float, MOM, 2>(jobs, n, P, steps, w, s) : muon_run<float, MOM, 1>(jobs, n, P, steps, w, s);
    if (dtype == DT_BF16) return prec == 3 ? muon_run<__bf16, MOM, 2>(jobs, n, P, steps, w, s) : muon_run<__bf16, MOM, 1>(jobs, n, P, steps, w, s);
    return prec == 3 ? muon_run<_Float16, MOM, 2>(jobs, n, P, steps, w, s) : muon_run<_Float16, MOM, 1>(jobs, n, P, steps, w, s);
}

}  // namespace fneus

using namespace fneus;

extern "C" long fneus_muon_scratch_bytes(const FneusMuonJob* jobs, int n_jobs, int prec) {
    long most = 0;
    if (!jobs) return 0;
    for (int first = 0; first < n_jobs; first += kMuonMaxJobs) {       // (a further round of launches uses the same memory: one stream)
        long off = kMuonTable;
        for (int q = first; q < n_jobs && q < first + kMuonMaxJobs; ++q)
            if (jobs[q].rows > 0 && jobs[q].cols > 0) off += muon_lay(jobs[q].rows, jobs[q].cols, prec == 3 ? 2 : 1).total;
        const int n = n_jobs - first < kMuonMaxJobs ? n_jobs - first : kMuonMaxJobs;
        if (muon_one_shape(jobs + first, n) && muon_shared(jobs[first].rows, jobs[first].cols, n, prec == 3 ? 2 : 1)) off += kMuonPartBytes;
        most = off > most ? off : most;
    }
    return most;
}

extern "C" int fneus_newton_schulz(const FneusMuonJob* jobs, int n_jobs, double a, double b, double c, int steps, double eps, int prec,
                                   int dtype, void* scratch, long scratch_bytes, fneus_stream_t stream) {
    fneus::clear_status();
    if (int rc = muon_check(jobs, n_jobs, steps, prec, dtype, scratch, scratch_bytes, false)) return rc;
    MuonNum P{};
    P.a = (float)a, P.b = (float)b, P.c = (float)c, P.eps = (float)eps;
    if (!(eps > 0.0) || !muon_scales(a, b, c, steps, P)) return muon_refuse("fneus_newton_schulz: eps > 0, a polynomial that keeps [0, 1] below 16 over the steps");
    if (n_jobs == 0) return 0;
    return muon_dispatch<false>(jobs, n_jobs, P, steps, prec, dtype, scratch, (hipStream_t)stream);
}

extern "C" int fneus_muon(const FneusMuonJob* jobs, int n_jobs, const float* lr, double mu, int nesterov, double weight_decay, double a,
                          double b, double c, int steps, double eps, int prec, int dtype, int zero_grad, void* scratch,
                          long scratch_bytes, fneus_stream_t stream) {
    fneus::clear_status();
    if (int rc = muon_check(jobs, n_jobs, steps, prec, dtype, scratch, scratch_bytes, true)) return rc;
    MuonNum P{};
    P.a = (float)a, P.b = (float)b, P.c = (float)c, P.eps = (float)eps;
    if (!lr || !(eps > 0.0) || !muon_scales(a, b, c, steps, P)) return muon_refuse("fneus_muon: lr, eps > 0, a polynomial that keeps [0, 1] below 16 over the steps");
    P.mu = (float)mu, P.omu = (float)(1.0 - mu), P.wd = (float)weight_decay, P.nesterov = nesterov, P.zero_grad = zero_grad, P.lr = lr;
    if (n_jobs == 0) return 0;
    return muon_dispatch<true>(jobs, n_jobs, P, steps, prec, dtype, scratch, (hipStream_t)stream);
}
