// Linear layer with bias, activation and residual in its epilogue, forward and backward, fp32 / bf16 / fp16:
//   z = x W^T + b,  y = act(z) + res;      delta = dy act'(z),  dx = delta W,  dW = delta^T x,  db = column sums of delta
// The three products are one form, D(i, j) = sum_k A(i, k) B(j, k), with either operand stored along k or along its rows.
#include "linear_act.h"
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

// 8 values of an operand for one lane, (i, k0 .. k0 + 7), zero beyond the matrix.  ROWS: stored along k (unaligned 16-byte loads),
// else element (i, k) at p[k ld + i] (the 32 lanes of a half read consecutive values)
template <class T, bool ROWS>
FN_DEV void lin_load8(const T* __restrict__ p, long ld, long i, long ni, long k0, long kend, float (&v)[8]) {
    const bool in = i < ni;
    if constexpr (ROWS) {
        const T* q = p + i * ld + k0;
        const long left = in ? kend - k0 : 0;
        constexpr int N = Chunk<T>::N;
        if (left >= 8) {
#pragma unroll
            for (int c = 0; c < 8 / N; ++c) {
                const typename Chunk<T>::type u = *reinterpret_cast<const typename Chunk<T>::type*>(q + c * N);
#pragma unroll
                for (int k = 0; k < N; ++k) v[c * N + k] = (float)u[k];
            }
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = k < left ? (float)q[k] : 0.0f;
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = in && k0 + k < kend ? (float)p[(k0 + k) * ld + i] : 0.0f;
    }
}

// The direct kernel: a workgroup owns a 32 x 32 tile of D, its 8 waves split the contraction, operands go from memory to the matrix
// instructions without LDS, the partial tiles are added in wave order (LDS).  For products too small for the tiled kernel to fill the
// chip, where a launch's latency is what counts: one launch forward, one backward.
template <class T, int KIND>
FN_DEV void lin_direct_tile(const LinProduct& P, long tile, float (*red)[16][65], float (*red_db)[32]) {
    constexpr bool AROWS = KIND != LIN_DW, BROWS = KIND == LIN_FWD;
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
    constexpr int U = 2;
    for (long k = kb; k < ke; k += 16 * U) {
        float av[U][8], bv[U][8], zv[U][8];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long k0 = k + 16 * u + 8 * h;
            lin_load8<T, AROWS>(a, P.lda, i0 + r, P.ni, k0, ke, av[u]);
            lin_load8<T, BROWS>(b, P.ldb, j0 + r, P.d ? P.nj : 0, k0, ke, bv[u]);      // (no D: the bias gradient alone)
            if (KIND != LIN_FWD && az) lin_load8<T, AROWS>(az, P.ldz, i0 + r, P.ni, k0, ke, zv[u]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (KIND != LIN_FWD && az) {
#pragma unroll
                for (int s = 0; s < 8; ++s) av[u][s] *= lin_dact(zv[u][s], P.act);
            }
            if constexpr (KIND == LIN_DW) {
#pragma unroll
                for (int s = 0; s < 8; ++s) asum += av[u][s];
            }
            LinFrag<T> fa, fb;
            lin_frag(av[u], fa);
            lin_frag(bv[u], fb);
            acc = lin_mfma32(fb, fa, acc);           // accumulator rows = j, columns (lanes) = i
        }
    }
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
template <class T>
__global__ void __launch_bounds__(512) linear_row_kernel(LinProduct P) {
    __shared__ float red[8][16][17];
    const int j0 = 16 * (int)blockIdx.x;
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const long part = ((P.nk + 7) / 8 + 31) / 32 * 32;
    const long kb = wave * part, ke = kb + part < P.nk ? kb + part : P.nk;
    const T *a = (const T*)P.a, *b = (const T*)P.b;
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    constexpr int U = 4;
    for (long k = kb; k < ke; k += 32 * U) {
        float av[U][8], bv[U][8];
#pragma unroll
        for (int u = 0; u < U; ++u) lin_load8<T, true>(b, P.ldb, j0 + r, P.nj, k + 32 * u + 8 * g, ke, bv[u]);
#pragma unroll
        for (int u = 0; u < U; ++u) lin_load8<T, true>(a, P.lda, r, P.ni, k + 32 * u + 8 * g, ke, av[u]);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            LinFrag<T> fa, fb;
            lin_frag(av[u], fa);
            lin_frag(bv[u], fb);
            acc = lin_mfma16(fb, fa, acc);
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) red[wave][4 * g + e][r] = acc[e];        // row j = 4 g + e, column i = r
    __syncthreads();
    if (threadIdx.x < 256) {
        const int jj = threadIdx.x & 15, ii = threadIdx.x >> 4;
        const int gj = j0 + jj;
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < 8; ++w) v += red[w][jj][ii];
        if (ii < P.ni && gj < P.nj) {
            if (P.bias) v += (float)((const T*)P.bias)[gj];
            if (P.z) ((T*)P.z)[ii * P.ldd + gj] = (T)v;
            v = lin_act(v, P.act);
            if (P.res) v += (float)((const T*)P.res)[ii * P.ldres + gj];
            ((T*)P.d)[ii * P.ldd + gj] = (T)v;
        }
    }
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

template <class T>
static int lin_fwd(const FneusLinear& f, hipStream_t stream) {
    LinProduct p{};
    p.a = f.x, p.lda = f.ldx, p.b = f.weight, p.ldb = f.n_in, p.bias = f.bias, p.res = f.residual, p.ldres = f.ld_residual;
    p.d = f.y, p.z = f.z, p.ldd = f.n_out, p.ni = f.rows, p.nj = f.n_out, p.nk = f.n_in, p.act = f.act;
    if (f.rows <= 16) {
        hipLaunchKernelGGL((linear_row_kernel<T>), dim3((unsigned)((f.n_out + 15) / 16)), dim3(512), 0, stream, p);
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

extern "C" long fneus_linear_scratch_bytes(const FneusLinear* f, int backward) { return 0; }

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
