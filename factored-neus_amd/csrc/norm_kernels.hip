// Layer norm over the last axis, forward and backward (fp32 / bf16 / fp16; statistics and sums in fp32).
//   row x[n]:  mu = mean(x),  var = mean((x - mu)^2),  r = 1 / sqrt(var + eps),  xh = (x - mu) r,  y = xh w + b
//   backward:  g = dy w,  dx = r (g - mean(g) - xh mean(g xh)),  dw = sum_rows dy xh,  db = sum_rows dy
// Memory bound: the forward reads x and writes y, the backward reads dy and x and writes dx.  A TEAM of TPR threads owns a row and
// holds it in registers (EPT values a thread, 16-byte chunks): one pass over memory, the variance from the centred values (two
// passes over registers: a row with a large mean keeps its digits).  TPR = 16 (sums by DPP), 64, 256 or 512 threads; wider rows
// take the streaming kernels, which read a row from the caches again; rows of fewer than 8 values a thread each.  A launch takes fewer than 2^32
// threads along a dimension, so grids are capped and their workgroups go on to further rows (the streaming kernels': a grid along two).
// The weight gradients: a team keeps its columns' sums of dy xh and dy in registers over all the rows it takes, the teams of a
// workgroup are added in LDS, every workgroup writes ONE partial row, and a second launch adds the partial rows in a fixed order: no
// atomics, the same bits in every run.
// MEASURED (MI355X, us): 4M x 3 fp32 forward 26, backward 43; forward 8192 x 8192 bf16 46 (5.8 TB/s with the caches' help; a copy of 1 GiB: 5.1), 65536 x 256 fp32 23 (5.8); backward
// of the latter 33 (5.8) + 4.6 for the fold; 4099 x 1031 fp16 11 / 15 / 5: latency, unaligned rows; one row of 4096 3.4.  A workgroup of 1024
// threads a row took 140 at 8192 x 8192: two rows a CU in flight, two barriers each.
#include "fneus_types.h"
#include "fneus_kernels.h"

namespace fneus {

constexpr int kNormMaxGrid = 1024;       // workgroups of the backward at most
constexpr long kNormFwdGrid = 2048;      // of the forward: 8 a CU
constexpr long kNormBwdGrid = 1L << 20;  // of the backward without weight gradients, and of the fold: the launch's limit alone

// sums of v over the team, in every thread of it.  `red`: LDS floats, 2 * TPR / 64 (TPR > 64); `flip` alternates the half used, so
// one barrier a sum is enough
template <int TPR>
FN_DEV float team_sum(float v, float* red, int& flip) {
    if constexpr (TPR == 16) return row16_sum(v);
    v = wave_sum(v);
    if constexpr (TPR > 64) {
        constexpr int W = TPR / 64;
        float* r = red + flip * W;
        flip ^= 1;
        if ((threadIdx.x & 63) == 0) r[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) v += r[w];
    }
    return v;
}

template <class T, class P>
struct NormArgs {
    const T *x, *dy;
    const P *w, *b;
    T *y, *dx;
    float *mean, *rstd;
    float* partial;          // [grid][2][n]
    long ldx, ldy, lddy, lddx;
    long rows;
    int n;
    float eps;
};

// rows blockIdx, blockIdx + grid, ...: the weights stay in registers
template <class T, class P, int TPR, int EPT>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256) layer_norm_fwd_kernel(NormArgs<T, P> a) {
    constexpr int V = Chunk<T>::N, NC = EPT / V, TEAMS = TPR > 256 ? 1 : 256 / TPR;
    __shared__ float red[2 * (TPR > 64 ? TPR / 64 : 1)];
    int flip = 0;
    const int t = threadIdx.x % TPR;
    P w[NC][V], b[NC][V];                            // (in their own type: half the registers for 16 bits)
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int col = (c * TPR + t) * V;
        float q[V];
        if (a.w) load_row_run<P, V>(a.w, col, a.n, q);
#pragma unroll
        for (int k = 0; k < V; ++k) w[c][k] = a.w ? (P)q[k] : (P)1.0f;
        if (a.b) load_row_run<P, V>(a.b, col, a.n, q);
#pragma unroll
        for (int k = 0; k < V; ++k) b[c][k] = a.b ? (P)q[k] : (P)0.0f;
    }
    const float len = (float)a.n;                    // (divisions, not a reciprocal: the mean of equal values is that value)
    for (long base = (long)blockIdx.x * TEAMS; base < a.rows; base += (long)gridDim.x * TEAMS) {
        const long row = base + threadIdx.x / TPR;
        const bool live = row < a.rows;              // (TPR > 64: one team, always live: every wave meets the barriers)
        const T* __restrict__ x = a.x + (live ? row : 0) * a.ldx;
        float v[NC][V];
        float s = 0.0f;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            load_row<T>(x, (c * TPR + t) * V, a.n, v[c]);
        }
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int k = 0; k < V; ++k) s += v[c][k];
        const float mu = team_sum<TPR>(s, red, flip) / len;
        float q = 0.0f;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int left = a.n - (c * TPR + t) * V;
#pragma unroll
            for (int k = 0; k < V; ++k) {
                v[c][k] -= mu;
                q += k < left ? v[c][k] * v[c][k] : 0.0f;
            }
        }
        const float r = 1.0f / sqrtf(team_sum<TPR>(q, red, flip) / len + a.eps);
        if (!live) continue;
        T* __restrict__ y = a.y + row * a.ldy;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int col = (c * TPR + t) * V, left = a.n - col;
            if (left <= 0) break;
            float o[V];
#pragma unroll
            for (int k = 0; k < V; ++k) o[k] = v[c][k] * r * (float)w[c][k] + (float)b[c][k];
            store_chunk<T>(y + col, left, o);
        }
        if (t == 0) {
            a.mean[row] = mu;
            a.rstd[row] = r;
        }
    }
}

// Rows of fewer than 8 values: a thread a row (a row is a few bytes, less than one chunk), rows blockIdx * 256 + thread, then a grid's further
constexpr int kThin = 8;
template <class T>
FN_DEV void load_thin(const T* p, int n, float (&v)[kThin - 1]) {
    T q[kThin - 1];
#pragma unroll
    for (int k = 0; k < kThin - 1; ++k) q[k] = p[k < n ? k : n - 1];
#pragma unroll
    for (int k = 0; k < kThin - 1; ++k) v[k] = k < n ? (float)q[k] : 0.0f;
}
template <class T, class P>
__global__ void __launch_bounds__(256) layer_norm_fwd_thin_kernel(NormArgs<T, P> a) {
    float w[kThin - 1], b[kThin - 1];
#pragma unroll
    for (int k = 0; k < kThin - 1; ++k) {
        w[k] = a.w && k < a.n ? (float)a.w[k] : 1.0f;
        b[k] = a.b && k < a.n ? (float)a.b[k] : 0.0f;
    }
    const float len = (float)a.n;
    for (long row = (long)blockIdx.x * 256 + threadIdx.x; row < a.rows; row += (long)gridDim.x * 256) {
        float v[kThin - 1], s = 0.0f, q = 0.0f;
        load_thin<T>(a.x + row * a.ldx, a.n, v);
#pragma unroll
        for (int k = 0; k < kThin - 1; ++k) s += v[k];
        const float mu = s / len;
#pragma unroll
        for (int k = 0; k < kThin - 1; ++k) {
            v[k] -= mu;
            q += k < a.n ? v[k] * v[k] : 0.0f;
        }
        const float r = 1.0f / sqrtf(q / len + a.eps);
        T* y = a.y + row * a.ldy;
#pragma unroll
        for (int k = 0; k < kThin - 1; ++k)
            if (k < a.n) y[k] = (T)(v[k] * r * w[k] + b[k]);
        a.mean[row] = mu;
        a.rstd[row] = r;
    }
}

// dx, and with PARAMS this workgroup's partial row of (dw, db): a thread's sums over its rows, the wave's, the four waves' in order
template <class T, class P, bool PARAMS>
__global__ void __launch_bounds__(256) layer_norm_bwd_thin_kernel(NormArgs<T, P> a) {
    float w[kThin - 1], sum[2][kThin - 1];
#pragma unroll
    for (int k = 0; k < kThin - 1; ++k) {
        w[k] = a.w && k < a.n ? (float)a.w[k] : 1.0f;
        sum[0][k] = sum[1][k] = 0.0f;
    }
    const float inv_n = 1.0f / (float)a.n;
    for (long row = (long)blockIdx.x * 256 + threadIdx.x; row < a.rows; row += (long)gridDim.x * 256) {
        float h[kThin - 1], g[kThin - 1], s1 = 0.0f, s2 = 0.0f;
        load_thin<T>(a.x + row * a.ldx, a.n, h);
        load_thin<T>(a.dy + row * a.lddy, a.n, g);
        const float mu = a.mean[row], r = a.rstd[row];
#pragma unroll
        for (int k = 0; k < kThin - 1; ++k) {
            h[k] = k < a.n ? (h[k] - mu) * r : 0.0f;
            if constexpr (PARAMS) {
                sum[0][k] += g[k] * h[k];
                sum[1][k] += g[k];
            }
            g[k] *= w[k];
            s1 += g[k];
            s2 += g[k] * h[k];
        }
        s1 *= inv_n;
        s2 *= inv_n;
        T* dx = a.dx + row * a.lddx;
#pragma unroll
        for (int k = 0; k < kThin - 1; ++k)
            if (k < a.n) dx[k] = (T)(r * (g[k] - s1 - h[k] * s2));
    }
    if constexpr (PARAMS) {
        __shared__ float red[4][2][kThin];
#pragma unroll
        for (int which = 0; which < 2; ++which)
#pragma unroll
            for (int k = 0; k < kThin - 1; ++k) {
                const float s = wave_sum(sum[which][k]);
                if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6][which][k] = s;
            }
        __syncthreads();
        const int which = threadIdx.x / kThin, k = threadIdx.x % kThin;
        if (which < 2 && k < a.n)
            a.partial[((long)blockIdx.x * 2 + which) * a.n + k] = red[0][which][k] + red[1][which][k] + red[2][which][k] + red[3][which][k];
    }
}

// rows wider than a team's registers: a workgroup a row, three passes (the second and third from the caches).  (Workgroups that go on to
// further rows: 442 us against 374 at 8192 x 20000 bf16.)
template <class T, class P>
__global__ void __launch_bounds__(1024) layer_norm_fwd_stream_kernel(NormArgs<T, P> a) {
    constexpr int V = Chunk<T>::N;
    __shared__ float red[32];
    int flip = 0;
    const long row = wide_block();
    if (row >= a.rows) return;
    const T* x = a.x + row * a.ldx;
    const float len = (float)a.n;
    float s = 0.0f, v[V];
    for (long col = (long)threadIdx.x * V; col < a.n; col += 1024 * V) {
        load_chunk<T>(x + col, (int)(a.n - col), v);
#pragma unroll
        for (int k = 0; k < V; ++k) s += v[k];
    }
    const float mu = team_sum<1024>(s, red, flip) / len;
    float q = 0.0f;
    for (long col = (long)threadIdx.x * V; col < a.n; col += 1024 * V) {
        const int left = (int)(a.n - col);
        load_chunk<T>(x + col, left, v);
#pragma unroll
        for (int k = 0; k < V; ++k) q += k < left ? (v[k] - mu) * (v[k] - mu) : 0.0f;
    }
    const float r = 1.0f / sqrtf(team_sum<1024>(q, red, flip) / len + a.eps);
    for (long col = (long)threadIdx.x * V; col < a.n; col += 1024 * V) {
        const int left = (int)(a.n - col);
        load_chunk<T>(x + col, left, v);
#pragma unroll
        for (int k = 0; k < V; ++k)
            if (k < left) v[k] = (v[k] - mu) * r * (a.w ? (float)a.w[col + k] : 1.0f) + (a.b ? (float)a.b[col + k] : 0.0f);
        store_chunk<T>(a.y + row * a.ldy + col, left, v);
    }
    if (threadIdx.x == 0) {
        a.mean[row] = mu;
        a.rstd[row] = r;
    }
}

// dx of the rows blockIdx, blockIdx + grid, ... and, PARAMS, this workgroup's partial row of (dw, db)
template <class T, class P, int TPR, int EPT, bool PARAMS>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256) layer_norm_bwd_kernel(NormArgs<T, P> a) {
    constexpr int V = Chunk<T>::N, NC = EPT / V, TEAMS = TPR > 256 ? 1 : 256 / TPR;
    __shared__ float red[2 * (TPR > 64 ? TPR / 64 : 1)];
    __shared__ float fold[PARAMS && TEAMS > 1 ? TEAMS : 1][PARAMS && TEAMS > 1 ? TPR * EPT : 1];
    int flip = 0;
    const int t = threadIdx.x % TPR, team = threadIdx.x / TPR;
    float w[NC][V], dw[NC][V], db[NC][V];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int col = (c * TPR + t) * V;
        if (a.w) load_row_run<P, V>(a.w, col, a.n, w[c]);
#pragma unroll
        for (int k = 0; k < V; ++k) {
            if (!a.w) w[c][k] = 1.0f;
            dw[c][k] = 0.0f;
            db[c][k] = 0.0f;
        }
    }
    const float inv_n = 1.0f / (float)a.n;
    for (long base = (long)blockIdx.x * TEAMS; base < a.rows; base += (long)gridDim.x * TEAMS) {
        const long row = base + team;
        const bool live = row < a.rows;               // (TPR > 64: one team, always live: every wave meets the barriers)
        const long at = live ? row : 0;
        const T* __restrict__ x = a.x + at * a.ldx;
        const T* __restrict__ dy = a.dy + at * a.lddy;
        float xh[NC][V], d[NC][V];
        const float mu = a.mean[at], r = live ? a.rstd[at] : 0.0f;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            load_row<T>(x, (c * TPR + t) * V, a.n, xh[c]);
            load_row<T>(dy, (c * TPR + t) * V, a.n, d[c]);
        }
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int left = live ? a.n - (c * TPR + t) * V : 0;
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float h = k < left ? (xh[c][k] - mu) * r : 0.0f;
                const float dk = k < left ? d[c][k] : 0.0f;
                if constexpr (PARAMS) {
                    dw[c][k] += dk * h;
                    db[c][k] += dk;
                }
                const float g = dk * w[c][k];
                s1 += g;
                s2 += g * h;
                xh[c][k] = h;
                d[c][k] = g;
            }
        }
        s1 = team_sum<TPR>(s1, red, flip) * inv_n;
        s2 = team_sum<TPR>(s2, red, flip) * inv_n;
        T* __restrict__ dx = a.dx + row * a.lddx;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int col = (c * TPR + t) * V, left = live ? a.n - col : 0;
            if (left <= 0) break;
            float o[V];
#pragma unroll
            for (int k = 0; k < V; ++k) o[k] = r * (d[c][k] - s1 - xh[c][k] * s2);
            store_chunk<T>(dx + col, left, o);
        }
    }
    if constexpr (PARAMS) {
        float* out = a.partial + (long)blockIdx.x * 2 * a.n;
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            if constexpr (TEAMS > 1) {
                __syncthreads();
#pragma unroll
                for (int c = 0; c < NC; ++c)
#pragma unroll
                    for (int k = 0; k < V; ++k) fold[team][(c * TPR + t) * V + k] = which ? db[c][k] : dw[c][k];
                __syncthreads();
                for (int col = threadIdx.x; col < a.n; col += 256) {
                    float s = 0.0f;
#pragma unroll
                    for (int m = 0; m < TEAMS; ++m) s += fold[m][col];
                    out[which * (long)a.n + col] = s;
                }
            } else {
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    const int col = (c * TPR + t) * V;
#pragma unroll
                    for (int k = 0; k < V; ++k)
                        if (col + k < a.n) out[which * (long)a.n + col + k] = which ? db[c][k] : dw[c][k];
                }
            }
        }
    }
}

template <class T, class P>
__global__ void __launch_bounds__(1024) layer_norm_bwd_stream_kernel(NormArgs<T, P> a) {
    constexpr int V = Chunk<T>::N;
    __shared__ float red[32];
    int flip = 0;
    const long row = wide_block();
    if (row >= a.rows) return;
    const T *x = a.x + row * a.ldx, *dy = a.dy + row * a.lddy;
    const float mu = a.mean[row], r = a.rstd[row], inv_n = 1.0f / (float)a.n;
    float s1 = 0.0f, s2 = 0.0f, v[V], d[V];
    for (long col = (long)threadIdx.x * V; col < a.n; col += 1024 * V) {
        const int left = (int)(a.n - col);
        load_chunk<T>(x + col, left, v);
        load_chunk<T>(dy + col, left, d);
#pragma unroll
        for (int k = 0; k < V; ++k)
            if (k < left) {
                const float g = d[k] * (a.w ? (float)a.w[col + k] : 1.0f);
                s1 += g;
                s2 += g * (v[k] - mu) * r;
            }
    }
    s1 = team_sum<1024>(s1, red, flip) * inv_n;
    s2 = team_sum<1024>(s2, red, flip) * inv_n;
    for (long col = (long)threadIdx.x * V; col < a.n; col += 1024 * V) {
        const int left = (int)(a.n - col);
        load_chunk<T>(x + col, left, v);
        load_chunk<T>(dy + col, left, d);
#pragma unroll
        for (int k = 0; k < V; ++k)
            if (k < left) v[k] = r * (d[k] * (a.w ? (float)a.w[col + k] : 1.0f) - s1 - (v[k] - mu) * r * s2);
        store_chunk<T>(a.dx + row * a.lddx + col, left, v);
    }
}

// the streaming form's partial rows: a thread a column, the rows blockIdx.y, blockIdx.y + gridDim.y, ...
template <class T, class P>
__global__ void __launch_bounds__(256) layer_norm_params_kernel(NormArgs<T, P> a) {
    const long col = (long)blockIdx.x * 256 + threadIdx.x;
    if (col >= a.n) return;
    float dw = 0.0f, db = 0.0f;
    for (long row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const float d = (float)a.dy[row * a.lddy + col];
        dw += d * (((float)a.x[row * a.ldx + col] - a.mean[row]) * a.rstd[row]);
        db += d;
    }
    float* out = a.partial + (long)blockIdx.y * 2 * a.n;
    out[col] = dw;
    out[a.n + col] = db;
}

// dw, db = the sums of the partial rows
template <class P>
__global__ void __launch_bounds__(1024) layer_norm_fold_kernel(const float* __restrict__ partial, int parts, int n, P* __restrict__ dw,
                                                               P* __restrict__ db) {
    __shared__ float red[128][9];
    for (long col0 = 8L * blockIdx.x; col0 < 2L * n; col0 += 8L * gridDim.x) {          // of the 2 n columns
        const long col = col0 + threadIdx.x;
        const float s = fold_rows8(partial, parts, 2L * n, col0, 2L * n, red);
        if (threadIdx.x < 8 && col < 2L * n) {
            if (col < n) {
                if (dw) dw[col] = (P)s;
            } else if (db) {
                db[col - n] = (P)s;
            }
        }
        __syncthreads();                 // (the next columns' sums go to the same cells)
    }
}

struct NormShape { int tpr, ept; };      // tpr 0: streaming, 1: a thread a row

// The narrowest team whose threads hold the row in at most 32 values each (the backward keeps five registers a value); 16 threads up to
// 256 values (sums by DPP, four rows a wave), one wave up to 2048 (no barrier), four and eight waves up to 8192 and 16384
static NormShape norm_shape(int n) {
    if (n < kThin) return {1, 0};         // (a chunk does not fit the row)
    if (n <= 256) return {16, 16};
    if (n <= 2048) return {64, 8 * ((n + 511) / 512)};
    if (n <= 8192) return {256, 8 * ((n + 2047) / 2048)};
    if (n <= 16384) return {512, 8 * ((n + 4095) / 4096)};
    return {0, 0};
}

static int norm_teams(const NormShape& s) { return s.tpr == 0 || s.tpr > 256 ? 1 : 256 / s.tpr; }

// workgroups of the backward = partial rows of the weight gradients
static int norm_grid(long rows, int n) {
    const NormShape s = norm_shape(n);
    const long need = (rows + norm_teams(s) - 1) / norm_teams(s);
    const long most = s.tpr == 0 ? 64 : (s.tpr >= 64 ? 512 : kNormMaxGrid);
    return (int)(need < most ? need : most);
}

#define FN_NORM_SHAPES(CALL) \
    switch (s.tpr * 100 + s.ept) { \
        case 1616: CALL(16, 16); break; \
        case 6408: CALL(64, 8); break; \
        case 6416: CALL(64, 16); break; \
        case 6424: CALL(64, 24); break; \
        case 6432: CALL(64, 32); break; \
        case 25616: CALL(256, 16); break; \
        case 25624: CALL(256, 24); break; \
        case 25632: CALL(256, 32); break; \
        case 51224: CALL(512, 24); break; \
        default: CALL(512, 32); break; \
    }

template <class T, class P>
static void norm_fwd_launch(const NormArgs<T, P>& a, hipStream_t stream) {
    const NormShape s = norm_shape(a.n);
    const int threads = s.tpr > 256 ? s.tpr : 256, teams = norm_teams(s);
    const long need = (a.rows + teams - 1) / teams;
    const dim3 grid((unsigned)(need < kNormFwdGrid ? need : kNormFwdGrid));
    if (s.tpr == 0) {
        hipLaunchKernelGGL((layer_norm_fwd_stream_kernel<T, P>), wide_grid(a.rows), dim3(1024), 0, stream, a);
        return;
    }
    if (s.tpr == 1) {
        hipLaunchKernelGGL((layer_norm_fwd_thin_kernel<T, P>), grid, dim3(256), 0, stream, a);
        return;
    }
#define CALL(TPR, EPT) hipLaunchKernelGGL((layer_norm_fwd_kernel<T, P, TPR, EPT>), grid, dim3(threads), 0, stream, a)
    FN_NORM_SHAPES(CALL)
#undef CALL
}

template <class T, class P>
static void norm_bwd_launch(const NormArgs<T, P>& a, P* dw, P* db, hipStream_t stream) {
    const NormShape s = norm_shape(a.n);
    const int grid = norm_grid(a.rows, a.n);
    const bool params = dw || db;
    if (s.tpr == 1) {
        if (params) hipLaunchKernelGGL((layer_norm_bwd_thin_kernel<T, P, true>), dim3((unsigned)grid), dim3(256), 0, stream, a);
        else hipLaunchKernelGGL((layer_norm_bwd_thin_kernel<T, P, false>), dim3((unsigned)grid), dim3(256), 0, stream, a);
    } else if (s.tpr == 0) {
        hipLaunchKernelGGL((layer_norm_bwd_stream_kernel<T, P>), wide_grid(a.rows), dim3(1024), 0, stream, a);
        if (params) hipLaunchKernelGGL((layer_norm_params_kernel<T, P>), dim3((unsigned)((a.n + 255) / 256), (unsigned)grid), dim3(256), 0, stream, a);
    } else {
        const int threads = s.tpr > 256 ? s.tpr : 256, teams = threads / s.tpr;
        const long need = (a.rows + teams - 1) / teams;
        const unsigned all = (unsigned)(need < kNormBwdGrid ? need : kNormBwdGrid);
        if (params) {
#define CALL(TPR, EPT) hipLaunchKernelGGL((layer_norm_bwd_kernel<T, P, TPR, EPT, true>), dim3((unsigned)grid), dim3(threads), 0, stream, a)
            FN_NORM_SHAPES(CALL)
#undef CALL
        } else {
#define CALL(TPR, EPT) hipLaunchKernelGGL((layer_norm_bwd_kernel<T, P, TPR, EPT, false>), dim3(all), dim3(threads), 0, stream, a)
            FN_NORM_SHAPES(CALL)
#undef CALL
        }
    }
    if (params) {
        const long folds = (2L * a.n + 7) / 8;
        hipLaunchKernelGGL((layer_norm_fold_kernel<P>), dim3((unsigned)(folds < kNormBwdGrid ? folds : kNormBwdGrid)), dim3(1024), 0, stream, a.partial,
                           grid, a.n, dw, db);
    }
}

static int norm_check(const char* what, const void* x, const void* out, const void* mean, const void* rstd, long rows, int n, int dtype,
                      int wtype, long ld0, long ld1) {
    if (rows < 0 || n <= 0 || rows > 0x7fffffffL) { set_last_error(what); return -2; }
    if (dtype < 0 || dtype > 2 || (wtype != dtype && wtype != DT_F32) || ld0 < n || ld1 < n) { set_last_error(what); return -2; }
    if (rows > 0 && (!x || !out || !mean || !rstd)) { set_last_error(what); return -2; }
    return 0;
}

}  // namespace fneus

using namespace fneus;

#define FN_NORM_TYPES(CALL) \
    if (dtype == DT_F32) CALL(float, float) \
    else if (dtype == DT_BF16 && wtype == DT_BF16) CALL(__bf16, __bf16) \
    else if (dtype == DT_BF16) CALL(__bf16, float) \
    else if (wtype == DT_F16) CALL(_Float16, _Float16) \
    else CALL(_Float16, float)

extern "C" int fneus_layer_norm_fwd(const void* x, long ldx, const void* weight, const void* bias, void* y, long ldy, float* mean,
                                    float* rstd, long rows, int n, float eps, int dtype, int wtype, fneus_stream_t stream_) {
    hipStream_t stream = (hipStream_t)stream_;
    fneus::clear_status();
    if (int rc = norm_check("fneus_layer_norm_fwd: 0 <= rows < 2^31, n > 0, row strides >= n, dtype 0..2, weights of the same type or fp32, x, y, "
                            "mean and rstd given", x, y, mean, rstd, rows, n, dtype, wtype, ldx, ldy)) return rc;
    if (rows == 0) return 0;
#define CALL(T, P) { NormArgs<T, P> a{}; a.x = (const T*)x; a.w = (const P*)weight; a.b = (const P*)bias; a.y = (T*)y; a.mean = mean; \
        a.rstd = rstd; a.ldx = ldx; a.ldy = ldy; a.rows = rows; a.n = n; a.eps = eps; norm_fwd_launch<T, P>(a, stream); }
    FN_NORM_TYPES(CALL)
#undef CALL
    return fneus::launch_status();
}

extern "C" long fneus_layer_norm_bwd_scratch_floats(long rows, int n) {
    if (rows <= 0 || n <= 0) return 0;
    return (long)norm_grid(rows, n) * 2 * n;
}

extern "C" int fneus_layer_norm_bwd(const void* dy, long lddy, const void* x, long ldx, const void* weight, const float* mean,
                                    const float* rstd, void* dx, long lddx, void* dweight, void* dbias, float* scratch, long rows,
                                    int n, int dtype, int wtype, fneus_stream_t stream_) {
    hipStream_t stream = (hipStream_t)stream_;
    fneus::clear_status();
    const char* what = "fneus_layer_norm_bwd: 0 < rows < 2^31, n > 0, row strides >= n, dtype 0..2, weights of the same type or fp32, dy, x, mean, "
                       "rstd, dx (and scratch for the weight gradients) given";
    if (int rc = norm_check(what, x, dx, mean, rstd, rows, n, dtype, wtype, ldx, lddx)) return rc;
    if (lddy < n || rows == 0 || !dy || ((dweight || dbias) && !scratch)) { fneus::set_last_error(what); return -2; }
#define CALL(T, P) { NormArgs<T, P> a{}; a.x = (const T*)x; a.dy = (const T*)dy; a.w = (const P*)weight; a.dx = (T*)dx; \
        a.mean = const_cast<float*>(mean); a.rstd = const_cast<float*>(rstd); a.partial = scratch; a.ldx = ldx; a.lddy = lddy; \
        a.lddx = lddx; a.rows = rows; a.n = n; norm_bwd_launch<T, P>(a, (P*)dweight, (P*)dbias, stream); }
    FN_NORM_TYPES(CALL)
#undef CALL
    return fneus::launch_status();
}
