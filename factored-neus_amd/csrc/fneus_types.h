// Element types of the operators that take fp32, bf16 and fp16 tensors (norm_kernels.hip, linear_kernels.hip, muon_kernels.hip):
// conversions, and 16-byte chunks that may start at any element.  Global loads and stores of this target need no alignment beyond the
// element's, so a row of odd length or stride takes the same wide accesses as an aligned one (the chunk types say aligned(element)).
#pragma once
#include "fneus_common.h"

namespace fneus {

enum { DT_F32 = 0, DT_BF16 = 1, DT_F16 = 2 };

typedef float f32x4_u __attribute__((ext_vector_type(4), aligned(4)));
typedef __bf16 bf16x8_u __attribute__((ext_vector_type(8), aligned(2)));
typedef _Float16 f16x8_u __attribute__((ext_vector_type(8), aligned(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

template <class T> struct Chunk;
template <> struct Chunk<float> { typedef f32x4_u type; static constexpr int N = 4; };
template <> struct Chunk<__bf16> { typedef bf16x8_u type; static constexpr int N = 8; };
template <> struct Chunk<_Float16> { typedef f16x8_u type; static constexpr int N = 8; };

// N values at p of which the first `valid` (1 .. N - 1) exist: every load is made, the last value's again beyond it, so that all are in flight
// at once (a load under a condition of its own is waited for inside it)
template <class T, int N>
FN_DEV void load_part(const T* p, int valid, float (&v)[N]) {
    T q[N];
#pragma unroll
    for (int k = 0; k < N; ++k) q[k] = p[k < valid ? k : valid - 1];
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = k < valid ? (float)q[k] : 0.0f;
}

// N values at p, of which the first `valid` exist (the others: 0)
template <class T>
FN_DEV void load_chunk(const T* p, int valid, float (&v)[Chunk<T>::N]) {
    constexpr int N = Chunk<T>::N;
    if (valid >= N) {
        const typename Chunk<T>::type c = *reinterpret_cast<const typename Chunk<T>::type*>(p);
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = (float)c[k];
    } else if (valid > 0) {
        load_part<T, N>(p, valid, v);
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = 0.0f;
    }
}

template <class T>
FN_DEV void store_chunk(T* p, int valid, const float (&v)[Chunk<T>::N]) {
    constexpr int N = Chunk<T>::N;
    if (valid >= N) {
        typename Chunk<T>::type c;
#pragma unroll
        for (int k = 0; k < N; ++k) c[k] = (T)v[k];
        *reinterpret_cast<typename Chunk<T>::type*>(p) = c;
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (k < valid) p[k] = (T)v[k];
    }
}

// four consecutive values, valid >= 1
template <class T> struct Quad;
template <> struct Quad<float> { typedef float type __attribute__((ext_vector_type(4), aligned(4))); };
template <> struct Quad<__bf16> { typedef __bf16 type __attribute__((ext_vector_type(4), aligned(2))); };
template <> struct Quad<_Float16> { typedef _Float16 type __attribute__((ext_vector_type(4), aligned(2))); };

template <class T>
FN_DEV void quad_load(const T* p, int valid, float (&v)[4]) {
    if (valid >= 4) {
        const typename Quad<T>::type q = *reinterpret_cast<const typename Quad<T>::type*>(p);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = (float)q[k];
    } else {
        load_part<T, 4>(p, valid, v);
    }
}
template <class T>
FN_DEV void quad_store(T* p, int valid, const float (&v)[4]) {
    if (valid >= 4) {
        typename Quad<T>::type q;
#pragma unroll
        for (int k = 0; k < 4; ++k) q[k] = (T)v[k];
        *reinterpret_cast<typename Quad<T>::type*>(p) = q;
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (k < valid) p[k] = (T)v[k];
    }
}

// N values of a row of n >= N at column `col`, zeros beyond it, WITHOUT a branch (so that a thread's loads are all in flight at once): the 16
// bytes that end with the row at the latest, shifted down to `col`
template <class T>
FN_DEV void load_row(const T* row, int col, int n, float (&v)[Chunk<T>::N]) {
    constexpr int N = Chunk<T>::N;
    const int start = col < n - N ? col : n - N, by = (col - start) * (int)sizeof(T) * 8;        // bits; >= 128: nothing of it exists
    typename Chunk<T>::type c = *reinterpret_cast<const typename Chunk<T>::type*>(row + start);
    if (n % N) {                                    // (the same for every thread)
        u32x4 w;
        __builtin_memcpy(&w, &c, 16);
        const unsigned long lo = ((unsigned long)w[1] << 32) | w[0], hi = ((unsigned long)w[3] << 32) | w[2];
        const unsigned long up = by < 64 ? hi >> (by & 63) : 0;
        const unsigned long dn = by < 64 ? (lo >> (by & 63)) | ((hi << 1) << (63 - (by & 63))) : (by < 128 ? hi >> (by & 63) : 0);
        w = u32x4{(unsigned)dn, (unsigned)(dn >> 32), (unsigned)up, (unsigned)(up >> 32)};
        __builtin_memcpy(&c, &w, 16);
    }
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = n % N || by == 0 ? (float)c[k] : 0.0f;
}
template <class T, int V>
FN_DEV void load_row_run(const T* row, int col, int n, float (&v)[V]) {
    constexpr int N = Chunk<T>::N;
#pragma unroll
    for (int c = 0; c < V / N; ++c) {
        float q[N];
        load_row<T>(row, col + c * N, n, q);
#pragma unroll
        for (int k = 0; k < N; ++k) v[c * N + k] = q[k];
    }
}

// Sums of `parts` rows of partial sums (row p at partial + p * stride) for the 8 columns col0 .. col0 + 7 by 1024 threads: 128 threads a
// column, then a tree in LDS: a fixed order.  The result of column c is in the threads c < 8.
FN_DEV float fold_rows8(const float* __restrict__ partial, int parts, long stride, long col0, long cols, float (&red)[128][9]) {
    const int c = threadIdx.x & 7, g = threadIdx.x >> 3;
    float s = 0.0f;
    if (col0 + c < cols) {
#pragma unroll 4
        for (int p = g; p < parts; p += 128) s += partial[p * stride + col0 + c];
    }
    red[g][c] = s;
#pragma unroll
    for (int d = 64; d; d >>= 1) {
        __syncthreads();
        if (g < d) red[g][c] += red[g + d][c];
    }
    return red[0][c];                      // (g == 0 has written it itself)
}

// sum over the 16 lanes of a DPP row, in every lane (quad permutes, half mirror, mirror: no LDS traffic)
FN_DEV float row16_sum(float v) {
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0xB1, 0xF, 0xF, true));
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x4E, 0xF, 0xF, true));
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x141, 0xF, 0xF, true));
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x140, 0xF, 0xF, true));
    return v;
}

FN_DEV float wave_sum(float v) {
    v = row16_sum(v);
    v += __shfl_xor(v, 16, 64);
    v += __shfl_xor(v, 32, 64);
    return v;
}

// A launch takes fewer than 2^32 threads along a dimension: more than kWideGrid workgroups go along two.  wide_block() is a workgroup's number,
// of which the last may lie beyond the count.
constexpr long kWideGrid = 1L << 15;
inline dim3 wide_grid(long groups) {
    return groups <= kWideGrid ? dim3((unsigned)groups) : dim3((unsigned)kWideGrid, (unsigned)((groups + kWideGrid - 1) / kWideGrid));
}
FN_DEV long wide_block() { return (long)blockIdx.y * gridDim.x + blockIdx.x; }

}  // namespace fneus
