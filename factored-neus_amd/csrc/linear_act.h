// Activations of the linear layer's epilogue and their derivatives, in fp32 (linear_kernels.hip).
// Codes: 0 none, 1 ReLU, 2 LeakyReLU(0.2), 3 sigmoid (fneus_mlp_*'s), 4 softplus(beta 100) (the SDF network's), 5 GELU (erf), 6 SiLU.
#pragma once
#include "fneus_types.h"

namespace fneus {

constexpr int kLinActs = 7;

// exp by the base-2 instruction, 1 / x by the reciprocal instruction (1 ulp each): sigmoid to 1e-7 absolute (its largest values lie next to 1, where an
// ulp is 6e-8)
FN_DEV float lin_exp(float x) { return fast_exp2(x * kLog2e); }
FN_DEV float lin_sigmoid(float z) { return fast_rcp(1.0f + lin_exp(-z)); }

// Phi(z), the normal distribution's integral, and e = exp(-z^2 / 2).  With x = |z| / sqrt 2 the tail is e erfcx(x) / 2, erfcx(x) = exp(x^2) erfc(x)
// as t P(t), t = 1 / (1 + x / 2): P of degree 8, the minimax fit of the RELATIVE error over x <= 9.5 (4e-8; e is 0 beyond), so that the small
// side keeps its digits: z^2 x 2e-7 relative from the exponential's argument, 1e-6 from the rest (a fit of erfc's absolute error, 1.5e-7, left 5e-4
// of the value at z = -4).
FN_DEV float lin_phi(float z, float& e) {
    const float x = fabsf(z) * 0.70710678118654752f;
    e = lin_exp(-x * x);
    const float t = fast_rcp(1.0f + 0.5f * x);
    float p = -0.0588905998f;
    p = p * t + 0.283701122f;
    p = p * t - 0.485381961f;
    p = p * t + 0.275976181f;
    p = p * t - 0.0251763277f;
    p = p * t + 0.202069268f;
    p = p * t + 0.243261144f;
    p = p * t + 0.282353461f;
    p = p * t + 0.282087684f;
    const float tail = 0.5f * (p * t) * e;
    return z < 0.0f ? tail : 1.0f - tail;
}

FN_DEV float lin_act(float z, int act) {
    switch (act) {
        case 1: return z > 0.0f ? z : (z != z ? z : 0.0f);
        case 2: return z > 0.0f ? z : 0.2f * z;
        case 3: return lin_sigmoid(z);
        case 4: {
            const float e = lin_exp(-100.0f * fabsf(z));
            const float l = e < 0.01f ? e * (1.0f - e * (0.5f - e * 0.33333333f)) : fast_log2(1.0f + e) * kLn2;
            return (z > 0.0f ? z : (z != z ? z : 0.0f)) + l * 0.01f;
        }
        case 5: { float e; return z * lin_phi(z, e); }
        case 6: return z * lin_sigmoid(z);
        default: return z;
    }
}

// the same by CLASS of codes, for a kernel that holds one class's instructions only: 0 the piecewise linear ones (none, ReLU, leaky: `slope`
// of the negative side), 3 sigmoid and SiLU (`times`: times z), 4 softplus, 5 GELU
__host__ __device__ constexpr int lin_class(int act) { return act <= 2 ? 0 : (act == 6 ? 3 : act); }
template <int CLASS>
FN_DEV float lin_act_of(float z, float slope, bool times) {
    if constexpr (CLASS == 0) return z > 0.0f || z != z ? z : (slope == 0.0f ? 0.0f : slope * z);
    else if constexpr (CLASS == 3) { const float s = lin_sigmoid(z); return times ? z * s : s; }
    else return lin_act(z, CLASS);
}

FN_DEV float lin_near(float z) { return fabsf(z) > 128.0f ? 0.0f : z; }
// act'(z); at 0 the ReLUs take the slope of the negative side.  An infinite z has the limit (an fp16 z beyond 65504 is stored as infinity, its output
// may be finite): GELU's and SiLU's z times a factor that is 0 from |z| = 128 on is formed with z = 0 there, not as infinity times 0.
FN_DEV float lin_dact(float z, int act) {
    switch (act) {
        case 1: return z > 0.0f ? 1.0f : 0.0f;
        case 2: return z > 0.0f ? 1.0f : 0.2f;
        case 3: { const float s = lin_sigmoid(z); return s * (1.0f - s); }
        case 4: return lin_sigmoid(100.0f * z);
        case 5: { float e; const float p = lin_phi(z, e); return p + lin_near(z) * (0.39894228040143268f * e); }
        case 6: { const float s = lin_sigmoid(z); return s * (1.0f + lin_near(z) * (1.0f - s)); }
        default: return 1.0f;
    }
}

// Operands of the 32x32x16 / 16x16x32 matrix instructions: 8 consecutive values of the contraction a lane.  bf16 and fp16 enter as
// they are.  An fp32 value enters as THREE bf16 terms x = t0 + t1 + t2 (each the rounding of what is left: 24 bits for 2^-110 <= |x| < 3.39e38;
// below, the last terms' bits fall under bf16's smallest value, 2^-133), a product as the six term pairs down to 2^-24 of it, smallest first:
// fp32's accuracy at 6 bf16 MFMAs (16 k in 192 cycles; the fp32 MFMA takes 512).  An infinity, and a finite value that rounds above bf16's
// largest (3.39e38), has NaN as its second term, so it comes out as NaN.
template <class T> struct LinFrag;
template <> struct LinFrag<__bf16> { bf16x8 t; };
template <> struct LinFrag<_Float16> { fn_f16x8 t; };
template <> struct LinFrag<float> { bf16x8 t0, t1, t2; };

FN_DEV void lin_frag(const float (&v)[8], LinFrag<__bf16>& f) {
#pragma unroll
    for (int k = 0; k < 8; ++k) f.t[k] = (__bf16)v[k];
}
FN_DEV void lin_frag(const float (&v)[8], LinFrag<_Float16>& f) {
#pragma unroll
    for (int k = 0; k < 8; ++k) f.t[k] = (_Float16)v[k];
}
FN_DEV void lin_frag(const float (&v)[8], LinFrag<float>& f) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        f.t0[k] = (__bf16)v[k];
        const float r = v[k] - (float)f.t0[k];
        f.t1[k] = (__bf16)r;
        f.t2[k] = (__bf16)(r - (float)f.t1[k]);
    }
}

FN_DEV f32x16 lin_mfma32(const LinFrag<__bf16>& a, const LinFrag<__bf16>& b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.t, b.t, c, 0, 0, 0);
}
FN_DEV f32x16 lin_mfma32(const LinFrag<_Float16>& a, const LinFrag<_Float16>& b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a.t, b.t, c, 0, 0, 0);
}
FN_DEV f32x16 lin_mfma32(const LinFrag<float>& a, const LinFrag<float>& b, f32x16 c) {
    c = mfma32(a.t2, b.t0, c);
    c = mfma32(a.t0, b.t2, c);
    c = mfma32(a.t1, b.t1, c);
    c = mfma32(a.t1, b.t0, c);
    c = mfma32(a.t0, b.t1, c);
    return mfma32(a.t0, b.t0, c);
}
FN_DEV f32x4 lin_mfma16(const LinFrag<__bf16>& a, const LinFrag<__bf16>& b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.t, b.t, c, 0, 0, 0);
}
FN_DEV f32x4 lin_mfma16(const LinFrag<_Float16>& a, const LinFrag<_Float16>& b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a.t, b.t, c, 0, 0, 0);
}
FN_DEV f32x4 lin_mfma16(const LinFrag<float>& a, const LinFrag<float>& b, f32x4 c) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.t2, b.t0, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.t0, b.t2, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.t1, b.t1, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.t1, b.t0, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.t0, b.t1, c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.t0, b.t0, c, 0, 0, 0);
}

}  // namespace fneus
