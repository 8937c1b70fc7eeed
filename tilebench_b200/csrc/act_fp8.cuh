// The 8-bit form of an activation and the gate functions of the feed-forward block, shared by the kernels that save,
// restore and use activation checkpoints.
//
// A 1 x 128 block of a row is stored as e4m3 codes and one power-of-two scale: the smallest 2^e (e >= -126) with
// amax <= 448 * 2^e.  e4m3 carries its own exponent, so a finer scale would not make a code more precise; a power of
// two makes x / s and code * s exact, so every code is the correctly rounded one whatever order the work is done in,
// and restoring to bf16 or fp32 rounds nothing.  Infinities and NaN do not enter amax and are stored as NaN.
#pragma once

#include "common.cuh"

#include <cuda_fp8.h>
#include <float.h>

namespace tb200 {

constexpr int kActBlock = 128;

#ifdef __CUDACC__

// |v|, 0 for infinities and NaN.  fmaxf passes over NaN by itself, so a block's amax is first taken as the plain
// maximum of |v|, and only a block where that is infinite is looked at again with act_size.
__device__ __forceinline__ float act_size(float v) {
    const float a = fabsf(v);
    return a <= FLT_MAX ? a : 0.0f;
}
// (scale, 1 / scale) of a block: both are powers of two within the normal range, so both are exact.
__device__ __forceinline__ float2 act_scale(float amax) {
    const uint32_t b = __float_as_uint(amax);
    int e = static_cast<int>(b >> 23) - 8 + ((b & 0x7FFFFFu) > 0x600000u ? 1 : 0);      // 448 = 1.75 * 2^8
    e = amax > 0.0f ? max(e, 1) : 127;
    return make_float2(__uint_as_float(static_cast<uint32_t>(e) << 23), __uint_as_float(static_cast<uint32_t>(254 - e) << 23));
}
// Codes of numbers times 1 / scale.  The hardware conversion makes NaN of NaN but saturates infinities, so a block that
// holds any goes through act_scaled first (finite values are at most 448 here).
__device__ __forceinline__ float act_scaled(float v, float inv) {
    const float y = v * inv;
    return fabsf(y) <= 448.0f ? y : __int_as_float(0x7FC00000);
}
__device__ __forceinline__ uint32_t act_codes2(float a, float b) {
    return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint32_t act_codes4(float a, float b, float c, float d, float inv) {
    return act_codes2(a * inv, b * inv) | (act_codes2(c * inv, d * inv) << 16);
}
__device__ __forceinline__ uint32_t act_codes4_checked(float a, float b, float c, float d, float inv) {
    return act_codes2(act_scaled(a, inv), act_scaled(b, inv)) | (act_codes2(act_scaled(c, inv), act_scaled(d, inv)) << 16);
}
__device__ __forceinline__ float2 act_values2(uint32_t codes) { // two codes in the low half, as numbers (exact)
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(codes), __NV_E4M3);
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
// code * scale, held within +-top: a block whose amax is close to the type's largest value may round up beyond it,
// which takes a scale above top / 448.
__device__ __forceinline__ bool act_may_exceed(float s, float top) { return fabsf(s) > top * (1.0f / 448.0f) * 0.999f; }
__device__ __forceinline__ float act_held(float v, float top) {
    return fabsf(v) > top ? copysignf(top, v) : v;              // NaN stays NaN
}

template <typename T> struct ActType;
template <> struct ActType<float> {
    static constexpr float kTop = FLT_MAX;
    static __device__ __forceinline__ float store(float v) { return v; }
};
template <> struct ActType<__half> {
    static constexpr float kTop = 65504.0f;
    static __device__ __forceinline__ __half store(float v) { return __float2half_rn(v); }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
};
template <> struct ActType<__nv_bfloat16> {
    static constexpr float kTop = 3.38953138925153547590470800371487866880e+38f;
    static __device__ __forceinline__ __nv_bfloat16 store(float v) { return __float2bfloat16_rn(v); }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t w) {
        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    }
};

// ---- gate functions: f(g), and f'(g) ---------------------------------------------------------------------------
// All in fp32, with the hardware's power of two and reciprocal (2^-22 and 2^-23 of the value).  exp(x) takes a power of two of
// x log2(e) rounded to 32 bits, so its error grows with |x|: 2^-20 of the value at 20, 2^-18 at 60 and beyond; still far below the
// 2^-8 (bf16) or 2^-11 (fp16) of the rounding that follows.  Results below 2^-126 come as zero, which takes |g| * 2^-126 off a
// gate's value at most.  The error-function and tanh forms are written so that nothing cancels
// for large negative g: the normal tail instead of 1 + erf, and (1 + tanh z) / 2 as the logistic function of 2 z.
__device__ __forceinline__ float fast_exp(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * 1.44269504088896340736f));
    return y;
}
__device__ __forceinline__ float fast_reciprocal(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float gate_logistic(float z) { return fast_reciprocal(1.0f + fast_exp(-z)); }

// (Phi(g), exp(-g^2 / 2)) of the normal distribution.  The tail is Phi(-|g|) = exp(-g^2 / 2) t P(t) with
// t = 1 / (1 + 0.3 |g|); P has degree 7 and was fitted here to exp(g^2 / 2) erfc(|g| / sqrt 2) / (2 t), least largest relative error
// over |g| <= 14: 1.64e-7 with the coefficients as rounded here.  In 32 bits the exponential's argument g^2 / 2 sets the error: 9e-7 of the
// value up to |g| = 4, 2.7e-6 up to 8, 7.7e-6 at 13 (the steps' own roundings, evaluated).  CUDA's erfcf in its
// place took 6.9 us of a 128 x 256 accumulator's epilogue where the whole of it takes 3.
__device__ __forceinline__ float2 gate_normal(float g) {
    const float z = fabsf(g), e = fast_exp(-0.5f * g * g), t = fast_reciprocal(fmaf(0.3f, z, 1.0f));
    float p = 0.03567477688193321f;
    p = fmaf(p, t, -0.15720310807228088f);
    p = fmaf(p, t, 0.20635353028774261f);
    p = fmaf(p, t, -0.05368367210030556f);
    p = fmaf(p, t, 0.12856164574623108f);
    p = fmaf(p, t, 0.09991348534822464f);
    p = fmaf(p, t, 0.12075395882129669f);
    p = fmaf(p, t, 0.11962930113077164f);
    const float tail = p * t * e;
    return make_float2(g < 0.0f ? tail : 1.0f - tail, e);
}

constexpr float kInvSqrt2Pi = 0.39894228040143267794f;
constexpr float kTanhA = 0.79788456080286535588f;               // sqrt(2 / pi)
constexpr float kTanhB = 0.044715f;

template <int ACT>
__device__ __forceinline__ float gate_value(float g) {
    if constexpr (ACT == TB200_ACT_SILU) {
        return g * gate_logistic(g);
    } else if constexpr (ACT == TB200_ACT_GELU) {
        return g * gate_normal(g).x;
    } else if constexpr (ACT == TB200_ACT_GELU_TANH) {
        return g * gate_logistic(2.0f * kTanhA * (g + kTanhB * g * g * g));
    } else {
        return g <= 0.0f ? 0.0f : g;                            // NaN stays NaN
    }
}
// f(g) and f'(g) together
template <int ACT>
__device__ __forceinline__ float2 gate_both(float g) {
    if constexpr (ACT == TB200_ACT_SILU) {
        const float s = gate_logistic(g);
        return make_float2(g * s, s * (1.0f + g * (1.0f - s)));
    } else if constexpr (ACT == TB200_ACT_GELU) {
        const float2 n = gate_normal(g);
        return make_float2(g * n.x, n.x + g * kInvSqrt2Pi * n.y);
    } else if constexpr (ACT == TB200_ACT_GELU_TANH) {
        const float s = gate_logistic(2.0f * kTanhA * (g + kTanhB * g * g * g));
        // s (1 - s) is 0 long before g^2 leaves fp32's range, and has to stay 0 there
        return make_float2(g * s, s + 2.0f * kTanhA * (s * (1.0f - s)) * g * (1.0f + 3.0f * kTanhB * fminf(g * g, 1e30f)));
    } else {
        return make_float2(g <= 0.0f ? 0.0f : g, g > 0.0f ? 1.0f : 0.0f);
    }
}
#endif  // __CUDACC__

// ---- launches that overlap their set-up with the end of the kernel before ----------------------------------------
// Every kernel of the block lets the next one of its stream begin once all its CTAs have (let_next_begin), and the matrix
// products are launched so that they may: their launch, barriers, tensor memory and tensor maps overlap with the end of
// the kernel before, and they wait for it to be complete (wait_for_previous) before they touch global memory.  So are the two
// kernels that make fp16's power of two and use it.  The others, which stream, begin when the kernel before has ended (some 2 us later): they read
// through the read-only path, which is for what nothing writes while the kernel is there, be it before it waits.  With ordinary loads
// behind the wait they could overlap as well; that is not done.
#ifdef __CUDACC__
__device__ __forceinline__ void let_next_begin() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
template <typename Args, typename Maps>
int launch_over_previous(void (*kern)(Maps, Args), int grid, int block, int smem, int cluster, cudaStream_t st, const Maps& maps, const Args& args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(grid), 1, 1);
    cfg.blockDim = dim3(static_cast<unsigned>(block), 1, 1);
    cfg.dynamicSmemBytes = static_cast<size_t>(smem);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    TB200_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, maps, args));
    return TB200_OK;
}
#endif

// ---- launchers shared between the files of the feed-forward block ----------------------------------------------
// dg and du lie in rows of whole 128-byte lines: a copy of 128 bytes that begins elsewhere moves a fifth sector (12756 rows of
// 1264 x 19937: 2547 us with rows of 39888 bytes, 2282 so).
//
// In fp16 they are held times a power of two, the same for all of them: dh times projections may be far below fp16's normal numbers
// (with dh of 1e-6 half of the bits of the weights' gradients were lost, which are normal numbers themselves) or above its largest.  The
// power brings the bound max|dh| * 512 * max(scale of g or u) to between 2^13 and 2^15 (|u| <= 448 s, |f(g)| <= |g|, |f'| <= 1.13, and
// 448 * 1.13 < 512), over the finite values; what is within 2^-27 of the bound keeps all of its bits.  Products carry it exactly, and
// the factor that takes it off again is applied to their 32-bit sums.  That factor lies in the last four bytes of dg's first row; behind du's rows lie the
// maxima that it comes from.  So an fp16 row has room for four bytes behind its last whole piece of 8 numbers.
constexpr int64_t grad_pitch(int64_t f, int dtype) {
    return ((dtype == TB200_DT_F16 ? (f + 7) / 8 * 8 + 2 : f) + 63) / 64 * 64;
}
template <typename P>
P* behind_row(void* grads, int64_t ldg) { return reinterpret_cast<P*>(static_cast<uint8_t*>(grads) + 2 * ldg - sizeof(P)); }

// The backward pass's two intermediates, dg = dh * u * f'(g) and du = dh * f(g) with row pitch ldg = grad_pitch(f, dtype), in fp16 times
// a power of two whose inverse is left at behind_row<float>(dg, ldg); and, where xq is given, the
// block's input [m, k] restored from its 8-bit form with row pitch ldx (k and ldx multiples of 8; ldx = k unless xq lies on an 8-byte
// boundary).
int launch_gated_act_bwd(const void* dh, const void* gq, const float* gs, const void* uq, const float* us, void* dg, void* du,
                         int64_t m, int64_t f, int64_t ldg, const void* xq, const float* xs, void* x, int64_t k, int64_t ldx, int act, int dtype,
                         cudaStream_t st);

}  // namespace tb200
