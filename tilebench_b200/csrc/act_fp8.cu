// Activation checkpoints in 8 bits: saving (tb200_act_checkpoint_fp8), restoring (tb200_act_restore_fp8) and the
// elementwise part of the gated feed-forward block's backward pass, which reads them.  All are streaming kernels bound
// by HBM: saving moves size + 1 bytes per element, restoring 1 + size, the backward step 4 in and 4 out.
#include "act_fp8.cuh"

namespace tb200 {
namespace {

constexpr int kThreads = 256;
constexpr int kSeg = 1024;                      // columns that a warp of the staged kernels takes at a time
constexpr int kSegBlocks = kSeg / kActBlock;

template <typename T>
__device__ __forceinline__ void load8(const T* __restrict__ p, float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        const float4 a = __ldcs(reinterpret_cast<const float4*>(p)), b = __ldcs(reinterpret_cast<const float4*>(p) + 1);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
        const uint4 a = __ldcs(reinterpret_cast<const uint4*>(p));
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = ActType<T>::unpack(w[i]);
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
}

// Saving, rows on 16-byte boundaries.  Half a warp per block, 8 elements per lane; U pairs of blocks per warp are in
// flight at once.  A short last block is handled by leaving lanes out (cols is a multiple of 8).
template <typename T, int U>
__global__ void __launch_bounds__(kThreads) k_save(const T* __restrict__ x, uint8_t* __restrict__ q, float* __restrict__ scales,
                                                   uint32_t total, uint32_t nblk, int64_t cols, int64_t ldx) {
    const int lane = threadIdx.x & 31, sub = lane & 15;
    const uint32_t warps = gridDim.x * (kThreads / 32);
    const uint32_t groups = (total + 2 * U - 1) / (2 * U);
    for (uint32_t g = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); g < groups; g += warps) {
        float v[U][8];
        int64_t at[U];                          // offset of the lane's codes, -1 where it has none
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const uint32_t blk = g * (2 * U) + 2 * j + (lane >> 4);
            const uint32_t row = blk / nblk, col = (blk - row * nblk) * kActBlock + sub * 8;
            at[j] = blk < total && col < cols ? static_cast<int64_t>(row) * cols + col : -1;
            if (at[j] >= 0) {
                load8(x + static_cast<int64_t>(row) * ldx + col, v[j]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[j][i] = 0.0f;
            }
        }
#pragma unroll
        for (int j = 0; j < U; ++j) {
            float amax = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) amax = fmaxf(amax, act_size(v[j][i]));
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
            const float2 s = act_scale(amax);
            if (at[j] >= 0) {
                uint2 o;
                o.x = act_codes4(v[j][0], v[j][1], v[j][2], v[j][3], s.y);
                o.y = act_codes4(v[j][4], v[j][5], v[j][6], v[j][7], s.y);
                *reinterpret_cast<uint2*>(q + at[j]) = o;
                if (sub == 0) scales[g * (2 * U) + 2 * j + (lane >> 4)] = s.x;
            }
        }
    }
}

// Moves n elements between global memory at any alignment and a shared buffer that has the same address modulo 16:
// single elements up to the first 16-byte boundary and behind the last one, 16-byte pieces between.
template <typename T>
__device__ __forceinline__ T* same_offset(uint8_t* buf, const T* global) { return reinterpret_cast<T*>(buf + (reinterpret_cast<uintptr_t>(global) & 15)); }
template <typename T, typename Dst, typename Src>
__device__ __forceinline__ void copy_any(Dst* dst, const Src* src, int n, int lane) {
    constexpr int V = 16 / sizeof(T);
    const int head = min(n, static_cast<int>(((16 - (reinterpret_cast<uintptr_t>(src) & 15)) & 15) / sizeof(T)));
    const int vecs = (n - head) / V, tail0 = head + vecs * V;
    if (lane < head) dst[lane] = src[lane];
    for (int i = lane; i < vecs; i += 32) *reinterpret_cast<uint4*>(dst + head + i * V) = *reinterpret_cast<const uint4*>(src + head + i * V);
    if (tail0 + lane < n) dst[tail0 + lane] = src[tail0 + lane];
}

// Saving, any width, stride and alignment: a warp stages up to 1024 columns of a row in shared memory, so that global
// memory sees 16-byte accesses although a row may begin at any byte.
template <typename T>
__global__ void __launch_bounds__(kThreads) k_save_any(const T* __restrict__ x, uint8_t* __restrict__ q, float* __restrict__ scales,
                                                       int64_t segments, uint32_t nseg, uint32_t nblk, int64_t cols, int64_t ldx) {
    __shared__ __align__(16) uint8_t xs[kThreads / 32][kSeg * sizeof(T) + 16];
    __shared__ __align__(16) uint8_t qs[kThreads / 32][kSeg + 16];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int64_t s = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + warp; s < segments; s += static_cast<int64_t>(gridDim.x) * (kThreads / 32)) {
        const int64_t row = s / nseg;
        const int64_t col = (s - row * nseg) * kSeg;
        const int n = static_cast<int>(min(static_cast<int64_t>(kSeg), cols - col));
        const T* src = x + row * ldx + col;
        uint8_t* dst = q + row * cols + col;
        T* xb = same_offset(xs[warp], src);
        uint8_t* qb = same_offset(qs[warp], dst);
        copy_any<T>(xb, src, n, lane);
        __syncwarp();
#pragma unroll 2
        for (int b = 0; b * kActBlock < n; ++b) {
            float v[4], amax = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int i = b * kActBlock + j * 32 + lane;
                v[j] = i < n ? ActType<T>::load(xb[i]) : 0.0f;
                amax = fmaxf(amax, act_size(v[j]));
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
            const float2 sc = act_scale(amax);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int i = b * kActBlock + j * 32 + lane;
                if (i < n) qb[i] = static_cast<uint8_t>(act_codes2(act_scaled(v[j], sc.y), 0.0f) & 0xFFu);
            }
            if (lane == 0) scales[row * nblk + col / kActBlock + b] = sc.x;
        }
        __syncwarp();
        copy_any<uint8_t>(dst, qb, n, lane);
        __syncwarp();
    }
}

// 16 codes -> 16 values of T, 16-byte stores
template <typename T>
__device__ __forceinline__ void restore16(T* __restrict__ out, const uint4& c, float s) {
    const uint32_t w[4] = {c.x, c.y, c.z, c.w};
    float v[16];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 a = act_values2(w[i] & 0xFFFFu), b = act_values2(w[i] >> 16);
        v[4 * i] = act_restored(a.x, s, ActType<T>::kTop);
        v[4 * i + 1] = act_restored(a.y, s, ActType<T>::kTop);
        v[4 * i + 2] = act_restored(b.x, s, ActType<T>::kTop);
        v[4 * i + 3] = act_restored(b.y, s, ActType<T>::kTop);
    }
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) reinterpret_cast<float4*>(out)[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            reinterpret_cast<uint4*>(out)[i] = make_uint4(ActType<T>::pack(v[8 * i], v[8 * i + 1]), ActType<T>::pack(v[8 * i + 2], v[8 * i + 3]),
                                                          ActType<T>::pack(v[8 * i + 4], v[8 * i + 5]), ActType<T>::pack(v[8 * i + 6], v[8 * i + 7]));
    }
}

// Restoring, widths that are multiples of 16: 16 codes per lane, U independent loads in flight.
template <typename T, int U>
__global__ void __launch_bounds__(kThreads) k_restore(const uint4* __restrict__ q, const float* __restrict__ scales, T* __restrict__ out,
                                                      int64_t total, uint32_t per_row, uint32_t nblk) {
    const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads;
    for (int64_t i0 = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i0 < total; i0 += U * step) {
        uint4 c[U];
        float s[U];
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int64_t i = i0 + j * step;
            if (i < total) {
                c[j] = __ldcs(q + i);
                const int64_t row = i / per_row;
                s[j] = __ldg(scales + row * nblk + static_cast<uint32_t>(i - row * per_row) / 8);
            }
        }
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int64_t i = i0 + j * step;
            if (i < total) restore16(out + 16 * i, c[j], s[j]);
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) k_restore_any(const uint8_t* __restrict__ q, const float* __restrict__ scales, T* __restrict__ out,
                                                          int64_t segments, uint32_t nseg, uint32_t nblk, int64_t cols) {
    __shared__ __align__(16) uint8_t ys[kThreads / 32][kSeg * sizeof(T) + 16];
    __shared__ __align__(16) uint8_t qs[kThreads / 32][kSeg + 16];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int64_t s = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + warp; s < segments; s += static_cast<int64_t>(gridDim.x) * (kThreads / 32)) {
        const int64_t row = s / nseg;
        const int64_t col = (s - row * nseg) * kSeg;
        const int n = static_cast<int>(min(static_cast<int64_t>(kSeg), cols - col));
        const uint8_t* src = q + row * cols + col;
        T* dst = out + row * cols + col;
        uint8_t* qb = same_offset(qs[warp], src);
        T* yb = same_offset(ys[warp], dst);
        copy_any<uint8_t>(qb, src, n, lane);
        __syncwarp();
        for (int b = 0; b * kActBlock < n; ++b) {
            const float sc = __ldg(scales + row * nblk + col / kActBlock + b);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int i = b * kActBlock + j * 32 + lane;
                if (i < n) yb[i] = ActType<T>::store(act_restored(act_values2(qb[i]).x, sc, ActType<T>::kTop));
            }
        }
        __syncwarp();
        copy_any<T>(dst, yb, n, lane);
        __syncwarp();
    }
}

// dg = dh * u * f'(g), du = dh * f(g); 8 elements per thread, rows of multiples of 8.
template <typename T, int ACT>
__global__ void __launch_bounds__(kThreads) k_gated_bwd(const uint4* __restrict__ dh, const uint2* __restrict__ gq, const float* __restrict__ gs,
                                                        const uint2* __restrict__ uq, const float* __restrict__ us, uint4* __restrict__ dg,
                                                        uint4* __restrict__ du, int64_t total, uint32_t per_row, uint32_t nblk) {
    const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < total; i += step) {
        const int64_t row = i / per_row;
        const int64_t blk = row * nblk + static_cast<uint32_t>(i - row * per_row) / 16;
        const uint4 d = __ldcs(dh + i);
        const uint2 cg = __ldcs(gq + i), cu = __ldcs(uq + i);
        const float sg = __ldg(gs + blk), su = __ldg(us + blk);
        const uint32_t dw[4] = {d.x, d.y, d.z, d.w};
        uint32_t og[4], ou[4];
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            const uint32_t hg = (p < 2 ? cg.x : cg.y) >> (16 * (p & 1)) & 0xFFFFu, hu = (p < 2 ? cu.x : cu.y) >> (16 * (p & 1)) & 0xFFFFu;
            const float2 g = act_values2(hg), u = act_values2(hu), e = ActType<T>::unpack(dw[p]);
            const float2 a = gate_both<ACT>(act_restored(g.x, sg, FLT_MAX)), b = gate_both<ACT>(act_restored(g.y, sg, FLT_MAX));
            og[p] = ActType<T>::pack(e.x * act_restored(u.x, su, FLT_MAX) * a.y, e.y * act_restored(u.y, su, FLT_MAX) * b.y);
            ou[p] = ActType<T>::pack(e.x * a.x, e.y * b.x);
        }
        dg[i] = make_uint4(og[0], og[1], og[2], og[3]);
        du[i] = make_uint4(ou[0], ou[1], ou[2], ou[3]);
    }
}

// The same for any width: single elements, neighbouring lanes on neighbouring columns.
template <typename T, int ACT>
__global__ void __launch_bounds__(kThreads) k_gated_bwd_any(const T* __restrict__ dh, const uint8_t* __restrict__ gq, const float* __restrict__ gs,
                                                            const uint8_t* __restrict__ uq, const float* __restrict__ us, T* __restrict__ dg,
                                                            T* __restrict__ du, int64_t total, int64_t f, int64_t ldg, uint32_t nblk) {
    const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < total; i += step) {
        const int64_t row = i / f, col = i - row * f, blk = row * nblk + col / kActBlock;
        const float g = act_restored(act_values2(gq[i]).x, gs[blk], FLT_MAX), u = act_restored(act_values2(uq[i]).x, us[blk], FLT_MAX);
        const float e = ActType<T>::load(dh[i]);
        const float2 a = gate_both<ACT>(g);
        dg[row * ldg + col] = ActType<T>::store(e * u * a.y);
        du[row * ldg + col] = ActType<T>::store(e * a.x);
    }
}

int capped(int64_t ctas, int per_sm) {
    const int64_t cap = static_cast<int64_t>(num_sms()) * per_sm;
    return static_cast<int>(ctas < 1 ? 1 : ctas < cap ? ctas : cap);
}

template <typename T>
int launch_save(const T* x, uint8_t* q, float* scales, int64_t rows, int64_t cols, int64_t ldx, cudaStream_t st) {
    const uint32_t nblk = static_cast<uint32_t>((cols + kActBlock - 1) / kActBlock);
    const bool vec = cols % 8 == 0 && aligned16(x) && (ldx * sizeof(T)) % 16 == 0 && (reinterpret_cast<uintptr_t>(q) & 7) == 0;
    if (vec) {
        const uint32_t total = static_cast<uint32_t>(rows * nblk);
        constexpr int U = 4;
        k_save<T, U><<<capped((total + 16 * U - 1) / (16 * U), 8), kThreads, 0, st>>>(x, q, scales, total, nblk, cols, ldx);
    } else {
        const uint32_t nseg = static_cast<uint32_t>((cols + kSeg - 1) / kSeg);
        k_save_any<T><<<capped((rows * nseg + 7) / 8, 8), kThreads, 0, st>>>(x, q, scales, rows * nseg, nseg, nblk, cols, ldx);
    }
    TB200_CUDA_TRY(cudaGetLastError());
    return TB200_OK;
}

template <typename T>
int launch_restore(const uint8_t* q, const float* scales, T* out, int64_t rows, int64_t cols, cudaStream_t st) {
    const uint32_t nblk = static_cast<uint32_t>((cols + kActBlock - 1) / kActBlock);
    if (cols % 16 == 0 && aligned16(q) && aligned16(out)) {
        const int64_t total = rows * (cols / 16);
        constexpr int U = 4;
        k_restore<T, U><<<capped((total + kThreads * U - 1) / (kThreads * U), 8), kThreads, 0, st>>>(
            reinterpret_cast<const uint4*>(q), scales, out, total, static_cast<uint32_t>(cols / 16), nblk);
    } else {
        const uint32_t nseg = static_cast<uint32_t>((cols + kSeg - 1) / kSeg);
        k_restore_any<T><<<capped((rows * nseg + 7) / 8, 8), kThreads, 0, st>>>(q, scales, out, rows * nseg, nseg, nblk, cols);
    }
    TB200_CUDA_TRY(cudaGetLastError());
    return TB200_OK;
}

template <typename T, int ACT>
int launch_gated(const void* dh, const void* gq, const float* gs, const void* uq, const float* us, void* dg, void* du, int64_t m, int64_t f,
                 int64_t ldg, cudaStream_t st) {
    const uint32_t nblk = static_cast<uint32_t>((f + kActBlock - 1) / kActBlock);
    const bool vec = f % 8 == 0 && ldg == f && aligned16(dh) && (reinterpret_cast<uintptr_t>(gq) & 7) == 0 && (reinterpret_cast<uintptr_t>(uq) & 7) == 0;
    if (vec) {
        const int64_t total = m * (f / 8);
        k_gated_bwd<T, ACT><<<capped((total + kThreads - 1) / kThreads, 8), kThreads, 0, st>>>(
            static_cast<const uint4*>(dh), static_cast<const uint2*>(gq), gs, static_cast<const uint2*>(uq), us, static_cast<uint4*>(dg),
            static_cast<uint4*>(du), total, static_cast<uint32_t>(f / 8), nblk);
    } else {
        k_gated_bwd_any<T, ACT><<<capped((m * f + kThreads - 1) / kThreads, 8), kThreads, 0, st>>>(
            static_cast<const T*>(dh), static_cast<const uint8_t*>(gq), gs, static_cast<const uint8_t*>(uq), us, static_cast<T*>(dg),
            static_cast<T*>(du), m * f, f, ldg, nblk);
    }
    TB200_CUDA_TRY(cudaGetLastError());
    return TB200_OK;
}

template <typename T>
int launch_gated_act(const void* dh, const void* gq, const float* gs, const void* uq, const float* us, void* dg, void* du, int64_t m, int64_t f,
                     int64_t ldg, int act, cudaStream_t st) {
    switch (act) {
        case TB200_ACT_SILU: return launch_gated<T, TB200_ACT_SILU>(dh, gq, gs, uq, us, dg, du, m, f, ldg, st);
        case TB200_ACT_GELU: return launch_gated<T, TB200_ACT_GELU>(dh, gq, gs, uq, us, dg, du, m, f, ldg, st);
        case TB200_ACT_GELU_TANH: return launch_gated<T, TB200_ACT_GELU_TANH>(dh, gq, gs, uq, us, dg, du, m, f, ldg, st);
        default: return launch_gated<T, TB200_ACT_RELU>(dh, gq, gs, uq, us, dg, du, m, f, ldg, st);
    }
}

int check_sizes(const char* what, int64_t rows, int64_t cols) {
    if (rows < 0 || cols <= 0) return fail(TB200_ERR_ARG, "%s: rows=%lld cols=%lld (rows >= 0, cols > 0)", what, (long long)rows, (long long)cols);
    if (cols > (1ll << 31) || rows > (1ll << 40) / cols) return fail(TB200_ERR_UNSUPPORTED, "%s: rows=%lld cols=%lld is too large", what, (long long)rows, (long long)cols);
    if (rows * ((cols + kActBlock - 1) / kActBlock) > 0x7fffffffll)
        return fail(TB200_ERR_UNSUPPORTED, "%s: more than 2^31 blocks of %d", what, kActBlock);
    return TB200_OK;
}

}  // namespace

int launch_gated_act_bwd(const void* dh, const void* gq, const float* gs, const void* uq, const float* us, void* dg, void* du,
                         int64_t m, int64_t f, int64_t ldg, int act, int dtype, cudaStream_t st) {
    return dtype == TB200_DT_F16 ? launch_gated_act<__half>(dh, gq, gs, uq, us, dg, du, m, f, ldg, act, st)
                                 : launch_gated_act<__nv_bfloat16>(dh, gq, gs, uq, us, dg, du, m, f, ldg, act, st);
}

int launch_act_restore(const void* q, const float* scales, void* out, int dtype, int64_t rows, int64_t cols, cudaStream_t st) {
    const uint8_t* c = static_cast<const uint8_t*>(q);
    if (dtype == TB200_DT_F32) return launch_restore<float>(c, scales, static_cast<float*>(out), rows, cols, st);
    if (dtype == TB200_DT_F16) return launch_restore<__half>(c, scales, static_cast<__half*>(out), rows, cols, st);
    return launch_restore<__nv_bfloat16>(c, scales, static_cast<__nv_bfloat16*>(out), rows, cols, st);
}

}  // namespace tb200

using namespace tb200;

extern "C" int tb200_act_checkpoint_fp8(const void* x, void* q, float* scales, int64_t rows, int64_t cols, int64_t ldx, int dtype,
                                        void* stream) {
    clear_error();
    int rc = check_sizes("act_checkpoint_fp8", rows, cols);
    if (rc != TB200_OK) return rc;
    if (dtype != TB200_DT_F32 && dtype != TB200_DT_F16 && dtype != TB200_DT_BF16)
        return fail(TB200_ERR_UNSUPPORTED, "act_checkpoint_fp8: dtype %d is not one of F32, F16, BF16", dtype);
    if (rows == 0) return TB200_OK;
    if (!x || !q || !scales) return fail(TB200_ERR_ARG, "act_checkpoint_fp8: null pointer");
    if (rows > 1 && ldx < cols) return fail(TB200_ERR_ARG, "act_checkpoint_fp8: row stride %lld is below cols=%lld", (long long)ldx, (long long)cols);
    const int64_t size = dtype == TB200_DT_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(x) % size || reinterpret_cast<uintptr_t>(scales) & 3)
        return fail(TB200_ERR_ALIGN, "act_checkpoint_fp8: x and scales must be aligned to their elements");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    uint8_t* c = static_cast<uint8_t*>(q);
    if (dtype == TB200_DT_F32) return launch_save(static_cast<const float*>(x), c, scales, rows, cols, ldx, st);
    if (dtype == TB200_DT_F16) return launch_save(static_cast<const __half*>(x), c, scales, rows, cols, ldx, st);
    return launch_save(static_cast<const __nv_bfloat16*>(x), c, scales, rows, cols, ldx, st);
}

extern "C" int tb200_act_restore_fp8(const void* q, const float* scales, void* out, int64_t rows, int64_t cols, int dtype, void* stream) {
    clear_error();
    int rc = check_sizes("act_restore_fp8", rows, cols);
    if (rc != TB200_OK) return rc;
    if (dtype != TB200_DT_F32 && dtype != TB200_DT_F16 && dtype != TB200_DT_BF16)
        return fail(TB200_ERR_UNSUPPORTED, "act_restore_fp8: dtype %d is not one of F32, F16, BF16", dtype);
    if (rows == 0) return TB200_OK;
    if (!q || !scales || !out) return fail(TB200_ERR_ARG, "act_restore_fp8: null pointer");
    const int64_t size = dtype == TB200_DT_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(out) % size || reinterpret_cast<uintptr_t>(scales) & 3)
        return fail(TB200_ERR_ALIGN, "act_restore_fp8: out and scales must be aligned to their elements");
    return launch_act_restore(q, scales, out, dtype, rows, cols, static_cast<cudaStream_t>(stream));
}
