// Activation checkpoints in 8 bits: saving (tb200_act_checkpoint_fp8), restoring (tb200_act_restore_fp8) and the
// elementwise part of the gated feed-forward block's backward pass, which reads them.  All are streaming kernels bound
// by HBM: saving moves size + 1 bytes per element, restoring 1 + size, the backward step 4 in and 4 out.
#include "act_fp8.cuh"

namespace tb200 {
namespace {

constexpr int kThreads = 256;
template <typename T> constexpr bool kRanged = ActType<T>::kTop < 1e5f;      // fp16, whose dg and du are held times a power of two

__device__ __forceinline__ void load_once(const void* p, uint32_t (&r)[8]) {     // 32 bytes, read once
    asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "l"(p));
}
// 32 bytes on a boundary of 16, the second half only where it is there; the halves share a sector, which L1 keeps between them
__device__ __forceinline__ void load_halves(const void* p, bool both, uint32_t (&r)[8]) {
    const uint4 a = __ldg(static_cast<const uint4*>(p)), b = both ? __ldg(static_cast<const uint4*>(p) + 1) : make_uint4(0, 0, 0, 0);
    r[0] = a.x; r[1] = a.y; r[2] = a.z; r[3] = a.w;
    r[4] = b.x; r[5] = b.y; r[6] = b.z; r[7] = b.w;
}
__device__ __forceinline__ void store_piece(void* p, const uint32_t (&r)[4]) { *static_cast<uint4*>(p) = make_uint4(r[0], r[1], r[2], r[3]); }
__device__ __forceinline__ void store_piece(void* p, const uint32_t (&r)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]),
                 "r"(r[6]), "r"(r[7]) : "memory");
}

// N words of memory <-> the 4 N / sizeof(T) numbers that they hold
template <typename T, int N>
__device__ __forceinline__ void numbers(const uint32_t (&w)[N], float (&v)[4 * N / sizeof(T)]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if constexpr (sizeof(T) == 4) {
            v[i] = __uint_as_float(w[i]);
        } else {
            const float2 f = ActType<T>::unpack(w[i]);
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
}
template <typename T, int N>
__device__ __forceinline__ void words(const float (&v)[4 * N / sizeof(T)], uint32_t (&w)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(v[i]);
        else w[i] = ActType<T>::pack(v[2 * i], v[2 * i + 1]);
    }
}
// The scale of a block whose E numbers per lane lie in 128 / E neighbouring lanes, and the lane's codes.
template <int E>
__device__ __forceinline__ float encode(const float (&v)[E], uint32_t (&codes)[E / 4]) {
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) amax = fmaxf(amax, fabsf(v[i]));
#pragma unroll
    for (int o = kActBlock / E / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    const bool infinite = amax > FLT_MAX;                        // the same in all lanes of the block
    if (__any_sync(0xffffffffu, infinite)) {
        float size = 0.0f;
#pragma unroll
        for (int i = 0; i < E; ++i) size = fmaxf(size, act_size(v[i]));
#pragma unroll
        for (int o = kActBlock / E / 2; o > 0; o >>= 1) size = fmaxf(size, __shfl_xor_sync(0xffffffffu, size, o));
        amax = size;
    }
    const float2 s = act_scale(amax);
    if (infinite) {
#pragma unroll
        for (int i = 0; i < E / 4; ++i) codes[i] = act_codes4_checked(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3], s.y);
    } else {
#pragma unroll
        for (int i = 0; i < E / 4; ++i) codes[i] = act_codes4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3], s.y);
    }
    return s.x;
}
template <int E>
__device__ __forceinline__ void decode(const uint32_t (&codes)[E / 4], float s, float top, float (&v)[E]) {
#pragma unroll
    for (int i = 0; i < E / 4; ++i) {
        const float2 a = act_values2(codes[i] & 0xFFFFu), b = act_values2(codes[i] >> 16);
        v[4 * i] = a.x * s;
        v[4 * i + 1] = a.y * s;
        v[4 * i + 2] = b.x * s;
        v[4 * i + 3] = b.y * s;
    }
    if (act_may_exceed(s, top)) {
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] = act_held(v[i], top);
    }
}

// N words of codes, on a boundary of their size
template <int N>
__device__ __forceinline__ void load_codes(const uint8_t* p, uint32_t (&c)[N]) {
    if constexpr (N == 4) {
        const uint4 v = __ldcs(reinterpret_cast<const uint4*>(p));
        c[0] = v.x; c[1] = v.y; c[2] = v.z; c[3] = v.w;
    } else if constexpr (N == 2) {
        const uint2 v = __ldcs(reinterpret_cast<const uint2*>(p));
        c[0] = v.x; c[1] = v.y;
    } else {
        c[0] = __ldcs(reinterpret_cast<const uint32_t*>(p));
    }
}
template <int N>
__device__ __forceinline__ void store_codes(uint8_t* p, const uint32_t (&c)[N]) {
    if constexpr (N == 4) *reinterpret_cast<uint4*>(p) = make_uint4(c[0], c[1], c[2], c[3]);
    else if constexpr (N == 2) *reinterpret_cast<uint2*>(p) = make_uint2(c[0], c[1]);
    else *reinterpret_cast<uint32_t*>(p) = c[0];
}

// ---- rows on 32- or 16-byte boundaries: one such piece of x per lane and access ---------------------------------

// Saving.  E numbers (32 bytes) per lane, 128 / E lanes per block, U pieces in flight; a row ends inside a block where cols is not a
// multiple of 128 (lanes past it hold zeros).  FLAT: rows are whole blocks and adjacent, so the piece's number is its place.
// HALVES: rows begin on 16-byte boundaries and may end with half a piece.  (Pieces of 16 bytes instead, at twice the shuffles per
// number: 33390 x 5464 in 163 us where this takes 99.)
template <typename T, int U, bool FLAT, bool HALVES>
__global__ void __launch_bounds__(kThreads) tb200_k_act_save(const T* __restrict__ x, uint8_t* __restrict__ q, float* __restrict__ scales,
                                                   uint32_t blocks, uint32_t nblk, int64_t cols, int64_t ldx) {
    let_next_begin();
    constexpr int E = 32 / sizeof(T), kLanes = kActBlock / E;
    const uint64_t total = static_cast<uint64_t>(blocks) * kLanes, step = static_cast<uint64_t>(gridDim.x) * kThreads;
    for (uint64_t i0 = static_cast<uint64_t>(blockIdx.x) * kThreads + threadIdx.x; i0 - (threadIdx.x & 31) < total; i0 += U * step) {
        uint32_t w[U][8];
        int64_t at[U];                                           // place of the lane's codes, -1 where it has none
        bool both[U];                                            // whether the piece is whole
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const uint64_t i = i0 + j * step;
            at[j] = -1;
            both[j] = true;
            if (i < total) {
                if constexpr (FLAT) {
                    at[j] = static_cast<int64_t>(i) * E;
                    load_once(x + at[j], w[j]);
                } else {
                    const uint32_t blk = static_cast<uint32_t>(i / kLanes), row = blk / nblk;
                    const int64_t col = static_cast<int64_t>(blk - row * nblk) * kActBlock + (i % kLanes) * E;
                    if (col < cols) {
                        at[j] = static_cast<int64_t>(row) * cols + col;
                        const T* from = x + static_cast<int64_t>(row) * ldx + col;
                        if constexpr (HALVES) {
                            both[j] = col + E <= cols;
                            load_halves(from, both[j], w[j]);
                        } else {
                            load_once(from, w[j]);
                        }
                    }
                }
            }
            if (at[j] < 0) {
#pragma unroll
                for (int e = 0; e < 8; ++e) w[j][e] = 0;
            }
        }
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const uint64_t i = i0 + j * step;
            float v[E];
            uint32_t c[E / 4];
            numbers<T, 8>(w[j], v);
            const float s = encode<E>(v, c);
            if (at[j] >= 0) {
                if constexpr (HALVES) {
                    constexpr int H = E / 8;
                    uint32_t c0[H], c1[H];
#pragma unroll
                    for (int e = 0; e < H; ++e) {
                        c0[e] = c[e];
                        c1[e] = c[H + e];
                    }
                    store_codes<H>(q + at[j], c0);
                    if (both[j]) store_codes<H>(q + at[j] + E / 2, c1);
                } else {
                    store_codes<E / 4>(q + at[j], c);
                }
                if (i % kLanes == 0) scales[i / kLanes] = s;
            }
        }
    }
}

// Restoring: E codes per lane make one piece.  Rows of the result lie ldo apart.
template <typename T, int E, int U, bool FLAT>
__global__ void __launch_bounds__(kThreads) tb200_k_act_restore(const uint8_t* __restrict__ q, const float* __restrict__ scales, T* __restrict__ out,
                                                      uint32_t blocks, uint32_t nblk, int64_t cols, int64_t ldo) {
    let_next_begin();
    constexpr int kLanes = kActBlock / E, kWords = E * sizeof(T) / 4;
    const uint64_t total = static_cast<uint64_t>(blocks) * kLanes, step = static_cast<uint64_t>(gridDim.x) * kThreads;
    for (uint64_t i0 = static_cast<uint64_t>(blockIdx.x) * kThreads + threadIdx.x; i0 < total; i0 += U * step) {
        uint32_t c[U][E / 4];
        float s[U];
        int64_t to[U];                                           // place of the lane's numbers, -1 where it has none
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const uint64_t i = i0 + j * step;
            to[j] = -1;
            if (i < total) {
                const uint32_t blk = static_cast<uint32_t>(i / kLanes);
                int64_t from = static_cast<int64_t>(i) * E;
                if constexpr (FLAT) {
                    to[j] = from;
                } else {
                    const uint32_t row = blk / nblk;
                    const int64_t col = static_cast<int64_t>(blk - row * nblk) * kActBlock + (i % kLanes) * E;
                    from = static_cast<int64_t>(row) * cols + col;
                    if (col < cols) to[j] = static_cast<int64_t>(row) * ldo + col;
                }
                if (to[j] >= 0) {
                    load_codes<E / 4>(q + from, c[j]);
                    s[j] = __ldg(scales + blk);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < U; ++j) {
            if (to[j] >= 0) {
                float v[E];
                uint32_t w[kWords];
                decode<E>(c[j], s[j], ActType<T>::kTop, v);
                words<T, kWords>(v, w);
                store_piece(out + to[j], w);
            }
        }
    }
}

// ---- any width, stride and alignment ---------------------------------------------------------------------------
// A warp walks a span of one row in parts of 32 lanes with E neighbouring numbers each.  Loads are of aligned 4-byte words, one
// more than the numbers fill, shifted into place: every lane of a row has the same shift, and the neighbour's word comes from
// L1.  Saving is bound by that: every load instruction touches 32 sectors (one per lane), and the L1 data path is busy 89 % of the time at
// 16396 x 5461 in fp16 (80 us, 37 % of the DRAM rate, issue slots 55 %).  16-byte pieces joined by shuffles and selects took a third
// more time.  Rows of x on boundaries come here too where the codes' rows are odd.
// Stores of codes are of aligned words too, of the previous lane's last codes and the lane's own.  Loads that reach outside
// the tensor and stores that reach outside the span are made byte by byte.

// N words at p, on a boundary of their size, of which the first n bytes are there; the others come as zeros.
template <int N>
__device__ __forceinline__ void load_piece(const uint8_t* p, int n, uint32_t (&r)[N]) {
    if (n >= 4 * N) {
        load_codes<N>(p, r);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) r[i] = 0;
#pragma unroll 1
        for (int i = 0; i < n; ++i) {
            const uint32_t byte = static_cast<uint32_t>(p[i]) << (8 * (i & 3));
#pragma unroll
            for (int w = 0; w < N; ++w) r[w] |= i / 4 == w ? byte : 0;
        }
    }
}
// The N + 1 aligned words around N words at p, whatever its alignment.  inside: they all lie inside the tensor [begin, end), in
// every lane; where not, what does is fetched byte by byte.
template <int N>
__device__ __forceinline__ void load_words(const uint8_t* p, const uint8_t* begin, const uint8_t* end, bool inside, uint32_t (&a)[N + 1]) {
    const uint8_t* q = p - (reinterpret_cast<uintptr_t>(p) & 3);
    if (inside) {
#pragma unroll
        for (int i = 0; i <= N; ++i) a[i] = __ldg(reinterpret_cast<const uint32_t*>(q) + i);
    } else {
#pragma unroll
        for (int i = 0; i <= N; ++i) a[i] = 0;
#pragma unroll 1
        for (int i = 0; i < 4 * N + 4 && q + i < end; ++i) {
            if (q + i >= begin) {
                const uint32_t byte = static_cast<uint32_t>(q[i]) << (8 * (i & 3));
#pragma unroll
                for (int w = 0; w <= N; ++w) a[w] |= i / 4 == w ? byte : 0;
            }
        }
    }
}
template <int N>
__device__ __forceinline__ void into_place(const uint32_t (&a)[N + 1], const uint8_t* p, uint32_t (&r)[N]) {
    const uint32_t sh = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p) & 3) * 8;
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = __funnelshift_r(a[i], a[i + 1], sh);
}
// Whether all words of a part whose lane 0 begins at p and whose lanes have N words each lie inside the tensor.
template <int N>
__device__ __forceinline__ bool part_inside(const uint8_t* p, const uint8_t* begin, const uint8_t* end) {
    return p - (reinterpret_cast<uintptr_t>(p) & 3) >= begin && p + 32 * 4 * N + 4 <= end;
}
// Stores the word at byte b of a row's codes, as far as it lies in [lo, hi).
__device__ __forceinline__ void store_word(uint8_t* row, int b, int lo, int hi, uint32_t w) {
    if (b >= lo && b + 4 <= hi) {
        *reinterpret_cast<uint32_t*>(row + b) = w;
    } else if (b + 4 > lo && b < hi) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (b + i >= lo && b + i < hi) row[b + i] = static_cast<uint8_t>(w >> (8 * i));
    }
}
// spans: warps' shares of the rows, per_row of them in a row, `width` columns each (a multiple of the part).  PIECE: bytes per lane.
// 32 halve the shuffles per number (33390 x 5465 in bf16, with its restoring: 298 us with pieces of 16, 271 so), 16 leave fewer lanes
// idle in narrow rows (100000 x 130: 48 us against 62).
template <typename T, int PIECE>
__global__ void __launch_bounds__(kThreads) tb200_k_act_save_any(const T* __restrict__ x, uint8_t* __restrict__ q, float* __restrict__ scales,
                                                       int64_t spans, uint32_t per_row, int width, uint32_t nblk, int64_t rows, int64_t cols,
                                                       int64_t ldx) {
    let_next_begin();
    constexpr int E = PIECE / sizeof(T), N = E / 4, W = PIECE / 4, kLanes = kActBlock / E, kCols = 32 * E;
    const int lane = threadIdx.x & 31;
    const uint8_t *begin = reinterpret_cast<const uint8_t*>(x), *end = reinterpret_cast<const uint8_t*>(x + (rows - 1) * ldx + cols);
    for (int64_t s = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5); s < spans; s += static_cast<int64_t>(gridDim.x) * (kThreads / 32)) {
        const int64_t row = s / per_row, first = (s - row * per_row) * width;
        const int n = static_cast<int>(min(static_cast<int64_t>(width), cols - first));
        const uint8_t* const from = reinterpret_cast<const uint8_t*>(x + row * ldx + first);
        uint8_t* const to = q + row * cols + first;
        float* const sc = scales + row * nblk + first / kActBlock;
        const int mis = static_cast<int>(reinterpret_cast<uintptr_t>(to) & 3);
        uint32_t before = 0;                                     // lane 31's last word of the part before
        uint32_t ahead[W + 1];                                       // the next part's words, on the way while one is worked on
        auto fetch = [&](int col) {
            const uint8_t* p = from + static_cast<int64_t>(col) * sizeof(T);
            load_words<W>(p + lane * PIECE, begin, end, part_inside<W>(p, begin, end), ahead);
        };
        fetch(0);
#pragma unroll 2
        for (int col = 0; col < n; col += kCols) {
            uint32_t r[W], c[N];
            float v[E];
            const int at = col + lane * E;                       // the lane's first column in the span
            into_place<W>(ahead, from, r);
            if (col + kCols < n) fetch(col + kCols);
            numbers<T, W>(r, v);
            if (at + E > n) {
#pragma unroll
                for (int i = 0; i < E; ++i) v[i] = at + i < n ? v[i] : 0.0f;
            }
            const float scale = encode<E>(v, c);
            if (lane % kLanes == 0 && at < n) sc[at / kActBlock] = scale;
            // aligned words: the last `mis` bytes of the codes before and the first of the lane's own
            const uint32_t last = c[N - 1], first_before = __shfl_sync(0xffffffffu, lane == 31 ? before : last, (lane + 31) & 31);
#pragma unroll
            for (int i = 0; i < N; ++i) store_word(to, at + 4 * i - mis, 0, n, __funnelshift_l(i == 0 ? first_before : c[i > 0 ? i - 1 : 0], c[i], 8 * mis));
            before = last;
        }
        const int end = (n + kCols - 1) / kCols * kCols;         // codes of lane 31 that belong to the word behind the last part's
        if (lane == 31 && mis != 0) store_word(to, end - mis, 0, n, __funnelshift_l(before, 0, 8 * mis));
    }
}

// Restoring, any width of at least 16 columns, q on 16-byte and out on 32-byte boundaries: codes and numbers are both without gaps
// between rows, so pieces of 16 (8 for fp32) are taken across the ends of rows and blocks.  At most two ends lie inside a piece (those
// of a whole block and of a last one that is shorter than a piece); each code takes the scale of its side.
template <typename T, int U>
__global__ void __launch_bounds__(kThreads) tb200_k_act_restore_across(const uint8_t* __restrict__ q, const float* __restrict__ scales, T* __restrict__ out,
                                                             int64_t total, uint32_t nblk, int64_t cols) {
    let_next_begin();
    constexpr int E = 32 / sizeof(T);
    // a warp takes U * 32 neighbouring pieces at a time: their first place is divided once, the lanes' by 32-bit steps
    constexpr int kWarpCols = U * 32 * E;
    const int lane = threadIdx.x & 31;
    const int64_t step = static_cast<int64_t>(gridDim.x) * (kThreads / 32) * kWarpCols;
    for (int64_t w0 = (static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5)) * kWarpCols; w0 < total; w0 += step) {
        const int64_t row0 = w0 / cols;
        const uint32_t col0 = static_cast<uint32_t>(w0 - row0 * cols), width = static_cast<uint32_t>(cols);
        const float* sc = scales + row0 * nblk;
        uint32_t c[U][E / 4];
        float s0[U], s1[U], s2[U];
        uint32_t cut[U], cut2[U];                                // codes from here on take s1, and s2
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int64_t at = w0 + (j * 32 + lane) * E;
            if (at >= total) continue;
            load_piece<E / 4>(q + at, static_cast<int>(min(total - at, static_cast<int64_t>(E))), c[j]);
            uint32_t col = col0 + (j * 32 + lane) * E, row = 0;
            if (col >= width) {
                row = width >= kWarpCols ? 1 : col / width;      // 1: col0 < width, and the warp's share is no wider
                col -= row * width;
            }
            const float* p = sc + static_cast<int64_t>(row) * nblk + col / kActBlock;
            const uint32_t end = min(width, (col / kActBlock + 1) * kActBlock);                   // of the block
            cut[j] = min(end - col, static_cast<uint32_t>(E));
            cut2[j] = end < width ? min(width - col, static_cast<uint32_t>(E)) : E;
            s0[j] = __ldg(p);                                    // scales have no gaps either
            s1[j] = cut[j] < E && at + cut[j] < total ? __ldg(p + 1) : s0[j];
            s2[j] = cut2[j] < E && at + cut2[j] < total ? __ldg(p + 2) : s1[j];
        }
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int64_t at = w0 + (j * 32 + lane) * E;
            if (at >= total) continue;
            float v[E];
            uint32_t w[8];
            decode<E>(c[j], 1.0f, FLT_MAX, v);
            if (cut[j] == E) {
#pragma unroll
                for (int e = 0; e < E; ++e) v[e] *= s0[j];
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) v[e] *= e < cut[j] ? s0[j] : e < cut2[j] ? s1[j] : s2[j];
            }
            if (act_may_exceed(fmaxf(fabsf(s0[j]), fmaxf(fabsf(s1[j]), fabsf(s2[j]))), ActType<T>::kTop)) {
#pragma unroll
                for (int e = 0; e < E; ++e) v[e] = act_held(v[e], ActType<T>::kTop);
            }
            words<T, 8>(v, w);
            if (at + E <= total) store_piece(out + at, w);
            else {
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (at + e < total) out[at + e] = ActType<T>::store(v[e]);
            }
        }
    }
}

// Restoring at any alignment and width, one number per thread.
template <typename T>
__global__ void __launch_bounds__(kThreads) tb200_k_act_restore_any(const uint8_t* __restrict__ q, const float* __restrict__ scales, T* __restrict__ out,
                                                          int64_t total, uint32_t nblk, int64_t cols) {
    let_next_begin();
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * kThreads) {
        const int64_t row = i / cols;
        out[i] = ActType<T>::store(act_held(act_values2(q[i]).x * scales[row * nblk + (i - row * cols) / kActBlock], ActType<T>::kTop));
    }
}

// The backward pass's input, where it is small, restored by the last CTAs of the kernel that makes dg and du (a launch of its own
// takes 3 us whatever the work): 8 codes per thread, columns a multiple of 8, so that no piece has two scales.
struct RestoreJob {
    const uint2* q;
    const float* scales;
    uint4* out;
    uint32_t total, per_row, out_row, nblk;                      // pieces of 8, in all, per row and from row to row of the result; blocks per row
    int ctas;                                                    // 0: nothing to restore
};
template <typename T>
__device__ __forceinline__ void restore_job(const RestoreJob& job, uint32_t cta) {
    constexpr int U = 2;
    const uint64_t step = static_cast<uint64_t>(job.ctas) * kThreads;
    for (uint64_t i0 = static_cast<uint64_t>(cta) * kThreads + threadIdx.x; i0 < job.total; i0 += U * step) {
        uint2 c[U];
        float s[U];
        uint32_t to[U];
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const uint64_t i = i0 + j * step;
            if (i < job.total) {
                const uint32_t row = static_cast<uint32_t>(i) / job.per_row, col = static_cast<uint32_t>(i) - row * job.per_row;
                to[j] = row * job.out_row + col;
                c[j] = __ldcs(job.q + i);
                s[j] = __ldg(job.scales + static_cast<int64_t>(row) * job.nblk + col / 16);
            }
        }
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const uint64_t i = i0 + j * step;
            if (i < job.total) {
                const uint32_t codes[2] = {c[j].x, c[j].y};
                float v[8];
                uint32_t w[4];
                decode<8>(codes, s[j], ActType<T>::kTop, v);
                words<T, 4>(v, w);
                job.out[to[j]] = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
    }
}

// ---- the power of two of an fp16 backward pass ------------------------------------------------------------------------
// Largest finite |dh| (its bits, in the upper half of a word) and largest finite |scale| (the upper half of its bits, in the lower) of a
// CTA's share, written behind row blockIdx.x of du: there are at most m CTAs.  Bound by reading dh once, 2 bytes of the 16 or so that a
// number of dh costs in all (16384 x 8192: 46 us, 6.0 TB/s), and by a launch more: a captured backward pass in fp16 takes 5 us longer for it at 1023 rows of 1048 x 2731
// (39 -> 45) and at 4 of 2048 x 5632 (33 -> 38), 7 at 64 of 4096 x 14336 (108 -> 115).  The launch overlaps with the end of the
// kernel before, so nothing is read through the read-only path; the next kernel may begin once that one is complete.
__device__ __forceinline__ void load_plain(const void* p, uint32_t (&r)[8]) {    // 32 bytes
    asm volatile("ld.global.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "l"(p) : "memory");
}
constexpr int kRangeThreads = 512, kMostMaxima = kThreads;       // one for each thread that reads them
template <int WARPS>
__device__ __forceinline__ uint32_t block_max2(uint32_t v, uint32_t* shared) {                   // of both halves, in all threads
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = __vmaxu2(v, __shfl_xor_sync(0xffffffffu, v, o));
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WARPS; ++i) v = __vmaxu2(v, shared[i]);
    return v;
}
__global__ void __launch_bounds__(kRangeThreads) tb200_k_ffn_grad_range(const __half* dh, int64_t n, const float* gs, const float* us, int64_t blocks, uint32_t* maxima,
                                                              int64_t pitch) {
    wait_for_previous();
    let_next_begin();
    __shared__ uint32_t shared[kRangeThreads / 32];
    constexpr int E = 16, U = 4;
    const int64_t first = static_cast<int64_t>(blockIdx.x) * kRangeThreads + threadIdx.x, step = static_cast<int64_t>(gridDim.x) * kRangeThreads;
    // 32-byte pieces between the first such boundary and the last; up to 15 numbers before and 15 behind
    const int64_t skip = static_cast<int64_t>((32 - (reinterpret_cast<uintptr_t>(dh) & 31)) & 31) / 2, head = skip < n ? skip : n;
    const int64_t pieces = (n - head) / E, tail = head + pieces * E;
    const uint16_t* const bits = reinterpret_cast<const uint16_t*>(dh);
    uint32_t top = 0;                                            // of even and odd numbers
    auto take = [&](uint32_t w) {
        w &= 0x7FFF7FFFu;
        const uint32_t most = 0x7BFF7BFFu;                       // infinities and NaN do not count
        top = __vmaxu2(top, w & __hle2_mask(*reinterpret_cast<const __half2*>(&w), *reinterpret_cast<const __half2*>(&most)));
    };
    // the first of each kind on the way together
    const uint32_t before = first < head ? __ldcg(bits + first) : 0, behind = tail + first < n ? __ldcg(bits + tail + first) : 0;
    const float g0 = first < blocks ? __ldcg(gs + first) : 0.0f, u0 = first < blocks ? __ldcg(us + first) : 0.0f;
    for (int64_t i0 = first; i0 < pieces; i0 += U * step) {
        uint32_t w[U][8];
#pragma unroll
        for (int j = 0; j < U; ++j) {                            // past the end the last piece once more
            const int64_t i = i0 + j * step;
            load_plain(dh + head + (i < pieces ? i : pieces - 1) * E, w[j]);
        }
#pragma unroll
        for (int j = 0; j < U; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) take(w[j][e]);
    }
    take(before);
    take(behind);
    float size = fmaxf(act_size(g0), act_size(u0));
    for (int64_t i = first + step; i < blocks; i += step) size = fmaxf(size, fmaxf(act_size(__ldcg(gs + i)), act_size(__ldcg(us + i))));
    top = max(top & 0xFFFFu, top >> 16);
    const uint32_t all = block_max2<kRangeThreads / 32>(top << 16 | __float_as_uint(size) >> 16, shared);
    if (threadIdx.x == 0) maxima[blockIdx.x * pitch] = all;
}
// The power of two from those maxima, the same in all threads; the inverse is left at `inverse` by CTA 0.
struct GradRange { const uint32_t* maxima; float* inverse; int count; uint32_t pitch; };
__device__ __forceinline__ float grad_power(const GradRange& r) {
    __shared__ uint32_t shared[kThreads / 32];
    wait_for_previous();                                         // for the maxima: this kernel's launch overlaps with that one's end
    const int i = threadIdx.x;
    const uint32_t v = block_max2<kThreads / 32>(i < r.count ? __ldcg(r.maxima + static_cast<int64_t>(i) * r.pitch) : 0, shared);
    // 2^a <= |dh| < 2^(a + 1), 2^b <= scale < 2^(b + 1): the bound is below 2^(a + b + 11)
    const float largest = __half2float(__ushort_as_half(static_cast<unsigned short>(v >> 16)));
    const int a = static_cast<int>(__float_as_uint(largest) >> 23) - 127, b = static_cast<int>((v & 0xFFFFu) >> 7) - 127;
    const int e = min(max(15 - (a + b + 11), -100), 100);        // both powers stay far within fp32's range
    if (blockIdx.x == 0 && threadIdx.x == 0) *r.inverse = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
    return __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
}

// dg = dh * u * f'(g), du = dh * f(g) for 8 numbers of a lane, in fp32 and rounded once to T: they are operands of 16 bits in the
// products that follow (half a step, 2^-8 of the value in bf16 and 2^-11 in fp16, which the products' sums average out).  dh comes times `power` in fp16.
template <typename T, int ACT>
__device__ __forceinline__ void gated_bwd8(const uint32_t (&d)[4], const uint32_t (&cg)[2], const uint32_t (&cu)[2], float sg, float su, float power,
                                           uint4& dg, uint4& du) {
    float e[8], g[8], u[8];
    uint32_t og[4], ou[4];
    numbers<T, 4>(d, e);
    if constexpr (kRanged<T>) {
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] *= power;
    }
    decode<8>(cg, sg, FLT_MAX, g);
    decode<8>(cu, su, FLT_MAX, u);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float2 a = gate_both<ACT>(g[i]);
        g[i] = e[i] * u[i] * a.y;
        u[i] = e[i] * a.x;
    }
    words<T, 4>(g, og);
    words<T, 4>(u, ou);
    dg = make_uint4(og[0], og[1], og[2], og[3]);
    du = make_uint4(ou[0], ou[1], ou[2], ou[3]);
}

// Widths that are multiples of 8, 16-byte boundaries: 8 numbers per thread.
template <typename T, int ACT, int U>
__global__ void __launch_bounds__(kThreads) tb200_k_ffn_gated_bwd(const uint4* __restrict__ dh, const uint2* __restrict__ gq, const float* __restrict__ gs,
                                                        const uint2* __restrict__ uq, const float* __restrict__ us, uint4* __restrict__ dg,
                                                        uint4* __restrict__ du, uint32_t total, uint32_t per_row, uint32_t out_row, uint32_t nblk,
                                                        const RestoreJob job, const GradRange range) {
    let_next_begin();
    float power = 1.0f;
    if constexpr (kRanged<T>) power = grad_power(range);
    const uint32_t ctas = gridDim.x - job.ctas, step = ctas * kThreads;
    if (blockIdx.x >= ctas) return restore_job<T>(job, blockIdx.x - ctas);
    for (uint64_t i0 = blockIdx.x * kThreads + threadIdx.x; i0 < total; i0 += U * step) {
        uint4 d[U];
        uint2 cg[U], cu[U];
        float sg[U], su[U];
        uint32_t to[U];                                          // place in dg and du, whose rows lie out_row pieces apart
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const uint64_t i = i0 + j * step;
            if (i < total) {
                const uint32_t row = static_cast<uint32_t>(i) / per_row, col = static_cast<uint32_t>(i) - row * per_row, blk = row * nblk + col / 16;
                to[j] = row * out_row + col;
                d[j] = __ldcs(dh + i);
                cg[j] = __ldcs(gq + i);
                cu[j] = __ldcs(uq + i);
                sg[j] = __ldg(gs + blk);
                su[j] = __ldg(us + blk);
            }
        }
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const uint64_t i = i0 + j * step;
            if (i < total) {
                const uint32_t dw[4] = {d[j].x, d[j].y, d[j].z, d[j].w}, gw[2] = {cg[j].x, cg[j].y}, uw[2] = {cu[j].x, cu[j].y};
                uint4 a, b;
                gated_bwd8<T, ACT>(dw, gw, uw, sg[j], su[j], power, a, b);
                dg[to[j]] = a;
                du[to[j]] = b;
            }
        }
    }
}

// The same for any width and alignment of dh and the codes; dg and du have rows on 16-byte boundaries, ldg >= f a multiple of 8.
template <typename T, int ACT>
__global__ void __launch_bounds__(kThreads) tb200_k_ffn_gated_bwd_any(const T* __restrict__ dh, const uint8_t* __restrict__ gq, const float* __restrict__ gs,
                                                            const uint8_t* __restrict__ uq, const float* __restrict__ us, T* __restrict__ dg,
                                                            T* __restrict__ du, int64_t spans, uint32_t per_row, int width, int64_t m, int64_t f,
                                                            int64_t ldg, uint32_t nblk, const RestoreJob job, const GradRange range) {
    let_next_begin();
    float power = 1.0f;
    if constexpr (kRanged<T>) power = grad_power(range);
    const uint32_t ctas = gridDim.x - job.ctas;
    if (blockIdx.x >= ctas) return restore_job<T>(job, blockIdx.x - ctas);
    static_assert(sizeof(T) == 2, "8 numbers of 16 bits and 8 codes per lane");
    constexpr int E = 8, kCols = 32 * E;
    const int lane = threadIdx.x & 31;
    const int64_t total = m * f;
    for (int64_t s = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5); s < spans; s += static_cast<int64_t>(ctas) * (kThreads / 32)) {
        const int64_t row = s / per_row, first = (s - row * per_row) * width, at0 = row * f + first;
        const int n = static_cast<int>(min(static_cast<int64_t>(width), f - first));
        const int64_t blk = row * nblk + first / kActBlock;
        const uint8_t *const dh0 = reinterpret_cast<const uint8_t*>(dh), *const d0 = dh0 + 2 * at0, *const g0 = gq + at0, *const u0 = uq + at0;
        T *const to_g = dg + row * ldg + first, *const to_u = du + row * ldg + first;
        // the next part's words and scales, on the way while one is worked on
        uint32_t ad[5], ag[3], au[3];
        float asg, asu;
        auto fetch = [&](int col) {
            const int at = col + lane * E;
            const bool inside = part_inside<4>(d0 + 2 * col, dh0, dh0 + 2 * total) && part_inside<2>(g0 + col, gq, gq + total) && part_inside<2>(u0 + col, uq, uq + total);
            load_words<4>(d0 + 2 * at, dh0, dh0 + 2 * total, inside, ad);
            load_words<2>(g0 + at, gq, gq + total, inside, ag);
            load_words<2>(u0 + at, uq, uq + total, inside, au);
            asg = at < n ? __ldg(gs + blk + at / kActBlock) : 0.0f;
            asu = at < n ? __ldg(us + blk + at / kActBlock) : 0.0f;
        };
        fetch(0);
#pragma unroll 2
        for (int col = 0; col < n; col += kCols) {
            uint32_t d[4], cg[2], cu[2];
            const int at = col + lane * E;
            const bool here = at < n;
            const float sg = asg, su = asu;
            into_place<4>(ad, d0, d);
            into_place<2>(ag, g0, cg);
            into_place<2>(au, u0, cu);
            if (col + kCols < n) fetch(col + kCols);
            if (here) {
                uint4 a, b;
                gated_bwd8<T, ACT>(d, cg, cu, sg, su, power, a, b);
                *reinterpret_cast<uint4*>(to_g + at) = a;        // the row's padding takes what is behind its last column
                *reinterpret_cast<uint4*>(to_u + at) = b;
            }
        }
    }
}

// How tb200_k_act_save_any and tb200_k_ffn_gated_bwd_any share out their rows: spans of up to 4 parts, fewer where that leaves an SM less than 32
// warps' worth; neighbouring warps have neighbouring spans.  A whole row per warp has fewer ragged ends, but thousands of places
// of memory in use at once and a last round that is mostly idle (6525 x 27060: 404 us where this takes 277).
struct Spans { int64_t count; uint32_t per_row; int width; };
Spans spans_of(int64_t rows, int64_t cols, int part) {
    const int64_t parts = (cols + part - 1) / part, room = rows * parts / (static_cast<int64_t>(num_sms()) * 32);
    const int64_t most = room < 1 ? 1 : room > 4 ? 4 : room, per_row = (parts + most - 1) / most, each = (parts + per_row - 1) / per_row;
    return {rows * per_row, static_cast<uint32_t>(per_row), static_cast<int>(each * part)};
}

int capped(int64_t ctas, int per_sm) {
    const int64_t cap = static_cast<int64_t>(num_sms()) * per_sm;
    return static_cast<int>(ctas < 1 ? 1 : ctas < cap ? ctas : cap);
}

constexpr uint64_t aligned_to(uintptr_t bytes, const void* p, uintptr_t pitch_bytes) {
    return ((reinterpret_cast<uintptr_t>(p) | pitch_bytes) & (bytes - 1)) == 0;
}

// Pieces of 32 bytes where rows begin on such boundaries and are whole numbers of them, of 16 where that holds, else none of these.
// (bf16, 33390 x 5464, saved in 99 us, by shifted words in 171; restored in 101, across the ends of rows 123.)
int piece_bytes(const void* x, int64_t row_bytes, int64_t pitch_bytes, const void* codes, int size) {
    const uintptr_t all = reinterpret_cast<uintptr_t>(x) | static_cast<uintptr_t>(row_bytes) | static_cast<uintptr_t>(pitch_bytes);
    for (int b = 32; b >= 16; b /= 2)
        if (all % b == 0 && reinterpret_cast<uintptr_t>(codes) % (b / size) == 0) return b;
    return 0;
}

template <typename T>
int launch_save(const T* x, uint8_t* q, float* scales, int64_t rows, int64_t cols, int64_t ldx, cudaStream_t st) {
    constexpr int kSize = sizeof(T);
    const uint32_t nblk = static_cast<uint32_t>((cols + kActBlock - 1) / kActBlock);
    const int piece = piece_bytes(x, cols * kSize, rows > 1 ? ldx * kSize : 0, q, kSize);
    if (piece > 0) {
        constexpr int E = 32 / kSize, U = 4;
        const uint32_t blocks = static_cast<uint32_t>(rows * nblk);
        const int grid = capped((static_cast<int64_t>(blocks) * (kActBlock / E) + kThreads * U - 1) / (kThreads * U), 8);
        if (piece == 16) tb200_k_act_save<T, U, false, true><<<grid, kThreads, 0, st>>>(x, q, scales, blocks, nblk, cols, ldx);
        else if (cols % kActBlock == 0 && (ldx == cols || rows == 1)) tb200_k_act_save<T, U, true, false><<<grid, kThreads, 0, st>>>(x, q, scales, blocks, nblk, cols, ldx);
        else tb200_k_act_save<T, U, false, false><<<grid, kThreads, 0, st>>>(x, q, scales, blocks, nblk, cols, ldx);
    } else {
        // the wider pieces where rows have some four parts of them and at most a tenth more idle lanes
        const int64_t part = 32 * 32 / kSize, wide = (cols + part - 1) / part * part, narrow = (cols + part / 2 - 1) / (part / 2) * (part / 2);
        const bool by32 = cols > 3 * part && 10 * wide <= 11 * narrow;
        const Spans sp = spans_of(rows, cols, static_cast<int>(by32 ? part : part / 2));
        (by32 ? tb200_k_act_save_any<T, 32> : tb200_k_act_save_any<T, 16>)<<<capped((sp.count + 7) / 8, 8), kThreads, 0, st>>>(
            x, q, scales, sp.count, sp.per_row, sp.width, nblk, rows, cols, ldx);
    }
    TB200_CUDA_TRY(cudaGetLastError());
    return TB200_OK;
}

template <typename T, int E>
void launch_restore_pieces(const uint8_t* q, const float* scales, T* out, int64_t rows, int64_t cols, int64_t ldo, uint32_t nblk, cudaStream_t st) {
    constexpr int U = 128 / (E * static_cast<int>(sizeof(T)));
    const uint32_t blocks = static_cast<uint32_t>(rows * nblk);
    const int grid = capped((static_cast<int64_t>(blocks) * (kActBlock / E) + kThreads * U - 1) / (kThreads * U), 8);
    if (cols % kActBlock == 0 && ldo == cols) tb200_k_act_restore<T, E, U, true><<<grid, kThreads, 0, st>>>(q, scales, out, blocks, nblk, cols, ldo);
    else tb200_k_act_restore<T, E, U, false><<<grid, kThreads, 0, st>>>(q, scales, out, blocks, nblk, cols, ldo);
}

template <typename T>
int launch_restore(const uint8_t* q, const float* scales, T* out, int64_t rows, int64_t cols, int64_t ldo, cudaStream_t st) {
    constexpr int kSize = sizeof(T), E = 32 / kSize, U = 4;
    const uint32_t nblk = static_cast<uint32_t>((cols + kActBlock - 1) / kActBlock);
    const int piece = piece_bytes(out, cols * kSize, ldo * kSize, q, kSize);
    const int64_t total = rows * cols;
    if (piece == 32) {
        launch_restore_pieces<T, E>(q, scales, out, rows, cols, ldo, nblk, st);
    } else if (piece == 16) {
        launch_restore_pieces<T, E / 2>(q, scales, out, rows, cols, ldo, nblk, st);
    } else if (cols >= 16 && aligned_to(16, q, 0) && aligned_to(32, out, 0)) {
        tb200_k_act_restore_across<T, U><<<capped((total + kThreads * E * U - 1) / (kThreads * E * U), 8), kThreads, 0, st>>>(q, scales, out, total, nblk, cols);
    } else {
        tb200_k_act_restore_any<T><<<capped((total + kThreads - 1) / kThreads, 8), kThreads, 0, st>>>(q, scales, out, total, nblk, cols);
    }
    TB200_CUDA_TRY(cudaGetLastError());
    return TB200_OK;
}

template <typename Kernel, typename... Args>
int launch_over(bool over_previous, Kernel kern, int grid, int threads, cudaStream_t st, const Args&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(grid), 1, 1);
    cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = over_previous ? 1 : 0;
    TB200_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, args...));
    return TB200_OK;
}

template <typename T, int ACT>
int launch_gated(const void* dh, const void* gq, const float* gs, const void* uq, const float* us, void* dg, void* du, int64_t m, int64_t f,
                 int64_t ldg, const RestoreJob& job, cudaStream_t st) {
    const uint32_t nblk = static_cast<uint32_t>((f + kActBlock - 1) / kActBlock);
    GradRange range = {};
    if constexpr (kRanged<T>) {
        // one piece per thread, as far as there are rows to leave the maxima behind and threads to read them
        const int64_t wanted = (m * f + kRangeThreads * 16 - 1) / (kRangeThreads * 16), most = m < kMostMaxima ? m : kMostMaxima;
        uint32_t* const maxima = behind_row<uint32_t>(du, ldg);
        range = {maxima, behind_row<float>(dg, ldg), static_cast<int>(wanted < most ? wanted : most), static_cast<uint32_t>(ldg / 2)};
        const int rc = launch_over(true, tb200_k_ffn_grad_range, range.count, kRangeThreads, st, static_cast<const __half*>(dh), m * f, gs, us,
                                   m * static_cast<int64_t>(nblk), maxima, ldg / 2);
        if (rc != TB200_OK) return rc;
    }
    if (f % 8 == 0 && aligned_to(16, dh, 0) && aligned_to(8, gq, 0) && aligned_to(8, uq, 0) && m * (ldg / 8) <= 0xFFFFFFFFll) {
        const int64_t total = m * (f / 8);
        constexpr int U = 2;
        return launch_over(kRanged<T>, tb200_k_ffn_gated_bwd<T, ACT, U>, capped((total + kThreads * U - 1) / (kThreads * U), 8) + job.ctas, kThreads, st,
                           static_cast<const uint4*>(dh), static_cast<const uint2*>(gq), gs, static_cast<const uint2*>(uq), us,
                           static_cast<uint4*>(dg), static_cast<uint4*>(du), static_cast<uint32_t>(total), static_cast<uint32_t>(f / 8),
                           static_cast<uint32_t>(ldg / 8), nblk, job, range);
    }
    const Spans sp = spans_of(m, f, 256);
    return launch_over(kRanged<T>, tb200_k_ffn_gated_bwd_any<T, ACT>, capped((sp.count + 7) / 8, 8) + job.ctas, kThreads, st, static_cast<const T*>(dh),
                       static_cast<const uint8_t*>(gq), gs, static_cast<const uint8_t*>(uq), us, static_cast<T*>(dg), static_cast<T*>(du),
                       sp.count, sp.per_row, sp.width, m, f, ldg, nblk, job, range);
}

template <typename T>
int launch_gated_act(const void* dh, const void* gq, const float* gs, const void* uq, const float* us, void* dg, void* du, int64_t m, int64_t f,
                     int64_t ldg, const RestoreJob& job, int act, cudaStream_t st) {
    switch (act) {
        case TB200_ACT_SILU: return launch_gated<T, TB200_ACT_SILU>(dh, gq, gs, uq, us, dg, du, m, f, ldg, job, st);
        case TB200_ACT_GELU: return launch_gated<T, TB200_ACT_GELU>(dh, gq, gs, uq, us, dg, du, m, f, ldg, job, st);
        case TB200_ACT_GELU_TANH: return launch_gated<T, TB200_ACT_GELU_TANH>(dh, gq, gs, uq, us, dg, du, m, f, ldg, job, st);
        default: return launch_gated<T, TB200_ACT_RELU>(dh, gq, gs, uq, us, dg, du, m, f, ldg, job, st);
    }
}

// ldo: row pitch of out, cols unless rows of out and of q are whole 16-byte and 8-byte pieces on such boundaries.
int launch_act_restore(const void* q, const float* scales, void* out, int dtype, int64_t rows, int64_t cols, int64_t ldo, cudaStream_t st) {
    const uint8_t* c = static_cast<const uint8_t*>(q);
    if (dtype == TB200_DT_F32) return launch_restore<float>(c, scales, static_cast<float*>(out), rows, cols, ldo, st);
    if (dtype == TB200_DT_F16) return launch_restore<__half>(c, scales, static_cast<__half*>(out), rows, cols, ldo, st);
    return launch_restore<__nv_bfloat16>(c, scales, static_cast<__nv_bfloat16*>(out), rows, cols, ldo, st);
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
                         int64_t m, int64_t f, int64_t ldg, const void* xq, const float* xs, void* x, int64_t k, int64_t ldx, int act, int dtype,
                         cudaStream_t st) {
    RestoreJob job = {};
    if (xq) {
        const int64_t total = m * (k / 8);
        // up to 4 M numbers (5 us by themselves); 12867 x 3616 took 52 us together with dg and du, 40 in two launches
        if ((reinterpret_cast<uintptr_t>(xq) & 7) == 0 && m * k <= (4ll << 20)) {
            job = {static_cast<const uint2*>(xq), xs, static_cast<uint4*>(x), static_cast<uint32_t>(total), static_cast<uint32_t>(k / 8), static_cast<uint32_t>(ldx / 8),
                   static_cast<uint32_t>((k + kActBlock - 1) / kActBlock), capped((total + 2 * kThreads - 1) / (2 * kThreads), 8)};
        } else {
            const int rc = launch_act_restore(xq, xs, x, dtype, m, k, ldx, st);
            if (rc != TB200_OK) return rc;
        }
    }
    return dtype == TB200_DT_F16 ? launch_gated_act<__half>(dh, gq, gs, uq, us, dg, du, m, f, ldg, job, act, st)
                                 : launch_gated_act<__nv_bfloat16>(dh, gq, gs, uq, us, dg, du, m, f, ldg, job, act, st);
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
    return launch_act_restore(q, scales, out, dtype, rows, cols, cols, static_cast<cudaStream_t>(stream));
}
