// Matrix products of the gated feed-forward block, forward and backward, on tcgen05 (kind::f16, fp32 accumulation).
//
//   forward   g = x Wg^T, u = x Wu^T, h = f(g) * u         one kernel; the codes of g and u in 8 bits on request
//   backward  dx = dg Wg + du Wu                            one accumulator over both products
//             dWg = dg^T x, dWu = du^T x                    one kernel over the tiles of all three results
//
// Both are one CTA-pair kernel (cta_group::2): 256 x 256 accumulators in tensor memory, two of them, so that the
// epilogue of a tile runs under the main loop of the next.  Each CTA of a pair loads 128 rows of A and one 128-wide
// half of B per 64-deep stage.  What differs is where the operands lie:
//   forward   A = x and B = W with the contraction contiguous (K-major).  The leader's half of B is 128 rows of Wg,
//             the peer's the same 128 rows of Wu: columns 0..127 of the accumulator are g, columns 128..255 are u of the
//             same hidden units, so a thread of the epilogue holds both of its row and nothing is exchanged; a row's
//             1 x 128 block of g (or u) is one thread's, which is what makes the 8-bit codes free of any reduction.
//   dx        A = dg, then du (K-major); B = Wg, then Wu with the contraction strided (MN-major, read as stored).
//   dw        A = dg^T, du^T and B = x, both MN-major, read as stored: nothing is transposed in memory.
// Ragged sizes: copies that reach past a tensor's edge bring zeros, stores past it are left out.
// Every mbarrier wait is bounded and reports through g_status.
#include "act_fp8.cuh"

#include <cmath>
#include <cstring>
#include <type_traits>

namespace tb200 {
namespace {

constexpr int kBK = 64;                          // contraction per stage: 128 bytes of 16-bit elements
constexpr int kHalf = 128;                       // rows of A, and columns of B, that one CTA loads
// Stages in shared memory, and copies of the result under way per quarter: two places of 4 KB leave room for 6 stages.  Where dx has a
// kernel of its own, dw's tiles have a single stage: 4 are enough there, and four places keep more copies under way.
constexpr int stages_of(int kind) { return kind == 2 ? 4 : 6; }
constexpr int places_of(int kind) { return kind == 2 ? 4 : 2; }
constexpr int kOperandBytes = kHalf * 128;
constexpr int kStageBytes = 2 * kOperandBytes;
constexpr int kAtomBytes = kBK * 128;            // MN-major: one box of 64 contraction rows x 64 columns
constexpr int kEpiWarps = 16;                    // four per quarter of the tensor memory's lanes (32 rows), each a quarter of the columns
constexpr int kStagingBytes = 32 * 256;          // per quarter: 32 rows of 256 bytes
constexpr int kAmaxBytes = 4 * 32 * 8;           // per quarter: 32 rows' amax of g and of u
constexpr int kBarBytes = 256;
constexpr int kSmemBytes = 6 * kStageBytes + 4 * kStagingBytes + kAmaxBytes + kBarBytes + 1024;
constexpr int kTmemCols = 512;
constexpr int kThreads = 128 + 32 * kEpiWarps;   // TMA, MMA, two idle warps, epilogue
constexpr int kGroupM = 8;                       // tiles are walked in bands of 8 x 256 rows, so that B's tiles stay in L2

enum FfnKind : int { FK_FWD = 0, FK_BWD = 1, FK_DW = 2 };       // FK_DW: the backward pass without dx

template <int KIND> struct FfnMaps;
template <> struct FfnMaps<FK_FWD> { CUtensorMap a[1], b[2]; };                  // x; Wg, Wu
struct FfnBwdMaps {
    CUtensorMap a[2], b[2];                      // of dx: dg, du; Wg, Wu
    CUtensorMap at[2], x;                        // of dw: dg, du; x
    CUtensorMap out[3];                          // dx, dWg, dWu
};
template <> struct FfnMaps<FK_BWD> : FfnBwdMaps {};
template <> struct FfnMaps<FK_DW> : FfnBwdMaps {};
struct FfnArgs {
    void* out[3];                                // forward: h; backward: dx, dWg, dWu
    int m, f, k;
    int w;                                       // forward: hidden units per tile (128 with checkpoints)
    uint8_t* codes[2];                           // forward with checkpoints: codes of g and u, [m, f]
    float* scales[2];                            // and their scales, [m, ceil(f / 128)]
    float* sums[2];                              // backward, in shares: partial sums of dx [shares, m, k], of dw [shares, 2, f, k]
    int shares[2];                               // of the contraction of dx, and of dw; 0: not in this launch
    int early;                                   // backward, see item_at
    const float* factor;                         // backward in fp16: of the results, see grad_pitch
};

__device__ __forceinline__ uint64_t desc_mn(uint32_t smem_addr) {       // MN-major, 128-byte swizzle
    uint64_t d = 0;
    d |= static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4);
    d |= static_cast<uint64_t>(kAtomBytes >> 4) << 16;                  // from one 64-column box to the next
    d |= static_cast<uint64_t>(1024 >> 4) << 32;                        // from 8 contraction rows to the next 8
    d |= static_cast<uint64_t>(1) << 46;
    d |= static_cast<uint64_t>(2) << 61;
    return d;
}
__device__ __forceinline__ void mma_pair_if(uint32_t issue, uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
                 "@q tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem), "l"(a_desc), "l"(b_desc),
                 "r"(idesc), "r"(accumulate), "r"(issue) : "memory");
}

__device__ __forceinline__ void mma_if(uint32_t issue, uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem), "l"(a_desc), "l"(b_desc),
                 "r"(idesc), "r"(accumulate), "r"(issue) : "memory");
}

// Brings a box towards the SMs, as far as L2.  Nothing is read in the program's sense, so a weight that the kernel before is
// still writing may be asked for: L2 holds what is written last.
__device__ __forceinline__ void prefetch_2d(const CUtensorMap* m, int x, int y) {
    asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(reinterpret_cast<uint64_t>(m)), "r"(x), "r"(y) : "memory");
}

// ---- epilogue helpers --------------------------------------------------------------------------------------------
// The four warps of a quarter collect 32 rows of 256 bytes in shared memory, 16-byte piece c of row r at place
// c ^ (r & 15) (free of bank conflicts both ways); then each writes 8 of the rows out, neighbouring lanes on neighbouring bytes.
__device__ __forceinline__ uint8_t* staged(uint8_t* buf, int row, int piece) { return buf + row * 256 + ((piece ^ (row & 15)) << 4); }
__device__ __forceinline__ uint32_t shared_uint(uint32_t at) {
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(at));
    return v;
}
__device__ __forceinline__ uint32_t shared_byte(uint32_t at) {
    uint32_t v;
    asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(at));
    return v;
}
__device__ __forceinline__ uint4 shared_uint4(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
    return v;
}
__device__ __forceinline__ void quarter_sync(int quarter) { asm volatile("bar.sync %0, 128;" ::"r"(1 + quarter) : "memory"); }

// Columns [0, cols) of rows [r0, min(r0 + 8, rows)), r0 a multiple of 8, which begin at piece `first` (0 or 8), go to row r of
// dst; at most PIECES pieces of a row.  Rows that begin on 16-byte boundaries take 16-byte stores.  Others (f is odd, say) take a
// warp each: aligned words, shifted into place, and single bytes at either end.  Row r0 + i lies i * 256 bytes on, its piece c at
// place (c ^ r0 & 8) ^ i, which leaves one instruction per row to find a piece.
template <typename T, int PIECES>
__device__ __forceinline__ void flush(uint8_t* buf, int first, T* __restrict__ dst, int64_t pitch, int r0, int rows, int cols, int lane) {
    constexpr int kSize = sizeof(T), kPer = 32 / PIECES;
    const int bytes = min(cols * kSize, PIECES * 16), n = min(8, rows - r0);
    if (bytes <= 0 || n <= 0) return;
    const uint32_t base = smem_u32(buf) + r0 * 256;
    if (((reinterpret_cast<uintptr_t>(dst) | static_cast<uintptr_t>(pitch * kSize)) & 15) == 0) {
        const int c = lane % PIECES, sub = lane / PIECES;
        const uint32_t place = static_cast<uint32_t>((first + c) ^ (r0 & 8) ^ sub) << 4;
        uint8_t* p = reinterpret_cast<uint8_t*>(dst + (r0 + sub) * pitch) + 16 * c;
        if (16 * c + 16 <= bytes) {
#pragma unroll
            for (int i = 0; i < 8; i += kPer) {
                if (i + sub < n) *reinterpret_cast<uint4*>(p + i * pitch * kSize) = shared_uint4(base + sub * 256 + i * 256 + (place ^ (i << 4)));
            }
        } else if (16 * c < bytes) {
            for (int i = 0; i + sub < n; i += kPer) {
                const T* src = reinterpret_cast<const T*>(staged(buf, r0 + i + sub, first + c));
                for (int e = 0; 16 * c + e * kSize < bytes; ++e) reinterpret_cast<T*>(p + i * pitch * kSize)[e] = src[e];
            }
        }
    } else {
        // all words first, so that the rows do not wait for one another
        constexpr int kWords = PIECES / 8;
        const uint32_t place = (static_cast<uint32_t>((first + (lane >> 2)) ^ (r0 & 8)) << 4) + (lane & 3) * 4;
        uint8_t* const p0 = reinterpret_cast<uint8_t*>(dst + r0 * pitch);
        uint32_t w[8][kWords];
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int j = 0; j < kWords; ++j) w[i][j] = shared_uint(base + i * 256 + (place ^ (j << 7) ^ (i << 4)));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            uint8_t* const p = p0 + i * pitch * kSize;
            const int mis = static_cast<int>(reinterpret_cast<uintptr_t>(p) & 3), valid = i < n ? bytes : 0;
            uint32_t before = 0;
#pragma unroll
            for (int j = 0; j < kWords; ++j) {                   // lane l has the word that lies 4 (32 j + l) - mis bytes into the row
                const uint32_t w0 = __shfl_sync(0xffffffffu, lane == 31 ? before : w[i][j], (lane + 31) & 31);
                const int b = 4 * (32 * j + lane) - mis;
                if (b >= 0 && b + 4 <= valid) *reinterpret_cast<uint32_t*>(p + b) = __funnelshift_l(w0, w[i][j], 8 * mis);
                before = w[i][j];
            }
            const int head = min(-mis & 3, valid), tail = (valid - head) & 3, b = lane < head ? lane : valid - tail + lane - head;
            if (lane < head + tail) p[b] = static_cast<uint8_t>(shared_byte(base + i * 256 + ((((first + (b >> 4)) ^ (r0 & 8) ^ i) << 4) | (b & 15))));
        }
    }
}

// 16-bit numbers of 32 columns as 4 pieces, codes of 32 columns as 2
template <typename T>
__device__ __forceinline__ void stage32(uint8_t* buf, int row, int piece0, const uint32_t (&v)[32]) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = ActType<T>::pack(__uint_as_float(v[8 * q + 2 * e]), __uint_as_float(v[8 * q + 2 * e + 1]));
        *reinterpret_cast<uint4*>(staged(buf, row, piece0 + q)) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}
__device__ __forceinline__ void stage_codes32(uint8_t* buf, int row, int piece0, const uint32_t (&v)[32], float inv, bool checked) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = 16 * q + 4 * e;
            const float a = __uint_as_float(v[i]), b = __uint_as_float(v[i + 1]), c = __uint_as_float(v[i + 2]), d = __uint_as_float(v[i + 3]);
            w[e] = checked ? act_codes4_checked(a, b, c, d, inv) : act_codes4(a, b, c, d, inv);
        }
        *reinterpret_cast<uint4*>(staged(buf, row, piece0 + q)) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

template <int ACT>
__device__ __forceinline__ void gated32(uint32_t (&g)[32], const uint32_t (&u)[32]) {       // h in the place of g
#pragma unroll
    for (int i = 0; i < 32; ++i) g[i] = __float_as_uint(gate_value<ACT>(__uint_as_float(g[i])) * __uint_as_float(u[i]));
}

// The factor of an fp16 backward pass's results, which are then rounded; nothing in bf16.
template <typename T>
constexpr bool kFactor = ActType<T>::kTop < 1e5f;
template <typename T>
__device__ __forceinline__ float factor_of(const float* p) {
    if constexpr (kFactor<T>) return __ldcg(p);
    else return 1.0f;
}
template <typename T, int N>
__device__ __forceinline__ void times(uint32_t (&v)[N], float factor) {
    if constexpr (kFactor<T>) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * factor);
    }
}

// First step of share i of n.  (At most 2^25 steps and 16 shares.)
__device__ __forceinline__ int share_at(int steps, int i, int n) { return n == 1 ? i * steps : static_cast<int>(static_cast<uint32_t>(steps) * i / n); }

struct Tile { int m, n; };
__device__ __forceinline__ Tile tile_at(int t, int tiles_m, int tiles_n) {
    const int per_group = kGroupM * tiles_n;
    const int g = t / per_group, first = g * kGroupM, size = min(kGroupM, tiles_m - first), r = t - g * per_group;
    return {first + r % size, r / size};
}

// A pair's i-th piece of work: a share of a tile.  Backward: the items of dx, which are long, go round the pairs first.  Those
// of dw follow: where the last round of dx leaves pairs without an item, they take `early` ones of dw in its place; then all take
// turns, in an order that begins with them.  (dx and dw in launches of their own, each with a last round that is partly idle: 500
// rows of 4096 x 14336 211 us, 4096 rows 1368; in one: 198 and 1329.)
struct Item {
    bool any, dw;
    int sel, share;                              // dw: 0 dWg, 1 dWu
    Tile tile;                                   // of the result
    int st0, steps;                              // stages of the contraction; dx: dg Wg, then du Wu
};
__host__ __device__ __forceinline__ constexpr int ceil_to(int v, int n) { return (v + n - 1) / n; }
template <int KIND>
__device__ __forceinline__ Item item_at(const FfnArgs& p, int pair, int npairs, int i) {
    Item it = {};
    if constexpr (KIND == FK_FWD) {
        const int tiles_m = ceil_to(p.m, 2 * kHalf), tiles_n = ceil_to(p.f, p.w), t = pair + i * npairs;
        it.any = t < tiles_m * tiles_n;
        it.tile = tile_at(t, tiles_m, tiles_n);
        it.steps = ceil_to(p.k, kBK);
    } else {
        const int tiles_n = ceil_to(p.k, 2 * kHalf), tiles_x = ceil_to(p.m, 2 * kHalf) * tiles_n, tm = ceil_to(p.f, 2 * kHalf), tiles_w = 2 * tm * tiles_n;
        const int items_x = KIND == FK_BWD ? tiles_x * p.shares[0] : 0, rounds = items_x / npairs, last = items_x - rounds * npairs;   // pairs 0..last-1 have one more
        const bool more = pair < last;
        const int mine = rounds + more;
        if (KIND == FK_BWD && i < mine) {
            const int t = pair + i * npairs, n = p.shares[0], steps = 2 * ceil_to(p.f, kBK);
            it.any = true;
            it.share = n == 1 ? 0 : t / tiles_x;
            it.tile = tile_at(t - it.share * tiles_x, ceil_to(p.m, 2 * kHalf), tiles_n);
            it.st0 = share_at(steps, it.share, n);
            it.steps = share_at(steps, it.share + 1, n) - it.st0;
        } else {
            const int j = i - mine, n = p.shares[1], steps = ceil_to(p.m, kBK);
            int t;
            if (KIND == FK_DW) t = pair + i * npairs;
            else if (more) t = p.early * (npairs - last) + j * npairs + npairs - last + pair;
            else if (j < p.early) t = j * (npairs - last) + pair - last;
            else t = p.early * (npairs - last) + (j - p.early) * npairs + pair - last;
            it.any = t < tiles_w * n;
            if (!it.any) return it;
            it.dw = true;
            it.share = n == 1 ? 0 : t / tiles_w;
            it.tile = tile_at(t - it.share * tiles_w, 2 * tm, tiles_n);          // the tiles of dWg, then those of dWu
            it.sel = it.tile.m >= tm;
            it.tile.m -= it.sel * tm;
            it.st0 = share_at(steps, it.share, n);
            it.steps = share_at(steps, it.share + 1, n) - it.st0;
        }
    }
    return it;
}

// KIND as above; T fp16 or bf16; ACT the gate (forward only); SAVE writes the codes of g and u (forward only).
template <int KIND, typename T, int ACT, bool SAVE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
tb200_k_ffn_pair(const __grid_constant__ FfnMaps<KIND> maps, const __grid_constant__ FfnArgs p) {
    constexpr int S = stages_of(KIND), kPlaces = places_of(KIND), kStaging = kPlaces * (kStagingBytes / 2);
    static_assert(S * kStageBytes + 4 * kStaging <= 6 * kStageBytes + 4 * kStagingBytes, "shared memory");
    const int tile_cols = KIND == FK_FWD ? p.w : 2 * kHalf;     // columns of the result that a tile covers
    const int b_bytes = KIND == FK_FWD ? p.w * 128 : kOperandBytes;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* staging = smem + S * kStageBytes;
    uint32_t* amax = reinterpret_cast<uint32_t*>(staging + 4 * kStaging);      // [quarter][g, u][row], bits of non-negative numbers
    uint64_t* bar_full = reinterpret_cast<uint64_t*>(staging + 4 * kStaging + kAmaxBytes);
    uint64_t* bar_empty = bar_full + S;
    uint64_t* bar_afull = bar_empty + S;          // [2] accumulator complete
    uint64_t* bar_aempty = bar_afull + 2;         // [2] accumulator read (the epilogue warps of both CTAs)
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar_aempty + 2);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int rank = static_cast<int>(cluster_ctarank());       // 0 = leader
    const int pair = blockIdx.x >> 1;
    const int npairs = gridDim.x >> 1;

    let_next_begin();
    if (SAVE && threadIdx.x < kAmaxBytes / 4) amax[threadIdx.x] = 0;
    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(&bar_full[s], 1);
            mbar_init(&bar_empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&bar_afull[b], 1);
            mbar_init(&bar_aempty[b], 2 * kEpiWarps);
        }
        mbar_fence_init();
        const CUtensorMap* all = reinterpret_cast<const CUtensorMap*>(&maps);
        for (int i = 0; i < static_cast<int>(sizeof(maps) / sizeof(CUtensorMap)); ++i) tma_prefetch_desc(all + i);
    }
    if (warp == 1) {
        tmem_alloc_pair(tmem_slot, kTmemCols);
        tmem_relinquish_pair();
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();                                          // the peer's barriers exist before anything signals them
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    wait_for_previous();

    if (warp == 0) {
        // ---------------- TMA producer (both CTAs) ----------------
        if (lane == 0) {
            uint32_t s = 0, ph = 1;
            bool ok = true;
            const int KB = ceil_to(p.f, kBK);                    // stages of one of dx's products
            for (int i = 0; ok; ++i) {
                const Item it = item_at<KIND>(p, pair, npairs, i);
                if (!it.any) break;
                const int a_row = it.tile.m * 2 * kHalf + rank * kHalf;
                const int b_col = KIND == FK_FWD ? it.tile.n * tile_cols : it.tile.n * 2 * kHalf + rank * kHalf;
                // one loop per kind of item: the loops are what paces the pair, and carry no choice
                auto load = [&](auto dw) {
                    for (int st = it.st0; st < it.st0 + it.steps; ++st) {
                        if (!mbar_wait(&bar_empty[s], ph, ST_WAIT_SMEM_EMPTY, st)) { ok = false; break; }
                        uint8_t* stage = smem + s * kStageBytes;
                        if (rank == 0) mbar_expect_tx(&bar_full[s], 2 * (kOperandBytes + b_bytes));  // both CTAs' bytes
                        if constexpr (KIND == FK_FWD) {
                            tma_load_2d_pair(stage, &maps.a[0], &bar_full[s], st * kBK, a_row);
                            tma_load_2d_pair(stage + kOperandBytes, &maps.b[rank], &bar_full[s], st * kBK, b_col);
                        } else if constexpr (dw) {
                            tma_load_2d_pair(stage, &maps.at[it.sel], &bar_full[s], a_row, st * kBK);
                            tma_load_2d_pair(stage + kAtomBytes, &maps.at[it.sel], &bar_full[s], a_row + 64, st * kBK);
                            tma_load_2d_pair(stage + kOperandBytes, &maps.x, &bar_full[s], b_col, st * kBK);
                            tma_load_2d_pair(stage + kOperandBytes + kAtomBytes, &maps.x, &bar_full[s], b_col + 64, st * kBK);
                        } else {
                            const int prod = st >= KB ? 1 : 0, k0 = (st - prod * KB) * kBK;
                            tma_load_2d_pair(stage, &maps.a[prod], &bar_full[s], k0, a_row);
                            tma_load_2d_pair(stage + kOperandBytes, &maps.b[prod], &bar_full[s], b_col, k0);
                            tma_load_2d_pair(stage + kOperandBytes + kAtomBytes, &maps.b[prod], &bar_full[s], b_col + 64, k0);
                        }
                        if (++s == S) { s = 0; ph ^= 1; }
                    }
                };
                if (KIND == FK_DW || (KIND == FK_BWD && it.dw)) load(std::true_type());
                else if (KIND != FK_DW) load(std::false_type());
            }
            if (!ok) {
                // copies in flight land within microseconds; a bounded pause before the CTA may exit
                const long long t0 = clock64();
                while (clock64() - t0 < (1ll << 21)) {}
            }
        }
    } else if (warp == 1 && rank == 0) {
        // ---------------- MMA issuer (leader only; the whole warp walks the loop, lane 0 issues by predication) ------
        constexpr uint32_t fmt = sizeof(T) == 2 && ActType<T>::kTop > 1e6f ? 1u : 0u;            // 1 = bf16, 0 = fp16
        const uint32_t idesc0 = umma_idesc(fmt, fmt, 2 * kHalf, KIND == FK_FWD ? 2 * tile_cols : 2 * kHalf) | (KIND != FK_FWD ? 1u << 16 : 0u);
        constexpr uint32_t kStageDesc = kStageBytes >> 4;
        // 16 of the 64 contraction elements per MMA: 32 bytes along a K-major row, 16 rows of an MN-major box
        constexpr uint64_t kAlongRow = 2, kDownBox = 16 * 128 / 16, b_step = KIND != FK_FWD ? kDownBox : kAlongRow;
        const bool leader = lane == 0;
        const uint64_t b_desc0 = KIND != FK_FWD ? desc_mn(smem_u32(smem) + kOperandBytes) : umma_desc_sw128(smem_u32(smem) + kOperandBytes);
        uint32_t s = 0, ph = 0, cnt = 0;
        bool ready = false;
        bool ok = true;
        for (; ok; ++cnt) {
            const Item it = item_at<KIND>(p, pair, npairs, cnt);
            if (!it.any) break;
            const uint32_t acc = cnt & 1;
            if (!mbar_wait(&bar_aempty[acc], ((cnt >> 1) & 1) ^ 1, ST_WAIT_TMEM_EMPTY, cnt)) { ok = false; break; }
            tc_fence_after();
            const uint32_t d_tmem = tmem_base + acc * 256;
            auto multiply = [&](auto dw) {
                const uint32_t idesc = idesc0 | (dw ? 1u << 15 : 0u);
                const uint64_t a_desc0 = dw ? desc_mn(smem_u32(smem)) : umma_desc_sw128(smem_u32(smem));
                constexpr uint64_t a_step = dw ? kDownBox : kAlongRow;
                for (int st = 0; st < it.steps; ++st) {
                    if (!ready && !mbar_wait(&bar_full[s], ph, ST_WAIT_SMEM_FULL, st)) { ok = false; break; }
                    tc_fence_after();
                    const uint64_t a_desc = a_desc0 + s * kStageDesc;
                    const uint64_t b_desc = b_desc0 + s * kStageDesc;
                    uint64_t* const freed = &bar_empty[s];
                    if (++s == static_cast<uint32_t>(S)) { s = 0; ph ^= 1; }
                    mma_pair_if(leader, d_tmem, a_desc, b_desc, idesc, st > 0 ? 1u : 0u);
                    ready = mbar_test_wait(&bar_full[s], ph);
#pragma unroll
                    for (int k = 1; k < 4; ++k) mma_pair_if(leader, d_tmem, a_desc + k * a_step, b_desc + k * b_step, idesc, 1u);
                    if (leader) tc_commit_pair(freed, 0x3);
                }
            };
            if (KIND == FK_DW || (KIND == FK_BWD && it.dw)) multiply(std::true_type());
            else if (KIND != FK_DW) multiply(std::false_type());
            if (ok && leader) tc_commit_pair(&bar_afull[acc], 0x3);
        }
    } else if (warp >= 4) {
        // ---------------- epilogue (both CTAs; each owns 128 rows of the tile, each warp 32 rows of a quarter of the columns) ----
        const int quarter = (warp - 4) & 3, part = (warp - 4) >> 2, r8 = 8 * part;
        uint8_t* buf = staging + quarter * kStaging;
        const uint32_t t_lane = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
        const float factor = KIND == FK_FWD ? 1.0f : factor_of<T>(p.factor);
        uint32_t cnt = 0;
        bool ok = true;
        for (;; ++cnt) {
            const Item it = item_at<KIND>(p, pair, npairs, cnt);
            if (!it.any) break;
            const uint32_t acc = cnt & 1;
            const int all_rows = KIND != FK_FWD && it.dw ? p.f : p.m, all_cols = KIND == FK_FWD ? p.f : p.k;
            const int row0 = it.tile.m * 2 * kHalf + rank * kHalf + quarter * 32;                 // the quarter's first row
            const int rows = all_rows - row0;                                                     // valid rows (may be <= 0)
            const int col0 = it.tile.n * tile_cols, cols = all_cols - col0;
            const uint32_t t_acc = t_lane + acc * 256;
            // a wait that gave up ends the waiting, not the walk: the warps meet at barriers below
            ok = ok && mbar_wait(&bar_afull[acc], (cnt >> 1) & 1, ST_WAIT_TMEM_FULL, cnt);
            tc_fence_after();
            auto release = [&] {                                                                  // the warp has read its part of the accumulator
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_leader(&bar_aempty[acc]);
            };
            if constexpr (KIND == FK_FWD) {
                // columns [at, at + 32) of the tile; what lies beyond its w columns belongs to nobody and is not stored
                const int at = part * ((tile_cols / 4 + 7) / 8 * 8);
                const uint32_t t_g = t_acc + at, t_u = t_acc + tile_cols + at;
                uint32_t g[32], u[32];
                tmem_ld32(t_g, g);
                tmem_ld32(t_u, u);
                tmem_wait_ld();
                uint32_t* const row_amax = amax + quarter * 64 + lane;
                if constexpr (SAVE) {
                    float a = 0.0f, b = 0.0f;
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        a = fmaxf(a, fabsf(__uint_as_float(g[i])));
                        b = fmaxf(b, fabsf(__uint_as_float(u[i])));
                    }
                    atomicMax(row_amax, __float_as_uint(a));
                    atomicMax(row_amax + 32, __float_as_uint(b));
                } else {
                    release();
                }
                gated32<ACT>(g, u);
                stage32<T>(buf, lane, at / 8, g);
                quarter_sync(quarter);
                float ag = 0.0f, au = 0.0f;
                if constexpr (SAVE) {
                    ag = __uint_as_float(row_amax[0]);
                    au = __uint_as_float(row_amax[32]);
                }
                flush<T, 16>(buf, 0, static_cast<T*>(p.out[0]) + static_cast<int64_t>(row0) * p.f + col0, p.f, r8, rows, min(cols, tile_cols), lane);
                quarter_sync(quarter);
                if constexpr (SAVE) {
                    tmem_ld32(t_g, g);
                    tmem_ld32(t_u, u);
                    tmem_wait_ld();
                    release();
                    const bool infinite = __any_sync(0xffffffffu, fmaxf(ag, au) > FLT_MAX);       // the same in the quarter's warps
                    if (infinite) {                              // once more, over the finite values
                        if (part == 0) row_amax[0] = row_amax[32] = 0;
                        quarter_sync(quarter);
                        float a = 0.0f, b = 0.0f;
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            a = fmaxf(a, act_size(__uint_as_float(g[i])));
                            b = fmaxf(b, act_size(__uint_as_float(u[i])));
                        }
                        atomicMax(row_amax, __float_as_uint(a));
                        atomicMax(row_amax + 32, __float_as_uint(b));
                        quarter_sync(quarter);
                        ag = __uint_as_float(row_amax[0]);
                        au = __uint_as_float(row_amax[32]);
                    }
                    const float2 sg = act_scale(ag), su = act_scale(au);
                    const int64_t nblk = ceil_to(p.f, kHalf);
                    if (part < 2 && lane < rows) p.scales[part][(row0 + lane) * nblk + it.tile.n] = part == 0 ? sg.x : su.x;
                    stage_codes32(buf, lane, 2 * part, g, sg.y, infinite);
                    stage_codes32(buf, lane, 8 + 2 * part, u, su.y, infinite);
                    quarter_sync(quarter);
                    if (part == 0) row_amax[0] = row_amax[32] = 0;                                // all have read it, none adds before the next barrier
                    const int64_t to = static_cast<int64_t>(row0) * p.f + col0;
                    flush<uint8_t, 8>(buf, 0, p.codes[0] + to, p.f, r8, rows, cols, lane);
                    flush<uint8_t, 8>(buf, 8, p.codes[1] + to, p.f, r8, rows, cols, lane);
                    quarter_sync(quarter);
                }
            } else if (KIND == FK_BWD && p.shares[it.dw] > 1) {                    // partial sums in 32 bits, 64 columns at a time
                float* dst = p.sums[it.dw] + (static_cast<int64_t>(it.dw ? 2 * it.share + it.sel : it.share) * all_rows + row0) * p.k + col0;
                if (part == 0 && lane == 0) tma_store_wait_read<0>();     // the item before may have been stored by TMA
                quarter_sync(quarter);
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                    uint32_t v[16];
                    tmem_ld16(t_acc + c * 64 + part * 16, v);
                    tmem_wait_ld();
                    if (c == 3) release();
#pragma unroll
                    for (int q = 0; q < 4; ++q) *reinterpret_cast<uint4*>(staged(buf, lane, 4 * part + q)) = make_uint4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
                    quarter_sync(quarter);
                    flush<float, 16>(buf, 0, dst + c * 64, p.k, r8, rows, cols - c * 64, lane);
                    quarter_sync(quarter);
                }
            } else {
                // By TMA, which leaves out what lies beyond the result: 32 rows x 64 columns a copy, in the 128-byte swizzle, from the
                // places of the quarter's staging area in turn; its first lane, which issues the copies, waits for the place's last one.
                // Rows that do not begin on 32-byte boundaries are written by the warps, 256 bytes of a row at once: copies of 128
                // would leave twice as many sectors half written (6 rows of 7192 -> 28637: 221 us where this takes 182).
                const int which = it.dw ? 1 + it.sel : 0;
                if (p.k % 16 == 0) {
                    const bool issuer = part == 0 && lane == 0;
                    uint32_t v[4][16];
#pragma unroll
                    for (int c = 0; c < 4; ++c) tmem_ld16(t_acc + c * 64 + part * 16, v[c]);
                    tmem_wait_ld();
                    release();
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        times<T>(v[c], factor);
                        uint8_t* area = buf + c % kPlaces * (kStagingBytes / 2);
                        if (issuer) tma_store_wait_read<kPlaces - 1>();   // all but the other places'
                        quarter_sync(quarter);
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            uint32_t w[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) w[e] = ActType<T>::pack(__uint_as_float(v[c][8 * q + 2 * e]), __uint_as_float(v[c][8 * q + 2 * e + 1]));
                            *reinterpret_cast<uint4*>(area + lane * 128 + (((2 * part + q) ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                        fence_async_smem();
                        quarter_sync(quarter);
                        if (issuer) {
                            if (rows > 0 && c * 64 < cols) tma_store_2d(&maps.out[which], area, col0 + c * 64, row0);
                            tma_store_commit();
                        }
                    }
                } else {
                    uint32_t v[2][32];
                    tmem_ld32(t_acc + part * 32, v[0]);
                    tmem_ld32(t_acc + kHalf + part * 32, v[1]);
                    tmem_wait_ld();
                    release();
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        times<T>(v[c], factor);
                        stage32<T>(buf, lane, 4 * part, v[c]);
                        quarter_sync(quarter);
                        flush<T, 16>(buf, 0, static_cast<T*>(p.out[which]) + static_cast<int64_t>(row0) * p.k + col0 + c * kHalf, p.k, r8, rows, cols - c * kHalf, lane);
                        quarter_sync(quarter);
                    }
                }
            }
        }
        if (KIND != FK_FWD && part == 0 && lane == 0) tma_store_wait<0>();
    }

    // neither CTA may leave while the other can still read its shared memory or signal its barriers
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    tc_fence_after();
    if (warp == 1) {
        __syncwarp();
        tmem_dealloc_pair(tmem_base, kTmemCols);
    }
}

// ------------------------------------------------------------------------------------------------
// Forward block for a decoding batch (m <= 128 rows): bound by reading the weights, so every SM has to stream an equal share of
// them.  One CTA per tile of 128 rows x w hidden units (N = 2 w: w rows of Wg, w rows of Wu), with w, a multiple of 8, chosen per
// call so that the tiles fill one wave (or whole waves) of SMs.  More rows, in blocks of 128, where f is small.  Where f is too
// small for that, the CTAs of a cluster share the contraction of a tile (SPLIT): each leaves its sums in its shared
// memory, and each adds up a share of the columns in a fixed order, reading its peers' memory.
constexpr int kMaxStages = 8;
struct MidMaps { CUtensorMap x, wg, wu; };
struct MidArgs {
    void* h;
    int m, f, depth;
    int w, stages, x_rows;                       // hidden units per tile, stages in shared memory, rows of x per copy
    uint8_t* codes[2];                           // with checkpoints: codes of g and u, [m, f]
    float* scales[2];                            // and their scales, [m, ceil(f / 128)]
};
constexpr int kFewRows = 64, kFewCols = 128;     // rows of x, and columns of an accumulator, in the form for few rows
constexpr int kFewSums = kFewRows * 2 * kHalf * 4;
constexpr int kMidRing = 192 * 1024;             // in the form for few rows the sums take 32 KB of it beside the staging area
constexpr int kMidSmemBytes = kMidRing + 4 * kStagingBytes + kBarBytes + 1024;

__device__ __forceinline__ float4 peer_float4(uint32_t addr, uint32_t rank) {
    uint32_t at;
    float4 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(addr), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
    return v;
}

// g and u of four neighbouring hidden units c.. of row r, from sums that lie row by row, `pitch` apart, g first and u `w` on: in
// this CTA (SHARES = 1), or added up over the CTAs of the cluster.
template <int SHARES>
__device__ __forceinline__ void gather4(uint32_t base, int pitch, int w, int r, int c, float (&g)[4], float (&u)[4]) {
    const uint32_t at = base + 4 * (r * pitch + c);
    float4 gs[SHARES], us[SHARES];
#pragma unroll
    for (int o = 0; o < SHARES; ++o) {
        if constexpr (SHARES > 1) {
            gs[o] = peer_float4(at, o);
            us[o] = peer_float4(at + 4 * w, o);
        } else {
            const uint4 a = shared_uint4(at), b = shared_uint4(at + 4 * w);
            gs[o] = make_float4(__uint_as_float(a.x), __uint_as_float(a.y), __uint_as_float(a.z), __uint_as_float(a.w));
            us[o] = make_float4(__uint_as_float(b.x), __uint_as_float(b.y), __uint_as_float(b.z), __uint_as_float(b.w));
        }
    }
#pragma unroll
    for (int o = 1; o < SHARES; ++o) {
        gs[0].x += gs[o].x; gs[0].y += gs[o].y; gs[0].z += gs[o].z; gs[0].w += gs[o].w;
        us[0].x += us[o].x; us[0].y += us[o].y; us[0].z += us[o].z; us[0].w += us[o].w;
    }
    g[0] = gs[0].x; g[1] = gs[0].y; g[2] = gs[0].z; g[3] = gs[0].w;
    u[0] = us[0].x; u[1] = us[0].y; u[2] = us[0].z; u[3] = us[0].w;
}
// h of them, for row r and the result's columns col..; vec: four can be stored at once.
template <typename T, int ACT>
__device__ __forceinline__ void store4(const float (&g)[4], const float (&u)[4], T* __restrict__ out, int r, int col, int f, bool vec) {
    const float v[4] = {gate_value<ACT>(g[0]) * u[0], gate_value<ACT>(g[1]) * u[1], gate_value<ACT>(g[2]) * u[2], gate_value<ACT>(g[3]) * u[3]};
    T* h = out + static_cast<int64_t>(r) * f + col;
    if (vec && col < f) {
        *reinterpret_cast<uint2*>(h) = make_uint2(ActType<T>::pack(v[0], v[1]), ActType<T>::pack(v[2], v[3]));
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (col + e < f) h[e] = ActType<T>::store(v[e]);
    }
}
// Scale and codes of a row's 1 x 128 block, four numbers per lane of a warp.
__device__ __forceinline__ void save4(const float (&v)[4], uint8_t* __restrict__ codes, float* __restrict__ scale, int col, int f, bool vec, int lane) {
    float amax = fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    const bool infinite = amax > FLT_MAX;                        // the same in all lanes
    if (infinite) {
        amax = fmaxf(fmaxf(act_size(v[0]), act_size(v[1])), fmaxf(act_size(v[2]), act_size(v[3])));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    }
    const float2 s = act_scale(amax);
    const uint32_t c = infinite ? act_codes4_checked(v[0], v[1], v[2], v[3], s.y) : act_codes4(v[0], v[1], v[2], v[3], s.y);
    if (vec && col < f) {
        *reinterpret_cast<uint32_t*>(codes + col) = c;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (col + e < f) codes[col + e] = static_cast<uint8_t>(c >> (8 * e));
    }
    if (lane == 0) *scale = s.x;
}

// FEW: at most 64 rows.  The weights are the operand of 128 rows then (2 w rows, one or two blocks) and x that of 16 to 64
// columns, so that the tensor cores multiply by little that is not there: at 1 row of 4096 -> 14336, 128 rows of x cost 43.6 us a
// pass at the board's power limit, this form 39.6.
// SAVE (with FEW, tiles of 128 hidden units): a warp takes a row of the tile, which is one block of g and of u.
template <typename T, int ACT, int SHARES, bool FEW, bool SAVE>
__global__ void __launch_bounds__(kThreads, 1) tb200_k_ffn_mid(const __grid_constant__ MidMaps maps, const __grid_constant__ MidArgs p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* staging = smem + kMidRing;
    uint8_t* few_sums = staging + 4 * kStagingBytes - kFewSums;
    uint64_t* bar_full = reinterpret_cast<uint64_t*>(staging + 4 * kStagingBytes);
    uint64_t* bar_empty = bar_full + kMaxStages;
    uint64_t* bar_afull = bar_empty + kMaxStages;
    uint64_t* bar_aempty = bar_afull + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar_aempty + 2);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int S = p.stages, w = p.w;
    const int x_bytes = p.x_rows * 128, stage_bytes = x_bytes + 2 * w * 128;
    const int KB = (p.depth + kBK - 1) / kBK;
    constexpr bool SPLIT = SHARES > 1;
    const int share = SPLIT ? static_cast<int>(cluster_ctarank()) : 0;
    const int kb0 = KB * share / SHARES, kb1 = KB * (share + 1) / SHARES;
    const int blocks = FEW ? 1 : (p.m + kHalf - 1) / kHalf;      // of 128 rows; a tile's are neighbours, so that they share its weights in L2
    const int tiles = (p.f + w - 1) / w * blocks;
    const int t0 = static_cast<int>(blockIdx.x) / SHARES;
    const int t_step = SPLIT ? tiles : static_cast<int>(gridDim.x);                 // with SPLIT a CTA has one tile
    const bool vec = p.f % 4 == 0 && (reinterpret_cast<uintptr_t>(p.h) & 7) == 0 &&  // four of a row's results can be stored at once
                     ((reinterpret_cast<uintptr_t>(p.codes[0]) | reinterpret_cast<uintptr_t>(p.codes[1])) & 3) == 0;
    auto save_row = [&](uint32_t base, int pitch, int r, int t) {
        float g[4], u[4];
        gather4<SHARES>(base, pitch, kHalf, r, 4 * lane, g, u);
        const int col = t * kHalf + 4 * lane;
        const int64_t row = static_cast<int64_t>(r) * p.f, blk = static_cast<int64_t>(r) * ((p.f + kHalf - 1) / kHalf) + t;
        store4<T, ACT>(g, u, static_cast<T*>(p.h), r, col, p.f, vec);
        save4(g, p.codes[0] + row, p.scales[0] + blk, col, p.f, vec, lane);
        save4(u, p.codes[1] + row, p.scales[1] + blk, col, p.f, vec, lane);
    };

    let_next_begin();
    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(&bar_full[s], 1);
            mbar_init(&bar_empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&bar_afull[b], 1);
            mbar_init(&bar_aempty[b], kEpiWarps);
        }
        mbar_fence_init();
        tma_prefetch_desc(&maps.x);
        tma_prefetch_desc(&maps.wg);
        tma_prefetch_desc(&maps.wu);
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    if (warp == 0 && lane == 0 && t0 < tiles) {
        // the weights of the first stages, while the kernel before ends
        for (int kb = kb0; kb < min(kb1, kb0 + S); ++kb) {
            prefetch_2d(&maps.wg, kb * kBK, t0 / blocks * w);
            prefetch_2d(&maps.wu, kb * kBK, t0 / blocks * w);
        }
    }
    wait_for_previous();

    if (warp == 0) {
        // ---------------- TMA producer ----------------
        if (lane == 0) {
            uint32_t s = 0, ph = 1;
            bool ok = true;
            for (int t = t0; t < tiles && ok; t += t_step) {
                const int unit = t / blocks * w, row = t % blocks * kHalf;
                for (int kb = kb0; kb < kb1; ++kb) {
                    if (!mbar_wait(&bar_empty[s], ph, ST_WAIT_SMEM_EMPTY, kb)) { ok = false; break; }
                    uint8_t* stage = smem + s * stage_bytes;
                    mbar_expect_tx(&bar_full[s], stage_bytes);
                    tma_load_2d(stage + x_bytes, &maps.wg, &bar_full[s], kb * kBK, unit);
                    tma_load_2d(stage + x_bytes + w * 128, &maps.wu, &bar_full[s], kb * kBK, unit);
                    tma_load_2d(stage, &maps.x, &bar_full[s], kb * kBK, row);
                    if (++s == static_cast<uint32_t>(S)) { s = 0; ph ^= 1; }
                }
            }
            if (!ok) {
                // copies in flight land within microseconds; a bounded pause before the CTA may exit
                const long long c0 = clock64();
                while (clock64() - c0 < (1ll << 21)) {}
            }
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer ----------------
        // Rows of x beyond x_rows are whatever follows in shared memory: they reach only rows of the accumulator that
        // nothing reads.
        constexpr uint32_t fmt = ActType<T>::kTop > 1e6f ? 1u : 0u;
        const uint32_t idesc = FEW ? umma_idesc(fmt, fmt, kHalf, p.x_rows) : umma_idesc(fmt, fmt, kHalf, 2 * w);
        const bool leader = lane == 0;
        const uint64_t x_desc0 = umma_desc_sw128(smem_u32(smem)), w_desc0 = umma_desc_sw128(smem_u32(smem) + x_bytes);
        const uint64_t a_desc0 = FEW ? w_desc0 : x_desc0, b_desc0 = FEW ? x_desc0 : w_desc0;
        const bool two = FEW && 2 * w > kHalf;
        const uint32_t stage_desc = static_cast<uint32_t>(stage_bytes) >> 4;
        uint32_t s = 0, ph = 0, cnt = 0;
        bool ready = false;
        bool ok = true;
        for (int t = t0; t < tiles && ok; t += t_step, ++cnt) {
            const uint32_t acc = cnt & 1;
            if (!mbar_wait(&bar_aempty[acc], ((cnt >> 1) & 1) ^ 1, ST_WAIT_TMEM_EMPTY, t)) { ok = false; break; }
            tc_fence_after();
            const uint32_t d_tmem = tmem_base + acc * (FEW ? kFewCols : 256);
            for (int kb = kb0; kb < kb1; ++kb) {
                if (!ready && !mbar_wait(&bar_full[s], ph, ST_WAIT_SMEM_FULL, kb)) { ok = false; break; }
                tc_fence_after();
                const uint64_t a_desc = a_desc0 + s * stage_desc, b_desc = b_desc0 + s * stage_desc;
                uint64_t* const freed = &bar_empty[s];
                if (++s == static_cast<uint32_t>(S)) { s = 0; ph ^= 1; }
                mma_if(leader, d_tmem, a_desc, b_desc, idesc, kb > kb0 ? 1u : 0u);
                ready = mbar_test_wait(&bar_full[s], ph);
#pragma unroll
                for (int k = 1; k < 4; ++k) mma_if(leader, d_tmem, a_desc + 2 * k, b_desc + 2 * k, idesc, 1u);
                if (two) {                                       // rows 128.. of the weights, 16 KB on
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        mma_if(leader, d_tmem + kFewRows, a_desc + (kHalf * 128 >> 4) + 2 * k, b_desc + 2 * k, idesc, kb > kb0 || k > 0 ? 1u : 0u);
                }
                tc_commit_if(leader, freed);
            }
            if (ok && leader) tc_commit(&bar_afull[acc]);
        }
    } else if (warp >= 4) {
        // ---------------- epilogue: a warp has 32 rows (lanes) of a quarter of the columns ----------------
        const int quarter = (warp - 4) & 3, part = (warp - 4) >> 2, row0 = quarter * 32;
        uint8_t* buf = staging + quarter * kStagingBytes;
        const uint32_t t_lane = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
        uint32_t cnt = 0;
        bool ok = true;
        for (int t = t0; t < tiles; t += t_step, ++cnt) {
            const uint32_t acc = cnt & 1;
            // a wait that gave up ends the waiting, not the walk: the warps meet at barriers below
            ok = ok && mbar_wait(&bar_afull[acc], (cnt >> 1) & 1, ST_WAIT_TMEM_FULL, t);
            tc_fence_after();
            const uint32_t t_acc = t_lane + acc * (FEW ? kFewCols : 256);
            const int first_row = t % blocks * kHalf, rows = p.m - first_row;         // of the tile (may be more than 128)
            if constexpr (FEW) {
                // A lane has one row of the weights and 16 of the tokens at a time; the sums go token by token to where they are
                // combined: the ring (SPLIT, as below) or a place of their own.
                const int block = part >> 1, unit = kHalf * block + 32 * quarter + lane;
                const int pitch = SPLIT ? 2 * w + 4 : 2 * w;
                float* sums = reinterpret_cast<float*>(SPLIT ? smem : few_sums);
                for (int first = (part & 1) * 16; kHalf * block + 32 * quarter < 2 * w && first < p.m; first += 32) {
                    uint32_t v[16];
                    tmem_ld16(t_acc + block * kFewRows + first, v);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (unit < 2 * w && first + i < p.m) sums[(first + i) * pitch + unit] = __uint_as_float(v[i]);
                }
                if constexpr (!SPLIT) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&bar_aempty[acc]);
                    asm volatile("bar.sync 5, %0;" ::"n"(32 * kEpiWarps) : "memory");
                    if constexpr (SAVE) {
                        for (int r = warp - 4; r < p.m; r += kEpiWarps) save_row(smem_u32(sums), pitch, r, t);
                    } else {
                        const int quads = w / 4;
                        for (int i = threadIdx.x - 128; i < p.m * quads; i += 32 * kEpiWarps) {
                            const int r = i / quads, c = 4 * (i - r * quads);
                            float g[4], u[4];
                            gather4<1>(smem_u32(sums), pitch, w, r, c, g, u);
                            store4<T, ACT>(g, u, static_cast<T*>(p.h), r, t * w + c, p.f, vec);
                        }
                    }
                    asm volatile("bar.sync 5, %0;" ::"n"(32 * kEpiWarps) : "memory");
                }
            } else if constexpr (SPLIT) {
                // this CTA's sums, row by row.  A row pitch of 4 more than a multiple of 16 keeps eight lanes' (rows')
                // 16-byte pieces on different banks.  Every copy into the ring has landed and been used by the time the
                // accumulator is complete.
                if (row0 < rows) {
                    const int at = part * ((w / 2 + 7) / 8 * 8), n = min((w / 2 + 7) / 8 * 8, 2 * w - at);
                    float* mine = reinterpret_cast<float*>(smem) + (row0 + lane) * (2 * w + 4) + at;
#pragma unroll 1
                    for (int c = 0; c < n; c += 16) {
                        uint32_t v[16];
                        tmem_ld16(t_acc + at + c, v);
                        tmem_wait_ld();
                        if (row0 + lane < rows) {
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                if (c + 4 * i < n) *reinterpret_cast<uint4*>(mine + c + 4 * i) = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
                        }
                    }
                }
            } else {
                const int at = part * ((w / 4 + 7) / 8 * 8);
                if (row0 < rows && at < w) {
                    uint32_t g[32], u[32];
                    tmem_ld32(t_acc + at, g);
                    tmem_ld32(t_acc + w + at, u);
                    tmem_wait_ld();
                    gated32<ACT>(g, u);
                    stage32<T>(buf, lane, at / 8, g);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bar_aempty[acc]);
                quarter_sync(quarter);
                flush<T, 16>(buf, 0, static_cast<T*>(p.h) + static_cast<int64_t>(first_row + row0) * p.f + t / blocks * w, p.f, 8 * part, rows - row0, min(w, p.f - t / blocks * w), lane);
                quarter_sync(quarter);
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if constexpr (SPLIT) {
        cluster_sync_all();                                      // every share of the sums is in place
        const int quads = w / 4, q0 = quads * share / SHARES, qn = quads * (share + 1) / SHARES - q0;
        const uint32_t base = smem_u32(smem);
        if constexpr (SAVE) {
            for (int r = share + SHARES * warp; r < p.m; r += SHARES * (kThreads / 32)) save_row(base, 2 * w + 4, r, t0);
        } else {
            const int first_row = t0 % blocks * kHalf, rows = min(kHalf, p.m - first_row), unit = t0 / blocks * w;
            T* const h = static_cast<T*>(p.h) + static_cast<int64_t>(first_row) * p.f;
            for (int i = threadIdx.x; i < rows * qn; i += kThreads) {
                const int r = i / qn, c = 4 * (q0 + i - r * qn);
                float g[4], u[4];
                gather4<SHARES>(base, 2 * w + 4, w, r, c, g, u);
                store4<T, ACT>(g, u, h, r, unit + c, p.f, vec);
            }
        }
        cluster_sync_all();                                      // no CTA leaves while a peer reads its memory
    }
    if (warp == 1) {
        __syncwarp();
        tmem_dealloc(tmem_base, kTmemCols);
    }
}

// ------------------------------------------------------------------------------------------------
// dx for few rows (m <= 64): bound by reading the weights, as the forward block of a decoding batch is.  The weights, read as
// stored, are the operand of 128 rows (128 columns of dx), dg and du the one of 16 to 64; one CTA has 128 columns of dx and
// a share of the contraction over both products.  Sums go to [shares, m, k] in 32 bits, neighbouring lanes on neighbouring
// columns.  (4 rows of 4096 x 14336: 48 us, the pair kernel's 256-row tiles 60; at 100 of 2048 x 5632 it was 22 against 19.)
struct DxFewMaps { CUtensorMap d[2], w[2]; };    // dg, du; Wg, Wu
struct DxFewArgs {
    void* dx;                                    // with one share
    float* sums;                                 // with more
    int m, k, depth, shares;
    int rows, stages;                            // of dg per copy: m rounded up to 16; in shared memory
    const float* factor;                         // in fp16: of dx, where there is one share
};
constexpr int kDxCols = kFewRows;                     // columns of an accumulator
constexpr int kDxRing = 192 * 1024;
constexpr int kDxThreads = 256;
constexpr int kDxSmemBytes = kDxRing + kBarBytes + 1024;

template <typename T>
__global__ void __launch_bounds__(kDxThreads, 1) tb200_k_ffn_dx_few(const __grid_constant__ DxFewMaps maps, const __grid_constant__ DxFewArgs p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* bar_full = reinterpret_cast<uint64_t*>(smem + kDxRing);
    uint64_t* bar_empty = bar_full + kMaxStages;
    uint64_t* bar_afull = bar_empty + kMaxStages;
    uint64_t* bar_aempty = bar_afull + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar_aempty + 2);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int S = p.stages, d_bytes = p.rows * 128, stage_bytes = kOperandBytes + d_bytes;
    const int KB = (p.depth + kBK - 1) / kBK, steps = 2 * KB;
    const int tiles = (p.k + kHalf - 1) / kHalf, items = tiles * p.shares;

    let_next_begin();
    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(&bar_full[s], 1);
            mbar_init(&bar_empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&bar_afull[b], 1);
            mbar_init(&bar_aempty[b], 4);
        }
        mbar_fence_init();
        for (int i = 0; i < 2; ++i) {
            tma_prefetch_desc(&maps.d[i]);
            tma_prefetch_desc(&maps.w[i]);
        }
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, 2 * kDxCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    if (warp == 0 && lane == 0 && static_cast<int>(blockIdx.x) < items) {
        // the weights of the first stages, while the kernel before ends
        const int share = blockIdx.x / tiles, col = (blockIdx.x - share * tiles) * kHalf, st0 = share_at(steps, share, p.shares);
        for (int st = st0; st < min(st0 + S, share_at(steps, share + 1, p.shares)); ++st) {
            const int prod = st >= KB ? 1 : 0;
            prefetch_2d(&maps.w[prod], col, (st - prod * KB) * kBK);
            prefetch_2d(&maps.w[prod], col + 64, (st - prod * KB) * kBK);
        }
    }
    wait_for_previous();

    if (warp == 0) {
        // ---------------- TMA producer ----------------
        if (lane == 0) {
            uint32_t s = 0, ph = 1;
            bool ok = true;
            for (int t = blockIdx.x; t < items && ok; t += gridDim.x) {
                const int share = t / tiles, col = (t - share * tiles) * kHalf;
                for (int st = share_at(steps, share, p.shares); st < share_at(steps, share + 1, p.shares); ++st) {
                    if (!mbar_wait(&bar_empty[s], ph, ST_WAIT_SMEM_EMPTY, st)) { ok = false; break; }
                    uint8_t* stage = smem + s * stage_bytes;
                    mbar_expect_tx(&bar_full[s], stage_bytes);
                    const int prod = st >= KB ? 1 : 0, f0 = (st - prod * KB) * kBK;
                    tma_load_2d(stage, &maps.w[prod], &bar_full[s], col, f0);
                    tma_load_2d(stage + kAtomBytes, &maps.w[prod], &bar_full[s], col + 64, f0);
                    tma_load_2d(stage + kOperandBytes, &maps.d[prod], &bar_full[s], f0, 0);
                    if (++s == static_cast<uint32_t>(S)) { s = 0; ph ^= 1; }
                }
            }
            if (!ok) {
                // copies in flight land within microseconds; a bounded pause before the CTA may exit
                const long long c0 = clock64();
                while (clock64() - c0 < (1ll << 21)) {}
            }
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer ----------------
        constexpr uint32_t fmt = ActType<T>::kTop > 1e6f ? 1u : 0u;
        const uint32_t idesc = umma_idesc(fmt, fmt, kHalf, p.rows) | 1u << 15;                   // A is MN-major
        const bool leader = lane == 0;
        const uint64_t a_desc0 = desc_mn(smem_u32(smem)), b_desc0 = umma_desc_sw128(smem_u32(smem) + kOperandBytes);
        const uint32_t stage_desc = static_cast<uint32_t>(stage_bytes) >> 4;
        uint32_t s = 0, ph = 0, cnt = 0;
        bool ready = false;
        bool ok = true;
        for (int t = blockIdx.x; t < items && ok; t += gridDim.x, ++cnt) {
            const uint32_t acc = cnt & 1;
            if (!mbar_wait(&bar_aempty[acc], ((cnt >> 1) & 1) ^ 1, ST_WAIT_TMEM_EMPTY, t)) { ok = false; break; }
            tc_fence_after();
            const uint32_t d_tmem = tmem_base + acc * kDxCols;
            const int share = t / tiles, n = share_at(steps, share + 1, p.shares) - share_at(steps, share, p.shares);
            for (int st = 0; st < n; ++st) {
                if (!ready && !mbar_wait(&bar_full[s], ph, ST_WAIT_SMEM_FULL, st)) { ok = false; break; }
                tc_fence_after();
                const uint64_t a_desc = a_desc0 + s * stage_desc, b_desc = b_desc0 + s * stage_desc;
                uint64_t* const freed = &bar_empty[s];
                if (++s == static_cast<uint32_t>(S)) { s = 0; ph ^= 1; }
                mma_if(leader, d_tmem, a_desc, b_desc, idesc, st > 0 ? 1u : 0u);
                ready = mbar_test_wait(&bar_full[s], ph);
#pragma unroll
                for (int k = 1; k < 4; ++k) mma_if(leader, d_tmem, a_desc + k * (16 * 128 / 16), b_desc + 2 * k, idesc, 1u);
                tc_commit_if(leader, freed);
            }
            if (ok && leader) tc_commit(&bar_afull[acc]);
        }
    } else if (warp >= 4) {
        // ---------------- epilogue: a lane has one column of dx, a register one row ----------------
        const int quarter = warp - 4;
        const uint32_t t_lane = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
        const float factor = factor_of<T>(p.factor);
        uint32_t cnt = 0;
        bool ok = true;
        for (int t = blockIdx.x; t < items && ok; t += gridDim.x, ++cnt) {
            const uint32_t acc = cnt & 1;
            const int share = t / tiles, col = (t - share * tiles) * kHalf + quarter * 32 + lane;
            if (!mbar_wait(&bar_afull[acc], (cnt >> 1) & 1, ST_WAIT_TMEM_FULL, t)) { ok = false; break; }
            tc_fence_after();
#pragma unroll 1
            for (int r0 = 0; r0 < p.m; r0 += 16) {
                uint32_t v[16];
                tmem_ld16(t_lane + acc * kDxCols + r0, v);
                tmem_wait_ld();
                if (col < p.k) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        if (r0 + i < p.m) {
                            if (p.shares > 1) p.sums[(static_cast<int64_t>(share) * p.m + r0 + i) * p.k + col] = __uint_as_float(v[i]);
                            else static_cast<T*>(p.dx)[static_cast<int64_t>(r0 + i) * p.k + col] = ActType<T>::store(__uint_as_float(v[i]) * factor);
                        }
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar_aempty[acc]);
        }
    }

    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) {
        __syncwarp();
        tmem_dealloc(tmem_base, 2 * kDxCols);
    }
}

template <typename T>
constexpr CUtensorMapDataType tmap_type() { return ActType<T>::kTop > 1e6f ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16; }

// K-major operand: 128 rows x 64 of the contraction.  MN-major operand: 64 rows of the contraction x 64 columns.
template <typename T>
int map_k(CUtensorMap* m, const void* base, int64_t rows, int64_t cols, int64_t pitch, int box_rows = kHalf) {
    return encode_tmap_2d(m, base, tmap_type<T>(), 2, rows, cols, pitch * 2, box_rows, kBK, CU_TENSOR_MAP_SWIZZLE_128B);
}
template <typename T>
int map_mn(CUtensorMap* m, const void* base, int64_t rows, int64_t cols, int64_t pitch) {
    return encode_tmap_2d(m, base, tmap_type<T>(), 2, rows, cols, pitch * 2, kBK, 64, CU_TENSOR_MAP_SWIZZLE_128B);
}

// A result that is stored by TMA: 32 rows x 64 columns.
template <typename T>
int map_out(CUtensorMap* m, const void* base, int64_t rows, int64_t cols) {
    return encode_tmap_2d(m, base, tmap_type<T>(), 2, rows, cols, cols * 2, 32, 64, CU_TENSOR_MAP_SWIZZLE_128B);
}

// Pairs that the device holds at once.
template <int KIND, typename T, int ACT, bool SAVE>
int pairs_of(int* n) {
    auto kern = tb200_k_ffn_pair<KIND, T, ACT, SAVE>;
    static PerDeviceInt max_pairs_tab;
    int dev = 0;
    const int rc = current_device(&dev);
    if (rc != TB200_OK) return rc;
    int max_pairs = max_pairs_tab.v[dev].load(std::memory_order_acquire);
    if (max_pairs == 0) {
        TB200_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes));
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(static_cast<unsigned>(num_sms() & ~1), 1, 1);
        cfg.blockDim = dim3(kThreads, 1, 1);
        cfg.dynamicSmemBytes = kSmemBytes;
        TB200_CUDA_TRY(cudaOccupancyMaxActiveClusters(&max_pairs, kern, &cfg));
        if (max_pairs < 1) return fail(TB200_ERR_UNSUPPORTED, "ffn_gated: no CTA pair fits on this device");
        max_pairs_tab.v[dev].store(max_pairs, std::memory_order_release);
    }
    *n = max_pairs;
    return TB200_OK;
}

template <int KIND, typename T, int ACT, bool SAVE>
int launch_pair(const FfnMaps<KIND>& maps, const FfnArgs& args, int64_t items, cudaStream_t st) {
    int max_pairs = 0;
    const int rc = pairs_of<KIND, T, ACT, SAVE>(&max_pairs);
    if (rc != TB200_OK) return rc;
    if (items > 0x7fffffffll / kGroupM) return fail(TB200_ERR_UNSUPPORTED, "ffn_gated: too many tiles");
    const int pairs = static_cast<int>(items < max_pairs ? items : max_pairs);
    return launch_over_previous(tb200_k_ffn_pair<KIND, T, ACT, SAVE>, 2 * pairs, kThreads, kSmemBytes, 1, st, maps, args);
}

template <typename T, bool SAVE>
int launch_fwd(const FfnMaps<FK_FWD>& maps, const FfnArgs& args, int act, cudaStream_t st) {
    const int64_t items = static_cast<int64_t>(ceil_to(args.m, 2 * kHalf)) * ceil_to(args.f, args.w);
    switch (act) {
        case TB200_ACT_SILU: return launch_pair<FK_FWD, T, TB200_ACT_SILU, SAVE>(maps, args, items, st);
        case TB200_ACT_GELU: return launch_pair<FK_FWD, T, TB200_ACT_GELU, SAVE>(maps, args, items, st);
        case TB200_ACT_GELU_TANH: return launch_pair<FK_FWD, T, TB200_ACT_GELU_TANH, SAVE>(maps, args, items, st);
        default: return launch_pair<FK_FWD, T, TB200_ACT_RELU, SAVE>(maps, args, items, st);
    }
}

// ---- the decoding batch's tiles ----
struct MidPlan { int w, shares; float time; };

template <int SHARES>
int clusters_of(int* n) {                        // clusters of SHARES CTAs that the device holds at once
    static PerDeviceInt tab;
    int dev = 0;
    const int rc = current_device(&dev);
    if (rc != TB200_OK) return rc;
    *n = tab.v[dev].load(std::memory_order_acquire);
    if (*n == 0) {
        auto kern = tb200_k_ffn_mid<__nv_bfloat16, TB200_ACT_SILU, SHARES, false, false>;
        TB200_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMidSmemBytes));
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(static_cast<unsigned>(num_sms() / SHARES * SHARES), 1, 1);
        cfg.blockDim = dim3(kThreads, 1, 1);
        cfg.dynamicSmemBytes = kMidSmemBytes;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = SHARES;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        TB200_CUDA_TRY(cudaOccupancyMaxActiveClusters(n, kern, &cfg));
        if (*n < 1) *n = -1;
        tab.v[dev].store(*n, std::memory_order_release);
    }
    return TB200_OK;
}

// The width and the shares with the least time by a model fitted to measurements (1 to 128 rows, k 512..8192,
// f 512..28672; it picks within 8 % of the best measured plan).  A stage takes 0.25 us to issue whatever its size (0.37 in two
// blocks of weights), or what it takes to
// bring its bytes from L2 to the SM (95 GB/s each) or all CTAs' weights from HBM (6.4 TB/s); a wave takes its stages
// and 0.6 us; sharing costs 0.8 us and the peers' sums at 20 GB/s.
int mid_plan(int64_t m, int64_t f, int64_t k, int least_width, MidPlan* plan) {
    int clusters[4] = {num_sms(), 0, 0, 0};
    int rc = clusters_of<2>(&clusters[1]);
    if (rc == TB200_OK) rc = clusters_of<4>(&clusters[2]);
    if (rc == TB200_OK) rc = clusters_of<8>(&clusters[3]);
    if (rc != TB200_OK) return rc;
    const int KB = static_cast<int>((k + kBK - 1) / kBK), x_rows = static_cast<int>(m < kHalf ? (m + 7) / 8 * 8 : kHalf);
    const int64_t blocks = (m + kHalf - 1) / kHalf;
    float best = 0.0f;
    for (int i = 0; i < 4; ++i) {
        const int shares = 1 << i;
        if (shares > KB || clusters[i] < 1) break;               // every share has a stage
        for (int w = least_width; w <= kHalf; w += 8) {
            const int64_t tiles = (f + w - 1) / w * blocks;
            if (shares > 1 && tiles > clusters[i]) continue;     // shared tiles run in one wave: further ones, whose CTAs begin anew, gain nothing
            const int64_t waves = (tiles + clusters[i] - 1) / clusters[i], at_once = (tiles < clusters[i] ? tiles : clusters[i]) * shares;
            const float link = static_cast<float>(x_rows + 2 * w) * (128.0f / 95e3f), hbm = static_cast<float>(at_once) * (2 * w) * (128.0f / 6.4e6f) / static_cast<float>(blocks);
            const float stage = fmaxf(m <= kFewRows && 2 * w > kHalf ? 0.37f : 0.25f, fmaxf(link, hbm));
            const float t = static_cast<float>(waves) * static_cast<float>((KB + shares - 1) / shares) * stage +
                            (shares > 1 ? 0.8f + static_cast<float>(x_rows) * (8 * w) / 20e3f : 0.6f * static_cast<float>(waves) + 0.012f * w);
            if (best == 0.0f || t < best) {
                best = t;
                *plan = {w, shares, t};
            }
        }
    }
    return TB200_OK;
}

template <typename T, int ACT, int SHARES, bool FEW, bool SAVE>
int launch_mid(const MidMaps& maps, const MidArgs& args, cudaStream_t st) {
    auto kern = tb200_k_ffn_mid<T, ACT, SHARES, FEW, SAVE>;
    static PerDeviceInt attr_set;
    const int rc = ensure_max_smem(attr_set, reinterpret_cast<const void*>(kern), kMidSmemBytes);
    if (rc != TB200_OK) return rc;
    const int64_t tiles = static_cast<int64_t>((args.f + args.w - 1) / args.w) * ((args.m + kHalf - 1) / kHalf);
    if (tiles > 0x7fffffffll / 8) return fail(TB200_ERR_UNSUPPORTED, "ffn_gated: too many tiles");
    return launch_over_previous(kern, static_cast<int>(SHARES > 1 ? tiles * SHARES : tiles < num_sms() ? tiles : num_sms()), kThreads, kMidSmemBytes, SHARES, st, maps, args);
}

template <typename T, int ACT, bool FEW, bool SAVE>
int launch_mid_shares(const MidMaps& maps, const MidArgs& args, int shares, cudaStream_t st) {
    switch (shares) {
        case 1: return launch_mid<T, ACT, 1, FEW, SAVE>(maps, args, st);
        case 2: return launch_mid<T, ACT, 2, FEW, SAVE>(maps, args, st);
        case 4: return launch_mid<T, ACT, 4, FEW, SAVE>(maps, args, st);
        default: return launch_mid<T, ACT, 8, FEW, SAVE>(maps, args, st);
    }
}
template <typename T, bool FEW, bool SAVE>
int launch_mid_act(const MidMaps& maps, const MidArgs& args, int shares, int act, cudaStream_t st) {
    switch (act) {
        case TB200_ACT_SILU: return launch_mid_shares<T, TB200_ACT_SILU, FEW, SAVE>(maps, args, shares, st);
        case TB200_ACT_GELU: return launch_mid_shares<T, TB200_ACT_GELU, FEW, SAVE>(maps, args, shares, st);
        case TB200_ACT_GELU_TANH: return launch_mid_shares<T, TB200_ACT_GELU_TANH, FEW, SAVE>(maps, args, shares, st);
        default: return launch_mid_shares<T, TB200_ACT_RELU, FEW, SAVE>(maps, args, shares, st);
    }
}

template <typename T>
int ffn_mid(const void* x, const void* wg, const void* wu, void* h, void* gq, float* gs, void* uq, float* us, int64_t m, int64_t f, int64_t k,
            int64_t ldx, int act, const MidPlan& plan, cudaStream_t st) {
    MidArgs args = {};
    args.h = h;
    args.codes[0] = static_cast<uint8_t*>(gq);
    args.codes[1] = static_cast<uint8_t*>(uq);
    args.scales[0] = gs;
    args.scales[1] = us;
    args.m = static_cast<int>(m);
    args.f = static_cast<int>(f);
    args.depth = static_cast<int>(k);
    args.w = plan.w;
    const bool few = m <= kFewRows;
    args.x_rows = static_cast<int>(few ? (m + 15) / 16 * 16 : m < kHalf ? (m + 7) / 8 * 8 : kHalf);
    const int stage = (args.x_rows + 2 * plan.w) * 128;
    const int ring = few ? kMidRing + 4 * kStagingBytes - kFewSums : kMidRing;
    args.stages = ring / stage < kMaxStages ? ring / stage : kMaxStages;
    MidMaps maps;
    memset(&maps, 0, sizeof(maps));
    int rc = map_k<T>(&maps.x, x, m, k, ldx, args.x_rows);
    if (rc == TB200_OK) rc = map_k<T>(&maps.wg, wg, f, k, k, plan.w);
    if (rc == TB200_OK) rc = map_k<T>(&maps.wu, wu, f, k, k, plan.w);
    if (rc != TB200_OK) return rc;
    if (gq) return launch_mid_act<T, true, true>(maps, args, plan.shares, act, st);
    return few ? launch_mid_act<T, true, false>(maps, args, plan.shares, act, st) : launch_mid_act<T, false, false>(maps, args, plan.shares, act, st);
}

// Hidden units per tile of the pair kernel: 128, or the multiple of 16 (a pair's MMA is 32 columns or a multiple wide) that leaves
// the least idle at the end.  A wave's time
// hardly falls with its tiles' width, since a stage takes 0.27 us to issue whatever its width (measured at k = 2048: 12.1 us
// a wave of 128-wide tiles, 9.8 of 64-wide ones): it goes as the width + 200.
int pair_width(int64_t m, int64_t f, int64_t* waves) {
    const int64_t pairs = num_sms() / 2, tm = (m + 2 * kHalf - 1) / (2 * kHalf);
    int best = kHalf;
    int64_t least = 0;
    for (int w = kHalf; w >= 64; w -= 16) {
        const int64_t n = (tm * ((f + w - 1) / w) + pairs - 1) / pairs, cost = n * (w + 200);
        if (least == 0 || cost < least) {
            least = cost;
            best = w;
            *waves = n;
        }
    }
    return best;
}

template <typename T>
int ffn_forward(const void* x, const void* wg, const void* wu, void* h, void* gq, float* gs, void* uq, float* us, int64_t m, int64_t f,
                int64_t k, int64_t ldx, int act, int w, cudaStream_t st) {
    FfnMaps<FK_FWD> maps;
    memset(&maps, 0, sizeof(maps));
    int rc = map_k<T>(&maps.a[0], x, m, k, ldx);
    if (rc == TB200_OK) rc = map_k<T>(&maps.b[0], wg, f, k, k, w);
    if (rc == TB200_OK) rc = map_k<T>(&maps.b[1], wu, f, k, k, w);
    if (rc != TB200_OK) return rc;
    FfnArgs args = {};
    args.w = w;
    args.out[0] = h;
    args.m = static_cast<int>(m);
    args.f = static_cast<int>(f);
    args.k = static_cast<int>(k);
    args.codes[0] = static_cast<uint8_t*>(gq);
    args.codes[1] = static_cast<uint8_t*>(uq);
    args.scales[0] = gs;
    args.scales[1] = us;
    return gq ? launch_fwd<T, true>(maps, args, act, st) : launch_fwd<T, false>(maps, args, act, st);
}

// Up to 128 rows one CTA's accumulator holds them all and narrow tiles share the weights out evenly (1 row of 4096 -> 14336: 40 us
// against the pair kernel's 70).  Beyond, two CTAs share each weight tile, unless that leaves most of them idle: up to 1024 rows
// the shorter time by the two models decides (247 rows of 3960 -> 1164: 25 us in pairs, 17 so).  Checkpoints need whole 128-wide
// blocks: tiles of that width for up to 64 rows, the pair kernel's beyond.
template <typename T>
int forward(const void* x, const void* wg, const void* wu, void* h, void* gq, float* gs, void* uq, float* us, int64_t m, int64_t f, int64_t k,
            int64_t ldx, int act, cudaStream_t st) {
    int64_t waves = 0;
    const int w = gq ? kHalf : pair_width(m, f, &waves);
    if (m <= (gq ? kFewRows : 8 * kHalf)) {
        MidPlan plan = {kHalf, 1, 0.0f};
        const int rc = mid_plan(m, f, k, gq ? kHalf : 8, &plan);
        if (rc != TB200_OK) return rc;
        const float pair = static_cast<float>(waves) * (static_cast<float>((k + kBK - 1) / kBK) * 0.27f * static_cast<float>(w + 200) / 328.0f + 0.5f) + 3.0f;
        if (m <= kHalf || plan.time + 1.0f < pair) return ffn_mid<T>(x, wg, wu, h, gq, gs, uq, us, m, f, k, ldx, act, plan, st);
    }
    return ffn_forward<T>(x, wg, wu, h, gq, gs, uq, us, m, f, k, ldx, act, w, st);
}

// ---- the backward pass's shares ----
// A model of time in stages of 0.27 us.  An item of dx costs some 6 beside its own stages, one of dw 3; shares are written and
// added up in 32 bits, at 5 TB/s, by a kernel that costs some 10 more.
constexpr int kMostShares = 16, kLeastStages = 8;               // of a share
constexpr double kStagesPerByte = 1.0 / (5e6 * 0.27);

// dx for few rows, by a kernel of its own; a stage takes longer where it waits for the weights: 0.38 us at 148 CTAs.
int dx_few_shares(int64_t m, int64_t f, int64_t k) {
    const int64_t places = num_sms(), tiles = (k + kHalf - 1) / kHalf, steps = 2 * ((f + kBK - 1) / kBK);
    int best = 1;
    double least = 0.0;
    for (int s = 1; s <= kMostShares && steps >= kLeastStages * (s - 1); ++s) {
        const int64_t at_once = tiles * s < places ? tiles * s : places;
        const double stage = fmax(1.0, 1.4 * static_cast<double>(at_once) / static_cast<double>(places));
        const double cost = static_cast<double>((tiles * s + places - 1) / places) * (static_cast<double>((steps + s - 1) / s) * stage + 6.0) +
                            (s > 1 ? 10.0 + static_cast<double>(m) * k * 8.0 * s * kStagesPerByte : 0.0);
        if (s == 1 || cost < least) {
            least = cost;
            best = s;
        }
    }
    return best;
}

// Whether dx goes to that kernel: few rows, and weights of more than 100 MB in both, where its narrower tiles gain more than a launch
// shared with dw does.  Captured calls with cold inputs, in a kernel of its own against together, at 1 / 16 / 64 rows: 57 MB (512 x 28000)
// 47 / 49 / 57 us against 41 / 43 / 45; 84 MB (4096 x 5120) 49 / 51 / 55 against 53 / 53 / 53; 103 MB (3584 x 7168) 57 / 59 / 64 against
// 57 / 59 / 61; 117 MB (4096 x 7168) 61 / 64 / 70 against 66 / 66 / 68; 180 MB (4096 x 11008) 84 / 86 / 92 against 92 / 92 / 94;
// 235 MB (4096 x 14336) 104 / 107 / 113 against 115 / 117 / 119.  Between 80 and 150 MB it is a matter of 8 % either way, by rows and k.
bool dx_alone(int64_t m, int64_t f, int64_t k) { return m <= kFewRows && f * k > (24ll << 20); }

struct BwdPlan { int dx, dw, early; bool apart; }; // shares; early: see item_at; dx and dw in launches of their own
// Time of nx items of dx and nw of dw (cx and cw each) on the pairs, with the better number of early ones.
double bwd_time(int64_t nx, double cx, int64_t nw, double cw, int64_t pairs, int* early) {
    const int64_t rounds = nx / pairs, last = nx % pairs, idle = pairs - last;
    double least = 0.0;
    for (int64_t more = 0; more < 2; ++more) {
        const int64_t most = nw / idle, e = last == 0 ? 0 : static_cast<int64_t>(cx / cw) + more < most ? static_cast<int64_t>(cx / cw) + more : most;
        const int64_t rest = nw - e * idle, left = rest % pairs;
        const double busy = static_cast<double>(rounds + (last > 0)) * cx + static_cast<double>(rest / pairs + (left > idle)) * cw;
        const double other = static_cast<double>(rounds) * cx + static_cast<double>(e + rest / pairs + (left > 0)) * cw;
        if (more == 0 || fmax(busy, other) < least) {
            least = fmax(busy, other);
            *early = static_cast<int>(e);
        }
    }
    return least;
}
BwdPlan bwd_plan(int64_t m, int64_t f, int64_t k) {
    const bool few = dx_alone(m, f, k);
    const int64_t pairs = num_sms() / 2, tn = (k + 2 * kHalf - 1) / (2 * kHalf);
    const int64_t tx = few ? 0 : (m + 2 * kHalf - 1) / (2 * kHalf) * tn, tw = 2 * ((f + 2 * kHalf - 1) / (2 * kHalf)) * tn;
    const int64_t x_steps = 2 * ((f + kBK - 1) / kBK), w_steps = (m + kBK - 1) / kBK;
    BwdPlan best = {1, 1, 0, false};
    double least = 0.0;
    // more shares than it takes to give every pair two items are not looked at
    for (int sx = 1; sx <= kMostShares && x_steps >= kLeastStages * (sx - 1) && tx * (sx - 1) < 2 * pairs; ++sx) {
        for (int sw = 1; sw <= kMostShares && w_steps >= kLeastStages * (sw - 1) && tw * (sw - 1) < 2 * pairs; ++sw) {
            int early = 0;
            const double cx = static_cast<double>((x_steps + sx - 1) / sx) + 6.0, cw = static_cast<double>((w_steps + sw - 1) / sw) + 3.0;
            double cost = bwd_time(tx * sx, cx, tw * sw, cw, pairs, &early);
            // Items of both kinds at once read more of memory, in no common order: where one launch saves less than 5 % there are two
            // (16000 rows of 2048 x 8192: 1589 us against 1608; 4096 of 4096 x 14336, where it saves 9 %: 1368 against 1329).
            const double two = static_cast<double>((tx * sx + pairs - 1) / pairs) * cx + static_cast<double>((tw * sw + pairs - 1) / pairs) * cw + 10.0;
            const bool apart = cost > 0.95 * two;
            if (sx > 1 || sw > 1) cost += 10.0;
            if (sx > 1) cost += static_cast<double>(m) * k * 8.0 * sx * kStagesPerByte;
            if (sw > 1) cost += static_cast<double>(f) * k * 16.0 * sw * kStagesPerByte;
            if (least == 0.0 || cost < least) {
                least = cost;
                best = {sx, sw, early, apart};
            }
        }
        if (few) break;
    }
    if (few) best.dx = dx_few_shares(m, f, k);
    return best;
}

// out = the sum of `splits` arrays of n8 pieces of 8 numbers that lie `stride8` pieces apart, in order; 8 numbers per thread.  One
// result per row of the grid.
struct SumJob { const float4* sums; uint4* out; int64_t n8, stride8; int splits; };
struct SumJobs { SumJob job[3]; const float* factor; };         // factor: in fp16, of the results
template <typename T>
__global__ void __launch_bounds__(256) tb200_k_ffn_sum_shares(const __grid_constant__ SumJobs jobs) {
    let_next_begin();
    const SumJob& q = jobs.job[blockIdx.y];
    const float4* const __restrict__ sums = q.sums;
    const float factor = factor_of<T>(jobs.factor);
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < q.n8; i += static_cast<int64_t>(gridDim.x) * 256) {
        float4 a = sums[2 * i], b = sums[2 * i + 1];
#pragma unroll 4
        for (int s = 1; s < q.splits; ++s) {
            const float4 c = sums[2 * (s * q.stride8 + i)], d = sums[2 * (s * q.stride8 + i) + 1];
            a.x += c.x; a.y += c.y; a.z += c.z; a.w += c.w;
            b.x += d.x; b.y += d.y; b.z += d.z; b.w += d.w;
        }
        if constexpr (kFactor<T>) {
            a.x *= factor; a.y *= factor; a.z *= factor; a.w *= factor;
            b.x *= factor; b.y *= factor; b.z *= factor; b.w *= factor;
        }
        q.out[i] = make_uint4(ActType<T>::pack(a.x, a.y), ActType<T>::pack(a.z, a.w), ActType<T>::pack(b.x, b.y), ActType<T>::pack(b.z, b.w));
    }
}

template <typename T>
int dx_few(const void* dg, const void* du, int64_t ldg, const float* factor, const void* wg, const void* wu, void* dx, float* sums, int splits,
           int64_t m, int64_t f, int64_t k, cudaStream_t st) {
    auto kern = tb200_k_ffn_dx_few<T>;
    static PerDeviceInt attr_set;
    int rc = ensure_max_smem(attr_set, reinterpret_cast<const void*>(kern), kDxSmemBytes);
    if (rc != TB200_OK) return rc;
    DxFewArgs args = {};
    args.dx = dx;
    args.sums = sums;
    args.m = static_cast<int>(m);
    args.k = static_cast<int>(k);
    args.depth = static_cast<int>(f);
    args.shares = splits;
    args.rows = static_cast<int>((m + 15) / 16 * 16);
    args.factor = factor;
    const int stage = kOperandBytes + args.rows * 128;
    args.stages = kDxRing / stage < kMaxStages ? kDxRing / stage : kMaxStages;
    DxFewMaps maps;
    memset(&maps, 0, sizeof(maps));
    rc = map_k<T>(&maps.d[0], dg, m, f, ldg, args.rows);
    if (rc == TB200_OK) rc = map_k<T>(&maps.d[1], du, m, f, ldg, args.rows);
    if (rc == TB200_OK) rc = map_mn<T>(&maps.w[0], wg, f, k, k);
    if (rc == TB200_OK) rc = map_mn<T>(&maps.w[1], wu, f, k, k);
    if (rc != TB200_OK) return rc;
    const int64_t items = (k + kHalf - 1) / kHalf * splits;
    return launch_over_previous(kern, static_cast<int>(items < num_sms() ? items : num_sms()), kDxThreads, kDxSmemBytes, 1, st, maps, args);
}

// dg, du: [m, ldg], in fp16 with the results' factor behind dg's first row; x: [m, k]; sums: room for the plan's arrays of dx [m, k], then for those of dw [2, f, k], where they are more than 1
template <typename T>
int ffn_products_bwd(void* dg, const void* du, int64_t ldg, const void* x, int64_t ldx, const void* wg, const void* wu, void* dx, void* dwg,
                     void* dwu, float* sums, int64_t m, int64_t f, int64_t k, cudaStream_t st) {
    const BwdPlan plan = bwd_plan(m, f, k);
    const bool few = dx_alone(m, f, k);
    const float* const factor = kFactor<T> ? behind_row<float>(dg, ldg) : nullptr;
    float* const sums_w = sums + (plan.dx > 1 ? plan.dx * m * k : 0);
    int rc = few ? dx_few<T>(dg, du, ldg, factor, wg, wu, dx, sums, plan.dx, m, f, k, st) : TB200_OK;
    FfnBwdMaps maps;
    memset(&maps, 0, sizeof(maps));
    const void* const grads[2] = {dg, du};
    const void* const weights[2] = {wg, wu};
    for (int i = 0; i < 2; ++i) {
        if (rc == TB200_OK) rc = map_k<T>(&maps.a[i], grads[i], m, f, ldg);
        if (rc == TB200_OK) rc = map_mn<T>(&maps.b[i], weights[i], f, k, k);
        if (rc == TB200_OK) rc = map_mn<T>(&maps.at[i], grads[i], m, f, ldg);
    }
    if (rc == TB200_OK) rc = map_mn<T>(&maps.x, x, m, k, ldx);
    if (rc == TB200_OK) rc = map_out<T>(&maps.out[0], dx, m, k);
    if (rc == TB200_OK) rc = map_out<T>(&maps.out[1], dwg, f, k);
    if (rc == TB200_OK) rc = map_out<T>(&maps.out[2], dwu, f, k);
    if (rc != TB200_OK) return rc;
    FfnArgs args = {};
    args.out[0] = dx;
    args.out[1] = dwg;
    args.out[2] = dwu;
    args.m = static_cast<int>(m);
    args.f = static_cast<int>(f);
    args.k = static_cast<int>(k);
    args.sums[0] = sums;
    args.sums[1] = sums_w;
    args.shares[0] = plan.dx;
    args.shares[1] = plan.dw;
    args.early = plan.early;
    args.factor = factor;
    const int64_t tn = (k + 2 * kHalf - 1) / (2 * kHalf);
    const int64_t items_x = plan.dx * ((m + 2 * kHalf - 1) / (2 * kHalf)) * tn, items_w = plan.dw * 2 * ((f + 2 * kHalf - 1) / (2 * kHalf)) * tn;
    if (few) {
        rc = launch_pair<FK_DW, T, 0, false>({maps}, args, items_w, st);
    } else if (plan.apart) {
        FfnArgs first = args;
        first.shares[1] = first.early = args.shares[0] = args.early = 0;
        rc = launch_pair<FK_BWD, T, 0, false>({maps}, first, items_x, st);
        if (rc == TB200_OK) rc = launch_pair<FK_BWD, T, 0, false>({maps}, args, items_w, st);
    } else {
        rc = launch_pair<FK_BWD, T, 0, false>({maps}, args, items_x + items_w, st);
    }
    if (rc != TB200_OK) return rc;

    SumJobs jobs = {};
    jobs.factor = factor;
    int n = 0;
    int64_t most = 0;
    auto add = [&](const float* from, void* to, int64_t count, int64_t stride, int splits) {
        jobs.job[n++] = {reinterpret_cast<const float4*>(from), static_cast<uint4*>(to), count / 8, stride / 8, splits};
        most = count > most ? count : most;
    };
    if (plan.dx > 1) add(sums, dx, m * k, m * k, plan.dx);
    if (plan.dw > 1) add(sums_w, dwg, f * k, 2 * f * k, plan.dw);
    if (plan.dw > 1) add(sums_w + f * k, dwu, f * k, 2 * f * k, plan.dw);
    if (n > 0) {
        const int64_t ctas = (most / 8 + 255) / 256, cap = static_cast<int64_t>(num_sms()) * 8;
        tb200_k_ffn_sum_shares<T><<<dim3(static_cast<unsigned>(ctas < cap ? ctas : cap), static_cast<unsigned>(n)), 256, 0, st>>>(jobs);
        TB200_CUDA_TRY(cudaGetLastError());
    }
    return TB200_OK;
}

bool to_elements(const void* p, uintptr_t size) { return reinterpret_cast<uintptr_t>(p) % size == 0; }
constexpr int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }
int64_t x_pitch(int64_t k) { return round_up(k, 64); }          // of a restored x: whole 128-byte lines, as for dg and du
int64_t grad_bytes(int64_t m, int64_t f, int dtype) { return round_up(m * grad_pitch(f, dtype) * 2, 256); }

int check_common(const char* what, int64_t m, int64_t f, int64_t k, int act, int dtype) {
    if (m < 0 || f <= 0 || k <= 0)
        return fail(TB200_ERR_ARG, "%s: m=%lld f=%lld k=%lld (m >= 0, f > 0, k > 0)", what, (long long)m, (long long)f, (long long)k);
    if (m > (1ll << 30) || f > (1ll << 30) || k > (1ll << 30)) return fail(TB200_ERR_UNSUPPORTED, "%s: dimension too large", what);
    if (k % 8 != 0) return fail(TB200_ERR_UNSUPPORTED, "%s: k=%lld must be a multiple of 8 (rows of 16-byte pieces)", what, (long long)k);
    if (dtype != TB200_DT_F16 && dtype != TB200_DT_BF16) return fail(TB200_ERR_UNSUPPORTED, "%s: dtype %d is not one of F16, BF16", what, dtype);
    if (act < TB200_ACT_SILU || act > TB200_ACT_RELU) return fail(TB200_ERR_UNSUPPORTED, "%s: unknown activation %d", what, act);
    return TB200_OK;
}

}  // namespace
}  // namespace tb200

using namespace tb200;

TB200_DEFINE_STATUS_HOOKS(gemm_ffn)

extern "C" int tb200_ffn_gated(const void* x, const void* wg, const void* wu, void* h, void* gq, float* gs, void* uq, float* us, int64_t m,
                               int64_t f, int64_t k, int64_t ldx, int act, int dtype, void* stream) {
    clear_error();
    const int rc = check_common("ffn_gated", m, f, k, act, dtype);
    if (rc != TB200_OK) return rc;
    if (m == 0) return TB200_OK;
    if (!x || !wg || !wu || !h) return fail(TB200_ERR_ARG, "ffn_gated: null pointer");
    const int given = (gq != nullptr) + (gs != nullptr) + (uq != nullptr) + (us != nullptr);
    if (given != 0 && given != 4) return fail(TB200_ERR_ARG, "ffn_gated: gq, gs, uq, us are given together or not at all");
    if (m == 1) ldx = k;
    if (ldx < k || ldx % 8 != 0) return fail(TB200_ERR_ALIGN, "ffn_gated: row stride of x %lld must be a multiple of 8 and at least k", (long long)ldx);
    if (!aligned16(x) || !aligned16(wg) || !aligned16(wu)) return fail(TB200_ERR_ALIGN, "ffn_gated: x, wg, wu must be 16-byte aligned");
    if (!to_elements(h, 2) || !to_elements(gs, 4) || !to_elements(us, 4)) return fail(TB200_ERR_ALIGN, "ffn_gated: h, gs, us must be aligned to their elements");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return dtype == TB200_DT_F16 ? forward<__half>(x, wg, wu, h, gq, gs, uq, us, m, f, k, ldx, act, st)
                                 : forward<__nv_bfloat16>(x, wg, wu, h, gq, gs, uq, us, m, f, k, ldx, act, st);
}

extern "C" size_t tb200_ffn_gated_bwd_workspace_bytes(int64_t m, int64_t f, int64_t k, int x_codes) {
    if (m <= 0 || f <= 0 || k <= 0) return 0;
    const BwdPlan plan = bwd_plan(m, f, k);
    return static_cast<size_t>(2 * grad_bytes(m, f, TB200_DT_F16) + (x_codes ? round_up(m * x_pitch(k) * 2, 256) : 0) +     // no less than in bf16
                               (plan.dx > 1 ? plan.dx * m * k * 4 : 0) + (plan.dw > 1 ? plan.dw * 2 * f * k * 4 : 0));
}

extern "C" int tb200_ffn_gated_bwd(const void* dh, const void* wg, const void* wu, const void* x, const float* xs, const void* gq,
                                   const float* gs, const void* uq, const float* us, void* dx, void* dwg, void* dwu, int64_t m, int64_t f,
                                   int64_t k, int64_t ldx, int act, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
    clear_error();
    int rc = check_common("ffn_gated_bwd", m, f, k, act, dtype);
    if (rc != TB200_OK) return rc;
    if (!dwg || !dwu) return fail(TB200_ERR_ARG, "ffn_gated_bwd: null pointer");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (m == 0) {                                                // no token: the weights' gradients are zero
        TB200_CUDA_TRY(cudaMemsetAsync(dwg, 0, static_cast<size_t>(f) * k * 2, st));
        TB200_CUDA_TRY(cudaMemsetAsync(dwu, 0, static_cast<size_t>(f) * k * 2, st));
        return TB200_OK;
    }
    if (!dh || !wg || !wu || !x || !gq || !gs || !uq || !us || !dx) return fail(TB200_ERR_ARG, "ffn_gated_bwd: null pointer");
    const bool codes = xs != nullptr;
    if (codes || m == 1) ldx = k;                                // no pitch of the caller's, or none that matters
    if (ldx < k || ldx % 8 != 0) return fail(TB200_ERR_ALIGN, "ffn_gated_bwd: row stride of x %lld must be a multiple of 8 and at least k", (long long)ldx);
    if (!aligned16(wg) || !aligned16(wu) || !aligned16(dx) || !aligned16(dwg) || !aligned16(dwu) || (!codes && !aligned16(x)))
        return fail(TB200_ERR_ALIGN, "ffn_gated_bwd: x, wg, wu, dx, dwg, dwu must be 16-byte aligned");
    if (!to_elements(dh, 2) || !to_elements(gs, 4) || !to_elements(us, 4) || !to_elements(xs, 4))
        return fail(TB200_ERR_ALIGN, "ffn_gated_bwd: dh, gs, us, xs must be aligned to their elements");
    if (m > (1ll << 40) / f) return fail(TB200_ERR_UNSUPPORTED, "ffn_gated_bwd: m=%lld f=%lld is too large", (long long)m, (long long)f);
    const size_t need = tb200_ffn_gated_bwd_workspace_bytes(m, f, k, codes ? 1 : 0);
    if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255) != 0)
        return fail(TB200_ERR_WORKSPACE, "ffn_gated_bwd: needs a 256-byte aligned workspace of %zu bytes, got %zu", need, workspace ? workspace_bytes : size_t(0));
    const int64_t ldg = grad_pitch(f, dtype);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    void* dg = ws;
    void* du = ws + grad_bytes(m, f, dtype);
    void* xr = ws + 2 * grad_bytes(m, f, dtype);
    float* sums = reinterpret_cast<float*>(static_cast<uint8_t*>(xr) + (codes ? round_up(m * x_pitch(k) * 2, 256) : 0));
    if (codes) ldx = reinterpret_cast<uintptr_t>(x) % 8 == 0 ? x_pitch(k) : k;
    rc = launch_gated_act_bwd(dh, gq, gs, uq, us, dg, du, m, f, ldg, codes ? x : nullptr, xs, xr, k, ldx, act, dtype, st);
    if (rc != TB200_OK) return rc;
    if (codes) x = xr;
    return dtype == TB200_DT_F16 ? ffn_products_bwd<__half>(dg, du, ldg, x, ldx, wg, wu, dx, dwg, dwu, sums, m, f, k, st)
                                 : ffn_products_bwd<__nv_bfloat16>(dg, du, ldg, x, ldx, wg, wu, dx, dwg, dwu, sums, m, f, k, st);
}
