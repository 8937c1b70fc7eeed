// Matrix products of the gated feed-forward block, forward and backward, on tcgen05 (kind::f16, fp32 accumulation).
//
//   forward   g = x Wg^T, u = x Wu^T, h = f(g) * u         one kernel; the codes of g and u in 8 bits on request
//   dx        dx = dg Wg + du Wu                            one kernel, one accumulator over both products
//   dw        dWg = dg^T x, dWu = du^T x                    one launch over the tiles of both results
//
// All three are one CTA-pair kernel (cta_group::2): 256 x 256 accumulators in tensor memory, two of them, so that the
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

#include <cstring>

namespace tb200 {
namespace {

constexpr int kBK = 64;                          // contraction per stage: 128 bytes of 16-bit elements
constexpr int kHalf = 128;                       // rows of A, and columns of B, that one CTA loads
constexpr int kStages = 6;
constexpr int kOperandBytes = kHalf * 128;
constexpr int kStageBytes = 2 * kOperandBytes;
constexpr int kAtomBytes = kBK * 128;            // MN-major: one box of 64 contraction rows x 64 columns
constexpr int kStagingBytes = 32 * 256;          // per epilogue warp: 32 rows x 128 16-bit columns
constexpr int kBarBytes = 256;
constexpr int kSmemBytes = kStages * kStageBytes + 4 * kStagingBytes + kBarBytes + 1024;
constexpr int kTmemCols = 512;
constexpr int kThreads = 256;
constexpr int kGroupM = 8;                       // tiles are walked in bands of 8 x 256 rows, so that B's tiles stay in L2

enum FfnKind : int { FK_FWD = 0, FK_DX = 1, FK_DW = 2 };

struct FfnMaps {
    CUtensorMap a[2];                            // forward: x, -      dx: dg, du     dw: dg, du
    CUtensorMap b[2];                            // forward: Wg, Wu    dx: Wg, Wu     dw: x, -
};
struct FfnArgs {
    void* out[2];                                // forward: h, -      dx: dx, -      dw: dWg, dWu
    int rows, cols, depth;                       // of one result, and of one product's contraction
    int64_t ldo;                                 // row pitch of the result, in elements
    uint8_t* codes[2];                           // forward with checkpoints: codes of g and u, [rows, cols]
    float* scales[2];                            // and their scales, [rows, ceil(cols / 128)]
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

// ---- epilogue helpers --------------------------------------------------------------------------------------------
// A warp collects 32 rows of 256 bytes in shared memory, 16-byte piece c of row r at place c ^ (r & 15) (free of bank
// conflicts both ways), and writes them out with neighbouring lanes on neighbouring bytes.
__device__ __forceinline__ uint4* staged(uint8_t* buf, int row, int piece) {
    return reinterpret_cast<uint4*>(buf + row * 256 + ((piece ^ (row & 15)) << 4));
}
// Pieces [first, first + count) of every row are `count` * 16 bytes of row r of dst; rows and columns beyond the valid
// ones are left out.  T: the element.  Rows that do not lie on 16-byte boundaries are written element by element.
template <typename T>
__device__ __forceinline__ void flush(uint8_t* buf, int first, int count, T* __restrict__ dst, int64_t pitch, int rows, int cols, int lane) {
    constexpr int V = 16 / sizeof(T);
    if (rows > 32) rows = 32;
    const bool vec = (reinterpret_cast<uintptr_t>(dst) & 15) == 0 && (pitch * sizeof(T)) % 16 == 0;
    if (vec) {
        const int per = 32 / count, sub = lane / count, piece = lane % count;
        for (int r = sub; r < rows; r += per) {
            const uint4 v = *staged(buf, r, first + piece);
            T* p = dst + r * pitch + piece * V;
            if (piece * V + V <= cols) {
                *reinterpret_cast<uint4*>(p) = v;
            } else {
                const T* e = reinterpret_cast<const T*>(staged(buf, r, first + piece));
                for (int i = 0; i < cols - piece * V; ++i) p[i] = e[i];
            }
        }
    } else {
        for (int r = 0; r < rows; ++r)
            for (int c = lane; c < count * V && c < cols; c += 32)
                dst[r * pitch + c] = reinterpret_cast<const T*>(staged(buf, r, first + c / V))[c % V];
    }
}

template <typename T>
__device__ __forceinline__ void stage32(uint8_t* buf, int row, int piece0, const float (&v)[32]) {      // 32 columns: 4 pieces
#pragma unroll
    for (int q = 0; q < 4; ++q)
        *staged(buf, row, piece0 + q) = make_uint4(ActType<T>::pack(v[8 * q], v[8 * q + 1]), ActType<T>::pack(v[8 * q + 2], v[8 * q + 3]),
                                                   ActType<T>::pack(v[8 * q + 4], v[8 * q + 5]), ActType<T>::pack(v[8 * q + 6], v[8 * q + 7]));
}
__device__ __forceinline__ void stage_codes32(uint8_t* buf, int row, int piece0, const uint32_t (&v)[32], float inv) {  // 2 pieces
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = 16 * q + 4 * e;
            w[e] = act_codes4(__uint_as_float(v[i]), __uint_as_float(v[i + 1]), __uint_as_float(v[i + 2]), __uint_as_float(v[i + 3]), inv);
        }
        *staged(buf, row, piece0 + q) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

template <int ACT>
__device__ __forceinline__ void gated32(const uint32_t (&g)[32], const uint32_t (&u)[32], float (&h)[32]) {
#pragma unroll
    for (int i = 0; i < 32; ++i) h[i] = gate_value<ACT>(__uint_as_float(g[i])) * __uint_as_float(u[i]);
}

struct Tile { int m, n; };
__device__ __forceinline__ Tile tile_at(int t, int tiles_m, int tiles_n) {
    const int per_group = kGroupM * tiles_n;
    const int g = t / per_group, first = g * kGroupM, size = min(kGroupM, tiles_m - first), r = t - g * per_group;
    return {first + r % size, r / size};
}

// KIND as above; T fp16 or bf16; ACT the gate (forward only); SAVE writes the codes of g and u (forward only).
template <int KIND, typename T, int ACT, bool SAVE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
k_ffn_pair(const __grid_constant__ FfnMaps maps, const __grid_constant__ FfnArgs p) {
    constexpr int S = kStages;
    constexpr bool kAMn = KIND == FK_DW, kBMn = KIND != FK_FWD;
    constexpr int kTileCols = KIND == FK_FWD ? 128 : 256;       // columns of the result that a tile covers
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* staging = smem + S * kStageBytes;
    uint64_t* bar_full = reinterpret_cast<uint64_t*>(staging + 4 * kStagingBytes);
    uint64_t* bar_empty = bar_full + S;
    uint64_t* bar_afull = bar_empty + S;          // [2] accumulator complete
    uint64_t* bar_aempty = bar_afull + 2;         // [2] accumulator read (4 epilogue warps in each CTA)
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar_aempty + 2);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int rank = static_cast<int>(cluster_ctarank());       // 0 = leader
    const int pair = blockIdx.x >> 1;
    const int npairs = gridDim.x >> 1;
    const int KB = (p.depth + kBK - 1) / kBK;                   // stages of one product
    const int steps = KIND == FK_DX ? 2 * KB : KB;
    const int tm1 = (p.rows + 2 * kHalf - 1) / (2 * kHalf);
    const int tiles_m = KIND == FK_DW ? 2 * tm1 : tm1;          // dw: the tiles of dWg, then those of dWu
    const int tiles_n = (p.cols + kTileCols - 1) / kTileCols;
    const int tiles = tiles_m * tiles_n;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(&bar_full[s], 1);
            mbar_init(&bar_empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&bar_afull[b], 1);
            mbar_init(&bar_aempty[b], 8);
        }
        mbar_fence_init();
        tma_prefetch_desc(&maps.a[0]);
        tma_prefetch_desc(&maps.b[0]);
        if (KIND != FK_FWD) tma_prefetch_desc(&maps.a[1]);
        if (KIND != FK_DW) tma_prefetch_desc(&maps.b[1]);
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

    if (warp == 0) {
        // ---------------- TMA producer (both CTAs) ----------------
        if (lane == 0) {
            uint32_t s = 0, ph = 1;
            bool ok = true;
            for (int t = pair; t < tiles && ok; t += npairs) {
                const Tile tc = tile_at(t, tiles_m, tiles_n);
                const int sel = KIND == FK_DW && tc.m >= tm1 ? 1 : 0;
                const int a_row = (tc.m - sel * tm1) * 2 * kHalf + rank * kHalf;
                const int b_col = KIND == FK_FWD ? tc.n * kHalf : tc.n * 2 * kHalf + rank * kHalf;
                for (int st = 0; st < steps; ++st) {
                    if (!mbar_wait(&bar_empty[s], ph, ST_WAIT_SMEM_EMPTY, st)) { ok = false; break; }
                    uint8_t* stage = smem + s * kStageBytes;
                    if (rank == 0) mbar_expect_tx(&bar_full[s], 2 * kStageBytes);               // both CTAs' bytes
                    const int prod = KIND == FK_DX && st >= KB ? 1 : 0;
                    const int k0 = (st - prod * KB) * kBK;
                    if constexpr (kAMn) {
                        tma_load_2d_pair(stage, &maps.a[sel], &bar_full[s], a_row, k0);
                        tma_load_2d_pair(stage + kAtomBytes, &maps.a[sel], &bar_full[s], a_row + 64, k0);
                    } else {
                        tma_load_2d_pair(stage, &maps.a[prod], &bar_full[s], k0, a_row);
                    }
                    if constexpr (kBMn) {
                        tma_load_2d_pair(stage + kOperandBytes, &maps.b[prod], &bar_full[s], b_col, k0);
                        tma_load_2d_pair(stage + kOperandBytes + kAtomBytes, &maps.b[prod], &bar_full[s], b_col + 64, k0);
                    } else {
                        tma_load_2d_pair(stage + kOperandBytes, &maps.b[rank], &bar_full[s], k0, b_col);
                    }
                    if (++s == S) { s = 0; ph ^= 1; }
                }
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
        constexpr uint32_t idesc = umma_idesc(fmt, fmt, 2 * kHalf, 2 * kHalf) | (kAMn ? 1u << 15 : 0u) | (kBMn ? 1u << 16 : 0u);
        constexpr uint32_t kStageDesc = kStageBytes >> 4;
        // 16 of the 64 contraction elements per MMA: 32 bytes along a K-major row, 16 rows of an MN-major box
        constexpr uint64_t a_step = kAMn ? 16 * 128 / 16 : 2, b_step = kBMn ? 16 * 128 / 16 : 2;
        const bool leader = lane == 0;
        const uint64_t a_desc0 = kAMn ? desc_mn(smem_u32(smem)) : umma_desc_sw128(smem_u32(smem));
        const uint64_t b_desc0 = kBMn ? desc_mn(smem_u32(smem) + kOperandBytes) : umma_desc_sw128(smem_u32(smem) + kOperandBytes);
        uint32_t s = 0, ph = 0, cnt = 0;
        bool ready = false;
        bool ok = true;
        for (int t = pair; t < tiles && ok; t += npairs, ++cnt) {
            const uint32_t acc = cnt & 1;
            if (!mbar_wait(&bar_aempty[acc], ((cnt >> 1) & 1) ^ 1, ST_WAIT_TMEM_EMPTY, t)) { ok = false; break; }
            tc_fence_after();
            const uint32_t d_tmem = tmem_base + acc * 256;
            for (int st = 0; st < steps; ++st) {
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
            if (ok && leader) tc_commit_pair(&bar_afull[acc], 0x3);
        }
    } else if (warp >= 4) {
        // ---------------- epilogue (both CTAs; each owns 128 rows of the tile, each warp 32 of them) ----------------
        const int ew = warp - 4;
        uint8_t* buf = staging + ew * kStagingBytes;
        const uint32_t t_lane = tmem_base + (static_cast<uint32_t>(ew * 32) << 16);
        uint32_t cnt = 0;
        bool ok = true;
        for (int t = pair; t < tiles && ok; t += npairs, ++cnt) {
            const Tile tc = tile_at(t, tiles_m, tiles_n);
            const int sel = KIND == FK_DW && tc.m >= tm1 ? 1 : 0;
            const uint32_t acc = cnt & 1;
            const int row0 = (tc.m - sel * tm1) * 2 * kHalf + rank * kHalf + ew * 32;             // the warp's first row
            const int rows = p.rows - row0;                                                       // valid rows (may be <= 0)
            const int col0 = tc.n * kTileCols, cols = p.cols - col0;
            const uint32_t t_acc = t_lane + acc * 256;
            if (!mbar_wait(&bar_afull[acc], (cnt >> 1) & 1, ST_WAIT_TMEM_FULL, t)) { ok = false; break; }
            tc_fence_after();
            T* dst = static_cast<T*>(p.out[sel]) + static_cast<int64_t>(row0) * p.ldo + col0;
            if constexpr (KIND == FK_FWD) {
                uint32_t g[32], u[32];
                float amax_g = 0.0f, amax_u = 0.0f;
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                    tmem_ld32(t_acc + c * 32, g);
                    tmem_ld32(t_acc + kHalf + c * 32, u);
                    tmem_wait_ld();
                    if (!SAVE && c == 3) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive_leader(&bar_aempty[acc]);
                    }
                    if constexpr (SAVE) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            amax_g = fmaxf(amax_g, act_size(__uint_as_float(g[i])));
                            amax_u = fmaxf(amax_u, act_size(__uint_as_float(u[i])));
                        }
                    }
                    float h[32];
                    gated32<ACT>(g, u, h);
                    stage32<T>(buf, lane, 4 * c, h);
                }
                __syncwarp();
                flush<T>(buf, 0, 16, dst, p.ldo, rows, cols, lane);
                __syncwarp();
                if constexpr (SAVE) {
                    const int64_t nblk = (p.cols + kHalf - 1) / kHalf;
                    const float2 sg = act_scale(amax_g), su = act_scale(amax_u);
                    if (lane < rows) {
                        p.scales[0][(row0 + lane) * nblk + tc.n] = sg.x;
                        p.scales[1][(row0 + lane) * nblk + tc.n] = su.x;
                    }
#pragma unroll 1
                    for (int c = 0; c < 4; ++c) {
                        tmem_ld32(t_acc + c * 32, g);
                        tmem_ld32(t_acc + kHalf + c * 32, u);
                        tmem_wait_ld();
                        if (c == 3) {
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) mbar_arrive_leader(&bar_aempty[acc]);
                        }
                        stage_codes32(buf, lane, 2 * c, g, sg.y);
                        stage_codes32(buf, lane, 8 + 2 * c, u, su.y);
                    }
                    __syncwarp();
                    const int64_t at = static_cast<int64_t>(row0) * p.cols + col0;
                    flush<uint8_t>(buf, 0, 8, p.codes[0] + at, p.cols, rows, cols, lane);
                    flush<uint8_t>(buf, 8, 8, p.codes[1] + at, p.cols, rows, cols, lane);
                    __syncwarp();
                }
            } else {
#pragma unroll 1
                for (int half = 0; half < 2; ++half) {
#pragma unroll 1
                    for (int c = 0; c < 4; ++c) {
                        uint32_t v[32];
                        float w[32];
                        tmem_ld32(t_acc + half * kHalf + c * 32, v);
                        tmem_wait_ld();
                        if (half == 1 && c == 3) {
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) mbar_arrive_leader(&bar_aempty[acc]);
                        }
#pragma unroll
                        for (int i = 0; i < 32; ++i) w[i] = __uint_as_float(v[i]);
                        stage32<T>(buf, lane, 4 * c, w);
                    }
                    __syncwarp();
                    flush<T>(buf, 0, 16, dst + half * kHalf, p.ldo, rows, cols - half * kHalf, lane);
                    __syncwarp();
                }
            }
        }
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

template <typename T>
constexpr CUtensorMapDataType tmap_type() { return ActType<T>::kTop > 1e6f ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16; }

// K-major operand: 128 rows x 64 of the contraction.  MN-major operand: 64 rows of the contraction x 64 columns.
template <typename T>
int map_k(CUtensorMap* m, const void* base, int64_t rows, int64_t cols, int64_t pitch) {
    return encode_tmap_2d(m, base, tmap_type<T>(), 2, rows, cols, pitch * 2, kHalf, kBK, CU_TENSOR_MAP_SWIZZLE_128B);
}
template <typename T>
int map_mn(CUtensorMap* m, const void* base, int64_t rows, int64_t cols, int64_t pitch) {
    return encode_tmap_2d(m, base, tmap_type<T>(), 2, rows, cols, pitch * 2, kBK, 64, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int KIND, typename T, int ACT, bool SAVE>
int launch_pair(const FfnMaps& maps, const FfnArgs& args, cudaStream_t st) {
    auto kern = k_ffn_pair<KIND, T, ACT, SAVE>;
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
        int clusters = 0;
        TB200_CUDA_TRY(cudaOccupancyMaxActiveClusters(&clusters, kern, &cfg));
        if (clusters < 1) return fail(TB200_ERR_UNSUPPORTED, "ffn_gated: no CTA pair fits on this device");
        max_pairs = clusters;
        max_pairs_tab.v[dev].store(clusters, std::memory_order_release);
    }
    const int64_t tile_cols = KIND == FK_FWD ? kHalf : 2 * kHalf;
    const int64_t tiles = (KIND == FK_DW ? 2 : 1) * ((args.rows + 2 * kHalf - 1) / (2 * kHalf)) * ((args.cols + tile_cols - 1) / tile_cols);
    if (tiles > 0x7fffffffll / kGroupM) return fail(TB200_ERR_UNSUPPORTED, "ffn_gated: too many tiles");
    const int pairs = static_cast<int>(tiles < max_pairs ? tiles : max_pairs);
    kern<<<2 * pairs, kThreads, kSmemBytes, st>>>(maps, args);
    TB200_CUDA_TRY(cudaGetLastError());
    return TB200_OK;
}

template <typename T, bool SAVE>
int launch_fwd(const FfnMaps& maps, const FfnArgs& args, int act, cudaStream_t st) {
    switch (act) {
        case TB200_ACT_SILU: return launch_pair<FK_FWD, T, TB200_ACT_SILU, SAVE>(maps, args, st);
        case TB200_ACT_GELU: return launch_pair<FK_FWD, T, TB200_ACT_GELU, SAVE>(maps, args, st);
        case TB200_ACT_GELU_TANH: return launch_pair<FK_FWD, T, TB200_ACT_GELU_TANH, SAVE>(maps, args, st);
        default: return launch_pair<FK_FWD, T, TB200_ACT_RELU, SAVE>(maps, args, st);
    }
}

template <typename T>
int ffn_forward(const void* x, const void* wg, const void* wu, void* h, void* gq, float* gs, void* uq, float* us, int64_t m, int64_t f,
                int64_t k, int64_t ldx, int act, cudaStream_t st) {
    FfnMaps maps;
    memset(&maps, 0, sizeof(maps));
    int rc = map_k<T>(&maps.a[0], x, m, k, ldx);
    if (rc == TB200_OK) rc = map_k<T>(&maps.b[0], wg, f, k, k);
    if (rc == TB200_OK) rc = map_k<T>(&maps.b[1], wu, f, k, k);
    if (rc != TB200_OK) return rc;
    FfnArgs args = {};
    args.out[0] = h;
    args.rows = static_cast<int>(m);
    args.cols = static_cast<int>(f);
    args.depth = static_cast<int>(k);
    args.ldo = f;
    args.codes[0] = static_cast<uint8_t*>(gq);
    args.codes[1] = static_cast<uint8_t*>(uq);
    args.scales[0] = gs;
    args.scales[1] = us;
    return gq ? launch_fwd<T, true>(maps, args, act, st) : launch_fwd<T, false>(maps, args, act, st);
}

// dg, du: [m, ldg]; x: [m, k]
template <typename T>
int ffn_products_bwd(const void* dg, const void* du, int64_t ldg, const void* x, int64_t ldx, const void* wg, const void* wu, void* dx, void* dwg,
                     void* dwu, int64_t m, int64_t f, int64_t k, cudaStream_t st) {
    FfnMaps maps;
    memset(&maps, 0, sizeof(maps));
    int rc = map_k<T>(&maps.a[0], dg, m, f, ldg);
    if (rc == TB200_OK) rc = map_k<T>(&maps.a[1], du, m, f, ldg);
    if (rc == TB200_OK) rc = map_mn<T>(&maps.b[0], wg, f, k, k);
    if (rc == TB200_OK) rc = map_mn<T>(&maps.b[1], wu, f, k, k);
    if (rc != TB200_OK) return rc;
    FfnArgs args = {};
    args.out[0] = dx;
    args.rows = static_cast<int>(m);
    args.cols = static_cast<int>(k);
    args.depth = static_cast<int>(f);
    args.ldo = k;
    rc = launch_pair<FK_DX, T, 0, false>(maps, args, st);
    if (rc != TB200_OK) return rc;

    memset(&maps, 0, sizeof(maps));
    rc = map_mn<T>(&maps.a[0], dg, m, f, ldg);
    if (rc == TB200_OK) rc = map_mn<T>(&maps.a[1], du, m, f, ldg);
    if (rc == TB200_OK) rc = map_mn<T>(&maps.b[0], x, m, k, ldx);
    if (rc != TB200_OK) return rc;
    args.out[0] = dwg;
    args.out[1] = dwu;
    args.rows = static_cast<int>(f);
    args.depth = static_cast<int>(m);
    return launch_pair<FK_DW, T, 0, false>(maps, args, st);
}

constexpr int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }
int64_t pitch_of(int64_t f) { return round_up(f, 8); }          // rows of dg and du begin on 16-byte boundaries

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
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return dtype == TB200_DT_F16 ? ffn_forward<__half>(x, wg, wu, h, gq, gs, uq, us, m, f, k, ldx, act, st)
                                 : ffn_forward<__nv_bfloat16>(x, wg, wu, h, gq, gs, uq, us, m, f, k, ldx, act, st);
}

extern "C" size_t tb200_ffn_gated_bwd_workspace_bytes(int64_t m, int64_t f, int64_t k, int x_codes) {
    if (m <= 0 || f <= 0 || k <= 0) return 0;
    return static_cast<size_t>(2 * round_up(m * pitch_of(f) * 2, 256) + (x_codes ? round_up(m * k * 2, 256) : 0));
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
    if (codes || m == 1) ldx = k;
    if (ldx < k || ldx % 8 != 0) return fail(TB200_ERR_ALIGN, "ffn_gated_bwd: row stride of x %lld must be a multiple of 8 and at least k", (long long)ldx);
    if (!aligned16(wg) || !aligned16(wu) || !aligned16(dx) || !aligned16(dwg) || !aligned16(dwu) || (!codes && !aligned16(x)))
        return fail(TB200_ERR_ALIGN, "ffn_gated_bwd: x, wg, wu, dx, dwg, dwu must be 16-byte aligned");
    if (reinterpret_cast<uintptr_t>(dh) & 1) return fail(TB200_ERR_ALIGN, "ffn_gated_bwd: dh must be aligned to its elements");
    if (m > (1ll << 40) / f) return fail(TB200_ERR_UNSUPPORTED, "ffn_gated_bwd: m=%lld f=%lld is too large", (long long)m, (long long)f);
    const size_t need = tb200_ffn_gated_bwd_workspace_bytes(m, f, k, codes ? 1 : 0);
    if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255) != 0)
        return fail(TB200_ERR_WORKSPACE, "ffn_gated_bwd: needs a 256-byte aligned workspace of %zu bytes, got %zu", need, workspace ? workspace_bytes : size_t(0));
    const int64_t ldg = pitch_of(f);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    void* dg = ws;
    void* du = ws + round_up(m * ldg * 2, 256);
    void* xr = ws + 2 * round_up(m * ldg * 2, 256);
    rc = launch_gated_act_bwd(dh, gq, gs, uq, us, dg, du, m, f, ldg, act, dtype, st);
    if (rc != TB200_OK) return rc;
    if (codes) {
        rc = launch_act_restore(x, xs, xr, dtype, m, k, st);
        if (rc != TB200_OK) return rc;
        x = xr;
    }
    return dtype == TB200_DT_F16 ? ffn_products_bwd<__half>(dg, du, ldg, x, ldx, wg, wu, dx, dwg, dwu, m, f, k, st)
                                 : ffn_products_bwd<__nv_bfloat16>(dg, du, ldg, x, ldx, wg, wu, dx, dwg, dwu, m, f, k, st);
}
