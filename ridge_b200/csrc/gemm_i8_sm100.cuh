// The 8-bit GEMM for B200 (sm_100a):
//
//   C[i, j] = sa[i] * sb[j] * sum_k A[i, k] * B[j, k]  (+ bias[j])
//
//   A   signed 8-bit, row-major M x K (lda), one FP32 scale per row (token)
//   B   signed 8-bit, N x K with K contiguous (ldb), one FP32 scale per row (channel)
//   C   FP16, BF16 or FP32, row-major M x N (ldc)
//
// tcgen05.mma kind::i8 accumulates in 32-bit integers in TMEM. |A B| <= 2^14, so
// with K < 2^17 no sum can overflow and the product is exact whatever the order
// of the sum or the split of K. The epilogue rounds the integer to FP32, applies
// sb, sa and the bias there, and rounds once more to the type of C.
//
// The first two kernels below feed one MMA thread from a ring of 128-byte-wide K blocks
// (one 128B swizzle row, 128 values of K, four K = 32 MMAs) filled by one TMA
// thread, as the FP16 family does. They differ in which operand lies along the
// 128 TMEM lanes:
//
//   ridge_gemm_i8_tile    rows of A on the lanes: 256 x BN tiles by 2-CTA pairs,
//                         persistent, two accumulators, so that a tile's drain
//                         hides behind the next one's MMAs. For work that fills the
//                         GPU. Bound by the tensor cores and, in long runs, by the
//                         power they take: 8192^3 326 us (3370 TOP/s) in a burst,
//                         384 us back to back; 2048 x 14336 x 4096 82 us (tensor
//                         pipe 78 to 83% of active cycles, the rest the first loads, the
//                         last drain and the strips of the last round). A short K
//                         leaves the drain uncovered: 8192 x 8192 x 512 50 us, 3.2
//                         us a tile, against 22 us for its bytes.
//   ridge_gemm_i8_stream  rows of B on the lanes, up to 256 rows of A as columns,
//                         so few tokens waste no lanes: the MMA's cost falls with
//                         the columns. K is split over the CTAs of a cluster, which
//                         add their integer sums through distributed shared memory:
//                         exact in any order, no workspace, nothing to clear. For
//                         few tokens. Bound by the bytes of B and a fixed 3.5 us of
//                         launch, set-up, exchange and stores: 8 x 8192 x 8192 14.6
//                         us (4.6 TB/s), 1 x 16384 x 16384 44 us (6.1 TB/s); with
//                         128 tokens 17.8 us, when A passes through every CTA as
//                         well.
//   ridge_gemm_i8_vec     a token or a few and few enough bytes of B: no tensor
//                         cores, no set-up.

#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "ptx_sm100.cuh"

namespace ridge_b200 {

constexpr int kI8BK = 128;          // K block: bytes of one swizzle row
constexpr int kI8MaxStages = 12;
constexpr int kI8BarrierBytes = 256;
constexpr int kI8AlignSlack = 1024;

struct I8Params {
    const float* sa;
    const float* sb;
    const void* bias;  // N values of C's type, or null
    void* C;
    int M, N, K;
    long long ldc;
    int bn;         // tile: columns of C per tile (64, 128, 192, 256); stream: rows of A (16..256)
    int whole;      // tile: tiles computed bn wide; each later one is cut into `cut` narrower
    int cut;        // ones (1 to 4, widths of whole 64s) that fill the last round
    int stages;
    int sub;        // stream: K blocks to a ring stage (1 or 2)
    int groupM;
    int tma_store;  // tile: C is stored through its tensor map; 0: from shared memory by threads
    int vec_store;  // stream: rows of C start on four elements
    int* err;
};

template <typename T>
struct OutType;
template <>
struct OutType<__half> {
    __device__ static float up(__half v) { return __half2float(v); }
    __device__ static __half down(float v) { return __float2half_rn(v); }
    __device__ static uint32_t pack(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
};
template <>
struct OutType<__nv_bfloat16> {
    __device__ static float up(__nv_bfloat16 v) { return __bfloat162float(v); }
    __device__ static __nv_bfloat16 down(float v) { return __float2bfloat16_rn(v); }
    __device__ static uint32_t pack(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
};
template <>
struct OutType<float> {
    __device__ static float up(float v) { return v; }
    __device__ static float down(float v) { return v; }
};

// ------------------------------------------------------------------ tiles by 2-CTA pairs

constexpr int kI8TileThreads = 10 * 32;  // producer, MMA, 8 epilogue warps
constexpr int kI8TileStageOut = 4096;  // 32 rows x 128 bytes of C per epilogue warp
constexpr int kI8TileCols = 2 * 64;    // columns of a tile that one epilogue warp drains
constexpr int kI8TileEpiBytes = 8 * (kI8TileStageOut + kI8TileCols * 8);

__host__ __device__ constexpr int i8_tile_stage_bytes(int bn) {
    return 128 * kI8BK + (bn / 2) * kI8BK;
}
constexpr int i8_tile_smem(int bn, int stages) {
    return kI8AlignSlack + stages * i8_tile_stage_bytes(bn) + kI8TileEpiBytes + kI8BarrierBytes;
}

// Abort path of a producer that has filled `issued` stages in turn: the loads in
// flight, at most one filling of each ring slot, land before the CTA can exit.
__device__ __forceinline__ void i8_drain_loads(uint32_t full_bar0, int stages, long long issued,
                                               int* err) {
    for (long long i = issued > stages ? issued - stages : 0; i < issued; ++i)
        mbar_wait(full_bar0 + 8u * uint32_t(i % stages), uint32_t((i / stages) & 1), nullptr, err,
                  kErrTimeoutDrain);
}

// One unit of work of the tile kernel: rows from 256 * tm, columns [col, col + width).
struct I8Item {
    int tm, tn, col, width;
};

// Item i: the tiles in grouped-M order (the FP16 family's: groupM row tiles at a
// time, column by column inside the group), those from `whole` on cut into
// column strips. A last round of few tiles then takes all pairs for less than a
// tile's time instead of a few pairs for all of it.
__device__ __forceinline__ bool i8_item(const I8Params& p, int i, int num_m, int num_n, I8Item& w) {
    int tile = i, strip = 0, cut = 1;
    if (i >= p.whole) {
        cut = p.cut;
        tile = p.whole + (i - p.whole) / cut;
        strip = (i - p.whole) % cut;
    }
    if (tile >= num_m * num_n) return false;
    const int per_group = p.groupM * num_n;
    const int group = tile / per_group;
    const int first_m = group * p.groupM;
    const int rows = min(num_m - first_m, p.groupM);
    const int in_group = tile - group * per_group;
    w.tm = first_m + in_group % rows;
    w.tn = in_group / rows;
    w.width = p.bn / cut;
    w.col = w.tn * p.bn + strip * w.width;
    return true;
}

template <typename T>
__global__ void __launch_bounds__(kI8TileThreads, 1)
    ridge_gemm_i8_tile(const __grid_constant__ CUtensorMap tmap_a,
                       const __grid_constant__ CUtensorMap tmap_b,
                       const __grid_constant__ CUtensorMap tmap_strip,
                       const __grid_constant__ CUtensorMap tmap_c, const I8Params p) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_addr = smem_u32(smem_raw);
    const uint32_t base = (raw_addr + 1023u) & ~1023u;
    uint8_t* base_ptr = smem_raw + (base - raw_addr);

    const int stages = p.stages;
    const int bn = p.bn;
    const uint32_t stage_bytes = uint32_t(i8_tile_stage_bytes(bn));
    const uint32_t epi_base = base + stages * stage_bytes;
    const uint32_t bars = epi_base + kI8TileEpiBytes;
    auto full_bar = [&](int s) { return bars + 8u * s; };
    auto empty_bar = [&](int s) { return bars + 8u * (kI8MaxStages + s); };
    auto tfull_bar = [&](int b) { return bars + 8u * (2 * kI8MaxStages + b); };
    auto tempty_bar = [&](int b) { return bars + 8u * (2 * kI8MaxStages + 2 + b); };
    const uint32_t drain_bar = bars + 8u * (2 * kI8MaxStages + 4);
    uint32_t* tmem_slot =
        reinterpret_cast<uint32_t*>(base_ptr + (bars - base) + 8 * (2 * kI8MaxStages + 5));
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t rank = cluster_cta_rank();
    const bool leader = rank == 0;

    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(tfull_bar(b), 1);
            mbar_init(tempty_bar(b), 2 * 8);
        }
        mbar_init(drain_bar, 1);
        *abort_flag = 0;
        fence_barrier_init();
        tma_prefetch_desc(&tmap_a);
        tma_prefetch_desc(&tmap_b);
        if (p.tma_store) tma_prefetch_desc(&tmap_c);
    }
    if (warp == 1) {
        tmem_alloc<2>(smem_u32(tmem_slot), 512);
        tmem_relinquish<2>();
    }
    tc_fence_before();
    __syncwarp();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    const int num_m = (p.M + 255) / 256;
    const int num_n = (p.N + bn - 1) / bn;
    const int num_kb = (p.K + kI8BK - 1) / kI8BK;
    const int unit = blockIdx.x / 2;
    const int num_units = gridDim.x / 2;

    if (warp == 0 && lane == 0) {
        // ------------------------------------------------------ TMA producer
        const uint32_t leader_full0 = map_to_cta(full_bar(0), 0);
        int stage = 0;
        uint32_t phase = 0;
        long long issued = 0;
        bool ok = true;
        I8Item w;
        for (int it = unit; ok && i8_item(p, it, num_m, num_n, w); it += num_units) {
            const int rows_b = w.width / 2;  // rows of B held by this CTA
            const int a_row = w.tm * 256 + int(rank) * 128;
            const int b_row = w.col + int(rank) * rows_b;
            const void* map_b = w.width == bn ? &tmap_b : &tmap_strip;
            const uint32_t bytes = uint32_t(i8_tile_stage_bytes(w.width));
            for (int kb = 0; kb < num_kb; ++kb) {
                if (!mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag, p.err,
                               kErrTimeoutProducer)) {
                    ok = false;
                    break;
                }
                const uint32_t sa = base + stage * stage_bytes;
                const uint32_t fb = leader_full0 + 8u * uint32_t(stage);
                if (leader) mbar_arrive_expect_tx(full_bar(stage), 2 * bytes);
                tma_load_2d_pair(sa, &tmap_a, fb, kb * kI8BK, a_row);
                tma_load_2d_pair(sa + 128 * kI8BK, map_b, fb, kb * kI8BK, b_row);
                ++issued;
                if (++stage == stages) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
        }
        // The leader's barriers count the follower's bytes too, and neither CTA
        // leaves before the last cluster barrier.
        if (!ok && leader) i8_drain_loads(full_bar(0), stages, issued, p.err);
    } else if (warp == 1 && leader) {
        // ------------------------------------------------------ MMA issuer
        // The whole warp walks the ring and one elected lane issues: with every
        // address warp-uniform an MMA takes a few instructions to issue, against
        // about 75 cycles each from a lane that the compiler sees as divergent.
        int stage = 0;
        uint32_t phase = 0;
        int acc = 0;
        uint32_t acc_phase = 0;
        bool ok = true;
        I8Item w;
        for (int it = unit; ok && i8_item(p, it, num_m, num_n, w); it += num_units) {
            const uint32_t idesc = make_idesc_i8_s32(256, w.width);
            ok = __all_sync(0xffffffffu, mbar_wait<true>(tempty_bar(acc), acc_phase ^ 1u,
                                                         abort_flag, p.err, kErrTimeoutMma));
            if (!ok) break;
            tc_fence_after();
            const uint32_t d = tmem_base + uint32_t(acc * 256);
            for (int kb = 0; kb < num_kb; ++kb) {
                ok = __all_sync(0xffffffffu, mbar_wait(full_bar(stage), phase, abort_flag, p.err,
                                                       kErrTimeoutMma));
                if (!ok) break;
                tc_fence_after();
                const uint32_t sa = base + stage * stage_bytes;
                const uint64_t da = make_smem_desc<128>(sa);
                const uint64_t db = make_smem_desc<128>(sa + 128 * kI8BK);
                if (elect_one()) {
#pragma unroll
                    for (int kk = 0; kk < kI8BK / 32; ++kk)  // 32 bytes on: 2 in address >> 4
                        umma_i8<2>(d, da + 2 * kk, db + 2 * kk, idesc,
                                   (kb > 0 || kk > 0) ? 1u : 0u);
                    umma_commit_pair(empty_bar(stage), 0x3);
                }
                __syncwarp();
                if (++stage == stages) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
            if (!ok) break;
            if (elect_one()) umma_commit_pair(tfull_bar(acc), 0x3);
            __syncwarp();
            acc ^= 1;
            if (acc == 0) acc_phase ^= 1u;
        }
        if (!ok && elect_one()) {
            umma_commit_pair(drain_bar, 0x1);
            mbar_wait(drain_bar, 0, nullptr, p.err, kErrTimeoutDrain);
        }
    } else if (warp >= 2) {
        // ------------------------------------------------------ epilogue
        // A warp drains 32 rows x 64 columns at a time (two column groups of four
        // warps take alternate 64s): TMEM -> registers -> scaled -> 4 KB of
        // shared memory (rows of 128 bytes, 128B-swizzled) -> C.
        const int epi = warp - 2;
        const int quad = warp & 3;
        const int group = epi >> 2;
        const uint32_t tempty0 = map_to_cta(tempty_bar(0), 0);
        const uint32_t sbuf = epi_base + uint32_t(epi * kI8TileStageOut);
        uint8_t* sbuf_ptr = base_ptr + (sbuf - base);
        // Channel scales and biases of this warp's columns of the tile.
        float* cols = reinterpret_cast<float*>(base_ptr + (epi_base - base) + 8 * kI8TileStageOut) +
                      epi * 2 * kI8TileCols;
        const uint32_t row_addr = sbuf + uint32_t(lane * 128);
        const uint32_t sw = uint32_t(lane & 7);
        const T* bias = static_cast<const T*>(p.bias);
        T* C = static_cast<T*>(p.C);
        int acc = 0;
        uint32_t acc_phase = 0;

        // 32 rows x 128 bytes, staged by the warp's lanes, to C at (row0, col0).
        // A tensor-map store clips rows at M but columns only at the next 16-byte
        // boundary of C (measured: with N = 333 it also wrote columns 333..335),
        // so a box that runs past an N that is none is stored by threads.
        constexpr int kBoxCols = 128 / int(sizeof(T));
        auto store_staged = [&](const uint32_t (&word)[32], int row0, int col0) {
            const bool by_map =
                p.tma_store &&
                (col0 + kBoxCols <= p.N || p.N % (16 / int(sizeof(T))) == 0);
            if (p.tma_store) {
                if (lane == 0) tma_store_wait_read<0>();
            }
            __syncwarp();
#pragma unroll
            for (int c = 0; c < 8; ++c)
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(
                                 row_addr + ((uint32_t(c) ^ sw) << 4)),
                             "r"(word[4 * c]), "r"(word[4 * c + 1]), "r"(word[4 * c + 2]),
                             "r"(word[4 * c + 3])
                             : "memory");
            if (by_map) {
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    tma_store_2d(&tmap_c, sbuf, col0, row0);
                    tma_store_commit();
                }
            } else {
                // C's rows start anywhere: one row at a time, lane by lane.
                __syncwarp();
                constexpr int kPer = 4 / int(sizeof(T));  // elements per staged word
                for (int r = 0; r < 32 && row0 + r < p.M; ++r) {
                    const uint32_t off =
                        uint32_t(r * 128) +
                        (((uint32_t(lane >> 2)) ^ uint32_t(r & 7)) << 4) + uint32_t((lane & 3) * 4);
                    const uint32_t bits = *reinterpret_cast<const uint32_t*>(sbuf_ptr + off);
                    const T* e = reinterpret_cast<const T*>(&bits);
                    T* dst = C + (long long)(row0 + r) * p.ldc;
#pragma unroll
                    for (int i = 0; i < kPer; ++i) {
                        const int col = col0 + lane * kPer + i;
                        if (col < p.N) dst[col] = e[i];
                    }
                }
                __syncwarp();
            }
        };
        // Integers to values of C in place: r[j] = bits of (float(r[j]) * sb) * sa + bias.
        auto scale_half = [&](uint32_t (&r)[32], float row_scale, const float* col) {
#pragma unroll
            for (int g = 0; g < 8; ++g) {
                const float4 s = *reinterpret_cast<const float4*>(col + 4 * g);
                float4 b = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (bias) b = *reinterpret_cast<const float4*>(col + kI8TileCols + 4 * g);
                r[4 * g] = __float_as_uint(fmaf(float(int(r[4 * g])) * s.x, row_scale, b.x));
                r[4 * g + 1] = __float_as_uint(fmaf(float(int(r[4 * g + 1])) * s.y, row_scale, b.y));
                r[4 * g + 2] = __float_as_uint(fmaf(float(int(r[4 * g + 2])) * s.z, row_scale, b.z));
                r[4 * g + 3] = __float_as_uint(fmaf(float(int(r[4 * g + 3])) * s.w, row_scale, b.w));
            }
        };

        // An item's scales and biases go through registers to shared memory, fetched
        // while the item before it is drained: read from global memory in the drain
        // itself they made a 256 x 256 tile's epilogue 6.4 us long.
        constexpr int kFetch = kI8TileCols / 32;
        float next_sa = 0.0f, next_sb[kFetch], next_bias[kFetch];
        I8Item w, next;
        auto fetch = [&](const I8Item& t) {
            const int row = t.tm * 256 + int(rank) * 128 + quad * 32 + lane;
            next_sa = row < p.M ? p.sa[row] : 0.0f;
#pragma unroll
            for (int i = 0; i < kFetch; ++i) {
                const int col = t.col + (group + 2 * (i / 2)) * 64 + (i % 2) * 32 + lane;
                next_sb[i] = col < p.N ? p.sb[col] : 0.0f;
                next_bias[i] = bias && col < p.N ? OutType<T>::up(bias[col]) : 0.0f;
            }
        };
        bool more = i8_item(p, unit, num_m, num_n, next);
        if (more) fetch(next);
        for (int it = unit; more; it += num_units) {
            w = next;
            const int units = w.width / 64;
            const int row0 = w.tm * 256 + int(rank) * 128 + quad * 32;
            const float row_scale = next_sa;
            __syncwarp();
#pragma unroll
            for (int i = 0; i < kFetch; ++i) {
                cols[i * 32 + lane] = next_sb[i];
                if (bias) cols[kI8TileCols + i * 32 + lane] = next_bias[i];
            }
            __syncwarp();
            more = i8_item(p, it + num_units, num_m, num_n, next);
            if (more) fetch(next);
            int ok = 1;
            if (lane == 0)
                ok = mbar_wait(tfull_bar(acc), acc_phase, abort_flag, p.err, kErrTimeoutEpilogue);
            ok = __shfl_sync(0xffffffffu, ok, 0);
            if (!ok) break;
            tc_fence_after();
            for (int u = group; u < units; u += 2) {
                const int col0 = w.col + u * 64;
                if (row0 >= p.M || col0 >= p.N) break;  // nothing of this warp's is in C
                uint32_t ra[32], rb[32];
                const uint32_t taddr = tmem_base + (uint32_t(quad * 32) << 16) +
                                       uint32_t(acc * 256 + u * 64);
                tmem_ld_32x32b_x32(taddr, ra);
                tmem_ld_32x32b_x32(taddr + 32, rb);
                tmem_wait_ld(ra);
                tmem_wait_ld(rb);
                const float* col = cols + (u >> 1) * 64;
                scale_half(ra, row_scale, col);
                scale_half(rb, row_scale, col + 32);
                if constexpr (sizeof(T) == 4) {
                    store_staged(ra, row0, col0);
                    if (col0 + 32 < p.N) store_staged(rb, row0, col0 + 32);
                } else {
                    uint32_t word[32];
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        word[e] = OutType<T>::pack(__uint_as_float(ra[2 * e]),
                                                   __uint_as_float(ra[2 * e + 1]));
                        word[16 + e] = OutType<T>::pack(__uint_as_float(rb[2 * e]),
                                                        __uint_as_float(rb[2 * e + 1]));
                    }
                    store_staged(word, row0, col0);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(tempty0 + 8u * acc);
            acc ^= 1;
            if (acc == 0) acc_phase ^= 1u;
        }
        if (p.tma_store && lane == 0) tma_store_wait_all<0>();
    }

    tc_fence_before();
    __syncwarp();
    cluster_sync();  // neither CTA frees TMEM or exits while its peer may still use it
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc<2>(tmem_base, 512);
    }
}

// ------------------------------------------------------------------ B streamed past few rows of A

constexpr int kI8StreamThreads = 6 * 32;  // producer, MMA, 4 epilogue warps

constexpr int kI8StreamScales = (256 + 128 + 128) * 4;  // token and channel scales, biases

__host__ __device__ constexpr int i8_stream_block_bytes(int bn) { return (128 + bn) * kI8BK; }
constexpr int i8_stream_smem(int bn, int blocks) {
    return kI8AlignSlack + blocks * i8_stream_block_bytes(bn) + kI8StreamScales + kI8BarrierBytes;
}

template <bool kRemote>
__device__ __forceinline__ int4 ld_sums(uint32_t addr) {
    int4 v;
    if constexpr (kRemote)
        asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                     : "r"(addr));
    else
        asm volatile("ld.shared.v4.s32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                     : "r"(addr));
    return v;
}

// Four values of C at dst, the first `n` of them inside it.
template <typename T>
__device__ __forceinline__ void store4(T* dst, float4 v, int n, bool vec) {
    if (vec && n >= 4) {
        if constexpr (sizeof(T) == 4)
            *reinterpret_cast<float4*>(dst) = v;
        else
            *reinterpret_cast<uint2*>(dst) =
                make_uint2(OutType<T>::pack(v.x, v.y), OutType<T>::pack(v.z, v.w));
        return;
    }
    if (n > 0) dst[0] = OutType<T>::down(v.x);
    if (n > 1) dst[1] = OutType<T>::down(v.y);
    if (n > 2) dst[2] = OutType<T>::down(v.z);
    if (n > 3) dst[3] = OutType<T>::down(v.w);
}

// SPLIT CTAs of one cluster share a tile of 128 channels x bn tokens, each with a
// contiguous range of K blocks. blockIdx.x = channel tile * SPLIT + rank,
// blockIdx.y = token tile.
template <typename T, int SPLIT>
__global__ void __launch_bounds__(kI8StreamThreads)
    ridge_gemm_i8_stream(const __grid_constant__ CUtensorMap tmap_a,
                         const __grid_constant__ CUtensorMap tmap_b, const I8Params p) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_addr = smem_u32(smem_raw);
    const uint32_t base = (raw_addr + 1023u) & ~1023u;
    uint8_t* base_ptr = smem_raw + (base - raw_addr);

    const int stages = p.stages;
    const int bn = p.bn;
    const int sub = p.sub;
    const uint32_t block_bytes = uint32_t(i8_stream_block_bytes(bn));
    const uint32_t stage_bytes = uint32_t(sub) * block_bytes;
    const uint32_t bars = base + stages * stage_bytes + kI8StreamScales;
    float* token_scale = reinterpret_cast<float*>(base_ptr + stages * stage_bytes);
    float* channel_scale = token_scale + 256;
    float* channel_bias = channel_scale + 128;
    auto full_bar = [&](int s) { return bars + 8u * s; };
    auto empty_bar = [&](int s) { return bars + 8u * (kI8MaxStages + s); };
    const uint32_t done_bar = bars + 8u * (2 * kI8MaxStages);
    const uint32_t drain_bar = bars + 8u * (2 * kI8MaxStages + 1);
    uint32_t* tmem_slot =
        reinterpret_cast<uint32_t*>(base_ptr + (bars - base) + 8 * (2 * kI8MaxStages + 2));
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int rank = SPLIT > 1 ? int(cluster_cta_rank()) : 0;
    uint32_t tmem_cols = 32;
    while (int(tmem_cols) < bn) tmem_cols *= 2;

    const int f0 = int(blockIdx.x / SPLIT) * 128;
    const int t0 = int(blockIdx.y) * bn;
    const int num_kb = (p.K + kI8BK - 1) / kI8BK;
    const int kb0 = int((long long)num_kb * rank / SPLIT);
    const int kb1 = int((long long)num_kb * (rank + 1) / SPLIT);
    const int blocks = kb1 - kb0;
    const int steps = (blocks + sub - 1) / sub;
    // K block of this CTA's i-th place, and the loads of a step. CTAs start at
    // different places of their K range (the sum does not depend on the order):
    // 1 x 8192 x 8192 14.3 us, against 14.9 with all in step. Tiles of the other
    // kernel share panels and are 2 to 5% faster in step.
    const int spread = 3 * int(blockIdx.x / SPLIT) + 5 * int(blockIdx.y);
    const int turn = blocks < 16 ? spread % blocks : spread & 15;
    auto load = [&](int stage, int step) {
        const int n = min(sub, blocks - step * sub);
        mbar_arrive_expect_tx(full_bar(stage), uint32_t(n) * block_bytes);
        for (int j = 0; j < n; ++j) {
            const int place = kb0 + turn + step * sub + j;
            const int x = (place < kb1 ? place : place - blocks) * kI8BK;
            const uint32_t at = base + stage * stage_bytes + j * block_bytes;
            tma_load_2d(at, &tmap_b, full_bar(stage), x, f0);
            tma_load_2d(at + 128 * kI8BK, &tmap_a, full_bar(stage), x, t0);
        }
    };

    if (threadIdx.x == 0) {
        tma_prefetch_desc(&tmap_b);
        tma_prefetch_desc(&tmap_a);
        for (int s = 0; s < stages; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        mbar_init(done_bar, 1);
        mbar_init(drain_bar, 1);
        *abort_flag = 0;
        fence_barrier_init();
        // The first loads do not wait for the rest of the set-up.
        for (int s = 0; s < min(stages, steps); ++s) load(s, s);
    }
    if (warp == 1) {
        tmem_alloc<1>(smem_u32(tmem_slot), tmem_cols);
        tmem_relinquish<1>();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    const int quad = warp & 3;
    const uint32_t lane_taddr = tmem_base + (uint32_t(quad * 32) << 16);
    const T* bias = static_cast<const T*>(p.bias);
    T* C = static_cast<T*>(p.C);

    if (warp == 0 && lane == 0) {
        const int first = min(stages, steps);  // under way already
        int stage = first == stages ? 0 : first;
        uint32_t phase = first == stages ? 1u : 0u;
        int i = first;
        for (; i < steps; ++i) {
            if (!mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag, p.err, kErrTimeoutProducer))
                break;
            load(stage, i);
            if (++stage == stages) {
                stage = 0;
                phase ^= 1u;
            }
        }
        if (i < steps) i8_drain_loads(full_bar(0), stages, i, p.err);
    } else if (warp == 1) {
        const uint32_t idesc = make_idesc_i8_s32(128, bn);
        int stage = 0;
        uint32_t phase = 0;
        bool live = true;
        for (int i = 0; i < steps; ++i) {
            live = __all_sync(0xffffffffu, mbar_wait(full_bar(stage), phase, abort_flag, p.err,
                                                     kErrTimeoutMma));
            if (!live) break;
            tc_fence_after();
            const uint32_t sb = base + stage * stage_bytes;
            const int n = min(sub, blocks - i * sub);
            if (elect_one()) {
                for (int j = 0; j < n; ++j) {
                    const uint64_t db = make_smem_desc<128>(sb + j * block_bytes);
                    const uint64_t da = make_smem_desc<128>(sb + j * block_bytes + 128 * kI8BK);
#pragma unroll
                    for (int kk = 0; kk < kI8BK / 32; ++kk)
                        umma_i8<1>(tmem_base, db + 2 * kk, da + 2 * kk, idesc,
                                   (i > 0 || j > 0 || kk > 0) ? 1u : 0u);
                }
                umma_commit(empty_bar(stage));
            }
            __syncwarp();
            if (++stage == stages) {
                stage = 0;
                phase ^= 1u;
            }
        }
        if (elect_one()) {
            if (live) {
                umma_commit(done_bar);
            } else {
                umma_commit(drain_bar);
                mbar_wait(drain_bar, 0, nullptr, p.err, kErrTimeoutDrain);
            }
        }
    } else if (warp >= 2) {
        for (int i = int(threadIdx.x) - 64; i < bn; i += 128)
            token_scale[i] = t0 + i < p.M ? p.sa[t0 + i] : 0.0f;
        {
            const int i = int(threadIdx.x) - 64;
            channel_scale[i] = f0 + i < p.N ? p.sb[f0 + i] : 0.0f;
            channel_bias[i] = bias && f0 + i < p.N ? OutType<T>::up(bias[f0 + i]) : 0.0f;
        }
        int ok = 1;
        if (lane == 0) ok = mbar_wait(done_bar, 0, abort_flag, p.err, kErrTimeoutEpilogue);
        ok = __shfl_sync(0xffffffffu, ok, 0);
        tc_fence_after();
        // Every load has landed and every MMA has read it, so the ring can hold
        // this CTA's sums: token t, channel c at int t * 128 + c.
        int* part = reinterpret_cast<int*>(base_ptr) + quad * 32 + lane;
        for (int c = 0; ok && c < bn && t0 + c < p.M; c += 16) {
            uint32_t r[16];
            tmem_ld_32x32b_x16(lane_taddr + uint32_t(c), r);
            tmem_wait_ld(r);
#pragma unroll
            for (int i = 0; i < 16; ++i) part[(c + i) * 128] = int(r[i]);
        }
    }

    tc_fence_before();
    __syncthreads();
    // TMEM goes back before this CTA waits for its cluster. A rank may itself be
    // waiting for TMEM, held by a CTA of another kernel that waits for TMEM held
    // here (a pair of the FP16 family, launched on another stream).
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc<1>(tmem_base, tmem_cols);
    }
    __syncwarp();
    if constexpr (SPLIT > 1) cluster_sync();  // every rank's sums are in its shared memory
    if (!*abort_flag) {
        // A warp takes whole tokens, four channels to a lane, so that the sums
        // are read and C is written in full lines; the tokens are dealt to the
        // ranks and their warps (all of them by now idle) in turn, several at a
        // time in flight.
        const int f = f0 + lane * 4;
        const int in = p.N - f;  // channels of this lane inside C
        const float4 channel = *reinterpret_cast<const float4*>(channel_scale + lane * 4);
        const float4 b = *reinterpret_cast<const float4*>(channel_bias + lane * 4);
        const int live = min(bn, p.M - t0);  // tokens of this tile
        // The other ranks' sums, and this CTA's own without the way over the cluster.
        uint32_t peer[SPLIT];
        peer[0] = base + uint32_t(lane * 16);
#pragma unroll
        for (int s = 1; s < SPLIT; ++s) peer[s] = map_to_cta(peer[0], uint32_t((rank + s) % SPLIT));
        constexpr int kStep = (kI8StreamThreads / 32) * SPLIT;  // tokens between two of a warp's
        constexpr int kFlight = SPLIT >= 8 ? 2 : SPLIT >= 4 ? 4 : 8;
        for (int t = rank + warp * SPLIT; t < live; t += kFlight * kStep) {
            int4 sum[kFlight];
#pragma unroll
            for (int i = 0; i < kFlight; ++i) {
                const int ti = t + i * kStep;
                sum[i] = make_int4(0, 0, 0, 0);
                if (ti < live) {
                    sum[i] = ld_sums<false>(peer[0] + uint32_t(ti) * 512u);
#pragma unroll
                    for (int s = 1; s < SPLIT; ++s) {
                        const int4 v = ld_sums<true>(peer[s] + uint32_t(ti) * 512u);
                        sum[i].x += v.x;
                        sum[i].y += v.y;
                        sum[i].z += v.z;
                        sum[i].w += v.w;
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < kFlight; ++i) {
                const int ti = t + i * kStep;
                if (ti >= live) break;
                const float token = token_scale[ti];
                float4 v;
                v.x = fmaf(float(sum[i].x) * channel.x, token, b.x);
                v.y = fmaf(float(sum[i].y) * channel.y, token, b.y);
                v.z = fmaf(float(sum[i].z) * channel.z, token, b.z);
                v.w = fmaf(float(sum[i].w) * channel.w, token, b.w);
                store4<T>(C + (long long)(t0 + ti) * p.ldc + f, v, in, p.vec_store);
            }
        }
    }
    if constexpr (SPLIT > 1) {
        __syncwarp();
        cluster_sync();  // no rank leaves while another reads its sums
    }
}

// ------------------------------------------------------------------ one to four tokens

constexpr int kI8VecWarps = 8;

// 16 bytes of B, read once: not kept in L1.
__device__ __forceinline__ int4 ld_once(const int8_t* p) {
    int4 v;
    asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.s32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}

__device__ __forceinline__ int dot16(int4 a, int4 b, int sum) {
    sum = __dp4a(a.x, b.x, sum);
    sum = __dp4a(a.y, b.y, sum);
    sum = __dp4a(a.z, b.z, sum);
    return __dp4a(a.w, b.w, sum);
}

// Two channels at a time by a warp, whose lanes take 16 bytes of each in turn;
// `ksplit` warps of a CTA share the channels' K. A comes from L1, once for both
// channels. No set-up and no barrier stand before the first load (the streaming
// kernel's 3.5 us), and lanes multiply four bytes an instruction: bound by the
// bytes of B as long as a token or two share them, then by reading A again and
// again. 1 x 4096 x 4096 5.1 us (the streaming kernel 6.9), 1 x 1000 x 1000 2.6
// (4.3), 1 x 8192 x 8192 13.6 (13.8).
constexpr int kI8VecRows = 2;

template <typename T, int TOKENS>
__global__ void __launch_bounds__(kI8VecWarps * 32)
    ridge_gemm_i8_vec(const int8_t* __restrict__ A, const int8_t* __restrict__ B, long long lda,
                      long long ldb, int ksplit, const I8Params p) {
    __shared__ int s_sum[kI8VecWarps][kI8VecRows * TOKENS];
    constexpr int ROWS = kI8VecRows;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int group = warp / ksplit, part = warp - group * ksplit;
    const long long f0 = ((long long)blockIdx.x * (kI8VecWarps / ksplit) + group) * ROWS;
    const int chunks = p.K / 16;
    const int c0 = int((long long)chunks * part / ksplit);
    const int c1 = int((long long)chunks * (part + 1) / ksplit);
    // Channels and tokens past the end repeat the last one and are not stored.
    const int8_t* b[ROWS];
    const int8_t* a[TOKENS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) b[r] = B + min(f0 + r, (long long)p.N - 1) * ldb;
#pragma unroll
    for (int t = 0; t < TOKENS; ++t) a[t] = A + min(t, p.M - 1) * lda;
    int sum[ROWS][TOKENS] = {};
    constexpr int kUnroll = 4;  // 128 bytes of B in flight per lane
    int c = c0 + lane;
    for (; c + 32 * (kUnroll - 1) < c1; c += 32 * kUnroll) {
        int4 vb[kUnroll][ROWS];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
#pragma unroll
            for (int r = 0; r < ROWS; ++r) vb[u][r] = ld_once(b[r] + 16ll * (c + 32 * u));
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
#pragma unroll
            for (int t = 0; t < TOKENS; ++t) {
                const int4 va = *reinterpret_cast<const int4*>(a[t] + 16ll * (c + 32 * u));
#pragma unroll
                for (int r = 0; r < ROWS; ++r) sum[r][t] = dot16(va, vb[u][r], sum[r][t]);
            }
    }
    for (; c < c1; c += 32)
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const int4 vb = ld_once(b[r] + 16ll * c);
#pragma unroll
            for (int t = 0; t < TOKENS; ++t)
                sum[r][t] =
                    dot16(*reinterpret_cast<const int4*>(a[t] + 16ll * c), vb, sum[r][t]);
        }
    // The last K % 16 bytes of a row, one to a lane: nothing past them is read.
    if (part == 0 && lane < p.K - chunks * 16) {
        const int k = chunks * 16 + lane;
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
#pragma unroll
            for (int t = 0; t < TOKENS; ++t) sum[r][t] += int(a[t][k]) * int(b[r][k]);
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
        for (int t = 0; t < TOKENS; ++t)
            sum[r][t] = __reduce_add_sync(0xffffffffu, sum[r][t]);
    if (ksplit > 1) {
        if (lane == 0)
#pragma unroll
            for (int i = 0; i < ROWS * TOKENS; ++i) s_sum[warp][i] = sum[i / TOKENS][i % TOKENS];
        __syncthreads();
        if (part != 0) return;
        for (int w = 1; w < ksplit; ++w)
#pragma unroll
            for (int i = 0; i < ROWS * TOKENS; ++i)
                sum[i / TOKENS][i % TOKENS] += s_sum[warp + w][i];
    }
    const T* bias = static_cast<const T*>(p.bias);
    T* C = static_cast<T*>(p.C);
#pragma unroll
    for (int i = 0; i < ROWS * TOKENS; ++i) {
        const int r = i / TOKENS, t = i % TOKENS;
        const long long f = f0 + r;
        if (lane == i && f < p.N && t < p.M)
            C[t * p.ldc + f] = OutType<T>::down(fmaf(float(sum[r][t]) * p.sb[f], p.sa[t],
                                                     bias ? OutType<T>::up(bias[f]) : 0.0f));
    }
}

}  // namespace ridge_b200
