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
// Both kernels below feed one MMA thread from a ring of 128-byte-wide K blocks
// (one 128B swizzle row, 128 values of K, four K = 32 MMAs) filled by one TMA
// thread, as the FP16 family does. They differ in which operand lies along the
// 128 TMEM lanes:
//
//   ridge_gemm_i8_tile    rows of A on the lanes: 256 x BN tiles by 2-CTA pairs,
//                         persistent, two accumulators. For work that fills the
//                         GPU; bound by the tensor cores.
//   ridge_gemm_i8_stream  rows of B on the lanes, up to 256 rows of A as columns,
//                         so few tokens waste no lanes: the MMA's cost falls with
//                         the columns, not below 128 tokens' worth. K is split over
//                         the CTAs of a cluster, which add their integer sums
//                         through distributed shared memory. For few tokens; bound
//                         by the bytes of B.

#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "ptx_sm100.cuh"

namespace ridge_b200 {

constexpr int kI8BK = 128;          // K per ring stage: bytes of one swizzle row
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
    int stages;
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

// Where a tile or split starts in its K range: tiles that share a panel would
// otherwise read the same lines of it at the same moment, and a few lines do not
// spread over the L2 slices. The integer sum does not depend on the order.
__device__ __forceinline__ int i8_first_block(int seed, int num_kb) {
    return num_kb < 16 ? seed % num_kb : seed & 15;
}

// Tile t of the grouped-M order (the FP16 family's order): groupM row tiles at
// a time, column by column inside the group.
__device__ __forceinline__ void i8_tile_coords(int tile, int num_m, int num_n, int groupM, int& tm,
                                               int& tn) {
    const int per_group = groupM * num_n;
    const int group = tile / per_group;
    const int first_m = group * groupM;
    const int rows = min(num_m - first_m, groupM);
    const int in_group = tile - group * per_group;
    tm = first_m + in_group % rows;
    tn = in_group / rows;
}

template <typename T>
__global__ void __launch_bounds__(kI8TileThreads, 1)
    ridge_gemm_i8_tile(const __grid_constant__ CUtensorMap tmap_a,
                       const __grid_constant__ CUtensorMap tmap_b,
                       const __grid_constant__ CUtensorMap tmap_c, const I8Params p) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_addr = smem_u32(smem_raw);
    const uint32_t base = (raw_addr + 1023u) & ~1023u;
    uint8_t* base_ptr = smem_raw + (base - raw_addr);

    const int stages = p.stages;
    const int bn = p.bn;
    const int rows_b = bn / 2;  // rows of B held by this CTA
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
    const int num_tiles = num_m * num_n;
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
        for (int tile = unit; ok && tile < num_tiles; tile += num_units) {
            int tm, tn;
            i8_tile_coords(tile, num_m, num_n, p.groupM, tm, tn);
            const int a_row = tm * 256 + int(rank) * 128;
            const int b_row = tn * bn + int(rank) * rows_b;
            int kb = i8_first_block(3 * tm + 5 * tn, num_kb);
            for (int i = 0; i < num_kb; ++i) {
                if (!mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag, p.err,
                               kErrTimeoutProducer)) {
                    ok = false;
                    break;
                }
                const uint32_t sa = base + stage * stage_bytes;
                const uint32_t fb = leader_full0 + 8u * uint32_t(stage);
                if (leader) mbar_arrive_expect_tx(full_bar(stage), 2 * stage_bytes);
                tma_load_2d_pair(sa, &tmap_a, fb, kb * kI8BK, a_row);
                tma_load_2d_pair(sa + 128 * kI8BK, &tmap_b, fb, kb * kI8BK, b_row);
                if (++kb == num_kb) kb = 0;
                ++issued;
                if (++stage == stages) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
        }
        if (!ok && leader) {
            // Abort path: loads in flight land before the pair can exit (the
            // leader's barriers count the follower's bytes too).
            const long long first = issued > stages ? issued - stages : 0;
            for (long long i = first; i < issued; ++i)
                mbar_wait(full_bar(int(i % stages)), uint32_t((i / stages) & 1), nullptr, p.err,
                          kErrTimeoutDrain);
        }
    } else if (warp == 1 && lane == 0 && leader) {
        // ------------------------------------------------------ MMA issuer
        const uint32_t idesc = make_idesc_i8_s32(256, bn);
        int stage = 0;
        uint32_t phase = 0;
        int acc = 0;
        uint32_t acc_phase = 0;
        bool ok = true;
        for (int tile = unit; ok && tile < num_tiles; tile += num_units) {
            if (!mbar_wait<true>(tempty_bar(acc), acc_phase ^ 1u, abort_flag, p.err,
                                 kErrTimeoutMma)) {
                ok = false;
                break;
            }
            tc_fence_after();
            const uint32_t d = tmem_base + uint32_t(acc * 256);
            for (int kb = 0; kb < num_kb; ++kb) {
                if (!mbar_wait(full_bar(stage), phase, abort_flag, p.err, kErrTimeoutMma)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t sa = base + stage * stage_bytes;
                const uint32_t sb = sa + 128 * kI8BK;
#pragma unroll
                for (int kk = 0; kk < kI8BK / 32; ++kk)
                    umma_i8<2>(d, make_smem_desc<128>(sa + kk * 32),
                               make_smem_desc<128>(sb + kk * 32), idesc,
                               (kb > 0 || kk > 0) ? 1u : 0u);
                umma_commit_pair(empty_bar(stage), 0x3);
                if (++stage == stages) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
            if (!ok) break;
            umma_commit_pair(tfull_bar(acc), 0x3);
            acc ^= 1;
            if (acc == 0) acc_phase ^= 1u;
        }
        if (!ok) {
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
        const int units = bn / 64;
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
                    const uint32_t w = *reinterpret_cast<const uint32_t*>(sbuf_ptr + off);
                    const T* e = reinterpret_cast<const T*>(&w);
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

        for (int tile = unit; tile < num_tiles; tile += num_units) {
            int tm, tn;
            i8_tile_coords(tile, num_m, num_n, p.groupM, tm, tn);
            const int row0 = tm * 256 + int(rank) * 128 + quad * 32;
            const float row_scale = row0 + lane < p.M ? p.sa[row0 + lane] : 0.0f;
            // Fetched while the tile's MMAs still run: read from global memory in
            // the drain itself they made a 256 x 256 tile's epilogue 6.4 us long.
            __syncwarp();
#pragma unroll
            for (int i = 0; i < kI8TileCols / 32; ++i) {
                const int col = tn * bn + (group + 2 * (i / 2)) * 64 + (i % 2) * 32 + lane;
                const bool in = col < p.N;
                cols[i * 32 + lane] = in ? p.sb[col] : 0.0f;
                if (bias) cols[kI8TileCols + i * 32 + lane] = in ? OutType<T>::up(bias[col]) : 0.0f;
            }
            __syncwarp();
            int ok = 1;
            if (lane == 0)
                ok = mbar_wait(tfull_bar(acc), acc_phase, abort_flag, p.err, kErrTimeoutEpilogue);
            ok = __shfl_sync(0xffffffffu, ok, 0);
            if (!ok) break;
            tc_fence_after();
            for (int u = group; u < units; u += 2) {
                const int col0 = tn * bn + u * 64;
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

constexpr int kI8StreamScales = 256 * 4;  // token scales of the tile

__host__ __device__ constexpr int i8_stream_stage_bytes(int bn) { return (128 + bn) * kI8BK; }
constexpr int i8_stream_smem(int bn, int stages) {
    return kI8AlignSlack + stages * i8_stream_stage_bytes(bn) + kI8StreamScales + kI8BarrierBytes;
}

__device__ __forceinline__ int4 ld_cluster_v4(uint32_t addr) {
    int4 v;
    asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(addr)
                 : "memory");
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
    const uint32_t stage_bytes = uint32_t(i8_stream_stage_bytes(bn));
    const uint32_t bars = base + stages * stage_bytes + kI8StreamScales;
    float* token_scale = reinterpret_cast<float*>(base_ptr + stages * stage_bytes);
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

    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        mbar_init(done_bar, 1);
        mbar_init(drain_bar, 1);
        *abort_flag = 0;
        fence_barrier_init();
        tma_prefetch_desc(&tmap_a);
        tma_prefetch_desc(&tmap_b);
    }
    if (warp == 1) {
        tmem_alloc<1>(smem_u32(tmem_slot), tmem_cols);
        tmem_relinquish<1>();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    const int f0 = int(blockIdx.x / SPLIT) * 128;
    const int t0 = int(blockIdx.y) * bn;
    const int num_kb = (p.K + kI8BK - 1) / kI8BK;
    const int kb0 = int((long long)num_kb * rank / SPLIT);
    const int kb1 = int((long long)num_kb * (rank + 1) / SPLIT);
    const int quad = warp & 3;
    const uint32_t lane_taddr = tmem_base + (uint32_t(quad * 32) << 16);
    const T* bias = static_cast<const T*>(p.bias);
    T* C = static_cast<T*>(p.C);
    int ok = 1;

    if (warp == 0 && lane == 0) {
        int stage = 0;
        uint32_t phase = 0;
        int issued = 0;
        bool live = true;
        int kb = kb0 + i8_first_block(3 * int(blockIdx.x / SPLIT) + 5 * int(blockIdx.y), kb1 - kb0);
        for (int i = kb0; i < kb1; ++i) {
            if (!mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag, p.err, kErrTimeoutProducer)) {
                live = false;
                break;
            }
            const uint32_t sb = base + stage * stage_bytes;
            mbar_arrive_expect_tx(full_bar(stage), stage_bytes);
            tma_load_2d(sb, &tmap_b, full_bar(stage), kb * kI8BK, f0);
            tma_load_2d(sb + 128 * kI8BK, &tmap_a, full_bar(stage), kb * kI8BK, t0);
            if (++kb == kb1) kb = kb0;
            ++issued;
            if (++stage == stages) {
                stage = 0;
                phase ^= 1u;
            }
        }
        if (!live) {
            for (int i = issued > stages ? issued - stages : 0; i < issued; ++i)
                mbar_wait(full_bar(i % stages), uint32_t((i / stages) & 1), nullptr, p.err,
                          kErrTimeoutDrain);
        }
    } else if (warp == 1 && lane == 0) {
        const uint32_t idesc = make_idesc_i8_s32(128, bn);
        int stage = 0;
        uint32_t phase = 0;
        bool live = true;
        for (int kb = kb0; kb < kb1; ++kb) {
            if (!mbar_wait(full_bar(stage), phase, abort_flag, p.err, kErrTimeoutMma)) {
                live = false;
                break;
            }
            tc_fence_after();
            const uint32_t sb = base + stage * stage_bytes;
            const uint32_t sa = sb + 128 * kI8BK;
#pragma unroll
            for (int kk = 0; kk < kI8BK / 32; ++kk)
                umma_i8<1>(tmem_base, make_smem_desc<128>(sb + kk * 32),
                           make_smem_desc<128>(sa + kk * 32), idesc,
                           (kb > kb0 || kk > 0) ? 1u : 0u);
            umma_commit(empty_bar(stage));
            if (++stage == stages) {
                stage = 0;
                phase ^= 1u;
            }
        }
        if (live) {
            umma_commit(done_bar);
        } else {
            umma_commit(drain_bar);
            mbar_wait(drain_bar, 0, nullptr, p.err, kErrTimeoutDrain);
        }
    } else if (warp >= 2) {
        for (int i = int(threadIdx.x) - 64; i < bn; i += 128)
            token_scale[i] = t0 + i < p.M ? p.sa[t0 + i] : 0.0f;
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
    __syncwarp();
    if constexpr (SPLIT > 1)
        cluster_sync();  // every rank's sums are in its shared memory
    else
        __syncthreads();
    if (warp >= 2 && ok) {
        // A warp takes whole tokens, four channels to a lane, so that the sums
        // are read and C is written in full lines; the tokens are dealt to the
        // ranks and their warps in turn, four at a time in flight.
        const int f = f0 + lane * 4;
        const int in = p.N - f;  // channels of this lane inside C
        float4 channel, b;
        channel.x = in > 0 ? p.sb[f] : 0.0f;
        channel.y = in > 1 ? p.sb[f + 1] : 0.0f;
        channel.z = in > 2 ? p.sb[f + 2] : 0.0f;
        channel.w = in > 3 ? p.sb[f + 3] : 0.0f;
        b.x = bias && in > 0 ? OutType<T>::up(bias[f]) : 0.0f;
        b.y = bias && in > 1 ? OutType<T>::up(bias[f + 1]) : 0.0f;
        b.z = bias && in > 2 ? OutType<T>::up(bias[f + 2]) : 0.0f;
        b.w = bias && in > 3 ? OutType<T>::up(bias[f + 3]) : 0.0f;
        const int live = min(bn, p.M - t0);  // tokens of this tile
        uint32_t peer[SPLIT];
#pragma unroll
        for (int s = 0; s < SPLIT; ++s)
            peer[s] = SPLIT > 1 ? map_to_cta(base + uint32_t(lane * 16), s)
                                : base + uint32_t(lane * 16);
        constexpr int kStep = 4 * SPLIT;  // tokens between two of one warp's
        constexpr int kFlight = SPLIT >= 8 ? 2 : 4;
        for (int t = rank + (warp - 2) * SPLIT; t < live; t += kFlight * kStep) {
            int4 sum[kFlight];
#pragma unroll
            for (int i = 0; i < kFlight; ++i) {
                const int ti = t + i * kStep;
                sum[i] = make_int4(0, 0, 0, 0);
                if (ti < live) {
#pragma unroll
                    for (int s = 0; s < SPLIT; ++s) {
                        const int4 v = ld_cluster_v4(peer[s] + uint32_t(ti) * 512u);
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
    } else {
        __syncthreads();
    }
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc<1>(tmem_base, tmem_cols);
    }
}

}  // namespace ridge_b200
