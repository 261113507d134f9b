// C-ABI front end of the 8-bit GEMM (gemm_i8_sm100.cuh, include/ridge_b200.h):
// argument checks, tensor maps, and the choice of kernel and tile.

#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstring>

#include "../../include/ridge_b200.h"
#include "device_info.h"
#include "gemm_i8_sm100.cuh"
#include "row_arrays.h"

namespace ridge_b200 {
namespace {

constexpr int kMaxDevices = 64;
constexpr int kMaxDynSmem = 232448;  // 227 KB opt-in limit per CTA on sm_100
constexpr int kSmemPerSm = 233472;   // 228 KB per SM
constexpr int kSmemReservedPerCta = 1024;
constexpr int kTmemColsPerSm = 512;

// K = 0: no sum, C is the bias (a non-finite scale still makes its row or column NaN).
template <typename T>
__global__ void ridge_gemm_i8_empty(const I8Params p) {
    const int col = int(blockIdx.x) * blockDim.x + threadIdx.x;
    if (col >= p.N) return;
    const float s = 0.0f * p.sb[col];
    const float b = p.bias ? OutType<T>::up(static_cast<const T*>(p.bias)[col]) : 0.0f;
    for (long long row = blockIdx.y; row < p.M; row += gridDim.y)
        static_cast<T*>(p.C)[row * p.ldc + col] = OutType<T>::down(fmaf(s, p.sa[row], b));
}

// One launch: which kernel, its tile and its ring.
struct Plan {
    bool stream;
    int bn, stages;
    int sub;          // stream: K blocks to a stage
    int split;        // stream: CTAs of a cluster that share K
    int64_t items;    // units of work: tiles and strips, or CTAs of the streaming kernel
    int64_t whole;    // tile: see I8Params
    int cut;
};

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

int stages_for(int stage_bytes, int fixed, int budget) {
    return std::min(kI8MaxStages, (budget - fixed) / stage_bytes);
}

// The tile kernel's grid for tiles bn wide on `pairs` resident pairs: full rounds
// of whole tiles, and a last round whose tiles are cut into as many strips (of
// whole 64 columns) as there are pairs to take them.
Plan tile_plan(int64_t M, int64_t N, int bn, int pairs) {
    Plan p{};
    p.bn = bn;
    p.stages = stages_for(i8_tile_stage_bytes(bn), i8_tile_smem(bn, 0), kMaxDynSmem);
    p.split = 1;
    const int64_t tiles = ceil_div(M, 256) * ceil_div(N, bn);
    const int64_t last = tiles % pairs;
    p.cut = 1;
    for (int cut = 2; last > 0 && cut <= bn / 64; ++cut)
        if (bn % (64 * cut) == 0 && last * cut <= pairs) p.cut = cut;
    p.whole = p.cut > 1 ? tiles - last : tiles;
    p.items = p.whole + (tiles - p.whole) * p.cut;
    return p;
}

// CTAs of the streaming kernel that share an SM with this ring.
int stream_residents(int bn, int blocks) {
    int cols = 32;
    while (cols < bn) cols *= 2;
    const int by_smem = kSmemPerSm / (i8_stream_smem(bn, blocks) + kSmemReservedPerCta);
    return std::max(1, std::min(by_smem, kTmemColsPerSm / cols));
}

// Up to `bn` tokens to a tile, evened out over the tiles, and the ring: all of
// the shared memory when every CTA can have an SM to itself, else half of it
// where that leaves three K blocks.
Plan stream_plan(int64_t M, int64_t N, int64_t K, int bn, int split, int num_sms) {
    Plan p{};
    p.stream = true;
    p.split = split;
    const int64_t token_tiles = ceil_div(M, bn);
    p.bn = int(ceil_div(ceil_div(M, token_tiles), 16) * 16);
    p.items = ceil_div(N, 128) * ceil_div(M, p.bn) * split;
    // Two K blocks to a stage halve the barrier waits a block costs (1 x 1024 x
    // 4096 5.6 -> 5.2 us, 16 x 11008 x 512 4.8 -> 4.3); from 128 tokens on the ring
    // has too few stages left for it (128 x 8192 x 8192 19.2 -> 19.6).
    p.sub = p.bn <= 64 ? 2 : 1;
    const int fixed = i8_stream_smem(p.bn, 0);
    const int stage = p.sub * i8_stream_block_bytes(p.bn);
    p.stages = stages_for(stage, fixed, kMaxDynSmem);
    if (p.items > num_sms) {
        const int half = stages_for(stage, fixed, kSmemPerSm / 2 - kSmemReservedPerCta);
        if (half * p.sub >= 3) p.stages = half;
    }
    // No more than K fills, so that short products leave room for more CTAs, but
    // enough to hold the sums of the tile (bn tokens x 128 channels) at the end.
    const int64_t steps = ceil_div(ceil_div(ceil_div(K, kI8BK), split), p.sub);
    const int64_t sums = ceil_div(int64_t(p.bn) * 512, stage);
    p.stages = int(std::min<int64_t>(p.stages, std::max(steps, sums)));
    return p;
}

// Estimated times in microseconds, good for ranking plans: fitted to some 2,700
// timed launches of 107 shapes (1 to 8192 tokens, K of 256 to 16384, every tile,
// split and ring below) and 20 more with K from 64. The plans they pick are on
// average within 1% of the best of a shape.
//
// A streaming CTA takes 0.26 us for a K block of its own (0.23 with two to a
// stage) and an SM takes in 97 bytes/ns for all of its CTAs; sums leave at 20 ns a
// token, over a cluster with 1 us + 70 ns a rank for the exchange; each wave of
// CTAs after the first takes 0.8 us to start. Clusters of 4 and 8 do not find room
// on every SM.
double stream_time(const Plan& p, int64_t num_kb, int num_sms) {
    const double room = p.split == 8 ? 0.757 : p.split == 4 ? 0.892 : 1.0;
    const int64_t at_once = std::max<int64_t>(
        1, int64_t(stream_residents(p.bn, p.stages * p.sub) * room * num_sms));
    const int64_t waves = ceil_div(p.items, at_once);
    const int64_t per_sm = std::max(waves, ceil_div(p.items, num_sms));
    const double steps = double(ceil_div(num_kb, p.split));
    const double out = (p.split > 1 ? 1.0 + 0.07 * p.split : 0.25) + 0.02 * p.bn;
    const double feed = i8_stream_block_bytes(p.bn) / 97e3;
    const double step = p.sub == 2 ? 0.23 : 0.26;
    return 3.4 + waves * (0.8 + out) + steps * std::max(step * waves, feed * per_sm);
}

// A pair takes 0.35 to 0.38 us for a K block, little less for narrow tiles (5%
// more for strips, whose ring is no deeper than that of the tiles they are cut
// from), and 1.5 us + 5.5 ns a column to drain a tile into 16-bit C, 1.45 times
// that into 32-bit C. The drain of a tile overlaps the next one's K blocks.
double tile_time(const Plan& p, int64_t num_kb, int elem_size, int pairs) {
    double shorter = 0;
    auto round = [&](int width, double extra) {
        const double block = width == 256 ? 0.38 : width == 192 ? 0.36 : 0.35;
        const double blocks = block * num_kb * extra;
        const double drain = (1.5 + 0.0055 * width) * (elem_size == 4 ? 1.45 : 1.0);
        shorter = std::min(blocks, drain);
        return std::max(blocks, drain);
    };
    const int64_t rounds = p.cut > 1 ? p.whole / pairs : ceil_div(p.items, pairs);
    double t = 4.6 + rounds * round(p.bn, 1.0);
    if (p.cut > 1) t += round(p.bn / p.cut, 1.05);
    return t + shorter;
}

// The kernel and tile with the least estimated time. Sums are exact integers, so
// results do not depend on the choice.
Plan make_plan(int64_t M, int64_t N, int64_t K, int elem_size, int num_sms, int pairs) {
    const int64_t num_kb = ceil_div(K, kI8BK);
    Plan best{};
    double best_time = 0;
    auto offer = [&](const Plan& p, double t) {
        if (best.bn == 0 || t < best_time) {
            best = p;
            best_time = t;
        }
    };
    for (int bn : {256, 192, 128, 64}) {
        const Plan p = tile_plan(M, N, bn, pairs);
        offer(p, tile_time(p, num_kb, elem_size, pairs));
    }
    for (int bn : {64, 128, 256}) {
        if (ceil_div(M, bn) > 65535) continue;  // the grid's second dimension
        for (int split = 1; split <= 8 && split <= num_kb; split *= 2) {
            const Plan p = stream_plan(M, N, K, bn, split, num_sms);
            offer(p, stream_time(p, num_kb, num_sms));
        }
        if (M <= bn) break;  // one token tile already
    }
    return best;
}

// rows x cols bytes, pitch ld, read in boxes of box_rows x 128 bytes.
int operand_map(CUtensorMap* map, const void* ptr, int64_t rows, int64_t cols, int64_t ld,
                int box_rows) {
    auto enc = tensor_map_encode_fn();
    if (!enc) return RIDGE_ENOTSUP;
    cuuint64_t dims[2] = {cuuint64_t(cols), cuuint64_t(rows)};
    cuuint64_t strides[1] = {cuuint64_t(ld)};
    cuuint32_t box[2] = {cuuint32_t(kI8BK), cuuint32_t(box_rows)};
    cuuint32_t estr[2] = {1, 1};
    const CUresult r =
        enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box,
            estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? RIDGE_OK : RIDGE_EINVAL;
}

// C in boxes of 32 rows x 128 bytes.
int output_map(CUtensorMap* map, void* ptr, int32_t type, int64_t rows, int64_t cols, int64_t ld) {
    auto enc = tensor_map_encode_fn();
    if (!enc) return RIDGE_ENOTSUP;
    const int size = type == RIDGE_F32 ? 4 : 2;
    const CUtensorMapDataType dt = type == RIDGE_F16    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                   : type == RIDGE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                        : CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
    cuuint64_t dims[2] = {cuuint64_t(cols), cuuint64_t(rows)};
    cuuint64_t strides[1] = {cuuint64_t(ld) * size};
    cuuint32_t box[2] = {cuuint32_t(128 / size), 32};
    cuuint32_t estr[2] = {1, 1};
    const CUresult r = enc(map, dt, 2, ptr, dims, strides, box, estr,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                           CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? RIDGE_OK : RIDGE_EINVAL;
}

// Raises a kernel's shared-memory limit once per device.
int allow_smem(const void* func, std::atomic<bool>* done) {
    if (done->load(std::memory_order_acquire)) return RIDGE_OK;
    const cudaError_t e =
        cudaFuncSetAttribute(func, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxDynSmem);
    if (e != cudaSuccess) return int(e);
    done->store(true, std::memory_order_release);
    return RIDGE_OK;
}

void set_cluster(cudaLaunchConfig_t* cfg, cudaLaunchAttribute* attr, unsigned ctas) {
    attr->id = cudaLaunchAttributeClusterDimension;
    attr->val.clusterDim.x = ctas;
    attr->val.clusterDim.y = 1;
    attr->val.clusterDim.z = 1;
    cfg->attrs = attr;
    cfg->numAttrs = 1;
}

// Pairs of the tile kernel that run at once (for the full shared memory, one CTA
// per SM). The two CTAs of a pair sit on one TPC, so it is asked of the runtime.
template <typename T>
int resident_pairs(const DeviceInfo& dev, int* pairs) {
    static std::atomic<bool> ready[kMaxDevices];
    static std::atomic<int> known[kMaxDevices];  // 0 = not asked yet
    const void* func = reinterpret_cast<const void*>(&ridge_gemm_i8_tile<T>);
    const int st = allow_smem(func, &ready[dev.device]);
    if (st != RIDGE_OK) return st;
    *pairs = known[dev.device].load(std::memory_order_relaxed);
    if (*pairs > 0) return RIDGE_OK;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(4);
    cfg.blockDim = dim3(kI8TileThreads);
    cfg.dynamicSmemBytes = kMaxDynSmem;
    cudaLaunchAttribute attr[1];
    set_cluster(&cfg, attr, 2);
    if (cudaOccupancyMaxActiveClusters(pairs, func, &cfg) != cudaSuccess || *pairs <= 0) {
        cudaGetLastError();
        *pairs = std::max(1, dev.num_sms / 2);
    }
    known[dev.device].store(*pairs, std::memory_order_relaxed);
    return RIDGE_OK;
}

template <typename T, int SPLIT>
int launch_stream(const Plan& plan, const CUtensorMap& a, const CUtensorMap& b,
                  const I8Params& p, const DeviceInfo& dev, cudaStream_t stream) {
    static std::atomic<bool> ready[kMaxDevices];
    const int st = allow_smem(reinterpret_cast<const void*>(&ridge_gemm_i8_stream<T, SPLIT>),
                              &ready[dev.device]);
    if (st != RIDGE_OK) return st;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(ceil_div(p.N, 128) * SPLIT), unsigned(ceil_div(p.M, plan.bn)));
    if (cfg.gridDim.y > 65535) return RIDGE_EINVAL;
    cfg.blockDim = dim3(kI8StreamThreads);
    cfg.dynamicSmemBytes = size_t(i8_stream_smem(plan.bn, plan.stages * plan.sub));
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    if (SPLIT > 1) set_cluster(&cfg, attr, SPLIT);
    return int(cudaLaunchKernelEx(&cfg, ridge_gemm_i8_stream<T, SPLIT>, a, b, p));
}

// Products that go to ridge_gemm_i8_vec: one token while B is at most 64 MB, two
// tokens 16 MB, four 8 MB, the latter with at most 4096 channels. At the edges,
// against the streaming kernel: 1 x 8192 x 8192 13.6 us to 13.8, 1 x 14336 x 4096
// 13.2 to 12.3; 2 x 4096 x 4096 5.9 to 6.9, 2 x 8192 x 8192 14.6 to 13.9, 2 x 11008 x
// 512 4.3 to 3.8; 4 x 1024 x 4096 3.5 to 4.9, 4 x 4096 x 4096 7.8 to 7.0.
bool vec_serves(int64_t M, int64_t N, int64_t K) {
    const int64_t bytes = N * K;
    if (M == 1) return bytes <= int64_t(1) << 26;
    return N <= 4096 && ((M == 2 && bytes <= int64_t(1) << 24) ||
                         (M <= 4 && bytes <= int64_t(1) << 23));
}

// As many warps to a channel's K as keep all warps within 32 on every SM (8192
// channels 1, 4096 channels 2, whatever K), each with at least 1024 bytes of it.
template <typename T, int TOKENS>
int launch_vec(const int8_t* A, const int8_t* B, int64_t lda, int64_t ldb, const I8Params& p,
               const DeviceInfo& dev, cudaStream_t stream) {
    int ksplit = 1;
    while (ksplit < kI8VecWarps && p.K / (ksplit * 2) >= 1024 &&
           ceil_div(p.N, kI8VecRows) * ksplit * 2 <= int64_t(dev.num_sms) * 32)
        ksplit *= 2;
    const unsigned grid = unsigned(ceil_div(p.N, kI8VecRows * (kI8VecWarps / ksplit)));
    ridge_gemm_i8_vec<T, TOKENS><<<grid, kI8VecWarps * 32, 0, stream>>>(A, B, lda, ldb, ksplit, p);
    return int(cudaGetLastError());
}

template <typename T>
int launch_empty(const I8Params& p, cudaStream_t stream) {
    const dim3 grid(unsigned(ceil_div(p.N, 256)), unsigned(std::min(p.M, 65535)));
    ridge_gemm_i8_empty<T><<<grid, 256, 0, stream>>>(p);
    return int(cudaGetLastError());
}

template <typename T>
int run_product(const int8_t* A, const int8_t* B, int32_t type, int64_t lda, int64_t ldb,
                I8Params p, const DeviceInfo& dev, cudaStream_t stream) {
    if (vec_serves(p.M, p.N, p.K)) {
        if (p.M == 1) return launch_vec<T, 1>(A, B, lda, ldb, p, dev, stream);
        if (p.M == 2) return launch_vec<T, 2>(A, B, lda, ldb, p, dev, stream);
        return launch_vec<T, 4>(A, B, lda, ldb, p, dev, stream);
    }
    int pairs = 0;
    int st = resident_pairs<T>(dev, &pairs);
    if (st != RIDGE_OK) return st;
    const Plan plan = make_plan(p.M, p.N, p.K, int(sizeof(T)), dev.num_sms, pairs);
    p.bn = plan.bn;
    p.stages = plan.stages;
    p.sub = plan.sub;
    CUtensorMap a, b;
    st = operand_map(&a, A, p.M, p.K, lda, plan.stream ? plan.bn : 128);
    if (st != RIDGE_OK) return st;
    st = operand_map(&b, B, p.N, p.K, ldb, plan.stream ? 128 : plan.bn / 2);
    if (st != RIDGE_OK) return st;
    if (plan.stream) {
        p.vec_store = reinterpret_cast<uintptr_t>(p.C) % (4 * sizeof(T)) == 0 && p.ldc % 4 == 0;
        switch (plan.split) {
            case 1: return launch_stream<T, 1>(plan, a, b, p, dev, stream);
            case 2: return launch_stream<T, 2>(plan, a, b, p, dev, stream);
            case 4: return launch_stream<T, 4>(plan, a, b, p, dev, stream);
            default: return launch_stream<T, 8>(plan, a, b, p, dev, stream);
        }
    }
    if (plan.items > int64_t(1) << 30) return RIDGE_EINVAL;
    // Row tiles taken together: 16 share more of B in L2 while K is long (8192^3 328
    // us against 340 with 8), 8 write C in a better order while it is short
    // (8192 x 8192 x 512 50 us against 54.6).
    p.groupM = p.K >= 4096 ? 16 : 8;
    p.whole = int(plan.whole);
    p.cut = plan.cut;
    CUtensorMap strip = b, c;
    if (plan.cut > 1) {
        st = operand_map(&strip, B, p.N, p.K, ldb, plan.bn / plan.cut / 2);
        if (st != RIDGE_OK) return st;
    }
    // Stores through the tensor map need 16-byte aligned rows of C.
    std::memset(&c, 0, sizeof(c));
    p.tma_store = (reinterpret_cast<uintptr_t>(p.C) & 15) == 0 && (p.ldc * sizeof(T)) % 16 == 0;
    if (p.tma_store) {
        st = output_map(&c, p.C, type, p.M, p.N, p.ldc);
        if (st != RIDGE_OK) return st;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(std::min<int64_t>(plan.items, pairs)) * 2);
    cfg.blockDim = dim3(kI8TileThreads);
    cfg.dynamicSmemBytes = size_t(i8_tile_smem(plan.bn, plan.stages));
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    set_cluster(&cfg, attr, 2);
    return int(cudaLaunchKernelEx(&cfg, ridge_gemm_i8_tile<T>, a, b, strip, c, p));
}

}  // namespace
}  // namespace ridge_b200

using namespace ridge_b200;

extern "C" int ridge_gemm_i8(const int8_t* A, const float* scale_a, const int8_t* B,
                             const float* scale_b, const void* bias, int32_t type, void* C,
                             int64_t M, int64_t N, int64_t K, int64_t lda, int64_t ldb,
                             int64_t ldc, void* stream_v) {
    const int size = type_size(type);
    const int64_t kExtent = int64_t(1) << 30;  // a tile past the last row still has 32-bit indices
    if (size == 0 || M < 0 || N < 0 || K < 0 || M > kExtent || N > kExtent) return RIDGE_EINVAL;
    if (K >= int64_t(1) << 17) return RIDGE_EINVAL;  // 2^17 products of 2^14 could overflow
    // One row has no pitch of its own: any that the tensor map takes will do.
    const int64_t whole = (std::max<int64_t>(K, 1) + 15) / 16 * 16;
    if (M <= 1 || K == 0) lda = whole;
    if (N <= 1 || K == 0) ldb = whole;
    if (M <= 1) ldc = (N * size + 15) / 16 * 16 / size;
    const int64_t kPitch = int64_t(1) << 40;  // the tensor map's limit on a stride, in bytes
    if (lda % 16 != 0 || ldb % 16 != 0 || lda >= kPitch || ldb >= kPitch || ldc >= kPitch / size)
        return RIDGE_EINVAL;
    if (M == 0 || N == 0) return RIDGE_OK;
    if (!array_ok(A, M, K, lda, 16) || !array_ok(B, N, K, ldb, 16) ||
        !array_ok(C, M, N, ldc, size) || !array_ok(scale_a, 1, M, M, 4) ||
        !array_ok(scale_b, 1, N, N, 4) || (bias && !array_ok(bias, 1, N, N, size)))
        return RIDGE_EINVAL;
    const RowArray c = {C, M, ldc * size, N * size};
    if (overlaps(c, {A, M, lda, K}) || overlaps(c, {B, N, ldb, K}) ||
        overlaps(c, {scale_a, 1, M * 4, M * 4}) || overlaps(c, {scale_b, 1, N * 4, N * 4}) ||
        overlaps(c, {bias, 1, N * size, N * size}))
        return RIDGE_EINVAL;
    DeviceInfo dev;
    int st = device_info(&dev);
    if (st != RIDGE_OK) return st;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_v);

    I8Params p{};
    p.sa = scale_a;
    p.sb = scale_b;
    p.bias = bias;
    p.C = C;
    p.M = int(M);
    p.N = int(N);
    p.K = int(K);
    p.ldc = ldc;
    p.err = dev.err_word;
    if (K == 0)
        return type == RIDGE_F16    ? launch_empty<__half>(p, stream)
               : type == RIDGE_BF16 ? launch_empty<__nv_bfloat16>(p, stream)
                                    : launch_empty<float>(p, stream);

    if (type == RIDGE_F16) return run_product<__half>(A, B, type, lda, ldb, p, dev, stream);
    if (type == RIDGE_BF16)
        return run_product<__nv_bfloat16>(A, B, type, lda, ldb, p, dev, stream);
    return run_product<float>(A, B, type, lda, ldb, p, dev, stream);
}
