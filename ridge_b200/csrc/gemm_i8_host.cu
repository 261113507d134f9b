// C-ABI front end of the 8-bit GEMM (gemm_i8_sm100.cuh, include/ridge_b200.h):
// argument checks, tensor maps, and the choice of kernel and tile.

#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdlib>
#include <cstdio>
#include <cstring>

#include "../../include/ridge_b200.h"
#include "device_info.h"
#include "gemm_i8_sm100.cuh"
#include "row_arrays.h"

namespace ridge_b200 {
namespace {

constexpr int kMaxDevices = 64;
constexpr int kMaxDynSmem = 232448;  // 227 KB opt-in limit per CTA on sm_100

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
    int bn, stages, split;
};

int ceil_div(int64_t a, int64_t b) { return int((a + b - 1) / b); }

int stages_for(int stage_bytes, int fixed, int budget) {
    return std::min(kI8MaxStages, (budget - fixed) / stage_bytes);
}

Plan make_plan(int64_t M, int64_t N, int64_t K, int num_sms) {
    Plan p{};
    const int num_kb = ceil_div(K, kI8BK);
#ifdef RIDGE_I8_PROBE
    if (const char* v = std::getenv("RIDGE_I8_PLAN")) {
        int s = 0;
        std::sscanf(v, "%d,%d,%d,%d", &s, &p.bn, &p.stages, &p.split);
        p.stream = s != 0;
        if (p.stream) p.bn = std::min(p.bn, ceil_div(M, 16) * 16);
        return p;
    }
#endif
    if (M <= 256) {
        p.stream = true;
        p.bn = ceil_div(M, 16) * 16;
        const int tiles = ceil_div(N, 128);
        p.split = 1;
        while (p.split < 8 && tiles * p.split * 2 <= num_sms && num_kb >= p.split * 2 * 4)
            p.split *= 2;
        p.stages = stages_for(i8_stream_stage_bytes(p.bn), i8_stream_smem(0, 0), kMaxDynSmem);
        return p;
    }
    p.stream = false;
    p.bn = 256;
    p.stages = stages_for(i8_tile_stage_bytes(p.bn), i8_tile_smem(p.bn, 0), kMaxDynSmem);
    p.split = 1;
    return p;
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

template <typename T>
int launch_tile(const Plan& plan, const CUtensorMap& a, const CUtensorMap& b,
                const CUtensorMap& c, const I8Params& p, const DeviceInfo& dev,
                cudaStream_t stream) {
    static std::atomic<bool> ready[kMaxDevices];
    static std::atomic<int> pairs[kMaxDevices];  // 0 = not asked yet
    const void* func = reinterpret_cast<const void*>(&ridge_gemm_i8_tile<T>);
    const int st = allow_smem(func, &ready[dev.device]);
    if (st != RIDGE_OK) return st;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(kI8TileThreads);
    cfg.dynamicSmemBytes = size_t(i8_tile_smem(plan.bn, plan.stages));
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    set_cluster(&cfg, attr, 2);
    // The two CTAs of a pair sit on one TPC, so how many pairs run at once is
    // asked of the runtime (for the full shared memory: one CTA per SM).
    int units = pairs[dev.device].load(std::memory_order_relaxed);
    if (units == 0) {
        cudaLaunchConfig_t q = cfg;
        q.gridDim = dim3(4);
        q.dynamicSmemBytes = kMaxDynSmem;
        if (cudaOccupancyMaxActiveClusters(&units, func, &q) != cudaSuccess || units <= 0) {
            cudaGetLastError();
            units = dev.num_sms / 2;
        }
        pairs[dev.device].store(units, std::memory_order_relaxed);
    }
    const int64_t tiles = int64_t(ceil_div(p.M, 256)) * ceil_div(p.N, plan.bn);
    if (tiles > int64_t(1) << 30) return RIDGE_EINVAL;
    cfg.gridDim = dim3(unsigned(std::min<int64_t>(tiles, units)) * 2);
    return int(cudaLaunchKernelEx(&cfg, ridge_gemm_i8_tile<T>, a, b, c, p));
}

template <typename T, int SPLIT>
int launch_stream_n(const Plan& plan, const CUtensorMap& a, const CUtensorMap& b,
                    const I8Params& p, const DeviceInfo& dev, cudaStream_t stream) {
    static std::atomic<bool> ready[kMaxDevices];
    const int st = allow_smem(reinterpret_cast<const void*>(&ridge_gemm_i8_stream<T, SPLIT>),
                              &ready[dev.device]);
    if (st != RIDGE_OK) return st;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(ceil_div(p.N, 128)) * SPLIT, unsigned(ceil_div(p.M, plan.bn)));
    if (cfg.gridDim.y > 65535) return RIDGE_EINVAL;
    cfg.blockDim = dim3(kI8StreamThreads);
    cfg.dynamicSmemBytes = size_t(i8_stream_smem(plan.bn, plan.stages));
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    if (SPLIT > 1) set_cluster(&cfg, attr, SPLIT);
    return int(cudaLaunchKernelEx(&cfg, ridge_gemm_i8_stream<T, SPLIT>, a, b, p));
}

template <typename T>
int launch_typed(const Plan& plan, const CUtensorMap& a, const CUtensorMap& b,
                 const CUtensorMap& c, const I8Params& p, const DeviceInfo& dev,
                 cudaStream_t stream) {
    if (!plan.stream) return launch_tile<T>(plan, a, b, c, p, dev, stream);
    switch (plan.split) {
        case 1: return launch_stream_n<T, 1>(plan, a, b, p, dev, stream);
        case 2: return launch_stream_n<T, 2>(plan, a, b, p, dev, stream);
        case 4: return launch_stream_n<T, 4>(plan, a, b, p, dev, stream);
        default: return launch_stream_n<T, 8>(plan, a, b, p, dev, stream);
    }
}

template <typename T>
int launch_empty(const I8Params& p, cudaStream_t stream) {
    const dim3 grid(unsigned(ceil_div(p.N, 256)), unsigned(std::min(p.M, 65535)));
    ridge_gemm_i8_empty<T><<<grid, 256, 0, stream>>>(p);
    return int(cudaGetLastError());
}

}  // namespace
}  // namespace ridge_b200

using namespace ridge_b200;

extern "C" int ridge_gemm_i8(const int8_t* A, const float* scale_a, const int8_t* B,
                             const float* scale_b, const void* bias, int32_t type, void* C,
                             int64_t M, int64_t N, int64_t K, int64_t lda, int64_t ldb,
                             int64_t ldc, void* stream_v) {
    const int size = type_size(type);
    const int64_t kExtent = int64_t(1) << 31;
    if (size == 0 || M < 0 || N < 0 || K < 0 || M >= kExtent || N >= kExtent) return RIDGE_EINVAL;
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

    const Plan plan = make_plan(M, N, K, dev.num_sms);
    p.bn = plan.bn;
    p.stages = plan.stages;
    p.groupM = 8;
    p.vec_store = reinterpret_cast<uintptr_t>(C) % uintptr_t(4 * size) == 0 && ldc % 4 == 0;
    // Stores through the tensor map need 16-byte aligned rows of C.
    p.tma_store = (reinterpret_cast<uintptr_t>(C) & 15) == 0 && (ldc * size) % 16 == 0;
    CUtensorMap tmap_a, tmap_b, tmap_c;
    std::memset(&tmap_c, 0, sizeof(tmap_c));
    st = operand_map(&tmap_a, A, M, K, lda, plan.stream ? plan.bn : 128);
    if (st != RIDGE_OK) return st;
    st = operand_map(&tmap_b, B, N, K, ldb, plan.stream ? 128 : plan.bn / 2);
    if (st != RIDGE_OK) return st;
    if (!plan.stream && p.tma_store) {
        st = output_map(&tmap_c, C, type, M, N, ldc);
        if (st != RIDGE_OK) return st;
    }
    if (type == RIDGE_F16)
        return launch_typed<__half>(plan, tmap_a, tmap_b, tmap_c, p, dev, stream);
    if (type == RIDGE_BF16)
        return launch_typed<__nv_bfloat16>(plan, tmap_a, tmap_b, tmap_c, p, dev, stream);
    return launch_typed<float>(plan, tmap_a, tmap_b, tmap_c, p, dev, stream);
}
