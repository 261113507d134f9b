// C-ABI front end of the row operators (quant_i8.cuh) and the kernel that turns
// 8-bit rows and their scales back into values (include/ridge_b200.h).

#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "../../include/ridge_b200.h"
#include "device_info.h"
#include "quant_i8.cuh"
#include "row_arrays.h"

namespace ridge_b200 {
namespace {

bool extents_ok(int64_t M, int64_t D) {
    return M >= 0 && D >= 0 && M < (int64_t(1) << 31) && D < (int64_t(1) << 31);
}

int run(int op, int32_t type, RowParams p, int64_t M, int64_t D, void* stream_v) {
    const int size = type_size(type);
    if (size == 0 || !extents_ok(M, D)) return RIDGE_EINVAL;
    const bool has_r = op == kNormAdd || op == kSiluMul;
    const bool has_w = op == kNorm || op == kNormAdd;
    if (M == 0) return RIDGE_OK;
    if (!array_ok(p.x, M, D, p.ldx, size) || !array_ok(p.q, M, D, p.ldq, 1) ||
        !array_ok(p.scale, M, 1, 1, 4))
        return RIDGE_EINVAL;
    if (has_r && !array_ok(p.r, M, D, p.ldr, size)) return RIDGE_EINVAL;
    if (has_w && !array_ok(p.w, 1, D, D, size)) return RIDGE_EINVAL;
    if (op == kNormAdd && !array_ok(p.h, M, D, p.ldh, size)) return RIDGE_EINVAL;
    if (M == 1) p.ldx = p.ldr = p.ldh = p.ldq = D;
    // Outputs against inputs and against one another. h may be x or r itself.
    const RowArray in[3] = {{p.x, M, p.ldx * size, D * size},
                            {has_r ? p.r : nullptr, M, p.ldr * size, D * size},
                            {has_w ? p.w : nullptr, 1, D * size, D * size}};
    const RowArray q = {p.q, M, p.ldq, D}, sc = {p.scale, 1, M * 4, M * 4};
    const RowArray h = {op == kNormAdd ? p.h : nullptr, M, p.ldh * size, D * size};
    for (const RowArray& a : in) {
        if (overlaps(q, a) || overlaps(sc, a)) return RIDGE_EINVAL;
        if (overlaps(h, a) && !(a.p == h.p && a.pitch == h.pitch && a.rows == h.rows))
            return RIDGE_EINVAL;
    }
    if (overlaps(q, h) || overlaps(sc, h) || overlaps(q, sc)) return RIDGE_EINVAL;
    DeviceInfo dev;
    const int st = device_info(&dev);
    if (st != RIDGE_OK) return st;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
    if (D == 0) return int(cudaMemsetAsync(p.scale, 0, size_t(M) * 4, stream));
    p.M = int(M);
    p.D = int(D);
    cudaError_t e;
    if (type == RIDGE_F16) e = run_rows_f16(op, p, dev.num_sms, stream);
    else if (type == RIDGE_BF16) e = run_rows_bf16(op, p, dev.num_sms, stream);
    else e = run_rows_f32(op, p, dev.num_sms, stream);
    return int(e);
}

// Values of 8-bit rows: out = scale[row] * q, one rounding to T. A thread takes
// 16 values (one 16-byte load, 32 or 64 bytes of stores) at a time; blockDim.x
// threads walk a row and blockDim.y rows share a CTA, so short rows fill one. The
// last rows go first: behind a quantising kernel they are the ones still in L2
// (14336 x 4096 BF16, both ways 63.8 -> 62.6 us). 8192 x 8192 to BF16 33 us, 6.1 TB/s.
template <typename T>
__global__ void __launch_bounds__(256)
    ridge_dequantize_i8(const int8_t* __restrict__ q, const float* __restrict__ scale,
                        T* __restrict__ out, int M, int D, int64_t ldq, int64_t ldo) {
    const int64_t row = int64_t(M) - 1 - (int64_t(blockIdx.x) * blockDim.y + threadIdx.y);
    if (row < 0) return;
    const float s = scale[row];
    const int8_t* src = q + row * ldq;
    T* dst = out + row * ldo;
    const int64_t first = (int64_t(blockIdx.y) * blockDim.x + threadIdx.x) * 16;
    const int64_t step = int64_t(gridDim.y) * blockDim.x * 16;
    for (int64_t e = first; e < D; e += step) {
        const Chunk<int8_t, 16> in = *reinterpret_cast<const Chunk<int8_t, 16>*>(src + e);
        constexpr int V = kVecOf<T>;
#pragma unroll
        for (int g = 0; g < 16 / V; ++g) {
            float f[V];
#pragma unroll
            for (int i = 0; i < V; ++i) f[i] = float(in.raw[g * V + i]) * s;
            Chunk<T, V> o;
            o.set(f);
            *reinterpret_cast<Chunk<T, V>*>(dst + e + g * V) = o;
        }
    }
}

// V bytes from anywhere in a row of D: two aligned words and a shift where both lie
// inside the row, single bytes at its ends (zeros outside it).
template <int V>
__device__ __forceinline__ Chunk<int8_t, V> load_bytes(const int8_t* row, int64_t e, int64_t D) {
    static_assert(V == 4 || V == 8, "one word");
    using Word = typename std::conditional<V == 8, uint64_t, uint32_t>::type;
    Chunk<int8_t, V> c{};
    const int8_t* at = row + e;
    const int s = int(reinterpret_cast<uintptr_t>(at) % V);
    if (e >= s && e - s + 2 * V <= D) {
        const Word* word = reinterpret_cast<const Word*>(at - s);
        Word w = word[0];
        if (s) w = (w >> (8 * s)) | (word[1] << (8 * (V - s)));
        *reinterpret_cast<Word*>(&c) = w;
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (e + i >= 0 && e + i < D) c.raw[i] = at[i];
    }
    return c;
}

// The same for rows that start anywhere: windows of VEC values between two 16-byte
// boundaries of `out`, one store each; elements one by one at a row's ends.
template <typename T>
__global__ void __launch_bounds__(256)
    ridge_dequantize_i8_odd(const int8_t* __restrict__ q, const float* __restrict__ scale,
                            T* __restrict__ out, int M, int D, int64_t ldq, int64_t ldo) {
    constexpr int V = kVecOf<T>;
    const int64_t row = int64_t(M) - 1 - (int64_t(blockIdx.x) * blockDim.y + threadIdx.y);
    if (row < 0) return;
    const float s = scale[row];
    const int8_t* src = q + row * ldq;
    T* dst = out + row * ldo;
    // The first window holds the elements before the row's first boundary.
    const int before = int(reinterpret_cast<uintptr_t>(dst) & 15u) / int(sizeof(T));
    const int64_t first = (int64_t(blockIdx.y) * blockDim.x + threadIdx.x) * V - before;
    const int64_t step = int64_t(gridDim.y) * blockDim.x * V;
    for (int64_t e = first; e < D; e += step) {
        const Chunk<int8_t, V> in = load_bytes<V>(src, e, D);
        float f[V];
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = float(in.raw[i]) * s;
        if (e >= 0 && e + V <= D) {
            Chunk<T, V> o;
            o.set(f);
            *reinterpret_cast<Chunk<T, V>*>(dst + e) = o;
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (e + i >= 0 && e + i < D) dst[e + i] = from_f32<T>(f[i]);
        }
    }
}

template <typename T>
cudaError_t run_dequantize(const int8_t* q, const float* scale, void* out_v, int M, int D,
                           int64_t ldq, int64_t ldo, int num_sms, cudaStream_t stream) {
    T* out = static_cast<T*>(out_v);
    // 32-bit values leave lane by lane in the windows' way too: 16 of them to a thread
    // would be 64 bytes from the next thread's (8192 x 8192 74 us, against 68).
    const bool vec = sizeof(T) == 2 && D % 16 == 0 && ldq % 16 == 0 && (ldo * int64_t(sizeof(T))) % 16 == 0 &&
                     reinterpret_cast<uintptr_t>(q) % 16 == 0 &&
                     reinterpret_cast<uintptr_t>(out) % 16 == 0;
    constexpr int V = kVecOf<T>;
    const int64_t per_row = vec ? D / 16 : int64_t(D) / V + 2;  // windows: one more at each end
    int tx = 32;
    while (tx < 256 && tx < per_row) tx *= 2;
    const int ty = 256 / tx;
    const int64_t row_ctas = (int64_t(M) + ty - 1) / ty;
    // With fewer rows than would fill the GPU a row is split over several CTAs.
    const int64_t want = std::max<int64_t>(1, int64_t(num_sms) * 8 / row_ctas);
    const int64_t most = (per_row + tx - 1) / tx;
    const dim3 grid(unsigned(row_ctas), unsigned(std::min<int64_t>({want, most, 65535})));
    const dim3 block(static_cast<unsigned>(tx), static_cast<unsigned>(ty));
    if (vec)
        ridge_dequantize_i8<T><<<grid, block, 0, stream>>>(q, scale, out, M, D, ldq, ldo);
    else
        ridge_dequantize_i8_odd<T><<<grid, block, 0, stream>>>(q, scale, out, M, D, ldq, ldo);
    return cudaGetLastError();
}

}  // namespace
}  // namespace ridge_b200

using namespace ridge_b200;

extern "C" {

int ridge_quantize_i8(const void* x, int32_t type, int8_t* q, float* scale, int64_t M, int64_t D,
                      int64_t ldx, int64_t ldq, void* stream) {
    RowParams p{};
    p.x = x;
    p.q = q;
    p.scale = scale;
    p.ldx = ldx;
    p.ldq = ldq;
    return run(kQuant, type, p, M, D, stream);
}

int ridge_rms_norm_i8(const void* x, const void* residual, const void* weight, int32_t type,
                      void* residual_out, int8_t* q, float* scale, int64_t M, int64_t D,
                      int64_t ldx, int64_t ldr, int64_t ldro, int64_t ldq, float eps,
                      void* stream) {
    if (!(eps > 0.0f) || !std::isfinite(eps)) return RIDGE_EINVAL;
    if ((residual == nullptr) != (residual_out == nullptr) && M > 0 && D > 0) return RIDGE_EINVAL;
    RowParams p{};
    p.x = x;
    p.r = residual;
    p.w = weight;
    p.h = residual_out;
    p.q = q;
    p.scale = scale;
    p.ldx = ldx;
    p.ldr = ldr;
    p.ldh = ldro;
    p.ldq = ldq;
    p.eps = eps;
    return run(residual ? kNormAdd : kNorm, type, p, M, D, stream);
}

int ridge_silu_mul_i8(const void* gate, const void* up, int32_t type, int8_t* q, float* scale,
                      int64_t M, int64_t D, int64_t ldg, int64_t ldu, int64_t ldq, void* stream) {
    RowParams p{};
    p.x = gate;
    p.r = up;
    p.q = q;
    p.scale = scale;
    p.ldx = ldg;
    p.ldr = ldu;
    p.ldq = ldq;
    return run(kSiluMul, type, p, M, D, stream);
}

int ridge_dequantize_i8(const int8_t* q, const float* scale, int32_t type, void* out, int64_t M,
                        int64_t D, int64_t ldq, int64_t ldo, void* stream_v) {
    const int size = type_size(type);
    if (size == 0 || !extents_ok(M, D)) return RIDGE_EINVAL;
    if (M == 0 || D == 0) return RIDGE_OK;
    if (!array_ok(q, M, D, ldq, 1) || !array_ok(scale, M, 1, 1, 4) ||
        !array_ok(out, M, D, ldo, size))
        return RIDGE_EINVAL;
    if (M == 1) ldq = ldo = D;
    const RowArray o = {out, M, ldo * size, D * size};
    if (overlaps(o, {q, M, ldq, D}) || overlaps(o, {scale, 1, M * 4, M * 4})) return RIDGE_EINVAL;
    DeviceInfo dev;
    const int st = device_info(&dev);
    if (st != RIDGE_OK) return st;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
    cudaError_t e;
    if (type == RIDGE_F16)
        e = run_dequantize<__half>(q, scale, out, int(M), int(D), ldq, ldo, dev.num_sms, stream);
    else if (type == RIDGE_BF16)
        e = run_dequantize<__nv_bfloat16>(q, scale, out, int(M), int(D), ldq, ldo, dev.num_sms,
                                          stream);
    else
        e = run_dequantize<float>(q, scale, out, int(M), int(D), ldq, ldo, dev.num_sms, stream);
    return int(e);
}

}  // extern "C"
