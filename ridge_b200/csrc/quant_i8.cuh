// Row operators that write 8-bit GEMM operands: each row of y becomes signed
// 8-bit values q in -127..127 and one FP32 scale, y ~ scale * q, with
//
//   scale = max_j |y_j| / 127,   q_j = round_to_even(y_j / scale).
//
//   kQuant    y = x
//   kNorm     y = w h / sqrt(mean(h^2) + eps),  h = x
//   kNormAdd  the same with h = x + r, h also stored (rounded once, to the type of x;
//             the norm reads the FP32 sum, not the rounded one)
//   kSiluMul  y = x r / (1 + exp(-x))          (r is the up projection)
//
// One pass over the data: a row sits in the registers of the threads that read
// it. The norm needs two sums over a row, of h^2 and the maximum of |y|, but
// its factor 1 / sqrt(mean + eps) is the same for the whole row, so with
// v = w h both are taken in one reduction:
//
//   scale = max|v| rstd / 127,   q_j = round(v_j * (127 / max|v|)),
//
// and rstd never touches the elements. The other operators have v = y, rstd = 1.
//
// Bound by memory: 8192 x 8192 BF16 with a residual (read 2, write 1 and the 8-bit
// rows) 72 us, 6.5 TB/s; gate and up of 4096 x 14336 FP16 52 us, 5.7 TB/s;
// quantising 14336 x 4096 BF16 30 us, 5.8 TB/s; one row of 4096 2 us, a launch.
// Rows that start anywhere take 1.6 to 2 times as long (below).
//
// Numerics: everything between load and store is FP32. q_j is v_j * inv + 1.5 * 2^23
// in one fused multiply-add: the sum's unit is 1, so the add rounds the exact
// product to the nearest whole number (ties to even) and the low byte of its
// bits is q_j. inv = 127 / max|v| is rounded once, so a v_j within 2^-24 relative
// of a rounding border may go to the other side; |q_j| <= 127 always. Rows whose
// maximum is below 2^-100 are first scaled by 2^64 so that inv cannot overflow.
// A row of zeros has scale 0. A row holding an infinity or a NaN has an
// infinite or NaN scale and q = 0, so that whatever is computed from it is NaN
// and other rows are untouched.

#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

namespace ridge_b200 {

enum RowOp { kQuant = 0, kNorm = 1, kNormAdd = 2, kSiluMul = 3 };

struct RowParams {
    const void* x;
    const void* r;  // kNormAdd: residual; kSiluMul: up projection
    const void* w;  // kNorm, kNormAdd: gain
    void* h;        // kNormAdd: x + r
    int8_t* q;
    float* scale;
    int64_t ldx, ldr, ldh, ldq;  // row pitches in elements
    int M, D;
    float eps;
};

// Elements of one 16-byte load.
template <typename T>
constexpr int kVecOf = 16 / int(sizeof(T));

// One element, or the two 16-bit elements of a 32-bit word.
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// VEC elements as they lie in memory: one 16-byte load, or a single element
// where the row's start or length is no multiple of 16 bytes.
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Chunk {
    static constexpr bool kPairs = sizeof(T) == 2 && VEC > 1;
    using Raw = typename std::conditional<kPairs, uint32_t, T>::type;
    static constexpr int kRaw = kPairs ? VEC / 2 : VEC;
    Raw raw[kRaw];

    __device__ __forceinline__ void get(float (&f)[VEC]) const {
#pragma unroll
        for (int i = 0; i < kRaw; ++i) {
            if constexpr (kPairs) {
                const float2 v = unpack2<T>(raw[i]);
                f[2 * i] = v.x;
                f[2 * i + 1] = v.y;
            } else {
                f[i] = to_f32(raw[i]);
            }
        }
    }
    __device__ __forceinline__ void set(const float (&f)[VEC]) {
#pragma unroll
        for (int i = 0; i < kRaw; ++i) {
            if constexpr (kPairs)
                raw[i] = pack2<T>(f[2 * i], f[2 * i + 1]);
            else
                raw[i] = from_f32<T>(f[i]);
        }
    }
};

// Low bytes of the rounded sums v * inv + 1.5 * 2^23, four to a word.
__device__ __forceinline__ uint32_t round_bits(float v, float inv) {
    return __float_as_uint(fmaf(v, inv, 12582912.0f));
}

template <int VEC>
__device__ __forceinline__ void store_q(int8_t* dst, const float (&v)[VEC], float inv, bool zero) {
    if constexpr (VEC == 1) {
        const uint32_t b = round_bits(v[0], inv);
        *dst = zero ? int8_t(0) : int8_t(b & 0xffu);
    } else {
        uint32_t word[VEC / 4];
#pragma unroll
        for (int i = 0; i < VEC / 4; ++i) {
            const uint32_t lo = __byte_perm(round_bits(v[4 * i], inv),
                                            round_bits(v[4 * i + 1], inv), 0x0040);
            const uint32_t hi = __byte_perm(round_bits(v[4 * i + 2], inv),
                                            round_bits(v[4 * i + 3], inv), 0x0040);
            word[i] = zero ? 0u : __byte_perm(lo, hi, 0x5410);
        }
        if constexpr (VEC == 8)
            *reinterpret_cast<uint2*>(dst) = make_uint2(word[0], word[1]);
        else
            *reinterpret_cast<uint32_t*>(dst) = word[0];
    }
}

// max(|a|, |b|, |c|), NaN if any is.
__device__ __forceinline__ float max_abs(float a, float b, float c) {
    float m;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
    return m;
}

// x / (1 + e^-x), with one ex2 and one reciprocal of the hardware's (each within
// 2^-22.5 relative; the exponent's rounding adds |x| 2^-23.4 to e^-x, which reaches
// the result times e^-x / (1 + e^-x)). Where 1 + e^-x passes 2^126 the reciprocal
// and the result, under 1e-36, are flushed to 0; x = -inf gives NaN, as the formula
// does.
__device__ __forceinline__ float silu(float x) {
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x * -1.4426950408889634f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    return x * r;
}

// v and, for kNormAdd, the stored sum of one chunk; adds to the row's sum of
// squares and raises the row's maximum of |v|, which keeps a NaN.
template <typename T, int OP, int VEC>
__device__ __forceinline__ void take_chunk(const Chunk<T, VEC>& x, const Chunk<T, VEC>& r,
                                           const Chunk<T, VEC>& w, Chunk<T, VEC>& h,
                                           float (&v)[VEC], float& sumsq, float& top) {
    float other[VEC];
    x.get(v);
    if constexpr (OP == kNormAdd) {
        r.get(other);
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] += other[i];
        h.set(v);
    }
    if constexpr (OP == kNorm || OP == kNormAdd) {
        w.get(other);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            sumsq = fmaf(v[i], v[i], sumsq);
            v[i] *= other[i];
        }
    }
    if constexpr (OP == kSiluMul) {
        r.get(other);
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = silu(v[i]) * other[i];
    }
    if constexpr (VEC == 1) {
        top = max_abs(top, v[0], v[0]);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; i += 2) top = max_abs(top, v[i], v[i + 1]);
    }
}

// What a row's two reductions make of its elements.
struct RowScale {
    float scale, pre, inv;
    bool zero;
};

template <int OP>
__device__ __forceinline__ RowScale row_scale(float sumsq, float amax, int D, float eps) {
    float rstd = 1.0f;
    if constexpr (OP == kNorm || OP == kNormAdd) rstd = 1.0f / sqrtf(sumsq / float(D) + eps);
    RowScale s;
    s.scale = amax == 0.0f ? 0.0f : amax * rstd / 127.0f;
    s.zero = !(s.scale > 0.0f && s.scale < __uint_as_float(0x7f800000u));
    s.pre = amax < 7.8886091e-31f ? 18446744073709551616.0f : 1.0f;  // 2^-100, 2^64
    s.inv = 127.0f / (amax * s.pre);
    return s;
}

// A row so small that 127 / max would overflow is scaled up first.
template <int N>
__device__ __forceinline__ void prescale(const RowScale& s, float (&v)[N]) {
    if (s.pre != 1.0f) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] *= s.pre;
    }
}

// Sum and maximum over the G warps of a row (one warp: shuffles alone). Every
// thread gets both; the order of the sum is fixed.
__device__ __forceinline__ void reduce_row(float& sumsq, float& amax, bool with_sum) {
    __shared__ float s_sum[32];
    __shared__ uint32_t s_top[32];
    if (with_sum) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sumsq += __shfl_xor_sync(0xffffffffu, sumsq, o);
    }
    // |v| as bits: unsigned order is that of the values, every NaN above infinity.
    uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(amax) & 0x7fffffffu);
    amax = __uint_as_float(top);
    const int G = blockDim.x >> 5;
    if (G == 1) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) {
        s_sum[warp] = sumsq;
        s_top[warp] = top;
    }
    __syncthreads();
    top = __reduce_max_sync(0xffffffffu, lane < G ? s_top[lane] : 0u);
    amax = __uint_as_float(top);
    if (with_sum) {
        sumsq = lane < G ? s_sum[lane] : 0.0f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sumsq += __shfl_xor_sync(0xffffffffu, sumsq, o);
    }
}

// A chunk that is read once and is large beside the 8-bit rows: it leaves L2 first,
// so that more of q is still there for what reads it next (with a dequantise behind
// it, quantising 14336 x 4096 65.2 -> 63.8 us, the gate of 4096 x 14336 90.2 -> 88.1).
// Not where x + r is written too: that norm alone took 74.4 us for 72.1.
template <typename C>
__device__ __forceinline__ C load_once(const void* at) {
    static_assert(sizeof(C) == 16, "one 16-byte load");
    C c;
    *reinterpret_cast<uint4*>(&c) = __ldcs(static_cast<const uint4*>(at));
    return c;
}

// One row per blockDim.x threads (a multiple of 32), blockDim.y rows per CTA
// (more than one only for single-warp rows, which need no barrier). CH chunks
// of VEC elements per thread.
template <typename T, int OP, int VEC, int CH, int MAXT>
__global__ void __launch_bounds__(MAXT, 1024 / MAXT) ridge_row_i8(const RowParams p) {
    constexpr bool kR = OP == kNormAdd || OP == kSiluMul;
    constexpr bool kW = OP == kNorm || OP == kNormAdd;
    const int64_t row = int64_t(blockIdx.x) * blockDim.y + threadIdx.y;
    if (row >= p.M) return;
    const T* x = static_cast<const T*>(p.x) + row * p.ldx;
    const T* r = static_cast<const T*>(p.r) + (kR ? row * p.ldr : 0);
    const T* w = static_cast<const T*>(p.w);
    using C = Chunk<T, VEC>;
    // Every load of the row is issued before the first value is used. The gain
    // is among them where it is cheap. With four 16-byte chunks a thread it is not:
    // its registers (112 against 64 a thread) would halve the rows in flight on an
    // SM, and all rows share it, so it comes from L1 or L2 when it is needed
    // (8192 x 8192 BF16 with a residual: 136 us with it early, 78 without).
    constexpr bool kEarlyW = kW && CH <= 2;
    C cx[CH], cr[kR ? CH : 1], cw[kEarlyW ? CH : 1];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int e = (c * int(blockDim.x) + int(threadIdx.x)) * VEC;
        if (e < p.D) {
            if constexpr (OP == kNormAdd) {
                cx[c] = *reinterpret_cast<const C*>(x + e);
                cr[c] = *reinterpret_cast<const C*>(r + e);
            } else {
                cx[c] = load_once<C>(x + e);
                if constexpr (kR) cr[c] = load_once<C>(r + e);
            }
            if constexpr (kEarlyW) cw[c] = *reinterpret_cast<const C*>(w + e);
        }
    }
    float v[CH][VEC];
    float sumsq = 0.0f;
    float top = 0.0f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int e = (c * int(blockDim.x) + int(threadIdx.x)) * VEC;
        if (e < p.D) {
            C h, gain = cw[kEarlyW ? c : 0];
            if constexpr (kW && !kEarlyW) gain = *reinterpret_cast<const C*>(w + e);
            take_chunk<T, OP, VEC>(cx[c], cr[kR ? c : 0], gain, h, v[c], sumsq, top);
            if constexpr (OP == kNormAdd)
                *reinterpret_cast<C*>(static_cast<T*>(p.h) + row * p.ldh + e) = h;
        }
    }
    reduce_row(sumsq, top, kW);
    const RowScale s = row_scale<OP>(sumsq, top, p.D, p.eps);
    int8_t* q = p.q + row * p.ldq;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int e = (c * int(blockDim.x) + int(threadIdx.x)) * VEC;
        prescale(s, v[c]);
        if (e < p.D) store_q<VEC>(q + e, v[c], s.inv, s.zero);
    }
    if (threadIdx.x == 0) p.scale[row] = s.scale;
}

// ------------------------------------------------------------------ rows that start anywhere
//
// A row whose start or length is no multiple of 16 bytes is cut into the same
// windows of VEC elements (16 bytes) from its start. A window lies across two
// aligned 16-byte words of memory, at the same offset `s` for the whole row, so
// it is read as two loads and a shift. The sum x + r goes through shared memory,
// where the reduction's barrier stands anyway, and is written as aligned words.
// Only words that lie inside the row are touched as a whole; at its two ends
// elements go one by one.
// Against reading every element by itself, 8192 x 8191 BF16: quantise 58 us
// (154), norm with a residual 153 (210), gate 92 (151).

// 16 bytes from `s` bytes into the 32 of lo and hi.
__device__ __forceinline__ uint4 shift_words(const uint4& lo, const uint4& hi, uint32_t s) {
    const uint32_t b = (s & 3u) * 8u;
    switch (s >> 2) {
        case 0:
            return make_uint4(__funnelshift_r(lo.x, lo.y, b), __funnelshift_r(lo.y, lo.z, b),
                              __funnelshift_r(lo.z, lo.w, b), __funnelshift_r(lo.w, hi.x, b));
        case 1:
            return make_uint4(__funnelshift_r(lo.y, lo.z, b), __funnelshift_r(lo.z, lo.w, b),
                              __funnelshift_r(lo.w, hi.x, b), __funnelshift_r(hi.x, hi.y, b));
        case 2:
            return make_uint4(__funnelshift_r(lo.z, lo.w, b), __funnelshift_r(lo.w, hi.x, b),
                              __funnelshift_r(hi.x, hi.y, b), __funnelshift_r(hi.y, hi.z, b));
        default:
            return make_uint4(__funnelshift_r(lo.w, hi.x, b), __funnelshift_r(hi.x, hi.y, b),
                              __funnelshift_r(hi.y, hi.z, b), __funnelshift_r(hi.z, hi.w, b));
    }
}

template <typename T>
using Window = Chunk<T, kVecOf<T>>;

// Elements e .. e + VEC - 1 of a row of D; zeros past its end.
template <typename T>
__device__ __forceinline__ Window<T> load_window(const T* row, int64_t e, int64_t D) {
    constexpr int V = kVecOf<T>;
    union {
        uint4 words;
        T elems[V];
    } u;
    const T* at = row + e;
    const uint32_t s = uint32_t(reinterpret_cast<uintptr_t>(at) & 15u);
    const int before = int(s) / int(sizeof(T));  // elements between the aligned word and `at`
    const uint4* word = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(at) - s);
    if (s == 0 && e + V <= D) {
        u.words = word[0];
    } else if (e >= before && e - before + 2 * V <= D) {
        u.words = shift_words(word[0], word[1], s);
    } else {
        u.words = make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (e + i < D) u.elems[i] = at[i];
    }
    Window<T> c;
    *reinterpret_cast<uint4*>(&c) = u.words;
    return c;
}

// The window at e to a row of D, by all lanes of a warp whose windows follow one
// another (the long rows' way, without shared memory).
template <typename T>
__device__ __forceinline__ void store_window(T* row, int64_t e, int64_t D, const Window<T>& c) {
    constexpr int V = kVecOf<T>;
    union {
        uint4 words;
        T elems[V];
    } u;
    u.words = *reinterpret_cast<const uint4*>(&c);
    uint4 next;  // the next lane's window
    next.x = __shfl_down_sync(0xffffffffu, u.words.x, 1);
    next.y = __shfl_down_sync(0xffffffffu, u.words.y, 1);
    next.z = __shfl_down_sync(0xffffffffu, u.words.z, 1);
    next.w = __shfl_down_sync(0xffffffffu, u.words.w, 1);
    T* at = row + e;
    const int lane = threadIdx.x & 31;
    // Bytes and elements from the window's start to the next 16-byte boundary.
    const uint32_t off = uint32_t(16 - (reinterpret_cast<uintptr_t>(at) & 15u)) & 15u;
    const int head = int(off) / int(sizeof(T));
    // From the boundary on: one store with the next lane's first elements, which
    // that lane then leaves out.
    const bool joined = e + head + V <= D && (lane < 31 || off == 0);
    if (joined) *reinterpret_cast<uint4*>(at + head) = shift_words(u.words, next, off);
    const bool keep_head = lane == 0 || e + head > D;
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (e + i < D && (i < head ? keep_head : !joined)) at[i] = u.elems[i];
}

// The 8-bit values of a window.
template <int V>
__device__ __forceinline__ void store_q_window(int8_t* row, int64_t e, int64_t D,
                                               const float (&v)[V], float inv, bool zero) {
    if (e + V <= D) {
        store_q<V>(row + e, v, inv, zero);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (e + i < D) row[e + i] = zero ? int8_t(0) : int8_t(round_bits(v[i], inv) & 0xffu);
    }
}

// ridge_row_i8 for such rows; q itself starts on VEC bytes.
template <typename T, int OP, int CH, int MAXT>
__global__ void __launch_bounds__(MAXT) ridge_row_i8_odd(const RowParams p) {
    constexpr bool kR = OP == kNormAdd || OP == kSiluMul;
    constexpr bool kW = OP == kNorm || OP == kNormAdd;
    constexpr int V = kVecOf<T>;
    const int64_t row = int64_t(blockIdx.x) * blockDim.y + threadIdx.y;
    if (row >= p.M) return;
    const T* x = static_cast<const T*>(p.x) + row * p.ldx;
    const T* r = static_cast<const T*>(p.r) + (kR ? row * p.ldr : 0);
    const T* w = static_cast<const T*>(p.w);
    // kNormAdd: the row of sums as it will be stored, and one word that is read past it.
    extern __shared__ uint4 s_rows[];
    uint4* s_row = s_rows + threadIdx.y * (CH * blockDim.x + 1);
    Window<T> cx[CH], cr[kR ? CH : 1];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int e = (c * int(blockDim.x) + int(threadIdx.x)) * V;
        cx[c] = load_window(x, e, p.D);
        if constexpr (kR) cr[c] = load_window(r, e, p.D);
    }
    float v[CH][V];
    float sumsq = 0.0f;
    float top = 0.0f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int e = (c * int(blockDim.x) + int(threadIdx.x)) * V;
        Window<T> h, gain = cx[c];
        if constexpr (kW) gain = load_window(w, e, p.D);
        take_chunk<T, OP, V>(cx[c], cr[kR ? c : 0], gain, h, v[c], sumsq, top);
        if constexpr (OP == kNormAdd)
            s_row[c * int(blockDim.x) + int(threadIdx.x)] = *reinterpret_cast<const uint4*>(&h);
    }
    reduce_row(sumsq, top, kW);
    if constexpr (OP == kNormAdd) {
        __syncwarp();  // a row of one warp passes no barrier in reduce_row
        T* out = static_cast<T*>(p.h) + row * p.ldh;
        const T* sums = reinterpret_cast<const T*>(s_row);
        // Elements, and bytes, before the row's first 16-byte boundary.
        const uint32_t off = uint32_t(16 - (reinterpret_cast<uintptr_t>(out) & 15u)) & 15u;
        const int head = int(off) / int(sizeof(T));
        if (int(threadIdx.x) < min(head, p.D)) out[threadIdx.x] = sums[threadIdx.x];
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int i = c * int(blockDim.x) + int(threadIdx.x), e = head + i * V;
            if (e + V <= p.D)
                *reinterpret_cast<uint4*>(out + e) = shift_words(s_row[i], s_row[i + 1], off);
            else
                for (int k = e; k < p.D; ++k) out[k] = sums[k];
        }
    }
    const RowScale s = row_scale<OP>(sumsq, top, p.D, p.eps);
    int8_t* q = p.q + row * p.ldq;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int e = (c * int(blockDim.x) + int(threadIdx.x)) * V;
        prescale(s, v[c]);
        store_q_window(q, e, p.D, v[c], s.inv, s.zero);
    }
    if (threadIdx.x == 0) p.scale[row] = s.scale;
}

// Rows longer than a CTA's registers hold: read twice (the second time mostly
// from L2), reduce in the first pass and write in the second. x + r is stored
// in the second pass only. With windows (kWindows) that start anywhere; without,
// element by element, for a q that does not start on VEC bytes.
//
// h may be x or r here too: each element is read in the second pass by the warp
// that stores it, and a warp stores its windows after it has read them. (Its two
// outer words may be read by a neighbouring warp as well, whose elements beside
// the boundary are its own alone: what it takes from such a word it stores itself.)
template <typename T, int OP, bool kWindows>
__global__ void __launch_bounds__(1024) ridge_row_i8_long(const RowParams p) {
    constexpr bool kR = OP == kNormAdd || OP == kSiluMul;
    constexpr bool kW = OP == kNorm || OP == kNormAdd;
    constexpr int V = kWindows ? kVecOf<T> : 1;
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(p.x) + row * p.ldx;
    const T* r = static_cast<const T*>(p.r) + (kR ? row * p.ldr : 0);
    const T* w = static_cast<const T*>(p.w);
    T* h_row = static_cast<T*>(p.h) + (OP == kNormAdd ? row * p.ldh : 0);
    using C = Chunk<T, V>;
    const int64_t step = int64_t(blockDim.x) * V;
    float sumsq = 0.0f;
    float top = 0.0f;
    C cx, cr, cw, h;
    float v[V];
    auto load = [&](const T* from, int64_t e) -> C {
        if constexpr (kWindows) return load_window(from, e, p.D);
        C c{};
        if (e < p.D) c.raw[0] = *reinterpret_cast<const typename C::Raw*>(from + e);
        return c;
    };
    auto take = [&](int64_t e, float& sum, float& max) {
        cx = load(x, e);
        if constexpr (kR) cr = load(r, e);
        if constexpr (kW) cw = load(w, e);
        take_chunk<T, OP, V>(cx, cr, cw, h, v, sum, max);
    };
    // Whole warps take part to the end of the row (first element of the warp's windows).
    const int64_t mine = int64_t(threadIdx.x) * V, first = int64_t(threadIdx.x & ~31u) * V;
    for (int64_t e = 0; first + e < p.D; e += step) take(mine + e, sumsq, top);
    reduce_row(sumsq, top, kW);
    const RowScale s = row_scale<OP>(sumsq, top, p.D, p.eps);
    int8_t* q = p.q + row * p.ldq;
    float unused_sum = 0.0f, unused_top = 0.0f;
    for (int64_t i = 0; first + i < p.D; i += step) {
        const int64_t e = mine + i;
        take(e, unused_sum, unused_top);
        prescale(s, v);
        if constexpr (kWindows) {
            if constexpr (OP == kNormAdd) store_window(h_row, e, p.D, h);
            store_q_window(q, e, p.D, v, s.inv, s.zero);
        } else if (e < p.D) {
            if constexpr (OP == kNormAdd) *reinterpret_cast<C*>(h_row + e) = h;
            store_q<V>(q + e, v, s.inv, s.zero);
        }
    }
    if (threadIdx.x == 0) p.scale[row] = s.scale;
}

// The launch shape of a row of `chunks` 16-byte chunks. Rows of up to 128 chunks
// take one warp, four rows to a CTA (no barrier). Longer rows take a CTA with as few
// chunks per thread as fit when there are fewer rows than SMs -- one row's
// latency is then all that counts -- and four per thread otherwise (two for rows
// that start anywhere, whose windows take two loads each), so that several CTAs
// share an SM and one row's reduction hides behind another's loads.
template <typename T, int OP>
cudaError_t run_rows(const RowParams& p, bool aligned, int num_sms, cudaStream_t stream) {
    constexpr int V = kVecOf<T>;
    const int64_t chunks = (int64_t(p.D) + V - 1) / V;
    auto launch = [&](void (*kernel)(RowParams), int per, int rows_per_cta) {
        const int threads = chunks <= 128 ? 32 : int(((chunks + per - 1) / per + 31) / 32 * 32);
        const dim3 block(static_cast<unsigned>(threads), static_cast<unsigned>(rows_per_cta));
        const unsigned grid = unsigned((int64_t(p.M) + rows_per_cta - 1) / rows_per_cta);
        const size_t smem =
            !aligned && OP == kNormAdd ? size_t(per * threads + 1) * rows_per_cta * 16 : 0;
        kernel<<<grid, block, smem, stream>>>(p);
        return cudaGetLastError();
    };
    const bool few = p.M <= num_sms;
    if (aligned) {
        if (chunks <= 32) return launch(ridge_row_i8<T, OP, V, 1, 1024>, 1, 4);
        if (chunks <= 64) return launch(ridge_row_i8<T, OP, V, 2, 1024>, 2, 4);
        if (chunks <= 128) return launch(ridge_row_i8<T, OP, V, 4, 512>, 4, 4);
        if (few && chunks <= 1024) return launch(ridge_row_i8<T, OP, V, 1, 1024>, 1, 1);
        if (few && chunks <= 2048) return launch(ridge_row_i8<T, OP, V, 2, 1024>, 2, 1);
        if (chunks <= 2048) return launch(ridge_row_i8<T, OP, V, 4, 512>, 4, 1);
        if (chunks <= 4096) return launch(ridge_row_i8<T, OP, V, 4, 1024>, 4, 1);
    } else {
        if (chunks <= 32) return launch(ridge_row_i8_odd<T, OP, 1, 1024>, 1, 4);
        if (chunks <= 64) return launch(ridge_row_i8_odd<T, OP, 2, 512>, 2, 4);
        if (chunks <= 128) return launch(ridge_row_i8_odd<T, OP, 4, 128>, 4, 4);
        if (few && chunks <= 1024) return launch(ridge_row_i8_odd<T, OP, 1, 1024>, 1, 1);
        if (chunks <= 1024) return launch(ridge_row_i8_odd<T, OP, 2, 512>, 2, 1);
        if (chunks <= 2048) return launch(ridge_row_i8_odd<T, OP, 2, 1024>, 2, 1);
    }
    ridge_row_i8_long<T, OP, true><<<unsigned(p.M), 1024, 0, stream>>>(p);
    return cudaGetLastError();
}

// Rows are read by plain 16-byte chunks when every row of every operand starts on
// 16 bytes and D is whole chunks, by windows otherwise. Either way q takes stores of
// VEC bytes; one that does not start on them is written byte by byte.
template <typename T, int OP>
cudaError_t run_op(const RowParams& p, int num_sms, cudaStream_t stream) {
    constexpr int V = kVecOf<T>;
    auto fits = [](const void* ptr, int64_t ld, int size, int bytes) {
        return (reinterpret_cast<uintptr_t>(ptr) % bytes) == 0 && (ld * size) % bytes == 0;
    };
    if (!fits(p.q, p.ldq, 1, V)) {
        ridge_row_i8_long<T, OP, false><<<unsigned(p.M), 1024, 0, stream>>>(p);
        return cudaGetLastError();
    }
    bool aligned = p.D % V == 0 && fits(p.x, p.ldx, sizeof(T), 16);
    if (OP == kNormAdd || OP == kSiluMul) aligned = aligned && fits(p.r, p.ldr, sizeof(T), 16);
    if (OP == kNorm || OP == kNormAdd) aligned = aligned && fits(p.w, 0, 1, 16);
    if (OP == kNormAdd) aligned = aligned && fits(p.h, p.ldh, sizeof(T), 16);
    return run_rows<T, OP>(p, aligned, num_sms, stream);
}

template <typename T>
cudaError_t run_type(int op, const RowParams& p, int num_sms, cudaStream_t stream) {
    switch (op) {
        case kQuant: return run_op<T, kQuant>(p, num_sms, stream);
        case kNorm: return run_op<T, kNorm>(p, num_sms, stream);
        case kNormAdd: return run_op<T, kNormAdd>(p, num_sms, stream);
        default: return run_op<T, kSiluMul>(p, num_sms, stream);
    }
}

// One translation unit per element type (quant_i8_*.cu).
cudaError_t run_rows_f16(int op, const RowParams& p, int num_sms, cudaStream_t stream);
cudaError_t run_rows_bf16(int op, const RowParams& p, int num_sms, cudaStream_t stream);
cudaError_t run_rows_f32(int op, const RowParams& p, int num_sms, cudaStream_t stream);

}  // namespace ridge_b200
