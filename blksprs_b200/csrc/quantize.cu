// 8-bit values with a scale for each block of 128: the operands of the scaled product.
//
//   scale = max(a / F, 2^-126), a the block's largest magnitude, F the type's largest value
//   q     = value / scale, rounded to nearest even (a / scale is F within one rounding, so nothing saturates)
//
// The floor of 2^-126 keeps the quotient finite for blocks of zeros and of subnormal magnitudes.
// Magnitudes are compared as bit patterns: NaN > infinity > any finite value, so that one NaN or
// infinity decides its block's scale.
#include <cuda_fp8.h>

#include "common.cuh"

namespace bsp {
namespace {

constexpr int kBlock = 128;
constexpr float kSmallestScale = 1.17549435e-38f;   // 2^-126

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }

__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

__device__ __forceinline__ float scale_of(uint32_t largest, float type_max) {
    const float s = __uint_as_float(largest) / type_max;
    return s < kSmallestScale ? kSmallestScale : s;      // a NaN stays
}

// value / scale, correctly rounded, for one scale and many values: with y the correctly rounded reciprocal and
// q = x * y, the residual r = x - q * scale is exact and q + r * y rounds to the quotient (Markstein 1990).
// That needs residuals that do not underflow: for a scale above 2^-60 a quotient of at least 2^-18 (smaller ones
// round to zero in either type) has a residual above 2^-103.  Other scales divide.
struct Divider {
    float scale, reciprocal;
    bool fast;
    __device__ __forceinline__ explicit Divider(float s)
        : scale(s), reciprocal(1.0f / s), fast(s > 8.67e-19f && s < 1.0e30f) {}
    __device__ __forceinline__ float operator()(float x) const {
        if (!fast) return x / scale;
        const float q = x * reciprocal;
        return fmaf(fmaf(-q, scale, x), reciprocal, q);
    }
};

template <bool E5M2>
__device__ __forceinline__ uint32_t round2(float a, float b) {
    return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, E5M2 ? __NV_E5M2 : __NV_E4M3);
}
template <bool E5M2>
__device__ __forceinline__ uint2 round8(const float* v, const Divider& over) {
    uint32_t out[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) out[j] = round2<E5M2>(over(v[2 * j]), over(v[2 * j + 1]));
    return make_uint2(out[0] | (out[1] << 16), out[2] | (out[3] << 16));
}

// Eight values as they lie in memory: 16 or 32 bytes, kept unconverted in registers.
template <typename T>
struct Eight {
    static constexpr int kVectors = sizeof(T) / 2;
    int4 raw[kVectors];
    __device__ __forceinline__ void load(const T* src) {
#pragma unroll
        for (int i = 0; i < kVectors; ++i) raw[i] = __ldg(reinterpret_cast<const int4*>(src) + i);
    }
    // element by element, `stride` apart, zeros behind `left`
    __device__ __forceinline__ void gather(const T* src, int64_t stride, int64_t left) {
        T* e = reinterpret_cast<T*>(raw);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (j < left) e[j] = src[j * stride];
            else e[j] = T(0.0f);
        }
    }
    __device__ __forceinline__ float at(int j) const { return as_float(reinterpret_cast<const T*>(raw)[j]); }
    __device__ __forceinline__ uint32_t largest() const {
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max(m, magnitude(at(j)));
        return m;
    }
};

__device__ __forceinline__ void store_tail(uint8_t* dst, uint2 v, int64_t left) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (j < left) dst[j] = (uint8_t)((j < 4 ? v.x : v.y) >> (8 * (j & 3)));
}

// ---- rows: a scale for each 1 x 128 ----------------------------------------------------
// 16 lanes per block, 8 neighbouring values each; every half warp takes kAhead blocks at a time, whose loads
// are under way together.  HBM-bound: each value once in (2 or 4 bytes) and once out (1 byte).
constexpr int kAhead = 4;

template <typename T, bool E5M2, bool VEC>
__global__ void __launch_bounds__(256)
quantize_rows_kernel(const T* __restrict__ x, int64_t ld, int64_t rows, int64_t width, int64_t blocks,
                     uint8_t* __restrict__ q, float* __restrict__ scale) {
    const float type_max = E5M2 ? 57344.0f : 448.0f;
    const int sub = threadIdx.x & 15;
    const int64_t total = rows * blocks, stride = (int64_t)gridDim.x * 16;
    const int64_t row_step = stride / blocks, block_step = stride - row_step * blocks;
    // half warp h of the grid takes blocks h, h + stride, ...; both halves of a warp run the loop equally often
    // (the shuffles below take all lanes)
    int64_t i = (int64_t)blockIdx.x * 16 + threadIdx.x / 16;
    int64_t row = i / blocks, block = i - row * blocks;
    for (int64_t first = (int64_t)blockIdx.x * 16 + threadIdx.x / 32 * 2; first < total; first += kAhead * stride) {
        Eight<T> v[kAhead];
        int64_t at[kAhead], to[kAhead], left[kAhead];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            const int64_t col = block * kBlock + sub * 8;
            at[a] = i;
            to[a] = row * width + col;
            left[a] = i < total ? width - col : 0;
            if (VEC && left[a] >= 8) v[a].load(x + row * ld + col);
            else v[a].gather(x + row * ld + col, 1, left[a]);
            i += stride;
            row += row_step;
            block += block_step;
            if (block >= blocks) {
                block -= blocks;
                ++row;
            }
        }
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            uint32_t m = v[a].largest();
#pragma unroll
            for (int d = 8; d; d >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
            const Divider over(scale_of(m, type_max));
            if (at[a] < total && sub == 0) scale[at[a]] = over.scale;
            float f[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = v[a].at(j);
            const uint2 out = round8<E5M2>(f, over);
            if (VEC && left[a] >= 8) *reinterpret_cast<uint2*>(q + to[a]) = out;
            else if (left[a] > 0) store_tail(q + to[a], out, left[a]);
        }
    }
}

// ---- weights: a scale for each 128 x 128 -------------------------------------------------
// One CTA of 256 threads per block.  Every thread holds its 64 values in registers between the two passes
// (largest magnitude, rounding), so that the weights are read once; q is stored with the depth innermost.
// DEPTH_INNER: w is stored that way too, a thread has 8 neighbouring depths of 8 columns and writes them as they
// are.  Otherwise it has 8 neighbouring columns of 8 neighbouring depths, and the rounded block goes through
// shared memory: column n, 8-byte piece k at piece k ^ (n / 8 mod 16), free of bank conflicts both ways.
template <typename T, bool E5M2, bool DEPTH_INNER>
__global__ void __launch_bounds__(256)
quantize_blocks_kernel(const T* __restrict__ w, int64_t sg, int64_t sk, int64_t sn, int64_t depth, int64_t cols,
                       int64_t k_blocks, int64_t n_blocks, bool vec, uint8_t* __restrict__ q,
                       float* __restrict__ scale) {
    __shared__ uint2 staged[DEPTH_INNER ? 1 : kBlock * 16];
    __shared__ uint32_t largest[8];
    const float type_max = E5M2 ? 57344.0f : 448.0f;
    const int64_t per_group = k_blocks * n_blocks;
    const int64_t g = blockIdx.x / per_group, block = blockIdx.x - g * per_group;
    const int64_t k0 = block / n_blocks * kBlock, n0 = block % n_blocks * kBlock;
    const int inner = threadIdx.x & 15, outer = threadIdx.x >> 4;
    const int64_t ks = min((int64_t)kBlock, depth - k0), ns = min((int64_t)kBlock, cols - n0);
    const T* src = w + g * sg + k0 * sk + n0 * sn;
    // piece j: 8 values along the inner dimension from inner * 8; the other index
    auto other = [&](int j) { return DEPTH_INNER ? outer + 16 * j : outer * 8 + j; };
    const int64_t inner_left = (DEPTH_INNER ? ks : ns) - inner * 8, others = DEPTH_INNER ? ns : ks;
    Eight<T> v[8];
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int o = other(j);
        const T* from = src + (DEPTH_INNER ? inner * 8 * sk + o * sn : inner * 8 * sn + o * sk);
        if (vec && inner_left >= 8 && o < others) v[j].load(from);
        else v[j].gather(from, DEPTH_INNER ? sk : sn, o < others ? inner_left : 0);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, v[j].largest());
#pragma unroll
    for (int d = 16; d; d >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
    if ((threadIdx.x & 31) == 0) largest[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, largest[i]);
    const Divider over(scale_of(m, type_max));
    if (threadIdx.x == 0) scale[blockIdx.x] = over.scale;
    uint8_t* dst = q + g * depth * cols + n0 * depth + k0;
    const bool wide = (depth & 7) == 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        float f[8];
        if (DEPTH_INNER) {
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = v[j].at(i);
            const uint2 out = round8<E5M2>(f, over);
            const int n = other(j);
            if (n < ns && inner_left > 0) {
                uint8_t* to = dst + n * depth + inner * 8;
                if (wide && inner_left >= 8) *reinterpret_cast<uint2*>(to) = out;
                else store_tail(to, out, inner_left);
            }
        } else {
            // column inner * 8 + j, its 8 depths from outer * 8
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = v[i].at(j);
            staged[(inner * 8 + j) * 16 + (outer ^ inner)] = round8<E5M2>(f, over);
        }
    }
    if (DEPTH_INNER) return;
    __syncthreads();
    const int64_t left = ks - inner * 8;
    for (int n = outer; n < ns; n += 16) {
        const uint2 out = staged[n * 16 + (inner ^ (n >> 3))];
        uint8_t* to = dst + n * depth + inner * 8;
        if (wide && left >= 8) *reinterpret_cast<uint2*>(to) = out;
        else if (left > 0) store_tail(to, out, left);
    }
}

template <typename T, bool E5M2>
int launch_rows(const void* x, int64_t ld, int64_t rows, int64_t width, void* q, float* scale, cudaStream_t stream) {
    const int64_t blocks = ceil_div(width, kBlock), total = rows * blocks;
    int64_t ctas = ceil_div(total, 16);
    if (ctas > 148 * 8) ctas = 148 * 8;
    // 16-byte loads and 8-byte stores need every row to start on such a boundary
    const bool vec = (ld * (int64_t)sizeof(T)) % 16 == 0 && width % 8 == 0 &&
                     (reinterpret_cast<uintptr_t>(x) & 15) == 0 && (reinterpret_cast<uintptr_t>(q) & 7) == 0;
    if (vec) quantize_rows_kernel<T, E5M2, true><<<(unsigned)ctas, 256, 0, stream>>>((const T*)x, ld, rows, width, blocks, (uint8_t*)q, scale);
    else quantize_rows_kernel<T, E5M2, false><<<(unsigned)ctas, 256, 0, stream>>>((const T*)x, ld, rows, width, blocks, (uint8_t*)q, scale);
    BSP_LAUNCH_CHECK();
    return BSP_OK;
}

template <typename T, bool E5M2>
int launch_blocks(const void* w, int64_t sg, int64_t sk, int64_t sn, int64_t groups, int64_t depth, int64_t cols,
                  void* q, float* scale, cudaStream_t stream) {
    const int64_t kb = ceil_div(depth, kBlock), nb = ceil_div(cols, kBlock), total = groups * kb * nb;
    if (total > 0x7fffffffLL) return BSP_ERR_UNSUPPORTED;
    // 8 values of a thread are 16-byte vectors if every row of the inner dimension starts on such a boundary
    const bool depth_inner = sk == 1 && sn != 1;
    const int64_t size = sizeof(T), outer = depth_inner ? sn : sk;
    const bool vec = (depth_inner || sn == 1) && (reinterpret_cast<uintptr_t>(w) & 15) == 0 && outer * size % 16 == 0 &&
                     sg * size % 16 == 0;
    if (depth_inner)
        quantize_blocks_kernel<T, E5M2, true><<<(unsigned)total, 256, 0, stream>>>((const T*)w, sg, sk, sn, depth, cols, kb, nb, vec, (uint8_t*)q, scale);
    else
        quantize_blocks_kernel<T, E5M2, false><<<(unsigned)total, 256, 0, stream>>>((const T*)w, sg, sk, sn, depth, cols, kb, nb, vec, (uint8_t*)q, scale);
    BSP_LAUNCH_CHECK();
    return BSP_OK;
}

template <typename F>
int dispatch(int dtype, int type_q, F&& f) {
    if (type_q != BSP_E4M3 && type_q != BSP_E5M2) return BSP_ERR_UNSUPPORTED;
    switch (dtype) {
        case BSP_F16: return f(__half{}, type_q == BSP_E5M2);
        case BSP_BF16: return f(__nv_bfloat16{}, type_q == BSP_E5M2);
        case BSP_F32: return f(float{}, type_q == BSP_E5M2);
        default: return BSP_ERR_UNSUPPORTED;
    }
}

}  // namespace
}  // namespace bsp

using namespace bsp;

extern "C" int bsp_quantize_rows(const void* x, int64_t ld_x, int64_t rows, int64_t width, int dtype, void* q,
                                 int type_q, float* scale, void* stream) {
    if (rows < 0 || width < 0 || ld_x < 0) return BSP_ERR_INVALID_ARG;
    if (rows == 0 || width == 0) return BSP_OK;
    if (!x || !q || !scale) return BSP_ERR_INVALID_ARG;
    return dispatch(dtype, type_q, [&](auto t, bool e5m2) {
        using T = decltype(t);
        return e5m2 ? launch_rows<T, true>(x, ld_x, rows, width, q, scale, (cudaStream_t)stream)
                    : launch_rows<T, false>(x, ld_x, rows, width, q, scale, (cudaStream_t)stream);
    });
}

extern "C" int bsp_quantize_blocks(const void* w, int64_t group_stride_w, int64_t stride_depth, int64_t stride_cols,
                                   int64_t groups, int64_t depth, int64_t cols, int dtype, void* q, int type_q,
                                   float* scale, void* stream) {
    if (groups < 0 || depth < 0 || cols < 0) return BSP_ERR_INVALID_ARG;
    if (groups == 0 || depth == 0 || cols == 0) return BSP_OK;
    if (!w || !q || !scale || (reinterpret_cast<uintptr_t>(q) & 7)) return BSP_ERR_INVALID_ARG;
    return dispatch(dtype, type_q, [&](auto t, bool e5m2) {
        using T = decltype(t);
        return e5m2 ? launch_blocks<T, true>(w, group_stride_w, stride_depth, stride_cols, groups, depth, cols, q, scale, (cudaStream_t)stream)
                    : launch_blocks<T, false>(w, group_stride_w, stride_depth, stride_cols, groups, depth, cols, q, scale, (cudaStream_t)stream);
    });
}
