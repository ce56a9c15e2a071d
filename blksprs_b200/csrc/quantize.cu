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

template <bool E5M2>
__device__ __forceinline__ uint32_t round2(float a, float b) {
    return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, E5M2 ? __NV_E5M2 : __NV_E4M3);
}

// ---- rows: a scale for each 1 x 128 ----------------------------------------------------
// 16 lanes per block, 8 neighbouring values each: a warp takes two blocks at a time.  HBM-bound:
// each value once in (2 or 4 bytes) and once out (1 byte).
template <typename T, bool E5M2, bool VEC>
__global__ void __launch_bounds__(256)
quantize_rows_kernel(const T* __restrict__ x, int64_t ld, int64_t rows, int64_t width, int64_t blocks,
                     uint8_t* __restrict__ q, float* __restrict__ scale) {
    const float type_max = E5M2 ? 57344.0f : 448.0f;
    const int sub = threadIdx.x & 15;
    const int64_t total = rows * blocks, stride = (int64_t)gridDim.x * (blockDim.x / 16);
    // every warp stays whole in the loop (the shuffles below take all its lanes)
    for (int64_t first = (int64_t)blockIdx.x * (blockDim.x / 16) + (threadIdx.x / 32) * 2; first < total; first += stride) {
        const int64_t i = first + ((threadIdx.x >> 4) & 1);
        const bool ok = i < total;
        const int64_t row = ok ? i / blocks : 0, block = ok ? i - row * blocks : 0;
        const int64_t col = block * kBlock + sub * 8;
        const int64_t left = ok ? width - col : 0;        // values this lane has
        float v[8];
        const T* src = x + row * ld + col;
        if (VEC && left >= 8) {
            constexpr int N = 16 / sizeof(T);
#pragma unroll
            for (int part = 0; part < 8 / N; ++part) {
                const int4 raw = __ldg(reinterpret_cast<const int4*>(src) + part);
                const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
                for (int j = 0; j < N; ++j) v[part * N + j] = as_float(e[j]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = j < left ? as_float(src[j]) : 0.0f;
        }
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max(m, magnitude(v[j]));
#pragma unroll
        for (int d = 8; d; d >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
        const float s = scale_of(m, type_max);
        if (ok && sub == 0) scale[i] = s;
        uint32_t out[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) out[j] = round2<E5M2>(v[2 * j] / s, v[2 * j + 1] / s);
        uint8_t* dst = q + row * width + col;
        if (VEC && left >= 8) {
            *reinterpret_cast<uint2*>(dst) = make_uint2(out[0] | (out[1] << 16), out[2] | (out[3] << 16));
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (j < left) dst[j] = (uint8_t)(out[j / 2] >> (8 * (j & 1)));
        }
    }
}

// ---- weights: a scale for each 128 x 128 -------------------------------------------------
// One CTA of 256 threads per block.  Every thread holds its 64 values in registers between the two
// passes (largest magnitude, rounding), so that the weights are read once; the rounded block goes
// through shared memory, because q is stored with the depth innermost whatever the order of w.
template <typename T, bool E5M2>
__global__ void __launch_bounds__(256)
quantize_blocks_kernel(const T* __restrict__ w, int64_t sg, int64_t sk, int64_t sn, int64_t depth, int64_t cols,
                       int64_t k_blocks, int64_t n_blocks, uint8_t* __restrict__ q, float* __restrict__ scale) {
    constexpr int kPitch = kBlock + 4;        // bytes per column of the staged block
    __shared__ uint32_t staged[kBlock * kPitch / 4];
    __shared__ uint32_t largest[8];
    const float type_max = E5M2 ? 57344.0f : 448.0f;
    const int64_t per_group = k_blocks * n_blocks;
    const int64_t g = blockIdx.x / per_group, at = blockIdx.x - g * per_group;
    const int64_t k0 = at / n_blocks * kBlock, n0 = at % n_blocks * kBlock;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const T* src = w + g * sg;
    // a thread's values: 16 pieces of 4 neighbouring depths in one column.  Lanes run over the
    // contiguous dimension: over columns if it is that one, else over depths.
    const bool cols_inner = sn == 1;
    float v[16][4];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int n = cols_inner ? lane + 32 * (i & 3) : warp + 8 * i;
        const int k = cols_inner ? 4 * (warp + 8 * (i >> 2)) : 4 * lane;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bool ok = k0 + k + j < depth && n0 + n < cols;
            v[i][j] = ok ? as_float(src[(k0 + k + j) * sk + (n0 + n) * sn]) : 0.0f;
            m = max(m, magnitude(v[i][j]));
        }
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
    if (lane == 0) largest[warp] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, largest[i]);
    const float s = scale_of(m, type_max);
    if (threadIdx.x == 0) scale[blockIdx.x] = s;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int n = cols_inner ? lane + 32 * (i & 3) : warp + 8 * i;
        const int k = cols_inner ? 4 * (warp + 8 * (i >> 2)) : 4 * lane;
        staged[n * (kPitch / 4) + k / 4] =
            round2<E5M2>(v[i][0] / s, v[i][1] / s) | (round2<E5M2>(v[i][2] / s, v[i][3] / s) << 16);
    }
    __syncthreads();
    uint8_t* dst = q + g * depth * cols + n0 * depth + k0;
    const int ks = (int)min((int64_t)kBlock, depth - k0), ns = (int)min((int64_t)kBlock, cols - n0);
    const bool words = (depth & 3) == 0;
    for (int n = warp; n < ns; n += 8) {
        const uint32_t four = staged[n * (kPitch / 4) + lane];
        if (words) {
            if (4 * lane < ks) *reinterpret_cast<uint32_t*>(dst + n * depth + 4 * lane) = four;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (4 * lane + j < ks) dst[n * depth + 4 * lane + j] = (uint8_t)(four >> (8 * j));
        }
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
    quantize_blocks_kernel<T, E5M2><<<(unsigned)total, 256, 0, stream>>>((const T*)w, sg, sk, sn, depth, cols, kb, nb, (uint8_t*)q, scale);
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
    if (!w || !q || !scale || (reinterpret_cast<uintptr_t>(q) & 3)) return BSP_ERR_INVALID_ARG;
    return dispatch(dtype, type_q, [&](auto t, bool e5m2) {
        using T = decltype(t);
        return e5m2 ? launch_blocks<T, true>(w, group_stride_w, stride_depth, stride_cols, groups, depth, cols, q, scale, (cudaStream_t)stream)
                    : launch_blocks<T, false>(w, group_stride_w, stride_depth, stride_cols, groups, depth, cols, q, scale, (cudaStream_t)stream);
    });
}
