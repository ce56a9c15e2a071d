// 8-bit values with a scale for each block of 128: the operands of the scaled product.
//
//   scale = max(a * (1 / F), 2^-126), a the block's largest magnitude, F the type's largest value, its reciprocal
//           rounded (a product, as elementwise libraries divide by a constant: the same scales to the last bit)
//   q     = value / scale, rounded to nearest even (a / scale is F within two roundings, so nothing saturates)
//
// The floor of 2^-126 keeps the quotient finite for blocks of zeros and of subnormal magnitudes.
// Magnitudes are compared as bit patterns: NaN > infinity > any finite value, so that one NaN or
// infinity decides its block's scale.
#include <cuda_fp8.h>

#include "common.cuh"
#include "umma_common.cuh"

namespace bsp {
namespace {

constexpr int kBlock = 128;
constexpr float kSmallestScale = 1.17549435e-38f;   // 2^-126

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }

__device__ __forceinline__ float scale_of(float largest, float reciprocal_of_max) {
    const float s = largest * reciprocal_of_max;
    return s < kSmallestScale ? kSmallestScale : s;      // a NaN stays
}

// value / scale, correctly rounded, for one scale and many values: with y the correctly rounded reciprocal and
// q = x * y, the residual r = x - q * scale corrects q to q + r * y (Markstein 1990).  Where q is within one last place the
// residual is exact; q can be off by one and a half, and then it may not be (about 1 % of random pairs).  The result was
// the quotient all the same in 4e8 of them, and what it is rounded to afterwards has 2 or 3 bits.
// That needs residuals that do not underflow: for a scale above 2^-60 a quotient of at least 2^-18 (smaller ones
// round to zero in either type) has a residual above 2^-103.  Other scales divide.
struct Divider {
    float scale, reciprocal;
    __device__ __forceinline__ bool fast() const { return scale > 8.67e-19f && scale < 1.0e30f; }
    __device__ __forceinline__ float quick(float x) const {
        const float q = x * reciprocal;
        // the residual's negative, so that what is exact leaves q as it is: -0 stays -0
        return fmaf(-fmaf(q, scale, -x), reciprocal, q);
    }
};
__device__ __forceinline__ Divider divide_by(float scale) { return {scale, 1.0f / scale}; }

template <bool E5M2>
__device__ __forceinline__ uint32_t round2(float a, float b) {
    return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, E5M2 ? __NV_E5M2 : __NV_E4M3);
}
template <bool E5M2>
__device__ __forceinline__ uint2 round8(float* v, const Divider& over) {
    if (over.fast()) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = over.quick(v[j]);
    } else {
#pragma unroll 1
        for (int j = 0; j < 8; ++j) {
            // one at a time: this is rare, and eight divisions in line would be most of the kernel's code
            const float q = v[0] / over.scale;
#pragma unroll
            for (int i = 0; i < 7; ++i) v[i] = v[i + 1];
            v[7] = q;
        }
    }
    uint32_t out[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) out[j] = round2<E5M2>(v[2 * j], v[2 * j + 1]);
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
    // Largest magnitude as a bit pattern; 16-bit types: of the even and of the odd values, in either half.
    __device__ __forceinline__ uint32_t largest() const {
        const uint32_t* word = reinterpret_cast<const uint32_t*>(raw);
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 4 * kVectors; ++i)
            m = sizeof(T) == 2 ? __vmaxu2(m, word[i] & 0x7fff7fffu) : max(m, word[i] & 0x7fffffffu);
        return m;
    }
    static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
        return sizeof(T) == 2 ? __vmaxu2(a, b) : max(a, b);
    }
    // What largest() found, as a number.
    static __device__ __forceinline__ float value_of(uint32_t m) {
        if (sizeof(T) == 4) return __uint_as_float(m);
        const uint16_t h = (uint16_t)max(m & 0xffffu, m >> 16);
        return as_float(*reinterpret_cast<const T*>(&h));
    }
};

__device__ __forceinline__ void store_tail(uint8_t* dst, uint2 v, int64_t left) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (j < left) dst[j] = (uint8_t)((j < 4 ? v.x : v.y) >> (8 * (j & 3)));
}

// ---- rows: a scale for each 1 x 128 ----------------------------------------------------
// 8 lanes per block, 16 neighbouring values each (37 us on 16384 x 4096 bf16, 5.4 TB/s; fp32: 54 us, 6.2 TB/s; with 16
// lanes of 8 values 49 us in bf16: more shuffles and index arithmetic per value); every quarter warp takes kAhead blocks at
// a time, whose loads are under way together.
// HBM-bound: each value once in (2 or 4 bytes) and once out (1 byte).
constexpr int kAhead = 4;       // the lanes that divide (below) are as many

template <typename T, bool E5M2, bool VEC>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 3 : 2)
quantize_rows_kernel(const T* __restrict__ x, int64_t ld, int rows, int width, int blocks, uint8_t* __restrict__ q,
                     float* __restrict__ scale) {
    constexpr float reciprocal_of_max = E5M2 ? 1.0f / 57344.0f : 1.0f / 448.0f;
    const int lane = threadIdx.x & 31, sub = lane & 7;
    const int64_t stride = (int64_t)gridDim.x * 32;
    const int row_step = (int)(stride / blocks), block_step = (int)(stride - (int64_t)row_step * blocks);
    // quarter warp h of the grid takes blocks h, h + stride, ...; all quarters of a warp run the loop equally
    // often (the shuffles below take all lanes)
    const int64_t quarter = (int64_t)blockIdx.x * 32 + threadIdx.x / 8;
    int64_t row = quarter / blocks;
    int block = (int)(quarter - row * blocks);
    const int64_t total = (int64_t)rows * blocks;
    for (int64_t first = (int64_t)blockIdx.x * 32 + threadIdx.x / 32 * 4; first < total; first += kAhead * stride) {
        Eight<T> v[kAhead][2];
        int64_t rows_at[kAhead];
        int blocks_at[kAhead];
        uint32_t m[kAhead];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            const int col = block * kBlock + sub * 16;
            rows_at[a] = row;
            blocks_at[a] = block;
            const int left = row < rows ? width - col : 0;
            const T* from = x + row * ld + col;
            if (VEC && left >= 16) {
                v[a][0].load(from);
                v[a][1].load(from + 8);
            } else {
                v[a][0].gather(from, 1, left);
                v[a][1].gather(from + 8, 1, left - 8);
            }
            row += row_step;
            block += block_step;
            if (block >= blocks) {
                block -= blocks;
                ++row;
            }
        }
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            m[a] = Eight<T>::larger(v[a][0].largest(), v[a][1].largest());
#pragma unroll
            for (int d = 4; d; d >>= 1) m[a] = Eight<T>::larger(m[a], __shfl_xor_sync(0xffffffffu, m[a], d));
        }
        // the divisions of the four blocks side by side: lanes 0-3 of a quarter warp have one each
        const uint32_t mine = (lane & 2) ? ((lane & 1) ? m[3] : m[2]) : ((lane & 1) ? m[1] : m[0]);
        const Divider of_mine = divide_by(scale_of(Eight<T>::value_of(mine), reciprocal_of_max));
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            Divider over;
            over.scale = __shfl_sync(0xffffffffu, of_mine.scale, a, 8);
            over.reciprocal = __shfl_sync(0xffffffffu, of_mine.reciprocal, a, 8);
            if (rows_at[a] < rows) {
                const int col = blocks_at[a] * kBlock + sub * 16, left = width - col;
                if (sub == 0) scale[rows_at[a] * blocks + blocks_at[a]] = over.scale;
                uint2 out[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float f[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) f[j] = v[a][h].at(j);
                    out[h] = round8<E5M2>(f, over);
                }
                uint8_t* to = q + rows_at[a] * width + col;
                if (VEC && left >= 16) {
                    *reinterpret_cast<uint4*>(to) = make_uint4(out[0].x, out[0].y, out[1].x, out[1].y);
                } else if (left > 0) {
                    store_tail(to, out[0], left);
                    store_tail(to + 8, out[1], left - 8);
                }
            }
        }
    }
}

// ---- weights: a scale for each 128 x 128 -------------------------------------------------
// One CTA of 256 threads per block.  Every thread holds its 64 values in registers between the two passes
// (largest magnitude, rounding), so that the weights are read once (32 x 4096 x 2048 bf16: 137 us, 5.9 TB/s; the issue
// slots are 79 % busy; 16-bit weights stored depth-innermost spill 24 bytes per thread at the four CTAs per SM that fit);
// q is stored with the depth innermost.
// DEPTH_INNER: w is stored that way too, a thread has 8 neighbouring depths of 8 columns and writes them as they
// are.  Otherwise it has 8 neighbouring columns of 8 neighbouring depths, and the rounded block goes through
// shared memory: column n, 8-byte piece k at piece k ^ (n / 8 mod 16), free of bank conflicts both ways.
template <typename T, bool E5M2, bool DEPTH_INNER>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 4 : 2)
quantize_blocks_kernel(const T* __restrict__ w, int64_t sg, int64_t sk, int64_t sn, int64_t depth, int64_t cols,
                       int64_t k_blocks, int64_t n_blocks, bool vec, uint8_t* __restrict__ q,
                       float* __restrict__ scale) {
    __shared__ uint2 staged[DEPTH_INNER ? 1 : kBlock * 16];
    __shared__ uint32_t largest[8];
    constexpr float reciprocal_of_max = E5M2 ? 1.0f / 57344.0f : 1.0f / 448.0f;
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
    for (int j = 0; j < 8; ++j) m = Eight<T>::larger(m, v[j].largest());
#pragma unroll
    for (int d = 16; d; d >>= 1) m = Eight<T>::larger(m, __shfl_xor_sync(0xffffffffu, m, d));
    if ((threadIdx.x & 31) == 0) largest[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) m = Eight<T>::larger(m, largest[i]);
    const Divider over = divide_by(scale_of(Eight<T>::value_of(m), reciprocal_of_max));
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
    int64_t ctas = ceil_div(total, 32);
    const int sms = umma::num_sms();
    if (sms <= 0) return BSP_ERR_CUDA;
    // what is resident at once, as the kernel's launch bounds have it (16384 x 4096 bf16: 37 us, 24 per SM in waves 44; fp32:
    // 54 us, with three per SM, of which one waits for the others' end, 64)
    const int resident = sizeof(T) == 2 ? 3 : 2;
    if (ctas > sms * resident) ctas = sms * resident;
    // 16-byte loads and stores need every row to start on such a boundary
    const bool vec = (ld * (int64_t)sizeof(T)) % 16 == 0 && width % 16 == 0 &&
                     (reinterpret_cast<uintptr_t>(x) & 15) == 0 && (reinterpret_cast<uintptr_t>(q) & 15) == 0;
    auto kern = vec ? quantize_rows_kernel<T, E5M2, true> : quantize_rows_kernel<T, E5M2, false>;
    kern<<<(unsigned)ctas, 256, 0, stream>>>((const T*)x, ld, (int)rows, (int)width, (int)blocks, (uint8_t*)q, scale);
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
    auto kern = depth_inner ? quantize_blocks_kernel<T, E5M2, true> : quantize_blocks_kernel<T, E5M2, false>;
    kern<<<(unsigned)total, 256, 0, stream>>>((const T*)w, sg, sk, sn, depth, cols, kb, nb, vec, (uint8_t*)q, scale);
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
    if (rows > 0x7fffffffLL || width > 0x7fffffffLL - 256) return BSP_ERR_UNSUPPORTED;
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
