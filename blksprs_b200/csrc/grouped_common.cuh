// Shared by the grouped products (grouped.cu: tiles of CTA pairs; grouped_few.cu: few rows per group): launch
// parameters, bounded waits, cluster and epilogue pieces, tensor maps.
#pragma once

#include <stdio.h>

#include "common.cuh"
#include "umma_common.cuh"

namespace bsp {
namespace grouped {

using namespace umma;

constexpr int kMaxGroups = 1024;      // bounded by the group table in shared memory

struct Params {
    const void* offsets;
    int offsets_i64;
    int groups;
    int rows;        // T
    int cols;        // extent of the output's contiguous dimension
    int out_rows;    // weight gradient: rows of one group's output
    int parts;       // weight gradient: parts that a group's rows are split into (more than one: fp32 sums to be joined)
    int depth;       // rows product: contraction length
    void* out;
    int out_dtype;
    uint32_t idesc;  // instruction descriptor without N
    const float* scale_x;
    int64_t sx_row, sx_block;
    const float* scale_w;
    int64_t sw_group, sw_k, sw_n;
    int32_t* status;
};

// ---- clusters ----------------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t map_to_rank(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Arrival on a barrier of either CTA.  The plain form publishes no writes to the other CTA (tensor-memory reads
// are ordered by the tcgen05 fence before it): with release at cluster scope every arrival waited for all of the
// warp's memory traffic, 2000 cycles per 8-bit step.
__device__ __forceinline__ void mbar_arrive_pair(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// The forms that do: writes of this warp before the arrival are visible behind a wait that saw it in the other CTA.
__device__ __forceinline__ void mbar_publish_pair(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait_cluster(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    return done != 0;
}
// mbar_wait without a call: a call would have the epilogue's sums saved around it.
__device__ __forceinline__ bool bounded_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int32_t* status,
                                             bool honor_abort = true) {
    if (mbar_try_wait(bar, parity)) return true;
    unsigned long long t0 = 0;
    for (uint32_t it = 1;; ++it) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((it & 0xff) == 0) {
            if (honor_abort && *abort_flag) return false;
            if (t0 == 0) {
                t0 = global_timer();
            } else if (global_timer() - t0 > kWaitLimitNs) {
                *abort_flag = 1;
                if (status) *status = BSP_ERR_DEVICE_TIMEOUT;
                return false;
            }
        }
    }
}
__device__ __forceinline__ void copy_async_4(uint32_t to, const float* from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ float shared_float(uint32_t at) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ float4 shared_float4(uint32_t at) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
    return v;
}
// ---- scales of 8-bit steps -----------------------------------------------------------
// A step's sums are multiplied by two scales.  Their product is one factor, unless it leaves fp32's normal numbers: then
// it would be infinite (and infinity times a sum of 0 is NaN), have lost bits, or be 0, where the sum times both need not
// be.  Such a step multiplies twice: by the larger first where the product is small, by the smaller first where it is
// large, so that what lies between overflows or vanishes only if the result does (sums are 0 or 2^-32 .. 2^39).
__device__ __forceinline__ bool in_range(float product) {
    return fabsf(product) >= 1.17549435e-38f && fabsf(product) <= 3.40282347e38f;
}
// The two factors, in order; {1, product} where that is in range, or a scale is 0.
__device__ __forceinline__ float2 in_order(float a, float b) {
    const float product = a * b;
    if (in_range(product) || a == 0.0f || b == 0.0f) return make_float2(1.0f, product);
    const bool smaller_first = fabsf(product) > 1.0f;
    return (fabsf(a) > fabsf(b)) == smaller_first ? make_float2(b, a) : make_float2(a, b);
}
// sums += values * first * second, two neighbouring ones at a time.
__device__ __forceinline__ void add_pair(float& x, float& y, uint32_t v, uint32_t w, float2 factors) {
    asm("{\n\t.reg .b64 s, v, f;\n\tmov.b64 s, {%0, %1};\n\tmov.b64 v, {%2, %3};\n\tmov.b64 f, {%4, %4};\n\tmul.rn.f32x2 v, v, f;\n\t"
        "mov.b64 f, {%5, %5};\n\tfma.rn.f32x2 s, v, f, s;\n\tmov.b64 {%0, %1}, s;\n\t}"
        : "+f"(x), "+f"(y) : "r"(v), "r"(w), "f"(factors.x), "f"(factors.y));
}

// A bounded wait of a whole warp: true only if it succeeded for every lane, so that the lanes go on or leave
// together.  The first try is a straight line: 27 cycles on a barrier that is through, against 76 for the loop.
// progress: for waits that last as long as a whole contraction (the sums of 2^28 rows and more take a second): entries
// of the ring asked for so far.  The time then counts from when that number last changed; a ring that stands still is
// found by the roles that wait for its entries.
// CLUSTER: acquires what the other CTA published with its arrival.
template <bool CLUSTER = false>
__device__ __forceinline__ bool wait_all(uint32_t bar, uint32_t parity, volatile int* abort_flag, int32_t* status,
                                         const volatile int* progress = nullptr) {
    auto through = [&] { return CLUSTER ? mbar_try_wait_cluster(bar, parity) : mbar_try_wait(bar, parity); };
    if (__all_sync(0xffffffffu, through())) return true;
    unsigned long long t0 = 0;
    int seen = 0;
    for (uint32_t it = 1;; ++it) {
        if (__all_sync(0xffffffffu, through())) return true;
        if ((it & 0xff) == 0) {
            const unsigned long long now = global_timer();
            if (t0 == 0) t0 = now;
            if (progress && *progress != seen) {
                seen = *progress;
                t0 = now;
            }
            const bool late = now - t0 > kWaitLimitNs && now > t0;
            if (late) {
                *abort_flag = 1;
                if (status) *status = BSP_ERR_DEVICE_TIMEOUT;
            }
            if (__any_sync(0xffffffffu, late || *abort_flag)) return false;
        }
    }
}
// A value all lanes of a converged warp hold, told to the compiler: MMA operands then live in uniform registers.
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }

__device__ __forceinline__ int round_up(int v, int to) { return (v + to - 1) / to * to; }

// Programmatic dependent launch: the next launch of the stream may set up (barriers, tensor memory) on SMs this one
// leaves; no launch touches global memory before the one before it has finished.
__device__ __forceinline__ void let_next_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous_launch() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// ---- epilogue pieces ----------------------------------------------------------------
// A warp's staging area holds 32 output rows x 64 bytes; the 16-byte pieces of row r are permuted by
// (r / 2) mod 4, which keeps both the writes below and the reads free of bank conflicts.
__device__ __forceinline__ uint32_t staged_at(int row, int piece) { return row * 64 + ((piece ^ ((row >> 1) & 3)) << 4); }

// Stores the staged rows: four lanes write the 64 bytes of a row, eight rows per instruction.
__device__ __forceinline__ void store_staged(uint32_t staging, char* out, int64_t row_bytes, int rows, int bytes) {
    const int lane = threadIdx.x & 31;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = 8 * i + (lane >> 2), piece = lane & 3;
        uint32_t v[4];
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(staging + staged_at(row, piece)));
        if (row < rows && piece * 16 < bytes) st_global_16B(out + row * row_bytes + piece * 16, v);
    }
    __syncwarp();
}

// 16 lanes x 32 columns of tensor memory as four 8-column groups: r[4g], r[4g + 1] = lane t / 4, columns
// 8g + 2 (t mod 4) + {0, 1}; r[4g + 2], r[4g + 3] = lane t / 4 + 8, same columns.
__device__ __forceinline__ void tc_ld16x32(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr) : "memory");
}

// 32 lanes (output columns) x 32 accumulator columns (output rows) as two tc_ld16x32 deliver them: the pairs a thread
// holds are 8 x 8 matrices of neighbouring rows, stored transposed, so that a staged row is 32 neighbouring output
// columns.  (Exchanging words between lanes and storing them one by one took 40 instead of 12 shared-memory and
// shuffle instructions for the same 2 KiB.)
// words: v[2j], v[2j + 1] packed, in that order.
__device__ __forceinline__ void stage_transposed(uint32_t staging, const uint32_t* words) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const uint32_t at = staging + staged_at(8 * g + (lane & 7), lane >> 3);
        asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};"
                     ::"r"(at), "r"(words[2 * g]), "r"(words[2 * g + 1]), "r"(words[8 + 2 * g]), "r"(words[8 + 2 * g + 1])
                     : "memory");
    }
}

// 64 bytes of one output row per lane.
__device__ __forceinline__ void stage_row(uint32_t staging, const uint32_t* words) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};"
                     ::"r"(staging + staged_at(lane, i)), "r"(words[4 * i]), "r"(words[4 * i + 1]), "r"(words[4 * i + 2]),
                       "r"(words[4 * i + 3]) : "memory");
}

// ---- host side ---------------------------------------------------------------------

inline int make_map(CUtensorMap* map, const void* base, int elem, int rank, const int64_t* dims, const int64_t* strides_bytes,
             const int* box) {
    EncodeTiledFn fn = get_encode_fn();
    if (!fn) {
        set_cuda_error(cudaErrorNotSupported, "cuTensorMapEncodeTiled entry point");
        return BSP_ERR_CUDA;
    }
    cuuint64_t d[3], s[2];
    cuuint32_t b[3], e[3] = {1, 1, 1};
    for (int i = 0; i < rank; ++i) {
        d[i] = (cuuint64_t)dims[i];
        b[i] = (cuuint32_t)box[i];
    }
    for (int i = 0; i + 1 < rank; ++i) s[i] = (cuuint64_t)strides_bytes[i];
    const CUtensorMapDataType type = elem == BSP_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                   : elem == BSP_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                      : CU_TENSOR_MAP_DATA_TYPE_UINT8;
    auto encode = [&] {
        return fn(map, type, rank, const_cast<void*>(base), d, s, b, e, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    };
    CUresult r = encode();
    if (r == CUDA_ERROR_INVALID_CONTEXT) {
        // the encoder is a driver call and needs the device's context current in this thread; a thread that has made
        // no runtime call yet (the first backward of a process runs in one) does not have it
        int dev = 0;
        BSP_CUDA_TRY(cudaGetDevice(&dev));
        BSP_CUDA_TRY(cudaSetDevice(dev));
        r = encode();
    }
    if (r != CUDA_SUCCESS) {
        char what[64];
        snprintf(what, sizeof(what), "cuTensorMapEncodeTiled: CUresult %d", (int)r);
        set_cuda_error(cudaErrorInvalidValue, what);
        return BSP_ERR_CUDA;
    }
    return BSP_OK;
}

// A launch in clusters of `cluster` CTAs whose set-up overlaps the end of the launch before it.
template <typename K, typename... Args>
inline int launch_overlapped(K kernel, dim3 grid, int threads, int smem, int cluster, cudaStream_t stream, const Args&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    BSP_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, args...));
    return BSP_OK;
}

inline bool is_f8(int type) { return type == BSP_E4M3 || type == BSP_E5M2; }
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Rows (T, depth) with a row stride of ld elements; boxes of 128 bytes x `box_rows`.
inline int rows_map(CUtensorMap* map, const void* base, int elem, int64_t rows, int64_t width, int64_t ld, int box_rows) {
    const int esize = is_f8(elem) ? 1 : 2;
    const int64_t dims[2] = {width, rows}, strides[1] = {ld * esize};
    const int box[2] = {128 / esize, box_rows};
    return make_map(map, base, elem, 2, dims, strides, box);
}

// Product of few rows per group (grouped_few.cu); same operands as the products it stands in for: the weights in boxes
// of 128 features, the rows in boxes of 64 and of 32.
int launch_few(bool f8, bool a_mn, const CUtensorMap& weights, const CUtensorMap& rows_64, const CUtensorMap& rows_32,
               const Params& p, cudaStream_t stream);
bool few_applies(int64_t rows, int64_t groups, int64_t cols, bool f8);

}  // namespace grouped
}  // namespace bsp
