// Matrix products grouped by expert, on 5th-generation tensor cores (tcgen05.mma, accumulators in
// tensor memory): the rows of x are sorted by expert, offsets[e] .. offsets[e + 1] are the rows of
// expert e, and
//   rows product      out[t, :] = x[t, :] * w[e]                  (forward; with dY and W^T: dX)
//   weight gradient   out[e]    = sum over the rows t of e of x[t, :]^T * dY[t, :]
//   scaled product    the rows product of 8-bit operands, every 128 contraction values of a row of x
//                     and every 128 x 128 block of w with a scale of its own
// Group lengths are known on the device only; nothing is read back to the host.
//
// Roles of the operands.  The tensor core multiplies A (M = 128 rows) by B (N columns, any multiple
// of 16 up to 256).  M is the contiguous dimension of the output (the output features of a weight)
// and N runs over the rows, so that a group's last tile costs what its rows cost (N = its length
// rounded up to 32) and one row costs an MMA of N = 32, not a tile of 128.  Accumulator lanes are
// output columns: a warp's 32 lanes hold 32 neighbouring elements of one output row.
//
// One persistent CTA per SM, 12 warps: warp 0 copies tiles with TMA into a ring in shared memory
// (128 bytes of contraction per row: 64 values of 16 bits or 128 of 8), warp 1 issues the MMAs,
// warp 2 owns tensor memory, warps 4-11 are the epilogue.  Two accumulators of 256 columns: the
// epilogue of one tile runs under the MMAs of the next.
//
// Rows of a tile behind the end of its group belong to other groups: they only reach accumulator
// columns that are not stored.  In the weight gradient the rows are the contraction, so there the
// last (partial) step of a group is cut to a multiple of 16 rows and what is left of those 16 is
// zeroed in shared memory before the MMA reads it.
//
// Every mbarrier wait is bounded (about one second): one that runs out records
// BSP_ERR_DEVICE_TIMEOUT in the status word, all roles leave, copies in flight are waited for,
// tensor memory is freed.  Offsets that decrease or leave 0 .. T record BSP_ERR_DEVICE_RANGE and
// are clamped, so every access stays in bounds whatever they hold.
#include <stdio.h>

#include <atomic>

#include "common.cuh"
#include "umma_common.cuh"

namespace bsp {

using namespace umma;

namespace {

constexpr int kThreads = 384;
constexpr int kEpiWarps = 8;
constexpr int kTileM = 128;           // output columns of a tile
constexpr int kTileN = 256;           // rows of a tile (at most)
constexpr int kStages = 4;
constexpr int kABytes = kTileM * 128;
constexpr int kBBytes = kTileN * 128;
constexpr int kStageBytes = kABytes + kBBytes;
constexpr int kMaxGroups = 1024;      // bounded by the group table in shared memory
constexpr int kBand = 8;              // row tiles that are walked together for every column tile

constexpr int kModeRows = 0, kModeContract = 1;

struct Smem {
    static constexpr int kData = kStages * kStageBytes;
    static constexpr int kScale = 2 * kTileN * 4;
    static constexpr int kTable = 2 * (kMaxGroups + 1) * 4;
    static constexpr int kBars = (2 * kStages + 5) * 8;
    static constexpr int kTotal = kData + kScale + kTable + kBars + 64 + 1024;
};

struct Params {
    const void* offsets;
    int offsets_i64;
    int groups;
    int rows;        // T
    int cols;        // extent of the output's contiguous dimension
    int out_rows;    // weight gradient: rows of one group's output
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

struct Tile {
    int group;
    int r0, rows;    // first output row (of the whole output, or of the group's output), rows to store
    int c0;
    int t0;          // weight gradient: first contraction row
    int depth;       // contraction length
};

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}
__device__ __forceinline__ void tc_mma_f8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                          uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}

// A bounded wait of a whole warp: true only if it succeeded for every lane, so that the lanes go on or leave together.
__device__ __forceinline__ bool wait_all(uint32_t bar, uint32_t parity, volatile int* abort_flag, int32_t* status) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, status));
}

__device__ __forceinline__ int round_up(int v, int to) { return (v + to - 1) / to * to; }

// Rows of a group are cut into the fewest tiles of at most kTileN rows, all of about the same height.
__device__ __forceinline__ int tile_height(int m) {
    const int n = (m + kTileN - 1) / kTileN;
    return n == 0 ? 0 : round_up((m + n - 1) / n, 32);
}

template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// 32 accumulator columns of one warp = 32 rows of the output, lane = output column.
template <typename T>
__device__ __forceinline__ void store_columns(T* out, int64_t ld, const float* v, int rows, bool col_ok) {
    if (!col_ok) return;
#pragma unroll
    for (int j = 0; j < 32; ++j)
        if (j < rows) out[j * ld] = from_float<T>(v[j]);
}

template <int MODE, bool F8, bool A_MN>
__global__ void __launch_bounds__(kThreads, 1)
grouped_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
               const __grid_constant__ CUtensorMap map_b_small, const Params p) {
    extern __shared__ unsigned char smem_raw[];
    const uint32_t raw = smem_addr(smem_raw);
    const uint32_t data = (raw + 1023u) & ~1023u;
    unsigned char* data_ptr = smem_raw + (data - raw);
    float* scale_s = reinterpret_cast<float*>(data_ptr + Smem::kData);
    int* row_start = reinterpret_cast<int*>(data_ptr + Smem::kData + Smem::kScale);   // groups + 1
    int* tile_start = row_start + kMaxGroups + 1;                                     // groups + 1
    const uint32_t bars = data + Smem::kData + Smem::kScale + ((Smem::kTable + 7) & ~7);
    const uint32_t full_bar = bars, empty_bar = bars + 8 * kStages, tfull_bar = bars + 16 * kStages,
                   tempty_bar = tfull_bar + 16, drain_bar = tempty_bar + 16;
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_word;
    __shared__ int issued_stages;
    volatile int* abort_flag = &abort_word;

    constexpr int KE = F8 ? 128 : 64;        // contraction values of a ring entry
    constexpr int KSTEP = F8 ? 32 : 16;      // contraction values of one MMA
    constexpr bool B_MN = MODE == kModeContract;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(full_bar + 8 * s, 1);
            mbar_init(empty_bar + 8 * s, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(tfull_bar + 8 * i, 1);
            mbar_init(tempty_bar + 8 * i, kEpiWarps);
        }
        mbar_init(drain_bar, 1);
        abort_word = 0;
        issued_stages = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async;" ::: "memory");
    }
    // group table: clamped offsets, then (warp 0) their running maximum and the tiles before each group
    for (int i = threadIdx.x; i <= p.groups; i += kThreads) {
        const long long v = p.offsets_i64 ? reinterpret_cast<const long long*>(p.offsets)[i]
                                          : (long long)reinterpret_cast<const int*>(p.offsets)[i];
        const long long c = v < 0 ? 0 : v > p.rows ? p.rows : v;
        if (c != v && p.status) *p.status = BSP_ERR_DEVICE_RANGE;
        row_start[i] = (int)c;
    }
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;"
                     ::"r"(smem_addr(&tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    const int c_tiles = (p.cols + kTileM - 1) / kTileM;
    if (warp == 0) {
        int high = 0, before = 0;
        for (int base = 0; base <= p.groups; base += 32) {
            const int i = base + lane;
            int v = i <= p.groups ? row_start[i] : 0;
            const int own = v;
            for (int d = 1; d < 32; d <<= 1) {
                const int o = __shfl_up_sync(0xffffffffu, v, d);
                if (lane >= d) v = max(v, o);
            }
            v = max(v, high);
            if (i <= p.groups && v != own && p.status) *p.status = BSP_ERR_DEVICE_RANGE;
            high = __shfl_sync(0xffffffffu, v, 31);
            if (i <= p.groups) row_start[i] = v;
        }
        __syncwarp();
        if (MODE == kModeRows) {
            for (int base = 0; base < p.groups; base += 32) {
                const int i = base + lane;
                int n = 0;
                if (i < p.groups) n = (row_start[i + 1] - row_start[i] + kTileN - 1) / kTileN * c_tiles;
                const int own = n;
                for (int d = 1; d < 32; d <<= 1) {
                    const int o = __shfl_up_sync(0xffffffffu, n, d);
                    if (lane >= d) n += o;
                }
                if (i < p.groups) tile_start[i] = before + n - own;
                before += __shfl_sync(0xffffffffu, n, 31);
            }
            if (lane == 0) tile_start[p.groups] = before;
        }
    }
    __syncthreads();

    const int r_tiles_all = (p.out_rows + kTileN - 1) / kTileN;
    const int n_tiles = MODE == kModeRows ? tile_start[p.groups] : p.groups * c_tiles * r_tiles_all;

    auto tile_at = [&](int t) -> Tile {
        Tile o;
        int local, r_tiles;
        if (MODE == kModeRows) {
            int lo = 0, hi = p.groups - 1;          // the last group whose first tile is at or before t
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (tile_start[mid] <= t) lo = mid; else hi = mid - 1;
            }
            o.group = lo;
            local = t - tile_start[lo];
            r_tiles = (row_start[lo + 1] - row_start[lo] + kTileN - 1) / kTileN;
        } else {
            r_tiles = r_tiles_all;
            o.group = t / (c_tiles * r_tiles);
            local = t - o.group * c_tiles * r_tiles;
        }
        const int band = local / (kBand * c_tiles);
        const int in_band = min(kBand, r_tiles - band * kBand);
        const int rest = local - band * kBand * c_tiles;
        const int c = rest / in_band, r = band * kBand + rest - c * in_band;
        o.c0 = c * kTileM;
        const int first = row_start[o.group], m = row_start[o.group + 1] - first;
        if (MODE == kModeRows) {
            const int h = tile_height(m);
            o.r0 = first + r * h;
            o.rows = min(h, m - r * h);
            o.t0 = 0;
            o.depth = p.depth;
        } else {
            o.r0 = r * kTileN;
            o.rows = min(kTileN, p.out_rows - o.r0);
            o.t0 = first;
            o.depth = m;
        }
        return o;
    };

    if (warp == 0) {
        // ---------------- copies ----------------
        if (lane == 0) {
            uint32_t it = 0;
            bool alive = true;
            for (int t = blockIdx.x; t < n_tiles && alive; t += gridDim.x) {
                const Tile o = tile_at(t);
                const int n = round_up(o.rows, 32);
                const int steps = (o.depth + KE - 1) / KE;
                for (int k = 0; k < steps; ++k, ++it) {
                    const uint32_t s = it % kStages;
                    if (it >= kStages &&
                        !mbar_wait(empty_bar + 8 * s, (it / kStages - 1) & 1, abort_flag, p.status)) {
                        alive = false;
                        break;
                    }
                    const uint32_t a = data + s * kStageBytes, b = a + kABytes, bar = full_bar + 8 * s;
                    const int b_bytes = B_MN ? (n + 63) / 64 * 8192 : n * 128;
                    mbar_arrive_expect_tx(bar, kABytes + b_bytes);
                    issued_stages = (int)it + 1;
                    if (MODE == kModeRows) {
                        if (A_MN) {
                            tma_load_3d(a, &map_a, o.c0, k * KE, o.group, bar);
                            tma_load_3d(a + 8192, &map_a, o.c0 + 64, k * KE, o.group, bar);
                        } else {
                            tma_load_3d(a, &map_a, k * KE, o.c0, o.group, bar);
                        }
                        int r = 0;
                        for (; r + 128 <= n; r += 128) tma_load_2d(b + r * 128, &map_b, k * KE, o.r0 + r, bar);
                        for (; r < n; r += 32) tma_load_2d(b + r * 128, &map_b_small, k * KE, o.r0 + r, bar);
                    } else {
                        tma_load_2d(a, &map_a, o.c0, o.t0 + k * KE, bar);
                        tma_load_2d(a + 8192, &map_a, o.c0 + 64, o.t0 + k * KE, bar);
                        for (int r = 0; r < n; r += 64)
                            tma_load_2d(b + r * 128, &map_b, o.r0 + r, o.t0 + k * KE, bar);
                    }
                }
            }
        }
    } else if (warp == 1) {
        // ---------------- MMAs (the whole warp walks, lane 0 issues) ----------------
        uint32_t it = 0, acc = 0;
        bool alive = true;
        for (int t = blockIdx.x; t < n_tiles && alive; t += gridDim.x) {
            const Tile o = tile_at(t);
            const int n = round_up(o.rows, 32);
            const int steps = (o.depth + KE - 1) / KE;
            const uint32_t idesc = p.idesc | ((uint32_t)(n >> 3) << 17);
            for (int k = 0; k < steps; ++k, ++it) {
                const uint32_t s = it % kStages;
                // a new accumulator: per tile, and for 8-bit operands per step (every step has its own scales)
                if (F8 || k == 0) {
                    alive = acc < 2 || wait_all(tempty_bar + 8 * (acc & 1), (acc / 2 - 1) & 1, abort_flag, p.status);
                    if (!alive) break;
                    tc_fence_after();
                }
                alive = wait_all(full_bar + 8 * s, (it / kStages) & 1, abort_flag, p.status);
                if (!alive) break;
                const uint32_t a = data + s * kStageBytes, b = a + kABytes;
                const int valid = min(KE, o.depth - k * KE);
                const int mmas = (valid + KSTEP - 1) / KSTEP;
                if (MODE == kModeContract && (valid & (KSTEP - 1))) {
                    // rows of the next group inside the last 16: zero them in every 64-wide atom
                    const int pieces = (mmas * KSTEP - valid) * 8;     // 16-byte pieces per atom
                    const int atoms = 2 + (n + 63) / 64;
                    for (int i = lane; i < atoms * pieces; i += 32) {
                        const int atom = i / pieces, at = i - atom * pieces;
                        const uint32_t dst = (atom < 2 ? a + atom * 8192 : b + (atom - 2) * 8192) + valid * 128 + at * 16;
                        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(dst), "r"(0) : "memory");
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                }
                tc_fence_after();
                if (lane == 0) {
                    const uint32_t d = tmem + (acc & 1) * kTileN;
                    for (int kk = 0; kk < mmas; ++kk) {
                        const uint64_t ad = A_MN ? make_smem_desc(a + kk * 2048, 8192, 1024) : make_smem_desc(a + kk * 32, 16, 1024);
                        const uint64_t bd = B_MN ? make_smem_desc(b + kk * 2048, 8192, 1024) : make_smem_desc(b + kk * 32, 16, 1024);
                        const uint32_t accumulate = kk > 0 || (!F8 && k > 0);
                        if (F8) tc_mma_f8(d, ad, bd, idesc, accumulate);
                        else tc_mma_f16(d, ad, bd, idesc, accumulate);
                    }
                    tc_commit(empty_bar + 8 * s);
                    if (F8 || k == steps - 1) tc_commit(tfull_bar + 8 * (acc & 1));
                }
                __syncwarp();
                if (F8 || k == steps - 1) ++acc;
            }
        }
        if (!alive && lane == 0) {
            // the MMAs issued so far finish before tensor memory is given back
            tc_commit(drain_bar);
            mbar_wait_slow(drain_bar, 0, abort_flag, nullptr, kWaitLimitNs, false);
        }
        __syncwarp();
    } else if (warp >= 4) {
        // ---------------- epilogue ----------------
        const int quarter = warp & 3, half = (warp - 4) >> 2;
        const int epi_thread = threadIdx.x - 128;
        // rows outside every group are zero
        if (MODE == kModeRows) {
            const int64_t head = row_start[0], tail0 = row_start[p.groups];
            const int64_t outside = head + (p.rows - tail0);
            const int esize = p.out_dtype == BSP_F32 ? 4 : 2;
            const int64_t row_bytes = (int64_t)p.cols * esize, pieces = row_bytes / 16;
            for (int64_t i = (int64_t)blockIdx.x * 256 + epi_thread; i < outside * pieces; i += (int64_t)gridDim.x * 256) {
                const int64_t r = i / pieces, at = i - r * pieces;
                const int64_t row = r < head ? r : tail0 + (r - head);
                *reinterpret_cast<int4*>((char*)p.out + row * row_bytes + at * 16) = make_int4(0, 0, 0, 0);
            }
        }
        uint32_t acc = 0;
        bool alive = true;
        // 8-bit operands: a wait that ran out ends no loop early, the eight warps keep meeting at their
        // barrier and only skip what the wait was for
        for (int t = blockIdx.x; t < n_tiles && (F8 || alive); t += gridDim.x) {
            const Tile o = tile_at(t);
            const int n = round_up(o.rows, 32);
            const int steps = (o.depth + KE - 1) / KE;
            const int c = o.c0 + quarter * 32 + lane;
            const bool col_ok = c < p.cols;
            const int64_t first = MODE == kModeRows ? o.r0 : (int64_t)o.group * p.out_rows + o.r0;
            const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
            auto store = [&](int c32, const float* v) {
                const int rows = o.rows - c32;
                const int64_t at = (first + c32) * p.cols + c;
                if (p.out_dtype == BSP_F32) store_columns((float*)p.out + at, p.cols, v, rows, col_ok);
                else if (p.out_dtype == BSP_F16) store_columns((__half*)p.out + at, p.cols, v, rows, col_ok);
                else store_columns((__nv_bfloat16*)p.out + at, p.cols, v, rows, col_ok);
            };
            if (F8) {
                // every step's 128 products per element come back from tensor memory, are multiplied by
                // the step's scales and added up in fp32 registers
                float sum[4][32];
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 32; ++j) sum[i][j] = 0.0f;
                const bool row_ok = epi_thread < o.rows;
                const float* sx = p.scale_x + (int64_t)(o.r0 + epi_thread) * p.sx_row;
                const float* sw = p.scale_w + (int64_t)o.group * p.sw_group + (int64_t)(o.c0 / 128) * p.sw_n;
                float next = row_ok ? sx[0] * sw[0] : 0.0f;
                for (int k = 0; k < steps; ++k, ++acc) {
                    float* scale_now = scale_s + (acc & 1) * kTileN;
                    scale_now[epi_thread] = next;
                    if (k + 1 < steps)
                        next = row_ok ? sx[(int64_t)(k + 1) * p.sx_block] * sw[(int64_t)(k + 1) * p.sw_k] : 0.0f;
                    asm volatile("bar.sync 1, 256;" ::: "memory");
                    if (alive) alive = wait_all(tfull_bar + 8 * (acc & 1), (acc / 2) & 1, abort_flag, p.status);
                    if (alive) {
                        tc_fence_after();
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int c32 = (2 * i + half) * 32;
                            if (c32 < n) {
                                uint32_t v[32];
                                tc_ld32(lanes + (acc & 1) * kTileN + c32, v);
                                tc_wait_ld();
#pragma unroll
                                for (int j = 0; j < 32; j += 4) {
                                    const float4 f = *reinterpret_cast<const float4*>(scale_now + c32 + j);
                                    sum[i][j] += __uint_as_float(v[j]) * f.x;
                                    sum[i][j + 1] += __uint_as_float(v[j + 1]) * f.y;
                                    sum[i][j + 2] += __uint_as_float(v[j + 2]) * f.z;
                                    sum[i][j + 3] += __uint_as_float(v[j + 3]) * f.w;
                                }
                            }
                        }
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(tempty_bar + 8 * (acc & 1));
                }
                if (alive) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int c32 = (2 * i + half) * 32;
                        if (c32 < n) store(c32, sum[i]);
                    }
                }
            } else {
                const bool computed = steps > 0;    // a group without rows has a gradient of zero
                if (computed) {
                    alive = wait_all(tfull_bar + 8 * (acc & 1), (acc / 2) & 1, abort_flag, p.status);
                    if (!alive) break;
                    tc_fence_after();
                }
#pragma unroll 1
                for (int i = 0; i < 4; ++i) {
                    const int c32 = (2 * i + half) * 32;
                    if (c32 < n) {
                        uint32_t v[32];
                        if (computed) {
                            tc_ld32(lanes + (acc & 1) * kTileN + c32, v);
                            tc_wait_ld();
                        } else {
#pragma unroll
                            for (int j = 0; j < 32; ++j) v[j] = 0;
                        }
                        store(c32, reinterpret_cast<const float*>(v));
                    }
                }
                if (computed) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(tempty_bar + 8 * (acc & 1));
                    ++acc;
                }
            }
        }
    }

    // ---------------- teardown ----------------
    tc_fence_before();
    __syncthreads();
    if (abort_word) {
        // copies in flight land before the block may leave
        if (threadIdx.x == 0) {
            const int last = issued_stages;
            for (int i = last > kStages ? last - kStages : 0; i < last; ++i)
                mbar_wait_slow(full_bar + 8 * (i % kStages), (i / kStages) & 1, abort_flag, nullptr, kWaitLimitNs, false);
        }
        __syncthreads();
    }
    if (warp == 2) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

// ---- host side ---------------------------------------------------------------------

int make_map(CUtensorMap* map, const void* base, int elem, int rank, const int64_t* dims, const int64_t* strides_bytes,
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
    const CUresult r = fn(map, type, rank, const_cast<void*>(base), d, s, b, e, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        char what[64];
        snprintf(what, sizeof(what), "cuTensorMapEncodeTiled: CUresult %d", (int)r);
        set_cuda_error(cudaErrorInvalidValue, what);
        return BSP_ERR_CUDA;
    }
    return BSP_OK;
}

// The encoder is a driver call and needs the device's context current in this thread; a thread that has
// made no runtime call yet (the first backward of a process runs in one) does not have it.
int bind_context() {
    int dev = 0;
    BSP_CUDA_TRY(cudaGetDevice(&dev));
    BSP_CUDA_TRY(cudaSetDevice(dev));
    return BSP_OK;
}

bool is_f8(int type) { return type == BSP_E4M3 || type == BSP_E5M2; }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Rows (T, depth) with a row stride of ld elements; boxes of 128 bytes x `box_rows`.
int rows_map(CUtensorMap* map, const void* base, int elem, int64_t rows, int64_t width, int64_t ld, int box_rows) {
    const int esize = is_f8(elem) ? 1 : 2;
    const int64_t dims[2] = {width, rows}, strides[1] = {ld * esize};
    const int box[2] = {128 / esize, box_rows};
    return make_map(map, base, elem, 2, dims, strides, box);
}

template <int MODE, bool F8, bool A_MN>
int launch(const CUtensorMap& ma, const CUtensorMap& mb, const CUtensorMap& mbs, const Params& p, int64_t most_tiles,
           cudaStream_t stream) {
    auto kern = grouped_kernel<MODE, F8, A_MN>;
    static std::atomic<uint64_t> opted_in{0};
    int dev = 0;
    BSP_CUDA_TRY(cudaGetDevice(&dev));
    const uint64_t dev_bit = dev >= 0 && dev < 64 ? (1ull << dev) : 0;
    if (!(opted_in.load(std::memory_order_acquire) & dev_bit)) {
        BSP_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem::kTotal));
        opted_in.fetch_or(dev_bit, std::memory_order_release);
    }
    const int sms = num_sms();
    if (sms <= 0) return BSP_ERR_CUDA;
    const int ctas = (int)(most_tiles < sms ? (most_tiles < 1 ? 1 : most_tiles) : sms);
    kern<<<ctas, kThreads, Smem::kTotal, stream>>>(ma, mb, mbs, p);
    BSP_LAUNCH_CHECK();
    return BSP_OK;
}

// Tiles of a rows product: a group of m rows has ceil(m / kTileN) <= m / kTileN + 1 row tiles, and no more
// groups than rows have any.
int64_t most_row_tiles(int64_t rows, int64_t groups) {
    return rows / kTileN + (groups < rows ? groups : rows);
}

int check_sizes(int64_t rows, int64_t groups, int64_t depth, int64_t cols, const void* offsets) {
    if (rows < 0 || groups < 1 || depth < 1 || cols < 1 || !offsets) return BSP_ERR_INVALID_ARG;
    if (groups > kMaxGroups || rows > 0x7fffffffLL - 512 || depth > 0x7fffffffLL - 512 || cols > 0x7fffffffLL - 512)
        return BSP_ERR_UNSUPPORTED;
    if ((rows / kTileN + groups) * ceil_div(cols, kTileM) > 0x7fffffffLL - 65536) return BSP_ERR_UNSUPPORTED;
    return BSP_OK;
}

}  // namespace
}  // namespace bsp

using namespace bsp;

extern "C" int bsp_grouped_max_groups(void) { return kMaxGroups; }

extern "C" int bsp_grouped_matmul(const void* x, int64_t ld_x, const void* w, int64_t group_stride_w, int64_t ld_w,
                                  int w_cols_inner, const void* offsets, int offsets_i64, int64_t rows, int64_t groups,
                                  int64_t depth, int64_t cols, void* out, int dtype, int32_t* status_word,
                                  void* stream_) {
    if (rows == 0) return BSP_OK;
    int st = check_sizes(rows, groups, depth, cols, offsets);
    if (st != BSP_OK) return st;
    if (dtype != BSP_F16 && dtype != BSP_BF16) return BSP_ERR_UNSUPPORTED;
    if (!x || !w || !out || !aligned16(x) || !aligned16(w) || !aligned16(out)) return BSP_ERR_INVALID_ARG;
    const int64_t inner = w_cols_inner ? cols : depth, outer = w_cols_inner ? depth : cols;
    if ((depth & 7) || (cols & 7) || (ld_x & 7) || (ld_w & 7) || (group_stride_w & 7) || ld_x < depth || ld_w < inner ||
        group_stride_w < 0 || (groups > 1 && group_stride_w < 8))
        return BSP_ERR_INVALID_ARG;
    if ((st = bind_context()) != BSP_OK) return st;
    CUtensorMap ma, mb, mbs;
    const int64_t dims[3] = {inner, outer, groups};
    const int64_t strides[2] = {ld_w * 2, (groups > 1 ? group_stride_w : outer * ld_w) * 2};
    const int box[3] = {64, w_cols_inner ? 64 : kTileM, 1};
    if ((st = make_map(&ma, w, dtype, 3, dims, strides, box)) != BSP_OK) return st;
    if ((st = rows_map(&mb, x, dtype, rows, depth, ld_x, 128)) != BSP_OK) return st;
    if ((st = rows_map(&mbs, x, dtype, rows, depth, ld_x, 32)) != BSP_OK) return st;
    Params p = {};
    p.offsets = offsets;
    p.offsets_i64 = offsets_i64;
    p.groups = (int)groups;
    p.rows = (int)rows;
    p.cols = (int)cols;
    p.depth = (int)depth;
    p.out = out;
    p.out_dtype = dtype;
    const uint32_t fmt = dtype == BSP_BF16 ? 1u : 0u;
    p.idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | ((w_cols_inner ? 1u : 0u) << 15) | ((uint32_t)(kTileM >> 4) << 24);
    p.status = status_word;
    const int64_t tiles = most_row_tiles(rows, groups) * ceil_div(cols, kTileM);
    cudaStream_t stream = (cudaStream_t)stream_;
    return w_cols_inner ? launch<kModeRows, false, true>(ma, mb, mbs, p, tiles, stream)
                        : launch<kModeRows, false, false>(ma, mb, mbs, p, tiles, stream);
}

extern "C" int bsp_grouped_weight_grad(const void* x, int64_t ld_x, const void* grad, int64_t ld_grad,
                                       const void* offsets, int offsets_i64, int64_t rows, int64_t groups,
                                       int64_t depth, int64_t cols, void* out, int dtype, int32_t* status_word,
                                       void* stream_) {
    int st = check_sizes(rows, groups, depth, cols, offsets);
    if (st != BSP_OK) return st;
    if (rows < 1) return BSP_ERR_INVALID_ARG;
    if (dtype != BSP_F16 && dtype != BSP_BF16) return BSP_ERR_UNSUPPORTED;
    if (!x || !grad || !out || !aligned16(x) || !aligned16(grad) || !aligned16(out)) return BSP_ERR_INVALID_ARG;
    if ((depth & 7) || (cols & 7) || (ld_x & 7) || (ld_grad & 7) || ld_x < depth || ld_grad < cols)
        return BSP_ERR_INVALID_ARG;
    const int64_t tiles = groups * ceil_div(depth, kTileN) * ceil_div(cols, kTileM);
    if (tiles > 0x7fffffffLL - 65536) return BSP_ERR_UNSUPPORTED;
    if ((st = bind_context()) != BSP_OK) return st;
    CUtensorMap ma, mb;
    if ((st = rows_map(&ma, grad, dtype, rows, cols, ld_grad, 64)) != BSP_OK) return st;
    if ((st = rows_map(&mb, x, dtype, rows, depth, ld_x, 64)) != BSP_OK) return st;
    Params p = {};
    p.offsets = offsets;
    p.offsets_i64 = offsets_i64;
    p.groups = (int)groups;
    p.rows = (int)rows;
    p.cols = (int)cols;
    p.out_rows = (int)depth;
    p.out = out;
    p.out_dtype = dtype;
    const uint32_t fmt = dtype == BSP_BF16 ? 1u : 0u;
    p.idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | (1u << 15) | (1u << 16) | ((uint32_t)(kTileM >> 4) << 24);
    p.status = status_word;
    return launch<kModeContract, false, true>(ma, mb, mb, p, tiles, (cudaStream_t)stream_);
}

extern "C" int bsp_grouped_matmul_scaled(const void* x, int64_t ld_x, int type_x, const float* scale_x,
                                         int64_t sx_row, int64_t sx_block, const void* w, int64_t group_stride_w,
                                         int64_t ld_w, int type_w, const float* scale_w, int64_t sw_group,
                                         int64_t sw_k, int64_t sw_n, const void* offsets, int offsets_i64,
                                         int64_t rows, int64_t groups, int64_t depth, int64_t cols, void* out,
                                         int out_dtype, int32_t* status_word, void* stream_) {
    if (rows == 0) return BSP_OK;
    int st = check_sizes(rows, groups, depth, cols, offsets);
    if (st != BSP_OK) return st;
    if (!is_f8(type_x) || !is_f8(type_w)) return BSP_ERR_UNSUPPORTED;
    if (out_dtype != BSP_F16 && out_dtype != BSP_BF16 && out_dtype != BSP_F32) return BSP_ERR_UNSUPPORTED;
    if (!x || !w || !out || !scale_x || !scale_w || !aligned16(x) || !aligned16(w) || !aligned16(out))
        return BSP_ERR_INVALID_ARG;
    if ((depth & 15) || (cols & 7) || (ld_x & 15) || (ld_w & 15) || (group_stride_w & 15) || ld_x < depth ||
        ld_w < depth || group_stride_w < 0 || (groups > 1 && group_stride_w < 16))
        return BSP_ERR_INVALID_ARG;
    if ((st = bind_context()) != BSP_OK) return st;
    CUtensorMap ma, mb, mbs;
    const int64_t dims[3] = {depth, cols, groups};
    const int64_t strides[2] = {ld_w, groups > 1 ? group_stride_w : cols * ld_w};
    const int box[3] = {128, kTileM, 1};
    if ((st = make_map(&ma, w, type_w, 3, dims, strides, box)) != BSP_OK) return st;
    if ((st = rows_map(&mb, x, type_x, rows, depth, ld_x, 128)) != BSP_OK) return st;
    if ((st = rows_map(&mbs, x, type_x, rows, depth, ld_x, 32)) != BSP_OK) return st;
    Params p = {};
    p.offsets = offsets;
    p.offsets_i64 = offsets_i64;
    p.groups = (int)groups;
    p.rows = (int)rows;
    p.cols = (int)cols;
    p.depth = (int)depth;
    p.out = out;
    p.out_dtype = out_dtype;
    p.idesc = (1u << 4) | ((type_w == BSP_E5M2 ? 1u : 0u) << 7) | ((type_x == BSP_E5M2 ? 1u : 0u) << 10) |
              ((uint32_t)(kTileM >> 4) << 24);
    p.scale_x = scale_x;
    p.sx_row = sx_row;
    p.sx_block = sx_block;
    p.scale_w = scale_w;
    p.sw_group = sw_group;
    p.sw_k = sw_k;
    p.sw_n = sw_n;
    p.status = status_word;
    const int64_t tiles = most_row_tiles(rows, groups) * ceil_div(cols, kTileM);
    return launch<kModeRows, true, false>(ma, mb, mbs, p, tiles, (cudaStream_t)stream_);
}
