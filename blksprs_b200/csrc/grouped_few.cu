// Products grouped by expert where the groups are short (a decoding step: one to a few rows for each expert): the
// rows product and the scaled product of grouped.cu, same operands, other shape.
//
// What bounds it is streaming the weights of the groups that have rows, and below a few tens of megabytes the
// latency of a launch.  So the tiles are small (128 output features x up to 64 rows, one CTA each, two CTAs per SM
// with 96 KiB of copies under way), and where there are too few of them to fill the GPU the contraction is split
// over a cluster of 2, 4 or 8 CTAs: each leaves its partial sums in its own shared memory, and after a cluster
// barrier each adds up a share of the rows over all of them, always in the same order.  No workspace, no atomics,
// the same bits on every run.
//
// A = weights (M = 128 features, accumulator lanes), B = rows (N = their number rounded up to 16).  8 bits: the
// scale of a step belongs to the accumulator's columns; two factors for each are read from shared memory as vectors.
// (A second multiplication costs nothing here; whether one is needed, decided in the epilogue, cost 1-3 of 45 us.)
//
// What it measured on a B200: 128 rows over 32 groups, 4096 x 2048 bf16: 77 us, 521 MB
// of weights at 6.8 TB/s (a plain copy moves 6.5); in 8 bits 45 us, 5.8 TB/s.  Two rows of two groups, 2048 x 4096 bf16
// (33 MB): 9.1 us; one row, 4096 x 4096 in 8 bits (17 MB): 7.8 us: launch, offsets, one copy's way and the
// cluster's exchange are most of both.
//
// Warp 0 copies, warp 1 issues the MMAs and owns tensor memory, warps 2-5 are the epilogue, warp 6 stages scales.
// Waits are bounded and offsets are clamped as in grouped.cu.
#include <atomic>

#include "grouped_common.cuh"

namespace bsp {
namespace grouped {

namespace {

constexpr int kFewThreads = 7 * 32;
constexpr int kFewM = 128;
constexpr int kFewN = 64;
constexpr int kFewStages = 4;
constexpr int kFewStageBytes = kFewM * 128 + kFewN * 128;
constexpr int kFewAccs = 2;                    // 8 bits: one per step, 16 bits: the first one
constexpr int kFewScaleSlots = 3;              // steps in groups of four
constexpr int kFewScaleSlot = 4 * kFewN * 2;   // floats: two factors per step and row

struct FewSmem {
    static constexpr int kData = kFewStages * kFewStageBytes;   // afterwards the partial sums, 64 x 128 floats
    static constexpr int kStaging = 4 * 2048;
    static constexpr int kScales = kFewScaleSlots * kFewScaleSlot * 4;
    static constexpr int kBars = (2 * kFewStages + 2 * kFewAccs + 1 + 2 * kFewScaleSlots) * 8;
    static constexpr int kTotal = kData + kStaging + kScales + kBars + 1024;     // two CTAs per SM
    static_assert(kFewN * kFewM * 4 <= kData, "partial sums reuse the ring");
    static_assert((kMaxGroups + 1) * 4 <= kStaging, "the offsets lie in the staging area until the tile is known");
    static_assert(2 * (kTotal + 64 + 1024) <= 228 * 1024, "two CTAs per SM");
};

template <bool F8>
__device__ __forceinline__ void few_mma(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    if (F8)
        asm volatile(
            "{\n\t.reg .pred p, e;\n\t"
            "elect.sync _|e, 0xffffffff;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "@e tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
            ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
    else
        tc_mma_f16_elect(d_tmem, adesc, bdesc, idesc, accumulate);
}

__device__ __forceinline__ void few_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}
__device__ __forceinline__ float2 cluster_float2(uint32_t addr) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}

// grid: x = cluster rank (split of the contraction) + split * column tile, y = row tile.
template <bool F8, bool A_MN>
__global__ void __launch_bounds__(kFewThreads, 2)
grouped_few_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x_64,
                   const __grid_constant__ CUtensorMap map_x_32, const Params p, const int split) {
    extern __shared__ unsigned char smem_raw[];
    const uint32_t raw = smem_addr(smem_raw);
    const uint32_t data = (raw + 1023u) & ~1023u;
    unsigned char* data_ptr = smem_raw + (data - raw);
    const uint32_t scales = data + FewSmem::kData + FewSmem::kStaging;
    int* row_start = reinterpret_cast<int*>(data_ptr + FewSmem::kData);      // groups + 1
    const uint32_t bars = scales + FewSmem::kScales;
    const uint32_t full_bar = bars, empty_bar = full_bar + 8 * kFewStages, tfull_bar = empty_bar + 8 * kFewStages,
                   tempty_bar = tfull_bar + 8 * kFewAccs, drain_bar = tempty_bar + 8 * kFewAccs,
                   sfull_bar = drain_bar + 8, sempty_bar = sfull_bar + 8 * kFewScaleSlots;
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_word, issued_stages;
    __shared__ int tile_s[5];              // group, first row, rows (0: nothing to do), rows before and behind all groups
    volatile int* abort_flag = &abort_word;

    constexpr int KE = F8 ? 128 : 64;
    constexpr int KSTEP = F8 ? 32 : 16;
    constexpr uint32_t kColumns = F8 ? 128 : 64;     // of tensor memory

    const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int rank = split > 1 ? (int)cluster_rank() : 0;
    let_next_launch();
    if (threadIdx.x == 0) {
        for (int s = 0; s < kFewStages; ++s) {
            mbar_init(full_bar + 8 * s, 1);
            mbar_init(empty_bar + 8 * s, 1);
        }
        for (int i = 0; i < kFewAccs; ++i) {
            mbar_init(tfull_bar + 8 * i, 1);
            mbar_init(tempty_bar + 8 * i, 4);
        }
        mbar_init(drain_bar, 1);
        for (int i = 0; i < kFewScaleSlots; ++i) {
            mbar_init(sfull_bar + 8 * i, 32);
            mbar_init(sempty_bar + 8 * i, 4);
        }
        abort_word = issued_stages = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_addr(&tmem_slot)), "r"(kColumns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    wait_for_previous_launch();
    for (int i = threadIdx.x; i <= p.groups; i += kFewThreads) {
        const long long v = p.offsets_i64 ? reinterpret_cast<const long long*>(p.offsets)[i]
                                          : (long long)reinterpret_cast<const int*>(p.offsets)[i];
        const long long c = v < 0 ? 0 : v > p.rows ? p.rows : v;
        if (c != v && p.status) *p.status = BSP_ERR_DEVICE_RANGE;
        row_start[i] = (int)c;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = uniform(tmem_slot);
    if (warp == 0) {
        // running maximum of the offsets; the group that row tile blockIdx.y falls into
        int high = 0, before = 0;
        const int want = (int)blockIdx.y;
        if (lane < 5) tile_s[lane] = 0;
        __syncwarp();
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
            // group i - 1 ends at v and starts where the lane before is
            int start = __shfl_up_sync(0xffffffffu, v, 1);
            if (lane == 0) start = high;
            const int tiles = i >= 1 && i <= p.groups ? (v - start + kFewN - 1) / kFewN : 0;
            int sum = tiles;
            for (int d = 1; d < 32; d <<= 1) {
                const int o = __shfl_up_sync(0xffffffffu, sum, d);
                if (lane >= d) sum += o;
            }
            const int first = before + sum - tiles;
            if (tiles > 0 && want >= first && want < first + tiles) {
                tile_s[0] = i - 1;
                tile_s[1] = start + (want - first) * kFewN;
                tile_s[2] = min(kFewN, v - tile_s[1]);
            }
            if (i == 0) tile_s[3] = v;
            if (i == p.groups) tile_s[4] = v;
            before += __shfl_sync(0xffffffffu, sum, 31);
            high = __shfl_sync(0xffffffffu, v, 31);
        }
    }
    __syncthreads();
    const int group = uniform(tile_s[0]), r0 = uniform(tile_s[1]), rows = uniform(tile_s[2]);
    const int c0 = (int)(blockIdx.x / split) * kFewM;
    const int n = round_up(rows, 16);
    const int all_steps = (p.depth + KE - 1) / KE, share = (all_steps + split - 1) / split;
    const int first_step = min(all_steps, rank * share);
    const int steps = rows > 0 ? min(all_steps, first_step + share) - first_step : 0;
    const int esize = p.out_dtype == BSP_F32 ? 4 : 2;
    const int64_t row_bytes = (int64_t)p.cols * esize;

    if (warp == 0) {
        // ---------------- copies ----------------
        if (lane == 0) {
            const int b_bytes = n > 32 ? 8192 : 4096;
            for (int k = 0; k < steps; ++k) {
                const int s = k % kFewStages;
                if (k >= kFewStages && !bounded_wait(empty_bar + 8 * s, (k / kFewStages - 1) & 1, abort_flag, p.status)) break;
                const uint32_t a = data + s * kFewStageBytes, b = a + kFewM * 128, bar = full_bar + 8 * s;
                const int x0 = (first_step + k) * KE;
                mbar_arrive_expect_tx(bar, kFewM * 128 + b_bytes);
                issued_stages = k + 1;
                if (A_MN) {
                    few_load_3d(a, &map_w, c0, x0, group, bar);
                    few_load_3d(a + 8192, &map_w, c0 + 64, x0, group, bar);
                } else {
                    few_load_3d(a, &map_w, x0, c0, group, bar);
                }
                tma_load_2d(b, n > 32 ? &map_x_64 : &map_x_32, x0, r0, bar);
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ---------------- MMAs ----------------
        const uint32_t idesc = p.idesc | ((uint32_t)(n >> 3) << 17);
        bool alive = true;
        for (int k = 0; k < steps; ++k) {
            const int s = k % kFewStages;
            if (F8 && k >= kFewAccs) {
                alive = wait_all(tempty_bar + 8 * (k % kFewAccs), (k / kFewAccs - 1) & 1, abort_flag, p.status);
                if (!alive) break;
            }
            alive = wait_all(full_bar + 8 * s, (k / kFewStages) & 1, abort_flag, p.status);
            if (!alive) break;
            tc_fence_after();
            const uint32_t a = data + s * kFewStageBytes, b = a + kFewM * 128;
            const int valid = min(KE, p.depth - (first_step + k) * KE), mmas = (valid + KSTEP - 1) / KSTEP;
            const uint32_t d = tmem + (F8 ? k % kFewAccs * kFewN : 0);
            const uint64_t ad = A_MN ? make_smem_desc(a, 8192, 1024) : make_smem_desc(a, 16, 1024);
            const uint64_t bd = make_smem_desc(b, 16, 1024);
            for (int kk = 0; kk < mmas; ++kk)
                few_mma<F8>(d, ad + kk * (A_MN ? 128 : 2), bd + kk * 2, idesc, kk > 0 || (!F8 && k > 0));
            tc_commit_elect(empty_bar + 8 * s);
            if (F8) tc_commit_elect(tfull_bar + 8 * (k % kFewAccs));
            else if (k == steps - 1) tc_commit_elect(tfull_bar);
        }
        if (!alive) {
            // the MMAs issued so far finish before tensor memory is given back
            tc_commit_elect(drain_bar);
            bounded_wait(drain_bar, 0, abort_flag, nullptr, false);
        }
        __syncwarp();
    } else if (warp == 6) {
        // ---------------- scales of four steps at a time (8 bits) ----------------
        if (F8) {
            // two factors for every step and row: what its two scales come to (one lane has two rows)
            const float* sx = p.scale_x + (int64_t)(r0 + lane) * p.sx_row;
            const float* sw = p.scale_w + (int64_t)group * p.sw_group + (int64_t)(c0 / 128) * p.sw_n;
            float x[2][4], w[4];
            auto load = [&](int k0) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int64_t k = first_step + k0 + j;
                    w[j] = k0 + j < steps ? sw[k * p.sw_k] : 0.0f;
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        x[h][j] = k0 + j < steps && h * 32 + lane < rows ? sx[h * 32 * p.sx_row + k * p.sx_block] : 0.0f;
                }
            };
            load(0);
            for (int k0 = 0, at = 0; k0 < steps; k0 += 4, ++at) {
                const int slot = at % kFewScaleSlots;
                if (at >= kFewScaleSlots &&
                    !wait_all(sempty_bar + 8 * slot, (at / kFewScaleSlots - 1) & 1, abort_flag, p.status))
                    break;
                const uint32_t to = scales + slot * kFewScaleSlot * 4;
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float2 f = in_order(x[h][j], w[j]);
                        asm volatile("st.shared.v2.f32 [%0], {%1, %2};"
                                     ::"r"(to + (j * kFewN + h * 32 + lane) * 8), "f"(f.x), "f"(f.y) : "memory");
                    }
                mbar_arrive(sfull_bar + 8 * slot);
                load(k0 + 4);
            }
            __syncwarp();
        }
    }

    // ---------------- epilogue warps: lane = output column, accumulator column = output row ----------------
    const int quarter = warp & 3;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
    float sum[2][32];
    bool complete = rows > 0;
    if (warp >= 2 && warp < 6) {
        // rows outside every group are zero
        const int64_t ctas = (int64_t)gridDim.x * gridDim.y, cta = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
        const int64_t before = tile_s[3], behind = tile_s[4], pieces = row_bytes / 16;
        const int64_t outside = before + (p.rows - behind);
        for (int64_t i = cta * 128 + threadIdx.x - 64; i < outside * pieces; i += ctas * 128) {
            const int64_t r = i / pieces, at = i - r * pieces;
            const int64_t row = r < before ? r : behind + (r - before);
            *reinterpret_cast<int4*>((char*)p.out + row * row_bytes + at * 16) = make_int4(0, 0, 0, 0);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < 32; ++j) sum[h][j] = 0.0f;
        if (F8) {
            for (int k = 0; k < steps; ++k) {
                const int slot = k / 4 % kFewScaleSlots;
                const uint32_t from = scales + slot * kFewScaleSlot * 4 + (k & 3) * kFewN * 8;
                complete = ((k & 3) != 0 || wait_all(sfull_bar + 8 * slot, (k / 4 / kFewScaleSlots) & 1, abort_flag, p.status)) &&
                           wait_all(tfull_bar + 8 * (k % kFewAccs), (k / kFewAccs) & 1, abort_flag, p.status);
                if (!complete) break;
                tc_fence_after();
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (h * 32 < n) {
                        // columns behind n hold anything: they are not stored
                        uint32_t v[32];
                        tc_ld32(lanes + k % kFewAccs * kFewN + h * 32, v);
                        tc_wait_ld();
#pragma unroll
                        for (int j = 0; j < 32; j += 2) {
                            const float4 f = shared_float4(from + (h * 32 + j) * 8);
                            sum[h][j] = fmaf(__uint_as_float(v[j]) * f.x, f.y, sum[h][j]);
                            sum[h][j + 1] = fmaf(__uint_as_float(v[j + 1]) * f.z, f.w, sum[h][j + 1]);
                        }
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(tempty_bar + 8 * (k % kFewAccs));
                    if ((k & 3) == 3 || k == steps - 1) mbar_arrive(sempty_bar + 8 * slot);
                }
            }
        } else if (steps > 0) {
            complete = wait_all(tfull_bar, 0, abort_flag, p.status, &issued_stages);
            if (complete) {
                tc_fence_after();
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (h * 32 < n) {
                        // stored by this CTA: as stage_transposed takes them; else a column per lane
                        uint32_t v[32];
                        if (split == 1) {
                            tc_ld16x32(lanes + h * 32, v);
                            tc_ld16x32(lanes + h * 32 + (16u << 16), v + 16);
                        } else {
                            tc_ld32(lanes + h * 32, v);
                        }
                        tc_wait_ld();
#pragma unroll
                        for (int j = 0; j < 32; ++j) sum[h][j] = __uint_as_float(v[j]);
                    }
                }
                tc_fence_before();
            }
        }
        if (split == 1 && complete) {
            const uint32_t staging = data + FewSmem::kData + (warp - 2) * 2048;
            const int c = c0 + quarter * 32;
            char* out = (char*)p.out + r0 * row_bytes + (int64_t)c * esize;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (h * 32 < rows) {
                    if (F8) {
                        // a column per lane: 64 bytes (fp32: 128) of a row per warp and store
#pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            char* at = out + (h * 32 + j) * row_bytes + lane * esize;
                            if (h * 32 + j < rows && c + lane < p.cols) {
                                if (p.out_dtype == BSP_F32) *reinterpret_cast<float*>(at) = sum[h][j];
                                else if (p.out_dtype == BSP_F16) *reinterpret_cast<__half*>(at) = __float2half_rn(sum[h][j]);
                                else *reinterpret_cast<__nv_bfloat16*>(at) = __float2bfloat16_rn(sum[h][j]);
                            }
                        }
                    } else {
                        uint32_t words[16];
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            words[j] = p.out_dtype == BSP_F16 ? pack2<__half>(sum[h][2 * j], sum[h][2 * j + 1])
                                                              : pack2<__nv_bfloat16>(sum[h][2 * j], sum[h][2 * j + 1]);
                        stage_transposed(staging, words);
                        store_staged(staging, out + h * 32 * row_bytes, row_bytes, rows - h * 32, min(p.cols - c, 32) * 2);
                    }
                }
            }
        }
    }

    // ---------------- teardown ----------------
    tc_fence_before();
    __syncthreads();
    if (abort_word && threadIdx.x == 0) {
        // copies in flight land before the block may leave (or its shared memory is used again)
        const int last = issued_stages;
        for (int i = last > kFewStages ? last - kFewStages : 0; i < last; ++i)
            bounded_wait(full_bar + 8 * (i % kFewStages), (i / kFewStages) & 1, abort_flag, nullptr, false);
    }
    __syncthreads();
    if (split > 1) {
        // partial sums [row][column] over the ring, which every copy and MMA is through with; fp32, joined in fp32 and
        // rounded once at the end
        if (warp >= 2 && warp < 6) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < 32; ++j)
                    if (h * 32 + j < rows)
                        asm volatile("st.shared.f32 [%0], %1;"
                                     ::"r"(data + ((h * 32 + j) * kFewM + quarter * 32 + lane) * 4), "f"(sum[h][j]) : "memory");
        }
        cluster_sync();
        const int pair = threadIdx.x & 63;                       // two columns of one row per thread
        const int c = c0 + 2 * pair;
        if (threadIdx.x < 192 && c < p.cols) {
            for (int r = rank * 3 + (threadIdx.x >> 6); r < rows; r += split * 3) {
                float2 total = make_float2(0.0f, 0.0f);
                for (int q = 0; q < split; ++q) {
                    const float2 part = cluster_float2(map_to_rank(data + (r * kFewM + 2 * pair) * 4, q));
                    total.x += part.x;
                    total.y += part.y;
                }
                char* out = (char*)p.out + (r0 + r) * row_bytes + (int64_t)c * esize;
                if (p.out_dtype == BSP_F32) *reinterpret_cast<float2*>(out) = total;
                else *reinterpret_cast<uint32_t*>(out) = p.out_dtype == BSP_F16 ? pack2<__half>(total.x, total.y)
                                                                                : pack2<__nv_bfloat16>(total.x, total.y);
            }
        }
        cluster_sync();      // no CTA leaves while another still reads its sums
    }
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kColumns) : "memory");
    }
}

template <bool F8, bool A_MN>
int launch_kernel(const CUtensorMap& weights, const CUtensorMap& rows_64, const CUtensorMap& rows_32, const Params& p,
                  cudaStream_t stream) {
    auto kern = grouped_few_kernel<F8, A_MN>;
    static std::atomic<uint64_t> opted_in{0};
    int dev = 0;
    BSP_CUDA_TRY(cudaGetDevice(&dev));
    const uint64_t dev_bit = dev >= 0 && dev < 64 ? (1ull << dev) : 0;
    if (!(opted_in.load(std::memory_order_acquire) & dev_bit)) {
        BSP_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, FewSmem::kTotal));
        opted_in.fetch_or(dev_bit, std::memory_order_release);
    }
    const int sms = num_sms();
    if (sms <= 0) return BSP_ERR_CUDA;
    const int64_t c_tiles = ceil_div(p.cols, kFewM);
    const int64_t hit = p.groups < p.rows ? p.groups : p.rows;
    const int64_t row_tiles = p.rows / kFewN + hit;              // at most
    if (c_tiles * 8 > 0x7fffffffLL || row_tiles > 65535) return BSP_ERR_UNSUPPORTED;
    // Split the contraction while all CTAs fit the GPU at once (two per SM) and each keeps four steps.
    const int64_t steps = ceil_div(p.depth, F8 ? 128 : 64);
    int split = 1;
    while (split < 8 && c_tiles * hit * split * 2 <= 2 * sms && steps >= 8 * split) split *= 2;
    return launch_overlapped(kern, dim3((unsigned)(c_tiles * split), (unsigned)row_tiles), kFewThreads, FewSmem::kTotal,
                             split, stream, weights, rows_64, rows_32, p, split);
}

}  // namespace

// Which of the two: by the mean rows of the groups that can have rows, and by whether either kernel's tiles fill the GPU.
// Measured (us, few / pairs; groups, depth x columns, rows per group):
//   16 bits   64, 2048 x 1024: 32: 48 / 49, 48: 51 / 50, 128: 80 / 56     16, 4096 x 4096: 4: 77 / 87, 48: 89 / 90
//             8, 2048 x 2048: 8: 14.9 / 14.6, 16: 15.5 / 14.7, 48: 23 / 15
//             4, 1024 x 1024: 4: 5.7 / 8.8, 64: 8.4 / 9.4, 128: 13 / 10   1, 4096 x 4096: 64: 15 / 22, 96: 21 / 22
//   8 bits    64, 2048 x 1024: 48: 35 / 42, 64: 44 / 43                   16, 4096 x 4096: 4: 45 / 64, 64: 68 / 75
//             8, 2048 x 2048: 32: 14 / 15, 48: 18 / 15                    1, 4096 x 4096: 64: 14 / 18, 96: 19 / 19
// The bounds are on the device, so the mean decides also where all rows went to one of the groups.  Such a batch, beside the
// even one and beside the same rows as a group of their own (us): 16 bits, 64 groups, 2048 x 1024, 2048 rows: 17.8, 47.5,
// 16.2; 16 groups, 4096 x 4096, 192 rows: 21.6, 81.2, 23.3; 8 bits, 64 groups, 2048 x 1024, 2048 rows: 19.8, 30.8, 13.6; 16
// groups, 4096 x 4096, 768 rows: 53.4, 55.3, 22.8 (twelve row tiles read the weights, from L2).
bool few_applies(int64_t rows, int64_t groups, int64_t cols, bool f8) {
    const int64_t hit = groups < rows ? groups : rows;
    if (rows / kFewN + hit > 65535) return false;
    const bool fills = hit * ceil_div(cols, kFewM) >= 512;                   // a tile per group and 128 columns
    const bool pairs_idle = 4 * hit * ceil_div(cols, 256) <= num_sms();      // less than half of the pairs have a tile
    const int64_t most = pairs_idle ? (f8 ? 96 : 72) : fills ? (f8 ? 64 : 40) : (f8 ? 40 : 12);
    return rows <= most * hit;
}

int launch_few(bool f8, bool a_mn, const CUtensorMap& weights, const CUtensorMap& rows_64, const CUtensorMap& rows_32,
               const Params& p, cudaStream_t stream) {
    if (f8) return launch_kernel<true, false>(weights, rows_64, rows_32, p, stream);
    return a_mn ? launch_kernel<false, true>(weights, rows_64, rows_32, p, stream)
                : launch_kernel<false, false>(weights, rows_64, rows_32, p, stream);
}

}  // namespace grouped
}  // namespace bsp
