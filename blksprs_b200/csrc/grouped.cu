// Matrix products grouped by expert, on 5th-generation tensor cores (tcgen05.mma, accumulators in
// tensor memory): the rows of x are sorted by expert, offsets[e] .. offsets[e + 1] are the rows of
// expert e, and
//   rows product      out[t, :] = x[t, :] * w[e]                  (forward; with dY and W^T: dX)
//   weight gradient   out[e]    = sum over the rows t of e of x[t, :]^T * dY[t, :]
//   scaled product    the rows product of 8-bit operands, every 128 contraction values of a row of x
//                     and every 128 x 128 block of w with a scale of its own
// Group lengths are known on the device only; nothing is read back to the host.
//
// Two SMs share a tile (cta_group::2): M = 256, 128 accumulator lanes in each SM.  Each SM stages half of
// either operand, 32 KiB per 128 bytes of contraction and 256 columns; one SM alone with a tile of
// 128 x 256 would stage 48 KiB for the same 512 cycles of tensor-core work, and shared memory would
// be the bound (written once by TMA, read once by the MMA at 128 bytes per cycle: 768 cycles).
// Where groups are long a 16-bit tile has 512 rows, two accumulators that share what is staged of A.
//
// Roles of the operands.
//   16 bits: M runs over the output's contiguous dimension (output features), N over its rows.  N is any
//   multiple of 32, so a group's last tile costs what its rows cost.  Lanes are output columns.
//   8 bits: M runs over the rows, N over the output features.  A lane is a row of x, so a step's scale
//   (one for each row and each 128 features) is one register per thread.
//
// What it measured on a B200 (time, rate; bf16): forward, dX and dW of 8 groups of 2048 rows, 4096 x 4096:
// 370, 363-375 and 376-454 us, 1486, 1466-1514 and 1210-1462 TFLOP/s, the tensor pipe 76-83 % busy at the 1.51-1.56 GHz
// that the power cap leaves (a plain library product of 8192^3: 1404 TFLOP/s sustained, 1687 in a burst).  16
// groups of 1024 rows, 2048 x 4096: 206 us, 1335 TFLOP/s; the same in 8 bits, 4096 x 4096: 298 us, 1845
// TFLOP/s, tensor pipe 54 %: there the epilogue bounds, 128 multiply-adds per thread and 512 cycles of MMAs, with
// the waits around them (timed inside the kernel: 700 cycles per step).  64 groups of 64 rows, 2048 x 1024: 52
// us, HBM 65 % busy; 64 groups of 128 rows: 55 us, 318 MB at 5.8 TB/s.
//
// Persistent CTA pairs, 12 warps per CTA: warp 0 copies tiles with TMA into a ring in shared memory,
// warp 1 of the first CTA issues the MMAs, warp 2 owns tensor memory, warps 4-11 are the epilogue.
// Two accumulators of 256 columns: the epilogue of one tile (8 bits: of one step; tall tiles: of one half)
// runs under the MMAs of the next.
//
// Rows of a tile behind the end of its group belong to other groups: they only reach accumulator rows
// that are not stored.  In the weight gradient the rows are the contraction, so there the last
// (partial) step of a group is cut to a multiple of 16 rows and what is left of those 16 is zeroed in
// shared memory before the MMA reads it.
//
// Every mbarrier wait is bounded (about one second): one that runs out records
// BSP_ERR_DEVICE_TIMEOUT in the status word, all roles leave, copies and MMAs in flight are waited
// for, tensor memory is freed.  Offsets that decrease or leave 0 .. T record BSP_ERR_DEVICE_RANGE and
// are clamped, so every access stays in bounds whatever they hold.
#include <atomic>

#include "grouped_common.cuh"

namespace bsp {

using namespace grouped;

namespace {

constexpr int kThreads = 384;
constexpr int kEpiWarps = 8;
constexpr int kTile = 256;            // M of a pair's tile, and most of an MMA's N
constexpr int kHalf = 128;            // M in either CTA
constexpr int kScaleSlots = 4;        // groups of four steps whose scales are staged ahead
constexpr int kScaleSlot = 4 * kHalf + 12;  // words of a slot: four scales per row of the CTA's half, four of either block of
constexpr int kScaleFlag = (4 * kHalf + 8) * 4;     // w, whether these steps are multiplied by both, and three unused
constexpr int kBand = 8;              // row tiles that are walked together for every column tile

enum Mode { kRows16, kGrad16, kRows8 };

// N of an MMA, accumulators in tensor memory (512 columns in all), ring stages.  (8 bits with four accumulators of
// N = 128 instead, on 16 groups of 1024 rows, 4096 x 4096: 389 against 310 us with tiles of 128 features, 347 against
// 300 with halves of 256; the hand-over of an accumulator costs about the same whatever its width.)
constexpr int kN = 256, kAccs = 2;
constexpr int ring_stages(int halves) { return halves == 2 ? 4 : 6; }

template <int MODE, int HALVES>
struct Smem {
    static constexpr int kStages = ring_stages(HALVES);
    static constexpr int kABytes = kHalf * 128, kBBytes = kN / 2 * 128;       // of one half
    static constexpr int kStageBytes = kABytes + HALVES * kBBytes;
    static constexpr int kData = kStages * kStageBytes;
    static constexpr int kStaging = kEpiWarps * 2048;
    static constexpr int kTable = (2 * (kMaxGroups + 1) * 4 + 7) & ~7;
    static constexpr int kScales = MODE == kRows8 ? kScaleSlots * kScaleSlot * 4 : 0;
    static constexpr int kBars = (3 * kStages + 2 * kAccs + 1 + 2 * kScaleSlots) * 8;
    static constexpr int kTotal = kData + kStaging + kTable + kScales + kBars + 1024;
};

struct Tile {
    int group;       // weight gradient in parts: part * groups + group
    int r0, rows;    // first output row (of the whole output, or of the group's output), rows to store
    int c0, cols;    // first output column, columns to store
    int n;           // accumulator columns, in two halves if more than kTile
    int t0;          // weight gradient: first contraction row
    int depth;       // contraction length
};

// ---- PTX of CTA pairs --------------------------------------------------------------
// Copies into this CTA's shared memory that report to a barrier of either CTA of the pair.
__device__ __forceinline__ void pair_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
        ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ void pair_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}
// The MMAs of a whole ring entry (four; fewer only at the end of the contraction), then the stage's release, and
// for a finished accumulator its hand-over.  Called by a converged warp, issued by one elected lane, in one piece:
// the issue of an entry has to stay below the 512 cycles its MMAs take.  One by one, each with its own election,
// descriptors and loop test, they took 740; from inside `if (lane == 0)` 850.
// STEP_A / STEP_B: descriptor distance (16-byte units) of neighbouring MMAs.
#define BSP_PAIR_MMA(KIND)                                                                                     \
    asm volatile(                                                                                              \
        "{\n\t.reg .pred p, t, e, f, r;\n\t.reg .b64 a, b;\n\t"                                                 \
        "elect.sync _|e, 0xffffffff;\n\t"                                                                     \
        "setp.ne.b32 p, %4, 0;\n\t"                                                                           \
        "setp.ne.and.b32 f, %7, 0, e;\n\t"                                                                    \
        "setp.ne.and.b32 r, %11, 0, e;\n\t"                                                                   \
        "setp.eq.b32 t, 0, 0;\n\t"                                                                            \
        "@e tcgen05.mma.cta_group::2.kind::" KIND " [%0], %1, %2, %3, p;\n\t"                                 \
        "add.s64 a, %1, %8;\n\tadd.s64 b, %2, %9;\n\t"                                                       \
        "@e tcgen05.mma.cta_group::2.kind::" KIND " [%0], a, b, %3, t;\n\t"                                   \
        "add.s64 a, a, %8;\n\tadd.s64 b, b, %9;\n\t"                                                         \
        "@e tcgen05.mma.cta_group::2.kind::" KIND " [%0], a, b, %3, t;\n\t"                                   \
        "add.s64 a, a, %8;\n\tadd.s64 b, b, %9;\n\t"                                                         \
        "@e tcgen05.mma.cta_group::2.kind::" KIND " [%0], a, b, %3, t;\n\t"                                   \
        "@r tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%5], %10;\n\t" \
        "@f tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%6], %10;\n\t}" \
        ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(release_bar), "r"(done_bar),   \
          "r"(done), "n"(STEP_A), "n"(STEP_B), "h"((uint16_t)3), "r"(release) : "memory")
template <bool F8, int STEP_A, int STEP_B>
__device__ __forceinline__ void pair_mma_entry(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                               uint32_t accumulate, uint32_t release_bar, uint32_t release,
                                               uint32_t done_bar, uint32_t done) {
    if (F8) BSP_PAIR_MMA("f8f6f4");
    else BSP_PAIR_MMA("f16");
}
#undef BSP_PAIR_MMA
template <bool F8>
__device__ __forceinline__ void pair_mma(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                         uint32_t accumulate) {
    if (F8)
        asm volatile(
            "{\n\t.reg .pred p, e;\n\t"
            "elect.sync _|e, 0xffffffff;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "@e tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
            ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p, e;\n\t"
            "elect.sync _|e, 0xffffffff;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "@e tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
            ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
// Arrives on the barrier at this offset in both CTAs when the MMAs issued so far are done (converged warp).
__device__ __forceinline__ void pair_commit(uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}"
        ::"r"(bar), "h"((uint16_t)3) : "memory");
}

// 16 bits: the rows of a group are cut into the fewest tiles of at most `most` rows, all of about the same height.
// (The largest m are close to 2^31: m + n - 1 would pass it.)
__device__ __forceinline__ int tile_height(int m, int most) {
    const int n = (m + most - 1) / most;
    return n == 0 ? 0 : round_up((m - 1) / n + 1, 32);
}
// N of either half's MMAs.
__device__ __forceinline__ int half_n(int n, int half) {
    const int first = n <= kTile ? n : round_up(n / 2, 32);
    return half ? n - first : first;
}

// Rows of the copy that brings `share` rows of B.
__device__ __forceinline__ int copied_rows(int share) { return share > 64 ? 128 : share > 32 ? 64 : share > 0 ? 32 : 0; }

// HALVES: accumulators a tile may take (16 bits: 256 or 512 rows; 8 bits: one).
template <int MODE, bool A_MN, int HALVES>
__global__ void __launch_bounds__(kThreads, 1)
grouped_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
               const __grid_constant__ CUtensorMap map_b_64, const __grid_constant__ CUtensorMap map_b_32, const Params p) {
    using L = Smem<MODE, HALVES>;
    constexpr int kHalves = HALVES;
    constexpr int kStages = L::kStages, kStageBytes = L::kStageBytes, kABytes = L::kABytes, kBBytes = L::kBBytes;
    extern __shared__ unsigned char smem_raw[];
    const uint32_t raw = smem_addr(smem_raw);
    const uint32_t data = (raw + 1023u) & ~1023u;
    unsigned char* data_ptr = smem_raw + (data - raw);
    const uint32_t scales = data + L::kData + L::kStaging;
    int* row_start = reinterpret_cast<int*>(data_ptr + L::kData + L::kStaging + L::kScales);   // groups + 1
    int* tile_start = row_start + kMaxGroups + 1;                                              // groups + 1
    const uint32_t bars = scales + L::kScales + L::kTable;
    const uint32_t full_bar = bars, empty_bar = full_bar + 8 * kStages, zeroed_bar = empty_bar + 8 * kStages,
                   tfull_bar = zeroed_bar + 8 * kStages, tempty_bar = tfull_bar + 8 * kAccs,
                   drain_bar = tempty_bar + 8 * kAccs, sfull_bar = drain_bar + 8, sempty_bar = sfull_bar + 8 * kScaleSlots;
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_word;
    __shared__ int issued_stages;
    __shared__ int issued_tails[kStages];
    volatile int* abort_flag = &abort_word;

    constexpr bool F8 = MODE == kRows8;
    constexpr int KE = F8 ? 128 : 64;        // contraction values of a ring entry (128 bytes)
    constexpr int KSTEP = F8 ? 32 : 16;      // contraction values of one MMA
    constexpr bool B_MN = MODE == kGrad16;

    const uint32_t rank = cluster_rank();
    const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    let_next_launch();
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(full_bar + 8 * s, 1);
            mbar_init(empty_bar + 8 * s, 1);
            mbar_init(zeroed_bar + 8 * s, 1);
            issued_tails[s] = 0;
        }
        for (int i = 0; i < kAccs; ++i) {
            mbar_init(tfull_bar + 8 * i, 1);
            mbar_init(tempty_bar + 8 * i, 2 * kEpiWarps);
        }
        mbar_init(drain_bar, 1);
        for (int i = 0; i < kScaleSlots; ++i) {
            mbar_init(sfull_bar + 8 * i, 32);
            mbar_init(sempty_bar + 8 * i, kEpiWarps);
        }
        abort_word = 0;
        issued_stages = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async;" ::: "memory");
    }
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;"
                     ::"r"(smem_addr(&tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    wait_for_previous_launch();
    // group table: clamped offsets, then (warp 0) their running maximum and the tiles before each group
    for (int i = threadIdx.x; i <= p.groups; i += kThreads) {
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
    constexpr int kTileCols = MODE == kRows8 ? kN : kTile;       // of the output
    const int c_tiles = (p.cols + kTileCols - 1) / kTileCols;
    constexpr int tile_rows = HALVES * kTile;
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
        if (MODE != kGrad16) {
            for (int base = 0; base < p.groups; base += 32) {
                const int i = base + lane;
                int n = 0;
                if (i < p.groups) n = (row_start[i + 1] - row_start[i] + tile_rows - 1) / tile_rows * c_tiles;
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
    cluster_sync();      // the other CTA's barriers and tensor memory are ready

    const int r_tiles_all = (p.out_rows + tile_rows - 1) / tile_rows;
    const int n_tiles = uniform(MODE != kGrad16 ? tile_start[p.groups] : p.groups * p.parts * c_tiles * r_tiles_all);
    const int first_tile = blockIdx.x >> 1, tile_step = gridDim.x >> 1;

    auto tile_at = [&](int t) -> Tile {
        Tile o;
        int local, r_tiles;
        if (MODE != kGrad16) {
            int lo = 0, hi = p.groups - 1;          // the last group whose first tile is at or before t
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (tile_start[mid] <= t) lo = mid; else hi = mid - 1;
            }
            o.group = lo;
            local = t - tile_start[lo];
            r_tiles = (row_start[lo + 1] - row_start[lo] + tile_rows - 1) / tile_rows;
        } else {
            r_tiles = r_tiles_all;
            o.group = t / (c_tiles * r_tiles);
            local = t - o.group * c_tiles * r_tiles;
        }
        const int band = local / (kBand * c_tiles);
        const int in_band = min(kBand, r_tiles - band * kBand);
        const int rest = local - band * kBand * c_tiles;
        const int c = rest / in_band, r = band * kBand + rest - c * in_band;
        o.c0 = c * kTileCols;
        o.cols = min(kTileCols, p.cols - o.c0);
        const int g = MODE == kGrad16 ? o.group % p.groups : o.group;
        const int first = row_start[g], m = row_start[g + 1] - first;
        if (MODE == kGrad16) {
            const int h = tile_height(p.out_rows, tile_rows);
            o.r0 = r * h;
            o.rows = min(h, p.out_rows - o.r0);
            // whole ring entries per part, so that only a group's last part may have rows to zero
            const int share = round_up((m + p.parts - 1) / p.parts, KE);
            const int skipped = (int)min((int64_t)(o.group / p.groups) * share, (int64_t)m);
            o.t0 = first + skipped;
            o.depth = min(share, m - skipped);
        } else {
            const int h = MODE == kRows16 ? tile_height(m, tile_rows) : kTile;
            o.r0 = first + r * h;
            o.rows = min(h, m - r * h);
            o.t0 = 0;
            o.depth = p.depth;
        }
        o.n = round_up(MODE == kRows8 ? o.cols : o.rows, 32);
        return o;
    };

    // 8 bits: an epilogue thread holds 128 sums and 32 values on their way from tensor memory.  The warps of
    // the first warpgroup give 112 registers per thread, those of the other two take 56: nothing is left over.
    if (warp < 4) {
        if (F8) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == 0) {
            // ---------------- copies: each CTA its half of either operand ----------------
            if (lane == 0) {
                uint32_t it = 0;
                bool alive = true;
                for (int t = first_tile; t < n_tiles && alive; t += tile_step) {
                    const Tile o = tile_at(t);
                    const int steps = (o.depth + KE - 1) / KE;
                    // rows of B one CTA copies for either half, and their bytes.  One copy of 32, 64 or 128 rows, also where that
                    // brings rows that no accumulator column takes: 96 rows in three copies kept a step at 1100 cycles, 128 in one
                    // let it go at the MMAs' 770.
                    const int share[2] = {half_n(o.n, 0) / 2, half_n(o.n, 1) / 2};
                    int b_bytes = 0;
#pragma unroll
                    for (int h = 0; h < kHalves; ++h)
                        b_bytes += B_MN ? (share[h] + 63) / 64 * 8192 : copied_rows(share[h]) * 128;
                    for (int k = 0; k < steps; ++k, ++it) {
                        const uint32_t s = it % kStages;
                        if (it >= kStages &&
                            !bounded_wait(empty_bar + 8 * s, (it / kStages - 1) & 1, abort_flag, p.status)) {
                            alive = false;
                            break;
                        }
                        const uint32_t a = data + s * kStageBytes, b = a + kABytes;
                        // both halves report to the first CTA's barrier; in a step whose last rows have to be
                        // zeroed the second CTA's half reports to the stage's barrier there, which has no other use
                        const bool split = MODE == kGrad16 && ((o.depth - k * KE) & (KSTEP - 1)) && k == steps - 1;
                        uint32_t bar = map_to_rank(full_bar + 8 * s, 0);
                        issued_stages = (int)it + 1;
                        if (rank == 0) {
                            mbar_arrive_expect_tx(full_bar + 8 * s, (kABytes + b_bytes) * (split ? 1 : 2));
                        } else if (split) {
                            bar = map_to_rank(full_bar + 8 * s, 1);
                            mbar_arrive_expect_tx(full_bar + 8 * s, kABytes + b_bytes);
                            ++issued_tails[s];
                        }
                        if (MODE == kRows8) {
                            pair_load_2d(a, &map_a, k * KE, o.r0 + rank * kHalf, bar);
                        } else if (MODE == kGrad16) {
                            pair_load_2d(a, &map_a, o.c0 + rank * kHalf, o.t0 + k * KE, bar);
                            pair_load_2d(a + 8192, &map_a, o.c0 + rank * kHalf + 64, o.t0 + k * KE, bar);
                        } else if (A_MN) {
                            pair_load_3d(a, &map_a, o.c0 + rank * kHalf, k * KE, o.group, bar);
                            pair_load_3d(a + 8192, &map_a, o.c0 + rank * kHalf + 64, k * KE, o.group, bar);
                        } else {
                            pair_load_3d(a, &map_a, k * KE, o.c0 + rank * kHalf, o.group, bar);
                        }
#pragma unroll
                        for (int h = 0; h < kHalves; ++h) {
                            const uint32_t to = b + h * kBBytes;
                            const int from = (MODE == kRows8 ? o.c0 : o.r0) + (h ? 2 * share[0] : 0) + rank * share[h];
                            if (B_MN) {
                                for (int r = 0; r < share[h]; r += 64) pair_load_2d(to + r * 128, &map_b, from + r, o.t0 + k * KE, bar);
                            } else if (share[h] > 0) {
                                const CUtensorMap* map = share[h] > 64 ? &map_b : share[h] > 32 ? &map_b_64 : &map_b_32;
                                if (MODE == kRows8) pair_load_3d(to, map, k * KE, from, o.group, bar);
                                else pair_load_2d(to, map, k * KE, from, bar);
                            }
                        }
                    }
                }
                // the last arrivals from the first CTA's MMAs land before this CTA may leave
                for (uint32_t i = it > kStages ? it - kStages : 0; i < it && alive; ++i)
                    alive = bounded_wait(empty_bar + 8 * (i % kStages), (i / kStages) & 1, abort_flag, p.status);
            }
            __syncwarp();
        } else if (warp == 1 && (rank == 0 || MODE == kGrad16)) {
            // ---------------- MMAs (first CTA); zeroing of last rows (both) ----------------
            uint32_t it = 0, acc = 0;
            uint32_t tail_parity = 0;       // one bit per stage: uses of its barriers for zeroed rows
            bool alive = true;
            for (int t = first_tile; t < n_tiles && alive; t += tile_step) {
                const Tile o = tile_at(t);
                const int depth = uniform(o.depth), n = uniform(o.n);
                const int steps = (depth + KE - 1) / KE;
                const int halves = kHalves > 1 && n > kTile ? 2 : 1;
                for (int k = 0; k < steps; ++k, ++it) {
                    const uint32_t s = it % kStages;
                    const uint32_t a = data + s * kStageBytes, b = a + kABytes;
                    const int valid = min(KE, depth - k * KE);
                    const int mmas = (valid + KSTEP - 1) / KSTEP;
                    const bool zero_rows = MODE == kGrad16 && (valid & (KSTEP - 1));
                    if (rank == 0) {
                        alive = wait_all(full_bar + 8 * s, (it / kStages) & 1, abort_flag, p.status);
                    } else if (zero_rows) {
                        alive = wait_all(full_bar + 8 * s, (tail_parity >> s) & 1, abort_flag, p.status, &issued_stages);
                    }
                    if (!alive) break;
                    if (zero_rows) {
                        // rows of the next group inside the last 16: zero them in every 64-wide atom
                        const int pieces = (mmas * KSTEP - valid) * 8;     // 16-byte pieces per atom
                        const int atoms = 2 + (half_n(n, 0) / 2 + 63) / 64, more = (half_n(n, 1) / 2 + 63) / 64;
                        for (int atom = 0; atom < atoms + more; ++atom) {
                            const uint32_t dst = (atom < 2 ? a + atom * 8192 : atom < atoms ? b + (atom - 2) * 8192
                                                                                             : b + kBBytes + (atom - atoms) * 8192) + valid * 128;
                            for (int i = lane; i < pieces; i += 32)
                                asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(dst + i * 16), "r"(0) : "memory");
                        }
                        // what is zeroed here is read by this SM's tensor core, in an MMA that the first CTA issues: the
                        // second CTA's zeros pass to the async proxy here and to the first CTA with the arrival (release
                        // at cluster scope; one per group and tile, so its cost does not count)
                        asm volatile("fence.proxy.async;" ::: "memory");
                        __syncwarp();
                        if (rank == 1) {
                            if (lane == 0) mbar_publish_pair(map_to_rank(zeroed_bar + 8 * s, 0));
                        } else {
                            alive = wait_all<true>(zeroed_bar + 8 * s, (tail_parity >> s) & 1, abort_flag, p.status);
                            if (!alive) break;
                        }
                        tail_parity ^= 1u << s;
                    }
                    if (rank == 0) {
                        const uint64_t ad = A_MN ? make_smem_desc(a, 8192, 1024) : make_smem_desc(a, 16, 1024);
                        constexpr int STEP_A = A_MN ? 128 : 2, STEP_B = B_MN ? 128 : 2;
                        const bool done = F8 || k == steps - 1;
                        for (int h = 0; h < halves; ++h) {
                            // a new accumulator: per tile, and for 8-bit operands per step (every step has its own scales)
                            const uint32_t at = acc + h, slot = at % kAccs;
                            if (F8 || k == 0) {
                                alive = at < kAccs || wait_all(tempty_bar + 8 * slot, (at / kAccs - 1) & 1, abort_flag, p.status);
                                if (!alive) break;
                            }
                            tc_fence_after();
                            const uint32_t d = tmem + slot * kN, bh = b + h * kBBytes;
                            const uint32_t idesc = p.idesc | ((uint32_t)(half_n(n, h) >> 3) << 17);
                            const uint64_t bd = B_MN ? make_smem_desc(bh, 8192, 1024) : make_smem_desc(bh, 16, 1024);
                            const bool last = h == halves - 1;
                            if (mmas == 4) {
                                pair_mma_entry<F8, STEP_A, STEP_B>(d, ad, bd, idesc, !F8 && k > 0, empty_bar + 8 * s, last,
                                                                   tfull_bar + 8 * slot, done);
                            } else {
                                for (int kk = 0; kk < mmas; ++kk)
                                    pair_mma<F8>(d, ad + kk * STEP_A, bd + kk * STEP_B, idesc, kk > 0 || (!F8 && k > 0));
                                if (last) pair_commit(empty_bar + 8 * s);
                                if (done) pair_commit(tfull_bar + 8 * slot);
                            }
                        }
                        if (!alive) break;
                        if (done) acc += halves;
                    }
                }
            }
            if (!alive && rank == 0) {
                // the MMAs issued so far finish before tensor memory is given back
                pair_commit(drain_bar);
                bounded_wait(drain_bar, 0, abort_flag, nullptr, false);
            }
            __syncwarp();
        } else if (F8 && warp == 3) {
            // ---------------- scales: this CTA's rows' and the tile's two blocks of w's, steps ahead ----------------
            // Four steps' scales are on their way while those of the four before are looked at: whether a product of theirs may
            // leave fp32's range.  The least and the greatest of either operand's tell (a finer answer for 32 rows and one
            // block of w cost 25 us of 300, and asking in the epilogue 10), and fewer than four steps count as one that may.
            uint32_t at = 0;
            bool alive = true;
            int rows_before = 0, cols_before = 0, steps_before = 0;       // of what is on its way
            auto publish = [&](uint32_t slot) {
                __syncwarp();
                const uint32_t from = scales + slot * kScaleSlot * 4;
                float x_low = 1.0f, x_high = 1.0f, w_low = 1.0f, w_high = 1.0f;
                auto bound = [](float& low, float& high, const float4& v) {
                    low = fminf(fminf(low, fminf(fabsf(v.x), fabsf(v.y))), fminf(fabsf(v.z), fabsf(v.w)));
                    high = fmaxf(fmaxf(high, fmaxf(fabsf(v.x), fabsf(v.y))), fmaxf(fabsf(v.z), fabsf(v.w)));
                };
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (i * 32 + lane < rows_before) bound(x_low, x_high, shared_float4(from + (i * 32 + lane) * 16));
                bound(w_low, w_high, shared_float4(from + kHalf * 16));
                if (cols_before > 128) bound(w_low, w_high, shared_float4(from + kHalf * 16 + 16));
                const bool twice = steps_before < 4 || __any_sync(0xffffffffu, !in_range(x_low * w_low) || !in_range(x_high * w_high));
                if (lane == 0) asm volatile("st.shared.b32 [%0], %1;" ::"r"(from + kScaleFlag), "r"((int)twice) : "memory");
                __syncwarp();
                mbar_arrive(sfull_bar + 8 * slot);
            };
            for (int t = first_tile; t < n_tiles && alive; t += tile_step) {
                const Tile o = tile_at(t);
                const int steps = (o.depth + KE - 1) / KE;
                const int first = (int)rank * kHalf;
                const float* sx = p.scale_x + (int64_t)(o.r0 + first + lane) * p.sx_row;
                const float* sw = p.scale_w + (int64_t)o.group * p.sw_group + (int64_t)(o.c0 / 128 + ((lane >> 2) & 1)) * p.sw_n;
                for (int k = 0; k < steps; k += 4, ++at) {
                    const uint32_t slot = at % kScaleSlots;
                    if (at >= kScaleSlots) alive = wait_all(sempty_bar + 8 * slot, (at / kScaleSlots - 1) & 1, abort_flag, p.status);
                    if (!alive) break;
                    const uint32_t to = scales + slot * kScaleSlot * 4;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (first + i * 32 + lane < o.rows)
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                if (k + j < steps)
                                    copy_async_4(to + (i * 32 + lane) * 16 + j * 4, sx + i * 32 * p.sx_row + (k + j) * p.sx_block);
                    if (lane < 8 && k + (lane & 3) < steps && (lane >> 2) * 128 < o.cols)
                        copy_async_4(to + kHalf * 16 + lane * 4, sw + (k + (lane & 3)) * p.sw_k);
                    asm volatile("cp.async.commit_group;" ::: "memory");
                    if (at > 0) {
                        asm volatile("cp.async.wait_group 1;" ::: "memory");
                        publish((at - 1) % kScaleSlots);
                    }
                    rows_before = o.rows - first;
                    cols_before = o.cols;
                    steps_before = steps - k;
                }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            if (at > 0 && alive) publish((at - 1) % kScaleSlots);
            __syncwarp();
        }
    } else {
        if (F8) asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        // ---------------- epilogue ----------------
        const int quarter = warp & 3, part = (warp - 4) >> 2;
        const uint32_t staging = data + L::kData + (warp - 4) * 2048;
        const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
        const uint32_t tempty_first = map_to_rank(tempty_bar, 0);
        const int esize = p.out_dtype == BSP_F32 ? 4 : 2;
        const int64_t row_bytes = (int64_t)p.cols * esize;
        // rows outside every group are zero
        if (MODE != kGrad16) {
            const int64_t before = row_start[0], behind = row_start[p.groups], pieces = row_bytes / 16;
            const int64_t outside = before + (p.rows - behind);
            for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x - 128; i < outside * pieces; i += (int64_t)gridDim.x * 256) {
                const int64_t r = i / pieces, at = i - r * pieces;
                const int64_t row = r < before ? r : behind + (r - before);
                *reinterpret_cast<int4*>((char*)p.out + row * row_bytes + at * 16) = make_int4(0, 0, 0, 0);
            }
        }
        uint32_t acc = 0, scale_group = 0;
        bool alive = true;
        for (int t = first_tile; t < n_tiles && alive; t += tile_step) {
            const Tile o = tile_at(t);
            const int steps = (o.depth + KE - 1) / KE;
            if (F8) {
                // lane = row of x.  Every step's 128 products per element come back from tensor memory, are
                // multiplied by the step's scale and added up in fp32 registers, 128 columns per thread.
                float sum[128];
#pragma unroll
                for (int j = 0; j < 128; ++j) sum[j] = 0.0f;
                // one step's sums, 32 columns at a time; columns behind n, and rows behind the tile's, hold what came
                // before: they are not stored
                auto each_32_of_step = [&](auto add) {
                    if (!wait_all(tfull_bar + 8 * (acc % kAccs), (acc / kAccs) & 1, abort_flag, p.status)) return false;
                    tc_fence_after();
                    const uint32_t from = lanes + acc % kAccs * kN + part * 128;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t v[32];
                        tc_ld32(from + i * 32, v);
                        tc_wait_ld();
                        if (i == 3) {
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) mbar_arrive_pair(tempty_first + 8 * (acc % kAccs));
                        }
                        add(i, v);
                    }
                    ++acc;
                    return true;
                };
                // the scales of four steps (this row's times the one of these 128 columns), or `twice`: a product may leave
                // fp32's range, and both scales stay where they are for these steps
                float scale[4];
                bool twice = false;
                auto release = [&]() {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(sempty_bar + 8 * (scale_group % kScaleSlots));
                    ++scale_group;
                };
                auto scales_at = [&]() { return scales + scale_group % kScaleSlots * kScaleSlot * 4; };
                auto fetch = [&]() {
                    const uint32_t slot = scale_group % kScaleSlots, from = scales_at();
                    if (!wait_all(sfull_bar + 8 * slot, (scale_group / kScaleSlots) & 1, abort_flag, p.status)) return false;
                    const float4 x = shared_float4(from + (quarter * 32 + lane) * 16), w = shared_float4(from + kHalf * 16 + part * 16);
                    twice = __float_as_int(shared_float(from + kScaleFlag)) != 0;
                    if (!twice) release();
                    scale[0] = x.x * w.x;
                    scale[1] = x.y * w.y;
                    scale[2] = x.z * w.z;
                    scale[3] = x.w * w.w;
                    return true;
                };
                for (int k0 = 0; k0 < steps && alive; k0 += 4) {
                    alive = fetch();
                    if (!alive) break;
                    if (twice) {
                        // (with every step so: 341-371 instead of 304 us)
#pragma unroll 1
                        for (int kk = 0; kk < 4 && k0 + kk < steps && alive; ++kk) {
                            const float2 factors = in_order(shared_float(scales_at() + (quarter * 32 + lane) * 16 + kk * 4),
                                                            shared_float(scales_at() + kHalf * 16 + part * 16 + kk * 4));
                            alive = each_32_of_step([&](int i, const uint32_t* v) {
#pragma unroll
                                for (int j = 0; j < 32; j += 2) add_pair(sum[32 * i + j], sum[32 * i + j + 1], v[j], v[j + 1], factors);
                            });
                        }
                        release();
                        continue;
                    }
#pragma unroll 1
                    for (int kk = 0; kk < 4 && k0 + kk < steps && alive; ++kk) {
                        const float f = kk == 0 ? scale[0] : kk == 1 ? scale[1] : kk == 2 ? scale[2] : scale[3];
                        alive = each_32_of_step([&](int i, const uint32_t* v) {
#pragma unroll
                            for (int j = 0; j < 32; ++j) sum[32 * i + j] = fmaf(__uint_as_float(v[j]), f, sum[32 * i + j]);
                        });
                    }
                }
                if (!alive) break;
                const int first_row = (int)rank * kHalf + quarter * 32, rows = o.rows - first_row;
                char* out = (char*)p.out + (o.r0 + first_row) * row_bytes + (int64_t)(o.c0 + part * 128) * esize;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int left = (o.cols - part * 128 - i * 32) * esize;
                    if (left > 0) {
                        uint32_t words[16];
                        if (p.out_dtype == BSP_F32) {
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
#pragma unroll
                                for (int j = 0; j < 16; ++j) words[j] = __float_as_uint(sum[32 * i + 16 * h + j]);
                                stage_row(staging, words);
                                store_staged(staging, out + i * 128 + h * 64, row_bytes, rows, left - h * 64);
                            }
                        } else {
#pragma unroll
                            for (int j = 0; j < 16; ++j)
                                words[j] = p.out_dtype == BSP_F16 ? pack2<__half>(sum[32 * i + 2 * j], sum[32 * i + 2 * j + 1])
                                                                  : pack2<__nv_bfloat16>(sum[32 * i + 2 * j], sum[32 * i + 2 * j + 1]);
                            stage_row(staging, words);
                            store_staged(staging, out + i * 64, row_bytes, rows, left);
                        }
                    }
                }
            } else {
                // lane = output column
                const int c = o.c0 + (int)rank * kHalf + quarter * 32;
                const int64_t first = MODE == kRows16 ? o.r0 : (int64_t)o.group * p.out_rows + o.r0;
                char* out = (char*)p.out + first * row_bytes + (int64_t)c * esize;
                const int bytes = min(p.cols - c, 32) * 2;
                const bool computed = steps > 0;    // a group without rows has a gradient of zero
#pragma unroll 1
                for (int h = 0; h < kHalves; ++h) {
                    const int n = half_n(o.n, h), above = h ? half_n(o.n, 0) : 0;
                    if (n == 0) break;
                    // first everything out of tensor memory, as packed words, so that the accumulator is free again
                    // (the next tile's MMAs wait for it); then through the staging area into rows.  The sums are fp32 until
                    // here and rounded once, to the type of the operands: what a dense layer of that type returns
                    if (MODE == kGrad16 && HALVES == 1 && p.out_dtype == BSP_F32) {
                        // a part's sums, as they are; a column per lane, 128 bytes of a row per store
                        if (computed) {
                            alive = wait_all(tfull_bar + 8 * (acc % kAccs), (acc / kAccs) & 1, abort_flag, p.status, &issued_stages);
                            if (!alive) break;
                            tc_fence_after();
                        }
#pragma unroll 1
                        for (int c32 = part * 32; c32 < n; c32 += 64) {
                            uint32_t v[32];
                            if (computed) {
                                tc_ld32(lanes + acc % kAccs * kN + c32, v);
                                tc_wait_ld();
                            } else {
#pragma unroll
                                for (int j = 0; j < 32; ++j) v[j] = 0;
                            }
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                if (c32 + j < o.rows && c + lane < p.cols)
                                    *reinterpret_cast<uint32_t*>(out + (c32 + j) * row_bytes + lane * 4) = v[j];
                        }
                        if (computed) {
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) mbar_arrive_pair(tempty_first + 8 * (acc % kAccs));
                            ++acc;
                        }
                        continue;
                    }
                    uint32_t words[4][16];
                    if (computed) {
                        alive = wait_all(tfull_bar + 8 * (acc % kAccs), (acc / kAccs) & 1, abort_flag, p.status, &issued_stages);
                        if (!alive) break;
                        tc_fence_after();
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int c32 = part * 32 + i * 64;
                        if (c32 < n) {
                            uint32_t v[32];
                            if (computed) {
                                const uint32_t from = lanes + acc % kAccs * kN + c32;
                                tc_ld16x32(from, v);
                                tc_ld16x32(from + (16u << 16), v + 16);
                                tc_wait_ld();
                            } else {
#pragma unroll
                                for (int j = 0; j < 32; ++j) v[j] = 0;
                            }
                            const float* f = reinterpret_cast<const float*>(v);
#pragma unroll
                            for (int j = 0; j < 16; ++j)
                                words[i][j] = p.out_dtype == BSP_F16 ? pack2<__half>(f[2 * j], f[2 * j + 1])
                                                                     : pack2<__nv_bfloat16>(f[2 * j], f[2 * j + 1]);
                        }
                    }
                    if (computed) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive_pair(tempty_first + 8 * (acc % kAccs));
                        ++acc;
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int c32 = part * 32 + i * 64;
                        if (c32 < n) {
                            stage_transposed(staging, words[i]);
                            store_staged(staging, out + (above + c32) * row_bytes, row_bytes, o.rows - above - c32, bytes);
                        }
                    }
                }
            }
        }
    }

    // ---------------- teardown ----------------
    tc_fence_before();
    __syncthreads();
    if (abort_word && threadIdx.x == 0) {
        // copies in flight land before the block may leave (the first CTA's barriers cover both halves)
        if (rank == 0) {
            const int last = issued_stages;
            for (int i = last > kStages ? last - kStages : 0; i < last; ++i)
                bounded_wait(full_bar + 8 * (i % kStages), (i / kStages) & 1, abort_flag, nullptr, false);
        } else {
            for (int s = 0; s < kStages; ++s)
                if (issued_tails[s] > 0)
                    bounded_wait(full_bar + 8 * s, (issued_tails[s] - 1) & 1, abort_flag, nullptr, false);
        }
    }
    __syncthreads();
    cluster_sync();      // neither CTA leaves, nor frees tensor memory, while the other may still reach it
    if (warp == 2) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

// Sums of the parts, added up in their order and rounded once.  Four values per thread.
// The launch before writes `sums` while this one may already have started, so they are not declared unchanging
// (__restrict__ would let their loads go ahead of the wait for that launch).
constexpr int kJoinThreads = 128;
template <typename T>
__global__ void __launch_bounds__(kJoinThreads)
join_parts_kernel(const float4* sums, int64_t quads, int parts, uint2* out) {
    let_next_launch();
    wait_for_previous_launch();
    const int64_t i = (int64_t)blockIdx.x * kJoinThreads + threadIdx.x;
    if (i >= quads) return;
    float4 total = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int first = 0; first < parts; first += 8) {
        float4 v[8];         // eight loads under way, the last ones too
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = first + k < parts ? sums[(first + k) * quads + i] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            total.x += v[k].x;
            total.y += v[k].y;
            total.z += v[k].z;
            total.w += v[k].w;
        }
    }
    out[i] = make_uint2(pack2<T>(total.x, total.y), pack2<T>(total.z, total.w));
}

// ---- host side ---------------------------------------------------------------------

template <int MODE, bool A_MN, int HALVES>
int launch(const CUtensorMap& ma, const CUtensorMap (&mb)[3], const Params& p, int64_t most_tiles,
           cudaStream_t stream) {
    auto kern = grouped_kernel<MODE, A_MN, HALVES>;
    static std::atomic<uint64_t> opted_in{0};
    int dev = 0;
    BSP_CUDA_TRY(cudaGetDevice(&dev));
    const uint64_t dev_bit = dev >= 0 && dev < 64 ? (1ull << dev) : 0;
    if (!(opted_in.load(std::memory_order_acquire) & dev_bit)) {
        BSP_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<MODE, HALVES>::kTotal));
        opted_in.fetch_or(dev_bit, std::memory_order_release);
    }
    const int pairs = num_sms() / 2;
    if (pairs <= 0) return BSP_ERR_CUDA;
    const int ctas = 2 * (int)(most_tiles < pairs ? (most_tiles < 1 ? 1 : most_tiles) : pairs);
    return launch_overlapped(kern, dim3(ctas), kThreads, Smem<MODE, HALVES>::kTotal, 2, stream, ma, mb[0], mb[1], mb[2], p);
}

// Tiles of a rows product: a group of m rows has ceil(m / height) <= m / height + 1 row tiles, and no more groups
// than rows have any.
int64_t most_row_tiles(int64_t rows, int64_t groups, int64_t height) {
    return rows / height + (groups < rows ? groups : rows);
}

// Accumulators of a 16-bit tile.  Two: A is staged once for both, 24 KiB per CTA and 512 cycles of MMAs instead of
// 32 (what L2 delivers, about 55 bytes per cycle and SM, is what bounds the ring); one where two would leave the
// pairs fewer than four tiles each, or where the mean group would not fill them (192 rows: 71 / 81 us; 64 groups of
// 64 rows: 53 / 60 us; 33 groups of 60 rows, 1032 x 1496: 34 / 42 us).  Measured, one / two: 16 groups of 1024 rows,
// 2048 x 4096: 215 / 213 us; weight gradient of 8 groups of 2048 rows, 4096 x 4096: 559 / 380 us.
// With all rows in one group, which the host does not see (us, beside the same rows as a group of their own): 64 groups,
// 2048 x 4096, 12288 rows 140 / 144; 8 groups, 4096 x 4096, 3072 rows 73 / 72.
int tile_halves(int64_t tiles_of_two, int64_t rows, int64_t groups) {
    return tiles_of_two >= 4 * (num_sms() / 2) && rows >= 384 * (groups < rows ? groups : rows) ? 2 : 1;
}

// Parts that the rows of every group are split into for the weight gradient, where its tiles leave pairs idle: each
// part of a tile has a pair of its own, leaves its sums in the workspace, and a second launch adds them up.  A step of
// 64 rows takes a pair 0.39 us; a part more costs about 0.08 us per tile (its 256 KiB written and read), so the time
// is least near parts^2 = rows * 0.39 / 64 / (tiles * 0.08).  Measured, one part / parts, us: one group of 256 x 256,
// 1024 rows 12.1 / 9.2, 16384 rows 106 / 15.8; 8 groups, 256 x 256, 1024 rows each 12.5 / 11.4, 4096 rows 31.8 / 15.2;
// 4 groups, 512 x 520, 16384 rows 108 / 47.7.  Below 1024 rows the second launch costs what it saves (8 groups of 512
// rows: 9.3 / 10.4), as it does for parts of fewer than 256.
// The number goes by the mean of the groups.  With all rows in one of them (us, beside the even batch and the same rows as
// a group of their own): 8 groups, 256 x 256, 8192 rows 28 / 12 / 14; 32 groups, 512 x 512, 8192 rows 59 / 12 / 15; 8 groups,
// 2048 x 2048, 4096 rows 44 / 37 / 34.
constexpr int64_t kRowsToSplit = 1024, kPartRows = 256, kPartCost = 13;
int64_t gradient_parts(int64_t rows, int64_t groups, int64_t depth, int64_t cols) {
    const int64_t tiles = groups * ceil_div(depth, kTile) * ceil_div(cols, kTile), fit = num_sms() / 2 / tiles;
    const int64_t mean = rows / (groups < rows ? groups : rows);
    if (mean < kRowsToSplit) return 1;
    int64_t parts = 1;
    while (parts < fit && (parts + 1) * kPartRows <= mean && (parts + 1) * (parts + 1) * tiles * kPartCost <= mean) ++parts;
    return parts;
}

int check_sizes(int64_t rows, int64_t groups, int64_t depth, int64_t cols, const void* offsets) {
    if (rows < 0 || groups < 1 || depth < 1 || cols < 1 || !offsets) return BSP_ERR_INVALID_ARG;
    if (groups > kMaxGroups || rows > 0x7fffffffLL - 512 || depth > 0x7fffffffLL - 512 || cols > 0x7fffffffLL - 512)
        return BSP_ERR_UNSUPPORTED;
    if ((rows / kTile + groups) * ceil_div(cols, 128) > 0x7fffffffLL - 65536) return BSP_ERR_UNSUPPORTED;
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
    CUtensorMap ma, mb[3];
    const int64_t dims[3] = {inner, outer, groups};
    const int64_t strides[2] = {ld_w * 2, (groups > 1 ? group_stride_w : outer * ld_w) * 2};
    const int box[3] = {64, w_cols_inner ? 64 : kHalf, 1};
    if ((st = make_map(&ma, w, dtype, 3, dims, strides, box)) != BSP_OK) return st;
    const bool few = few_applies(rows, groups, cols, false);
    for (int i = few ? 1 : 0; i < 3; ++i)
        if ((st = rows_map(&mb[i], x, dtype, rows, depth, ld_x, 128 >> i)) != BSP_OK) return st;
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
    p.idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | ((w_cols_inner ? 1u : 0u) << 15) | ((uint32_t)(kTile >> 4) << 24);
    p.status = status_word;
    cudaStream_t stream = (cudaStream_t)stream_;
    if (few) {
        p.idesc = (p.idesc & 0x00ffffffu) | (128u >> 4 << 24);
        return launch_few(false, w_cols_inner != 0, ma, mb[1], mb[2], p, stream);
    }
    const int halves = tile_halves(most_row_tiles(rows, groups, 2 * kTile) * ceil_div(cols, kTile), rows, groups);
    const int64_t tiles = most_row_tiles(rows, groups, halves * kTile) * ceil_div(cols, kTile);
    if (w_cols_inner)
        return halves == 2 ? launch<kRows16, true, 2>(ma, mb, p, tiles, stream)
                           : launch<kRows16, true, 1>(ma, mb, p, tiles, stream);
    return halves == 2 ? launch<kRows16, false, 2>(ma, mb, p, tiles, stream)
                       : launch<kRows16, false, 1>(ma, mb, p, tiles, stream);
}

extern "C" int64_t bsp_grouped_weight_grad_workspace(int64_t rows, int64_t groups, int64_t depth, int64_t cols) {
    if (rows < 1 || groups < 1 || depth < 1 || cols < 1 || groups > kMaxGroups || depth > 0x7fffffffLL || cols > 0x7fffffffLL)
        return 0;
    const int64_t parts = gradient_parts(rows, groups, depth, cols);
    return parts > 1 ? parts * groups * depth * cols * 4 : 0;
}

extern "C" int bsp_grouped_weight_grad(const void* x, int64_t ld_x, const void* grad, int64_t ld_grad,
                                       const void* offsets, int offsets_i64, int64_t rows, int64_t groups,
                                       int64_t depth, int64_t cols, void* out, int dtype, void* workspace,
                                       int64_t workspace_bytes, int32_t* status_word, void* stream_) {
    int st = check_sizes(rows, groups, depth, cols, offsets);
    if (st != BSP_OK) return st;
    if (rows < 1) return BSP_ERR_INVALID_ARG;
    if (dtype != BSP_F16 && dtype != BSP_BF16) return BSP_ERR_UNSUPPORTED;
    if (!x || !grad || !out || !aligned16(x) || !aligned16(grad) || !aligned16(out)) return BSP_ERR_INVALID_ARG;
    if ((depth & 7) || (cols & 7) || (ld_x & 7) || (ld_grad & 7) || ld_x < depth || ld_grad < cols)
        return BSP_ERR_INVALID_ARG;
    const int64_t tiles = groups * ceil_div(depth, kTile) * ceil_div(cols, kTile);
    if (tiles > 0x7fffffffLL - 65536) return BSP_ERR_UNSUPPORTED;
    const int parts = (int)gradient_parts(rows, groups, depth, cols);
    if (parts > 1 && (!workspace || !aligned16(workspace) || workspace_bytes < parts * groups * depth * cols * 4))
        return BSP_ERR_INVALID_ARG;
    CUtensorMap ma, mb[3] = {};
    if ((st = rows_map(&ma, grad, dtype, rows, cols, ld_grad, 64)) != BSP_OK) return st;
    if ((st = rows_map(&mb[0], x, dtype, rows, depth, ld_x, 64)) != BSP_OK) return st;
    Params p = {};
    p.offsets = offsets;
    p.offsets_i64 = offsets_i64;
    p.groups = (int)groups;
    p.rows = (int)rows;
    p.cols = (int)cols;
    p.out_rows = (int)depth;
    p.parts = parts;
    p.out = parts > 1 ? workspace : out;
    p.out_dtype = parts > 1 ? BSP_F32 : dtype;
    const uint32_t fmt = dtype == BSP_BF16 ? 1u : 0u;
    p.idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | (1u << 15) | (1u << 16) | ((uint32_t)(kTile >> 4) << 24);
    p.status = status_word;
    cudaStream_t stream = (cudaStream_t)stream_;
    if (parts > 1) {
        if ((st = launch<kGrad16, true, 1>(ma, mb, p, tiles * parts, stream)) != BSP_OK) return st;
        const int64_t quads = groups * depth * cols / 4;
        auto join = dtype == BSP_F16 ? join_parts_kernel<__half> : join_parts_kernel<__nv_bfloat16>;
        return launch_overlapped(join, dim3((unsigned)ceil_div(quads, kJoinThreads)), kJoinThreads, 0, 1, stream,
                                 (const float4*)workspace, quads, parts, (uint2*)out);
    }
    const bool two = tile_halves(groups * ceil_div(depth, 2 * kTile) * ceil_div(cols, kTile), rows, groups) == 2;
    return two ? launch<kGrad16, true, 2>(ma, mb, p, tiles, stream)
               : launch<kGrad16, true, 1>(ma, mb, p, tiles, stream);
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
    CUtensorMap ma, ma_32, mb[3];
    const int64_t dims[3] = {depth, cols, groups};
    const int64_t strides[2] = {ld_w, groups > 1 ? group_stride_w : cols * ld_w};
    const bool few = few_applies(rows, groups, cols, true);
    for (int i = 0; i < (few ? 1 : 3); ++i) {
        const int box[3] = {128, 128 >> i, 1};
        if ((st = make_map(&mb[i], w, type_w, 3, dims, strides, box)) != BSP_OK) return st;
    }
    if ((st = rows_map(&ma, x, type_x, rows, depth, ld_x, few ? 64 : kHalf)) != BSP_OK) return st;
    if (few && (st = rows_map(&ma_32, x, type_x, rows, depth, ld_x, 32)) != BSP_OK) return st;
    Params p = {};
    p.offsets = offsets;
    p.offsets_i64 = offsets_i64;
    p.groups = (int)groups;
    p.rows = (int)rows;
    p.cols = (int)cols;
    p.depth = (int)depth;
    p.out = out;
    p.out_dtype = out_dtype;
    p.idesc = (1u << 4) | ((type_x == BSP_E5M2 ? 1u : 0u) << 7) | ((type_w == BSP_E5M2 ? 1u : 0u) << 10) |
              ((uint32_t)(kTile >> 4) << 24);
    p.scale_x = scale_x;
    p.sx_row = sx_row;
    p.sx_block = sx_block;
    p.scale_w = scale_w;
    p.sw_group = sw_group;
    p.sw_k = sw_k;
    p.sw_n = sw_n;
    p.status = status_word;
    if (few) {
        // the weights are A there
        p.idesc = (1u << 4) | ((type_w == BSP_E5M2 ? 1u : 0u) << 7) | ((type_x == BSP_E5M2 ? 1u : 0u) << 10) |
                  (128u >> 4 << 24);
        return launch_few(true, false, mb[0], ma, ma_32, p, (cudaStream_t)stream_);
    }
    const int64_t tiles = most_row_tiles(rows, groups, kTile) * ceil_div(cols, kN);
    return launch<kRows8, false, 1>(ma, mb, p, tiles, (cudaStream_t)stream_);
}
