// grouped_mm.cu -- one matrix product per expert over ragged row segments, and
// its two gradients, on the 5th-generation tensor cores (tcgen05 + TMEM,
// TMA-fed), sm_100a.  With w [E, N, K] and the rows of segment s belonging to
// expert e = seg_expert[s] (or s):
//   forward  y[r]  = w[e] . x[r]             A = x rows,    B = w[e],    reduced over K
//   dgrad    dx[r] = w[e]^T . dy[r]          A = dy rows,   B = w[e]^T,  reduced over N
//   wgrad    dw[s] = sum_r dy[r] x[r]^T      A = dy^T,      B = x^T,     reduced over the segment's rows
// fp32 accumulation in TMEM, results rounded once to 16 bits.
//
// All three are C[128 x 256] tiles of A . B^T with 64-wide K steps; they
// differ in which operand is stored with the reduced dimension innermost.
// One that is (x and w in the forward) is a K-major tile, as in the expert FFN.  One
// that is not (w in dgrad, both in wgrad) is loaded by TMA as boxes of 64
// consecutive columns x 64 reduced rows and read by the MMA as an MN-major
// operand: no transposed copy of weights or activations is ever made.
//
// One CTA per SM, 7 warps: TMA producer, MMA issuer, 4 epilogue warps (TMEM
// accumulator double-buffered, so the epilogue of one tile runs under the MMAs
// of the next), tile scheduler.  Four forms share the code:
//   few     one SM per 32 x 128 tile: for segments of a few rows, where the
//           time is that of reading the weights and narrow tiles bring more
//           SMs to it; only 32 rows of A are loaded (the MMA's other 96 rows
//           are whatever lies behind them and are not read back)
//   narrow  one SM per 128 x 64 tile: for products of so few wider tiles that
//           most SMs would be idle
//   single  one SM per 128 x 256 tile, 48 KB a K step, 4 stages: for short
//           segments, where a taller tile would be half empty
//   pair    an SM pair (cluster of 2) per 256 x 256 tile: each CTA stages its
//           128 rows of A and half of B, 32 KB a K step, 6 stages.  One SM
//           cannot feed its tensor core at full rate (48 KB are written to and
//           read from shared memory per 512 cycles); a pair can.
// Forward and dgrad tiles cost the same, and a persistent grid deals them
// round-robin.  A wgrad tile costs as much as its segment has rows; there the
// grid is one CTA per tile and running ones take over waiting ones (cluster
// launch control), which balances any routing.
//
// wgrad runs on single SMs (a pair would have to exchange the cleared ends of
// segments).  Its last K step of a segment holds rows of the next segment: the
// MMA warp clears them in shared memory in both operands (so that no infinity
// or NaN there meets a zero) and issues only the 16-row MMAs that hold rows.
//
// The tensor core's queue holds about one K step: the loop of the issuing
// thread has to come around within one MMA (128 cycles), so it does nothing
// but wait, add to descriptors, issue and commit, and it runs under the
// warp's elected thread (see elect_one): a K step of a small tile takes 300
// cycles so, 600 under `lane == 0` (one row, 4096 x 4096: 13.5 us against 22.3).
// Results leave through TMA stores from the swizzled staging tile.  Every wait
// is bounded, as in the expert FFN; those for a whole tile have 64 ns more for each
// index of the sum (a 64-wide K step takes 350 ns: a segment of 360 M rows passes
// the 2 s that a wait has otherwise).
//
// Measured on one B200, bf16, back to back (the power limit holds the SM clock
// near 1.2 to 1.4 GHz then, and cuBLAS at 1340 TFLOP/s for one product of this
// size): 60 even segments of 1024 rows, 2816 x 2048: forward 570 to 610 us (1160
// to 1240 TFLOP/s), dgrad 590, wgrad 695 (1020); 65536 Zipf-routed rows: 665,
// 660, 813.
// wgrad of 128 short segments (7992 rows, 712 x 1096), 79 us, writes 200 MB at
// 2.5 TB/s; a plain fill of memory reaches 3.9 TB/s on this card.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "common.cuh"
#include "gemm_epilogue.cuh"
#include "per_device.cuh"
#include "tcgen05.cuh"

namespace moe_b200 {

int fail(int code, const char* fmt, ...);
int cuda_fail(cudaError_t err, const char* where);

enum { kMmForward = 0, kMmDgrad = 1, kMmWgrad = 2 };

constexpr int kMmTileK = 64;
constexpr int kMmThreads = 7 * 32;
constexpr uint32_t kMmBoxBytes = 64 * 64 * 2;            // one MN-major box: 64 columns x 64 reduced rows
constexpr uint32_t kMmTmemCols = 512;
constexpr int kMmBufCols = 256;                          // TMEM columns of one accumulator
constexpr int kMmMaxSegments = 1024;
constexpr int kMmMaxSize = INT32_MAX - 4095;             // rows, N, K: indices that run past a tile's end stay 32-bit
constexpr int kSchedSlots = 4;
enum { kMmFew = 0, kMmSingle = 1, kMmPair = 2, kMmNarrow = 3 };
template <int FORM> struct MmGeo {
    static constexpr int kCtas = FORM == kMmPair ? 2 : 1;
    static constexpr int kTileM = FORM == kMmFew ? 32 : 128;  // rows of A per CTA
    static constexpr int kTileN = FORM == kMmNarrow ? 64 : FORM == kMmFew ? 128 : 256;
    static constexpr int kBlockRows = kTileM * kCtas;         // rows per tile
    static constexpr int kBCols = kTileN / kCtas;             // columns of B a CTA holds
    static constexpr uint32_t kABytes = kTileM * kMmTileK * 2;
    static constexpr uint32_t kBBytes = kBCols * kMmTileK * 2;
    static constexpr uint32_t kStageBytes = kABytes + kBBytes;
    static constexpr int kStages =                            // 180 or 192 KB
        FORM == kMmFew ? 9 : FORM == kMmNarrow ? 8 : FORM == kMmSingle ? 4 : 6;
};
constexpr int kMmMaxStages = 9;

struct MmSmem {
    uint64_t full[kMmMaxStages];
    uint64_t empty[kMmMaxStages];
    uint64_t tmem_full[2];
    uint64_t tmem_empty[2];
    uint64_t sched_full[kSchedSlots];
    uint64_t sched_empty[kSchedSlots];
    uint64_t clc_full;  // answers of cluster launch control
    uint64_t drained;   // after a wait gave up: the MMAs in flight are through
    uint4 clc;
    int next[kSchedSlots];  // tiles handed to the warps
    uint32_t tmem_base;
    int abort_flag;
    int total_blocks;
};

struct MmArgs {
    const int32_t* seg_start;
    const int32_t* seg_expert;
    int nseg, rows, experts;
    int kdim;      // reduced length (forward, dgrad)
    int m_blocks;  // wgrad: row blocks of dw
    int n_blocks;  // column blocks of the output
    int m_out;     // wgrad: rows of dw per expert
    int n_out;     // output columns
    uint16_t* out;
    uint32_t* status;
};

// Shared-memory descriptor of an MN-major operand, 128-byte swizzle: rows of
// 128 bytes hold 64 consecutive columns of one reduced index, 8 reduced
// indices are 1024 bytes (stride offset), the next 64 columns lie one box
// further (leading offset).
__device__ __forceinline__ uint64_t umma_desc_mn_sw128(uint32_t smem_addr) {
    uint64_t d = 0;
    d |= uint64_t((smem_addr >> 4) & 0x3FFF);
    d |= uint64_t(kMmBoxBytes >> 4) << 16;
    d |= uint64_t(1024 >> 4) << 32;
    d |= uint64_t(1) << 46;
    d |= uint64_t(2) << 61;
    return d;
}

__device__ __forceinline__ void tma_load_3d(void* smem_dst, const CUtensorMap* map, int x, int y, int z,
                                            uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(smem_dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
        : "memory");
}

// Asks the hardware for a CTA of this grid that has not started; the 16-byte
// answer arrives in shared memory.
__device__ __forceinline__ void clc_try_cancel(uint4* response, uint64_t* bar) {
    asm volatile(
        "clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
            smem_u32(response)),
        "r"(smem_u32(bar))
        : "memory");
}
// blockIdx.x of the CTA taken over, or -1 when none was left.
__device__ __forceinline__ int clc_result(const uint4* response) {
    uint32_t ok, x;
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b128 r;\n\t"
        "ld.shared.b128 r, [%2];\n\t"
        "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t"
        "mov.u32 %1, 0;\n\t"
        "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, r;\n\t}"
        : "=r"(ok), "=r"(x)
        : "r"(smem_u32(response))
        : "memory");
    return ok ? int(x) : -1;
}

// Completion of this thread's MMAs arrives on the barrier at this offset in
// both CTAs of the pair.
__device__ __forceinline__ void umma_commit_both(uint64_t* bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_u32(bar)),
        "h"(uint16_t(3))
        : "memory");
}
__device__ __forceinline__ void tma_load_3d_pair(void* smem_dst, const CUtensorMap* map, int x, int y, int z,
                                                uint32_t cluster_bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(smem_dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(cluster_bar)
        : "memory");
}

// Tiled TMA store of a staged box; its elements past the tensor's bounds are not written.
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, const void* smem_src, int x, int y, int z) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(
                     reinterpret_cast<uint64_t>(map)),
                 "r"(x), "r"(y), "r"(z), "r"(smem_u32(smem_src))
                 : "memory");
}

// Clears the reduced rows [from, to), 128 bytes each, of `boxes` MN-major boxes at `base`, by one warp.
__device__ __forceinline__ void clear_rows(uint32_t base, int boxes, int from, int to, int lane) {
    const int n = to - from;
    for (int i = lane; i < n * 8 * boxes; i += 32) {
        const int box = i / (n * 8), r = (i >> 3) % n, c = i & 7;
        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(base + box * kMmBoxBytes + (from + r) * 128 + c * 16),
                     "r"(0)
                     : "memory");
    }
}

template <int MODE, int DT, int FORM>
__global__ void __launch_bounds__(kMmThreads, 1)
grouped_mm_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                  const __grid_constant__ CUtensorMap tmap_c, const MmArgs a) {
    constexpr bool kDynamic = MODE == kMmWgrad;
    using GEO = MmGeo<FORM>;
    constexpr int CG = GEO::kCtas, kStages = GEO::kStages, kMmTileN = GEO::kTileN;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* base = reinterpret_cast<unsigned char*>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    unsigned char* sA = base;  // [stages][A, B]: B follows A, so a stage's boxes are consecutive
    constexpr uint32_t kStage = GEO::kStageBytes;
    unsigned char* s_stage = base + kStages * kStage;
    MmSmem* ctl = reinterpret_cast<MmSmem*>(s_stage + kStageBytes);
    int32_t* blk_prefix = reinterpret_cast<int32_t*>(ctl + 1);  // [nseg + 1] row blocks before a segment
    int32_t* s_start = blk_prefix + (a.nseg + 1);               // [nseg] first row
    int32_t* s_rows = s_start + a.nseg;                         // [nseg] rows
    int32_t* s_exp = s_rows + a.nseg;                           // [nseg] expert

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile int* abort_flag = &ctl->abort_flag;
    const uint64_t tile_limit = kWaitLimitNs + uint64_t(MODE == kMmWgrad ? a.rows : a.kdim) * 64;
    // Pair coordinates: rank 0 is the leader, which issues the MMAs and finds the tiles.
    const uint32_t crank = CG == 2 ? cluster_rank() : 0u;
    const int tile0 = CG == 2 ? int(cluster_id_x()) : int(blockIdx.x);
    const int tile_step = CG == 2 ? int(num_clusters_x()) : int(gridDim.x);

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&ctl->full[s], 1);
            mbar_init(&ctl->empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&ctl->tmem_full[b], 1);
            mbar_init(&ctl->tmem_empty[b], 4 * CG);
        }
        for (int b = 0; b < kSchedSlots; ++b) {
            mbar_init(&ctl->sched_full[b], 1);
            mbar_init(&ctl->sched_empty[b], 7);  // one arrival per warp
        }
        mbar_init(&ctl->clc_full, 1);
        mbar_init(&ctl->drained, 1);
        ctl->abort_flag = 0;
        mbar_fence_init();
        prefetch_tmap(&tmap_a);
        prefetch_tmap(&tmap_b);
        prefetch_tmap(&tmap_c);
    }
    if (warp == 0) {
        // Offsets are held ascending inside [0, rows]: no bad table leads a
        // store outside the output or makes more tiles than the host counted.
        int run = 0, reached = 0;
        for (int s0 = 0; s0 < a.nseg; s0 += 32) {
            const int i = s0 + lane;
            int cnt = 0;
            int lo = i < a.nseg ? min(max(a.seg_start[i], 0), a.rows) : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, lo, o);
                if (lane >= o) lo = max(lo, v);
            }
            lo = max(lo, reached);
            const int hi = i < a.nseg ? max(min(a.seg_start[i + 1], a.rows), lo) : lo;
            reached = __shfl_sync(0xffffffffu, hi, 31);
            if (i < a.nseg) {
                s_start[i] = lo;
                s_rows[i] = hi - lo;
                const int e = a.seg_expert ? a.seg_expert[i] : i;
                s_exp[i] = e >= 0 && e < a.experts ? e : -1;
                cnt = (s_rows[i] + GEO::kBlockRows - 1) / GEO::kBlockRows;
            }
            int incl = cnt;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += v;
            }
            if (i < a.nseg) blk_prefix[i] = run + incl - cnt;
            run += __shfl_sync(0xffffffffu, incl, 31);
        }
        if (lane == 0) {
            blk_prefix[a.nseg] = run;
            ctl->total_blocks = run;
        }
    }
    if (warp == 1) {
        if (CG == 1) {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                             smem_u32(&ctl->tmem_base)),
                         "r"(kMmTmemCols)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                             smem_u32(&ctl->tmem_base)),
                         "r"(kMmTmemCols)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        }
    }
    tc_fence_before();
    __syncthreads();
    if (CG == 2) cluster_sync();  // both CTAs' barriers initialised before any cross-CTA signal
    tc_fence_after();

    const uint32_t tmem = ctl->tmem_base;
    const int total_tiles = MODE == kMmWgrad ? a.nseg * a.m_blocks * a.n_blocks : ctl->total_blocks * a.n_blocks;
    const int first_tile = tile0 < total_tiles ? tile0 : -1;

    // The tile after `tile`, or -1.  Called by whole warps.
    uint32_t sidx = 0;
    auto next_tile = [&](int tile) -> int {
        if (!kDynamic) {
            const int n = tile + tile_step;
            return n < total_tiles && !__any_sync(0xffffffffu, *abort_flag) ? n : -1;
        }
        const int slot = int(sidx % kSchedSlots);
        const bool ok = wait_or_abort(&ctl->sched_full[slot], (sidx / kSchedSlots) & 1u, abort_flag, a.status, tile_limit);
        const int n = ok ? *const_cast<volatile int*>(&ctl->next[slot]) : -1;
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl->sched_empty[slot]);
        ++sidx;
        return __all_sync(0xffffffffu, ok) ? n : -1;
    };
    // Segment, row block, column block and K steps of a tile.
    auto locate = [&](int tile, int& s, int& m, int& n) -> int {
        if (MODE == kMmWgrad) {
            n = tile % a.n_blocks;
            const int g = tile / a.n_blocks;
            m = g % a.m_blocks;
            s = g / a.m_blocks;
            return (s_rows[s] + kMmTileK - 1) / kMmTileK;
        }
        const int g = tile / a.n_blocks;
        n = tile % a.n_blocks;
        s = find_segment(blk_prefix, a.nseg, g);
        m = g - blk_prefix[s];
        // No expert: no steps, and the epilogue writes zeros.  (Weights that read
        // as zeros would not do: a NaN or infinity in the rows would meet them.)
        return s_exp[s] < 0 ? 0 : (a.kdim + kMmTileK - 1) / kMmTileK;
    };
    const uint32_t leader_full0 = CG == 2 ? map_to_rank(&ctl->full[0], 0) : 0u;

    if (warp == 0) {
        // ---------------- TMA producer ----------------
        uint32_t it = 0;
        int leader = 0;
        for (int tile = first_tile; tile >= 0; tile = next_tile(tile)) {
            int s, m, n;
            const int nk = locate(tile, s, m, n);
            if (elect_one(leader)) {
                const int e = s_exp[s], row0 = s_start[s];
                const int a0 = m * GEO::kBlockRows + int(crank) * GEO::kTileM;    // rows of A (wgrad: columns of dy)
                const int b0 = n * kMmTileN + int(crank) * GEO::kBCols;        // columns of the output
                // A pair's second half past the segment reads zeros from beyond the
                // tensor instead of other segments' rows: no traffic, and less power.
                const int a_row = CG == 1 || a0 < s_rows[s] ? row0 + a0 : a.rows;
                for (int kb = 0; kb < nk; ++kb, ++it) {
                    const int st = int(it % kStages);
                    if (!wait_or_abort(&ctl->empty[st], ((it / kStages) & 1u) ^ 1u, abort_flag, a.status)) break;
                    unsigned char* pa = sA + st * kStage;
                    unsigned char* pb = pa + GEO::kABytes;
                    const int k0 = kb * kMmTileK;
                    if (CG == 1) {
                        uint64_t* bar = &ctl->full[st];
                        mbar_arrive_expect_tx(bar, kStage);
                        if (MODE == kMmWgrad) {
                            for (int i = 0; i < GEO::kTileM / 64; ++i)
                                tma_load_2d(pa + i * kMmBoxBytes, &tmap_a, a0 + i * 64, row0 + k0, bar);
                            for (int i = 0; i < GEO::kBCols / 64; ++i)
                                tma_load_2d(pb + i * kMmBoxBytes, &tmap_b, b0 + i * 64, row0 + k0, bar);
                        } else {
                            tma_load_2d(pa, &tmap_a, k0, a_row, bar);
                            if (MODE == kMmForward) {
                                tma_load_3d(pb, &tmap_b, k0, b0, e, bar);
                            } else {
                                for (int i = 0; i < GEO::kBCols / 64; ++i)
                                    tma_load_3d(pb + i * kMmBoxBytes, &tmap_b, b0 + i * 64, k0, e, bar);
                            }
                        }
                    } else {
                        // Both CTAs' bytes land on the leader's barrier.
                        const uint32_t bar = leader_full0 + uint32_t(st) * 8u;
                        if (crank == 0) mbar_arrive_expect_tx(&ctl->full[st], 2 * kStage);
                        tma_load_2d_pair(pa, &tmap_a, k0, a_row, bar);
                        if (MODE == kMmForward) {
                            tma_load_3d_pair(pb, &tmap_b, k0, b0, e, bar);
                        } else {
                            for (int i = 0; i < GEO::kBCols / 64; ++i)
                                tma_load_3d_pair(pb + i * kMmBoxBytes, &tmap_b, b0 + i * 64, k0, e, bar);
                        }
                    }
                }
            }
            __syncwarp();
        }
        // (the pair's loads complete on the leader's barriers; the last cluster
        // barrier keeps the peer resident until the leader has drained them)
        if (lane == leader && crank == 0 && *abort_flag) drain_stages(ctl->full, it, kStages);
    } else if (warp == 1) {
        // ---------------- MMA issuer (the pair's leader) ----------------
        // Bits 15 / 16 of the instruction descriptor: A / B is MN-major.
        const uint32_t idesc = umma_idesc_mn(DT == MOE_B200_BF16 ? 1 : 0, 128 * CG, kMmTileN) |
                               (MODE == kMmWgrad ? 1u << 15 : 0u) | (MODE != kMmForward ? 1u << 16 : 0u);
        // Descriptor steps (16-byte units) per 16 reduced indices and per stage.
        constexpr uint32_t a_step = (MODE == kMmWgrad ? 2048 : 32) >> 4, b_step = (MODE != kMmForward ? 2048 : 32) >> 4;
        constexpr uint32_t stage_step = kStage >> 4;
        const uint64_t adesc0 = MODE == kMmWgrad ? umma_desc_mn_sw128(smem_u32(sA)) : umma_desc_sw128(smem_u32(sA));
        const uint64_t bdesc0 = MODE != kMmForward ? umma_desc_mn_sw128(smem_u32(sA) + GEO::kABytes)
                                                   : umma_desc_sw128(smem_u32(sA) + GEO::kABytes);
        int st = 0;
        uint32_t phase = 0, j = 0;
        bool ok = crank == 0;
        int leader = 0;
        auto issue = [&](uint32_t d_tmem, int kk, uint32_t acc) {
            const uint64_t ad = adesc0 + uint32_t(st) * stage_step + uint32_t(kk) * a_step;
            const uint64_t bd = bdesc0 + uint32_t(st) * stage_step + uint32_t(kk) * b_step;
            if (CG == 1) umma_f16(d_tmem, ad, bd, idesc, acc);
            else umma_f16_pair(d_tmem, ad, bd, idesc, acc);
        };
        auto commit = [&](uint64_t* bar) {
            if (CG == 1) umma_commit(bar);
            else umma_commit_both(bar);
        };
        auto next_stage = [&]() {
            if (++st == kStages) st = 0, phase ^= 1;
        };
        for (int tile = first_tile; ok && tile >= 0; tile = next_tile(tile)) {
            int s, m, n;
            const int nk = locate(tile, s, m, n);
            if (nk == 0) continue;  // an empty segment or no expert: the epilogue writes zeros
            const int buf = int(j & 1u);
            const int rem = MODE == kMmWgrad ? s_rows[s] % kMmTileK : 0;  // rows of a last, partial step
            const int nfull = nk - (rem > 0 ? 1 : 0);
            const uint32_t d_tmem = tmem + uint32_t(buf) * kMmBufCols;
            if (elect_one(leader)) {
                ok = wait_or_abort(&ctl->tmem_empty[buf], ((j >> 1) & 1u) ^ 1u, abort_flag, a.status, tile_limit);
                tc_fence_after();
                for (int kb = 0; ok && kb < nfull; ++kb) {
                    ok = wait_or_abort(&ctl->full[st], phase, abort_flag, a.status);
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll
                    for (int kk = 0; kk < kMmTileK / 16; ++kk) issue(d_tmem, kk, (kb | kk) != 0 ? 1u : 0u);
                    commit(&ctl->empty[st]);
                    next_stage();
                }
            }
            ++j;
            if (MODE == kMmWgrad) {
                ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, leader) != 0;
                st = __shfl_sync(0xffffffffu, st, leader);
                phase = __shfl_sync(0xffffffffu, phase, leader);
                if (ok && rem > 0) {
                    ok = __all_sync(0xffffffffu, wait_or_abort(&ctl->full[st], phase, abort_flag, a.status));
                    if (ok) {
                        const int k16 = (rem + 15) / 16;
                        clear_rows(smem_u32(sA) + st * kStage, int(kStage / kMmBoxBytes), rem, k16 * 16, lane);
                        fence_proxy_async_smem();
                        __syncwarp();
                        tc_fence_after();
                        if (lane == leader) {  // (elect_one costs the few MMAs more than it saves: 81 us against 79 ragged)
                            for (int kk = 0; kk < k16; ++kk) issue(d_tmem, kk, (nfull | kk) != 0 ? 1u : 0u);
                            commit(&ctl->empty[st]);
                        }
                        next_stage();
                    }
                }
            }
            ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, leader) != 0;
            if (ok && elect_one(leader)) commit(&ctl->tmem_full[buf]);
        }
    } else if (warp < 6) {
        // ---------------- epilogue (warps 2..5) ----------------
        const int quad = warp & 3;  // TMEM lanes 32*quad .. 32*quad+31
        unsigned char* stg = s_stage + quad * kWarpStageBytes;
        const uint32_t leader_tmem_empty0 = CG == 2 ? map_to_rank(&ctl->tmem_empty[0], 0) : 0u;
        uint32_t j = 0;
        for (int tile = first_tile; tile >= 0; tile = next_tile(tile)) {
            int s, m, n;
            const int nk = locate(tile, s, m, n);
            const int w_row0 = m * GEO::kBlockRows + int(crank) * GEO::kTileM + quad * 32;
            // Of a 32-row tile only the first warp has rows; behind them lie the next tile's.
            const int nrows_w = quad * 32 < GEO::kTileM ? (MODE == kMmWgrad ? a.m_out : s_rows[s]) - w_row0 : 0;
            const int64_t out_row = (MODE == kMmWgrad ? int64_t(s) * a.m_out : int64_t(s_start[s])) + w_row0;
            uint16_t* dst = a.out + out_row * a.n_out;
            // The staged 32 x 64 piece has the layout of a 128-byte-swizzled TMA
            // box: one store instruction writes it.  Only a segment's last rows
            // (forward, dgrad), behind which other segments' rows lie, are
            // written by the lanes; dw ends with its tensor map.
            const bool by_tma = MODE == kMmWgrad || nrows_w >= 32;
            const int buf = int(j & 1u);
            if (nk > 0) {
                const bool ok = wait_or_abort(&ctl->tmem_full[buf], (j >> 1) & 1u, abort_flag, a.status, tile_limit);
                if (!__all_sync(0xffffffffu, ok)) break;
                ++j;
                tc_fence_after();
            }
            const uint32_t t_row = tmem + uint32_t(buf) * kMmBufCols + (uint32_t(quad * 32) << 16);
#pragma unroll 1
            for (int c = 0; c < kMmTileN; c += 64) {
                if (n * kMmTileN + c >= a.n_out || nrows_w <= 0) break;
                uint32_t v[4][16];
                if (nk > 0) {
#pragma unroll
                    for (int q4 = 0; q4 < 4; ++q4) tmem_ld16(t_row + c + 16 * q4, v[q4]);
                    tmem_wait_ld();
                } else {
#pragma unroll
                    for (int q4 = 0; q4 < 4; ++q4)
#pragma unroll
                        for (int q = 0; q < 16; ++q) v[q4][q] = 0;
                }
                if (lane == 0) bulk_wait_read<0>();  // the piece before is read
                __syncwarp();
#pragma unroll
                for (int q4 = 0; q4 < 4; ++q4) {
                    uint32_t o[8];
#pragma unroll
                    for (int q = 0; q < 8; ++q)
                        o[q] = pack2<DT>(__uint_as_float(v[q4][2 * q]), __uint_as_float(v[q4][2 * q + 1]));
                    stage_put(stg, lane, 2 * q4, make_uint4(o[0], o[1], o[2], o[3]));
                    stage_put(stg, lane, 2 * q4 + 1, make_uint4(o[4], o[5], o[6], o[7]));
                }
                if (by_tma) {
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        tma_store_3d(&tmap_c, stg, n * kMmTileN + c, MODE == kMmWgrad ? w_row0 : int(out_row),
                                     MODE == kMmWgrad ? s : 0);
                        bulk_commit();
                    }
                } else {
                    stage_flush(stg, lane, dst, a.n_out, nrows_w, n * kMmTileN + c, a.n_out, nullptr);
                }
            }
            if (nk > 0) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (CG == 1) mbar_arrive(&ctl->tmem_empty[buf]);
                    else mbar_arrive_cluster(leader_tmem_empty0 + uint32_t(buf) * 8u);
                }
            }
        }
        if (lane == 0) bulk_wait<0>();
    } else if (kDynamic) {
        // ---------------- tile scheduler (warp 6) ----------------
        // Keeps the slots filled ahead of the other warps and stops after the
        // first answer that names no CTA.
        int tile = first_tile;
        uint32_t asked = 0;
        while (tile >= 0) {
            const int slot = int(sidx % kSchedSlots);
            bool ok = wait_or_abort(&ctl->sched_empty[slot], ((sidx / kSchedSlots) & 1u) ^ 1u, abort_flag, a.status, tile_limit);
            if (!__all_sync(0xffffffffu, ok)) break;
            if (lane == 0) {
                mbar_arrive_expect_tx(&ctl->clc_full, 16);
                clc_try_cancel(&ctl->clc, &ctl->clc_full);
            }
            __syncwarp();
            ok = wait_or_abort(&ctl->clc_full, asked & 1u, abort_flag, a.status);
            if (!__all_sync(0xffffffffu, ok)) {
                mbar_wait(&ctl->clc_full, asked & 1u);  // the answer still in flight has landed
                break;
            }
            ++asked;
            const int next = clc_result(&ctl->clc);
            fence_proxy_async_smem();  // the answer is read before the next one is written
            __syncwarp();
            if (lane == 0) {
                *const_cast<volatile int*>(&ctl->next[slot]) = next;
                mbar_arrive(&ctl->sched_full[slot]);
            }
            __syncwarp();
            tile = next_tile(tile);
        }
    }

    tc_fence_before();
    __syncthreads();
    // After a wait gave up nobody has waited for the last MMAs, which must not
    // run into the TMEM and shared memory of the next CTA.
    if (warp == 1 && crank == 0 && *abort_flag) {
        int issuer;
        if (elect_one(issuer)) {
            if (CG == 1) umma_commit(&ctl->drained);
            else umma_commit_both(&ctl->drained);
            mbar_wait(&ctl->drained, 0);
        }
        __syncwarp();
    }
    if (CG == 2) cluster_sync();  // no CTA leaves while its pair may still signal it
    tc_fence_after();
    if (warp == 1) {
        __syncwarp();
        if (CG == 1)
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kMmTmemCols)
                         : "memory");
        else
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kMmTmemCols)
                         : "memory");
    }
}

// ----------------------------------------------------------------- host ----

// 3-D map over w [E, N, K] 16-bit; box = 64 columns x box_rows rows of one expert, 128B swizzle.
static bool make_map_experts(CUtensorMap* map, const void* base, int64_t experts, int64_t rows, int64_t cols,
                             int box_rows, int dtype) {
    const cuuint64_t dims[3] = {cuuint64_t(cols), cuuint64_t(rows), cuuint64_t(experts)};
    const cuuint64_t strides[2] = {cuuint64_t(cols) * 2, cuuint64_t(cols) * cuuint64_t(rows) * 2};
    const cuuint32_t box[3] = {64u, cuuint32_t(box_rows), 1u};
    return encode_tiled(map, map_type(dtype), 3, base, dims, strides, box);
}

template <int MODE, int DT, int FORM>
static cudaError_t launch_mm(const CUtensorMap& ma, const CUtensorMap& mb, const CUtensorMap& mc, MmArgs a,
                             cudaStream_t s) {
    using GEO = MmGeo<FORM>;
    constexpr int CG = GEO::kCtas;
    auto kern = grouped_mm_kernel<MODE, DT, FORM>;
    const size_t smem = 1024 + size_t(GEO::kStages) * GEO::kStageBytes + kStageBytes + sizeof(MmSmem) +
                        size_t(4 * a.nseg + 1) * 4;
    static SmemLimit limit;
    const cudaError_t err = limit.open(reinterpret_cast<const void*>(kern));
    if (err != cudaSuccess) return err;
    a.m_blocks = (a.m_out + GEO::kBlockRows - 1) / GEO::kBlockRows;
    a.n_blocks = (a.n_out + GEO::kTileN - 1) / GEO::kTileN;
    cudaLaunchConfig_t cfg = pdl_config(dim3(1), dim3(kMmThreads), smem, s);
    cudaLaunchAttribute attr[1];
    if (CG == 2) {
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = 2;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
    }
    int64_t groups;
    if (MODE == kMmWgrad) {
        groups = int64_t(a.nseg) * a.m_blocks * a.n_blocks;
    } else {
        groups = (int64_t(a.rows) / GEO::kBlockRows + a.nseg) * a.n_blocks;  // a segment may add one partial block
        int fit = device_sm_count() / CG;
        if (CG == 2) {  // not every SM has a partner: a pair left waiting would run its share behind all others
            static DeviceCount pairs;
            const int n = pairs.get([&] {
                int most = 0;
                cfg.gridDim = dim3(unsigned(2 * fit));
                if (cudaOccupancyMaxActiveClusters(&most, kern, &cfg) != cudaSuccess || most < 1) most = fit;
                cudaGetLastError();
                return most;
            });
            if (n < fit) fit = n;
        }
        if (groups > fit) groups = fit;
    }
    cfg.gridDim = dim3(unsigned(CG * groups));
    return cudaLaunchKernelEx(&cfg, kern, ma, mb, mc, a);
}

template <int MODE>
static cudaError_t launch_mm_as(int dtype, int form, const CUtensorMap& ma, const CUtensorMap& mb,
                                const CUtensorMap& mc, const MmArgs& a, cudaStream_t s) {
    const bool bf = dtype == MOE_B200_BF16;
    if constexpr (MODE != kMmWgrad) {
        if (form == kMmPair)
            return bf ? launch_mm<MODE, MOE_B200_BF16, kMmPair>(ma, mb, mc, a, s)
                      : launch_mm<MODE, MOE_B200_F16, kMmPair>(ma, mb, mc, a, s);
        if (form == kMmFew)
            return bf ? launch_mm<MODE, MOE_B200_BF16, kMmFew>(ma, mb, mc, a, s)
                      : launch_mm<MODE, MOE_B200_F16, kMmFew>(ma, mb, mc, a, s);
        if (form == kMmNarrow)
            return bf ? launch_mm<MODE, MOE_B200_BF16, kMmNarrow>(ma, mb, mc, a, s)
                      : launch_mm<MODE, MOE_B200_F16, kMmNarrow>(ma, mb, mc, a, s);
    }
    return bf ? launch_mm<MODE, MOE_B200_BF16, kMmSingle>(ma, mb, mc, a, s)
              : launch_mm<MODE, MOE_B200_F16, kMmSingle>(ma, mb, mc, a, s);
}

// Rows a tile loads and columns of its B that a CTA loads.
static int form_rows(int form) { return form == kMmFew ? MmGeo<kMmFew>::kTileM : MmGeo<kMmSingle>::kTileM; }
static int form_cols(int form) {
    return form == kMmFew      ? MmGeo<kMmFew>::kBCols
           : form == kMmNarrow ? MmGeo<kMmNarrow>::kBCols
           : form == kMmPair   ? MmGeo<kMmPair>::kBCols
                               : MmGeo<kMmSingle>::kBCols;
}

// The form of forward and dgrad, from what the host knows.  Measured on one
// B200, bf16, in captured graphs, us of forward / dgrad:
//  few     segments of at most 16 rows on average.  60 experts of 1408 x 2048,
//          15 rows: even 59 / 59 against 65 / 62 as single tiles, Zipf 61 / 61
//          against 64 / 60; 20 rows: even 61 / 60 against 67 / 64, Zipf 70 / 67
//          against 64 / 61; 40 rows: even 78 / 81 against 66 / 63.  4 experts of
//          2816 x 1024, 16 rows: 8.3 / 12.7 against 11.2 / 12.0 as narrow tiles.
//          (All 900 rows on one of the 60 experts: 23 / 23 against 16 / 13.)
//  narrow  at most two narrow tiles an SM.  One expert of 1408 x 2048 (22 / 32
//          tiles for 128 rows), 256 rows: 10.1 / 8.4 against 16.6 / 13.5 as
//          single tiles; 1024 rows: 15.9 / 13.1 against 16.4 / 13.8; 2048 rows:
//          21.5 / 21.6 against 16.8 / 14.3.
//  pair    segments of 384 rows on average and two rounds of pair tiles.  60
//          experts of 2816 x 2048, 512 rows: even 311 / 305 against 358 / 347 as
//          single tiles, Zipf 343 / 342 against 367 / 362; 384 rows: even (every
//          other pair tile half empty) 278 / 272 against 265 / 252, Zipf 287 /
//          280 against 298 / 296; 128 rows: even 138 / 137 against 125 / 125,
//          Zipf 163 / 163 against 156 / 151.  (With 256 rows pairs would win: even
//          152 / 156 against 174 / 172, Zipf 209 / 204 against 220 / 218.)  One
//          round (16 x 512 rows of 1024 x 1024): equal, 27 / 27.
static int mm_form(int mode, int rows, int nseg, int wide) {
    if (mode == kMmWgrad) return kMmSingle;
    const int sms = device_sm_count();
    const int64_t columns = (int64_t(wide) + 255) / 256;
    if (rows <= 16 * int64_t(nseg)) return kMmFew;
    const int64_t blocks = rows / 128 + (rows < nseg ? rows : nseg);  // at most
    if (blocks * ((int64_t(wide) + 63) / 64) <= 2 * int64_t(sms)) return kMmNarrow;
    return rows >= 384 * int64_t(nseg) && rows / 256 * columns >= sms ? kMmPair : kMmSingle;
}

static int grouped_mm_impl(const char* who, int mode, const void* pa, const void* pb, const int32_t* seg_start,
                           const int32_t* seg_expert, int nseg, int rows, int N, int K, int E, int dtype, void* out,
                           cudaStream_t s) {
    if (nseg < 1 || rows < 0 || N < 1 || K < 1 || E < 1)
        return fail(MOE_B200_ERR_INVALID_ARG, "%s: need nseg>=1, rows>=0, N>=1, K>=1, E>=1", who);
    if (nseg > kMmMaxSegments)
        return fail(MOE_B200_ERR_UNSUPPORTED, "%s: %d segments exceed %d", who, nseg, kMmMaxSegments);
    if (dtype != MOE_B200_F16 && dtype != MOE_B200_BF16)
        return fail(MOE_B200_ERR_INVALID_ARG, "%s: dtype %d is neither F16 nor BF16", who, dtype);
    if (N % 8 != 0 || K % 8 != 0)
        return fail(MOE_B200_ERR_UNSUPPORTED, "%s: N and K must be multiples of 8 (N=%d K=%d)", who, N, K);
    if (rows > kMmMaxSize || N > kMmMaxSize || K > kMmMaxSize)
        return fail(MOE_B200_ERR_UNSUPPORTED, "%s: rows, N and K may be at most %d", who, kMmMaxSize);
    if (rows == 0 && mode != kMmWgrad) return MOE_B200_OK;
    if (!seg_start || !out || (rows > 0 && (!pa || !pb)) || (mode != kMmWgrad && !pb))
        return fail(MOE_B200_ERR_INVALID_ARG, "%s: null pointer", who);
    const uintptr_t al = reinterpret_cast<uintptr_t>(pa) | reinterpret_cast<uintptr_t>(pb) | reinterpret_cast<uintptr_t>(out);
    if (al % 16 != 0) return fail(MOE_B200_ERR_INVALID_ARG, "%s: pointers must be 16-byte aligned", who);
    if (inside_element({seg_start, seg_expert}, 4))
        return fail(MOE_B200_ERR_INVALID_ARG, "%s: the segment tables must be 4-byte aligned", who);
    const int64_t row_n = 2 * int64_t(N), row_k = 2 * int64_t(K), weights = row_k * N;
    const bool wg = mode == kMmWgrad;
    if (overlaps_any(whole(out, wg ? nseg * weights : rows * (mode == kMmForward ? row_n : row_k)),
                     {whole(pa, rows * (mode == kMmForward ? row_k : row_n)), whole(pb, wg ? rows * row_k : E * weights),
                      whole(seg_start, 4 * (int64_t(nseg) + 1)), whole(seg_expert, 4 * int64_t(nseg))}))
        return fail(MOE_B200_ERR_INVALID_ARG, "%s: the result overlaps an operand", who);
    MmArgs a{};
    a.seg_start = seg_start;
    a.seg_expert = seg_expert;
    a.nseg = nseg;
    a.rows = rows;
    a.experts = E;
    a.out = static_cast<uint16_t*>(out);
    const int wide = mode == kMmForward ? N : K;  // output columns
    a.n_out = wide;
    a.kdim = mode == kMmForward ? K : N;
    a.m_out = N;
    const int64_t n_most = (int64_t(wide) + 127) / 128, m_most = (int64_t(N) + 127) / 128;  // of the smallest tiles
    if ((int64_t(rows) / 32 + nseg) * 2 * n_most > INT32_MAX || nseg * m_most * n_most > INT32_MAX)
        return fail(MOE_B200_ERR_UNSUPPORTED, "%s: too many tiles", who);
    if (rows == 0) {  // wgrad: sums over no row
        const cudaError_t err = cudaMemsetAsync(out, 0, size_t(nseg) * size_t(N) * size_t(K) * 2, s);
        return err == cudaSuccess ? MOE_B200_OK : cuda_fail(err, who);
    }
    a.status = device_status_word();
    if (!a.status) return fail(MOE_B200_ERR_CUDA, "%s: device status word unavailable", who);
    const int form = mm_form(mode, rows, nseg, wide);
    CUtensorMap ma, mb, mc;
    bool ok = mode == kMmWgrad ? make_map_experts(&mc, out, nseg, N, K, 32, dtype)
                               : make_map_experts(&mc, out, 1, rows, wide, 32, dtype);
    if (mode == kMmWgrad)
        ok = ok && make_map(&ma, pa, rows, N, kMmTileK, dtype) && make_map(&mb, pb, rows, K, kMmTileK, dtype);
    else
        ok = ok && make_map(&ma, pa, rows, a.kdim, form_rows(form), dtype) &&
             make_map_experts(&mb, pb, E, N, K, mode == kMmForward ? form_cols(form) : kMmTileK, dtype);
    if (!ok) return fail(MOE_B200_ERR_CUDA, "%s: cuTensorMapEncodeTiled failed", who);
    const cudaError_t err = mode == kMmForward ? launch_mm_as<kMmForward>(dtype, form, ma, mb, mc, a, s)
                            : mode == kMmDgrad ? launch_mm_as<kMmDgrad>(dtype, form, ma, mb, mc, a, s)
                                               : launch_mm_as<kMmWgrad>(dtype, form, ma, mb, mc, a, s);
    return err == cudaSuccess ? MOE_B200_OK : cuda_fail(err, who);
}

}  // namespace moe_b200

extern "C" int moe_b200_grouped_mm(const void* x, const int32_t* seg_start, const int32_t* seg_expert, int nseg,
                                   int rows, int N, int K, int E, const void* w, int dtype, void* y, void* stream) {
    return moe_b200::grouped_mm_impl("grouped_mm", moe_b200::kMmForward, x, w, seg_start, seg_expert, nseg, rows, N, K,
                                     E, dtype, y, static_cast<cudaStream_t>(stream));
}

extern "C" int moe_b200_grouped_mm_dgrad(const void* dy, const int32_t* seg_start, const int32_t* seg_expert, int nseg,
                                         int rows, int N, int K, int E, const void* w, int dtype, void* dx,
                                         void* stream) {
    return moe_b200::grouped_mm_impl("grouped_mm_dgrad", moe_b200::kMmDgrad, dy, w, seg_start, seg_expert, nseg, rows,
                                     N, K, E, dtype, dx, static_cast<cudaStream_t>(stream));
}

extern "C" int moe_b200_grouped_mm_wgrad(const void* dy, const void* x, const int32_t* seg_start, int nseg, int rows,
                                         int N, int K, int dtype, void* dw, void* stream) {
    return moe_b200::grouped_mm_impl("grouped_mm_wgrad", moe_b200::kMmWgrad, dy, x, seg_start, nullptr, nseg, rows, N,
                                     K, nseg, dtype, dw, static_cast<cudaStream_t>(stream));
}
