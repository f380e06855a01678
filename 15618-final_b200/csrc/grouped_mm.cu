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
// of the next), tile scheduler.  Forward and dgrad tiles cost the same, and a
// persistent grid deals them round-robin.  A wgrad tile costs as much as its
// segment has rows; there the grid is one CTA per tile and running CTAs take
// over waiting ones (cluster launch control), which balances any routing.
//
// wgrad's last K step of a segment holds rows of the next segment: the MMA
// warp clears those rows of both operands in shared memory (so that no
// infinity or NaN there meets a zero) and issues only the 16-row MMAs that
// hold rows.  Every wait is bounded, as in the expert FFN.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "common.cuh"
#include "gemm_epilogue.cuh"
#include "tcgen05.cuh"

namespace moe_b200 {

int fail(int code, const char* fmt, ...);
int cuda_fail(cudaError_t err, const char* where);

enum { kMmForward = 0, kMmDgrad = 1, kMmWgrad = 2 };

constexpr int kMmTileM = 128;
constexpr int kMmTileN = 256;
constexpr int kMmTileK = 64;
constexpr int kMmThreads = 7 * 32;
constexpr int kMmStages = 4;
constexpr uint32_t kMmABytes = kMmTileM * kMmTileK * 2;  // 16 KB
constexpr uint32_t kMmBBytes = kMmTileN * kMmTileK * 2;  // 32 KB
constexpr uint32_t kMmBoxBytes = 64 * 64 * 2;            // one MN-major box: 64 columns x 64 reduced rows
constexpr uint32_t kMmTmemCols = 512;
constexpr int kMmMaxSegments = 1024;
constexpr int kSchedSlots = 2;

struct MmSmem {
    uint64_t full[kMmStages];
    uint64_t empty[kMmStages];
    uint64_t tmem_full[2];
    uint64_t tmem_empty[2];
    uint64_t sched_full[kSchedSlots];
    uint64_t sched_empty[kSchedSlots];
    uint4 sched[kSchedSlots];  // cluster launch control responses
    uint32_t tmem_base;
    int abort_flag;
    int total_blocks;
};

struct MmArgs {
    const int32_t* seg_start;
    const int32_t* seg_expert;
    int nseg, rows;
    int kdim;      // reduced length (forward, dgrad)
    int m_blocks;  // wgrad: 128-row blocks of dw
    int n_blocks;  // 256-column blocks of the output
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

template <int MODE, int DT>
__global__ void __launch_bounds__(kMmThreads, 1)
grouped_mm_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                  const MmArgs a) {
    constexpr bool kDynamic = MODE == kMmWgrad;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* base = reinterpret_cast<unsigned char*>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    unsigned char* sA = base;
    unsigned char* sB = sA + kMmStages * kMmABytes;
    unsigned char* s_stage = sB + kMmStages * kMmBBytes;
    MmSmem* ctl = reinterpret_cast<MmSmem*>(s_stage + kStageBytes);
    int32_t* blk_prefix = reinterpret_cast<int32_t*>(ctl + 1);  // [nseg + 1] row blocks before a segment
    int32_t* s_start = blk_prefix + (a.nseg + 1);               // [nseg] first row
    int32_t* s_rows = s_start + a.nseg;                         // [nseg] rows
    int32_t* s_exp = s_rows + a.nseg;                           // [nseg] expert

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile int* abort_flag = &ctl->abort_flag;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kMmStages; ++s) {
            mbar_init(&ctl->full[s], 1);
            mbar_init(&ctl->empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&ctl->tmem_full[b], 1);
            mbar_init(&ctl->tmem_empty[b], 4);
        }
        for (int b = 0; b < kSchedSlots; ++b) {
            mbar_init(&ctl->sched_full[b], 1);
            mbar_init(&ctl->sched_empty[b], 7);  // one arrival per warp
        }
        ctl->abort_flag = 0;
        mbar_fence_init();
        prefetch_tmap(&tmap_a);
        prefetch_tmap(&tmap_b);
    }
    if (warp == 0) {
        // Offsets are held inside [0, rows], so that no bad table leads a store outside the output.
        int run = 0;
        for (int s0 = 0; s0 < a.nseg; s0 += 32) {
            const int i = s0 + lane;
            int cnt = 0;
            if (i < a.nseg) {
                const int lo = min(max(a.seg_start[i], 0), a.rows), hi = min(max(a.seg_start[i + 1], 0), a.rows);
                s_start[i] = lo;
                s_rows[i] = max(hi - lo, 0);
                s_exp[i] = a.seg_expert ? a.seg_expert[i] : i;
                cnt = (s_rows[i] + kMmTileM - 1) / kMmTileM;
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
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_u32(&ctl->tmem_base)),
                     "r"(kMmTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();

    const uint32_t tmem = ctl->tmem_base;
    const int total_tiles = MODE == kMmWgrad ? a.nseg * a.m_blocks * a.n_blocks : ctl->total_blocks * a.n_blocks;
    const int first_tile = int(blockIdx.x) < total_tiles ? int(blockIdx.x) : -1;

    // The tile after `tile`, or -1.  Called by whole warps.
    uint32_t sidx = 0;
    auto next_tile = [&](int tile) -> int {
        if (!kDynamic) {
            const int n = tile + int(gridDim.x);
            return n < total_tiles && !__any_sync(0xffffffffu, *abort_flag) ? n : -1;
        }
        const int slot = int(sidx % kSchedSlots);
        const bool ok = wait_or_abort(&ctl->sched_full[slot], (sidx / kSchedSlots) & 1u, abort_flag, a.status);
        const int n = ok ? clc_result(&ctl->sched[slot]) : -1;
        fence_proxy_async_smem();  // the answer is read before the next one is written
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
        return (a.kdim + kMmTileK - 1) / kMmTileK;
    };

    if (warp == 0) {
        // ---------------- TMA producer ----------------
        uint32_t it = 0;
        for (int tile = first_tile; tile >= 0; tile = next_tile(tile)) {
            int s, m, n;
            const int nk = locate(tile, s, m, n);
            if (lane == 0) {
                const int e = s_exp[s], row0 = s_start[s];
                for (int kb = 0; kb < nk; ++kb, ++it) {
                    const int st = int(it % kMmStages);
                    if (!wait_or_abort(&ctl->empty[st], ((it / kMmStages) & 1u) ^ 1u, abort_flag, a.status)) break;
                    uint64_t* bar = &ctl->full[st];
                    mbar_arrive_expect_tx(bar, kMmABytes + kMmBBytes);
                    unsigned char* pa = sA + st * kMmABytes;
                    unsigned char* pb = sB + st * kMmBBytes;
                    if (MODE == kMmWgrad) {
                        for (int i = 0; i < kMmTileM / 64; ++i)
                            tma_load_2d(pa + i * kMmBoxBytes, &tmap_a, m * kMmTileM + i * 64, row0 + kb * kMmTileK, bar);
                        for (int i = 0; i < kMmTileN / 64; ++i)
                            tma_load_2d(pb + i * kMmBoxBytes, &tmap_b, n * kMmTileN + i * 64, row0 + kb * kMmTileK, bar);
                    } else {
                        tma_load_2d(pa, &tmap_a, kb * kMmTileK, row0 + m * kMmTileM, bar);
                        if (MODE == kMmForward) {
                            tma_load_3d(pb, &tmap_b, kb * kMmTileK, n * kMmTileN, e, bar);
                        } else {
                            for (int i = 0; i < kMmTileN / 64; ++i)
                                tma_load_3d(pb + i * kMmBoxBytes, &tmap_b, n * kMmTileN + i * 64, kb * kMmTileK, e, bar);
                        }
                    }
                }
            }
            __syncwarp();
        }
        if (lane == 0 && *abort_flag) drain_stages(ctl->full, it, kMmStages);
    } else if (warp == 1) {
        // ---------------- MMA issuer ----------------
        // Bits 15 / 16 of the instruction descriptor: A / B is MN-major.
        const uint32_t idesc = umma_idesc_mn(DT == MOE_B200_BF16 ? 1 : 0, kMmTileM, kMmTileN) |
                               (MODE == kMmWgrad ? 1u << 15 : 0u) | (MODE != kMmForward ? 1u << 16 : 0u);
        constexpr uint32_t a_step = MODE == kMmWgrad ? 2048 : 32;  // bytes per 16 reduced indices
        constexpr uint32_t b_step = MODE != kMmForward ? 2048 : 32;
        uint32_t it = 0, j = 0;
        bool ok = true;
        for (int tile = first_tile; ok && tile >= 0; tile = next_tile(tile)) {
            int s, m, n;
            const int nk = locate(tile, s, m, n);
            if (nk == 0) continue;  // an empty segment: the epilogue writes zeros
            const int buf = int(j & 1u);
            ok = __all_sync(0xffffffffu, wait_or_abort(&ctl->tmem_empty[buf], ((j >> 1) & 1u) ^ 1u, abort_flag, a.status));
            ++j;
            tc_fence_after();
            const uint32_t d_tmem = tmem + uint32_t(buf) * kMmTileN;
            for (int kb = 0; ok && kb < nk; ++kb, ++it) {
                const int st = int(it % kMmStages);
                ok = __all_sync(0xffffffffu, wait_or_abort(&ctl->full[st], (it / kMmStages) & 1u, abort_flag, a.status));
                if (!ok) break;
                const uint32_t a_addr = smem_u32(sA + st * kMmABytes), b_addr = smem_u32(sB + st * kMmBBytes);
                int k16 = kMmTileK / 16;
                if (MODE == kMmWgrad) {
                    const int rem = s_rows[s] - kb * kMmTileK;
                    if (rem < kMmTileK) {
                        k16 = (rem + 15) / 16;
                        // rows [rem, 16 * k16) of the 6 boxes: 128 bytes each, 8 lanes a row
                        const int clear = k16 * 16 - rem;
                        for (int i = lane; i < clear * 8 * 6; i += 32) {
                            const int box = i / (clear * 8), r = (i >> 3) % clear, c = i & 7;
                            const uint32_t at = (box < 2 ? a_addr + box * kMmBoxBytes : b_addr + (box - 2) * kMmBoxBytes) +
                                                (rem + r) * 128 + c * 16;
                            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(at), "r"(0) : "memory");
                        }
                        fence_proxy_async_smem();
                        __syncwarp();
                    }
                }
                tc_fence_after();
                if (lane == 0) {
                    for (int kk = 0; kk < k16; ++kk) {
                        const uint64_t ad = MODE == kMmWgrad ? umma_desc_mn_sw128(a_addr + kk * a_step)
                                                             : umma_desc_sw128(a_addr + kk * a_step);
                        const uint64_t bd = MODE != kMmForward ? umma_desc_mn_sw128(b_addr + kk * b_step)
                                                               : umma_desc_sw128(b_addr + kk * b_step);
                        umma_f16(d_tmem, ad, bd, idesc, (kb > 0 || kk > 0) ? 1u : 0u);
                    }
                    umma_commit(&ctl->empty[st]);
                    if (kb == nk - 1) umma_commit(&ctl->tmem_full[buf]);
                }
                __syncwarp();
            }
        }
    } else if (warp < 6) {
        // ---------------- epilogue (warps 2..5) ----------------
        const int quad = warp & 3;  // TMEM lanes 32*quad .. 32*quad+31
        unsigned char* stg = s_stage + quad * kWarpStageBytes;
        uint32_t j = 0;
        for (int tile = first_tile; tile >= 0; tile = next_tile(tile)) {
            int s, m, n;
            const int nk = locate(tile, s, m, n);
            const int w_row0 = m * kMmTileM + quad * 32;
            const int nrows_w = (MODE == kMmWgrad ? a.m_out : s_rows[s]) - w_row0;
            const int64_t out_row = (MODE == kMmWgrad ? int64_t(s) * a.m_out : int64_t(s_start[s])) + w_row0;
            uint16_t* dst = a.out + out_row * a.n_out;
            const int buf = int(j & 1u);
            if (nk > 0) {
                const bool ok = wait_or_abort(&ctl->tmem_full[buf], (j >> 1) & 1u, abort_flag, a.status);
                if (!__all_sync(0xffffffffu, ok)) break;
                ++j;
                tc_fence_after();
            }
            const uint32_t t_row = tmem + uint32_t(buf) * kMmTileN + (uint32_t(quad * 32) << 16);
#pragma unroll 1
            for (int c = 0; c < kMmTileN; c += 64) {
                if (n * kMmTileN + c >= a.n_out) break;
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
#pragma unroll
                for (int q4 = 0; q4 < 4; ++q4) {
                    uint32_t o[8];
#pragma unroll
                    for (int q = 0; q < 8; ++q)
                        o[q] = pack2<DT>(__uint_as_float(v[q4][2 * q]), __uint_as_float(v[q4][2 * q + 1]));
                    stage_put(stg, lane, 2 * q4, make_uint4(o[0], o[1], o[2], o[3]));
                    stage_put(stg, lane, 2 * q4 + 1, make_uint4(o[4], o[5], o[6], o[7]));
                }
                stage_flush(stg, lane, dst, a.n_out, nrows_w, n * kMmTileN + c, a.n_out, nullptr);
            }
            if (nk > 0) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&ctl->tmem_empty[buf]);
            }
        }
    } else if (kDynamic) {
        // ---------------- tile scheduler (warp 6) ----------------
        // Fills the answer slots ahead of the other warps and stops after the
        // first answer that names no CTA.
        int tile = first_tile;
        while (tile >= 0) {
            const int slot = int(sidx % kSchedSlots);
            const bool ok =
                wait_or_abort(&ctl->sched_empty[slot], ((sidx / kSchedSlots) & 1u) ^ 1u, abort_flag, a.status);
            if (!__all_sync(0xffffffffu, ok)) break;
            if (lane == 0) {
                mbar_arrive_expect_tx(&ctl->sched_full[slot], 16);
                clc_try_cancel(&ctl->sched[slot], &ctl->sched_full[slot]);
            }
            __syncwarp();
            tile = next_tile(tile);
        }
    }

    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) {
        __syncwarp();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kMmTmemCols) : "memory");
    }
}

// ----------------------------------------------------------------- host ----

// 3-D map over w [E, N, K] 16-bit; box = 64 columns x box_rows rows of one expert, 128B swizzle.
static bool make_map_experts(CUtensorMap* map, const void* base, int64_t experts, int64_t rows, int64_t cols,
                             int box_rows, int dtype) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    cuuint64_t dims[3] = {cuuint64_t(cols), cuuint64_t(rows), cuuint64_t(experts)};
    cuuint64_t strides[2] = {cuuint64_t(cols) * 2, cuuint64_t(cols) * cuuint64_t(rows) * 2};
    cuuint32_t box[3] = {64u, cuuint32_t(box_rows), 1u};
    cuuint32_t estr[3] = {1, 1, 1};
    return fn(map, dtype == MOE_B200_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
              const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

static int sm_count_mm() {
    int dev = 0, n = 148;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    return n > 0 ? n : 148;
}

template <int MODE, int DT>
static cudaError_t launch_mm(const CUtensorMap& ma, const CUtensorMap& mb, const MmArgs& a, cudaStream_t s) {
    auto kern = grouped_mm_kernel<MODE, DT>;
    const size_t smem = 1024 + size_t(kMmStages) * (kMmABytes + kMmBBytes) + kStageBytes + sizeof(MmSmem) +
                        size_t(4 * a.nseg + 1) * 4;
    cudaError_t err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
    if (err != cudaSuccess) return err;
    int64_t grid;
    if (MODE == kMmWgrad) {
        grid = int64_t(a.nseg) * a.m_blocks * a.n_blocks;
    } else {
        grid = (int64_t(a.rows) / kMmTileM + a.nseg) * a.n_blocks;  // each segment may add one partial block
        if (grid > sm_count_mm()) grid = sm_count_mm();
    }
    kern<<<unsigned(grid), kMmThreads, smem, s>>>(ma, mb, a);
    return cudaGetLastError();
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
    if (rows == 0 && mode != kMmWgrad) return MOE_B200_OK;
    if (!seg_start || !out || (rows > 0 && (!pa || !pb)) || (mode != kMmWgrad && !pb))
        return fail(MOE_B200_ERR_INVALID_ARG, "%s: null pointer", who);
    const uintptr_t al = reinterpret_cast<uintptr_t>(pa) | reinterpret_cast<uintptr_t>(pb) | reinterpret_cast<uintptr_t>(out);
    if (al % 16 != 0) return fail(MOE_B200_ERR_INVALID_ARG, "%s: pointers must be 16-byte aligned", who);
    MmArgs a{};
    a.seg_start = seg_start;
    a.seg_expert = seg_expert;
    a.nseg = nseg;
    a.rows = rows;
    a.out = static_cast<uint16_t*>(out);
    const int wide = mode == kMmForward ? N : K;  // output columns
    a.n_out = wide;
    a.n_blocks = (wide + kMmTileN - 1) / kMmTileN;
    a.kdim = mode == kMmForward ? K : N;
    a.m_out = N;
    a.m_blocks = (N + kMmTileM - 1) / kMmTileM;
    if ((int64_t(rows) / kMmTileM + nseg) * a.n_blocks > INT32_MAX || int64_t(nseg) * a.m_blocks * a.n_blocks > INT32_MAX)
        return fail(MOE_B200_ERR_UNSUPPORTED, "%s: too many tiles", who);
    if (rows == 0) {  // wgrad: sums over no row
        const cudaError_t err = cudaMemsetAsync(out, 0, size_t(nseg) * size_t(N) * size_t(K) * 2, s);
        return err == cudaSuccess ? MOE_B200_OK : cuda_fail(err, who);
    }
    a.status = device_status_word();
    if (!a.status) return fail(MOE_B200_ERR_CUDA, "%s: device status word unavailable", who);
    CUtensorMap ma, mb;
    bool ok;
    if (mode == kMmWgrad)
        ok = make_map(&ma, pa, rows, N, kMmTileK, dtype) && make_map(&mb, pb, rows, K, kMmTileK, dtype);
    else
        ok = make_map(&ma, pa, rows, a.kdim, kMmTileM, dtype) &&
             make_map_experts(&mb, pb, E, N, K, mode == kMmForward ? kMmTileN : kMmTileK, dtype);
    if (!ok) return fail(MOE_B200_ERR_CUDA, "%s: cuTensorMapEncodeTiled failed", who);
    const bool bf = dtype == MOE_B200_BF16;
    cudaError_t err;
    if (mode == kMmForward)
        err = bf ? launch_mm<kMmForward, MOE_B200_BF16>(ma, mb, a, s) : launch_mm<kMmForward, MOE_B200_F16>(ma, mb, a, s);
    else if (mode == kMmDgrad)
        err = bf ? launch_mm<kMmDgrad, MOE_B200_BF16>(ma, mb, a, s) : launch_mm<kMmDgrad, MOE_B200_F16>(ma, mb, a, s);
    else
        err = bf ? launch_mm<kMmWgrad, MOE_B200_BF16>(ma, mb, a, s) : launch_mm<kMmWgrad, MOE_B200_F16>(ma, mb, a, s);
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
