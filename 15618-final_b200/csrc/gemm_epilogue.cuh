// gemm_epilogue.cuh -- what the grouped tensor-core kernels share behind the
// accumulator: rounding, the staged row-wise stores, the segment lookup.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "common.cuh"

namespace moe_b200 {

template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if (DT == MOE_B200_BF16) {
        __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<uint32_t*>(&v);
    } else {
        __half2 v = __floats2half2_rn(a, b);
        return *reinterpret_cast<uint32_t*>(&v);
    }
}

// Epilogue staging: each epilogue warp owns 32 rows x 128 bytes (64 16-bit
// columns) of shared memory.  Lane r writes its accumulator row r; the 16-byte
// chunk j of row r sits at slot j ^ (r & 7), so that both the row-wise writes
// (8 lanes cover all 32 banks) and the chunk-wise reads are conflict-free.
constexpr uint32_t kWarpStageBytes = 32 * 128;
constexpr uint32_t kStageBytes = 4 * kWarpStageBytes;

__device__ __forceinline__ void stage_put(unsigned char* stg, int row, int chunk, const uint4& v) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(smem_u32(stg + row * 128 + ((chunk ^ (row & 7)) << 4))),
                 "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
                 : "memory");
}

// Writes the warp's staged 32 x 64 columns to its rows 0..nrows-1 (columns
// col0 .. col0+63, clipped at n_out): 4 rows x 128 contiguous bytes per warp
// store instruction instead of 32 scattered 16-byte pieces.  Row r goes to
// dst + r * stride, or, when lane_row is given (scatter mode), to the row
// address lane r holds in lane_row.
__device__ __forceinline__ void stage_flush(const unsigned char* stg, int lane, uint16_t* dst, int64_t stride,
                                            int nrows, int col0, int n_out, uint16_t* lane_row) {
    __syncwarp();
    const int ch = lane & 7;
    const bool col_ok = col0 + ch * 8 < n_out;
#pragma unroll
    for (int it = 0; it < 8; ++it) {
        const int r = it * 4 + (lane >> 3);
        uint4 v;
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                     : "r"(smem_u32(stg + r * 128 + ((ch ^ (r & 7)) << 4)))
                     : "memory");
        uint16_t* row = dst ? dst + int64_t(r) * stride
                            : reinterpret_cast<uint16_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(lane_row), r));
        if (r < nrows && col_ok) st_v4(reinterpret_cast<uint4*>(row + col0) + ch, v);
    }
    __syncwarp();
}

// Maps a linear 128-row block index to (segment, block within segment).
__device__ __forceinline__ int find_segment(const int32_t* blk_prefix, int nseg, int g) {
    int lo = 0, hi = nseg - 1;
    while (lo < hi) {
        int mid = (lo + hi + 1) >> 1;
        if (blk_prefix[mid] <= g) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

}  // namespace moe_b200
