// expert_w4.cu -- products of few token rows with 4-bit expert weights:
// the serving form of the expert products for decode batches.
//
//   y[s, n] = sum_k x[row(s), k] * (q[e, n, k] - z[e, n, k / G]) * w_scale[e, n, k / G],   e = asgn[s]
// for slot s = (token, choice); row(s) is the token's row or the slot's own
// row of x.  With MOE_B200_ACT_SWIGLU the N = 2I columns are gate and up and
// the output is silu(y[:, :I]) * y[:, I:].
//
// With a few rows per expert the time is that of reading the chosen experts'
// weights once (half a byte per weight), so the kernel streams them:
//  - A CTA belongs to one expert (found from asgn on the device, no packing
//    pass) and to a range of its weight rows; it lists the expert's slots and
//    serves up to NT * 8 of them for one read of the weights.
//  - Weights keep their natural layout.  Each warp streams 32 weight rows x
//    128 k (2 KB) per step through its own cp.async ring of kStages steps, so
//    no registers and no barriers are spent on loads in flight.
//  - mma.sync m16n8k16 with the weights as the 16-row operand and 8 slots as
//    the columns.  A 32-bit word holds 8 consecutive k of one row; the order
//    of k inside a product does not matter as long as both operands agree, so
//    word s*4+t of a row is lane t's operand of step s and the nibbles are
//    taken in pairs (k, k+4): one shift and one logic op give two values.  x
//    is staged in shared memory in that order.
//  - q - z is an exact 16-bit integer and a product of it with x is exact in
//    fp32, so weights are never rounded: the group's fp32 sum is multiplied
//    by its scale.
//  - The k blocks are split over the CTA's warps (WK ways) and joined in
//    shared memory in warp order: results do not depend on timing.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "common.cuh"

namespace moe_b200 {

int fail(int code, const char* fmt, ...);
int cuda_fail(cudaError_t err, const char* where);

constexpr int kW4Warps = 8;
constexpr int kW4Threads = kW4Warps * 32;
constexpr int kW4Stages = 4;
constexpr int kW4Block = 128;       // k per step
constexpr int kW4TileRows = 32;     // weight rows per warp step: two 16-row operands
constexpr int kW4StageBytes = kW4TileRows * kW4Block / 2;
constexpr int kW4MaxSlots = 4096;
// Dynamic shared memory a CTA may ask for.
constexpr size_t kW4SmemLimit = 227 * 1024 - 1024;

struct W4Args {
    const void* x;
    const int32_t* asgn;
    const uint8_t* wq;
    const void* scale;
    const uint8_t* zero;
    void* out;
    uint32_t* status;
    int slots, x_div;    // slot s reads row s / x_div of x
    int E, N, K;
    int swiglu;          // 1: gate rows [0, N/2), up rows [N/2, N)
    int n_out;           // output columns
    int tiles;           // warp tiles per expert
    int tiles_per_cta, wk;
    int by_slot;         // 1: blockIdx.y is a slot, the first slot of an expert serves it
    int x_pitch;         // bytes of a staged x row
    int s_x, s_red, s_list;  // offsets of the staged x, the join buffer and the slot list
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool ok) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool ok) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(ok ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
}

// 16-bit integers 0..15 as floats with an offset: 0x6400 | q is 1024 + q in
// fp16, 0x4300 | q is 128 + q in bf16, both exact.
template <int DT> __device__ __forceinline__ constexpr uint32_t magic() {
    return DT == MOE_B200_BF16 ? 0x43004300u : 0x64006400u;
}
template <int DT> __device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b) {
    if (DT == MOE_B200_BF16) {
        __nv_bfloat162 r = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
        return *reinterpret_cast<uint32_t*>(&r);
    }
    __half2 r = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<uint32_t*>(&r);
}
// (nibble i, nibble i+4) - z for i = 0..3 of a word
template <int DT> __device__ __forceinline__ void unpack8(uint32_t w, uint32_t z2, uint32_t (&o)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = sub2<DT>(((w >> (4 * i)) & 0x000f000fu) | magic<DT>(), z2);
}

// Eight consecutive x in the order of a weight word's nibbles: (0,4) (1,5) (2,6) (3,7).
__device__ __forceinline__ uint4 x_pairs(const uint4& v) {
    return make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410),
                      __byte_perm(v.y, v.w, 0x7632));
}

template <int DT>
__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          uint32_t b0, uint32_t b1) {
    if (DT == MOE_B200_BF16)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <int DT> __device__ __forceinline__ float w4_from16(uint32_t b) {
    return DT == MOE_B200_BF16 ? __uint_as_float(b << 16) : __half2float(__ushort_as_half(uint16_t(b)));
}
template <int DT> __device__ __forceinline__ uint16_t w4_to16(float f) {
    return DT == MOE_B200_BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(f)) : __half_as_ushort(__float2half_rn(f));
}

// Row `r` (0..31) of tile `tile`: its weight row, or -1 past the last one.
// SwiGLU: rows 0..15 are gate rows, rows 16..31 the matching up rows.
__device__ __forceinline__ int w4_row(const W4Args& a, int tile, int r) {
    if (a.swiglu) {
        const int n = tile * 16 + (r & 15);
        return n < a.n_out ? n + (r >> 4) * a.n_out : -1;
    }
    const int n = tile * kW4TileRows + r;
    return n < a.N ? n : -1;
}

// Bytes of one ring step: weights, then per row and group a 4-byte word
// holding its scale and one holding its zero point.
template <int G> constexpr int w4_step_bytes() { return kW4StageBytes + 32 * (kW4Block / G) * 8; }

// XS: x is staged in shared memory; otherwise (rows too long for it) each lane
// reads its pieces of x from global memory, where they stay in L1 / L2.
template <int DT, int G, int NT, bool XS>
__global__ void __launch_bounds__(kW4Threads)
expert_linear_w4_kernel(const W4Args a) {
    extern __shared__ __align__(128) unsigned char smem[];
    constexpr int kGroups = kW4Block / G;  // groups of a row per step
    constexpr int kStep = w4_step_bytes<G>();
    uint16_t* s_list = reinterpret_cast<uint16_t*>(smem + a.s_list);
    __shared__ int s_warp[kW4Warps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;

    int e = int(blockIdx.y);
    if (a.by_slot) e = a.asgn[blockIdx.y];
    const bool e_ok = e >= 0 && e < a.E;

    const int wk = a.wk, wn_count = kW4Warps / wk, kw = warp % wk, wn = warp / wk;
    const int tile0 = int(blockIdx.x) * a.tiles_per_cta;
    const int tile_end = min(tile0 + a.tiles_per_cta, a.tiles);
    const int steps = (a.tiles_per_cta + wn_count - 1) / wn_count;  // tiles a warp walks
    const int blocks = (a.K + kW4Block - 1) / kW4Block;
    const int my_blocks = blocks > kw ? (blocks - kw + wk - 1) / wk : 0;
    const int iters = steps * my_blocks;  // of one pass over the weights
    const int ngroups = a.K / G;
    const uint32_t ring = smem_u32(smem) + warp * (kW4Stages * kStep);
    const int64_t row_bytes = a.K / 2;

    // Step `i` of a pass: tile tile0 + (i / my_blocks) * wn_count + wn, k block kw + (i % my_blocks) * wk.
    auto issue = [&](int i) {
        if (i < iters && e_ok) {
            const int tile = tile0 + (i / my_blocks) * wn_count + wn, b = kw + (i % my_blocks) * wk;
            const uint32_t dst = ring + (i % kW4Stages) * kStep;
            const bool tile_ok = tile < tile_end;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int r = j * 8 + g;  // 8 rows x 64 bytes per instruction
                const int n = tile_ok ? w4_row(a, tile, r) : -1;
                const bool ok = n >= 0 && b * kW4Block + t * 32 < a.K;
                const uint8_t* src = ok ? a.wq + (int64_t(e) * a.N + n) * row_bytes + b * (kW4Block / 2) + t * 16 : a.wq;
                // 16-byte pieces of a row sit at piece ^ (row / 2 mod 4): word reads are free of bank conflicts
                cp_async16(dst + r * 64 + ((t ^ ((r >> 1) & 3)) << 4), src, ok);
            }
            const int n = tile_ok ? w4_row(a, tile, lane) : -1;
#pragma unroll
            for (int q = 0; q < kGroups; ++q) {
                const int grp = b * kGroups + q;
                const bool ok = n >= 0 && grp < ngroups;
                const int64_t at = ok ? (int64_t(e) * a.N + n) * ngroups + grp : 0;
                const uint32_t d = dst + kW4StageBytes + (q * 32 + lane) * 8;
                cp_async4(d, static_cast<const uint16_t*>(a.scale) + (at & ~int64_t(1)), ok);
                if (a.zero) cp_async4(d + 4, a.zero + (at & ~int64_t(3)), ok);
            }
        }
        cp_commit();
    };
#pragma unroll
    for (int i = 0; i < kW4Stages - 1; ++i) issue(i);

    // The expert's slots in ascending order; slots without an expert (-1 or
    // out of range) get rows of zeros from the first row of CTAs.
    int count = 0;
    bool earlier = false;
    for (int s0 = 0; s0 < a.slots; s0 += kW4Threads) {
        const int s = s0 + threadIdx.x;
        const int v = s < a.slots ? a.asgn[s] : -1;
        const bool mine = e_ok && s < a.slots && v == e;
        if (mine && a.by_slot && s < int(blockIdx.y)) earlier = true;
        const uint32_t m = __ballot_sync(0xffffffffu, mine);
        if (lane == 0) s_warp[warp] = __popc(m);
        __syncthreads();
        int at = count;
        for (int w = 0; w < kW4Warps; ++w) {
            if (w < warp) at += s_warp[w];
            count += s_warp[w];
        }
        if (mine) s_list[at + __popc(m & lanemask_lt())] = uint16_t(s);
        if (blockIdx.y == 0 && s < a.slots && (v < 0 || v >= a.E)) {
            if (v != -1 && blockIdx.x == 0) atomicOr(a.status, MOE_B200_DEV_BAD_ASSIGNMENT);
            const int per = a.swiglu ? 16 : kW4TileRows;
            for (int c = tile0 * per; c < min(tile_end * per, a.n_out); ++c)
                static_cast<uint16_t*>(a.out)[int64_t(s) * a.n_out + c] = 0;
        }
        __syncthreads();
    }
    if (__syncthreads_or(earlier ? 1 : 0) || count == 0) {
        cp_wait<0>();
        return;
    }

    const uint32_t sx = smem_u32(smem + a.s_x);
    float* s_red = reinterpret_cast<float*>(smem + a.s_red);
    for (int r0 = 0; r0 < count; r0 += NT * 8) {
        const int nrows = min(count - r0, NT * 8);
        const int nt = (nrows + 7) >> 3;
        if (r0 > 0) {  // the next rows read the weights again (from L2)
#pragma unroll
            for (int i = 0; i < kW4Stages - 1; ++i) issue(i);
        }
        // Stage x, zeros past K and past the last row.
        const uint16_t* x_row[NT];
        if (XS) {
            const int chunks = blocks * (kW4Block / 8);
            for (int c = threadIdx.x; c < nt * 8 * chunks; c += kW4Threads) {
                const int r = c / chunks, k8 = c - r * chunks;
                uint4 v = make_uint4(0, 0, 0, 0);
                if (r < nrows && k8 * 8 < a.K)
                    v = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.x) +
                                                        int64_t(s_list[r0 + r] / a.x_div) * a.K + k8 * 8);
                *reinterpret_cast<uint4*>(smem + a.s_x + r * a.x_pitch + k8 * 16) = x_pairs(v);
            }
            __syncthreads();
        } else {
#pragma unroll
            for (int q = 0; q < NT; ++q)
                x_row[q] = q * 8 + g < nrows ? static_cast<const uint16_t*>(a.x) +
                                                   int64_t(s_list[r0 + q * 8 + g] / a.x_div) * a.K + t * 8
                                             : nullptr;
        }

        int i = 0;
        for (int step = 0; step < steps; ++step) {
            const int tile = tile0 + step * wn_count + wn;
            float acc[2][NT][4];
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int q = 0; q < NT; ++q)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[m][q][j] = 0.f;
            for (int jb = 0; jb < my_blocks; ++jb, ++i) {
                cp_wait<kW4Stages - 2>();
                __syncwarp();
                issue(i + kW4Stages - 1);  // into the step read last time
                const uint32_t st = ring + (i % kW4Stages) * kStep;
                const int b = kw + jb * wk;
                const uint32_t xb = sx + b * (kW4Block * 2) + t * 16;
#pragma unroll
                for (int q4 = 0; q4 < kGroups; ++q4) {
                    // scales and zero points of this lane's four rows
                    float sc[2][2];
                    uint32_t z2[2][2];
#pragma unroll
                    for (int m = 0; m < 2; ++m)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int r = m * 16 + h * 8 + g;
                            const uint32_t d = st + kW4StageBytes + (q4 * 32 + r) * 8;
                            const int n = w4_row(a, tile, r);
                            const uint32_t at = uint32_t(e * a.N + n) * uint32_t(ngroups) + uint32_t(b * kGroups + q4);
                            const uint32_t sw = lds32(d);
                            sc[m][h] = w4_from16<DT>((at & 1) ? (sw >> 16) : (sw & 0xffffu));
                            uint32_t z = 8;
                            if (a.zero) z = (lds32(d + 4) >> (8 * (at & 3))) & 0xffu;
                            z2[m][h] = z * 0x00010001u | magic<DT>();
                        }
                    float d4[2][NT][4];
#pragma unroll
                    for (int m = 0; m < 2; ++m)
#pragma unroll
                        for (int q = 0; q < NT; ++q)
#pragma unroll
                            for (int j = 0; j < 4; ++j) d4[m][q][j] = 0.f;
#pragma unroll
                    for (int s4 = 0; s4 < G / 32; ++s4) {
                        const int s = q4 * (G / 32) + s4;  // 32 k of the block
                        uint4 xv[NT];
#pragma unroll
                        for (int q = 0; q < NT; ++q)
                            if (XS) {
                                if (q < nt) xv[q] = lds128(xb + (q * 8 + g) * a.x_pitch + s * 64);
                            } else {
                                const int k = b * kW4Block + s * 32;
                                xv[q] = make_uint4(0, 0, 0, 0);
                                if (x_row[q] && k < a.K) xv[q] = x_pairs(*reinterpret_cast<const uint4*>(x_row[q] + k));
                            }
#pragma unroll
                        for (int m = 0; m < 2; ++m) {
                            uint32_t lo[4], hi[4];
                            const int ra = m * 16 + g, rb = ra + 8;
                            unpack8<DT>(lds32(st + ra * 64 + ((s ^ ((ra >> 1) & 3)) << 4) + t * 4), z2[m][0], lo);
                            unpack8<DT>(lds32(st + rb * 64 + ((s ^ ((rb >> 1) & 3)) << 4) + t * 4), z2[m][1], hi);
#pragma unroll
                            for (int q = 0; q < NT; ++q)
                                if (q < nt) {
                                    mma_16816<DT>(d4[m][q], lo[0], hi[0], lo[1], hi[1], xv[q].x, xv[q].y);
                                    mma_16816<DT>(d4[m][q], lo[2], hi[2], lo[3], hi[3], xv[q].z, xv[q].w);
                                }
                        }
                    }
#pragma unroll
                    for (int m = 0; m < 2; ++m)
#pragma unroll
                        for (int q = 0; q < NT; ++q)
#pragma unroll
                            for (int j = 0; j < 4; ++j) acc[m][q][j] += sc[m][j >> 1] * d4[m][q][j];
                }
                __syncwarp();  // the step is read before its refill
            }
            // Join the WK parts: [warp][m][q][lane][4] floats.
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int q = 0; q < NT; ++q)
                    if (q < nt)
                        *reinterpret_cast<float4*>(s_red + (((warp * 2 + m) * NT + q) * 32 + lane) * 4) =
                            make_float4(acc[m][q][0], acc[m][q][1], acc[m][q][2], acc[m][q][3]);
            __syncthreads();
            // One output a thread and turn: value j of lane l of the fragment
            // is row l/4 + 8*(j/2), column (l%4)*2 + j%2.
            const int per = (a.swiglu ? 1 : 2) * nt * 128;
            for (int o = threadIdx.x; o < wn_count * per; o += kW4Threads) {
                const int w2 = o / per, rem = o - w2 * per, f = rem >> 7, l = (rem & 127) >> 2, j = rem & 3;
                const int m = a.swiglu ? 0 : f / nt, q = a.swiglu ? f : f - m * nt;
                float v0 = 0.f, v1 = 0.f;
                for (int w = 0; w < wk; ++w) {
                    const float* p = s_red + ((((w2 * wk + w) * 2 + m) * NT + q) * 32 + l) * 4 + j;
                    v0 += p[0];
                    if (a.swiglu) v1 += p[NT * 128];
                }
                const int tl = tile0 + step * wn_count + w2, col = q * 8 + (l & 3) * 2 + (j & 1);
                const int rr = (l >> 2) + (j >> 1) * 8;
                const int n = a.swiglu ? tl * 16 + rr : tl * kW4TileRows + m * 16 + rr;
                if (tl < tile_end && n < a.n_out && col < nrows) {
                    if (a.swiglu) v0 = v0 / (1.0f + __expf(-v0)) * v1;
                    static_cast<uint16_t*>(a.out)[int64_t(s_list[r0 + col]) * a.n_out + n] = w4_to16<DT>(v0);
                }
            }
            __syncthreads();
        }
    }
    cp_wait<0>();
}

// ----------------------------------------------------------------- host ----

static int sm_count_w4() {
    int dev = 0, n = 148;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    return n > 0 ? n : 148;
}

// Shared memory of a CTA and its layout; xs: with x staged.
template <int G>
static size_t w4_layout(W4Args& a, int nt, bool xs) {
    const int blocks = (a.K + kW4Block - 1) / kW4Block;
    a.x_pitch = blocks * kW4Block * 2 + 64;  // 64 bytes off a multiple of 128: rows of a fragment on other banks
    size_t off = size_t(kW4Warps) * kW4Stages * w4_step_bytes<G>();
    a.s_x = int(off);
    off += xs ? size_t(nt) * 8 * a.x_pitch : 0;
    a.s_red = int(off);
    off += size_t(kW4Warps) * 2 * nt * 128 * 4;
    a.s_list = int(off);
    off += (size_t(a.slots) * 2 + 15) & ~size_t(15);
    return off;
}

template <int DT, int G, int NT, bool XS>
static cudaError_t launch_w4(W4Args a, dim3 grid, cudaStream_t s) {
    const size_t smem = w4_layout<G>(a, NT, XS);
    auto kern = expert_linear_w4_kernel<DT, G, NT, XS>;
    const cudaError_t err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
    if (err != cudaSuccess) return err;
    kern<<<grid, kW4Threads, smem, s>>>(a);
    return cudaGetLastError();
}

template <int DT, int G>
static cudaError_t run_w4(W4Args a, cudaStream_t s) {
    a.by_slot = a.slots < a.E;
    const int served = a.by_slot ? a.slots : a.E;  // experts that may have work
    // Rows served per read of the weights: 8, or 16 when some expert may have more and they fit.
    const bool two = a.slots > 8 && w4_layout<G>(a, 2, true) <= kW4SmemLimit;
    const bool staged = two || w4_layout<G>(a, 1, true) <= kW4SmemLimit;
    a.wk = 8;
    const int64_t units = int64_t(a.tiles) * served;
    a.tiles_per_cta = int(units / (int64_t(sm_count_w4()) * 8));
    if (a.tiles_per_cta < 1) a.tiles_per_cta = 1;
    if (a.tiles_per_cta > 8) a.tiles_per_cta = 8;
    const dim3 grid((a.tiles + a.tiles_per_cta - 1) / a.tiles_per_cta, served);
    if (two) return launch_w4<DT, G, 2, true>(a, grid, s);
    return staged ? launch_w4<DT, G, 1, true>(a, grid, s) : launch_w4<DT, G, 1, false>(a, grid, s);
}

}  // namespace moe_b200

extern "C" int moe_b200_expert_linear_w4(const void* x, int x_per_slot, const int32_t* asgn, int T, int K, int E, int d,
                                         int N, const void* w_q, const void* w_scale, const void* w_zero, int group,
                                         int act, int dtype, void* out, void* stream) {
    using namespace moe_b200;
    if (T < 0 || K < 1 || E < 1 || d < 1 || N < 1)
        return fail(MOE_B200_ERR_INVALID_ARG, "expert_linear_w4: need T>=0, K>=1, E>=1, d>=1, N>=1");
    if (dtype != MOE_B200_F16 && dtype != MOE_B200_BF16)
        return fail(MOE_B200_ERR_INVALID_ARG, "expert_linear_w4: dtype %d is neither F16 nor BF16", dtype);
    if (act != MOE_B200_ACT_NONE && act != MOE_B200_ACT_SWIGLU)
        return fail(MOE_B200_ERR_INVALID_ARG, "expert_linear_w4: unknown activation %d", act);
    if (group != 32 && group != 64 && group != 128)
        return fail(MOE_B200_ERR_UNSUPPORTED, "expert_linear_w4: group %d is not 32, 64 or 128", group);
    if (d % group != 0) return fail(MOE_B200_ERR_UNSUPPORTED, "expert_linear_w4: d=%d is no multiple of group=%d", d, group);
    if (N % (act == MOE_B200_ACT_SWIGLU ? 16 : 8) != 0)
        return fail(MOE_B200_ERR_UNSUPPORTED, "expert_linear_w4: N=%d must be a multiple of 8 (SwiGLU: 16)", N);
    if (E > MOE_B200_MAX_EXPERTS)
        return fail(MOE_B200_ERR_UNSUPPORTED, "expert_linear_w4: %d experts exceed %d", E, MOE_B200_MAX_EXPERTS);
    if (int64_t(T) * K > kW4MaxSlots)
        return fail(MOE_B200_ERR_UNSUPPORTED, "expert_linear_w4: %lld slots exceed %d", static_cast<long long>(T) * K,
                    kW4MaxSlots);
    if (T == 0) return MOE_B200_OK;
    if (!x || !asgn || !w_q || !w_scale || !out) return fail(MOE_B200_ERR_INVALID_ARG, "expert_linear_w4: null pointer");
    const uintptr_t al = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w_q) |
                         reinterpret_cast<uintptr_t>(w_scale) | reinterpret_cast<uintptr_t>(w_zero) |
                         reinterpret_cast<uintptr_t>(out);
    if (al % 16 != 0) return fail(MOE_B200_ERR_INVALID_ARG, "expert_linear_w4: pointers must be 16-byte aligned");
    uint32_t* st = device_status_word();
    if (!st) return fail(MOE_B200_ERR_CUDA, "expert_linear_w4: device status word unavailable");
    W4Args a{};
    a.x = x;
    a.asgn = asgn;
    a.wq = static_cast<const uint8_t*>(w_q);
    a.scale = w_scale;
    a.zero = static_cast<const uint8_t*>(w_zero);
    a.out = out;
    a.status = st;
    a.slots = T * K;
    a.x_div = x_per_slot ? 1 : K;
    a.E = E;
    a.N = N;
    a.K = d;
    a.swiglu = act == MOE_B200_ACT_SWIGLU;
    a.n_out = a.swiglu ? N / 2 : N;
    a.tiles = a.swiglu ? (a.n_out + 15) / 16 : (N + kW4TileRows - 1) / kW4TileRows;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool bf = dtype == MOE_B200_BF16;
    cudaError_t err;
    if (group == 32) err = bf ? run_w4<MOE_B200_BF16, 32>(a, s) : run_w4<MOE_B200_F16, 32>(a, s);
    else if (group == 64) err = bf ? run_w4<MOE_B200_BF16, 64>(a, s) : run_w4<MOE_B200_F16, 64>(a, s);
    else err = bf ? run_w4<MOE_B200_BF16, 128>(a, s) : run_w4<MOE_B200_F16, 128>(a, s);
    return err == cudaSuccess ? MOE_B200_OK : cuda_fail(err, "expert_linear_w4 launch");
}
