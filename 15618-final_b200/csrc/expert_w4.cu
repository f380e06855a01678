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
//  - Every CTA sorts the slots by expert in shared memory (a few hundred
//    words, no packing pass) and takes an even share of all (expert, weight
//    rows) units, so that any routing is balanced; up to NT * 8 slots of an
//    expert are served by one read of its weights.
//  - Weights keep their natural layout.  Each warp streams 32 weight rows x
//    256 k (4 KB) per step through its own ring: two TMA boxes of 16 rows x
//    128 bytes, whose 128-byte swizzle makes the word reads free of bank
//    conflicts; no registers and no barriers are spent on loads in flight.
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
// What bounds it: for one token latency (launch, slot list, one trip to memory
// for x and for the weights); for batches the work between the MMAs, spread
// over all of it, done by 4 warps a scheduler (128 registers each), and their
// stalls: a pass over a weight executes 2.9 instructions a lane with groups of 128 and
// up to 8 rows of x (63% of the issue slots at 1.81 GHz) and 5.2 with groups of 32,
// zero points and up to 16 rows (55%): unpacking, x and scales from shared memory
// and by shuffles, the groups' sums.  The tensor pipe is not it: mma.sync m16n8k16 takes
// 8 cycles a scheduler, 21 to 23% of the time, and a unit with 8 rows of x costs
// about as much as one with 16, so that shares weighted by rows are worse (66 to
// 78 us against 62).  tcgen05.mma with the unpacked weights in tensor memory was
// built and measured too: the chain from unpacking to reading the groups'
// accumulators back is longer (64 tokens 75 us, one token 11, in a graph;
// this form 50 and 7).  Measured on one B200, 60 experts, 4 a token (bf16, groups
// of 128, gate/up 2816 x 2048 with SwiGLU): 1 token 12.7 us, 64 tokens 52 us;
// down 2048 x 1408 (fp16, groups of 32, zero points), 147 tokens: 64 to 83 us by
// routing.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "common.cuh"
#include "per_device.cuh"
#include "tcgen05.cuh"

namespace moe_b200 {

int fail(int code, const char* fmt, ...);
int cuda_fail(cudaError_t err, const char* where);

constexpr int kW4Parts = 8;         // stretches of slots that are listed side by side
constexpr int kW4Stages = 2;
constexpr int kW4Block = 256;       // k per step
constexpr int kW4TileRows = 32;     // weight rows per warp step: two 16-row operands
constexpr int kW4StageBytes = kW4TileRows * kW4Block / 2;
constexpr int kW4MaxSlots = 4096;
constexpr int kW4MaxSize = 1 << 29;  // d and N: bytes of a staged row of x and row indices stay 32-bit
// Dynamic shared memory a CTA may ask for.
constexpr size_t kW4SmemLimit = 227 * 1024 - 1024;

struct W4Args {
    const void* x;
    const int32_t* asgn;
    const void* scale;
    const uint8_t* zero;
    void* out;
    uint32_t* status;
    int slots, x_div;    // slot s reads row s / x_div of x
    int E, N, K;
    int swiglu;          // 1: gate rows [0, N/2), up rows [N/2, N)
    int n_out;           // output columns
    int tiles;           // warp tiles per expert
    int wk;              // warps that share a tile's k blocks
    int units;           // units (8 / wk neighbouring tiles) per expert and pass
    int x_pitch;         // bytes of a staged x row
    int s_x, s_red, s_tab;  // offsets of the staged x, the join buffer and the slot tables
};

__device__ __forceinline__ void tma_load_rows(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
            smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
        : "memory");
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
// (w & mask) | bits in one instruction
__device__ __forceinline__ uint32_t and_or(uint32_t w, uint32_t mask, uint32_t bits) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(w), "r"(mask), "r"(bits));
    return r;
}
// (nibble i, nibble i+4) - z for i = 0..3 of a word, z2 = the magic number + z twice
template <int DT> __device__ __forceinline__ void unpack8(uint32_t w, uint32_t z2, uint32_t (&o)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = sub2<DT>(and_or(i ? w >> (4 * i) : w, 0x000f000fu, magic<DT>()), z2);
}

// Eight consecutive x in the order of a weight word's nibbles: (0,4) (1,5) (2,6) (3,7).
__device__ __forceinline__ uint4 x_pairs(const uint4& v) {
    return make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410),
                      __byte_perm(v.y, v.w, 0x7632));
}

// c = A . B (FIRST) or c += A . B
template <int DT, bool FIRST>
__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          uint32_t b0, uint32_t b1) {
    const float i0 = FIRST ? 0.f : c[0], i1 = FIRST ? 0.f : c[1], i2 = FIRST ? 0.f : c[2], i3 = FIRST ? 0.f : c[3];
    if (DT == MOE_B200_BF16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%10, %11, %12, %13};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(i0), "f"(i1), "f"(i2), "f"(i3));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%10, %11, %12, %13};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(i0), "f"(i1), "f"(i2), "f"(i3));
}

template <int DT> __device__ __forceinline__ float w4_from16(uint32_t b) {
    return DT == MOE_B200_BF16 ? __uint_as_float(b << 16) : __half2float(__ushort_as_half(uint16_t(b)));
}
template <int DT> __device__ __forceinline__ uint16_t w4_to16(float f) {
    return DT == MOE_B200_BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(f)) : __half_as_ushort(__float2half_rn(f));
}

// XS: x is staged in shared memory; otherwise (rows too long for it) each lane
// reads its pieces of x from global memory, where they stay in L1 / L2.
// W: warps of the CTA.  With 16 rows of x a CTA fills an SM by itself, and 16
// warps share them (147 tokens, 2048 x 1408: 71 us against 76 with 8).
template <int DT, int G, int NT, bool XS, int W>
__global__ void __launch_bounds__(W * 32, 16 / W)
expert_linear_w4_kernel(const __grid_constant__ CUtensorMap tmap, const W4Args a) {
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ uint64_t s_full[W][kW4Stages];
    constexpr int kGroups = kW4Block / G;  // groups of a row per step
    constexpr int kThreads = W * 32;
    int* s_expert = reinterpret_cast<int*>(smem + a.s_tab);  // [entries] experts served (or all of them)
    int* s_cnt = s_expert + a.E;                             // [entries] slots of an expert
    int* s_first = s_cnt + a.E;                              // [entries] its first place in s_slots
    int* s_unit = s_first + a.E;                             // [entries + 1] units of the experts before
    int* s_cur = s_unit + a.E + 1;                           // [kW4Parts][E] next place, by stretch
    uint16_t* s_slots = reinterpret_cast<uint16_t*>(s_cur + kW4Parts * a.E);  // [slots] by expert, ascending
    __shared__ int s_entries, s_none;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;

    // Slots by expert, ascending within an expert (every CTA has to find the
    // same order: CTAs share an expert's slots by their places in it).
    bool none = false;
    if (a.slots <= 32) {
        // One warp, a lane per slot; the experts in the order of their first slots.
        if (warp == 0) {
            const int e = lane < a.slots ? a.asgn[lane] : -1;
            const bool ok = e >= 0 && e < a.E;
            if (lane < a.slots && !ok && e != -1 && blockIdx.x == 0) atomicOr(a.status, MOE_B200_DEV_BAD_ASSIGNMENT);
            const uint32_t same = __match_any_sync(0xffffffffu, ok ? e : -1), lt = lanemask_lt();
            const bool leads = ok && (same & lt) == 0;
            const uint32_t leaders = __ballot_sync(0xffffffffu, leads);
            const int c = leads ? __popc(same) : 0, u = (c + NT * 8 - 1) / (NT * 8) * a.units;
            int rows = c, units = u;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int rv = __shfl_up_sync(0xffffffffu, rows, o), uv = __shfl_up_sync(0xffffffffu, units, o);
                if (lane >= o) rows += rv, units += uv;
            }
            const int first = __shfl_sync(0xffffffffu, rows - c, __ffs(same) - 1);
            if (leads) {
                const int i = __popc(leaders & lt);
                s_expert[i] = e;
                s_cnt[i] = c;
                s_first[i] = rows - c;
                s_unit[i + 1] = units;
            }
            if (ok) s_slots[first + __popc(same & lt)] = uint16_t(lane);
            none = __any_sync(0xffffffffu, lane < a.slots && !ok);
            if (lane == 0) {
                s_unit[0] = 0;
                s_entries = __popc(leaders);
                s_none = none;
            }
        }
        __syncthreads();
    } else {
        // The first warps count and deal one stretch of the slots each.
        const int part = ((a.slots + kW4Parts * 32 - 1) / (kW4Parts * 32)) * 32;
        const int s_lo = warp < kW4Parts ? warp * part : a.slots, s_hi = min(s_lo + part, a.slots);
        const int first_e = s_lo + lane < s_hi ? a.asgn[s_lo + lane] : -1;
        for (int i = threadIdx.x; i < kW4Parts * a.E; i += kThreads) s_cur[i] = 0;
        __syncthreads();
        for (int s = s_lo + lane; s < s_hi; s += 32) {
            const int e = s == s_lo + lane ? first_e : a.asgn[s];
            if (e >= 0 && e < a.E) atomicAdd(&s_cur[warp * a.E + e], 1);
            else if (e != -1 && blockIdx.x == 0) atomicOr(a.status, MOE_B200_DEV_BAD_ASSIGNMENT);
            none |= e < 0 || e >= a.E;
        }
        none = __syncthreads_or(none);
        if (warp == 0) {
            int rows = 0, units = 0;
            for (int e0 = 0; e0 < a.E; e0 += 32) {
                const int e = e0 + lane;
                int n[kW4Parts], c = 0;
#pragma unroll
                for (int w = 0; w < kW4Parts; ++w) {
                    n[w] = e < a.E ? s_cur[w * a.E + e] : 0;
                    c += n[w];
                }
                int r = c, u = (c + NT * 8 - 1) / (NT * 8) * a.units;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int rv = __shfl_up_sync(0xffffffffu, r, o), uv = __shfl_up_sync(0xffffffffu, u, o);
                    if (lane >= o) r += rv, u += uv;
                }
                if (e < a.E) {
                    s_expert[e] = e;
                    s_cnt[e] = c;
                    int at = rows + r - c;
                    s_first[e] = at;
#pragma unroll
                    for (int w = 0; w < kW4Parts; ++w) {
                        s_cur[w * a.E + e] = at;
                        at += n[w];
                    }
                    s_unit[e + 1] = units + u;
                }
                rows += __shfl_sync(0xffffffffu, r, 31);
                units += __shfl_sync(0xffffffffu, u, 31);
            }
            if (lane == 0) {
                s_unit[0] = 0;
                s_entries = a.E;
                s_none = none;
            }
        }
        __syncthreads();
        for (int s0 = s_lo; s0 < s_hi; s0 += 32) {
            const int s = s0 + lane;
            const int e = s0 == s_lo ? first_e : s < s_hi ? a.asgn[s] : -1;
            const bool ok = e >= 0 && e < a.E;
            const uint32_t same = __match_any_sync(0xffffffffu, ok ? e : -1);
            int base = 0;
            if (ok) base = s_cur[warp * a.E + e];
            __syncwarp();
            if (ok) {
                s_slots[base + __popc(same & lanemask_lt())] = uint16_t(s);
                if ((same & lanemask_lt()) == 0) s_cur[warp * a.E + e] = base + __popc(same);
            }
            __syncwarp();
        }
        __syncthreads();
    }
    const int entries = s_entries;
    // Slots without an expert get rows of zeros, dealt over the grid.
    for (int s = blockIdx.x; s_none && s < a.slots; s += gridDim.x) {
        const int e = a.asgn[s];
        if (e >= 0 && e < a.E) continue;
        for (int c = threadIdx.x; c < a.n_out; c += kThreads)
            static_cast<uint16_t*>(a.out)[int64_t(s) * a.n_out + c] = 0;
    }

    // This CTA's even share of all units.
    const int total = s_unit[entries], share = total / int(gridDim.x), more = total - share * int(gridDim.x);
    const int u_begin = share * int(blockIdx.x) + min(int(blockIdx.x), more);
    const int u_end = u_begin + share + (int(blockIdx.x) < more ? 1 : 0);
    if (u_begin >= u_end) return;

    const int wk = a.wk, wn_count = W / wk, kw = warp % wk, wn = warp / wk;
    const int blocks = (a.K + kW4Block - 1) / kW4Block;
    const int my_blocks = blocks > kw ? (blocks - kw + wk - 1) / wk : 0;
    const int ngroups = a.K / G;

    // A place in the walk over units: entry and its expert, unit of its current pass, pass.
    struct Place {
        int u, i, e, tg, pass;
    };
    auto entry_of = [&](int u) {  // last entry with s_unit[i] <= u
        int lo = 0, hi = entries - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (s_unit[mid] <= u) lo = mid;
            else hi = mid - 1;
        }
        return lo;
    };
    auto place_at = [&](int u) {
        Place p;
        p.u = u;
        p.i = entry_of(u);
        p.e = s_expert[p.i];
        const int local = u - s_unit[p.i];
        p.pass = local / a.units;
        p.tg = local - p.pass * a.units;
        return p;
    };
    auto advance = [&](Place& p) {
        ++p.u;
        if (++p.tg < a.units) return;
        p.tg = 0;
        ++p.pass;
        if (p.u < u_end && p.u >= s_unit[p.i + 1]) {
            p.i = entry_of(p.u);
            p.e = s_expert[p.i];
            p.pass = 0;
        }
    };

    // The next step of a warp, fetched while it works on one: its weights by
    // TMA into the other half of its ring, and the scales and zero points of
    // tile row `lane` into registers (handed out by shuffles).
    unsigned char* ring = smem + warp * (kW4Stages * kW4StageBytes);
    uint32_t sc_raw[kGroups], z_raw[kGroups];
    auto fetch = [&](const Place& p, int b, int slot) {
        const int n = (p.tg * wn_count + wn) * (a.swiglu ? 16 : kW4TileRows);
        if (lane == 0) {  // rows past N and columns past K read as zeros
            unsigned char* dst = ring + slot * kW4StageBytes;
            uint64_t* bar = &s_full[warp][slot];
            mbar_arrive_expect_tx(bar, kW4StageBytes);
            tma_load_rows(dst, &tmap, b * (kW4Block / 2), n, p.e, bar);
            tma_load_rows(dst + kW4StageBytes / 2, &tmap, b * (kW4Block / 2), n + (a.swiglu ? a.n_out : 16), p.e, bar);
        }
        const int r = n + (a.swiglu ? lane & 15 : lane);
        const bool row_ok = r < a.n_out;
        const int64_t base = (int64_t(p.e) * a.N + r + (a.swiglu ? (lane >> 4) * a.n_out : 0)) * ngroups + b * kGroups;
        const uint16_t* sp = static_cast<const uint16_t*>(a.scale) + base;
        const uint8_t* zp = a.zero + base;
#pragma unroll
        for (int q = 0; q < kGroups; ++q) {
            const bool ok = row_ok && b * kGroups + q < ngroups;
            sc_raw[q] = ok ? sp[q] : 0u;
            z_raw[q] = 0u;
            if (a.zero) z_raw[q] = ok ? zp[q] : 0u;
        }
    };
    if (lane == 0) {
        for (int i = 0; i < kW4Stages; ++i) mbar_init(&s_full[warp][i], 1);
        mbar_fence_init();
    }
    __syncwarp();
    Place at = place_at(u_begin);
    if (my_blocks > 0) fetch(at, kw, 0);

    float* s_red = reinterpret_cast<float*>(smem + a.s_red);
    int piece[kW4Block / 32];  // where the 16-byte pieces of this lane's rows sit
#pragma unroll
    for (int s = 0; s < kW4Block / 32; ++s) piece[s] = (s ^ g) << 4;
    int staged_e = -1, staged_pass = 0, nrows = 0, nt = 0, list0 = 0, slot = 0;
    uint32_t parity = 0;
    const uint16_t* x_row[NT];
    while (at.u < u_end) {
        Place next = at;
        advance(next);
        if (at.e != staged_e || at.pass != staged_pass) {
            staged_e = at.e, staged_pass = at.pass;
            const int cnt = s_cnt[at.i];
            list0 = s_first[at.i] + at.pass * NT * 8;
            nrows = min(cnt - at.pass * NT * 8, NT * 8);
            nt = (nrows + 7) >> 3;
            if (XS) {  // zeros past K; columns of the product past the last row are not written
                const int chunks = blocks * (kW4Block / 8), all = nrows * chunks;
                for (int c0 = threadIdx.x; c0 < all; c0 += 4 * kThreads) {
                    uint4 v[4];
                    int r[4], k8[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {  // four loads in flight
                        const int c = c0 + i * kThreads;
                        r[i] = c / chunks, k8[i] = c - r[i] * chunks;
                        v[i] = make_uint4(0, 0, 0, 0);
                        if (c < all && k8[i] * 8 < a.K)
                            v[i] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.x) +
                                                                   int64_t(s_slots[list0 + r[i]] / a.x_div) * a.K + k8[i] * 8);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (c0 + i * kThreads < all)
                            *reinterpret_cast<uint4*>(smem + a.s_x + r[i] * a.x_pitch + k8[i] * 16) = x_pairs(v[i]);
                }
                __syncthreads();
            } else {
#pragma unroll
                for (int q = 0; q < NT; ++q)
                    x_row[q] = q * 8 + g < nrows ? static_cast<const uint16_t*>(a.x) +
                                                       int64_t(s_slots[list0 + q * 8 + g] / a.x_div) * a.K + t * 8
                                                 : nullptr;
            }
        }
        float acc[2][NT][4];
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int q = 0; q < NT; ++q)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[m][q][j] = 0.f;
#pragma unroll 1
        for (int jb = 0; jb < my_blocks; ++jb) {
            const int b = kw + jb * wk;
            // scale in the upper half, zero point in the lower
            uint32_t sz[kGroups];
#pragma unroll
            for (int q = 0; q < kGroups; ++q) sz[q] = sc_raw[q] << 16 | z_raw[q];
            if (jb + 1 < my_blocks) fetch(at, b + wk, slot ^ 1);
            else if (next.u < u_end) fetch(next, kw, slot ^ 1);
            if (!mbar_wait(&s_full[warp][slot], parity)) atomicOr(a.status, MOE_B200_DEV_WAIT_TIMEOUT);
            const unsigned char* wb = ring + slot * kW4StageBytes + g * 128 + t * 4;
            parity ^= uint32_t(slot);
            slot ^= 1;
            const unsigned char* xb = smem + a.s_x + b * (kW4Block * 2) + t * 16 + g * a.x_pitch;
#pragma unroll
            for (int q4 = 0; q4 < kGroups; ++q4) {
                float sc[2][2];
                uint32_t z2[2][2];
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t v = __shfl_sync(0xffffffffu, sz[q4], m * 16 + h * 8 + g);
                        sc[m][h] = DT == MOE_B200_BF16 ? __uint_as_float(v & 0xffff0000u) : w4_from16<DT>(v >> 16);
                        z2[m][h] = magic<DT>() + 8 * 0x00010001u;
                        if (a.zero) z2[m][h] = (v & 0xffu) * 0x00010001u + magic<DT>();
                    }
                float d4[2][NT][4];
#pragma unroll
                for (int s4 = 0; s4 < G / 32; ++s4) {
                    const int s = q4 * (G / 32) + s4;  // 32 k of the step
                    uint4 xv[NT];
#pragma unroll
                    for (int q = 0; q < NT; ++q)
                        if (XS) {
                            if (q == 0 || q < nt) xv[q] = *reinterpret_cast<const uint4*>(xb + q * 8 * a.x_pitch + s * 64);
                        } else {
                            const int k = b * kW4Block + s * 32;
                            xv[q] = make_uint4(0, 0, 0, 0);
                            if (x_row[q] && k < a.K) xv[q] = x_pairs(*reinterpret_cast<const uint4*>(x_row[q] + k));
                        }
#pragma unroll
                    for (int m = 0; m < 2; ++m) {
                        uint32_t lo[4], hi[4];
                        // 16-byte piece s of row r sits at piece s ^ (r mod 8); r mod 8 = g
                        const unsigned char* wa = wb + (m * 2048 + piece[s]);
                        unpack8<DT>(*reinterpret_cast<const uint32_t*>(wa), z2[m][0], lo);
                        unpack8<DT>(*reinterpret_cast<const uint32_t*>(wa + 1024), z2[m][1], hi);
#pragma unroll
                        for (int q = 0; q < NT; ++q)
                            if (q == 0 || q < nt) {
                                if (s4 == 0) mma_16816<DT, true>(d4[m][q], lo[0], hi[0], lo[1], hi[1], xv[q].x, xv[q].y);
                                else mma_16816<DT, false>(d4[m][q], lo[0], hi[0], lo[1], hi[1], xv[q].x, xv[q].y);
                                mma_16816<DT, false>(d4[m][q], lo[2], hi[2], lo[3], hi[3], xv[q].z, xv[q].w);
                            }
                    }
                }
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int q = 0; q < NT; ++q)
                        if (q == 0 || q < nt) {
#pragma unroll
                            for (int j = 0; j < 4; ++j) acc[m][q][j] += sc[m][j >> 1] * d4[m][q][j];
                        }
            }
            __syncwarp();  // the step is read before its refill
        }
        // Join the WK parts: [warp][m][q][lane][4] floats.  Value j of lane l
        // is row l/4 + 8*(j/2), column (l%4)*2 + j%2 of the 16 x 8 fragment.
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int q = 0; q < NT; ++q)
                *reinterpret_cast<float4*>(s_red + (((warp * 2 + m) * NT + q) * 32 + lane) * 4) =
                    make_float4(acc[m][q][0], acc[m][q][1], acc[m][q][2], acc[m][q][3]);
        __syncthreads();
        // A thread sums one value of (tile, q) for both m and writes them, or their SwiGLU.
        for (int o = threadIdx.x; o < wn_count * NT * 128; o += kThreads) {
            const int q = (o >> 7) % NT, w2 = (o >> 7) / NT, l = (o & 127) >> 2, j = o & 3;
            const int tl = at.tg * wn_count + w2, col = q * 8 + (l & 3) * 2 + (j & 1), rr = (l >> 2) + (j >> 1) * 8;
            if (col >= nrows || tl >= a.tiles) continue;
            float v[2] = {0.f, 0.f};
            const float* p = s_red + ((w2 * wk * 2 * NT + q) * 32 + l) * 4 + j;
            for (int w = 0; w < wk; ++w) {
                v[0] += p[w * (2 * NT * 128)];
                v[1] += p[w * (2 * NT * 128) + NT * 128];
            }
            uint16_t* out = static_cast<uint16_t*>(a.out) + int64_t(s_slots[list0 + col]) * a.n_out;
            if (a.swiglu) {
                const int n = tl * 16 + rr;
                if (n < a.n_out) out[n] = w4_to16<DT>(__fdividef(v[0], 1.0f + __expf(-v[0])) * v[1]);
            } else {
                const int n = tl * kW4TileRows + rr;
                if (n < a.N) out[n] = w4_to16<DT>(v[0]);
                if (n + 16 < a.N) out[n + 16] = w4_to16<DT>(v[1]);
            }
        }
        __syncthreads();
        at = next;
    }
}

// ----------------------------------------------------------------- host ----

// Shared memory of a CTA of `warps` and its layout; xs: with x staged.
static size_t w4_layout(W4Args& a, int nt, bool xs, int warps) {
    const int blocks = (a.K + kW4Block - 1) / kW4Block;
    a.x_pitch = blocks * kW4Block * 2 + 64;  // 64 bytes off a multiple of 128: rows of a fragment on other banks
    size_t off = size_t(warps) * kW4Stages * kW4StageBytes;
    a.s_x = int(off);
    off += xs ? size_t(nt) * 8 * a.x_pitch : 0;
    a.s_red = int(off);
    off += size_t(warps) * 2 * nt * 128 * 4;
    a.s_tab = int(off);
    off += size_t((4 + kW4Parts) * a.E + 1) * 4 + ((size_t(a.slots) * 2 + 15) & ~size_t(15));
    return off;
}

template <int DT, int G, int NT, bool XS, int W>
static cudaError_t launch_w4(const CUtensorMap& map, W4Args a, int served, cudaStream_t s) {
    const size_t smem = w4_layout(a, NT, XS, W);
    auto kern = expert_linear_w4_kernel<DT, G, NT, XS, W>;
    static SmemLimit limit;
    const cudaError_t err = limit.open(reinterpret_cast<const void*>(kern));
    if (err != cudaSuccess) return err;
    int64_t grid = 16 / W * device_sm_count();
    // Warps that share a tile's k: few, as each joint costs about as much as a
    // step, but so that every CTA gets several units, and none that loses more
    // than an eighth of its steps to an uneven split.  Shared 1 / 2 / 4 / 8 ways,
    // us in captured graphs: one token, 4 experts of 2816 x 2048 (8 blocks of k;
    // 8 taken) 13.8 / 8.8 / 8.4 / 7.6; one row of 4096 x 4096 (8) 23 / 13.7 / 8.7 /
    // 6.2; 64 tokens (4) 51.1 / 51.1 / 51.2 / 54.3; 147 tokens, 2048 x 1408 (6 blocks;
    // 2) 67 / 63 / 67 / 72.  The bound on uneven splits is for batches: one
    // token there takes 9.4 in 2 parts and would take 7.0 in 8.
    const int blocks = (a.K + kW4Block - 1) / kW4Block;
    a.wk = 8;
    while (a.wk > 1 && (8 * blocks < 7 * a.wk * ((blocks + a.wk - 1) / a.wk) ||
                        int64_t(a.tiles) * served * a.wk > 16 * W * grid))
        a.wk /= 2;
    a.units = (a.tiles + W / a.wk - 1) / (W / a.wk);
    const int64_t most = int64_t(a.units) * (a.slots < a.E ? a.slots : a.E + a.slots / 8);
    if (grid > most) grid = most;
    kern<<<unsigned(grid), W * 32, smem, s>>>(map, a);
    return cudaGetLastError();
}

template <int DT, int G>
static cudaError_t run_w4(const CUtensorMap& map, W4Args a, cudaStream_t s) {
    const int served = a.slots < a.E ? a.slots : a.E;  // experts that may have work
    // Rows served per read of the weights: 8, or 16 when experts have more than
    // 8 on average and they fit (with 16 warps where those fit too).
    if (a.slots > 8 * served) {
        if (w4_layout(a, 2, true, 16) <= kW4SmemLimit) return launch_w4<DT, G, 2, true, 16>(map, a, served, s);
        if (w4_layout(a, 2, true, 8) <= kW4SmemLimit) return launch_w4<DT, G, 2, true, 8>(map, a, served, s);
    }
    if (w4_layout(a, 1, true, 8) <= kW4SmemLimit) return launch_w4<DT, G, 1, true, 8>(map, a, served, s);
    return launch_w4<DT, G, 1, false, 8>(map, a, served, s);
}

// 3-D map over w_q [E, N, d/2] bytes; box = 128 bytes x 16 rows of one expert, 128B swizzle.
static bool make_map_w4(CUtensorMap* map, const void* base, int E, int N, int K) {
    const cuuint64_t dims[3] = {cuuint64_t(K / 2), cuuint64_t(N), cuuint64_t(E)};
    const cuuint64_t strides[2] = {cuuint64_t(K / 2), cuuint64_t(K / 2) * cuuint64_t(N)};
    const cuuint32_t box[3] = {128u, 16u, 1u};
    return encode_tiled(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, base, dims, strides, box);
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
    if (d > kW4MaxSize || N > kW4MaxSize)
        return fail(MOE_B200_ERR_UNSUPPORTED, "expert_linear_w4: d and N may be at most %d", kW4MaxSize);
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
    if (inside_element({asgn}, 4)) return fail(MOE_B200_ERR_INVALID_ARG, "expert_linear_w4: asgn must be 4-byte aligned");
    const int64_t slots = int64_t(T) * K, weights = int64_t(E) * N * d;
    if (overlaps_any(whole(out, 2 * slots * (act == MOE_B200_ACT_SWIGLU ? N / 2 : N)),
                     {whole(x, 2 * int64_t(d) * (x_per_slot ? slots : T)), whole(asgn, 4 * slots), whole(w_q, weights / 2),
                      whole(w_scale, weights / group * 2), whole(w_zero, weights / group)}))
        return fail(MOE_B200_ERR_INVALID_ARG, "expert_linear_w4: out overlaps an operand");
    uint32_t* st = device_status_word();
    if (!st) return fail(MOE_B200_ERR_CUDA, "expert_linear_w4: device status word unavailable");
    W4Args a{};
    a.x = x;
    a.asgn = asgn;
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
    CUtensorMap map;
    if (!make_map_w4(&map, w_q, E, N, d)) return fail(MOE_B200_ERR_CUDA, "expert_linear_w4: cuTensorMapEncodeTiled failed");
    const bool bf = dtype == MOE_B200_BF16;
    cudaError_t err;
    if (group == 32) err = bf ? run_w4<MOE_B200_BF16, 32>(map, a, s) : run_w4<MOE_B200_F16, 32>(map, a, s);
    else if (group == 64) err = bf ? run_w4<MOE_B200_BF16, 64>(map, a, s) : run_w4<MOE_B200_F16, 64>(map, a, s);
    else err = bf ? run_w4<MOE_B200_BF16, 128>(map, a, s) : run_w4<MOE_B200_F16, 128>(map, a, s);
    return err == cudaSuccess ? MOE_B200_OK : cuda_fail(err, "expert_linear_w4 launch");
}
