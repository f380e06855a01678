// block_norm.cu -- RMS norms behind and before a block of a residual network,
// fused with the block's gate and residual scale, forward and backward.
//
//   rms(v) = v * rsqrt(mean(v^2) + eps)                       (per row, d columns)
//   z  = rms(y) * w_post        (w_post NULL: z = y)
//   r' = r + scale * gate * z   (y NULL: r' = r; gate NULL: 1)
//   n  = rms(r') * w_pre        (w_pre NULL: none)
// Backward, at the stored r', for the gradients dr' and dn:
//   c  = rsqrt(mean(r'^2) + eps),  u = dn * w_pre
//   ds = dr' + c * (u - r' * c^2 * mean(u * r')),   dr = ds
//   a  = rsqrt(mean(y^2) + eps),  yh = a * y,  q = scale * gate * ds,  v = q * w_post
//   dy = a * (v - yh * mean(v * yh))
//   dw_pre = sum_t dn * c * r',  dw_post = sum_t q * yh,  dgate = scale * ds * z (summed where it was broadcast)
//
// Both directions are bound by memory: every row is read once and every result
// is written once; all sums are fp32, outputs are rounded once (n comes from
// the unrounded r').
//
// A row belongs to a warp or to a CTA, so that its sums are one or two short
// reductions, and a thread to fixed columns.  Rows come through a ring of
// shared-memory stages that bulk copies fill: loads in flight cost no registers.
// The instructions count nearly as much as the bytes (per element 4 to 7 values
// are unpacked, and 12 to 30 fp32 operations done): conversions are packed, the
// backward works on pairs of fp32, calls of the usual form have kernels
// without branches.  Barriers are whole-CTA ones: a named barrier with a
// register for its number reserves 16 of them, which left 25% occupancy.
// Measured on one B200 (bf16, cases back to back): forward with both norms and
// a gate per token, 16384 x 2048: 47 us, 5.7 TB/s, 0.87 of the copy bandwidth;
// backward with a channel gate, 8192 x 4096: 83 us, 4.8 TB/s (77 us for the
// rows, where 2.3 instructions a cycle of 4 are issued, and the rest for
// adding up the CTAs' column sums).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <initializer_list>
#include <type_traits>

#include "common.cuh"

namespace moe_b200 {

int fail(int code, const char* fmt, ...);
int cuda_fail(cudaError_t err, const char* where);

constexpr int kNormMaxD = 16384;

enum { kGateNone = MOE_B200_GATE_NONE, kGateToken = MOE_B200_GATE_TOKEN, kGateChannel = MOE_B200_GATE_CHANNEL,
       kGateFull = MOE_B200_GATE_FULL };

// One 16-bit word <-> fp32.
template <int DT> __device__ __forceinline__ float from16(uint16_t b) {
    return DT == MOE_B200_BF16 ? __uint_as_float(uint32_t(b) << 16) : __half2float(__ushort_as_half(b));
}
template <int DT> __device__ __forceinline__ uint16_t to16(float f) {
    return DT == MOE_B200_BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(f)) : __half_as_ushort(__float2half_rn(f));
}

// Two fp32 values to a word of two 16-bit ones.
template <int DT> __device__ __forceinline__ uint32_t pack16(float a, float b) {
    if (DT == MOE_B200_BF16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// Pairs of fp32 values in one 64-bit register: sm_100a multiplies and adds two
// at a time (each half rounded as the single operation).
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 pair(float lo, float hi) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void split(f32x2 v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float sum2(f32x2 v) {
    float lo, hi;
    split(v, lo, hi);
    return lo + hi;
}

// A row's columns as a thread holds them: V chunks of 8.  Aligned rows
// (ALIGNED: d, strides and pointers in 16-byte steps) give a thread 8
// consecutive columns per chunk, one 16-byte access (two for fp32); other rows
// are read element by element, neighbouring threads on neighbouring columns.
template <bool ALIGNED>
__device__ __forceinline__ int col_of(int chunk, int j, int t, int nt) {
    return ALIGNED ? (chunk * nt + t) * 8 + j : (chunk * 8 + j) * nt + t;
}

// Eight columns of a chunk as raw words: 16-bit rows use w[0..3] (two columns
// a word), fp32 rows w[0..7].  Aligned rows end with a chunk, and the caller
// asks chunk_in() once per chunk; of other rows, columns past d read as zero,
// which adds nothing to any sum.
template <bool ALIGNED> __device__ __forceinline__ bool chunk_in(int chunk, int t, int nt, int d) {
    return !ALIGNED || (chunk * nt + t) * 8 < d;
}
template <bool F32> struct Raw {
    uint32_t w[F32 ? 8 : 4];
};

template <bool ALIGNED, bool F32>
__device__ __forceinline__ Raw<F32> load_raw(const void* row, int chunk, int t, int nt, int d) {
    Raw<F32> r;
    if (ALIGNED) {
        const uint4* p = reinterpret_cast<const uint4*>(static_cast<const char*>(row) +
                                                        col_of<true>(chunk, 0, t, nt) * (F32 ? 4 : 2));
#pragma unroll
        for (int h = 0; h < (F32 ? 2 : 1); ++h) {
            const uint4 v = p[h];
            r.w[4 * h] = v.x, r.w[4 * h + 1] = v.y, r.w[4 * h + 2] = v.z, r.w[4 * h + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int c = col_of<false>(chunk, j, t, nt);
            uint32_t v = 0;
            if (c < d) v = F32 ? static_cast<const uint32_t*>(row)[c] : uint32_t(static_cast<const uint16_t*>(row)[c]);
            if (F32) r.w[j % (F32 ? 8 : 4)] = v;
            else if (j & 1) r.w[(j >> 1) % 4] |= v << 16;
            else r.w[(j >> 1) % 4] = v;
        }
    }
    return r;
}

template <int DT, bool F32>
__device__ __forceinline__ float raw_get(const Raw<F32>& r, int j) {
    if (F32) return __uint_as_float(r.w[j % (F32 ? 8 : 4)]);
    const uint32_t w = r.w[(j >> 1) % 4];
    if (DT == MOE_B200_BF16) return __uint_as_float((j & 1) ? (w & 0xffff0000u) : (w << 16));
    return from16<DT>(uint16_t((j & 1) ? (w >> 16) : w));
}

// Columns 2j and 2j + 1 of a chunk as a pair.
template <int DT, bool F32>
__device__ __forceinline__ f32x2 raw_pair(const Raw<F32>& r, int j) {
    return pair(raw_get<DT, F32>(r, 2 * j), raw_get<DT, F32>(r, 2 * j + 1));
}

// Eight fp32 values to a row of 16-bit or fp32 columns.
template <int DT, bool ALIGNED, bool F32>
__device__ __forceinline__ void store8(void* row, const float (&x)[8], int chunk, int t, int nt, int d) {
    if (ALIGNED) {
        uint4* p = reinterpret_cast<uint4*>(static_cast<char*>(row) + col_of<true>(chunk, 0, t, nt) * (F32 ? 4 : 2));
        if (F32) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
                st_v4(p + h, make_uint4(__float_as_uint(x[4 * h]), __float_as_uint(x[4 * h + 1]),
                                        __float_as_uint(x[4 * h + 2]), __float_as_uint(x[4 * h + 3])));
        } else {
            uint32_t o[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = pack16<DT>(x[2 * j], x[2 * j + 1]);
            st_v4(p, make_uint4(o[0], o[1], o[2], o[3]));
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int c = col_of<false>(chunk, j, t, nt);
            if (c < d) {
                if (F32) static_cast<float*>(row)[c] = x[j];
                else static_cast<uint16_t*>(row)[c] = to16<DT>(x[j]);
            }
        }
    }
}

// Sums of N <= 4 values over a row's threads: a warp (WARP) or the whole CTA,
// the same bits in every thread.  `red` holds two buffers of [N][warps] floats
// (the number of warps rounded up to 4, the rest zeros); `phase` alternates
// them, so one barrier a reduction is enough: a buffer is written again only
// after the next reduction's barrier, which no thread passes before it has
// read this one.
constexpr int kRedFloats = 2 * 4 * 32;
template <bool WARP, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float* red, int& phase) {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    if (WARP) return;
    const int nw = ((blockDim.x >> 5) + 3) & ~3;
    float* b = red + phase * (4 * 32);
    phase ^= 1;
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) b[i * 32 + (threadIdx.x >> 5)] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        float4 s = *reinterpret_cast<const float4*>(b + i * 32);
        for (int w = 4; w < nw; w += 4) {
            const float4 u = *reinterpret_cast<const float4*>(b + i * 32 + w);
            s.x += u.x, s.y += u.y, s.z += u.z, s.w += u.w;
        }
        v[i] = (s.x + s.y) + (s.z + s.w);
    }
}
// Zeros for the places of warps that do not exist; before the first row_sum.
template <bool WARP> __device__ __forceinline__ void row_sum_init(float* red) {
    if (!WARP) {
        for (int i = threadIdx.x; i < kRedFloats; i += blockDim.x) red[i] = 0.f;
        __syncthreads();
    }
}

template <int DT, bool ALIGNED, bool F32>
__device__ __forceinline__ void store8(void* row, const f32x2 (&x)[4], int chunk, int t, int nt, int d) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) split(x[j], v[2 * j], v[2 * j + 1]);
    store8<DT, ALIGNED, F32>(row, v, chunk, t, nt, d);
}

struct NormArgs {
    const void *y, *residual, *w_post, *w_pre, *gate;
    int64_t y_stride, res_stride;  // elements
    int gate_form;
    float scale, eps;
    int T, d;
    void *residual_out, *normed;
    // Ring of rows in shared memory (RING): rows in flight, bytes of a staged
    // row and where y and a full gate lie in it (the residual comes first).
    int stages, row_bytes, off_y, off_gate;
    uint32_t* status;
};

constexpr int kNormStages = 4;  // rows in flight, at most

// What a call consists of, where it is known when compiling (the forms that
// models run all the time); kFormAny asks the arguments.  A column gate is one
// per channel or per element: its rows lie 0 or d apart.
enum { kFormAny = 0, kFormFull = 1, kFormFullColGate = 2, kFormAddNorm = 3, kFormNorm = 4 };
template <int FORM> struct Form {
    static constexpr bool any = FORM == kFormAny;
    static constexpr bool y = FORM != kFormNorm, post = FORM == kFormFull || FORM == kFormFullColGate;
    static constexpr bool col = FORM == kFormFullColGate;
};

// A row belongs to one warp (WARP: CTAs of 4 rows) or to a CTA; each thread
// holds V chunks of 8 columns.  The grid fits the card and walks the rows; the
// weights stay packed in registers.  RING: rows come through a ring of shared-
// memory stages filled by bulk copies some rows ahead; otherwise (rows not in
// 16-byte steps, too wide, or at most one row a CTA) by plain loads.
template <int DT, bool RES32, bool ALIGNED, bool RING, bool WARP, int V, int MAXT, int FORM>
__global__ void __launch_bounds__(MAXT, MAXT <= 256 ? 768 / MAXT : 1)  // 80 registers: 24 warps an SM
block_norm_kernel(const NormArgs a) {
    using F = Form<FORM>;
    extern __shared__ __align__(128) unsigned char s_dyn[];
    __shared__ __align__(16) float s_red[kRedFloats];
    __shared__ uint64_t s_full[4 * kNormStages], s_empty[4 * kNormStages];
    const bool has_y = F::any ? a.y != nullptr : F::y, has_post = F::any ? a.w_post != nullptr : F::post;
    const bool has_col = F::any ? a.gate_form >= kGateChannel : F::col, has_pre = F::any ? a.w_pre != nullptr : true;
    const int nt = WARP ? 32 : blockDim.x, t = WARP ? (threadIdx.x & 31) : threadIdx.x;
    const int groups = WARP ? blockDim.x >> 5 : 1, group = WARP ? threadIdx.x >> 5 : 0;
    const int64_t step = int64_t(gridDim.x) * groups;
    const int64_t row0 = int64_t(blockIdx.x) * groups + group;
    row_sum_init<WARP>(s_red);
    if (row0 >= a.T) return;
    int phase = 0;
    const int d = a.d;
    const float inv_d = 1.0f / float(d);
    constexpr int kRes = RES32 ? 4 : 2;
    const bool gate_rows = has_col && a.gate_form == kGateFull;
    uint64_t *full = s_full + group * kNormStages, *empty = s_empty + group * kNormStages;
    unsigned char* ring = s_dyn + group * a.stages * a.row_bytes;

    // Rows of the operands: of the next one to fetch.
    const char* res_row = static_cast<const char*>(a.residual) + row0 * a.res_stride * kRes;
    const uint16_t* y_row = static_cast<const uint16_t*>(a.y) + row0 * a.y_stride;
    const uint16_t* g_row = static_cast<const uint16_t*>(a.gate) + (gate_rows ? row0 * d : 0);
    auto next_rows = [&]() {
        res_row += step * a.res_stride * kRes;
        if (has_y) y_row += step * a.y_stride;
        if (gate_rows) g_row += step * d;
    };
    auto fill = [&](int s) {  // one thread
        unsigned char* p = ring + s * a.row_bytes;
        mbar_arrive_expect_tx(full + s, a.row_bytes);
        bulk_g2s(p, res_row, d * kRes, full + s);
        if (has_y) bulk_g2s(p + a.off_y, y_row, d * 2, full + s);
        if (gate_rows) bulk_g2s(p + a.off_gate, g_row, d * 2, full + s);
        next_rows();
    };
    if (RING) {
        if (t == 0) {
            for (int s = 0; s < a.stages; ++s) {
                mbar_init(full + s, 1);
                mbar_init(empty + s, nt >> 5);
            }
            mbar_fence_init();
        }
        if (WARP) __syncwarp();
        else __syncthreads();
        if (t == 0)
            for (int s = 0; s < a.stages; ++s)
                if (row0 + s * step < a.T) fill(s);
    }
    Raw<false> wp[V], wn[V], gc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        if (!chunk_in<ALIGNED>(i, t, nt, d)) continue;
        if (has_post) wp[i] = load_raw<ALIGNED, false>(a.w_post, i, t, nt, d);
        if (has_pre) wn[i] = load_raw<ALIGNED, false>(a.w_pre, i, t, nt, d);
        if (has_col && !gate_rows) gc[i] = load_raw<ALIGNED, false>(a.gate, i, t, nt, d);
    }
    int st = 0;
    uint32_t ph = 0;
    char* res_out = static_cast<char*>(a.residual_out) + row0 * d * kRes;
    uint16_t* norm_out = static_cast<uint16_t*>(a.normed) + row0 * d;
    for (int64_t row = row0; row < a.T; row += step) {
        const unsigned char* p = ring + st * a.row_bytes;
        if (RING) {
            // Refill the stage of the row before, once all its warps have read it.
            if (t == 0 && row > row0 && row + (a.stages - 1) * step < a.T) {
                const int prev = st == 0 ? a.stages - 1 : st - 1;
                if (!mbar_wait(empty + prev, st == 0 ? ph ^ 1u : ph)) atomicOr(a.status, MOE_B200_DEV_WAIT_TIMEOUT);
                fill(prev);
            }
            if (!mbar_wait(full + st, ph)) atomicOr(a.status, MOE_B200_DEV_WAIT_TIMEOUT);
        }
        float r[V][8], z[V][8];
        float s[1] = {0.f};
        float f = a.scale;
        if (has_y && !has_col && a.gate_form == kGateToken) f *= from16<DT>(static_cast<const uint16_t*>(a.gate)[row]);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (!chunk_in<ALIGNED>(i, t, nt, d)) continue;
            const Raw<RES32> res = RING ? load_raw<ALIGNED, RES32>(p, i, t, nt, d) : load_raw<ALIGNED, RES32>(res_row, i, t, nt, d);
            Raw<false> yr, gr;
            if (has_y) yr = RING ? load_raw<ALIGNED, false>(p + a.off_y, i, t, nt, d) : load_raw<ALIGNED, false>(y_row, i, t, nt, d);
            if (has_col) {
                gr = gc[i];
                if (gate_rows)
                    gr = RING ? load_raw<ALIGNED, false>(p + a.off_gate, i, t, nt, d) : load_raw<ALIGNED, false>(g_row, i, t, nt, d);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) r[i][j] = raw_get<DT, RES32>(res, j);
            if (has_y) {
#pragma unroll
                for (int j = 0; j < 8; ++j) z[i][j] = raw_get<DT, false>(yr, j);
                if (has_post) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        s[0] += z[i][j] * z[i][j];
                        z[i][j] *= raw_get<DT, false>(wp[i], j);
                    }
                }
                if (has_col) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) z[i][j] *= raw_get<DT, false>(gr, j);
                }
            }
        }
        if (RING) {  // the stage is read
            __syncwarp();
            if ((threadIdx.x & 31) == 0) mbar_arrive(empty + st);
            if (++st == a.stages) st = 0, ph ^= 1;
        } else {
            next_rows();
        }
        if (has_y) {
            if (has_post) {
                row_sum<WARP>(s, s_red, phase);
                f *= rsqrtf(s[0] * inv_d + a.eps);
            }
#pragma unroll
            for (int i = 0; i < V; ++i) {
                if (!chunk_in<ALIGNED>(i, t, nt, d)) continue;
#pragma unroll
                for (int j = 0; j < 8; ++j) r[i][j] += z[i][j] * f;
                store8<DT, ALIGNED, RES32>(res_out, r[i], i, t, nt, d);
            }
            res_out += step * d * kRes;
        }
        if (has_pre) {
            s[0] = 0.f;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                if (!chunk_in<ALIGNED>(i, t, nt, d)) continue;
#pragma unroll
                for (int j = 0; j < 8; ++j) s[0] += r[i][j] * r[i][j];
            }
            row_sum<WARP>(s, s_red, phase);
            const float c = rsqrtf(s[0] * inv_d + a.eps);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                if (!chunk_in<ALIGNED>(i, t, nt, d)) continue;
#pragma unroll
                for (int j = 0; j < 8; ++j) r[i][j] *= c * raw_get<DT, false>(wn[i], j);
                store8<DT, ALIGNED, false>(norm_out, r[i], i, t, nt, d);
            }
            norm_out += step * d;
        }
    }
}

struct NormGradArgs {
    const void *d_res_out, *d_normed, *res_out, *y, *w_post, *w_pre, *gate;
    int64_t y_stride, res_stride;
    int gate_form;
    float scale, eps;
    int T, d;
    void *d_res, *d_y, *d_gate;
    // Column sums of each CTA: up to three vectors of d floats, [vector][CTA][d].
    float* part;
    int sum_pre, sum_post, sum_gate;  // index of the vector, or -1
    // Ring of rows in shared memory (RING): bytes of a staged row and where its
    // parts lie in it (-1: absent).
    int row_bytes, off_ds, off_rr, off_dn, off_y, off_gate;
    int stages, off_w;  // rows in flight; the weights' copies (w_pre, w_post, channel gate) behind the ring
    uint32_t* status;
};

// Rows are dealt to a grid that fits the card, so that each thread keeps its
// columns' sums over its rows in registers and the column gradients cost one
// row of partial sums a CTA.  RING: the rows come through a ring of shared-
// memory stages filled by bulk copies some rows ahead, which costs no registers,
// and the weights are copied there once; otherwise (rows not in 16-byte steps, or too wide for the ring)
// they are read from global memory at each of the two uses.
// GATE: the gate's form, or -1 where the call is of a rarer kind (a norm or
// the residual's gradient missing) and the arguments are asked.
template <int DT, bool RES32, bool ALIGNED, bool RING, bool WARP, int V, int MAXT, int GATE>
__global__ void __launch_bounds__(MAXT)
block_norm_backward_kernel(const NormGradArgs a) {
    extern __shared__ __align__(128) unsigned char s_dyn[];
    __shared__ __align__(16) float s_red[kRedFloats];
    __shared__ uint64_t s_full[4 * kNormStages], s_empty[4 * kNormStages];
    constexpr bool kAny = GATE < 0;
    const bool has_y = kAny ? a.y != nullptr : true, has_post = kAny ? a.w_post != nullptr : true;
    const bool has_pre = kAny ? a.w_pre != nullptr : true, has_ds = kAny ? a.d_res_out != nullptr : true;
    const int gate_form = kAny ? a.gate_form : GATE;
    const int nt = WARP ? 32 : blockDim.x, t = WARP ? (threadIdx.x & 31) : threadIdx.x;
    const int groups = WARP ? blockDim.x >> 5 : 1, group = WARP ? threadIdx.x >> 5 : 0;
    const int64_t step = int64_t(gridDim.x) * groups;
    const int64_t row0 = int64_t(blockIdx.x) * groups + group;
    int phase = 0;
    const int d = a.d;
    const float inv_d = 1.0f / float(d);
    constexpr int kRes = RES32 ? 4 : 2;
    uint64_t *full = s_full + group * kNormStages, *empty = s_empty + group * kNormStages;
    unsigned char* ring = s_dyn + size_t(group) * a.stages * a.row_bytes;
    unsigned char *s_wpre = s_dyn + a.off_w, *s_wpost = s_wpre + (has_pre ? d * 2 : 0), *s_wgate = s_wpost + (has_post ? d * 2 : 0);

    auto ds_row = [&](int64_t r) { return static_cast<const char*>(a.d_res_out) + r * d * kRes; };
    auto rr_row = [&](int64_t r) { return static_cast<const char*>(a.res_out) + r * a.res_stride * kRes; };
    auto dn_row = [&](int64_t r) { return static_cast<const char*>(a.d_normed) + r * d * 2; };
    auto y_row = [&](int64_t r) { return static_cast<const char*>(a.y) + r * a.y_stride * 2; };
    auto g_row = [&](int64_t r) { return static_cast<const char*>(a.gate) + r * d * 2; };
    auto fill = [&](int64_t r, int s) {  // one thread
        unsigned char* p = ring + size_t(s) * a.row_bytes;
        mbar_arrive_expect_tx(full + s, a.row_bytes);
        if (has_ds) bulk_g2s(p + a.off_ds, ds_row(r), d * kRes, full + s);
        if (has_pre) bulk_g2s(p + a.off_rr, rr_row(r), d * kRes, full + s);
        if (has_pre) bulk_g2s(p + a.off_dn, dn_row(r), d * 2, full + s);
        if (has_y) bulk_g2s(p + a.off_y, y_row(r), d * 2, full + s);
        if (gate_form == kGateFull) bulk_g2s(p + a.off_gate, g_row(r), d * 2, full + s);
    };
    row_sum_init<WARP>(s_red);
    if (RING) {
        if (t == 0) {
            for (int s = 0; s < a.stages; ++s) {
                mbar_init(full + s, 1);
                mbar_init(empty + s, nt >> 5);
            }
            mbar_fence_init();
        }
        for (int c = threadIdx.x * 8; c < d; c += blockDim.x * 8) {
            if (has_pre) *reinterpret_cast<uint4*>(s_wpre + c * 2) = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.w_pre) + c);
            if (has_post) *reinterpret_cast<uint4*>(s_wpost + c * 2) = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.w_post) + c);
            if (gate_form == kGateChannel) *reinterpret_cast<uint4*>(s_wgate + c * 2) = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.gate) + c);
        }
        __syncthreads();
        if (t == 0)
            for (int s = 0; s < a.stages; ++s)
                if (row0 + s * step < a.T) fill(row0 + s * step, s);
    }

    // Column sums.  A channel gate and w_post share one: with A = sum ds yh,
    // d_w_post = scale * gate * A and d_gate = scale * w_post * A.
    f32x2 s_pre[V][4], s_post[V][4];
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s_pre[i][j] = s_post[i][j] = 0;

    uint32_t n = 0;
    int st = 0;         // ring stage and its phase
    uint32_t ph = 0;
    char* dres_out = static_cast<char*>(a.d_res) + row0 * d * kRes;
    uint16_t* dy_out = static_cast<uint16_t*>(a.d_y) + row0 * d;
    uint16_t* dg_out = static_cast<uint16_t*>(a.d_gate) + row0 * d;
    for (int64_t row = row0; row < a.T; row += step, ++n) {
        const unsigned char* p = ring + st * a.row_bytes;
        if (RING) {
            // Refill the stage of the row before, once all its warps are through with it.
            const int64_t ahead = row + (a.stages - 1) * step;
            if (t == 0 && n > 0 && ahead < a.T) {
                const int prev = st == 0 ? a.stages - 1 : st - 1;
                if (!mbar_wait(empty + prev, st == 0 ? ph ^ 1u : ph)) atomicOr(a.status, MOE_B200_DEV_WAIT_TIMEOUT);
                fill(ahead, prev);
            }
            if (!mbar_wait(full + st, ph)) atomicOr(a.status, MOE_B200_DEV_WAIT_TIMEOUT);
        }
        auto get16 = [&](int off, const char* g, int i) {
            return RING ? load_raw<ALIGNED, false>(p + off, i, t, nt, d) : load_raw<ALIGNED, false>(g, i, t, nt, d);
        };
        auto getres = [&](int off, const char* g, int i) {
            return RING ? load_raw<ALIGNED, RES32>(p + off, i, t, nt, d) : load_raw<ALIGNED, RES32>(g, i, t, nt, d);
        };
        auto getw = [&](const unsigned char* s, const void* g, int i) {
            return RING ? load_raw<ALIGNED, false>(s, i, t, nt, d) : load_raw<ALIGNED, false>(g, i, t, nt, d);
        };
        f32x2 p_rr = 0, p_ur = 0, p_yy = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (!chunk_in<ALIGNED>(i, t, nt, d)) continue;
            if (has_pre) {
                const Raw<false> wn = getw(s_wpre, a.w_pre, i);
                const Raw<false> dn = get16(a.off_dn, dn_row(row), i);
                const Raw<RES32> rr = getres(a.off_rr, rr_row(row), i);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const f32x2 r = raw_pair<DT, RES32>(rr, j);
                    p_rr = fma2(r, r, p_rr);
                    p_ur = fma2(mul2(raw_pair<DT, false>(dn, j), raw_pair<DT, false>(wn, j)), r, p_ur);
                }
            }
            if (has_post) {
                const Raw<false> yr = get16(a.off_y, y_row(row), i);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const f32x2 y = raw_pair<DT, false>(yr, j);
                    p_yy = fma2(y, y, p_yy);
                }
            }
        }
        float sums[3] = {sum2(p_rr), sum2(p_ur), sum2(p_yy)};  // sum r'^2, sum u r', sum y^2
        if (has_pre || has_post) row_sum<WARP>(sums, s_red, phase);
        const float c = rsqrtf(sums[0] * inv_d + a.eps);
        const float k = sums[1] * inv_d * c * c;  // ds = dr' + c dn w_pre - (c r') k
        const float post = has_post ? rsqrtf(sums[2] * inv_d + a.eps) : 1.0f;
        const float gate_t =
            gate_form == kGateToken ? from16<DT>(static_cast<const uint16_t*>(a.gate)[row]) : 1.0f;
        // q is first ds, then ds * (column gate) * w_post, without the row's scale f
        const float f = a.scale * gate_t;
        const float fa = gate_form == kGateChannel ? post : f * post;  // of the sum behind w_post
        const f32x2 c2 = pair(c, c), k2 = pair(-k, -k), fa2 = pair(fa, fa), dg2 = pair(a.scale * post, a.scale * post);
        f32x2 p_qy = 0;
        f32x2 q[V][4];
        Raw<false> yr[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (!chunk_in<ALIGNED>(i, t, nt, d)) continue;
            if (has_ds) {
                const Raw<RES32> ds = getres(a.off_ds, ds_row(row), i);
#pragma unroll
                for (int j = 0; j < 4; ++j) q[i][j] = raw_pair<DT, RES32>(ds, j);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) q[i][j] = 0;
            }
            if (has_pre) {
                const Raw<false> wn = getw(s_wpre, a.w_pre, i);
                const Raw<false> dn = get16(a.off_dn, dn_row(row), i);
                const Raw<RES32> rr = getres(a.off_rr, rr_row(row), i);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const f32x2 rc = mul2(raw_pair<DT, RES32>(rr, j), c2), dnj = raw_pair<DT, false>(dn, j);
                    s_pre[i][j] = fma2(dnj, rc, s_pre[i][j]);
                    q[i][j] = fma2(c2, mul2(dnj, raw_pair<DT, false>(wn, j)), fma2(rc, k2, q[i][j]));
                }
            }
            store8<DT, ALIGNED, RES32>(dres_out, q[i], i, t, nt, d);
            if (has_y) {
                yr[i] = get16(a.off_y, y_row(row), i);
                Raw<false> wp, gr;
                if (has_post) wp = getw(s_wpost, a.w_post, i);
                if (gate_form == kGateChannel) gr = getw(s_wgate, a.gate, i);
                if (gate_form == kGateFull) {
                    gr = get16(a.off_gate, g_row(row), i);
                    f32x2 dg[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        dg[j] = mul2(mul2(q[i][j], dg2), raw_pair<DT, false>(yr[i], j));
                        if (has_post) dg[j] = mul2(dg[j], raw_pair<DT, false>(wp, j));
                        q[i][j] = mul2(q[i][j], raw_pair<DT, false>(gr, j));
                    }
                    store8<DT, ALIGNED, false>(dg_out, dg, i, t, nt, d);
                }
                if (has_post || gate_form == kGateChannel) {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        s_post[i][j] = fma2(q[i][j], mul2(fa2, raw_pair<DT, false>(yr[i], j)), s_post[i][j]);
                }
                if (gate_form == kGateChannel) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) q[i][j] = mul2(q[i][j], raw_pair<DT, false>(gr, j));
                }
                if (has_post) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) q[i][j] = mul2(q[i][j], raw_pair<DT, false>(wp, j));
                }
                if (has_post || gate_form == kGateToken) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) p_qy = fma2(q[i][j], raw_pair<DT, false>(yr[i], j), p_qy);
                }
            }
        }
        if (RING) {  // the stage is read
            __syncwarp();
            if ((threadIdx.x & 31) == 0) mbar_arrive(empty + st);
            if (++st == a.stages) st = 0, ph ^= 1;
        }
        if (has_y) {
            float qy[1] = {sum2(p_qy)};  // sum q y
            if (has_post || gate_form == kGateToken) row_sum<WARP>(qy, s_red, phase);
            if (gate_form == kGateToken && t == 0) static_cast<float*>(a.d_gate)[row] = a.scale * post * qy[0];
            const float fp = f * post, m = -qy[0] * inv_d * post * post * fp;
            const f32x2 fp2 = pair(fp, fp), m2 = pair(m, m), f2 = pair(f, f);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                if (!chunk_in<ALIGNED>(i, t, nt, d)) continue;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    q[i][j] = has_post ? fma2(fp2, q[i][j], mul2(raw_pair<DT, false>(yr[i], j), m2)) : mul2(q[i][j], f2);
                store8<DT, ALIGNED, false>(dy_out, q[i], i, t, nt, d);
            }
        }
        dres_out += step * d * kRes;
        dy_out += step * d;
        dg_out += step * d;
    }

    // Column sums: the CTA's rows side by side add up through shared memory in
    // warp order, then the CTA writes its rows of partial sums.
    __syncthreads();  // the ring is free
    float* s_col = reinterpret_cast<float*>(s_dyn);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        if (which == 0 ? a.sum_pre < 0 : a.sum_post < 0 && a.sum_gate < 0) continue;
        float s[V][8];
#pragma unroll
        for (int i = 0; i < V; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) split(which == 0 ? s_pre[i][j] : s_post[i][j], s[i][2 * j], s[i][2 * j + 1]);
        for (int g = 0; g < groups - 1; ++g) {
            if (group == g) {
#pragma unroll
                for (int i = 0; i < V; ++i)
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int col = col_of<ALIGNED>(i, j, t, nt);
                        if (col < d) s_col[col] = g == 0 ? s[i][j] : s_col[col] + s[i][j];
                    }
            }
            __syncthreads();
        }
        if (group == groups - 1) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                if (!chunk_in<ALIGNED>(i, t, nt, d)) continue;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int col = col_of<ALIGNED>(i, j, t, nt);
                    if (groups > 1 && col < d) s[i][j] += s_col[col];
                }
                auto row_of = [&](int vec) { return a.part + (int64_t(vec) * gridDim.x + blockIdx.x) * d; };
                if (which == 0) {
                    store8<DT, ALIGNED, true>(row_of(a.sum_pre), s[i], i, t, nt, d);
                } else if (a.sum_gate < 0) {
                    store8<DT, ALIGNED, true>(row_of(a.sum_post), s[i], i, t, nt, d);
                } else {
                    const Raw<false> gr = load_raw<ALIGNED, false>(a.gate, i, t, nt, d);
                    float v[8];
                    if (has_post) {
                        const Raw<false> wp = load_raw<ALIGNED, false>(a.w_post, i, t, nt, d);
#pragma unroll
                        for (int j = 0; j < 8; ++j) v[j] = a.scale * raw_get<DT, false>(gr, j) * s[i][j];
                        store8<DT, ALIGNED, true>(row_of(a.sum_post), v, i, t, nt, d);
#pragma unroll
                        for (int j = 0; j < 8; ++j) s[i][j] *= raw_get<DT, false>(wp, j);
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] = a.scale * s[i][j];
                    store8<DT, ALIGNED, true>(row_of(a.sum_gate), v, i, t, nt, d);
                }
            }
        }
        __syncthreads();
    }
    pdl_launch_dependents();
}

// Adds the CTAs' partial rows: a CTA per 32 columns of one vector, its 32
// warps split the rows; each output is a fixed-order sum.
__global__ void __launch_bounds__(1024)
block_norm_columns_kernel(const float* __restrict__ part, int nparts, int d, float* out0, float* out1, float* out2) {
    __shared__ float s[32][33];
    pdl_wait_primary();
    float* out = blockIdx.y == 0 ? out0 : blockIdx.y == 1 ? out1 : out2;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, col = blockIdx.x * 32 + lane;
    const float* p = part + int64_t(blockIdx.y) * nparts * d;
    float v = 0.f;
    if (col < d) {
#pragma unroll 8
        for (int i = warp; i < nparts; i += 32) v += p[int64_t(i) * d + col];
    }
    s[warp][lane] = v;
    __syncthreads();
    v = s[lane][warp];  // column `warp` of the 32, part `lane`
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    const int mine = blockIdx.x * 32 + warp;
    if (lane == 0 && mine < d) out[mine] = v;
}

// ----------------------------------------------------------------- host ----

// Smallest power of two >= 32 of threads that covers d with V chunks of 8.
static int row_threads_for(int d, int v) {
    int nt = 32;
    while (nt * 8 * v < d) nt *= 2;
    return nt;
}

static bool aligned16(std::initializer_list<const void*> ps) {
    uintptr_t x = 0;
    for (const void* p : ps) x |= reinterpret_cast<uintptr_t>(p);
    return x % 16 == 0;
}

// The column vectors a backward call sums over the tokens.
static int column_vectors(bool pre, bool post, int gate_form) {
    return int(pre) + int(post) + int(gate_form == kGateChannel);
}

// Backward geometry: chunks a thread, threads a row, CTA threads and grid.
struct NormGradPlan {
    int v, row_threads, cta_threads, grid;
};
static NormGradPlan plan_norm_backward(int T, int d) {
    NormGradPlan p{};
    // Two chunks a thread and up to 512 threads: 32 column sums and the row in
    // hand fit 128 registers; the widest rows take four.
    p.v = d <= 8192 ? 2 : 4;
    p.row_threads = row_threads_for(d, p.v);
    p.cta_threads = p.row_threads == 32 ? 128 : p.row_threads;
    const int groups = p.cta_threads / p.row_threads;
    const int64_t need = (int64_t(T) + groups - 1) / groups;
    const int64_t fit = int64_t(device_sm_count()) * (512 / p.cta_threads);
    p.grid = int(need < fit ? need : fit);
    if (p.grid < 1) p.grid = 1;
    return p;
}

static int check_norm(const char* who, int T, int d, int dtype, int gate_form, const void* gate, const void* y,
                      const void* w_post, const void* w_pre, float eps) {
    if (T < 0 || d < 1) return fail(MOE_B200_ERR_INVALID_ARG, "%s: need T>=0, d>=1", who);
    if (d > kNormMaxD) return fail(MOE_B200_ERR_UNSUPPORTED, "%s: d=%d exceeds %d", who, d, kNormMaxD);
    if (dtype != MOE_B200_F16 && dtype != MOE_B200_BF16)
        return fail(MOE_B200_ERR_INVALID_ARG, "%s: dtype %d is neither F16 nor BF16", who, dtype);
    if (gate_form < kGateNone || gate_form > kGateFull)
        return fail(MOE_B200_ERR_INVALID_ARG, "%s: unknown gate form %d", who, gate_form);
    if ((gate_form == kGateNone) != (gate == nullptr))
        return fail(MOE_B200_ERR_INVALID_ARG, "%s: the gate and its form do not agree", who);
    if (!y && (w_post || gate)) return fail(MOE_B200_ERR_INVALID_ARG, "%s: w_post and gate need y", who);
    if (!y && !w_pre) return fail(MOE_B200_ERR_INVALID_ARG, "%s: nothing to do without y and w_pre", who);
    if (!(eps >= 0.f)) return fail(MOE_B200_ERR_INVALID_ARG, "%s: eps must be >= 0", who);
    return MOE_B200_OK;
}

template <int DT, bool RES32, bool AL, bool RING, bool WARP, int MAXT, int FORM>
static cudaError_t launch_norm_as(NormArgs a, int cta, int64_t grid, size_t smem, cudaStream_t s) {
    auto kern = block_norm_kernel<DT, RES32, AL, RING, WARP, 2, MAXT, FORM>;
    if (smem > 40 * 1024) {  // beyond what a kernel may use unasked
        const cudaError_t err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
        if (err != cudaSuccess) return err;
    }
    kern<<<unsigned(grid), cta, smem, s>>>(a);
    return cudaGetLastError();
}

template <int DT, bool RES32, bool AL, bool RING, int FORM>
static cudaError_t launch_norm_form(const NormArgs& a, int nt, int64_t grid, size_t smem, cudaStream_t s) {
    if (nt == 32) return launch_norm_as<DT, RES32, AL, RING, true, 128, FORM>(a, 128, grid, smem, s);
    if (nt <= 128) return launch_norm_as<DT, RES32, AL, RING, false, 128, FORM>(a, nt, grid, smem, s);
    if (nt <= 256) return launch_norm_as<DT, RES32, AL, RING, false, 256, FORM>(a, nt, grid, smem, s);
    return launch_norm_as<DT, RES32, AL, RING, false, 1024, FORM>(a, nt, grid, smem, s);
}

template <int DT, bool RES32, bool AL>
static cudaError_t launch_norm(const NormArgs& a0, cudaStream_t s) {
    NormArgs a = a0;
    const int nt = row_threads_for(a.d, 2), cta = nt == 32 ? 128 : nt, groups = cta / nt;
    const int per_sm = cta <= 256 ? 768 / cta : 1024 / cta;  // what the registers allow
    const int64_t need = (int64_t(a.T) + groups - 1) / groups, most = int64_t(device_sm_count()) * per_sm;
    if constexpr (AL) {
        a.off_y = a.d * (RES32 ? 4 : 2);
        a.off_gate = a.off_y + (a.y ? a.d * 2 : 0);
        a.row_bytes = a.off_gate + (a.gate_form == kGateFull ? a.d * 2 : 0);
        const size_t share = 227 * 1024 / per_sm - 3 * 1024;
        a.stages = kNormStages;
        while (a.stages > 1 && size_t(groups) * a.stages * a.row_bytes > share) --a.stages;
        if (need > most && a.stages > 1) {
            const size_t smem = size_t(groups) * a.stages * a.row_bytes;
            if (a.w_pre) {
                if (!a.y) return launch_norm_form<DT, RES32, true, true, kFormNorm>(a, nt, most, smem, s);
                if (a.w_post)
                    return a.gate_form >= kGateChannel
                               ? launch_norm_form<DT, RES32, true, true, kFormFullColGate>(a, nt, most, smem, s)
                               : launch_norm_form<DT, RES32, true, true, kFormFull>(a, nt, most, smem, s);
                if (a.gate_form < kGateChannel)
                    return launch_norm_form<DT, RES32, true, true, kFormAddNorm>(a, nt, most, smem, s);
            }
            return launch_norm_form<DT, RES32, true, true, kFormAny>(a, nt, most, smem, s);
        }
    }
    return launch_norm_form<DT, RES32, AL, false, kFormAny>(a, nt, need < most ? need : most, 0, s);
}

template <int DT, bool RES32, bool AL, bool RING, bool WARP, int V, int GATE = -1>
static cudaError_t launch_norm_backward_as(const NormGradArgs& a, const NormGradPlan& p, size_t smem, cudaStream_t s) {
    constexpr int kMax = WARP ? 128 : 512;
    auto kern = block_norm_backward_kernel<DT, RES32, AL, RING, WARP, V, kMax, GATE>;
    if (smem > 40 * 1024) {  // beyond what a kernel may use unasked
        const cudaError_t err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
        if (err != cudaSuccess) return err;
    }
    kern<<<p.grid, p.cta_threads, smem, s>>>(a);
    return cudaGetLastError();
}

template <int DT, bool RES32, bool WARP>
static cudaError_t launch_norm_backward_ring(const NormGradArgs& a, const NormGradPlan& p, size_t smem, cudaStream_t s) {
    if (a.w_pre && a.w_post && a.d_res_out) {
        if (a.gate_form == kGateNone) return launch_norm_backward_as<DT, RES32, true, true, WARP, 2, kGateNone>(a, p, smem, s);
        if (a.gate_form == kGateToken) return launch_norm_backward_as<DT, RES32, true, true, WARP, 2, kGateToken>(a, p, smem, s);
        if (a.gate_form == kGateChannel)
            return launch_norm_backward_as<DT, RES32, true, true, WARP, 2, kGateChannel>(a, p, smem, s);
        return launch_norm_backward_as<DT, RES32, true, true, WARP, 2, kGateFull>(a, p, smem, s);
    }
    return launch_norm_backward_as<DT, RES32, true, true, WARP, 2>(a, p, smem, s);
}

template <int DT, bool RES32, bool AL>
static cudaError_t launch_norm_backward(const NormGradArgs& a0, const NormGradPlan& p, cudaStream_t s) {
    NormGradArgs a = a0;
    const int groups = p.cta_threads / p.row_threads;
    int off = 0;
    auto part = [&](bool present, int bytes) {
        const int at = present ? off : -1;
        off += present ? bytes : 0;
        return at;
    };
    a.off_ds = part(a.d_res_out != nullptr, a.d * (RES32 ? 4 : 2));
    a.off_rr = part(a.w_pre != nullptr, a.d * (RES32 ? 4 : 2));
    a.off_dn = part(a.w_pre != nullptr, a.d * 2);
    a.off_y = part(a.y != nullptr, a.d * 2);
    a.off_gate = part(a.gate_form == kGateFull, a.d * 2);
    a.row_bytes = off;
    const size_t cols = groups > 1 ? size_t(a.d) * 4 : 0;
    // Ring: as many rows as fit the share of an SM's shared memory that each
    // of the CTAs it holds may take, two at least.
    const size_t weights = size_t(column_vectors(a.w_pre != nullptr, a.w_post != nullptr, a.gate_form)) * a.d * 2;
    const size_t share = 227 * 1024 / (512 / p.cta_threads) - 3 * 1024;
    a.stages = kNormStages;
    while (a.stages > 1 && size_t(groups) * a.stages * off + weights > share) --a.stages;
    a.off_w = groups * a.stages * off;
    const size_t ring = size_t(a.off_w) + weights;
    const bool use_ring = AL && p.v == 2 && a.stages > 1;
    const size_t smem = use_ring && ring > cols ? ring : cols;
    const bool warp = p.row_threads == 32;
    if constexpr (AL) {
        if (use_ring) {
            if (warp) return launch_norm_backward_ring<DT, RES32, true>(a, p, smem, s);
            return launch_norm_backward_ring<DT, RES32, false>(a, p, smem, s);
        }
    }
    if (warp) return launch_norm_backward_as<DT, RES32, AL, false, true, 2>(a, p, smem, s);
    if (p.v == 2) return launch_norm_backward_as<DT, RES32, AL, false, false, 2>(a, p, smem, s);
    return launch_norm_backward_as<DT, RES32, AL, false, false, 4>(a, p, smem, s);
}

template <typename F>
static cudaError_t by_form(int dtype, bool res32, bool al, F&& f) {
    using std::integral_constant;
    const int k = (dtype == MOE_B200_BF16 ? 4 : 0) | (res32 ? 2 : 0) | (al ? 1 : 0);
    constexpr int H = MOE_B200_F16, B = MOE_B200_BF16;
    switch (k) {
        case 0: return f(integral_constant<int, H>{}, std::false_type{}, std::false_type{});
        case 1: return f(integral_constant<int, H>{}, std::false_type{}, std::true_type{});
        case 2: return f(integral_constant<int, H>{}, std::true_type{}, std::false_type{});
        case 3: return f(integral_constant<int, H>{}, std::true_type{}, std::true_type{});
        case 4: return f(integral_constant<int, B>{}, std::false_type{}, std::false_type{});
        case 5: return f(integral_constant<int, B>{}, std::false_type{}, std::true_type{});
        case 6: return f(integral_constant<int, B>{}, std::true_type{}, std::false_type{});
        default: return f(integral_constant<int, B>{}, std::true_type{}, std::true_type{});
    }
}

}  // namespace moe_b200

extern "C" int moe_b200_block_norm(const void* y, int64_t y_stride, const void* residual, int64_t residual_stride,
                                   int residual_f32, const void* w_post, const void* w_pre, const void* gate,
                                   int gate_form, float scale, float eps, int T, int d, int dtype, void* residual_out,
                                   void* normed, void* stream) {
    using namespace moe_b200;
    const int rc = check_norm("block_norm", T, d, dtype, gate_form, gate, y, w_post, w_pre, eps);
    if (rc != MOE_B200_OK) return rc;
    if (!residual || (y && !residual_out) || (w_pre && !normed))
        return fail(MOE_B200_ERR_INVALID_ARG, "block_norm: null pointer");
    if (residual_stride < d || (y && y_stride < d))
        return fail(MOE_B200_ERR_INVALID_ARG, "block_norm: row strides below d=%d", d);
    if (T == 0) return MOE_B200_OK;
    uint32_t* status = device_status_word();
    if (!status) return fail(MOE_B200_ERR_CUDA, "block_norm: device status word unavailable");
    const NormArgs a{y, residual, w_post, w_pre, gate, y ? y_stride : 0, residual_stride, gate_form, scale, eps, T, d,
                     y ? residual_out : nullptr, w_pre ? normed : nullptr, 0, 0, 0, 0, status};
    const bool al = d % 8 == 0 && (!y || y_stride % 8 == 0) && residual_stride % (residual_f32 ? 4 : 8) == 0 &&
                    aligned16({y, residual, w_post, w_pre, gate_form >= kGateChannel ? gate : nullptr, a.residual_out,
                               a.normed});
    const cudaError_t err = by_form(dtype, residual_f32 != 0, al, [&](auto dt, auto r32, auto ali) {
        return launch_norm<decltype(dt)::value, decltype(r32)::value, decltype(ali)::value>(
            a, static_cast<cudaStream_t>(stream));
    });
    return err == cudaSuccess ? MOE_B200_OK : cuda_fail(err, "block_norm launch");
}

extern "C" size_t moe_b200_block_norm_backward_workspace_bytes(int T, int d) {
    using namespace moe_b200;
    if (T < 0 || d < 1 || d > kNormMaxD) return 0;
    return align256(size_t(3) * size_t(plan_norm_backward(T, d).grid) * size_t(d) * 4);
}

extern "C" int moe_b200_block_norm_backward(const void* d_residual_out, const void* d_normed,
                                            const void* residual_out, int64_t residual_stride, int residual_f32,
                                            const void* y, int64_t y_stride, const void* w_post, const void* w_pre,
                                            const void* gate, int gate_form, float scale, float eps, int T, int d,
                                            int dtype, void* d_residual, void* d_y, float* d_w_post, float* d_w_pre,
                                            void* d_gate, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace moe_b200;
    const int rc = check_norm("block_norm_backward", T, d, dtype, gate_form, gate, y, w_post, w_pre, eps);
    if (rc != MOE_B200_OK) return rc;
    if (!d_residual || (w_pre && (!d_normed || !residual_out || !d_w_pre)) || (!w_pre && !d_residual_out) ||
        (y && !d_y) || (w_post && !d_w_post) || (gate && !d_gate))
        return fail(MOE_B200_ERR_INVALID_ARG, "block_norm_backward: null pointer");
    if ((w_pre && residual_stride < d) || (y && y_stride < d))
        return fail(MOE_B200_ERR_INVALID_ARG, "block_norm_backward: row strides below d=%d", d);
    const bool res32 = residual_f32 != 0;
    const NormGradPlan p = plan_norm_backward(T, d);
    const int vectors = column_vectors(w_pre != nullptr, w_post != nullptr, gate_form);
    if (vectors && (!workspace || workspace_bytes < align256(size_t(vectors) * p.grid * size_t(d) * 4)))
        return fail(MOE_B200_ERR_WORKSPACE, "block_norm_backward: workspace too small");
    if (reinterpret_cast<uintptr_t>(workspace) % 256 != 0)
        return fail(MOE_B200_ERR_INVALID_ARG, "block_norm_backward: workspace must be 256-byte aligned");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    float* outs[3] = {nullptr, nullptr, nullptr};
    int n = 0, i_pre = -1, i_post = -1, i_gate = -1;
    if (w_pre) outs[i_pre = n++] = d_w_pre;
    if (w_post) outs[i_post = n++] = d_w_post;
    if (gate_form == kGateChannel) outs[i_gate = n++] = static_cast<float*>(d_gate);
    if (T == 0) {  // sums over no token
        for (int i = 0; i < n; ++i) {
            const cudaError_t err = cudaMemsetAsync(outs[i], 0, size_t(d) * 4, s);
            if (err != cudaSuccess) return cuda_fail(err, "block_norm_backward");
        }
        return MOE_B200_OK;
    }
    uint32_t* status = device_status_word();
    if (!status) return fail(MOE_B200_ERR_CUDA, "block_norm_backward: device status word unavailable");
    const NormGradArgs a{d_residual_out, d_normed, residual_out, y, w_post, w_pre, gate, y ? y_stride : 0,
                         w_pre ? residual_stride : 0, gate_form, scale, eps, T, d, d_residual, d_y, d_gate,
                         static_cast<float*>(workspace), i_pre, i_post, i_gate, 0, -1, -1, -1, -1, -1, 0, 0, status};
    const bool al = d % 8 == 0 && a.y_stride % 8 == 0 && a.res_stride % (res32 ? 4 : 8) == 0 &&
                    aligned16({d_residual_out, d_normed, residual_out, y, w_post, w_pre,
                               gate_form >= kGateChannel ? gate : nullptr, d_residual, d_y,
                               gate_form == kGateFull ? d_gate : nullptr});
    cudaError_t err = by_form(dtype, res32, al, [&](auto dt, auto r32, auto ali) {
        return launch_norm_backward<decltype(dt)::value, decltype(r32)::value, decltype(ali)::value>(a, p, s);
    });
    if (err == cudaSuccess && n > 0) {
        cudaLaunchConfig_t cfg = pdl_config(dim3((d + 31) / 32, n), dim3(1024), 0, s);
        cudaLaunchAttribute attr[1] = {pdl_attr()};
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        err = cudaLaunchKernelEx(&cfg, block_norm_columns_kernel, static_cast<const float*>(a.part), p.grid, d, outs[0],
                                 outs[1], outs[2]);
    }
    return err == cudaSuccess ? MOE_B200_OK : cuda_fail(err, "block_norm_backward launch");
}
