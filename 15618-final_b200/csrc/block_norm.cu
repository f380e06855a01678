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
// Both directions are bound by memory: every row is read once into registers
// and every result is written once; all sums are fp32, outputs are rounded
// once (n comes from the unrounded r').
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
constexpr int kNormMaxThreads = 1024;

enum { kGateNone = MOE_B200_GATE_NONE, kGateToken = MOE_B200_GATE_TOKEN, kGateChannel = MOE_B200_GATE_CHANNEL,
       kGateFull = MOE_B200_GATE_FULL };

// One 16-bit word <-> fp32.
template <int DT> __device__ __forceinline__ float from16(uint16_t b) {
    return DT == MOE_B200_BF16 ? __uint_as_float(uint32_t(b) << 16) : __half2float(__ushort_as_half(b));
}
template <int DT> __device__ __forceinline__ uint16_t to16(float f) {
    return DT == MOE_B200_BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(f)) : __half_as_ushort(__float2half_rn(f));
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
// a word), fp32 rows w[0..7].  Columns past d read as zero, which adds nothing
// to any sum.
template <bool F32> struct Raw {
    uint32_t w[F32 ? 8 : 4];
};

template <bool ALIGNED, bool F32>
__device__ __forceinline__ Raw<F32> load_raw(const void* row, int chunk, int t, int nt, int d) {
    Raw<F32> r;
    if (ALIGNED) {
        const int c = col_of<true>(chunk, 0, t, nt);
        if (c < d) {
            const uint4* p = reinterpret_cast<const uint4*>(static_cast<const char*>(row) + size_t(c) * (F32 ? 4 : 2));
#pragma unroll
            for (int h = 0; h < (F32 ? 2 : 1); ++h) {
                const uint4 v = p[h];
                r.w[4 * h] = v.x, r.w[4 * h + 1] = v.y, r.w[4 * h + 2] = v.z, r.w[4 * h + 3] = v.w;
            }
        } else {
#pragma unroll
            for (int j = 0; j < (F32 ? 8 : 4); ++j) r.w[j] = 0;
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

// Eight fp32 values to a row of 16-bit or fp32 columns.
template <int DT, bool ALIGNED, bool F32>
__device__ __forceinline__ void store8(void* row, const float (&x)[8], int chunk, int t, int nt, int d) {
    if (ALIGNED) {
        const int c = col_of<true>(chunk, 0, t, nt);
        if (c >= d) return;
        uint4* p = reinterpret_cast<uint4*>(static_cast<char*>(row) + size_t(c) * (F32 ? 4 : 2));
        if (F32) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
                st_v4(p + h, make_uint4(__float_as_uint(x[4 * h]), __float_as_uint(x[4 * h + 1]),
                                        __float_as_uint(x[4 * h + 2]), __float_as_uint(x[4 * h + 3])));
        } else {
            uint32_t o[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                o[j] = uint32_t(to16<DT>(x[2 * j])) | (uint32_t(to16<DT>(x[2 * j + 1])) << 16);
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

// Sums of N values over the `nt` threads of a row group (nt a multiple of 32),
// the same bits in every thread.  `red` holds two buffers of N floats a warp;
// `phase` alternates them, so one barrier a reduction is enough: a buffer is
// written again only after the next reduction's barrier, which no thread
// passes before it has read this one.
template <int N>
__device__ __forceinline__ void group_sum(float (&v)[N], float* red, int nt, int group, int warp_in_group, int& phase) {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    if (nt == 32) return;
    const int nw = nt >> 5;
    float* b = red + (phase & 1) * (nw * 4);
    ++phase;
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) b[warp_in_group * 4 + i] = v[i];
    }
    asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(nt) : "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = 0.f;
    for (int w = 0; w < nw; ++w) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += b[w * 4 + i];
    }
}

struct NormArgs {
    const void *y, *residual, *w_post, *w_pre, *gate;
    int64_t y_stride, res_stride;  // elements
    int gate_form;
    float scale, eps;
    int T, d, row_threads;
    void *residual_out, *normed;
};

// A group of `row_threads` threads per row, V chunks of 8 columns a thread, a
// CTA of at least 128 threads.  No loop over rows: the grid's many small CTAs
// keep enough loads in flight.
template <int DT, bool RES32, bool ALIGNED, int V>
__global__ void __launch_bounds__(kNormMaxThreads)
block_norm_kernel(const NormArgs a) {
    __shared__ float s_red[2 * 4 * 32];
    const int nt = a.row_threads, group = threadIdx.x / nt, t = threadIdx.x - group * nt, wig = t >> 5;
    const int64_t row = int64_t(blockIdx.x) * (blockDim.x / nt) + group;
    if (row >= a.T) return;  // whole groups leave together; barriers are per group
    float* red = s_red + group * (nt >> 5) * 8;
    int phase = 0;
    const int d = a.d;
    const float inv_d = 1.0f / float(d);
    const char* res_row = static_cast<const char*>(a.residual) + row * a.res_stride * (RES32 ? 4 : 2);
    const uint16_t* y_row = static_cast<const uint16_t*>(a.y) + row * a.y_stride;
    Raw<RES32> res[V];
    Raw<false> yr[V], wp[V], gr[V], wn[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        res[i] = load_raw<ALIGNED, RES32>(res_row, i, t, nt, d);
        if (a.y) yr[i] = load_raw<ALIGNED, false>(y_row, i, t, nt, d);
        if (a.gate_form == kGateFull)
            gr[i] = load_raw<ALIGNED, false>(static_cast<const uint16_t*>(a.gate) + row * d, i, t, nt, d);
        if (a.gate_form == kGateChannel) gr[i] = load_raw<ALIGNED, false>(a.gate, i, t, nt, d);
        if (a.w_post) wp[i] = load_raw<ALIGNED, false>(a.w_post, i, t, nt, d);
        if (a.w_pre) wn[i] = load_raw<ALIGNED, false>(a.w_pre, i, t, nt, d);
    }
    float r[V][8];
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) r[i][j] = raw_get<DT, RES32>(res[i], j);
    if (a.y) {
        float f = a.scale;
        if (a.gate_form == kGateToken) f *= from16<DT>(static_cast<const uint16_t*>(a.gate)[row]);
        if (a.w_post) {
            float s[1] = {0.f};
#pragma unroll
            for (int i = 0; i < V; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float y = raw_get<DT, false>(yr[i], j);
                    s[0] += y * y;
                }
            group_sum(s, red, nt, group, wig, phase);
            f *= rsqrtf(s[0] * inv_d + a.eps);
        }
#pragma unroll
        for (int i = 0; i < V; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float z = raw_get<DT, false>(yr[i], j) * f;
                if (a.w_post) z *= raw_get<DT, false>(wp[i], j);
                if (a.gate_form >= kGateChannel) z *= raw_get<DT, false>(gr[i], j);
                r[i][j] += z;
            }
        char* out = static_cast<char*>(a.residual_out) + row * d * (RES32 ? 4 : 2);
#pragma unroll
        for (int i = 0; i < V; ++i) store8<DT, ALIGNED, RES32>(out, r[i], i, t, nt, d);
    }
    if (a.w_pre) {
        float s[1] = {0.f};
#pragma unroll
        for (int i = 0; i < V; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) s[0] += r[i][j] * r[i][j];
        group_sum(s, red, nt, group, wig, phase);
        const float c = rsqrtf(s[0] * inv_d + a.eps);
        uint16_t* out = static_cast<uint16_t*>(a.normed) + row * d;
#pragma unroll
        for (int i = 0; i < V; ++i) {
#pragma unroll
            for (int j = 0; j < 8; ++j) r[i][j] *= c * raw_get<DT, false>(wn[i], j);
            store8<DT, ALIGNED, false>(out, r[i], i, t, nt, d);
        }
    }
}

struct NormGradArgs {
    const void *d_res_out, *d_normed, *res_out, *y, *w_post, *w_pre, *gate;
    int64_t y_stride, res_stride;
    int gate_form;
    float scale, eps;
    int T, d, row_threads;
    void *d_res, *d_y, *d_gate;
    // Column sums of each CTA: up to three vectors of d floats, [vector][CTA][d].
    float* part;
    int sum_pre, sum_post, sum_gate;  // index of the vector, or -1
};

// Rows are dealt to the groups of a grid that fits the card, so that each
// thread keeps its columns' sums over its rows in registers and the column
// gradients cost one row of partial sums a CTA.  Row data stays packed as
// loaded until it is used.
template <int DT, bool RES32, bool ALIGNED, int V, int MAXT>
__global__ void __launch_bounds__(MAXT)
block_norm_backward_kernel(const NormGradArgs a) {
    extern __shared__ float s_dyn[];  // [2 * 4 * 32] reduction words, then (several groups) [d] column sums
    const int nt = a.row_threads, group = threadIdx.x / nt, t = threadIdx.x - group * nt, wig = t >> 5;
    const int groups = blockDim.x / nt;
    float* red = s_dyn + group * (nt >> 5) * 8;
    int phase = 0;
    const int d = a.d;
    const float inv_d = 1.0f / float(d);
    float s_pre[V][8], s_post[V][8], s_gate[V][8];
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) s_pre[i][j] = s_post[i][j] = s_gate[i][j] = 0.f;

    for (int64_t row = int64_t(blockIdx.x) * groups + group; row < a.T; row += int64_t(gridDim.x) * groups) {
        Raw<RES32> ds[V], rr[V];
        Raw<false> dn[V], yr[V], gr[V];
        const char* ds_row = static_cast<const char*>(a.d_res_out) + row * d * (RES32 ? 4 : 2);
        const char* rr_row = static_cast<const char*>(a.res_out) + row * a.res_stride * (RES32 ? 4 : 2);
        const uint16_t* dn_row = static_cast<const uint16_t*>(a.d_normed) + row * d;
        const uint16_t* y_row = static_cast<const uint16_t*>(a.y) + row * a.y_stride;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (a.w_pre) {
                rr[i] = load_raw<ALIGNED, RES32>(rr_row, i, t, nt, d);
                dn[i] = load_raw<ALIGNED, false>(dn_row, i, t, nt, d);
            }
            if (a.y) yr[i] = load_raw<ALIGNED, false>(y_row, i, t, nt, d);
            if (a.d_res_out) ds[i] = load_raw<ALIGNED, RES32>(ds_row, i, t, nt, d);
            if (a.gate_form == kGateFull)
                gr[i] = load_raw<ALIGNED, false>(static_cast<const uint16_t*>(a.gate) + row * d, i, t, nt, d);
            if (a.gate_form == kGateChannel) gr[i] = load_raw<ALIGNED, false>(a.gate, i, t, nt, d);
        }
        float sums[3] = {0.f, 0.f, 0.f};  // sum r'^2, sum u r', sum y^2
        float q[V][8];
        if (a.w_pre) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const Raw<false> wn = load_raw<ALIGNED, false>(a.w_pre, i, t, nt, d);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float r = raw_get<DT, RES32>(rr[i], j);
                    q[i][j] = raw_get<DT, false>(dn[i], j) * raw_get<DT, false>(wn, j);
                    sums[0] += r * r;
                    sums[1] += q[i][j] * r;
                }
            }
        }
        if (a.w_post) {
#pragma unroll
            for (int i = 0; i < V; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float y = raw_get<DT, false>(yr[i], j);
                    sums[2] += y * y;
                }
        }
        if (a.w_pre || a.w_post) group_sum(sums, red, nt, group, wig, phase);
        const float c = rsqrtf(sums[0] * inv_d + a.eps);
        const float k = sums[1] * inv_d * c * c;
        const float post = a.w_post ? rsqrtf(sums[2] * inv_d + a.eps) : 1.0f;
        char* dres_out = static_cast<char*>(a.d_res) + row * d * (RES32 ? 4 : 2);
        float f = a.scale;
        if (a.gate_form == kGateToken) f *= from16<DT>(static_cast<const uint16_t*>(a.gate)[row]);
        float sums2[2] = {0.f, 0.f};  // sum v yh, sum ds z (gate per token)
#pragma unroll
        for (int i = 0; i < V; ++i) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float g = a.d_res_out ? raw_get<DT, RES32>(ds[i], j) : 0.f;
                if (a.w_pre) {
                    const float r = raw_get<DT, RES32>(rr[i], j);
                    g += c * (q[i][j] - r * k);
                    s_pre[i][j] += raw_get<DT, false>(dn[i], j) * (r * c);
                }
                q[i][j] = g;
            }
            store8<DT, ALIGNED, RES32>(dres_out, q[i], i, t, nt, d);
        }
        if (a.y) {
            float dg[8];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                Raw<false> wp;
                if (a.w_post) wp = load_raw<ALIGNED, false>(a.w_post, i, t, nt, d);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float yh = raw_get<DT, false>(yr[i], j) * post;
                    const float w = a.w_post ? raw_get<DT, false>(wp, j) : 1.0f;
                    const float g = q[i][j];
                    if (a.gate_form != kGateNone) dg[j] = a.scale * g * (yh * w);
                    float v = g * f;
                    if (a.gate_form >= kGateChannel) v *= raw_get<DT, false>(gr[i], j);
                    if (a.w_post) {
                        s_post[i][j] += v * yh;
                        v *= w;
                        sums2[0] += v * yh;
                    }
                    q[i][j] = v;
                    if (a.gate_form == kGateToken) sums2[1] += dg[j];
                    if (a.gate_form == kGateChannel) s_gate[i][j] += dg[j];
                }
                if (a.gate_form == kGateFull)
                    store8<DT, ALIGNED, false>(static_cast<uint16_t*>(a.d_gate) + row * d, dg, i, t, nt, d);
            }
            if (a.w_post || a.gate_form == kGateToken) group_sum(sums2, red, nt, group, wig, phase);
            if (a.gate_form == kGateToken && t == 0) static_cast<float*>(a.d_gate)[row] = sums2[1];
            const float m = sums2[0] * inv_d;
            uint16_t* dy_out = static_cast<uint16_t*>(a.d_y) + row * d;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                if (a.w_post) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) q[i][j] = post * (q[i][j] - raw_get<DT, false>(yr[i], j) * post * m);
                }
                store8<DT, ALIGNED, false>(dy_out, q[i], i, t, nt, d);
            }
        }
    }

    // Column sums: the groups of the CTA add up through shared memory in group
    // order, then the CTA writes its row of partial sums.
    float* s_col = s_dyn + 2 * 4 * 32;
#pragma unroll
    for (int which = 0; which < 3; ++which) {
        const int vec = which == 0 ? a.sum_pre : which == 1 ? a.sum_post : a.sum_gate;
        if (vec < 0) continue;
        float* part = a.part + (int64_t(vec) * gridDim.x + blockIdx.x) * d;
        float(&s)[V][8] = which == 0 ? s_pre : which == 1 ? s_post : s_gate;
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
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int col = col_of<ALIGNED>(i, j, t, nt);
                    if (groups > 1 && col < d) s[i][j] += s_col[col];
                }
                store8<DT, ALIGNED, true>(part, s[i], i, t, nt, d);
            }
        }
        __syncthreads();
    }
    pdl_launch_dependents();
}

// Adds the CTAs' partial rows: a warp per 32 columns of one vector, 8 warps
// split the rows; each output is a fixed-order sum.
__global__ void __launch_bounds__(256)
block_norm_columns_kernel(const float* __restrict__ part, int nparts, int d, float* out0, float* out1, float* out2) {
    __shared__ float s[8][33];
    pdl_wait_primary();
    float* out = blockIdx.y == 0 ? out0 : blockIdx.y == 1 ? out1 : out2;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, col = blockIdx.x * 32 + lane;
    const float* p = part + int64_t(blockIdx.y) * nparts * d;
    float v = 0.f;
    if (col < d)
        for (int i = warp; i < nparts; i += 8) v += p[int64_t(i) * d + col];
    s[warp][lane] = v;
    __syncthreads();
    if (warp == 0 && col < d) {
#pragma unroll
        for (int w = 1; w < 8; ++w) v += s[w][lane];
        out[col] = v;
    }
}

// ----------------------------------------------------------------- host ----

static int sm_count_norm() {
    int dev = 0, n = 148;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    return n > 0 ? n : 148;
}

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
static NormGradPlan plan_norm_backward(int T, int d, bool res32) {
    NormGradPlan p{};
    // Two chunks a thread and up to 512 threads: 48 sums and the packed row
    // fit 128 registers; fp32 residuals (twice the words) take one chunk while
    // 512 threads cover the row; the widest rows take four.
    p.v = (res32 && d <= 4096) ? 1 : d <= 8192 ? 2 : 4;
    p.row_threads = row_threads_for(d, p.v);
    p.cta_threads = p.row_threads < 128 ? 128 : p.row_threads;
    const int groups = p.cta_threads / p.row_threads;
    const int64_t need = (int64_t(T) + groups - 1) / groups;
    const int64_t fit = int64_t(sm_count_norm()) * (512 / p.cta_threads);
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

template <int DT, bool RES32, bool AL>
static cudaError_t launch_norm(const NormArgs& a0, cudaStream_t s) {
    NormArgs a = a0;
    a.row_threads = row_threads_for(a.d, 2);
    const int cta = a.row_threads < 128 ? 128 : a.row_threads;
    const int groups = cta / a.row_threads;
    const unsigned grid = unsigned((int64_t(a.T) + groups - 1) / groups);
    block_norm_kernel<DT, RES32, AL, 2><<<grid, cta, 0, s>>>(a);
    return cudaGetLastError();
}

template <int DT, bool RES32, bool AL, int V, int MAXT>
static cudaError_t launch_norm_backward_v(const NormGradArgs& a, const NormGradPlan& p, cudaStream_t s) {
    const int groups = p.cta_threads / p.row_threads;
    const size_t smem = sizeof(float) * (2 * 4 * 32 + (groups > 1 ? a.d : 0));
    block_norm_backward_kernel<DT, RES32, AL, V, MAXT><<<p.grid, p.cta_threads, smem, s>>>(a);
    return cudaGetLastError();
}

template <int DT, bool RES32, bool AL>
static cudaError_t launch_norm_backward(const NormGradArgs& a, const NormGradPlan& p, cudaStream_t s) {
    if (p.v == 1) return launch_norm_backward_v<DT, RES32, AL, 1, 512>(a, p, s);
    if (p.v == 2) return launch_norm_backward_v<DT, RES32, AL, 2, 512>(a, p, s);
    return launch_norm_backward_v<DT, RES32, AL, 4, 512>(a, p, s);
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
    const NormArgs a{y, residual, w_post, w_pre, gate, y ? y_stride : 0, residual_stride, gate_form, scale, eps, T, d,
                     0, y ? residual_out : nullptr, w_pre ? normed : nullptr};
    const bool al = d % 8 == 0 && (!y || y_stride % 8 == 0) && residual_stride % (residual_f32 ? 4 : 8) == 0 &&
                    aligned16({y, residual, w_post, w_pre, gate_form >= kGateChannel ? gate : nullptr, a.residual_out,
                               a.normed});
    const cudaError_t err = by_form(dtype, residual_f32 != 0, al, [&](auto dt, auto r32, auto ali) {
        return launch_norm<decltype(dt)::value, decltype(r32)::value, decltype(ali)::value>(
            a, static_cast<cudaStream_t>(stream));
    });
    return err == cudaSuccess ? MOE_B200_OK : cuda_fail(err, "block_norm launch");
}

extern "C" size_t moe_b200_block_norm_backward_workspace_bytes(int T, int d, int residual_f32) {
    using namespace moe_b200;
    if (T < 0 || d < 1 || d > kNormMaxD) return 0;
    return align256(size_t(3) * size_t(plan_norm_backward(T, d, residual_f32 != 0).grid) * size_t(d) * 4);
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
    const NormGradPlan p = plan_norm_backward(T, d, res32);
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
    const NormGradArgs a{d_residual_out, d_normed, residual_out, y, w_post, w_pre, gate, y ? y_stride : 0,
                         w_pre ? residual_stride : 0, gate_form, scale, eps, T, d, p.row_threads, d_residual, d_y,
                         d_gate, static_cast<float*>(workspace), i_pre, i_post, i_gate};
    const bool al = d % 8 == 0 && a.y_stride % 8 == 0 && a.res_stride % (res32 ? 4 : 8) == 0 &&
                    aligned16({d_residual_out, d_normed, residual_out, y, w_post, w_pre,
                               gate_form >= kGateChannel ? gate : nullptr, d_residual, d_y,
                               gate_form == kGateFull ? d_gate : nullptr});
    cudaError_t err = by_form(dtype, res32, al, [&](auto dt, auto r32, auto ali) {
        return launch_norm_backward<decltype(dt)::value, decltype(r32)::value, decltype(ali)::value>(a, p, s);
    });
    if (err == cudaSuccess && n > 0) {
        cudaLaunchConfig_t cfg = pdl_config(dim3((d + 31) / 32, n), dim3(256), 0, s);
        cudaLaunchAttribute attr[1] = {pdl_attr()};
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        err = cudaLaunchKernelEx(&cfg, block_norm_columns_kernel, static_cast<const float*>(a.part), p.grid, d, outs[0],
                                 outs[1], outs[2]);
    }
    return err == cudaSuccess ? MOE_B200_OK : cuda_fail(err, "block_norm_backward launch");
}
