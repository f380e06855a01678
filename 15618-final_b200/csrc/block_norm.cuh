// block_norm.cuh -- what the forward (block_norm.cu) and the backward
// (block_norm_backward.cu) of the norms around a block share: how a thread
// holds a row's columns, sums over a row, the checks and the choice of access.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <initializer_list>
#include <type_traits>

#include "common.cuh"
#include "per_device.cuh"

namespace moe_b200 {

int fail(int code, const char* fmt, ...);
int cuda_fail(cudaError_t err, const char* where);

constexpr int kNormMaxD = 16384;
constexpr int kNormStages = 4;  // rows in flight, at most

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

// A row's columns as a thread holds them: V chunks of 8, by what the rows allow.
//   kChunks  d, strides and pointers in 16-byte steps: 8 consecutive columns a
//            chunk, one 16-byte access (two for fp32)
//   kPairs   rows that begin an even number of columns from an aligned place,
//            or all an odd number: columns in pairs, neighbouring threads on
//            neighbouring pairs, a 4-byte access each (8 for fp32).  With odd
//            d every other row begins in the middle of a word; there (`odd`)
//            the pairs are (-1, 0), (1, 2), ..  A thread's rows are all of one
//            kind (the grid steps by an even number of rows), so its columns
//            stay its own.
//   kSingle  other rows: element by element, neighbours on neighbours
// 3475 rows of 3545, gate per token, in a captured graph: fp16 with fp32
// residual 50 us in pairs and 68 one by one, backward 110 and 125; bf16 with
// bf16 residual 41 and 65, backward 99 and 193.  Rows of 3544, in chunks: 29 and
// 49, 19 and 40.
enum { kSingle = 0, kPairs = 1, kChunks = 2 };
enum { kOddRow = 1, kHalfPair = 2 };  // of `odd`: the row begins inside a word; a pair of this thread has one column only
template <int AL>
__device__ __forceinline__ int col_of(int chunk, int j, int t, int nt, int odd) {
    return AL == kChunks  ? (chunk * nt + t) * 8 + j
           : AL == kPairs ? ((chunk * 4 + (j >> 1)) * nt + t) * 2 + (j & 1) - (odd & kOddRow)
                          : (chunk * 8 + j) * nt + t;
}

// Eight columns of a chunk as raw words: 16-bit rows use w[0..3] (two columns
// a word), fp32 rows w[0..7].  Rows in chunks end with one, and the caller
// asks chunk_in() once per chunk; of other rows, columns outside [0, d) read as
// zero, which adds nothing to any sum.
// (A row of pairs held by a warp may end before a chunk; a CTA's does not, and
// a test there would keep the loads of its chunks apart.)
template <int AL, bool WARP> __device__ __forceinline__ bool chunk_in(int chunk, int t, int nt, int d) {
    return AL == kChunks ? (chunk * nt + t) * 8 < d : AL == kPairs && WARP ? chunk * 256 <= d : true;
}
// `odd` of a row: whether it begins inside a word, and whether this thread has
// a pair that sticks out of it on one side (pairs: few threads do, and all
// others skip the halves).
template <int AL> __device__ __forceinline__ int odd_of(int64_t row, int t, int nt, int d) {
    if (AL != kPairs) return 0;
    const int odd = int(row) & d & 1;
    bool half = odd && t == 0;  // column 0 alone
    const int last = (d - 1 + odd) >> 1;  // pair of the last column
    half |= ((d - 1 + odd) & 1) == 0 && last % nt == t;
    return odd | (half ? kHalfPair : 0);
}
template <bool F32> struct Raw {
    uint32_t w[F32 ? 8 : 4];
};

// Pairs: BRANCH puts the columns that are alone in their word behind a branch
// that few threads take; otherwise they are predicated accesses, and all of a
// row's loads start at once.  The backward takes the branch (rows and types as
// above: 110 us against 118, bf16 99 against 112; even 3546 columns 93 against
// 116), the forward does not (50 against 54, bf16 41 against 45; only with 3546
// columns the branch is better, 46 against 49).
template <int AL, bool F32, bool BRANCH = false>
__device__ __forceinline__ Raw<F32> load_raw(const void* row, int chunk, int t, int nt, int d, int odd) {
    Raw<F32> r;
    if (AL == kChunks) {
        const uint4* p = reinterpret_cast<const uint4*>(static_cast<const char*>(row) +
                                                        col_of<kChunks>(chunk, 0, t, nt, 0) * (F32 ? 4 : 2));
#pragma unroll
        for (int h = 0; h < (F32 ? 2 : 1); ++h) {
            const uint4 v = p[h];
            r.w[4 * h] = v.x, r.w[4 * h + 1] = v.y, r.w[4 * h + 2] = v.z, r.w[4 * h + 3] = v.w;
        }
    } else if (AL == kPairs) {
        const uint16_t* p16 = static_cast<const uint16_t*>(row);
        const uint32_t* p32 = static_cast<const uint32_t*>(row);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int c = col_of<kPairs>(chunk, 2 * k, t, nt, odd);
            const bool lo = c >= 0 && c < d, hi = c + 1 < d;
            if (F32) {
                uint2 v = make_uint2(0, 0);
                if (lo && hi) v = *reinterpret_cast<const uint2*>(p32 + c);
                else if (!BRANCH && lo) v.x = p32[c];
                else if (!BRANCH && hi) v.y = p32[c + 1];
                r.w[2 * k % (F32 ? 8 : 4)] = v.x, r.w[(2 * k + 1) % (F32 ? 8 : 4)] = v.y;
            } else {
                uint32_t v = 0;
                if (lo && hi) v = *reinterpret_cast<const uint32_t*>(p16 + c);
                else if (!BRANCH && lo) v = p16[c];
                else if (!BRANCH && hi) v = uint32_t(p16[c + 1]) << 16;
                r.w[k] = v;
            }
        }
        if (BRANCH && (odd & kHalfPair)) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int c = col_of<kPairs>(chunk, 2 * k, t, nt, odd);
                if (c == -1) {
                    if (F32) r.w[(2 * k + 1) % (F32 ? 8 : 4)] = p32[0];
                    else r.w[k] = uint32_t(p16[0]) << 16;
                } else if (c + 1 == d) {
                    if (F32) r.w[2 * k % (F32 ? 8 : 4)] = p32[c];
                    else r.w[k] = p16[c];
                }
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int c = col_of<kSingle>(chunk, j, t, nt, 0);
            uint32_t v = 0;
            if (c < d) v = F32 ? static_cast<const uint32_t*>(row)[c] : uint32_t(static_cast<const uint16_t*>(row)[c]);
            if (F32) r.w[j % (F32 ? 8 : 4)] = v;
            else if (j & 1) r.w[(j >> 1) % 4] |= v << 16;
            else r.w[(j >> 1) % 4] = v;
        }
    }
    return r;
}
// The same columns of a vector [d] (weights, channel gate), which begins where it begins.
template <int AL>
__device__ __forceinline__ Raw<false> load_vec(const void* vec, int chunk, int t, int nt, int d, int odd) {
    if constexpr (AL != kPairs) {
        return load_raw<AL, false>(vec, chunk, t, nt, d, odd);
    } else {
        Raw<false> r;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int c = col_of<kPairs>(chunk, j, t, nt, odd);
            const uint32_t v = c >= 0 && c < d ? static_cast<const uint16_t*>(vec)[c] : 0u;
            if (j & 1) r.w[j >> 1] |= v << 16;
            else r.w[j >> 1] = v;
        }
        return r;
    }
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
template <int DT, int AL, bool F32, bool BRANCH = false>
__device__ __forceinline__ void store8(void* row, const float (&x)[8], int chunk, int t, int nt, int d, int odd) {
    float* p32 = static_cast<float*>(row);
    uint16_t* p16 = static_cast<uint16_t*>(row);
    if (AL == kChunks) {
        uint4* p = reinterpret_cast<uint4*>(static_cast<char*>(row) + col_of<kChunks>(chunk, 0, t, nt, 0) * (F32 ? 4 : 2));
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
    } else if (AL == kPairs) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int c = col_of<kPairs>(chunk, 2 * k, t, nt, odd);
            const bool lo = c >= 0 && c < d, hi = c + 1 < d;
            const uint32_t v = F32 ? 0u : pack16<DT>(x[2 * k], x[2 * k + 1]);
            if (lo && hi) {
                if (F32) *reinterpret_cast<float2*>(p32 + c) = make_float2(x[2 * k], x[2 * k + 1]);
                else *reinterpret_cast<uint32_t*>(p16 + c) = v;
            } else if (!BRANCH && lo) {
                if (F32) p32[c] = x[2 * k];
                else p16[c] = uint16_t(v);
            } else if (!BRANCH && hi) {
                if (F32) p32[c + 1] = x[2 * k + 1];
                else p16[c + 1] = uint16_t(v >> 16);
            }
        }
        if (BRANCH && (odd & kHalfPair)) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int c = col_of<kPairs>(chunk, 2 * k, t, nt, odd);
                if (c == -1) {
                    if (F32) p32[0] = x[2 * k + 1];
                    else p16[0] = to16<DT>(x[2 * k + 1]);
                } else if (c + 1 == d) {
                    if (F32) p32[c] = x[2 * k];
                    else p16[c] = to16<DT>(x[2 * k]);
                }
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int c = col_of<kSingle>(chunk, j, t, nt, 0);
            if (c < d) {
                if (F32) p32[c] = x[j];
                else p16[c] = to16<DT>(x[j]);
            }
        }
    }
}
// The same columns of a vector of d floats, which begins where it begins.
template <int DT, int AL>
__device__ __forceinline__ void store_vec(float* vec, const float (&x)[8], int chunk, int t, int nt, int d, int odd) {
    if constexpr (AL != kPairs) {
        store8<DT, AL, true>(vec, x, chunk, t, nt, d, odd);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int c = col_of<kPairs>(chunk, j, t, nt, odd);
            if (c >= 0 && c < d) vec[c] = x[j];
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

template <int DT, int AL, bool F32>
__device__ __forceinline__ void store8(void* row, const f32x2 (&x)[4], int chunk, int t, int nt, int d, int odd) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) split(x[j], v[2 * j], v[2 * j + 1]);
    store8<DT, AL, F32, true>(row, v, chunk, t, nt, d, odd);  // (the backward's)
}

// ----------------------------------------------------------------- host ----

// Smallest power of two >= 32 of threads that covers d with V chunks of 8.
inline int row_threads_for(int d, int v) {
    int nt = 32;
    while (nt * 8 * v < d) nt *= 2;
    return nt;
}

// A grid whose CTAs, of `groups` rows each, keep to rows of one kind in pairs.
template <int AL> inline int64_t steps(int64_t grid, int groups, int d) {
    return AL == kPairs && (d & 1) && groups == 1 && grid > 1 ? grid & ~int64_t(1) : grid;
}

inline int check_norm(const char* who, int T, int d, int dtype, int gate_form, const void* gate, const void* y,
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

// How a call's rows may be accessed.  `rows`: pointers to rows of d columns,
// with their strides in elements and whether they are fp32; vectors: w_post,
// w_pre and a channel gate.
struct NormRows {
    const void* p;
    int64_t stride;
    bool f32;
};
inline int access_of(int d, std::initializer_list<NormRows> rows, std::initializer_list<const void*> vectors) {
    bool chunks = d % 8 == 0, pairs = true;
    for (const NormRows& r : rows) {
        if (!r.p) continue;
        const uintptr_t at = reinterpret_cast<uintptr_t>(r.p);
        chunks = chunks && at % 16 == 0 && r.stride % (r.f32 ? 4 : 8) == 0;
        pairs = pairs && at % (r.f32 ? 8 : 4) == 0 && (r.stride - d) % 2 == 0;
    }
    for (const void* v : vectors) chunks = chunks && reinterpret_cast<uintptr_t>(v) % 16 == 0;
    return chunks ? kChunks : pairs ? kPairs : kSingle;
}

template <typename F>
inline cudaError_t by_form(int dtype, bool res32, int access, F&& f) {
    using std::integral_constant;
    auto with_access = [&](auto dt, auto r32) {
        if (access == kChunks) return f(dt, r32, integral_constant<int, kChunks>{});
        if (access == kPairs) return f(dt, r32, integral_constant<int, kPairs>{});
        return f(dt, r32, integral_constant<int, kSingle>{});
    };
    auto with_residual = [&](auto dt) {
        return res32 ? with_access(dt, std::true_type{}) : with_access(dt, std::false_type{});
    };
    return dtype == MOE_B200_BF16 ? with_residual(integral_constant<int, MOE_B200_BF16>{})
                                  : with_residual(integral_constant<int, MOE_B200_F16>{});
}

}  // namespace moe_b200
