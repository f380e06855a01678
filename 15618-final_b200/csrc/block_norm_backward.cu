// block_norm_backward.cu -- gradients of the norms around a block; the formulas
// and what bounds them stand in block_norm.cu.
#include "block_norm.cuh"

namespace moe_b200 {

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
template <int DT, bool RES32, int AL, bool RING, bool WARP, int V, int MAXT, int GATE>
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
    const int odd = odd_of<AL>(row0, t, nt, a.d);
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

    // In pairs: this thread's columns of the weights, as it will need them.
    uint32_t* s_own = reinterpret_cast<uint32_t*>(s_dyn) + threadIdx.x;
    if (AL == kPairs) {
        auto keep = [&](const void* vec, int at) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const Raw<false> w = load_vec<AL>(vec, i, t, nt, d, odd);
#pragma unroll
                for (int k = 0; k < 4; ++k) s_own[((at * V + i) * 4 + k) * blockDim.x] = w.w[k];
            }
        };
        if (has_pre) keep(a.w_pre, 0);
        if (has_post) keep(a.w_post, has_pre);
        if (gate_form == kGateChannel) keep(a.gate, has_pre + has_post);
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
            return RING ? load_raw<AL, false, true>(p + off, i, t, nt, d, odd) : load_raw<AL, false, true>(g, i, t, nt, d, odd);
        };
        auto getres = [&](int off, const char* g, int i) {
            return RING ? load_raw<AL, RES32, true>(p + off, i, t, nt, d, odd) : load_raw<AL, RES32, true>(g, i, t, nt, d, odd);
        };
        auto getw = [&](const unsigned char* s, const void* g, int vec, int i) {
            if constexpr (AL != kPairs) {
                return load_raw<AL, false, true>(RING ? s : g, i, t, nt, d, 0);
            } else {
                Raw<false> w;
#pragma unroll
                for (int k = 0; k < 4; ++k) w.w[k] = s_own[((vec * V + i) * 4 + k) * blockDim.x];
                return w;
            }
        };
        f32x2 p_rr = 0, p_ur = 0, p_yy = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (!chunk_in<AL, WARP>(i, t, nt, d)) continue;
            if (has_pre) {
                const Raw<false> wn = getw(s_wpre, a.w_pre, 0, i);
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
            if (!chunk_in<AL, WARP>(i, t, nt, d)) continue;
            if (has_ds) {
                const Raw<RES32> ds = getres(a.off_ds, ds_row(row), i);
#pragma unroll
                for (int j = 0; j < 4; ++j) q[i][j] = raw_pair<DT, RES32>(ds, j);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) q[i][j] = 0;
            }
            if (has_pre) {
                const Raw<false> wn = getw(s_wpre, a.w_pre, 0, i);
                const Raw<false> dn = get16(a.off_dn, dn_row(row), i);
                const Raw<RES32> rr = getres(a.off_rr, rr_row(row), i);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const f32x2 rc = mul2(raw_pair<DT, RES32>(rr, j), c2), dnj = raw_pair<DT, false>(dn, j);
                    s_pre[i][j] = fma2(dnj, rc, s_pre[i][j]);
                    q[i][j] = fma2(c2, mul2(dnj, raw_pair<DT, false>(wn, j)), fma2(rc, k2, q[i][j]));
                }
            }
            store8<DT, AL, RES32>(dres_out, q[i], i, t, nt, d, odd);
            if (has_y) {
                yr[i] = get16(a.off_y, y_row(row), i);
                Raw<false> wp, gr;
                if (has_post) wp = getw(s_wpost, a.w_post, has_pre, i);
                if (gate_form == kGateChannel) gr = getw(s_wgate, a.gate, has_pre + has_post, i);
                if (gate_form == kGateFull) {
                    gr = get16(a.off_gate, g_row(row), i);
                    f32x2 dg[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        dg[j] = mul2(mul2(q[i][j], dg2), raw_pair<DT, false>(yr[i], j));
                        if (has_post) dg[j] = mul2(dg[j], raw_pair<DT, false>(wp, j));
                        q[i][j] = mul2(q[i][j], raw_pair<DT, false>(gr, j));
                    }
                    store8<DT, AL, false>(dg_out, dg, i, t, nt, d, odd);
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
                if (!chunk_in<AL, WARP>(i, t, nt, d)) continue;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    q[i][j] = has_post ? fma2(fp2, q[i][j], mul2(raw_pair<DT, false>(yr[i], j), m2)) : mul2(q[i][j], f2);
                store8<DT, AL, false>(dy_out, q[i], i, t, nt, d, odd);
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
                        const int col = col_of<AL>(i, j, t, nt, odd);
                        if (col >= 0 && col < d) s_col[col] = g == 0 ? s[i][j] : s_col[col] + s[i][j];
                    }
            }
            __syncthreads();
        }
        if (group == groups - 1) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                if (!chunk_in<AL, WARP>(i, t, nt, d)) continue;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int col = col_of<AL>(i, j, t, nt, odd);
                    if (groups > 1 && col >= 0 && col < d) s[i][j] += s_col[col];
                }
                auto row_of = [&](int vec) { return a.part + (int64_t(vec) * gridDim.x + blockIdx.x) * d; };
                if (which == 0) {
                    store_vec<DT, AL>(row_of(a.sum_pre), s[i], i, t, nt, d, odd);
                } else if (a.sum_gate < 0) {
                    store_vec<DT, AL>(row_of(a.sum_post), s[i], i, t, nt, d, odd);
                } else {
                    const Raw<false> gr = load_vec<AL>(a.gate, i, t, nt, d, odd);
                    float v[8];
                    if (has_post) {
                        const Raw<false> wp = load_vec<AL>(a.w_post, i, t, nt, d, odd);
#pragma unroll
                        for (int j = 0; j < 8; ++j) v[j] = a.scale * raw_get<DT, false>(gr, j) * s[i][j];
                        store_vec<DT, AL>(row_of(a.sum_post), v, i, t, nt, d, odd);
#pragma unroll
                        for (int j = 0; j < 8; ++j) s[i][j] *= raw_get<DT, false>(wp, j);
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] = a.scale * s[i][j];
                    store_vec<DT, AL>(row_of(a.sum_gate), v, i, t, nt, d, odd);
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
    // hand fit 128 registers.  The widest rows take four, without a ring, and
    // spill: 152 to 184 bytes in chunks, 416 to 440 in pairs, 792 to 880 one by
    // one (2048 x 16384, bf16: 201 us; 2000 x 16383: 394).
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

template <int DT, bool RES32, int AL, bool RING, bool WARP, int V, int GATE = -1>
static cudaError_t launch_norm_backward_as(const NormGradArgs& a, const NormGradPlan& p, size_t smem, cudaStream_t s) {
    constexpr int kMax = WARP ? 128 : 512;
    auto kern = block_norm_backward_kernel<DT, RES32, AL, RING, WARP, V, kMax, GATE>;
    if (smem > 40 * 1024) {  // beyond what a kernel may use unasked
        static SmemLimit limit;
        const cudaError_t err = limit.open(reinterpret_cast<const void*>(kern));
        if (err != cudaSuccess) return err;
    }
    kern<<<p.grid, p.cta_threads, smem, s>>>(a);
    return cudaGetLastError();
}

template <int DT, bool RES32, bool WARP>
static cudaError_t launch_norm_backward_ring(const NormGradArgs& a, const NormGradPlan& p, size_t smem, cudaStream_t s) {
    if (a.w_pre && a.w_post && a.d_res_out) {
        if (a.gate_form == kGateNone) return launch_norm_backward_as<DT, RES32, kChunks, true, WARP, 2, kGateNone>(a, p, smem, s);
        if (a.gate_form == kGateToken) return launch_norm_backward_as<DT, RES32, kChunks, true, WARP, 2, kGateToken>(a, p, smem, s);
        if (a.gate_form == kGateChannel)
            return launch_norm_backward_as<DT, RES32, kChunks, true, WARP, 2, kGateChannel>(a, p, smem, s);
        return launch_norm_backward_as<DT, RES32, kChunks, true, WARP, 2, kGateFull>(a, p, smem, s);
    }
    return launch_norm_backward_as<DT, RES32, kChunks, true, WARP, 2>(a, p, smem, s);
}

template <int DT, bool RES32, int AL>
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
    const bool use_ring = AL == kChunks && p.v == 2 && a.stages > 1;
    const size_t own = AL == kPairs ? size_t(p.cta_threads) * p.v * 16 * (weights / (2 * size_t(a.d))) : 0;
    size_t smem = use_ring ? ring : own;
    if (smem < cols) smem = cols;
    const bool warp = p.row_threads == 32;
    if constexpr (AL == kChunks) {
        if (use_ring) {
            if (warp) return launch_norm_backward_ring<DT, RES32, true>(a, p, smem, s);
            return launch_norm_backward_ring<DT, RES32, false>(a, p, smem, s);
        }
    }
    if (warp) return launch_norm_backward_as<DT, RES32, AL, false, true, 2>(a, p, smem, s);
    if (p.v == 2) return launch_norm_backward_as<DT, RES32, AL, false, false, 2>(a, p, smem, s);
    return launch_norm_backward_as<DT, RES32, AL, false, false, 4>(a, p, smem, s);
}

}  // namespace moe_b200

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
    if (inside_element({y, w_post, w_pre, gate, w_pre ? d_normed : nullptr, y ? d_y : nullptr}, 2) ||
        inside_element({d_residual_out, w_pre ? residual_out : nullptr, d_residual}, res32 ? 4 : 2) ||
        inside_element({w_post ? d_w_post : nullptr, w_pre ? d_w_pre : nullptr}, 4) ||
        inside_element({gate ? d_gate : nullptr}, gate_form == kGateFull ? 2 : 4))
        return fail(MOE_B200_ERR_INVALID_ARG, "block_norm_backward: a pointer is not aligned to its elements");
    NormGradPlan p = plan_norm_backward(T, d);
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
    const int64_t w16 = 2 * int64_t(d), w32 = 4 * int64_t(d), w_res = (res32 ? 4 : 2) * int64_t(d);
    const bool full = gate_form == kGateFull;
    const RowSet in_ds{d_residual_out, w_res, w_res, T}, in_rr{w_pre ? residual_out : nullptr, (res32 ? 4 : 2) * residual_stride, w_res, T};
    const RowSet in_dn{w_pre ? d_normed : nullptr, w16, w16, T}, in_y{y, 2 * y_stride, w16, T};
    const RowSet in_gate = full ? RowSet{gate, w16, w16, T} : whole(gate, gate_form == kGateToken ? 2 * int64_t(T) : w16);
    const RowSet out_r{d_residual, w_res, w_res, T}, out_y{y ? d_y : nullptr, w16, w16, T};
    const RowSet out_g = !gate  ? whole(nullptr, 0)
                         : full ? RowSet{d_gate, w16, w16, T}
                                : whole(d_gate, gate_form == kGateToken ? 4 * int64_t(T) : w32);
    const RowSet flat[] = {whole(w_post ? d_w_post : nullptr, w32), whole(w_pre ? d_w_pre : nullptr, w32),
                           whole(vectors ? workspace : nullptr, int64_t(align256(size_t(vectors) * p.grid * size_t(d) * 4)))};
    // A thread reads its columns of a row, then writes d_residual, then reads the
    // row's y and gate, then writes d_gate and d_y: a result may be rows that are
    // read before it is written, but not lie on others.
    auto on = [](const RowSet& out, std::initializer_list<RowSet> others) {
        for (const RowSet& o : others)
            if (!same_rows(out, o) && rows_overlap(out, o)) return true;
        return false;
    };
    bool overlap = on(out_r, {in_ds, in_rr, in_dn}) || overlaps_any(out_r, {in_y, in_gate, out_y, out_g}) ||
                   on(out_y, {in_ds, in_rr, in_dn, in_y, in_gate}) || on(out_g, {in_ds, in_rr, in_dn, in_y, in_gate}) ||
                   rows_overlap(out_y, out_g) || rows_overlap(flat[0], flat[1]) || rows_overlap(flat[0], flat[2]) ||
                   rows_overlap(flat[1], flat[2]);
    for (const RowSet& out : {out_r, out_y, out_g}) overlap = overlap || overlaps_any(out, {whole(w_post, w16), whole(w_pre, w16)});
    for (const RowSet& f : flat)
        overlap = overlap || overlaps_any(f, {in_ds, in_rr, in_dn, in_y, in_gate, whole(w_post, w16), whole(w_pre, w16), out_r, out_y, out_g});
    if (overlap) return fail(MOE_B200_ERR_INVALID_ARG, "block_norm_backward: a result overlaps an operand or another result");
    uint32_t* status = device_status_word();
    if (!status) return fail(MOE_B200_ERR_CUDA, "block_norm_backward: device status word unavailable");
    const NormGradArgs a{d_residual_out, d_normed, residual_out, y, w_post, w_pre, gate, y ? y_stride : 0,
                         w_pre ? residual_stride : 0, gate_form, scale, eps, T, d, d_residual, d_y, d_gate,
                         static_cast<float*>(workspace), i_pre, i_post, i_gate, 0, -1, -1, -1, -1, -1, 0, 0, status};
    const int access = access_of(d,
                                 {{d_residual_out, d, res32}, {d_normed, d, false}, {w_pre ? residual_out : nullptr, residual_stride, res32},
                                  {y, y_stride, false}, {d_residual, d, res32}, {d_y, d, false},
                                  {gate_form == kGateFull ? gate : nullptr, d, false},
                                  {gate_form == kGateFull ? d_gate : nullptr, d, false}},
                                 {w_post, w_pre, gate_form == kGateChannel ? gate : nullptr});
    if (access == kPairs && int64_t(p.grid) * (p.cta_threads / p.row_threads) < T)
        p.grid = int(steps<kPairs>(p.grid, p.cta_threads / p.row_threads, d));
    cudaError_t err = by_form(dtype, res32, access, [&](auto dt, auto r32, auto ali) {
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
