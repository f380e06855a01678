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
// The instructions count nearly as much as the bytes (25 an element in the
// forward, 44 in the backward with a channel gate): conversions are packed, the
// backward works on pairs of fp32, calls of the usual form have kernels
// without branches.  Barriers are whole-CTA ones: a named barrier with a
// register for its number reserves 16 of them, which left 25% occupancy.
// Measured on one B200 (bf16, cases back to back): forward with both norms and
// a gate per token, 16384 x 2048: 47 us, 5.7 TB/s, 0.87 of the copy bandwidth;
// backward with a channel gate, 8192 x 4096: 83 us, 4.8 TB/s (77 us for the
// rows, where 2.3 instructions a cycle of 4 are issued at 1.88 GHz, and the rest
// for adding up the CTAs' column sums).
// Wider rows, 33.5 M elements each, gate per token (floor 41 us, backward 61):
// 4096 x 8192: 55 us, backward 95; rows of 4104 columns and more need 512
// threads, whose kernel has 64 registers a thread and spills 4 to 200 bytes of
// them by form.  6553 x 5120: 68 and 120 (those 512 threads hold 8192 columns);
// 3276 x 10240: 85 and 237, 2048 x 16384: 67 and 201 (no ring in the backward).
#include "block_norm.cuh"

namespace moe_b200 {

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
template <int DT, bool RES32, int AL, bool RING, bool WARP, int V, int MAXT, int FORM>
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
    const int odd = odd_of<AL>(row0, t, nt, a.d);
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
        if (!chunk_in<AL, WARP>(i, t, nt, d)) continue;
        if (has_post) wp[i] = load_vec<AL>(a.w_post, i, t, nt, d, odd);
        if (has_pre) wn[i] = load_vec<AL>(a.w_pre, i, t, nt, d, odd);
        if (has_col && !gate_rows) gc[i] = load_vec<AL>(a.gate, i, t, nt, d, odd);
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
            if (!chunk_in<AL, WARP>(i, t, nt, d)) continue;
            const Raw<RES32> res = RING ? load_raw<AL, RES32>(p, i, t, nt, d, odd) : load_raw<AL, RES32>(res_row, i, t, nt, d, odd);
            Raw<false> yr, gr;
            if (has_y) yr = RING ? load_raw<AL, false>(p + a.off_y, i, t, nt, d, odd) : load_raw<AL, false>(y_row, i, t, nt, d, odd);
            if (has_col) {
                gr = gc[i];
                if (gate_rows)
                    gr = RING ? load_raw<AL, false>(p + a.off_gate, i, t, nt, d, odd) : load_raw<AL, false>(g_row, i, t, nt, d, odd);
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
                if (!chunk_in<AL, WARP>(i, t, nt, d)) continue;
#pragma unroll
                for (int j = 0; j < 8; ++j) r[i][j] += z[i][j] * f;
                store8<DT, AL, RES32>(res_out, r[i], i, t, nt, d, odd);
            }
            res_out += step * d * kRes;
        }
        if (has_pre) {
            s[0] = 0.f;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                if (!chunk_in<AL, WARP>(i, t, nt, d)) continue;
#pragma unroll
                for (int j = 0; j < 8; ++j) s[0] += r[i][j] * r[i][j];
            }
            row_sum<WARP>(s, s_red, phase);
            const float c = rsqrtf(s[0] * inv_d + a.eps);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                if (!chunk_in<AL, WARP>(i, t, nt, d)) continue;
#pragma unroll
                for (int j = 0; j < 8; ++j) r[i][j] *= c * raw_get<DT, false>(wn[i], j);
                store8<DT, AL, false>(norm_out, r[i], i, t, nt, d, odd);
            }
            norm_out += step * d;
        }
    }
}

// ----------------------------------------------------------------- host ----

template <int DT, bool RES32, int AL, bool RING, bool WARP, int MAXT, int FORM>
static cudaError_t launch_norm_as(NormArgs a, int cta, int64_t grid, size_t smem, cudaStream_t s) {
    auto kern = block_norm_kernel<DT, RES32, AL, RING, WARP, 2, MAXT, FORM>;
    if (smem > 40 * 1024) {  // beyond what a kernel may use unasked
        static SmemLimit limit;
        const cudaError_t err = limit.open(reinterpret_cast<const void*>(kern));
        if (err != cudaSuccess) return err;
    }
    kern<<<unsigned(grid), cta, smem, s>>>(a);
    return cudaGetLastError();
}

template <int DT, bool RES32, int AL, bool RING, int FORM>
static cudaError_t launch_norm_form(const NormArgs& a, int nt, int64_t grid, size_t smem, cudaStream_t s) {
    if (nt == 32) return launch_norm_as<DT, RES32, AL, RING, true, 128, FORM>(a, 128, grid, smem, s);
    if (nt <= 128) return launch_norm_as<DT, RES32, AL, RING, false, 128, FORM>(a, nt, grid, smem, s);
    if (nt <= 256) return launch_norm_as<DT, RES32, AL, RING, false, 256, FORM>(a, nt, grid, smem, s);
    return launch_norm_as<DT, RES32, AL, RING, false, 1024, FORM>(a, nt, grid, smem, s);
}

template <int DT, bool RES32, int AL>
static cudaError_t launch_norm(const NormArgs& a0, cudaStream_t s) {
    NormArgs a = a0;
    const int nt = row_threads_for(a.d, 2), cta = nt == 32 ? 128 : nt, groups = cta / nt;
    const int per_sm = cta <= 256 ? 768 / cta : 1024 / cta;  // what the registers allow
    const int64_t need = (int64_t(a.T) + groups - 1) / groups, most = int64_t(device_sm_count()) * per_sm;
    if constexpr (AL == kChunks) {
        a.off_y = a.d * (RES32 ? 4 : 2);
        a.off_gate = a.off_y + (a.y ? a.d * 2 : 0);
        a.row_bytes = a.off_gate + (a.gate_form == kGateFull ? a.d * 2 : 0);
        const size_t share = 227 * 1024 / per_sm - 3 * 1024;
        a.stages = kNormStages;
        while (a.stages > 1 && size_t(groups) * a.stages * a.row_bytes > share) --a.stages;
        if (need > most && a.stages > 1) {
            const size_t smem = size_t(groups) * a.stages * a.row_bytes;
            if (a.w_pre) {
                if (!a.y) return launch_norm_form<DT, RES32, AL, true, kFormNorm>(a, nt, most, smem, s);
                if (a.w_post)
                    return a.gate_form >= kGateChannel
                               ? launch_norm_form<DT, RES32, AL, true, kFormFullColGate>(a, nt, most, smem, s)
                               : launch_norm_form<DT, RES32, AL, true, kFormFull>(a, nt, most, smem, s);
                if (a.gate_form < kGateChannel)
                    return launch_norm_form<DT, RES32, AL, true, kFormAddNorm>(a, nt, most, smem, s);
            }
            return launch_norm_form<DT, RES32, AL, true, kFormAny>(a, nt, most, smem, s);
        }
    }
    return launch_norm_form<DT, RES32, AL, false, kFormAny>(a, nt, need < most ? need : steps<AL>(most, groups, a.d), 0, s);
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
    NormArgs a{y, residual, w_post, w_pre, gate, y ? y_stride : 0, residual_stride, gate_form, scale, eps, T, d,
               y ? residual_out : nullptr, w_pre ? normed : nullptr, 0, 0, 0, 0, nullptr};
    const bool res32 = residual_f32 != 0;
    if (inside_element({y, w_post, w_pre, gate, a.normed}, 2) || inside_element({residual, a.residual_out}, res32 ? 4 : 2))
        return fail(MOE_B200_ERR_INVALID_ARG, "block_norm: a pointer is not aligned to its elements");
    const int64_t w16 = 2 * int64_t(d), w_res = (res32 ? 4 : 2) * int64_t(d);
    const RowSet ro{a.residual_out, w_res, w_res, T}, no{a.normed, w16, w16, T};
    const RowSet rows_in[] = {{y, 2 * a.y_stride, w16, T}, {residual, (res32 ? 4 : 2) * residual_stride, w_res, T},
                              {gate_form == kGateFull ? gate : nullptr, w16, w16, T}};
    // A row is read in full before it is written, each column by the thread that
    // writes it: a result may be rows that are read, but not lie on others.
    bool overlap = rows_overlap(ro, no);
    for (const RowSet& out : {ro, no}) {
        for (const RowSet& in : rows_in) overlap = overlap || (!same_rows(out, in) && rows_overlap(out, in));
        overlap = overlap || overlaps_any(out, {whole(w_post, w16), whole(w_pre, w16),
                                                whole(gate_form == kGateFull ? nullptr : gate, gate_form == kGateToken ? 2 * int64_t(T) : w16)});
    }
    if (overlap) return fail(MOE_B200_ERR_INVALID_ARG, "block_norm: a result overlaps an operand or the other result");
    a.status = device_status_word();
    if (!a.status) return fail(MOE_B200_ERR_CUDA, "block_norm: device status word unavailable");
    const int access = access_of(d,
                                 {{y, y_stride, false}, {residual, residual_stride, res32}, {a.residual_out, d, res32},
                                  {a.normed, d, false}, {gate_form == kGateFull ? gate : nullptr, d, false}},
                                 {w_post, w_pre, gate_form == kGateChannel ? gate : nullptr});
    const cudaError_t err = by_form(dtype, res32, access, [&](auto dt, auto r32, auto ali) {
        return launch_norm<decltype(dt)::value, decltype(r32)::value, decltype(ali)::value>(
            a, static_cast<cudaStream_t>(stream));
    });
    return err == cudaSuccess ? MOE_B200_OK : cuda_fail(err, "block_norm launch");
}
