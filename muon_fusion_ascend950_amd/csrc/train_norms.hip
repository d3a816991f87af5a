// train_norms.hip — the norms before and after a block, its gate and its residual scale,
// forward and backward (include/muon_train.h; the formulas are there).
//
// A workgroup holds whole rows in registers, so every operand is read once and every
// result written once: the passes are bound by memory.  Forward: y and residual in,
// residual_out and normed out.  Backward: both again with the two gradients in, d_y and
// d_residual out, R formed anew from y and residual (a saved R would cost the same read)
// with the saved ρ1 and ρ2, so that two row sums remain:
//
//     m = R·ρ2, dm = dh·w2        dR = dR' + ρ2·(dm − m·mean(dm·m))
//     d_residual = scale·dR       du = gate·dR, dn = du·w1
//     d_y = ρ1·(dn − n·mean(dn·n))
//
// Sums over rows (the gradients of weights, of a gate that rows share and of the scale)
// are kept by the thread that owns the column, in registers or (rows past 8192 columns) in
// LDS, over the rows of its workgroup; each workgroup writes them once and a second kernel adds the workgroups'
// in index order.  With a gate that all rows of a sequence share, one sum serves two
// gradients: C = Σ dR·n gives d_w1 = gate·C and d_gate = w1·C.
#include "train_common.hpp"

#include <mutex>
#include <utility>

namespace muon_train {

namespace {

using Args = muon_train_norms_args;

// Over a wave, in a fixed order; the same in every lane.
__device__ __forceinline__ double wave_total(double v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
    return v;
}

__device__ __forceinline__ int clamp8(int64_t n) { return n < 0 ? 0 : n > 8 ? 8 : int(n); }

// NT threads take a row, V pieces of 8 columns each: thread t has the pieces t, t + NT, ..
template <class TY, class TR, int NT, int V>
__global__ __launch_bounds__(NT) void norms_forward_kernel(Args a) {
    using RawY = typename TY::Raw;
    using RawR = typename TR::Raw;
    __shared__ float red[2][NT / 64];
    BlockSum<NT / 64, 1> block(red);
    const int tid = threadIdx.x;
    const float inv_d = 1.0f / float(a.d), eps = float(a.eps);
    const float number = a.scale_kind == MUON_TRAIN_SCALE_SCALAR ? a.scale[0] : float(a.scale_value);

    int col[V], valid[V];
    float w1[V][8], w2[V][8], sc[V][8];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        col[v] = (v * NT + tid) * 8;
        valid[v] = clamp8(a.d - col[v]);
#pragma unroll
        for (int i = 0; i < 8; ++i) w1[v][i] = w2[v][i] = 1.0f, sc[v][i] = number;
        if (a.post_weight) load8_any(a.post_weight, col[v], valid[v], a.weight_dtype, w1[v]);
        if (a.pre_weight) load8_any(a.pre_weight, col[v], valid[v], a.weight_dtype, w2[v]);
        if (a.scale_kind == MUON_TRAIN_SCALE_VECTOR)
            load8_any(a.scale, col[v], valid[v], MUON_TRAIN_F32, sc[v]);
        if (a.gate_kind == MUON_TRAIN_GATE_CHANNEL) {
            float g[8];
            load8_any(a.gate, col[v], valid[v], a.gate_dtype, g);
#pragma unroll
            for (int i = 0; i < 8; ++i) w1[v][i] *= g[i];
        }
    }
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        Piece<TY> py[V];
        Piece<TR> pr[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            py[v].load(static_cast<const RawY *>(a.y) + row * a.ld_y + col[v], valid[v]);
            pr[v].load(static_cast<const RawR *>(a.residual) + row * a.ld_residual + col[v], valid[v]);
        }
        float t[V][8];
        float ss = 0.0f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            py[v].get(t[v]);
#pragma unroll
            for (int i = 0; i < 8; ++i) ss = fmaf(t[v][i], t[v][i], ss);
        }
        const float rho1 = a.post_norm ? 1.0f / sqrtf(block.sum(ss) * inv_d + eps) : 1.0f;
        float f = rho1;
        if (a.gate_kind == MUON_TRAIN_GATE_TOKEN) f *= load_any(a.gate, row, a.gate_dtype);
        ss = 0.0f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float r[8];
            pr[v].get(r);
            if (a.gate_kind == MUON_TRAIN_GATE_SEQUENCE || a.gate_kind == MUON_TRAIN_GATE_FULL) {
                const int64_t at = a.gate_kind == MUON_TRAIN_GATE_FULL ? row : row / a.rows_per_sequence;
                float g[8];
                load8_any(a.gate, at * a.d + col[v], valid[v], a.gate_dtype, g);
#pragma unroll
                for (int i = 0; i < 8; ++i) t[v][i] *= g[i];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                t[v][i] = fmaf(sc[v][i], r[i], t[v][i] * f * w1[v][i]);
                ss = fmaf(t[v][i], t[v][i], ss);
            }
            Piece<TR> o;
            o.set(t[v]);
            o.store(static_cast<RawR *>(a.residual_out) + row * a.d + col[v], valid[v]);
        }
        float rho2 = 1.0f;
        if (a.pre_norm) {
            rho2 = 1.0f / sqrtf(block.sum(ss) * inv_d + eps);
#pragma unroll
            for (int v = 0; v < V; ++v) {
#pragma unroll
                for (int i = 0; i < 8; ++i) t[v][i] = t[v][i] * rho2 * w2[v][i];
                Piece<TY> o;
                o.set(t[v]);
                o.store(static_cast<RawY *>(a.normed) + row * a.d + col[v], valid[v]);
            }
        }
        if (a.stats && tid == 0) {
            a.stats[2 * row] = rho1;
            a.stats[2 * row + 1] = rho2;
        }
    }
}

// What a workgroup of the backward pass leaves: one fp64 word for a scalar scale's gradient
// [groups], then its column sums [groups][sums][d] fp32.
enum { kSumPost = 0, kSumPre = 1, kSumScale = 2 };

struct BackwardPlan {
    int nt, v;                 // threads of a workgroup, pieces of a thread
    int64_t groups;            // workgroups
    int64_t groups_per_sequence; // with a sequence gate: a group's rows lie in one sequence
    int sums;                  // column sums: 2, or 3 with a scale vector
    size_t bytes;              // workspace
};

// kGeneral: a gate of y's shape or a scale vector, whose rows and columns have values of
// their own; without, the gate that rows share is folded into post_weight, a token's is one
// number (it leaves the row's sum Σ dn·n, taken before it, as the gate's own gradient), and
// the scale is one number.
//
// Where registers allow (one piece a thread, not kGeneral) the next row's pieces are under way
// while a row is worked on, whose two sums each wait for the whole workgroup: 16384 rows of
// 4096 in bf16 take 165 us, without 181 to 195 (805 MB: 4.9 TB/s).
template <class TY, class TR, int NT, int V, bool kGeneral>
__global__ __launch_bounds__(NT, V == 1 && !kGeneral ? 4 : 1) void norms_backward_kernel(Args a, BackwardPlan plan,
                                                                           int64_t first_group, float *part,
                                                                           double *part_scale) {
    using RawY = typename TY::Raw;
    using RawR = typename TR::Raw;
    __shared__ float red[2][NT / 64];
    BlockSum<NT / 64, 1> block(red);
    const int tid = threadIdx.x;
    const float inv_d = 1.0f / float(a.d);
    const float number = a.scale_kind == MUON_TRAIN_SCALE_SCALAR ? a.scale[0] : float(a.scale_value);
    const bool seq_gate = a.gate_kind == MUON_TRAIN_GATE_SEQUENCE;
    const bool token_gate = a.gate_kind == MUON_TRAIN_GATE_TOKEN;
    const bool full_gate = kGeneral && a.gate_kind == MUON_TRAIN_GATE_FULL;
    const bool vector_scale = kGeneral && a.scale_kind == MUON_TRAIN_SCALE_VECTOR;
    // Of one channel, dn − n·mean(dn·n) = dn·(1 − n²) = dn·eps·ρ² is all cancellation in
    // fp32: it is formed as that product.
    const bool single = a.d == 1;
    const float eps = float(a.eps);

    // rows of this workgroup, `group` of all: first, first + step, .. below end
    const int64_t group = first_group + blockIdx.x;
    int64_t first = group, step = plan.groups, end = a.rows;
    int64_t sequence = 0;
    if (seq_gate) {
        sequence = group / plan.groups_per_sequence;
        first = sequence * a.rows_per_sequence + group % plan.groups_per_sequence;
        step = plan.groups_per_sequence;
        end = (sequence + 1) * a.rows_per_sequence;
    }

    int col[V], valid[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        col[v] = (v * NT + tid) * 8;
        valid[v] = clamp8(a.d - col[v]);
    }
    constexpr bool kWide = NT == 1024;  // sums in LDS, weights not held
    float held1[kWide ? 1 : V][8], held2[kWide ? 1 : V][8], held_sum[2][kWide ? 1 : V][8];
    __shared__ muon_polar::f32x4 lds_sum[kWide ? 4 * V * NT : 1];
    float sum_scale[kGeneral ? V : 1][8];
    // w1: post_weight times a gate that rows share; w2: pre_weight.
    auto read_weights = [&](int v, float (&w1)[8], float (&w2)[8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) w1[i] = w2[i] = 1.0f;
        if (a.post_weight) load8_any(a.post_weight, col[v], valid[v], a.weight_dtype, w1);
        if (a.pre_weight) load8_any(a.pre_weight, col[v], valid[v], a.weight_dtype, w2);
        if (a.gate_kind == MUON_TRAIN_GATE_CHANNEL || seq_gate) {
            float g[8];
            load8_any(a.gate, sequence * a.d + col[v], valid[v], a.gate_dtype, g);
#pragma unroll
            for (int i = 0; i < 8; ++i) w1[i] *= g[i];
        }
    };
    auto weights = [&](int v, float (&w1)[8], float (&w2)[8]) {
        if constexpr (kWide) {
            read_weights(v, w1, w2);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) w1[i] = held1[v][i], w2[i] = held2[v][i];
        }
    };
    auto get_sum = [&](int which, int v, float (&x)[8]) {
        if constexpr (kWide) {
            const muon_polar::f32x4 lo = lds_sum[(2 * (which * V + v)) * NT + tid], hi = lds_sum[(2 * (which * V + v) + 1) * NT + tid];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = lo[i], x[4 + i] = hi[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = held_sum[which][v][i];
        }
    };
    auto put_sum = [&](int which, int v, const float (&x)[8]) {
        if constexpr (kWide) {
            lds_sum[(2 * (which * V + v)) * NT + tid] = muon_polar::f32x4{x[0], x[1], x[2], x[3]};
            lds_sum[(2 * (which * V + v) + 1) * NT + tid] = muon_polar::f32x4{x[4], x[5], x[6], x[7]};
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) held_sum[which][v][i] = x[i];
        }
    };
    double scale_total = 0.0;  // a scalar scale's gradient: one sum over all elements, which cancel
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const float zero[8] = {};
        put_sum(kSumPost, v, zero);
        put_sum(kSumPre, v, zero);
        if (kGeneral)
#pragma unroll
            for (int i = 0; i < 8; ++i) sum_scale[v][i] = 0.0f;
        if constexpr (!kWide) read_weights(v, held1[v], held2[v]);
    }
    const bool has_dh = a.d_normed && a.pre_norm, has_dt = a.d_residual_out != nullptr;
    struct Row {
        Piece<TY> y[V], h[V];
        Piece<TR> r[V], t[V];
        float rho1, rho2, gate;
    };
    auto fetch = [&](int64_t row, Row &x) {
        x.rho1 = a.stats[2 * row];
        x.rho2 = a.stats[2 * row + 1];
        x.gate = token_gate ? load_any(a.gate, row, a.gate_dtype) : 1.0f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            x.y[v].load(static_cast<const RawY *>(a.y) + row * a.ld_y + col[v], valid[v]);
            x.r[v].load(static_cast<const RawR *>(a.residual) + row * a.ld_residual + col[v], valid[v]);
            if (has_dh) x.h[v].load(static_cast<const RawY *>(a.d_normed) + row * a.d + col[v], valid[v]);
            else x.h[v].zero();
            if (has_dt) x.t[v].load(static_cast<const RawR *>(a.d_residual_out) + row * a.d + col[v], valid[v]);
            else x.t[v].zero();
        }
    };
    constexpr bool kAhead = V == 1 && !kGeneral;
    Row next;
    if (kAhead && first < end) fetch(first, next);
    for (int64_t row = first; row < end; row += step) {
        if (!kAhead) fetch(row, next);
        const Row x = next;
        if (kAhead && row + step < end) fetch(row + step, next);
        const float rho1 = x.rho1, rho2 = x.rho2;
        float n[V][8], m[V][8], dm[V][8], gate[kGeneral ? V : 1][8], sc[kGeneral ? V : 1][8];
        float dot = 0.0f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float r[8], dh[8], w1[8], w2[8], sum_pre[8];
            weights(v, w1, w2);
            get_sum(kSumPre, v, sum_pre);
            x.y[v].get(n[v]);
            x.r[v].get(r);
            x.h[v].get(dh);
            if constexpr (kGeneral) {
#pragma unroll
                for (int i = 0; i < 8; ++i) gate[v][i] = 1.0f, sc[v][i] = number;
                if (full_gate) load8_any(a.gate, row * a.d + col[v], valid[v], a.gate_dtype, gate[v]);
                if (vector_scale) load8_any(a.scale, col[v], valid[v], MUON_TRAIN_F32, sc[v]);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                n[v][i] *= rho1;
                float u = x.gate * (n[v][i] * w1[i]);
                if constexpr (kGeneral) u *= gate[v][i];
                m[v][i] = fmaf(kGeneral ? sc[v][i] : number, r[i], u) * rho2;
                dm[v][i] = dh[i] * w2[i];
                dot = fmaf(dm[v][i], m[v][i], dot);
                sum_pre[i] = fmaf(dh[i], m[v][i], sum_pre[i]);
            }
            put_sum(kSumPre, v, sum_pre);
        }
        const float mean2 = a.pre_norm && !single ? block.sum(dot) * inv_d : 0.0f;
        const float f2 = !a.pre_norm ? 0.0f : single ? rho2 * eps * rho2 * rho2 : rho2;
        float row_dot = 0.0f, row_scale = 0.0f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float r[8], dt[8], out[8], dgate[8], w1[8], w2[8], sum_post[8];
            weights(v, w1, w2);
            get_sum(kSumPost, v, sum_post);
            x.r[v].get(r);
            x.t[v].get(dt);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float d_total = fmaf(f2, dm[v][i] - m[v][i] * mean2, dt[i]);
                out[i] = (kGeneral ? sc[v][i] : number) * d_total;
                row_scale = fmaf(d_total, r[i], row_scale);
                const float with_n = d_total * n[v][i];
                dm[v][i] = d_total * w1[i];  // dn from here on, but for the token's gate
                float weighed = with_n * x.gate;
                if constexpr (kGeneral) {
                    sum_scale[v][i] = fmaf(d_total, r[i], sum_scale[v][i]);
                    dgate[i] = with_n * w1[i];
                    weighed *= gate[v][i];
                    dm[v][i] *= gate[v][i];
                }
                sum_post[i] += weighed;
                row_dot = fmaf(dm[v][i], n[v][i], row_dot);
            }
            put_sum(kSumPost, v, sum_post);
            Piece<TR> o;
            o.set(out);
            o.store(static_cast<RawR *>(a.d_residual) + row * a.d + col[v], valid[v]);
            if (full_gate && a.d_gate)
                store8_any(a.d_gate, row * a.d + col[v], valid[v], a.gate_dtype, dgate);
        }
        scale_total += row_scale;
        row_dot = block.sum(row_dot);
        if (token_gate && a.d_gate && tid == 0) store_any(a.d_gate, row, a.gate_dtype, row_dot);
        const float mean1 = a.post_norm && !single ? row_dot * inv_d : 0.0f;
        const float f1 = x.gate * (a.post_norm && single ? rho1 * eps * rho1 * rho1 : rho1);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float out[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) out[i] = f1 * (dm[v][i] - n[v][i] * mean1);
            Piece<TY> o;
            o.set(out);
            o.store(static_cast<RawY *>(a.d_y) + row * a.d + col[v], valid[v]);
        }
    }
    float *mine = part + group * plan.sums * a.d;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        float sum[8];
        get_sum(kSumPost, v, sum);
        store8_any(mine, kSumPost * a.d + col[v], valid[v], MUON_TRAIN_F32, sum);
        get_sum(kSumPre, v, sum);
        store8_any(mine, kSumPre * a.d + col[v], valid[v], MUON_TRAIN_F32, sum);
        if constexpr (kGeneral)
            if (plan.sums > kSumScale)
                store8_any(mine, kSumScale * a.d + col[v], valid[v], MUON_TRAIN_F32, sum_scale[v]);
    }
    if (a.scale_kind != MUON_TRAIN_SCALE_SCALAR) return;
    __shared__ double totals[NT / 64];
    scale_total = wave_total(scale_total);
    if ((tid & 63) == 0) totals[tid >> 6] = scale_total;
    __syncthreads();
    if (tid == 0) {
        double t = totals[0];
        for (int w = 1; w < NT / 64; ++w) t += totals[w];
        part_scale[group] = t;
    }
}

// Adds the workgroups' column sums, in index order within each of 16 runs and then run by
// run.  blockIdx.y: the sum.  A workgroup of 64 x 16 threads takes 64 columns.
constexpr int kFinishRuns = 16;
__global__ __launch_bounds__(64 * kFinishRuns) void norms_finish_kernel(Args a, BackwardPlan plan,
                                                                        const float *part,
                                                                        const double *part_scale) {
    __shared__ float red[kFinishRuns][64];
    const int lane = threadIdx.x & 63, run = threadIdx.x >> 6;
    const int64_t d = a.d, stride = plan.sums * d;
    if (int(blockIdx.y) == plan.sums) {  // a scalar scale's gradient
        if (blockIdx.x != 0 || run != 0) return;
        double t = 0.0;
        for (int64_t g = lane; g < plan.groups; g += 64) t += part_scale[g];
        t = wave_total(t);
        if (lane == 0) a.d_scale[0] = static_cast<float>(t);
        return;
    }
    const int which = blockIdx.y;
    const int64_t c = int64_t(blockIdx.x) * 64 + lane;
    const bool in = c < d;
    const float *p = part + which * d + c;
    auto over_runs = [&](float t) {
        __syncthreads();
        red[run][lane] = t;
        __syncthreads();
        float s = red[0][lane];
#pragma unroll
        for (int r = 1; r < kFinishRuns; ++r) s += red[r][lane];
        return s;
    };
    auto sum = [&](int64_t g0, int64_t g1) {  // of the groups [g0, g1)
        const int64_t share = (g1 - g0 + kFinishRuns - 1) / kFinishRuns;
        const int64_t lo = g0 + run * share, hi = lo + share < g1 ? lo + share : g1;
        float t = 0.0f;
        if (in) {
#pragma unroll 8
            for (int64_t g = lo; g < hi; ++g) t += p[g * stride];
        }
        return over_runs(t);
    };
    if (which != kSumPost || a.gate_kind != MUON_TRAIN_GATE_SEQUENCE) {
        const float t = sum(0, plan.groups);
        if (!in || run != 0) return;
        if (which == kSumScale) {
            if (a.d_scale) a.d_scale[c] = t;
        } else if (which == kSumPre) {
            if (a.d_pre_weight) store_any(a.d_pre_weight, c, a.weight_dtype, t);
        } else if (a.gate_kind == MUON_TRAIN_GATE_CHANNEL) {
            const float w = a.post_weight ? load_any(a.post_weight, c, a.weight_dtype) : 1.0f;
            if (a.d_post_weight)
                store_any(a.d_post_weight, c, a.weight_dtype, t * load_any(a.gate, c, a.gate_dtype));
            if (a.d_gate) store_any(a.d_gate, c, a.gate_dtype, t * w);
        } else if (a.d_post_weight) {
            store_any(a.d_post_weight, c, a.weight_dtype, t);
        }
        return;
    }
    // a gate for each sequence: with 16 sequences or more each run takes whole ones, with
    // fewer all runs share each
    const int64_t sequences = plan.groups / plan.groups_per_sequence;
    const float w = in && a.post_weight ? load_any(a.post_weight, c, a.weight_dtype) : 1.0f;
    float total = 0.0f;
    auto finish_sequence = [&](int64_t b, float t) {
        if (a.d_gate) store_any(a.d_gate, b * d + c, a.gate_dtype, t * w);
        total = fmaf(t, load_any(a.gate, b * d + c, a.gate_dtype), total);
    };
    if (sequences >= kFinishRuns) {
        for (int64_t b = run; in && b < sequences; b += kFinishRuns) {
            float t = 0.0f;
            const float *q = p + b * plan.groups_per_sequence * stride;
#pragma unroll 4
            for (int64_t g = 0; g < plan.groups_per_sequence; ++g) t += q[g * stride];
            finish_sequence(b, t);
        }
        total = over_runs(total);
    } else {
        for (int64_t b = 0; b < sequences; ++b) {
            const float t = sum(b * plan.groups_per_sequence, (b + 1) * plan.groups_per_sequence);
            if (in && run == 0) finish_sequence(b, t);
        }
    }
    if (in && run == 0 && a.d_post_weight) store_any(a.d_post_weight, c, a.weight_dtype, total);
}

// Threads and pieces of a row.  Forward: one piece a thread up to 512 columns and from 1025 to
// 2048 (64 registers, 32 waves a compute unit), otherwise two (up to 111, 16 waves).  Backward, which holds more: two pieces and up to 256
// registers, 8 waves a compute unit; in bf16 with values that rows share one piece, whose 128
// registers also hold the next row's, 16 waves, as far as 512 threads go.  16384 rows: of 4096
// in bf16 161 us with one piece, 169 with two; with an fp32 residual 284 with one (some spilled)
// and 237 with two, all in fp32 365 and 308; of 5120 (1024 threads would spill more, three in
// eight of them idle) in bf16 254 and 250, fp32 residual 506 and 299, all in fp32 658 and 383.
// Past 8192 columns two pieces of 1024 threads have 128 registers: their column sums lie in LDS
// and the weights are read anew for each row (8192 rows of 16384 in bf16 388 to 413 us, 75 to 80 %
// of the copy rate, in fp32 657, 94 %; with all of it held, 330 registers spilled, 809 and 1395; a gate
// of y's shape still spills 100, 939 us and 44 %).
struct Shape {
    int nt, v;
};
Shape forward_shape(int64_t d) {
    if (d <= 512) return {64, 1};
    if (d <= 1024) return {64, 2};
    if (d <= 2048) return {256, 1};
    if (d <= 4096) return {256, 2};
    if (d <= 8192) return {512, 2};
    return {1024, 2};
}
bool general(const Args &a) {
    return a.gate_kind == MUON_TRAIN_GATE_FULL || a.scale_kind == MUON_TRAIN_SCALE_VECTOR;
}
bool one_piece(const Args &a) {
    return a.y_dtype == MUON_TRAIN_BF16 && a.residual_dtype == MUON_TRAIN_BF16 && !general(a);
}
Shape backward_shape(const Args &a) {
    if (a.d <= 512) return {64, 1};
    const bool one = a.d <= 4096 && one_piece(a);
    for (int nt = 64; nt < 512; nt *= 2)
        if (a.d <= 16 * nt) return one ? Shape{2 * nt, 1} : Shape{nt, 2};
    return {a.d <= 8192 ? 512 : 1024, 2};
}

template <class F>
void with_forward_shape(Shape s, F &&f) {
    using std::integral_constant;
    if (s.nt == 64 && s.v == 1) f(integral_constant<int, 64>{}, integral_constant<int, 1>{});
    else if (s.nt == 64) f(integral_constant<int, 64>{}, integral_constant<int, 2>{});
    else if (s.nt == 256 && s.v == 1) f(integral_constant<int, 256>{}, integral_constant<int, 1>{});
    else if (s.nt == 256) f(integral_constant<int, 256>{}, integral_constant<int, 2>{});
    else if (s.nt == 512) f(integral_constant<int, 512>{}, integral_constant<int, 2>{});
    else f(integral_constant<int, 1024>{}, integral_constant<int, 2>{});
}
template <bool kOnePiece, class F>
void with_backward_shape(Shape s, F &&f) {
    using std::integral_constant;
    constexpr integral_constant<int, 1> one{};
    constexpr integral_constant<int, 2> two{};
    if (s.nt == 1024) return f(integral_constant<int, 1024>{}, two);
    if (s.nt == 512 && s.v == 2) return f(integral_constant<int, 512>{}, two);
    if (s.nt == 64 && s.v == 1) return f(integral_constant<int, 64>{}, one);
    if constexpr (kOnePiece) {
        if (s.nt == 128) f(integral_constant<int, 128>{}, one);
        else if (s.nt == 256) f(integral_constant<int, 256>{}, one);
        else f(integral_constant<int, 512>{}, one);
    } else {
        if (s.nt == 64) f(integral_constant<int, 64>{}, two);
        else if (s.nt == 128) f(integral_constant<int, 128>{}, two);
        else f(integral_constant<int, 256>{}, two);
    }
}
template <class F>
void with_types(const Args &a, F &&f) {
    if (a.y_dtype == MUON_TRAIN_BF16 && a.residual_dtype == MUON_TRAIN_BF16) f(Bf16{}, Bf16{});
    else if (a.y_dtype == MUON_TRAIN_BF16) f(Bf16{}, F32{});
    else if (a.residual_dtype == MUON_TRAIN_BF16) f(F32{}, Bf16{});
    else f(F32{}, F32{});
}

BackwardPlan backward_plan(const Args &a, int cus) {
    const Shape s = backward_shape(a);
    BackwardPlan p{};
    p.nt = s.nt;
    p.v = s.v;
    // workgroups that the card holds at once: 16 waves a compute unit, 8 of two pieces
    const int64_t resident = int64_t(cus) * (s.v == 1 || s.nt == 1024 ? 1024 / s.nt : 512 / s.nt);
    p.groups_per_sequence = 1;
    if (a.gate_kind == MUON_TRAIN_GATE_SEQUENCE && a.rows > 0) {
        const int64_t sequences = a.rows / a.rows_per_sequence;
        p.groups_per_sequence = (resident + sequences - 1) / sequences;
        if (p.groups_per_sequence > a.rows_per_sequence) p.groups_per_sequence = a.rows_per_sequence;
        p.groups = sequences * p.groups_per_sequence;
    } else {
        p.groups = a.rows < resident ? a.rows : resident;
    }
    p.sums = a.scale_kind == MUON_TRAIN_SCALE_VECTOR ? 3 : 2;
    p.bytes = size_t(p.groups) * (sizeof(double) + sizeof(float) * size_t(p.sums) * size_t(a.d));
    return p;
}

bool dtype_ok(int t) { return t == MUON_TRAIN_F32 || t == MUON_TRAIN_BF16; }

int check(const Args *a) {
    if (!a) return invalid("norms: args is null");
    if (a->rows < 0 || a->d < 1 || a->d > 16384 || a->rows > (int64_t(1) << 40))
        return invalid("norms: rows must not be negative and d must be 1 to 16384");
    if (!dtype_ok(a->y_dtype) || !dtype_ok(a->residual_dtype) || !dtype_ok(a->weight_dtype) ||
        !dtype_ok(a->gate_dtype))
        return invalid("norms: dtypes must be float32 or bfloat16");
    if (a->gate_kind < MUON_TRAIN_GATE_NONE || a->gate_kind > MUON_TRAIN_GATE_FULL ||
        a->scale_kind < MUON_TRAIN_SCALE_NUMBER || a->scale_kind > MUON_TRAIN_SCALE_VECTOR)
        return invalid("norms: unknown kind of gate or scale");
    if (a->gate_kind == MUON_TRAIN_GATE_SEQUENCE &&
        (a->rows_per_sequence < 1 || a->rows % a->rows_per_sequence != 0))
        return invalid("norms: rows_per_sequence must divide rows");
    if (a->rows == 0) return MUON_POLAR_OK;
    if (!a->y || !a->residual || (a->gate_kind != MUON_TRAIN_GATE_NONE && !a->gate) ||
        (a->scale_kind != MUON_TRAIN_SCALE_NUMBER && !a->scale))
        return invalid("norms: null pointer");
    if (a->ld_y < a->d || a->ld_residual < a->d)
        return invalid("norms: rows of y and residual must not overlap");
    return MUON_POLAR_OK;
}

// Whether an output [rows, d] meets one of the inputs that a pass reads, or another output.
bool outputs_meet(const Args &a, const void *r_out, const void *y_out, const void *r_in,
                  const void *y_in) {
    const int64_t sy = a.y_dtype == MUON_TRAIN_BF16 ? 2 : 4, sr = a.residual_dtype == MUON_TRAIN_BF16 ? 2 : 4;
    const int64_t whole_y = a.rows * a.d * sy, whole_r = a.rows * a.d * sr;
    const int64_t span_y = ((a.rows - 1) * a.ld_y + a.d) * sy;
    const int64_t span_r = ((a.rows - 1) * a.ld_residual + a.d) * sr;
    bool bad = meet(r_out, whole_r, y_out, whole_y);
    const std::pair<const void *, int64_t> outs[] = {{r_out, whole_r}, {y_out, whole_y}};
    for (const auto &[out, bytes] : outs)
        bad = bad || meet(out, bytes, a.y, span_y) || meet(out, bytes, a.residual, span_r) ||
              meet(out, bytes, r_in, whole_r) || meet(out, bytes, y_in, whole_y);
    return bad;
}

}  // namespace

int compute_units() noexcept {
    static std::mutex mutex;
    static int known[64];
    int device = 0;
    if (hipGetDevice(&device) != hipSuccess || device < 0 || device >= 64) return 0;
    std::lock_guard<std::mutex> lock(mutex);
    if (known[device] == 0) {
        int n = 0;
        if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess)
            return 0;
        known[device] = n;
    }
    return known[device];
}

}  // namespace muon_train

using namespace muon_train;

extern "C" int muon_train_norms_forward(const muon_train_norms_args *args, hipStream_t stream) {
    int st = check(args);
    if (st != MUON_POLAR_OK || args->rows == 0) return st;
    const Args a = *args;
    if (!a.residual_out || (a.pre_norm && !a.normed)) return invalid("norms: null output");
    if (outputs_meet(a, a.residual_out, a.pre_norm ? a.normed : nullptr, nullptr, nullptr))
        return invalid("norms: outputs must not overlap inputs or each other");
    const int cus = compute_units();
    if (cus <= 0) return muon_polar::report(MUON_POLAR_ERR_HIP, "norms: no device");
    const Shape s = forward_shape(a.d);
    // up to 32 waves a compute unit: each workgroup keeps its weights over its rows
    const int64_t resident = int64_t(cus) * (2048 / s.nt);
    const dim3 grid(static_cast<uint32_t>(a.rows < resident ? a.rows : resident));
    Launches launch{stream};
    with_types(a, [&](auto ty, auto tr) {
        with_forward_shape(s, [&](auto nt, auto v) {
            launch(norms_forward_kernel<decltype(ty), decltype(tr), decltype(nt)::value, decltype(v)::value>,
                   grid, s.nt, a);
        });
    });
    return launch.result("norms_forward");
}

extern "C" int muon_train_norms_workspace(const muon_train_norms_args *args, size_t *bytes) {
    const int st = check(args);
    if (st != MUON_POLAR_OK) return st;
    if (!bytes) return invalid("norms: bytes is null");
    const int cus = compute_units();
    if (cus <= 0) return muon_polar::report(MUON_POLAR_ERR_HIP, "norms: no device");
    *bytes = backward_plan(*args, cus).bytes;
    return MUON_POLAR_OK;
}

extern "C" int muon_train_norms_backward(const muon_train_norms_args *args, void *workspace,
                                         size_t workspace_bytes, hipStream_t stream) {
    int st = check(args);
    if (st != MUON_POLAR_OK) return st;
    const Args a = *args;
    const int cus = compute_units();
    if (cus <= 0) return muon_polar::report(MUON_POLAR_ERR_HIP, "norms: no device");
    if (a.rows > 0 && (!a.stats || !a.d_y || !a.d_residual)) return invalid("norms: null output");
    if (a.rows > 0 && outputs_meet(a, a.d_residual, a.d_y, a.d_residual_out, a.d_normed))
        return invalid("norms: outputs must not overlap inputs or each other");
    const BackwardPlan p = backward_plan(a, cus);
    if (workspace_bytes < p.bytes || (p.bytes > 0 && !workspace))
        return muon_polar::report(MUON_POLAR_ERR_WORKSPACE, "norms: workspace missing or too small");
    if (reinterpret_cast<uintptr_t>(workspace) % 8 != 0)
        return invalid("norms: workspace must be 8-byte aligned");
    double *part_scale = static_cast<double *>(workspace);
    float *part = reinterpret_cast<float *>(part_scale + p.groups);
    Launches launch{stream};
    if (a.rows > 0) {
        with_types(a, [&](auto ty, auto tr) {
            auto go = [&](auto is_general) {
                constexpr bool kGeneral = decltype(is_general)::value;
                constexpr bool kOnePiece = std::is_same_v<decltype(ty), Bf16> && std::is_same_v<decltype(tr), Bf16> && !kGeneral;
                with_backward_shape<kOnePiece>({p.nt, p.v}, [&](auto nt, auto v) {
                    // one launch but for gates of very many sequences
                    const int64_t most = kMaxThreads / p.nt;
                    for (int64_t g = 0; g < p.groups; g += most) {
                        const dim3 grid(static_cast<uint32_t>(p.groups - g < most ? p.groups - g : most));
                        launch(norms_backward_kernel<decltype(ty), decltype(tr), decltype(nt)::value, decltype(v)::value, kGeneral>,
                               grid, p.nt, a, p, g, part, part_scale);
                    }
                });
            };
            if (general(a)) go(std::true_type{});
            else go(std::false_type{});
        });
        st = launch.result("norms_backward");
        if (st != MUON_POLAR_OK) return st;
    }
    const bool scalar = a.scale_kind == MUON_TRAIN_SCALE_SCALAR && a.d_scale;
    const bool shared_gate = a.d_gate && (a.gate_kind == MUON_TRAIN_GATE_CHANNEL ||
                                          a.gate_kind == MUON_TRAIN_GATE_SEQUENCE);
    if (!a.d_post_weight && !a.d_pre_weight && !a.d_scale && !shared_gate) return MUON_POLAR_OK;
    const dim3 grid(static_cast<uint32_t>((a.d + 63) / 64), p.sums + (scalar ? 1 : 0));
    launch(norms_finish_kernel, grid, 64 * kFinishRuns, a, p, part, part_scale);
    return launch.result("norms_finish");
}
