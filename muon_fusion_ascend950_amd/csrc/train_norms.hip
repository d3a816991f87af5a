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
// are kept in registers by the thread that owns the column, over the rows of its
// workgroup; each workgroup writes them once and a second kernel adds the workgroups'
// in index order.  With a gate that all rows of a sequence share, one sum serves two
// gradients: C = Σ dR·n gives d_w1 = gate·C and d_gate = w1·C.
#include "train_common.hpp"

#include <mutex>

namespace muon_train {

namespace {

using Args = muon_train_norms_args;

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

// The column sums a workgroup of the backward pass leaves, [groups][sums][d] fp32, then
// one word a group for a scalar scale's gradient.
enum { kSumPost = 0, kSumPre = 1, kSumScale = 2 };

struct BackwardPlan {
    int nt, v;                 // threads of a workgroup, pieces of a thread
    int64_t groups;            // workgroups
    int64_t groups_per_sequence; // with a sequence gate: a group's rows lie in one sequence
    int sums;                  // column sums: 2, or 3 with a scale vector
    size_t bytes;              // workspace
};

template <class TY, class TR, int NT, int V>
__global__ __launch_bounds__(NT) void norms_backward_kernel(Args a, BackwardPlan plan, float *part,
                                                            float *part_scale) {
    using RawY = typename TY::Raw;
    using RawR = typename TR::Raw;
    __shared__ float red[2][NT / 64 * 3];
    BlockSum<NT / 64, 3> block(red);
    const int tid = threadIdx.x;
    const float inv_d = 1.0f / float(a.d);
    const float number = a.scale_kind == MUON_TRAIN_SCALE_SCALAR ? a.scale[0] : float(a.scale_value);
    const bool seq_gate = a.gate_kind == MUON_TRAIN_GATE_SEQUENCE;
    // Of one channel, dn − n·mean(dn·n) = dn·(1 − n²) = dn·eps·ρ² is all cancellation in
    // fp32: it is formed as that product.
    const bool single = a.d == 1;
    const float eps = float(a.eps);

    // rows of this workgroup: first, first + step, .. below end
    int64_t first = blockIdx.x, step = gridDim.x, end = a.rows;
    int64_t sequence = 0;
    if (seq_gate) {
        sequence = blockIdx.x / plan.groups_per_sequence;
        first = sequence * a.rows_per_sequence + blockIdx.x % plan.groups_per_sequence;
        step = plan.groups_per_sequence;
        end = (sequence + 1) * a.rows_per_sequence;
    }

    int col[V], valid[V];
    float w1[V][8], w2[V][8], gate[V][8], sc[V][8];
    float sum_post[V][8], sum_pre[V][8], sum_scale[V][8], scale_total = 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        col[v] = (v * NT + tid) * 8;
        valid[v] = clamp8(a.d - col[v]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            w1[v][i] = w2[v][i] = gate[v][i] = 1.0f;
            sc[v][i] = number;
            sum_post[v][i] = sum_pre[v][i] = sum_scale[v][i] = 0.0f;
        }
        if (a.post_weight) load8_any(a.post_weight, col[v], valid[v], a.weight_dtype, w1[v]);
        if (a.pre_weight) load8_any(a.pre_weight, col[v], valid[v], a.weight_dtype, w2[v]);
        if (a.scale_kind == MUON_TRAIN_SCALE_VECTOR)
            load8_any(a.scale, col[v], valid[v], MUON_TRAIN_F32, sc[v]);
        if (a.gate_kind == MUON_TRAIN_GATE_CHANNEL || seq_gate)
            load8_any(a.gate, sequence * a.d + col[v], valid[v], a.gate_dtype, gate[v]);
    }
    for (int64_t row = first; row < end; row += step) {
        Piece<TY> py[V], ph[V];
        Piece<TR> pr[V], pt[V];
        const float rho1 = a.stats[2 * row], rho2 = a.stats[2 * row + 1];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            py[v].load(static_cast<const RawY *>(a.y) + row * a.ld_y + col[v], valid[v]);
            pr[v].load(static_cast<const RawR *>(a.residual) + row * a.ld_residual + col[v], valid[v]);
            if (a.d_normed && a.pre_norm)
                ph[v].load(static_cast<const RawY *>(a.d_normed) + row * a.d + col[v], valid[v]);
            else
                ph[v].zero();
            if (a.d_residual_out)
                pt[v].load(static_cast<const RawR *>(a.d_residual_out) + row * a.d + col[v], valid[v]);
            else
                pt[v].zero();
        }
        float token = 1.0f;
        if (a.gate_kind == MUON_TRAIN_GATE_TOKEN) {
            token = load_any(a.gate, row, a.gate_dtype);
#pragma unroll
            for (int v = 0; v < V; ++v)
#pragma unroll
                for (int i = 0; i < 8; ++i) gate[v][i] = token;
        } else if (a.gate_kind == MUON_TRAIN_GATE_FULL) {
#pragma unroll
            for (int v = 0; v < V; ++v)
                load8_any(a.gate, row * a.d + col[v], valid[v], a.gate_dtype, gate[v]);
        }
        float n[V][8], m[V][8], dm[V][8];
        float dot = 0.0f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float r[8], dh[8];
            py[v].get(n[v]);
            pr[v].get(r);
            ph[v].get(dh);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                n[v][i] *= rho1;
                m[v][i] = fmaf(sc[v][i], r[i], gate[v][i] * (n[v][i] * w1[v][i])) * rho2;
                dm[v][i] = dh[i] * w2[v][i];
                dot = fmaf(dm[v][i], m[v][i], dot);
                sum_pre[v][i] = fmaf(dh[i], m[v][i], sum_pre[v][i]);
            }
        }
        const float mean2 = a.pre_norm && !single ? block.sum(dot) * inv_d : 0.0f;
        const float f2 = single ? rho2 * eps * rho2 * rho2 : rho2;
        float s[2] = {0.0f, 0.0f};
        float total_scale = 0.0f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float r[8], dt[8], out[8], dgate[8];
            pr[v].get(r);
            pt[v].get(dt);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float d_total =
                    a.pre_norm ? fmaf(f2, dm[v][i] - m[v][i] * mean2, dt[i]) : dt[i];
                out[i] = sc[v][i] * d_total;
                total_scale = fmaf(d_total, r[i], total_scale);
                sum_scale[v][i] = fmaf(d_total, r[i], sum_scale[v][i]);
                const float with_n = d_total * n[v][i];
                dgate[i] = with_n * w1[v][i];
                s[1] += dgate[i];
                const bool shared = a.gate_kind <= MUON_TRAIN_GATE_SEQUENCE;
                sum_post[v][i] += shared ? with_n : with_n * gate[v][i];
                dm[v][i] = d_total * gate[v][i] * w1[v][i];  // dn from here on
                s[0] = fmaf(dm[v][i], n[v][i], s[0]);
            }
            Piece<TR> o;
            o.set(out);
            o.store(static_cast<RawR *>(a.d_residual) + row * a.d + col[v], valid[v]);
            if (a.gate_kind == MUON_TRAIN_GATE_FULL && a.d_gate)
                store8_any(a.d_gate, row * a.d + col[v], valid[v], a.gate_dtype, dgate);
        }
        scale_total += total_scale;
        block.sum(s);
        if (a.gate_kind == MUON_TRAIN_GATE_TOKEN && a.d_gate && tid == 0)
            store_any(a.d_gate, row, a.gate_dtype, s[1]);
        const float mean1 = a.post_norm && !single ? s[0] * inv_d : 0.0f;
        const float f1 = a.post_norm && single ? rho1 * eps * rho1 * rho1 : rho1;
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
    float *mine = part + int64_t(blockIdx.x) * plan.sums * a.d;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        store8_any(mine, kSumPost * a.d + col[v], valid[v], MUON_TRAIN_F32, sum_post[v]);
        store8_any(mine, kSumPre * a.d + col[v], valid[v], MUON_TRAIN_F32, sum_pre[v]);
        if (plan.sums > kSumScale)
            store8_any(mine, kSumScale * a.d + col[v], valid[v], MUON_TRAIN_F32, sum_scale[v]);
    }
    const float t = block.sum(scale_total);
    if (tid == 0) part_scale[blockIdx.x] = t;
}

// Adds the workgroups' column sums, in index order within each of 16 runs and then run by
// run.  blockIdx.y: the sum.  A workgroup of 64 x 16 threads takes 64 columns.
constexpr int kFinishRuns = 16;
__global__ __launch_bounds__(64 * kFinishRuns) void norms_finish_kernel(Args a, BackwardPlan plan,
                                                                        const float *part,
                                                                        const float *part_scale) {
    __shared__ float red[kFinishRuns][64];
    const int lane = threadIdx.x & 63, run = threadIdx.x >> 6;
    const int64_t d = a.d, stride = plan.sums * d;
    if (int(blockIdx.y) == plan.sums) {  // a scalar scale's gradient
        if (blockIdx.x != 0 || run != 0) return;
        float t = 0.0f;
        for (int64_t g = lane; g < plan.groups; g += 64) t += part_scale[g];
        t = wave_total(t);
        if (lane == 0) a.d_scale[0] = t;
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
#pragma unroll 4
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
    // a gate for each sequence: each run takes whole sequences
    const int64_t sequences = plan.groups / plan.groups_per_sequence;
    const float w = in && a.post_weight ? load_any(a.post_weight, c, a.weight_dtype) : 1.0f;
    float total = 0.0f;
    if (in) {
        for (int64_t b = run; b < sequences; b += kFinishRuns) {
            float t = 0.0f;
            const float *q = p + b * plan.groups_per_sequence * stride;
#pragma unroll 4
            for (int64_t g = 0; g < plan.groups_per_sequence; ++g) t += q[g * stride];
            if (a.d_gate) store_any(a.d_gate, b * d + c, a.gate_dtype, t * w);
            total = fmaf(t, load_any(a.gate, b * d + c, a.gate_dtype), total);
        }
    }
    total = over_runs(total);
    if (in && run == 0 && a.d_post_weight) store_any(a.d_post_weight, c, a.weight_dtype, total);
}

// Threads and pieces of a row: one piece a thread up to 512 columns in one wave, two up to
// 1024; then as many waves as two pieces a thread fill, so that weights and sums stay in
// registers.
struct Shape {
    int nt, v;
};
Shape row_shape(int64_t d) {
    if (d <= 512) return {64, 1};
    if (d <= 1024) return {64, 2};
    if (d <= 2048) return {256, 1};
    if (d <= 4096) return {256, 2};
    if (d <= 8192) return {512, 2};
    return {1024, 2};
}

template <class F>
void with_shape(Shape s, F &&f) {
    using std::integral_constant;
    if (s.nt == 64 && s.v == 1) f(integral_constant<int, 64>{}, integral_constant<int, 1>{});
    else if (s.nt == 64) f(integral_constant<int, 64>{}, integral_constant<int, 2>{});
    else if (s.nt == 256 && s.v == 1) f(integral_constant<int, 256>{}, integral_constant<int, 1>{});
    else if (s.nt == 256) f(integral_constant<int, 256>{}, integral_constant<int, 2>{});
    else if (s.nt == 512) f(integral_constant<int, 512>{}, integral_constant<int, 2>{});
    else f(integral_constant<int, 1024>{}, integral_constant<int, 2>{});
}
template <class F>
void with_types(const Args &a, F &&f) {
    if (a.y_dtype == MUON_TRAIN_BF16 && a.residual_dtype == MUON_TRAIN_BF16) f(Bf16{}, Bf16{});
    else if (a.y_dtype == MUON_TRAIN_BF16) f(Bf16{}, F32{});
    else if (a.residual_dtype == MUON_TRAIN_BF16) f(F32{}, Bf16{});
    else f(F32{}, F32{});
}

BackwardPlan backward_plan(const Args &a, int cus) {
    const Shape s = row_shape(a.d);
    BackwardPlan p{};
    p.nt = s.nt;
    p.v = s.v;
    // workgroups that the card holds at once (about eight waves a compute unit)
    const int64_t resident = int64_t(cus) * (512 / s.nt > 1 ? 512 / s.nt : 1);
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
    p.bytes = sizeof(float) * size_t(p.groups) * (size_t(p.sums) * size_t(a.d) + 1);
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
    const int cus = compute_units();
    if (cus <= 0) return muon_polar::report(MUON_POLAR_ERR_HIP, "norms: no device");
    const Shape s = row_shape(a.d);
    // as many workgroups as stay resident: each keeps its weights over its rows
    const int64_t resident = int64_t(cus) * (2048 / s.nt);
    const dim3 grid(static_cast<uint32_t>(a.rows < resident ? a.rows : resident));
    with_types(a, [&](auto ty, auto tr) {
        with_shape(s, [&](auto nt, auto v) {
            norms_forward_kernel<decltype(ty), decltype(tr), decltype(nt)::value, decltype(v)::value>
                <<<grid, s.nt, 0, stream>>>(a);
        });
    });
    return launched("norms_forward");
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
    const BackwardPlan p = backward_plan(a, cus);
    if (workspace_bytes < p.bytes || (p.bytes > 0 && !workspace))
        return muon_polar::report(MUON_POLAR_ERR_WORKSPACE, "norms: workspace missing or too small");
    if (reinterpret_cast<uintptr_t>(workspace) % 4 != 0)
        return invalid("norms: workspace must be 4-byte aligned");
    float *part = static_cast<float *>(workspace);
    float *part_scale = part + p.groups * p.sums * a.d;
    if (a.rows > 0) {
        with_types(a, [&](auto ty, auto tr) {
            with_shape({p.nt, p.v}, [&](auto nt, auto v) {
                norms_backward_kernel<decltype(ty), decltype(tr), decltype(nt)::value,
                                      decltype(v)::value>
                    <<<dim3(static_cast<uint32_t>(p.groups)), p.nt, 0, stream>>>(a, p, part, part_scale);
            });
        });
        st = launched("norms_backward");
        if (st != MUON_POLAR_OK) return st;
    }
    const bool scalar = a.scale_kind == MUON_TRAIN_SCALE_SCALAR && a.d_scale;
    const bool shared_gate = a.d_gate && (a.gate_kind == MUON_TRAIN_GATE_CHANNEL ||
                                          a.gate_kind == MUON_TRAIN_GATE_SEQUENCE);
    if (!a.d_post_weight && !a.d_pre_weight && !a.d_scale && !shared_gate) return MUON_POLAR_OK;
    const dim3 grid(static_cast<uint32_t>((a.d + 63) / 64), p.sums + (scalar ? 1 : 0));
    norms_finish_kernel<<<grid, 64 * kFinishRuns, 0, stream>>>(a, p, part, part_scale);
    return launched("norms_finish");
}
