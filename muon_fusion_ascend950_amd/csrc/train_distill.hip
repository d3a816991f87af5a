// train_distill.hip — the loss against a teacher's top logits, its gradient, and both in
// one pass (include/muon_train.h; the formulas are there).
//
// One workgroup a row.  The row is loaded into registers whole (up to 256 KiB: 1024
// threads with 16 pieces of 16 bytes each), its maximum and its sum of exponentials are
// taken from there, and the gradient is written from there: the logits cross memory once
// in and once out, which is what bounds the pass.  Of a longer row the threads take the
// rest with a running maximum and sum, and read it again for the gradient.
//
// The gradient is the softmax everywhere but at the teacher's indices and the label.  All
// of the row is written as softmax first; then, past a barrier, each entry overwrites its
// element with the softmax less the sum of all amounts that lie on that index (the same
// bits from every entry of an index that occurs twice).
#include "train_common.hpp"

namespace muon_train {

namespace {

using Args = muon_train_distill_args;

constexpr int kMaxTop = 1024;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kNegInf = -__builtin_inff();

// 16 bytes of a row: 8 bf16 or 4 fp32 logits; those past the row's end read as −inf.
template <class T>
struct Chunk {
    static constexpr int kElems = 16 / sizeof(typename T::Raw);
    u32x4 v;
    __device__ __forceinline__ void load(const typename T::Raw *p, int valid) {
        if (valid >= kElems) {
            __builtin_memcpy(&v, p, 16);
        } else if constexpr (kElems == 8) {
            uint32_t h[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) h[i] = i < valid ? p[i] : 0xff80u;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = h[2 * i] | (h[2 * i + 1] << 16);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = i < valid ? __float_as_uint(p[i]) : 0xff800000u;
        }
    }
    __device__ __forceinline__ void get(float (&f)[kElems]) const {
        if constexpr (kElems == 8) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                f[2 * i] = __uint_as_float(v[i] << 16);
                f[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(v[i]);
        }
    }
    __device__ __forceinline__ void set(const float (&f)[kElems]) {
        if constexpr (kElems == 8) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                v[i] = f32_to_bf16_bits(f[2 * i]) | uint32_t(f32_to_bf16_bits(f[2 * i + 1])) << 16;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = __float_as_uint(f[i]);
        }
    }
    __device__ __forceinline__ void store(typename T::Raw *p, int valid) const {
        if (valid >= kElems) {
            __builtin_memcpy(p, &v, 16);
        } else {
#pragma unroll
            for (int i = 0; i < kElems; ++i)
                if (i < valid) {
                    if constexpr (kElems == 8)
                        p[i] = static_cast<uint16_t>(v[i / 2] >> (16 * (i & 1)));
                    else
                        p[i] = __uint_as_float(v[i]);
                }
        }
    }
};

__device__ __forceinline__ int64_t load_index(const Args &a, int64_t i) {
    return a.index_bytes == 4 ? static_cast<const int32_t *>(a.teacher_indices)[i]
                              : static_cast<const int64_t *>(a.teacher_indices)[i];
}
// 2^x by the hardware instruction (1 ulp; results under the normal range become 0, as
// their share of a sum whose largest term is 1 does).
__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

enum { kLoss = 0, kLossAndGrad = 1, kGradFromStats = 2 };

// NT threads a row, R chunks of it in each thread's registers.  kHard: with labels.
template <class T, int NT, int R, int MODE, bool kHard>
__global__ __launch_bounds__(NT) void distill_kernel(Args a) {
    using Raw = typename T::Raw;
    using C = Chunk<T>;
    constexpr int E = C::kElems, NW = NT / 64, kTops = kMaxTop / NT;
    __shared__ float red[2][NW * 3];
    __shared__ int entry_at[kMaxTop + 1];
    __shared__ float entry_amount[kMaxTop + 1];
    BlockSum<NW, 3> block(red);
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.x;
    const int vocab = static_cast<int>(a.vocab), k = static_cast<int>(a.k);
    const Raw *z = static_cast<const Raw *>(a.logits) + row * a.ld_logits;
    const float tau = float(a.temperature), lam = kHard ? float(a.label_weight) : 0.0f;
    const float c = kLog2e / tau;  // exponents in powers of two

    C zr[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int at = (r * NT + tid) * E;
        zr[r].load(z + at, vocab - at);
    }
    constexpr int kHeld = R * NT * E;  // elements of the row that registers hold

    // the teacher's entries of this thread, and the student's logits there
    float t[kTops], zk[kTops];
    int index[kTops];
    float top[2] = {kNegInf, kNegInf};  // of z, of t
#pragma unroll
    for (int j = 0; j < kTops; ++j) {
        const int e = j * NT + tid;
        index[j] = -1;
        t[j] = kNegInf;
        zk[j] = 0.0f;
        if (e < k) {
            const int64_t i = load_index(a, row * k + e);
            if (i >= 0 && i < a.vocab) {
                index[j] = static_cast<int>(i);
                t[j] = load_any(a.teacher_logits, row * k + e, a.teacher_dtype);
                zk[j] = to_f32(z[i]);
            }
            top[1] = fmaxf(top[1], t[j]);
        }
    }
    int64_t label = -1;
    float z_label = 0.0f;
    if constexpr (kHard) {
        label = a.labels[row];
        if (label < 0 || label >= a.vocab) label = -1;
        if (label >= 0) z_label = to_f32(z[label]);
    }

    // maxima; of the part past the registers a running sum too
    float run_max = kNegInf, run_sum = 0.0f, run_hard = 0.0f;
    if constexpr (MODE != kGradFromStats) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float f[E];
            zr[r].get(f);
#pragma unroll
            for (int i = 0; i < E; ++i) top[0] = fmaxf(top[0], f[i]);
        }
        for (int at = kHeld + tid * E; at < vocab; at += NT * E) {
            C x;
            float f[E];
            x.load(z + at, vocab - at);
            x.get(f);
            float m = run_max;
#pragma unroll
            for (int i = 0; i < E; ++i) m = fmaxf(m, f[i]);
            if (m > run_max) {
                run_sum *= exp2_hw((run_max - m) * c);
                if constexpr (kHard) run_hard *= exp2_hw((run_max - m) * kLog2e);
                run_max = m;
            }
            if (run_max > kNegInf) {
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    run_sum += exp2_hw((f[i] - run_max) * c);
                    if constexpr (kHard) run_hard += exp2_hw((f[i] - run_max) * kLog2e);
                }
            } else {  // −inf so far, or a NaN, which the maximum passes over
#pragma unroll
                for (int i = 0; i < E; ++i) run_sum += f[i] != f[i] ? f[i] : 0.0f;
            }
        }
        top[0] = fmaxf(top[0], run_max);
    }
    block.max(top);
    const float t_max = top[1];
    float z_max = top[0];

    float sum[3] = {0.0f, 0.0f, 0.0f};  // of the student at τ, of the teacher, of the student at 1
    float pe[kTops];
#pragma unroll
    for (int j = 0; j < kTops; ++j) {
        pe[j] = index[j] >= 0 && t_max > kNegInf ? exp2_hw((t[j] - t_max) * c) : 0.0f;
        if (index[j] >= 0 && t[j] != t[j]) pe[j] = t[j];
        sum[1] += pe[j];
    }
    if constexpr (MODE != kGradFromStats) {
        if (run_max > kNegInf) {
            sum[0] = run_sum * exp2_hw((run_max - z_max) * c);
            if constexpr (kHard) sum[2] = run_hard * exp2_hw((run_max - z_max) * kLog2e);
        } else {
            sum[0] = run_sum;
            if constexpr (kHard) sum[2] = run_sum;
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float f[E];
            zr[r].get(f);
#pragma unroll
            for (int i = 0; i < E; ++i) {
                sum[0] += exp2_hw((f[i] - z_max) * c);
                if constexpr (kHard) sum[2] += exp2_hw((f[i] - z_max) * kLog2e);
            }
        }
    }
    block.sum(sum);
    float inv_sum, inv_hard = 0.0f;
    if constexpr (MODE == kGradFromStats) {
        z_max = a.stats[4 * row];
        inv_sum = a.stats[4 * row + 1];
        inv_hard = a.stats[4 * row + 2];
    } else {
        inv_sum = 1.0f / sum[0];
        if constexpr (kHard) inv_hard = 1.0f / sum[2];
    }
    const bool taught = sum[1] != 0.0f;
    const float inv_teacher = taught ? 1.0f / sum[1] : 0.0f;

    if constexpr (MODE != kGradFromStats) {
        // τ²·p·(log p − log q), the differences of logits scaled by τ alone: neither overflows
        // where the loss does not
        const float logs = tau * (logf(sum[0]) - (taught ? logf(sum[1]) : 0.0f));
        float kl[1] = {0.0f};
#pragma unroll
        for (int j = 0; j < kTops; ++j) {
            const float p = pe[j] * inv_teacher;
            if (p != 0.0f)
                kl[0] += p * (tau * (((t[j] - t_max) - (zk[j] - z_max)) + logs));
        }
        block.sum(kl);
        if (tid == 0) {
            float loss = (1.0f - lam) * kl[0];
            if constexpr (kHard)
                if (label >= 0) loss += lam * (logf(sum[2]) - (z_label - z_max));
            a.loss[row] = loss;
            if (a.stats) {
                a.stats[4 * row] = z_max;
                a.stats[4 * row + 1] = inv_sum;
                a.stats[4 * row + 2] = inv_hard;
                a.stats[4 * row + 3] = 0.0f;
            }
        }
    }
    if constexpr (MODE != kLoss) {
        const float g = a.grad_loss ? a.grad_loss[row] : float(a.grad_value);
        const float soft = taught ? (1.0f - lam) * tau : 0.0f;
        const float f_soft = g * soft * inv_sum, f_hard = label >= 0 ? g * lam * inv_hard : 0.0f;
        auto softmax = [&](float x) {
            float d = f_soft * exp2_hw((x - z_max) * c);
            if constexpr (kHard) d = fmaf(f_hard, exp2_hw((x - z_max) * kLog2e), d);
            return d;
        };
        Raw *out = static_cast<Raw *>(a.grad) + row * a.ld_grad;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int at = (r * NT + tid) * E;
            float f[E];
            zr[r].get(f);
#pragma unroll
            for (int i = 0; i < E; ++i) f[i] = softmax(f[i]);
            zr[r].set(f);
            zr[r].store(out + at, vocab - at);
        }
        for (int at = kHeld + tid * E; at < vocab; at += NT * E) {
            C x;
            float f[E];
            x.load(z + at, vocab - at);
            x.get(f);
#pragma unroll
            for (int i = 0; i < E; ++i) f[i] = softmax(f[i]);
            x.set(f);
            x.store(out + at, vocab - at);
        }
        // what the entries take away, then their elements once more
#pragma unroll
        for (int j = 0; j < kTops; ++j) {
            const int e = j * NT + tid;
            if (e < k) {
                entry_at[e] = index[j];
                entry_amount[e] = soft * (pe[j] * inv_teacher);
            }
        }
        if (tid == 0) {
            entry_at[k] = static_cast<int>(label);
            entry_amount[k] = label >= 0 ? lam : 0.0f;
        }
        __syncthreads();
        const int entries = k + (kHard ? 1 : 0);
        auto overwrite = [&](int at, float x) {
            float amount = 0.0f;
#pragma unroll 8
            for (int e = 0; e < entries; ++e) amount += entry_at[e] == at ? entry_amount[e] : 0.0f;
            const float d = softmax(x) - g * amount;
            if constexpr (E == 8)
                out[at] = f32_to_bf16_bits(d);
            else
                out[at] = d;
        };
#pragma unroll
        for (int j = 0; j < kTops; ++j)
            if (index[j] >= 0) overwrite(index[j], zk[j]);
        if constexpr (kHard)
            if (tid == NT - 1 && label >= 0) overwrite(static_cast<int>(label), z_label);
    }
}

int check(const Args *a) {
    if (!a) return invalid("distill: args is null");
    if (a->rows < 0 || a->rows > INT32_MAX || a->vocab < 1 || a->vocab > (1 << 30))
        return invalid("distill: rows must not be negative and vocab must be 1 to 2^30");
    if (a->k < 1 || a->k > kMaxTop) return invalid("distill: k must be 1 to 1024");
    if ((a->logits_dtype != MUON_TRAIN_F32 && a->logits_dtype != MUON_TRAIN_BF16) ||
        (a->teacher_dtype != MUON_TRAIN_F32 && a->teacher_dtype != MUON_TRAIN_BF16))
        return invalid("distill: dtypes must be float32 or bfloat16");
    if (a->index_bytes != 4 && a->index_bytes != 8)
        return invalid("distill: indices must be int32 or int64");
    if (!(a->temperature > 0.0) || !(a->temperature < 1e30))
        return invalid("distill: temperature must be positive");
    if (!(a->label_weight >= 0.0 && a->label_weight <= 1.0))
        return invalid("distill: label_weight must be 0 to 1");
    if (a->rows == 0) return MUON_POLAR_OK;
    if (!a->logits || !a->teacher_logits || !a->teacher_indices) return invalid("distill: null pointer");
    if (a->ld_logits < a->vocab) return invalid("distill: rows of logits must not overlap");
    if (a->grad) {
        if (a->ld_grad < a->vocab) return invalid("distill: rows of grad must not overlap");
        const int64_t size = a->logits_dtype == MUON_TRAIN_BF16 ? 2 : 4;
        const char *z = static_cast<const char *>(a->logits);
        const char *g = static_cast<const char *>(a->grad);
        const char *z_end = z + ((a->rows - 1) * a->ld_logits + a->vocab) * size;
        const char *g_end = g + ((a->rows - 1) * a->ld_grad + a->vocab) * size;
        if (z < g_end && g < z_end && (z != g || a->ld_logits != a->ld_grad))
            return invalid("distill: grad must be logits itself or not overlap it");
    }
    return MUON_POLAR_OK;
}

// Threads and register chunks by the row's bytes: the fewest chunks that hold it, 256
// threads up to 32 KiB and 1024 beyond.
template <class T, int MODE, bool kHard>
void launch(const Args &a, hipStream_t stream) {
    const int64_t bytes = a.vocab * int64_t(sizeof(typename T::Raw));
    const dim3 grid(static_cast<uint32_t>(a.rows));
    auto go = [&](auto nt, auto r) {
        distill_kernel<T, decltype(nt)::value, decltype(r)::value, MODE, kHard>
            <<<grid, decltype(nt)::value, 0, stream>>>(a);
    };
    using std::integral_constant;
    if (bytes <= 256 * 2 * 16) go(integral_constant<int, 256>{}, integral_constant<int, 2>{});
    else if (bytes <= 256 * 8 * 16) go(integral_constant<int, 256>{}, integral_constant<int, 8>{});
    else if (bytes <= 1024 * 4 * 16) go(integral_constant<int, 1024>{}, integral_constant<int, 4>{});
    else if (bytes <= 1024 * 8 * 16) go(integral_constant<int, 1024>{}, integral_constant<int, 8>{});
    else go(integral_constant<int, 1024>{}, integral_constant<int, 16>{});
}
template <int MODE>
void launch(const Args &a, hipStream_t stream) {
    const bool hard = a.labels != nullptr;
    if (a.logits_dtype == MUON_TRAIN_BF16)
        hard ? launch<Bf16, MODE, true>(a, stream) : launch<Bf16, MODE, false>(a, stream);
    else
        hard ? launch<F32, MODE, true>(a, stream) : launch<F32, MODE, false>(a, stream);
}

}  // namespace

}  // namespace muon_train

using namespace muon_train;

extern "C" int muon_train_distill_forward(const muon_train_distill_args *args, hipStream_t stream) {
    const int st = check(args);
    if (st != MUON_POLAR_OK || args->rows == 0) return st;
    if (!args->loss) return invalid("distill: null output");
    if (args->grad)
        launch<kLossAndGrad>(*args, stream);
    else
        launch<kLoss>(*args, stream);
    return launched("distill_forward");
}

extern "C" int muon_train_distill_backward(const muon_train_distill_args *args, hipStream_t stream) {
    const int st = check(args);
    if (st != MUON_POLAR_OK || args->rows == 0) return st;
    if (!args->grad || !args->stats) return invalid("distill: null output");
    launch<kGradFromStats>(*args, stream);
    return launched("distill_backward");
}
