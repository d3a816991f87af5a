// train_distill.hip — the loss against a teacher's top logits, its gradient, and both in
// one pass (include/muon_train.h; the formulas are there).
//
// Loss and gradient in one pass: one workgroup a row, which it loads into registers whole
// (up to 256 KiB: 1024 threads with 16 pieces of 16 bytes each); maximum and sum of
// exponentials are taken from there, and the gradient is written from there: the logits
// cross memory once in and once out, which is what bounds the pass.  Of a longer row the
// threads take the rest with a running maximum and sum, keep the next 128 KiB in LDS, and read
// what lies past that again for the gradient.
// Loss alone, and the gradient from a forward pass's stats, hold no row: it streams by.
//
// The gradient is the softmax everywhere but at the teacher's indices and the label.  All
// of the row is written as softmax first; then, past a barrier, each entry overwrites its
// element with the softmax less the sum of all amounts that lie on that index (the same
// bits from every entry of an index that occurs twice).
#include "train_common.hpp"

#include <cfloat>

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
        if (valid < kElems) {
#pragma unroll
            for (int i = 0; i < kElems; ++i)
                if (i < valid) {
                    if constexpr (kElems == 8)
                        p[i] = static_cast<uint16_t>(v[i / 2] >> (16 * (i & 1)));
                    else
                        p[i] = __uint_as_float(v[i]);
                }
        } else {
            __builtin_memcpy(p, &v, 16);
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

// The teacher's entries of one row, kTops in each of NT threads, and the label.
template <int NT, bool kHard>
struct Targets {
    static constexpr int kTops = kMaxTop / NT;
    float t[kTops], zk[kTops], pe[kTops];  // logits of teacher and student, exp of the former
    int index[kTops];
    int label = -1;
    float z_label = 0.0f;

    // Loads; returns the largest of the thread's teacher logits.
    template <class Raw>
    __device__ __forceinline__ float load(const Args &a, int64_t row, const Raw *z) {
        float top = kNegInf;
#pragma unroll
        for (int j = 0; j < kTops; ++j) {
            const int e = j * NT + threadIdx.x;
            index[j] = -1;
            t[j] = kNegInf;
            zk[j] = 0.0f;
            if (e < a.k) {
                const int64_t i = load_index(a, row * a.k + e);
                if (i >= 0 && i < a.vocab) {
                    index[j] = static_cast<int>(i);
                    t[j] = load_any(a.teacher_logits, row * a.k + e, a.teacher_dtype);
                    zk[j] = to_f32(z[i]);
                }
                top = fmaxf(top, t[j]);
            }
        }
        if constexpr (kHard) {
            const int64_t y = a.labels[row];
            label = y >= 0 && y < a.vocab ? static_cast<int>(y) : -1;
            if (label >= 0) z_label = to_f32(z[label]);
        }
        return top;
    }
    // The thread's share of Σ exp((t − t_max) / τ); c = log2(e) / τ.
    __device__ __forceinline__ float weigh(float t_max, float c) {
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < kTops; ++j) {
            pe[j] = index[j] >= 0 && t_max > kNegInf ? exp2_hw((t[j] - t_max) * c) : 0.0f;
            if (index[j] >= 0 && t[j] != t[j]) pe[j] = t[j];
            sum += pe[j];
        }
        return sum;
    }
    // The thread's share of τ²·Σ p·(log p − log q): the differences of logits are scaled by
    // τ alone, so that neither overflows where the loss does not.
    __device__ __forceinline__ float divergence(float tau, float t_max, float t_sum, float z_max,
                                                float z_sum) const {
        const bool taught = t_sum != 0.0f;
        const float inv = taught ? 1.0f / t_sum : 0.0f;
        const float logs = tau * (logf(z_sum) - (taught ? logf(t_sum) : 0.0f));
        float kl = 0.0f;
#pragma unroll
        for (int j = 0; j < kTops; ++j) {
            const float p = pe[j] * inv;
            if (p != 0.0f) kl += p * (tau * (((t[j] - t_max) - (zk[j] - z_max)) + logs));
        }
        return kl;
    }
};

// One chunk's arithmetic at a time.
__device__ __forceinline__ void chunk_done() { __builtin_amdgcn_sched_barrier(0); }
// Makes the compiler forget what it knows of held chunks: it would keep what one pass over
// them works out (fp32 values, exponentials: twice the registers of bf16 chunks) for the
// next, and spill.
template <int R, class C>
__device__ __forceinline__ void forget(C *held) {
#pragma unroll
    for (int r = 0; r < R; ++r) asm volatile("" : "+v"(held[r].v));
}

// Largest logit and sums of exponentials of a part of a row, taken piece by piece: the sums
// are relative to the largest so far (to 0 while that is −inf, so that −inf adds nothing
// and a NaN stays one).
template <bool kHard>
struct Running {
    float top = kNegInf, sum = 0.0f, hard = 0.0f;
    __device__ __forceinline__ static float against(float top) { return top == kNegInf ? 0.0f : top; }
    __device__ __forceinline__ void rebase(float m, float c) {
        const float d = top - against(m);
        sum *= exp2_hw(d * c);
        if constexpr (kHard) hard *= exp2_hw(d * kLog2e);
        top = m;
    }
    template <int N>
    __device__ __forceinline__ void add(const float (&f)[N], float c) {
        const float ref = against(top);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            sum += exp2_hw((f[i] - ref) * c);
            if constexpr (kHard) hard += exp2_hw((f[i] - ref) * kLog2e);
        }
    }
};

// Takes kAhead chunks of a thread into its running sums.  Every kernel takes a row's chunks
// in the same groups and order, so the loss has the same bits with and without a gradient.
constexpr int kAhead = 4;
template <class C, bool kHard>
__device__ __forceinline__ void take(Running<kHard> &run, C *x, float c) {
    float m = run.top;
#pragma unroll
    for (int r = 0; r < kAhead; ++r) {
        float f[C::kElems];
        x[r].get(f);
#pragma unroll
        for (int i = 0; i < C::kElems; ++i) m = fmaxf(m, f[i]);
        chunk_done();
    }
    forget<kAhead>(x);
    run.rebase(m, c);
#pragma unroll
    for (int r = 0; r < kAhead; ++r) {
        float f[C::kElems];
        x[r].get(f);
        run.add(f, c);
        chunk_done();
    }
}

// 1 / a sum of exponentials; of a row that is all −inf, whose softmax is 0 / 0, NaN.
__device__ __forceinline__ float inverse_sum(float sum) {
    return sum == 0.0f ? __builtin_nanf("") : 1.0f / sum;
}
// What the gradient needs of a row: softmax(z / τ) times f_soft plus softmax(z) times f_hard,
// 0 for a term that the row does not have.  Logits that are NaN, +inf or all −inf make that
// factor NaN where the term counts; the exponentials themselves are held to [0, 1], with 0 for
// NaN (a modifier of the instruction: no time), so that where it does not they add nothing.
template <bool kHard>
struct Slope {
    float z_max, c, f_soft, f_hard;
    __device__ __forceinline__ static float within(float x) { return __builtin_amdgcn_fmed3f(x, 0.0f, 1.0f); }
    __device__ __forceinline__ float operator()(float x) const {
        float d = f_soft * within(exp2_hw((x - z_max) * c));
        if constexpr (kHard) d = fmaf(f_hard, within(exp2_hw((x - z_max) * kLog2e)), d);
        return d;
    }
};

// Entries of a row in LDS, (index, bits of the amount), read sixteen at a time by whoever looks
// for an element's: one by one, each read waited for, an entry took 100 clocks of every
// workgroup (4096 x 65536, 64 entries 225 us, 1024 entries 1008; so 213 and 472).
using u32x2 = uint32_t __attribute__((ext_vector_type(2)));
constexpr int kEntryGroup = 16;
struct Entries {
    u32x2 of[kMaxTop + 2 * kEntryGroup];
};
// Past a barrier behind the whole row's softmax: the elements of the entries in [lo, hi).
template <class T, int NT, bool kHard>
__device__ __forceinline__ void overwrite_entries(const Args &a, const Targets<NT, kHard> &y,
                                                  const Slope<kHard> &slope, float g, float soft,
                                                  float inv_teacher, typename T::Raw *out, int lo,
                                                  int hi, Entries &entry) {
    const int k = static_cast<int>(a.k), tid = threadIdx.x, entries = k + (kHard ? 1 : 0);
#pragma unroll
    for (int j = 0; j < y.kTops; ++j) {
        const int e = j * NT + tid;
        if (e < k) entry.of[e] = u32x2{static_cast<uint32_t>(y.index[j]), __float_as_uint(soft * (y.pe[j] * inv_teacher))};
    }
    if (kHard && tid == 0)
        entry.of[k] = u32x2{static_cast<uint32_t>(y.label), __float_as_uint(y.label >= 0 ? float(a.label_weight) : 0.0f)};
    if (tid < kEntryGroup) entry.of[entries + tid] = u32x2{~0u, 0u};  // to a whole group
    __syncthreads();
    auto overwrite = [&](int at, float x) {
        float amount = 0.0f;
        for (int e = 0; e < entries; e += kEntryGroup) {
            u32x4 two[kEntryGroup / 2];
#pragma unroll
            for (int i = 0; i < kEntryGroup / 2; ++i)
                two[i] = *reinterpret_cast<const u32x4 *>(&entry.of[e + 2 * i]);
#pragma unroll
            for (int i = 0; i < kEntryGroup; ++i)
                amount += two[i / 2][2 * (i % 2)] == static_cast<uint32_t>(at)
                              ? __uint_as_float(two[i / 2][2 * (i % 2) + 1]) : 0.0f;
        }
        const float d = slope(x) - g * amount;
        if constexpr (sizeof(typename T::Raw) == 2)
            out[at] = f32_to_bf16_bits(d);
        else
            out[at] = d;
    };
#pragma unroll
    for (int j = 0; j < y.kTops; ++j)
        if (y.index[j] >= lo && y.index[j] < hi) overwrite(y.index[j], y.zk[j]);
    if (kHard && tid == NT - 1 && y.label >= lo && y.label < hi) overwrite(y.label, y.z_label);
}

template <bool kHard>
__device__ __forceinline__ void write_row(const Args &a, int64_t row, float kl, float z_max,
                                          float z_sum, float z_hard, float t_sum, int label,
                                          float z_label) {
    const float lam = kHard ? float(a.label_weight) : 0.0f;
    float loss = (1.0f - lam) * kl;
    if (kHard && label >= 0) loss += lam * (logf(z_hard) - (z_label - z_max));
    a.loss[row] = loss;
    if (a.stats) {
        a.stats[4 * row] = z_max;
        a.stats[4 * row + 1] = inverse_sum(z_sum);
        a.stats[4 * row + 2] = kHard ? inverse_sum(z_hard) : 0.0f;
        a.stats[4 * row + 3] = t_sum != 0.0f ? 1.0f / t_sum : 0.0f;
    }
}

// Calls f(r, offset of the stripe, offset in it, elements of the chunk inside the row) for
// the R stripes of NT chunks from `at` on; of a stripe that lies inside whole, without a
// mask.
template <int NT, int R, int E, class F>
__device__ __forceinline__ void over_chunks(int at, int end, F &&f) {
    const uint32_t own = threadIdx.x * E;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int base = at + r * NT * E;
        if (base + NT * E <= end)
            f(r, base, own, E);
        else
            f(r, base, own, end - (base + static_cast<int>(own)));
    }
}
// Loss alone: the row streams by, kAhead chunks of each thread in flight.
template <class T, int NT, bool kHard>
__global__ __launch_bounds__(NT) void distill_loss_kernel(Args a) {
    using C = Chunk<T>;
    constexpr int E = C::kElems, NW = NT / 64, kStep = kAhead * NT * E;
    __shared__ float red[2][NW * 3];
    BlockSum<NW, 3> block(red);
    const int64_t row = blockIdx.x;
    const int vocab = static_cast<int>(a.vocab);
    const auto *z = static_cast<const typename T::Raw *>(a.logits) + row * a.ld_logits;
    const float tau = float(a.temperature), c = kLog2e / tau;

    C next[kAhead];
    auto fetch = [&](int at) {
        over_chunks<NT, kAhead, E>(at, vocab, [&](int r, int base, uint32_t own, int valid) {
            next[r].load((z + base) + own, valid);
        });
    };
    fetch(0);
    Targets<NT, kHard> y;
    float top[2];
    top[1] = y.load(a, row, z);
    Running<kHard> run;
    for (int at = 0; at < vocab; at += kStep) {
        C now[kAhead];
#pragma unroll
        for (int r = 0; r < kAhead; ++r) now[r] = next[r];
        if (at + kStep < vocab) fetch(at + kStep);
        take(run, now, c);
    }
    top[0] = run.top;
    block.max(top);
    run.rebase(top[0], c);
    float sum[3] = {run.sum, y.weigh(top[1], c), run.hard};
    block.sum(sum);
    const float kl = block.sum(y.divergence(tau, top[1], sum[1], top[0], sum[0]));
    if (threadIdx.x == 0)
        write_row<kHard>(a, row, kl, top[0], sum[0], sum[2], sum[1], y.label, y.z_label);
}

// Loss and gradient: NT threads hold R chunks each of the row in registers, 16 waves a
// compute unit whatever NT is, and L chunks more each in LDS: rows
// up to 384 KiB are read once (4096 rows of 160000 in bf16, with labels 656 -> 642 us, without 556
// -> 549; 2048 rows of 98304 in fp32 344 -> 322), longer ones twice past that.
template <class T, int NT, int R, int L, bool kHard>
__global__ __launch_bounds__(NT, 4) void distill_both_kernel(Args a) {
    using Raw = typename T::Raw;
    using C = Chunk<T>;
    constexpr int E = C::kElems, NW = NT / 64, kHeld = R * NT * E;
    constexpr int kKept = kHeld + L * NT * E;
    static_assert(L % kAhead == 0, "whole groups");
    __shared__ u32x4 kept[L > 0 ? L * NT : 1];
    __shared__ float red[2][NW * 3];
    __shared__ __attribute__((aligned(16))) Entries entry;
    BlockSum<NW, 3> block(red);
    const int64_t row = blockIdx.x;
    const int vocab = static_cast<int>(a.vocab);
    const Raw *z = static_cast<const Raw *>(a.logits) + row * a.ld_logits;
    const float tau = float(a.temperature), lam = kHard ? float(a.label_weight) : 0.0f;
    const float c = kLog2e / tau;  // exponents in powers of two

    C held[R];
    over_chunks<NT, R, E>(0, vocab, [&](int r, int base, uint32_t own, int valid) {
        held[r].load((z + base) + own, valid);
    });
    Targets<NT, kHard> y;
    float top[2];
    top[1] = y.load(a, row, z);
    Running<kHard> run;
    static_assert(R % kAhead == 0, "whole groups");
#pragma unroll
    for (int r = 0; r < R; r += kAhead) take(run, held + r, c);
    for (int at = kHeld; at < vocab; at += kAhead * NT * E) {  // what registers do not hold
        C x[kAhead];
        over_chunks<NT, kAhead, E>(at, vocab, [&](int r, int base, uint32_t own, int valid) {
            x[r].load((z + base) + own, valid);
        });
        if (L > 0 && at < kKept)
#pragma unroll
            for (int r = 0; r < kAhead; ++r) kept[(at - kHeld) / E + r * NT + threadIdx.x] = x[r].v;
        take(run, x, c);
    }
    top[0] = run.top;
    block.max(top);
    run.rebase(top[0], c);
    float sum[3] = {run.sum, y.weigh(top[1], c), run.hard};
    forget<R>(held);
    block.sum(sum);
    const float kl = block.sum(y.divergence(tau, top[1], sum[1], top[0], sum[0]));
    if (threadIdx.x == 0)
        write_row<kHard>(a, row, kl, top[0], sum[0], sum[2], sum[1], y.label, y.z_label);

    const bool taught = sum[1] != 0.0f;
    const float g = a.grad_loss ? a.grad_loss[row] : float(a.grad_value);
    const float soft = taught ? (1.0f - lam) * tau : 0.0f;
    const Slope<kHard> slope{top[0], c, taught ? g * soft * inverse_sum(sum[0]) : 0.0f,
                             kHard && y.label >= 0 ? g * lam * inverse_sum(sum[2]) : 0.0f};
    Raw *out = static_cast<Raw *>(a.grad) + row * a.ld_grad;
    over_chunks<NT, R, E>(0, vocab, [&](int r, int base, uint32_t own, int valid) {
        float f[E];
        held[r].get(f);
#pragma unroll
        for (int i = 0; i < E; ++i) f[i] = slope(f[i]);
        C x;
        x.set(f);
        x.store((out + base) + own, valid);
        chunk_done();
    });
    for (int at = kHeld + threadIdx.x * E; at < vocab; at += NT * E) {
        C x;
        float f[E];
        if (L > 0 && at < kKept)
            x.v = kept[(at - kHeld) / E];
        else
            x.load(z + at, vocab - at);
        x.get(f);
#pragma unroll
        for (int i = 0; i < E; ++i) f[i] = slope(f[i]);
        x.set(f);
        x.store(out + at, vocab - at);
    }
    overwrite_entries<T, NT, kHard>(a, y, slope, g, soft, taught ? 1.0f / sum[1] : 0.0f, out, 0,
                                    vocab, entry);
}

// Gradient from a forward pass's stats: no sums over the row, which streams by; blockIdx.y
// takes the columns [y·width, (y + 1)·width).
constexpr int kGradThreads = 256;
template <class T, bool kHard>
__global__ __launch_bounds__(kGradThreads) void distill_grad_kernel(Args a, int width) {
    using Raw = typename T::Raw;
    using C = Chunk<T>;
    constexpr int NT = kGradThreads, E = C::kElems, NW = NT / 64, kStep = kAhead * NT * E;
    __shared__ float red[2][NW];
    __shared__ __attribute__((aligned(16))) Entries entry;
    BlockSum<NW, 1> block(red);
    const int64_t row = blockIdx.x;
    const int lo = blockIdx.y * width;
    const int hi = width < a.vocab - lo ? lo + width : static_cast<int>(a.vocab);
    const Raw *z = static_cast<const Raw *>(a.logits) + row * a.ld_logits;
    Raw *out = static_cast<Raw *>(a.grad) + row * a.ld_grad;
    const float tau = float(a.temperature), lam = kHard ? float(a.label_weight) : 0.0f;
    const float c = kLog2e / tau;

    C next[kAhead];
    auto fetch = [&](int at) {
        over_chunks<NT, kAhead, E>(at, hi, [&](int r, int base, uint32_t own, int valid) {
            next[r].load((z + base) + own, valid);
        });
    };
    fetch(lo);
    Targets<NT, kHard> y;
    float t_max[1] = {y.load(a, row, z)};
    block.max(t_max);
    y.weigh(t_max[0], c);
    const float inv_teacher = a.stats[4 * row + 3];
    const bool taught = inv_teacher != 0.0f;
    const float g = a.grad_loss ? a.grad_loss[row] : float(a.grad_value);
    const float soft = taught ? (1.0f - lam) * tau : 0.0f;
    const Slope<kHard> slope{a.stats[4 * row], c, taught ? g * soft * a.stats[4 * row + 1] : 0.0f,
                             kHard && y.label >= 0 ? g * lam * a.stats[4 * row + 2] : 0.0f};
    for (int at = lo; at < hi; at += kStep) {
        C now[kAhead];
#pragma unroll
        for (int r = 0; r < kAhead; ++r) now[r] = next[r];
        if (at + kStep < hi) fetch(at + kStep);
        over_chunks<NT, kAhead, E>(at, hi, [&](int r, int base, uint32_t own, int valid) {
            float f[E];
            now[r].get(f);
#pragma unroll
            for (int i = 0; i < E; ++i) f[i] = slope(f[i]);
            now[r].set(f);
            now[r].store((out + base) + own, valid);
            chunk_done();
        });
    }
    overwrite_entries<T, NT, kHard>(a, y, slope, g, soft, inv_teacher, out, lo, hi,
                                    entry);
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
    // log2(e) / temperature has to be finite in fp32
    if (!(a->temperature >= double(FLT_MIN)) || !(a->temperature < 1e30))
        return invalid("distill: temperature must be a positive normal fp32 number below 1e30");
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

using std::integral_constant;

// Threads of a row: rows that fill the card take as few as hold them with up to 16 chunks
// each, so that several workgroups share a compute unit and one's loads and stores run
// beside another's sums; fewer rows take 1024 threads, and the row arrives sooner.
int row_threads(const Args &a, int64_t chunks, int cus) {
    const bool many = a.rows >= 2 * int64_t(cus);
    if (chunks <= 256 * 4 || (many && chunks <= 256 * 16)) return 256;
    return many && chunks <= 512 * 16 ? 512 : 1024;
}
template <class T>
int64_t row_chunks(const Args &a) {
    return (a.vocab * int64_t(sizeof(typename T::Raw)) + 15) / 16;
}

template <class T, bool kHard>
void launch_loss(const Args &a, int cus, Launches &launch) {
    const dim3 grid(static_cast<uint32_t>(a.rows));
    const int nt = row_threads(a, row_chunks<T>(a), cus);
    if (nt == 256) launch(distill_loss_kernel<T, 256, kHard>, grid, nt, a);
    else if (nt == 512) launch(distill_loss_kernel<T, 512, kHard>, grid, nt, a);
    else launch(distill_loss_kernel<T, 1024, kHard>, grid, nt, a);
}
template <class T, bool kHard>
void launch_both(const Args &a, int cus, Launches &launch) {
    const int64_t chunks = row_chunks<T>(a);
    const int nt = row_threads(a, chunks, cus);
    const dim3 grid(static_cast<uint32_t>(a.rows));
    auto go = [&](auto threads, auto r, auto l) {
        launch(distill_both_kernel<T, decltype(threads)::value, decltype(r)::value, decltype(l)::value, kHard>,
               grid, nt, a);
    };
    constexpr integral_constant<int, 0> none{};
    if (nt == 256 && chunks <= 256 * 4) go(integral_constant<int, 256>{}, integral_constant<int, 4>{}, none);
    else if (nt == 256 && chunks <= 256 * 8) go(integral_constant<int, 256>{}, integral_constant<int, 8>{}, none);
    else if (nt == 256) go(integral_constant<int, 256>{}, integral_constant<int, 16>{}, none);
    else if (nt == 512) go(integral_constant<int, 512>{}, integral_constant<int, 16>{}, none);
    else if (chunks <= 1024 * 8) go(integral_constant<int, 1024>{}, integral_constant<int, 8>{}, none);
    else if (chunks <= 1024 * 16) go(integral_constant<int, 1024>{}, integral_constant<int, 16>{}, none);
    else go(integral_constant<int, 1024>{}, integral_constant<int, 16>{}, integral_constant<int, 8>{});
}
// Gradient alone: rows are cut where there are too few to fill the card, into parts of 16
// KiB at least.
template <class T, bool kHard>
void launch_grad(const Args &a, int cus, Launches &launch) {
    const int64_t least = 16384 / int64_t(sizeof(typename T::Raw));
    int64_t parts = (8 * int64_t(cus) + a.rows - 1) / a.rows;
    const int64_t most = (a.vocab + least - 1) / least;
    parts = parts < most ? parts : most;
    int64_t width = (a.vocab + parts - 1) / parts;
    width = (width + 7) / 8 * 8;  // parts begin where 16-byte chunks do
    const dim3 grid(static_cast<uint32_t>(a.rows), static_cast<uint32_t>((a.vocab + width - 1) / width));
    launch(distill_grad_kernel<T, kHard>, grid, kGradThreads, a, static_cast<int>(width));
}
#define MUON_TRAIN_LAUNCH(which)                                                              \
    do {                                                                                      \
        const bool hard = a.labels != nullptr;                                                \
        if (a.logits_dtype == MUON_TRAIN_BF16)                                                \
            hard ? which<Bf16, true>(a, cus, launch) : which<Bf16, false>(a, cus, launch);    \
        else                                                                                  \
            hard ? which<F32, true>(a, cus, launch) : which<F32, false>(a, cus, launch);      \
    } while (0)

}  // namespace

}  // namespace muon_train

using namespace muon_train;

namespace muon_train {
namespace {

// Calls f with the arguments of up to kSlice rows after another: of one launch's threads (a row
// takes 1024 at most).  Slices of one size, so that all take the kernel of many rows.
template <class F>
void over_slices(const Args &args, F &&f) {
    constexpr int64_t kSlice = int64_t(1) << 21;
    static_assert(kSlice * 1024 <= kMaxThreads, "threads of a launch");
    const int64_t size = args.logits_dtype == MUON_TRAIN_BF16 ? 2 : 4;
    const int64_t teacher_size = args.teacher_dtype == MUON_TRAIN_BF16 ? 2 : 4;
    auto past = [](auto *p, int64_t bytes) {
        return p ? reinterpret_cast<decltype(p)>(reinterpret_cast<uintptr_t>(p) + static_cast<uintptr_t>(bytes)) : p;
    };
    const int64_t slices = (args.rows + kSlice - 1) / kSlice, each = (args.rows + slices - 1) / slices;
    for (int64_t row = 0; row < args.rows; row += each) {
        Args a = args;
        a.rows = args.rows - row < each ? args.rows - row : each;
        a.logits = past(args.logits, row * args.ld_logits * size);
        a.grad = past(args.grad, row * args.ld_grad * size);
        a.teacher_logits = past(args.teacher_logits, row * args.k * teacher_size);
        a.teacher_indices = past(args.teacher_indices, row * args.k * args.index_bytes);
        a.labels = past(args.labels, row * int64_t(sizeof(int64_t)));
        a.grad_loss = past(args.grad_loss, row * int64_t(sizeof(float)));
        a.loss = past(args.loss, row * int64_t(sizeof(float)));
        a.stats = past(args.stats, row * int64_t(4 * sizeof(float)));
        f(a);
    }
}

}  // namespace
}  // namespace muon_train

extern "C" int muon_train_distill_forward(const muon_train_distill_args *args, hipStream_t stream) {
    const int st = check(args);
    if (st != MUON_POLAR_OK || args->rows == 0) return st;
    if (!args->loss) return invalid("distill: null output");
    const int cus = compute_units();
    if (cus <= 0) return muon_polar::report(MUON_POLAR_ERR_HIP, "distill: no device");
    Launches launch{stream};
    over_slices(*args, [&](const Args &a) {
        if (a.grad)
            MUON_TRAIN_LAUNCH(launch_both);
        else
            MUON_TRAIN_LAUNCH(launch_loss);
    });
    return launch.result("distill_forward");
}

extern "C" int muon_train_distill_backward(const muon_train_distill_args *args, hipStream_t stream) {
    const int st = check(args);
    if (st != MUON_POLAR_OK || args->rows == 0) return st;
    if (!args->grad || !args->stats) return invalid("distill: null output");
    const int cus = compute_units();
    if (cus <= 0) return muon_polar::report(MUON_POLAR_ERR_HIP, "distill: no device");
    Launches launch{stream};
    over_slices(*args, [&](const Args &a) { MUON_TRAIN_LAUNCH(launch_grad); });
    return launch.result("distill_backward");
}
