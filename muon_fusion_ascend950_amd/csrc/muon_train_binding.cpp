// muon_train_binding.cpp — registers the operators of a training step around the Muon
// update (include/muon_train.h) as torch operators of the muon_ascend950 library.  No
// reference counterpart.
//
// Two layers: operators that launch kernels (norms_forward, distill_backward, ...; device
// kernels here, FakeTensor kernels in _loader.py), and the ones that users call
// (block_norms, distill_topk, ...), which check their arguments and carry the gradient.
// Checks and autograd are here and not in Python for the calls whose kernels take a few
// microseconds: forward and backward of 1001 x 2051 norms took 137 us of host time with
// both in Python, four times their kernels.
#include <ATen/ATen.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include <cfloat>

#include "muon_train.h"

namespace {

using OptTensor = std::optional<at::Tensor>;

int dtype_of(const at::Tensor &t, const char *what) {
    TORCH_CHECK(t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16, what,
                " must be float32 or bfloat16");
    return t.scalar_type() == at::kFloat ? MUON_TRAIN_F32 : MUON_TRAIN_BF16;
}

bool given(const OptTensor &t) { return t.has_value() && t->defined(); }

hipStream_t stream_of(const at::Tensor &t) {
    return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

// t [.., d] as rows: the tensor itself where its rows lie evenly apart and unbroken,
// otherwise a contiguous copy.
struct Rows {
    at::Tensor t;
    int64_t rows, ld;
};
Rows as_rows(const at::Tensor &t) {
    const int64_t d = t.size(-1), rows = d > 0 ? t.numel() / d : 0;
    if (t.is_contiguous()) return {t, rows, d};
    at::Tensor r = t.reshape({rows, d});
    if (d > 1 && r.stride(1) == 1 && r.stride(0) >= d) return {r, rows, r.stride(0)};
    return {r.contiguous(), rows, d};
}

at::Tensor none(const at::Tensor &like) { return at::empty({0}, like.options()); }

// ---------------------------------------------------------------------------- norms
struct Norms {
    muon_train_norms_args a{};
    Rows y, residual;
    at::Tensor post, pre, gate, scale;

    Norms(const at::Tensor &y_, const at::Tensor &residual_, const OptTensor &post_weight,
          const OptTensor &gate_, const OptTensor &scale_, double scale_value,
          const OptTensor &pre_weight, int64_t gate_kind, int64_t rows_per_sequence,
          bool post_norm, bool pre_norm, double eps) {
        TORCH_CHECK(y_.device().is_cuda() && residual_.device() == y_.device(),
                    "block_norms: y and residual must be on one ROCm (HIP) device");
        TORCH_CHECK(y_.dim() >= 1 && y_.sizes() == residual_.sizes(),
                    "block_norms: y and residual must have one shape");
        a.d = y_.size(-1);
        a.y_dtype = dtype_of(y_, "block_norms: y");
        a.residual_dtype = dtype_of(residual_, "block_norms: residual");
        y = as_rows(y_);
        residual = as_rows(residual_);
        a.rows = y.rows;
        a.ld_y = y.ld;
        a.ld_residual = residual.ld;
        a.y = y.t.data_ptr();
        a.residual = residual.t.data_ptr();
        auto vector = [&](const OptTensor &t, int64_t numel, const char *what) {
            TORCH_CHECK(t->device() == y_.device() && t->numel() == numel, "block_norms: ", what,
                        " has the wrong device or size");
            return t->contiguous();
        };
        if (given(post_weight)) {
            post = vector(post_weight, a.d, "post_weight");
            a.weight_dtype = dtype_of(post, "block_norms: post_weight");
            a.post_weight = post.data_ptr();
        }
        if (given(pre_weight)) {
            pre = vector(pre_weight, a.d, "pre_weight");
            a.weight_dtype = dtype_of(pre, "block_norms: pre_weight");
            a.pre_weight = pre.data_ptr();
            TORCH_CHECK(!post.defined() || post.scalar_type() == pre.scalar_type(),
                        "block_norms: post_weight and pre_weight must have one dtype");
        }
        a.gate_kind = static_cast<int>(gate_kind);
        // sequences of no tokens: no rows, whatever number of gate vectors
        const bool no_tokens = gate_kind == MUON_TRAIN_GATE_SEQUENCE && rows_per_sequence == 0 && a.rows == 0;
        a.rows_per_sequence = no_tokens ? 1 : rows_per_sequence;
        if (gate_kind != MUON_TRAIN_GATE_NONE) {
            TORCH_CHECK(given(gate_), "block_norms: gate is missing");
            TORCH_CHECK(gate_kind != MUON_TRAIN_GATE_SEQUENCE || a.rows_per_sequence > 0,
                        "block_norms: rows_per_sequence must be positive");
            const int64_t numel = gate_kind == MUON_TRAIN_GATE_CHANNEL ? a.d
                                  : no_tokens                          ? gate_->numel()
                                  : gate_kind == MUON_TRAIN_GATE_SEQUENCE
                                      ? a.rows / rows_per_sequence * a.d
                                  : gate_kind == MUON_TRAIN_GATE_TOKEN ? a.rows
                                                                       : a.rows * a.d;
            gate = vector(gate_, numel, "gate");
            a.gate_dtype = dtype_of(gate, "block_norms: gate");
            a.gate = gate.data_ptr();
        }
        a.scale_value = scale_value;
        if (given(scale_)) {
            a.scale_kind = scale_->numel() == 1 ? MUON_TRAIN_SCALE_SCALAR : MUON_TRAIN_SCALE_VECTOR;
            scale = vector(scale_, scale_->numel() == 1 ? 1 : a.d, "residual_scale");
            TORCH_CHECK(scale.scalar_type() == at::kFloat,
                        "block_norms: residual_scale must be float32");
            a.scale = scale.data_ptr<float>();
        }
        a.post_norm = post_norm;
        a.pre_norm = pre_norm;
        a.eps = eps;
    }
};

std::tuple<at::Tensor, at::Tensor, at::Tensor> NormsForward(
    const at::Tensor &y, const at::Tensor &residual, const OptTensor &post_weight,
    const OptTensor &gate, const OptTensor &scale, double scale_value, const OptTensor &pre_weight,
    int64_t gate_kind, int64_t rows_per_sequence, bool post_norm, bool pre_norm, double eps,
    bool save) {
    const c10::OptionalDeviceGuard device_guard(y.device());
    Norms n(y, residual, post_weight, gate, scale, scale_value, pre_weight, gate_kind,
            rows_per_sequence, post_norm, pre_norm, eps);
    at::Tensor out = at::empty(y.sizes(), residual.options());
    at::Tensor normed = pre_norm ? at::empty(y.sizes(), y.options()) : none(y);
    at::Tensor stats;
    if (save) stats = at::empty({n.a.rows, 2}, y.options().dtype(at::kFloat));
    n.a.residual_out = out.data_ptr();
    if (pre_norm) n.a.normed = normed.data_ptr();
    if (save) n.a.stats = stats.data_ptr<float>();
    const int st = muon_train_norms_forward(&n.a, stream_of(y));
    TORCH_CHECK(st == MUON_POLAR_OK, "block_norms: ", muon_polar_last_error());
    return {out, normed, stats};
}

// wanted: bits of the gradients wanted (1 post_weight, 2 gate, 4 scale, 8 pre_weight); y's
// and residual's are always formed.
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> NormsBackward(
    const at::Tensor &y, const at::Tensor &residual, const OptTensor &post_weight,
    const OptTensor &gate, const OptTensor &scale, double scale_value, const OptTensor &pre_weight,
    int64_t gate_kind, int64_t rows_per_sequence, bool post_norm, bool pre_norm, double eps,
    const at::Tensor &stats, const OptTensor &d_residual_out, const OptTensor &d_normed,
    int64_t wanted) {
    const c10::OptionalDeviceGuard device_guard(y.device());
    Norms n(y, residual, post_weight, gate, scale, scale_value, pre_weight, gate_kind,
            rows_per_sequence, post_norm, pre_norm, eps);
    TORCH_CHECK(stats.is_contiguous() && stats.scalar_type() == at::kFloat &&
                    stats.numel() == 2 * n.a.rows,
                "block_norms: stats of another forward pass");
    n.a.stats = stats.data_ptr<float>();
    at::Tensor dro, dno;
    if (given(d_residual_out)) {
        TORCH_CHECK(d_residual_out->sizes() == y.sizes() &&
                        d_residual_out->scalar_type() == residual.scalar_type(),
                    "block_norms: the gradient of residual_out has another shape or dtype");
        dro = d_residual_out->contiguous();
        n.a.d_residual_out = dro.data_ptr();
    }
    if (given(d_normed) && pre_norm) {
        TORCH_CHECK(d_normed->sizes() == y.sizes() && d_normed->scalar_type() == y.scalar_type(),
                    "block_norms: the gradient of normed has another shape or dtype");
        dno = d_normed->contiguous();
        n.a.d_normed = dno.data_ptr();
    }
    at::Tensor dy = at::empty(y.sizes(), y.options());
    at::Tensor dr = at::empty(y.sizes(), residual.options());
    auto grad = [&](const at::Tensor &t, int64_t bit) {
        return (wanted & bit) && t.defined() ? at::empty(t.sizes(), t.options()) : none(y);
    };
    at::Tensor d_post = grad(n.post, 1), d_gate = grad(n.gate, 2), d_scale = grad(n.scale, 4),
               d_pre = grad(n.pre, 8);
    if (n.a.rows == 0 && d_gate.numel() > 0) d_gate.zero_();  // of sequences without tokens
    n.a.d_y = dy.data_ptr();
    n.a.d_residual = dr.data_ptr();
    if ((wanted & 1) && n.post.defined()) n.a.d_post_weight = d_post.data_ptr();
    if ((wanted & 2) && n.gate.defined()) n.a.d_gate = d_gate.data_ptr();
    if ((wanted & 4) && n.scale.defined()) n.a.d_scale = d_scale.data_ptr<float>();
    if ((wanted & 8) && n.pre.defined()) n.a.d_pre_weight = d_pre.data_ptr();
    size_t bytes = 0;
    int st = muon_train_norms_workspace(&n.a, &bytes);
    TORCH_CHECK(st == MUON_POLAR_OK, "block_norms: ", muon_polar_last_error());
    at::Tensor workspace =
        at::empty({static_cast<int64_t>(bytes)}, y.options().dtype(at::kByte));
    st = muon_train_norms_backward(&n.a, workspace.data_ptr(), bytes, stream_of(y));
    TORCH_CHECK(st == MUON_POLAR_OK, "block_norms: ", muon_polar_last_error());
    return {dy, dr, d_post, d_gate, d_scale, d_pre};
}

// -------------------------------------------------------------------------- distill
struct Distill {
    muon_train_distill_args a{};
    Rows logits;
    at::Tensor teacher, indices, labels, grad_loss;

    Distill(const at::Tensor &logits_, const at::Tensor &teacher_, const at::Tensor &indices_,
            const OptTensor &labels_, double temperature, double label_weight) {
        TORCH_CHECK(logits_.device().is_cuda(), "distill_topk: logits must be a ROCm (HIP) device tensor");
        TORCH_CHECK(logits_.dim() >= 1 && teacher_.dim() == logits_.dim() &&
                        teacher_.sizes() == indices_.sizes(),
                    "distill_topk: logits [.., V], teacher_logits and teacher_indices [.., K]");
        for (int64_t i = 0; i + 1 < logits_.dim(); ++i)
            TORCH_CHECK(teacher_.size(i) == logits_.size(i),
                        "distill_topk: logits and teacher_logits must have the same rows");
        logits = as_rows(logits_);
        a.rows = logits.rows;
        a.vocab = logits_.size(-1);
        a.k = teacher_.size(-1);
        a.ld_logits = logits.ld;
        a.logits_dtype = dtype_of(logits_, "distill_topk: logits");
        a.logits = logits.t.data_ptr();
        auto on_device = [&](const at::Tensor &t, const char *what) {
            TORCH_CHECK(t.device() == logits_.device(), "distill_topk: ", what, " is on another device");
            return t.contiguous();
        };
        teacher = on_device(teacher_, "teacher_logits");
        a.teacher_dtype = dtype_of(teacher, "distill_topk: teacher_logits");
        a.teacher_logits = teacher.data_ptr();
        indices = on_device(indices_, "teacher_indices");
        TORCH_CHECK(indices.scalar_type() == at::kInt || indices.scalar_type() == at::kLong,
                    "distill_topk: teacher_indices must be int32 or int64");
        a.index_bytes = indices.scalar_type() == at::kInt ? 4 : 8;
        a.teacher_indices = indices.data_ptr();
        if (given(labels_)) {
            labels = on_device(*labels_, "labels");
            TORCH_CHECK(labels.scalar_type() == at::kLong && labels.numel() == a.rows,
                        "distill_topk: labels must be int64, one a row");
            a.labels = labels.data_ptr<int64_t>();
        }
        a.temperature = temperature;
        a.label_weight = label_weight;
    }
    void set_grad_loss(const OptTensor &t, double value) {
        a.grad_value = value;
        if (!given(t)) return;
        TORCH_CHECK(t->device() == logits.t.device() && t->scalar_type() == at::kFloat &&
                        t->numel() == a.rows,
                    "distill_topk: grad_loss must be float32, one a row");
        grad_loss = t->contiguous();
        a.grad_loss = grad_loss.data_ptr<float>();
    }
    at::Tensor per_row(const at::Tensor &like) const {
        return at::empty(like.sizes().slice(0, like.dim() - 1), like.options().dtype(at::kFloat));
    }
};

std::tuple<at::Tensor, at::Tensor> DistillForward(const at::Tensor &logits,
                                                  const at::Tensor &teacher_logits,
                                                  const at::Tensor &teacher_indices,
                                                  const OptTensor &labels, double temperature,
                                                  double label_weight, bool save) {
    const c10::OptionalDeviceGuard device_guard(logits.device());
    Distill d(logits, teacher_logits, teacher_indices, labels, temperature, label_weight);
    at::Tensor loss = d.per_row(logits);
    at::Tensor stats;
    if (save) stats = at::empty({d.a.rows, 4}, loss.options());
    d.a.loss = loss.data_ptr<float>();
    if (save) d.a.stats = stats.data_ptr<float>();
    const int st = muon_train_distill_forward(&d.a, stream_of(logits));
    TORCH_CHECK(st == MUON_POLAR_OK, "distill_topk: ", muon_polar_last_error());
    return {loss, stats};
}

at::Tensor DistillBackward(const at::Tensor &logits, const at::Tensor &teacher_logits,
                           const at::Tensor &teacher_indices, const OptTensor &labels,
                           double temperature, double label_weight, const at::Tensor &stats,
                           const at::Tensor &grad_loss) {
    const c10::OptionalDeviceGuard device_guard(logits.device());
    Distill d(logits, teacher_logits, teacher_indices, labels, temperature, label_weight);
    TORCH_CHECK(stats.is_contiguous() && stats.scalar_type() == at::kFloat &&
                    stats.numel() == 4 * d.a.rows,
                "distill_topk: stats of another forward pass");
    d.set_grad_loss(grad_loss, 0.0);
    at::Tensor grad = at::empty(logits.sizes(), logits.options());
    d.a.stats = stats.data_ptr<float>();
    d.a.grad = grad.data_ptr();
    d.a.ld_grad = d.a.vocab;
    const int st = muon_train_distill_backward(&d.a, stream_of(logits));
    TORCH_CHECK(st == MUON_POLAR_OK, "distill_topk: ", muon_polar_last_error());
    return grad;
}

// Loss, and the gradient into `grad`, which may be logits itself.
at::Tensor DistillWithGrad(const at::Tensor &logits, const at::Tensor &teacher_logits,
                           const at::Tensor &teacher_indices, const OptTensor &labels,
                           double temperature, double label_weight, const OptTensor &grad_loss,
                           double grad_value, const at::Tensor &grad) {
    const c10::OptionalDeviceGuard device_guard(logits.device());
    Distill d(logits, teacher_logits, teacher_indices, labels, temperature, label_weight);
    TORCH_CHECK(grad.sizes() == logits.sizes() && grad.scalar_type() == logits.scalar_type() &&
                    grad.device() == logits.device(),
                "distill_topk: out must have the shape, dtype and device of logits");
    d.set_grad_loss(grad_loss, grad_value);
    const Rows out = as_rows(grad);
    TORCH_CHECK(grad.numel() == 0 || out.t.data_ptr() == grad.data_ptr(),
                "distill_topk: the rows of out must lie evenly apart, each unbroken");
    at::Tensor loss = d.per_row(logits);
    d.a.loss = loss.data_ptr<float>();
    d.a.grad = out.t.data_ptr();
    d.a.ld_grad = out.ld;
    const int st = muon_train_distill_forward(&d.a, stream_of(logits));
    TORCH_CHECK(st == MUON_POLAR_OK, "distill_topk: ", muon_polar_last_error());
    return loss;
}

// ------------------------------------------------------------------------------ fp8
constexpr int64_t kBlock = 128;
int64_t blocks(int64_t n) { return (n + kBlock - 1) / kBlock; }

// A matrix held as e4m3 values [rows, blocks(cols) * 128] and scales
// [rows or blocks(rows), blocks(cols)].
struct Held {
    at::Tensor values, scales;
};
Held empty_held(const at::Tensor &like, int64_t rows, int64_t cols, int64_t block_rows) {
    const auto f32 = like.options().dtype(at::kFloat);
    Held h;
    h.values = at::empty({rows, blocks(cols) * kBlock}, like.options().dtype(at::kFloat8_e4m3fn));
    h.scales = block_rows == 1 ? at::empty({blocks(cols), rows}, f32).t()
                               : at::empty({blocks(rows), blocks(cols)}, f32);
    return h;
}

Held quantize(const at::Tensor &x, int64_t block_rows) {
    TORCH_CHECK(x.device().is_cuda() && x.dim() == 2, "fp8: a matrix on a ROCm (HIP) device is needed");
    const Rows r = as_rows(x);
    muon_train_fp8_quantize_args a{};
    a.rows = x.size(0);
    a.cols = x.size(1);
    a.ld_x = r.ld;
    a.x = r.t.data_ptr();
    a.x_dtype = dtype_of(x, "fp8: a matrix to quantise");
    a.block_rows = static_cast<int>(block_rows);
    Held h = empty_held(x, a.rows, a.cols, block_rows);
    a.values = h.values.data_ptr();
    a.scales = h.scales.data_ptr<float>();
    const int st = muon_train_fp8_quantize(&a, stream_of(x));
    TORCH_CHECK(st == MUON_POLAR_OK, "fp8: ", muon_polar_last_error());
    return h;
}

muon_train_fp8_operand operand(Held &h, const at::Tensor &like) {
    TORCH_CHECK(h.values.device() == like.device() && h.scales.device() == like.device(),
                "fp8: operands must be on one device");
    TORCH_CHECK(h.values.dim() == 2 && h.values.scalar_type() == at::kFloat8_e4m3fn &&
                    h.values.size(1) % kBlock == 0,
                "fp8: values must be float8_e4m3fn [rows, a multiple of 128]");
    const int64_t rows = h.values.size(0), kb = h.values.size(1) / kBlock;
    TORCH_CHECK(h.scales.dim() == 2 && h.scales.scalar_type() == at::kFloat &&
                    h.scales.size(1) == kb &&
                    (h.scales.size(0) == rows || h.scales.size(0) == blocks(rows)),
                "fp8: scales must be float32 [rows or ceil(rows / 128), cols / 128]");
    if (h.values.stride(1) != 1 || h.values.stride(0) % 16 != 0 ||
        h.values.stride(0) < h.values.size(1) ||
        reinterpret_cast<uintptr_t>(h.values.data_ptr()) % 16 != 0)
        h.values = h.values.clone(at::MemoryFormat::Contiguous);
    muon_train_fp8_operand o{};
    o.block_rows = h.scales.size(0) == rows ? 1 : static_cast<int>(kBlock);
    if (o.block_rows == 1 && rows > 1 && (h.scales.stride(0) != 1 || h.scales.stride(1) < rows))
        h.scales = h.scales.t().contiguous().t();
    o.values = h.values.data_ptr();
    o.scales = h.scales.data_ptr<float>();
    o.ld = h.values.stride(0);
    o.scale_row = o.block_rows == 1 ? 1 : h.scales.stride(0);
    o.scale_col = h.scales.stride(1);
    return o;
}

// With the workspace that the product asks for (few tiles of a long K).
void multiply(const muon_train_fp8_matmul_args &g, const at::Tensor &c) {
    size_t bytes = 0;
    int st = muon_train_fp8_matmul_workspace(&g, &bytes);
    at::Tensor workspace;
    if (st == MUON_POLAR_OK && bytes > 0)
        workspace = at::empty({static_cast<int64_t>(bytes)}, c.options().dtype(at::kByte));
    if (st == MUON_POLAR_OK)
        st = muon_train_fp8_matmul_in(&g, workspace.defined() ? workspace.data_ptr() : nullptr, bytes, stream_of(c));
    TORCH_CHECK(st == MUON_POLAR_OK, "fp8: ", muon_polar_last_error());
}

// c [m, n] = a · bᵀ
void matmul(Held a, Held b, at::Tensor &c) {
    muon_train_fp8_matmul_args g{};
    g.a = operand(a, c);
    g.b = operand(b, c);
    TORCH_CHECK(a.values.size(1) == b.values.size(1), "fp8: operands of different width");
    g.m = c.size(0);
    g.n = c.size(1);
    g.k = a.values.size(1);
    TORCH_CHECK(g.m == a.values.size(0) && g.n == b.values.size(0), "fp8: result of another shape");
    g.c = c.data_ptr();
    g.ldc = g.n;
    g.c_dtype = dtype_of(c, "fp8: the result");
    multiply(g, c);
}

std::tuple<at::Tensor, at::Tensor> QuantizeFp8(const at::Tensor &x, int64_t block_rows) {
    const c10::OptionalDeviceGuard device_guard(x.device());
    Held h = quantize(x, block_rows);
    return {h.values, h.scales};
}

at::Tensor Fp8Matmul(const at::Tensor &a, const at::Tensor &a_scales, const at::Tensor &b,
                     const at::Tensor &b_scales, at::ScalarType dtype) {
    const c10::OptionalDeviceGuard device_guard(a.device());
    at::Tensor c = at::empty({a.size(0), b.size(0)}, a.options().dtype(dtype));
    matmul({a, a_scales}, {b, b_scales}, c);
    return c;
}

// What a linear layer holds for itself, values and scales in one buffer: x (or a gradient)
// in rows, or the weight in 128 x 128 blocks, as they are or transposed.
struct Layout {
    int64_t rows, cols; // of the held matrix
    int64_t block_rows;
    bool turned; // a transposed weight: its scales lie in the weight's own order
    int64_t width() const { return blocks(cols) * kBlock; }
    int64_t scales_at() const { return (rows * width() + 255) / 256 * 256; }
    int64_t bytes() const {
        return scales_at() + 4 * blocks(cols) * (block_rows == 1 ? rows : blocks(rows));
    }
    at::Tensor empty(const at::Tensor &like) const {
        return at::empty({bytes()}, like.options().dtype(at::kByte));
    }
    uint8_t *values(const at::Tensor &t) const { return t.data_ptr<uint8_t>(); }
    float *scales(const at::Tensor &t) const {
        return reinterpret_cast<float *>(t.data_ptr<uint8_t>() + scales_at());
    }
    muon_train_fp8_operand operand(const at::Tensor &t) const {
        muon_train_fp8_operand o{};
        o.values = values(t);
        o.scales = scales(t);
        o.ld = width();
        o.block_rows = static_cast<int>(block_rows);
        o.scale_row = block_rows == 1 || turned ? 1 : blocks(cols);
        o.scale_col = block_rows == 1 ? rows : turned ? blocks(rows) : 1;
        return o;
    }
};

// x [.., cols] as rows, held and / or transposed and held (buffers may be undefined).
void hold_rows(const at::Tensor &x, const at::Tensor &plain, const at::Tensor &turned) {
    const Rows r = as_rows(x);
    const int64_t cols = x.size(-1);
    const Layout p{r.rows, cols, 1, false}, t{cols, r.rows, 1, false};
    muon_train_fp8_quantize_args a{};
    a.rows = r.rows;
    a.cols = cols;
    a.ld_x = r.ld;
    a.x = r.t.data_ptr();
    a.x_dtype = dtype_of(x, "fp8: a matrix to quantise");
    a.block_rows = 1;
    if (plain.defined()) a.values = p.values(plain), a.scales = p.scales(plain);
    if (turned.defined()) a.values_t = t.values(turned), a.scales_t = t.scales(turned);
    const int st = muon_train_fp8_quantize(&a, stream_of(x));
    TORCH_CHECK(st == MUON_POLAR_OK, "fp8: ", muon_polar_last_error());
}

void multiply(const muon_train_fp8_operand &a, int64_t m, const muon_train_fp8_operand &b, int64_t n,
              int64_t k, const at::Tensor &c) {
    muon_train_fp8_matmul_args g{};
    g.a = a;
    g.b = b;
    g.m = m;
    g.n = g.ldc = n;
    g.k = k;
    g.c = c.data_ptr();
    g.c_dtype = dtype_of(c, "fp8: the result");
    multiply(g, c);
}

int64_t rows_of(const at::Tensor &x) { return x.size(-1) > 0 ? x.numel() / x.size(-1) : 0; }
at::Tensor result_like(const at::Tensor &x, int64_t n) {
    auto sizes = x.sizes().vec();
    sizes.back() = n;
    return at::empty(sizes, x.options());
}

// y = x · wᵀ on a held weight.
at::Tensor Fp8Linear(const at::Tensor &x, const at::Tensor &values, const at::Tensor &scales) {
    const c10::OptionalDeviceGuard device_guard(x.device());
    const int64_t rows = rows_of(x), cols = x.size(-1);
    at::Tensor y = result_like(x, values.size(0));
    Held held{values, scales};
    const muon_train_fp8_operand w = operand(held, x);
    TORCH_CHECK(blocks(cols) * kBlock == values.size(1), "fp8: operands of different width");
    // Up to 16 rows can be quantised in the product's own kernel.  Each workgroup then does that
    // work, four rows and 4096 columns a pass of some 1 us; a launch of its own takes 3 us.
    // (12 rows of 4096 columns, three passes: 2.4 us over the product of held rows; 16, four
    // passes: 3.5; one row of 14336 2.7, five rows 7.6, 16 rows 17.7.)  The bits are the same.
    const int64_t passes = (rows + 3) / 4 * ((cols + 4095) / 4096);
    if (rows <= 16 && passes < 4 && w.block_rows == kBlock) {
        muon_train_fp8_decode_args a{};
        const Rows r = as_rows(x);
        a.w = w;
        a.m = rows;
        a.n = a.ldc = values.size(0);
        a.cols = cols;
        a.ld_x = r.ld;
        a.x = r.t.data_ptr();
        a.x_dtype = a.c_dtype = dtype_of(x, "fp8: a matrix to quantise");
        a.c = y.data_ptr();
        const int st = muon_train_fp8_decode(&a, stream_of(x));
        TORCH_CHECK(st == MUON_POLAR_OK, "fp8: ", muon_polar_last_error());
        return y;
    }
    const Layout q{rows, cols, 1, false};
    const at::Tensor xq = q.empty(x);
    hold_rows(x, xq, {});
    multiply(q.operand(xq), rows, w, values.size(0), q.width(), y);
    return y;
}

// y = x · weightᵀ, and what the backward pass needs: the transposed x along the tokens
// (save & 1, for the weight's gradient) and the transposed weight (save & 2, for x's).
std::tuple<at::Tensor, at::Tensor, at::Tensor> Fp8LinearForward(const at::Tensor &x,
                                                                const at::Tensor &weight,
                                                                int64_t save) {
    const c10::OptionalDeviceGuard device_guard(x.device());
    TORCH_CHECK(x.device().is_cuda() && weight.device() == x.device() && weight.dim() == 2 &&
                    x.dim() >= 1 && weight.size(1) == x.size(-1) && weight.numel() > 0,
                "fp8: x [.., K] and weight [N, K] on one ROCm (HIP) device");
    const int64_t rows = rows_of(x), k = weight.size(1), n = weight.size(0);
    const Layout q{rows, k, 1, false}, xt{k, rows, 1, false}, w{n, k, kBlock, false},
        wt{k, n, kBlock, true};
    at::Tensor y = result_like(x, n), xq = q.empty(x), wq = w.empty(x);
    at::Tensor saved_x = (save & 1) ? xt.empty(x) : at::Tensor();
    at::Tensor saved_w = (save & 2) ? wt.empty(x) : at::Tensor();
    hold_rows(x, xq, saved_x);
    const Rows r = as_rows(weight);
    muon_train_fp8_quantize_args a{};
    a.rows = n;
    a.cols = k;
    a.ld_x = r.ld;
    a.x = r.t.data_ptr();
    a.x_dtype = dtype_of(weight, "fp8: the weight");
    a.block_rows = static_cast<int>(kBlock);
    a.values = w.values(wq);
    muon_train_fp8_operand held = w.operand(wq);
    if (saved_w.defined()) {  // one set of scales serves both
        a.values_t = wt.values(saved_w);
        held.scales = wt.scales(saved_w);
    }
    a.scales = const_cast<float *>(held.scales);
    const int st = muon_train_fp8_quantize(&a, stream_of(x));
    TORCH_CHECK(st == MUON_POLAR_OK, "fp8: ", muon_polar_last_error());
    multiply(q.operand(xq), rows, held, n, q.width(), y);
    for (at::Tensor *t : {&saved_x, &saved_w})
        if (!t->defined()) *t = none(x);
    return {y, saved_x, saved_w};
}

// Gradients of x (with the saved transposed weight) and of the weight (with the saved
// transposed x) of k columns, as wanted (1: x, 2: weight).
std::tuple<at::Tensor, at::Tensor> Fp8LinearBackward(const at::Tensor &dy, const at::Tensor &saved_x,
                                                     const at::Tensor &saved_w, int64_t k,
                                                     at::ScalarType weight_dtype, int64_t wanted) {
    const c10::OptionalDeviceGuard device_guard(dy.device());
    TORCH_CHECK(dy.device().is_cuda() && dy.dim() >= 1 && dy.size(-1) > 0,
                "fp8: a gradient [.., N] on a ROCm (HIP) device is needed");
    const int64_t rows = rows_of(dy), n = dy.size(-1);
    const Layout g{rows, n, 1, false}, gt{n, rows, 1, false}, xt{k, rows, 1, false},
        wt{k, n, kBlock, true};
    TORCH_CHECK(!(wanted & 1) || saved_w.numel() == wt.bytes(), "fp8: saved for another gradient");
    TORCH_CHECK(!(wanted & 2) || saved_x.numel() == xt.bytes(), "fp8: saved for another gradient");
    const at::Tensor gq = (wanted & 1) ? g.empty(dy) : at::Tensor();
    const at::Tensor gtq = (wanted & 2) ? gt.empty(dy) : at::Tensor();
    if (wanted & 3) hold_rows(dy, gq, gtq);
    at::Tensor dx = none(dy), dw = none(dy);
    if (wanted & 1) {
        dx = result_like(dy, k);
        multiply(g.operand(gq), rows, wt.operand(saved_w), k, g.width(), dx);
    }
    if (wanted & 2) {
        dw = at::empty({n, k}, dy.options().dtype(weight_dtype));
        multiply(gt.operand(gtq), n, xt.operand(saved_x), k, gt.width(), dw);
    }
    return {dx, dw};
}

// =============================================================== what users call
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// The operator of this library with f's signature, through the dispatcher (so that
// FakeTensor and tracing modes see it).
template <class F>
c10::TypedOperatorHandle<F> find(const char *name, F *) {
    return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}
#define MUON_TRAIN_OP(name, function)                                              \
    ([]() -> auto & {                                                              \
        static const auto op = find("muon_ascend950::" name, &function);           \
        return op;                                                                 \
    }())

void check_tensor(const char *name, const at::Tensor &t, const at::Tensor *like,
                  at::ArrayRef<at::ScalarType> types) {
    if (!like) {
        TORCH_CHECK_VALUE(t.device().is_cuda(), name, " must be on a ROCm GPU, got ", t.device());
    } else {
        TORCH_CHECK_VALUE(t.device() == like->device(), name, " must be on ", like->device(),
                          ", got ", t.device());
    }
    for (at::ScalarType type : types)
        if (t.scalar_type() == type) return;
    std::string names;
    for (at::ScalarType type : types)
        names += (names.empty() ? "torch." : " or torch.") +
                 std::string(type == at::kFloat      ? "float32"
                             : type == at::kBFloat16 ? "bfloat16"
                             : type == at::kInt      ? "int32"
                             : type == at::kLong     ? "int64"
                                                     : "float8_e4m3fn");
    TORCH_CHECK_TYPE(false, name, " must use ", names, ", got ", t.scalar_type());
}
constexpr at::ScalarType kFloats[] = {at::kFloat, at::kBFloat16};
constexpr at::ScalarType kFloat32[] = {at::kFloat};
constexpr at::ScalarType kInts[] = {at::kInt, at::kLong};
constexpr at::ScalarType kInt64[] = {at::kLong};
constexpr at::ScalarType kFp8[] = {at::kFloat8_e4m3fn};

bool wants_grad(const at::Tensor &t) { return t.requires_grad(); }
bool wants_grad(const OptTensor &t) { return given(t) && t->requires_grad(); }
OptTensor maybe(const at::Tensor &t) { return t.defined() ? OptTensor(t) : OptTensor(); }
// No operator has a derivative in forward mode: a tangent that reaches one is refused here, or
// it would be lost with the result none the wiser (an operator that is called without a
// reverse-mode gradient leaves autograd behind).  Level 0 is the only one there is.
bool has_tangent(const at::Tensor &t) { return t.defined() && t._fw_grad(0).defined(); }
bool has_tangent(const OptTensor &t) { return t.has_value() && has_tangent(*t); }
template <class... T>
void refuse_tangents(const char *what, const T &...t) {
    TORCH_CHECK_NOT_IMPLEMENTED(!(has_tangent(t) || ...), what, ": no derivative in forward mode");
}
// Gradients that have none of their own: in a pass that keeps its graph, asking them for one
// is an error.
variable_list only_once(variable_list grads, const char *what) {
    if (!at::GradMode::is_enabled()) return grads;
    for (at::Tensor &g : grads) {
        if (!g.defined()) continue;
        g = g.detach();
        g.set_requires_grad(true);
    }
    const auto error = std::make_shared<torch::autograd::DelayedError>(
        std::string(what) + ": its gradient has no gradient of its own",
        static_cast<int64_t>(grads.size()));
    return (*error)(std::move(grads));
}

// ---------------------------------------------------------------------------- norms
constexpr int64_t kMaxChannels = 16384;

// Kind of a gate for y, and how many rows share one vector of it.
std::pair<int64_t, int64_t> gate_kind(const at::Tensor &y, const at::Tensor &gate) {
    const auto want = y.sizes(), got = gate.sizes();
    const int64_t dims = y.dim(), d = want.back();
    bool ones = gate.dim() >= 1 && gate.dim() <= dims && got.back() == d;
    for (int64_t i = 0; ones && i + 1 < gate.dim(); ++i) ones = got[i] == 1;
    if (ones) return {MUON_TRAIN_GATE_CHANNEL, 1};
    if (got == want) return {MUON_TRAIN_GATE_FULL, 1};
    if (gate.dim() == dims && got.slice(0, dims - 1) == want.slice(0, dims - 1) && got.back() == 1)
        return {MUON_TRAIN_GATE_TOKEN, 1};
    if (dims >= 3 && gate.dim() == dims && got[0] == want[0] && got.back() == d) {
        int64_t rows = 1;
        for (int64_t i = 1; ones = got[i] == 1, ones && i + 1 < dims - 1; ++i) rows *= want[i];
        if (ones) return {MUON_TRAIN_GATE_SEQUENCE, rows * want[dims - 2]};
    }
    TORCH_CHECK_VALUE(false, "gate of shape ", got, " does not fit y of shape ", want,
                      ": expected [D], [..., 1], [B, 1, D] or y's own shape");
}

struct BlockNormsFunction : torch::autograd::Function<BlockNormsFunction> {
    static variable_list forward(AutogradContext *ctx, const at::Tensor &y,
                                 const at::Tensor &residual, const OptTensor &post_weight,
                                 const OptTensor &gate, const OptTensor &scale,
                                 const OptTensor &pre_weight, double value, int64_t kind,
                                 int64_t per_sequence, bool post_norm, bool pre_norm, double eps,
                                 int64_t wanted) {
        const at::AutoDispatchBelowADInplaceOrView below;
        auto [out, normed, stats] = MUON_TRAIN_OP("norms_forward", NormsForward)
                                        .call(y, residual, post_weight, gate, scale, value,
                                              pre_weight, kind, per_sequence, post_norm, pre_norm,
                                              eps, true);
        auto held = [](const OptTensor &t) { return given(t) ? *t : at::Tensor(); };
        ctx->save_for_backward({y, residual, held(post_weight), held(gate), held(scale),
                                held(pre_weight), stats});
        ctx->saved_data["numbers"] = std::vector<double>{value, eps};
        ctx->saved_data["choices"] =
            std::vector<int64_t>{kind, per_sequence, post_norm, pre_norm, wanted};
        ctx->set_materialize_grads(false);
        if (!pre_norm) ctx->mark_non_differentiable({normed});
        return {out, normed};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        variable_list result(13);
        const bool pre_norm = ctx->saved_data["choices"].toIntVector()[3];
        if (!grads[0].defined() && !(grads[1].defined() && pre_norm)) return result;
        refuse_tangents("block_norms", grads[0], grads[1]);
        const auto t = ctx->get_saved_variables();
        const auto numbers = ctx->saved_data["numbers"].toDoubleVector();
        const auto choices = ctx->saved_data["choices"].toIntVector();
        const int64_t wanted = choices[4];
        const at::AutoDispatchBelowADInplaceOrView below;
        auto [dy, dr, d_post, d_gate, d_scale, d_pre] =
            MUON_TRAIN_OP("norms_backward", NormsBackward)
                .call(t[0], t[1], maybe(t[2]), maybe(t[3]), maybe(t[4]), numbers[0], maybe(t[5]),
                      choices[0], choices[1], choices[2], choices[3], numbers[1], t[6],
                      maybe(grads[0]), maybe(grads[1]), wanted & 15);
        if (wanted & 16) result[0] = dy;
        if (wanted & 32) result[1] = dr;
        if (wanted & 1) result[2] = d_post;
        if (wanted & 2) result[3] = d_gate;
        if (wanted & 4) result[4] = d_scale;
        if (wanted & 8) result[5] = d_pre;
        return only_once(std::move(result), "block_norms");
    }
};

std::tuple<at::Tensor, at::Tensor> BlockNorms(const at::Tensor &y, const at::Tensor &residual,
                                              const OptTensor &post_weight, const OptTensor &gate,
                                              const OptTensor &scale, double value,
                                              const OptTensor &pre_weight, bool post_norm,
                                              bool pre_norm, double eps) {
    check_tensor("y", y, nullptr, kFloats);
    check_tensor("residual", residual, &y, kFloats);
    TORCH_CHECK_VALUE(y.dim() >= 1 && residual.sizes() == y.sizes(),
                      "y and residual must have one shape [..., D], got ", y.sizes(), " and ",
                      residual.sizes());
    const int64_t d = y.size(-1);
    TORCH_CHECK_VALUE(d >= 1 && d <= kMaxChannels, "D must be 1 to ", kMaxChannels, ", got ", d);
    const std::pair<const char *, const OptTensor &> weights[] = {{"post_weight", post_weight},
                                                                  {"pre_weight", pre_weight}};
    for (const auto &[name, w] : weights) {
        if (!given(w)) continue;
        check_tensor(name, *w, &y, kFloats);
        TORCH_CHECK_VALUE(w->dim() == 1 && w->size(0) == d, name, " must have shape [", d,
                          "], got ", w->sizes());
    }
    TORCH_CHECK_TYPE(!given(post_weight) || !given(pre_weight) ||
                         post_weight->scalar_type() == pre_weight->scalar_type(),
                     "post_weight and pre_weight must have one dtype");
    TORCH_CHECK_VALUE(!given(pre_weight) || pre_norm, "pre_weight needs pre_norm");
    std::pair<int64_t, int64_t> kind{MUON_TRAIN_GATE_NONE, 1};
    if (given(gate)) {
        check_tensor("gate", *gate, &y, kFloats);
        kind = gate_kind(y, *gate);
    }
    if (given(scale)) {
        check_tensor("residual_scale", *scale, &y, kFloat32);
        TORCH_CHECK_VALUE(scale->dim() == 0 || (scale->dim() == 1 && (scale->size(0) == 1 ||
                                                                      scale->size(0) == d)),
                          "residual_scale must have one or ", d, " elements, got shape ",
                          scale->sizes());
    }
    TORCH_CHECK_VALUE(eps >= 0.0, "eps must not be negative, got ", eps);
    refuse_tangents("block_norms", y, residual, post_weight, gate, scale, pre_weight);
    int64_t wanted = 0;
    if (at::GradMode::is_enabled())
        wanted = int64_t(wants_grad(post_weight)) | wants_grad(gate) << 1 | wants_grad(scale) << 2 |
                 wants_grad(pre_weight) << 3 | wants_grad(y) << 4 | wants_grad(residual) << 5;
    if (wanted) {
        const variable_list r = BlockNormsFunction::apply(
            y, residual, post_weight, gate, scale, pre_weight, value, kind.first, kind.second,
            post_norm, pre_norm, eps, wanted);
        return {r[0], r[1]};
    }
    auto [out, normed, stats] =
        MUON_TRAIN_OP("norms_forward", NormsForward)
            .call(y, residual, post_weight, gate, scale, value, pre_weight, kind.first, kind.second,
                  post_norm, pre_norm, eps, false);
    return {out, normed};
}

// -------------------------------------------------------------------------- distill
constexpr int64_t kMaxTop = 1024;

// Checks the operands; false where the labels carry no weight.
bool check_distill(const at::Tensor &logits, const at::Tensor &teacher_logits,
                   const at::Tensor &teacher_indices, const OptTensor &labels, double temperature,
                   double label_weight) {
    check_tensor("logits", logits, nullptr, kFloats);
    check_tensor("teacher_logits", teacher_logits, &logits, kFloats);
    check_tensor("teacher_indices", teacher_indices, &logits, kInts);
    TORCH_CHECK_VALUE(logits.dim() >= 1 && logits.size(-1) >= 1,
                      "logits must have shape [..., V], got ", logits.sizes());
    const auto lead = logits.sizes().slice(0, logits.dim() - 1);
    TORCH_CHECK_VALUE(teacher_logits.dim() == logits.dim() &&
                          teacher_logits.sizes().slice(0, logits.dim() - 1) == lead &&
                          teacher_indices.sizes() == teacher_logits.sizes(),
                      "teacher_logits and teacher_indices must have shape ", lead, " + [K], got ",
                      teacher_logits.sizes(), " and ", teacher_indices.sizes());
    const int64_t k = teacher_logits.size(-1);
    TORCH_CHECK_VALUE(k >= 1 && k <= kMaxTop, "K must be 1 to ", kMaxTop, ", got ", k);
    TORCH_CHECK_VALUE(temperature >= double(FLT_MIN) && temperature < 1e30,
                      "temperature must be a positive normal float32 number below 1e30, got ",
                      temperature);
    TORCH_CHECK_VALUE(label_weight >= 0.0 && label_weight <= 1.0,
                      "label_weight must be 0 to 1, got ", label_weight);
    if (!given(labels)) {
        TORCH_CHECK_VALUE(label_weight == 0.0, "label_weight needs labels");
        return false;
    }
    check_tensor("labels", *labels, &logits, kInt64);
    TORCH_CHECK_VALUE(labels->sizes() == lead, "labels must have shape ", lead, ", got ",
                      labels->sizes());
    return label_weight != 0.0;
}

struct DistillFunction : torch::autograd::Function<DistillFunction> {
    static at::Tensor forward(AutogradContext *ctx, const at::Tensor &logits,
                              const at::Tensor &teacher_logits, const at::Tensor &teacher_indices,
                              const OptTensor &labels, double temperature, double label_weight) {
        const at::AutoDispatchBelowADInplaceOrView below;
        auto [loss, stats] = MUON_TRAIN_OP("distill_forward", DistillForward)
                                 .call(logits, teacher_logits, teacher_indices, labels,
                                       temperature, label_weight, true);
        ctx->save_for_backward({logits, teacher_logits, teacher_indices,
                                given(labels) ? *labels : at::Tensor(), stats});
        ctx->saved_data["numbers"] = std::vector<double>{temperature, label_weight};
        return loss;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        refuse_tangents("distill_topk", grads[0]);
        const at::AutoDispatchBelowADInplaceOrView below;
        const auto t = ctx->get_saved_variables();
        const auto numbers = ctx->saved_data["numbers"].toDoubleVector();
        variable_list result(6);
        result[0] = MUON_TRAIN_OP("distill_backward", DistillBackward)
                        .call(t[0], t[1], t[2], maybe(t[3]), numbers[0], numbers[1], t[4], grads[0]);
        return only_once(std::move(result), "distill_topk");
    }
};

at::Tensor DistillTopk(const at::Tensor &logits, const at::Tensor &teacher_logits,
                       const at::Tensor &teacher_indices, const OptTensor &labels,
                       double temperature, double label_weight) {
    const bool hard = check_distill(logits, teacher_logits, teacher_indices, labels, temperature,
                                    label_weight);
    refuse_tangents("distill_topk", logits, teacher_logits);
    const OptTensor used = hard ? labels : OptTensor();
    if (at::GradMode::is_enabled() && wants_grad(logits))
        return DistillFunction::apply(logits, teacher_logits.detach(), teacher_indices, used,
                                      temperature, label_weight);
    return std::get<0>(MUON_TRAIN_OP("distill_forward", DistillForward)
                           .call(logits, teacher_logits, teacher_indices, used, temperature,
                                 label_weight, false));
}

// (loss, gradient), the gradient empty where it went into `out`.
std::tuple<at::Tensor, at::Tensor> DistillTopkWithGrad(
    const at::Tensor &logits, const at::Tensor &teacher_logits, const at::Tensor &teacher_indices,
    const OptTensor &labels, double temperature, double label_weight, const OptTensor &grad_loss,
    double grad_value, const OptTensor &out) {
    const bool hard = check_distill(logits, teacher_logits, teacher_indices, labels, temperature,
                                    label_weight);
    if (given(grad_loss)) {
        check_tensor("grad_loss", *grad_loss, &logits, kFloat32);
        const auto lead = logits.sizes().slice(0, logits.dim() - 1);
        TORCH_CHECK_VALUE(grad_loss->sizes() == lead, "grad_loss must have shape ", lead, ", got ",
                          grad_loss->sizes());
    }
    refuse_tangents("distill_topk_with_grad", logits, teacher_logits, grad_loss, out);
    const at::NoGradGuard no_grad;
    at::Tensor grad;
    if (given(out)) {
        const at::ScalarType type[] = {logits.scalar_type()};
        check_tensor("out", *out, &logits, type);
        TORCH_CHECK_VALUE(out->sizes() == logits.sizes(), "out must have shape ", logits.sizes(),
                          ", got ", out->sizes());
        grad = *out;
    } else {
        grad = at::empty(logits.sizes(), logits.options());
    }
    at::Tensor loss = MUON_TRAIN_OP("distill_with_grad", DistillWithGrad)
                          .call(logits, teacher_logits, teacher_indices, hard ? labels : OptTensor(),
                                temperature, label_weight, grad_loss, grad_value, grad);
    if (!given(out)) return {loss, grad};
    if (!out->is_inference()) out->unsafeGetTensorImpl()->bump_version();
    return {loss, none(loss)};
}

// ------------------------------------------------------------------------------ fp8
struct Fp8LinearFunction : torch::autograd::Function<Fp8LinearFunction> {
    static at::Tensor forward(AutogradContext *ctx, const at::Tensor &x, const at::Tensor &weight,
                              int64_t wanted) {
        const at::AutoDispatchBelowADInplaceOrView below;
        // wanted: 1 x, 2 weight; the weight's gradient needs x saved and the other way round
        const int64_t save = (wanted & 2) >> 1 | (wanted & 1) << 1;
        auto [y, xt, wt] = MUON_TRAIN_OP("fp8_linear_forward", Fp8LinearForward).call(x, weight, save);
        ctx->save_for_backward({xt, wt});
        ctx->saved_data["choices"] = std::vector<int64_t>{
            wanted, static_cast<int64_t>(weight.scalar_type()), weight.size(1)};
        return y;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        refuse_tangents("fp8_linear", grads[0]);
        const at::AutoDispatchBelowADInplaceOrView below;
        const auto t = ctx->get_saved_variables();
        const auto choices = ctx->saved_data["choices"].toIntVector();
        auto [dx, dw] = MUON_TRAIN_OP("fp8_linear_backward", Fp8LinearBackward)
                            .call(grads[0], t[0], t[1], choices[2],
                                  static_cast<at::ScalarType>(choices[1]), choices[0]);
        variable_list result(3);
        if (choices[0] & 1) result[0] = dx;
        if (choices[0] & 2) result[1] = dw;
        return only_once(std::move(result), "fp8_linear");
    }
};

// Whether an operand of a product, rows of `width` values with `scales` scales in each column of
// blocks, lies within what a product reaches (include/muon_train.h).
bool reached(int64_t width, int64_t scales) {
    return blocks(width) * kBlock <= MUON_TRAIN_FP8_MAX_LD &&
           scales <= MUON_TRAIN_FP8_MAX_SCALES / (blocks(width) + 1);
}

at::Tensor Fp8LinearTrain(const at::Tensor &x, const at::Tensor &weight) {
    check_tensor("x", x, nullptr, kFloats);
    TORCH_CHECK_VALUE(x.dim() >= 1, "x must have shape [..., K]");
    check_tensor("weight", weight, &x, kFloats);
    TORCH_CHECK_VALUE(weight.dim() == 2 && weight.size(1) == x.size(-1),
                      "weight must have shape [N, ", x.size(-1), "], got ", weight.sizes());
    TORCH_CHECK_VALUE(weight.numel() > 0, "weight's dimensions must be positive");
    refuse_tangents("fp8_linear", x, weight);
    // what the backward pass would refuse: dy [tokens, N], and both operands transposed
    const int64_t tokens = rows_of(x), n = weight.size(0), k = weight.size(1);
    if (at::GradMode::is_enabled())
        TORCH_CHECK_VALUE((!wants_grad(x) || reached(n, tokens)) &&
                              (!wants_grad(weight) || (reached(tokens, n) && reached(tokens, k))),
                          "too many tokens for a backward pass in one call, ", tokens, " of ", k, " to ", n,
                          " columns");
    if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(weight)))
        return Fp8LinearFunction::apply(x, weight,
                                        int64_t(wants_grad(x)) | wants_grad(weight) << 1);
    return std::get<0>(
        MUON_TRAIN_OP("fp8_linear_forward", Fp8LinearForward).call(x, weight, 0));
}

at::Tensor Fp8LinearServe(const at::Tensor &x, const at::Tensor &values, const at::Tensor &scales,
                          int64_t cols) {
    check_tensor("x", x, nullptr, kFloats);
    TORCH_CHECK_VALUE(x.dim() >= 1, "x must have shape [..., K]");
    check_tensor("weight", values, &x, kFp8);
    TORCH_CHECK_VALUE(cols == x.size(-1), "x must have ", cols, " columns, got shape ", x.sizes());
    TORCH_CHECK_VALUE(!(at::GradMode::is_enabled() && wants_grad(x)),
                      "a quantised weight has no gradient: pass the float32 or bfloat16 one");
    refuse_tangents("fp8_linear", x, scales);
    return MUON_TRAIN_OP("fp8_linear", Fp8Linear).call(x, values, scales);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(muon_ascend950, m) {
    m.def("norms_forward(Tensor y, Tensor residual, Tensor? post_weight, Tensor? gate, "
          "Tensor? scale, float scale_value, Tensor? pre_weight, int gate_kind, "
          "int rows_per_sequence, bool post_norm, bool pre_norm, float eps, bool save) -> "
          "(Tensor, Tensor, Tensor)");
    m.def("norms_backward(Tensor y, Tensor residual, Tensor? post_weight, Tensor? gate, "
          "Tensor? scale, float scale_value, Tensor? pre_weight, int gate_kind, "
          "int rows_per_sequence, bool post_norm, bool pre_norm, float eps, Tensor stats, "
          "Tensor? d_residual_out, Tensor? d_normed, int wanted) -> "
          "(Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)");
    m.def("distill_forward(Tensor logits, Tensor teacher_logits, Tensor teacher_indices, "
          "Tensor? labels, float temperature, float label_weight, bool save) -> (Tensor, Tensor)");
    m.def("distill_backward(Tensor logits, Tensor teacher_logits, Tensor teacher_indices, "
          "Tensor? labels, float temperature, float label_weight, Tensor stats, "
          "Tensor grad_loss) -> Tensor");
    m.def("distill_with_grad(Tensor logits, Tensor teacher_logits, Tensor teacher_indices, "
          "Tensor? labels, float temperature, float label_weight, Tensor? grad_loss, "
          "float grad_value, Tensor(a!) grad) -> Tensor");
    m.def("quantize_fp8(Tensor x, int block_rows) -> (Tensor, Tensor)");
    m.def("fp8_matmul(Tensor a, Tensor a_scales, Tensor b, Tensor b_scales, ScalarType dtype) -> "
          "Tensor");
    m.def("fp8_linear(Tensor x, Tensor values, Tensor scales) -> Tensor");
    m.def("fp8_linear_forward(Tensor x, Tensor weight, int save) -> (Tensor, Tensor, Tensor)");
    m.def("fp8_linear_backward(Tensor dy, Tensor saved_x, Tensor saved_w, int k, "
          "ScalarType weight_dtype, int wanted) -> (Tensor, Tensor)");

    m.def("block_norms(Tensor y, Tensor residual, Tensor? post_weight, Tensor? gate, "
          "Tensor? scale, float scale_value, Tensor? pre_weight, bool post_norm, bool pre_norm, "
          "float eps) -> (Tensor, Tensor)", &BlockNorms);
    m.def("distill_topk(Tensor logits, Tensor teacher_logits, Tensor teacher_indices, "
          "Tensor? labels, float temperature, float label_weight) -> Tensor", &DistillTopk);
    m.def("distill_topk_with_grad(Tensor logits, Tensor teacher_logits, Tensor teacher_indices, "
          "Tensor? labels, float temperature, float label_weight, Tensor? grad_loss, "
          "float grad_value, Tensor(a!)? out) -> (Tensor, Tensor)", &DistillTopkWithGrad);
    m.def("fp8_linear_train(Tensor x, Tensor weight) -> Tensor", &Fp8LinearTrain);
    m.def("fp8_linear_serve(Tensor x, Tensor values, Tensor scales, int cols) -> Tensor",
          &Fp8LinearServe);
}

TORCH_LIBRARY_IMPL(muon_ascend950, CUDA, m) {
    m.impl("norms_forward", &NormsForward);
    m.impl("norms_backward", &NormsBackward);
    m.impl("distill_forward", &DistillForward);
    m.impl("distill_backward", &DistillBackward);
    m.impl("distill_with_grad", &DistillWithGrad);
    m.impl("quantize_fp8", &QuantizeFp8);
    m.impl("fp8_matmul", &Fp8Matmul);
    m.impl("fp8_linear", &Fp8Linear);
    m.impl("fp8_linear_forward", &Fp8LinearForward);
    m.impl("fp8_linear_backward", &Fp8LinearBackward);
}
