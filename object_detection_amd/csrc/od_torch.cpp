// torch binding of the operators that train a head: group norm with an activation, and the losses over a large vocabulary.
// Outputs and scratch come from torch's allocator, the launches go to the current stream, and the backward passes are
// autograd nodes in C++: a step over a small map is bound by the host, and a Python node costs the autograd thread its turn
// at the interpreter twice (158 -> 81 us for a training step of a 2 x 96 x 61 x 47 map).  The arguments are checked by the
// Python functions that call this (norm.py, det_utils.py); the kernels are those of the C ABI.
#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/utils/pybind.h>

#include "../../include/od_boxes.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> OptTensor;

int dtype_code(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return OD_DTYPE_F32;
        case at::kHalf: return OD_DTYPE_F16;
        case at::kBFloat16: return OD_DTYPE_BF16;
        default: break;
    }
    TORCH_CHECK_TYPE(false, "element type ", t.scalar_type(), " is not supported (float32, float16, bfloat16)");
}

void* stream_of(const Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

void check(int code, const char* what) {
    TORCH_CHECK(code == 0, what, code < 0 ? ": rejected with code " : ": HIP runtime error ", code);
}

Tensor bytes(int64_t n, const Tensor& like) { return at::empty({n}, like.options().dtype(at::kByte)); }

const void* address(const Tensor& t) { return t.defined() && t.numel() > 0 ? t.const_data_ptr() : nullptr; }
void* address_mut(const Tensor& t) { return t.defined() && t.numel() > 0 ? t.data_ptr() : nullptr; }

// Gradients that come out of kernels have no graph behind them: under create_graph they raise when they are differentiated
// again, instead of counting as constants.
variable_list once(variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    variable_list out(grads.size());
    for (size_t i = 0; i < grads.size(); ++i) {
        if (!grads[i].defined()) continue;
        auto stop = std::make_shared<torch::autograd::DelayedError>(
            "trying to differentiate twice a function that can be differentiated only once (once_differentiable)", 1);
        Tensor part = grads[i].detach();
        part.set_requires_grad(true);                               // or the node would not become part of the graph
        out[i] = (*stop)({part})[0];
    }
    return out;
}

// A step recorded into a graph must not share leaves with an earlier step on the default stream whose results still live: its
// backward pass would make that stream, on which the leaves' accumulators came to be, wait for the recorded one.  The default
// stream cannot become part of a recording, and the process would end there.  Such a call is refused before it records
// anything.  A stream of another kind becomes part of the recording and is joined at the end of the backward pass.
void check_recording(const Tensor& on, std::initializer_list<const Tensor*> inputs) {
    if (!at::GradMode::is_enabled() || !on.is_cuda()) return;
    const c10::Stream refused = c10::impl::VirtualGuardImpl(on.device().type()).getDefaultStream(on.device());
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing((hipStream_t)stream_of(on), &status) != hipSuccess || status == hipStreamCaptureStatusNone) return;
    for (const Tensor* t : inputs) {
        if (!t->defined() || !t->requires_grad() || !t->is_leaf()) continue;
        const auto accumulator = torch::autograd::impl::try_get_grad_accumulator(*t);
        if (accumulator && accumulator->stream() && *accumulator->stream() == refused)
            TORCH_CHECK(false, "a training step cannot be recorded while results of an earlier one with the same parameters, on "
                               "the default stream, are alive: drop them first");
    }
}

// ---- group norm with an activation -----------------------------------------------------------------------------
// [B, C, H, W] as dense channels-last memory
Tensor dense_map(const Tensor& x) {
    return x.is_contiguous(at::MemoryFormat::ChannelsLast) ? x : x.permute({0, 2, 3, 1}).contiguous().permute({0, 3, 1, 2});
}

// One pixel is both orders at once; under channels-last strides torch's convolution to one output channel refuses it.
Tensor empty_map(const Tensor& like) {
    const bool pixel = like.size(2) * like.size(3) == 1;
    return at::empty(like.sizes(), like.options(), pixel ? at::MemoryFormat::Contiguous : at::MemoryFormat::ChannelsLast);
}

struct NormSizes {
    int64_t batch, pixels, channels;
    explicit NormSizes(const Tensor& x) : batch(x.size(0)), pixels(x.size(2) * x.size(3)), channels(x.size(1)) {}
};

struct GroupNormAct : torch::autograd::Function<GroupNormAct> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x_in, const OptTensor& weight, const OptTensor& bias,
                          int64_t groups, double eps, int64_t activation, int64_t workspace) {
        const c10::OptionalDeviceGuard guard(x_in.device());
        const Tensor x = dense_map(x_in);
        const Tensor w = weight ? weight->contiguous() : Tensor(), b = bias ? bias->contiguous() : Tensor();
        const NormSizes s(x);
        const Tensor y = empty_map(x), stats = at::empty({s.batch, groups, 2}, x.options().dtype(at::kDouble));
        const Tensor ws = bytes(workspace, x);
        const int pcode = w.defined() ? dtype_code(w) : b.defined() ? dtype_code(b) : OD_DTYPE_F32;
        check(od_group_norm_act_forward(address(x), dtype_code(x), s.batch, s.pixels, (int32_t)s.channels, (int32_t)groups,
                                        address(w), address(b), pcode, (float)eps, (int32_t)activation, address_mut(y),
                                        (double*)address_mut(stats), ws.data_ptr(), ws.numel(), stream_of(x)),
              "od_group_norm_act_forward");
        ctx->save_for_backward({x, w, b, stats});
        ctx->saved_data["groups"] = groups;
        ctx->saved_data["activation"] = activation;
        ctx->saved_data["workspace"] = workspace;
        return y;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grad) {
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &w = saved[1], &b = saved[2], &stats = saved[3];
        const int64_t groups = ctx->saved_data["groups"].toInt();
        const c10::OptionalDeviceGuard guard(x.device());
        const NormSizes s(x);
        const Tensor dy = dense_map(grad[0]);
        const bool empty = x.numel() == 0;                          // no launch fills the sums of an empty map
        auto fresh = [&](const Tensor& t, size_t edge) {
            if (!t.defined() || !ctx->needs_input_grad(edge)) return Tensor();
            return empty ? at::zeros_like(t) : at::empty_like(t);
        };
        const Tensor dx = ctx->needs_input_grad(0) ? empty_map(x) : Tensor();
        const Tensor dw = fresh(w, 1), db = fresh(b, w.defined() ? 2 : 1);      // a missing tensor has no edge
        const Tensor ws = bytes(ctx->saved_data["workspace"].toInt(), x);
        const int pcode = w.defined() ? dtype_code(w) : b.defined() ? dtype_code(b) : OD_DTYPE_F32;
        check(od_group_norm_act_backward(address(x), address(dy), dtype_code(x), s.batch, s.pixels, (int32_t)s.channels,
                                         (int32_t)groups, address(w), address(b), pcode,
                                         (int32_t)ctx->saved_data["activation"].toInt(), (const double*)address(stats),
                                         address_mut(dx), address_mut(dw), address_mut(db), ws.data_ptr(), ws.numel(),
                                         stream_of(x)),
              "od_group_norm_act_backward");
        variable_list out = once({dx, dw, db});
        out.resize(7);
        return out;
    }
};

// ---- losses over a large vocabulary ------------------------------------------------------------------------------
// [rows, n] with contiguous rows that do not overlap
Tensor dense_rows(const Tensor& t) {
    const bool fine = (t.size(1) <= 1 || t.stride(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1));
    return fine ? t : t.contiguous();
}
int64_t pitch_of(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

struct VocabLoss : torch::autograd::Function<VocabLoss> {
    static Tensor forward(AutogradContext* ctx, const Tensor& features, const Tensor& weight_in, const OptTensor& bias,
                          const Tensor& targets_in, const OptTensor& teacher_logits, double temperature, int64_t reduction,
                          int64_t saved_bytes, int64_t forward_bytes, int64_t backward_bytes) {
        const c10::OptionalDeviceGuard guard(features.device());
        const Tensor f = dense_rows(features), w = dense_rows(weight_in), t = targets_in.contiguous();
        const Tensor b = bias ? bias->contiguous() : Tensor();
        const Tensor logits = teacher_logits ? teacher_logits->contiguous() : Tensor();
        const int64_t rows = f.size(0), dim = f.size(1), classes = w.size(0);
        const int32_t top = logits.defined() ? (int32_t)t.size(1) : 0;
        const auto f32 = f.options().dtype(at::kFloat);
        const Tensor row_loss = at::empty({rows}, f32);
        const Tensor loss = reduction == OD_REDUCE_NONE ? Tensor() : at::empty({}, f32);
        const Tensor saved = bytes(saved_bytes, f), ws = bytes(forward_bytes, f);
        check(od_vocab_loss_forward(address(f), pitch_of(f), address(w), pitch_of(w), address(b), dtype_code(f), rows, classes,
                                    (int32_t)dim, (const int64_t*)address(t), top, address(logits),
                                    logits.defined() ? dtype_code(logits) : dtype_code(f), (float)temperature,
                                    (int32_t)reduction, (float*)address_mut(row_loss), (float*)address_mut(loss),
                                    saved.data_ptr(), saved.numel(), ws.data_ptr(), ws.numel(), stream_of(f)),
              "od_vocab_loss_forward");
        if (features.requires_grad() || weight_in.requires_grad() || (bias && bias->requires_grad())) {
            ctx->save_for_backward({w, b, t, saved});
            ctx->saved_data["temperature"] = temperature;
            ctx->saved_data["reduction"] = reduction;
            ctx->saved_data["workspace"] = backward_bytes;
        }
        return reduction == OD_REDUCE_NONE ? row_loss : loss;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grad) {
        const variable_list kept = ctx->get_saved_variables();
        const Tensor &w = kept[0], &b = kept[1], &t = kept[2], &saved = kept[3];
        const c10::OptionalDeviceGuard guard(w.device());
        const int64_t rows = t.size(0), classes = w.size(0), dim = w.size(1);
        const Tensor up = grad[0].to(at::kFloat).contiguous();
        auto fresh = [&](at::IntArrayRef shape, bool wanted) {
            if (!wanted) return Tensor();
            return rows == 0 ? at::zeros(shape, w.options()) : at::empty(shape, w.options());
        };
        const Tensor df = fresh({rows, dim}, ctx->needs_input_grad(0)), dw = fresh({classes, dim}, ctx->needs_input_grad(1));
        const Tensor db = fresh({classes}, b.defined() && ctx->needs_input_grad(2));
        const Tensor ws = bytes(ctx->saved_data["workspace"].toInt(), w);
        check(od_vocab_loss_backward(address(w), pitch_of(w), address(b), dtype_code(w), rows, classes, (int32_t)dim,
                                     (const int64_t*)address(t), t.dim() == 2 ? (int32_t)t.size(1) : 0,
                                     (float)ctx->saved_data["temperature"].toDouble(),
                                     (int32_t)ctx->saved_data["reduction"].toInt(), (const float*)address(up),
                                     saved.const_data_ptr(), saved.numel(), address_mut(df), address_mut(dw), address_mut(db),
                                     ws.data_ptr(), ws.numel(), stream_of(w)),
              "od_vocab_loss_backward");
        variable_list out = once({df, dw, db});
        out.resize(10);
        return out;
    }
};

}  // namespace

PYBIND11_MODULE(_od_torch, m) {
    m.def("group_norm_act",
          [](const Tensor& x, int64_t groups, const OptTensor& weight, const OptTensor& bias, double eps, int64_t activation,
             int64_t workspace) {
              const Tensor none;
              check_recording(x, {&x, weight ? &*weight : &none, bias ? &*bias : &none});
              return GroupNormAct::apply(x, weight, bias, groups, eps, activation, workspace);
          },
          pybind11::call_guard<pybind11::gil_scoped_release>());
    m.def("vocab_loss",
          [](const Tensor& features, const Tensor& weight, const OptTensor& bias, const Tensor& targets,
             const OptTensor& teacher_logits, double temperature, int64_t reduction, int64_t saved_bytes,
             int64_t forward_bytes, int64_t backward_bytes) {
              const Tensor none;
              check_recording(features, {&features, &weight, bias ? &*bias : &none});
              return VocabLoss::apply(features, weight, bias, targets, teacher_logits, temperature, reduction, saved_bytes,
                                      forward_bytes, backward_bytes);
          },
          pybind11::call_guard<pybind11::gil_scoped_release>());
}
