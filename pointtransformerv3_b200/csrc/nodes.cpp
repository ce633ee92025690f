// Calls and autograd nodes of the operators behind a network's logits (functional.py, ops.py): outputs and the forward call of the C ABI, and, on
// the engine's thread, the backward call, without Python on the way.  Short calls are bounded by the host: a training step on 64 x 20 logits
// took 104 us with a node in Python, most of it in a thread that has just woken up, and takes 56 so (one of torch's own log_softmax: 49).
//
// The checks of arguments stand in functional.py, ahead of these calls.  Gradients are of first order: one that is to be differentiated again
// is an error node, as torch's once_differentiable leaves it.
#include <c10/core/DeviceGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include "../../include/ptv3_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void check(int rc, const char* what) { TORCH_CHECK(rc == PTV3_OK, what, " failed (", rc, "): ", ptv3_last_error()); }
void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
int dtype_of(const Tensor& t) { return t.scalar_type() == at::kBFloat16 ? PTV3_DTYPE_BF16 : PTV3_DTYPE_F32; }
void* pointer(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
int64_t row_step(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }
Tensor floats(at::IntArrayRef shape, const Tensor& like) { return at::empty(shape, like.options().dtype(at::kFloat)); }
// a tensor made in inference mode counts no changes and cannot be kept for a backward pass
Tensor kept(const Tensor& t) { return t.defined() && t.is_inference() ? t.clone() : t; }

Tensor first_order(Tensor grad)
{
    if (!at::GradMode::is_enabled()) return grad;
    grad = grad.detach().requires_grad_(true);
    torch::autograd::DelayedError error("trying to differentiate twice an operator whose gradients are of first order", 1);
    return error({grad})[0];
}

// outputs of rows that are scored; those that nobody wants are undefined
struct Scores {
    Tensor log_prob, entropy, values, classes;
    Scores(const Tensor& rows, bool labelled, int64_t top)
    {
        const int64_t n = rows.size(0);
        if (labelled) log_prob = floats({n}, rows);
        entropy = floats({n}, rows);
        if (top) {
            values = floats({n, top}, rows);
            classes = at::empty({n, top}, rows.options().dtype(at::kInt));
        }
    }
    using Given = std::optional<Tensor>;
    static Given given(const Tensor& t) { return t.defined() ? Given(t) : Given(); }
    std::tuple<Given, Given, Given, Given> all() const { return {given(log_prob), given(entropy), given(values), given(classes)}; }
};
Scores run_class_scores(const Tensor& logits, const Tensor& labels, int64_t top, double temperature, int64_t ignore, const Tensor& status,
                        const Tensor& stats)
{
    const Scores s(logits, labels.defined(), top);
    check(ptv3_class_scores_fwd(logits.data_ptr(), row_step(logits), pointer(labels), labels.defined() ? (int)labels.element_size() : 0, ignore,
                                (float*)pointer(s.log_prob), (float*)pointer(s.entropy), (float*)pointer(s.values), (int32_t*)pointer(s.classes),
                                (float*)pointer(stats), logits.size(0), (int)logits.size(1), (int)top, (float)temperature, dtype_of(logits),
                                (uint32_t*)pointer(status), stream_of(logits)),
          "ptv3_class_scores_fwd");
    return s;
}
Tensor run_distill(const Tensor& logits, const Tensor& teacher, const Tensor& classes, double temperature, bool rest, const Tensor& status,
                   const Tensor& stats)
{
    const Tensor loss = floats({logits.size(0)}, logits);
    check(ptv3_distill_topk_fwd(logits.data_ptr(), row_step(logits), teacher.data_ptr(), dtype_of(teacher), classes.data_ptr(),
                                (int)classes.element_size(), (int)classes.size(1), (float*)loss.data_ptr(), (float*)pointer(stats), logits.size(0),
                                (int)logits.size(1), (float)temperature, rest, dtype_of(logits), (uint32_t*)status.data_ptr(), stream_of(logits)),
          "ptv3_distill_topk_fwd");
    return loss;
}

struct ClassScores : torch::autograd::Function<ClassScores> {
    static variable_list forward(AutogradContext* ctx, const Tensor& logits, const std::optional<Tensor>& given_labels, int64_t top,
                                 double temperature, int64_t ignore, const std::optional<Tensor>& status)
    {
        const Tensor labels = given_labels.value_or(Tensor()), stats = floats({logits.size(0), 4}, logits);
        const Scores s = run_class_scores(logits, labels, top, temperature, ignore, status.value_or(Tensor()), stats);
        const Tensor &log_prob = s.log_prob, &entropy = s.entropy, &values = s.values, &classes = s.classes;
        ctx->save_for_backward({logits, kept(labels), classes, stats});
        ctx->saved_data["temperature"] = temperature;
        ctx->saved_data["ignore"] = ignore;
        ctx->set_materialize_grads(false);
        // (those that there are)
        variable_list out = {entropy};
        if (labels.defined()) out.push_back(log_prob);
        if (top) {
            out.push_back(values);
            out.push_back(classes);
            ctx->mark_non_differentiable({classes});
        }
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &logits = saved[0], &labels = saved[1], &classes = saved[2], &stats = saved[3];
        const Tensor dentropy = grads[0], dlog_prob = labels.defined() ? grads[1] : Tensor();
        Tensor dtop = classes.defined() ? grads[labels.defined() ? 2 : 1] : Tensor();
        Tensor dlogits;
        if (dentropy.defined() || dlog_prob.defined() || dtop.defined()) {
            const c10::DeviceGuard guard(logits.device());
            const int64_t n = logits.size(0), K = logits.size(1);
            if (dtop.defined()) dtop = dtop.contiguous();
            dlogits = at::empty({n, K}, logits.options());
            check(ptv3_class_scores_bwd(logits.data_ptr(), row_step(logits), pointer(labels), labels.defined() ? (int)labels.element_size() : 0,
                                        ctx->saved_data["ignore"].toInt(), (const int32_t*)pointer(classes), (const float*)stats.data_ptr(),
                                        (const float*)pointer(dlog_prob), dlog_prob.defined() ? dlog_prob.stride(0) : 0,
                                        (const float*)pointer(dentropy), dentropy.defined() ? dentropy.stride(0) : 0,
                                        (const float*)pointer(dtop), dlogits.data_ptr(), n, (int)K,
                                        classes.defined() ? (int)classes.size(1) : 0, (float)ctx->saved_data["temperature"].toDouble(),
                                        dtype_of(logits), stream_of(logits)),
                  "ptv3_class_scores_bwd");
            dlogits = first_order(dlogits);
        }
        return {dlogits, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

struct DistillTopk : torch::autograd::Function<DistillTopk> {
    static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& teacher, const Tensor& classes, double temperature,
                          bool rest, const Tensor& status)
    {
        const Tensor stats = floats({logits.size(0), 4}, logits);
        const Tensor loss = run_distill(logits, teacher, classes, temperature, rest, status, stats);
        ctx->save_for_backward({logits, kept(teacher), kept(classes), stats});
        ctx->saved_data["temperature"] = temperature;
        ctx->saved_data["rest"] = rest;
        return loss;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &logits = saved[0], &teacher = saved[1], &classes = saved[2], &stats = saved[3], &dloss = grads[0];
        const c10::DeviceGuard guard(logits.device());
        const int64_t n = logits.size(0), K = logits.size(1);
        const Tensor dlogits = at::empty({n, K}, logits.options());
        check(ptv3_distill_topk_bwd(logits.data_ptr(), row_step(logits), teacher.data_ptr(), dtype_of(teacher), classes.data_ptr(),
                                    (int)classes.element_size(), (int)classes.size(1), (const float*)stats.data_ptr(),
                                    (const float*)dloss.data_ptr(), dloss.stride(0), dlogits.data_ptr(), n, (int)K,
                                    (float)ctx->saved_data["temperature"].toDouble(), ctx->saved_data["rest"].toBool(), dtype_of(logits),
                                    stream_of(logits)),
              "ptv3_distill_topk_bwd");
        return {first_order(dlogits), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

bool wants_grad(const Tensor& t) { return at::GradMode::is_enabled() && t.requires_grad(); }

// ---- arguments as they ordinarily are: what needs no copy, no message and no read of a status word -------------------------------------
bool logits_are_plain(const Tensor& t)
{
    return t.is_cuda() && t.dim() == 2 && (t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16) && t.size(0) > 1 && t.size(1) >= 1 &&
           t.size(1) <= 1 << 18 && t.stride(1) == 1 && t.stride(0) >= t.size(1);
}
bool is_plain(const Tensor& t, const Tensor& like, bool type) { return type && t.device() == like.device() && t.is_contiguous(); }
bool is_index(const Tensor& t) { return t.scalar_type() == at::kInt || t.scalar_type() == at::kLong; }
bool status_is_plain(const Tensor& t, const Tensor& like) { return is_plain(t, like, t.scalar_type() == at::kInt) && t.numel() > 0; }
bool temperature_is_plain(double t) { return t >= 1e-6 && t <= 1e6; }

using Given = std::optional<Tensor>;
using Answers = std::tuple<Given, Given, Given, Given>;

// -> log_prob (None without labels), entropy, the alternatives' values and classes (None with top = 0)
Answers class_scores(const Tensor& logits, const Given& labels, int64_t top, double temperature, int64_t ignore, const Given& status)
{
    const c10::DeviceGuard guard(logits.device());
    if (!wants_grad(logits))
        return run_class_scores(logits, labels.value_or(Tensor()), top, temperature, ignore, status.value_or(Tensor()), Tensor()).all();
    const variable_list out = ClassScores::apply(logits, labels, top, temperature, ignore, status);
    const size_t at = labels ? 2 : 1;
    return {labels ? Given(out[1]) : Given(), out[0], top ? Given(out[at]) : Given(), top ? Given(out[at + 1]) : Given()};
}
Tensor distill_topk(const Tensor& logits, const Tensor& teacher, const Tensor& classes, double temperature, bool rest, const Tensor& status)
{
    const c10::DeviceGuard guard(logits.device());
    if (!wants_grad(logits)) return run_distill(logits, teacher, classes, temperature, rest, status, Tensor());
    return DistillTopk::apply(logits, teacher, classes, temperature, rest, status);
}
Answers seg_head_scores(const Tensor& feat, const Tensor& weight, const Given& bias, const Given& given_labels, int64_t top, double temperature,
                        int64_t ignore, const Tensor& status)
{
    const c10::DeviceGuard guard(feat.device());
    const Tensor labels = given_labels.value_or(Tensor());
    const Scores s(feat, labels.defined(), top);
    check(ptv3_seg_head_scores_fwd(feat.data_ptr(), weight.data_ptr(), pointer(bias.value_or(Tensor())), pointer(labels),
                                   labels.defined() ? (int)labels.element_size() : 0, ignore, (float*)pointer(s.log_prob),
                                   (float*)pointer(s.entropy), (float*)pointer(s.values), (int32_t*)pointer(s.classes), feat.size(0),
                                   (int)feat.size(1), (int)weight.size(0), (int)top, (float)temperature, dtype_of(feat),
                                   (uint32_t*)status.data_ptr(), stream_of(feat)),
          "ptv3_seg_head_scores_fwd");
    return s.all();
}
bool labels_are_plain(const Given& labels, const Tensor& rows)
{
    return !labels || (labels->dim() == 1 && labels->size(0) == rows.size(0) && is_plain(*labels, rows, is_index(*labels)));
}

}  // namespace

// The functions whose names begin with plain_ return None where an argument is not as ordinary ones are; functional.py and ops.py then check them
// one by one.
PYBIND11_MODULE(ptv3_nodes, m)
{
    m.def("class_scores", &class_scores);
    m.def("distill_topk", &distill_topk);
    m.def("seg_head_scores", &seg_head_scores);
    m.def("plain_class_scores", [](const Tensor& logits, const Given& labels, int64_t top, double temperature, int64_t ignore,
                                   const Given& status) -> std::optional<Answers> {
        if (!logits_are_plain(logits) || !labels_are_plain(labels, logits) || top < 0 || top > 64 || !temperature_is_plain(temperature) ||
            (labels && !(status && status_is_plain(*status, logits))))
            return std::nullopt;
        return class_scores(logits, labels, top, temperature, ignore, status);
    });
    m.def("plain_distill_topk", [](const Tensor& logits, const Tensor& teacher, const Tensor& classes, double temperature, bool rest,
                                   const Given& status) -> Given {
        if (!logits_are_plain(logits) || classes.dim() != 2 || classes.size(0) != logits.size(0) || classes.size(1) < 1 || classes.size(1) > 64 ||
            !is_plain(classes, logits, is_index(classes)) || teacher.sizes() != classes.sizes() || wants_grad(teacher) ||
            !is_plain(teacher, logits, teacher.scalar_type() == at::kFloat || teacher.scalar_type() == at::kBFloat16) ||
            !temperature_is_plain(temperature) || !status || !status_is_plain(*status, logits))
            return std::nullopt;
        return distill_topk(logits, teacher, classes, temperature, rest, *status);
    });
    m.def("plain_seg_head_scores", [](const Tensor& feat, const Tensor& weight, const Given& bias, const Given& labels, int64_t top, double temperature,
                                      int64_t ignore, const Given& status) -> std::optional<Answers> {
        auto bf16 = [&](const Tensor& t, int64_t dim, bool wide) {
            return t.dim() == dim && is_plain(t, feat, t.scalar_type() == at::kBFloat16) && !wants_grad(t) &&
                   (!wide || ((uintptr_t)t.data_ptr() & 15) == 0);
        };
        if (!feat.is_cuda() || !bf16(feat, 2, true) || !bf16(weight, 2, true) || weight.size(1) != feat.size(1) || weight.size(0) < 1 ||
            weight.size(0) > 1 << 18 || (bias && !(bf16(*bias, 1, false) && bias->size(0) == weight.size(0))) || feat.size(1) % 8 ||
            feat.size(1) < 8 || feat.size(1) > 512 || !labels_are_plain(labels, feat) || top < 0 || top > PTV3_HEAD_TOP_MAX ||
            !temperature_is_plain(temperature) || !status || !status_is_plain(*status, feat))
            return std::nullopt;
        return seg_head_scores(feat, weight, bias, labels, top, temperature, ignore, *status);
    });
}
