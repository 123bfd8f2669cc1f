// Front end in C++ of the fine-tuning operators: residual join, log-probability losses, gradient
// norm and clipped AdamW.  The kernels are those of the native library; here are their autograd
// nodes and the memory they need, so that a call costs microseconds of host time (a forward and
// backward pass of the residual join through Python functions: 208 us; through these 95 us, of which
// torch's autograd engine takes some 65).
//
// Arguments are checked in Python (gpubridge_b200/ops); an entry point here only answers None where
// they are not what the kernels take, and Python then says why.
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <ATen/autocast_mode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <atomic>
#include <cmath>
#include <vector>

extern "C" {
const char* gb_error_string(int code);
int gb_residual_norm_fwd(int s, int u, int y, int vec, const void* residual, long long residual_stride,
                         const void* update, long long update_stride, void* stream, void* normed, float* stats,
                         const void* weight, const void* bias, const void* post_weight, const void* post_bias,
                         int param_code, const void* gate, int gate_code, long long rows, long long group_rows, int d,
                         int layer, float scale, float eps, cudaStream_t cuda_stream);
void gb_residual_norm_workers(long long rows, int d, int vec, int* blocks, int* owners);
int gb_residual_norm_bwd(int s, int u, int y, int vec, const void* d_stream, const void* d_normed, const void* stream,
                         const void* update, long long update_stride, const float* stats, const void* weight,
                         const void* bias, const void* post_weight, const void* post_bias, int param_code,
                         const void* gate, int gate_code, void* d_residual, void* d_update, float* part,
                         float* gate_part, void* out0, void* out1, void* out2, void* out3, void* gate_out,
                         long long rows, long long group_rows, int d, int layer, float scale, cudaStream_t cuda_stream);
int gb_token_logprobs(int dtype, const void* logits, long long batch_stride, long long row_stride, long long inner,
                      long long rows, int vocab, int ld, const long long* targets, double temperature, float* logprobs,
                      float* stats, cudaStream_t stream);
int gb_policy_loss(int dtype, const void* logits, long long batch_stride, long long row_stride, long long inner,
                   long long rows, int vocab, int ld, const long long* targets, double temperature, const float* old,
                   const float* advantages, const float* ref, const float* weights, const float* denominator,
                   float clip_low, float clip_high, float kl_coef, float* logprobs, float* stats, float* coef,
                   float* scratch, float* loss, float* kl, float* clipped, void* grad, cudaStream_t stream);
int gb_logprob_grad(int dtype, const void* logits, long long batch_stride, long long row_stride, long long inner,
                    long long rows, int vocab, int ld, const long long* targets, double temperature, const float* stats,
                    const float* coef, const float* upstream, void* grad, cudaStream_t stream);
int gb_preference_loss(const float* logprobs, const long long* targets, const long long* offsets, long long rows,
                       long long length, int sequences, int vocab, int average, const void* ref, int ref_double,
                       double beta, double smoothing, double* sums, float* seq_coef, float* loss, float* rewards,
                       float* seq_logprobs, float* coef, cudaStream_t stream);
int gb_grad_norm_max_tensors();
int gb_grad_norm_parts(void* const* ptrs, const long long* sizes, int count);
int gb_grad_norm_partial(int dtype, int maximum, void* const* ptrs, const long long* sizes, int count, double* part,
                         cudaStream_t stream);
int gb_grad_norm_finish(int maximum, const double* part, int parts, double scale, double max_norm, float* result,
                        cudaStream_t stream);
int gb_grad_clip_coef(const float* norm, double max_norm, float* result, cudaStream_t stream);
int gb_grad_scale(int dtype, void* const* ptrs, const long long* sizes, int count, const float* coef,
                  cudaStream_t stream);
int gb_adamw_clipped(float* p, float* g, float* m, float* v, size_t n, void* state, double lr, double beta1,
                     double beta2, double eps, double weight_decay, float grad_scale, const float* coef, int zero_grad,
                     cudaStream_t stream);
}

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;
using Maybe = std::optional<Tensor>;

std::atomic<long long> g_launches{0};

void check(int code, const char* what, int launches) {
    TORCH_CHECK(code == 0, "gpubridge native call ", what, " failed: ", gb_error_string(code), " (CUDA error ", code, ")");
    g_launches += launches;
}

int code_of(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return 0;
        case at::kBFloat16: return 1;
        case at::kHalf: return 2;
        default: return -1;
    }
}

// An ordinary tensor of a GPU: values in strided memory, no subclass that dispatches on its own.
bool plain(const Tensor& t) {
    return t.is_cuda() && t.layout() == at::kStrided && !t.key_set().has(c10::DispatchKey::Python);
}

bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }
Tensor of(const Maybe& t) { return t.has_value() ? *t : Tensor(); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
cudaStream_t stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
Tensor floats(at::IntArrayRef shape, const Tensor& like) { return at::empty(shape, like.options().dtype(at::kFloat)); }

// Gradients that have no derivative of their own: with create_graph the second backward says so.
variable_list once(variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    variable_list given;
    for (auto& g : grads) if (g.defined()) given.push_back(g.detach().set_requires_grad(true));
    if (given.empty()) return grads;
    auto fail = std::make_shared<torch::autograd::DelayedError>(
        "trying to differentiate twice a function that has no second derivative here", (int)given.size());
    given = (*fail)(std::move(given));
    size_t next = 0;
    for (auto& g : grads) if (g.defined()) g = given[next++];
    return grads;
}

// -- residual join ---------------------------------------------------------------------------------

// [rows, d] whose rows are dense: a view where the strides allow it.
Tensor rows_of(const Tensor& t, int64_t d) {
    Tensor flat = t.reshape({-1, d});
    return d == 1 || flat.stride(1) == 1 ? flat : flat.contiguous();
}

// Whether every row begins on a boundary of eight values.
bool aligned(const Tensor& t) {
    return !t.defined() || (reinterpret_cast<uintptr_t>(t.data_ptr()) % (8 * t.element_size()) == 0 &&
                            (t.size(0) <= 1 || t.stride(0) % 8 == 0));
}

struct Join {
    Tensor residual, update, weight, bias, post_weight, post_bias, gate;
    double scale, eps;
    bool layer;
    at::ScalarType out;
    int param_code() const {
        return weight.defined() ? code_of(weight.scalar_type()) : post_weight.defined() ? code_of(post_weight.scalar_type()) : 0;
    }
    int gate_code() const { return gate.defined() ? code_of(gate.scalar_type()) : 0; }
    int64_t groups() const { return !gate.defined() || gate.dim() == 1 ? 1 : gate.size(0); }
};

// stream, normed (or nothing), stats (or nothing)
std::tuple<Tensor, Tensor, Tensor> join_forward(const Join& a, bool keep) {
    const int64_t d = a.residual.size(-1);
    const Tensor r = rows_of(a.residual, d), u = rows_of(a.update, d);
    const int64_t rows = r.size(0);
    Tensor stream = at::empty(a.residual.sizes(), a.residual.options()), normed, stats;
    if (a.weight.defined()) normed = at::empty(a.residual.sizes(), a.residual.options().dtype(a.out));
    if (keep) stats = floats({rows, 4}, a.residual);
    if (rows) {
        c10::cuda::CUDAGuard guard(a.residual.device());
        const int vec = d % 8 == 0 && aligned(r) && aligned(u) ? 8 : 1;
        check(gb_residual_norm_fwd(code_of(r.scalar_type()), code_of(u.scalar_type()), code_of(a.out), vec, r.data_ptr(),
                                   r.stride(0), u.data_ptr(), u.stride(0), stream.data_ptr(), ptr(normed),
                                   static_cast<float*>(ptr(stats)), ptr(a.weight), ptr(a.bias), ptr(a.post_weight),
                                   ptr(a.post_bias), a.param_code(), ptr(a.gate), a.gate_code(), rows, rows / a.groups(),
                                   (int)d, a.layer, (float)a.scale, (float)a.eps, stream_of(r)),
              "gb_residual_norm_fwd", 1);
    }
    return {stream, normed, stats};
}

struct ResidualNorm : Function<ResidualNorm> {
    static variable_list forward(AutogradContext* ctx, const Tensor& residual, const Tensor& update, const Maybe& weight,
                                 const Maybe& bias, const Maybe& post_weight, const Maybe& post_bias, const Maybe& gate,
                                 double scale, double eps, bool layer, int64_t out) {
        const Join a{residual, update, of(weight), of(bias), of(post_weight), of(post_bias), of(gate), scale, eps, layer,
                     static_cast<at::ScalarType>(out)};
        auto [stream, normed, stats] = join_forward(a, true);
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({update, stream, stats, a.weight, a.bias, a.post_weight, a.post_bias, a.gate});
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["layer"] = layer;
        ctx->saved_data["out"] = out;
        ctx->saved_data["residual"] = residual.requires_grad();
        if (!normed.defined()) return {stream};
        return {stream, normed};
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor &update = saved[0], &stream = saved[1], &stats = saved[2];
        Join a{Tensor(), update, saved[3], saved[4], saved[5], saved[6], saved[7], ctx->saved_data["scale"].toDouble(), 0.0,
               ctx->saved_data["layer"].toBool(), static_cast<at::ScalarType>(ctx->saved_data["out"].toInt())};
        const int param_code = a.param_code();
        variable_list result(11);
        Tensor d_stream = grads[0], d_normed = grads.size() > 1 ? grads[1] : Tensor();
        if (!d_stream.defined() && !d_normed.defined()) return result;
        if (d_stream.defined()) d_stream = d_stream.contiguous();
        if (d_normed.defined()) d_normed = d_normed.contiguous();
        else { a.weight = Tensor(); a.bias = Tensor(); }         // the following norm took no part
        const int64_t d = stream.size(-1);
        const Tensor u = rows_of(update, d);
        const int64_t rows = u.size(0), groups = a.groups();
        // without a norm or a gate of its own the update's gradient is scale times the stream's, and
        // without a following norm the stream's is the one that came
        const bool own = a.post_weight.defined() || a.gate.defined();
        const bool same = !own && a.scale == 1.0 && update.scalar_type() == stream.scalar_type();
        const bool through = !own && !d_normed.defined();
        if (through && (same || !rows)) {
            result[0] = d_stream;
            result[1] = rows ? d_stream : at::empty(update.sizes(), update.options());
            return once(std::move(result));
        }
        if (through) result[0] = d_stream;
        else if (ctx->saved_data["residual"].toBool() || same) result[0] = at::empty(stream.sizes(), stream.options());
        result[1] = same ? result[0] : at::empty(update.sizes(), update.options());
        const Tensor* params[4] = {&a.weight, &a.bias, &a.post_weight, &a.post_bias};
        void* slots[4] = {};
        int64_t sums = 0;
        for (int i = 0; i < 4; ++i) {
            if (!params[i]->defined()) continue;
            result[2 + i] = at::empty(params[i]->sizes(), params[i]->options());
            slots[sums++] = result[2 + i].data_ptr();
        }
        if (a.gate.defined()) result[6] = at::empty(a.gate.sizes(), a.gate.options());
        if (!rows) {
            for (int i = 2; i < 7; ++i) if (result[i].defined()) result[i].zero_();
            return once(std::move(result));
        }
        c10::cuda::CUDAGuard guard(stream.device());
        auto flat = [&](const Tensor& t) { return t.defined() ? t.view({-1, d}) : t; };
        const int vec = d % 8 == 0 && aligned(u) && aligned(flat(d_stream)) && aligned(flat(d_normed)) ? 8 : 1;
        int blocks = 0, owners = 0;
        gb_residual_norm_workers(rows, (int)d, vec, &blocks, &owners);
        const int64_t part = blocks * sums * d, gate_part = a.gate.defined() ? (owners + groups - 1) * d : 0;
        const int64_t apart = (part + 63) / 64 * 64;             // both begin on a vector's boundary
        const Tensor scratch = floats({apart + gate_part}, stream);
        float* at = static_cast<float*>(scratch.data_ptr());
        check(gb_residual_norm_bwd(code_of(stream.scalar_type()), code_of(u.scalar_type()), code_of(a.out), vec,
                                   ptr(d_stream), ptr(d_normed), stream.data_ptr(), u.data_ptr(), u.stride(0),
                                   static_cast<float*>(stats.data_ptr()), ptr(a.weight), ptr(a.bias), ptr(a.post_weight),
                                   ptr(a.post_bias), param_code, ptr(a.gate), a.gate_code(),
                                   through ? nullptr : ptr(result[0]), same ? nullptr : result[1].data_ptr(), at, at + apart, slots[0], slots[1], slots[2], slots[3],
                                   ptr(result[6]), rows, rows / groups, (int)d, a.layer, (float)a.scale, stream_of(stream)),
              "gb_residual_norm_bwd", 2);
        return once(std::move(result));
    }
};

constexpr int64_t MAX_WIDTH = 8192;

// None where Python has to look at the arguments.
std::optional<std::tuple<Tensor, Maybe>> residual_norm(const Tensor& residual, Tensor update, const Maybe& weight_,
                                                       const Maybe& bias_, const Maybe& post_weight_,
                                                       const Maybe& post_bias_, const Maybe& gate_, double scale,
                                                       double eps, const std::string& kind,
                                                       const std::optional<at::ScalarType>& out_dtype) {
    if (!plain(residual) || !plain(update) || residual.dim() < 1 || !update.sizes().equals(residual.sizes())) return std::nullopt;
    const int64_t d = residual.size(-1);
    const bool layer = kind == "layer";
    if (d < 1 || d > MAX_WIDTH || (!layer && kind != "rms")) return std::nullopt;
    at::ScalarType out = residual.scalar_type();
    if (out_dtype.has_value()) out = *out_dtype;
    else if (out == at::kFloat && at::autocast::is_autocast_enabled(at::kCUDA)) out = at::autocast::get_autocast_dtype(at::kCUDA);
    if (code_of(residual.scalar_type()) < 0 || code_of(out) < 0) return std::nullopt;
    if (residual.scalar_type() != at::kFloat && out != residual.scalar_type()) return std::nullopt;
    if (update.device() != residual.device()) return std::nullopt;
    // a stream and an update in fp32 are joined and normed in fp32; only the result is then rounded
    const at::ScalarType asked = out;
    if (residual.scalar_type() == at::kFloat && update.scalar_type() == at::kFloat) out = at::kFloat;
    if (update.scalar_type() != out) update = update.to(out);
    Tensor params[4] = {of(weight_), of(bias_), of(post_weight_), of(post_bias_)};
    if ((params[1].defined() && !params[0].defined()) || (params[3].defined() && !params[2].defined())) return std::nullopt;
    const Tensor& first = params[0].defined() ? params[0] : params[2];
    for (auto& p : params) {
        if (!p.defined()) continue;
        if (!plain(p) || p.device() != residual.device() || p.dim() != 1 || p.size(0) != d || code_of(p.scalar_type()) < 0) return std::nullopt;
        if (p.scalar_type() != first.scalar_type()) p = p.to(first.scalar_type());
        if (!p.is_contiguous()) p = p.contiguous();
    }
    Tensor gate = of(gate_);
    if (gate.defined()) {
        if (!plain(gate) || gate.device() != residual.device() || code_of(gate.scalar_type()) < 0) return std::nullopt;
        bool good = gate.dim() == 1 && gate.size(0) == d;
        if (!good && gate.dim() == residual.dim() && gate.dim() > 1) {
            good = gate.size(0) == residual.size(0) && gate.size(-1) == d;
            for (int64_t i = 1; i + 1 < gate.dim(); ++i) good = good && gate.size(i) == 1;
        }
        if (!good) return std::nullopt;
        gate = gate.contiguous();
    }
    bool needs = wants_grad(residual) || wants_grad(update) || wants_grad(gate);
    for (auto& p : params) needs = needs || wants_grad(p);
    if (!needs || !at::GradMode::is_enabled()) {
        at::NoGradGuard no_grad;
        auto [stream, normed, stats] = join_forward(
            Join{residual, update, params[0], params[1], params[2], params[3], gate, scale, eps, layer, out}, false);
        return std::make_tuple(stream, normed.defined() ? Maybe(normed.to(asked)) : Maybe());
    }
    auto maybe = [](const Tensor& t) { return t.defined() ? Maybe(t) : Maybe(); };
    auto got = ResidualNorm::apply(residual, update, maybe(params[0]), maybe(params[1]), maybe(params[2]), maybe(params[3]),
                                   maybe(gate), scale, eps, layer, static_cast<int64_t>(out));
    return std::make_tuple(got[0], got.size() > 1 ? Maybe(got[1].to(asked)) : Maybe());
}

// -- log-probabilities -------------------------------------------------------------------------------

// The rows of a logits tensor as the kernels take them, and room for their gradient.
struct Rows {
    Tensor logits;
    int code, vocab, ld, skew;
    long long batch, row, inner, rows;
    Rows(const Tensor& given, int64_t vocab_) : logits(given), vocab((int)vocab_) {
        const int64_t width = given.size(-1), step = 16 / given.element_size();
        bool strided = (given.dim() == 2 || given.dim() == 3) && (width == 1 || given.stride(-1) == 1) && width % step == 0 &&
                       reinterpret_cast<uintptr_t>(given.data_ptr()) % 16 == 0;
        for (int64_t i = 0; i + 1 < given.dim(); ++i) strided = strided && given.stride(i) % step == 0;
        if (!given.is_contiguous() && !strided) logits = given.contiguous();
        code = code_of(logits.scalar_type());
        ld = (int)width;
        rows = logits.numel() / width;
        inner = rows > 0 ? rows : 1;
        batch = 0;
        row = width;
        if (!logits.is_contiguous()) {
            row = logits.stride(-2);
            if (logits.dim() == 3) { batch = logits.stride(0); inner = logits.size(1); }
        }
        skew = (int)(reinterpret_cast<uintptr_t>(logits.data_ptr()) % 16 / logits.element_size());
    }
    // [..., ld] without gaps, as far from a 16-byte boundary as the logits
    Tensor grad() const {
        if (!skew) return at::empty(logits.sizes(), logits.options());
        return at::empty({logits.numel() + skew}, logits.options()).slice(0, skew).view(logits.sizes());
    }
};

#define GB_ROWS(r) (r).code, (r).logits.data_ptr(), (r).batch, (r).row, (r).inner, (r).rows, (r).vocab, (r).ld

const long long* targets_of(const Tensor& t) { return reinterpret_cast<const long long*>(t.data_ptr<int64_t>()); }
float* f32(const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }

Tensor logits_grad(const Tensor& logits, int64_t vocab, const Tensor& targets, double temperature, const Tensor& stats,
                   const Tensor& coef, const Tensor& upstream) {
    const Rows r(logits, vocab);
    Tensor grad = r.grad();
    if (r.rows) {
        c10::cuda::CUDAGuard guard(grad.device());
        check(gb_logprob_grad(GB_ROWS(r), targets_of(targets), temperature, f32(stats), f32(coef), f32(upstream),
                              grad.data_ptr(), stream_of(grad)), "gb_logprob_grad", 1);
    }
    return grad;
}

std::tuple<Tensor, Tensor> logprobs_of(const Rows& r, const Tensor& targets, double temperature, bool keep) {
    Tensor logprobs = floats(targets.sizes(), r.logits), stats;
    if (keep) stats = floats({r.rows, 2}, r.logits);
    if (r.rows) {
        c10::cuda::CUDAGuard guard(logprobs.device());
        check(gb_token_logprobs(GB_ROWS(r), targets_of(targets), temperature, f32(logprobs), f32(stats),
                                stream_of(logprobs)), "gb_token_logprobs", 1);
    }
    return {logprobs, stats};
}

struct TokenLogprobs : Function<TokenLogprobs> {
    static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& targets, int64_t vocab, double temperature) {
        auto [logprobs, stats] = logprobs_of(Rows(logits, vocab), targets, temperature, true);
        ctx->save_for_backward({logits, targets, stats});
        ctx->saved_data["vocab"] = vocab;
        ctx->saved_data["temperature"] = temperature;
        return logprobs;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto s = ctx->get_saved_variables();
        variable_list result(4);
        result[0] = logits_grad(s[0], ctx->saved_data["vocab"].toInt(), s[1], ctx->saved_data["temperature"].toDouble(), s[2],
                                grads[0].contiguous(), Tensor());
        return once(std::move(result));
    }
};

Tensor token_logprobs(const Tensor& logits, const Tensor& targets, int64_t vocab, double temperature) {
    if (at::GradMode::is_enabled() && logits.requires_grad()) return TokenLogprobs::apply(logits, targets, vocab, temperature);
    at::NoGradGuard no_grad;
    return std::get<0>(logprobs_of(Rows(logits, vocab), targets, temperature, false));
}

struct Policy {
    Tensor old, advantages, ref, weights, denominator;
    double clip_low, clip_high, kl_coef, temperature;
};

struct PolicyResult {
    Tensor loss, logprobs, kl, clipped, stats, coef, grad;
};

PolicyResult policy_forward(const Tensor& logits, const Tensor& targets, int64_t vocab, const Policy& p, bool needs, bool unit) {
    const Rows r(logits, vocab);
    PolicyResult out;
    out.loss = floats({}, logits);
    out.kl = floats({}, logits);
    out.clipped = floats({}, logits);
    out.logprobs = floats(targets.sizes(), logits);
    if (needs && unit) out.grad = r.grad();
    if (needs && !unit) out.stats = floats({r.rows, 2}, logits);
    if (!r.rows) {
        out.loss.zero_();
        out.kl.zero_();
        out.clipped.zero_();
        out.coef = floats({0}, logits);
        return out;
    }
    const Tensor scratch = floats({4 * r.rows + 1}, logits);
    out.coef = scratch.slice(0, 3 * r.rows + 1);
    c10::cuda::CUDAGuard guard(logits.device());
    check(gb_policy_loss(GB_ROWS(r), targets_of(targets), p.temperature, f32(p.old), f32(p.advantages), f32(p.ref),
                         f32(p.weights), f32(p.denominator), (float)p.clip_low, (float)p.clip_high, (float)p.kl_coef,
                         f32(out.logprobs), f32(out.stats), f32(out.coef), f32(scratch), f32(out.loss), f32(out.kl),
                         f32(out.clipped), ptr(out.grad), stream_of(logits)), "gb_policy_loss", 2);
    return out;
}

struct PolicyLoss : Function<PolicyLoss> {
    static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& targets, int64_t vocab,
                                 const Tensor& old, const Tensor& advantages, const Maybe& ref, const Maybe& weights,
                                 const Maybe& denominator, double low, double high, double kl_coef, double temperature,
                                 bool unit) {
        const Policy p{old, advantages, of(ref), of(weights), of(denominator), low, high, kl_coef, temperature};
        PolicyResult out = policy_forward(logits, targets, vocab, p, true, unit);
        if (unit) ctx->saved_data["grad"] = out.grad;
        else ctx->save_for_backward({logits, targets, out.stats, out.coef});
        ctx->saved_data["unit"] = unit;
        ctx->saved_data["vocab"] = vocab;
        ctx->saved_data["temperature"] = temperature;
        ctx->mark_non_differentiable({out.logprobs, out.kl, out.clipped});
        return {out.loss, out.logprobs, out.kl, out.clipped};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        variable_list result(13);
        if (ctx->saved_data["unit"].toBool()) {
            TORCH_CHECK(ctx->saved_data["grad"].isTensor(), "policy_loss(unit_grad=True) hands its gradient out once: "
                        "leave unit_grad away for a second backward pass");
            result[0] = ctx->saved_data["grad"].toTensor();
            ctx->saved_data["grad"] = c10::IValue();
        } else {
            const auto s = ctx->get_saved_variables();
            result[0] = logits_grad(s[0], ctx->saved_data["vocab"].toInt(), s[1], ctx->saved_data["temperature"].toDouble(),
                                    s[2], s[3], grads[0].to(at::kFloat).contiguous());
        }
        return once(std::move(result));
    }
};

std::tuple<Tensor, Tensor, Tensor, Tensor> policy_loss(const Tensor& logits, const Tensor& targets, int64_t vocab,
                                                       const Tensor& old, const Tensor& advantages, const Maybe& ref,
                                                       const Maybe& weights, const Maybe& denominator, double low,
                                                       double high, double kl_coef, double temperature, bool unit) {
    if (at::GradMode::is_enabled() && logits.requires_grad()) {
        auto v = PolicyLoss::apply(logits, targets, vocab, old, advantages, ref, weights, denominator, low, high, kl_coef,
                                   temperature, unit);
        return {v[0], v[1], v[2], v[3]};
    }
    at::NoGradGuard no_grad;
    auto out = policy_forward(logits, targets, vocab,
                              Policy{old, advantages, of(ref), of(weights), of(denominator), low, high, kl_coef, temperature},
                              false, false);
    return {out.loss, out.logprobs, out.kl, out.clipped};
}

struct PreferenceResult {
    Tensor loss, rewards, logprobs, stats, coef;
};

PreferenceResult preference_forward(const Tensor& logits, const Tensor& targets, int64_t vocab, const Tensor& ref,
                                    const Tensor& offsets, double beta, double smoothing, bool average, bool needs) {
    const Rows r(logits, vocab);
    const int64_t sequences = ref.numel();
    PreferenceResult out;
    auto [logprobs, stats] = logprobs_of(r, targets, 1.0, needs);
    out.stats = stats;
    out.loss = floats({}, logits);
    out.rewards = floats({sequences}, logits);
    out.logprobs = floats({sequences}, logits);
    out.coef = floats({r.rows}, logits);
    const Tensor scratch = at::empty({sequences * 2}, logits.options().dtype(at::kDouble));
    double* sums = scratch.data_ptr<double>();
    c10::cuda::CUDAGuard guard(logits.device());
    check(gb_preference_loss(f32(logprobs), targets_of(targets), offsets.defined() ? targets_of(offsets) : nullptr, r.rows,
                             r.rows / sequences, (int)sequences, r.vocab, average, ref.data_ptr(),
                             ref.scalar_type() == at::kDouble, beta, smoothing, sums,
                             reinterpret_cast<float*>(sums + sequences), f32(out.loss), f32(out.rewards),
                             f32(out.logprobs), f32(out.coef), stream_of(logits)), "gb_preference_loss", 1);
    return out;
}

struct PreferenceLoss : Function<PreferenceLoss> {
    static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& targets, int64_t vocab,
                                 const Tensor& ref, const Maybe& offsets, double beta, double smoothing, bool average) {
        auto out = preference_forward(logits, targets, vocab, ref, of(offsets), beta, smoothing, average, true);
        ctx->save_for_backward({logits, targets, out.stats, out.coef});
        ctx->saved_data["vocab"] = vocab;
        ctx->mark_non_differentiable({out.rewards, out.logprobs});
        return {out.loss, out.rewards, out.logprobs};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto s = ctx->get_saved_variables();
        variable_list result(8);
        result[0] = logits_grad(s[0], ctx->saved_data["vocab"].toInt(), s[1], 1.0, s[2], s[3],
                                grads[0].to(at::kFloat).contiguous());
        return once(std::move(result));
    }
};

std::tuple<Tensor, Tensor, Tensor> preference_loss(const Tensor& logits, const Tensor& targets, int64_t vocab,
                                                   const Tensor& ref, const Maybe& offsets, double beta, double smoothing,
                                                   bool average) {
    if (at::GradMode::is_enabled() && logits.requires_grad()) {
        auto v = PreferenceLoss::apply(logits, targets, vocab, ref, offsets, beta, smoothing, average);
        return {v[0], v[1], v[2]};
    }
    at::NoGradGuard no_grad;
    auto out = preference_forward(logits, targets, vocab, ref, of(offsets), beta, smoothing, average, false);
    return {out.loss, out.rewards, out.logprobs};
}

// -- gradient norm -------------------------------------------------------------------------------------

// One launch's tensors: one type, at most as many as a launch carries.
struct Group {
    int code;
    std::vector<void*> ptrs;
    std::vector<long long> sizes;
    int count() const { return (int)ptrs.size(); }
};

std::vector<Group> groups_of(const std::vector<Tensor>& tensors) {
    static const size_t most = (size_t)gb_grad_norm_max_tensors();
    std::vector<Group> done, open(3);
    for (const Tensor& t : tensors) {
        const long long n = t.numel();
        if (!n) continue;
        const int code = code_of(t.scalar_type());
        Group& g = open[code];
        g.code = code;
        g.ptrs.push_back(t.data_ptr());
        g.sizes.push_back(n);
        if (g.ptrs.size() == most) {
            done.push_back(std::move(g));
            g = Group();
        }
    }
    for (Group& g : open) if (g.count()) done.push_back(std::move(g));
    return done;
}

// Whether the list is what the kernels take: floating tensors of one GPU, without gaps.
bool simple_grads(const std::vector<Tensor>& tensors) {
    if (tensors.empty()) return false;
    for (const Tensor& t : tensors) {
        if (!plain(t) || t.device() != tensors[0].device() || code_of(t.scalar_type()) < 0 || !t.is_non_overlapping_and_dense())
            return false;
    }
    return true;
}

// Two floats: the norm times |scale|, and the factor that clips it to max_norm.
Tensor norm_of(const std::vector<Tensor>& tensors, bool maximum, double scale, double max_norm) {
    const auto groups = groups_of(tensors);
    std::vector<int> counts;
    long long total = 0;
    for (const Group& g : groups) {
        counts.push_back(gb_grad_norm_parts(g.ptrs.data(), g.sizes.data(), g.count()));
        TORCH_CHECK_VALUE(counts.back() >= 0, "too many gradient values for one call");
        total += counts.back();
    }
    const Tensor part = at::empty({std::max<long long>(1, total)}, tensors[0].options().dtype(at::kDouble));
    Tensor result = floats({2}, tensors[0]);
    c10::cuda::CUDAGuard guard(result.device());
    const cudaStream_t stream = stream_of(result);
    double* at = part.data_ptr<double>();
    for (size_t i = 0; i < groups.size(); ++i) {
        const Group& g = groups[i];
        check(gb_grad_norm_partial(g.code, maximum, g.ptrs.data(), g.sizes.data(), g.count(), at, stream),
              "gb_grad_norm_partial", 1);
        at += counts[i];
    }
    check(gb_grad_norm_finish(maximum, part.data_ptr<double>(), (int)total, scale, max_norm, f32(result), stream),
          "gb_grad_norm_finish", 1);
    return result;
}

// None where Python has to look at the list.
std::optional<Tensor> grad_norm(const std::vector<Tensor>& tensors, bool maximum, double scale, double max_norm) {
    if (!simple_grads(tensors)) return std::nullopt;
    at::NoGradGuard no_grad;
    return norm_of(tensors, maximum, scale, max_norm);
}

Tensor grad_coef(const Tensor& norm, double max_norm) {
    Tensor result = floats({2}, norm);
    c10::cuda::CUDAGuard guard(norm.device());
    check(gb_grad_clip_coef(f32(norm), max_norm, f32(result), stream_of(norm)), "gb_grad_clip_coef", 1);
    return result;
}

// Every value of the tensors (without gaps, on one GPU) times result[1].
void grad_scale(const std::vector<Tensor>& tensors, const Tensor& result) {
    c10::cuda::CUDAGuard guard(result.device());
    for (const Group& g : groups_of(tensors))
        check(gb_grad_scale(g.code, g.ptrs.data(), g.sizes.data(), g.count(), f32(result) + 1, stream_of(result)),
              "gb_grad_scale", 1);
}

// Norm and clipped update in one call; returns the norm and its factor.
Tensor adamw_clipped(const Tensor& p, const Tensor& g, const Tensor& m, const Tensor& v, const Tensor& state, double lr,
                     double beta1, double beta2, double eps, double weight_decay, double scale, double max_norm,
                     bool zero_grad) {
    at::NoGradGuard no_grad;
    Tensor result = norm_of({g}, false, scale, max_norm);
    c10::cuda::CUDAGuard guard(p.device());
    check(gb_adamw_clipped(f32(p), f32(g), f32(m), f32(v), (size_t)p.numel(), state.data_ptr(), lr, beta1, beta2, eps,
                           weight_decay, (float)scale, f32(result) + 1, zero_grad, stream_of(p)), "gb_adamw_clipped", 1);
    return result;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.def("launches", [] { return g_launches.load(); });
    m.def("residual_norm", &residual_norm);
    m.def("token_logprobs", &token_logprobs);
    m.def("policy_loss", &policy_loss);
    m.def("preference_loss", &preference_loss);
    m.def("grad_norm", &grad_norm);
    m.def("grad_coef", &grad_coef);
    m.def("grad_scale", &grad_scale);
    m.def("adamw_clipped", &adamw_clipped);
}
