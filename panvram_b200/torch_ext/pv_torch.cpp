// pv_torch.cpp - the operators of a training step as torch sees them: argument checks, outputs from torch's allocator, and
// autograd nodes over the C entry points (include/panvram_b200.h pv_logprobs ... pv_clip_grads). panvram_b200/train.py is
// the public face and its documentation.
//
// The nodes are C++ because a Python backward pass costs a hand-over of the interpreter to autograd's own thread: the
// preference loss and its gradient over 4 windows of 512 take 115 us that way and 64 so, 11 of them on the device.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/extension.h>

#include <cmath>
#include <limits>

#include "panvram_b200.h"

namespace {

using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
using MaybeTensor = std::optional<Tensor>;

[[noreturn]] void failed(const char* what) { TORCH_CHECK(false, "panvram_b200 ", what, ": ", pv_kernels_last_error()); }
void* stream_of(const at::Device& d) { return (void*)at::cuda::getCurrentCUDAStream(d.index()).stream(); }

int type_of(at::ScalarType t) {
    return t == at::kBFloat16 ? PV_T_BF16 : t == at::kHalf ? PV_T_FP16 : t == at::kFloat ? PV_T_FP32 : -1;
}

// the kernels take a tensor's memory as it lies
void check_memory(const Tensor& t, const char* name) {
    TORCH_CHECK_VALUE(!t.is_neg() && !t._is_zerotensor(), name, ": a view whose negation torch has put off, or zeros without memory; pass t.clone()");
    TORCH_CHECK_VALUE(t.has_storage() && (t.numel() == 0 || t.storage().data() != nullptr), name,
                      ": a tensor without memory of its own (in a wrapper class, as sharded tensors are, or in a function transform such as vmap); "
                      "pass the tensor inside, a shard's local part");
}

void check_device(const Tensor& t, const char* what) {
    TORCH_CHECK(t.is_cuda(), "panvram_b200 runs on the GPU only: ", what, " on ", t.device());
    TORCH_CHECK(at::cuda::getDeviceProperties(t.get_device())->major >= 10, "panvram_b200 is built for sm_100a (B200); ",
                at::cuda::getDeviceProperties(t.get_device())->name, " is not one");
}

// where a batch's tensors lie (no mask: an undefined one)
void place(pv_scored& b, const Tensor& logits, const Tensor& tokens, const Tensor& mask) {
    b.logits = logits.data_ptr();
    b.logits_n = logits.stride(0); b.logits_w = logits.stride(1);
    b.tokens = tokens.data_ptr();
    b.tokens_n = tokens.stride(0); b.tokens_w = tokens.stride(1);
    if (!mask.defined()) return;
    b.mask = mask.data_ptr();
    b.mask_n = mask.stride(0); b.mask_w = mask.stride(1);
}

// the arguments that all operators over logits share, checked -> pv_scored without a gradient
pv_scored batch_of(const Tensor& logits, const Tensor& tokens, const MaybeTensor& mask, int64_t shift, std::optional<int64_t> ignore) {
    TORCH_CHECK_VALUE(logits.dim() == 3 && logits.layout() == at::kStrided && type_of(logits.scalar_type()) >= 0,
                      "logits: a bf16, fp16 or fp32 tensor [n, W, V]");
    const int64_t n = logits.size(0), W = logits.size(1), V = logits.size(2);
    TORCH_CHECK_VALUE(V >= 1 && (V == 1 || logits.stride(2) == 1), "logits: at least one word, and a position's words contiguous");
    TORCH_CHECK_VALUE(W < (int64_t(1) << 31) && V < (int64_t(1) << 30), "logits: W below 2^31 and V below 2^30");
    TORCH_CHECK_VALUE(n <= (int64_t(1) << 56) / std::max<int64_t>(W, 1), "logits: n W up to 2^56");
    const bool ids = tokens.scalar_type() == at::kLong;
    TORCH_CHECK_VALUE(tokens.dim() == 2 && tokens.size(0) == n && tokens.size(1) == W && tokens.layout() == at::kStrided &&
                          (ids || tokens.scalar_type() == at::kByte),
                      "tokens: a uint8 or int64 tensor [n, W]");
    if (mask)
        TORCH_CHECK_VALUE(mask->dim() == 2 && mask->size(0) == n && mask->size(1) == W && mask->layout() == at::kStrided &&
                              (mask->scalar_type() == at::kBool || mask->scalar_type() == at::kByte || mask->scalar_type() == at::kFloat),
                          "mask: a bool, uint8 or float32 tensor [n, W]");
    TORCH_CHECK_VALUE(shift >= 0 && shift < (int64_t(1) << 31), "shift: 0 or more");
    TORCH_CHECK(!logits._fw_grad(0).defined(), "panvram_b200: no forward-mode derivative");
    check_memory(logits, "logits");
    check_memory(tokens, "tokens");
    if (mask) check_memory(*mask, "mask");
    check_device(logits, "logits");
    TORCH_CHECK_VALUE(tokens.device() == logits.device(), "tokens: on ", tokens.device(), ", the logits on ", logits.device());
    if (mask) TORCH_CHECK_VALUE(mask->device() == logits.device(), "mask: on ", mask->device(), ", the logits on ", logits.device());
    pv_scored b = {};
    b.n = n; b.W = W; b.V = V;
    place(b, logits, tokens, mask ? *mask : Tensor());
    if (mask) b.mask_bytes = (int32_t)mask->element_size();
    b.ignore = ignore ? *ignore : ids ? -100 : 4;
    b.shift = (int32_t)shift;
    b.type = type_of(logits.scalar_type());
    b.token_bytes = ids ? 8 : 1;
    return b;
}

// a float32 tensor [n] or [n, W] (each allowed or not) on the logits' device
void check_floats(const Tensor& t, const char* name, const pv_scored& b, const Tensor& logits, bool one, bool each) {
    const bool shape = (one && t.dim() == 1 && t.size(0) == b.n) || (each && t.dim() == 2 && t.size(0) == b.n && t.size(1) == b.W);
    TORCH_CHECK_VALUE(shape && t.scalar_type() == at::kFloat && t.layout() == at::kStrided, name, ": a float32 tensor ", one ? "[n]" : "",
                      one && each ? " or " : "", each ? "[n, W]" : "");
    TORCH_CHECK_VALUE(t.device() == logits.device(), name, ": on ", t.device(), ", the logits on ", logits.device());
    check_memory(t, name);
}
float number(double v, const char* name, double low, double high = std::numeric_limits<double>::infinity()) {
    const bool ok = v >= low && v <= high && std::isfinite((float)v);
    if (std::isinf(high)) TORCH_CHECK_VALUE(ok, name, ": finite (in 32 bits), ", low, " or more");
    TORCH_CHECK_VALUE(ok, name, ": from ", low, " to ", high);
    return (float)v;
}

// `more` bytes (rounded up to 16) and behind them the scratch of a batch
struct Buffer {
    Tensor t;
    size_t more = 0, need = 0;
    Buffer() = default;
    Buffer(const pv_scored& b, const Tensor& like, size_t more_) : more((more_ + 15) / 16 * 16), need(pv_score_work_bytes(&b)) {
        t = at::empty({(int64_t)(more + need)}, like.options().dtype(at::kByte).requires_grad(false));
    }
    char* front() const { return (char*)t.data_ptr(); }
    void* work() const { return front() + more; }
};

bool wants_grad(const Tensor& logits) { return at::GradMode::is_enabled() && logits.requires_grad(); }
Tensor scalar_like(const Tensor& logits) { return at::empty({}, logits.options().dtype(at::kFloat).requires_grad(false)); }
// a new gradient of the logits, entered in b
Tensor grad_into(pv_scored& b, const Tensor& logits) {
    Tensor g = at::empty(logits.sizes(), logits.options().requires_grad(false));
    b.grad = g.data_ptr();
    b.grad_n = g.stride(0);
    b.grad_w = g.stride(1);
    return g;
}

// What the backward passes have in common: the batch, whose tensors autograd keeps (and refuses when one was changed in place
// meanwhile), and a gradient that may be used but not differentiated.
struct BatchNode : Node {
    SavedVariable logits, tokens, mask;
    pv_scored b;
    Buffer buf;              // what the forward pass leaves: the rows' statistics (`stat` bytes) and what the node puts behind them
    size_t stat = 0;
    c10::Device device = c10::Device(c10::kCUDA, 0);
    void keep(const Tensor& l, const Tensor& t, const MaybeTensor& m, const pv_scored& batch) {
        logits = SavedVariable(l, false);
        tokens = SavedVariable(t, false);
        if (m) mask = SavedVariable(*m, false);
        b = batch;
        device = l.device();
        set_next_edges(torch::autograd::collect_next_edges(l));
    }
    // a saved tensor; hooks on saved tensors (offloading to the host, checkpoints) may bring it back at another address and
    // laid out otherwise, so what the forward pass noted of either is not used again
    Tensor back(SavedVariable& s) {
        Tensor t = s.unpack();
        TORCH_CHECK(!t.defined() || t.device() == device, "panvram_b200: a saved tensor came back on ", t.device(), ", it was on ", device);
        return t;
    }
    variable_list apply(variable_list&& ups) override {
        std::lock_guard<std::mutex> lock(mutex_);
        const Tensor saved = back(logits), t = back(tokens), m = back(mask);
        Tensor l = saved, up = ups[0], g;
        if (!up.defined()) return {Tensor()};
        {
            at::AutoGradMode off(false);
            const c10::cuda::CUDAGuard guard(device);
            TORCH_CHECK(l.sizes() == at::IntArrayRef({b.n, b.W, b.V}) && type_of(l.scalar_type()) == b.type && t.sizes() == at::IntArrayRef({b.n, b.W}) &&
                            (int)t.element_size() == b.token_bytes && (!m.defined() || (m.sizes() == t.sizes() && (int)m.element_size() == b.mask_bytes)),
                        "panvram_b200: a saved tensor came back with another shape or type");
            if (b.V > 1 && l.stride(2) != 1) l = l.contiguous();
            pv_scored now = b;
            place(now, l, t, m);
            // torch may have put a negation or the zeros themselves off
            up = up._is_zerotensor() ? at::zeros(up.sizes(), l.options().dtype(at::kFloat)) : up.resolve_neg();
            g = grad(now, l, t, up);
        }
        if (at::GradMode::is_enabled())
            torch::autograd::set_history(g, std::make_shared<torch::autograd::Error>("panvram_b200: no second derivative",
                                                                                     torch::autograd::collect_next_edges(saved)));
        return {g};
    }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        logits.reset_data();
        tokens.reset_data();
        mask.reset_data();
        let_go();
    }
    virtual Tensor grad(pv_scored& b, const Tensor& l, const Tensor& t, const Tensor& up) = 0;
    virtual void let_go() { buf = Buffer(); }
    // the gradient of logits whose log-probabilities have the derivative `up`, times *scale
    Tensor from_logprobs(pv_scored& b, const Tensor& l, const float* up, int64_t up_n, int64_t up_w, const float* scale, const char* what) {
        Tensor g = grad_into(b, l), again, logp;
        const char* rows = stat ? buf.front() : nullptr;
        const size_t need = pv_score_stat_bytes(&b);
        if (need && !stat) {                        // rows that came back astride one more 16-byte piece, enough to need statistics
            again = at::empty({(int64_t)need}, l.options().dtype(at::kByte));
            logp = at::empty({b.n, b.W}, l.options().dtype(at::kFloat));
            rows = (const char*)again.data_ptr();
            if (pv_logprobs(&b, logp.data_ptr<float>(), nullptr, again.data_ptr(), nullptr, 0, stream_of(device))) failed(what);
        }
        if (pv_logprobs_grad(&b, up, up_n, up_w, rows, scale, stream_of(device))) failed(what);
        return g;
    }
};
template <typename N> std::shared_ptr<N> node() { return std::shared_ptr<N>(new N(), torch::autograd::deleteNode); }

// ---------------------------------------------------------------- log-probabilities
struct LogProbs : BatchNode {
    std::string name() const override { return "panvram_b200::LogProbs"; }
    Tensor grad(pv_scored& b, const Tensor& l, const Tensor&, const Tensor& up) override {
        return from_logprobs(b, l, up.data_ptr<float>(), up.stride(0), up.dim() == 2 ? up.stride(1) : 0, nullptr, "log-probabilities' gradient");
    }
};

Tensor window_logprobs(const Tensor& logits, const Tensor& tokens, const MaybeTensor& mask, int64_t shift, std::optional<int64_t> ignore, bool window) {
    const pv_scored b = batch_of(logits, tokens, mask, shift, ignore);
    const c10::cuda::CUDAGuard guard(logits.device());
    const bool keep = wants_grad(logits);
    Tensor out = at::empty(window ? at::IntArrayRef({b.n}) : at::IntArrayRef({b.n, b.W}), logits.options().dtype(at::kFloat).requires_grad(false));
    const size_t stat = keep ? pv_score_stat_bytes(&b) : 0;
    Buffer buf;
    if (window || stat) buf = Buffer(b, logits, stat);
    if (pv_logprobs(&b, window ? nullptr : out.data_ptr<float>(), window ? out.data_ptr<float>() : nullptr, stat ? buf.front() : nullptr,
                    buf.need ? buf.work() : nullptr, buf.need, stream_of(logits.device())))
        failed("log-probabilities");
    if (keep) {
        auto fn = node<LogProbs>();
        fn->keep(logits, tokens, mask, b);
        if (stat) fn->buf = buf;
        fn->stat = stat;
        torch::autograd::set_history(out, fn);
    }
    return out;
}

// ---------------------------------------------------------------- preference
struct Preference : BatchNode {      // buf: the rows' statistics, each window's derivative
    std::string name() const override { return "panvram_b200::PreferenceLoss"; }
    Tensor grad(pv_scored& b, const Tensor& l, const Tensor&, const Tensor& up) override {
        return from_logprobs(b, l, (const float*)(buf.front() + stat), 1, 0, up.data_ptr<float>(), "preference loss's gradient");
    }
};

std::pair<Tensor, MaybeTensor> preference_loss(const Tensor& logits, const Tensor& tokens, const Tensor& ref, double beta, double smoothing,
                                               const MaybeTensor& mask, int64_t shift, std::optional<int64_t> ignore, bool margins) {
    const float be = number(beta, "beta", 0.0), sm = number(smoothing, "label_smoothing", 0.0, 1.0);
    const pv_scored b = batch_of(logits, tokens, mask, shift, ignore);
    TORCH_CHECK_VALUE(b.n % 2 == 0, "logits: an even number of windows, the preferred ones first");
    check_floats(ref, "ref_logp", b, logits, true, false);
    const c10::cuda::CUDAGuard guard(logits.device());
    const bool keep = wants_grad(logits);
    Tensor loss = scalar_like(logits);
    MaybeTensor m;
    if (margins) m = at::empty({b.n / 2}, loss.options());
    const size_t stat = keep ? pv_score_stat_bytes(&b) : 0;
    const Buffer buf(b, logits, stat + 4 * b.n);
    if (pv_preference(&b, ref.data_ptr<float>(), ref.stride(0), be, sm, loss.data_ptr<float>(), m ? m->data_ptr<float>() : nullptr,
                      (float*)(buf.front() + stat), stat ? buf.front() : nullptr, buf.work(), buf.need, stream_of(logits.device())))
        failed("preference loss");
    if (keep) {
        auto fn = node<Preference>();
        fn->keep(logits, tokens, mask, b);
        fn->buf = buf;
        fn->stat = stat;
        torch::autograd::set_history(loss, fn);
    }
    return {loss, m};
}

// ---------------------------------------------------------------- policy
void place_policy(pv_policy_args& a, const Tensor& old, const Tensor& adv, const Tensor& ref) {
    a.old = old.data_ptr<float>();
    a.old_n = old.stride(0); a.old_w = old.stride(1);
    a.adv = adv.data_ptr<float>();
    a.adv_n = adv.stride(0); a.adv_w = adv.dim() == 2 ? adv.stride(1) : 0;
    if (!ref.defined()) return;
    a.ref = ref.data_ptr<float>();
    a.ref_n = ref.stride(0); a.ref_w = ref.stride(1);
}

// A position's weight is known from the tokens alone, so the loss's pass over the logits forms their gradient too and the
// logits are read once: backward finds it made where its upstream gradient is 1, and forms it again where it is not (found
// out on the device, without a wait). Half-precision logits come with a loss scale that keeps their gradient in range, so
// theirs is left to backward.
struct Policy : BatchNode {          // buf: the windows' weights, the loss's scratch again: it is done with, and long rows need some
    SavedVariable old, adv, ref;
    pv_policy_args a;
    Tensor made;                     // the gradient, until it is handed out
    std::string name() const override { return "panvram_b200::PolicyLoss"; }
    void let_go() override {
        old.reset_data();
        adv.reset_data();
        ref.reset_data();
        buf = Buffer();
        made = Tensor();
    }
    Tensor grad(pv_scored& b, const Tensor& l, const Tensor& t, const Tensor& up) override {
        const Tensor o = back(old), v = back(adv), r = back(ref);
        TORCH_CHECK(o.sizes() == t.sizes() && v.dim() == adv_dim && v.size(0) == b.n && v.size(-1) == (adv_dim == 2 ? b.W : b.n) &&
                        (!r.defined() || r.sizes() == t.sizes()) && o.scalar_type() == at::kFloat && v.scalar_type() == at::kFloat &&
                        (!r.defined() || r.scalar_type() == at::kFloat),
                    "panvram_b200: a saved tensor came back with another shape or type");
        pv_policy_args now = a;
        place_policy(now, o, v, r);
        Tensor g = std::move(made), scratch;
        made = Tensor();
        const bool skip = g.defined();
        if (skip) {
            b.grad = g.data_ptr();
            b.grad_n = g.stride(0);
            b.grad_w = g.stride(1);
        } else {
            g = grad_into(b, l);
        }
        void* work = buf.work();
        const size_t need = pv_score_work_bytes(&b);
        if (need > buf.need) {                      // rows that came back astride one more 16-byte piece
            scratch = at::empty({(int64_t)need}, l.options().dtype(at::kByte));
            work = scratch.data_ptr();
        }
        if (pv_policy_grad(&b, &now, (const double*)buf.front(), up.data_ptr<float>(), skip, work, need, stream_of(device)))
            failed("policy loss's gradient");
        return g;
    }
    int64_t adv_dim = 1;
};

Tensor policy_loss(const Tensor& logits, const Tensor& tokens, const Tensor& old, const Tensor& adv, const MaybeTensor& ref, double low, double high,
                   double kl, const MaybeTensor& mask, int64_t shift, std::optional<int64_t> ignore, bool by_window, double scale) {
    pv_policy_args a = {};
    a.clip_low = number(low, "clip", 0.0);
    a.clip_high = number(high, "clip", 0.0);
    a.kl = number(kl, "kl", 0.0);
    a.scale = number(scale, "scale", 0.0);
    a.by_window = by_window;
    TORCH_CHECK_VALUE(a.kl == 0.f || ref, "kl: a KL term needs ref_logp");
    const pv_scored b = batch_of(logits, tokens, mask, shift, ignore);
    check_floats(old, "old_logp", b, logits, false, true);
    check_floats(adv, "advantages", b, logits, true, true);
    const bool kl_term = a.kl != 0.f;
    if (kl_term) check_floats(*ref, "ref_logp", b, logits, false, true);
    place_policy(a, old, adv, kl_term ? *ref : Tensor());
    const c10::cuda::CUDAGuard guard(logits.device());
    const bool keep = wants_grad(logits);
    Tensor loss = scalar_like(logits), made;
    const Buffer buf(b, logits, 8 * b.n);
    pv_scored run = b;
    if (keep && b.type != PV_T_FP16) made = grad_into(run, logits);
    if (pv_policy(&run, &a, loss.data_ptr<float>(), (double*)buf.front(), buf.work(), buf.need, stream_of(logits.device()))) failed("policy loss");
    if (keep) {
        auto fn = node<Policy>();
        fn->keep(logits, tokens, mask, b);
        fn->a = a;
        fn->old = SavedVariable(old.detach(), false);
        fn->adv = SavedVariable(adv.detach(), false);
        fn->adv_dim = adv.dim();
        if (kl_term) fn->ref = SavedVariable(ref->detach(), false);
        fn->buf = buf;
        fn->made = made;
        torch::autograd::set_history(loss, fn);
    }
    return loss;
}

// ---------------------------------------------------------------- gradients
struct List {
    std::vector<uint64_t> ptr;
    std::vector<int64_t> numel;
    std::vector<uint8_t> type;
    pv_tensors g;
    List(const std::vector<Tensor>& ts, const char* name) {
        TORCH_CHECK_VALUE(!ts.empty(), name, ": no tensors");
        ptr.reserve(ts.size());
        numel.reserve(ts.size());
        type.reserve(ts.size());
        for (const Tensor& t : ts) {
            TORCH_CHECK_VALUE(t.defined() && t.layout() == at::kStrided && type_of(t.scalar_type()) >= 0, name, ": bf16, fp16 or fp32 tensors");
            TORCH_CHECK_VALUE(t.is_contiguous() || t.is_non_overlapping_and_dense(), name, ": tensors that are dense in memory (no gaps, no expanded dimensions)");
            TORCH_CHECK_VALUE(t.device() == ts[0].device(), name, ": on one device");
            check_memory(t, name);
            ptr.push_back((uint64_t)t.data_ptr());
            numel.push_back(t.numel());
            type.push_back((uint8_t)type_of(t.scalar_type()));
        }
        g = {ptr.data(), numel.data(), type.data(), (int64_t)ts.size()};
    }
};

Tensor grad_norm(const std::vector<Tensor>& grads) {
    const List l(grads, "grads");
    check_device(grads[0], "gradients");
    const c10::cuda::CUDAGuard guard(grads[0].device());
    const auto options = at::TensorOptions().device(grads[0].device());
    Tensor norm = at::empty({}, options.dtype(at::kFloat)), work = at::empty({(int64_t)pv_grads_work_bytes(&l.g)}, options.dtype(at::kByte));
    if (pv_grad_norm(&l.g, norm.data_ptr<float>(), work.data_ptr(), work.numel(), stream_of(grads[0].device()))) failed("gradient norm");
    return norm;
}

Tensor clip_grads(const std::vector<Tensor>& grads, double max_norm, const std::optional<std::vector<Tensor>>& out) {
    TORCH_CHECK_VALUE(max_norm >= 0 && std::isinf(max_norm) == std::isinf((float)max_norm), "max_norm: 0 or more, in float32's range or infinity");
    const List l(grads, "grads");
    std::optional<List> o;
    if (out) {
        o.emplace(*out, "out");
        TORCH_CHECK_VALUE(out->size() == grads.size(), "out: one tensor per gradient, of its size and laid out alike");
        for (size_t i = 0; i < grads.size(); i++) {
            const Tensor &a = grads[i], &b = (*out)[i];
            const bool alike = a.is_contiguous() && b.is_contiguous() ? a.numel() == b.numel() : a.sizes() == b.sizes() && a.strides() == b.strides();
            TORCH_CHECK_VALUE(alike, "out: one tensor per gradient, of its size and laid out alike");
            TORCH_CHECK_VALUE(l.type[i] == o->type[i] || o->type[i] == PV_T_FP32, "out: of the gradient's type, or float32");
        }
        TORCH_CHECK_VALUE((*out)[0].device() == grads[0].device(), "out: on the gradients' device");
    }
    const std::vector<Tensor>& written = out ? *out : grads;
    for (const Tensor& t : written)
        TORCH_CHECK_VALUE(!t.requires_grad(), "clip_grads: pass gradients (p.grad), not parameters, and none that autograd has a graph for");
    check_device(grads[0], "gradients");
    const c10::cuda::CUDAGuard guard(grads[0].device());
    const auto options = at::TensorOptions().device(grads[0].device());
    Tensor norm = at::empty({}, options.dtype(at::kFloat)), work = at::empty({(int64_t)pv_grads_work_bytes(&l.g)}, options.dtype(at::kByte));
    const int code = pv_clip_grads(&l.g, o ? &o->g : nullptr, (float)max_norm, norm.data_ptr<float>(), work.data_ptr(), work.numel(),
                                   stream_of(grads[0].device()));
    TORCH_CHECK_VALUE(code != PV_EARG, pv_kernels_last_error());
    if (code) failed("gradient clipping");
    for (const Tensor& t : written)
        if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();      // written behind autograd's back: saved ones are refused
    return norm;
}

}  // namespace

PYBIND11_MODULE(_train, m) {
    // without the interpreter's lock; an exception of Python's own (a hook's on saved tensors) goes back as it is
    m.def("window_logprobs", torch::wrap_pybind_function_no_gil(&window_logprobs));
    m.def("preference_loss", torch::wrap_pybind_function_no_gil(&preference_loss));
    m.def("policy_loss", torch::wrap_pybind_function_no_gil(&policy_loss));
    m.def("grad_norm", torch::wrap_pybind_function_no_gil(&grad_norm));
    m.def("clip_grads", torch::wrap_pybind_function_no_gil(&clip_grads));
}
