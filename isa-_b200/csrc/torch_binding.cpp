// torch_binding.cpp — tensors in, C ABI calls out: the digital operators' entry
// points for Python (layer norm with its autograd node, orthogonalisation, the Muon
// step).  In C++ because these calls are short: a forward and backward of a small
// layer norm took 150 us through a Python autograd Function, most of it in the
// interpreter.  The library's entry points are handed over by address (bind), so
// this module works with whichever build of the library is loaded.

#include <ATen/cuda/CUDAEvent.h>
#include <c10/core/AutogradState.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <algorithm>
#include <array>
#include <climits>
#include <cmath>
#include <map>
#include <tuple>
#include <vector>

#include "cimekv.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

struct Library {
    decltype(&cimekv_last_error) last_error = nullptr;
    decltype(&cimekv_layer_norm_forward) norm_forward = nullptr;
    decltype(&cimekv_layer_norm_backward) norm_backward = nullptr;
    decltype(&cimekv_layer_norm_workspace_bytes) norm_workspace = nullptr;
    decltype(&cimekv_orthogonalize) orthogonalize = nullptr;
    decltype(&cimekv_orthogonalize_workspace_bytes) orthogonalize_workspace = nullptr;
    decltype(&cimekv_muon_shares) muon_shares = nullptr;
    decltype(&cimekv_muon_step_weighted) muon_step = nullptr;
} lib;

void bind(const std::map<std::string, uintptr_t>& at) {
    const auto get = [&](auto& fn, const char* name) { fn = reinterpret_cast<std::decay_t<decltype(fn)>>(at.at(name)); };
    get(lib.last_error, "cimekv_last_error");
    get(lib.norm_forward, "cimekv_layer_norm_forward");
    get(lib.norm_backward, "cimekv_layer_norm_backward");
    get(lib.norm_workspace, "cimekv_layer_norm_workspace_bytes");
    get(lib.orthogonalize, "cimekv_orthogonalize");
    get(lib.orthogonalize_workspace, "cimekv_orthogonalize_workspace_bytes");
    get(lib.muon_shares, "cimekv_muon_shares");
    get(lib.muon_step, "cimekv_muon_step_weighted");
}

// A number of steps as the library's int; one that does not fit is none that it takes.
int steps_of(int64_t steps) { return (int)std::clamp<int64_t>(steps, -1, INT_MAX); }

void check(int rc, const char* what) { TORCH_CHECK(rc == 0, what, " failed (status ", rc, "): ", lib.last_error()); }

bool available(at::ScalarType t) { return t == at::kFloat || t == at::kBFloat16 || t == at::kHalf; }
int code(at::ScalarType t) { return t == at::kFloat ? CIMEKV_F32 : t == at::kBFloat16 ? CIMEKV_BF16 : CIMEKV_F16; }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// The kernels get addresses, so whatever follows a call by its tensors alone sees only the outputs'
// allocation.  A trace would hand out memory that nothing writes.
void check_not_traced(const char* what) {
    TORCH_CHECK(!torch::jit::tracer::isTracing() &&
                    !c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY),
                what, " cannot be traced: a trace would miss its kernels");
}
// A forward-mode tangent would be lost, and read as zero; a subclass that carries its values itself has no
// memory of its own to hand over.
void check_plain(const Tensor& t, const char* name, const char* what) {
    TORCH_CHECK(!t._fw_grad(0).defined() || !c10::AutogradState::get_tls_state().get_fw_grad_mode(), name,
                " has a forward-mode tangent: ", what, " has no forward-mode derivative");
    TORCH_CHECK(!t.unsafeGetTensorImpl()->is_python_dispatch(), name, " is a tensor subclass with its own dispatch: ", what,
                " takes plain tensors");
}

// The values that memory holds for a tensor: a view with its negative bit set is written out.
Tensor values(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }

void* stream() { return c10::cuda::getCurrentCUDAStream().stream(); }

// ------------------------------------------------------------- layer norm ---

// A tensor as rows of contiguous elements, and their stride.
struct Rows {
    Tensor t;
    int64_t stride;
};
Rows rows_of(const Tensor& view, int64_t cols) {
    const Tensor t = values(view);
    if (t.is_contiguous()) return {t, cols};
    Tensor r = t.dim() == 2 ? t : t.reshape({-1, cols});
    if (cols > 1 && r.stride(1) != 1) r = r.contiguous();
    return {r, r.size(0) > 1 ? r.stride(0) : cols};
}

void check_norm(const Tensor& x, const OptTensor& delta, const OptTensor& weight, const OptTensor& bias, double eps,
                at::ScalarType out) {
    check_not_traced("layer norm");
    check_plain(x, "x", "layer norm");
    if (delta) check_plain(*delta, "delta", "layer norm");
    if (weight) check_plain(*weight, "weight", "layer norm");
    if (bias) check_plain(*bias, "bias", "layer norm");
    TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor: the layer norm kernels have no CPU implementation");
    TORCH_CHECK(x.dim() >= 1, "x must have at least one axis");
    TORCH_CHECK(available(x.scalar_type()), "x must be float32, bfloat16 or float16, got ", x.scalar_type());
    const int64_t cols = x.size(-1);
    TORCH_CHECK(cols >= 1 && cols <= CIMEKV_LAYER_NORM_MAX_COLS, "layer norm takes 1 to ", CIMEKV_LAYER_NORM_MAX_COLS,
                " columns, got ", cols);
    TORCH_CHECK(eps >= 0.0, "eps must be >= 0, got ", eps);
    TORCH_CHECK(available(out) && (x.scalar_type() == at::kFloat || out == x.scalar_type() || out == at::kFloat), "out_dtype ",
                out, " is not available for ", x.scalar_type(), " inputs");
    const auto check_columns = [&](const OptTensor& t, const char* name) {
        if (!t) return;
        TORCH_CHECK(t->device() == x.device(), name, " must be on the device of x");
        TORCH_CHECK(available(t->scalar_type()), name, " must be float32, bfloat16 or float16, got ", t->scalar_type());
        TORCH_CHECK(t->dim() == 1 && t->size(0) == cols, name, " must have shape (", cols, ",), got ", t->sizes());
    };
    check_columns(weight, "weight");
    check_columns(bias, "bias");
    TORCH_CHECK(!weight || !bias || weight->scalar_type() == bias->scalar_type(), "weight and bias must have one type");
    if (delta) {
        TORCH_CHECK(delta->device() == x.device(), "delta must be on the device of x");
        TORCH_CHECK(delta->sizes() == x.sizes(), "delta must have the shape of x: ", delta->sizes(), ", ", x.sizes());
        TORCH_CHECK(available(delta->scalar_type()) &&
                        (x.scalar_type() == at::kFloat || delta->scalar_type() == x.scalar_type()),
                    "delta ", delta->scalar_type(), " is not available for ", x.scalar_type(), " streams");
    }
}

struct Normed {
    Tensor y, h, stats, weight;
};

// stats: mean and rstd [2][rows], kept for a backward.
Normed norm_forward(const Tensor& x, const OptTensor& delta, const OptTensor& weight, const OptTensor& bias, double eps,
                    at::ScalarType out, bool keep) {
    const c10::cuda::CUDAGuard guard(x.device());
    const int64_t cols = x.size(-1), rows = x.numel() / cols;
    const Rows x2 = rows_of(x, cols);
    const Rows d2 = delta ? rows_of(*delta, cols) : Rows{Tensor(), 0};
    Normed r;
    r.weight = weight ? values(*weight).contiguous() : Tensor();
    const Tensor b = bias ? values(*bias).contiguous() : Tensor();
    r.y = at::empty(x.sizes(), x.options().dtype(out));
    if (delta) r.h = at::empty(x.sizes(), x.options());
    if (keep) r.stats = at::empty({2, rows}, x.options().dtype(at::kFloat));
    float* mean = keep ? r.stats.data_ptr<float>() : nullptr;
    const Tensor& affine = weight ? r.weight : b;
    check(lib.norm_forward(x2.t.data_ptr(), code(x.scalar_type()), x2.stride, ptr(d2.t),
                           delta ? code(delta->scalar_type()) : 0, d2.stride, ptr(r.weight), ptr(b),
                           affine.defined() ? code(affine.scalar_type()) : 0, rows, (int)cols, (float)eps, ptr(r.h),
                           r.y.data_ptr(), code(out), mean, mean ? mean + rows : nullptr, stream()),
          "cimekv_layer_norm_forward");
    return r;
}

// Bits of the saved word: which gradients are wanted, types of branch and weights.
constexpr int64_t kNeedX = 1, kNeedDelta = 2, kNeedWeight = 4, kNeedBias = 8;

class NormNode : public torch::autograd::Function<NormNode> {
public:
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptTensor& delta, const OptTensor& weight,
                                 const OptTensor& bias, double eps, int64_t out) {
        const Normed r = norm_forward(x, delta, weight, bias, eps, (at::ScalarType)out, true);
        ctx->save_for_backward({delta ? r.h : x, r.weight, r.stats});
        const auto wants = [](const OptTensor& t, int64_t bit) { return t && t->requires_grad() ? bit : 0; };
        const at::ScalarType w = weight ? weight->scalar_type() : bias ? bias->scalar_type() : at::kFloat;
        ctx->saved_data["call"] = wants(x, kNeedX) | wants(delta, kNeedDelta) | wants(weight, kNeedWeight) |
                                  wants(bias, kNeedBias) | (int64_t)w << 8 |
                                  (int64_t)(delta ? delta->scalar_type() : x.scalar_type()) << 16;
        ctx->set_materialize_grads(false);
        if (!delta) return {r.y};
        return {r.y, r.h};
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        check_capture();
        variable_list out(6);
        const Tensor dy = grads[0], dh = grads.size() > 1 ? grads[1] : Tensor();
        if (!dy.defined() && !dh.defined()) return out;
        {
            const at::NoGradGuard no_grad;
            run(ctx, dy, dh, out);
        }
        if (at::GradMode::is_enabled()) {  // the gradients have no graph behind them: using one raises
            for (Tensor& g : out)
                if (g.defined()) g = g.detach().set_requires_grad(true);
            out = (*std::make_shared<torch::autograd::DelayedError>(
                "layer norm's backward cannot be differentiated again", (int64_t)out.size()))(std::move(out));
        }
        return out;
    }

private:
    // A captured backward that reaches leaves whose accumulators an eager graph has
    // made on the default stream would pull that stream into the capture, which
    // spoils the capture or ends the process.  Refused here while it is still an error.
    static void check_capture() {
        if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return;
        const auto* only = torch::autograd::get_current_graph_task_exec_info();  // autograd.grad(): what it needs
        const auto node = torch::autograd::get_current_node();
        if (!node) return;
        for (const auto& edge : node->next_edges()) {
            if (!edge.function || !dynamic_cast<torch::autograd::AccumulateGrad*>(edge.function.get())) continue;
            if (only && !only->empty()) {
                const auto it = only->find(edge.function.get());
                if (it == only->end() || !it->second.should_execute()) continue;
            }
            const auto made_on = edge.function->stream();
            TORCH_CHECK(!made_on || *made_on != c10::cuda::getDefaultCUDAStream(made_on->device_index()).unwrap(),
                        "this backward is being captured while an eager graph of the same parameters is alive (made on the "
                        "default stream): drop its outputs before the capture, or make it on a side stream");
        }
    }

    static void run(AutogradContext* ctx, const Tensor& dy, const Tensor& dh, variable_list& out) {
        const auto saved = ctx->get_saved_variables();
        const Tensor &src = saved[0], &weight = saved[1], &stats = saved[2];
        const int64_t call = ctx->saved_data["call"].toInt();
        const auto w_type = (at::ScalarType)(call >> 8 & 255), d_type = (at::ScalarType)(call >> 16 & 255);
        const int64_t cols = src.size(-1), rows = src.numel() / cols;
        const c10::cuda::CUDAGuard guard(src.device());
        if (!dy.defined()) {  // only the sum was used
            if (call & kNeedX) out[0] = dh;
            if (call & kNeedDelta) out[1] = dh.to(d_type);
            if (call & kNeedWeight) out[2] = at::zeros({cols}, src.options().dtype(w_type));
            if (call & kNeedBias) out[3] = at::zeros({cols}, src.options().dtype(w_type));
            return;
        }
        const Rows g = rows_of(dy, cols), h = rows_of(src, cols);
        const Rows s = dh.defined() ? rows_of(dh, cols) : Rows{Tensor(), 0};
        // one gradient for both where stream and branch have one type
        const bool shared = (call & kNeedDelta) && d_type == src.scalar_type();
        Tensor dx, dd, dw, db, ws;
        if ((call & kNeedX) || shared) dx = at::empty(src.sizes(), src.options());
        if ((call & kNeedDelta) && !shared) dd = at::empty(src.sizes(), src.options().dtype(d_type));
        if (call & kNeedWeight) dw = at::empty({cols}, src.options().dtype(w_type));
        if (call & kNeedBias) db = at::empty({cols}, src.options().dtype(w_type));
        size_t ws_bytes = 0;
        if (dw.defined() || db.defined()) {
            ws_bytes = lib.norm_workspace(rows, (int)cols);
            ws = at::empty({(int64_t)ws_bytes}, src.options().dtype(at::kByte));
        }
        const float* mean = rows ? stats.data_ptr<float>() : nullptr;
        check(lib.norm_backward(g.t.data_ptr(), code(dy.scalar_type()), g.stride, ptr(s.t), s.stride, h.t.data_ptr(),
                                code(src.scalar_type()), h.stride, ptr(weight), code(w_type), mean,
                                mean ? mean + rows : nullptr, rows, (int)cols, ptr(dx), ptr(dd), code(d_type), ptr(dw),
                                ptr(db), ptr(ws), ws_bytes, stream()),
              "cimekv_layer_norm_backward");
        if (call & kNeedX) out[0] = dx;
        if (call & kNeedDelta) out[1] = shared ? dx : dd;
        out[2] = dw;
        out[3] = db;
    }
};

bool wants_grad(std::initializer_list<const OptTensor*> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const OptTensor* t : ts)
        if (*t && (*t)->requires_grad()) return true;
    return false;
}

Tensor layer_norm(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps,
                  std::optional<at::ScalarType> out_dtype) {
    const at::ScalarType out = out_dtype.value_or(x.scalar_type());
    check_norm(x, std::nullopt, weight, bias, eps, out);
    const OptTensor xo = x;
    if (!wants_grad({&xo, &weight, &bias})) return norm_forward(x, std::nullopt, weight, bias, eps, out, false).y;
    return NormNode::apply(x, OptTensor(), weight, bias, eps, (int64_t)out)[0];
}

std::tuple<Tensor, Tensor> add_layer_norm(const Tensor& x, const Tensor& delta, const OptTensor& weight,
                                          const OptTensor& bias, double eps, std::optional<at::ScalarType> out_dtype) {
    const at::ScalarType out = out_dtype.value_or(x.scalar_type());
    const OptTensor xo = x, d = delta;
    check_norm(x, d, weight, bias, eps, out);
    if (!wants_grad({&xo, &d, &weight, &bias})) {
        const Normed r = norm_forward(x, d, weight, bias, eps, out, false);
        return {r.y, r.h};
    }
    const variable_list r = NormNode::apply(x, d, weight, bias, eps, (int64_t)out);
    return {r[0], r[1]};
}

// ------------------------------------------------------------------ muon ----

void check_matrix(const Tensor& t, const char* name) {
    TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor: the Newton-Schulz kernels have no CPU implementation");
    TORCH_CHECK(available(t.scalar_type()), name, " must be float32, bfloat16 or float16, got ", t.scalar_type());
    TORCH_CHECK(t.dim() >= 2, name, " must have at least two axes, got shape ", t.sizes());
    TORCH_CHECK(t.size(-2) <= CIMEKV_ORTHOGONALIZE_MAX_SIDE && t.size(-1) <= CIMEKV_ORTHOGONALIZE_MAX_SIDE, name,
                " must have sides of at most ", CIMEKV_ORTHOGONALIZE_MAX_SIDE, ", got shape ", t.sizes());
}

// Matrices of one launch: at most `most`, and no more than `room` bytes of workspace hold (one matrix takes what it
// takes), in launches of about one size.  Matrices this large fill the chip by themselves: 16 of 4,096 x 4,096
// take 3,490 us each in one launch (4 GB of workspace) and 3,460 in two.
constexpr int64_t kRoom = 2ll << 30;
int64_t at_once(int64_t count, int64_t rows, int64_t cols, int64_t most, int64_t room = kRoom) {
    const int64_t one = std::max<int64_t>(1, (int64_t)lib.orthogonalize_workspace(1, (int)rows, (int)cols));
    const int64_t fit = std::clamp<int64_t>(room / one, 1, most), calls = (count + fit - 1) / fit;
    return (count + calls - 1) / calls;
}

Tensor workspace(const Tensor& like, int64_t bytes) { return at::empty({bytes}, like.options().dtype(at::kByte)); }

Tensor orthogonalize(const Tensor& g, int64_t steps, std::array<double, 3> c, double eps) {
    const at::NoGradGuard no_grad;
    check_not_traced("orthogonalize");
    check_plain(g, "g", "orthogonalize");
    check_matrix(g, "g");
    const int64_t rows = g.size(-2), cols = g.size(-1);
    Tensor out = at::empty(g.sizes(), g.options());
    if (g.numel() == 0) return out;
    Tensor g3 = values(g);
    if (g3.dim() != 3) g3 = g3.reshape({-1, rows, cols});
    if (cols > 1 && g3.stride(2) != 1) g3 = g3.contiguous();
    const int64_t batch = g3.size(0);
    TORCH_CHECK(batch <= 65535, "orthogonalize takes at most 65535 matrices, got ", batch);
    const c10::cuda::CUDAGuard guard(g.device());
    const int64_t each = at_once(batch, rows, cols, batch), size = g.element_size();
    const Tensor ws = workspace(g, (int64_t)lib.orthogonalize_workspace((int)each, (int)rows, (int)cols));
    for (int64_t i = 0; i < batch; i += each)
        check(lib.orthogonalize(static_cast<const char*>(g3.data_ptr()) + i * g3.stride(0) * size, code(g.scalar_type()),
                                g3.stride(0), g3.stride(1), (int)std::min(each, batch - i), (int)rows, (int)cols,
                                steps_of(steps), (float)c[0], (float)c[1], (float)c[2], (float)eps,
                                static_cast<char*>(out.data_ptr()) + i * rows * cols * size, ws.data_ptr(),
                                (size_t)ws.numel(), stream()),
              "cimekv_orthogonalize");
    return out;
}

struct Group {
    std::vector<void*> params;
    std::vector<const void*> grads;
    std::vector<float*> momenta;
};

// Streams beside the current one: they begin after what it has been given so far, and
// join() (or the end, if a launch failed) lets it wait for them.
class Beside {
public:
    explicit Beside(c10::DeviceIndex device) : main_(c10::cuda::getCurrentCUDAStream(device)) { begin_.record(main_); }
    ~Beside() {
        try {
            join();
        } catch (...) {
        }
    }
    // (the current stream itself if all of the pool's are taken)
    c10::cuda::CUDAStream next() {
        for (int i = 0; i < 32; ++i) {
            const auto s = c10::cuda::getStreamFromPool(false, main_.device_index());
            const auto theirs = capture_of(s);
            if (theirs && theirs != capture_of(main_)) continue;  // part of somebody else's capture
            begin_.block(s);
            sides_.push_back(s);
            return s;
        }
        return main_;
    }
    void join() {
        while (!sides_.empty()) {
            const auto s = sides_.back();
            sides_.pop_back();
            at::cuda::CUDAEvent end;
            end.record(s);
            end.block(main_);
        }
    }

private:
    // The capture that a stream is part of; 0: none.
    static unsigned long long capture_of(const c10::cuda::CUDAStream& s) {
        cudaStreamCaptureStatus status;
        unsigned long long id = 0;
        C10_CUDA_CHECK(cudaStreamGetCaptureInfo(s.stream(), &status, &id));
        return status == cudaStreamCaptureStatusNone ? 0 : id;
    }

    c10::cuda::CUDAStream main_;
    at::cuda::CUDAEvent begin_;
    std::vector<c10::cuda::CUDAStream> sides_;
};

void muon_step(const std::vector<Tensor>& params, const std::vector<Tensor>& grads, const std::vector<Tensor>& momenta,
               double lr, const OptTensor& lr_tensor, double momentum, bool nesterov, double weight_decay, int64_t steps,
               std::array<double, 3> c, double eps, bool match_rms) {
    const at::NoGradGuard no_grad;
    TORCH_CHECK(params.size() == grads.size() && params.size() == momenta.size(),
                "expected as many gradients and momenta as parameters, got ", params.size(), ", ", grads.size(), ", ",
                momenta.size());
    check_not_traced("the Muon step");
    using Key = std::tuple<int64_t, int64_t, at::ScalarType, at::ScalarType>;
    std::vector<std::pair<Key, Group>> groups;
    std::vector<Tensor> keep;  // contiguous copies of gradients, alive until the launches
    for (size_t i = 0; i < params.size(); ++i) {
        const Tensor &p = params[i], &m = momenta[i];
        Tensor g = grads[i];
        check_plain(p, "parameter", "the Muon step");
        check_plain(g, "gradient", "the Muon step");
        check_plain(m, "momentum", "the Muon step");
        check_matrix(p, "parameter");
        TORCH_CHECK(g.sizes() == p.sizes() && m.sizes() == p.sizes(), "shape mismatch: parameter ", p.sizes(), ", gradient ",
                    g.sizes(), ", momentum ", m.sizes());
        TORCH_CHECK(g.device() == p.device() && m.device() == p.device() && p.device() == params[0].device(),
                    "parameters, gradients and momenta must be on one device");
        TORCH_CHECK(available(g.scalar_type()), "gradient must be float32, bfloat16 or float16, got ", g.scalar_type());
        TORCH_CHECK(m.scalar_type() == at::kFloat, "momentum must be float32, got ", m.scalar_type());
        TORCH_CHECK(p.is_contiguous() && m.is_contiguous() && !p.is_neg() && !m.is_neg(),
                    "parameters and momenta are updated in place and must be contiguous, without a negative bit");
    }
    if (lr_tensor)
        TORCH_CHECK(lr_tensor->numel() == 1 && lr_tensor->scalar_type() == at::kFloat && !params.empty() &&
                        lr_tensor->device() == params[0].device(),
                    "lr must be a float or a one-element float32 tensor on the parameters' device");
    if (params.empty()) return;
    // What is written must be memory of its own, checked before anything is: a
    // refused call leaves every parameter as it was.
    struct Range {
        uintptr_t begin, end;
        bool written;
        bool operator<(const Range& o) const { return begin < o.begin; }
    };
    std::vector<Range> ranges;
    const auto add = [&](const Tensor& t, bool written) {
        if (t.numel() && (written || (t.is_contiguous() && !t.is_neg())))  // other gradients are copied first
            ranges.push_back({(uintptr_t)t.data_ptr(), (uintptr_t)t.data_ptr() + t.numel() * t.element_size(), written});
    };
    for (size_t i = 0; i < params.size(); ++i) {
        add(params[i], true);
        add(momenta[i], true);
        add(grads[i], false);
    }
    std::sort(ranges.begin(), ranges.end());
    uintptr_t written_to = 0, read_to = 0;  // ends of what was seen so far
    for (const Range& r : ranges) {
        TORCH_CHECK(r.begin >= written_to && (!r.written || r.begin >= read_to),
                    "parameters and momenta must not overlap each other or a gradient");
        (r.written ? written_to : read_to) = std::max(r.written ? written_to : read_to, r.end);
    }
    const c10::cuda::CUDAGuard guard(params[0].device());
    for (size_t i = 0; i < params.size(); ++i) {
        const Tensor &p = params[i], &m = momenta[i];
        if (p.numel() == 0) continue;
        Tensor g = grads[i];
        if (!g.is_contiguous() || g.is_neg()) keep.push_back(g = values(g).contiguous());
        const Key key{p.size(-2), p.size(-1), p.scalar_type(), g.scalar_type()};
        size_t k = 0;
        while (k < groups.size() && groups[k].first != key) ++k;
        if (k == groups.size()) groups.emplace_back(key, Group());
        Group& to = groups[k].second;
        const int64_t each = p.size(-2) * p.size(-1);
        for (int64_t at = 0; at < p.numel(); at += each) {
            to.params.push_back(static_cast<char*>(p.data_ptr()) + at * p.element_size());
            to.grads.push_back(static_cast<const char*>(g.data_ptr()) + at * g.element_size());
            to.momenta.push_back(m.data_ptr<float>() + at);
        }
    }
    struct Room {
        Tensor ws;
        int64_t each, bytes;  // matrices of a launch, and what these take
    };
    const auto step = [&](const std::pair<Key, Group>& of, const Room& room, int share, void* on) {
        const auto& [key, group] = of;
        const auto& [rows, cols, p_type, g_type] = key;
        const double scale = match_rms ? 0.2 * std::sqrt((double)std::max(rows, cols))
                                       : std::sqrt(std::max(1.0, (double)rows / (double)cols));
        const int64_t count = (int64_t)group.params.size();
        for (int64_t i = 0; i < count; i += room.each)
            check(lib.muon_step(share, (int)std::min(room.each, count - i), group.params.data() + i, group.grads.data() + i,
                                group.momenta.data() + i, code(p_type), code(g_type), (int)rows, (int)cols, (float)lr,
                                lr_tensor ? lr_tensor->data_ptr<float>() : nullptr, (float)momentum,
                                (float)(1.0 - momentum), nesterov, (float)weight_decay, (float)scale, steps_of(steps),
                                (float)c[0], (float)c[1], (float)c[2], (float)eps, room.ws.data_ptr(),
                                (size_t)room.ws.numel(), on),
                  "cimekv_muon_step");
    };
    const auto room = [&](const std::pair<Key, Group>& of, int64_t beside) {
        const int64_t rows = std::get<0>(of.first), cols = std::get<1>(of.first);
        const int64_t each = at_once((int64_t)of.second.params.size(), rows, cols, CIMEKV_MUON_MAX_MATRICES, kRoom / beside);
        return Room{Tensor(), each, (int64_t)lib.orthogonalize_workspace((int)each, (int)rows, (int)cols)};
    };
    // small matrices of several shapes run side by side, each on its share of the SMs
    std::vector<int> counts, rows, cols, shares(groups.size(), 0);
    if (groups.size() > 1) {
        for (const auto& [key, group] : groups) {
            counts.push_back((int)group.params.size());
            rows.push_back((int)std::get<0>(key));
            cols.push_back((int)std::get<1>(key));
        }
        check(lib.muon_shares((int)groups.size(), counts.data(), rows.data(), cols.data(), (float)c[2], 0, shares.data()),
              "cimekv_muon_shares");
    }
    // All memory is asked for before anything is written: a call that it fails leaves every parameter as it was.
    const int64_t apart = std::count(shares.begin(), shares.end(), 0), beside = (int64_t)groups.size() - apart;
    std::vector<Room> rooms;  // those side by side have one each, until the streams have joined
    Tensor shared;            // for the others, one after the other
    for (size_t k = 0; k < groups.size(); ++k) {
        rooms.push_back(room(groups[k], shares[k] ? beside : 1));
        Room& r = rooms.back();
        if (!shares[k] && r.bytes > (shared.defined() ? shared.numel() : 0)) {
            shared = Tensor();
            shared = workspace(params[0], r.bytes);
        }
        if (shares[k]) r.ws = workspace(params[0], r.bytes);
    }
    for (size_t k = 0; k < groups.size(); ++k) {
        if (shares[k]) continue;
        rooms[k].ws = shared;
        step(groups[k], rooms[k], 0, stream());
    }
    if (beside) {
        Beside sides(params[0].device().index());
        bool first = true;
        for (size_t k = 0; k < groups.size(); ++k) {
            if (!shares[k]) continue;
            void* on = first ? stream() : (void*)sides.next().stream();
            first = false;
            step(groups[k], rooms[k], shares[k], on);
        }
        sides.join();
    }
    // autograd must see that these were written
    for (const auto* list : {&params, &momenta})
        for (const Tensor& t : *list)
            if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.def("bind", &bind);
    m.def("layer_norm", &layer_norm);
    m.def("add_layer_norm", &add_layer_norm);
    m.def("orthogonalize", &orthogonalize);
    m.def("muon_step", &muon_step);
}
