// The operators of include/ntc_ops.h on torch tensors: checks of arguments, allocation of results and workspaces on the current
// stream, and the autograd nodes. In C++ because a call's cost is otherwise the interpreter's: a layer forward and backward 224 us of
// host work from Python nodes against the kernels' 60 to 100.
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <dlfcn.h>

#include <cmath>
#include <cstring>
#include <optional>
#include <vector>

#include "ntc_ops.h"

using at::Tensor;
using std::optional;
namespace py = pybind11;

namespace {

int type_of(const Tensor& t) { return t.scalar_type() == at::kFloat ? NTC_F32 : t.scalar_type() == at::kBFloat16 ? NTC_BF16 : t.scalar_type() == at::kHalf ? NTC_F16 : -1; }
int type_of(at::ScalarType t) { return t == at::kFloat ? NTC_F32 : t == at::kBFloat16 ? NTC_BF16 : t == at::kHalf ? NTC_F16 : -1; }

void on_gpu(const char* name, const Tensor& t) { TORCH_CHECK_VALUE(t.defined() && t.is_cuda(), name, " must be a tensor on the GPU"); }
void floats(const char* name, const Tensor& t) {
    on_gpu(name, t);
    TORCH_CHECK_VALUE(type_of(t) >= 0, name, " is ", t.scalar_type(), "; it can be float32, bfloat16, float16");
}

// Forward-mode derivatives are not there either: a tangent would be dropped without a word.
void no_tangent(const char* name, const Tensor& t) {
    TORCH_CHECK_VALUE(!c10::AutogradState::get_tls_state().get_fw_grad_mode() || !t._fw_grad(0).defined(), name, " has a tangent; there is no forward-mode derivative");
}

// One entry point on a device's current stream: a refusal is a ValueError, an error of the runtime a RuntimeError.
template <class F> void call(const c10::Device& device, F entry) {
    const c10::DeviceGuard guard(device);
    char why[256] = "";
    const int rc = entry((void*)c10::hip::getCurrentHIPStream(device.index()).stream(), why, sizeof(why));
    TORCH_CHECK_VALUE(rc != 1, why);
    TORCH_CHECK(rc == 0, why);
}

// The files of the HIP runtimes that the kernels' library and torch use. They name theirs differently, so that both end up in a process that loads
// the library first, and torch's streams are not the library's then.
std::pair<std::string, std::string> runtimes() {
    const auto file = [](const void* p) {
        Dl_info info{};
        return p && dladdr(p, &info) && info.dli_fname ? std::string(info.dli_fname) : std::string();
    };
    const void* torchs = dlsym(dlopen(nullptr, RTLD_LAZY), "hipStreamSynchronize");   // (what is in the global scope comes before a library's own)
    if (!torchs)
        if (void* c10 = dlopen("libc10_hip.so", RTLD_NOLOAD | RTLD_LAZY)) torchs = dlsym(c10, "hipStreamSynchronize");
    return { file(ntc_op_runtime()), file(torchs) };
}

Tensor bytes(int64_t n, const Tensor& like) { return at::empty({ n }, like.options().dtype(at::kByte).requires_grad(false)); }

// Gradients of gradients are not there: asked for, they raise instead of counting as zero.
Tensor once(const Tensor& grad, const char* op) {
    if (!grad.defined() || !at::GradMode::is_enabled()) return grad;
    auto error = std::make_shared<torch::autograd::DelayedError>(std::string(op) + " is differentiable once", 1);
    Tensor g = grad.detach();
    g.requires_grad_(true);
    return (*error)({ g })[0];
}

// ---------------------------------------------------------------- token log probabilities
struct Rows { int64_t rows, inner, outer_stride, inner_stride; };
Rows rows_of(const Tensor& t, int64_t lead, const char* name) {
    if (lead == 0) return { 1, 1, 0, 0 };
    if (lead == 1) return { t.size(0), std::max<int64_t>(1, t.size(0)), 0, t.stride(0) };
    for (int64_t a = 0; a < lead; a++) if (t.size(a) == 0) return { 0, 1, 0, 0 };
    // axes but the last one joined into one stride
    int64_t outer = 1, stride = 0;
    for (int64_t a = lead - 2; a >= 0; a--) {
        if (t.size(a) != 1) {
            TORCH_CHECK_VALUE(outer == 1 || t.stride(a) == stride * outer, "the rows of ", name, " must lie at two strides at most");
            if (outer == 1) stride = t.stride(a);
        }
        outer *= t.size(a);
    }
    return { outer * t.size(lead - 1), std::max<int64_t>(1, t.size(lead - 1)), stride, t.stride(lead - 1) };
}

ntc_logprobs_desc logprobs_desc(const Tensor& logits, const Tensor& tokens, int64_t top, double temperature, int64_t ignore) {
    const int64_t lead = logits.dim() - 1;
    const Rows a = rows_of(logits, lead, "logits"), b = rows_of(tokens, lead, "tokens");
    ntc_logprobs_desc d = {};
    d.logits = logits.const_data_ptr();
    d.tokens = tokens.const_data_ptr();
    d.rows = a.rows;
    d.inner_rows = a.inner;
    d.V = logits.size(-1);
    d.outer_stride = a.outer_stride;
    d.inner_stride = a.inner_stride;
    d.token_outer_stride = b.outer_stride;
    d.token_inner_stride = b.inner_stride;
    d.ignore_index = ignore;
    d.dtype = type_of(logits);
    d.token_bytes = (int32_t)tokens.element_size();
    d.top = (int32_t)top;
    d.temperature = (float)temperature;
    return d;
}

struct Logprobs { Tensor logprob, entropy, ids, top, stats; };
Logprobs logprobs_forward(const Tensor& logits, const Tensor& tokens, int64_t top, double temperature, int64_t ignore) {
    ntc_logprobs_desc d = logprobs_desc(logits, tokens, top, temperature, ignore);
    const auto f = logits.options().dtype(at::kFloat).requires_grad(false);
    Logprobs r;
    r.logprob = at::empty(tokens.sizes(), f);
    r.entropy = at::empty(tokens.sizes(), f);
    r.stats = at::empty({ d.rows, 2 }, f);
    d.logprob = r.logprob.mutable_data_ptr<float>();
    d.entropy = r.entropy.mutable_data_ptr<float>();
    d.stats = r.stats.mutable_data_ptr<float>();
    if (top) {
        std::vector<int64_t> shape = tokens.sizes().vec();
        shape.push_back(top);
        r.ids = at::empty(shape, f.dtype(at::kLong));
        r.top = at::empty(shape, f);
        d.top_ids = r.ids.mutable_data_ptr<int64_t>();
        d.top_logprobs = r.top.mutable_data_ptr<float>();
    }
    const size_t size = ntc_op_token_logprobs_workspace(d.rows, d.V, d.dtype, d.top);
    const Tensor work = size ? bytes((int64_t)size, logits) : Tensor();
    d.workspace = size ? work.mutable_data_ptr() : nullptr;
    call(logits.device(), [&](void* s, char* why, size_t cap) { return ntc_op_token_logprobs(&d, s, why, cap); });
    return r;
}

struct LogprobsNode : torch::autograd::Function<LogprobsNode> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& logits, const Tensor& tokens, int64_t top, double temperature, int64_t ignore) {
        const Logprobs r = logprobs_forward(logits, tokens, top, temperature, ignore);
        ctx->save_for_backward({ logits, tokens, r.entropy, r.stats, r.ids });
        ctx->saved_data["top"] = top;
        ctx->saved_data["temperature"] = temperature;
        ctx->saved_data["ignore"] = ignore;
        ctx->set_materialize_grads(false);
        if (!top) return { r.logprob, r.entropy };
        ctx->mark_non_differentiable({ r.ids });
        return { r.logprob, r.entropy, r.ids, r.top };
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list g) {
        const auto saved = ctx->get_saved_variables();
        const Tensor &logits = saved[0], &tokens = saved[1];
        const int64_t top = ctx->saved_data["top"].toInt();
        Tensor grads[3] = { g[0], g[1], top ? g[3] : Tensor() };
        Tensor dlogits;
        if (grads[0].defined() || grads[1].defined() || grads[2].defined()) {
            ntc_logprobs_desc d = logprobs_desc(logits, tokens, top, ctx->saved_data["temperature"].toDouble(), ctx->saved_data["ignore"].toInt());
            const float* p[3];
            for (int i = 0; i < 3; i++) {
                if (grads[i].defined()) grads[i] = grads[i].contiguous();
                p[i] = grads[i].defined() ? grads[i].const_data_ptr<float>() : nullptr;
            }
            dlogits = at::empty(logits.sizes(), logits.options().requires_grad(false));
            d.entropy = saved[2].data_ptr<float>();
            d.stats = saved[3].data_ptr<float>();
            d.top_ids = top ? saved[4].data_ptr<int64_t>() : nullptr;
            d.g_logprob = p[0];
            d.g_entropy = p[1];
            d.g_top = p[2];
            d.dlogits = dlogits.mutable_data_ptr();
            call(logits.device(), [&](void* s, char* why, size_t cap) { return ntc_op_token_logprobs_backward(&d, s, why, cap); });
        }
        return { once(dlogits, "token_logprobs"), Tensor(), Tensor(), Tensor(), Tensor() };
    }
};

py::tuple token_logprobs(const Tensor& logits, Tensor tokens, int64_t top, double temperature, int64_t ignore) {
    floats("logits", logits);
    no_tangent("logits", logits);
    on_gpu("tokens", tokens);
    TORCH_CHECK_VALUE(tokens.scalar_type() == at::kLong || tokens.scalar_type() == at::kInt, "tokens is ", tokens.scalar_type(), "; it can be int64, int32");
    TORCH_CHECK_VALUE(logits.dim() >= 1 && tokens.sizes() == logits.sizes().slice(0, logits.dim() - 1) && tokens.device() == logits.device(),
                      "tokens ", tokens.sizes(), " must have the shape of logits ", logits.sizes(), " without its last axis, on its device");
    const int64_t V = logits.size(-1);
    TORCH_CHECK_VALUE(V >= 1 && (V == 1 || logits.stride(-1) == 1), "a row of logits must hold at least one value, contiguous");
    TORCH_CHECK_VALUE(top >= 0 && top <= std::min<int64_t>(NTC_MAX_TOP, V), "top is 0 to ", std::min<int64_t>(NTC_MAX_TOP, V), ", not ", top);
    TORCH_CHECK_VALUE(temperature >= 0x1p-127 && temperature <= 0x1p120, "temperature must be from 2^-127 to 2^120, not ", temperature);
    if (tokens.dim() > 2) tokens = tokens.contiguous();
    if (logits.requires_grad() && at::GradMode::is_enabled()) {
        auto r = LogprobsNode::apply(logits, tokens, top, temperature, ignore);
        return top ? py::make_tuple(r[0], r[1], r[2], r[3]) : py::make_tuple(r[0], r[1], py::none(), py::none());
    }
    const Logprobs r = logprobs_forward(logits, tokens, top, temperature, ignore);
    return top ? py::make_tuple(r.logprob, r.entropy, r.ids, r.top) : py::make_tuple(r.logprob, r.entropy, py::none(), py::none());
}

// ---------------------------------------------------------------- 8-bit floating point in blocks
int64_t blocks_of(int64_t n, int64_t b) { return (n + b - 1) / b; }

// A matrix in 8 bits inside a buffer, from `at` on: codes, then exponents, then up to a multiple of 16 bytes.
struct Held {
    Tensor buffer;
    int64_t R = 0, K = 0, block = 1, at = 0;
    uint8_t* codes() const { return buffer.defined() ? (uint8_t*)buffer.data_ptr() + at : nullptr; }
    uint8_t* exps() const { return buffer.defined() ? codes() + R * ntc_fp8_code_stride(K) : nullptr; }
    int64_t size() const { return (R * ntc_fp8_code_stride(K) + blocks_of(R, block) * ntc_fp8_exp_stride(K) + 15) / 16 * 16; }
    Held() = default;
    Held(int64_t r, int64_t k, int64_t b) : R(r), K(k), block(b) {}
    Held(int64_t r, int64_t k, int64_t b, const Tensor& like) : Held(r, k, b) { buffer = bytes(size(), like); }
};
// One buffer for two of them, or for those that are wanted.
Tensor hold(Held& a, bool want_a, Held& b, bool want_b, const Tensor& like) {
    if (!want_a && !want_b) return {};
    const Tensor buffer = bytes((want_a ? a.size() : 0) + (want_b ? b.size() : 0), like);
    b.at = want_a ? a.size() : 0;
    if (want_a) a.buffer = buffer;
    if (want_b) b.buffer = buffer;
    return buffer;
}

ntc_fp8_quantize_desc quantize_desc(const Tensor& x, int64_t block, const Held& plain, const Held& transposed) {
    return { x.const_data_ptr(), x.size(0), x.size(1), x.stride(0), type_of(x), (int32_t)block, plain.codes(), plain.exps(), transposed.codes(), transposed.exps() };
}
void run_quantize(const Tensor& x, const Held& plain, const Held& transposed) {
    if (!x.numel()) return;
    const ntc_fp8_quantize_desc d = quantize_desc(x, plain.block, plain, transposed);
    call(x.device(), [&](void* s, char* why, size_t cap) { return ntc_op_fp8_quantize(&d, s, why, cap); });
}
void run_quantize_pair(const Tensor& x, const Held& xq, const Held& xt, const Tensor& w, const Held& wq, const Held& wt) {
    if (!x.numel() || !w.numel()) { run_quantize(x, xq, xt); run_quantize(w, wq, wt); return; }
    const ntc_fp8_quantize_desc a = quantize_desc(x, 1, xq, xt), b = quantize_desc(w, 128, wq, wt);
    call(x.device(), [&](void* s, char* why, size_t cap) { return ntc_op_fp8_quantize_pair(&a, &b, s, why, cap); });
}
Tensor rows_contiguous(const Tensor& x) { return (x.size(1) > 1 && x.stride(1) != 1) || x.stride(0) < 0 ? x.contiguous() : x; }

struct Operand { const void* p; const uint8_t* exps; int64_t rows, stride; int type, block; };
Operand operand(const Held& h) { return { h.codes(), h.exps(), h.R, 0, NTC_FP8, (int)h.block }; }
void run_matmul(const Operand& a, const Operand& b, int64_t K, const Tensor& c) {
    if (!a.rows || !b.rows) return;
    if (!K) { c.zero_(); return; }
    const size_t size = ntc_op_fp8_matmul_workspace(a.rows, b.rows, K, a.type);
    const Tensor work = size ? bytes((int64_t)size, c) : Tensor();
    const ntc_fp8_matmul_desc d = { a.p, a.exps, (const uint8_t*)b.p, b.exps, c.mutable_data_ptr(), size ? work.mutable_data_ptr() : nullptr, a.rows, b.rows, K, a.stride, c.stride(0),
                                    a.type, a.block, b.block, type_of(c) };
    call(c.device(), [&](void* s, char* why, size_t cap) { return ntc_op_fp8_matmul(&d, s, why, cap); });
}
Tensor matrix(int64_t m, int64_t n, at::ScalarType t, const Tensor& like) { return at::empty({ m, n }, like.options().dtype(t).requires_grad(false)); }

py::tuple quantize(const Tensor& x_, int64_t block, bool plain, bool transposed) {
    floats("x", x_);
    TORCH_CHECK_VALUE(x_.dim() == 2, "a matrix is needed, not ", x_.sizes());
    TORCH_CHECK_VALUE(block == 1 || block == 128, "blocks have 1 or 128 rows, not ", block);
    const Tensor x = rows_contiguous(x_);
    const int64_t R = x.size(0), K = x.size(1);
    const auto o = x.options().dtype(at::kByte).requires_grad(false);
    const auto make = [&](int64_t r, int64_t k) { return std::make_pair(at::empty({ r, ntc_fp8_code_stride(k) }, o), at::empty({ blocks_of(r, block), ntc_fp8_exp_stride(k) }, o)); };
    std::pair<Tensor, Tensor> q, t;
    if (plain) q = make(R, K);
    if (transposed) t = make(K, R);
    const auto at_ = [](const Tensor& b) { return b.defined() ? (uint8_t*)b.data_ptr() : nullptr; };
    if (x.numel()) {
        const ntc_fp8_quantize_desc d = { x.const_data_ptr(), R, K, x.stride(0), type_of(x), (int32_t)block, at_(q.first), at_(q.second), at_(t.first), at_(t.second) };
        call(x.device(), [&](void* s, char* why, size_t cap) { return ntc_op_fp8_quantize(&d, s, why, cap); });
    }
    return py::make_tuple(plain ? py::cast(q) : py::none(), transposed ? py::cast(t) : py::none());
}

Operand given(const char* name, const Tensor& codes, const Tensor& exps, int64_t R, int64_t K, int64_t block) {
    on_gpu(name, codes);
    on_gpu(name, exps);
    const bool ok = (block == 1 || block == 128) && codes.scalar_type() == at::kByte && exps.scalar_type() == at::kByte && codes.is_contiguous() && exps.is_contiguous() &&
                    codes.device() == exps.device() && R >= 0 && K >= 0;
    TORCH_CHECK_VALUE(ok && codes.sizes() == at::IntArrayRef({ R, ntc_fp8_code_stride(K) }) && (uintptr_t)codes.const_data_ptr() % 16 == 0, name, ".codes must be uint8, contiguous, start at a multiple of 16 bytes and be [",
                      R, ", ", ntc_fp8_code_stride(K), "]");
    TORCH_CHECK_VALUE(exps.sizes() == at::IntArrayRef({ blocks_of(R, block), ntc_fp8_exp_stride(K) }) && (uintptr_t)exps.const_data_ptr() % 4 == 0, name,
                      ".exps must be uint8, contiguous, start at a multiple of 4 bytes and be [", blocks_of(R, block), ", ", ntc_fp8_exp_stride(K), "]");
    return { codes.const_data_ptr(), (const uint8_t*)exps.const_data_ptr(), R, 0, NTC_FP8, (int)block };
}

Tensor matmul(const Tensor& ac, const Tensor& ae, int64_t M, int64_t ka, int64_t a_block, const Tensor& bc, const Tensor& be, int64_t N, int64_t kb, int64_t b_block, at::ScalarType type) {
    const Operand a = given("a", ac, ae, M, ka, a_block), b = given("b", bc, be, N, kb, b_block);
    TORCH_CHECK_VALUE(ka == kb && ac.device() == bc.device(), "a [", M, ", ", ka, "] and b [", N, ", ", kb, "] must have as many columns, on one device");
    TORCH_CHECK_VALUE(type_of(type) >= 0, "products are float32, bfloat16 or float16, not ", type);
    const Tensor c = matrix(M, N, type, ac);
    run_matmul(a, b, ka, c);
    return c;
}

// Rows that one product may sum over (a multiple of its blocks): the weights' gradient of more is the sum of several, in 32 bits.
constexpr int64_t kMostSum = 1 << 23;

struct LinearNode : torch::autograd::Function<LinearNode> {
    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& w) {
        const int64_t M = x.size(0), K = x.size(1), N = w.size(0);
        const bool need_x = x.requires_grad(), need_w = w.requires_grad();
        Held xq(M, K, 1), wq(N, K, 128), xt(K, M, 1), wt(K, N, 128);
        hold(xq, true, wq, true, x);
        const bool parts = need_w && M > kMostSum;
        const Tensor kept = hold(xt, need_w && !parts, wt, need_x, x);
        run_quantize_pair(x, xq, xt, w, wq, wt);
        torch::autograd::variable_list saved = { kept };
        for (int64_t m = 0; parts && m < M; m += kMostSum) {
            const Held t(K, std::min(kMostSum, M - m), 1, x);
            run_quantize(x.narrow(0, m, t.K), {}, t);
            saved.push_back(t.buffer);
        }
        const Tensor y = matrix(M, N, x.scalar_type(), x);
        run_matmul(operand(xq), operand(wq), K, y);
        ctx->save_for_backward(saved);
        ctx->saved_data["call"] = std::vector<int64_t>{ M, N, K, need_x, need_w, (int64_t)x.scalar_type(), (int64_t)w.scalar_type() };
        ctx->set_materialize_grads(false);
        return y;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list g) {
        if (!g[0].defined()) return { Tensor(), Tensor() };
        const auto saved = ctx->get_saved_variables();
        const std::vector<int64_t> of = ctx->saved_data["call"].toIntVector();
        const int64_t M = of[0], N = of[1], K = of[2];
        const bool need_x = of[3], need_w = of[4];
        const Tensor dy = rows_contiguous(g[0]);
        Held dq(M, N, 1), dt(N, M, 1), xt(K, M, 1), wt(K, N, 128);
        const bool parts = need_w && M > kMostSum;
        hold(dq, need_x, dt, need_w && !parts, dy);
        if (need_w && !parts) xt.buffer = saved[0];
        if (need_x) wt.buffer = saved[0];
        wt.at = xt.buffer.defined() ? xt.size() : 0;
        if (need_x || !parts) run_quantize(dy, dq, dt);
        Tensor dx, dw;
        if (need_x) {
            dx = matrix(M, K, (at::ScalarType)of[5], dy);
            run_matmul(operand(dq), operand(wt), N, dx);
        }
        if (parts) {
            for (int64_t m = 0; m < M; m += kMostSum) {
                Held part(K, std::min(kMostSum, M - m), 1);
                part.buffer = saved[1 + m / kMostSum];
                const Held t(N, part.K, 1, dy);
                run_quantize(dy.narrow(0, m, part.K), {}, t);
                const Tensor sum = matrix(N, K, at::kFloat, dy);
                run_matmul(operand(t), operand(part), part.K, sum);
                if (m) dw += sum; else dw = sum;
            }
            dw = dw.to((at::ScalarType)of[6]);
        } else if (need_w) {
            dw = matrix(N, K, (at::ScalarType)of[6], dy);
            run_matmul(operand(dt), operand(xt), M, dw);
        }
        return { once(dx, "fp8_linear"), once(dw, "fp8_linear") };
    }
};

Tensor as_rows(const Tensor& x) {
    int64_t rows = 1;
    for (int64_t a = 0; a + 1 < x.dim(); a++) rows *= x.size(a);
    return x.dim() == 2 ? x : x.reshape({ rows, x.size(-1) });
}
Tensor like_rows(const Tensor& y, const Tensor& x) {
    if (x.dim() == 2) return y;
    std::vector<int64_t> shape = x.sizes().vec();
    shape.back() = y.size(1);
    return y.view(shape);
}

Tensor linear(const Tensor& x, const Tensor& w) {
    floats("x", x);
    floats("w", w);
    no_tangent("x", x);
    no_tangent("w", w);
    TORCH_CHECK_VALUE(x.dim() >= 1, "x must have at least one axis");
    TORCH_CHECK_VALUE(w.dim() == 2 && w.size(1) == x.size(-1) && w.device() == x.device(), "w ", w.sizes(), " must be a matrix with x's ", x.size(-1), " columns, on its device");
    const bool grad = at::GradMode::is_enabled() && (x.requires_grad() || w.requires_grad());
    const Tensor x2 = rows_contiguous(as_rows(x)), w2 = rows_contiguous(w);
    if (grad) return like_rows(LinearNode::apply(x2, w2), x);
    Held xq(x2.size(0), x2.size(1), 1), wq(w2.size(0), w2.size(1), 128);
    hold(xq, true, wq, true, x2);
    run_quantize_pair(x2, xq, {}, w2, wq, {});
    const Tensor y = matrix(x2.size(0), w2.size(0), x.scalar_type(), x2);
    run_matmul(operand(xq), operand(wq), x2.size(1), y);
    return like_rows(y, x);
}

Tensor linear_fp8(const Tensor& x, const Tensor& codes, const Tensor& exps, int64_t N, int64_t K, int64_t block) {
    floats("x", x);
    no_tangent("x", x);
    const Operand b = given("w", codes, exps, N, K, block);
    TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) == K && x.device() == codes.device(), "x ", x.sizes(), " must have w's ", K, " columns, on its device");
    TORCH_CHECK_VALUE(!(x.requires_grad() && at::GradMode::is_enabled()), "w in 8 bits is for inference: give the weights themselves for a gradient");
    const Tensor x2 = rows_contiguous(as_rows(x));
    const int64_t M = x2.size(0);
    const Tensor y = matrix(M, N, x.scalar_type(), x2);
    if (M <= ntc_op_fp8_matmul_float_rows()) {
        run_matmul({ x2.const_data_ptr(), nullptr, M, x2.stride(0), type_of(x2), 1 }, b, K, y);
    } else {
        const Held xq(M, K, 1, x2);
        run_quantize(x2, xq, {});
        run_matmul(operand(xq), b, K, y);
    }
    return like_rows(y, x);
}

// ---------------------------------------------------------------- AdamW
void state_tensor(const char* name, const Tensor& t, at::ScalarType type, int64_t n, const c10::Device& device) {
    TORCH_CHECK_VALUE(t.defined() && t.device() == device && t.scalar_type() == type && t.numel() == n && t.is_contiguous(), name, " must be ", n, " contiguous values of ", type, " on ", device);
}
// Of n values in 32 bits, or in 8 with their exponents (undefined otherwise).
void state_tensors(const Tensor& m, const Tensor& v, const Tensor& me, const Tensor& ve, int64_t bits, int64_t n, const c10::Device& device) {
    const auto type = bits == 8 ? at::kByte : at::kFloat;
    state_tensor("exp_avg", m, type, n, device);
    state_tensor("exp_avg_sq", v, type, n, device);
    if (bits != 8) return;
    state_tensor("exp_avg_exp", me, at::kByte, n / NTC_STATE_BLOCK, device);
    state_tensor("exp_avg_sq_exp", ve, at::kByte, n / NTC_STATE_BLOCK, device);
}

// The tensors of an optimizer, and what their step needs beside its state.
struct AdamwPlan {
    std::vector<Tensor> params;
    std::vector<const void*> pointers;
    std::vector<int64_t> numels;
    std::vector<int32_t> kinds;
    Tensor tables;                                          // on the device: the tensors, then each chunk's
    const ntc_adamw_tensor* table = nullptr;
    const int32_t* chunk_tensor = nullptr;
    std::vector<int64_t> first_chunk, offsets;
    std::vector<int32_t> steps;
    int64_t size = 0, calls = 0;

    explicit AdamwPlan(std::vector<Tensor> p) : params(std::move(p)) {
        TORCH_CHECK_VALUE(!params.empty(), "no parameters");
        std::vector<std::pair<uintptr_t, uintptr_t>> spans;
        std::vector<ntc_adamw_tensor> rows;
        std::vector<int32_t> of_chunk;
        first_chunk.push_back(0);
        for (const Tensor& t : params) {
            floats("a parameter", t);
            TORCH_CHECK_VALUE(t.is_contiguous() && t.device() == params[0].device(), "parameters are contiguous and on one device");
            const int64_t n = t.numel(), chunks = blocks_of(n, NTC_ADAMW_CHUNK);
            const uintptr_t at = (uintptr_t)t.const_data_ptr();
            if (n) spans.push_back({ at, at + (uintptr_t)(n * t.element_size()) });
            TORCH_CHECK_VALUE(first_chunk.back() + chunks < (int64_t)1 << 31, "too many weights");
            rows.push_back({ (void*)at, n, size, type_of(t), (int32_t)first_chunk.back() });
            of_chunk.insert(of_chunk.end(), (size_t)chunks, (int32_t)pointers.size());
            pointers.push_back((const void*)at);
            numels.push_back(n);
            kinds.push_back(type_of(t));
            offsets.push_back(size);
            size += blocks_of(n, NTC_STATE_BLOCK) * NTC_STATE_BLOCK;
            first_chunk.push_back(first_chunk.back() + chunks);
        }
        std::sort(spans.begin(), spans.end());
        for (size_t i = 1; i < spans.size(); i++) TORCH_CHECK_VALUE(spans[i - 1].second <= spans[i].first, "parameters overlap");
        const c10::DeviceGuard guard(params[0].device());
        // one copy to the device for both: it waits, and costs more than what it moves
        const size_t rows_size = rows.size() * sizeof(rows[0]), chunks_size = of_chunk.size() * sizeof(of_chunk[0]);
        std::vector<uint8_t> both(rows_size + chunks_size);
        std::memcpy(both.data(), rows.data(), rows_size);
        if (chunks_size) std::memcpy(both.data() + rows_size, of_chunk.data(), chunks_size);
        tables = at::from_blob(both.data(), { (int64_t)both.size() }, at::kByte).to(params[0].device());
        table = (const ntc_adamw_tensor*)tables.const_data_ptr();
        chunk_tensor = (const int32_t*)((const uint8_t*)tables.const_data_ptr() + rows_size);
        steps.resize(params.size());
    }

    // one gradient or None a parameter; None for all: the parameters' own
    void step(const optional<std::vector<optional<Tensor>>>& given, const Tensor& m, const Tensor& v, const optional<Tensor>& me, const optional<Tensor>& ve, const optional<Tensor>& master, int64_t bits,
              double lr, double b1, double b2, double eps, double decay, uint64_t seed) {
        const size_t n = params.size();
        TORCH_CHECK_VALUE(!given || given->size() == n, given ? given->size() : 0, " gradients for ", n, " parameters");
        std::vector<Tensor> keep;                           // copies of gradients that are not contiguous, until their launch
        std::vector<const void*> g(n, nullptr);
        std::vector<int32_t> types(n, 0), next(steps);
        const auto device = params[0].device();
        state_tensors(m, v, me ? *me : undefined, ve ? *ve : undefined, bits, size, device);
        if (master) state_tensor("master", *master, at::kFloat, size, device);
        for (size_t i = 0; i < n; i++) {
            const Tensor& p = params[i];
            TORCH_CHECK_VALUE(p.const_data_ptr() == pointers[i], "a parameter has moved to other memory since the optimizer was made");
            TORCH_CHECK_VALUE(p.numel() == numels[i] && type_of(p) == kinds[i] && p.is_contiguous(), "a parameter has another size, type or layout than when the optimizer was made");
            const Tensor& t = given ? ((*given)[i] ? *(*given)[i] : undefined) : params[i].grad();
            if (!t.defined()) continue;
            types[i] = type_of(t);
            TORCH_CHECK_VALUE(types[i] >= 0 && t.device() == device && t.sizes() == params[i].sizes(), "gradient ", i, " must have its parameter's shape ", params[i].sizes(),
                              ", be on its device, and be float32, bfloat16 or float16");
            if (t.is_contiguous()) g[i] = t.const_data_ptr();
            else { keep.push_back(t.contiguous()); g[i] = keep.back().const_data_ptr(); }
            next[i]++;
        }
        const auto at_ = [](const optional<Tensor>& t) { return t ? t->data_ptr() : nullptr; };
        ntc_adamw_desc d = {};
        d.tensors = table;
        d.chunk_tensor = chunk_tensor;
        d.first_chunk = first_chunk.data();
        d.grads = g.data();
        d.grad_types = types.data();
        d.steps = next.data();
        d.n = (int64_t)n;
        d.exp_avg = m.data_ptr();
        d.exp_avg_sq = v.data_ptr();
        d.exp_avg_exp = (uint8_t*)at_(me);
        d.exp_avg_sq_exp = (uint8_t*)at_(ve);
        d.master = (float*)at_(master);
        d.lr = lr;
        d.beta1 = b1;
        d.beta2 = b2;
        d.eps = eps;
        d.weight_decay = decay;
        d.seed = seed;
        d.calls = (uint32_t)(calls + 1);
        d.state_bits = (int32_t)bits;
        call(device, [&](void* s, char* why, size_t cap) { return ntc_op_adamw(&d, s, why, cap); });
        for (size_t i = 0; i < n; i++)                       // (changed in place, behind autograd's back; those left alone have not changed)
            if (g[i] && !params[i].is_inference()) params[i].unsafeGetTensorImpl()->bump_version();
        steps = next;
        calls++;
    }
    const Tensor undefined;
};

std::pair<Tensor, Tensor> adamw_moments(const Tensor& m, const Tensor& v, const Tensor& me, const Tensor& ve) {
    on_gpu("exp_avg", m);
    TORCH_CHECK_VALUE(m.numel() % NTC_STATE_BLOCK == 0, "a state is a multiple of 256 values");
    state_tensors(m, v, me, ve, 8, m.numel(), m.device());
    const Tensor a = at::empty(m.sizes(), m.options().dtype(at::kFloat)), b = at::empty(m.sizes(), m.options().dtype(at::kFloat));
    call(m.device(), [&](void* s, char* why, size_t cap) {
        return ntc_op_adamw_moments(m.const_data_ptr(), v.const_data_ptr(), (const uint8_t*)me.const_data_ptr(), (const uint8_t*)ve.const_data_ptr(), m.numel(), a.mutable_data_ptr<float>(),
                                    b.mutable_data_ptr<float>(), s, why, cap);
    });
    return { a, b };
}
void adamw_encode(const Tensor& m, const Tensor& v, const Tensor& cm, const Tensor& cv, const Tensor& me, const Tensor& ve) {
    on_gpu("m", m);
    state_tensor("m", m, at::kFloat, m.numel(), m.device());
    state_tensor("v", v, at::kFloat, m.numel(), m.device());
    state_tensors(cm, cv, me, ve, 8, m.numel(), m.device());
    call(m.device(), [&](void* s, char* why, size_t cap) {
        return ntc_op_adamw_encode(m.const_data_ptr<float>(), v.const_data_ptr<float>(), m.numel(), cm.data_ptr(), cv.data_ptr(), (uint8_t*)me.data_ptr(), (uint8_t*)ve.data_ptr(), s, why, cap);
    });
}

}  // namespace

PYBIND11_MODULE(_ops, m) {
    m.doc() = "The operators of ops.py on torch tensors";
    m.def("runtimes", &runtimes);
    m.def("token_logprobs", &token_logprobs);
    m.def("quantize", &quantize);
    m.def("matmul", [](const Tensor& ac, const Tensor& ae, int64_t M, int64_t ka, int64_t a_block, const Tensor& bc, const Tensor& be, int64_t N, int64_t kb, int64_t b_block, py::object type) {
        return matmul(ac, ae, M, ka, a_block, bc, be, N, kb, b_block, torch::python::detail::py_object_to_dtype(type));
    });
    m.def("linear", &linear);
    m.def("linear_fp8", &linear_fp8);
    m.def("adamw_moments", &adamw_moments);
    m.def("adamw_encode", &adamw_encode);
    py::class_<AdamwPlan>(m, "AdamwPlan")
        .def(py::init<std::vector<Tensor>>())
        .def("step", &AdamwPlan::step)
        .def_readonly("offsets", &AdamwPlan::offsets)
        .def_readonly("size", &AdamwPlan::size)
        .def_readwrite("calls", &AdamwPlan::calls)
        .def_readwrite("steps", &AdamwPlan::steps);
}
