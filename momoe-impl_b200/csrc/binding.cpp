// Host side of the operators around the expert layer: argument checks, buffers and autograd nodes for torch tensors above
// the C ABI.  In C++ because these operators are short: one call costs 10 us here and 25 to 60 us in Python, where the
// kernels of a decoded token take 3 us and those of a training step 20 to 100 us.
//
// The module does not link libmomoe_b200.so; it is handed the path of the library that the package has loaded and takes
// the entry points from it.
#include <dlfcn.h>

#include <atomic>
#include <optional>

#include <ATen/cuda/CUDAContext.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/extension.h>

#include "../../include/momoe_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

#define ENTRY_POINTS(X)                         \
    X(momoe_rms_norm)                           \
    X(momoe_rms_norm_backward_workspace_bytes)  \
    X(momoe_rms_norm_backward)                  \
    X(momoe_balance_loss_workspace_bytes)       \
    X(momoe_balance_loss)                       \
    X(momoe_balance_loss_backward)              \
    X(momoe_fp8_experts_workspace_bytes)        \
    X(momoe_fp8_experts_launches)               \
    X(momoe_fp8_experts_forward)

struct Api {
#define X(name) decltype(&::name) name = nullptr;
    ENTRY_POINTS(X)
#undef X
} api;

std::atomic<int64_t> n_launches{0};

void bind(const std::string& path) {
    void* lib = dlopen(path.c_str(), RTLD_NOW | RTLD_LOCAL);
    TORCH_CHECK(lib != nullptr, "cannot load ", path, ": ", dlerror());
#define X(name)                                                                  \
    api.name = reinterpret_cast<decltype(&::name)>(dlsym(lib, #name));           \
    TORCH_CHECK(api.name != nullptr, path, " has no ", #name);
    ENTRY_POINTS(X)
#undef X
}

void check(int rc, const char* what, int64_t launches) {
    if (rc == 0) {
        n_launches += launches;
        return;
    }
    const char* why = rc == -1   ? "bad argument (null pointer, size or alignment)"
                      : rc == -2 ? "unsupported shape or type"
                      : rc == -3 ? "a CUDA call failed"
                      : rc == -4 ? "exceeds a fixed capacity"
                                 : "unknown code";
    TORCH_CHECK(false, what, " failed: ", why);
}

void require_device(const Tensor& t, const at::Device& dev) {
    TORCH_CHECK(t.is_cuda(), "momoe (B200 build) runs on CUDA tensors only; there is no CPU path");
    TORCH_CHECK(t.device() == dev, "all tensors must be on the same device, but got: ", dev, " and ", t.device());
}
at::Device cuda_device(const Tensor& t) {
    TORCH_CHECK(t.is_cuda(), "momoe (B200 build) runs on CUDA tensors only; there is no CPU path");
    return t.device();
}
void no_second_derivative(const char* what) {
    TORCH_CHECK(!at::GradMode::is_enabled(), what, " has no second derivative (create_graph=True)");
}

// There are no forward-mode derivatives: a tangent would be lost, so it is refused.
template <typename... T>
void no_tangent(const char* what, const T&... inputs) {
    if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
    const auto dual = [](const Tensor& t) { return t.defined() && t._fw_grad(/*level=*/0).defined(); };
    TORCH_CHECK(!(dual(inputs) || ...), what, " has no forward-mode derivative");
}

int type_code(at::ScalarType t) { return t == at::kBFloat16 ? 0 : t == at::kHalf ? 1 : t == at::kFloat ? 2 : -1; }

bool is_aligned(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }
// t itself where it is contiguous and starts on a 16-byte boundary, a copy otherwise.
Tensor dense(const Tensor& t) {
    Tensor c = t.contiguous();
    return is_aligned(c) ? c : c.clone();
}
// Whole numbers as contiguous int32; ones that int32 does not hold are first brought into [lo, hi], which keeps the ones
// outside outside.  In 64 bits, since a narrow type does not hold the limits either (-1 wraps around in an unsigned one).
Tensor whole32(const Tensor& t, int64_t lo, int64_t hi) {
    switch (t.scalar_type()) {
        case at::kInt:
            return t.contiguous();
        case at::kLong:
        case at::kUInt32:
        case at::kUInt64:
            return t.to(at::kLong).clamp(lo, hi).to(at::kInt).contiguous();
        default:
            return t.to(at::kInt).contiguous();
    }
}
// t [..., D] as [M, D] with contiguous columns, a row pitch of a multiple of 8 elements and a 16-byte aligned start: a
// view where the layout allows it.
Tensor as_rows(const Tensor& t) {
    Tensor r = t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
    if (r.is_contiguous()) return is_aligned(r) ? r : r.clone();
    if (r.stride(1) != 1 || r.stride(0) % 8 != 0 || r.stride(0) < 0 || !is_aligned(r)) return r.contiguous();
    return r;
}
int64_t pitch(const Tensor& r) { return r.size(0) > 1 ? r.stride(0) : r.size(1); }
void* data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* stream_of(const at::Device& dev) { return at::cuda::getCurrentCUDAStream(dev.index()).stream(); }
int32_t i32(int64_t v, const char* what) {
    TORCH_CHECK(v >= 0 && v <= INT32_MAX, what, " is out of range: ", v);
    return static_cast<int32_t>(v);
}

// ------------------------------------------------------------------------------------------------ norm
constexpr int64_t kBlock = 128, kMaxNorm = 16384;

void norm_check(const Tensor& x, const Tensor& weight, const OptTensor& residual) {
    const at::Device dev = cuda_device(x);
    require_device(weight, dev);
    TORCH_CHECK(type_code(x.scalar_type()) >= 0, "rms_norm works on bfloat16, float16 or float32, but got: ", x.dtype());
    const int64_t D = x.dim() > 0 ? x.size(-1) : 0;
    TORCH_CHECK(D > 0 && D % 8 == 0 && D <= kMaxNorm, "the normed width must be a multiple of 8 up to ", kMaxNorm,
                ", but got: ", D);
    TORCH_CHECK(weight.dim() == 1 && weight.size(0) == D &&
                    (weight.scalar_type() == x.scalar_type() || weight.scalar_type() == at::kFloat),
                "the weight must be [", D, "] in ", x.dtype(), " or float32, but got: ", weight.sizes(), " in ",
                weight.dtype());
    if (residual) {
        require_device(*residual, dev);
        TORCH_CHECK(residual->sizes() == x.sizes() && residual->scalar_type() == x.scalar_type(),
                    "the residual must be like x, ", x.sizes(), " in ", x.dtype(), ", but got: ", residual->sizes(), " in ",
                    residual->dtype());
    }
    no_tangent("rms_norm", x, weight, residual ? *residual : Tensor());
}

struct Norm {
    Tensor rows, w, y, r, rstd, q, scale;     // rows: x as read; r: the sum, undefined without a residual
};
Norm norm_forward(const Tensor& x, const Tensor& weight, const OptTensor& residual, double eps, bool want_rstd,
                  bool want_rows8) {
    Norm o;
    const at::Device dev = x.device();
    const c10::cuda::CUDAGuard guard(dev);
    o.rows = as_rows(x);
    o.w = dense(weight);
    const int64_t M = o.rows.size(0), D = o.rows.size(1);
    const auto opt = o.rows.options();
    // outputs keep the shape of x; they are contiguous, so the kernel sees rows
    o.y = at::empty(x.sizes(), opt);
    Tensor res;
    if (residual) {
        res = as_rows(*residual);
        o.r = at::empty(x.sizes(), opt);
    }
    if (want_rstd) o.rstd = at::empty({M}, opt.dtype(at::kFloat));
    if (want_rows8) {
        o.q = at::empty({M, D}, opt.dtype(at::kFloat8_e4m3fn));
        o.scale = at::empty({M, (D + kBlock - 1) / kBlock}, opt.dtype(at::kFloat8_e8m0fnu));
    }
    if (M > 0)
        check(api.momoe_rms_norm(o.rows.data_ptr(), pitch(o.rows), data(res), res.defined() ? pitch(res) : 0,
                                 o.w.data_ptr(), type_code(x.scalar_type()), type_code(o.w.scalar_type()), i32(M, "M"),
                                 static_cast<int32_t>(D), static_cast<float>(eps), data(o.r), o.y.data_ptr(),
                                 static_cast<float*>(data(o.rstd)), static_cast<uint8_t*>(data(o.q)),
                                 static_cast<uint8_t*>(data(o.scale)), stream_of(dev)),
              "momoe_rms_norm", 1);
    return o;
}

struct NormFunction : torch::autograd::Function<NormFunction> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const OptTensor& residual,
                                 double eps) {
        ctx->set_materialize_grads(false);
        Norm o = norm_forward(x, weight, residual, eps, true, false);
        // what the backward pass reads: the sum as it was returned, or x as the kernel read it
        ctx->save_for_backward({residual ? o.r : o.rows, o.w, o.rstd});
        ctx->saved_data["shape"] = x.sizes();
        return residual ? variable_list{o.y, o.r} : variable_list{o.y};
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        no_second_derivative("rms_norm");
        const auto saved = ctx->get_saved_variables();
        Tensor r = saved[0];
        const Tensor &w = saved[1], &rstd = saved[2];
        const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
        const bool has_residual = g.size() > 1;      // an input that was not a tensor gets no gradient
        Tensor gy = g[0], gr = has_residual ? g[1] : Tensor();
        if (!gy.defined())                     // only the sum was used, or nothing
            return {gr, need_w && gr.defined() ? at::zeros_like(w) : Tensor(), gr, Tensor()};
        const at::Device dev = w.device();
        const c10::cuda::CUDAGuard guard(dev);
        const int64_t D = w.size(0);
        if (r.dim() != 2) r = r.view({-1, D});
        const int64_t M = r.size(0);
        gy = dense(gy);
        if (gr.defined()) gr = dense(gr);
        Tensor gx = at::empty(ctx->saved_data["shape"].toIntVector(), r.options());
        Tensor gw = need_w ? at::empty_like(w) : Tensor(), ws;
        if (M > 0) {
            size_t bytes = 0;
            if (need_w) {
                bytes = api.momoe_rms_norm_backward_workspace_bytes(static_cast<int32_t>(M), static_cast<int32_t>(D));
                ws = at::empty({static_cast<int64_t>(bytes)}, r.options().dtype(at::kByte));
            }
            check(api.momoe_rms_norm_backward(gy.data_ptr(), data(gr), r.data_ptr(), pitch(r), w.data_ptr(),
                                              rstd.data_ptr<float>(), type_code(r.scalar_type()),
                                              type_code(w.scalar_type()), static_cast<int32_t>(M),
                                              static_cast<int32_t>(D), gx.data_ptr(), data(gw), data(ws), bytes,
                                              stream_of(dev)),
                  "momoe_rms_norm_backward", need_w ? 2 : 1);
        } else if (need_w) {
            gw.zero_();
        }
        return {need_x ? gx : Tensor(), gw, has_residual ? gx : Tensor(), Tensor()};
    }
};

bool learns(const Tensor& x, const Tensor& weight, const OptTensor& residual) {
    return at::GradMode::is_enabled() &&
           (x.requires_grad() || weight.requires_grad() || (residual && residual->requires_grad()));
}

// [y] or [y, r]
std::vector<Tensor> rms_norm(const Tensor& x, const Tensor& weight, const OptTensor& residual, double eps) {
    norm_check(x, weight, residual);
    if (learns(x, weight, residual)) return NormFunction::apply(x, weight, residual, eps);
    Norm o = norm_forward(x, weight, residual, eps, false, false);
    return residual ? std::vector<Tensor>{o.y, o.r} : std::vector<Tensor>{o.y};
}

// [y, q, scale] or [y, q, scale, r]
std::vector<Tensor> rms_norm_fp8(const Tensor& x, const Tensor& weight, const OptTensor& residual, double eps) {
    norm_check(x, weight, residual);
    TORCH_CHECK(!learns(x, weight, residual), "rms_norm_fp8 has no backward pass: call it under torch.no_grad()");
    Norm o = norm_forward(x, weight, residual, eps, false, true);
    return residual ? std::vector<Tensor>{o.y, o.q, o.scale, o.r} : std::vector<Tensor>{o.y, o.q, o.scale};
}

// ------------------------------------------------------------------------------------------------ balance loss
// Contiguous logits and ids -> loss [], counts [B, N], coefficients of the backward pass [B, N].
std::vector<Tensor> balance_forward(const Tensor& logits, const Tensor& idx, int64_t Ks, double balance_coef, double z_coef,
                                    const OptTensor& cu, int64_t seq_len, int64_t B) {
    const at::Device dev = logits.device();
    const c10::cuda::CUDAGuard guard(dev);
    const int64_t M = logits.size(0), N = logits.size(1);
    const auto opt = logits.options().dtype(at::kFloat);
    if (M == 0) return {at::zeros({}, opt), at::zeros({B, N}, opt.dtype(at::kLong)), at::zeros({B, N}, opt)};
    Tensor loss = at::empty({}, opt), counts = at::empty({B, N}, opt.dtype(at::kLong)), g = at::empty({B, N}, opt);
    const int32_t m = i32(M, "M"), n = i32(N, "N"), b = i32(B, "B");
    const size_t bytes = api.momoe_balance_loss_workspace_bytes(m, n, b);
    Tensor ws = at::empty({static_cast<int64_t>(bytes)}, opt.dtype(at::kByte));
    check(api.momoe_balance_loss(logits.data_ptr(), type_code(logits.scalar_type()), idx.data_ptr<int32_t>(),
                                 cu ? cu->data_ptr<int32_t>() : nullptr, i32(seq_len, "seq_len"), m, n,
                                 i32(idx.size(1), "K"), static_cast<int32_t>(Ks), b, static_cast<float>(balance_coef),
                                 static_cast<float>(z_coef), loss.data_ptr<float>(), counts.data_ptr<int64_t>(),
                                 g.data_ptr<float>(), ws.data_ptr(), bytes, stream_of(dev)),
          "momoe_balance_loss", 2);
    return {loss, counts, g};
}

// Gradient of the logits; `add` (in the type of the logits): a gradient from elsewhere, overwritten with the sum.
Tensor balance_backward(const Tensor& logits, const Tensor& g, int64_t Ks, double z_coef, const OptTensor& cu,
                        int64_t seq_len, const Tensor& G_loss, const OptTensor& add) {
    const at::Device dev = logits.device();
    const c10::cuda::CUDAGuard guard(dev);
    Tensor out = add ? *add : at::empty_like(logits);
    if (logits.size(0) == 0) return out;
    const Tensor up = G_loss.scalar_type() == at::kFloat ? G_loss : G_loss.to(at::kFloat);
    check(api.momoe_balance_loss_backward(logits.data_ptr(), type_code(logits.scalar_type()),
                                          cu ? cu->data_ptr<int32_t>() : nullptr, static_cast<int32_t>(seq_len),
                                          g.data_ptr<float>(), static_cast<int32_t>(logits.size(0)),
                                          static_cast<int32_t>(logits.size(1)), static_cast<int32_t>(Ks),
                                          static_cast<int32_t>(g.size(0)), static_cast<float>(z_coef),
                                          up.data_ptr<float>(), add ? add->data_ptr() : nullptr, out.data_ptr(),
                                          stream_of(dev)),
          "momoe_balance_loss_backward", 1);
    return out;
}

struct BalanceFunction : torch::autograd::Function<BalanceFunction> {
    static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& idx, int64_t Ks,
                                 double balance_coef, double z_coef, const OptTensor& cu, int64_t seq_len, int64_t B) {
        ctx->set_materialize_grads(false);
        const c10::cuda::CUDAGuard guard(logits.device());
        const Tensor x = dense(logits);
        auto o = balance_forward(x, idx, Ks, balance_coef, z_coef, cu, seq_len, B);
        ctx->save_for_backward({x, o[2], cu ? *cu : Tensor()});
        ctx->saved_data["Ks"] = Ks;
        ctx->saved_data["z"] = z_coef;
        ctx->saved_data["S"] = seq_len;
        ctx->mark_non_differentiable({o[1]});
        return {o[0], o[1]};
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        no_second_derivative("balance_loss");
        variable_list grads(8);
        if (!g[0].defined()) return grads;
        const auto saved = ctx->get_saved_variables();
        grads[0] = balance_backward(saved[0], saved[1], ctx->saved_data["Ks"].toInt(), ctx->saved_data["z"].toDouble(),
                                    saved[2].defined() ? OptTensor(saved[2]) : OptTensor(), ctx->saved_data["S"].toInt(),
                                    g[0], {});
        return grads;
    }
};

// [loss, counts]
std::vector<Tensor> balance_loss(const Tensor& logits, const Tensor& topk_idx, int64_t Ks, double balance_coef,
                                 double z_coef, const OptTensor& cu_seqlens, std::optional<int64_t> seq_len) {
    const at::Device dev = cuda_device(logits);
    require_device(topk_idx, dev);
    TORCH_CHECK(logits.scalar_type() == at::kBFloat16 || logits.scalar_type() == at::kFloat,
                "the logits must be bfloat16 or float32, but got: ", logits.dtype());
    TORCH_CHECK(logits.dim() == 2 && topk_idx.dim() == 2 && topk_idx.size(0) == logits.size(0),
                "the logits must be [M, N] and the expert ids [M, K], but got: ", logits.sizes(), " and ",
                topk_idx.sizes());
    TORCH_CHECK(at::isIntegralType(topk_idx.scalar_type(), false), "the expert ids must be whole numbers, but got: ",
                topk_idx.dtype());
    const int64_t M = logits.size(0), N = logits.size(1), K = topk_idx.size(1);
    TORCH_CHECK(0 <= Ks && Ks < K && K <= N && N <= 1024,
                "0 <= shared experts < K <= N <= 1024 is needed, but got: Ks = ", Ks, ", K = ", K, ", N = ", N);
    TORCH_CHECK(!(cu_seqlens && seq_len), "give cu_seqlens or seq_len, not both");
    no_tangent("balance_loss", logits);
    const c10::cuda::CUDAGuard guard(dev);
    const Tensor idx = whole32(topk_idx, -1, N);
    OptTensor cu;
    int64_t S = 0, B = 0;
    if (cu_seqlens) {
        require_device(*cu_seqlens, dev);
        TORCH_CHECK(cu_seqlens->dim() == 1 && cu_seqlens->size(0) >= 2 &&
                        at::isIntegralType(cu_seqlens->scalar_type(), false),
                    "cu_seqlens must be whole numbers [B + 1], but got: ", cu_seqlens->sizes(), " in ",
                    cu_seqlens->dtype());
        cu = whole32(*cu_seqlens, 0, M);
        B = cu->size(0) - 1;
    } else {
        const int64_t most = M > 0 ? M : 1;
        S = seq_len ? *seq_len : most;
        TORCH_CHECK(S > 0, "seq_len must be positive, but got: ", S);
        S = S < most ? S : most;
        B = (most + S - 1) / S;
    }
    TORCH_CHECK(B <= 65535, "at most 65535 sequences, but got: ", B);
    return BalanceFunction::apply(logits, idx, Ks, balance_coef, z_coef, cu, S, B);
}

// ------------------------------------------------------------------------------------------------ 8-bit experts
void weight_check(const Tensor& t, const char* name, at::IntArrayRef shape, at::ScalarType type, const at::Device& dev) {
    require_device(t, dev);
    TORCH_CHECK(t.sizes() == shape && t.scalar_type() == type && t.is_contiguous(), name, " must be a contiguous ", type,
                " of shape ", shape, ", but got: ", t.dtype(), " of shape ", t.sizes(), ", strides ", t.strides());
    TORCH_CHECK(is_aligned(t), name, " must start on a 16-byte boundary");
}

// x: float rows, or e4m3 rows with their scales.  [y, tokens_per_expert]
std::vector<Tensor> experts_forward(const Tensor& x, const OptTensor& scale, const Tensor& topk_idx, const Tensor& topk_w,
                                    const Tensor& W1, const Tensor& S1, const Tensor& W2, const Tensor& S2,
                                    int64_t stream_max_avg_rows, const Tensor& status) {
    const at::Device dev = cuda_device(x);
    require_device(topk_idx, dev);
    require_device(topk_w, dev);
    TORCH_CHECK(!(at::GradMode::is_enabled() && (x.requires_grad() || topk_w.requires_grad())),
                "8-bit experts have no backward pass: call them under torch.no_grad()");
    no_tangent("the forward pass of 8-bit experts", x, topk_w);
    TORCH_CHECK(W2.dim() == 3 && x.dim() == 2 && topk_idx.dim() == 2 && topk_idx.size(0) == x.size(0),
                "x must be [M, D], topk_idx_MK [M, K] and the weights [N, 2H, D] and [N, D, H], but got: ", x.sizes(), ", ",
                topk_idx.sizes(), ", ", W1.sizes(), " and ", W2.sizes());
    const int64_t N = W2.size(0), D = W2.size(1), H = W2.size(2), M = x.size(0), K = topk_idx.size(1);
    TORCH_CHECK(D > 0 && H > 0 && D % 16 == 0 && H % 16 == 0,
                "8-bit experts need D and H in multiples of 16, but got: D = ", D, ", H = ", H);
    const auto blocks = [](int64_t n) { return (n + kBlock - 1) / kBlock; };
    weight_check(W1, "W1_N2HD", {N, 2 * H, D}, at::kFloat8_e4m3fn, dev);
    weight_check(W2, "W2_NDH", {N, D, H}, at::kFloat8_e4m3fn, dev);
    weight_check(S1, "S1", {N, 2, blocks(H), blocks(D)}, at::kFloat8_e8m0fnu, dev);
    weight_check(S2, "S2", {N, blocks(D), blocks(H)}, at::kFloat8_e8m0fnu, dev);
    TORCH_CHECK(K >= 1 && K <= N, "each token needs 1 to N = ", N, " experts, but got K = ", K);
    TORCH_CHECK(topk_w.sizes() == topk_idx.sizes(), "topk_w_MK must be like topk_idx_MK, ", topk_idx.sizes(),
                ", but got: ", topk_w.sizes());
    TORCH_CHECK(at::isIntegralType(topk_idx.scalar_type(), false), "the expert ids must be whole numbers, but got: ",
                topk_idx.dtype());
    TORCH_CHECK(x.size(1) == D && at::isFloatingType(x.scalar_type()), "x must be floating-point [M, ", D,
                "], but got: ", x.dtype(), " ", x.sizes());
    const c10::cuda::CUDAGuard guard(dev);
    Tensor rows, sc;
    if (scale) {
        require_device(*scale, dev);
        TORCH_CHECK(x.scalar_type() == at::kFloat8_e4m3fn && scale->scalar_type() == at::kFloat8_e8m0fnu,
                    "8-bit rows are float8_e4m3fn with float8_e8m0fnu scales, but got: ", x.dtype(), " and ",
                    scale->dtype());
        TORCH_CHECK(scale->dim() == 2 && scale->size(0) == M && scale->size(1) == blocks(D), "the scales must be [", M,
                    ", ", blocks(D), "], but got: ", scale->sizes());
        rows = dense(x);
        sc = scale->contiguous();
    } else {
        TORCH_CHECK(type_code(x.scalar_type()) >= 0 || x.scalar_type() == at::kDouble,
                    "rows of ", x.dtype(), " need their scales: pass Fp8Rows");
        rows = dense(x.to(at::kBFloat16));
    }
    const Tensor idx = whole32(topk_idx, -1, N), w = topk_w.to(at::kFloat).contiguous();
    const auto opt = rows.options();
    Tensor y = at::empty({M, D}, opt.dtype(at::kBFloat16));
    if (M == 0) return {y, at::zeros({N}, opt.dtype(at::kLong))};
    Tensor sizes = at::empty({N}, opt.dtype(at::kLong));
    const int32_t m = i32(M, "M"), n = i32(N, "N"), k = i32(K, "K"), d = i32(D, "D"), h = i32(H, "H");
    const size_t bytes = api.momoe_fp8_experts_workspace_bytes(m, n, k, d, h);
    Tensor ws = at::empty({static_cast<int64_t>(bytes)}, opt.dtype(at::kByte));
    const auto u8 = [](const Tensor& t) { return static_cast<const uint8_t*>(data(t)); };
    check(api.momoe_fp8_experts_forward(rows.data_ptr(), u8(sc), idx.data_ptr<int32_t>(), w.data_ptr<float>(), m, n, k, d,
                                        h, u8(W1), u8(S1), u8(W2), u8(S2), i32(stream_max_avg_rows, "stream_max_avg_rows"),
                                        y.data_ptr(), sizes.data_ptr<int64_t>(), ws.data_ptr(), bytes,
                                        status.data_ptr<int32_t>(), stream_of(dev)),
          "momoe_fp8_experts_forward", api.momoe_fp8_experts_launches(m, n, k));
    return {y, sizes};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    using Release = pybind11::call_guard<pybind11::gil_scoped_release>;
    m.attr("built_for") = MOMOE_BUILT_FOR;
    m.def("bind", &bind);
    m.def("launches", [] { return n_launches.load(); });
    m.def("rms_norm", &rms_norm, Release());
    m.def("rms_norm_fp8", &rms_norm_fp8, Release());
    m.def("balance_loss", &balance_loss, Release());
    m.def("balance_forward", &balance_forward, Release());
    m.def("balance_backward", &balance_backward, Release());
    m.def("experts_forward", &experts_forward, Release());
}
