// PyTorch C++ extension over libqlka.so's C ABI: the pybind module the reference's packages import as `_ext`
// (Weighted_Abs_Sum/csrc/binding.cpp:442-453, Weighted_Laplace_Sum/csrc/binding.cpp:102-105), with the same function
// names, arguments, checks and TORCH_CHECK messages, plus the autograd Functions of weighted_abs_sum(_full)
// (Weighted_Abs_Sum/weighted_abs_sum/ops.py:72-104) in C++, so that neither a call nor its backward runs Python.
//
// Host code only: every computation is a libqlka.so entry point (the gfx950 kernels). Outputs and workspaces come from
// torch's caching allocator on q's device, launches go on that device's current stream under a device guard.
#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>

#include <cstdint>
#include <tuple>

#include "qlka.h"

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::tensor_list;

void check_rc(int rc) {
    if (rc != 0) {
        const char* msg = qlka_last_error();
        TORCH_CHECK(false, (msg && *msg) ? msg : "libqlka error");
    }
}

void* stream_of(const Tensor& t) { return (void*)at::hip::getCurrentHIPStream(t.device().index()).stream(); }

float* fptr(const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }
float* fptr(const OptTensor& t) { return (t.has_value() && t->defined()) ? t->data_ptr<float>() : nullptr; }

struct Dims { int P, D, N, M, C; };

// check_qkv of Weighted_Abs_Sum/csrc/binding.cpp:69-84, same messages
Dims check_qkv(const Tensor& q, const Tensor& k, const Tensor& v) {
    TORCH_CHECK(q.is_cuda() && k.is_cuda() && v.is_cuda(), "q, k, and v must be CUDA tensors");
    TORCH_CHECK(q.device() == k.device() && q.device() == v.device(), "q, k, and v must be on the same CUDA device");
    TORCH_CHECK(q.scalar_type() == at::kFloat && k.scalar_type() == at::kFloat && v.scalar_type() == at::kFloat,
                "q, k, and v must be float32");
    TORCH_CHECK(q.dim() == 3 && k.dim() == 3 && v.dim() == 3, "q, k, and v must be 3D tensors");
    TORCH_CHECK(q.size(0) == k.size(0) && q.size(0) == v.size(0), "Batch size of q, k, and v must match");
    TORCH_CHECK(q.size(1) == k.size(1), "q and k must have same feature dimension");
    TORCH_CHECK(k.size(2) == v.size(1), "k and v must have same length");
    TORCH_CHECK(q.is_contiguous() && k.is_contiguous() && v.is_contiguous(), "q, k, and v must be contiguous");
    const int64_t P = q.size(0), D = q.size(1), N = k.size(2), C = v.size(2), M = q.size(2);
    TORCH_CHECK(M > 0 && N > 0 && D > 0, "N, M and D must be > 0");
    TORCH_CHECK(1 <= C && C <= 128, "C (v.size(2)) must be in [1, 128]");
    TORCH_CHECK(N <= 131072 && M <= 131072, "N and M must be <= 131072");
    TORCH_CHECK(P * D * std::max(N, M) <= INT32_MAX, "P*D*max(N,M) must fit int32 (cub sort offsets)");
    return {(int)P, (int)D, (int)N, (int)M, (int)C};
}

// the g / g_w / g_u checks (binding.cpp:251-262, 388-393)
void check_grad(const char* name, const Tensor& g, const Tensor& q, at::IntArrayRef shape) {
    TORCH_CHECK(g.is_cuda() && g.device() == q.device(), name, " must be on q's CUDA device");
    TORCH_CHECK(g.scalar_type() == at::kFloat, name, " must be float32");
    if (shape.size() == 3) {
        TORCH_CHECK(g.dim() == 3, name, " must be 3D");
        TORCH_CHECK(g.sizes() == shape, name, " must have shape (P, M, C)");
    } else {
        TORCH_CHECK(g.dim() == 2 && g.sizes() == shape, name, " must have shape (P, M)");
    }
    TORCH_CHECK(g.is_contiguous(), name, " must be contiguous");
}

void check_path(int64_t path) {
    TORCH_CHECK(-1 <= path && path <= 1, "path must be -1 (auto), 0 (global) or 1 (fused)");
}

Tensor workspace(size_t bytes, const Tensor& like) {
    return at::empty({(int64_t)std::max<size_t>(bytes, 1)}, like.options().dtype(at::kByte));
}

Tensor empty_f(at::IntArrayRef shape, const Tensor& like) { return at::empty(shape, like.options()); }

// ---- weighted_abs_sum

std::tuple<Tensor, OptTensor> abs_forward(const Tensor& q, const Tensor& k, const Tensor& v, int64_t path, bool full) {
    const Dims d = check_qkv(q, k, v);
    check_path(path);
    c10::DeviceGuard guard(q.device());
    Tensor out = empty_f({d.P, d.M, d.C}, q);
    OptTensor out_u;
    if (full) out_u = empty_f({d.P, d.M}, q);
    Tensor ws = workspace(qlka_abs_fwd_ws_bytes(d.P, d.D, d.N, d.M, d.C), q);
    check_rc(qlka_abs_fwd(fptr(q), fptr(k), fptr(v), fptr(out), fptr(out_u), d.P, d.D, d.N, d.M, d.C, (int)path,
                          ws.data_ptr(), (size_t)ws.numel(), stream_of(q)));
    return {out, out_u};
}

Tensor weighted_abs_sum_forward(const Tensor& q, const Tensor& k, const Tensor& v, int64_t path) {
    return std::get<0>(abs_forward(q, k, v, path, false));
}

std::tuple<Tensor, Tensor> weighted_abs_sum_full_forward(const Tensor& q, const Tensor& k, const Tensor& v,
                                                         int64_t path) {
    auto r = abs_forward(q, k, v, path, true);
    return {std::get<0>(r), *std::get<1>(r)};
}

// forward that also keeps the sorted k and q (with their permutations) when the backward at this shape walks
std::tuple<Tensor, OptTensor, std::vector<Tensor>> abs_forward_keep(const Tensor& q, const Tensor& k, const Tensor& v,
                                                                    int64_t path, bool full) {
    const Dims d = check_qkv(q, k, v);
    check_path(path);
    c10::DeviceGuard guard(q.device());
    Tensor out = empty_f({d.P, d.M, d.C}, q);
    OptTensor out_u;
    if (full) out_u = empty_f({d.P, d.M}, q);
    Tensor ws = workspace(qlka_abs_fwd_ws_bytes(d.P, d.D, d.N, d.M, d.C), q);
    std::vector<Tensor> srt;
    if (!qlka_abs_bwd_walks(d.P, d.N, d.M)) {
        check_rc(qlka_abs_fwd(fptr(q), fptr(k), fptr(v), fptr(out), fptr(out_u), d.P, d.D, d.N, d.M, d.C, (int)path,
                              ws.data_ptr(), (size_t)ws.numel(), stream_of(q)));
        return {out, out_u, srt};
    }
    const auto i32 = q.options().dtype(at::kInt);
    srt = {empty_f({d.P, d.D, d.N}, q), at::empty({d.P, d.D, d.N}, i32), empty_f({d.P, d.D, d.M}, q),
           at::empty({d.P, d.D, d.M}, i32)};
    // the walk's range states and bounds too, so that the backward's grad_q walk skips its range passes
    Tensor states = at::empty({(int64_t)qlka_abs_keep_state_bytes(d.P, d.D, d.N, d.M, d.C)},
                              q.options().dtype(at::kByte));
    int kept = 0;
    check_rc(qlka_abs_fwd_keep(fptr(q), fptr(k), fptr(v), fptr(out), fptr(out_u), d.P, d.D, d.N, d.M, d.C, (int)path,
                               fptr(srt[0]), (uint32_t*)srt[1].data_ptr<int32_t>(), fptr(srt[2]),
                               (uint32_t*)srt[3].data_ptr<int32_t>(), states.numel() ? states.data_ptr() : nullptr,
                               &kept, ws.data_ptr(), (size_t)ws.numel(), stream_of(q)));
    if (!kept) srt.clear();
    else if (kept & 2) srt.push_back(states);
    return {out, out_u, srt};
}

// The dense route's forward that keeps its kernel matrix A (P, M, (N + 3) & ~3) for the backward, and that backward
// (qlka_abs_fwd_dense_keep / qlka_abs_bwd_dense_kept): only where qlka_abs_dense_keep_bytes is nonzero.
std::tuple<Tensor, OptTensor, Tensor> abs_forward_dense_keep(const Tensor& q, const Tensor& k, const Tensor& v,
                                                             bool full) {
    const Dims d = check_qkv(q, k, v);
    c10::DeviceGuard guard(q.device());
    Tensor out = empty_f({d.P, d.M, d.C}, q);
    OptTensor out_u;
    if (full) out_u = empty_f({d.P, d.M}, q);
    Tensor A = empty_f({d.P, d.M, (d.N + 3) & ~int64_t(3)}, q);
    check_rc(qlka_abs_fwd_dense_keep(fptr(q), fptr(k), fptr(v), fptr(out), fptr(out_u), fptr(A), d.P, d.D, d.N, d.M,
                                     d.C, stream_of(q)));
    return {out, out_u, A};
}

std::tuple<Tensor, Tensor, Tensor> abs_backward_dense_kept(const Tensor& q, const Tensor& k, const Tensor& v,
                                                           const Tensor& g_w, const OptTensor& g_u, const Tensor& A) {
    const Dims d = check_qkv(q, k, v);
    check_grad("g_w", g_w, q, {d.P, d.M, d.C});
    if (g_u.has_value()) check_grad("g_u", *g_u, q, {d.P, d.M});
    TORCH_CHECK(A.sizes() == at::IntArrayRef({d.P, d.M, (d.N + 3) & ~int64_t(3)}) && A.is_contiguous(),
                "kept kernel matrix does not match q and k");
    c10::DeviceGuard guard(q.device());
    Tensor gq = empty_f({d.P, d.D, d.M}, q), gk = empty_f({d.P, d.D, d.N}, q), gv = empty_f({d.P, d.N, d.C}, q);
    check_rc(qlka_abs_bwd_dense_kept(fptr(q), fptr(k), fptr(v), fptr(g_w), fptr(g_u), fptr(gq), fptr(gk), fptr(gv),
                                     fptr(A), d.P, d.D, d.N, d.M, d.C, stream_of(q)));
    return {gq, gk, gv};
}

std::tuple<Tensor, Tensor, Tensor> abs_backward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g_w,
                                                const OptTensor& g_u) {
    const Dims d = check_qkv(q, k, v);
    check_grad("g_w", g_w, q, {d.P, d.M, d.C});
    if (g_u.has_value()) check_grad("g_u", *g_u, q, {d.P, d.M});
    c10::DeviceGuard guard(q.device());
    Tensor gq = empty_f({d.P, d.D, d.M}, q), gk = empty_f({d.P, d.D, d.N}, q), gv = empty_f({d.P, d.N, d.C}, q);
    Tensor ws = workspace(qlka_abs_bwd_ws_bytes(d.P, d.D, d.N, d.M, d.C), q);
    check_rc(qlka_abs_bwd(fptr(q), fptr(k), fptr(v), fptr(g_w), fptr(g_u), fptr(gq), fptr(gk), fptr(gv), d.P, d.D,
                          d.N, d.M, d.C, ws.data_ptr(), (size_t)ws.numel(), stream_of(q)));
    return {gq, gk, gv};
}

std::tuple<Tensor, Tensor, Tensor> weighted_abs_sum_backward(const Tensor& q, const Tensor& k, const Tensor& v,
                                                             const Tensor& g_w) {
    return abs_backward(q, k, v, g_w, c10::nullopt);
}

std::tuple<Tensor, Tensor, Tensor> weighted_abs_sum_full_backward(const Tensor& q, const Tensor& k, const Tensor& v,
                                                                  const Tensor& g_w, const Tensor& g_u) {
    return abs_backward(q, k, v, g_w, g_u);
}

std::tuple<Tensor, Tensor, Tensor> abs_backward_sorted(const Tensor& q, const Tensor& k, const Tensor& v,
                                                       const Tensor& g_w, const OptTensor& g_u,
                                                       const std::vector<Tensor>& srt) {
    const Dims d = check_qkv(q, k, v);
    check_grad("g_w", g_w, q, {d.P, d.M, d.C});
    if (g_u.has_value()) check_grad("g_u", *g_u, q, {d.P, d.M});
    TORCH_CHECK((srt.size() == 4 || srt.size() == 5) && srt[0].sizes() == at::IntArrayRef({d.P, d.D, d.N}) &&
                    srt[1].sizes() == at::IntArrayRef({d.P, d.D, d.N}) &&
                    srt[2].sizes() == at::IntArrayRef({d.P, d.D, d.M}) &&
                    srt[3].sizes() == at::IntArrayRef({d.P, d.D, d.M}),
                "sorted arrays do not match q and k");
    const void* states = nullptr;
    if (srt.size() == 5) {
        TORCH_CHECK(srt[4].numel() == (int64_t)qlka_abs_keep_state_bytes(d.P, d.D, d.N, d.M, d.C) &&
                        srt[4].scalar_type() == at::kByte && srt[4].is_contiguous(),
                    "kept range states do not match q and k");
        states = srt[4].data_ptr();
    }
    c10::DeviceGuard guard(q.device());
    Tensor gq = empty_f({d.P, d.D, d.M}, q), gk = empty_f({d.P, d.D, d.N}, q), gv = empty_f({d.P, d.N, d.C}, q);
    Tensor ws = workspace(qlka_abs_bwd_ws_bytes(d.P, d.D, d.N, d.M, d.C), q);
    check_rc(qlka_abs_bwd_sorted(fptr(q), fptr(k), fptr(v), fptr(g_w), fptr(g_u), fptr(gq), fptr(gk), fptr(gv), d.P,
                                 d.D, d.N, d.M, d.C, fptr(srt[0]), (const uint32_t*)srt[1].data_ptr<int32_t>(),
                                 fptr(srt[2]), (const uint32_t*)srt[3].data_ptr<int32_t>(), states, ws.data_ptr(),
                                 (size_t)ws.numel(), stream_of(q)));
    return {gq, gk, gv};
}

Tensor weighted_sgn_sum_forward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g) {
    const Dims d = check_qkv(q, k, v);
    check_grad("g", g, q, {d.P, d.M, d.C});
    c10::DeviceGuard guard(q.device());
    Tensor out = empty_f({d.P, d.D, d.M}, q);
    Tensor ws = workspace(qlka_sgn_fwd_ws_bytes(d.P, d.D, d.N, d.M, d.C), q);
    check_rc(qlka_sgn_fwd(fptr(q), fptr(k), fptr(v), fptr(g), fptr(out), d.P, d.D, d.N, d.M, d.C, ws.data_ptr(),
                          (size_t)ws.numel(), stream_of(q)));
    return out;
}

// ---- dense evaluation (the "keops" route)

std::tuple<Tensor, OptTensor> direct_forward(const Tensor& q, const Tensor& k, const Tensor& v, bool full) {
    const Dims d = check_qkv(q, k, v);
    c10::DeviceGuard guard(q.device());
    Tensor out = empty_f({d.P, d.M, d.C}, q);
    OptTensor out_u;
    if (full) out_u = empty_f({d.P, d.M}, q);
    check_rc(qlka_direct_fwd(0, fptr(q), fptr(k), fptr(v), fptr(out), fptr(out_u), d.P, d.D, d.N, d.M, d.C,
                             stream_of(q)));
    return {out, out_u};
}

std::tuple<Tensor, Tensor, Tensor> direct_backward(const Tensor& q, const Tensor& k, const Tensor& v,
                                                   const Tensor& g_w, const OptTensor& g_u, double tie) {
    const Dims d = check_qkv(q, k, v);
    check_grad("g_w", g_w, q, {d.P, d.M, d.C});
    if (g_u.has_value()) check_grad("g_u", *g_u, q, {d.P, d.M});
    c10::DeviceGuard guard(q.device());
    Tensor gq = empty_f({d.P, d.D, d.M}, q), gk = empty_f({d.P, d.D, d.N}, q), gv = empty_f({d.P, d.N, d.C}, q);
    check_rc(qlka_direct_bwd((float)tie, fptr(q), fptr(k), fptr(v), fptr(g_w), fptr(g_u), fptr(gq), fptr(gk),
                             fptr(gv), d.P, d.D, d.N, d.M, d.C, stream_of(q)));
    return {gq, gk, gv};
}

Tensor direct_sgn(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, double tie) {
    const Dims d = check_qkv(q, k, v);
    check_grad("g", g, q, {d.P, d.M, d.C});
    c10::DeviceGuard guard(q.device());
    Tensor out = empty_f({d.P, d.D, d.M}, q);
    check_rc(qlka_direct_sgn((float)tie, fptr(q), fptr(k), fptr(v), fptr(g), fptr(out), d.P, d.D, d.N, d.M, d.C,
                             stream_of(q)));
    return out;
}

// ---- weighted_laplace_sum (Weighted_Laplace_Sum/csrc/binding.cpp:63-105, its messages)

std::tuple<Tensor, Tensor> weighted_laplace_sum_forward(const Tensor& q, const Tensor& k, const Tensor& v) {
    TORCH_CHECK(q.is_cuda() && k.is_cuda() && v.is_cuda(), "q, k and v must be CUDA tensors");
    TORCH_CHECK(q.device() == k.device() && q.device() == v.device(), "q, k and v must be on one device");
    TORCH_CHECK(q.scalar_type() == at::kFloat && k.scalar_type() == at::kFloat && v.scalar_type() == at::kFloat,
                "q, k and v must be float32");
    TORCH_CHECK(q.dim() == 3 && k.dim() == 3 && v.dim() == 3, "q, k and v must be 3D");
    TORCH_CHECK(q.size(0) == k.size(0) && q.size(0) == v.size(0), "batch size must match");
    TORCH_CHECK(q.size(1) == k.size(1), "q and k must have the same feature dimension");
    TORCH_CHECK(k.size(2) == v.size(1), "k and v must have the same length");
    TORCH_CHECK(q.is_contiguous() && k.is_contiguous() && v.is_contiguous(), "q, k and v must be contiguous");
    const int64_t P = q.size(0), D = q.size(1), N = k.size(2), C = v.size(2), M = q.size(2);
    TORCH_CHECK(M > 0 && N > 0 && D > 0, "N, M and D must be > 0");
    TORCH_CHECK(1 <= C && C <= 128, "C (v.size(2)) must be in [1, 128]");
    TORCH_CHECK(N <= 131072 && M <= 131072, "N and M must be <= 131072");
    TORCH_CHECK(P * D * std::max(N, M) <= INT32_MAX, "P*D*max(N,M) must fit int32 (cub sort offsets)");
    c10::DeviceGuard guard(q.device());
    Tensor out = empty_f({P, M, C}, q), out_u = empty_f({P, M}, q);
    Tensor ws = workspace(qlka_laplace_fwd_ws_bytes((int)P, (int)D, (int)N, (int)M, (int)C), q);
    check_rc(qlka_laplace_fwd(fptr(q), fptr(k), fptr(v), fptr(out), fptr(out_u), (int)P, (int)D, (int)N, (int)M,
                              (int)C, ws.data_ptr(), (size_t)ws.numel(), stream_of(q)));
    return {out, out_u};
}

// ---- autograd (Weighted_Abs_Sum/weighted_abs_sum/ops.py:72-104)
//
// path: -1 / 0 / 1 as the C entries take it, or DIRECT for the "keops" route (dense forward on contiguous copies,
// its gradient with sign(0) = 0). keep: keep the forward's sorts for the backward when a gradient is wanted.
constexpr int64_t DIRECT = 2;

struct AbsSumFn : public torch::autograd::Function<AbsSumFn> {
    static tensor_list forward(AutogradContext* ctx, Tensor q, Tensor k, Tensor v, int64_t path, bool full,
                               bool keep) {
        ctx->set_materialize_grads(false);
        ctx->saved_data["path"] = path;
        ctx->saved_data["full"] = full;
        std::vector<Tensor> srt;
        Tensor out;
        OptTensor out_u;
        bool dense_a = false;                 // srt holds the dense route's kernel matrix
        if (path == DIRECT) {
            q = q.contiguous();
            k = k.contiguous();
            v = v.contiguous();
            std::tie(out, out_u) = direct_forward(q, k, v, full);
        } else if (keep && q.dim() == 3 && k.dim() == 3 && v.dim() == 3 &&     // else check_qkv raises below
                   qlka_abs_dense_keep_bytes((int)q.size(0), (int)q.size(1), (int)k.size(2), (int)q.size(2),
                                             (int)v.size(2)) > 0) {
            Tensor A;
            std::tie(out, out_u, A) = abs_forward_dense_keep(q, k, v, full);
            srt = {A};
            dense_a = true;
        } else if (keep) {
            std::tie(out, out_u, srt) = abs_forward_keep(q, k, v, path, full);
        } else {
            std::tie(out, out_u) = abs_forward(q, k, v, path, full);
        }
        ctx->saved_data["sorted"] = !srt.empty() && !dense_a;
        ctx->saved_data["dense_a"] = dense_a;
        std::vector<Tensor> saved = {q, k, v};
        saved.insert(saved.end(), srt.begin(), srt.end());
        ctx->save_for_backward(saved);
        if (full) return {out, *out_u};
        return {out};
    }

    static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor& q = saved[0];
        const Tensor& k = saved[1];
        const Tensor& v = saved[2];
        const int64_t path = ctx->saved_data["path"].toInt();
        const bool full = ctx->saved_data["full"].toBool();
        Tensor g_w = grads[0];
        OptTensor g_u;
        if (full && grads.size() > 1 && grads[1].defined()) g_u = grads[1].contiguous();
        if (!g_w.defined()) g_w = at::zeros({q.size(0), q.size(2), v.size(2)}, q.options());
        g_w = g_w.contiguous();
        Tensor gq, gk, gv;
        if (path == DIRECT)
            std::tie(gq, gk, gv) = direct_backward(q, k, v, g_w, g_u, 0.0);
        else if (ctx->saved_data["dense_a"].toBool())
            std::tie(gq, gk, gv) = abs_backward_dense_kept(q, k, v, g_w, g_u, saved[3]);
        else if (ctx->saved_data["sorted"].toBool())
            std::tie(gq, gk, gv) = abs_backward_sorted(q, k, v, g_w, g_u,
                                                       std::vector<Tensor>(saved.begin() + 3, saved.end()));
        else
            std::tie(gq, gk, gv) = abs_backward(q, k, v, g_w, g_u);
        return {gq, gk, gv, Tensor(), Tensor(), Tensor()};
    }
};

std::vector<Tensor> abs_sum_autograd(const Tensor& q, const Tensor& k, const Tensor& v, int64_t path, bool full,
                                     bool keep) {
    return AbsSumFn::apply(q, k, v, path, full, keep);
}

// ---- softmax attention to a sequence of another length, and the bucketed position bias (qlka_softmax_*,
// qlka_bias_map_*)

struct SoftmaxCall {
    Tensor q, k, v, table, keep;      // table and keep may be undefined
    double scale;
    bool causal;
    int64_t start;
    std::vector<int64_t> border;
    bool both;
};

int64_t bucket_count(const std::vector<int64_t>& border, bool both) {
    return ((int64_t)border.size() + 1) * (both ? 2 : 1);
}

void check_table(const Tensor& table, int64_t heads, const std::vector<int64_t>& border, bool both) {
    TORCH_CHECK(table.scalar_type() == at::kFloat, "table must be float32");
    TORCH_CHECK(table.dim() == 2 && table.size(0) == bucket_count(border, both) && table.size(1) == heads,
                "table must be (num_buckets, H) = (", bucket_count(border, both), ", ", heads, "), got ",
                table.sizes());
}

void check_start(int64_t start) { TORCH_CHECK(std::abs(start) <= (1 << 28), "|start| must be <= 2^28"); }

void check_softmax(const SoftmaxCall& c) {
    const Tensor &q = c.q, &k = c.k, &v = c.v;
    TORCH_CHECK(q.is_cuda() && k.is_cuda() && v.is_cuda(), "q, k and v must be CUDA tensors");
    TORCH_CHECK(q.device() == k.device() && q.device() == v.device(), "q, k and v must be on one device");
    TORCH_CHECK(q.scalar_type() == at::kFloat || q.scalar_type() == at::kBFloat16, "q must be float32 or bfloat16");
    TORCH_CHECK(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(),
                "q, k and v must have the same dtype");
    TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && v.dim() == 4, "q, k and v must be 4D: (B, heads, length, D)");
    TORCH_CHECK(k.sizes() == v.sizes(), "k and v must have the same shape");
    TORCH_CHECK(q.size(0) == k.size(0), "batch size must match");
    TORCH_CHECK(q.size(3) == k.size(3), "q and k must have the same head dimension");
    TORCH_CHECK(q.size(1) >= 1 && k.size(1) >= 1 && q.size(1) % k.size(1) == 0,
                "the heads of q must be a multiple of those of k and v");
    TORCH_CHECK(1 <= q.size(3) && q.size(3) <= 128, "the head dimension must be in [1, 128]");
    TORCH_CHECK(q.size(2) <= (1 << 28) && k.size(2) <= (1 << 28), "lengths must be <= 2^28");
    TORCH_CHECK(q.size(0) <= INT32_MAX && q.size(1) <= INT32_MAX &&
                    (double)q.size(0) * q.size(1) * q.size(2) <= INT32_MAX &&
                    (double)k.size(0) * k.size(1) * k.size(2) <= INT32_MAX,
                "batch * heads * length must fit int32");
    check_start(c.start);
    if (c.table.defined()) {
        TORCH_CHECK(c.table.device() == q.device(), "table must be on q's device");
        check_table(c.table, q.size(1), c.border, c.both);
        TORCH_CHECK(c.table.is_contiguous(), "table must be contiguous");
    }
    if (c.keep.defined()) {
        TORCH_CHECK(c.keep.device() == q.device(), "keep must be on q's device");
        TORCH_CHECK(c.keep.scalar_type() == at::kBool || c.keep.scalar_type() == at::kByte,
                    "keep must be bool or uint8");
        TORCH_CHECK(c.keep.dim() == 2 && c.keep.size(0) == q.size(0) && c.keep.size(1) == k.size(2),
                    "keep must be (B, N) = (", q.size(0), ", ", k.size(2), "), got ", c.keep.sizes());
    }
}

// whether the kernels can read t's rows: their elements next to each other, each row at a multiple of 16 bytes
bool readable(const Tensor& t) {
    const int64_t piece = 16 / t.element_size();
    if (t.stride(3) != 1 || (uintptr_t)t.data_ptr() % 16) return false;
    for (int i = 0; i < 3; ++i)
        if (t.size(i) > 1 && t.stride(i) % piece) return false;
    return true;
}
Tensor packed_rows(const Tensor& t) {
    return t.numel() == 0 || readable(t) ? t : t.clone(at::MemoryFormat::Contiguous);
}
// an output laid out as t is
Tensor empty_rows(const Tensor& t) {
    Tensor r = at::empty_like(t);
    return r.numel() == 0 || readable(r) ? r : at::empty(t.sizes(), t.options());
}
void set_strides(int64_t* to, const Tensor& t) {
    for (int i = 0; i < 3; ++i) to[i] = t.stride(i);
}

// Sizes, inputs and the bias of a call; border has to outlive the arguments.
qlka_softmax_args softmax_args(const SoftmaxCall& c, const std::vector<int>& border) {
    qlka_softmax_args a{};
    a.dtype = c.q.scalar_type() == at::kFloat ? QLKA_F32 : QLKA_BF16;
    a.B = (int)c.q.size(0); a.H = (int)c.q.size(1); a.G = (int)c.k.size(1);
    a.M = (int)c.q.size(2); a.N = (int)c.k.size(2); a.D = (int)c.q.size(3);
    a.causal = c.causal;
    a.start = (int)c.start;
    a.scale = (float)c.scale;
    a.q = c.q.data_ptr(); a.k = c.k.data_ptr(); a.v = c.v.data_ptr();
    set_strides(a.q_stride, c.q); set_strides(a.k_stride, c.k); set_strides(a.v_stride, c.v);
    if (c.keep.defined()) {
        a.keep = (const uint8_t*)c.keep.data_ptr();
        a.keep_stride = c.keep.stride(0);
    }
    if (c.table.defined()) {
        a.table = c.table.data_ptr<float>();
        a.border = border.data();
        a.num_borders = (int)border.size();
        a.bidirectional = c.both;
    }
    return a;
}

// (out, out before its rounding to bfloat16, the rows' log sums in two floats); the last where a gradient will be
// wanted, the second where one through the scores will (v's needs none)
std::tuple<Tensor, Tensor, Tensor> softmax_forward(SoftmaxCall& c, bool train, bool train_scores, bool train_table) {
    check_softmax(c);
    c10::DeviceGuard guard(c.q.device());
    c.q = packed_rows(c.q);
    c.k = packed_rows(c.k);
    c.v = packed_rows(c.v);
    if (c.keep.defined() && c.keep.size(1) > 1 && c.keep.stride(1) != 1) c.keep = c.keep.contiguous();
    Tensor out = empty_rows(c.q), full, lse;
    const std::vector<int> border(c.border.begin(), c.border.end());
    qlka_softmax_args a = softmax_args(c, border);
    a.out = out.data_ptr();
    set_strides(a.out_stride, out);
    if (train) {
        lse = at::empty({2, a.B, a.H, a.M}, c.q.options().dtype(at::kFloat));
        a.log_sums = lse.data_ptr<float>();
        if (a.dtype == QLKA_BF16 && train_scores) {
            a.table_kept = !train_table;
            full = at::empty({a.B, a.H, a.M, a.D}, lse.options());
            a.out_full = full.data_ptr<float>();
        }
    }
    const size_t bytes = qlka_softmax_fwd_ws_bytes(&a);
    Tensor ws;
    if (bytes) ws = workspace(bytes, c.q);
    check_rc(qlka_softmax_fwd(&a, bytes ? ws.data_ptr() : nullptr, bytes, stream_of(c.q)));
    return {out, full, lse};
}

struct SoftmaxFn : public torch::autograd::Function<SoftmaxFn> {
    static Tensor forward(AutogradContext* ctx, Tensor q, Tensor k, Tensor v, OptTensor table_, OptTensor keep_,
                          double scale, bool causal, int64_t start, std::vector<int64_t> border, bool both) {
        ctx->set_materialize_grads(false);
        const Tensor table = table_.value_or(Tensor()), keep = keep_.value_or(Tensor());
        SoftmaxCall c{q, k, v, table, keep, scale, causal, start, border, both};
        Tensor out, full, lse;
        const bool train_table = table.defined() && table.requires_grad();
        const bool train_scores = q.requires_grad() || k.requires_grad() || train_table;
        std::tie(out, full, lse) = softmax_forward(c, true, train_scores, train_table);
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["causal"] = causal;
        ctx->saved_data["start"] = start;
        ctx->saved_data["border"] = border;
        ctx->saved_data["both"] = both;
        ctx->save_for_backward({c.q, c.k, c.v, c.table, c.keep, out, full, lse});
        return out;
    }

    static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "softmax_attention has no second derivative");
        tensor_list r(10);
        if (!grads[0].defined()) return r;
        const auto s = ctx->get_saved_variables();
        const SoftmaxCall c{s[0], s[1], s[2], s[3], s[4], ctx->saved_data["scale"].toDouble(),
                            ctx->saved_data["causal"].toBool(), ctx->saved_data["start"].toInt(),
                            ctx->saved_data["border"].toIntVector(), ctx->saved_data["both"].toBool()};
        const Tensor &out = s[5], &full = s[6], &lse = s[7];
        c10::DeviceGuard guard(c.q.device());
        const std::vector<int> border(c.border.begin(), c.border.end());
        qlka_softmax_args a = softmax_args(c, border);
        const Tensor g = packed_rows(grads[0]);
        a.out = out.data_ptr();
        set_strides(a.out_stride, out);
        if (full.defined()) a.out_full = full.data_ptr<float>();
        a.log_sums = lse.data_ptr<float>();
        a.g_out = g.data_ptr();
        set_strides(a.g_out_stride, g);
        if (ctx->needs_input_grad(0)) {
            r[0] = empty_rows(c.q);
            a.g_q = r[0].data_ptr();
            set_strides(a.g_q_stride, r[0]);
        }
        if (ctx->needs_input_grad(1) || ctx->needs_input_grad(2)) {
            r[1] = empty_rows(c.k);
            r[2] = empty_rows(c.v);
            a.g_k = r[1].data_ptr();
            a.g_v = r[2].data_ptr();
            set_strides(a.g_k_stride, r[1]);
            set_strides(a.g_v_stride, r[2]);
        }
        if (c.table.defined() && ctx->needs_input_grad(3)) {
            r[3] = at::empty_like(c.table);
            a.g_table = r[3].data_ptr<float>();
        }
        const size_t bytes = qlka_softmax_bwd_ws_bytes(&a);
        Tensor ws;
        if (bytes) ws = workspace(bytes, c.q);
        check_rc(qlka_softmax_bwd(&a, bytes ? ws.data_ptr() : nullptr, bytes, stream_of(c.q)));
        return r;
    }
};

Tensor softmax_attention(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& table,
                         const OptTensor& keep, double scale, bool causal, int64_t start,
                         const std::vector<int64_t>& border, bool both) {
    // a call without a gradient goes around the autograd function, which would refuse a tangent
    for (const Tensor& t : {q, k, v, table.value_or(Tensor())})
        TORCH_CHECK(!t.defined() || !t._fw_grad(0).defined(), "softmax_attention has no forward-mode derivative");
    if (q.dim() == 4 && k.dim() == 4 && v.dim() == 4 && q.size(3) % 8 && q.size(3) == k.size(3) &&
        q.size(3) == v.size(3)) {
        // zeros up to a multiple of 8 change no product
        const auto padded = [&](const Tensor& t) { return at::constant_pad_nd(t, {0, 8 - t.size(3) % 8}); };
        return softmax_attention(padded(q), padded(k), padded(v), table, keep, scale, causal, start, border, both)
            .narrow(3, 0, q.size(3));
    }
    const Tensor t = table.value_or(Tensor()), m = keep.value_or(Tensor());
    if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad() ||
                                       (t.defined() && t.requires_grad())))
        return SoftmaxFn::apply(q, k, v, table, keep, scale, causal, start, border, both);
    SoftmaxCall c{q, k, v, t, m, scale, causal, start, border, both};
    return std::get<0>(softmax_forward(c, false, false, false));
}

struct BiasMapFn : public torch::autograd::Function<BiasMapFn> {
    static Tensor forward(AutogradContext* ctx, Tensor table, int64_t M, int64_t N, int64_t start,
                          std::vector<int64_t> border, bool both) {
        TORCH_CHECK(table.is_cuda(), "table must be a CUDA tensor");
        TORCH_CHECK(table.dim() == 2 && table.size(1) >= 1, "table must be (num_buckets, H)");
        check_table(table, table.size(1), border, both);
        TORCH_CHECK(M >= 0 && N >= 0 && M <= (1 << 21) && N <= (1 << 21), "lengths must be in [0, 2^21]");
        check_start(start);
        c10::DeviceGuard guard(table.device());
        const Tensor t = table.contiguous();
        const std::vector<int> b(border.begin(), border.end());
        Tensor out = at::empty({t.size(1), M, N}, t.options());
        check_rc(qlka_bias_map_fwd(t.data_ptr<float>(), b.data(), (int)b.size(), both, out.data_ptr<float>(),
                                   (int)t.size(1), (int)M, (int)N, (int)start, stream_of(t)));
        ctx->saved_data["start"] = start;
        ctx->saved_data["border"] = border;
        ctx->saved_data["both"] = both;
        return out;
    }

    static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "relative_bias has no second derivative");
        const Tensor g = grads[0].contiguous();
        const std::vector<int64_t> border = ctx->saved_data["border"].toIntVector();
        const bool both = ctx->saved_data["both"].toBool();
        const std::vector<int> b(border.begin(), border.end());
        const int H = (int)g.size(0), M = (int)g.size(1), N = (int)g.size(2);
        c10::DeviceGuard guard(g.device());
        Tensor gt = at::empty({bucket_count(border, both), H}, g.options());
        const size_t bytes = qlka_bias_map_bwd_ws_bytes((int)b.size(), both, H, M, N);
        Tensor ws = workspace(bytes, g);
        check_rc(qlka_bias_map_bwd(g.data_ptr<float>(), b.data(), (int)b.size(), both, gt.data_ptr<float>(), H, M, N,
                                   (int)ctx->saved_data["start"].toInt(), ws.data_ptr(), bytes, stream_of(g)));
        return {gt, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

Tensor relative_bias(const Tensor& table, int64_t M, int64_t N, int64_t start, const std::vector<int64_t>& border,
                     bool both) {
    return BiasMapFn::apply(table, M, N, start, border, both);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    namespace py = pybind11;
    m.doc() = "weighted_abs_sum / weighted_laplace_sum entry points over libqlka.so (gfx950)";
    m.def("weighted_abs_sum_forward", &weighted_abs_sum_forward, py::arg("q"), py::arg("k"), py::arg("v"),
          py::arg("path") = -1, "out[p,m,c] = sum_{n,d} |k[p,d,n] - q[p,d,m]| * v[p,n,c] (binding.cpp:229-233)");
    m.def("weighted_abs_sum_full_forward", &weighted_abs_sum_full_forward, py::arg("q"), py::arg("k"), py::arg("v"),
          py::arg("path") = -1, "(out_w, out_u), out_u[p,m] = sum_{n,d} |k - q| (binding.cpp:235-239)");
    m.def("weighted_abs_sum_backward", &weighted_abs_sum_backward, py::arg("q"), py::arg("k"), py::arg("v"),
          py::arg("g_w"), "(grad_q, grad_k, grad_v) of weighted_abs_sum (binding.cpp:370-374)");
    m.def("weighted_abs_sum_full_backward", &weighted_abs_sum_full_backward, py::arg("q"), py::arg("k"),
          py::arg("v"), py::arg("g_w"), py::arg("g_u"),
          "(grad_q, grad_k, grad_v) of weighted_abs_sum_full (binding.cpp:376-380)");
    m.def("weighted_sgn_sum_forward", &weighted_sgn_sum_forward, py::arg("q"), py::arg("k"), py::arg("v"),
          py::arg("g"), "out[p,d,m] = sum_n sgn(k - q) dot(v[n], g[m]), a tie counted +1 (binding.cpp:383-439)");
    m.def("weighted_abs_sum_forward_keep", &abs_forward_keep, py::arg("q"), py::arg("k"), py::arg("v"),
          py::arg("path"), py::arg("full"),
          "(out_w, out_u or None, [k_sorted, k_perm, q_sorted, q_perm (, range states)] or []): the forward that "
          "keeps its sorts (and, when it walked, its range states) when the backward at this shape walks "
          "(qlka_abs_fwd_keep)");
    m.def("weighted_abs_sum_backward_sorted", &abs_backward_sorted, py::arg("q"), py::arg("k"), py::arg("v"),
          py::arg("g_w"), py::arg("g_u"), py::arg("srt"),
          "the backward over the sorts a weighted_abs_sum_forward_keep left (qlka_abs_bwd_sorted)");
    m.def("weighted_abs_sum_direct_forward", &direct_forward, py::arg("q"), py::arg("k"), py::arg("v"),
          py::arg("full"), "dense (out_w, out_u or None) without a sort (qlka_direct_fwd)");
    m.def("weighted_abs_sum_direct_backward", &direct_backward, py::arg("q"), py::arg("k"), py::arg("v"),
          py::arg("g_w"), py::arg("g_u"), py::arg("tie"), "dense backward with sign(0) = tie (qlka_direct_bwd)");
    m.def("weighted_sgn_sum_direct", &direct_sgn, py::arg("q"), py::arg("k"), py::arg("v"), py::arg("g"),
          py::arg("tie"), "dense weighted_sgn_sum with sign(0) = tie (qlka_direct_sgn)");
    m.def("weighted_laplace_sum_forward", &weighted_laplace_sum_forward, py::arg("q"), py::arg("k"), py::arg("v"),
          "(out_w, out_u) of the weighted Laplace sum (Weighted_Laplace_Sum/csrc/binding.cpp:102-105)");
    m.def("abs_sum_autograd", &abs_sum_autograd, py::arg("q"), py::arg("k"), py::arg("v"), py::arg("path"),
          py::arg("full"), py::arg("keep"),
          "differentiable weighted_abs_sum (full=False: [out]) / weighted_abs_sum_full ([out_w, out_u]); path "
          "-1/0/1, or 2 for the dense route with sign(0) = 0 in the backward");
    m.def("softmax_attention", &softmax_attention, py::arg("q"), py::arg("k"), py::arg("v"), py::arg("table"),
          py::arg("keep"), py::arg("scale"), py::arg("causal"), py::arg("start"), py::arg("border"), py::arg("both"),
          "differentiable softmax attention (qlka_softmax_fwd / qlka_softmax_bwd)");
    m.def("relative_bias", &relative_bias, py::arg("table"), py::arg("M"), py::arg("N"), py::arg("start"),
          py::arg("border"), py::arg("both"), "differentiable bias map (qlka_bias_map_fwd / qlka_bias_map_bwd)");
    m.attr("DIRECT") = DIRECT;
}
