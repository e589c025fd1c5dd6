// Torch binding of the serving entry points: _serve_native.
//
// A step of serving is a few microseconds on the device, so the host's way to it counts: taking the tensors apart in
// Python costs 15 to 30 us a call.  These functions check a call, allocate its results and scratch and pass it to the
// C ABI; a call that is not in order they decline by returning None, and the Python side then says what is wrong with it
// (_norm_rotate.py, _gather_cache.py).  Results and scratch are allocated per call, from the pool of a captured graph
// during its capture.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/extension.h>

#include <limits>
#include <unordered_set>

#include "../../include/att3_b200.h"

namespace {

using at::Tensor;
using MaybeTensor = std::optional<Tensor>;
using Tensors = std::vector<Tensor>;

void check(int status) {
    if (status != ATT3_OK) throw std::runtime_error(att3_last_error());
}

int type_of(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kBFloat16: return ATT3_BF16;
        case at::kHalf: return ATT3_FP16;
        case at::kFloat: return ATT3_FP32;
        default: return -1;
    }
}

bool on_16_bytes(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

bool small(int64_t n) { return n <= std::numeric_limits<int>::max(); }

// t [B,N,H,D] if the kernels can read its rows where they lie (16-byte aligned, contiguous), else a copy.
Tensor readable(const Tensor& t) {
    bool fine = on_16_bytes(t.const_data_ptr()) && t.stride(3) == 1;
    const int64_t step = 16 / static_cast<int64_t>(t.element_size());
    for (int k = 0; k < 3 && fine; ++k)
        if (t.size(k) > 1) fine = t.stride(k) % step == 0 && t.stride(k) >= 0 && (k == 0 || small(t.stride(k)));
    return fine ? t : t.clone(at::MemoryFormat::Contiguous);
}

void set_strides(int64_t (&to)[3], const Tensor& t) {
    for (int k = 0; k < 3; ++k) to[k] = t.size(k) > 1 ? t.stride(k) : 0;       // a dimension of one entry may carry any stride
}

bool is_scale(const Tensor& w, int64_t D, const at::Device& dev) {
    return w.dim() == 1 && w.size(0) == D && type_of(w) >= 0 && w.device() == dev;
}
Tensor readable_scale(const Tensor& w) {
    return w.is_contiguous() && on_16_bytes(w.const_data_ptr()) ? w : w.detach().clone(at::MemoryFormat::Contiguous);
}

bool is_table(const Tensor& t, int64_t D, const at::Device& dev) {
    return t.dim() == 2 && t.scalar_type() == at::kFloat && t.size(0) >= 1 && small(t.size(0)) && t.size(1) >= 8 && t.size(1) <= D &&
           t.size(1) % 8 == 0 && t.device() == dev;
}
Tensor readable_table(const Tensor& t) {
    return t.is_contiguous() && on_16_bytes(t.const_data_ptr()) ? t : t.clone(at::MemoryFormat::Contiguous);
}

// [B,N,heads,D] tensors of one type, batch, length, head dim and CUDA device.
bool are_heads(const Tensors& xs) {
    for (const Tensor& x : xs) {
        if (!x.defined() || x.dim() != 4 || !x.is_cuda() || x.scalar_type() != xs[0].scalar_type() || x.device() != xs[0].device() ||
            x.size(0) != xs[0].size(0) || x.size(1) != xs[0].size(1) || x.size(3) != xs[0].size(3) || x.size(2) < 1 || !small(x.size(2)))
            return false;
    }
    const int64_t D = xs[0].size(3);
    return type_of(xs[0]) >= 0 && (D == 16 || D == 32 || D == 64 || D == 128) && small(xs[0].size(0)) && small(xs[0].size(1));
}

// Whether autograd would miss something: a gradient that the call has none of, or a tangent of forward differentiation
// (which follows tensors that require no gradient, under no_grad too).
bool carries(const Tensor& t, bool gradient) { return t.defined() && ((gradient && t.requires_grad()) || t._fw_grad(0).defined()); }
bool carries(const MaybeTensor& t, bool gradient) { return t && carries(*t, gradient); }
template <typename List>
bool any_carries(const List& list, bool gradient) {
    for (const auto& t : list)
        if (carries(t, gradient)) return true;
    return false;
}

// ------------------------------------------------------------------ norms with rotation

struct Positions {
    const void* at = nullptr;
    int bytes = 0;
    int64_t b = 0, n = 0;
};

bool are_positions(const MaybeTensor& p, int64_t B, int64_t N, const at::Device& dev) {
    if (!p) return true;
    if ((p->scalar_type() != at::kInt && p->scalar_type() != at::kLong) || p->device() != dev) return false;
    return p->dim() == 1 ? p->size(0) == N : p->dim() == 2 && (p->size(0) == B || p->size(0) == 1) && p->size(1) == N;
}
Positions positions_of(const MaybeTensor& p) {
    if (!p) return {};
    return Positions{p->const_data_ptr(), static_cast<int>(p->element_size()), p->dim() == 2 && p->size(0) > 1 ? p->stride(0) : 0,
                     p->size(-1) > 1 ? p->stride(-1) : 0};
}

struct Call {
    MaybeTensor table, positions;
    double eps;
    bool interleaved, heads_first;
};

int rows_of(const MaybeTensor& t) { return t ? static_cast<int>(t->size(0)) : 0; }
int rot_of(const MaybeTensor& t) { return t ? static_cast<int>(t->size(1)) : 0; }
const float* table_of(const MaybeTensor& t) { return t ? t->const_data_ptr<float>() : nullptr; }

// ws[k] may be undefined: tensor k is not normed.
Tensors run_forward(const Tensors& xs, const Tensors& ws, const Call& c) {
    const int64_t B = xs[0].size(0), N = xs[0].size(1), D = xs[0].size(3);
    const c10::cuda::CUDAGuard guard(xs[0].device());
    const auto stream = at::cuda::getCurrentCUDAStream();
    att3_head_rows rows[5] = {};
    Tensors held, ys;
    const auto options = xs[0].options().dtype(at::kBFloat16).requires_grad(false);
    for (size_t k = 0; k < xs.size(); ++k) {
        const int64_t H = xs[k].size(2);
        Tensor x = readable(xs[k]), y = at::empty(c.heads_first ? at::IntArrayRef({B, H, N, D}) : at::IntArrayRef({B, N, H, D}), options);
        rows[k].x = x.const_data_ptr();
        set_strides(rows[k].x_stride, x);
        if (ws[k].defined()) {
            Tensor w = readable_scale(ws[k]);
            rows[k].w = w.const_data_ptr();
            rows[k].w_type = type_of(w);
            held.push_back(w);
        }
        rows[k].rotate = 1;
        rows[k].y = y.mutable_data_ptr();
        rows[k].y_stride[0] = N * H * D;
        rows[k].y_stride[1] = c.heads_first ? D : H * D;
        rows[k].y_stride[2] = c.heads_first ? N * D : D;
        rows[k].heads = H;
        held.push_back(x);
        ys.push_back(y);
    }
    const MaybeTensor table = c.table ? MaybeTensor(readable_table(*c.table)) : std::nullopt;
    const Positions p = positions_of(c.positions);
    check(att3_norm_rotate_forward(rows, static_cast<int>(xs.size()), type_of(xs[0]), table_of(table), rows_of(table), rot_of(table),
                                   c.interleaved, p.at, p.bytes, p.b, p.n, static_cast<int>(B), static_cast<int>(N), static_cast<int>(D),
                                   static_cast<float>(c.eps), stream));
    return ys;
}

Tensors run_backward(const Tensors& xs, const Tensors& ws, const Tensors& dys, const Call& c, Tensors& dws) {
    const int64_t B = xs[0].size(0), N = xs[0].size(1), D = xs[0].size(3);
    const c10::cuda::CUDAGuard guard(xs[0].device());
    const auto stream = at::cuda::getCurrentCUDAStream();
    att3_head_rows rows[5] = {};
    Tensors held, dxs;
    for (size_t k = 0; k < xs.size(); ++k) {
        const int64_t H = xs[k].size(2);
        Tensor x = readable(xs[k]);
        Tensor dy = dys[k].defined() ? dys[k].to(at::kBFloat16)
                                     : at::zeros(c.heads_first ? at::IntArrayRef({B, H, N, D}) : at::IntArrayRef({B, N, H, D}),
                                                 x.options().dtype(at::kBFloat16));
        dy = readable(c.heads_first ? dy.transpose(1, 2) : dy);
        Tensor dx = at::empty({B, N, H, D}, x.options()), dw;
        rows[k].x = x.const_data_ptr();
        set_strides(rows[k].x_stride, x);
        if (ws[k].defined()) {
            Tensor w = readable_scale(ws[k]);
            dw = at::empty({D}, w.options().dtype(at::kFloat));
            rows[k].w = w.const_data_ptr();
            rows[k].w_type = type_of(w);
            rows[k].dw = dw.mutable_data_ptr<float>();
            held.push_back(w);
        }
        rows[k].rotate = 1;
        rows[k].dy = dy.const_data_ptr();
        set_strides(rows[k].dy_stride, dy);
        rows[k].dx = dx.mutable_data_ptr();
        set_strides(rows[k].dx_stride, dx);
        rows[k].heads = H;
        held.push_back(x);
        held.push_back(dy);
        dxs.push_back(dx);
        dws.push_back(dw);
    }
    const MaybeTensor table = c.table ? MaybeTensor(readable_table(*c.table)) : std::nullopt;
    const Positions p = positions_of(c.positions);
    const size_t bytes = att3_norm_rotate_workspace_bytes(static_cast<int>(xs.size()), static_cast<int>(D));
    Tensor scratch = at::empty({static_cast<int64_t>(bytes)}, xs[0].options().dtype(at::kByte));
    check(att3_norm_rotate_backward(rows, static_cast<int>(xs.size()), type_of(xs[0]), table_of(table), rows_of(table), rot_of(table),
                                    c.interleaved, p.at, p.bytes, p.b, p.n, static_cast<int>(B), static_cast<int>(N),
                                    static_cast<int>(D), static_cast<float>(c.eps), scratch.mutable_data_ptr(), bytes, stream));
    for (size_t k = 0; k < ws.size(); ++k)
        if (ws[k].defined()) dws[k] = dws[k].to(ws[k].scalar_type());
    return dxs;
}

// Differentiable in its first argument: the inputs, then the scales that there are (`scaled`, a bit an input).
struct NormRotate : torch::autograd::Function<NormRotate> {
    static constexpr int OTHERS = 7;               // arguments behind the tensors

    static Tensors scales(at::TensorList tensors, int64_t n, int64_t scaled) {
        Tensors ws;
        for (int64_t k = 0, at = n; k < n; ++k) ws.push_back(scaled >> k & 1 ? tensors[at++] : Tensor());
        return ws;
    }
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, at::TensorList tensors, int64_t n, int64_t scaled,
                                                  const MaybeTensor& table, const MaybeTensor& positions, double eps, bool interleaved,
                                                  bool heads_first) {
        const Call c{table, positions, eps, interleaved, heads_first};
        Tensors saved(tensors.begin(), tensors.end());
        const Tensors ys = run_forward(Tensors(tensors.begin(), tensors.begin() + n), scales(tensors, n, scaled), c);
        saved.push_back(table ? *table : Tensor());
        saved.push_back(positions ? *positions : Tensor());
        ctx->save_for_backward(saved);
        ctx->saved_data["n"] = n;
        ctx->saved_data["scaled"] = scaled;
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["interleaved"] = interleaved;
        ctx->saved_data["heads_first"] = heads_first;
        return ys;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list dys) {
        if (at::GradMode::is_enabled())
            throw std::runtime_error("norm_rotate: its gradients have no gradients of their own (create_graph=True)");
        const Tensors saved = ctx->get_saved_variables();
        const int64_t n = ctx->saved_data["n"].toInt(), scaled = ctx->saved_data["scaled"].toInt();
        const size_t inputs = saved.size() - 2;
        const Tensor &table = saved[inputs], &positions = saved[inputs + 1];
        const Call c{table.defined() ? MaybeTensor(table) : std::nullopt, positions.defined() ? MaybeTensor(positions) : std::nullopt,
                     ctx->saved_data["eps"].toDouble(), ctx->saved_data["interleaved"].toBool(), ctx->saved_data["heads_first"].toBool()};
        Tensors dws;
        Tensors grads = run_backward(Tensors(saved.begin(), saved.begin() + n), scales(at::TensorList(saved).slice(0, inputs), n, scaled), dys, c, dws);
        for (const Tensor& dw : dws)
            if (dw.defined()) grads.push_back(dw);
        grads.resize(inputs + OTHERS);             // none for the rest
        return grads;
    }
};

// During a capture autograd runs a leaf's accumulation on the stream that the leaf's accumulator was made on.  One that an
// eager graph still keeps alive is of a stream outside the capture, and the backward pass would then end the capture, and
// with it the process; so the forward pass refuses.  The leaves are the inputs, or lie behind what the capture made of them
// (views, projections); what was computed before the capture is not gone through, since a captured backward pass has to end
// there in any case.
void check_capture(const Tensors& inputs) {
    if (at::cuda::currentStreamCaptureStatusMayInitCtx() == at::cuda::CaptureStatus::None) return;
    std::vector<std::shared_ptr<torch::autograd::Node>> todo;
    std::unordered_set<torch::autograd::Node*> seen;
    const auto add = [&](std::shared_ptr<torch::autograd::Node> node) {
        if (node && seen.insert(node.get()).second) todo.push_back(std::move(node));
    };
    for (const Tensor& t : inputs)
        if (t.requires_grad()) add(t.is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(t) : t.grad_fn());
    const auto here = at::cuda::getCurrentCUDAStream(inputs[0].device().index()).unwrap();
    while (!todo.empty()) {
        const std::shared_ptr<torch::autograd::Node> node = std::move(todo.back());
        todo.pop_back();
        const auto stream = node->stream();
        const bool outside = stream && *stream != here;
        if (dynamic_cast<torch::autograd::AccumulateGrad*>(node.get())) {
            if (outside)
                throw std::runtime_error("norm_rotate: an autograd graph of these leaves made outside the capture is still alive; release it first");
        } else if (!outside)
            for (const auto& edge : node->next_edges()) add(edge.function);
    }
}

py::object norm_rotate(const Tensors& xs, const std::vector<MaybeTensor>& weights, const MaybeTensor& table, const MaybeTensor& positions,
                       double eps, bool interleaved, bool heads_first) {
    if (xs.empty() || xs.size() > 5 || weights.size() != xs.size() || !are_heads(xs) || !(eps >= 0)) return py::none();
    const int64_t B = xs[0].size(0), N = xs[0].size(1), D = xs[0].size(3);
    const at::Device dev = xs[0].device();
    if (table && !is_table(*table, D, dev)) return py::none();
    if (!are_positions(positions, B, N, dev) || (table && !positions && N > table->size(0))) return py::none();
    if (any_carries(xs, false) || any_carries(weights, false) || carries(table, at::GradMode::is_enabled())) return py::none();
    Tensors tensors(xs), ws;
    int64_t scaled = 0;
    bool graph = false;
    for (size_t k = 0; k < xs.size(); ++k) {
        graph = graph || xs[k].requires_grad();
        if (weights[k]) {
            if (!is_scale(*weights[k], D, dev)) return py::none();
            scaled |= int64_t(1) << k;
            tensors.push_back(*weights[k]);
            graph = graph || weights[k]->requires_grad();
        }
        ws.push_back(weights[k] ? *weights[k] : Tensor());
    }
    Tensors ys;
    const c10::cuda::CUDAGuard guard(dev);         // the capture that is asked for is one of this device's stream
    if (graph && at::GradMode::is_enabled()) {
        check_capture(tensors);
        ys = NormRotate::apply(at::TensorList(tensors), static_cast<int64_t>(xs.size()), scaled, table, positions, eps, interleaved,
                               heads_first);
    } else
        ys = run_forward(xs, ws, Call{table, positions, eps, interleaved, heads_first});
    py::tuple out(ys.size());
    for (size_t k = 0; k < ys.size(); ++k) out[k] = py::cast(ys[k]);
    return out;
}

// ------------------------------------------------------------------ the cache

bool are_pools(const Tensors& pools) {
    if (pools.size() != 4) return false;
    for (const Tensor& p : pools) {
        if (!p.defined() || !p.is_cuda() || p.scalar_type() != at::kBFloat16 || p.dim() != 4 || !p.is_contiguous() || p.numel() == 0 ||
            p.sizes() != pools[0].sizes() || p.device() != pools[0].device() || !on_16_bytes(p.const_data_ptr()))
            return false;
    }
    return true;
}

bool is_page_table(const Tensor& t, const at::Device& dev) {
    return t.dim() == 2 && t.scalar_type() == at::kInt && t.size(1) >= 1 && (t.size(1) == 1 || t.stride(1) == 1) && t.device() == dev;
}

bool are_ints(const Tensor& t, int64_t B, const at::Device& dev) {
    return t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == B && t.is_contiguous() && t.device() == dev;
}

bool is_mass(const MaybeTensor& m, const Tensor& pool) {
    return !m || (m->scalar_type() == at::kFloat && m->is_contiguous() && m->sizes() == pool.sizes().slice(0, 3) && m->device() == pool.device());
}

att3_gather_pages pages_of(const Tensor& table, const Tensor& pool) {
    return att3_gather_pages{table.const_data_ptr<int32_t>(), table.stride(0), table.size(1), pool.size(0), pool.size(1)};
}

const int32_t* ints_of(const MaybeTensor& t) { return t ? t->const_data_ptr<int32_t>() : nullptr; }
float* mass_of(const MaybeTensor& t) { return t ? t->mutable_data_ptr<float>() : nullptr; }

// True, or the queries' rows, or None for a call that is not in order.
py::object append(const Tensors& pools, const Tensor& page_table, const Tensor& lengths, const Tensor& R, const Tensor& S, const Tensor& Vr,
                  const Tensor& Vs, const MaybeTensor& counts, const MaybeTensor& Q, const std::vector<MaybeTensor>& weights,
                  const MaybeTensor& table, const MaybeTensor& positions, const MaybeTensor& mass, double eps, bool interleaved) {
    if (!are_pools(pools) || weights.size() != 3 || !(eps >= 0)) return py::none();
    Tensors xs{R, S, Vr, Vs};
    if (Q) xs.push_back(*Q);
    if (!are_heads(xs)) return py::none();
    const Tensor& pool = pools[0];
    const at::Device dev = pool.device();
    const int64_t B = R.size(0), T = R.size(1), D = R.size(3), Hkv = pool.size(2);
    if (R.device() != dev || D != pool.size(3) || R.size(2) != Hkv || S.size(2) != Hkv || Vr.size(2) != Hkv || Vs.size(2) != Hkv) return py::none();
    if (!is_page_table(page_table, dev) || page_table.size(0) != B || !are_ints(lengths, B, dev)) return py::none();
    if ((counts && !are_ints(*counts, B, dev)) || (positions && !are_ints(*positions, B, dev)) || !is_mass(mass, pool)) return py::none();
    if (table && !is_table(*table, D, dev)) return py::none();
    for (const MaybeTensor& w : weights)
        if (w && !is_scale(*w, D, dev)) return py::none();
    const bool graph = at::GradMode::is_enabled();
    if (any_carries(xs, graph) || any_carries(weights, graph) || any_carries(pools, graph) || carries(table, graph) || carries(mass, graph))
        return py::none();
    const c10::cuda::CUDAGuard guard(dev);
    const auto stream = at::cuda::getCurrentCUDAStream();
    att3_head_rows rows[5] = {};
    Tensors held;
    Tensor out;
    const int scale_of[5] = {1, 2, -1, -1, 0};                 // weights are of Q, R and S
    for (size_t k = 0; k < xs.size(); ++k) {
        Tensor x = readable(xs[k]);
        rows[k].x = x.const_data_ptr();
        set_strides(rows[k].x_stride, x);
        held.push_back(x);
        rows[k].heads = x.size(2);
        if (scale_of[k] >= 0) {
            rows[k].rotate = table ? 1 : 0;
            if (const MaybeTensor& w = weights[scale_of[k]]) {
                Tensor r = readable_scale(*w);
                rows[k].w = r.const_data_ptr();
                rows[k].w_type = type_of(r);
                held.push_back(r);
            }
        }
        if (k < 4) rows[k].y = pools[k].mutable_data_ptr();
        else {
            const int64_t H = x.size(2);
            out = at::empty({B, T, H, D}, x.options().dtype(at::kBFloat16).requires_grad(false));
            rows[k].y = out.mutable_data_ptr();
            rows[k].y_stride[0] = T * H * D;
            rows[k].y_stride[1] = H * D;
            rows[k].y_stride[2] = D;
        }
    }
    const MaybeTensor angles = table ? MaybeTensor(readable_table(*table)) : std::nullopt;
    const att3_gather_pages pages = pages_of(page_table, pool);
    check(att3_gather_cache_append(rows, static_cast<int>(xs.size()), type_of(R), table_of(angles), rows_of(angles), rot_of(angles),
                                   interleaved, ints_of(positions), &pages, lengths.const_data_ptr<int32_t>(), ints_of(counts), mass_of(mass),
                                   static_cast<int>(B), static_cast<int>(T), static_cast<int>(D), static_cast<float>(eps), stream));
    return Q ? py::cast(out) : py::object(py::bool_(true));
}

py::object decode(const Tensor& Q, const Tensors& pools, const Tensor& page_table, const Tensor& lengths, int64_t window, int64_t sinks,
                  const MaybeTensor& mass) {
    if (!are_pools(pools) || !Q.is_cuda() || Q.dim() != 3 || !Q.is_floating_point()) return py::none();
    const Tensor& pool = pools[0];
    const at::Device dev = pool.device();
    const int64_t B = Q.size(0), Hq = Q.size(1), D = Q.size(2), Hkv = pool.size(2);
    if ((D != 64 && D != 128) || D != pool.size(3) || Hq < 1 || Hq % Hkv != 0 || Q.device() != dev || !small(B) || !small(Hq)) return py::none();
    if (!is_page_table(page_table, dev) || page_table.size(0) != B || !are_ints(lengths, B, dev)) return py::none();
    if (window < 0 || sinks < 0 || (sinks > 0 && window == 0) || !is_mass(mass, pool)) return py::none();
    const bool graph = at::GradMode::is_enabled();
    if (carries(Q, graph) || any_carries(pools, graph) || carries(mass, graph)) return py::none();
    const int64_t slots = page_table.size(1) * pool.size(1);
    if (!small(slots)) return py::none();
    window = std::min(window, slots);
    sinks = std::min(sinks, slots);
    const c10::cuda::CUDAGuard guard(dev);
    const auto stream = at::cuda::getCurrentCUDAStream();
    Tensor q = Q.to(at::kBFloat16).contiguous();
    if (!on_16_bytes(q.const_data_ptr())) q = q.clone();
    Tensor y = at::empty({B, Hq, D}, q.options().requires_grad(false));
    if (B > 0) {
        const int b = static_cast<int>(B), hq = static_cast<int>(Hq), hkv = static_cast<int>(Hkv), d = static_cast<int>(D);
        const size_t bytes = att3_sg_decode_workspace_bytes(b, hq, hkv, d, static_cast<int>(window), static_cast<int>(sinks),
                                                            static_cast<int>(slots), mass ? 1 : 0);
        Tensor scratch = at::empty({static_cast<int64_t>(bytes)}, q.options().dtype(at::kByte));
        const att3_gather_pages pages = pages_of(page_table, pool);
        check(att3_sg_decode(q.const_data_ptr(), pools[0].const_data_ptr(), pools[1].const_data_ptr(), pools[2].const_data_ptr(),
                             pools[3].const_data_ptr(), mass_of(mass), y.mutable_data_ptr(), &pages, lengths.const_data_ptr<int32_t>(), b, hq,
                             hkv, d, static_cast<int>(window), static_cast<int>(sinks), scratch.mutable_data_ptr(), bytes, stream));
    }
    return py::cast(y.to(Q.scalar_type()));
}

py::object evict(const Tensors& pools, const MaybeTensor& mass, const Tensor& page_table, const Tensor& lengths, int64_t keep, int64_t sinks,
                 int64_t recent, const MaybeTensor& out_table) {
    if (!are_pools(pools) || !mass || !is_mass(mass, pools[0])) return py::none();
    const Tensor& pool = pools[0];
    const at::Device dev = pool.device();
    const int64_t Hkv = pool.size(2), D = pool.size(3);
    if (D != 16 && D != 32 && D != 64 && D != 128) return py::none();
    if (!is_page_table(page_table, dev) || !small(page_table.size(0)) || !are_ints(lengths, page_table.size(0), dev)) return py::none();
    const bool graph = at::GradMode::is_enabled();
    if (any_carries(pools, graph) || carries(mass, graph)) return py::none();
    if (keep < 1 || !small(keep) || sinks < 0 || recent < 0 || sinks > keep || recent > keep || sinks + recent > keep) return py::none();
    const int64_t B = page_table.size(0), slots = page_table.size(1) * pool.size(1);
    if (out_table && (!is_page_table(*out_table, dev) || out_table->size(0) != B || out_table->size(1) * pool.size(1) < std::min(keep, slots)))
        return py::none();
    const c10::cuda::CUDAGuard guard(dev);
    const auto stream = at::cuda::getCurrentCUDAStream();
    Tensor kept = at::empty({B, Hkv, keep}, lengths.options()), left = at::empty({B}, lengths.options());
    if (B > 0) {
        const att3_gather_pages from = pages_of(page_table, pool), to = pages_of(out_table ? *out_table : page_table, pool);
        check(att3_gather_cache_evict(pools[0].mutable_data_ptr(), pools[1].mutable_data_ptr(), pools[2].mutable_data_ptr(),
                                      pools[3].mutable_data_ptr(), mass_of(mass), &from, &to, lengths.const_data_ptr<int32_t>(),
                                      left.mutable_data_ptr<int32_t>(), kept.mutable_data_ptr<int32_t>(), static_cast<int>(B),
                                      static_cast<int>(Hkv), static_cast<int>(D), static_cast<int>(keep), static_cast<int>(sinks),
                                      static_cast<int>(recent), stream));
    }
    return py::make_tuple(kept, left);
}

}  // namespace

PYBIND11_MODULE(_serve_native, m) {
    m.doc() = "Torch binding of the serving entry points of libatt3_b200.so; a call that is not in order gives None.";
    m.def("norm_rotate", &norm_rotate);
    m.def("append", &append);
    m.def("decode", &decode);
    m.def("evict", &evict);
}
