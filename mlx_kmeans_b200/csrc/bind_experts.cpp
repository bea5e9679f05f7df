// bind_experts.cpp -- torch tensors to the routed-experts entry points of include/kmc.h (the module _experts).
//
// These calls run once or more per layer and token, so their host time counts: checks, allocation of the results and
// the launch happen here in one call (5 to 7 us where ctypes and Python took 12 to 16).  Checks of the tensors raise
// ValueError; so do statuses KMC_ERR_INVALID and KMC_ERR_UNSUPPORTED, any other status raises RuntimeError.  Work goes
// to the current stream of the tensors' device; nothing synchronises but status().
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include <mutex>
#include <sstream>
#include <vector>

#include "../../include/kmc.h"

namespace {

using at::Tensor;
using Maybe = std::optional<Tensor>;

template <typename... Args>
[[noreturn]] void refuse(Args&&... args) {
    std::ostringstream s;
    (s << ... << args);
    throw py::value_error(s.str());
}

void check(int status, const char* who) {
    if (status == KMC_OK) return;
    const std::string text = std::string(who) + ": " + kmc_last_error();
    if (status == KMC_ERR_INVALID || status == KMC_ERR_UNSUPPORTED) throw py::value_error(text);
    throw std::runtime_error(text);
}

std::string shape(const Tensor& t) {
    std::ostringstream s;
    s << t.sizes();
    return s.str();
}

void on_gpu(const Tensor& t, const char* name, int64_t ndim = -1) {
    if (!t.defined() || !t.is_cuda()) refuse(name, " must be a CUDA tensor");
    if (ndim >= 0 && t.dim() != ndim) refuse(name, " must be ", ndim, "-D, got ", t.dim(), "-D");
}
void beside(const Tensor& t, const char* name, const Tensor& other) {
    if (t.device() != other.device()) refuse(name, " is on ", t.device(), ", not on ", other.device());
}
// An input whose derivative counts carries no tangent of forward-mode differentiation, which would be lost here.
void no_tangent(const Tensor& t, const char* name) {
    if (t._fw_grad(0).defined())
        throw std::runtime_error(std::string("route, expert_matmul and combine_rows have no forward-mode derivative (") + name + " has a tangent)");
}
void of_type(const Tensor& t, const char* name, at::ScalarType type) {
    if (t.scalar_type() != type) refuse(name, " must be ", type, ", got ", t.scalar_type());
}

int dtype_of(const Tensor& t, const char* name, bool f32) {
    switch (t.scalar_type()) {
        case at::kFloat:
            if (f32) return KMC_F32;
            break;
        case at::kBFloat16: return KMC_BF16;
        case at::kHalf: return KMC_F16;
        default: break;
    }
    refuse(name, " must be ", f32 ? "float32, bfloat16 or float16" : "bfloat16 or float16", ", got ", t.scalar_type());
}

// t (2-D) with unit stride along its rows, copied if it has none; rows may lie any distance apart
Tensor rows_of(const Tensor& t) {
    return (t.stride(1) == 1 || t.size(1) == 1) && t.stride(0) >= t.size(1) ? t : t.contiguous();
}
int64_t row_stride(const Tensor& t) { return std::max(t.stride(0), t.size(1)); }

Tensor empty(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) {
    return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}
void* data(const Tensor& t) { return t.data_ptr(); }
template <typename T>
T* ptr(const Tensor& t) { return static_cast<T*>(t.data_ptr()); }
void* stream(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

int as_int(int64_t v, const char* name) {
    if (v > INT32_MAX || v < INT32_MIN) refuse(name, " of ", v, " is out of range");
    return (int)v;
}

// Per device: the int32 a kernel sets when it gave up on a barrier.  It lies in pinned host memory, which the host clears
// at its first use without a stream, so that use may be inside a graph capture (whose mode is relaxed for the
// allocation); and it stays for the life of the process, as a graph may keep its address.
std::mutex g_mutex;
std::vector<Tensor>& error_words() {
    static auto* words = new std::vector<Tensor>(64);
    return *words;
}

const char* kGaveUp = "expert_matmul: a kernel gave up waiting on a barrier; its result is incomplete";

Tensor error_tensor(int64_t i) {
    std::lock_guard<std::mutex> lock(g_mutex);
    Tensor& word = error_words().at(i);
    if (!word.defined()) {
        const c10::cuda::CUDAStreamCaptureModeGuard relaxed(cudaStreamCaptureModeRelaxed);
        const Tensor fresh = at::empty({1}, at::TensorOptions(at::kInt).pinned_memory(true));
        *ptr<int32_t>(fresh) = 0;
        word = fresh;
    }
    return word;
}
// The word of a call on the device of `like`; an earlier kernel's that is set raises first, and is cleared.  (The host
// only looks at its memory: what a kernel still running has not written yet, the next call sees, or expert_status.)
int32_t* error_word(const Tensor& like) {
    int32_t* word = ptr<int32_t>(error_tensor(like.device().index()));
    if (*static_cast<volatile int32_t*>(word) != 0) {
        *word = 0;
        throw std::runtime_error(std::string("an earlier ") + kGaveUp);
    }
    return word;
}

void status(int64_t device) {
    volatile int32_t* word;
    {
        std::lock_guard<std::mutex> lock(g_mutex);
        if (device < 0 || device >= (int64_t)error_words().size() || !error_words()[device].defined()) return;
        word = ptr<int32_t>(error_words()[device]);
    }
    c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).synchronize();
    if (*word == 0) return;
    *word = 0;
    throw std::runtime_error(kGaveUp);
}

// ---------------------------------------------------------------- routing

std::tuple<Tensor, Tensor> route(const Tensor& logits0, int64_t top_k, int64_t flags, const Maybe& bias0, int64_t groups,
                                 int64_t top_groups, double scale, const Maybe& mask0) {
    on_gpu(logits0, "logits", 2);
    no_tangent(logits0, "logits");
    const int type = dtype_of(logits0, "logits", true);
    const Tensor logits = rows_of(logits0);
    const int64_t T = logits.size(0), E = logits.size(1);
    Tensor bias, mask;
    if (bias0) {
        on_gpu(*bias0, "bias", 1);
        of_type(*bias0, "bias", at::kFloat);
        beside(*bias0, "bias", logits);
        if (bias0->size(0) != E) refuse("bias has ", bias0->size(0), " values for ", E, " experts");
        bias = bias0->contiguous();
    }
    if (mask0) {
        on_gpu(*mask0, "mask", 1);
        of_type(*mask0, "mask", at::kBool);
        beside(*mask0, "mask", logits);
        if (mask0->size(0) != T) refuse("mask has ", mask0->size(0), " values for ", T, " rows");
        mask = mask0->contiguous();
    }
    if (top_k < 1 || top_k > E) refuse("route: ", top_k, " choices of ", E, " experts");
    const c10::cuda::CUDAGuard guard(logits.device());
    Tensor ids = empty({T, top_k}, at::kInt, logits), weights = empty({T, top_k}, at::kFloat, logits);
    check(kmc_route(data(logits), type, T, as_int(E, "n_experts"), row_stride(logits), bias0 ? ptr<float>(bias) : nullptr,
                    mask0 ? ptr<uint8_t>(mask) : nullptr, as_int(top_k, "top_k"), as_int(groups, "groups"),
                    as_int(top_groups, "top_groups"), (float)scale, (unsigned)flags, ptr<int32_t>(ids), ptr<float>(weights),
                    stream(logits)),
          "kmc_route");
    return {ids, weights};
}

Tensor route_grad(const Tensor& dweights, const Tensor& logits0, const Tensor& ids, int64_t flags, double scale) {
    on_gpu(logits0, "logits", 2);
    no_tangent(logits0, "logits");
    const int type = dtype_of(logits0, "logits", true);
    on_gpu(ids, "ids", 2);
    of_type(ids, "ids", at::kInt);
    beside(ids, "ids", logits0);
    on_gpu(dweights, "dweights", 2);
    no_tangent(dweights, "dweights");
    of_type(dweights, "dweights", at::kFloat);
    beside(dweights, "dweights", logits0);
    if (ids.sizes() != dweights.sizes() || ids.size(0) != logits0.size(0))
        refuse("dweights ", shape(dweights), ", ids ", shape(ids), " and logits ", shape(logits0), " do not belong together");
    const Tensor logits = rows_of(logits0), g = dweights.contiguous(), id = ids.contiguous();
    const c10::cuda::CUDAGuard guard(logits.device());
    Tensor dl = empty(logits.sizes(), logits.scalar_type(), logits);
    check(kmc_route_grad(ptr<float>(g), data(logits), type, logits.size(0), as_int(logits.size(1), "n_experts"),
                         row_stride(logits), ptr<int32_t>(id), as_int(id.size(1), "top_k"), (float)scale, (unsigned)flags,
                         data(dl), stream(logits)),
          "kmc_route_grad");
    return dl;
}

// ---------------------------------------------------------------- grouping

std::tuple<Tensor, Tensor, Tensor> group_rows(const Tensor& ids0, int64_t experts) {
    on_gpu(ids0, "ids");
    of_type(ids0, "ids", at::kInt);
    if (ids0.dim() != 1 && ids0.dim() != 2) refuse("ids must be 1-D or 2-D, got ", ids0.dim(), "-D");
    const Tensor ids = ids0.contiguous();
    const int64_t T = ids.size(0), k = ids.dim() == 2 ? ids.size(1) : 1;
    const int E = as_int(experts, "n_experts");
    const c10::cuda::CUDAGuard guard(ids.device());
    const size_t need = kmc_group_bytes(T * k, E);
    Tensor ws;
    if (need) ws = empty({(int64_t)need}, at::kByte, ids);
    Tensor offsets = empty({std::max(E, 0) + 1}, at::kInt, ids), rows = empty({T * k}, at::kInt, ids),
           slot = empty(ids.sizes(), at::kInt, ids);
    check(kmc_group_rows(ptr<int32_t>(ids), T, as_int(k, "choices"), E, ptr<int32_t>(offsets), ptr<int32_t>(rows),
                         ptr<int32_t>(slot), need ? data(ws) : nullptr, need, stream(ids)),
          "kmc_group_rows");
    return {offsets, rows, slot};
}

struct Groups {
    Tensor offsets, rows, slot;
    int64_t T, k, P, E;
    Groups(const Tensor& o, const Tensor& r, const Tensor& s, const Tensor& like) : offsets(o), rows(r), slot(s) {
        const char* names[] = {"groups.offsets", "groups.rows", "groups.slot"};
        const Tensor* all[] = {&o, &r, &s};
        for (int i = 0; i < 3; i++) {
            on_gpu(*all[i], names[i], i < 2 ? 1 : -1);
            of_type(*all[i], names[i], at::kInt);
            beside(*all[i], names[i], like);
            if (!all[i]->is_contiguous()) refuse(names[i], " must be contiguous (as group_rows gives it)");
        }
        if ((s.dim() != 1 && s.dim() != 2) || s.numel() != r.numel() || o.numel() < 2)
            refuse("groups of ", o.numel() - 1, " experts, ", r.numel(), " positions and slots of shape ", shape(s),
                   " do not belong together");
        T = s.size(0);
        k = s.dim() == 2 ? s.size(1) : 1;
        P = r.numel();
        E = o.numel() - 1;
    }
    const int32_t* off() const { return ptr<int32_t>(offsets); }
};

// ---------------------------------------------------------------- combination

Tensor workspace(size_t need, const Tensor& like) { return need ? empty({(int64_t)need}, at::kByte, like) : Tensor(); }

Tensor combine_of(const Tensor& y, int type, const Groups& g, const Tensor& weights) {
    Tensor out = empty({g.T, y.size(1)}, y.scalar_type(), y);
    check(kmc_combine(data(y), type, g.T, as_int(g.k, "choices"), as_int(y.size(1), "width"), ptr<int32_t>(g.slot),
                      weights.defined() ? ptr<float>(weights) : nullptr, data(out), stream(y)),
          "kmc_combine");
    return out;
}

Tensor weights_of(const Maybe& weights, const Groups& g, const Tensor& y) {
    if (!weights) return {};
    on_gpu(*weights, "weights");
    no_tangent(*weights, "weights");
    of_type(*weights, "weights", at::kFloat);
    beside(*weights, "weights", y);
    if (weights->sizes() != g.slot.sizes()) refuse("weights are ", shape(*weights), ", the groups' pairs ", shape(g.slot));
    return weights->contiguous();
}

Tensor combine(const Tensor& y0, const Tensor& offsets, const Tensor& rows, const Tensor& slot, const Maybe& weights) {
    on_gpu(y0, "y", 2);
    no_tangent(y0, "y");
    const int type = dtype_of(y0, "y", true);
    const Groups g(offsets, rows, slot, y0);
    if (y0.size(0) != g.P) refuse("y has ", y0.size(0), " rows for ", g.P, " positions");
    const c10::cuda::CUDAGuard guard(y0.device());
    return combine_of(y0.contiguous(), type, g, weights_of(weights, g, y0));
}

std::tuple<Tensor, Maybe> combine_grad(const Tensor& dout0, const Tensor& y0, const Tensor& offsets, const Tensor& rows,
                                       const Tensor& slot, const Maybe& weights0) {
    on_gpu(y0, "y", 2);
    no_tangent(y0, "y");
    const int type = dtype_of(y0, "y", true);
    const Groups g(offsets, rows, slot, y0);
    if (y0.size(0) != g.P) refuse("y has ", y0.size(0), " rows for ", g.P, " positions");
    on_gpu(dout0, "dout", 2);
    no_tangent(dout0, "dout");
    of_type(dout0, "dout", y0.scalar_type());
    beside(dout0, "dout", y0);
    if (dout0.size(0) != g.T || dout0.size(1) != y0.size(1))
        refuse("dout is ", shape(dout0), ", the result ", g.T, " x ", y0.size(1));
    const Tensor weights = weights_of(weights0, g, y0), dout = dout0.contiguous(), y = y0.contiguous();
    const c10::cuda::CUDAGuard guard(y.device());
    Tensor dy = empty(y.sizes(), y.scalar_type(), y);
    Maybe dw;
    if (weights0) dw = empty(weights.sizes(), at::kFloat, y);
    const int k = as_int(g.k, "choices");
    const size_t need = kmc_combine_bytes(g.T, k);
    const Tensor ws = workspace(need, y);
    check(kmc_combine_grad_slots(data(dout), data(y), type, g.T, k, as_int(y.size(1), "width"), ptr<int32_t>(slot),
                                 weights0 ? ptr<float>(weights) : nullptr, data(dy), dw ? ptr<float>(*dw) : nullptr,
                                 need ? data(ws) : nullptr, need, stream(y)),
          "kmc_combine_grad_slots");
    return {dy, dw};
}

// ---------------------------------------------------------------- products per expert

void check_x(const Tensor& x, int64_t d, at::ScalarType type, const Groups& g, bool gather) {
    on_gpu(x, "x", 2);
    no_tangent(x, "x");
    of_type(x, "x", type);
    if (x.size(1) != d) refuse("x has ", x.size(1), " columns, the matrices ", d);
    const int64_t want = gather ? g.T : g.P;
    if (x.size(0) != want) refuse("x has ", x.size(0), " rows, the groups want ", want, gather ? " (rows)" : " (positions)");
}
int check_w(const Tensor& w, const Groups& g) {
    if (w.size(0) != g.E) refuse("w has ", w.size(0), " matrices for ", g.E, " experts");
    return dtype_of(w, "w", false);
}
void check_dy(const Tensor& dy, int64_t n, at::ScalarType type, const Groups& g, const Tensor& like) {
    on_gpu(dy, "dy", 2);
    no_tangent(dy, "dy");
    of_type(dy, "dy", type);
    beside(dy, "dy", like);
    if (dy.size(0) != g.P || dy.size(1) != n) refuse("dy is ", shape(dy), ", the products ", g.P, " x ", n);
}

Tensor expert_matmul(const Tensor& x0, const Tensor& w0, const Tensor& offsets, const Tensor& rows, const Tensor& slot,
                     bool gather) {
    on_gpu(w0, "w", 3);
    no_tangent(w0, "w");
    const Groups g(offsets, rows, slot, w0);
    const int type = check_w(w0, g);
    check_x(x0, w0.size(2), w0.scalar_type(), g, gather);
    beside(x0, "x", w0);
    const c10::cuda::CUDAGuard guard(w0.device());
    const Tensor x = rows_of(x0), w = w0.contiguous();
    const int E = as_int(g.E, "n_experts"), N = as_int(w.size(1), "n"), D = as_int(w.size(2), "d");
    const int32_t* row = gather ? ptr<int32_t>(rows) : nullptr;
    const size_t need = kmc_expert_bytes(data(x), x.size(0), row_stride(x), row, data(w), nullptr, g.P, E, N, D);
    const Tensor ws = workspace(need, w);
    Tensor y = empty({g.P, N}, w.scalar_type(), w);
    check(kmc_expert_matmul(data(x), x.size(0), row_stride(x), row, data(w), g.off(), g.P, E, N, D, type, data(y),
                            need ? data(ws) : nullptr, need, error_word(w), stream(w)),
          "kmc_expert_matmul");
    return y;
}

Tensor expert_dx(const Tensor& dy0, const Tensor& w0, const Tensor& offsets, const Tensor& rows, const Tensor& slot,
                 bool gather) {
    on_gpu(w0, "w", 3);
    no_tangent(w0, "w");
    const Groups g(offsets, rows, slot, w0);
    const int type = check_w(w0, g);
    check_dy(dy0, w0.size(1), w0.scalar_type(), g, w0);
    const c10::cuda::CUDAGuard guard(w0.device());
    const Tensor dy = dy0.contiguous(), w = w0.contiguous();
    const int E = as_int(g.E, "n_experts"), N = as_int(w.size(1), "n"), D = as_int(w.size(2), "d");
    if (gather) {
        const int k = as_int(g.k, "choices");
        const size_t need = kmc_expert_dx_rows_bytes(data(w), data(dy), g.T, k, E, N, D);
        const Tensor ws = workspace(need, w);
        Tensor dx = empty({g.T, D}, w.scalar_type(), w);
        check(kmc_expert_matmul_dx_rows(data(dy), data(w), g.off(), ptr<int32_t>(slot), g.T, k, E, N, D, type, data(dx),
                                        need ? data(ws) : nullptr, need, error_word(w), stream(w)),
              "kmc_expert_matmul_dx_rows");
        return dx;
    }
    const size_t need = kmc_expert_bytes(nullptr, 0, D, nullptr, data(w), data(dy), g.P, E, N, D);
    const Tensor ws = workspace(need, w);
    Tensor dx = empty({g.P, D}, w.scalar_type(), w);
    check(kmc_expert_matmul_dx(data(dy), data(w), g.off(), g.P, E, N, D, type, data(dx), need ? data(ws) : nullptr, need,
                               error_word(w), stream(w)),
          "kmc_expert_matmul_dx");
    return dx;
}

Tensor expert_dw(const Tensor& dy0, const Tensor& x0, const Tensor& offsets, const Tensor& rows, const Tensor& slot,
                 bool gather) {
    on_gpu(x0, "x", 2);
    const int type = dtype_of(x0, "x", false);
    const Groups g(offsets, rows, slot, x0);
    check_x(x0, x0.size(1), x0.scalar_type(), g, gather);
    on_gpu(dy0, "dy", 2);
    check_dy(dy0, dy0.size(1), x0.scalar_type(), g, x0);
    const c10::cuda::CUDAGuard guard(x0.device());
    const Tensor dy = dy0.contiguous(), x = rows_of(x0);
    const int E = as_int(g.E, "n_experts"), N = as_int(dy.size(1), "n"), D = as_int(x.size(1), "d");
    const int32_t* row = gather ? ptr<int32_t>(rows) : nullptr;
    const size_t need = kmc_expert_bytes(data(x), x.size(0), row_stride(x), row, nullptr, data(dy), g.P, E, N, D);
    const Tensor ws = workspace(need, x);
    Tensor dw = empty({g.E, N, D}, x.scalar_type(), x);
    check(kmc_expert_matmul_dw(data(dy), data(x), x.size(0), row_stride(x), row, g.off(), g.P, E, N, D, type, data(dw),
                               need ? data(ws) : nullptr, need, error_word(x), stream(x)),
          "kmc_expert_matmul_dw");
    return dw;
}

}  // namespace

PYBIND11_MODULE(_experts, m) {
    m.def("route", &route);
    m.def("route_grad", &route_grad);
    m.def("group_rows", &group_rows);
    m.def("expert_matmul", &expert_matmul);
    m.def("expert_dx", &expert_dx);
    m.def("expert_dw", &expert_dw);
    m.def("combine", &combine);
    m.def("combine_grad", &combine_grad);
    m.def("status", &status);
    m.def("error_word", &error_tensor);
}
