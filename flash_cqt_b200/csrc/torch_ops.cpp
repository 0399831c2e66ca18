// Torch-facing fast path of the CUDA engines: the four whole-slice entry
// points of the C ABI (cqt_analysis, cqt_synthesis, cqt_adj_analysis,
// cqt_adj_synthesis) called from C++ with torch's current stream, and
// TrainableCQT's fwd / bwd as C++ autograd functions whose backward nodes run
// the transposes without entering Python.  The C-ABI library stays the only
// place with device code; this module receives its function pointers from the
// Python loader (no link-time dependency) and only moves tensors in and out.
//
// Mirrors trainable.py:141-191 of the reference (TrainableCQT.fwd / bwd: the
// forward returns per-group complex views, the backward of the analysis is
// the transpose of the analysis, that of the synthesis the transpose of the
// synthesis, nothing saved for backward).
//
// Also the per-call host work of AdamW.step (gradients, addresses and checks of
// every parameter) and of CoefCache.append / window, which have no counterpart
// there.
#include <torch/extension.h>

#include "flash_cqt_b200.h"

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>

#include <cstdint>
#include <string>
#include <unordered_map>
#include <vector>

namespace {

constexpr int64_t kDefaultN = 65536;
constexpr int kLayoutPlanar = 0;    // CQT_LAYOUT_PLANAR
constexpr int kLayoutComplex = 1;   // CQT_LAYOUT_COMPLEX
constexpr int64_t kWsHeader = 256;  // workspace header (the wait-status word)

// cqt_analysis / cqt_adj_synthesis: signal first
using FnSignalFirst = int (*)(const void*, const float*, float*, float*, int, int, void*,
                              size_t, void*);
// cqt_synthesis / cqt_adj_analysis: coefficients first
using FnCoefFirst = int (*)(const void*, const float*, const float*, int, float*, int, void*,
                            size_t, void*);
using FnWorkspace = size_t (*)(const void*, int);
// cqt_synthesis_sqerr / cqt_adj_synthesis_sqerr (the fused MSE loss)
using FnSynSqErr = int (*)(const void*, const float*, const float*, int, float*, const float*,
                           float*, float, int, void*, size_t, void*);
using FnAdjSynSqErr = int (*)(const void*, const float*, const float*, float, const float*,
                              float*, float*, int, int, void*, size_t, void*);
using FnLastError = const char* (*)();

// One filterbank's device tables on one device, with a grow-only workspace.
// Held by intrusive pointer from Python and from every autograd node that
// may still call it; it keeps the Python owner of the tables alive.
struct Ops : torch::CustomClassHolder {
    const void* tables = nullptr;
    c10::DeviceIndex device = 0;
    int64_t ncoef = 0;
    int64_t kN = kDefaultN;   // samples per slice (65536 or 32768)
    FnSignalFirst an = nullptr, adj_syn = nullptr;
    FnCoefFirst syn = nullptr, adj_an = nullptr;
    FnWorkspace ws_bytes = nullptr;
    FnLastError last_error = nullptr;
    FnSynSqErr syn_sqerr = nullptr;
    FnAdjSynSqErr adj_syn_sqerr = nullptr;
    PyObject* owner = nullptr;         // Python object owning `tables` (strong ref)
    at::Tensor ws;
    std::vector<at::Tensor> retired;   // outgrown workspaces: captured graphs may address them
    std::unordered_map<int64_t, size_t> need;
    std::vector<int64_t> sizes, bins, lens;   // per group: b * M, b, M
    int64_t ngroups = 0;                       // octave groups (the rest are side groups)
    // the heap and views of the last fwd, held weakly, so that bwd can
    // recognise untouched views by identity
    c10::weak_intrusive_ptr<c10::TensorImpl, c10::UndefinedTensorImpl> last_h{
        c10::intrusive_ptr<c10::TensorImpl, c10::UndefinedTensorImpl>()};
    std::vector<c10::weak_intrusive_ptr<c10::TensorImpl, c10::UndefinedTensorImpl>> last_v;

    ~Ops() override {
        if (owner && Py_IsInitialized()) {
            pybind11::gil_scoped_acquire gil;
            Py_DECREF(owner);
        }
    }

    void check(int rc, const char* what) const {
        if (rc != 0)
            TORCH_CHECK(false, what, " failed (", rc, "): ", last_error ? last_error() : "");
    }

    void* workspace(int64_t batch, size_t* bytes) {
        auto it = need.find(batch);
        size_t n;
        if (it == need.end()) {
            n = ws_bytes(tables, (int)batch);
            need.emplace(batch, n);
        } else {
            n = it->second;
        }
        if (!ws.defined() || (size_t)ws.numel() < n) {
            if (ws.defined()) retired.push_back(ws);
            ws = at::empty({(int64_t)std::max<size_t>(n, kWsHeader)},
                           at::TensorOptions().dtype(at::kByte).device(at::kCUDA, device));
            ws.narrow(0, 0, kWsHeader).zero_();   // the wait-status header
        }
        *bytes = (size_t)ws.numel();
        return ws.data_ptr();
    }

    void* stream() const { return at::cuda::getCurrentCUDAStream(device).stream(); }

    at::Tensor signal(const at::Tensor& t, const char* name) const {
        TORCH_CHECK_VALUE(t.defined() && t.is_cuda() && t.get_device() == device, name,
                          " must be a tensor on cuda:", (int)device);
        TORCH_CHECK_TYPE(t.scalar_type() == at::kFloat, name, " must be float32, got ",
                         t.scalar_type());
        TORCH_CHECK_VALUE(t.dim() == 2 && t.size(1) == kN, name, " must be [B, ", kN,
                          "], got ", t.sizes());
        at::Tensor c = t.contiguous();
        // the engines move signals as float2 / float4 vectors
        return (reinterpret_cast<uintptr_t>(c.data_ptr()) & 15u) ? c.clone() : c;
    }

    at::Tensor coef(const at::Tensor& t, const char* name) const {
        TORCH_CHECK_VALUE(t.defined() && t.is_cuda() && t.get_device() == device, name,
                          " must be a tensor on cuda:", (int)device);
        TORCH_CHECK_TYPE(t.scalar_type() == at::kComplexFloat, name,
                         " must be complex64, got ", t.scalar_type());
        TORCH_CHECK_VALUE(t.dim() == 2 && t.size(1) == ncoef, name, " must be [B, ", ncoef,
                          "], got ", t.sizes());
        return t.resolve_conj().contiguous();
    }

    // a float32 [B, ncoef] coefficient plane on this device; `out` planes
    // are written in place, so they must already be contiguous
    at::Tensor plane(const at::Tensor& t, const char* name, int64_t B, bool out) const {
        TORCH_CHECK_VALUE(t.defined() && t.is_cuda() && t.get_device() == device,
                          "coefficient plane ", name, " must be float32 on cuda:", (int)device);
        TORCH_CHECK_VALUE(t.scalar_type() == at::kFloat, "coefficient plane ", name,
                          " must be float32 on cuda:", (int)device);
        TORCH_CHECK_VALUE(t.dim() == 2 && t.size(1) == ncoef && (B < 0 || t.size(0) == B),
                          "coefficient plane ", name, " must be [B, ", ncoef, "]");
        if (out) {
            TORCH_CHECK_VALUE(t.is_contiguous(), "coefficient plane ", name,
                              " must be contiguous");
            return t;
        }
        return t.contiguous();
    }

    struct DeviceSwitch {   // switches only when the current device differs
        c10::optional<c10::cuda::CUDAGuard> g;
        explicit DeviceSwitch(c10::DeviceIndex d) {
            if (c10::cuda::current_device() != d) g.emplace(d);
        }
    };

    at::Tensor analysis(const at::Tensor& x_) {
        at::Tensor x = signal(x_, "x");
        DeviceSwitch sw(device);
        const int64_t B = x.size(0);
        at::Tensor out = at::empty({B, ncoef}, x.options().dtype(at::kComplexFloat));
        size_t wb;
        void* w = workspace(B, &wb);
        check(an(tables, x.data_ptr<float>(), reinterpret_cast<float*>(out.data_ptr()), nullptr,
                 kLayoutComplex, (int)B, w, wb, stream()),
              "cqt_analysis");
        return out;
    }

    // planar layout (FusedOctCQT): results go into the caller's tensors
    void analysis_planar(const at::Tensor& x_, const at::Tensor& kr_, const at::Tensor& ki_) {
        at::Tensor x = signal(x_, "x");
        const int64_t B = x.size(0);
        at::Tensor kr = plane(kr_, "re", B, true), ki = plane(ki_, "im", B, true);
        DeviceSwitch sw(device);
        size_t wb;
        void* w = workspace(B, &wb);
        check(an(tables, x.data_ptr<float>(), kr.data_ptr<float>(), ki.data_ptr<float>(),
                 kLayoutPlanar, (int)B, w, wb, stream()),
              "cqt_analysis");
    }

    void synthesis_planar(const at::Tensor& kr_, const at::Tensor& ki_, const at::Tensor& y) {
        at::Tensor kr = plane(kr_, "re", -1, false);
        const int64_t B = kr.size(0);
        at::Tensor ki = plane(ki_, "im", B, false);
        TORCH_CHECK_VALUE(y.defined() && y.is_cuda() && y.get_device() == device &&
                              y.scalar_type() == at::kFloat && y.dim() == 2 &&
                              y.size(0) == B && y.size(1) == kN && y.is_contiguous(),
                          "y must be a contiguous float32 [B, ", kN, "] tensor on cuda:",
                          (int)device);
        DeviceSwitch sw(device);
        size_t wb;
        void* w = workspace(B, &wb);
        check(syn(tables, kr.data_ptr<float>(), ki.data_ptr<float>(), kLayoutPlanar,
                  y.data_ptr<float>(), (int)B, w, wb, stream()),
              "cqt_synthesis");
    }

    at::Tensor synthesis(const at::Tensor& c_) {
        at::Tensor c = coef(c_, "coefficients");
        DeviceSwitch sw(device);
        const int64_t B = c.size(0);
        at::Tensor out = at::empty({B, kN}, c.options().dtype(at::kFloat));
        size_t wb;
        void* w = workspace(B, &wb);
        check(syn(tables, reinterpret_cast<const float*>(c.data_ptr()), nullptr, kLayoutComplex,
                  out.data_ptr<float>(), (int)B, w, wb, stream()),
              "cqt_synthesis");
        return out;
    }

    at::Tensor adj_analysis(const at::Tensor& g_) {
        at::Tensor g = coef(g_, "coefficient gradient");
        DeviceSwitch sw(device);
        const int64_t B = g.size(0);
        at::Tensor out = at::empty({B, kN}, g.options().dtype(at::kFloat));
        size_t wb;
        void* w = workspace(B, &wb);
        check(adj_an(tables, reinterpret_cast<const float*>(g.data_ptr()), nullptr,
                     kLayoutComplex, out.data_ptr<float>(), (int)B, w, wb, stream()),
              "cqt_adj_analysis");
        return out;
    }

    // synthesis + the squared-error sum against `target`: (loss = mean of
    // (y - target)^2 as a 0-dim float32 tensor, y)
    std::vector<at::Tensor> synthesis_sqerr(const at::Tensor& c_, const at::Tensor& target_) {
        at::Tensor c = coef(c_, "coefficients");
        const int64_t B = c.size(0);
        at::Tensor tgt = signal(target_, "target");
        TORCH_CHECK_VALUE(tgt.size(0) == B, "target must be [", B, ", ", kN, "], got ",
                          tgt.sizes());
        DeviceSwitch sw(device);
        at::Tensor y = at::empty({B, kN}, c.options().dtype(at::kFloat));
        at::Tensor loss = at::empty({}, c.options().dtype(at::kFloat));
        size_t wb;
        void* w = workspace(B, &wb);
        const float scale = B > 0 ? (float)(1.0 / ((double)B * (double)kN)) : 0.f;
        check(syn_sqerr(tables, reinterpret_cast<const float*>(c.data_ptr()), nullptr,
                        kLayoutComplex, y.data_ptr<float>(), tgt.data_ptr<float>(),
                        loss.data_ptr<float>(), scale, (int)B, w, wb, stream()),
              "cqt_synthesis_sqerr");
        return {loss, y, tgt};
    }

    // transpose of the synthesis applied to scale * (*g) * (y - target)
    at::Tensor adj_synthesis_sqerr(const at::Tensor& y, const at::Tensor& tgt, float scale,
                                   const at::Tensor& g) {
        DeviceSwitch sw(device);
        const int64_t B = y.size(0);
        at::Tensor out = at::empty({B, ncoef}, y.options().dtype(at::kComplexFloat));
        size_t wb;
        void* w = workspace(B, &wb);
        check(adj_syn_sqerr(tables, y.data_ptr<float>(), tgt.data_ptr<float>(), scale,
                            g.data_ptr<float>(), reinterpret_cast<float*>(out.data_ptr()),
                            nullptr, kLayoutComplex, (int)B, w, wb, stream()),
              "cqt_adj_synthesis_sqerr");
        return out;
    }

    at::Tensor adj_synthesis(const at::Tensor& gy_) {
        at::Tensor gy = signal(gy_, "signal gradient");
        DeviceSwitch sw(device);
        const int64_t B = gy.size(0);
        at::Tensor out = at::empty({B, ncoef}, gy.options().dtype(at::kComplexFloat));
        size_t wb;
        void* w = workspace(B, &wb);
        check(adj_syn(tables, gy.data_ptr<float>(), reinterpret_cast<float*>(out.data_ptr()),
                      nullptr, kLayoutComplex, (int)B, w, wb, stream()),
              "cqt_adj_synthesis");
        return out;
    }
};

Ops* ops_of(const torch::autograd::AutogradContext* ctx) {
    return static_cast<Ops*>(ctx->saved_data.at("ops").toCapsule().get());
}

// analysis with the transpose of the analysis as its backward
struct AnalysisFn : public torch::autograd::Function<AnalysisFn> {
    static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x,
                              const c10::intrusive_ptr<Ops>& ops) {
        ctx->saved_data["ops"] = c10::IValue::make_capsule(ops);
        return ops->analysis(x);
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                   torch::autograd::variable_list g) {
        if (!g[0].defined()) return {at::Tensor(), at::Tensor()};
        return {ops_of(ctx)->adj_analysis(g[0]), at::Tensor()};
    }
};

// synthesis with the transpose of the synthesis as its backward
struct SynthesisFn : public torch::autograd::Function<SynthesisFn> {
    static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& c,
                              const c10::intrusive_ptr<Ops>& ops) {
        ctx->saved_data["ops"] = c10::IValue::make_capsule(ops);
        return ops->synthesis(c);
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                   torch::autograd::variable_list g) {
        if (!g[0].defined()) return {at::Tensor(), at::Tensor()};
        return {ops_of(ctx)->adj_synthesis(g[0]), at::Tensor()};
    }
};

// synthesis + mean squared error against a target: outputs (loss, y), y not
// differentiable (it is a by-product for the caller); the backward runs the
// transpose of the synthesis with dL/dy = 2 dL/dloss (y - target) / n formed
// inside the kernel's load -- no elementwise loss kernels between the engines
struct SynthesisMSEFn : public torch::autograd::Function<SynthesisMSEFn> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx,
                                                  const at::Tensor& c, const at::Tensor& target,
                                                  const c10::intrusive_ptr<Ops>& ops) {
        ctx->saved_data["ops"] = c10::IValue::make_capsule(ops);
        std::vector<at::Tensor> r = ops->synthesis_sqerr(c, target);
        ctx->saved_data["y"] = r[1];
        ctx->saved_data["t"] = r[2];
        ctx->mark_non_differentiable({r[1]});
        ctx->set_materialize_grads(false);   // no zero gradient is built for y
        return {r[0], r[1]};
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                   torch::autograd::variable_list g) {
        if (!g[0].defined()) return {at::Tensor(), at::Tensor(), at::Tensor()};
        Ops* o = ops_of(ctx);
        at::Tensor y = ctx->saved_data.at("y").toTensor();
        at::Tensor t = ctx->saved_data.at("t").toTensor();
        at::Tensor gl = g[0].to(y.options()).contiguous();
        const float scale = y.numel() > 0 ? (float)(2.0 / (double)y.numel()) : 0.f;
        at::Tensor gc = o->adj_synthesis_sqerr(y, t, scale, gl);
        at::Tensor gt;
        if (ctx->needs_input_grad(1)) gt = (y - t) * (gl * -scale);
        return {gc, gt, at::Tensor()};
    }
};

// Python handle of an Ops
struct Handle {
    c10::intrusive_ptr<Ops> ops;

    Handle(uintptr_t tables, int device, int64_t ncoef, uintptr_t an, uintptr_t syn,
           uintptr_t adj_an, uintptr_t adj_syn, uintptr_t ws_bytes, uintptr_t last_error,
           uintptr_t syn_sqerr, uintptr_t adj_syn_sqerr, pybind11::object owner, std::vector<int64_t> bins, std::vector<int64_t> lens,
           int64_t ngroups)
        : ops(c10::make_intrusive<Ops>()) {
        TORCH_CHECK(bins.size() == lens.size() && ngroups <= (int64_t)bins.size(),
                    "bad group layout");
        Ops& o = *ops;
        o.tables = reinterpret_cast<const void*>(tables);
        o.device = (c10::DeviceIndex)device;
        o.ncoef = ncoef;
        o.an = reinterpret_cast<FnSignalFirst>(an);
        o.syn = reinterpret_cast<FnCoefFirst>(syn);
        o.adj_an = reinterpret_cast<FnCoefFirst>(adj_an);
        o.adj_syn = reinterpret_cast<FnSignalFirst>(adj_syn);
        o.ws_bytes = reinterpret_cast<FnWorkspace>(ws_bytes);
        o.last_error = reinterpret_cast<FnLastError>(last_error);
        o.syn_sqerr = reinterpret_cast<FnSynSqErr>(syn_sqerr);
        o.adj_syn_sqerr = reinterpret_cast<FnAdjSynSqErr>(adj_syn_sqerr);
        o.owner = owner.release().ptr();   // the strong reference moves into Ops
        int64_t total = 0;
        for (size_t i = 0; i < bins.size(); ++i) {
            o.sizes.push_back(bins[i] * lens[i]);
            total += bins[i] * lens[i];
        }
        TORCH_CHECK(total == ncoef, "group layout does not cover the heap");
        o.bins = std::move(bins);
        o.lens = std::move(lens);
        o.ngroups = ngroups;
    }

    // the grow-only scratch for `batch` slices (shared with ctypes callers)
    at::Tensor workspace(int64_t batch) {
        size_t b;
        ops->workspace(batch, &b);
        return ops->ws;
    }

    void set_slice_len(int64_t n) {
        TORCH_CHECK_VALUE(n == 65536 || n == 32768, "slice length must be 65536 or 32768");
        ops->kN = n;
    }

    at::Tensor analysis(const at::Tensor& x) { return ops->analysis(x); }
    void analysis_planar(const at::Tensor& x, const at::Tensor& kr, const at::Tensor& ki) {
        ops->analysis_planar(x, kr, ki);
    }
    void synthesis_planar(const at::Tensor& kr, const at::Tensor& ki, const at::Tensor& y) {
        ops->synthesis_planar(kr, ki, y);
    }
    at::Tensor synthesis(const at::Tensor& c) { return ops->synthesis(c); }
    at::Tensor adj_analysis(const at::Tensor& g) { return ops->adj_analysis(g); }
    at::Tensor adj_synthesis(const at::Tensor& gy) { return ops->adj_synthesis(gy); }

    // differentiable heap <-> signal, no per-group views
    at::Tensor analysis_heap(const at::Tensor& x) { return AnalysisFn::apply(x, ops); }
    at::Tensor synthesis_heap(const at::Tensor& h) { return SynthesisFn::apply(h, ops); }
    // heap [B, ncoef] and target [B, 65536] -> (mean squared error, y)
    pybind11::tuple mse(const at::Tensor& h, const at::Tensor& target) {
        torch::autograd::variable_list r = SynthesisMSEFn::apply(h, target, ops);
        return pybind11::make_tuple(r[0], r[1]);
    }

    // TrainableCQT.fwd: x [..., 65536] -> (blocks [..., b, M], side [..., 1, M])
    pybind11::tuple fwd(const at::Tensor& x) {
        Ops& o = *ops;
        TORCH_CHECK(x.dim() >= 1 && x.size(-1) == ops->kN, "x must be [..., ", ops->kN, "]");
        std::vector<int64_t> lead(x.sizes().begin(), x.sizes().end() - 1);
        int64_t B = 1;   // explicit: reshape cannot infer -1 for an empty batch
        for (int64_t d : lead) B *= d;
        // a [B, 65536] input goes in as it is: a no-op reshape would still
        // add a view node to the autograd graph
        at::Tensor h = AnalysisFn::apply(x.dim() == 2 ? x : x.reshape({B, ops->kN}), ops);
        std::vector<at::Tensor> parts = h.split_with_sizes(o.sizes, 1);
        pybind11::list blocks, side;
        o.last_v.clear();
        std::vector<int64_t> shape(lead);
        shape.push_back(0);
        shape.push_back(0);
        for (size_t i = 0; i < parts.size(); ++i) {
            shape[shape.size() - 2] = o.bins[i];
            shape[shape.size() - 1] = o.lens[i];
            at::Tensor v = parts[i].view(shape);
            o.last_v.emplace_back(v.getIntrusivePtr());
            if ((int64_t)i < o.ngroups) blocks.append(v);
            else side.append(v);
        }
        o.last_h = c10::weak_intrusive_ptr<c10::TensorImpl, c10::UndefinedTensorImpl>(
            h.getIntrusivePtr());
        return pybind11::make_tuple(blocks, side);
    }

    // the heap behind (blocks, side) when they are the untouched views the last
    // fwd returned (same tensor objects, the heap still alive), else None
    pybind11::object last_heap(const std::vector<at::Tensor>& all) {
        Ops& o = *ops;
        if (all.size() != o.last_v.size() || o.last_h.expired()) return pybind11::none();
        for (size_t i = 0; i < all.size(); ++i)
            if (o.last_v[i].expired() ||
                all[i].unsafeGetTensorImpl() != o.last_v[i]._unsafe_get_target())
                return pybind11::none();
        auto hp = o.last_h.lock();
        if (!hp) return pybind11::none();
        return pybind11::cast(at::Tensor(std::move(hp)));
    }

    // TrainableCQT.mse_loss in one call when (blocks, side) are the untouched
    // views of the last fwd: the target [lead..., 65536] is checked and
    // flattened here; (loss, y [lead..., 65536]) or None (the caller takes the
    // general path)
    pybind11::object mse_views(const std::vector<at::Tensor>& all, const at::Tensor& target) {
        pybind11::object h = last_heap(all);
        if (h.is_none()) return pybind11::none();
        at::Tensor heap = h.cast<at::Tensor>();
        const int64_t B = heap.size(0);
        std::vector<int64_t> lead(all[0].sizes().begin(), all[0].sizes().end() - 2);
        std::vector<int64_t> want(lead);
        want.push_back(ops->kN);
        TORCH_CHECK_VALUE(target.defined() && target.sizes().vec() == want, "target must be ",
                          c10::IntArrayRef(want), ", got ",
                          target.defined() ? target.sizes() : c10::IntArrayRef());
        torch::autograd::variable_list r =
            SynthesisMSEFn::apply(heap, target.dim() == 2 ? target : target.reshape({B, ops->kN}), ops);
        at::Tensor y = lead.size() == 1 ? r[1] : r[1].reshape(want);
        return pybind11::make_tuple(r[0], y);
    }
};

// ---------------------------------------------------------------------------
// AdamW: one step's host work
using FnGradNorm = decltype(&cqt_grad_norm);
using FnAdamw = decltype(&cqt_adamw_step);

// a kernel changes a tensor that autograd may have saved
void written(const at::Tensor& t) {
    if (t.defined() && !t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// whether the elements fill one stretch of memory and element i of a's is
// element i of b's (sizes are equal)
bool same_order(const at::Tensor& a, const at::Tensor& b) {
    for (int64_t d = 0; d < a.dim(); ++d)
        if (a.size(d) != 1 && a.stride(d) != b.stride(d)) return false;
    return true;
}

// The parameters of an optimizer with the states that it holds for them.  It
// remembers the Python objects that it was built from -- the lists of
// parameters, the state dictionary, every parameter's own dictionary and what
// is in them -- and refuses to step (the caller then checks them and builds
// another) when any of them has been replaced, or when what a tensor of the state
// holds is not of the type, device, size or order that the kernels take any
// more (its storage can be exchanged without replacing the object).
struct AdamWPlan {
    struct Slot {
        at::Tensor p;
        at::Tensor m, v, ms, vs, step, master;   // undefined: no state yet
        std::vector<int64_t> sizes, strides;     // of the parameter when it was checked
        at::ScalarType type;
        cqt_adamw_tensor d{};

        // whether a tensor has the parameter's sizes and strides of that time (the
        // codes of 8-bit moments are flat and do not show theirs)
        bool in_order(const at::Tensor& t) const {
            const at::IntArrayRef n = t.sizes(), s = t.strides();
            if (n.size() != sizes.size()) return false;
            for (size_t k = 0; k < sizes.size(); ++k)
                if (n[k] != sizes[k] || (s[k] != strides[k] && n[k] != 1)) return false;
            return true;
        }
        // plain memory on the device: usually seen by the same set of dispatch keys
        // as a tensor that is known to be
        static bool plain(const at::Tensor& t, at::ScalarType type, c10::DeviceIndex device,
                          const at::Tensor* known = nullptr) {
            return t.defined() && t.scalar_type() == type && t.get_device() == device &&
                   ((known && t.key_set() == known->key_set()) ||
                    (t.layout() == at::kStrided && !t.is_conj() && !t.is_neg()));
        }

        // whether the state is what the kernels take for the (plain) parameter
        bool fits(int bits, c10::DeviceIndex device) const {
            const auto like_p = [&](const at::Tensor& t, at::ScalarType type) {
                return plain(t, type, device, &p) && in_order(t);
            };
            const auto flat = [&](const at::Tensor& t, at::ScalarType type, int64_t n) {
                return plain(t, type, device, &p) && t.numel() == n && t.is_contiguous();
            };
            if (!plain(step, at::kLong, device, &p) || step.numel() != 1) return false;
            if (master.defined() && !like_p(master, at::kFloat)) return false;
            if (bits == 8) {
                const int64_t blocks = (d.numel + 255) / 256;
                return flat(m, at::kFloat8_e4m3fn, d.numel) && flat(v, at::kFloat8_e5m2, d.numel) &&
                       flat(ms, at::kFloat8_e8m0fnu, blocks) && flat(vs, at::kFloat8_e8m0fnu, blocks);
            }
            const at::ScalarType moments = type == at::kComplexFloat ? type : at::kFloat;
            return like_p(m, moments) && like_p(v, moments);
        }
    };
    struct Group {
        std::vector<Slot> slots;
        std::vector<PyObject*> params;   // the list's items (kept alive by `held`)
        int bits = 32;
        bool master = false;
    };
    std::vector<Group> groups;
    std::vector<PyObject*> seen;         // keys and values of the state, in order
    std::vector<pybind11::object> held;
    c10::DeviceIndex device;
    FnGradNorm norm_fn;
    FnAdamw step_fn;
    FnLastError last_error;
    std::vector<cqt_adamw_tensor> todo;
    std::vector<int64_t> ends;           // of each group in todo
    std::vector<at::Tensor> keep;
    std::vector<const Slot*> stepped;    // the parameters behind todo
    bool captured = false;               // a graph holds a step of this plan
    std::vector<at::Tensor> graphed;     // what it addresses beside the plan's own

    static int32_t type_of(const at::Tensor& p) {
        return p.scalar_type() == at::kBFloat16 ? CQT_BF16
               : p.scalar_type() == at::kHalf   ? CQT_F16
               : p.scalar_type() == at::kFloat || p.scalar_type() == at::kComplexFloat ? CQT_F32 : -1;
    }
    static void walk(PyObject* state, std::vector<PyObject*>& out) {
        PyObject *k, *v;
        Py_ssize_t at = 0;
        while (PyDict_Next(state, &at, &k, &v)) {
            out.push_back(k);
            out.push_back(v);
            if (!PyDict_Check(v)) continue;
            PyObject *kk, *vv;
            Py_ssize_t inner = 0;
            while (PyDict_Next(v, &inner, &kk, &vv)) out.push_back(vv);
        }
    }

    AdamWPlan(int device_, uintptr_t norm, uintptr_t step, uintptr_t error,
              pybind11::list param_groups, pybind11::dict state)
        : device((c10::DeviceIndex)device_), norm_fn(reinterpret_cast<FnGradNorm>(norm)),
          step_fn(reinterpret_cast<FnAdamw>(step)),
          last_error(reinterpret_cast<FnLastError>(error)) {
        int32_t ordinal = 0;
        for (auto g : param_groups) {
            pybind11::dict group = g.cast<pybind11::dict>();
            groups.emplace_back();
            Group& out = groups.back();
            out.bits = group["state_bits"].cast<int>();
            out.master = group["master"].cast<bool>();
            pybind11::list params = group["params"].cast<pybind11::list>();
            for (auto p : params) {
                held.push_back(pybind11::reinterpret_borrow<pybind11::object>(p));
                out.params.push_back(p.ptr());
                out.slots.emplace_back();
                Slot& s = out.slots.back();
                s.p = p.cast<at::Tensor>();
                s.type = s.p.scalar_type();
                s.sizes = s.p.sizes().vec();
                s.strides = s.p.strides().vec();
                s.d.ordinal = ordinal++;
                s.d.numel = s.p.numel() * (s.p.is_complex() ? 2 : 1);
                s.d.dtype = type_of(s.p);
                pybind11::object mine = pybind11::none();
                if (state.contains(p)) mine = state[p];
                if (!pybind11::isinstance<pybind11::dict>(mine)) continue;
                pybind11::dict d = mine.cast<pybind11::dict>();
                auto get = [&](const char* k) {
                    return d.contains(k) ? d[k].cast<at::Tensor>() : at::Tensor();
                };
                s.m = get("exp_avg");
                s.v = get("exp_avg_sq");
                s.step = get("step");
                if (out.bits == 8) {
                    s.ms = get("exp_avg_scale");
                    s.vs = get("exp_avg_sq_scale");
                }
                if (out.master && s.d.dtype != CQT_F32) s.master = get("master");
                // (a parameter without a gradient has not been checked by the caller)
                if (!plan_takes(s, out.bits, get("order")))
                    s.m = s.v = s.ms = s.vs = s.step = s.master = at::Tensor();
            }
        }
        walk(state.ptr(), seen);
        for (PyObject* o : seen) held.push_back(pybind11::reinterpret_borrow<pybind11::object>(o));
    }

    // whether a parameter is what the kernels take, in the memory order of its state
    // (of 8-bit moments: the sizes over the strides; those of a contiguous parameter
    // if nothing says it)
    bool plan_takes(const Slot& s, int bits, const at::Tensor& order) const {
        if (s.d.dtype < 0 || !Slot::plain(s.p, s.type, device) || !s.p.is_non_overlapping_and_dense())
            return false;
        if (bits != 8) return true;   // their own order is compared at each step
        if (!order.defined()) return s.p.is_contiguous();
        const int64_t dims = s.p.dim();
        if (order.scalar_type() != at::kLong || order.dim() != 2 || order.size(0) != 2 ||
            order.size(1) != dims)
            return false;
        const at::Tensor host = order.cpu().contiguous();
        const int64_t* n = host.data_ptr<int64_t>();
        for (int64_t k = 0; k < dims; ++k)
            if (n[k] != s.sizes[k] || (n[dims + k] != s.strides[k] && n[k] != 1)) return false;
        return true;
    }

    // whether what this was built from is still what the optimizer holds
    bool current(const pybind11::list& param_groups, const pybind11::dict& state) const {
        if (param_groups.size() != groups.size()) return false;
        PyObject *k, *v;
        Py_ssize_t at = 0;
        size_t i = 0;
        auto next = [&](PyObject* o) { return i < seen.size() && seen[i++] == o; };
        while (PyDict_Next(state.ptr(), &at, &k, &v)) {
            if (!next(k) || !next(v)) return false;
            if (!PyDict_Check(v)) continue;
            PyObject *kk, *vv;
            Py_ssize_t inner = 0;
            while (PyDict_Next(v, &inner, &kk, &vv))
                if (!next(vv)) return false;
        }
        return i == seen.size();
    }

    // fills `todo` with the parameters that have gradients; false where one of
    // them has no state yet, or not one for its present shape
    bool gather(const pybind11::list& param_groups) {
        todo.clear();
        ends.clear();
        keep.clear();
        stepped.clear();
        size_t k = 0;
        for (auto gr : param_groups) {
            Group& g = groups[k++];
            PyObject* group = gr.ptr();
            PyObject* params = PyDict_GetItemString(group, "params");
            if (!params || !PyList_Check(params) ||
                (size_t)PyList_GET_SIZE(params) != g.params.size() ||
                number(item(group, "state_bits")) != g.bits ||
                PyObject_IsTrue(item(group, "master")) != (g.master ? 1 : 0))
                return false;
            for (size_t i = 0; i < g.slots.size(); ++i) {
                if (PyList_GET_ITEM(params, (Py_ssize_t)i) != g.params[i]) return false;
                Slot& s = g.slots[i];
                const at::Tensor& p = s.p;
                const at::Tensor& grad = p.grad();
                if (!grad.defined() || p.numel() == 0) continue;
                if (!s.m.defined() || !s.v.defined() || !s.step.defined()) return false;
                TORCH_CHECK(grad.layout() == at::kStrided, "sparse gradients are not supported");
                TORCH_CHECK_VALUE(grad.scalar_type() == p.scalar_type() &&
                                      grad.device() == p.device() && grad.sizes() == p.sizes(),
                                  "a gradient must be ", p.scalar_type(), " ", p.sizes(), " on ",
                                  p.device(), ", got ", grad.scalar_type(), " ", grad.sizes(),
                                  " on ", grad.device());
                // the storage of a parameter or of a state may have been exchanged
                if (!Slot::plain(p, s.type, device) || !s.in_order(p) || !s.fits(g.bits, device))
                    return false;
                at::Tensor use = grad;
                if (grad.is_conj() || grad.is_neg() || !same_order(grad, p)) {
                    use = at::empty_like(p).copy_(grad);
                    keep.push_back(use);
                }
                s.d.param = p.data_ptr();
                s.d.grad = use.data_ptr();
                s.d.master = s.master.defined() ? s.master.data_ptr<float>() : nullptr;
                s.d.exp_avg = s.m.data_ptr();
                s.d.exp_avg_sq = s.v.data_ptr();
                s.d.exp_avg_scale =
                    s.ms.defined() ? static_cast<uint8_t*>(s.ms.data_ptr()) : nullptr;
                s.d.exp_avg_sq_scale =
                    s.vs.defined() ? static_cast<uint8_t*>(s.vs.data_ptr()) : nullptr;
                s.d.step = s.step.data_ptr<int64_t>();
                todo.push_back(s.d);
                stepped.push_back(&s);
            }
            ends.push_back((int64_t)todo.size());
        }
        return true;
    }

    // whether a step would take everything as it is
    bool fits(pybind11::list param_groups, pybind11::dict state) {
        at::NoGradGuard no_grad;
        const bool yes = current(param_groups, state) && gather(param_groups);
        keep.clear();
        return yes;
    }

    // an option of a parameter group
    static PyObject* item(PyObject* group, const char* key) {
        PyObject* o = PyDict_GetItemString(group, key);
        if (!o) throw pybind11::key_error(key);
        return o;
    }
    static double number(PyObject* o) {
        const double x = PyFloat_AsDouble(o);
        if (x == -1.0 && PyErr_Occurred()) throw pybind11::error_already_set();
        return x;
    }

    // Autograd refuses a backward pass through values that it saved before a step,
    // as behind any operation in place: marks what the launches write, behind
    // them (the GPU is at work meanwhile) and also behind one that failed.
    struct Marks {
        const AdamWPlan& plan;
        const at::Tensor* norm;
        ~Marks() {
            for (const Slot* x : plan.stepped)
                for (const at::Tensor* t : {&x->p, &x->m, &x->v, &x->ms, &x->vs, &x->step, &x->master})
                    written(*t);
            if (norm) written(*norm);
        }
    };

    // one step; false (nothing done) when the plan does not fit any more
    bool step(pybind11::list param_groups, pybind11::dict state, pybind11::object max_norm,
              uint32_t seed, const at::Tensor& ws, const c10::optional<at::Tensor>& norm) {
        at::NoGradGuard no_grad;
        if (!current(param_groups, state)) return false;
        Ops::DeviceSwitch sw(device);
        if (!gather(param_groups)) return false;
        void* stream = at::cuda::getCurrentCUDAStream(device).stream();
        auto check = [&](int rc, const char* what) {
            TORCH_CHECK(rc == 0, what, " failed (", rc, "): ", last_error());
        };
        // all options are read and checked before anything is changed
        std::vector<cqt_adamw_args> args;
        int use_norm = max_norm.is_none() ? 0 : 2;   // 1 after the launch behind the norm
        for (auto gr : param_groups) {
            PyObject* g = gr.ptr();
            PyObject* lr = item(g, "lr");
            cqt_adamw_args a{};
            a.max_norm = use_norm ? number(max_norm.ptr()) : 0.0;
            a.seed = seed;
            if (THPVariable_Check(lr) && THPVariable_Unpack(lr).is_cuda()) {
                const at::Tensor& t = THPVariable_Unpack(lr);
                TORCH_CHECK_TYPE(t.scalar_type() == at::kFloat, "a device lr must be float32, got ",
                                 t.scalar_type());
                TORCH_CHECK_VALUE(t.numel() == 1 && t.get_device() == device,
                                  "a device lr must hold one number on cuda:", (int)device);
                a.lr_dev = t.data_ptr<float>();
            } else {
                a.lr = THPVariable_Check(lr) ? THPVariable_Unpack(lr).item<double>() : number(lr);
            }
            pybind11::sequence bs = pybind11::reinterpret_borrow<pybind11::sequence>(item(g, "betas"));
            a.beta1 = bs[0].cast<double>();
            a.beta2 = bs[1].cast<double>();
            a.eps = number(item(g, "eps"));
            a.weight_decay = number(item(g, "weight_decay"));
            TORCH_CHECK_VALUE(a.lr >= 0, "lr must not be negative, got ", a.lr);
            TORCH_CHECK_VALUE(a.beta1 >= 0 && a.beta1 < 1 && a.beta2 >= 0 && a.beta2 < 1,
                              "betas must lie in [0, 1), got ", a.beta1, ", ", a.beta2);
            TORCH_CHECK_VALUE(a.eps >= 0 && a.weight_decay >= 0,
                              "eps and weight_decay must not be negative");
            args.push_back(a);
        }
        TORCH_CHECK_VALUE(!use_norm || args.empty() || args[0].max_norm > 0,
                          "max_norm must be positive");
        TORCH_CHECK_VALUE(!use_norm || (norm->get_device() == device && norm->numel() == 1 &&
                                        norm->scalar_type() == at::kFloat),
                          "grad_norm must hold one float32 number on cuda:", (int)device);
        if (c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) {
            // the graph addresses what this plan holds, the rates and the norm
            captured = true;
            if (use_norm) graphed.push_back(*norm);
            for (auto gr : param_groups)
                held.push_back(pybind11::reinterpret_borrow<pybind11::object>(item(gr.ptr(), "lr")));
        }
        const Marks marks{*this, use_norm ? &*norm : nullptr};
        if (use_norm) {
            check(norm_fn(todo.data(), (int)todo.size(), norm->data_ptr<float>(), ws.data_ptr(),
                          (size_t)ws.numel(), stream),
                  "cqt_grad_norm");
        }
        int64_t first = 0;
        for (size_t k = 0; k < args.size(); ++k) {
            const int64_t last = ends[k];
            if (last == first) continue;
            args[k].use_norm = use_norm;
            check(step_fn(todo.data() + first, (int)(last - first), groups[k].bits, &args[k],
                          ws.data_ptr(), (size_t)ws.numel(), stream),
                  "cqt_adamw_step");
            if (use_norm) use_norm = 1;
            first = last;
        }
        keep.clear();
        return true;
    }
};

// ---------------------------------------------------------------------------
// CoefCache: the per-call host work of append and window
using FnCacheAppend = decltype(&cqt_cache_append);
using FnCacheWindow = decltype(&cqt_cache_window);

struct CacheHandle {
    at::Tensor codes, scales, length, ws;
    at::Tensor own[3];   // the same storage, kept whatever is done to those objects
    std::vector<int64_t> lead;
    std::vector<int32_t> bands, lens;
    int64_t ngroups, rows = 1, ncoef = 0;
    c10::DeviceIndex device;
    cqt_cache desc{};
    FnCacheAppend append_fn;
    FnCacheWindow window_fn;
    FnLastError last_error;

    CacheHandle(uintptr_t append, uintptr_t window, uintptr_t error, at::Tensor codes_,
                at::Tensor scales_, at::Tensor length_, at::Tensor ws_, int64_t capacity,
                int format, std::vector<int32_t> bands_, std::vector<int32_t> lens_,
                int64_t ngroups_)
        : codes(std::move(codes_)), scales(std::move(scales_)), length(std::move(length_)),
          ws(std::move(ws_)), lead(length.sizes().vec()), bands(std::move(bands_)),
          lens(std::move(lens_)), ngroups(ngroups_), device((c10::DeviceIndex)codes.get_device()),
          append_fn(reinterpret_cast<FnCacheAppend>(append)),
          window_fn(reinterpret_cast<FnCacheWindow>(window)),
          last_error(reinterpret_cast<FnLastError>(error)) {
        for (int64_t d : lead) rows *= d;
        for (size_t k = 0; k < bands.size(); ++k) ncoef += (int64_t)bands[k] * lens[k];
        own[0] = codes.detach();
        own[1] = scales.detach();
        own[2] = length.detach();
        desc.codes = codes.data_ptr();
        desc.scales = static_cast<uint8_t*>(scales.data_ptr());
        desc.length = length.data_ptr<int64_t>();
        desc.workspace = ws.data_ptr();
        desc.rows = (int32_t)rows;
        desc.capacity = (int32_t)capacity;
        desc.format = format;
        desc.ngroups = (int32_t)bands.size();
        desc.group_count = bands.data();
        desc.group_len = lens.data();
    }
    CacheHandle(const CacheHandle&) = delete;   // desc points into the vectors

    void check(int rc, const char* what) const {
        TORCH_CHECK(rc == 0, what, " failed (", rc, "): ", last_error());
    }

    // the store's tensors are public, and their storage can be exchanged
    void check_store() const {
        TORCH_CHECK_VALUE(codes.data_ptr() == desc.codes && scales.data_ptr() == desc.scales &&
                              length.data_ptr() == desc.length,
                          "the cache's codes, scales or length have another storage than they "
                          "were made with (copy into them instead)");
    }

    const int64_t* numbers(const c10::optional<at::Tensor>& t, const char* name,
                           at::Tensor& hold) const {
        if (!t) return nullptr;
        TORCH_CHECK_VALUE(t->is_cuda() && t->get_device() == device &&
                              t->scalar_type() == at::kLong && t->sizes() == at::IntArrayRef(lead),
                          name, " must be an int64 tensor ", at::IntArrayRef(lead), " on cuda:",
                          (int)device);
        hold = t->contiguous();
        return hold.data_ptr<int64_t>();
    }

    // false (nothing done) for shapes that the caller has to sort out or refuse
    bool append(const std::vector<at::Tensor>& all, const c10::optional<at::Tensor>& counts) {
        at::NoGradGuard no_grad;
        check_store();
        const size_t L = lead.size();
        if (all.size() != bands.size() || all[0].dim() != (int64_t)L + 2) return false;
        const int64_t S = all[0].size((int64_t)L + 1) / lens[0];
        cqt_cache_part parts[16];
        for (size_t k = 0; k < all.size(); ++k) {
            const at::Tensor& c = all[k];
            if (!c.defined() || !c.is_cuda() || c.get_device() != device ||
                c.scalar_type() != at::kComplexFloat || c.is_conj() || c.is_neg())
                return false;
            const bool side = (int64_t)k >= ngroups;
            const int64_t b = bands[k], M = lens[k];
            const int64_t want = !side || c.dim() == (int64_t)L + 2 ? (int64_t)L + 2 : (int64_t)L + 3;
            if (c.dim() != want || c.sizes().slice(0, L) != at::IntArrayRef(lead)) return false;
            const bool one = side && want == (int64_t)L + 2;
            if (!side ? (c.size(L) != b || c.size(L + 1) != S * M)
                      : one ? (S != 1 || c.size(L) != b || c.size(L + 1) != M)
                            : (c.size(L) != S || c.size(L + 1) != b || c.size(L + 2) != M))
                return false;
            // the leading dimensions have to be one stride
            if (c.stride(-1) != 1 || reinterpret_cast<uintptr_t>(c.data_ptr()) % 8) return false;
            int64_t row = 0, span = 1;
            for (size_t d = L; d-- > 0;) {
                if (lead[d] == 1) continue;
                if (span == 1) row = c.stride((int64_t)d);
                else if (c.stride((int64_t)d) != row * span) return false;
                span *= lead[d];
            }
            parts[k].data = c.data_ptr();
            parts[k].row_stride = row;
            if (!side) {
                parts[k].slice_stride = M;
                parts[k].band_stride = c.stride((int64_t)L);
            } else {
                parts[k].slice_stride = one ? 0 : c.stride((int64_t)L);
                parts[k].band_stride = c.stride(one ? (int64_t)L : (int64_t)L + 1);
            }
        }
        at::Tensor hold;
        const int64_t* n = numbers(counts, "counts", hold);
        Ops::DeviceSwitch sw(device);
        check(append_fn(&desc, parts, (int)S, n, at::cuda::getCurrentCUDAStream(device).stream()),
              "cqt_cache_append");
        for (const at::Tensor* t : {&codes, &scales, &length}) written(*t);
        return true;
    }

    pybind11::tuple window(int64_t n, at::ScalarType dtype, int type,
                           const c10::optional<at::Tensor>& end) {
        at::NoGradGuard no_grad;
        check_store();
        at::Tensor hold;
        const int64_t* e = numbers(end, "end", hold);
        const bool cplx = dtype == at::kComplexFloat;
        const int64_t item = cplx ? 1 : 2;   // scalars of one coefficient
        Ops::DeviceSwitch sw(device);
        at::Tensor out = at::empty({rows * n * ncoef * item}, codes.options().dtype(dtype));
        char* base = static_cast<char*>(out.data_ptr());
        cqt_cache_part parts[16];
        pybind11::list blocks, side;
        int64_t off = 0;
        for (size_t k = 0; k < bands.size(); ++k) {
            const int64_t b = bands[k], M = lens[k], row = n * b * M;
            parts[k] = {base + (size_t)off * item * out.element_size(), row, M, n * M};
            std::vector<int64_t> sz(lead);
            if ((int64_t)k < ngroups) {
                sz.insert(sz.end(), {b, n * M});
            } else {
                parts[k].slice_stride = b * M;
                parts[k].band_stride = M;
                sz.insert(sz.end(), {n, b, M});
            }
            if (!cplx) sz.push_back(2);
            std::vector<int64_t> st(sz.size());
            int64_t step = 1;
            for (size_t d = sz.size(); d-- > 0;) {
                st[d] = step;
                step *= sz[d] > 1 ? sz[d] : 1;
            }
            at::Tensor v = out.as_strided(sz, st, off * item);
            if ((int64_t)k < ngroups) blocks.append(v);
            else side.append(v);
            off += rows * row;
        }
        check(window_fn(&desc, parts, (int)n, e, type,
                        at::cuda::getCurrentCUDAStream(device).stream()),
              "cqt_cache_window");
        return pybind11::make_tuple(blocks, side);
    }
};

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.doc() = "torch fast path of the flash_cqt_b200 C ABI";
    pybind11::class_<Handle>(m, "Handle")
        .def(pybind11::init<uintptr_t, int, int64_t, uintptr_t, uintptr_t, uintptr_t, uintptr_t,
                            uintptr_t, uintptr_t, uintptr_t, uintptr_t, pybind11::object,
                            std::vector<int64_t>, std::vector<int64_t>, int64_t>())
        .def("workspace", &Handle::workspace)
        .def("set_slice_len", &Handle::set_slice_len)
        .def("analysis", &Handle::analysis)
        .def("analysis_planar", &Handle::analysis_planar)
        .def("synthesis_planar", &Handle::synthesis_planar)
        .def("synthesis", &Handle::synthesis)
        .def("adj_analysis", &Handle::adj_analysis)
        .def("adj_synthesis", &Handle::adj_synthesis)
        .def("analysis_heap", &Handle::analysis_heap)
        .def("synthesis_heap", &Handle::synthesis_heap)
        .def("mse", &Handle::mse)
        .def("mse_views", &Handle::mse_views)
        .def("fwd", &Handle::fwd)
        .def("last_heap", &Handle::last_heap);
    pybind11::class_<AdamWPlan>(m, "AdamWPlan")
        .def(pybind11::init<int, uintptr_t, uintptr_t, uintptr_t, pybind11::list, pybind11::dict>())
        .def_readonly("captured", &AdamWPlan::captured)
        .def("fits", &AdamWPlan::fits)
        .def("step", &AdamWPlan::step);
    pybind11::class_<CacheHandle>(m, "CacheHandle")
        .def(pybind11::init<uintptr_t, uintptr_t, uintptr_t, at::Tensor, at::Tensor, at::Tensor,
                            at::Tensor, int64_t, int, std::vector<int32_t>, std::vector<int32_t>,
                            int64_t>())
        .def("append", &CacheHandle::append)
        .def("window", &CacheHandle::window);
}
