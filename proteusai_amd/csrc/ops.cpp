// The operators' host path in C++: allocations, launches and autograd nodes of geometric attention, of the two wavefunction embeddings, of the norm and rotation of
// queries and keys, of the gated feed-forward block, of the loss over a vocabulary, of the clipping of gradients and of AdamW's step for ordinary calls.
//
// Every function here takes a call only if it is the plain one -- ordinary tensors of the kernels' own types and layouts on the current GPU, and nothing that looks on (functional
// transforms, forward-mode differentiation, dispatch modes, tracing) -- and answers None otherwise: the Python functions, which convert, check and raise, do the
// rest, and the backward of a node hands whatever is not plain (gradients without memory of their own, saved tensors that hooks gave back in another form) to them, too.
// Us of a forward and backward that the host bounds, Python / this: attention of 64 tokens 86 to 170 / 46 to 80 (the higher figures are processes whose autograd thread
// waits longer for the interpreter's lock, which the backward no longer takes), with the spreads checked 110 to 193 / 56, embedding of 2 x 512 70 to 131 / 48; a forward alone 11.5 / 7.1 and
// 22.6 / 18.5 (the GPU's time).
#include <torch/extension.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>
#include <algorithm>
#include <climits>
#include <ATen/autocast_mode.h>
#include "proteus_hip.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

// ---- which calls ----

// Does nothing look on that expects torch operators?
bool unobserved()
{
    return !c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode) && !c10::impl::TorchDispatchModeTLS::any_modes_set() && !torch::jit::tracer::isTracing();
}

// A tensor with memory of its own on the current GPU that carries no tangent.
bool plain(const Tensor& t)
{
    if (!t.defined() || t.layout() != at::kStrided || !t.is_cuda()) return false;
    const auto keys = t.unsafeGetTensorImpl()->key_set();
    return !keys.has(c10::DispatchKey::Python) && !keys.has(c10::DispatchKey::FuncTorchBatched) && !keys.has(c10::DispatchKey::FuncTorchGradWrapper)
           && !keys.has(c10::DispatchKey::Functionalize) && !keys.has(c10::DispatchKey::ZeroTensor) && !keys.has(c10::DispatchKey::Negative)
           && t.has_storage() && !t._fw_grad(0).defined();
}

// The same of many tensors, where no forward-mode differentiation goes on: its keys in one look (500 tensors in five lists 73 us / 42).
bool plain_in_bulk(const Tensor& t)
{
    static const c10::DispatchKeySet wanted(c10::DispatchKey::CUDA), other({c10::DispatchKey::Python, c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Functionalize,
                                                                           c10::DispatchKey::ZeroTensor, c10::DispatchKey::Negative});
    if (!t.defined()) return false;
    const c10::TensorImpl* const i = t.unsafeGetTensorImpl();
    return i->key_set().has_all(wanted) && !i->key_set().has_any(other) && i->has_storage();
}

// The tensor behind a Python object that is exactly a Tensor or Parameter and plain, on device `dev` (any, the current one, where that is negative).
bool get(const py::object& o, Tensor& t, const int dev = -1)
{
    if (!THPVariable_CheckExact(o.ptr())) return false;
    t = THPVariable_Unpack(o.ptr());
    return plain(t) && (dev < 0 || t.get_device() == dev);
}

bool f32(const Tensor& t) { return t.scalar_type() == at::kFloat && t.is_contiguous(); }
const float* floats(const Tensor& t) { return static_cast<const float*>(t.const_data_ptr()); }
float* out_floats(const Tensor& t) { return static_cast<float*>(t.mutable_data_ptr()); }
const uint16_t* halves(const Tensor& t) { return static_cast<const uint16_t*>(t.const_data_ptr()); }
const uint8_t* bytes(const Tensor& t) { return t.defined() ? static_cast<const uint8_t*>(t.const_data_ptr()) : nullptr; }
bool off(const Tensor& t, const uintptr_t by) { return (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & (by - 1)) != 0; }

// An optional padding mask [Z, N]: None, or a dense bool tensor.
bool get_mask(const py::object& o, Tensor& m, const int dev, const int64_t Z, const int64_t N)
{
    if (o.is_none()) return true;
    return get(o, m, dev) && m.scalar_type() == at::kBool && m.is_contiguous() && m.dim() == 2 && m.size(0) == Z && m.size(1) == N;
}

bool current(const int dev)
{
    int now = -1;
    return hipGetDevice(&now) == hipSuccess && now == dev;
}

void* stream_of(const int dev) { return c10::hip::getCurrentHIPStream(static_cast<c10::DeviceIndex>(dev)).stream(); }

// What the library does not take, or could not launch, goes the general way, which says what is wrong with it (as a ValueError or a ProteusError).
struct Refused {};
void launched(const int rc) { if (rc != 0) throw Refused(); }

at::TensorOptions on(const Tensor& t, const at::ScalarType type) { return t.options().dtype(type).requires_grad(false); }

// ---- geometric attention ----

// Can the kernels read or write this [Z,H,N,d] tensor in place?  (Rows of d contiguous elements on multiples of 16 bytes, no negative or overlapping strides.)
bool rows_ok(const Tensor& t, const int64_t itemsize)
{
    if (off(t, 16)) return false;
    if (t.is_contiguous()) return true;
    const int64_t per16 = 16 / itemsize;
    if (t.stride(3) != 1 || t.stride(2) < t.size(3) || t.size(2) * t.stride(2) * itemsize >= (1LL << 31)) return false;
    for (int i = 0; i < 3; ++i) if (t.stride(i) < 0 || t.stride(i) % per16) return false;
    return (t.size(0) == 1 || t.stride(0) > 0) && (t.size(1) == 1 || t.stride(1) > 0);
}

struct Strides {
    int64_t v[21];
    bool dense = true;
    int n = 0;
    void add(const Tensor& t) { for (int i = 0; i < 3; ++i) v[n++] = t.stride(i); dense = dense && t.is_contiguous(); }
    const int64_t* get() const { return dense ? nullptr : v; }
};

struct Logits { bool legacy, f16; double min_rbf, max_rbf; };

std::pair<Tensor, Tensor> attention_forward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& coords, const Tensor& sigma, const Tensor& betas, const Tensor& mask,
                                            const Logits& how, const bool token_major)
{
    const int64_t Z = q.size(0), H = q.size(1), N = q.size(2), d = q.size(3);
    const auto opt = on(q, at::kFloat);
    const Tensor O = token_major ? at::empty({Z, N, H, d}, opt).permute({0, 2, 1, 3}) : at::empty({Z, H, N, d}, opt);
    const Tensor L = at::empty({Z, H, N}, opt);
    Strides st;
    for (const Tensor* t : {&q, &k, &v, &O}) st.add(*t);
    void* const stream = stream_of(q.get_device());
    if (!how.legacy) {
        const size_t need = proteus_geo_attn_fwd_workspace_bytes(Z, H, N, d, 0);
        Tensor ws;
        if (need) ws = at::empty({static_cast<int64_t>(need)}, on(q, at::kByte));
        launched(proteus_geo_attn_fwd_ws(halves(q), halves(k), halves(v), st.get(), floats(coords), floats(sigma), bytes(mask), out_floats(O), out_floats(L),
                                         need ? ws.mutable_data_ptr() : nullptr, need, Z, H, N, d, 0, stream));
    } else {
        // (contiguous tensors may have any stride along a dimension of size one, which the strided entry point would hold against them)
        const int type = how.f16 ? PROTEUS_OPERAND_F16 : PROTEUS_OPERAND_BF16;
        launched(st.get() ? proteus_geo_attn_legacy_fwd_strided(halves(q), halves(k), halves(v), st.get(), floats(coords), floats(sigma), floats(betas), bytes(mask), out_floats(O), out_floats(L),
                                                                Z, H, N, d, how.min_rbf, how.max_rbf, type, 0, stream)
                          : proteus_geo_attn_legacy_fwd(halves(q), halves(k), halves(v), floats(coords), floats(sigma), floats(betas), bytes(mask), out_floats(O), out_floats(L),
                                                        Z, H, N, d, how.min_rbf, how.max_rbf, type, 0, stream));
    }
    return {O, L};
}

PyObject* g_attention_backward = nullptr;        // the Python function (set once, when the module is set up)

// What is not plain: gradients and saved tensors as the Python function takes them.
variable_list attention_backward_general(const variable_list& s, const Tensor& dO, const Logits& how)
{
    py::gil_scoped_acquire gil;
    auto opt = [](const Tensor& t) -> py::object { return t.defined() ? py::cast(t) : py::none(); };
    const py::object got = py::reinterpret_borrow<py::object>(g_attention_backward)(s[0], s[1], s[2], s[3], s[4], dO, s[5], s[6], opt(s[8]), opt(s[7]), how.min_rbf, how.max_rbf, how.f16);
    variable_list out;
    for (const auto& o : py::reinterpret_borrow<py::tuple>(got)) out.push_back(o.is_none() ? Tensor() : o.cast<Tensor>());
    return out;                                  // dQ, dK, dV, d_sigma, d_betas
}

variable_list attention_backward_plain(const variable_list& s, const Tensor& dO, const Logits& how)
{
    const Tensor &q = s[0], &k = s[1], &v = s[2], &O = s[3], &L = s[4], &coords = s[5], &sigma = s[6], &betas = s[7], &mask = s[8];
    const auto op = how.f16 ? at::kHalf : at::kBFloat16;
    const auto type = dO.defined() ? dO.scalar_type() : at::kByte;
    bool ok = unobserved() && (type == at::kFloat || type == at::kBFloat16 || type == at::kHalf) && plain(dO) && current(dO.get_device()) && O.dim() == 4 && O.sizes() == dO.sizes();
    for (const Tensor* t : {&q, &k, &v}) ok = ok && plain(*t) && t->scalar_type() == op && t->sizes() == O.sizes() && rows_ok(*t, 2);
    for (const Tensor* t : {&L, &coords, &sigma}) ok = ok && plain(*t) && f32(*t);
    ok = ok && plain(O) && O.scalar_type() == at::kFloat;
    if (!ok) return attention_backward_general(s, dO, how);
    const int64_t Z = O.size(0), H = O.size(1), N = O.size(2), d = O.size(3);
    ok = L.numel() == Z * H * N && coords.numel() == Z * N * 3 && sigma.numel() == H;
    for (const Tensor* t : {&q, &k, &v, &O, &L, &coords, &sigma}) ok = ok && t->get_device() == dO.get_device();
    if (betas.defined()) ok = ok && plain(betas) && f32(betas) && betas.numel() == H && betas.get_device() == dO.get_device();
    if (mask.defined())  ok = ok && plain(mask) && mask.scalar_type() == at::kBool && mask.is_contiguous() && mask.numel() == Z * N && mask.get_device() == dO.get_device();
    ok = ok && !off(O, 16) && !off(dO, 4 * dO.element_size());
    if (!(O.is_contiguous() && dO.is_contiguous()))
        for (const Tensor* t : {&O, &dO}) {
            ok = ok && t->stride(3) == 1 && t->stride(2) >= d;
            for (int i = 0; i < 3; ++i) ok = ok && t->stride(i) % 4 == 0;
        }
    if (!ok) return attention_backward_general(s, dO, how);
    Tensor cast = dO;
    if (type != op) cast = at::empty_like(dO, on(dO, op));
    if (!rows_ok(cast, 2)) return attention_backward_general(s, dO, how);

    const auto opt = on(O, at::kFloat);
    const Tensor D = at::empty({Z, H, N}, opt), d_sigma = at::empty({H}, opt);
    const Tensor d_beta = betas.defined() ? at::empty({H}, opt) : Tensor();
    float* const to_beta = betas.defined() ? out_floats(d_beta) : nullptr;
    const int operand = how.f16 ? PROTEUS_OPERAND_F16 : PROTEUS_OPERAND_BF16;
    void* const stream = stream_of(O.get_device());
    Strides prep;
    for (const Tensor* t : {&O, &dO, static_cast<const Tensor*>(&cast)}) prep.add(*t);
    launched(proteus_geo_attn_prepare_bwd(floats(O), dO.const_data_ptr(), prep.get(), out_floats(D), type != op ? static_cast<uint16_t*>(cast.mutable_data_ptr()) : nullptr, out_floats(d_sigma),
                                          to_beta, Z, H, N, d, type == at::kFloat ? PROTEUS_DTYPE_F32 : type == at::kHalf ? PROTEUS_DTYPE_F16 : PROTEUS_DTYPE_BF16, operand, stream));
    // gradients in the memory order of their operands (dense) and in their type
    auto like = [&](const Tensor& t) {
        const Tensor g = at::empty_like(t, on(t, op));
        return rows_ok(g, 2) ? g : at::empty({Z, H, N, d}, on(t, op));
    };
    const Tensor dq = like(q), dk = like(k), dv = like(v);
    Strides st;
    for (const Tensor* t : {&q, &k, &v, static_cast<const Tensor*>(&cast), &dq, &dk, &dv}) st.add(*t);
    launched(proteus_geo_attn_bwd_typed(halves(q), halves(k), halves(v), halves(cast), st.get(), floats(coords), floats(sigma), betas.defined() ? floats(betas) : nullptr, bytes(mask),
                                        floats(L), floats(D), dq.mutable_data_ptr(), dk.mutable_data_ptr(), dv.mutable_data_ptr(), out_floats(d_sigma), to_beta, Z, H, N, d,
                                        how.legacy ? how.min_rbf : 0.0, how.legacy ? how.max_rbf : 1.0, operand, PROTEUS_GRAD_OPERAND, stream));
    return {dq, dk, dv, d_sigma, d_beta};
}

variable_list attention_backward(const variable_list& s, const Tensor& dO, const Logits& how)
{
    try {
        return attention_backward_plain(s, dO, how);
    } catch (const Refused&) {
        return attention_backward_general(s, dO, how);
    }
}

struct Attention : torch::autograd::Function<Attention> {
    static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& coords, const Tensor& spreads,
                          const std::optional<Tensor>& betas, const std::optional<Tensor>& mask, bool legacy, bool f16, double min_rbf, double max_rbf, bool token_major)
    {
        const Tensor b = betas.value_or(Tensor()), m = mask.value_or(Tensor());
        const auto [O, L] = attention_forward(q, k, v, coords, spreads, b, m, Logits{legacy, f16, min_rbf, max_rbf}, token_major);
        ctx->save_for_backward({q, k, v, O, L, coords, spreads, b, m});
        ctx->saved_data["legacy"] = legacy; ctx->saved_data["f16"] = f16;
        ctx->saved_data["min"] = min_rbf; ctx->saved_data["max"] = max_rbf;
        return O;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        const Logits how{ctx->saved_data["legacy"].toBool(), ctx->saved_data["f16"].toBool(), ctx->saved_data["min"].toDouble(), ctx->saved_data["max"].toDouble()};
        const variable_list g = attention_backward(ctx->get_saved_variables(), grads[0], how);
        return {g[0], g[1], g[2], Tensor(), g[3], g[4], Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

// The spreads' values on their way to the host while the kernels that read them are launched: a call that waited for them first left the GPU without work for
// as long as the host then takes to launch.
struct Arriving {
    Tensor host;
    hipEvent_t done = nullptr;
    Arriving(const Tensor& t, hipStream_t stream)
    {
        host = at::empty({t.numel()}, at::TensorOptions().dtype(at::kFloat).device(at::kCPU).pinned_memory(true));
        if (hipEventCreateWithFlags(&done, hipEventDisableTiming) != hipSuccess) { done = nullptr; return; }
        if (hipMemcpyAsync(host.mutable_data_ptr(), t.const_data_ptr(), t.numel() * 4, hipMemcpyDeviceToHost, stream) != hipSuccess || hipEventRecord(done, stream) != hipSuccess) {
            (void)hipStreamSynchronize(stream);
            (void)hipEventDestroy(done);
            done = nullptr;
        }
    }
    ~Arriving() { if (done) { (void)hipEventSynchronize(done); (void)hipEventDestroy(done); } }          // (the memory is written until then)
    // Once they are there: are all of them positive numbers?
    bool positive()
    {
        if (!done || hipEventSynchronize(done) != hipSuccess) return false;
        const float* v = floats(host);
        for (int64_t i = 0; i < host.numel(); ++i) if (!(v[i] > 0.0f)) return false;
        return true;
    }
};

// geometric_attn(...) with O in fp32, or None.
py::object attention(const py::object& Q, const py::object& K, const py::object& V, const py::object& coords_, const py::object& spreads_, const py::object& betas_, const py::object& mask_,
                     const double min_rbf, const double max_rbf, const bool check, const bool token_major, const bool f16)
{
    Tensor q, k, v, coords, spreads, betas, mask;
    if (!unobserved() || !get(Q, q) || q.dim() != 4) return py::none();
    const int dev = q.get_device();
    const int64_t Z = q.size(0), H = q.size(1), N = q.size(2), d = q.size(3);
    const auto op = f16 ? at::kHalf : at::kBFloat16;
    const bool legacy = !betas_.is_none();
    if ((f16 && !legacy) || !current(dev) || !get(K, k, dev) || !get(V, v, dev) || !get(coords_, coords, dev) || !get(spreads_, spreads, dev) || !get_mask(mask_, mask, dev, Z, N)
        || (legacy && !get(betas_, betas, dev))) return py::none();
    for (const Tensor* t : {&q, &k, &v}) if (t->scalar_type() != op || t->sizes() != q.sizes() || !rows_ok(*t, 2)) return py::none();
    if (Z <= 0 || H <= 0 || N <= 0 || (d != 32 && d != 64 && d != 128) || N > PROTEUS_ATTN_MAX_N || Z * H > 65535
        || !f32(coords) || coords.dim() != 3 || coords.size(0) != Z || coords.size(1) != N || coords.size(2) != 3
        || !f32(spreads) || spreads.dim() != 1 || spreads.size(0) != H || (legacy && (!f32(betas) || betas.dim() != 1 || betas.size(0) != H || !(max_rbf > min_rbf)))
        || N * H * d * 4 >= (1LL << 31)) return py::none();
    const hipStream_t stream = static_cast<hipStream_t>(stream_of(dev));
    std::optional<Arriving> arriving;
    if (check) {
        hipStreamCaptureStatus capturing = hipStreamCaptureStatusNone;
        if (hipStreamIsCapturing(stream, &capturing) != hipSuccess || capturing != hipStreamCaptureStatusNone) return py::none();
        arriving.emplace(spreads, stream);
    }
    const bool recording = at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad() || spreads.requires_grad() || (legacy && betas.requires_grad()));
    Tensor O;
    bool good = true;
    try {
        py::gil_scoped_release no_gil;
        const std::optional<Tensor> b = legacy ? std::optional<Tensor>(betas) : std::nullopt, m = mask.defined() ? std::optional<Tensor>(mask) : std::nullopt;
        if (recording) O = Attention::apply(q, k, v, coords, spreads, b, m, legacy, f16, min_rbf, max_rbf, token_major);
        else {
            at::NoGradGuard no_grad;
            O = attention_forward(q, k, v, coords, spreads, betas, mask, Logits{legacy, f16, min_rbf, max_rbf}, token_major).first;
        }
        if (arriving) good = arriving->positive();
    } catch (const Refused&) {
        return py::none();
    }
    return good ? py::cast(O) : py::none();                   // (what is wrong with the spreads is said by the general path)
}

// ---- wavefunction embedding ----

PyObject* g_embedding_backward = nullptr;
PyObject* g_aniso_backward = nullptr;

// A gradient, and what the forward kept for it, that the kernels may read.
bool backward_ok(const Tensor& dO, const variable_list& kept, const int64_t per_gradient)
{
    if (!unobserved() || !dO.defined() || !plain(dO) || !f32(dO) || dO.dim() != 3 || off(dO, 8) || !current(dO.get_device())) return false;
    for (const Tensor& t : kept)
        if (t.defined() && !(plain(t) && f32(t) && t.get_device() == dO.get_device() && t.numel() * per_gradient == dO.numel() && !off(t, 8))) return false;
    return true;
}

Tensor bwd_workspace(const Tensor& dO, const int64_t K)
{
    return at::empty({static_cast<int64_t>(proteus_we_bwd_workspace_bytes(dO.size(0), dO.size(1), K))}, on(dO, at::kByte));
}

std::array<Tensor, 3> embedding_forward(const Tensor& coords, const Tensor& wn, const Tensor& mask, const bool sums)
{
    const int64_t Z = coords.size(0), N = coords.size(1), K = wn.size(0);
    const auto opt = on(coords, at::kFloat);
    const Tensor out = at::empty({Z, N, 2 * K}, opt);
    const Tensor cs = sums ? at::empty({Z, N, K}, opt) : Tensor(), sn = sums ? at::empty({Z, N, K}, opt) : Tensor();
    const size_t need = proteus_we_fwd_workspace_bytes(Z, N, K, 0);
    Tensor ws;
    if (need) ws = at::empty({static_cast<int64_t>(need)}, on(coords, at::kByte));
    launched(proteus_we_fwd_ws(floats(coords), PROTEUS_COORDS_AOS, floats(wn), bytes(mask), out_floats(out), sums ? out_floats(cs) : nullptr, sums ? out_floats(sn) : nullptr,
                               need ? ws.mutable_data_ptr() : nullptr, need, Z, N, K, 0, stream_of(coords.get_device())));
    return {out, cs, sn};
}

struct Embedding : torch::autograd::Function<Embedding> {
    static Tensor forward(AutogradContext* ctx, const Tensor& coords, const Tensor& wn, const std::optional<Tensor>& mask)
    {
        const auto [out, cs, sn] = embedding_forward(coords, wn, mask.value_or(Tensor()), true);
        ctx->save_for_backward({cs, sn});
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        const variable_list s = ctx->get_saved_variables();
        const Tensor& dO = grads[0];
        if (backward_ok(dO, s, 2)) try {
            return {Tensor(), reduced(dO, s), Tensor()};
        } catch (const Refused&) {}
        py::gil_scoped_acquire gil;
        return {Tensor(), py::reinterpret_borrow<py::object>(g_embedding_backward)(dO, s[0], s[1]).cast<Tensor>(), Tensor()};
    }
    static Tensor reduced(const Tensor& dO, const variable_list& s)
    {
        const int64_t K = dO.size(2) / 2;
        const Tensor ws = bwd_workspace(dO, K), dk = at::empty({K}, on(dO, at::kFloat));
        launched(proteus_we_bwd(floats(dO), floats(s[0]), floats(s[1]), out_floats(dk), out_floats(ws), ws.numel(), dO.size(0), dO.size(1), K, stream_of(dO.get_device())));
        return dk;
    }
};

std::array<Tensor, 3> aniso_forward(const Tensor& a, const Tensor& b, const Tensor& cb, const Tensor& wn, const Tensor& mask, const bool partials)
{
    const int64_t Z = a.size(0), N = a.size(1), K = wn.size(0);
    const auto opt = on(a, at::kFloat);
    const Tensor out = at::empty({Z, N, 2 * K}, opt);
    const Tensor d_cb = partials ? at::empty({Z, N, 2 * K}, opt) : Tensor(), d_k = partials ? at::empty({Z, N, 2 * K}, opt) : Tensor();
    const size_t need = proteus_we_aniso_fwd_workspace_bytes(Z, N, K, partials, mask.defined(), 0);
    Tensor ws;
    if (need) ws = at::empty({static_cast<int64_t>(need)}, on(a, at::kByte));
    launched(proteus_we_aniso_fwd_ws(floats(a), floats(b), PROTEUS_COORDS_AOS, floats(cb), floats(wn), bytes(mask), out_floats(out), partials ? out_floats(d_cb) : nullptr,
                                     partials ? out_floats(d_k) : nullptr, need ? ws.mutable_data_ptr() : nullptr, need, Z, N, K, 0, stream_of(a.get_device())));
    return {out, d_cb, d_k};
}

struct Aniso : torch::autograd::Function<Aniso> {
    static Tensor forward(AutogradContext* ctx, const Tensor& a, const Tensor& b, const Tensor& cb, const Tensor& wn, const std::optional<Tensor>& mask)
    {
        const auto [out, d_cb, d_k] = aniso_forward(a, b, cb, wn, mask.value_or(Tensor()), true);
        ctx->save_for_backward({d_cb, d_k});
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        variable_list s = ctx->get_saved_variables();
        const Tensor& dO = grads[0];
        for (int i = 0; i < 2; ++i) if (!ctx->needs_input_grad(2 + i)) s[i] = Tensor();
        if (!s[0].defined() && !s[1].defined()) return {Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
        if (backward_ok(dO, s, 1)) try {
            return reduced(dO, s);
        } catch (const Refused&) {}
        py::gil_scoped_acquire gil;
        auto opt = [](const Tensor& t) -> py::object { return t.defined() ? py::cast(t) : py::none(); };
        const py::tuple got = py::reinterpret_borrow<py::object>(g_aniso_backward)(dO, opt(s[0]), opt(s[1]));
        auto back = [&](const int i) { const py::object o = got[i]; return o.is_none() ? Tensor() : o.cast<Tensor>(); };
        return {Tensor(), Tensor(), back(0), back(1), Tensor()};
    }
    static variable_list reduced(const Tensor& dO, const variable_list& s)
    {
        const int64_t K = dO.size(2) / 2;
        const Tensor ws = bwd_workspace(dO, K);
        Tensor g[2];
        for (int i = 0; i < 2; ++i) if (s[i].defined()) g[i] = at::empty({K}, on(dO, at::kFloat));
        launched(proteus_we_aniso_bwd(floats(dO), s[0].defined() ? floats(s[0]) : nullptr, s[1].defined() ? floats(s[1]) : nullptr, g[0].defined() ? out_floats(g[0]) : nullptr,
                                      g[1].defined() ? out_floats(g[1]) : nullptr, out_floats(ws), ws.numel(), dO.size(0), dO.size(1), K, stream_of(dO.get_device())));
        return {Tensor(), Tensor(), g[0], g[1], Tensor()};
    }
};

bool sizes_ok(const Tensor& coords, const Tensor& wn)
{
    return f32(coords) && coords.dim() == 3 && coords.size(2) == 3 && f32(wn) && wn.dim() == 1 && coords.size(0) > 0 && coords.size(0) <= 65535 && coords.size(1) > 0
           && coords.size(1) <= PROTEUS_WE_MAX_N && wn.size(0) > 0 && wn.size(0) <= PROTEUS_WE_MAX_K;
}

// wf_embedding(coords, wavenumbers, mask=mask), or None.
py::object embedding(const py::object& coords_, const py::object& wn_, const py::object& mask_)
{
    Tensor coords, wn, mask;
    if (!unobserved() || !get(coords_, coords) || !current(coords.get_device()) || !get(wn_, wn, coords.get_device()) || !sizes_ok(coords, wn)
        || !get_mask(mask_, mask, coords.get_device(), coords.size(0), coords.size(1)) || coords.requires_grad()) return py::none();
    Tensor out;
    try {
        py::gil_scoped_release no_gil;
        if (at::GradMode::is_enabled() && wn.requires_grad()) out = Embedding::apply(coords, wn, mask.defined() ? std::optional<Tensor>(mask) : std::nullopt);
        else { at::NoGradGuard no_grad; out = embedding_forward(coords, wn, mask, false)[0]; }
    } catch (const Refused&) {
        return py::none();
    }
    return py::cast(out);
}

// wf_embedding_learnCB(a, b, cb, wavenumbers, mask), or None.
py::object aniso(const py::object& a_, const py::object& b_, const py::object& cb_, const py::object& wn_, const py::object& mask_)
{
    Tensor a, b, cb, wn, mask;
    if (!unobserved() || !get(a_, a) || !current(a.get_device())) return py::none();
    const int dev = a.get_device();
    if (!get(b_, b, dev) || !get(cb_, cb, dev) || !get(wn_, wn, dev) || !sizes_ok(a, wn) || !f32(b) || b.sizes() != a.sizes() || !f32(cb) || cb.sizes() != wn.sizes()
        || !get_mask(mask_, mask, dev, a.size(0), a.size(1)) || a.requires_grad() || b.requires_grad()) return py::none();
    Tensor out;
    try {
        py::gil_scoped_release no_gil;
        if (at::GradMode::is_enabled() && (cb.requires_grad() || wn.requires_grad())) out = Aniso::apply(a, b, cb, wn, mask.defined() ? std::optional<Tensor>(mask) : std::nullopt);
        else { at::NoGradGuard no_grad; out = aniso_forward(a, b, cb, wn, mask, false)[0]; }
    } catch (const Refused&) {
        return py::none();
    }
    return py::cast(out);
}

// ---- norm and rotation of queries and keys ----

PyObject* g_qk_backward = nullptr;

int dtype_of(const at::ScalarType t) { return t == at::kFloat ? PROTEUS_DTYPE_F32 : t == at::kBFloat16 ? PROTEUS_DTYPE_BF16 : t == at::kHalf ? PROTEUS_DTYPE_F16 : -1; }

// Queries, keys or values of every head, [Z,heads,N,d], as they lie in a tensor (without making a view of it: 1 us each).
struct Heads {
    char* data;
    int64_t Z, heads, N, d, stride[3], last;
    int64_t item;
    Heads(const Tensor& t) : Heads(t, t.size(0), t.size(1), t.size(2), t.size(3), t.stride(0), t.stride(1), t.stride(2), t.stride(3), 0) {}
    // part i of a fused projection [Z,N,3,heads,d]
    Heads(const Tensor& t, const int i) : Heads(t, t.size(0), t.size(3), t.size(1), t.size(4), t.stride(0), t.stride(3), t.stride(1), t.stride(4), i * t.stride(2)) {}
    // Can the kernel read or write it in place?
    bool ok() const
    {
        if (reinterpret_cast<uintptr_t>(data) % 16 || last != 1) return false;
        for (const int64_t s : stride) if (s * item % 16) return false;
        return true;
    }
private:
    Heads(const Tensor& t, int64_t Z_, int64_t heads_, int64_t N_, int64_t d_, int64_t sz, int64_t sh, int64_t sn, int64_t sd, int64_t first)
        : data(static_cast<char*>(const_cast<void*>(t.const_data_ptr())) + first * t.element_size()), Z(Z_), heads(heads_), N(N_), d(d_),
          stride{Z_ > 1 ? sz : 0, heads_ > 1 ? sh : 0, N_ > 1 ? sn : 0}, last(sd), item(t.element_size()) {}
};
using HeadList = std::vector<Heads>;

// How the operator is called, beside its tensors.
struct Rotation {
    double base, eps;
    bool interleaved;
    at::ScalarType out;
};

HeadList heads_of(const Tensor& qkv) { return {Heads(qkv, 0), Heads(qkv, 1), Heads(qkv, 2)}; }

proteus_qk_args qk_args(const HeadList& x, const at::ScalarType type, const HeadList& dy, const HeadList& y, const Tensor& qw, const Tensor& kw, const Tensor& positions, const Tensor& mask,
                        const Rotation& how)
{
    proteus_qk_args a = {};
    for (size_t i = 0; i < x.size(); ++i) {
        a.x[i] = x[i].data;
        a.y[i] = y[i].data;
        std::copy(x[i].stride, x[i].stride + 3, a.x_strides[i]);
        std::copy(y[i].stride, y[i].stride + 3, a.y_strides[i]);
        if (!dy.empty()) { a.dy[i] = dy[i].data; std::copy(dy[i].stride, dy[i].stride + 3, a.dy_strides[i]); }
    }
    const Heads& q = x[0];
    const Tensor& w = qw.defined() ? qw : kw;
    a.weight[0] = qw.defined() ? qw.const_data_ptr() : nullptr;
    a.weight[1] = kw.defined() ? kw.const_data_ptr() : nullptr;
    a.positions = positions.defined() ? static_cast<const int64_t*>(positions.const_data_ptr()) : nullptr;
    a.positions_stride = positions.defined() && positions.dim() == 2 && positions.size(0) > 1 ? positions.stride(0) : 0;
    a.mask = bytes(mask);
    a.base = how.base; a.eps = static_cast<float>(how.eps);
    a.Z = q.Z; a.N = q.N; a.heads_q = q.heads; a.heads_k = x[1].heads; a.heads_v = x.size() > 2 ? x[2].heads : 0; a.d_head = q.d;
    a.x_type = dtype_of(type); a.y_type = dtype_of(how.out);
    a.weight_type = w.defined() ? dtype_of(w.scalar_type()) : PROTEUS_DTYPE_F32;
    a.per_head = w.defined() && w.dim() == 2;
    a.interleaved = how.interleaved;
    return a;
}

// Tensors in the memory order of t (dense).
Tensor heads_like(const Tensor& t, const at::ScalarType type)
{
    const Tensor y = at::empty_like(t, on(t, type));
    return Heads(y).ok() && y.is_non_overlapping_and_dense() ? y : at::empty(t.sizes(), on(t, type));
}

void qk_forward(const Tensor& in, const HeadList& x, const HeadList& y, const Tensor& qw, const Tensor& kw, const Tensor& positions, const Tensor& mask, const Rotation& how)
{
    const proteus_qk_args a = qk_args(x, in.scalar_type(), {}, y, qw, kw, positions, mask, how);
    launched(proteus_qk_norm_rotate_fwd(&a, stream_of(in.get_device())));
}
variable_list qk_separate(const Tensor& q, const Tensor& k, const Tensor& qw, const Tensor& kw, const Tensor& positions, const Tensor& mask, const Rotation& how)
{
    const Tensor y = heads_like(q, how.out), z = heads_like(k, how.out);
    qk_forward(q, {Heads(q), Heads(k)}, {Heads(y), Heads(z)}, qw, kw, positions, mask, how);
    return {y, z};
}
Tensor qk_fused(const Tensor& qkv, const Tensor& qw, const Tensor& kw, const Tensor& positions, const Tensor& mask, const Rotation& how)
{
    const Tensor y = at::empty(qkv.sizes(), on(qkv, how.out));
    qk_forward(qkv, heads_of(qkv), heads_of(y), qw, kw, positions, mask, how);
    return y;
}

// What the kernel takes of tensors of the operator's shapes (which the caller has looked at).
bool qk_ok(const HeadList& x, const at::ScalarType type, const Tensor& qw, const Tensor& kw, const Tensor& positions, const Tensor& mask, const Rotation& how)
{
    const int64_t Z = x[0].Z, N = x[0].N, d = x[0].d;
    if (dtype_of(type) < 0 || (how.out != type && !(type == at::kFloat && dtype_of(how.out) >= 0)) || Z <= 0 || N <= 0 || (d != 32 && d != 64 && d != 128)) return false;
    for (const Heads& t : x) if (t.Z != Z || t.N != N || t.d != d || t.heads <= 0 || !t.ok()) return false;
    for (int i = 0; i < 2; ++i) {
        const Tensor& w = i ? kw : qw;
        if (!w.defined()) continue;
        if (dtype_of(w.scalar_type()) < 0 || !w.is_contiguous() || !((w.dim() == 1 && w.size(0) == d) || (w.dim() == 2 && w.size(0) == x[i].heads && w.size(1) == d))) return false;
    }
    if (qw.defined() && kw.defined() && (qw.dim() != kw.dim() || qw.scalar_type() != kw.scalar_type())) return false;
    if (positions.defined() && !(positions.scalar_type() == at::kLong && ((positions.dim() == 1 && positions.size(0) == N) || (positions.dim() == 2 && positions.size(0) == Z && positions.size(1) == N))
                                 && (N == 1 || positions.stride(-1) == 1))) return false;
    return !mask.defined() || (mask.scalar_type() == at::kBool && mask.is_contiguous() && mask.dim() == 2 && mask.size(0) == Z && mask.size(1) == N);
}

std::optional<Tensor> maybe(const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }

// Gradients of (q, k) or (qkv), and of the two weights, from those of the results; None where the general way has to be gone.
variable_list qk_backward(const variable_list& saved, const variable_list& grads, const Rotation& how, const bool fused, const bool dqw, const bool dkw)
{
    const Tensor &qw = saved[2], &kw = saved[3], &positions = saved[4], &mask = saved[5];
    auto general = [&]() -> variable_list {
        py::gil_scoped_acquire gil;
        auto opt = [](const Tensor& t) -> py::object { return t.defined() ? py::cast(t) : py::none(); };
        py::list outs;
        for (const Tensor& g : grads) outs.append(opt(g));
        const py::object got = py::reinterpret_borrow<py::object>(g_qk_backward)(opt(saved[0]), opt(saved[1]), opt(qw), opt(kw), opt(positions), opt(mask), outs, how.base, how.eps, how.interleaved,
                                                                               static_cast<int>(dtype_of(how.out)), fused);
        variable_list out;
        for (const auto& o : py::reinterpret_borrow<py::tuple>(got)) out.push_back(o.is_none() ? Tensor() : o.cast<Tensor>());
        return out;
    };
    if (at::GradMode::is_enabled() || !unobserved()) return general();
    for (const Tensor* t : {&saved[0], &saved[1], &qw, &kw, &positions, &mask}) if (t->defined() && (!plain(*t) || t->get_device() != saved[0].get_device())) return general();
    const int dev = saved[0].get_device();
    if (!current(dev)) return general();
    if (fused ? saved[0].dim() != 5 || saved[0].size(2) != 3 : saved[0].dim() != 4 || saved[1].dim() != 4) return general();
    const auto type = saved[0].scalar_type();
    const HeadList x = fused ? heads_of(saved[0]) : HeadList{Heads(saved[0]), Heads(saved[1])};
    if (!qk_ok(x, type, qw, kw, positions, mask, how) || (!fused && saved[1].scalar_type() != type)) return general();
    HeadList dy;
    variable_list held;                              // (copies of gradients that lie otherwise)
    for (size_t i = 0; i < grads.size(); ++i) {
        const Tensor& g = grads[i];
        if (!g.defined() || !plain(g) || g.get_device() != dev || g.scalar_type() != how.out || g.sizes() != saved[i].sizes()) return general();
        HeadList parts = fused ? heads_of(g) : HeadList{Heads(g)};
        bool ok = true;
        for (const Heads& h : parts) ok = ok && h.ok();
        if (!ok) {
            held.push_back(g.clone(at::MemoryFormat::Contiguous));
            parts = fused ? heads_of(held.back()) : HeadList{Heads(held.back())};
        }
        dy.insert(dy.end(), parts.begin(), parts.end());
    }
    variable_list out;
    if (fused) out = {at::empty(saved[0].sizes(), on(saved[0], type))};
    else out = {heads_like(saved[0], type), heads_like(saved[1], type)};
    const HeadList dx = fused ? heads_of(out[0]) : HeadList{Heads(out[0]), Heads(out[1])};
    const Tensor gq = dqw ? at::empty_like(qw) : Tensor(), gk = dkw ? at::empty_like(kw) : Tensor();
    const proteus_qk_args a = qk_args(x, type, dy, dx, qw, kw, positions, mask, how);
    Tensor ws;
    if (gq.defined() || gk.defined())
        ws = at::empty({static_cast<int64_t>(proteus_qk_norm_rotate_bwd_workspace_bytes(a.Z, a.N, a.heads_q, a.heads_k, a.heads_v, a.d_head, a.per_head))}, on(saved[0], at::kByte));
    const int rc = proteus_qk_norm_rotate_bwd(&a, gq.defined() ? gq.mutable_data_ptr() : nullptr, gk.defined() ? gk.mutable_data_ptr() : nullptr, ws.defined() ? ws.mutable_data_ptr() : nullptr,
                                              ws.defined() ? ws.numel() : 0, stream_of(dev));
    if (rc != 0) return general();
    if (!fused) return {out[0], out[1], gq, gk};
    return {out[0], gq, gk};
}

void save_rotation(AutogradContext* ctx, const Rotation& how)
{
    ctx->saved_data["base"] = how.base; ctx->saved_data["eps"] = how.eps; ctx->saved_data["inter"] = how.interleaved; ctx->saved_data["out"] = static_cast<int64_t>(how.out);
}
Rotation saved_rotation(AutogradContext* ctx)
{
    return {ctx->saved_data["base"].toDouble(), ctx->saved_data["eps"].toDouble(), ctx->saved_data["inter"].toBool(), static_cast<at::ScalarType>(ctx->saved_data["out"].toInt())};
}

// Is a gradient asked of weight `i` (2: the queries', 3: the keys') among the saved tensors?  (Inputs that were left out are not counted: the weights that are
// there follow `first` others.)
bool wanted(AutogradContext* ctx, const variable_list& saved, const int i, const int first)
{
    return saved[i].defined() && ctx->needs_input_grad(first + (i == 3 && saved[2].defined()));
}

struct QkRotate : torch::autograd::Function<QkRotate> {
    static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const std::optional<Tensor>& qw, const std::optional<Tensor>& kw, const std::optional<Tensor>& positions, const std::optional<Tensor>& mask,
                                 double base, double eps, bool interleaved, int64_t out)
    {
        const Tensor a = qw.value_or(Tensor()), b = kw.value_or(Tensor()), p = positions.value_or(Tensor()), m = mask.value_or(Tensor());
        const Rotation how{base, eps, interleaved, static_cast<at::ScalarType>(out)};
        ctx->save_for_backward({q, k, a, b, p, m});
        save_rotation(ctx, how);
        return qk_separate(q, k, a, b, p, m, how);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        const variable_list s = ctx->get_saved_variables();
        const variable_list g = qk_backward(s, grads, saved_rotation(ctx), false, wanted(ctx, s, 2, 2), wanted(ctx, s, 3, 2));
        return {g[0], g[1], g[2], g[3], Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

struct QkvRotate : torch::autograd::Function<QkvRotate> {
    static Tensor forward(AutogradContext* ctx, const Tensor& qkv, const std::optional<Tensor>& qw, const std::optional<Tensor>& kw, const std::optional<Tensor>& positions, const std::optional<Tensor>& mask,
                          double base, double eps, bool interleaved, int64_t out)
    {
        const Tensor a = qw.value_or(Tensor()), b = kw.value_or(Tensor()), p = positions.value_or(Tensor()), m = mask.value_or(Tensor());
        const Rotation how{base, eps, interleaved, static_cast<at::ScalarType>(out)};
        ctx->save_for_backward({qkv, Tensor(), a, b, p, m});
        save_rotation(ctx, how);
        return qk_fused(qkv, a, b, p, m, how);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        const variable_list s = ctx->get_saved_variables();
        const variable_list g = qk_backward(s, grads, saved_rotation(ctx), true, wanted(ctx, s, 2, 1), wanted(ctx, s, 3, 1));
        return {g[0], g[1], g[2], Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

// qk_norm_rotate (k a tensor: the two results) or qk_norm_rotate_qkv (k None: q is the fused projection), or None.
py::object qk_norm_rotate(const py::object& q_, const py::object& k_, const py::object& qw_, const py::object& kw_, const py::object& positions_, const py::object& mask_,
                          const double base, const double eps, const bool interleaved, const int out_type)
{
    Tensor q, k, qw, kw, positions, mask;
    const bool fused = k_.is_none();
    if (!unobserved() || !get(q_, q) || !current(q.get_device())) return py::none();
    const int dev = q.get_device();
    if ((!fused && !get(k_, k, dev)) || (!qw_.is_none() && !get(qw_, qw, dev)) || (!kw_.is_none() && !get(kw_, kw, dev)) || (!positions_.is_none() && !get(positions_, positions, dev))
        || (!mask_.is_none() && !get(mask_, mask, dev))) return py::none();
    const auto out = out_type < 0 ? q.scalar_type() : out_type == PROTEUS_DTYPE_F32 ? at::kFloat : out_type == PROTEUS_DTYPE_BF16 ? at::kBFloat16 : at::kHalf;
    const Rotation how{base, eps, interleaved, out};
    if (q.dim() != (fused ? 5 : 4) || (fused && q.size(2) != 3)) return py::none();
    if (!fused && (k.dim() != 4 || k.scalar_type() != q.scalar_type())) return py::none();
    if (!qk_ok(fused ? heads_of(q) : HeadList{Heads(q), Heads(k)}, q.scalar_type(), qw, kw, positions, mask, how)) return py::none();
    const bool recording = at::GradMode::is_enabled() && (q.requires_grad() || (!fused && k.requires_grad()) || (qw.defined() && qw.requires_grad()) || (kw.defined() && kw.requires_grad()));
    variable_list y;
    try {
        py::gil_scoped_release no_gil;
        if (recording) {
            if (fused) y = {QkvRotate::apply(q, maybe(qw), maybe(kw), maybe(positions), maybe(mask), base, eps, interleaved, static_cast<int64_t>(out))};
            else y = QkRotate::apply(q, k, maybe(qw), maybe(kw), maybe(positions), maybe(mask), base, eps, interleaved, static_cast<int64_t>(out));
        } else {
            at::NoGradGuard no_grad;
            y = fused ? variable_list{qk_fused(q, qw, kw, positions, mask, how)} : qk_separate(q, k, qw, kw, positions, mask, how);
        }
    } catch (const Refused&) {
        return py::none();
    }
    if (fused) return py::cast(y[0]);
    return py::make_tuple(y[0], y[1]);
}

// ---- gated feed-forward block ----

PyObject* g_gated_backward = nullptr;

struct Block {
    long rows;
    int d_in, hidden, d_out, type;
};

// Dense on 16 bytes, of one type on one GPU (undefined: left out)
bool block_tensor(const Tensor& t, const at::ScalarType type, const int dev)
{
    return !t.defined() || (plain(t) && t.scalar_type() == type && t.get_device() == dev && t.is_contiguous() && !off(t, 16));
}

const void* address(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
Tensor bytes_like(const Tensor& t, const size_t n) { return n ? at::empty({static_cast<int64_t>(n)}, on(t, at::kByte)) : Tensor(); }
void* memory(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }

// y, and (keep) what the backward reads
std::pair<Tensor, Tensor> block_forward(const Tensor& x, const variable_list& p, const Block& b, const int act, const bool keep)
{
    std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
    shape.back() = b.d_out;
    const Tensor y = at::empty(shape, on(x, x.scalar_type()));
    const size_t kept_bytes = keep ? proteus_gated_mlp_kept_bytes(b.rows, b.d_in, b.hidden, b.d_out, b.type) : 0;
    const size_t ws_bytes = keep ? proteus_gated_mlp_train_fwd_bytes(b.rows, b.d_in, b.hidden, b.d_out, b.type) : proteus_gated_mlp_fwd_bytes(b.rows, b.d_in, b.hidden, b.d_out, b.type);
    const Tensor kept = bytes_like(x, kept_bytes), ws = bytes_like(x, ws_bytes);
    const void* const params[4] = {address(p[0]), address(p[1]), address(p[2]), address(p[3])};
    launched(proteus_gated_mlp_fwd(x.const_data_ptr(), params, y.mutable_data_ptr(), memory(kept), kept_bytes, memory(ws), ws_bytes, b.rows, b.d_in, b.hidden, b.d_out, act, b.type,
                                   stream_of(x.get_device())));
    return {y, kept};
}

// Gradients of x, W, b, Wo, bo
variable_list block_backward(const variable_list& s, const Tensor& dy_, const int act, const std::array<bool, 5>& need)
{
    const Tensor &x = s[0], &w = s[1], &wo = s[3], &kept = s[5];
    auto general = [&]() -> variable_list {
        py::gil_scoped_acquire gil;
        auto opt = [](const Tensor& t) -> py::object { return t.defined() ? py::cast(t) : py::none(); };
        py::list saved, needs;
        for (const Tensor& t : s) saved.append(opt(t));
        for (const bool n : need) needs.append(n);
        const py::object got = py::reinterpret_borrow<py::object>(g_gated_backward)(saved, opt(dy_), act, needs);
        variable_list out;
        for (const auto& o : py::reinterpret_borrow<py::tuple>(got)) out.push_back(o.is_none() ? Tensor() : o.cast<Tensor>());
        return out;
    };
    if (at::GradMode::is_enabled() || !unobserved() || !dy_.defined() || !plain(dy_)) return general();
    const int dev = dy_.get_device();
    const auto type = dy_.scalar_type();
    bool ok = current(dev) && x.defined() && w.defined() && wo.defined() && kept.defined();
    for (int i = 0; i < 5; ++i) ok = ok && block_tensor(s[i], type, dev);
    ok = ok && block_tensor(kept, at::kByte, dev) && !off(kept, 256) && w.dim() == 2 && wo.dim() == 2 && x.dim() >= 1;
    if (!ok) return general();
    const Block b = {static_cast<long>(x.size(-1) ? x.numel() / x.size(-1) : 0), static_cast<int>(w.size(1)), static_cast<int>(wo.size(1)), static_cast<int>(wo.size(0)), dtype_of(type)};
    if (w.size(0) != 2 * b.hidden || x.size(-1) != b.d_in || dy_.numel() != b.rows * b.d_out || (s[2].defined() && s[2].numel() != 2 * b.hidden) || (s[4].defined() && s[4].numel() != b.d_out)
        || static_cast<size_t>(kept.numel()) != proteus_gated_mlp_kept_bytes(b.rows, b.d_in, b.hidden, b.d_out, b.type)) return general();
    Tensor dy = dy_.is_contiguous() ? dy_ : dy_.contiguous();
    if (off(dy, 16)) dy = dy.clone();
    const Tensor dx = need[0] ? at::empty(x.sizes(), on(x, type)) : Tensor();
    variable_list grads(4);
    for (int i = 0; i < 4; ++i) if (need[1 + i] && s[1 + i].defined()) grads[i] = at::empty(s[1 + i].sizes(), on(x, type));
    const size_t n = proteus_gated_mlp_bwd_bytes(b.rows, b.d_in, b.hidden, b.d_out, b.type);
    const Tensor ws = bytes_like(x, n);
    const void* const params[4] = {address(w), address(s[2]), address(wo), address(s[4])};
    void* const to[4] = {memory(grads[0]), memory(grads[1]), memory(grads[2]), memory(grads[3])};
    if (proteus_gated_mlp_bwd(x.const_data_ptr(), params, dy.const_data_ptr(), memory(dx), to, kept.const_data_ptr(), kept.numel(), memory(ws), n, b.rows, b.d_in, b.hidden, b.d_out, act, b.type,
                              stream_of(dev)) != 0) return general();
    return {dx, grads[0], grads[1], grads[2], grads[3]};
}

struct GatedBlock : torch::autograd::Function<GatedBlock> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Tensor& wo, const std::optional<Tensor>& b, const std::optional<Tensor>& bo, int64_t rows, int64_t act)
    {
        const variable_list p = {w, b.value_or(Tensor()), wo, bo.value_or(Tensor())};
        const Block how = {static_cast<long>(rows), static_cast<int>(w.size(1)), static_cast<int>(wo.size(1)), static_cast<int>(wo.size(0)), dtype_of(x.scalar_type())};
        const auto [y, kept] = block_forward(x, p, how, static_cast<int>(act), true);
        ctx->save_for_backward({x, w, p[1], wo, p[3], kept});
        ctx->saved_data["act"] = act;
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        const variable_list s = ctx->get_saved_variables();
        // (inputs that were left out are not counted: x, W, Wo, then the biases that are there)
        const bool b = s[2].defined(), bo = s[4].defined();
        const variable_list g = block_backward(s, grads[0], static_cast<int>(ctx->saved_data["act"].toInt()),
                                               {ctx->needs_input_grad(0), ctx->needs_input_grad(1), b && ctx->needs_input_grad(3), ctx->needs_input_grad(2), bo && ctx->needs_input_grad(3 + b)});
        return {g[0], g[1], g[3], g[2], g[4], Tensor(), Tensor()};
    }
};

// gated_mlp(x, W, b, Wo, bo) with the activation's number, or None.
py::object gated_mlp(const py::object& x_, const py::object& w_, const py::object& b_, const py::object& wo_, const py::object& bo_, const int act)
{
    Tensor x, w, b, wo, bo;
    if (!unobserved() || at::autocast::is_autocast_enabled(at::kCUDA) || !get(x_, x) || !current(x.get_device())) return py::none();
    const int dev = x.get_device();
    const auto type = x.scalar_type();
    if ((type != at::kFloat && type != at::kBFloat16) || x.dim() < 1 || !get(w_, w, dev) || !get(wo_, wo, dev) || (!b_.is_none() && !get(b_, b, dev)) || (!bo_.is_none() && !get(bo_, bo, dev)))
        return py::none();
    for (const Tensor* t : {&x, &w, &b, &wo, &bo}) if (!block_tensor(*t, type, dev)) return py::none();
    if (w.dim() != 2 || wo.dim() != 2 || w.size(0) != 2 * wo.size(1) || x.size(-1) != w.size(1) || x.numel() == 0 || (b.defined() && (b.dim() != 1 || b.size(0) != w.size(0)))
        || (bo.defined() && (bo.dim() != 1 || bo.size(0) != wo.size(0))) || w.numel() > INT_MAX || wo.numel() > INT_MAX) return py::none();
    const Block how = {static_cast<long>(x.numel() / x.size(-1)), static_cast<int>(w.size(1)), static_cast<int>(wo.size(1)), static_cast<int>(wo.size(0)), dtype_of(type)};
    if (!proteus_gated_mlp_kept_bytes(how.rows, how.d_in, how.hidden, how.d_out, how.type)) return py::none();
    bool recording = false;
    if (at::GradMode::is_enabled()) for (const Tensor* t : {&x, &w, &b, &wo, &bo}) recording = recording || (t->defined() && t->requires_grad());
    Tensor y;
    try {
        py::gil_scoped_release no_gil;
        if (recording) y = GatedBlock::apply(x, w, wo, maybe(b), maybe(bo), static_cast<int64_t>(how.rows), static_cast<int64_t>(act));
        else { at::NoGradGuard no_grad; y = block_forward(x, {w, b, wo, bo}, how, act, false).first; }
    } catch (const Refused&) {
        return py::none();
    }
    return py::cast(y);
}

// ---- softmax cross entropy from features ----

PyObject* g_ce_backward = nullptr;

struct CeHow { int64_t ignored; double smoothing; int64_t reduction; };

proteus_ce_args ce_args(const Tensor& x, const Tensor& w, const Tensor& b, const Tensor& target, const CeHow& how)
{
    proteus_ce_args a = {};
    a.x = x.const_data_ptr(); a.weight = w.const_data_ptr(); a.bias = address(b); a.target = static_cast<const int64_t*>(target.const_data_ptr());
    a.ignore_index = how.ignored; a.label_smoothing = static_cast<float>(how.smoothing); a.reduction = static_cast<int>(how.reduction);
    a.rows = static_cast<long>(target.numel()); a.d = static_cast<int>(w.size(1)); a.vocab = static_cast<int>(w.size(0)); a.dtype = dtype_of(x.scalar_type());
    return a;
}

// The loss, and (keep) what the backward reads
std::pair<Tensor, Tensor> ce_forward(const Tensor& x, const Tensor& w, const Tensor& b, const Tensor& target, const CeHow& how, const bool keep)
{
    const proteus_ce_args a = ce_args(x, w, b, target, how);
    const Tensor loss = how.reduction == PROTEUS_CE_NONE ? at::empty(target.sizes(), on(x, at::kFloat)) : at::empty({}, on(x, at::kFloat));
    const size_t kept_bytes = keep ? proteus_linear_ce_kept_bytes(&a) : 0, n = proteus_linear_ce_fwd_bytes(&a);
    const Tensor kept = bytes_like(x, kept_bytes), ws = bytes_like(x, n);
    launched(proteus_linear_ce_fwd(&a, static_cast<float*>(loss.mutable_data_ptr()), memory(kept), kept_bytes, memory(ws), n, stream_of(x.get_device())));
    return {loss, kept};
}

// Gradients of x, W, b
variable_list ce_backward(const variable_list& s, const Tensor& d_, const CeHow& how, const std::array<bool, 3>& need)
{
    const Tensor &x = s[0], &w = s[1], &b = s[2], &target = s[3], &kept = s[4];
    auto general = [&]() -> variable_list {
        py::gil_scoped_acquire gil;
        auto opt = [](const Tensor& t) -> py::object { return t.defined() ? py::cast(t) : py::none(); };
        py::list saved, needs;
        for (const Tensor& t : s) saved.append(opt(t));
        for (const bool n : need) needs.append(n);
        const py::object got = py::reinterpret_borrow<py::object>(g_ce_backward)(saved, opt(d_), how.ignored, how.smoothing, how.reduction, needs);
        variable_list out;
        for (const auto& o : py::reinterpret_borrow<py::tuple>(got)) out.push_back(o.is_none() ? Tensor() : o.cast<Tensor>());
        return out;
    };
    if (at::GradMode::is_enabled() || !unobserved() || !d_.defined() || !plain(d_) || !x.defined() || !w.defined() || !target.defined() || !kept.defined()) return general();
    const int dev = d_.get_device();
    const auto type = w.scalar_type();
    bool ok = current(dev) && d_.scalar_type() == at::kFloat && dtype_of(type) >= 0;
    for (int i = 0; i < 3; ++i) ok = ok && block_tensor(s[i], type, dev);
    ok = ok && block_tensor(target, at::kLong, dev) && block_tensor(kept, at::kByte, dev) && w.dim() == 2;
    if (!ok || x.numel() != target.numel() * w.size(1) || (b.defined() && b.numel() != w.size(0)) || d_.numel() != (how.reduction == PROTEUS_CE_NONE ? target.numel() : 1)) return general();
    const proteus_ce_args a = ce_args(x, w, b, target, how);
    if (static_cast<size_t>(kept.numel()) != proteus_linear_ce_kept_bytes(&a)) return general();
    const Tensor d = d_.is_contiguous() ? d_ : d_.contiguous();
    Tensor grads[3];
    for (int i = 0; i < 3; ++i) if (need[i] && s[i].defined()) grads[i] = at::empty(s[i].sizes(), on(x, type));
    const size_t n = proteus_linear_ce_bwd_bytes(&a);
    const Tensor ws = bytes_like(x, n);
    if (proteus_linear_ce_bwd(&a, floats(d), kept.const_data_ptr(), kept.numel(), memory(grads[0]), memory(grads[1]), memory(grads[2]), memory(ws), n, stream_of(dev)) != 0) return general();
    return {grads[0], grads[1], grads[2]};
}

struct LinearCe : torch::autograd::Function<LinearCe> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Tensor& target, const std::optional<Tensor>& b, int64_t ignored, double smoothing, int64_t reduction)
    {
        const Tensor bias = b.value_or(Tensor());
        const auto [loss, kept] = ce_forward(x, w, bias, target, {ignored, smoothing, reduction}, true);
        ctx->save_for_backward({x, w, bias, target, kept});
        ctx->saved_data["ignored"] = ignored;
        ctx->saved_data["smoothing"] = smoothing;
        ctx->saved_data["reduction"] = reduction;
        return loss;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        const variable_list s = ctx->get_saved_variables();
        // (inputs that were left out are not counted: x, W, target, then the bias if there is one)
        const variable_list g = ce_backward(s, grads[0], {ctx->saved_data["ignored"].toInt(), ctx->saved_data["smoothing"].toDouble(), ctx->saved_data["reduction"].toInt()},
                                            {ctx->needs_input_grad(0), ctx->needs_input_grad(1), s[2].defined() && ctx->needs_input_grad(3)});
        return {g[0], g[1], Tensor(), g[2], Tensor(), Tensor(), Tensor()};
    }
};

// linear_cross_entropy(x, W, b, target), or None.
py::object linear_ce(const py::object& x_, const py::object& w_, const py::object& b_, const py::object& target_, const int64_t ignored, const double smoothing, const int64_t reduction)
{
    Tensor x, w, b, target;
    if (!unobserved() || at::autocast::is_autocast_enabled(at::kCUDA) || !get(x_, x) || !current(x.get_device())) return py::none();
    const int dev = x.get_device();
    const auto type = x.scalar_type();
    if (dtype_of(type) < 0 || x.dim() < 1 || !get(w_, w, dev) || !get(target_, target, dev) || (!b_.is_none() && !get(b_, b, dev))) return py::none();
    for (const Tensor* t : {&x, &w, &b}) if (!block_tensor(*t, type, dev)) return py::none();
    if (!block_tensor(target, at::kLong, dev) || w.dim() != 2 || w.size(1) != x.size(-1) || x.numel() == 0 || target.sizes() != x.sizes().slice(0, x.dim() - 1)
        || (b.defined() && (b.dim() != 1 || b.size(0) != w.size(0))) || w.size(0) > INT_MAX || w.size(1) > INT_MAX) return py::none();
    const CeHow how = {ignored, smoothing, reduction};
    const proteus_ce_args a = ce_args(x, w, b, target, how);
    if (proteus_linear_ce_check(&a) != 0) return py::none();
    bool recording = false;
    if (at::GradMode::is_enabled()) for (const Tensor* t : {&x, &w, &b}) recording = recording || (t->defined() && t->requires_grad());
    Tensor loss;
    try {
        py::gil_scoped_release no_gil;
        if (recording) loss = LinearCe::apply(x, w, target, maybe(b), ignored, smoothing, reduction);
        else { at::NoGradGuard no_grad; loss = ce_forward(x, w, b, target, how, false).first; }
    } catch (const Refused&) {
        return py::none();
    }
    return py::cast(loss);
}

// ---- the norm of gradients, and clipping ----

// Do two of the tensors written share memory, or one of them with another tensor that is read?  Pairs (from[i], to[i]) may be one and the same.
bool entangled(const std::vector<std::pair<uintptr_t, uintptr_t>>& from, const std::vector<std::pair<uintptr_t, uintptr_t>>& to)
{
    // mostly: what is written lies in ascending order, and is what is read or all beyond it
    bool ascending = true, same = true;
    uintptr_t lo = UINTPTR_MAX, hi = 0;
    for (size_t i = 0; i < to.size(); ++i) {
        same = same && to[i] == from[i];
        if (to[i].first == to[i].second) continue;
        ascending = ascending && to[i].first >= hi;
        lo = std::min(lo, to[i].first);
        hi = std::max(hi, to[i].second);
    }
    if (ascending) {
        bool clear = same;
        if (!same) {
            clear = true;
            for (const auto& f : from) clear = clear && (f.first == f.second || f.second <= lo || f.first >= hi);
        }
        if (clear) return false;
    }
    struct Span { uintptr_t begin, end; size_t of; bool written; };
    std::vector<Span> spans;
    for (size_t i = 0; i < to.size(); ++i) {
        if (to[i].first == to[i].second) continue;
        spans.push_back({to[i].first, to[i].second, i, true});
        if (from[i] != to[i]) spans.push_back({from[i].first, from[i].second, i, false});
    }
    std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& b) { return a.begin < b.begin; });
    uintptr_t written = 0, read = 0;                         // the furthest ends so far
    for (const Span& s : spans) {
        if (s.begin < written || (s.written && s.begin < read)) return true;
        (s.written ? written : read) = std::max(s.written ? written : read, s.end);
    }
    return false;
}

// The norm of `tensors` (of_parameters: of their gradients, where they have one), which are scaled into `outs` (None: not at all; the list itself: in place) where
// their norm is beyond max_norm; or None.
py::object clip(const py::list& tensors, const bool of_parameters, const py::object& outs, const int norm_type, const double max_norm)
{
    if (!unobserved()) return py::none();
    const bool in_place = outs.ptr() == tensors.ptr(), scaled = !outs.is_none();
    if (scaled && !in_place && (!py::isinstance<py::list>(outs) || py::len(outs) != tensors.size())) return py::none();
    // (the tensors' references are the list's and the parameters' own, which outlive the call)
    const size_t most = tensors.size();
    std::vector<const Tensor*> to;
    std::vector<const void*> src;
    std::vector<void*> dst;
    std::vector<int64_t> numel;
    std::vector<int> st, dt;
    std::vector<std::pair<uintptr_t, uintptr_t>> read, written;
    src.reserve(most); numel.reserve(most); st.reserve(most);
    if (scaled) { to.reserve(most); dst.reserve(most); dt.reserve(most); read.reserve(most); written.reserve(most); }
    const bool recording = at::GradMode::is_enabled(), inference = c10::InferenceMode::is_enabled();
    int dev = -1;
    const Tensor* any = nullptr;
    for (size_t i = 0; i < most; ++i) {
        PyObject* const o = PyList_GET_ITEM(tensors.ptr(), static_cast<Py_ssize_t>(i));
        if (!THPVariable_CheckExact(o)) return py::none();
        const Tensor* t = &THPVariable_Unpack(o);
        if (of_parameters) {
            t = &t->grad();
            if (!t->defined()) continue;
        }
        const int type = dtype_of(t->scalar_type());
        if (!plain(*t) || (dev >= 0 && t->get_device() != dev) || type < 0 || !t->is_non_overlapping_and_dense()) return py::none();
        dev = t->get_device();
        any = t;
        const int64_t n = t->numel();
        src.push_back(t->const_data_ptr()); numel.push_back(n); st.push_back(type);
        if (!scaled) continue;
        const Tensor* u = t;
        if (!in_place) {
            PyObject* const other = PyList_GET_ITEM(outs.ptr(), static_cast<Py_ssize_t>(i));
            if (!THPVariable_CheckExact(other)) return py::none();
            u = &THPVariable_Unpack(other);
            if (!plain(*u) || u->get_device() != dev || dtype_of(u->scalar_type()) < 0 || u->sizes() != t->sizes() || u->strides() != t->strides()) return py::none();
        }
        // (the Python function writes a tensor that is recorded without recording that, and refuses one made in inference mode outside of it)
        if ((recording && u->requires_grad()) || (u->is_inference() && !inference)) return py::none();
        to.push_back(u);
        dst.push_back(u->mutable_data_ptr()); dt.push_back(dtype_of(u->scalar_type()));
        const uintptr_t r = reinterpret_cast<uintptr_t>(src.back()), w = reinterpret_cast<uintptr_t>(dst.back());
        read.emplace_back(r, r + n * (type == PROTEUS_DTYPE_F32 ? 4 : 2));
        written.emplace_back(w, w + n * (dt.back() == PROTEUS_DTYPE_F32 ? 4 : 2));
    }
    if (src.empty() || !current(dev) || (scaled && entangled(read, written))) return py::none();
    const int n = static_cast<int>(src.size());
    const Tensor norm = at::empty({}, on(*any, at::kFloat));
    const Tensor ws = at::empty({static_cast<int64_t>(proteus_clip_grads_workspace_bytes(n))}, on(*any, at::kByte));
    if (proteus_clip_grads(src.data(), scaled ? dst.data() : nullptr, numel.data(), st.data(), scaled ? dt.data() : nullptr, n, norm_type, static_cast<float>(max_norm),
                           static_cast<float*>(norm.mutable_data_ptr()), ws.mutable_data_ptr(), ws.numel(), stream_of(dev)) != 0) return py::none();
    for (const Tensor* t : to) if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
    return py::cast(norm);
}

// ---- AdamW ----

// Does memory that is written overlap any other?  Spans of several lists: mostly each lies in ascending order, and then often in a stretch of its own; else merging them does (500 tensors in five lists merged 16 us).
struct Spans {
    struct Span { uintptr_t begin, end; };
    struct List { std::vector<Span> all; bool written, ascending = true, apart = true; uintptr_t end = 0; size_t at = 0; };      // apart: from one another
    std::vector<List> lists;
    int list(const bool written, const size_t most)
    {
        lists.emplace_back();
        lists.back().written = written;
        lists.back().all.reserve(most);
        return static_cast<int>(lists.size()) - 1;
    }
    void add(const int i, const void* p, const size_t n)
    {
        if (!n) return;
        const uintptr_t b = reinterpret_cast<uintptr_t>(p);
        List& l = lists[i];
        l.ascending = l.ascending && (l.all.empty() || l.all.back().begin <= b);
        l.apart = l.apart && b >= l.end;
        l.end = std::max(l.end, b + n);
        l.all.push_back({b, b + n});
    }
    bool overlap()
    {
        bool clear = true;
        for (size_t i = 0; i < lists.size() && clear; ++i) {
            const List& l = lists[i];
            if (l.all.empty() || !l.written) continue;
            clear = l.ascending && l.apart;
            for (size_t j = 0; j < lists.size() && clear; ++j) {
                const List& o = lists[j];
                clear = j == i || o.all.empty() || (o.ascending && (o.end <= l.all.front().begin || o.all.front().begin >= l.end));
            }
        }
        if (clear) return false;
        for (List& l : lists) if (!l.ascending) std::sort(l.all.begin(), l.all.end(), [](const Span& a, const Span& b) { return a.begin < b.begin; });
        uintptr_t written = 0, read = 0;
        for (;;) {
            List* next = nullptr;
            for (List& l : lists) if (l.at < l.all.size() && (!next || l.all[l.at].begin < next->all[next->at].begin)) next = &l;
            if (!next) return false;
            const Span s = next->all[next->at++];
            if (s.begin < written || (next->written && s.begin < read)) return true;
            uintptr_t& end = next->written ? written : read;
            end = std::max(end, s.end);
        }
    }
};

// One step on lists of tensors; seconds None: firsts are rows of 8 bits.  The entry point's code; or None, with nothing launched, where the Python function is to do it.
py::object adamw(const py::list& params, const py::list& grads, const py::list& firsts, const py::object& seconds, const py::object& masters, const py::object& step, const py::object& lr, const double beta1,
           const double beta2, const double eps, const double decay, const py::object& norm, const double max_norm, const uint32_t seed)
{
    const bool eight = seconds.is_none(), with_masters = !masters.is_none();
    const size_t count = params.size();
    if (!unobserved() || count == 0 || count > INT_MAX || grads.size() != count || firsts.size() != count) return py::none();
    if ((!eight && (!py::isinstance<py::list>(seconds) || py::len(seconds) != count)) || (with_masters && (!py::isinstance<py::list>(masters) || py::len(masters) != count))) return py::none();
    proteus_adamw_args a = {};
    int dev = -1;
    const bool inference = c10::InferenceMode::is_enabled(), tangents = torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr;
    std::vector<const Tensor*> written;
    std::vector<void*> p(count), s(count);
    std::vector<const void*> g(count);
    std::vector<float*> m(count), v(count), w(count);
    std::vector<int64_t> numel(count);
    std::vector<int> pt(count), gt(count);
    Spans spans;
    const int of_p = spans.list(true, count), of_g = spans.list(false, count), of_m = spans.list(true, count), of_v = spans.list(true, eight ? 0 : count), of_w = spans.list(true, with_masters ? count : 0),
              of_one = spans.list(true, 1), of_some = spans.list(false, 2);
    written.reserve(4 * count + 1);
    auto item = [&](const py::handle list, const size_t i) -> const Tensor* {
        PyObject* const o = PyList_GET_ITEM(list.ptr(), static_cast<Py_ssize_t>(i));
        if (!THPVariable_CheckExact(o)) return nullptr;
        const Tensor* t = &THPVariable_Unpack(o);
        if (!(tangents ? plain(*t) : plain_in_bulk(*t)) || (dev >= 0 && t->get_device() != dev) || (t->is_inference() && !inference)) return nullptr;
        return t;
    };
    for (size_t i = 0; i < count; ++i) {
        const Tensor* const x = item(params, i);
        if (!x) return py::none();
        dev = x->get_device();
        const Tensor *const d = item(grads, i), *const first = item(firsts, i), *const second = eight ? nullptr : item(seconds, i);
        if (!d || !first || (!eight && !second)) return py::none();
        numel[i] = x->numel();
        pt[i] = dtype_of(x->scalar_type());
        gt[i] = dtype_of(d->scalar_type());
        if (pt[i] < 0 || gt[i] < 0 || !x->is_non_overlapping_and_dense()) return py::none();
        auto alike = [&](const Tensor& t) { return t.sizes() == x->sizes() && t.strides() == x->strides(); };
        auto floats_like = [&](const Tensor& t) { return t.scalar_type() == at::kFloat && alike(t); };
        if (!alike(*d)) return py::none();
        if (eight ? first->scalar_type() != at::kByte || !first->is_contiguous() || static_cast<size_t>(first->numel()) != proteus_adamw_state_bytes(numel[i])
                  : !floats_like(*first) || !floats_like(*second)) return py::none();
        p[i] = x->mutable_data_ptr();
        g[i] = d->const_data_ptr();
        spans.add(of_p, p[i], numel[i] * x->itemsize());
        spans.add(of_g, g[i], numel[i] * d->itemsize());
        written.push_back(x);
        written.push_back(first);
        if (eight) {
            s[i] = first->mutable_data_ptr();
            spans.add(of_m, s[i], first->numel());
        } else {
            m[i] = static_cast<float*>(first->mutable_data_ptr());
            v[i] = static_cast<float*>(second->mutable_data_ptr());
            spans.add(of_m, m[i], numel[i] * 4);
            spans.add(of_v, v[i], numel[i] * 4);
            written.push_back(second);
        }
        if (with_masters && PyList_GET_ITEM(masters.ptr(), static_cast<Py_ssize_t>(i)) != Py_None) {
            const Tensor* const t = item(masters, i);
            if (!t || !floats_like(*t)) return py::none();
            w[i] = static_cast<float*>(t->mutable_data_ptr());
            spans.add(of_w, w[i], numel[i] * 4);
            written.push_back(t);
        }
    }
    if (!current(dev)) return py::none();
    auto scalar = [&](const py::object& o, const at::ScalarType type, const bool writes) -> void* {
        Tensor t;
        if (!get(o, t, dev) || t.scalar_type() != type || t.numel() != 1 || (t.is_inference() && !inference)) return nullptr;
        void* const at = t.data_ptr();
        spans.add(writes ? of_one : of_some, at, t.itemsize());
        return at;
    };
    const Tensor* counted = nullptr;
    if (THPVariable_Check(step.ptr())) {
        if (!(a.step_gpu = static_cast<int64_t*>(scalar(step, at::kLong, true)))) return py::none();
        counted = &THPVariable_Unpack(step.ptr());
        written.push_back(counted);
    } else if (!PyLong_CheckExact(step.ptr())) return py::none();
    else a.step = step.cast<int64_t>();
    if (THPVariable_Check(lr.ptr())) {
        if (!(a.lr_gpu = static_cast<const float*>(scalar(lr, at::kFloat, false)))) return py::none();
    } else a.lr = lr.cast<double>();
    if (!norm.is_none() && !(a.norm = static_cast<const float*>(scalar(norm, at::kFloat, false)))) return py::none();
    if (spans.overlap()) return py::none();
    a.params = p.data(); a.grads = g.data(); a.numel = numel.data(); a.param_types = pt.data(); a.grad_types = gt.data();
    a.masters = with_masters ? w.data() : nullptr;
    a.count = static_cast<int>(count);
    if (eight) a.states = s.data();
    else { a.exp_avgs = m.data(); a.exp_avg_sqs = v.data(); }
    a.beta1 = beta1; a.beta2 = beta2; a.eps = eps; a.weight_decay = decay; a.max_norm = static_cast<float>(max_norm); a.seed = seed;
    const int rc = proteus_adamw(&a, stream_of(dev));
    if (rc < 0) return py::none();                          // (refused before anything was launched)
    // (a launch that failed: those before it have written, so that the step must not be taken again)
    for (const Tensor* t : written) if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
    return py::cast(rc);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m)
{
    m.def("version", [] { return proteus_version(); });
    m.def("attention", &attention);
    m.def("embedding", &embedding);
    m.def("aniso", &aniso);
    m.def("qk_norm_rotate", &qk_norm_rotate);
    m.def("gated_mlp", &gated_mlp);
    m.def("linear_ce", &linear_ce);
    m.def("clip", &clip);
    m.def("adamw", &adamw);
    // the general backward functions (kept for as long as the process lives)
    m.def("set_general", [](py::object attention_bwd, py::object embedding_bwd, py::object aniso_bwd, py::object qk_bwd, py::object gated_bwd, py::object ce_bwd) {
        g_attention_backward = attention_bwd.release().ptr();
        g_embedding_backward = embedding_bwd.release().ptr();
        g_aniso_backward = aniso_bwd.release().ptr();
        g_qk_backward = qk_bwd.release().ptr();
        g_gated_backward = gated_bwd.release().ptr();
        g_ce_backward = ce_bwd.release().ptr();
    });
}
