// bindings.cpp -- the training operators as differentiable PyTorch functions (module _atlas_train): checks of arguments, outputs and workspaces from
// PyTorch's allocator, the current stream, autograd nodes. The kernels are behind the C-ABI of include/atlas_train.h, whose library is handed over by path.
//
// Native, because a step on a few tokens is bound by the host: through ctypes and Python autograd functions the dense layer's step on 41 tokens took
// 176 us of host time around 37 us of kernels, most of it in the backward pass, which the engine runs on a thread of its own that then waits for the
// interpreter.
#include <dlfcn.h>
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include "../../../include/atlas_train.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Refusal : std::runtime_error { using std::runtime_error::runtime_error; };

struct Api {
    decltype(&atlas_train_abi_version) abi_version;
    decltype(&atlas_attention_workspace_bytes) attention_workspace_bytes;
    decltype(&atlas_attention_forward) attention_forward;
    decltype(&atlas_attention_backward) attention_backward;
    decltype(&atlas_gemm_workspace_bytes) gemm_workspace_bytes;
    decltype(&atlas_gemm) gemm;
    decltype(&atlas_linear_dz_workspace_bytes) linear_dz_workspace_bytes;
    decltype(&atlas_linear_dz) linear_dz;
    decltype(&atlas_compress) compress;
    decltype(&atlas_decompress) decompress;
    decltype(&atlas_layer_norm_forward) layer_norm_forward;
    decltype(&atlas_layer_norm_workspace_bytes) layer_norm_workspace_bytes;
    decltype(&atlas_layer_norm_backward) layer_norm_backward;
} api;

template <class F> void symbol(void* lib, const char* name, F& f) {
    f = reinterpret_cast<F>(dlsym(lib, name));
    if (!f) throw Refusal(std::string("symbol missing: ") + name);
}
void bind(const std::string& path) {
    void* lib = dlopen(path.c_str(), RTLD_NOW | RTLD_LOCAL);
    if (!lib) throw Refusal(std::string("cannot load ") + path + ": " + dlerror());
    symbol(lib, "atlas_train_abi_version", api.abi_version);
    symbol(lib, "atlas_attention_workspace_bytes", api.attention_workspace_bytes);
    symbol(lib, "atlas_attention_forward", api.attention_forward);
    symbol(lib, "atlas_attention_backward", api.attention_backward);
    symbol(lib, "atlas_gemm_workspace_bytes", api.gemm_workspace_bytes);
    symbol(lib, "atlas_gemm", api.gemm);
    symbol(lib, "atlas_linear_dz_workspace_bytes", api.linear_dz_workspace_bytes);
    symbol(lib, "atlas_linear_dz", api.linear_dz);
    symbol(lib, "atlas_compress", api.compress);
    symbol(lib, "atlas_decompress", api.decompress);
    symbol(lib, "atlas_layer_norm_forward", api.layer_norm_forward);
    symbol(lib, "atlas_layer_norm_workspace_bytes", api.layer_norm_workspace_bytes);
    symbol(lib, "atlas_layer_norm_backward", api.layer_norm_backward);
    if (api.abi_version() != ATLAS_TRAIN_ABI_VERSION) throw Refusal(path + " has another ABI version than its binding");
}

// ---- checks ----
template <class... A> [[noreturn]] void refuse(const A&... a) { throw Refusal(c10::str(a...)); }
void ok(int rc, const char* what) {
    if (rc == 0) return;
    const char* names[3] = {"ATLAS_TRAIN_E_BADARG", "ATLAS_TRAIN_E_WORKSPACE", "ATLAS_TRAIN_E_UNSUPPORTED"};
    if (rc < 0 && rc >= -3) refuse(what, " failed: ", names[-rc - 1]);
    refuse(what, " failed: hipError_t ", rc);
}
int dtype_code(at::ScalarType t) {
    switch (t) {
        case at::kHalf: return ATLAS_TRAIN_F16;
        case at::kBFloat16: return ATLAS_TRAIN_BF16;
        case at::kFloat: return ATLAS_TRAIN_F32;
        default: return -1;
    }
}
// A kernel reads values. A trace would hold the empty result that it fills and nothing that fills it; a tensor of a function transform, a fake one or one of a
// class with a dispatch of its own has no values to read, or not all of them
void only_values(std::initializer_list<const Tensor*> tensors) {
    using c10::impl::TorchDispatchModeKey;
    using c10::impl::TorchDispatchModeTLS;
    bool traced = torch::jit::tracer::isTracing();
    if (TorchDispatchModeTLS::any_modes_set())
        for (const auto mode : {TorchDispatchModeKey::FAKE, TorchDispatchModeKey::PROXY, TorchDispatchModeKey::FUNCTIONAL}) traced |= TorchDispatchModeTLS::get_mode(mode).has_value();
    if (traced) refuse("a trace cannot hold the kernels of train_ops");
    constexpr c10::DispatchKeySet wrapped({c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::BatchedNestedTensor, c10::DispatchKey::FuncTorchGradWrapper,
                                           c10::DispatchKey::Batched, c10::DispatchKey::Functionalize, c10::DispatchKey::Python, c10::DispatchKey::ZeroTensor});
    for (const Tensor* t : tensors)
        if (t->defined() && t->key_set().has_any(wrapped)) refuse("a tensor of the call is no plain tensor: it is of a function transform, a fake one, or of a class with a dispatch of its own");
}
// Nor does it know derivatives: the tangent of a dual tensor would be lost without a word, which says that the derivative is zero
void no_tangents(std::initializer_list<const Tensor*> tensors) {
    only_values(tensors);
    for (const Tensor* t : tensors)
        if (t->defined() && t->_fw_grad(0).defined()) refuse("forward-mode derivatives are not implemented: a tensor of the call has a tangent");
}
// the values in memory: of a conjugate's imaginary part torch keeps the values' negatives and a flag
Tensor in_memory(const Tensor& t) { return t.defined() && t.is_neg() ? t.resolve_neg() : t; }
Tensor or_none(const c10::optional<Tensor>& t) { return t ? *t : Tensor(); }
// a tensor the kernels can take: on a GPU, of a known dtype, like the others of the call
void operand(const char* name, const Tensor& t, const Tensor* like = nullptr) {
    if (!t.is_cuda()) refuse(name, " is on ", t.device(), ": train_ops run on an MI355X only; there is no CPU / eager fallback");
    if (t.layout() != at::kStrided) refuse(name, ": only dense tensors");
    if (dtype_code(t.scalar_type()) < 0) refuse(name, ": unsupported dtype ", t.scalar_type());
    if (!like) return;
    if (t.scalar_type() != like->scalar_type()) refuse(name, " is ", t.scalar_type(), ", the call's other tensors are ", like->scalar_type());
    if (t.device() != like->device()) refuse(name, " is on ", t.device(), ", the call's other tensors on ", like->device());
}
// a 0 / 1 tensor as bytes of 0 and 1
Tensor decisions(const char* name, const Tensor& t, at::IntArrayRef shape, const Tensor& like) {
    only_values({&t});
    if ((t.scalar_type() != at::kBool && t.scalar_type() != at::kByte) || t.device() != like.device()) refuse(name, " has to be a bool or uint8 tensor on ", like.device());
    if (t.sizes() != shape) refuse(name, " has shape ", t.sizes(), ", expected ", shape);
    return t.scalar_type() == at::kByte ? t.ne(0) : t;
}

// the tensors' device as the current one, and its current stream
struct On {
    c10::OptionalDeviceGuard guard;
    void* stream;
    explicit On(const Tensor& t) : guard(t.device()), stream(c10::hip::getCurrentHIPStream(t.device().index()).stream()) {}
};

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
uint8_t* bytes(const Tensor& t) { return static_cast<uint8_t*>(ptr(t)); }
Tensor empty_bytes(int64_t n, const Tensor& like) { return at::empty({n}, like.options().dtype(at::kByte)); }

// any tensor as [rows, last dimension] with a contiguous last dimension, as a view where it is one already, and its row stride
struct Rows { Tensor t; int64_t m, n, ld; };
Rows rows(const Tensor& x) {
    const int64_t n = x.size(-1);
    Tensor t = x.dim() == 2 ? x : x.reshape({n ? x.numel() / n : 0, n});
    const int64_t m = t.size(0);
    if (m <= 1 || n == 0) return {t.contiguous(), m, n, n};
    if (t.stride(1) != 1 && n > 1) t = t.contiguous();
    return {t, m, n, t.stride(0)};
}

// What a forward pass saved: contiguous, but for those of `strided` (a bit each). Hooks on saved tensors may give back others: on the host, of other strides
variable_list saved(AutogradContext* ctx, const Tensor& like, unsigned strided) {
    at::NoGradGuard no_grad_inside;
    auto tensors = ctx->get_saved_variables();
    for (size_t i = 0; i < tensors.size(); ++i) {
        if (!tensors[i].defined()) continue;
        if (tensors[i].device() != like.device()) refuse("a saved tensor came back on ", tensors[i].device(), ", its gradient is on ", like.device());
        if (!(strided >> i & 1)) tensors[i] = tensors[i].contiguous();
    }
    return tensors;
}

// A backward pass here is differentiable once: under create_graph its gradients carry a node that says so when it is asked
variable_list once(variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    auto error = std::make_shared<torch::autograd::DelayedError>("atlas_amd.train_ops are differentiable once: trying to differentiate a gradient again",
                                                                 static_cast<int64_t>(grads.size()));
    for (auto& g : grads)
        if (g.defined()) g = g.detach().requires_grad_();
    return (*error)(std::move(grads));
}
bool wants(const Tensor& t) { return t.defined() && t.requires_grad(); }

// A backward pass runs a node on the stream that it was made on. Work on the default stream cannot be part of a capture, and trying to ends the process:
// a captured call refuses a tensor whose node was made there (a leaf's lives as long as some graph of it)
void capturable(std::initializer_list<const Tensor*> inputs, const On& on) {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    if (!on.stream || hipStreamIsCapturing(static_cast<hipStream_t>(on.stream), &status) != hipSuccess || status == hipStreamCaptureStatusNone) return;
    for (const Tensor* t : inputs) {
        if (!wants(*t)) continue;
        const auto node = t->grad_fn() ? t->grad_fn() : torch::autograd::impl::try_get_grad_accumulator(*t);
        const auto made = node ? node->stream() : c10::nullopt;
        if (made && *made == c10::impl::VirtualGuardImpl(t->device().type()).getDefaultStream(t->device()))
            refuse("captured into a graph, but a graph of the same tensors from the default stream is alive: a backward pass could not be captured; let go of it first");
    }
}

// ---- attention ----
struct AttentionRest { int64_t max_q, max_k, cols; double scale, keep_scale; };
struct AttentionFixed { Tensor q_offsets, k_offsets, key_mask, keep; AttentionRest r; };      // what takes no gradient (and may be undefined)

// [T, H, D] with a contiguous, 16-byte aligned last dimension and rows within the kernels' reach, as a view where it is one already
Tensor heads_ready(const Tensor& t) {
    const int64_t s = 16 / t.element_size();
    const bool fine = (t.stride(2) == 1 || t.size(2) == 1) && t.stride(0) % s == 0 && t.stride(1) % s == 0 && t.stride(0) < (s << 20) &&
                      reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
    if (fine) return t;
    const Tensor c = t.contiguous();                                         // (the same tensor where it only lies off a 16-byte border, or has a lone row of any stride)
    return c.is_same(t) ? t.clone(at::MemoryFormat::Contiguous) : c;
}
atlas_attention_args attention_args(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& q_offsets, const Tensor& k_offsets, const Tensor& key_mask,
                                    const Tensor& bits, const Tensor& out, const Tensor& out_rest, const Tensor& lse, const AttentionRest& r) {
    atlas_attention_args a = {};
    a.q = q.data_ptr(); a.k = k.data_ptr(); a.v = v.data_ptr();
    a.q_row = q.stride(0); a.q_head = q.stride(1); a.k_row = k.stride(0); a.k_head = k.stride(1); a.v_row = v.stride(0); a.v_head = v.stride(1);
    a.q_offsets = static_cast<const int32_t*>(q_offsets.data_ptr());
    a.k_offsets = static_cast<const int32_t*>(k_offsets.data_ptr());
    a.total_q = q.size(0); a.total_k = k.size(0);
    a.batch = static_cast<int>(q_offsets.numel() - 1);
    a.heads = static_cast<int>(q.size(1)); a.kv_heads = static_cast<int>(k.size(1)); a.dim = static_cast<int>(q.size(2));
    a.max_q = static_cast<int>(r.max_q); a.max_k = static_cast<int>(r.max_k);
    a.dtype = dtype_code(q.scalar_type());
    a.keep_cols = static_cast<int>(r.cols);
    a.key_mask = bytes(key_mask);
    a.keep_bits = static_cast<uint32_t*>(ptr(bits));
    a.scale = static_cast<float>(r.scale); a.keep_scale = static_cast<float>(r.keep_scale);
    a.out = out.data_ptr(); a.lse = static_cast<float*>(lse.data_ptr()); a.out_rest = bytes(out_rest);
    return a;
}
Tensor attention_workspace(atlas_attention_args& a, bool backward, const Tensor& like) {
    a.ws_bytes = api.attention_workspace_bytes(&a, backward);
    Tensor ws;
    if (a.ws_bytes) ws = empty_bytes(static_cast<int64_t>(a.ws_bytes), like);
    a.ws = ptr(ws);
    return ws;
}
struct AttentionSaved { Tensor out, lse, bits, out_rest; };
AttentionSaved attention_run(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& q_offsets, const Tensor& k_offsets, const Tensor& key_mask, const Tensor& keep,
                             const AttentionRest& r, bool train) {
    AttentionSaved s;
    s.out = at::empty(q.sizes(), q.options());
    s.lse = at::empty({q.size(1), q.size(0)}, q.options().dtype(at::kFloat));
    // the decisions as bits are what the backward pass reads (never an empty tensor: its pointer says "dropout")
    if (keep.defined() && train) s.bits = at::empty({std::max<int64_t>(1, s.lse.numel() * ((r.cols + 31) / 32))}, q.options().dtype(at::kInt));
    if (train && q.element_size() == 2) s.out_rest = empty_bytes(q.size(0) * q.size(1) * (q.size(2) <= 64 ? 64 : 128), q);       // (fp32: nothing that counts)
    auto a = attention_args(q, k, v, q_offsets, k_offsets, key_mask, s.bits, s.out, s.out_rest, s.lse, r);
    if (keep.defined()) {
        // no column to read, but dropout all the same: nothing is kept
        a.keep = keep.numel() ? bytes(keep) : static_cast<const uint8_t*>(q_offsets.data_ptr());
        a.keep_row = keep.size(0) > 1 ? keep.stride(0) : 0; a.keep_head = keep.stride(1);
    }
    const Tensor ws = attention_workspace(a, false, q);
    On on(q);
    ok(api.attention_forward(&a, on.stream), "atlas_attention_forward");
    return s;
}
struct Attention : torch::autograd::Function<Attention> {
    static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const AttentionFixed& f) {
        const AttentionRest& r = f.r;
        auto s = attention_run(q, k, v, f.q_offsets, f.k_offsets, f.key_mask, f.keep, r, true);
        ctx->save_for_backward({q, k, v, f.q_offsets, f.k_offsets, f.key_mask, s.bits, s.out, s.lse, s.out_rest});
        ctx->saved_data["rest"] = std::vector<int64_t>{r.max_q, r.max_k, r.cols};
        ctx->saved_data["scales"] = std::vector<double>{r.scale, r.keep_scale};
        return s.out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        no_tangents({&grads[0]});
        const auto t = saved(ctx, grads[0], 7);
        const auto rest = ctx->saved_data["rest"].toIntVector();
        const auto scales = ctx->saved_data["scales"].toDoubleVector();
        const AttentionRest r{rest[0], rest[1], rest[2], scales[0], scales[1]};
        const Tensor& lse = t[8];
        Tensor dq, dk, dv;
        {
        at::NoGradGuard no_grad_inside;
        const Tensor q = heads_ready(t[0]), k = heads_ready(t[1]), v = heads_ready(t[2]);
        const Tensor dout = heads_ready(in_memory(grads[0])), delta = at::empty_like(lse);
        dq = at::empty(q.sizes(), q.options()); dk = at::empty(k.sizes(), k.options()); dv = at::empty(v.sizes(), v.options());
        auto a = attention_args(q, k, v, t[3], t[4], t[5], t[6], t[7], t[9], lse, r);
        a.dout = dout.data_ptr(); a.dout_row = dout.stride(0); a.dout_head = dout.stride(1);
        a.dq = dq.data_ptr(); a.dk = dk.data_ptr(); a.dv = dv.data_ptr(); a.delta = static_cast<float*>(delta.data_ptr());
        const Tensor ws = attention_workspace(a, true, q);
        On on(q);
        ok(api.attention_backward(&a, on.stream), "atlas_attention_backward");
        }
        auto g = once({dq, dk, dv});
        return {g[0], g[1], g[2], {}};
    }
};
Tensor offsets(const char* name, const Tensor& t, const Tensor& like) {
    only_values({&t});
    if (t.dim() != 1 || t.numel() < 1 || (t.scalar_type() != at::kInt && t.scalar_type() != at::kLong) || t.device() != like.device())
        refuse(name, " has to be a 1-d int32 (or int64) tensor of batch + 1 offsets on ", like.device());
    return t.to(at::kInt).contiguous();
}
Tensor attention(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& q_offsets_, const c10::optional<Tensor>& k_offsets_, c10::optional<int64_t> max_q,
                 c10::optional<int64_t> max_k, const c10::optional<Tensor>& key_mask_, c10::optional<double> scale, const c10::optional<Tensor>& keep_, double keep_scale) {
    no_tangents({&q_, &k_, &v_});
    const Tensor q = in_memory(q_), k = in_memory(k_), v = in_memory(v_);
    operand("q", q);
    operand("k", k, &q);
    operand("v", v, &q);
    if (q.dim() != 3 || k.dim() != 3 || k.sizes() != v.sizes() || k.size(2) != q.size(2))
        refuse("attention takes q [Tq, H, D] and k, v [Tk, H', D]: got ", q.sizes(), ", ", k.sizes(), ", ", v.sizes());
    const int64_t dim = q.size(2);
    if (std::max({q.size(0), q.size(1), k.size(0), k.size(1), q_offsets_.numel()}) > INT32_MAX) refuse("attention: a dimension of 2^31 or more");
    if (dim == 0 || dim % 8 || dim > 128) refuse("attention: head dimension ", dim, "; multiples of 8 up to 128 are implemented");
    if (k.size(1) == 0 || q.size(1) == 0 || q.size(1) % k.size(1)) refuse("attention: ", q.size(1), " query heads cannot share ", k.size(1), " key heads evenly");
    const Tensor q_offsets = offsets("q_offsets", q_offsets_, q);
    if (!k_offsets_ && k.size(0) != q.size(0)) refuse("attention: k_offsets is needed where q and k have different rows");
    const Tensor k_offsets = k_offsets_ ? offsets("k_offsets", *k_offsets_, q) : q_offsets;
    if (k_offsets.numel() != q_offsets.numel()) refuse("attention: ", q_offsets.numel() - 1, " query sequences, ", k_offsets.numel() - 1, " key sequences");
    AttentionRest r;
    r.scale = scale ? *scale : 1.0 / std::sqrt(static_cast<double>(dim));
    if (!(static_cast<float>(r.scale) > 0.f) || !std::isfinite(static_cast<float>(r.scale))) refuse("attention: scale ", r.scale, " is not positive");
    r.keep_scale = keep_scale;
    r.cols = 0;
    Tensor key_mask, keep;
    if (key_mask_) key_mask = decisions("key_mask", *key_mask_, {k.size(0)}, q).contiguous();
    if (keep_) {
        r.cols = keep_->dim() == 3 ? keep_->size(2) : -1;
        keep = decisions("keep", *keep_, {q.size(0), q.size(1), r.cols}, q);
        if (r.cols > INT32_MAX) refuse("attention: keep has 2^31 columns or more");
        if ((keep.stride(2) != 1 && r.cols > 1) || keep.stride(0) >= 1 << 26) keep = keep.contiguous();
    }
    const auto longest = [](c10::optional<int64_t> given, int64_t n) { return std::min<int64_t>(given ? std::max<int64_t>(0, std::min(*given, n)) : n, INT32_MAX); };
    r.max_q = longest(max_q, q.size(0));
    r.max_k = longest(max_k, k.size(0));
    const Tensor q1 = heads_ready(q), k1 = heads_ready(k), v1 = heads_ready(v);
    if (at::GradMode::is_enabled() && (wants(q) || wants(k) || wants(v))) {
        capturable({&q, &k, &v}, On(q));
        return Attention::apply(q1, k1, v1, AttentionFixed{q_offsets, k_offsets, key_mask, keep, r});
    }
    return attention_run(q1, k1, v1, q_offsets, k_offsets, key_mask, keep, r, false).out;
}

// ---- 8-bit activations ----
std::pair<Tensor, Tensor> code_buffers(int64_t m, int64_t n, const Tensor& like) {
    const int64_t groups = (n + 31) / 32;
    const auto o = like.options().dtype(at::kByte);
    return {at::empty({m, groups * 32}, o), at::empty({m, groups}, o)};
}
std::pair<Tensor, Tensor> compress_rows(const Rows& x) {
    auto c = code_buffers(x.m, x.n, x.t);
    On on(x.t);
    ok(api.compress(x.t.data_ptr(), x.ld, x.m, static_cast<int>(x.n), dtype_code(x.t.scalar_type()), bytes(c.first), bytes(c.second), on.stream), "atlas_compress");
    return c;
}
std::pair<Tensor, Tensor> compress(const Tensor& x) {
    only_values({&x});
    operand("x", x);
    if (x.dim() < 1) refuse("compress takes a tensor of at least one dimension");
    if (x.size(-1) > (1 << 30)) refuse("compress: rows of more than 2^30 elements");
    at::NoGradGuard no_grad_inside;
    return compress_rows(rows(in_memory(x)));
}
Tensor decompress(const Tensor& codes, const Tensor& scales, std::vector<int64_t> shape, at::ScalarType dtype) {
    only_values({&codes, &scales});
    if (dtype_code(dtype) < 0) refuse("decode: unsupported dtype ", dtype);
    if (shape.empty() || shape.back() > (1 << 30) || *std::min_element(shape.begin(), shape.end()) < 0) refuse("decode: shape ", at::IntArrayRef(shape));
    const int64_t n = shape.back(), m = n ? c10::multiply_integers(shape) / n : 0, groups = (n + 31) / 32;
    const Tensor* both[2] = {&codes, &scales};
    for (int i = 0; i < 2; ++i) {
        const int64_t cols = i ? groups : groups * 32;
        if (!both[i]->is_cuda() || both[i]->device() != codes.device() || both[i]->scalar_type() != at::kByte || !both[i]->is_contiguous() || both[i]->dim() != 2 ||
            both[i]->size(0) != m || both[i]->size(1) != cols || (i == 0 && reinterpret_cast<uintptr_t>(codes.data_ptr()) % 16))
            refuse("decode: ", i ? "scales" : "codes", " have to be uint8 [", m, ", ", cols, "] for shape ", at::IntArrayRef(shape), ", as compress gives them");
    }
    Tensor out = at::empty(shape, codes.options().dtype(dtype));
    On on(out);
    ok(api.decompress(bytes(codes), bytes(scales), m, static_cast<int>(n), dtype_code(dtype), out.data_ptr(), on.stream), "atlas_decompress");
    return out;
}

// ---- dense layer ----
atlas_gemm_args product(const Tensor& a, int64_t lda, const Tensor& b, int64_t ldb, const Tensor& c, int64_t m, int64_t n, int64_t k, int a_layout, int b_layout) {
    atlas_gemm_args g = {};
    g.a = a.data_ptr(); g.b = ptr(b); g.lda = lda; g.ldb = ldb; g.ldc = n;
    g.m = static_cast<int>(m); g.n = static_cast<int>(n); g.k = static_cast<int>(k);
    g.dtype = dtype_code(a.scalar_type()); g.a_layout = a_layout; g.b_layout = b_layout;
    g.c = c.data_ptr();
    return g;
}
void run(atlas_gemm_args& g, const Tensor& like, void* stream) {
    const size_t need = api.gemm_workspace_bytes(&g);
    Tensor ws;
    if (need) {
        ws = empty_bytes(static_cast<int64_t>(need), like);
        g.ws = ws.data_ptr();
        g.ws_bytes = need;
    }
    ok(api.gemm(&g, stream), "atlas_gemm");
}
struct LinearRest { bool gelu, eight_bits; double keep_scale; bool need_x, need_w, need_b, need_r; Tensor keep; };
struct LinearSaved { Tensor y, z, z_codes, z_scales, x_codes, x_scales; };
LinearSaved linear_run(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& residual, const LinearRest& r) {
    LinearSaved s;
    const Rows x2 = rows(x), w2 = rows(weight);
    const int64_t m = x2.m, n = w2.m, k = w2.n;
    auto shape = x.sizes().vec();
    shape.back() = n;
    s.y = at::empty(shape, x.options());
    auto g = product(x2.t, x2.ld, w2.t, w2.ld, s.y, m, n, k, 0, 0);
    g.bias = ptr(bias);
    g.act = r.gelu;
    g.keep = bytes(r.keep);
    g.keep_scale = static_cast<float>(r.keep_scale);
    Rows r2{};
    if (residual.defined()) {
        r2 = rows(residual);
        g.residual = r2.t.data_ptr();
        g.ld_residual = r2.ld;
    }
    if (r.gelu && (r.need_x || r.need_w || r.need_b)) {                      // what the activation's slope is taken from
        if (r.eight_bits) {
            std::tie(s.z_codes, s.z_scales) = code_buffers(m, n, x);
            g.save_z_codes = bytes(s.z_codes);
            g.save_z_scales = bytes(s.z_scales);
        } else {
            s.z = at::empty({m, n}, x.options());
            g.save_z = s.z.data_ptr();
        }
    }
    {
        On on(x);
        run(g, x, on.stream);
    }
    if (r.eight_bits && r.need_w) std::tie(s.x_codes, s.x_scales) = compress_rows(x2);
    return s;
}
struct Linear : torch::autograd::Function<Linear> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const c10::optional<Tensor>& bias, const c10::optional<Tensor>& residual,
                          const LinearRest& r) {
        auto s = linear_run(x, weight, or_none(bias), or_none(residual), r);
        ctx->save_for_backward({r.need_w && !r.eight_bits ? x : Tensor(), s.x_codes, s.x_scales, weight, s.z, s.z_codes, s.z_scales, r.keep});
        ctx->saved_data["shape"] = x.sizes().vec();
        ctx->saved_data["keep_scale"] = r.keep_scale;
        ctx->saved_data["need"] = static_cast<int64_t>(r.need_x | r.need_w << 1 | r.need_b << 2 | r.need_r << 3);
        return s.y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        no_tangents({&grads[0]});
        const auto t = saved(ctx, grads[0], 9);
        const Tensor &x = t[0], &x_codes = t[1], &x_scales = t[2], &weight = t[3], &z = t[4], &z_codes = t[5], &z_scales = t[6], &keep = t[7];
        const int64_t need = ctx->saved_data["need"].toInt();
        const bool need_x = need & 1, need_w = need & 2, need_b = need & 4, need_r = need & 8;
        const float keep_scale = static_cast<float>(ctx->saved_data["keep_scale"].toDouble());
        Tensor dx, dw, db;
        {
            at::NoGradGuard no_grad_inside;
            const Tensor dy = in_memory(grads[0]);
            const int64_t n = weight.size(0), k = weight.size(1);
            const Rows d2 = rows(dy);
            const int64_t m = d2.m;
            const int dtype = dtype_code(dy.scalar_type());
            On on(dy);
            const bool changed = z.defined() || z_codes.defined() || keep.defined();     // dz is dy otherwise
            const bool want_dz = changed && (need_x || need_w);
            Tensor dz = d2.t;
            int64_t ldz = d2.ld;
            if (want_dz || need_b) {
                Tensor ws;
                if (want_dz) { dz = at::empty({m, n}, dy.options()); ldz = n; }
                if (need_b) {
                    db = at::empty({n}, dy.options());
                    ws = empty_bytes(static_cast<int64_t>(api.linear_dz_workspace_bytes(m, static_cast<int>(n))), dy);
                }
                ok(api.linear_dz(d2.t.data_ptr(), d2.ld, ptr(z), bytes(z_codes), bytes(z_scales), bytes(keep), keep_scale, m, static_cast<int>(n), dtype,
                                 want_dz ? dz.data_ptr() : nullptr, ptr(db), ptr(ws), ws.defined() ? ws.numel() : 0, on.stream), "atlas_linear_dz");
            }
            if (need_x) {
                const Rows w2 = rows(weight);
                dx = at::empty(ctx->saved_data["shape"].toIntVector(), dy.options());
                auto g = product(dz, ldz, w2.t, w2.ld, dx, m, k, n, 0, 1);
                run(g, dy, on.stream);
            }
            if (need_w) {
                dw = at::empty({n, k}, dy.options());
                if (x_codes.defined()) {
                    auto g = product(dz, ldz, Tensor(), x_codes.size(1), dw, n, k, m, 1, 1);
                    g.b_codes = bytes(x_codes);
                    g.b_scales = bytes(x_scales);
                    run(g, dy, on.stream);
                } else {
                    const Rows x2 = rows(x);
                    auto g = product(dz, ldz, x2.t, x2.ld, dw, n, k, m, 1, 1);
                    run(g, dy, on.stream);
                }
            }
        }
        Tensor dr;
        if (need_r) dr = grads[0];
        auto out = once({dx, dw, db});
        return {out[0], out[1], out[2], dr, {}};
    }
};
Tensor linear(const Tensor& x_, const Tensor& weight_, const c10::optional<Tensor>& bias_, const c10::optional<std::string>& activation, const c10::optional<Tensor>& keep_,
              double keep_scale, const c10::optional<Tensor>& residual_, const c10::optional<std::string>& checkpoint) {
    const Tensor bias_or_none = or_none(bias_), residual_or_none = or_none(residual_);
    no_tangents({&x_, &weight_, &bias_or_none, &residual_or_none});
    const Tensor x = in_memory(x_), weight = in_memory(weight_);
    operand("x", x);
    operand("weight", weight, &x);
    if (weight.dim() != 2 || x.dim() < 1 || x.size(-1) != weight.size(1)) refuse("linear takes x [..., K] and weight [N, K]: got ", x.sizes(), " and ", weight.sizes());
    const int64_t n = weight.size(0), k = weight.size(1);
    if (n == 0 || k == 0) refuse("linear: a layer of ", k, " inputs and ", n, " outputs");
    if (x.numel() / k > (1 << 30) || n > (1 << 30) || k > (1 << 30)) refuse("linear: a dimension of more than 2^30");
    auto shape = x.sizes().vec();
    shape.back() = n;
    c10::optional<Tensor> bias, residual;
    Tensor keep;
    if (bias_) {
        operand("bias", *bias_, &x);
        if (bias_->dim() != 1 || bias_->size(0) != n) refuse("bias has shape ", bias_->sizes(), ", expected [", n, "]");
        bias = in_memory(*bias_).contiguous();
    }
    if (residual_) {
        operand("residual", *residual_, &x);
        if (residual_->sizes() != at::IntArrayRef(shape)) refuse("residual has shape ", residual_->sizes(), ", expected ", shape);
        residual = in_memory(*residual_);
    }
    if (keep_) keep = decisions("keep", *keep_, shape, x).contiguous();
    if (activation && *activation != "gelu") refuse("activation='", *activation, "': None and the exact-erf 'gelu' are implemented");
    if (checkpoint && *checkpoint != "e4m3") refuse("checkpoint='", *checkpoint, "': None and 'e4m3' are implemented");
    LinearRest r{activation.has_value(), checkpoint.has_value(), keep_scale, wants(x), wants(weight), bias && wants(*bias), residual && wants(*residual), keep};
    if (at::GradMode::is_enabled() && (r.need_x || r.need_w || r.need_b || r.need_r)) {
        const Tensor none;
        capturable({&x, &weight, bias ? &*bias : &none, residual ? &*residual : &none}, On(x));
        return Linear::apply(x, weight, bias, residual, r);
    }
    r.need_x = r.need_w = r.need_b = r.need_r = false;
    return linear_run(x, weight, or_none(bias), or_none(residual), r).y;
}

// ---- layer norm ----
std::pair<Tensor, Tensor> layer_norm_run(const Tensor& x, const Tensor& weight, const Tensor& bias, double eps) {
    const Rows x2 = rows(x);
    Tensor y = at::empty(x.sizes(), x.options()), stats = at::empty({x2.m, 2}, x.options().dtype(at::kFloat));
    On on(x);
    ok(api.layer_norm_forward(x2.t.data_ptr(), x2.ld, weight.data_ptr(), bias.data_ptr(), static_cast<float>(eps), x2.m, static_cast<int>(x2.n),
                              dtype_code(x.scalar_type()), y.data_ptr(), static_cast<float*>(stats.data_ptr()), on.stream), "atlas_layer_norm_forward");
    return {y, stats};
}
struct LayerNorm : torch::autograd::Function<LayerNorm> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Tensor& bias, double eps) {
        auto s = layer_norm_run(x, weight, bias, eps);
        ctx->save_for_backward({x, weight, s.second});
        ctx->saved_data["need"] = static_cast<int64_t>(wants(x) | wants(weight) << 1 | wants(bias) << 2);
        return s.first;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        no_tangents({&grads[0]});
        const auto t = saved(ctx, grads[0], 1);
        const Tensor &x = t[0], &weight = t[1], &stats = t[2];
        const int64_t need = ctx->saved_data["need"].toInt();
        Tensor dx, dw, db;
        {
            at::NoGradGuard no_grad_inside;
            const Rows x2 = rows(x), d2 = rows(in_memory(grads[0]));
            Tensor ws;
            if (need & 1) dx = at::empty(x.sizes(), x.options());
            if (need & 6) {
                dw = at::empty(weight.sizes(), x.options());
                db = at::empty(weight.sizes(), x.options());
                ws = empty_bytes(static_cast<int64_t>(api.layer_norm_workspace_bytes(x2.m, static_cast<int>(x2.n))), x);
            }
            On on(x);
            ok(api.layer_norm_backward(x2.t.data_ptr(), x2.ld, weight.data_ptr(), static_cast<const float*>(stats.data_ptr()), d2.t.data_ptr(), d2.ld, x2.m,
                                       static_cast<int>(x2.n), dtype_code(x.scalar_type()), ptr(dx), ptr(dw), ptr(db), ptr(ws), ws.defined() ? ws.numel() : 0, on.stream),
               "atlas_layer_norm_backward");
        }
        if (!(need & 2)) dw = Tensor();
        if (!(need & 4)) db = Tensor();
        auto out = once({dx, dw, db});
        return {out[0], out[1], out[2], {}};
    }
};
Tensor layer_norm(const Tensor& x_, const Tensor& weight_, const Tensor& bias_, double eps) {
    no_tangents({&x_, &weight_, &bias_});
    const Tensor x = in_memory(x_), weight = in_memory(weight_), bias = in_memory(bias_);
    operand("x", x);
    if (x.dim() < 1) refuse("layer_norm takes a tensor of at least one dimension");
    if (x.size(-1) == 0) refuse("layer_norm: rows of length 0");
    if (x.size(-1) > (1 << 30)) refuse("layer_norm: rows of more than 2^30 elements");
    const Tensor* both[2] = {&weight, &bias};
    for (int i = 0; i < 2; ++i) {
        operand(i ? "bias" : "weight", *both[i], &x);
        if (both[i]->dim() != 1 || both[i]->size(0) != x.size(-1)) refuse(i ? "bias" : "weight", " has shape ", both[i]->sizes(), ", expected [", x.size(-1), "]");
    }
    if (!(eps >= 0.0) || !std::isfinite(eps)) refuse("layer_norm: eps ", eps);
    const Tensor w = weight.contiguous(), b = bias.contiguous();
    if (at::GradMode::is_enabled() && (wants(x) || wants(w) || wants(b))) {
        capturable({&x, &weight, &bias}, On(x));
        return LayerNorm::apply(x, w, b, eps);
    }
    return layer_norm_run(x, w, b, eps).first;
}

}  // namespace

PYBIND11_MODULE(_atlas_train, m) {
    static py::object error;                     // atlas_amd._lib.AtlasHipError, handed over by bind
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const Refusal& e) {
            PyErr_SetString(error ? error.ptr() : PyExc_RuntimeError, e.what());
        }
    });
    m.def("bind", [](const std::string& path, py::object error_class) { error = std::move(error_class); error.inc_ref(); bind(path); });
    typedef py::call_guard<py::gil_scoped_release> free_gil;
    m.def("attention", &attention, free_gil());
    m.def("compress", &compress, free_gil());
    m.def("decompress", [](const Tensor& c, const Tensor& s, std::vector<int64_t> shape, py::object dtype) {
        const auto t = torch::python::detail::py_object_to_dtype(std::move(dtype));
        py::gil_scoped_release r;
        return decompress(c, s, std::move(shape), t);
    });
    m.def("linear", &linear, free_gil());
    m.def("layer_norm", &layer_norm, free_gil());
}
