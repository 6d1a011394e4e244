// The gated scan and the 8-bit checkpoints for torch's dispatcher (torch.ops.sad_amd.*), with their autograd nodes.
//
// functional.py checks the arguments and calls these; they allocate, fill the argument structs and launch through libsad's
// C-ABI.  They are here and not in Python because the calls are short: a backward pass runs on autograd's device thread, where
// a Python node first has to take the interpreter lock from the thread that waits for it (a training call at [64, 23, 512]
// took 115 us with Python nodes; it takes 37 us in some processes and 60 in others, as fast as that thread wakes).
//
// The library's functions are handed in as addresses (sad_amd::bind), so this file does not link libsad and follows whichever
// build of it the package loaded.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include <cstring>
#include <dlfcn.h>

#include "../../include/sad.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

struct Api {
    decltype(&sad_last_error) last_error = nullptr;
    decltype(&sad_gated_scan_workspace_bytes) scan_ws = nullptr;
    decltype(&sad_gated_scan_kept_bytes) scan_kept = nullptr;
    decltype(&sad_gated_scan_codes_bytes) scan_codes = nullptr;
    decltype(&sad_gated_scan_fwd) scan_fwd = nullptr;
    decltype(&sad_gated_scan_bwd) scan_bwd = nullptr;
    decltype(&sad_gated_scan_step) scan_step = nullptr;
    decltype(&sad_checkpoint8_bytes) ckpt_bytes = nullptr;
    decltype(&sad_checkpoint8_save) ckpt_save = nullptr;
    decltype(&sad_checkpoint8_restore) ckpt_restore = nullptr;
    decltype(&sad_weight_grad8_workspace_bytes) wgrad_ws = nullptr;
    decltype(&sad_weight_grad8) wgrad = nullptr;
} api;

// Addresses in the order of Api's members.  The operator is public and its arguments are numbers: each has to be where a
// loaded library exports the function of that name.
void bind(at::IntArrayRef a) {
    TORCH_CHECK(a.size() == 12, "expected 12 addresses");
    auto look = [&](int i, const char* name) {
        Dl_info info{};
        void* p = reinterpret_cast<void*>(a[i]);
        TORCH_CHECK(dladdr(p, &info) != 0 && info.dli_saddr == p && info.dli_sname != nullptr && std::strcmp(info.dli_sname, name) == 0,
                    "address ", i, " is not ", name);
        return p;
    };
    Api next;
    int i = 0;
#define SAD_TAKE(member, name) next.member = reinterpret_cast<decltype(next.member)>(look(i++, #name))
    SAD_TAKE(last_error, sad_last_error);
    SAD_TAKE(scan_ws, sad_gated_scan_workspace_bytes);
    SAD_TAKE(scan_kept, sad_gated_scan_kept_bytes);
    SAD_TAKE(scan_codes, sad_gated_scan_codes_bytes);
    SAD_TAKE(scan_fwd, sad_gated_scan_fwd);
    SAD_TAKE(scan_bwd, sad_gated_scan_bwd);
    SAD_TAKE(scan_step, sad_gated_scan_step);
    SAD_TAKE(ckpt_bytes, sad_checkpoint8_bytes);
    SAD_TAKE(ckpt_save, sad_checkpoint8_save);
    SAD_TAKE(ckpt_restore, sad_checkpoint8_restore);
    SAD_TAKE(wgrad_ws, sad_weight_grad8_workspace_bytes);
    SAD_TAKE(wgrad, sad_weight_grad8);
#undef SAD_TAKE
    api = next;
}

void need_bound() { TORCH_CHECK(api.last_error != nullptr, "torch.ops.sad_amd is not bound to libsad: use sad_amd.functional"); }
void check(int rc, const char* what) { TORCH_CHECK(rc == 0, "libsad ", what, " failed (", rc, "): ", api.last_error()); }
size_t size_of(size_t n, const char* what) {
    TORCH_CHECK(n != 0, "libsad ", what, " failed: ", api.last_error());
    return n;
}
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
Tensor bytes(size_t n, const Tensor& like) { return at::empty({(int64_t)n}, like.options().dtype(at::kByte)); }
int kind_of(at::ScalarType t) {
    TORCH_CHECK(t == at::kFloat || t == at::kBFloat16 || t == at::kHalf, "expected float32, bfloat16 or float16, got ", t);
    return t == at::kFloat ? SAD_SRC_F32 : (t == at::kBFloat16 ? SAD_SRC_BF16 : SAD_SRC_F16);
}
template <class T> T* ptr(const Tensor& t) { return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr; }

// autograd.Function's once_differentiable: with create_graph the results raise when they are differentiated again
variable_list once(variable_list grads, const char* name) {
    if (!at::GradMode::is_enabled()) return grads;
    auto fn = std::make_shared<torch::autograd::DelayedError>(std::string(name) + " has no second derivative", (int64_t)grads.size());
    for (auto& g : grads)
        if (g.defined()) { g = g.detach(); g.requires_grad_(true); }
    return (*fn)(std::move(grads));
}

// The kernels follow data pointers: every tensor has to have memory on the device.  Fake and meta tensors (tracing) and the
// wrappers of function transforms have none.
void need_memory(const Tensor& t, const char* name, const char* what) {
    need_bound();
    TORCH_CHECK(t.has_storage() && t.storage().device_type() != at::kMeta, name, ": ", what,
                " has no memory (a meta or fake tensor, or the wrapper of a function transform); the operator cannot be traced");
    TORCH_CHECK(t.is_cuda(), name, ": ", what, " must be on the HIP device, got ", t.device(), "; there is no CPU path");
}
void need_matrix(const Tensor& t, const char* name, const char* what, at::ScalarType type, int64_t rows, int64_t cols, at::Device device) {
    need_memory(t, name, what);
    TORCH_CHECK(t.scalar_type() == type && t.dim() == 2 && t.size(0) == rows && t.size(1) == cols && t.stride(1) == 1 && t.device() == device,
                name, ": ", what, " must be ", type, " [", rows, ",", cols, "] with unit channel stride on ", device);
}
void need_vector(const Tensor& t, const char* name, const char* what, int64_t n, at::Device device) {
    need_memory(t, name, what);
    TORCH_CHECK(t.dim() == 1 && t.size(0) == n && t.device() == device, name, ": ", what, " must hold ", n, " entries on ", device);
}
int64_t channels_of(const Tensor& z, const char* name, int64_t dim, bool gated) {
    need_memory(z, name, "z");
    const int64_t parts = gated ? 3 : 2;
    TORCH_CHECK(z.dim() == dim && z.size(-1) % parts == 0 && z.size(-1) >= 2 * parts, name, ": z must hold ", parts, " parts of two channels or more, got ",
                z.sizes());
    return z.size(-1) / parts;
}

bool dual(const Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }
// the kernels write no tangents: a dual tensor's derivative would count as zero
void no_tangent(const char* name, const Tensor& a, const Tensor& b, const Tensor& c = Tensor()) {
    TORCH_CHECK(!dual(a) && !dual(b) && !dual(c), name, " has no forward-mode derivative");
}

// sizes go into 32-bit fields
int dim32(int64_t n) {
    TORCH_CHECK(n <= INT32_MAX, "a size of ", n, " is beyond the supported maximum");
    return (int)n;
}

// ---- gated scan -------------------------------------------------------------------------------------------------------
struct ScanShape {
    int64_t B, T, D, ws, kept, codes;
};
ScanShape scan_shape(const Tensor& z, bool gated) {
    ScanShape s;
    s.B = z.size(0); s.T = z.size(1); s.D = z.size(2) / (gated ? 3 : 2);
    const int B = dim32(s.B), T = dim32(s.T), D = dim32(s.D);
    s.ws = (int64_t)size_of(api.scan_ws(B, T, D), "sad_gated_scan_workspace_bytes");
    s.kept = ((int64_t)api.scan_kept(B, T, D) + 15) / 16 * 16;
    s.codes = (int64_t)api.scan_codes(B, T, D, gated);
    return s;
}

// (y, h_last, kept states and behind them the codes)
std::tuple<Tensor, Tensor, Tensor> scan_forward(const Tensor& z, const Tensor& h0, const Tensor& lengths, bool reverse, bool gated,
                                                bool int8, bool track) {
    const c10::DeviceGuard guard(z.device());
    const ScanShape s = scan_shape(z, gated);
    Tensor y;
    // in z's order, and no view: the results of an autograd node may then be modified in place
    if (s.B > 1 && s.T > 1 && z.stride(0) < z.stride(1)) y = at::empty_strided({s.B, s.T, s.D}, {s.D, s.B * s.D, 1}, z.options());
    else y = at::empty({s.B, s.T, s.D}, z.options());
    Tensor h_last = at::empty({s.B, s.D}, z.options().dtype(at::kFloat)), kept;
    if (track) kept = bytes(s.kept + (int8 ? s.codes : 0), z);
    const Tensor ws = s.ws > 16 ? bytes(s.ws, z) : h_last;      // any address where none is needed
    sad_scan_args a{};
    a.B = (int)s.B; a.T = (int)s.T; a.D = (int)s.D;
    a.kind = kind_of(z.scalar_type()); a.gated = gated; a.reverse = reverse;
    a.z = z.data_ptr(); a.z_stride_b = z.stride(0); a.z_stride_t = z.stride(1);
    a.lengths = ptr<int32_t>(lengths);
    a.h0 = ptr<float>(h0);
    a.y = y.data_ptr(); a.y_stride_b = y.stride(0); a.y_stride_t = y.stride(1);
    a.h_last = ptr<float>(h_last);
    if (track) {
        a.kept = ptr<float>(kept);
        if (int8) a.codes = ptr<char>(kept) + s.kept;
    }
    check(api.scan_fwd(&a, ws.data_ptr(), stream_of(z)), "sad_gated_scan_fwd");
    return {y, h_last, kept};
}

bool is_dense(at::IntArrayRef size, at::IntArrayRef stride) {      // a permutation of a contiguous [.., .., C]
    if (stride[2] != 1) return false;
    const int a = stride[0] < stride[1] ? 0 : 1, b = 1 - a;
    return (size[a] == 1 || stride[a] == size[2]) && (size[b] == 1 || stride[b] == size[2] * size[a]);
}

struct GatedScan : torch::autograd::Function<GatedScan> {
    static variable_list forward(AutogradContext* ctx, const Tensor& z, const OptTensor& h0, const OptTensor& lengths, bool reverse,
                                 bool gated, bool int8) {
        const Tensor l = lengths.value_or(Tensor());
        auto [y, h_last, kept] = scan_forward(z, h0.value_or(Tensor()), l, reverse, gated, int8, true);
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({int8 ? Tensor() : z, l, kept});
        ctx->saved_data["s"] = std::vector<int64_t>{z.size(0), z.size(1), z.size(2), z.stride(0), z.stride(1), z.stride(2),
                                                    (int64_t)z.scalar_type(), reverse, gated, h0.has_value(), kept.numel()};
        return {y, h_last};
    }
    static variable_list backward(AutogradContext* ctx, variable_list gout) {
        Tensor dy = gout[0], dh = gout[1];
        if (!dy.defined() && !dh.defined()) return variable_list(6);
        const auto saved = ctx->get_saved_variables();
        const auto v = ctx->saved_data["s"].toIntVector();
        const bool reverse = v[7] != 0, gated = v[8] != 0;
        const at::IntArrayRef size(v.data(), 3), stride(v.data() + 3, 3);
        // Saved tensors pass through the hooks of the program (save_on_cpu), which keep values and not layouts: what comes
        // back is read by its own strides.
        Tensor z = saved[0], lengths = saved[1], kept = saved[2];
        if (z.defined() && z.stride(2) != 1) z = z.contiguous();
        if (lengths.defined()) lengths = lengths.contiguous();
        kept = kept.contiguous();
        if ((size_t)kept.data_ptr() % 16) kept = kept.clone();
        TORCH_CHECK(!z.defined() || (z.sizes() == size && z.scalar_type() == (at::ScalarType)v[6] && z.device() == kept.device()),
                    "gated_scan: the saved z came back as another tensor");
        TORCH_CHECK(kept.is_cuda() && kept.scalar_type() == at::kByte && kept.numel() == v[10], "gated_scan: the kept states came back as another tensor");
        TORCH_CHECK(!lengths.defined() || (lengths.scalar_type() == at::kInt && lengths.numel() == size[0] && lengths.device() == kept.device()),
                    "gated_scan: the lengths came back as another tensor");
        const c10::DeviceGuard guard(kept.device());
        const auto options = kept.options().dtype((at::ScalarType)v[6]);
        // in z's order: its strides, or those of its axes without the gaps
        Tensor dz, dh0;
        if (is_dense(size, stride)) dz = at::empty_strided(size, stride, options);
        else if (size[0] > 1 && size[1] > 1 && stride[0] < stride[1]) dz = at::empty_strided(size, {size[2], size[0] * size[2], 1}, options);
        else dz = at::empty(size, options);
        const ScanShape s = scan_shape(dz, gated);
        if (dy.defined() && dy.stride(2) != 1) dy = dy.contiguous();
        if (dh.defined()) dh = dh.contiguous();
        if (v[9] && ctx->needs_input_grad(1)) dh0 = at::empty({s.B, s.D}, options.dtype(at::kFloat));
        const Tensor ws = s.ws > 16 ? bytes(s.ws, kept) : dz;
        sad_scan_args a{};
        a.B = (int)s.B; a.T = (int)s.T; a.D = (int)s.D;
        a.kind = kind_of(dz.scalar_type()); a.gated = gated; a.reverse = reverse;
        a.lengths = ptr<int32_t>(lengths);
        a.kept = ptr<float>(kept);
        if (z.defined()) { a.z = z.data_ptr(); a.z_stride_b = z.stride(0); a.z_stride_t = z.stride(1); }
        else a.codes = ptr<char>(kept) + s.kept;
        if (dy.defined()) { a.dy = dy.data_ptr(); a.dy_stride_b = dy.stride(0); a.dy_stride_t = dy.stride(1); }
        a.dh_last = ptr<float>(dh);
        a.dz = dz.data_ptr(); a.dz_stride_b = dz.stride(0); a.dz_stride_t = dz.stride(1);
        a.dh0 = ptr<float>(dh0);
        check(api.scan_bwd(&a, ws.data_ptr(), stream_of(kept)), "sad_gated_scan_bwd");
        if (!ctx->needs_input_grad(0)) dz = Tensor();
        return once({dz, dh0, Tensor(), Tensor(), Tensor(), Tensor()}, "gated_scan");
    }
};

std::tuple<Tensor, Tensor> gated_scan(const Tensor& z, const OptTensor& h0, const OptTensor& lengths, bool reverse, bool gated, bool int8) {
    no_tangent("gated_scan", z, h0.value_or(Tensor()));
    const int64_t D = channels_of(z, "gated_scan", 3, gated);
    TORCH_CHECK(z.stride(2) == 1, "gated_scan: z must have unit channel stride");
    if (h0.has_value()) {
        need_matrix(*h0, "gated_scan", "h0", at::kFloat, z.size(0), D, z.device());
        TORCH_CHECK(h0->is_contiguous(), "gated_scan: h0 must be contiguous");
    }
    if (lengths.has_value()) {
        need_vector(*lengths, "gated_scan", "lengths", z.size(0), z.device());
        TORCH_CHECK(lengths->scalar_type() == at::kInt && lengths->is_contiguous(), "gated_scan: lengths must be contiguous int32");
    }
    if (at::GradMode::is_enabled() && (z.requires_grad() || (h0.has_value() && h0->requires_grad()))) {
        auto r = GatedScan::apply(z, h0, lengths, reverse, gated, int8);
        return {r[0], r[1]};
    }
    auto [y, h_last, kept] = scan_forward(z, h0.value_or(Tensor()), lengths.value_or(Tensor()), reverse, gated, false, false);
    return {y, h_last};
}

// do the address ranges of two non-empty matrices meet
bool overlap(const Tensor& a, const Tensor& b) {
    const auto end = [](const Tensor& t) {
        return (const char*)t.data_ptr() + ((t.size(0) - 1) * t.stride(0) + (t.size(1) - 1) * t.stride(1) + 1) * (int64_t)t.element_size();
    };
    return (const char*)a.data_ptr() < end(b) && (const char*)b.data_ptr() < end(a);
}

// y; the new states go to h_out (h itself updates in place)
Tensor gated_scan_step(const Tensor& z, const Tensor& h, const OptTensor& alive, bool gated, const Tensor& h_out) {
    no_tangent("gated_scan_step", z, h, h_out);
    const int64_t D = channels_of(z, "gated_scan_step", 2, gated);
    need_matrix(h, "gated_scan_step", "h", at::kFloat, z.size(0), D, z.device());
    need_matrix(h_out, "gated_scan_step", "h_out", at::kFloat, z.size(0), D, z.device());
    // lanes read h and z while others write h_out
    TORCH_CHECK(h_out.size(0) < 2 || h_out.stride(0) >= D, "gated_scan_step: rows of h_out overlap");
    if (h.size(0) > 0) {
        const bool same = h_out.data_ptr() == h.data_ptr() && h_out.strides() == h.strides();
        TORCH_CHECK(same || !overlap(h_out, h), "gated_scan_step: h_out must be h itself or must not overlap it");
        TORCH_CHECK(!overlap(h_out, z), "gated_scan_step: h_out must not overlap z");
    }
    if (alive.has_value()) {
        need_vector(*alive, "gated_scan_step", "alive", z.size(0), z.device());
        TORCH_CHECK(alive->scalar_type() == at::kBool || alive->scalar_type() == at::kByte, "gated_scan_step: alive must be bool");
    }
    const c10::DeviceGuard guard(z.device());
    Tensor y = at::empty({h.size(0), h.size(1)}, z.options());
    if (h.size(0) == 0) return y;
    const Tensor zc = z.stride(1) == 1 ? z : z.contiguous(), ac = alive.has_value() ? alive->contiguous() : Tensor();
    check(api.scan_step(dim32(h.size(0)), dim32(h.size(1)), kind_of(z.scalar_type()), gated, zc.data_ptr(), zc.stride(0), ptr<float>(h),
                        h.stride(0), ptr<uint8_t>(ac), y.data_ptr(), y.stride(0), ptr<float>(h_out), h_out.stride(0), stream_of(z)),
          "sad_gated_scan_step");
    if (!h_out.is_inference()) h_out.unsafeGetTensorImpl()->bump_version();
    return y;
}

// ---- checkpoints, linear8 ------------------------------------------------------------------------------------------------------------
struct Rows {
    Tensor t;      // holds the memory
    int64_t n0, n1, s0, s1, C;
};
// the rows of t [..., C] in their order, without a copy where two strides say it
Rows rows_of(Tensor t) {
    if (t.dim() == 1) t = t.unsqueeze(0);
    if (t.stride(-1) != 1 && t.size(-1) != 1) t = t.contiguous();
    if (t.dim() > 3) t = t.flatten(0, -2);
    if (t.dim() == 2) return {t, 1, t.size(0), 0, t.stride(0), t.size(1)};
    return {t, t.size(0), t.size(1), t.stride(0), t.stride(1), t.size(2)};
}

// 8-bit checkpoint of x [..., C]
Tensor checkpoint8(const Tensor& x) {
    TORCH_CHECK(x.dim() > 0, "checkpoint8: x must have a channel axis");
    need_memory(x, "checkpoint8", "x");
    const c10::DeviceGuard guard(x.device());
    if (x.numel() == 0) return bytes(0, x);
    const Rows r = rows_of(x.detach());
    Tensor saved = bytes(size_of(api.ckpt_bytes(r.n0 * r.n1, r.C), "sad_checkpoint8_bytes"), x);
    check(api.ckpt_save(r.n0, r.n1, r.C, kind_of(x.scalar_type()), r.t.data_ptr(), r.s0, r.s1, saved.data_ptr(), stream_of(x)),
          "sad_checkpoint8_save");
    return saved;
}

// `saved` is the caller's to move, copy and slice: it has to be a whole checkpoint of rows x C entries, on the device
void need_saved(const Tensor& saved, int64_t rows, int64_t C) {
    need_bound();
    TORCH_CHECK(saved.scalar_type() == at::kByte && saved.is_contiguous(), "a checkpoint's codes are contiguous uint8, got ", saved.scalar_type(),
                saved.is_contiguous() ? "" : " (not contiguous)");
    const size_t n = rows > 0 && C > 0 ? size_of(api.ckpt_bytes(rows, C), "sad_checkpoint8_bytes") : 0;
    TORCH_CHECK((size_t)saved.numel() == n, "a checkpoint of ", rows, " x ", C, " entries holds ", n, " bytes, got ", saved.numel());
    need_memory(saved, "a checkpoint", "saved");
}

// the values a checkpoint stands for, contiguous
Tensor restore8(const Tensor& saved, at::IntArrayRef size, at::ScalarType dtype) {
    TORCH_CHECK(!size.empty(), "a checkpoint has a channel axis");
    const int64_t n = c10::multiply_integers(size), rows = n > 0 ? n / size.back() : 0;
    need_saved(saved, rows, size.back());
    const c10::DeviceGuard guard(saved.device());
    Tensor out = at::empty(size, saved.options().dtype(dtype));
    if (n == 0) return out;
    check(api.ckpt_restore(rows, size.back(), kind_of(dtype), saved.data_ptr(), out.data_ptr(), stream_of(saved)),
          "sad_checkpoint8_restore");
    return out;
}

// (dW [N,K], db [N] or an empty tensor)
std::tuple<Tensor, Tensor> weight_grad8(const Tensor& dy, const Tensor& saved, int64_t K, bool bias) {
    TORCH_CHECK(dy.dim() > 0, "dy must have a channel axis");
    const int64_t rows = c10::multiply_integers(dy.sizes().slice(0, dy.dim() - 1));
    need_saved(saved, rows, K);
    need_memory(dy, "weight_grad8", "dy");
    TORCH_CHECK(saved.device() == dy.device(), "dy is on ", dy.device(), ", the checkpoint on ", saved.device());
    const c10::DeviceGuard guard(dy.device());
    if (dy.numel() == 0 || K == 0) {
        const auto options = dy.options().dtype(at::kFloat);
        const Tensor dw = at::zeros({dy.size(-1), K}, options);
        if (!bias) return {dw, at::empty({0}, options)};
        return {dw, dy.numel() == 0 ? at::zeros({dy.size(-1)}, options) : dy.detach().to(at::kFloat).reshape({-1, dy.size(-1)}).sum(0)};
    }
    const Rows r = rows_of(dy.detach());
    const int kind = kind_of(dy.scalar_type());
    Tensor dw = at::empty({r.C, K}, dy.options().dtype(at::kFloat)), db = at::empty({bias ? r.C : 0}, dw.options());
    const Tensor ws = bytes(size_of(api.wgrad_ws(r.n0 * r.n1, r.C, K, kind), "sad_weight_grad8_workspace_bytes"), dy);
    check(api.wgrad(r.n0, r.n1, r.C, K, kind, r.t.data_ptr(), r.s0, r.s1, saved.data_ptr(), ptr<float>(dw), bias ? ptr<float>(db) : nullptr, ws.data_ptr(),
                    stream_of(dy)),
          "sad_weight_grad8");
    return {dw, db};
}

// x w^T + b for x [..., K].  A time-major activation seen as [B,T,K] is multiplied as its rows lie in memory, and y comes
// back in the same order.
Tensor linear_rows(const Tensor& x, const Tensor& w, const OptTensor& b) {
    const c10::impl::ExcludeDispatchKeyGuard no_autocast(c10::autocast_dispatch_keyset);      // x's type is the caller's choice
    const bool swap = x.dim() == 3 && !x.is_contiguous() && x.transpose(0, 1).is_contiguous();
    const Tensor xt = swap ? x.transpose(0, 1) : x;
    auto lead = xt.sizes().vec();
    const int64_t rows = c10::multiply_integers(lead.begin(), lead.end() - 1);      // x may have no channels
    const Tensor y = at::linear(xt.reshape({rows, x.size(-1)}), w, b);
    lead.back() = w.size(0);
    return swap ? y.view(lead).transpose(0, 1) : y.view(lead);
}

// The same where no derivative is taken through it: its result is no view for autograd, so that it may be modified in place
// (views made inside an autograd node or under no_grad may not).
Tensor linear_rows_fresh(const Tensor& x, const Tensor& w, const OptTensor& b) {
    const at::AutoDispatchBelowADInplaceOrView guard;
    return linear_rows(x, w, b);
}

struct Linear8 : torch::autograd::Function<Linear8> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const OptTensor& bias) {
        const Tensor w = weight.to(x.scalar_type());
        OptTensor b;
        if (bias.has_value()) b = bias->to(x.scalar_type());
        Tensor y = linear_rows_fresh(x, w, b), saved;
        const bool keep = weight.requires_grad() || (bias.has_value() && bias->requires_grad());
        if (keep) saved = checkpoint8(x);
        ctx->save_for_backward({x.requires_grad() ? w : Tensor(), saved});
        ctx->saved_data["s"] = std::vector<int64_t>{keep, bias.has_value(), weight.size(1), (int64_t)weight.scalar_type(),
                                                    bias.has_value() ? (int64_t)bias->scalar_type() : 0};
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list gout) {
        const Tensor& dy = gout[0];
        const auto saved = ctx->get_saved_variables();
        const auto v = ctx->saved_data["s"].toIntVector();
        Tensor dx, dw, db;
        {
            at::AutoGradMode no_grad(false);
            if (ctx->needs_input_grad(0)) dx = linear_rows(dy, saved[0].t(), std::nullopt);
            if (v[0]) {
                std::tie(dw, db) = weight_grad8(dy, saved[1], v[2], v[1] != 0);
                dw = ctx->needs_input_grad(1) ? dw.to((at::ScalarType)v[3]) : Tensor();
                db = v[1] && ctx->needs_input_grad(2) ? db.to((at::ScalarType)v[4]) : Tensor();
            }
        }
        return once({dx, dw, db}, "linear8");
    }
};

Tensor linear8(const Tensor& x, const Tensor& weight, const OptTensor& bias) {
    need_memory(x, "linear8", "x");
    need_memory(weight, "linear8", "weight");
    TORCH_CHECK(x.dim() > 0 && weight.dim() == 2 && x.size(-1) == weight.size(1) && weight.device() == x.device(), "linear8: x ", x.sizes(),
                " and weight ", weight.sizes(), " do not fit");
    if (bias.has_value()) need_vector(*bias, "linear8", "bias", weight.size(0), x.device());
    if (at::GradMode::is_enabled() && (x.requires_grad() || weight.requires_grad() || (bias.has_value() && bias->requires_grad())))
        return Linear8::apply(x, weight, bias);
    OptTensor b;
    if (bias.has_value()) b = bias->to(x.scalar_type());
    const Tensor w = weight.to(x.scalar_type());
    if (dual(x) || dual(w) || dual(b.value_or(Tensor()))) return linear_rows(x, w, b);      // forward-mode derivative
    return linear_rows_fresh(x, w, b);
}

}  // namespace

TORCH_LIBRARY(sad_amd, m) {
    m.def("bind(int[] addresses) -> ()", &bind);
    m.def("gated_scan(Tensor z, Tensor? h0, Tensor? lengths, bool reverse, bool gated, bool int8) -> (Tensor, Tensor)", &gated_scan);
    m.def("gated_scan_step(Tensor z, Tensor h, Tensor? alive, bool gated, Tensor(a!) h_out) -> Tensor", &gated_scan_step);
    m.def("checkpoint8(Tensor x) -> Tensor", &checkpoint8);
    m.def("restore8(Tensor saved, int[] size, ScalarType dtype) -> Tensor", &restore8);
    m.def("weight_grad8(Tensor dy, Tensor saved, int K, bool bias) -> (Tensor, Tensor)", &weight_grad8);
    m.def("linear8(Tensor x, Tensor weight, Tensor? bias) -> Tensor", &linear8);
}
