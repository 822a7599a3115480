// Host side of the two hottest wrappers in C++: a Python call of the fused RMSNorm+quant or
// SwiGLU+quant wrapper costs about 20 us when the output tensors are allocated from Python
// (three torch.empty calls, a ctypes marshal), more than the 12 us the kernel takes at the small
// benchmark shapes.  The same steps from C++ -- allocate through ATen, take the current stream,
// call the C ABI of include/linghe_b200.h -- cost a few microseconds.  Nothing here computes:
// this is the argument handling of linghe_b200/utils/norm.py and utils/silu.py, restated, in
// front of the same two entry points, with the same return contract as the upstream wrappers
// (linghe/utils/norm.py:343-502, linghe/utils/silu.py:279-335).
#include <torch/extension.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <cstdint>
#include <initializer_list>
#include <optional>
#include <string>
#include <tuple>
#include <utility>
#include <vector>

#include "linghe_b200.h"

namespace {

using OptT = std::optional<at::Tensor>;

[[noreturn]] void raise_assert(const std::string& msg) {
    PyErr_SetString(PyExc_AssertionError, msg.c_str());
    throw py::error_already_set();
}

int dtype_code(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kBFloat16: return LH_BF16;
        case at::kHalf: return LH_F16;
        case at::kFloat: return LH_F32;
        default: raise_assert("unsupported dtype");
    }
}

// argument errors are AssertionError (the upstream wrappers use bare asserts), CUDA errors RuntimeError
void check_rc(int rc, const char* name) {
    if (rc == LH_OK) return;
    const std::string msg = lh_last_error();
    if (rc == LH_ERR_ARG) raise_assert(msg);
    throw std::runtime_error(std::string("linghe_b200 ") + name + ": CUDA error " + std::to_string(rc) + ": " + msg);
}

void check_device(const at::Tensor& x) {
    if (!x.is_cuda()) throw std::runtime_error("linghe_b200 runs on CUDA tensors only (no CPU fallback)");
    static bool checked[64] = {};
    const int idx = x.get_device();
    if (idx >= 0 && idx < 64 && !checked[idx]) {
        if (lh_device_check(idx) != LH_OK) throw std::runtime_error(std::string("linghe_b200: ") + lh_last_error());
        checked[idx] = true;
    }
}

void* ptr(const OptT& t) { return t.has_value() ? t->data_ptr() : nullptr; }

// (out, scale, rms, transpose_output, transpose_scale); entries a mode does not produce and the
// caller did not pass are None, except the transposed pair, which upstream always allocates
std::tuple<OptT, OptT, at::Tensor, at::Tensor, at::Tensor> rms_norm_and_block_quant_forward(
    const at::Tensor& x, const at::Tensor& weight, double eps, OptT out, OptT scale, OptT rms, bool round_scale,
    int64_t output_mode) {
    if (!x.is_contiguous() || !weight.is_contiguous()) raise_assert("x and weight must be contiguous");
    if (x.dim() != 2) raise_assert("x must be 2-D");
    const int64_t M = x.size(0), n = x.size(1);
    if (n > 8192) raise_assert("n <= 8192");
    if (output_mode < 0 || output_mode > 2) raise_assert("output_mode in (0, 1, 2)");
    if (output_mode == 0 && rms.has_value()) raise_assert("rms must be None in output_mode 0");
    if (output_mode == 1 && !rms.has_value()) raise_assert("rms is required in output_mode 1");
    check_device(x);
    const c10::cuda::OptionalCUDAGuard guard(x.device());
    const auto fp8 = x.options().dtype(at::kFloat8_e4m3fn);
    const auto f32 = x.options().dtype(at::kFloat);
    if (output_mode != 1) {
        if (!out.has_value()) out = at::empty({M, n}, fp8);
        if (!scale.has_value()) scale = at::empty({n / 128, M}, f32);
    }
    at::Tensor tq, ts;
    if (output_mode != 0) {
        tq = at::empty({n, M}, fp8);
        ts = at::empty({(M + 127) / 128, n}, f32);
    }
    if (output_mode != 1) rms = at::empty({M}, f32);
    const int rc = lh_rmsnorm_blockquant_fwd(x.data_ptr(), weight.data_ptr(), dtype_code(x), M, n, float(eps),
                                             output_mode != 1 ? ptr(out) : nullptr,
                                             output_mode != 1 ? static_cast<float*>(ptr(scale)) : nullptr,
                                             static_cast<float*>(ptr(rms)), tq.defined() ? tq.data_ptr() : nullptr,
                                             ts.defined() ? static_cast<float*>(ts.data_ptr()) : nullptr, round_scale ? 1 : 0,
                                             int(output_mode), c10::cuda::getCurrentCUDAStream().stream());
    check_rc(rc, "lh_rmsnorm_blockquant_fwd");
    if (!tq.defined()) {   // not written in mode 0: allocated behind the launch, where it delays nothing
        tq = at::empty({n, M}, fp8);
        ts = at::empty({(M + 127) / 128, n}, f32);
    }
    return {out, scale, *rms, tq, ts};
}

// (out, scale, transpose_output, transpose_scale)
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> silu_and_block_quant_forward(const at::Tensor& x, OptT out,
                                                                                        OptT scale, bool round_scale,
                                                                                        int64_t output_mode) {
    if (!x.is_contiguous()) raise_assert("x must be contiguous");
    if (x.dim() != 2) raise_assert("x must be 2-D");
    const int64_t M = x.size(0), n = x.size(1) / 2;
    // upstream tiles the width by 128 columns, by 64 when only the transposed pair is written
    if (n % (output_mode == 1 ? 64 : 128) != 0) raise_assert("n % 128 == 0 (n % 64 == 0 in output_mode 1)");
    check_device(x);
    const c10::cuda::OptionalCUDAGuard guard(x.device());
    const auto fp8 = x.options().dtype(at::kFloat8_e4m3fn);
    const auto f32 = x.options().dtype(at::kFloat);
    if (!out.has_value()) out = at::empty({M, n}, fp8);
    if (!scale.has_value()) scale = at::empty({n / 128, M}, f32);
    at::Tensor tq, ts;
    if (output_mode != 0) {
        tq = at::empty({n, M}, fp8);
        ts = at::empty({(M + 127) / 128, n}, f32);
    }
    const int rc = lh_silu_blockquant_fwd(x.data_ptr(), dtype_code(x), M, n, out->data_ptr(),
                                          static_cast<float*>(scale->data_ptr()), tq.defined() ? tq.data_ptr() : nullptr,
                                          ts.defined() ? static_cast<float*>(ts.data_ptr()) : nullptr, round_scale ? 1 : 0,
                                          int(output_mode), c10::cuda::getCurrentCUDAStream().stream());
    check_rc(rc, "lh_silu_blockquant_fwd");
    if (!tq.defined()) {
        tq = at::empty({n, M}, fp8);
        ts = at::empty({(M + 127) / 128, n}, f32);
    }
    return {*out, *scale, tq, ts};
}

// Several uninitialised tensors on the device of `ref` from one call: specs = [(shape, code), ...]
// with code 0 e4m3, 1 float32, 2 bfloat16, 3 float16, 4 uint8, 5 int32, 6 int64, 7 int8.  One
// Python -> C++ transition instead of one per torch.empty.
std::vector<at::Tensor> empty_many(const at::Tensor& ref, const std::vector<std::pair<std::vector<int64_t>, int>>& specs) {
    static const at::ScalarType kinds[] = {at::kFloat8_e4m3fn, at::kFloat, at::kBFloat16, at::kHalf, at::kByte, at::kInt, at::kLong, at::kChar};
    if (!ref.is_cuda()) throw std::runtime_error("linghe_b200 runs on CUDA tensors only (no CPU fallback)");
    std::vector<at::Tensor> out;
    out.reserve(specs.size());
    const c10::cuda::OptionalCUDAGuard guard(ref.device());
    for (const auto& sp : specs) {
        if (sp.second < 0 || sp.second > 7) raise_assert("empty_many: unknown dtype code");
        out.push_back(at::empty(sp.first, ref.options().dtype(kinds[sp.second])));
    }
    return out;
}

uintptr_t current_stream(int device) { return reinterpret_cast<uintptr_t>(c10::cuda::getCurrentCUDAStream(device).stream()); }

// ---- the operators that keep activations in eight bits: the argument handling of utils/norm.py (rms_norm_pair_*),
// utils/silu.py (silu_and_checkpoint_*), quant/token.py and gemm/int8_gemm.py, restated ----

#define LH_NEED(cond, msg) \
    do { if (!(cond)) raise_assert(msg); } while (0)

// contiguous, on the device of `ref`, of `type` and `shape` (the checks of _lib.check_same)
void check_same(const at::Tensor& ref, at::ScalarType type, const char* name, const at::Tensor& t) {
    if (t.device() != ref.device()) raise_assert(std::string(name) + " is on " + t.device().str() + ", expected " + ref.device().str());
    if (t.scalar_type() != type) raise_assert(std::string(name) + " is " + c10::toString(t.scalar_type()) + ", expected " + c10::toString(type));
    if (!t.is_contiguous()) raise_assert(std::string(name) + " must be contiguous");
}
void check_same(const at::Tensor& ref, at::ScalarType type, const char* name, const at::Tensor& t, at::IntArrayRef shape) {
    check_same(ref, type, name, t);
    if (t.sizes() != shape) raise_assert(std::string(name) + " has another shape than expected");
}

// an uninitialised tensor on the device of `ref`, straight from the CUDA allocator (the dispatcher in front of at::empty costs
// as much as the allocation)
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& ref) {
    return at::detail::empty_cuda(sizes, type, ref.device(), std::nullopt);
}

const void* cptr(const OptT& t) { return t.has_value() ? t->data_ptr() : nullptr; }
float* fptr(const at::Tensor& t) { return static_cast<float*>(t.data_ptr()); }
const float* fptr(const OptT& t) { return t.has_value() ? static_cast<const float*>(t->data_ptr()) : nullptr; }

int checkpoint_code(const std::optional<at::ScalarType>& type) {
    if (!type.has_value()) return 0;
    if (*type == at::kChar) return 1;
    if (*type == at::kFloat8_e4m3fn) return 2;
    raise_assert("checkpoint must be torch.int8 or torch.float8_e4m3fn");
}

int64_t rows_cols(const at::Tensor& x, int64_t& n) {
    LH_NEED(x.dim() == 2 || x.dim() == 3, "x must be 2-D or 3-D");
    n = x.size(-1);
    return x.dim() == 3 ? x.size(0) * x.size(1) : x.size(0);
}

// rows of a gate whose shape is that of the last dimensions of x
int64_t gate_rows(const OptT& gate, const at::Tensor& x) {
    if (!gate.has_value()) return 0;
    at::IntArrayRef shape = gate->sizes();
    while (shape.size() > 1 && shape[0] == 1) shape = shape.slice(1);
    LH_NEED(!shape.empty() && int64_t(shape.size()) <= x.dim() && shape == x.sizes().slice(x.dim() - shape.size()),
            "gate must have the shape of the last dimensions of x");
    int64_t g = 1;
    for (size_t i = 0; i + 1 < shape.size(); ++i) g *= shape[i];
    return g;
}

using Saved = std::optional<std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor>>;

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, Saved> rms_norm_pair_forward(
    const at::Tensor& x, const at::Tensor& o, const at::Tensor& post, const at::Tensor& pre, const OptT& gate, double alpha, double eps,
    const std::optional<at::ScalarType>& checkpoint) {
    int64_t n = 0;
    const int64_t M = rows_cols(x, n);
    LH_NEED(n > 0 && n % 128 == 0 && n <= 8192, "need n % 128 == 0 and n <= 8192");
    const int codes = checkpoint_code(checkpoint), dt = dtype_code(x);
    check_device(x);
    const at::ScalarType type = x.scalar_type();
    check_same(x, type, "x", x);
    check_same(x, type, "o", o, x.sizes());
    check_same(x, type, "post_weight", post, {n});
    check_same(x, type, "pre_weight", pre, {n});
    if (gate.has_value()) check_same(x, type, "gate", *gate);
    const int64_t G = gate_rows(gate, x);
    const c10::cuda::OptionalCUDAGuard guard(x.device());
    const at::Tensor h = fresh(x.sizes(), x.scalar_type(), x), y = fresh(x.sizes(), x.scalar_type(), x), rp = fresh({M}, at::kFloat, x), rh = fresh({M}, at::kFloat, x);
    Saved saved;
    at::Tensor oq, os, hq, hs;
    if (codes) {
        oq = fresh(x.sizes(), *checkpoint, x); os = fresh({M, n / 128}, at::kFloat, x);
        hq = fresh(x.sizes(), *checkpoint, x); hs = fresh({M, n / 128}, at::kFloat, x);
        saved = std::make_tuple(oq, os, hq, hs);
    }
    check_rc(lh_rmsnorm_pair_fwd(x.data_ptr(), o.data_ptr(), post.data_ptr(), pre.data_ptr(), cptr(gate), dt, M, n, G, float(alpha), float(eps),
                                 codes, h.data_ptr(), y.data_ptr(), fptr(rp), fptr(rh), codes ? oq.data_ptr() : nullptr, codes ? fptr(os) : nullptr,
                                 codes ? hq.data_ptr() : nullptr, codes ? fptr(hs) : nullptr, c10::cuda::getCurrentCUDAStream().stream()),
             "lh_rmsnorm_pair_fwd");
    return {h, y, rp, rh, saved};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, OptT> rms_norm_pair_backward(
    const at::Tensor& dy, const OptT& dh, const at::Tensor& o, const at::Tensor& h, const at::Tensor& post, const at::Tensor& pre,
    const at::Tensor& rp, const at::Tensor& rh, const OptT& gate, double alpha, const OptT& os, const OptT& hs) {
    int64_t n = 0;
    const int64_t M = rows_cols(dy, n);
    LH_NEED(n > 0 && n % 128 == 0 && n <= 8192, "need n % 128 == 0 and n <= 8192");
    LH_NEED(os.has_value() == hs.has_value(), "o_scale and h_scale are given together");
    const int codes = os.has_value() ? checkpoint_code(o.scalar_type()) : 0, dt = dtype_code(dy);
    check_device(dy);
    const at::ScalarType type = dy.scalar_type(), kept = codes ? o.scalar_type() : type;
    check_same(dy, type, "grad_y", dy);
    if (dh.has_value()) check_same(dy, type, "grad_h", *dh, dy.sizes());
    check_same(dy, kept, "o", o, dy.sizes());
    check_same(dy, kept, "h", h, dy.sizes());
    if (codes) {
        check_same(dy, at::kFloat, "o_scale", *os, {M, n / 128});
        check_same(dy, at::kFloat, "h_scale", *hs, {M, n / 128});
    }
    check_same(dy, type, "post_weight", post, {n});
    check_same(dy, type, "pre_weight", pre, {n});
    check_same(dy, at::kFloat, "rms_post", rp, {M});
    check_same(dy, at::kFloat, "rms_pre", rh, {M});
    if (gate.has_value()) check_same(dy, type, "gate", *gate);
    const int64_t G = gate_rows(gate, dy);
    const c10::cuda::OptionalCUDAGuard guard(dy.device());
    const int64_t nbytes = lh_scratch_bytes("rmsnorm_pair_bwd", M, n);
    const at::Tensor dx = fresh(dy.sizes(), dy.scalar_type(), dy), dout = fresh(dy.sizes(), dy.scalar_type(), dy), dpost = fresh({n}, at::kFloat, dy),
                     dpre = fresh({n}, at::kFloat, dy), scratch = fresh({nbytes}, at::kByte, dy);
    OptT dgate;
    if (gate.has_value()) dgate = fresh(gate->sizes(), dy.scalar_type(), dy);
    check_rc(lh_rmsnorm_pair_bwd(dy.data_ptr(), cptr(dh), o.data_ptr(), fptr(os), h.data_ptr(), fptr(hs), post.data_ptr(), pre.data_ptr(),
                                 cptr(gate), fptr(rp), fptr(rh), dt, M, n, G, float(alpha), codes, dx.data_ptr(), dout.data_ptr(), fptr(dpost),
                                 fptr(dpre), ptr(dgate), scratch.data_ptr(), nbytes, c10::cuda::getCurrentCUDAStream().stream()),
             "lh_rmsnorm_pair_bwd");
    return {dx, dout, dpost, dpre, dgate};
}

int weight_code(const at::Tensor& ref, const OptT& w, int64_t M) {
    if (!w.has_value()) return LH_F32;
    check_same(ref, w->scalar_type(), "weight", *w, {M});
    return dtype_code(*w);
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> silu_and_checkpoint_forward(const at::Tensor& x, const OptT& w,
                                                                           const std::optional<at::ScalarType>& checkpoint) {
    LH_NEED(x.dim() == 2, "x must be 2-D");
    const int64_t M = x.size(0), N = x.size(1);
    LH_NEED(N > 0 && N % 256 == 0, "need N % 256 == 0");
    const int codes = checkpoint_code(checkpoint), dt = dtype_code(x);
    LH_NEED(codes != 0, "checkpoint must be torch.int8 or torch.float8_e4m3fn");
    check_device(x);
    check_same(x, x.scalar_type(), "x", x);
    const int wt = weight_code(x, w, M);
    const c10::cuda::OptionalCUDAGuard guard(x.device());
    const at::Tensor y = fresh({M, N / 2}, x.scalar_type(), x), q = fresh({M, N}, *checkpoint, x),
                     s = fresh({M, N / 128}, at::kFloat, x);
    check_rc(lh_silu_checkpoint_fwd(x.data_ptr(), cptr(w), dt, wt, codes, M, N / 2, y.data_ptr(), q.data_ptr(), fptr(s),
                                    c10::cuda::getCurrentCUDAStream().stream()),
             "lh_silu_checkpoint_fwd");
    return {y, q, s};
}

std::tuple<at::Tensor, OptT> silu_and_checkpoint_backward(const at::Tensor& g, const at::Tensor& q, const at::Tensor& s, const OptT& w) {
    LH_NEED(q.dim() == 2, "x_q must be 2-D");
    const int64_t M = q.size(0), N = q.size(1);
    LH_NEED(N > 0 && N % 256 == 0, "need N % 256 == 0");
    const int codes = checkpoint_code(q.scalar_type()), dt = dtype_code(g);
    check_device(g);
    check_same(g, g.scalar_type(), "g", g, {M, N / 2});
    check_same(g, q.scalar_type(), "x_q", q);
    check_same(g, at::kFloat, "x_scale", s, {M, N / 128});
    const int wt = weight_code(g, w, M);
    const c10::cuda::OptionalCUDAGuard guard(g.device());
    const at::Tensor dx = fresh({M, N}, g.scalar_type(), g);
    OptT dw;
    if (w.has_value()) dw = fresh({M}, w->scalar_type(), *w);
    check_rc(lh_silu_checkpoint_bwd(g.data_ptr(), q.data_ptr(), fptr(s), cptr(w), dt, wt, codes, M, N / 2, dx.data_ptr(), ptr(dw),
                                    c10::cuda::getCurrentCUDAStream().stream()),
             "lh_silu_checkpoint_bwd");
    return {dx, dw};
}

// sizes [..., K] -> [..., N]
std::vector<int64_t> last_dim(const at::Tensor& t, int64_t n) {
    std::vector<int64_t> v = t.sizes().vec();
    v.back() = n;
    return v;
}

std::tuple<at::Tensor, at::Tensor> token_quant_int8(const at::Tensor& x, const OptT& smooth, OptT out, OptT scale) {
    LH_NEED(x.dim() >= 1 && x.size(-1) > 0 && x.size(-1) % 16 == 0, "K must be a positive multiple of 16");
    const int64_t K = x.size(-1), M = x.numel() / K;
    const int dt = dtype_code(x);
    check_device(x);
    check_same(x, x.scalar_type(), "x", x);
    if (smooth.has_value()) check_same(x, at::kFloat, "smooth_scale", *smooth, {K});
    const c10::cuda::OptionalCUDAGuard guard(x.device());
    if (!out.has_value()) out = fresh(x.sizes(), at::kChar, x);
    if (!scale.has_value()) scale = fresh({M}, at::kFloat, x);
    check_same(x, at::kChar, "out", *out, x.sizes());
    check_same(x, at::kFloat, "scale", *scale, {M});
    check_rc(lh_token_quant_int8(x.data_ptr(), fptr(smooth), dt, M, K, out->data_ptr(), fptr(*scale), c10::cuda::getCurrentCUDAStream().stream()),
             "lh_token_quant_int8");
    return {*out, *scale};
}

// a gradient that would be lost without a word is refused
void no_gradient(std::initializer_list<const at::Tensor*> tensors) {
    if (!at::GradMode::is_enabled()) return;
    for (const at::Tensor* t : tensors)
        LH_NEED(t == nullptr || !t->requires_grad(), "the int8 product has no backward pass: call it under torch.no_grad() or on detached tensors");
}

int out_code(at::ScalarType t) {
    switch (t) {
        case at::kBFloat16: return LH_BF16;
        case at::kHalf: return LH_F16;
        case at::kFloat: return LH_F32;
        default: raise_assert("unsupported out_dtype");
    }
}

at::Tensor int8_gemm(const at::Tensor& a, const at::Tensor& b, const at::Tensor& a_s, const at::Tensor& b_s, at::ScalarType out_dtype) {
    no_gradient({&a_s, &b_s});
    const int od = out_code(out_dtype);
    LH_NEED(b.dim() == 2 && a.dim() >= 1 && a.size(-1) == b.size(1), "a and b must have the same number of columns");
    const int64_t N = b.size(0), K = b.size(1);
    LH_NEED(K > 0 && K % 16 == 0, "K must be a positive multiple of 16");
    const int64_t M = a.numel() / K;
    check_device(a);
    check_same(a, at::kChar, "a", a);
    check_same(a, at::kChar, "b", b);
    check_same(a, at::kFloat, "a_s", a_s, {M});
    check_same(a, at::kFloat, "b_s", b_s, {N});
    const c10::cuda::OptionalCUDAGuard guard(a.device());
    const at::Tensor c = fresh(last_dim(a, N), out_dtype, a);
    check_rc(lh_int8_gemm(a.data_ptr(), b.data_ptr(), fptr(a_s), fptr(b_s), c.data_ptr(), M, N, K, od, c10::cuda::getCurrentCUDAStream().stream()),
             "lh_int8_gemm");
    return c;
}

at::Tensor int8_linear(const at::Tensor& x, const at::Tensor& w, const at::Tensor& w_s, const OptT& smooth, const std::optional<at::ScalarType>& out_dtype) {
    no_gradient({&x, &w_s, smooth.has_value() ? &*smooth : nullptr});
    const at::ScalarType type = out_dtype.has_value() ? *out_dtype : x.scalar_type();
    const int od = out_code(type), dt = dtype_code(x);
    LH_NEED(w.dim() == 2 && x.dim() >= 1 && x.size(-1) == w.size(1), "x and w must have the same number of columns");
    const int64_t N = w.size(0), K = w.size(1);
    LH_NEED(K > 0 && K % 16 == 0, "K must be a positive multiple of 16");
    const int64_t M = x.numel() / K;
    check_device(x);
    check_same(x, x.scalar_type(), "x", x);
    check_same(x, at::kChar, "w", w);
    check_same(x, at::kFloat, "w_s", w_s, {N});
    if (smooth.has_value()) check_same(x, at::kFloat, "smooth_scale", *smooth, {K});
    const c10::cuda::OptionalCUDAGuard guard(x.device());
    const at::Tensor c = fresh(last_dim(x, N), type, x);
    const at::Tensor ws = fresh({M * K + 4 * M}, at::kByte, x);      // codes, then scales: K is a multiple of 16
    uint8_t* q = static_cast<uint8_t*>(ws.data_ptr());
    check_rc(lh_int8_linear(x.data_ptr(), fptr(smooth), dt, w.data_ptr(), fptr(w_s), q, reinterpret_cast<float*>(q + M * K), c.data_ptr(), M, N, K,
                            od, c10::cuda::getCurrentCUDAStream().stream()),
             "lh_int8_linear");
    return c;
}

}  // namespace

PYBIND11_MODULE(_lh_host, m) {
    m.doc() = "C++ argument handling for the hottest linghe_b200 wrappers (allocation + C-ABI call)";
    m.def("empty_many", &empty_many);
    m.def("current_stream", &current_stream);
#include "lh_host_bindings.inc"
    m.def("rms_norm_and_block_quant_forward", &rms_norm_and_block_quant_forward);
    m.def("silu_and_block_quant_forward", &silu_and_block_quant_forward);
    m.def("rms_norm_pair_forward", &rms_norm_pair_forward);
    m.def("rms_norm_pair_backward", &rms_norm_pair_backward);
    m.def("silu_and_checkpoint_forward", &silu_and_checkpoint_forward);
    m.def("silu_and_checkpoint_backward", &silu_and_checkpoint_backward);
    m.def("token_quant_int8", &token_quant_int8);
    m.def("int8_gemm", &int8_gemm);
    m.def("int8_linear", &int8_linear);
}
