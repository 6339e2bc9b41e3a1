// Thin PyTorch C++ extension over the C ABI of libksmm_cu.so.
//
// Same module surface as the reference's extension
// (src/ksmm_py/layer/kronecker_sparse/kernel.cpp:25-50): forward(input, factor,
// bs_last, a, b, c, d, dtype, vsize) -> output tensor on the input's device and
// current stream.  `dtype` and `vsize` are accepted for signature compatibility;
// the element type is the input tensor's and vector widths are chosen by the
// library.  chain_forward runs all factors of one KSLinear in one call.
//
// The package's own layers go through layer_forward, layer_train, factor_forward, fp8_forward and
// grouped_forward below, which hold everything between Python and the C ABI (argument checks, output and
// workspace allocation, stream): two factors (384 -> 1536, fp16) on 16 rows 48 -> 20 us against the same calls
// through ctypes, a training step of that layer 241 -> 151 us.  They return None where an
// argument is not what the call takes; the Python wrappers then run the same call through ctypes and raise
// what is wrong with it.  A status other than KSMM_OK comes back as that number; inside the autograd node of
// layer_train it raises what the wrappers raise for it.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <array>
#include <string>
#include <vector>

#include "../../include/ksmm_cu.h"

namespace {

int dtype_code(const torch::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return KSMM_F32;
    case at::kHalf: return KSMM_F16;
    case at::kBFloat16: return KSMM_BF16;
    default: TORCH_CHECK(false, "ksmm: unsupported tensor type ", t.scalar_type());
  }
  return -1;
}

void check_input(const torch::Tensor& x, const char* name) {
  TORCH_CHECK(x.device().is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(x.is_contiguous(), name, " must be contiguous");
}

void check_status(int st) { TORCH_CHECK(st == KSMM_OK, "libksmm_cu: ", ksmm_cu_last_error()); }

torch::Tensor forward(torch::Tensor input, torch::Tensor factor, int64_t bs_last, int64_t a, int64_t b,
                      int64_t c, int64_t d, const std::string& /*dtype*/, int64_t /*vsize*/) {
  check_input(input, "input");
  check_input(factor, "factor");
  TORCH_CHECK(input.dim() == 2 && factor.dim() == 2, "input and factor are 2-D");
  TORCH_CHECK(input.size(bs_last ? 0 : 1) == a * c * d, "input has ", input.size(bs_last ? 0 : 1),
              " features, the pattern expects ", a * c * d);
  TORCH_CHECK(factor.size(0) == a * d * c && factor.size(1) == b, "factor must be (a*d*c, b)");
  TORCH_CHECK(factor.scalar_type() == input.scalar_type() && factor.device() == input.device(),
              "factor and input must share type and device");
  const c10::cuda::CUDAGuard guard(input.device());
  const int64_t batch = input.size(bs_last ? 1 : 0);
  auto out = bs_last ? torch::empty({a * b * d, batch}, input.options())
                     : torch::empty({batch, a * b * d}, input.options());
  ksmm_forward_desc_t f = {};
  f.input = input.data_ptr();
  f.values = factor.data_ptr();
  f.output = out.data_ptr();
  f.batch = batch;
  f.a = static_cast<int>(a); f.b = static_cast<int>(b); f.c = static_cast<int>(c); f.d = static_cast<int>(d);
  f.in_dtype = f.out_dtype = dtype_code(input);
  f.bs_last = bs_last ? 1 : 0;
  f.algo = KSMM_ALGO_AUTO;
  f.config = -1;
  f.alpha = 1.f;
  torch::Tensor scratch;
  if (const size_t need = ksmm_cu_layout_scratch_bytes(&f)) {
    scratch = torch::empty({static_cast<int64_t>(need)}, input.options().dtype(at::kByte));
    f.scratch = scratch.data_ptr();
    f.scratch_bytes = need;
  }
  check_status(ksmm_cu_forward_ex(&f, at::cuda::getCurrentCUDAStream().stream()));
  return out;
}

torch::Tensor chain_forward(torch::Tensor input, std::vector<torch::Tensor> factors,
                            std::vector<std::vector<int64_t>> patterns, int64_t bs_last,
                            c10::optional<torch::Tensor> bias, int64_t activation) {
  check_input(input, "input");
  TORCH_CHECK(input.dim() == 2, "input is 2-D: (features, batch) batch-last, (batch, features) batch-first");
  TORCH_CHECK(!patterns.empty() && patterns.size() == factors.size(), "one factor per pattern");
  std::vector<int32_t> flat;
  std::vector<const void*> vals;
  int64_t feats = input.size(bs_last ? 0 : 1);  // features entering the next factor
  for (size_t f = 0; f < patterns.size(); ++f) {
    TORCH_CHECK(patterns[f].size() == 4, "a pattern is (a, b, c, d)");
    for (int64_t v : patterns[f])
      TORCH_CHECK(v > 0 && v <= 0x7fffffffLL, "pattern values are positive 32-bit integers, got ", v);
    const int64_t a = patterns[f][0], b = patterns[f][1], c = patterns[f][2], d = patterns[f][3];
    TORCH_CHECK(a * c * d == feats, "factor ", f, " expects ", a * c * d, " features but receives ", feats);
    check_input(factors[f], "factor");
    TORCH_CHECK(factors[f].dim() == 2 && factors[f].size(0) == a * d * c && factors[f].size(1) == b,
                "factor ", f, " must have shape (a*d*c, b) = (", a * d * c, ", ", b, ")");
    TORCH_CHECK(factors[f].scalar_type() == input.scalar_type(), "factors share the input's type");
    TORCH_CHECK(factors[f].device() == input.device(), "factors live on the input's device");
    for (int64_t v : patterns[f]) flat.push_back(static_cast<int32_t>(v));
    vals.push_back(factors[f].data_ptr());
    feats = a * b * d;
  }
  const c10::cuda::CUDAGuard guard(input.device());
  const int64_t batch = input.size(bs_last ? 1 : 0);
  const auto& pl = patterns.back();
  const int64_t n_out = pl[0] * pl[1] * pl[3];
  auto out = bs_last ? torch::empty({n_out, batch}, input.options())
                     : torch::empty({batch, n_out}, input.options());
  const int code = dtype_code(input);
  const size_t need = ksmm_cu_chain_workspace_bytes_ex(static_cast<int>(patterns.size()), flat.data(), batch,
                                                       code, bs_last ? 1 : 0);
  torch::Tensor ws;
  if (need > 0) ws = torch::empty({static_cast<int64_t>(need)}, input.options().dtype(at::kByte));
  const void* bptr = nullptr;
  if (bias.has_value()) {
    check_input(*bias, "bias");
    TORCH_CHECK(bias->numel() == n_out && bias->scalar_type() == input.scalar_type() &&
                    bias->device() == input.device(),
                "bias must hold out_size elements of the input's type on the input's device");
    bptr = bias->data_ptr();
  }
  check_status(ksmm_cu_chain_forward_act(input.data_ptr(), vals.data(), out.data_ptr(), bptr,
                                         need > 0 ? ws.data_ptr() : nullptr, need, batch,
                                         static_cast<int>(patterns.size()), flat.data(), code,
                                         bs_last ? 1 : 0, static_cast<int>(activation),
                                         at::cuda::getCurrentCUDAStream().stream()));
  return out;
}


// ---------------------------------------------------------------------------
// the package's own calls
// ---------------------------------------------------------------------------
struct Patterns {
  std::vector<int32_t> flat;
  int n = 0;
  int64_t in(int f) const { return static_cast<int64_t>(flat[4 * f]) * flat[4 * f + 2] * flat[4 * f + 3]; }
  int64_t out(int f) const { return static_cast<int64_t>(flat[4 * f]) * flat[4 * f + 1] * flat[4 * f + 3]; }
};

// a list of 4-tuples of positive ints; false for anything else
bool read_patterns(const py::handle& h, Patterns* p) {
  PyObject* seq = h.ptr();
  if (!PyList_Check(seq) && !PyTuple_Check(seq)) return false;
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(seq);
  if (n < 1 || n > 1024) return false;
  p->n = static_cast<int>(n);
  p->flat.reserve(4 * n);
  for (Py_ssize_t f = 0; f < n; ++f) {
    PyObject* q = PySequence_Fast_GET_ITEM(seq, f);
    if ((!PyList_Check(q) && !PyTuple_Check(q)) || PySequence_Fast_GET_SIZE(q) != 4) return false;
    for (int e = 0; e < 4; ++e) {
      PyObject* v = PySequence_Fast_GET_ITEM(q, e);
      if (!PyLong_Check(v)) return false;
      int overflow = 0;
      const long long x = PyLong_AsLongLongAndOverflow(v, &overflow);
      if (overflow || x <= 0 || x > 0x7fffffffLL) return false;
      p->flat.push_back(static_cast<int32_t>(x));
    }
  }
  return true;
}

bool plain_dtype(const at::Tensor& t) {
  return t.scalar_type() == at::kFloat || t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16;
}

// a plain strided CUDA tensor whose memory may be handed to the library
bool usable(const at::Tensor& t) {
  return t.defined() && t.is_cuda() && t.layout() == at::kStrided && t.is_contiguous() && !t.is_neg() && !t.is_conj();
}

// does the chain take these tensors?  groups: weights of several chains, one after the other
bool chain_fits(const at::Tensor& x, const std::vector<at::Tensor>& w, const Patterns& p, bool last, at::ScalarType wtype,
                int64_t groups = 1) {
  if (static_cast<int>(w.size()) != p.n || !usable(x) || x.dim() != 2 || x.size(last ? 0 : 1) != p.in(0)) return false;
  for (int f = 0; f < p.n; ++f) {
    if (!usable(w[f]) || w[f].dim() != 2 || w[f].scalar_type() != wtype || w[f].device() != x.device()) return false;
    if (w[f].size(0) != groups * p.flat[4 * f] * static_cast<int64_t>(p.flat[4 * f + 3]) * p.flat[4 * f + 2] ||
        w[f].size(1) != p.flat[4 * f + 1])
      return false;
    if (f > 0 && p.in(f) != p.out(f - 1)) return false;
  }
  return true;
}

bool bias_fits(const c10::optional<at::Tensor>& b, const at::Tensor& x, int64_t n, at::ScalarType type) {
  return !b.has_value() || (usable(*b) && b->numel() == n && b->scalar_type() == type && b->device() == x.device());
}

const void* ptr_or_null(const c10::optional<at::Tensor>& t) { return t.has_value() ? t->data_ptr() : nullptr; }

at::Tensor new_tensor(int64_t feats, int64_t batch, bool last, const at::TensorOptions& o) {
  return last ? at::empty({feats, batch}, o) : at::empty({batch, feats}, o);
}
at::Tensor new_bytes(size_t n, const at::Tensor& like) {
  return at::empty({static_cast<int64_t>(n)}, like.options().dtype(at::kByte));
}
void* stream_of(const at::Tensor& x) { return at::cuda::getCurrentCUDAStream(x.get_device()).stream(); }

std::vector<const void*> pointers(const std::vector<at::Tensor>& w) {
  std::vector<const void*> v(w.size());
  for (size_t f = 0; f < w.size(); ++f) v[f] = w[f].data_ptr();
  return v;
}

bool wants_grad(const at::Tensor& x, const std::vector<at::Tensor>& w, const c10::optional<at::Tensor>& b) {
  if (!at::GradMode::is_enabled()) return false;
  if (x.requires_grad() || (b.has_value() && b->requires_grad())) return true;
  for (const auto& t : w)
    if (t.requires_grad()) return true;
  return false;
}

py::object result(int st, const at::Tensor& out) { return st == KSMM_OK ? py::cast(out) : py::cast(st); }

// KSLinear without gradients: every factor, bias, activation and residual in one call
py::object layer_forward(const at::Tensor& x, const std::vector<at::Tensor>& factors, const py::handle& patterns, bool last,
                         bool out_last, const c10::optional<at::Tensor>& bias, int activation,
                         const c10::optional<at::Tensor>& residual) {
  Patterns p;
  if (!read_patterns(patterns, &p) || !usable(x) || !plain_dtype(x) || wants_grad(x, factors, bias) ||
      !chain_fits(x, factors, p, last, x.scalar_type()) || !bias_fits(bias, x, p.out(p.n - 1), x.scalar_type()))
    return py::none();
  const int64_t batch = x.size(last ? 1 : 0), n_out = p.out(p.n - 1);
  if (residual.has_value() && (!usable(*residual) || residual->scalar_type() != x.scalar_type() || residual->dim() != 2 ||
                               residual->size(out_last ? 0 : 1) != n_out || residual->size(out_last ? 1 : 0) != batch ||
                               residual->device() != x.device()))
    return py::none();
  int st;
  at::Tensor out;
  {
    py::gil_scoped_release nogil;
    const c10::cuda::CUDAGuard guard(x.device());
    const int code = dtype_code(x);
    out = new_tensor(n_out, batch, out_last, x.options());
    const size_t need = ksmm_cu_chain_workspace_bytes_layouts(p.n, p.flat.data(), batch, code, last, out_last);
    at::Tensor ws;
    if (need) ws = new_bytes(need, x);
    const auto vals = pointers(factors);
    ksmm_chain_desc_t d = {};
    d.input = x.data_ptr();
    d.values = vals.data();
    d.output = out.data_ptr();
    d.bias = ptr_or_null(bias);
    d.residual = ptr_or_null(residual);
    d.workspace = need ? ws.data_ptr() : nullptr;
    d.workspace_bytes = need;
    d.batch = batch;
    d.nfactors = p.n;
    d.patterns = p.flat.data();
    d.dtype = code;
    d.bs_last = last;
    d.out_layout = out_last ? 2 : 1;
    d.activation = activation;
    st = ksmm_cu_chain_forward_desc(&d, stream_of(x));
  }
  return result(st, out);
}

// Kernel.forward: one factor
py::object factor_forward(const at::Tensor& x, const at::Tensor& w, bool last, int64_t a, int64_t b, int64_t c, int64_t d) {
  if (a <= 0 || b <= 0 || c <= 0 || d <= 0 || a > 0x7fffffff || b > 0x7fffffff || c > 0x7fffffff || d > 0x7fffffff ||
      !usable(x) || !usable(w) || !plain_dtype(x) || x.dim() != 2 || w.dim() != 2 || w.scalar_type() != x.scalar_type() ||
      w.device() != x.device() || x.size(last ? 0 : 1) != a * c * d || w.size(0) != a * c * d || w.size(1) != b)
    return py::none();
  int st;
  at::Tensor out;
  {
    py::gil_scoped_release nogil;
    const c10::cuda::CUDAGuard guard(x.device());
    const int64_t batch = x.size(last ? 1 : 0);
    out = new_tensor(a * b * d, batch, last, x.options().requires_grad(false));
    ksmm_forward_desc_t f = {};
    f.input = x.data_ptr();
    f.values = w.data_ptr();
    f.output = out.data_ptr();
    f.batch = batch;
    f.a = static_cast<int>(a); f.b = static_cast<int>(b); f.c = static_cast<int>(c); f.d = static_cast<int>(d);
    f.in_dtype = f.out_dtype = dtype_code(x);
    f.bs_last = last;
    f.algo = KSMM_ALGO_AUTO;
    f.config = -1;
    f.alpha = 1.f;
    const size_t need = ksmm_cu_layout_scratch_bytes(&f);
    at::Tensor scratch;
    if (need) {
      scratch = new_bytes(need, x);
      f.scratch = scratch.data_ptr();
      f.scratch_bytes = need;
    }
    st = ksmm_cu_forward_ex(&f, stream_of(x));
  }
  return result(st, out);
}

// the factors of an fp8 layer
py::object fp8_forward(const at::Tensor& x, const std::vector<at::Tensor>& factors, const std::vector<float>& scales,
                       const py::handle& patterns, bool last, const c10::optional<at::Tensor>& bias) {
  Patterns p;
  if (!read_patterns(patterns, &p) || !usable(x) || !plain_dtype(x) || scales.size() != factors.size() ||
      !chain_fits(x, factors, p, last, at::kFloat8_e4m3fn) || !bias_fits(bias, x, p.out(p.n - 1), at::kBFloat16))
    return py::none();
  int st;
  at::Tensor out;
  {
    py::gil_scoped_release nogil;
    const c10::cuda::CUDAGuard guard(x.device());
    const int64_t batch = x.size(last ? 1 : 0);
    const int code = dtype_code(x);
    out = new_tensor(p.out(p.n - 1), batch, last, x.options().dtype(at::kBFloat16).requires_grad(false));
    const size_t need = ksmm_cu_chain_fp8_workspace_bytes(p.n, p.flat.data(), batch, code, last);
    const at::Tensor ws = new_bytes(need, x);
    const auto vals = pointers(factors);
    st = ksmm_cu_chain_forward_fp8(x.data_ptr(), code, vals.data(), scales.data(), out.data_ptr(), ptr_or_null(bias),
                                   ws.data_ptr(), need, batch, p.n, p.flat.data(), last, stream_of(x));
  }
  return result(st, out);
}

// several chains on one input, weights and bias stacked
py::object grouped_forward(const at::Tensor& x, const std::vector<at::Tensor>& factors, const py::handle& patterns, bool last,
                           int64_t groups, const c10::optional<at::Tensor>& bias) {
  Patterns p;
  if (groups < 1 || groups > 65535 || !read_patterns(patterns, &p) || !usable(x) || !plain_dtype(x) ||
      !chain_fits(x, factors, p, last, x.scalar_type(), groups) ||
      !bias_fits(bias, x, groups * p.out(p.n - 1), x.scalar_type()))
    return py::none();
  int st;
  at::Tensor out;
  {
    py::gil_scoped_release nogil;
    const c10::cuda::CUDAGuard guard(x.device());
    const int64_t batch = x.size(last ? 1 : 0), n_out = p.out(p.n - 1);
    const int code = dtype_code(x);
    const auto o = x.options().requires_grad(false);
    out = last ? at::empty({groups, n_out, batch}, o) : at::empty({groups, batch, n_out}, o);
    const size_t need = groups * ksmm_cu_chain_workspace_bytes_ex(p.n, p.flat.data(), batch, code, last);
    at::Tensor ws;
    if (need) ws = new_bytes(need, x);
    const auto vals = pointers(factors);
    st = ksmm_cu_grouped_chain_forward(x.data_ptr(), vals.data(), out.data_ptr(), ptr_or_null(bias),
                                       need ? ws.data_ptr() : nullptr, need, batch, p.n, p.flat.data(), code, last,
                                       static_cast<int>(groups), stream_of(x));
  }
  return result(st, out);
}

// Raises ksmm_b200.KsmmError for a status, on whichever thread autograd runs (with or without the GIL).
void raise_status(int st) {
  if (st == KSMM_OK) return;
  py::gil_scoped_acquire gil;
  py::module_::import("ksmm_b200._lib").attr("check")(st);
}

// A trainable layer as one autograd node: ksmm_b200.kernel.ChainFunction without Python in its backward.
at::Tensor aligned(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 ? t.clone() : t; }

struct ChainNode : torch::autograd::Function<ChainNode> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x_in, const c10::optional<at::Tensor>& bias,
                            at::TensorList factors, std::vector<int64_t> patterns, bool last) {
    const at::Tensor x = aligned(x_in);
    const c10::cuda::CUDAGuard guard(x.device());
    const int n = static_cast<int>(factors.size());
    std::vector<int32_t> flat(patterns.begin(), patterns.end());
    const int32_t* pl = flat.data() + 4 * (n - 1);
    const int64_t batch = x.size(last ? 1 : 0), n_out = static_cast<int64_t>(pl[0]) * pl[1] * pl[3];
    const int code = dtype_code(x);
    size_t bytes[3];
    raise_status(ksmm_cu_chain_train_bytes(n, flat.data(), batch, code, last, &bytes[0], &bytes[1], &bytes[2]));
    at::Tensor out = new_tensor(n_out, batch, last, x.options());
    const at::Tensor saved = new_bytes(bytes[0], x), scratch = new_bytes(bytes[1], x);
    std::vector<const void*> vals(n);
    for (int f = 0; f < n; ++f) vals[f] = factors[f].data_ptr();
    int32_t layouts[16] = {};
    raise_status(ksmm_cu_chain_train_forward(x.data_ptr(), vals.data(), out.data_ptr(), ptr_or_null(bias), saved.data_ptr(),
                                             bytes[0], scratch.data_ptr(), bytes[1], batch, n, flat.data(), code, last, layouts,
                                             stream_of(x)));
    torch::autograd::variable_list keep{x, saved};
    keep.insert(keep.end(), factors.begin(), factors.end());
    ctx->save_for_backward(std::move(keep));
    // number of factors, layout, bytes of the backward, patterns, layouts, the bias's shape
    std::vector<int64_t> meta{n, last, static_cast<int64_t>(bytes[2])};
    meta.insert(meta.end(), patterns.begin(), patterns.end());
    for (int f = 0; f + 1 < n; ++f) meta.push_back(layouts[f]);
    meta.push_back(bias.has_value());
    if (bias.has_value()) meta.insert(meta.end(), bias->sizes().begin(), bias->sizes().end());
    ctx->saved_data["chain"] = std::move(meta);
    return out;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto kept = ctx->get_saved_variables();
    const std::vector<int64_t> meta = ctx->saved_data["chain"].toIntVector();
    const int n = static_cast<int>(meta[0]);
    const bool last = meta[1] != 0;
    const size_t need = static_cast<size_t>(meta[2]);
    const std::vector<int32_t> flat(meta.begin() + 3, meta.begin() + 3 + 4 * n);
    std::vector<int32_t> layouts(meta.begin() + 3 + 4 * n, meta.begin() + 3 + 4 * n + n - 1);
    const bool has_bias = meta[3 + 4 * n + n - 1] != 0;
    layouts.push_back(0);
    const at::Tensor& x = kept[0];
    const at::Tensor& saved = kept[1];
    const c10::cuda::CUDAGuard guard(x.device());
    const at::Tensor g = aligned(grads[0].contiguous());
    // edges of the graph: the input, the bias if there is one, the factors
    at::Tensor gx, gb;
    if (ctx->needs_input_grad(0)) gx = at::empty(x.sizes(), x.options());
    if (has_bias && ctx->needs_input_grad(1))
      gb = at::empty(at::IntArrayRef(meta.data() + 3 + 4 * n + n, meta.size() - (3 + 4 * n + n)), x.options());
    std::vector<at::Tensor> gw(n);
    std::vector<const void*> vals(n);
    std::vector<void*> outs(n, nullptr);
    for (int f = 0; f < n; ++f) {
      const at::Tensor& w = kept[2 + f];
      vals[f] = w.data_ptr();
      if (ctx->needs_input_grad(1 + has_bias + f)) {
        gw[f] = at::empty(w.sizes(), w.options());
        outs[f] = gw[f].data_ptr();
      }
    }
    const at::Tensor ws = new_bytes(need, x);
    raise_status(ksmm_cu_chain_backward(x.data_ptr(), vals.data(), saved.data_ptr(), layouts.data(), g.data_ptr(),
                                        gx.defined() ? gx.data_ptr() : nullptr, outs.data(),
                                        gb.defined() ? gb.data_ptr() : nullptr, ws.data_ptr(), need, x.size(last ? 1 : 0), n,
                                        flat.data(), dtype_code(x), last, stream_of(x)));
    torch::autograd::variable_list r{gx, gb};
    r.insert(r.end(), gw.begin(), gw.end());
    r.emplace_back();  // patterns
    r.emplace_back();  // layout
    return r;
  }
};

py::object layer_train(const at::Tensor& x, const std::vector<at::Tensor>& factors, const py::handle& patterns, bool last,
                       const c10::optional<at::Tensor>& bias) {
  Patterns p;
  if (!read_patterns(patterns, &p) || p.n > 16 || !usable(x) || !plain_dtype(x) ||
      !chain_fits(x, factors, p, last, x.scalar_type()) || !bias_fits(bias, x, p.out(p.n - 1), x.scalar_type()))
    return py::none();
  at::Tensor out;
  {
    py::gil_scoped_release nogil;
    out = ChainNode::apply(x, bias, at::TensorList(factors), std::vector<int64_t>(p.flat.begin(), p.flat.end()), last);
  }
  return py::cast(out);
}

// A backward pass that is to be differentiated again would come back as a constant.
void differentiable_once() {
  TORCH_CHECK_NOT_IMPLEMENTED(!at::GradMode::is_enabled(), "this operator is differentiable once (create_graph=True)");
}

// a tangent of forward-mode differentiation, which a call through data pointers would lose
bool has_tangent(const at::Tensor& t) { return t.defined() && t._fw_grad(/*level=*/0).defined(); }

// a gated layer without gradients
bool gated_fits(const at::Tensor& x, const std::vector<at::Tensor>& factors, const Patterns& p, bool last,
                const c10::optional<at::Tensor>& bias) {
  if (has_tangent(x) || (bias.has_value() && has_tangent(*bias)) || std::any_of(factors.begin(), factors.end(), has_tangent)) return false;
  return p.n <= 16 && usable(x) && plain_dtype(x) && chain_fits(x, factors, p, last, x.scalar_type(), 2) &&
         bias_fits(bias, x, 2 * p.out(p.n - 1), x.scalar_type());
}

ksmm_gated_desc_t gated_desc(const at::Tensor& x, const void* const* values, const int32_t* patterns, int n, bool last, bool out_last,
                             int activation) {
  ksmm_gated_desc_t d = {};
  d.input = x.data_ptr();
  d.values = values;
  d.batch = x.size(last ? 1 : 0);
  d.nfactors = n;
  d.patterns = patterns;
  d.dtype = dtype_code(x);
  d.bs_last = last;
  d.out_layout = out_last ? 2 : 1;
  d.activation = activation;
  return d;
}

py::object gated_forward(const at::Tensor& x, const std::vector<at::Tensor>& factors, const py::handle& patterns, bool last,
                         bool out_last, const c10::optional<at::Tensor>& bias, int activation) {
  Patterns p;
  if (!read_patterns(patterns, &p) || !gated_fits(x, factors, p, last, bias)) return py::none();
  int st;
  at::Tensor out;
  {
    py::gil_scoped_release nogil;
    const c10::cuda::CUDAGuard guard(x.device());
    const auto vals = pointers(factors);
    ksmm_gated_desc_t d = gated_desc(x, vals.data(), p.flat.data(), p.n, last, out_last, activation);
    out = new_tensor(p.out(p.n - 1), d.batch, out_last, x.options().requires_grad(false));
    d.workspace_bytes = ksmm_cu_gated_workspace_bytes(p.n, p.flat.data(), d.batch, d.dtype, last, out_last);
    const at::Tensor ws = new_bytes(d.workspace_bytes, x);
    d.workspace = ws.data_ptr();
    d.output = out.data_ptr();
    d.bias = ptr_or_null(bias);
    st = ksmm_cu_gated_forward(&d, stream_of(x));
  }
  return result(st, out);
}

// A trainable gated layer as one autograd node: ksmm_b200.kernel.GatedFunction without Python in its backward.
struct GatedNode : torch::autograd::Function<GatedNode> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x_in, const c10::optional<at::Tensor>& bias,
                            at::TensorList factors, std::vector<int64_t> patterns, bool last, bool out_last, int64_t activation) {
    const at::Tensor x = aligned(x_in);
    const c10::cuda::CUDAGuard guard(x.device());
    const int n = static_cast<int>(factors.size());
    const std::vector<int32_t> flat(patterns.begin(), patterns.end());
    std::vector<const void*> vals(n);
    for (int f = 0; f < n; ++f) vals[f] = factors[f].data_ptr();
    ksmm_gated_desc_t d = gated_desc(x, vals.data(), flat.data(), n, last, out_last, static_cast<int>(activation));
    const int32_t* pl = flat.data() + 4 * (n - 1);
    size_t bytes[3];
    raise_status(ksmm_cu_gated_train_bytes(n, flat.data(), d.batch, d.dtype, last, out_last, &bytes[0], &bytes[1], &bytes[2]));
    at::Tensor out = new_tensor(static_cast<int64_t>(pl[0]) * pl[1] * pl[3], d.batch, out_last, x.options());
    // (an empty batch keeps nothing, but a saved pointer says that this is training)
    const at::Tensor saved = new_bytes(std::max<size_t>(bytes[0], 1), x), ws = new_bytes(bytes[1], x);
    int32_t layouts[16] = {};
    d.output = out.data_ptr();
    d.bias = ptr_or_null(bias);
    d.saved = saved.data_ptr();
    d.saved_bytes = bytes[0];
    d.workspace = ws.data_ptr();
    d.workspace_bytes = bytes[1];
    d.layouts = layouts;
    raise_status(ksmm_cu_gated_forward(&d, stream_of(x)));
    torch::autograd::variable_list keep{x, saved};
    keep.insert(keep.end(), factors.begin(), factors.end());
    ctx->save_for_backward(std::move(keep));
    // number of factors, layouts, activation, bytes of the backward, patterns, kept layouts, the bias's shape
    std::vector<int64_t> meta{n, last, out_last, activation, static_cast<int64_t>(bytes[2])};
    meta.insert(meta.end(), patterns.begin(), patterns.end());
    for (int f = 0; f < n; ++f) meta.push_back(layouts[f]);
    meta.push_back(bias.has_value());
    if (bias.has_value()) meta.insert(meta.end(), bias->sizes().begin(), bias->sizes().end());
    ctx->saved_data["gated"] = std::move(meta);
    return out;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    differentiable_once();
    const auto kept = ctx->get_saved_variables();
    const std::vector<int64_t> meta = ctx->saved_data["gated"].toIntVector();
    const int n = static_cast<int>(meta[0]);
    const bool last = meta[1] != 0, out_last = meta[2] != 0;
    const std::vector<int32_t> flat(meta.begin() + 5, meta.begin() + 5 + 4 * n);
    std::vector<int32_t> layouts(meta.begin() + 5 + 4 * n, meta.begin() + 5 + 5 * n);
    const size_t at_bias = 5 + 5 * static_cast<size_t>(n);
    const bool has_bias = meta[at_bias] != 0;
    const at::Tensor& x = kept[0];
    const c10::cuda::CUDAGuard guard(x.device());
    const at::Tensor g = aligned(grads[0].contiguous());
    // edges of the graph: the input, the bias if there is one, the factors
    at::Tensor gx, gb;
    if (ctx->needs_input_grad(0)) gx = at::empty(x.sizes(), x.options());
    if (has_bias && ctx->needs_input_grad(1))
      gb = at::empty(at::IntArrayRef(meta.data() + at_bias + 1, meta.size() - at_bias - 1), x.options());
    std::vector<at::Tensor> gw(n);
    std::vector<const void*> vals(n);
    std::vector<void*> outs(n, nullptr);
    for (int f = 0; f < n; ++f) {
      const at::Tensor& w = kept[2 + f];
      vals[f] = w.data_ptr();
      if (ctx->needs_input_grad(1 + has_bias + f)) {
        gw[f] = at::empty(w.sizes(), w.options());
        outs[f] = gw[f].data_ptr();
      }
    }
    ksmm_gated_desc_t d = gated_desc(x, vals.data(), flat.data(), n, last, out_last, static_cast<int>(meta[3]));
    const at::Tensor ws = new_bytes(static_cast<size_t>(meta[4]), x);
    d.workspace = ws.data_ptr();
    d.workspace_bytes = static_cast<size_t>(meta[4]);
    d.saved = kept[1].data_ptr();
    d.saved_bytes = static_cast<size_t>(kept[1].numel());
    d.layouts = layouts.data();
    raise_status(ksmm_cu_gated_backward(&d, g.data_ptr(), gx.defined() ? gx.data_ptr() : nullptr, outs.data(),
                                        gb.defined() ? gb.data_ptr() : nullptr, stream_of(x)));
    torch::autograd::variable_list r{gx, gb};
    r.insert(r.end(), gw.begin(), gw.end());
    for (int q = 0; q < 4; ++q) r.emplace_back();  // patterns, layouts, activation
    return r;
  }
};

// KSGatedLinear: with gradients where something learns
py::object gated_layer(const at::Tensor& x, const std::vector<at::Tensor>& factors, const py::handle& patterns, bool last,
                       bool out_last, const c10::optional<at::Tensor>& bias, int activation) {
  if (!wants_grad(x, factors, bias)) return gated_forward(x, factors, patterns, last, out_last, bias, activation);
  Patterns p;
  if (!read_patterns(patterns, &p) || !gated_fits(x, factors, p, last, bias)) return py::none();
  at::Tensor out;
  {
    py::gil_scoped_release nogil;
    out = GatedNode::apply(x, bias, at::TensorList(factors), std::vector<int64_t>(p.flat.begin(), p.flat.end()), last, out_last,
                           static_cast<int64_t>(activation));
  }
  return py::cast(out);
}

// ---------------------------------------------------------------------------
// residual_norm
// ---------------------------------------------------------------------------
constexpr int kNormParams = 7;  // weight, bias, post_weight, post_bias, scale, shift, gate
using NormParams = std::array<c10::optional<at::Tensor>, kNormParams>;

struct NormCall {
  int64_t norm, post_norm, bs_last;
  double alpha, eps;
  int64_t rows = 0, channels = 0, samples = 1;
  int param_dtype = 0;
};

// Tensors that the kernel takes as they are; everything else goes through Python, which converts or raises.
bool norm_fits(const at::Tensor& x, const c10::optional<at::Tensor>& y, const NormParams& p, NormCall* c) {
  if (has_tangent(x) || (y.has_value() && has_tangent(*y))) return false;
  if (!usable(x) || !plain_dtype(x) || x.dim() < 1 || x.dim() > 64 || c->norm < 0 || c->norm > 2 || c->post_norm < 0 || c->post_norm > 2)
    return false;
  c->channels = x.size(c->bs_last ? 0 : x.dim() - 1);
  if (c->channels <= 0 || c->channels > 0x7fffffff || (c->norm == 0 && !y.has_value())) return false;
  c->rows = x.numel() / c->channels;
  if (y.has_value()) {
    if (!usable(*y) || y->sizes() != x.sizes() || y->scalar_type() != x.scalar_type() || y->device() != x.device()) return false;
  } else if (c->post_norm || p[2].has_value() || p[3].has_value() || p[6].has_value()) {
    return false;
  }
  if ((!c->post_norm && (p[2].has_value() || p[3].has_value())) ||
      (!c->norm && (p[0].has_value() || p[1].has_value() || p[4].has_value() || p[5].has_value())))
    return false;
  at::ScalarType type = x.scalar_type();
  bool any = false;
  for (int q = 0; q < kNormParams; ++q) {
    if (!p[q].has_value()) continue;
    const at::Tensor& t = *p[q];
    if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || t.is_neg() || t.is_conj() || t.device() != x.device() || has_tangent(t)) return false;
    if (any && t.scalar_type() != type) return false;
    type = t.scalar_type();
    any = true;
    if (t.dim() == 1) {
      if (t.size(0) != c->channels || (t.stride(0) != 1 && c->channels != 1)) return false;
      continue;
    }
    if (q < 4 || t.dim() != 2 || t.size(1) != c->channels || t.size(0) < 1 || (t.stride(1) != 1 && c->channels != 1)) return false;
    if (t.size(0) > 1) {
      if (t.stride(0) <= 0 || (c->samples != 1 && c->samples != t.size(0))) return false;
      c->samples = t.size(0);
    }
  }
  if (type != x.scalar_type() && type != at::kFloat) return false;
  if (c->rows % c->samples) return false;
  c->param_dtype = type == at::kFloat ? KSMM_F32 : dtype_code(x);
  return true;
}

int64_t sample_stride(const at::Tensor& t) { return t.dim() == 2 && t.size(0) > 1 ? t.stride(0) : 0; }

ksmm_norm_desc_t norm_desc(const at::Tensor& x, const c10::optional<at::Tensor>& y, const NormParams& p, const NormCall& c) {
  ksmm_norm_desc_t d = {};
  d.x = x.data_ptr();
  d.y = ptr_or_null(y);
  d.weight = ptr_or_null(p[0]); d.bias = ptr_or_null(p[1]);
  d.post_weight = ptr_or_null(p[2]); d.post_bias = ptr_or_null(p[3]);
  d.scale = ptr_or_null(p[4]); d.shift = ptr_or_null(p[5]); d.gate = ptr_or_null(p[6]);
  if (p[4].has_value()) d.scale_stride = sample_stride(*p[4]);
  if (p[5].has_value()) d.shift_stride = sample_stride(*p[5]);
  if (p[6].has_value()) d.gate_stride = sample_stride(*p[6]);
  d.rows = c.rows; d.samples = c.samples; d.channels = static_cast<int32_t>(c.channels);
  d.norm = static_cast<int32_t>(c.norm); d.post_norm = static_cast<int32_t>(c.post_norm);
  d.bs_last = static_cast<int32_t>(c.bs_last);
  d.dtype = dtype_code(x); d.param_dtype = c.param_dtype;
  d.alpha = static_cast<float>(c.alpha); d.eps = static_cast<float>(c.eps);
  return d;
}

int norm_run(const at::Tensor& x, const c10::optional<at::Tensor>& y, const NormParams& p, const NormCall& c, at::Tensor* z,
             at::Tensor* h, at::Tensor* stats) {
  const c10::cuda::CUDAGuard guard(x.device());
  ksmm_norm_desc_t d = norm_desc(x, y, p, c);
  const auto o = x.options().requires_grad(false);
  if (y.has_value()) {
    *z = at::empty(x.sizes(), o);
    d.z = z->data_ptr();
  }
  if (c.norm) {
    *h = at::empty(x.sizes(), o);
    d.h = h->data_ptr();
  }
  if (stats) {
    *stats = at::empty({c.rows * 4}, o.dtype(at::kFloat));
    d.stats = stats->data_ptr<float>();
  }
  at::Tensor ws;
  const size_t need = c.bs_last ? ksmm_cu_norm_forward_workspace_bytes(&d) : 0;
  if (need) ws = new_bytes(need, x);
  return ksmm_cu_norm_forward(&d, need ? ws.data_ptr() : nullptr, need, stream_of(x));
}

// residual_norm as one autograd node: ksmm_b200.norm.NormFunction without Python in its backward.
struct NormNode : torch::autograd::Function<NormNode> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x,
                                                const c10::optional<at::Tensor>& y, const c10::optional<at::Tensor>& p0,
                                                const c10::optional<at::Tensor>& p1, const c10::optional<at::Tensor>& p2,
                                                const c10::optional<at::Tensor>& p3, const c10::optional<at::Tensor>& p4,
                                                const c10::optional<at::Tensor>& p5, const c10::optional<at::Tensor>& p6,
                                                std::vector<int64_t> ints, double alpha, double eps) {
    const NormParams p{p0, p1, p2, p3, p4, p5, p6};
    const NormCall c{ints[0], ints[1], ints[2], alpha, eps, ints[3], ints[4], ints[5], static_cast<int>(ints[6])};
    at::Tensor z, h, stats;
    raise_status(norm_run(x, y, p, c, &z, &h, &stats));
    // (what pre normalised: 16-bit calls form it again from x and y, unrounded)
    torch::autograd::variable_list keep{y.has_value() && x.scalar_type() == at::kFloat ? z : x, y.has_value() ? *y : at::Tensor(), stats};
    for (const auto& t : p) keep.push_back(t.has_value() ? *t : at::Tensor());
    ctx->save_for_backward(std::move(keep));
    ctx->saved_data["ints"] = std::move(ints);
    ctx->saved_data["alpha"] = alpha;
    ctx->saved_data["eps"] = eps;
    ctx->set_materialize_grads(false);
    torch::autograd::variable_list out;
    if (z.defined()) out.push_back(z);
    if (h.defined()) out.push_back(h);
    return out;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    differentiable_once();
    const auto kept = ctx->get_saved_variables();
    const std::vector<int64_t> ints = ctx->saved_data["ints"].toIntVector();
    const at::Tensor& x = kept[0];
    const bool has_y = kept[1].defined();
    c10::optional<at::Tensor> y;
    if (has_y) y = kept[1];
    NormParams p;
    for (int q = 0; q < kNormParams; ++q)
      if (kept[3 + q].defined()) p[q] = kept[3 + q];
    const NormCall c{ints[0], ints[1], ints[2], ctx->saved_data["alpha"].toDouble(), ctx->saved_data["eps"].toDouble(),
                     ints[3], ints[4], ints[5], static_cast<int>(ints[6])};
    torch::autograd::variable_list r(2 + kNormParams + 3);
    at::Tensor gz, gh;
    if (has_y) gz = grads[0];
    if (c.norm) gh = grads.back();
    if (!gz.defined() && !gh.defined()) return r;
    const c10::cuda::CUDAGuard guard(x.device());
    ksmm_norm_desc_t d = norm_desc(x, y, p, c);
    if (x.scalar_type() == at::kFloat) d.z = x.data_ptr();
    d.stats = kept[2].data_ptr<float>();
    if (gz.defined()) {
      gz = gz.to(x.scalar_type()).contiguous();
      d.grad_z = gz.data_ptr();
    }
    if (gh.defined()) {
      gh = gh.to(x.scalar_type()).contiguous();
      d.grad_h = gh.data_ptr();
    }
    // edges of the graph: x, y if there is one, the parameters that there are
    int edge = 0;
    auto wanted = [&](bool there, const at::Tensor& like, int at) -> void* {
      if (!there || !ctx->needs_input_grad(edge++)) return nullptr;
      r[at] = at::empty(like.sizes(), like.options().requires_grad(false));
      return r[at].data_ptr();
    };
    d.grad_x = wanted(true, x, 0);
    d.grad_y = wanted(has_y, x, 1);
    void** const outs[kNormParams] = {&d.grad_weight, &d.grad_bias, &d.grad_post_weight, &d.grad_post_bias,
                                      &d.grad_scale, &d.grad_shift, &d.grad_gate};
    for (int q = 0; q < kNormParams; ++q)
      *outs[q] = wanted(p[q].has_value(), p[q].has_value() ? *p[q] : x, 2 + q);
    // (sizes of a cut row are dense in a new tensor: the kernel writes rows one after the other)
    const size_t need = ksmm_cu_norm_backward_workspace_bytes(&d);
    at::Tensor ws;
    if (need) ws = new_bytes(need, x);
    raise_status(ksmm_cu_norm_backward(&d, need ? ws.data_ptr() : nullptr, need, stream_of(x)));
    return r;
  }
};

py::object residual_norm(const at::Tensor& x, const c10::optional<at::Tensor>& y, const c10::optional<at::Tensor>& weight,
                         const c10::optional<at::Tensor>& bias, const c10::optional<at::Tensor>& post_weight,
                         const c10::optional<at::Tensor>& post_bias, const c10::optional<at::Tensor>& scale,
                         const c10::optional<at::Tensor>& shift, const c10::optional<at::Tensor>& gate, int64_t norm, int64_t post_norm,
                         double alpha, double eps, bool bs_last) {
  const NormParams p{weight, bias, post_weight, post_bias, scale, shift, gate};
  NormCall c{norm, post_norm, bs_last, alpha, eps};
  if (!norm_fits(x, y, p, &c)) return py::none();
  bool learns = x.requires_grad() || (y.has_value() && y->requires_grad());
  for (const auto& t : p) learns = learns || (t.has_value() && t->requires_grad());
  if (learns && at::GradMode::is_enabled()) {
    torch::autograd::variable_list out;
    {
      py::gil_scoped_release nogil;
      out = NormNode::apply(x, y, p[0], p[1], p[2], p[3], p[4], p[5], p[6],
                            std::vector<int64_t>{norm, post_norm, bs_last, c.rows, c.channels, c.samples, c.param_dtype}, alpha, eps);
    }
    return out.size() > 1 ? py::object(py::make_tuple(out[0], out[1])) : py::cast(out[0]);
  }
  at::Tensor z, h;
  int st;
  {
    py::gil_scoped_release nogil;
    st = norm_run(x, y, p, c, &z, &h, nullptr);
  }
  if (st != KSMM_OK) return py::cast(st);
  if (z.defined() && h.defined()) return py::make_tuple(z, h);
  return py::cast(z.defined() ? z : h);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("forward", &forward, "One Kronecker-sparse factor (CUDA, libksmm_cu)");
  m.def("chain_forward", &chain_forward, "All factors of a KSLinear in one call (CUDA, libksmm_cu)",
        py::arg("input"), py::arg("factors"), py::arg("patterns"), py::arg("bs_last"),
        py::arg("bias") = py::none(), py::arg("activation") = 0);
  m.def("layer_forward", &layer_forward, "A KSLinear without gradients");
  m.def("layer_train", &layer_train, "A trainable KSLinear as one autograd node");
  m.def("factor_forward", &factor_forward, "One factor in its input's type");
  m.def("fp8_forward", &fp8_forward, "The factors of an fp8 KSLinear");
  m.def("grouped_forward", &grouped_forward, "Several chains on one input");
  m.def("residual_norm", &residual_norm, "Norms around a block, gate, residual scale and modulation");
  m.def("gated_forward", &gated_forward, "A gated layer without gradients");
  m.def("gated_layer", &gated_layer, "A gated layer, as one autograd node where something learns");
}
