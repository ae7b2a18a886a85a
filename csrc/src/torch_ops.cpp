// The operators of ops/gated_ffn.py and ops/mx4.py on torch tensors: allocation, stream and autograd around the C entry points.
//
// A call on a few tokens is bound by the host. Through Python's autograd.Function and ctypes a training step of the feed-forward block took 142 us
// of host time and a product with quantisation 14.6; the kernels of the smallest sizes take 20 and 6. Arguments are checked by the Python
// callers.
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <cuda_runtime.h>

#include <array>

#include "purlin/gated_ffn.h"
#include "purlin/mx4.h"

extern "C" const char* purlin_last_error();

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void check(int rc) {
  if (rc) throw std::runtime_error(std::string("purlin: ") + purlin_last_error());
}
int narrow(int64_t v) {      // of a size that the C entries count in 32 bits
  if (v < 0 || v > INT32_MAX) throw std::invalid_argument("a dimension of 2^31 or more");
  return int(v);
}
void* stream() { return c10::cuda::getCurrentCUDAStream().stream(); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor bytes(int64_t n, const Tensor& like) { return at::empty({n}, like.options().dtype(at::kByte)); }

// A kernel whose wait gave up leaves outputs unwritten and says so in four words, {code, where, tile, k-block}. They lie in host memory that every
// device can write (one set each, for the life of the process, captured graphs included), so that looking at them costs a call nothing: the first
// call on the device after such a kernel raises, whichever operator it is of, as does check_waits().
constexpr int kMaxDevices = 64, kWordsApart = 16;
uint32_t* waitWords(int64_t device) {
  static uint32_t* const all = [] {
    void* p = nullptr;
    const c10::cuda::CUDAStreamCaptureModeGuard relaxed(cudaStreamCaptureModeRelaxed);      // (the first call may be a captured one)
    const size_t size = size_t(kMaxDevices) * kWordsApart * sizeof(uint32_t);
    if (cudaHostAlloc(&p, size, cudaHostAllocPortable | cudaHostAllocMapped) != cudaSuccess) { cudaGetLastError(); throw std::runtime_error("purlin: no host memory for the words of waits"); }
    memset(p, 0, size);
    return static_cast<uint32_t*>(p);
  }();
  if (device < 0 || device >= kMaxDevices) throw std::invalid_argument("no such device");
  return all + device * kWordsApart;
}
std::array<uint32_t, 4> takeWaitReport(int64_t device) {      // and clears it
  uint32_t* const w = waitWords(device);
  const volatile uint32_t* v = w;
  if (!v[0]) return {};
  const std::array<uint32_t, 4> r{v[0], v[1], v[2], v[3]};
  return __atomic_exchange_n(w, 0u, __ATOMIC_ACQ_REL) ? r : std::array<uint32_t, 4>{};      // (one of two threads tells)
}
uint32_t* status(const Tensor& on) {
  const int64_t device = on.device().index();
  const auto r = takeWaitReport(device);
  if (r[0])
    throw std::runtime_error("purlin: a wait inside an earlier kernel of the operators on cuda:" + std::to_string(device) + " gave up (where " + std::to_string(r[1]) + ", " +
                             std::to_string(r[2]) + ", " + std::to_string(r[3]) + "): what it computed is not complete");
  return waitWords(device);
}

// The tangent of a dual tensor (forward-mode differentiation) would be dropped without a word: the kernels see the values alone.
void refuseTangents(const char* name, std::initializer_list<const Tensor*> inputs) {
  for (const Tensor* t : inputs)
    if (t->_fw_grad(/*level=*/0).defined()) throw std::runtime_error(std::string(name) + " has no forward-mode derivative");
}

// y and h, and the pre-activations where the backward will want them
std::tuple<Tensor, Tensor, Tensor> ffnForward(const Tensor& x, const Tensor& wGateUp, const Tensor& wDown, int64_t activation, bool keep) {
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t tokens = x.size(0), hidden = wDown.size(0), intermediate = wDown.size(1);
  Tensor y = at::empty_like(x), h = at::empty({tokens, intermediate}, x.options()), saved;
  if (keep) saved = bytes(int64_t(purlin_ffn_saved_bytes(narrow(tokens), narrow(intermediate))), x);
  if (tokens)
    check(purlin_ffn_forward(x.data_ptr(), wGateUp.data_ptr(), wDown.data_ptr(), h.data_ptr(), ptr(saved), y.data_ptr(), narrow(tokens), narrow(hidden), narrow(intermediate),
                             int(activation), status(x), stream()));
  return {y, h, saved};
}

struct GatedFfn : torch::autograd::Function<GatedFfn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& wGateUp, const Tensor& wDown, int64_t activation) {
    const bool needX = x.requires_grad(), needGateUp = wGateUp.requires_grad(), needDown = wDown.requires_grad();
    auto [y, h, saved] = ffnForward(x, wGateUp, wDown, activation, needX || needGateUp);
    ctx->saved_data["activation"] = activation;
    ctx->saved_data["needs"] = int64_t(needX) | int64_t(needGateUp) << 1 | int64_t(needDown) << 2;
    ctx->save_for_backward({x, wGateUp, wDown, needDown ? h : Tensor(), saved});
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    const Tensor &x = s[0], &wGateUp = s[1], &wDown = s[2], &h = s[3], &saved = s[4];
    int64_t needs = ctx->saved_data["needs"].toInt();
    for (int i = 0; i < 3; ++i) if (!ctx->needs_input_grad(size_t(i))) needs &= ~(int64_t(1) << i);      // (a pass that asks for some of them only)
    const int64_t tokens = x.size(0), hidden = wDown.size(0), intermediate = wDown.size(1);
    Tensor dx, dGateUp, dDown, dz;
    if (!grads[0].defined()) return {dx, dGateUp, dDown, Tensor()};
    refuseTangents("gated_ffn's backward pass", {&grads[0]});
    const bool again = at::GradMode::is_enabled() && (grads[0].requires_grad() || needs);
    {
      at::AutoGradMode off(false);
      const c10::cuda::CUDAGuard guard(x.device());
      if (needs & 1) dx = at::empty_like(x);
      if (needs & 2) dGateUp = at::empty_like(wGateUp);
      if (needs & 4) dDown = at::empty_like(wDown);
      if (tokens == 0) {
        if (dGateUp.defined()) dGateUp.zero_();
        if (dDown.defined()) dDown.zero_();
      } else {
        Tensor dy = grads[0].contiguous();
        if (reinterpret_cast<uintptr_t>(dy.data_ptr()) % 16) dy = dy.clone();
        if (needs & 3) dz = at::empty({tokens, 2 * intermediate}, x.options());
        Tensor work;
        if (const size_t n = purlin_ffn_workspace_bytes(narrow(tokens), narrow(hidden), narrow(intermediate), int(needs & 1), int(needs & 2), int(needs & 4))) work = bytes(int64_t(n), x);
        check(purlin_ffn_backward(x.data_ptr(), wGateUp.data_ptr(), wDown.data_ptr(), ptr(h), ptr(saved), dy.data_ptr(), ptr(dz), ptr(dx), ptr(dGateUp), ptr(dDown), ptr(work),
                                  work.defined() ? size_t(work.numel()) : 0, narrow(tokens), narrow(hidden), narrow(intermediate), int(ctx->saved_data["activation"].toInt()), status(x), stream()));
      }
    }
    variable_list out{dx, dGateUp, dDown};
    if (again) {      // a graph through these gradients would be cut here without a word: whoever differentiates them is told
      auto error = std::make_shared<torch::autograd::Error>("gated_ffn is differentiable once", torch::autograd::collect_next_edges(x, wGateUp, wDown, grads[0]));
      for (Tensor& t : out) if (t.defined()) torch::autograd::create_gradient_edge(t, error);
    }
    out.emplace_back();
    return out;
  }
};

Tensor gatedFfn(const Tensor& x, const Tensor& wGateUp, const Tensor& wDown, int64_t activation) {
  refuseTangents("gated_ffn", {&x, &wGateUp, &wDown});
  if (at::GradMode::is_enabled() && (x.requires_grad() || wGateUp.requires_grad() || wDown.requires_grad())) return GatedFfn::apply(x, wGateUp, wDown, activation);
  return std::get<0>(ffnForward(x, wGateUp, wDown, activation, false));
}

std::tuple<Tensor, Tensor> quantize(const Tensor& x, int64_t type, int64_t rows, int64_t cols) {
  refuseTangents("a 4-bit quantisation", {&x});
  const c10::cuda::CUDAGuard guard(x.device());
  Tensor data = at::empty({rows, cols / 2}, x.options().dtype(at::kByte)), scales = bytes(int64_t(purlin_mx4_scale_bytes(narrow(rows), narrow(cols))), x);
  if (rows) check(purlin_mx4_quantize(x.data_ptr(), int(type), data.data_ptr(), scales.data_ptr(), narrow(rows), narrow(cols), stream()));
  return {data, scales};
}

Tensor dequantize(const Tensor& data, const Tensor& scales, int64_t type) {
  const c10::cuda::CUDAGuard guard(data.device());
  const int64_t rows = data.size(0), cols = 2 * data.size(1);
  Tensor out = at::empty({rows, cols}, data.options().dtype(type == PURLIN_MX4_FP32 ? at::kFloat : at::kBFloat16));
  if (rows) check(purlin_mx4_dequantize(data.data_ptr(), scales.data_ptr(), out.data_ptr(), int(type), narrow(rows), narrow(cols), stream()));
  return out;
}

bool overlap(const Tensor& a, const Tensor& b) {
  const auto x = reinterpret_cast<uintptr_t>(a.data_ptr()), y = reinterpret_cast<uintptr_t>(b.data_ptr());
  return x < y + b.nbytes() && y < x + a.nbytes();
}

// out[rows of a, N or N / 2]; `a` is dense of type `type`, or quantised with its scales
void multiply(const Tensor& a, int64_t type, const std::optional<Tensor>& aScales, const Tensor& wData, const Tensor& wScales, const Tensor& out, int64_t rows, int64_t epilogue) {
  const c10::cuda::CUDAGuard guard(wData.device());
  const int64_t n = wData.size(0), k = 2 * wData.size(1);
  if (overlap(out, wData) || overlap(out, wScales) || (aScales && (overlap(out, a) || overlap(out, *aScales)))) throw std::invalid_argument("out overlaps a quantised operand");
  if (aScales) {
    check(purlin_mx4_gemm(a.data_ptr(), aScales->data_ptr(), wData.data_ptr(), wScales.data_ptr(), out.data_ptr(), narrow(rows), narrow(n), narrow(k), int(epilogue), status(wData), stream()));
  } else {
    Tensor work;
    size_t size = purlin_mx4_workspace_bytes(int(type), narrow(rows), narrow(k));
    if (!size && overlap(out, a)) size = size_t(rows) * size_t(k) / 2 + purlin_mx4_scale_bytes(narrow(rows), narrow(k));
    if (size) work = bytes(int64_t(size), wData);
    check(purlin_mx4_linear(a.data_ptr(), int(type), ptr(work), wData.data_ptr(), wScales.data_ptr(), out.data_ptr(), narrow(rows), narrow(n), narrow(k), int(epilogue), status(wData), stream()));
  }
}
// Nothing here is differentiable. A result that was computed from a tensor with a gradient says so to whoever differentiates it; with `out`, which is
// written in place, such a call is refused, as torch's own functions do.
constexpr char kNoGradient[] = "a 4-bit product is not differentiable";
void product(const Tensor& a, int64_t type, const std::optional<Tensor>& aScales, const Tensor& wData, const Tensor& wScales, const Tensor& out, int64_t rows, int64_t epilogue) {
  refuseTangents("a 4-bit product", {&a, &out});
  if (at::GradMode::is_enabled() && (a.requires_grad() || out.requires_grad()))
    throw std::runtime_error("a 4-bit product with out is not differentiable, but one of its arguments requires a gradient");
  if (rows) multiply(a, type, aScales, wData, wScales, out, rows, epilogue);
  if (!out.is_inference()) out.unsafeGetTensorImpl()->bump_version();      // a graph that kept the old values notices
}
Tensor newProduct(const Tensor& a, int64_t type, const std::optional<Tensor>& aScales, const Tensor& wData, const Tensor& wScales, std::vector<int64_t> shape, int64_t rows,
                  int64_t epilogue) {
  refuseTangents("a 4-bit product", {&a});
  Tensor out = at::empty(shape, wData.options().dtype(at::kBFloat16));
  if (rows) multiply(a, type, aScales, wData, wScales, out, rows, epilogue);
  if (at::GradMode::is_enabled() && a.requires_grad())
    torch::autograd::create_gradient_edge(out, std::make_shared<torch::autograd::Error>(kNoGradient, torch::autograd::collect_next_edges(a)));
  return out;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  using release = py::call_guard<py::gil_scoped_release>;
  m.def("wait_words", [](int64_t device) { return reinterpret_cast<uintptr_t>(waitWords(device)); });
  m.def("take_wait_report", &takeWaitReport);
  m.def("gated_ffn", &gatedFfn, release());
  m.def("mx4_quantize", &quantize, release());
  m.def("mx4_dequantize", &dequantize, release());
  m.def("mx4_product", &product, release());
  m.def("mx4_new_product", &newProduct, release());
}
