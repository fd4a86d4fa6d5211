// awq_torch_ext.cpp -- the PyTorch-facing host glue of the drop-in, in C++.
//
// kernels.awq_gemm.awq_gemm_forward (songqiuyu/Qwen2-7B-Triton_Engine kernels/awq_gemm.py:
// 237-284) runs once per linear layer per decode step, so its host cost is paid 112 times
// per token of Qwen2-7B.  This module does the per-call work of awq_b200.gemm --
// argument checks, the output allocation, the current stream, the per-(device, stream)
// split-K workspace -- in C++ and calls the library through its C ABI
// (include/awq_b200.h; no torch types cross that boundary).  The Python package uses it
// when it is built and keeps its ctypes path otherwise; both call the same entry points.
//
// Errors: the same exception types as the Python path -- TypeError for dtypes,
// ValueError for shapes, devices and CPU tensors ("... CUDA only ..."), and the
// package's AwqError (registered by set_error_class) for a non-zero return code.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <map>
#include <mutex>
#include <string>
#include <tuple>
#include <vector>

#include "../../include/awq_b200.h"

namespace {

PyObject* g_error_class = nullptr;   // awq_b200._lib.AwqError

[[noreturn]] void raise_awq(int rc) {
  const char* msg = awq_last_error();
  if (g_error_class) {
    PyObject* exc = PyObject_CallFunction(g_error_class, "is", rc, msg ? msg : "");
    if (exc) {
      PyErr_SetObject(g_error_class, exc);
      Py_DECREF(exc);
    }
    throw pybind11::error_already_set();
  }
  TORCH_CHECK(false, "libawq_b200 error ", rc, ": ", msg ? msg : "");
}

void require_cuda(const at::Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.is_cuda(), name, " is on ", t.device().str(),
                    "; the AWQ kernels run on CUDA only (no CPU fallback)");
}

// Contiguous and 16-byte aligned (copies only when needed).
at::Tensor dense16(const at::Tensor& t) {
  at::Tensor r = t.is_contiguous() ? t : t.contiguous();
  if (reinterpret_cast<uintptr_t>(r.data_ptr()) % 16) r = r.clone();
  return r;
}

// Validates the packed layout (model/qwen2.py:34-36); returns (K, N) with N =
// scales.shape[1] as in awq_gemm_forward (kernels/awq_gemm.py:247).
std::pair<int64_t, int64_t> check_weights(const at::Tensor& qw, const at::Tensor& qz,
                                          const at::Tensor& s, int64_t gs) {
  require_cuda(qw, "qweight");
  require_cuda(qz, "qzeros");
  require_cuda(s, "scales");
  TORCH_CHECK_VALUE(qw.dim() == 2 && qz.dim() == 2 && s.dim() == 2,
                    "qweight, qzeros and scales must be 2-D");
  TORCH_CHECK_TYPE(qw.scalar_type() == at::kInt && qz.scalar_type() == at::kInt,
                   "qweight and qzeros must be int32");
  TORCH_CHECK_TYPE(s.scalar_type() == at::kHalf, "scales must be float16");
  TORCH_CHECK_VALUE(qw.device() == qz.device() && qw.device() == s.device(),
                    "qweight, qzeros and scales must be on one device");
  const int64_t K = qw.size(0), N = s.size(1);
  TORCH_CHECK_VALUE(qw.size(1) * 8 == N, "scales.shape[1]=", N, " but qweight packs ",
                    qw.size(1) * 8, " columns");
  TORCH_CHECK_VALUE(gs > 0 && K % gs == 0, "K=", K, " is not a multiple of group_size=", gs);
  const int64_t G = K / gs;
  TORCH_CHECK_VALUE(qz.size(0) == G && qz.size(1) == N / 8 && s.size(0) == G,
                    "qzeros / scales do not match [K/group_size=", G, ", N/8=", N / 8, "] / [",
                    G, ", ", N, "]");
  return {K, N};
}

// Zero-initialised split-K workspace per (device, stream), grown on demand.  The kernels
// leave its counters at zero after every call, so it is zeroed once per allocation.  The calls
// that a stream records into one graph share a workspace of that graph's own memory, whose
// counters the graph zeroes: graphs may replay beside one another and beside other calls, and
// none is left with memory that a later, larger call has given back.
std::mutex g_mu;
std::map<std::pair<int, cudaStream_t>, at::Tensor> g_ws;
struct CaptureWorkspace {
  unsigned long long id = 0;      // of the capture
  at::Tensor ws;
};
std::map<std::pair<int, cudaStream_t>, CaptureWorkspace> g_capture_ws;
constexpr size_t kCounterBytes = 64 * 1024;   // head of a workspace that must start at zero
std::map<std::tuple<int, int64_t, int64_t, int64_t, int64_t, bool>, size_t> g_need;

size_t workspace_need(int dev, int64_t M, int64_t N, int64_t K, int64_t gs, bool silu) {
  const auto key = std::make_tuple(dev, M, N, K, gs, silu);
  {
    std::lock_guard<std::mutex> lk(g_mu);
    auto it = g_need.find(key);
    if (it != g_need.end()) return it->second;
  }
  const size_t need = silu ? awq_gemm_silu_mul_workspace_bytes(M, N, K, gs)
                           : awq_gemm_workspace_bytes(M, N, K, gs);
  std::lock_guard<std::mutex> lk(g_mu);
  if (g_need.size() > 65536) g_need.clear();
  g_need[key] = need;
  return need;
}

at::Tensor workspace_for(const at::Device& dev, cudaStream_t st, size_t need) {
  cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  if (cudaStreamGetCaptureInfo(st, &cap, &id) != cudaSuccess) {
    (void)cudaGetLastError();      // the launch that follows reports what is wrong
    cap = cudaStreamCaptureStatusNone;
  }
  const int64_t size = need > (size_t)(1 << 20) ? (int64_t)need : (int64_t)(1 << 20);
  const auto options = at::TensorOptions().dtype(at::kByte).device(dev);
  const std::pair<int, cudaStream_t> key(dev.index(), st);
  std::lock_guard<std::mutex> lk(g_mu);
  if (cap == cudaStreamCaptureStatusActive) {
    CaptureWorkspace& c = g_capture_ws[key];
    if (!c.ws.defined() || c.id != id || (size_t)c.ws.numel() < need) {
      at::Tensor ws = at::empty({size}, options);
      if (const int rc = awq_workspace_init(ws.data_ptr(), kCounterBytes, st)) raise_awq(rc);
      c.ws = ws;
      c.id = id;
    }
    return c.ws;
  }
  if (!g_capture_ws.empty()) g_capture_ws.erase(key);
  at::Tensor& ws = g_ws[key];
  if (!ws.defined() || (size_t)ws.numel() < need) ws = at::zeros({size}, options);
  return ws;
}

// The product behind gemm / forward: out fp16 [M, N] (or [M, N/2] with silu) on the
// current stream.
at::Tensor gemm_impl(at::Tensor x, at::Tensor qw, at::Tensor qz, at::Tensor s, int64_t gs,
                     int64_t path, c10::optional<at::Tensor> out_opt,
                     c10::optional<at::Tensor> bias_opt, bool silu) {
  auto [K, N] = check_weights(qw, qz, s, gs);
  qw = dense16(qw);
  qz = dense16(qz);
  s = dense16(s);
  require_cuda(x, "x");
  TORCH_CHECK_TYPE(x.scalar_type() == at::kHalf, "x must be float16, got ", x.scalar_type());
  TORCH_CHECK_VALUE(x.dim() == 2 && x.size(1) == K, "x must be [M, K=", K, "], got ", x.sizes());
  TORCH_CHECK_VALUE(x.device() == qw.device(), "x and the weights must be on one device");
  if (silu) TORCH_CHECK_VALUE(N % 2 == 0, "N=", N, " is not even: no gate / up halves");
  at::Tensor bias;
  if (bias_opt.has_value() && bias_opt->defined()) {
    bias = *bias_opt;
    require_cuda(bias, "bias");
    TORCH_CHECK_VALUE(bias.scalar_type() == at::kHalf && bias.dim() == 1 && bias.size(0) == N,
                      "bias must be float16 [N=", N, "]");
    TORCH_CHECK_VALUE(path == AWQ_PATH_AUTO, "the bias epilogue runs on the automatic kernel choice only");
    bias = bias.contiguous();
  }
  const int64_t M = x.size(0);
  const int64_t NO = silu ? N / 2 : N;
  at::Tensor out = out_opt.has_value() && out_opt->defined()
                       ? *out_opt
                       : at::empty({M, NO}, x.options());
  if (M == 0) return out;
  if (x.stride(1) != 1 || reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 || (x.stride(0) * 2) % 16) {
    x = x.contiguous();
    if (reinterpret_cast<uintptr_t>(x.data_ptr()) % 16) x = x.clone();
  }
  const c10::cuda::CUDAGuard guard(x.device());
  cudaStream_t st = at::cuda::getCurrentCUDAStream(x.device().index()).stream();
  const size_t need = workspace_need(x.device().index(), M, N, K, gs, silu);
  at::Tensor ws;
  if (need) ws = workspace_for(x.device(), st, need);
  void* wsp = ws.defined() ? ws.data_ptr() : nullptr;
  const size_t wsn = ws.defined() ? (size_t)ws.numel() : 0;
  int rc;
  if (silu) {
    rc = awq_gemm_f16_silu_mul(x.data_ptr(), x.stride(0), qw.data_ptr<int32_t>(), qz.data_ptr<int32_t>(),
                               s.data_ptr(), out.data_ptr(), out.stride(0), M, N, K, gs, wsp, wsn, st);
  } else if (bias.defined()) {
    rc = awq_gemm_f16_bias(x.data_ptr(), x.stride(0), qw.data_ptr<int32_t>(), qz.data_ptr<int32_t>(),
                           s.data_ptr(), bias.data_ptr(), out.data_ptr(), out.stride(0), M, N, K, gs,
                           wsp, wsn, st);
  } else {
    rc = awq_gemm_f16_ex(x.data_ptr(), x.stride(0), qw.data_ptr<int32_t>(), qz.data_ptr<int32_t>(),
                         s.data_ptr(), out.data_ptr(), out.stride(0), M, N, K, gs, wsp, wsn, st,
                         (int)path);
  }
  if (rc != AWQ_OK) raise_awq(rc);
  return out;
}

// awq_gemm_forward's shape handling (kernels/awq_gemm.py:244-284): x [..., K] -> [..., N].
at::Tensor forward_impl(const at::Tensor& x, const at::Tensor& qw, const at::Tensor& qz,
                        const at::Tensor& s, int64_t gs, c10::optional<at::Tensor> bias, bool silu) {
  TORCH_CHECK_VALUE(x.dim() >= 1, "x must have at least one dimension");
  const int64_t N = s.dim() == 2 ? s.size(1) : 0;
  at::Tensor out = gemm_impl(x.reshape({-1, x.size(-1)}), qw, qz, s, gs, AWQ_PATH_AUTO,
                             c10::nullopt, bias, silu);
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end() - 1);
  shape.push_back(silu ? N / 2 : N);
  return out.view(shape);
}

// ---- the operators between the products (awq_b200/layer.py has the same steps in Python) ----

using OptTensor = c10::optional<at::Tensor>;

bool given(const OptTensor& t) { return t.has_value() && t->defined(); }

void need(const at::Tensor& t, const char* name, at::ScalarType dtype, int64_t ndim,
          const at::Device* dev = nullptr) {
  require_cuda(t, name);
  TORCH_CHECK_TYPE(t.scalar_type() == dtype, name, " must be ", c10::toString(dtype), ", got ",
                   t.scalar_type());
  TORCH_CHECK_VALUE(t.dim() == ndim, name, " must be ", ndim, "-D, got shape ", t.sizes());
  if (dev) TORCH_CHECK_VALUE(t.device() == *dev, name, " is on ", t.device().str(), ", expected ", dev->str());
}

// A contiguous tensor of exactly this shape (state and outputs, never copied).
void need_dense(const at::Tensor& t, const char* name, at::ScalarType dtype, at::IntArrayRef shape,
                const at::Device& dev) {
  need(t, name, dtype, (int64_t)shape.size(), &dev);
  TORCH_CHECK_VALUE(t.sizes() == shape && t.is_contiguous(), name, " must be a contiguous ", shape,
                    " tensor, got ", t.sizes());
}

at::Tensor last_dense(const at::Tensor& t) {
  return t.size(-1) == 1 || t.stride(-1) == 1 ? t : t.contiguous();
}

// Whether the address ranges of two tensors overlap.
bool overlap(const at::Tensor& a, const at::Tensor& b) {
  auto span = [](const at::Tensor& t) {
    int64_t last = t.numel() ? 0 : -1;
    if (t.numel())
      for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * std::abs(t.stride(d));
    const char* p = static_cast<const char*>(t.data_ptr());
    return std::make_pair(p, p + (last + 1) * t.element_size());
  };
  const auto x = span(a), y = span(b);
  return x.first < y.second && y.first < x.second;
}

// Different columns of the same rows (views of one fused q/k/v tensor).
bool apart(const at::Tensor& o, const at::Tensor& y) {
  if (o.stride(0) != y.stride(0) || o.stride(0) <= 0 || o.stride(1) < 0 || y.stride(1) < 0) return false;
  const int64_t row = o.stride(0) * 2;
  auto cols = [](const at::Tensor& t) { return (t.size(1) - 1) * t.stride(1) * 2 + t.size(2) * 2; };
  int64_t d = (static_cast<const char*>(y.data_ptr()) - static_cast<const char*>(o.data_ptr())) % row;
  if (d < 0) d += row;
  return cols(o) <= d && d + cols(y) <= row;
}

// Whether no two rows of t [T, H, D] (last dimension dense) share an element: heads within tokens
// or tokens within heads, not expanded ones.
bool distinct(const at::Tensor& t) {
  const int64_t T = t.size(0), H = t.size(1), D = t.size(2), ts = t.stride(0), hs = t.stride(1);
  return t.numel() == 0 || ((H == 1 || hs >= D) && (T == 1 || ts >= (H - 1) * hs + D)) ||
         ((T == 1 || ts >= D) && (H == 1 || hs >= (T - 1) * ts + D));
}

uintptr_t address(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()); }

void check(int rc) {
  if (rc != AWQ_OK) raise_awq(rc);
}

int activation_code(const c10::optional<std::string>& name) {
  static const std::map<std::string, int> codes = {{"none", AWQ_ACT_NONE}, {"relu", AWQ_ACT_RELU},
                                                   {"silu", AWQ_ACT_SILU}, {"gelu", AWQ_ACT_GELU},
                                                   {"gelu_tanh", AWQ_ACT_GELU_TANH}};
  if (!name.has_value()) return AWQ_ACT_NONE;
  const auto it = codes.find(*name);
  TORCH_CHECK_VALUE(it != codes.end(), "activation '", *name,
                    "' is none of gelu, gelu_tanh, none, relu, silu");
  return it->second;
}

at::Tensor gemm_epilogue(at::Tensor x, at::Tensor qw, at::Tensor qz, at::Tensor s, int64_t gs,
                         OptTensor bias_opt, const c10::optional<std::string>& activation,
                         OptTensor res_opt, OptTensor out_opt) {
  auto [K, N] = check_weights(qw, qz, s, gs);
  qw = dense16(qw);
  qz = dense16(qz);
  s = dense16(s);
  require_cuda(x, "x");
  TORCH_CHECK_TYPE(x.scalar_type() == at::kHalf, "x must be float16, got ", x.scalar_type());
  TORCH_CHECK_VALUE(x.dim() == 2 && x.size(1) == K, "x must be [M, K=", K, "], got ", x.sizes());
  TORCH_CHECK_VALUE(x.device() == qw.device(), "x and the weights must be on one device");
  const at::Device dev = x.device();
  const int64_t M = x.size(0);
  const int act = activation_code(activation);
  at::Tensor bias, res;
  if (given(bias_opt)) {
    bias = *bias_opt;
    need(bias, "bias", at::kHalf, 1, &dev);
    TORCH_CHECK_VALUE(bias.size(0) == N, "bias must be [", N, "], got ", bias.sizes());
  }
  if (given(res_opt)) {
    res = *res_opt;
    need(res, "residual", at::kHalf, 2, &dev);
    TORCH_CHECK_VALUE(res.size(0) == M && res.size(1) == N, "residual must be [", M, ", ", N, "], got ", res.sizes());
  }
  at::Tensor out;
  if (given(out_opt)) {
    out = *out_opt;
    need(out, "out", at::kHalf, 2, &dev);
    TORCH_CHECK_VALUE(out.size(0) == M && out.size(1) == N && out.stride(1) == 1 &&
                          (M <= 1 || out.stride(0) >= N) && address(out) % 16 == 0 && out.stride(0) % 8 == 0,
                      "out must be a [", M, ", ", N, "] tensor with dense, 16-byte aligned rows");
    const bool same = res.defined() && out.data_ptr() == res.data_ptr() && out.strides() == res.strides();
    TORCH_CHECK_VALUE(!overlap(out, x) && !(bias.defined() && overlap(out, bias)) &&
                          !(res.defined() && !same && overlap(out, res)),
                      "out overlaps an input (it may only be the residual itself)");
  } else {
    out = at::empty({M, N}, x.options());
  }
  if (M == 0) return out;
  if (bias.defined()) bias = bias.contiguous();
  if (res.defined() && (res.stride(1) != 1 || (M > 1 && res.stride(0) < N))) res = res.contiguous();
  if (x.stride(1) != 1 || address(x) % 16 || (x.stride(0) * 2) % 16 || (M > 1 && x.stride(0) < K)) {
    x = x.contiguous();
    if (address(x) % 16) x = x.clone();
  }
  const c10::cuda::CUDAGuard guard(dev);
  cudaStream_t st = at::cuda::getCurrentCUDAStream(dev.index()).stream();
  const size_t nb = workspace_need(dev.index(), M, N, K, gs, false);
  at::Tensor ws;
  if (nb) ws = workspace_for(dev, st, nb);
  check(awq_gemm_f16_epilogue(x.data_ptr(), std::max(x.stride(0), K), qw.data_ptr<int32_t>(),
                              qz.data_ptr<int32_t>(), s.data_ptr(), bias.defined() ? bias.data_ptr() : nullptr,
                              act, res.defined() ? res.data_ptr() : nullptr,
                              res.defined() ? std::max(res.stride(0), N) : 0, out.data_ptr(),
                              std::max(out.stride(0), N), M, N, K, gs, ws.defined() ? ws.data_ptr() : nullptr,
                              ws.defined() ? (size_t)ws.numel() : 0, st));
  return out;
}

std::tuple<at::Tensor, at::Tensor> rope_axes(at::Tensor q, at::Tensor k, at::Tensor pos,
                                             const at::Tensor& inv_freq, const std::vector<int64_t>& sections,
                                             bool interleaved, OptTensor out_q, OptTensor out_k) {
  need(q, "q", at::kHalf, 3);
  const at::Device dev = q.device();
  need(k, "k", at::kHalf, 3, &dev);
  const int64_t T = q.size(0), D = q.size(2), A = (int64_t)sections.size();
  TORCH_CHECK_VALUE(k.size(0) == T && k.size(2) == D, "k ", k.sizes(), " does not match q ", q.sizes());
  int64_t half = 0;
  bool ok = A >= 1 && A <= 4;
  int32_t sec[4] = {};
  for (int64_t i = 0; i < A && ok; ++i) {
    ok = sections[i] >= 0 && sections[i] <= D;
    sec[i] = (int32_t)sections[i];
    half += sections[i];
  }
  TORCH_CHECK_VALUE(ok && half >= 1 && 2 * half <= D, "sections=", sections,
                    " must be 1 to 4 counts that rotate 2 to ", D, " channels");
  require_cuda(pos, "positions");
  if (pos.dim() == 1) pos = pos.unsqueeze(0);
  TORCH_CHECK_TYPE(pos.scalar_type() == at::kLong || pos.scalar_type() == at::kInt,
                   "positions must be int64 or int32, got ", pos.scalar_type());
  need(pos, "positions", pos.scalar_type(), 2, &dev);
  TORCH_CHECK_VALUE(pos.size(0) == A && pos.size(1) == T, "positions must be [", A, ", ", T, "], got ", pos.sizes());
  need_dense(inv_freq, "inv_freq", at::kFloat, {half}, dev);
  if (T) pos = last_dense(pos);
  if (T) q = last_dense(q), k = last_dense(k);
  at::Tensor outs[2];
  const OptTensor* asked[2] = {&out_q, &out_k};
  const at::Tensor ins[2] = {q, k};
  for (int i = 0; i < 2; ++i) {
    if (!given(*asked[i])) {
      outs[i] = at::empty(ins[i].sizes(), ins[i].options());
      continue;
    }
    const char* name = i ? "out_k" : "out_q";
    const at::Tensor& o = **asked[i];
    need(o, name, at::kHalf, 3, &dev);
    TORCH_CHECK_VALUE(o.sizes() == ins[i].sizes() && (D == 1 || o.stride(2) == 1) && distinct(o), name,
                      " must be ", ins[i].sizes(), " with a dense last dimension and rows that share no element");
    const bool same = o.data_ptr() == ins[i].data_ptr() && o.strides() == ins[i].strides();
    for (int j = 0; j < 2; ++j)
      TORCH_CHECK_VALUE(!overlap(o, ins[j]) || (same && i == j) || apart(o, ins[j]), name,
                        " overlaps an input other than as that input itself");
    outs[i] = o;
  }
  TORCH_CHECK_VALUE(!overlap(outs[0], outs[1]) || apart(outs[0], outs[1]), "out_q overlaps out_k");
  if (T == 0) return {outs[0], outs[1]};
  const c10::cuda::CUDAGuard guard(dev);
  check(awq_rope_axes(q.data_ptr(), q.stride(0), q.stride(1), q.size(1), k.data_ptr(), k.stride(0), k.stride(1),
                      k.size(1), T, D, pos.data_ptr(), pos.scalar_type() == at::kLong, pos.stride(0),
                      inv_freq.data_ptr<float>(), sec, (int)A, interleaved, outs[0].data_ptr(), outs[0].stride(0),
                      outs[0].stride(1), outs[1].data_ptr(), outs[1].stride(0), outs[1].stride(1),
                      at::cuda::getCurrentCUDAStream(dev.index()).stream()));
  return {outs[0], outs[1]};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> kv4_pages_step(
    const at::Tensor& table, const at::Tensor& held, const at::Tensor& free_pages, const at::Tensor& free_count,
    const at::Tensor& kv_lens, const at::Tensor& new_tokens, int64_t page_size, int64_t max_tokens,
    OptTensor reset) {
  need(table, "block_table", at::kInt, 2);
  const at::Device dev = table.device();
  const int64_t R = table.size(0), width = table.size(1);
  TORCH_CHECK_VALUE((!width || width == 1 || table.stride(1) == 1) && (R <= 1 || table.stride(0) >= width),
                    "block_table must have dense, non-overlapping rows");
  need_dense(held, "held", at::kInt, {R}, dev);
  need(free_pages, "free_pages", at::kInt, 1, &dev);
  TORCH_CHECK_VALUE(free_pages.is_contiguous(), "free_pages must be contiguous");
  need_dense(free_count, "free_count", at::kInt, {1}, dev);
  need_dense(kv_lens, "kv_lens", at::kInt, {R}, dev);
  need_dense(new_tokens, "new_tokens", at::kInt, {R}, dev);
  if (given(reset)) {
    require_cuda(*reset, "reset");
    TORCH_CHECK_TYPE(reset->scalar_type() == at::kBool || reset->scalar_type() == at::kByte,
                     "reset must be bool or uint8, got ", reset->scalar_type());
    need_dense(*reset, "reset", reset->scalar_type(), {R}, dev);
  }
  TORCH_CHECK_VALUE(page_size >= 1 && max_tokens >= 0, "page_size must be positive and max_tokens not negative");
  at::Tensor slots = at::empty({max_tokens}, table.options().dtype(at::kLong));
  at::Tensor ints = at::empty({max_tokens + 2 * R + 2}, table.options());
  int32_t* p = ints.data_ptr<int32_t>();
  const c10::cuda::CUDAGuard guard(dev);
  check(awq_kv4_pages_step(table.data_ptr<int32_t>(), R > 1 ? table.stride(0) : width, width,
                           held.data_ptr<int32_t>(), free_pages.data_ptr<int32_t>(), free_pages.numel(),
                           free_count.data_ptr<int32_t>(), kv_lens.data_ptr<int32_t>(),
                           new_tokens.data_ptr<int32_t>(),
                           given(reset) ? static_cast<const uint8_t*>(reset->data_ptr()) : nullptr, R, page_size,
                           slots.data_ptr<int64_t>(), p, max_tokens, p + max_tokens, p + max_tokens + R + 1,
                           p + max_tokens + 2 * R + 1, at::cuda::getCurrentCUDAStream(dev.index()).stream()));
  return {slots, ints.narrow(0, 0, max_tokens), ints.narrow(0, max_tokens, R + 1),
          ints.narrow(0, max_tokens + R + 1, R), ints.narrow(0, max_tokens + 2 * R + 1, 1)};
}

void kv4_append(at::Tensor k, at::Tensor v, at::Tensor slots, const at::Tensor& data, int64_t D, int64_t page,
                int64_t group) {
  require_cuda(data, "cache.data");
  const at::Device dev = data.device();
  need(k, "k", at::kHalf, 3, &dev);
  need(v, "v", at::kHalf, 3, &dev);
  need(slots, "slots", at::kLong, 1, &dev);
  const int64_t T = slots.size(0), H = data.size(1);
  const int64_t want[3] = {T, H, D};
  TORCH_CHECK_VALUE(k.sizes() == at::IntArrayRef(want, 3) && v.sizes() == at::IntArrayRef(want, 3), "k ", k.sizes(),
                    " and v ", v.sizes(), " must be [", T, ", ", H, ", ", D, "]");
  if (T == 0) return;
  k = last_dense(k);
  v = last_dense(v);
  slots = slots.contiguous();
  const c10::cuda::CUDAGuard guard(dev);
  check(awq_kv4_append(k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1),
                       slots.data_ptr<int64_t>(), T, data.data_ptr(), data.size(0), H, D, group, page,
                       at::cuda::getCurrentCUDAStream(dev.index()).stream()));
}

std::tuple<at::Tensor, at::Tensor> kv4_gather(const at::Tensor& data, int64_t D, int64_t page, int64_t group,
                                              at::Tensor slots) {
  require_cuda(data, "cache.data");
  const at::Device dev = data.device();
  need(slots, "slots", at::kLong, 1, &dev);
  const int64_t T = slots.size(0), H = data.size(1);
  at::Tensor k = at::empty({T, H, D}, data.options().dtype(at::kHalf)), v = at::empty_like(k);
  if (T == 0) return {k, v};
  slots = slots.contiguous();
  const c10::cuda::CUDAGuard guard(dev);
  check(awq_kv4_gather(data.data_ptr(), data.size(0), H, D, group, page, slots.data_ptr<int64_t>(), T, k.data_ptr(),
                       v.data_ptr(), at::cuda::getCurrentCUDAStream(dev.index()).stream()));
  return {k, v};
}

at::Tensor kv4_attention(at::Tensor q, const at::Tensor& data, int64_t D, int64_t page, int64_t group,
                         at::Tensor table, const at::Tensor& kv_lens, OptTensor cu_q, int64_t max_q,
                         c10::optional<double> scale, OptTensor out_opt) {
  require_cuda(data, "cache.data");
  const at::Device dev = data.device();
  need(q, "q", at::kHalf, 3, &dev);
  const int64_t T = q.size(0), H = q.size(1), Hk = data.size(1);
  TORCH_CHECK_VALUE(q.size(2) == D, "q has head_dim ", q.size(2), ", the cache ", D);
  TORCH_CHECK_VALUE(H >= 1 && H % Hk == 0, H, " query heads do not group over ", Hk, " kv heads");
  need(table, "block_table", at::kInt, 2, &dev);
  const int64_t R = table.size(0), width = table.size(1);
  if ((width > 1 && table.stride(1) != 1) || (R > 1 && table.stride(0) < width)) table = table.contiguous();
  need_dense(kv_lens, "kv_lens", at::kInt, {R}, dev);
  const bool ragged = given(cu_q);
  if (!ragged) {
    TORCH_CHECK_VALUE(T == R && max_q == 1, "without cu_q every request has one query row: ", T, " rows, ", R,
                      " requests, max_q=", max_q);
  } else {
    need_dense(*cu_q, "cu_q", at::kInt, {R + 1}, dev);
    TORCH_CHECK_VALUE(max_q >= 1, "max_q must be positive");
  }
  if (q.numel() && (q.stride(2) != 1 || address(q) % 16 || q.stride(0) % 8 || q.stride(1) % 8)) {
    q = q.contiguous();
    if (address(q) % 16) q = q.clone();
  }
  const c10::cuda::CUDAGuard guard(dev);
  at::Tensor out;
  if (given(out_opt)) {
    out = *out_opt;
    need(out, "out", at::kHalf, 3, &dev);
    TORCH_CHECK_VALUE(out.sizes() == q.sizes() && out.stride(2) == 1 && address(out) % 8 == 0 &&
                          out.stride(0) % 4 == 0 && out.stride(1) % 4 == 0 && distinct(out),
                      "out must be ", q.sizes(),
                      " with a dense last dimension, 8-byte aligned rows that share no element");
    TORCH_CHECK_VALUE(!overlap(out, q), "out overlaps q");
  } else {
    out = ragged ? at::zeros(q.sizes(), q.options()) : at::empty(q.sizes(), q.options());
  }
  if (T == 0 || R == 0) return out;
  const size_t nb = awq_kv4_attention_workspace_bytes(D, std::min(max_q, T) * (H / Hk));
  // a workspace of this call alone: graphs that replay at once must not share one
  at::Tensor ws = at::empty({(int64_t)nb}, data.options());
  check(awq_kv4_attention(q.data_ptr(), q.stride(0), q.stride(1), T, H, data.data_ptr(), data.size(0), Hk, D, group,
                          page, table.data_ptr<int32_t>(), R > 1 ? table.stride(0) : width, width,
                          kv_lens.data_ptr<int32_t>(), ragged ? cu_q->data_ptr<int32_t>() : nullptr, R, max_q,
                          (float)(scale.has_value() ? *scale : 1.0 / std::sqrt((double)D)), out.data_ptr(),
                          out.stride(0), out.stride(1), ws.data_ptr(), nb,
                          at::cuda::getCurrentCUDAStream(dev.index()).stream()));
  return out;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "C++ host glue of the AWQ drop-in (calls libawq_b200 through its C ABI)";
  m.def("set_error_class", [](pybind11::object cls) {
    Py_XDECREF(g_error_class);
    g_error_class = cls.ptr();
    Py_INCREF(g_error_class);
  });
  m.def("gemm", [](at::Tensor x, at::Tensor qw, at::Tensor qz, at::Tensor s, int64_t gs, int64_t path,
                   c10::optional<at::Tensor> out, c10::optional<at::Tensor> bias) {
          return gemm_impl(x, qw, qz, s, gs, path, out, bias, false);
        });
  m.def("gemm_silu_mul", [](at::Tensor x, at::Tensor qw, at::Tensor qz, at::Tensor s, int64_t gs,
                            c10::optional<at::Tensor> out) {
          return gemm_impl(x, qw, qz, s, gs, AWQ_PATH_AUTO, out, c10::nullopt, true);
        });
  m.def("forward", [](const at::Tensor& x, const at::Tensor& qw, const at::Tensor& qz,
                      const at::Tensor& s, int64_t gs) {
          return forward_impl(x, qw, qz, s, gs, c10::nullopt, false);
        });
  m.def("forward_bias", [](const at::Tensor& x, const at::Tensor& qw, const at::Tensor& qz,
                           const at::Tensor& s, const at::Tensor& bias, int64_t gs) {
          return forward_impl(x, qw, qz, s, gs, bias, false);
        });
  m.def("forward_silu_mul", [](const at::Tensor& x, const at::Tensor& qw, const at::Tensor& qz,
                               const at::Tensor& s, int64_t gs) {
          return forward_impl(x, qw, qz, s, gs, c10::nullopt, true);
        });
  m.def("workspace", [](int64_t device, int64_t stream, int64_t need) {   // of a call on that stream
    return workspace_for(at::Device(at::kCUDA, (c10::DeviceIndex)device),
                         reinterpret_cast<cudaStream_t>(stream), (size_t)need);
  });
  m.def("gemm_epilogue", &gemm_epilogue);
  m.def("rope_axes", &rope_axes);
  m.def("kv4_pages_step", &kv4_pages_step);
  m.def("kv4_append", &kv4_append);
  m.def("kv4_gather", &kv4_gather);
  m.def("kv4_attention", &kv4_attention);
}
