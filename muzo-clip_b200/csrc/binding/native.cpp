// Python module muzo_clip_b200._native: the gradient operators' calls from torch tensors to the C
// ABI, with their checks of arguments, their outputs and workspaces (torch's allocator, the current
// stream of the tensors' device) and their autograd node. A call's host side takes 9 to 16 us this
// way; the same steps in Python over ctypes took 30 to 60 us, and 200 us with the backward pass
// behind the interpreter lock: more than the kernels of a small model.
//
// The library's functions are handed over by address (bind), so that this module uses the very copy
// of libmuzo_b200.so that muzo_clip_b200._lib has loaded.
#include <torch/extension.h>

#include <ATen/cuda/CUDAContext.h>
#include <c10/core/InferenceMode.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>

#include <algorithm>
#include <array>
#include <cmath>
#include <mutex>
#include <optional>
#include <vector>

#include "muzo_b200.h"

namespace {

using torch::Tensor;
using OptTensor = std::optional<Tensor>;

// ---------------------------------------------------------------- the library

struct Library {
  decltype(&muzo_attention_max_lse) attention_forward = nullptr;
  decltype(&muzo_attention_backward) attention_backward = nullptr;
  decltype(&muzo_attention_backward_workspace) attention_workspace = nullptr;
  decltype(&muzo_grad_norm) grad_norm = nullptr;
  decltype(&muzo_grad_clip) grad_clip = nullptr;
  decltype(&muzo_grad_workspace) grad_workspace = nullptr;
  decltype(&muzo_status_string) status_string = nullptr;
  decltype(&muzo_last_cuda_error) last_cuda_error = nullptr;
};
Library lib;

struct Failure : std::runtime_error {
  using std::runtime_error::runtime_error;
};

void check(int status, const char* what) {
  if (status == MUZO_OK) return;
  std::string msg = std::string(what) + ": " + lib.status_string(status);
  if (status == MUZO_ERR_CUDA) msg += " (cudaError " + std::to_string(lib.last_cuda_error()) + ")";
  throw Failure(msg);
}

int dtype_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return MUZO_F32;
    case at::kBFloat16: return MUZO_BF16;
    case at::kHalf: return MUZO_F16;
    default: return -1;
  }
}

// Refuses what would be answered without its part: a tangent (forward-mode derivatives), torch.func's wrappers.
void check_plain(const Tensor& t, const char* what) {
  if (t.unsafeGetTensorImpl()->autograd_meta() != nullptr)
    TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(/*level=*/0).defined(), what, ": forward-mode derivatives are not supported");
  TORCH_CHECK_NOT_IMPLEMENTED(
      !t.key_set().has_any(c10::DispatchKeySet({c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper})),
      what, ": torch.func transforms (vmap, grad, jvp) are not supported");
}

void* stream_of(const Tensor& t) { return at::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

// ---------------------------------------------------------------- attention

// Two int32 words per GPU, shared by its attention launches: [0] the first nonzero timeout code, [1]
// a test's stall request. Created on first use, which may be under capture; they outlive any graph.
std::mutex status_mutex;
Tensor& status_words(int device) {
  static std::array<Tensor, 64>* words = new std::array<Tensor, 64>;   // never destroyed: tensors must not outlive CUDA
  TORCH_CHECK(device >= 0 && device < 64, "muzo_clip_b200: GPU index ", device);
  return (*words)[device];
}
// Whether any attention launch on the GPU can have used them.
bool attention_used(int device) {
  std::lock_guard<std::mutex> lock(status_mutex);
  return status_words(device).defined();
}
Tensor attention_status(int device) {
  std::lock_guard<std::mutex> lock(status_mutex);
  Tensor& t = status_words(device);
  if (t.defined()) return t;
  // On a stream of their own, which no capture can be on (a stream of torch's pool may be the capturing one: the
  // words would then lie in the graph's memory, and every replay would clear them), and cleared before any stream's
  // launch reads them.
  c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(device));
  c10::cuda::CUDAStreamCaptureModeGuard relaxed{cudaStreamCaptureModeRelaxed};
  c10::InferenceMode normal(false);   // a check outside it clears the words
  cudaStream_t own = nullptr;
  C10_CUDA_CHECK(cudaStreamCreateWithFlags(&own, cudaStreamNonBlocking));   // kept: the words' memory belongs to it
  Tensor fresh;
  {
    c10::cuda::CUDAStreamGuard side(c10::cuda::getStreamFromExternal(own, static_cast<c10::DeviceIndex>(device)));
    fresh = at::zeros({2}, at::TensorOptions().dtype(at::kInt).device(at::kCUDA, device));
  }
  C10_CUDA_CHECK(cudaStreamSynchronize(own));
  t = fresh;
  return t;
}

// Element strides of a [.., .., .., D] tensor's leading dimensions, as the kernels' 16-byte tile loads
// take them; a dimension of size 1 is never stepped over, and gets any valid stride.
using Strides = std::array<int64_t, 3>;

bool in_place(const Tensor& t, Strides& s) {
  for (int i = 0; i < 3; ++i) {
    s[i] = t.size(i) > 1 ? t.stride(i) : t.size(3);
    if (s[i] % 8 != 0 || s[i] <= 0) return false;
  }
  return (t.stride(3) == 1 || t.size(3) == 1) && reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0;
}

// `t`, copied where it could not be read in place (D strided, unaligned, expanded along a dimension).
Tensor readable(const Tensor& t, Strides& s) {
  if (in_place(t, s)) return t;
  Tensor c = t.clone(at::MemoryFormat::Contiguous);
  in_place(c, s);
  return c;
}

const void* ptr(const Tensor& t) { return t.numel() > 0 ? t.const_data_ptr() : nullptr; }
void* out_ptr(const Tensor& t) { return t.defined() && t.numel() > 0 ? t.data_ptr() : nullptr; }
const int32_t* range_ptr(const OptTensor& t) { return t ? t->const_data_ptr<int32_t>() : nullptr; }

// Refuses what the kernels do not compute; returns the scaling.
double check_attention(const Tensor& q, const Tensor& k, const Tensor& v, std::optional<double> scaling, const OptTensor& lo,
                       const OptTensor& hi) {
  for (const Tensor* t : {&q, &k, &v}) check_plain(*t, "attention_max");
  TORCH_CHECK_VALUE(q.dim() == 4 && k.dim() == 4 && v.dim() == 4,
                    "attention_max expects 4-D query, key and value [B, H, S, D]");
  TORCH_CHECK_VALUE(q.is_cuda(), "muzo_clip_b200 attention kernels run on CUDA tensors only");
  TORCH_CHECK_TYPE(q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf,
                   "attention_max supports bfloat16 and float16, not ", q.scalar_type());
  TORCH_CHECK_TYPE(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(),
                   "attention_max: query, key and value differ in type");
  TORCH_CHECK_VALUE(k.device() == q.device() && v.device() == q.device(),
                    "attention_max: query, key and value are on different devices");
  TORCH_CHECK_VALUE(k.sizes() == v.sizes() && k.size(0) == q.size(0) && k.size(3) == q.size(3), "attention_max: key ",
                    k.sizes(), " and value ", v.sizes(), " do not fit query ", q.sizes());
  TORCH_CHECK_VALUE(q.size(1) > 0 && k.size(1) > 0 && q.size(1) % k.size(1) == 0, "attention_max: ", q.size(1),
                    " query heads are not a multiple of ", k.size(1), " key heads");
  const int64_t d = q.size(3);
  TORCH_CHECK_VALUE(d % 8 == 0 && d >= 8 && d <= 128,
                    "attention_max supports head dimensions that are multiples of 8 up to 128, not ", d);
  for (const OptTensor* t : {&lo, &hi})
    TORCH_CHECK_VALUE(!*t || ((*t)->scalar_type() == at::kInt && (*t)->device() == q.device() && (*t)->dim() == 1 &&
                              (*t)->size(0) == q.size(0) && (*t)->is_contiguous()),
                      "attention_max: key_lo and key_hi must be contiguous int32 tensors of ", q.size(0), " values on ",
                      q.device());
  const double s = scaling ? *scaling : 1.0 / std::sqrt(static_cast<double>(d));
  TORCH_CHECK_VALUE(s > 0.0 && std::isfinite(static_cast<float>(s)) && static_cast<float>(s) > 0.0f,
                    "attention_max: the scaling must be positive and finite, not ", s);
  return s;
}

struct Forward {
  Tensor out, lse, smax, valid;
};

Forward attention_forward(const Tensor& query, const Tensor& key, const Tensor& value, double scaling, bool causal,
                          const OptTensor& lo, const OptTensor& hi, bool record, bool keep_lse) {
  const c10::cuda::CUDAGuard guard(query.device());
  const int64_t b = query.size(0), hq = query.size(1), sq = query.size(2), d = query.size(3);
  const int64_t hkv = key.size(1), sk = key.size(2);
  const auto opt = query.options();
  Forward f;
  f.out = at::empty({b, sq, hq, d}, opt);
  if (keep_lse) f.lse = at::empty({b, hq, sq}, opt.dtype(at::kFloat));
  if (f.out.numel() == 0) {
    if (record) {
      f.smax = at::full({hq}, -INFINITY, opt.dtype(at::kFloat));
      f.valid = at::ones({1}, opt.dtype(at::kInt));
    }
    return f;
  }
  if (record) {
    f.smax = at::empty({hq}, opt.dtype(at::kFloat));
    f.valid = at::empty({1}, opt.dtype(at::kInt));
  }
  Strides qs, ks, vs;
  const Tensor q = readable(query, qs), k = readable(key, ks), v = readable(value, vs);
  check(lib.attention_forward(ptr(q), ptr(k), ptr(v), f.out.data_ptr(), static_cast<float*>(out_ptr(f.lse)), dtype_code(q), b,
                              hq, hkv, sq, sk, d, qs[0], qs[1], qs[2], ks[0], ks[1], ks[2], vs[0], vs[1], vs[2],
                              sq * hq * d, d, hq * d, causal ? 1 : 0, static_cast<float>(scaling), range_ptr(lo),
                              range_ptr(hi), static_cast<float*>(out_ptr(f.smax)), static_cast<int32_t*>(out_ptr(f.valid)),
                              attention_status(query.device().index()).data_ptr<int32_t>(), stream_of(query)),
        "muzo_attention_max_lse");
  return f;
}

// A gradient of x [B, H, S, D]: x's own layout where the kernels can write it, else the projections'
// [B, S, H, D] memory.
Tensor gradient_like(const Tensor& x, Strides& s) {
  if (x.is_non_overlapping_and_dense()) {
    Tensor g = at::empty_like(x);
    if (in_place(g, s)) return g;
  }
  Tensor g = at::empty({x.size(0), x.size(2), x.size(1), x.size(3)}, x.options()).transpose(1, 2);
  in_place(g, s);
  return g;
}

std::array<Tensor, 3> attention_backward(const Tensor& grad_out, const Tensor& query, const Tensor& key, const Tensor& value,
                                         const Tensor& out, const Tensor& lse, double scaling, bool causal,
                                         const OptTensor& lo, const OptTensor& hi, const std::array<bool, 3>& wanted) {
  const c10::cuda::CUDAGuard guard(query.device());
  const int64_t b = query.size(0), hq = query.size(1), sq = query.size(2), d = query.size(3);
  const int64_t hkv = key.size(1), sk = key.size(2);
  std::array<Tensor, 3> grads;
  std::array<Strides, 3> gs{};
  const Tensor* inputs[3] = {&query, &key, &value};
  bool any = false;
  for (int i = 0; i < 3; ++i) {
    if (!wanted[i]) continue;
    any = true;
    grads[i] = gradient_like(*inputs[i], gs[i]);
    if (query.numel() == 0 || key.numel() == 0) grads[i].zero_();   // no pair of a query and a key
  }
  if (!any || query.numel() == 0 || key.numel() == 0) return grads;
  Strides qs, ks, vs, os, ds;
  const Tensor q = readable(query, qs), k = readable(key, ks), v = readable(value, vs), o = readable(out, os),
               dout = readable(grad_out, ds);
  const int64_t strides[24] = {qs[0], qs[1], qs[2], ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], os[0], os[2], os[1],
                               ds[0], ds[2], ds[1], gs[0][0], gs[0][1], gs[0][2], gs[1][0], gs[1][1], gs[1][2],
                               gs[2][0], gs[2][1], gs[2][2]};
  const int code = dtype_code(q);
  const int64_t size = lib.attention_workspace(code, b, hq, hkv, sq, sk, d, causal ? 1 : 0);
  if (size < 0) throw Failure("muzo_attention_backward: shape not supported");
  const Tensor workspace = at::empty({size}, q.options().dtype(at::kByte));
  check(lib.attention_backward(ptr(q), ptr(k), ptr(v), ptr(o), ptr(dout), lse.const_data_ptr<float>(), out_ptr(grads[0]),
                               out_ptr(grads[1]), out_ptr(grads[2]), code, b, hq, hkv, sq, sk, d, strides, causal ? 1 : 0,
                               static_cast<float>(scaling), range_ptr(lo), range_ptr(hi), workspace.data_ptr(), size,
                               attention_status(query.device().index()).data_ptr<int32_t>(), stream_of(query)),
        "muzo_attention_backward");
  return grads;
}

// The autograd node of attention_max: differentiable once; the maxima are not differentiable.
struct AttentionMax : torch::autograd::Function<AttentionMax> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& query, const Tensor& key,
                                                const Tensor& value, double scaling, bool causal, const OptTensor& lo,
                                                const OptTensor& hi, bool record) {
    Forward f = attention_forward(query, key, value, scaling, causal, lo, hi, record, true);
    ctx->save_for_backward({query, key, value, f.out, f.lse, lo ? *lo : Tensor(), hi ? *hi : Tensor()});
    ctx->saved_data["scaling"] = scaling;
    ctx->saved_data["causal"] = causal;
    if (!record) return {f.out};
    ctx->mark_non_differentiable({f.smax, f.valid});
    return {f.out, f.smax, f.valid};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "attention_max is differentiable once: its backward pass has no gradient of its own");
    const auto saved = ctx->get_saved_variables();
    std::array<bool, 3> wanted;
    for (int i = 0; i < 3; ++i) wanted[i] = ctx->needs_input_grad(i);
    Tensor grad_out = grads[0];
    if (!grad_out.defined()) grad_out = at::zeros_like(saved[3]);
    const OptTensor lo = saved[5].defined() ? OptTensor(saved[5]) : std::nullopt;
    const OptTensor hi = saved[6].defined() ? OptTensor(saved[6]) : std::nullopt;
    const auto g = attention_backward(grad_out, saved[0], saved[1], saved[2], saved[3], saved[4],
                                      ctx->saved_data["scaling"].toDouble(), ctx->saved_data["causal"].toBool(), lo, hi, wanted);
    return {g[0], g[1], g[2], Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

py::object or_none(const Tensor& t) { return t.defined() ? py::cast(t) : py::none(); }

py::tuple py_attention(const Tensor& query, const Tensor& key, const Tensor& value, std::optional<double> scaling, bool causal,
                       const OptTensor& lo, const OptTensor& hi, bool record) {
  const double s = check_attention(query, key, value, scaling, lo, hi);
  if (at::GradMode::is_enabled() && (query.requires_grad() || key.requires_grad() || value.requires_grad())) {
    const auto r = AttentionMax::apply(query, key, value, s, causal, lo, hi, record);
    return py::make_tuple(r[0], or_none(record ? r[1] : Tensor()), or_none(record ? r[2] : Tensor()));
  }
  at::NoGradGuard no_grad;
  const Forward f = attention_forward(query, key, value, s, causal, lo, hi, record, false);
  return py::make_tuple(f.out, or_none(f.smax), or_none(f.valid));
}

py::tuple py_forward(const Tensor& query, const Tensor& key, const Tensor& value, std::optional<double> scaling, bool causal,
                     const OptTensor& lo, const OptTensor& hi, bool record, bool keep_lse) {
  const double s = check_attention(query, key, value, scaling, lo, hi);
  at::NoGradGuard no_grad;
  const Forward f = attention_forward(query, key, value, s, causal, lo, hi, record, keep_lse);
  return py::make_tuple(f.out, or_none(f.lse), or_none(f.smax), or_none(f.valid));
}

py::tuple py_backward(const Tensor& grad_out, const Tensor& query, const Tensor& key, const Tensor& value, const Tensor& out,
                      const Tensor& lse, std::optional<double> scaling, bool causal, const OptTensor& lo, const OptTensor& hi,
                      const std::array<bool, 3>& wanted) {
  for (const Tensor* t : {&grad_out, &out, &lse}) check_plain(*t, "attention_max_backward");
  const double s = check_attention(query, key, value, scaling, lo, hi);
  const int64_t b = query.size(0), hq = query.size(1), sq = query.size(2), d = query.size(3);
  for (const Tensor* t : {&out, &grad_out})
    TORCH_CHECK_VALUE(t->dim() == 4 && t->size(0) == b && t->size(1) == sq && t->size(2) == hq && t->size(3) == d &&
                          t->scalar_type() == query.scalar_type() && t->device() == query.device(),
                      "attention_max_backward: out and grad_out must be [B, Sq, Hq, D] of the query's type and device");
  TORCH_CHECK_VALUE(lse.dim() == 3 && lse.size(0) == b && lse.size(1) == hq && lse.size(2) == sq &&
                        lse.scalar_type() == at::kFloat && lse.device() == query.device(),
                    "attention_max_backward: lse must be fp32 [B, Hq, Sq] on ", query.device());
  at::NoGradGuard no_grad;
  const auto g = attention_backward(grad_out, query, key, value, out, lse.contiguous(), s, causal, lo, hi, wanted);
  return py::make_tuple(or_none(g[0]), or_none(g[1]), or_none(g[2]));
}

// ---------------------------------------------------------------- gradient norm and clipping

// The tensors' common device; none without tensors.
std::optional<at::Device> check_grads(const std::vector<Tensor>& tensors, const char* what) {
  std::optional<at::Device> device;
  for (const Tensor& t : tensors) check_plain(t, what);
  for (const Tensor& t : tensors) {
    TORCH_CHECK_VALUE(t.layout() == at::kStrided, what, ": sparse gradients are not supported");
    TORCH_CHECK_TYPE(dtype_code(t) >= 0, what, " supports float32, bfloat16 and float16, not ", t.scalar_type());
    if (!device) {
      device = t.device();
      TORCH_CHECK_VALUE(t.is_cuda(), "muzo_clip_b200 gradient kernels run on CUDA tensors only");
    }
    TORCH_CHECK_VALUE(t.device() == *device, what, ": the tensors are on different devices");
  }
  return device;
}

// Whether t's elements fill its memory from data_ptr() on, in whatever order.
bool flat(const Tensor& t) { return t.is_contiguous() || t.is_non_overlapping_and_dense(); }

struct Columns {
  std::vector<uint64_t> address;
  std::vector<int64_t> numel;
  std::vector<int32_t> dtype;
  int64_t elements = 0;
  explicit Columns(const std::vector<Tensor>& tensors) {
    address.reserve(tensors.size());
    numel.reserve(tensors.size());
    dtype.reserve(tensors.size());
    for (const Tensor& t : tensors) {
      numel.push_back(t.numel());
      elements += t.numel();
      address.push_back(t.numel() ? reinterpret_cast<uint64_t>(t.const_data_ptr()) : 0);
      dtype.push_back(dtype_code(t));
    }
  }
};

Tensor grad_norm(std::vector<Tensor> grads, bool inf) {
  const auto device = check_grads(grads, "grad_norm");
  if (!device) return at::zeros({}, at::kFloat);
  at::NoGradGuard no_grad;
  const c10::cuda::CUDAGuard guard(*device);
  for (Tensor& t : grads)
    if (!flat(t)) t = t.contiguous();
  const Columns c(grads);
  const auto options = at::TensorOptions().device(*device);
  const Tensor norm = at::empty({}, options.dtype(at::kFloat));
  const int64_t size = lib.grad_workspace(static_cast<int64_t>(grads.size()), c.elements);
  const Tensor work = at::empty({size}, options.dtype(at::kByte));
  check(lib.grad_norm(c.address.data(), c.numel.data(), c.dtype.data(), static_cast<int64_t>(grads.size()), inf ? 1 : 0,
                      norm.data_ptr<float>(), work.data_ptr(), size, stream_of(norm)),
        "muzo_grad_norm");
  return norm;
}

// Whether sum c_k z_k == target has a solution with 0 <= z_k <= m_k (c_k > 0, by descending c_k). The strides of
// ordinary views leave one or two values to try per dimension; what takes longer counts as a solution.
struct Term { int64_t c, m; };
bool solvable(const std::vector<Term>& terms, size_t k, int64_t target, int64_t& budget) {
  if (target == 0) return true;
  if (k == terms.size() || --budget < 0) return budget < 0;
  int64_t rest = 0;   // the largest sum of the terms behind this one
  for (size_t i = k + 1; i < terms.size(); ++i) rest += terms[i].c * terms[i].m;
  const int64_t c = terms[k].c;
  const int64_t first = target > rest ? (target - rest + c - 1) / c : 0, last = std::min(terms[k].m, target / c);
  for (int64_t z = first; z <= last; ++z)
    if (solvable(terms, k + 1, target - c * z, budget)) return true;
  return false;
}
bool solvable(std::vector<Term> terms, int64_t target) {
  std::sort(terms.begin(), terms.end(), [](const Term& x, const Term& y) { return x.c > y.c; });
  std::vector<Term> merged;   // equal factors are one term
  for (const Term& t : terms) {
    if (t.c == 0 || t.m == 0) continue;
    if (!merged.empty() && merged.back().c == t.c) merged.back().m += t.m;
    else merged.push_back(t);
  }
  int64_t budget = 1 << 16;
  return target >= 0 && solvable(merged, 0, target, budget);
}

struct View {   // a tensor's bytes: dimensions of `m` steps of `c` bytes from `begin`, elements of `size` bytes
  int64_t begin, end, size;
  std::vector<Term> dims;
  size_t tensor;
  bool written;
  View(const Tensor& t, size_t i, bool w)
      : begin(reinterpret_cast<int64_t>(t.const_data_ptr())), end(0), size(t.element_size()), tensor(i), written(w) {
    end = begin + size;
    for (int64_t d = 0; d < t.dim(); ++d) {
      dims.push_back({t.stride(d) * size, t.size(d) - 1});
      end += dims.back().c * dims.back().m;
    }
  }
};
bool share_bytes(const View& a, const View& b) {   // a + x = b + y, with y counted from its end
  std::vector<Term> terms(a.dims);
  terms.insert(terms.end(), b.dims.begin(), b.dims.end());
  terms.push_back({1, a.size - 1 + b.size - 1});
  return solvable(std::move(terms), b.end - 1 - a.begin);
}
bool repeats_bytes(const View& v) {   // two indices, first different in dimension d, of one element
  for (size_t d = 0; d < v.dims.size(); ++d) {
    if (v.dims[d].m == 0) continue;
    if (v.dims[d].c == 0) return true;
    std::vector<Term> terms{{v.dims[d].c, v.dims[d].m - 1}};
    int64_t target = -v.dims[d].c;
    for (size_t e = d + 1; e < v.dims.size(); ++e) {
      terms.push_back({v.dims[e].c, 2 * v.dims[e].m});
      target += v.dims[e].c * v.dims[e].m;
    }
    if (solvable(std::move(terms), target)) return true;
  }
  return false;
}

// Whether anything that is written shares bytes with itself or with anything else that is written or read (a tensor
// scaled in place is only itself), for lists in which some tensors do not fill their memory; the library
// checks the others.
bool any_shared(const std::vector<Tensor>& grads, const std::vector<Tensor>& outs) {
  std::vector<View> views;
  for (size_t i = 0; i < grads.size(); ++i) {
    if (grads[i].numel() == 0) continue;
    views.emplace_back(outs[i], i, true);
    if (repeats_bytes(views.back())) return true;
    if (!(grads[i].const_data_ptr() == outs[i].const_data_ptr() && grads[i].scalar_type() == outs[i].scalar_type() &&
          grads[i].strides() == outs[i].strides()))
      views.emplace_back(grads[i], i, false);
  }
  std::sort(views.begin(), views.end(), [](const View& x, const View& y) { return x.begin < y.begin; });
  std::vector<const View*> open;   // those that reach beyond the present one's begin
  for (const View& v : views) {
    open.erase(std::remove_if(open.begin(), open.end(), [&](const View* o) { return o->end <= v.begin; }), open.end());
    for (const View* o : open)
      if ((o->written || v.written) && share_bytes(*o, v)) return true;
    open.push_back(&v);
  }
  return false;
}

constexpr char kOverlap[] = "gradient clipping: tensors that are written overlap in memory (the same one twice?)";

// Scales grads into outs (the same list: in place) and returns the norm before.
Tensor clip_grads(std::vector<Tensor> grads, const std::optional<std::vector<Tensor>>& outs, double max_norm, bool inf) {
  if (outs)
    for (const Tensor& t : *outs) check_plain(t, "clip_grads");
  const auto device = check_grads(grads, "clip_grads");
  if (outs) {
    check_grads(*outs, "clip_grads");
    TORCH_CHECK_VALUE(outs->size() == grads.size(), "clip_grads: ", grads.size(), " gradients but ", outs->size(), " outputs");
  }
  if (!device) return at::zeros({}, at::kFloat);
  at::NoGradGuard no_grad;
  const c10::cuda::CUDAGuard guard(*device);
  const std::vector<Tensor> written = outs ? *outs : grads;
  std::vector<Tensor> dst = written;
  std::vector<size_t> detours;   // what does not fill its memory, or lies in another order than its output
  for (size_t i = 0; i < grads.size(); ++i) {
    const Tensor &g = grads[i], &o = dst[i];
    TORCH_CHECK_VALUE(o.device() == *device && o.sizes() == g.sizes() &&
                          (o.scalar_type() == g.scalar_type() || o.scalar_type() == at::kFloat),
                      "clip_grads: an output must have its gradient's shape and device, and its type or fp32");
    if (!flat(g) || (g.strides() != o.strides() && g.numel() > 1)) detours.push_back(i);
  }
  TORCH_CHECK_VALUE(detours.empty() || !any_shared(grads, written), kOverlap);
  for (const size_t i : detours) {
    grads[i] = grads[i].contiguous();
    dst[i] = at::empty(dst[i].sizes(), dst[i].options());
  }
  const Columns from(grads), to(dst);
  const auto options = at::TensorOptions().device(*device);
  const Tensor norm = at::empty({}, options.dtype(at::kFloat));
  const int64_t size = lib.grad_workspace(static_cast<int64_t>(grads.size()), from.elements);
  const Tensor work = at::empty({size}, options.dtype(at::kByte));
  const int status = lib.grad_clip(from.address.data(), to.address.data(), from.numel.data(), from.dtype.data(),
                                   to.dtype.data(), static_cast<int64_t>(grads.size()), inf ? 1 : 0,
                                   static_cast<float>(max_norm), norm.data_ptr<float>(), work.data_ptr(), size, stream_of(norm));
  TORCH_CHECK_VALUE(status != MUZO_ERR_ARG, kOverlap);
  check(status, "muzo_grad_clip");
  size_t next = 0;
  for (size_t i = 0; i < dst.size(); ++i) {
    if (next < detours.size() && detours[next] == i) {
      ++next;
      written[i].copy_(dst[i]);
    } else if (!written[i].is_inference()) {
      written[i].unsafeGetTensorImpl()->bump_version();
    }
  }
  return norm;
}

// ---------------------------------------------------------------- module

py::object error_class;

void bind(const py::dict& addresses, py::object error) {
  auto at = [&](const char* name) { return reinterpret_cast<void*>(py::cast<uintptr_t>(addresses[name])); };
  lib.attention_forward = reinterpret_cast<decltype(lib.attention_forward)>(at("muzo_attention_max_lse"));
  lib.attention_backward = reinterpret_cast<decltype(lib.attention_backward)>(at("muzo_attention_backward"));
  lib.attention_workspace = reinterpret_cast<decltype(lib.attention_workspace)>(at("muzo_attention_backward_workspace"));
  lib.grad_norm = reinterpret_cast<decltype(lib.grad_norm)>(at("muzo_grad_norm"));
  lib.grad_clip = reinterpret_cast<decltype(lib.grad_clip)>(at("muzo_grad_clip"));
  lib.grad_workspace = reinterpret_cast<decltype(lib.grad_workspace)>(at("muzo_grad_workspace"));
  lib.status_string = reinterpret_cast<decltype(lib.status_string)>(at("muzo_status_string"));
  lib.last_cuda_error = reinterpret_cast<decltype(lib.last_cuda_error)>(at("muzo_last_cuda_error"));
  error_class = std::move(error);
  error_class.inc_ref();   // lives until the process ends
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const Failure& e) {
      PyErr_SetString(error_class ? error_class.ptr() : PyExc_RuntimeError, e.what());
    }
  });
  m.def("bind", &bind);
  m.def("attention", &py_attention);
  m.def("attention_forward", &py_forward);
  m.def("attention_backward", &py_backward);
  m.def("attention_status", &attention_status);
  m.def("attention_used", &attention_used);
  m.def("readable", [](const Tensor& t) {
    Strides s;
    const Tensor r = readable(t, s);
    return py::make_tuple(r, py::make_tuple(s[0], s[1], s[2]));
  });
  m.def("flat", &flat);
  m.def("grad_norm", &grad_norm);
  m.def("clip_grads", &clip_grads);
}
