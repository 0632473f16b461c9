// Python binding of the attention training operators (kernelcodegen_b200/ops.py) on torch tensors:
// argument checks, outputs, workspace, descriptor and launch of one call in one crossing.
//
// A call of these operators on one short sequence is host time and little else: through ctypes, with
// every tensor property read from Python, it takes 15 to 28 us, and 6 to 10 this way.  The kernels stay behind
// the C-ABI of include/kcg_capi.h: the functions are handed over as addresses once (bind), so that the
// library the process has loaded, the bounds-checking build included, is the one that is called.
#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/utils/pybind.h>

#include <array>
#include <limits>
#include <optional>

#include "../../include/kcg_capi.h"

namespace {

using at::Tensor;
using Opt = std::optional<Tensor>;
using Strides = std::array<int64_t, 3>;
using Shape = std::array<int64_t, 4>;

decltype(&kcg_fmha_fwd_lse_launch) fwd_lse;
decltype(&kcg_fmha_bwd_workspace_bytes) bwd_bytes;
decltype(&kcg_fmha_bwd_launch) bwd;
decltype(&kcg_qk_norm_rope_launch) rope;
decltype(&kcg_qk_norm_rope_bwd_workspace_bytes) rope_bwd_bytes;
decltype(&kcg_qk_norm_rope_bwd_launch) rope_bwd;

void bind(int64_t a, int64_t b, int64_t c, int64_t d, int64_t e, int64_t f) {
  fwd_lse = reinterpret_cast<decltype(fwd_lse)>(a);
  bwd_bytes = reinterpret_cast<decltype(bwd_bytes)>(b);
  bwd = reinterpret_cast<decltype(bwd)>(c);
  rope = reinterpret_cast<decltype(rope)>(d);
  rope_bwd_bytes = reinterpret_cast<decltype(rope_bwd_bytes)>(e);
  rope_bwd = reinterpret_cast<decltype(rope_bwd)>(f);
}

[[noreturn]] void bad_value(const std::string& what) { throw py::value_error(what); }
[[noreturn]] void bad_type(const std::string& what) { throw py::type_error(what); }

void same_device(const Tensor& t, at::Device dev) {
  if (t.device() != dev) throw std::runtime_error("all tensors must live on the same device");
}

at::Device cuda_device(const Tensor& t) {
  if (!t.is_cuda()) throw std::runtime_error("kernelcodegen_b200 operators need CUDA tensors; there is no CPU path");
  return t.device();
}

Shape shape4(const Tensor& t, const char* what) {
  if (t.dim() != 4) bad_value(what);
  return {t.size(0), t.size(1), t.size(2), t.size(3)};
}

// Batch, head and row stride of the [B, heads, S, D] view that is expected.
Strides view(const char* name, const Tensor& t, const Shape& shape, at::ScalarType dtype, at::Device dev) {
  bool same = t.dim() == 4;
  for (int i = 0; same && i < 4; ++i) same = t.size(i) == shape[i];
  if (!same) {
    std::string got, want;
    for (const int64_t n : t.sizes()) got += (got.empty() ? "" : ", ") + std::to_string(n);
    for (const int64_t n : shape) want += (want.empty() ? "" : ", ") + std::to_string(n);
    bad_value(std::string(name) + " has shape (" + got + "), expected (" + want + ")");
  }
  if (t.scalar_type() != dtype) bad_type(std::string(name) + " is " + toString(t.scalar_type()) + ", expected " + toString(dtype));
  same_device(t, dev);
  if (shape[3] != 1 && t.stride(3) != 1) bad_value(std::string(name) + " must have stride 1 in the last dimension");
  return {t.stride(0), t.stride(1), t.stride(2)};
}

Tensor contiguous(at::IntArrayRef shape, at::ScalarType dtype, at::Device dev) {
  std::array<int64_t, 4> strides;
  int64_t n = 1;
  for (size_t i = shape.size(); i-- > 0;) {
    strides[i] = n;
    n *= shape[i] > 0 ? shape[i] : 1;
  }
  return at::detail::empty_strided_cuda(shape, at::IntArrayRef(strides.data(), shape.size()), dtype, dev);
}

// The same, of a tensor that has to have memory of its own for every entry: what autograd hands out for a broadcast has not.
Strides own_view(const char* name, const Tensor& t, const Shape& shape, at::ScalarType dtype, at::Device dev) {
  for (int64_t i = 0; i < t.dim(); ++i)
    if (t.size(i) > 1 && t.stride(i) == 0)
      bad_value(std::string(name) + " is an expanded tensor (stride 0 in dimension " + std::to_string(i) + "): call .contiguous() on it first");
  return view(name, t, shape, dtype, dev);
}

// An output view: the one given, checked, or a new contiguous tensor.
Strides output(const char* name, const Opt& given, const Shape& shape, at::ScalarType dtype, at::Device dev, Tensor& out) {
  out = given ? *given : contiguous(shape, dtype, dev);
  return view(name, out, shape, dtype, dev);
}

void put(int64_t (&into)[3], const Strides& s) {
  for (int i = 0; i < 3; ++i) into[i] = s[i];
}

void* data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* data(const Opt& t) { return t ? t->data_ptr() : nullptr; }

struct Attn {
  kcg_attn_desc d{};
  at::Device dev{at::kCUDA, 0};
  Shape q, k;
  bool empty;      // no query, or no key: nothing to launch
};

Attn attention(const Tensor& q, const Tensor& k, const Tensor& v, double scale, bool causal) {
  Attn a;
  a.dev = cuda_device(q);
  const char* shapes = "expected Q [B,H,Sq,D] and K, V [B,Hkv,Skv,D]";
  a.q = shape4(q, shapes);
  a.k = shape4(k, shapes);
  if (shape4(v, shapes) != a.k || a.q[0] != a.k[0] || a.q[3] != a.k[3]) bad_value(shapes);
  const auto bf16 = at::kBFloat16;
  if (q.scalar_type() != bf16 || k.scalar_type() != bf16 || v.scalar_type() != bf16)
    bad_type("Q, K, V must be bfloat16: the gradients' contractions have no float32 form");
  if (a.k[1] == 0 ? a.q[1] != 0 : a.q[1] % a.k[1] != 0)
    bad_value("the number of query heads must be a multiple of the number of key/value heads");
  for (const int64_t n : {a.q[0], a.q[1], a.q[2], a.k[2]})
    if (n > INT32_MAX) bad_value("an extent does not fit 32 bits");
  a.d.B = static_cast<int32_t>(a.q[0]);
  a.d.H = static_cast<int32_t>(a.q[1]);
  a.d.Hkv = static_cast<int32_t>(a.k[1]);
  a.d.Sq = static_cast<int32_t>(a.q[2]);
  a.d.Skv = static_cast<int32_t>(a.k[2]);
  a.d.D = a.q[3] > INT32_MAX ? 0 : static_cast<int32_t>(a.q[3]);
  a.d.dtype = KCG_BF16;
  a.d.causal = causal;
  a.d.scale = static_cast<float>(scale);
  put(a.d.q, own_view("Q", q, a.q, bf16, a.dev));
  put(a.d.k, own_view("K", k, a.k, bf16, a.dev));
  put(a.d.v, own_view("V", v, a.k, bf16, a.dev));
  a.empty = q.numel() == 0 || k.numel() == 0;
  return a;
}

// A call without queries or keys is checked like any other: the status that it would have with extents of one.
int check_empty(kcg_attn_desc d) {
  for (int32_t* n : {&d.B, &d.H, &d.Hkv, &d.Sq, &d.Skv}) *n = 1;
  return bwd_bytes(&d) ? KCG_OK : fwd_lse(&d, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr);
}

std::tuple<int, Tensor, Tensor> fmha_with_lse(const Tensor& q, const Tensor& k, const Tensor& v, double scale, bool causal,
                                              const Opt& given) {
  Attn a = attention(q, k, v, scale, causal);
  Tensor out;
  put(a.d.o, output("out", given, a.q, at::kBFloat16, a.dev, out));
  Tensor lse = contiguous({a.q[0], a.q[1], a.q[2]}, at::kFloat, a.dev);
  const c10::cuda::CUDAGuard guard(a.dev);
  if (a.empty) {
    // a query that sees no key
    const int st = check_empty(a.d);
    if (st == KCG_OK) out.zero_(), lse.fill_(-std::numeric_limits<float>::infinity());
    return {st, out, lse};
  }
  const int st = fwd_lse(&a.d, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), static_cast<float*>(lse.data_ptr()),
                         c10::cuda::getCurrentCUDAStream(a.dev.index()).stream());
  return {st, out, lse};
}

std::tuple<int, Tensor, Tensor, Tensor> fmha_backward(const Tensor& dout, const Tensor& q, const Tensor& k, const Tensor& v,
                                                      const Tensor& out, const Tensor& lse, double scale, bool causal,
                                                      const Opt& dq_, const Opt& dk_, const Opt& dv_) {
  Attn a = attention(q, k, v, scale, causal);
  const auto bf16 = at::kBFloat16;
  put(a.d.d_o, own_view("dout", dout, a.q, bf16, a.dev));
  put(a.d.o, own_view("out", out, a.q, bf16, a.dev));
  if (lse.dim() != 3 || lse.size(0) != a.q[0] || lse.size(1) != a.q[1] || lse.size(2) != a.q[2] ||
      lse.scalar_type() != at::kFloat || !lse.is_contiguous())
    bad_value("lse must be the contiguous float32 [B,H,Sq] tensor of fmha_with_lse");
  same_device(lse, a.dev);
  Tensor dq, dk, dv;
  put(a.d.d_q, output("dq", dq_, a.q, bf16, a.dev, dq));
  put(a.d.d_k, output("dk", dk_, a.k, bf16, a.dev, dk));
  put(a.d.d_v, output("dv", dv_, a.k, bf16, a.dev, dv));
  const c10::cuda::CUDAGuard guard(a.dev);
  if (a.empty) {
    const int st = check_empty(a.d);
    if (st == KCG_OK) dq.zero_(), dk.zero_(), dv.zero_();
    return {st, dq, dk, dv};
  }
  // a buffer of this call alone, from the stream's allocator: two captured graphs never share it
  const size_t bytes = bwd_bytes(&a.d);
  const c10::DataPtr ws = c10::cuda::CUDACachingAllocator::get()->allocate(bytes);
  const int st = bwd(&a.d, dout.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                     static_cast<const float*>(lse.data_ptr()), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), ws.get(), bytes,
                     c10::cuda::getCurrentCUDAStream(a.dev.index()).stream());
  return {st, dq, dk, dv};
}

struct Rope {
  kcg_rope_desc d{};
  at::Device dev{at::kCUDA, 0};
  at::ScalarType dtype;
  Shape q, k;
  bool empty;
};

int32_t dtype_code(at::ScalarType t) {
  if (t == at::kFloat) return KCG_F32;
  if (t == at::kBFloat16) return KCG_BF16;
  bad_type(std::string("unsupported dtype ") + toString(t) + ": the kernels take float32 or bfloat16");
}

Rope rotation(const Tensor& q, const Opt& k, const Tensor& cos, const Tensor& sin, const Opt& wq, const Opt& wk,
              const Opt& positions, double eps, bool interleaved) {
  Rope r;
  r.q = shape4(q, "expected queries (and keys) as [B, heads, S, D]");
  r.dtype = q.scalar_type();
  r.d.dtype = dtype_code(r.dtype);
  r.dev = cuda_device(q);
  const int64_t B = r.q[0], S = r.q[2], D = r.q[3];
  put(r.d.q, view("q", q, r.q, r.dtype, r.dev));
  r.k = {B, 0, S, D};
  if (k) {
    r.k[1] = k->dim() == 4 ? k->size(1) : 0;
    put(r.d.k, view("k", *k, r.k, r.dtype, r.dev));
  } else if (wk) {
    bad_value("k_weight without keys");
  }
  r.empty = q.numel() == 0 && (!k || k->numel() == 0);
  if (cos.dim() != 2 || sin.dim() != 2 || cos.size(0) != sin.size(0) || cos.size(1) != sin.size(1) || 2 * cos.size(1) > D)
    bad_value("cos and sin must be [positions, R / 2] with R <= D");
  for (const Tensor* t : {&cos, &sin}) {
    if (t->scalar_type() != at::kFloat || !t->is_contiguous()) bad_type("cos and sin must be contiguous float32 tables");
    same_device(*t, r.dev);
  }
  r.d.dtype_w = KCG_F32;
  const Tensor* first = nullptr;
  for (const Opt* w : {&wq, &wk}) {
    if (!*w) continue;
    const Tensor& t = **w;
    if (!first) first = &t;
    if (t.dim() != 1 || t.size(0) != D || t.scalar_type() != first->scalar_type() || !t.is_contiguous())
      bad_value("the weights must be contiguous [D] tensors of one type");
    same_device(t, r.dev);
    r.d.dtype_w = dtype_code(t.scalar_type());
  }
  r.d.pos_bits = 32;
  if (positions) {
    const Tensor& t = *positions;
    if (t.scalar_type() != at::kInt && t.scalar_type() != at::kLong) bad_type("positions must be int32 or int64");
    if (t.dim() == 2 && t.size(0) == B && t.size(1) == S) r.d.pos[0] = t.stride(0);
    else if (t.dim() != 1 || t.size(0) != S) bad_value("positions must be [" + std::to_string(S) + "] or [" + std::to_string(B) + ", " + std::to_string(S) + "]");
    r.d.pos[1] = t.stride(-1);
    r.d.pos_bits = t.scalar_type() == at::kLong ? 64 : 32;
    same_device(t, r.dev);
  } else if (S > cos.size(0)) {
    bad_value("more tokens than rows of the tables");
  }
  for (const int64_t n : {B, r.q[1], r.k[1], S, D})
    if (n > INT32_MAX) bad_value("an extent does not fit 32 bits");
  r.d.B = static_cast<int32_t>(B);
  r.d.S = static_cast<int32_t>(S);
  r.d.H = static_cast<int32_t>(r.q[1]);
  r.d.Hk = static_cast<int32_t>(r.k[1]);
  r.d.D = static_cast<int32_t>(D);
  r.d.R = static_cast<int32_t>(2 * cos.size(1));
  r.d.interleaved = interleaved;
  r.d.table_rows = cos.size(0);
  r.d.eps = static_cast<float>(eps);
  return r;
}

std::tuple<int, Tensor, Opt> qk_norm_rope(const Tensor& q, const Opt& k, const Tensor& cos, const Tensor& sin, const Opt& wq,
                                          const Opt& wk, const Opt& positions, double eps, bool interleaved, const Opt& q_out_,
                                          const Opt& k_out_) {
  Rope r = rotation(q, k, cos, sin, wq, wk, positions, eps, interleaved);
  if (!k && k_out_) bad_value("k_out without keys");
  Tensor q_out, k_out;
  put(r.d.q_out, output("q_out", q_out_, r.q, r.dtype, r.dev, q_out));
  if (!r.empty && r.d.H == 0) {      // keys alone: they take the queries' place
    const auto keys = qk_norm_rope(*k, {}, cos, sin, wk, {}, positions, eps, interleaved, k_out_, {});
    return {std::get<0>(keys), q_out, std::get<1>(keys)};
  }
  if (k) put(r.d.k_out, output("k_out", k_out_, r.k, r.dtype, r.dev, k_out));
  int st = KCG_OK;
  if (!r.empty) {
    const c10::cuda::CUDAGuard guard(r.dev);
    st = rope(&r.d, q.data_ptr(), data(k), data(wq), data(wk), cos.data_ptr(), sin.data_ptr(), data(positions), q_out.data_ptr(),
              data(k_out), c10::cuda::getCurrentCUDAStream(r.dev.index()).stream());
  }
  return {st, q_out, k ? Opt(k_out) : Opt()};
}

std::tuple<int, Tensor, Opt, Opt, Opt> qk_norm_rope_backward(const Tensor& dq_out, const Opt& dk_out, const Tensor& q, const Opt& k,
                                                             const Tensor& cos, const Tensor& sin, const Opt& wq, const Opt& wk,
                                                             const Opt& positions, double eps, bool interleaved, const Opt& dq_,
                                                             const Opt& dk_) {
  Rope r = rotation(q, k, cos, sin, wq, wk, positions, eps, interleaved);
  if (dk_out.has_value() != k.has_value() || (!k && dk_)) bad_value("keys and their gradients go together");
  put(r.d.q_out, view("dq_out", dq_out, r.q, r.dtype, r.dev));
  Tensor dq, dk, dwq, dwk;
  put(r.d.d_q, output("dq", dq_, r.q, r.dtype, r.dev, dq));
  if (!r.empty && r.d.H == 0) {      // keys alone: they take the queries' place
    const auto keys = qk_norm_rope_backward(*dk_out, {}, *k, {}, cos, sin, wk, {}, positions, eps, interleaved, dk_, {});
    if (wq) dwq = contiguous({r.q[3]}, at::kFloat, r.dev).zero_();
    return {std::get<0>(keys), dq, std::get<1>(keys), wq ? Opt(dwq) : Opt(), std::get<3>(keys)};
  }
  if (k) {
    put(r.d.k_out, view("dk_out", *dk_out, r.k, r.dtype, r.dev));
    put(r.d.d_k, output("dk", dk_, r.k, r.dtype, r.dev, dk));
  }
  if (wq) dwq = contiguous({r.q[3]}, at::kFloat, r.dev);
  if (wk) dwk = contiguous({r.q[3]}, at::kFloat, r.dev);
  int st = KCG_OK;
  if (r.empty) {
    if (wq) dwq.zero_();
    if (wk) dwk.zero_();
  } else {
    const c10::cuda::CUDAGuard guard(r.dev);
    // a buffer of this call alone, from the stream's allocator: two captured graphs never share it
    const size_t bytes = wq || wk ? rope_bwd_bytes(&r.d) : 0;
    c10::DataPtr ws;
    if (bytes) ws = c10::cuda::CUDACachingAllocator::get()->allocate(bytes);
    st = rope_bwd(&r.d, dq_out.data_ptr(), data(dk_out), q.data_ptr(), data(k), data(wq), data(wk), cos.data_ptr(), sin.data_ptr(),
                  data(positions), dq.data_ptr(), data(dk), static_cast<float*>(data(dwq)), static_cast<float*>(data(dwk)), ws.get(),
                  bytes, c10::cuda::getCurrentCUDAStream(r.dev.index()).stream());
  }
  return {st, dq, k ? Opt(dk) : Opt(), wq ? Opt(dwq) : Opt(), wk ? Opt(dwk) : Opt()};
}

}  // namespace

PYBIND11_MODULE(_torch_binding, m) {
  m.attr("built_with") = KCG_BUILT_WITH;
  m.def("bind", &bind);
  // (wrapped: torch's own errors, out of memory among them, keep their Python types)
  m.def("fmha_with_lse", torch::wrap_pybind_function(fmha_with_lse));
  m.def("fmha_backward", torch::wrap_pybind_function(fmha_backward));
  m.def("qk_norm_rope", torch::wrap_pybind_function(qk_norm_rope));
  m.def("qk_norm_rope_backward", torch::wrap_pybind_function(qk_norm_rope_backward));
}
