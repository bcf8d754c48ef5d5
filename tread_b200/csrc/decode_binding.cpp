// Python binding of the decode-step operators (tread_b200.kernels.paged_append, paged_attn, adjust_logits).
//
// A decode step makes two such calls a layer, and for few sequences the host's time is what bounds it: the same
// checks and argument marshalling in Python with ctypes took 13 to 15 us a call, of which the launches are 3 to
// 5. Here a call is positional arguments in, checks on the tensors' own sizes and strides, the output from
// PyTorch's allocator, and the C ABI's entry point on the current stream of the tensors' device.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <utility>
#include <vector>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include "tread_b200.h"

namespace {

using at::Tensor;

bool given(PyObject* o) { return o != Py_None; }

const Tensor& tensor(PyObject* o, const char* name) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), name, " must be a tensor, got ", Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}

int dtype_code(const Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return TREAD_BF16;
    case at::kHalf: return TREAD_F16;
    case at::kFloat: return TREAD_F32;
    default:
      TORCH_CHECK_TYPE(false, name, ": unsupported dtype ", t.scalar_type(), "; expected float32, float16 or bfloat16");
  }
}

// every tensor of a call sits on one device: the kernels dereference them all there
void on(const Tensor& t, c10::DeviceIndex index, const char* name) {
  TORCH_CHECK_VALUE(t.is_cuda() && t.get_device() == index, name, " is on ", t.device(),
                    ", the call's other tensors on cuda:", (int)index);
}

c10::DeviceIndex device_of(const Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.is_cuda(), name, " must be a CUDA tensor (got ", t.device(), "); tread_b200 has no CPU path");
  return t.get_device();
}

// a contiguous [n] of a type, on the call's device
template <typename T>
const T* vector(const Tensor& t, int64_t n, at::ScalarType type, c10::DeviceIndex index, const char* name) {
  on(t, index, name);
  TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == n && t.scalar_type() == type && t.is_contiguous(), name,
                    " must be a contiguous ", type, " tensor of length ", n);
  return static_cast<const T*>(t.data_ptr());
}

int32_t small(int64_t n, const char* name) {
  TORCH_CHECK_VALUE(n <= INT32_MAX, name, " is too large: ", n);
  return (int32_t)n;
}

void* error_word(PyObject* o, c10::DeviceIndex index) {
  if (!given(o)) return nullptr;
  const Tensor& t = tensor(o, "err");
  on(t, index, "err");
  TORCH_CHECK_VALUE(t.scalar_type() == at::kInt && t.numel() >= 1, "err must be an int32 tensor of one element or more");
  return t.data_ptr();
}

// A pair of pools [N, Hkv, page_size, D] with contiguous [page_size, D] planes: a whole pool, or one layer of
// [N, L, Hkv, page_size, D].
struct Pools {
  int64_t pages, heads, size, dim, page_stride, head_stride;
};
Pools pools(const Tensor& k, const Tensor& v) {
  TORCH_CHECK_VALUE(k.dim() == 4 && k.sizes() == v.sizes() && k.strides() == v.strides(),
                    "k_pages and v_pages must be [pages, Hkv, page_size, D] of one shape and strides");
  const auto n = k.sizes();
  const auto s = k.strides();
  TORCH_CHECK_VALUE(s[3] == 1 && (s[2] == n[3] || n[2] == 1) && k.scalar_type() == v.scalar_type(),
                    "k_pages and v_pages must share a dtype and have contiguous [page_size, D] planes");
  return {n[0], n[1], n[2], n[3], s[0], s[1]};
}

const int32_t* page_table(const Tensor& t, c10::DeviceIndex index) {
  on(t, index, "table");
  TORCH_CHECK_VALUE(t.dim() == 2 && t.scalar_type() == at::kInt && (t.stride(1) == 1 || t.size(1) <= 1),
                    "table must be int32 [sequences, pages] with unit column stride");
  return static_cast<const int32_t*>(t.data_ptr());
}

// The runs of consecutive bytes of a tensor with unit last stride, in order of address.
std::vector<std::pair<uintptr_t, uintptr_t>> runs(const Tensor& t) {
  std::vector<std::pair<uintptr_t, uintptr_t>> r;
  const int64_t es = t.element_size(), width = t.size(-1) * es, d = t.dim();
  const int64_t n0 = t.size(0), n1 = d == 3 ? t.size(1) : 1, s0 = t.stride(0) * es, s1 = d == 3 ? t.stride(1) * es : 0;
  for (int64_t i = 0; i < n0; ++i)
    for (int64_t j = 0; j < n1; ++j) {
      const uintptr_t at = reinterpret_cast<uintptr_t>(t.data_ptr()) + i * s0 + j * s1;
      r.emplace_back(at, at + width);
    }
  std::sort(r.begin(), r.end());
  return r;
}

// An output may be an input itself (each element is read before it is written, by the thread that writes it) where
// `itself` says so, or lie apart from it; its elements over others of the input would be a race.
void apart(const Tensor& out, const Tensor& in, bool itself, const char* out_name, const char* in_name) {
  if (out.numel() == 0 || in.numel() == 0) return;
  auto end = [](const Tensor& t) {
    int64_t last = 1;
    for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
    return reinterpret_cast<uintptr_t>(t.data_ptr()) + last * t.element_size();
  };
  const uintptr_t a = reinterpret_cast<uintptr_t>(out.data_ptr()), b = reinterpret_cast<uintptr_t>(in.data_ptr());
  if (a >= end(in) || b >= end(out)) return;
  if (itself && a == b && out.scalar_type() == in.scalar_type() && out.sizes() == in.sizes()) {
    bool same = true;
    for (int64_t i = 0; i < out.dim(); ++i) same &= out.size(i) == 1 || out.stride(i) == in.stride(i);
    if (same) return;
  }
  const auto x = runs(out), y = runs(in);  // columns of one buffer may lie between each other
  for (size_t i = 0, j = 0; i < x.size() && j < y.size();) {
    TORCH_CHECK_VALUE(x[i].second <= y[j].first || y[j].second <= x[i].first, out_name, " overlaps ", in_name,
                      " in memory", itself ? ", but is not the same elements" : "");
    x[i].second <= y[j].first ? ++i : ++j;
  }
}

void check(int rc, const char* what) {
  TORCH_CHECK(rc == TREAD_OK, what, " failed (status ", rc, "): ", tread_last_error());
}

tread_stream_t stream_of(c10::DeviceIndex index) {
  return reinterpret_cast<tread_stream_t>(c10::cuda::getCurrentCUDAStream(index).stream());
}

// (k, v, k_pages, v_pages, table, pos, seq, inv_freq, rope_pos, attn_scaling, q, q_out, err)
PyObject* paged_append(PyObject*, PyObject* const* arg, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(count == 13, "paged_append: 13 arguments wanted");
  const Tensor &k = tensor(arg[0], "k"), &v = tensor(arg[1], "v"), &kp = tensor(arg[2], "k_pages"),
               &vp = tensor(arg[3], "v_pages"), &table = tensor(arg[4], "table"), &pos = tensor(arg[5], "pos");
  const auto index = device_of(kp, "k_pages");
  const Pools p = pools(kp, vp);
  on(vp, index, "v_pages"), on(k, index, "k"), on(v, index, "v");
  TORCH_CHECK_VALUE(k.dim() == 3 && k.size(1) == p.heads && k.size(2) == p.dim && k.stride(2) == 1 &&
                        v.sizes() == k.sizes() && v.stride(2) == 1,
                    "k and v must be [R, ", p.heads, ", ", p.dim, "] with unit last stride");
  TORCH_CHECK_TYPE(k.scalar_type() == v.scalar_type() && k.scalar_type() == kp.scalar_type(),
                   "k, v and the pages must share a dtype");
  const int64_t R = k.size(0);
  tread_paged_append_args a{};
  a.table = page_table(table, index);
  a.pos = vector<int64_t>(pos, R, at::kLong, index, "pos");
  if (given(arg[6]))
    a.seq = vector<int32_t>(tensor(arg[6], "seq"), R, at::kInt, index, "seq");
  else
    TORCH_CHECK_VALUE(R <= table.size(0), R, " rows without seq, but a table of ", table.size(0), " sequences");
  if (given(arg[7])) a.inv_freq = vector<float>(tensor(arg[7], "inv_freq"), p.dim / 2, at::kFloat, index, "inv_freq");
  if (given(arg[8])) a.rope_pos = vector<int64_t>(tensor(arg[8], "rope_pos"), R, at::kLong, index, "rope_pos");
  a.attn_scaling = (float)PyFloat_AsDouble(arg[9]);
  if (PyErr_Occurred()) throw python_error();
  a.err_flag = error_word(arg[12], index);
  c10::cuda::CUDAGuard guard(index);
  Tensor out;
  if (given(arg[10])) {
    const Tensor& q = tensor(arg[10], "q");
    on(q, index, "q");
    TORCH_CHECK_VALUE(q.dim() == 3 && q.size(0) == R && q.size(2) == p.dim && q.stride(2) == 1 &&
                          q.scalar_type() == k.scalar_type(),
                      "q must be [", R, ", Hq, ", p.dim, "] of k's dtype with unit last stride");
    TORCH_CHECK_VALUE(a.inv_freq, "q without inv_freq: nothing rotates it");
    if (given(arg[11])) {
      out = tensor(arg[11], "q_out");
      on(out, index, "q_out");
      TORCH_CHECK_VALUE(out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type() && out.is_contiguous(),
                        "q_out must be a contiguous tensor of q's shape and dtype");
      apart(out, q, true, "q_out", "q"), apart(out, k, false, "q_out", "k"), apart(out, v, false, "q_out", "v");
    } else {
      out = at::empty(q.sizes(), q.options());
    }
    a.q = q.data_ptr(), a.q_out = out.data_ptr(), a.q_ld = q.stride(0), a.q_sh = q.stride(1);
    a.Hq = small(q.size(1), "Hq");
  } else {
    TORCH_CHECK_VALUE(!given(arg[11]), "q_out without q");
  }
  a.k = k.data_ptr(), a.v = v.data_ptr(), a.k_pages = kp.data_ptr(), a.v_pages = vp.data_ptr();
  a.k_ld = k.stride(0), a.k_sh = k.stride(1), a.v_ld = v.stride(0), a.v_sh = v.stride(1);
  a.page_stride = p.page_stride, a.head_stride = p.head_stride, a.num_pages = p.pages, a.table_ld = table.stride(0);
  a.page_size = small(p.size, "page_size"), a.num_seqs = small(table.size(0), "table");
  a.max_pages = small(table.size(1), "table");
  a.R = small(R, "R"), a.Hkv = small(p.heads, "Hkv"), a.D = small(p.dim, "D"), a.dtype = dtype_code(k, "k");
  check(tread_paged_append(&a, stream_of(index)), "tread_paged_append");
  if (!out.defined()) Py_RETURN_NONE;
  if (given(arg[11])) return Py_NewRef(arg[11]);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// (q, k_pages, v_pages, table, lens, out, sm_scale, err)
PyObject* paged_attn(PyObject*, PyObject* const* arg, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(count == 8, "paged_attn: 8 arguments wanted");
  const Tensor &q = tensor(arg[0], "q"), &kp = tensor(arg[1], "k_pages"), &vp = tensor(arg[2], "v_pages"),
               &table = tensor(arg[3], "table"), &lens = tensor(arg[4], "lens");
  const auto index = device_of(kp, "k_pages");
  const Pools p = pools(kp, vp);
  on(vp, index, "v_pages"), on(q, index, "q");
  TORCH_CHECK_VALUE(q.dim() == 3 && q.size(2) == p.dim && q.stride(2) == 1 && (q.stride(1) == p.dim || q.size(1) <= 1) &&
                        q.scalar_type() == kp.scalar_type(),
                    "q must be [B, Hq, ", p.dim, "] of the pages' dtype with contiguous rows");
  const int64_t B = q.size(0);
  tread_paged_attn_args a{};
  a.table = page_table(table, index);
  TORCH_CHECK_VALUE(table.size(0) == B, "table must have a row for each of the ", B, " sequences");
  a.lens = vector<int64_t>(lens, B, at::kLong, index, "lens");
  a.err_flag = error_word(arg[7], index);
  if (given(arg[6])) {
    a.sm_scale = (float)PyFloat_AsDouble(arg[6]);
    if (PyErr_Occurred()) throw python_error();
  } else {
    a.sm_scale = (float)(1.0 / std::sqrt((double)p.dim));
  }
  c10::cuda::CUDAGuard guard(index);
  Tensor out;
  if (given(arg[5])) {
    out = tensor(arg[5], "out");
    on(out, index, "out");
    TORCH_CHECK_VALUE(out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type() && out.is_contiguous(),
                      "out must be a contiguous tensor of q's shape and dtype");
    apart(out, q, true, "out", "q");
  } else {
    out = at::empty(q.sizes(), q.options());
  }
  a.B = small(B, "B"), a.Hq = small(q.size(1), "Hq"), a.Hkv = small(p.heads, "Hkv"), a.D = small(p.dim, "D");
  // one workspace a call, from the allocator: calls of several streams, threads and graphs share none
  a.workspace_bytes = (int64_t)tread_paged_attn_workspace_bytes(a.Hq, a.Hkv, a.D);
  const Tensor ws = at::empty({a.workspace_bytes}, q.options().dtype(at::kByte));
  a.workspace = ws.data_ptr(), a.q = q.data_ptr(), a.k_pages = kp.data_ptr(), a.v_pages = vp.data_ptr();
  a.out = out.data_ptr();
  a.q_ld = q.stride(0), a.page_stride = p.page_stride, a.head_stride = p.head_stride, a.num_pages = p.pages;
  a.table_ld = table.stride(0), a.page_size = small(p.size, "page_size"), a.max_pages = small(table.size(1), "table");
  a.dtype = dtype_code(q, "q");
  check(tread_paged_attn(&a, stream_of(index)), "tread_paged_attn");
  if (given(arg[5])) return Py_NewRef(arg[5]);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// a penalty: one number, or fp32 [B]
void per_row(PyObject* o, int64_t B, c10::DeviceIndex index, const char* name, const float*& rows, float& all) {
  if (THPVariable_Check(o)) {
    rows = vector<float>(THPVariable_Unpack(o), B, at::kFloat, index, name);
    return;
  }
  all = (float)PyFloat_AsDouble(o);
  if (PyErr_Occurred()) throw python_error();
}

// row stride of [B, width], or 0 for one row [width] that serves every row
int64_t by_row(const Tensor& t, int64_t B, int64_t width, at::ScalarType type, c10::DeviceIndex index, const char* name) {
  on(t, index, name);
  const int64_t d = t.dim();
  TORCH_CHECK_VALUE(t.scalar_type() == type && ((d == 2 && t.size(0) == B) || d == 1) && t.size(d - 1) == width &&
                        (width <= 1 || t.stride(d - 1) == 1),
                    name, " must be ", type, " [", B, ", ", width, "] or [", width, "] with unit last stride");
  return d == 2 ? t.stride(0) : 0;
}

// (logits, tokens, lens, prompt_lens, repetition, presence, frequency, bias_ids, bias, allowed, out)
PyObject* adjust_logits(PyObject*, PyObject* const* arg, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(count == 11, "adjust_logits: 11 arguments wanted");
  const Tensor& x = tensor(arg[0], "logits");
  const auto index = device_of(x, "logits");
  TORCH_CHECK_VALUE(x.dim() == 2 && (x.size(1) <= 1 || x.stride(1) == 1), "logits must be [B, V] with unit column stride");
  const int64_t B = x.size(0), V = x.size(1);
  tread_adjust_logits_args a{};
  if (given(arg[1])) {
    const Tensor& tokens = tensor(arg[1], "tokens");
    on(tokens, index, "tokens");
    TORCH_CHECK_VALUE(tokens.dim() == 2 && tokens.size(0) == B && tokens.scalar_type() == at::kLong &&
                          (tokens.size(1) <= 1 || tokens.stride(1) == 1),
                      "tokens must be int64 [", B, ", H] with unit column stride");
    a.tokens = static_cast<const int64_t*>(tokens.data_ptr()), a.tokens_ld = tokens.stride(0);
    a.max_tokens = small(tokens.size(1), "tokens");
    if (given(arg[2])) a.lens = vector<int64_t>(tensor(arg[2], "lens"), B, at::kLong, index, "lens");
    if (given(arg[3])) a.prompt_lens = vector<int64_t>(tensor(arg[3], "prompt_lens"), B, at::kLong, index, "prompt_lens");
  } else {
    TORCH_CHECK_VALUE(!given(arg[2]) && !given(arg[3]), "lens and prompt_lens without tokens");
  }
  a.repetition_all = 1.f;
  per_row(arg[4], B, index, "repetition", a.repetition, a.repetition_all);
  per_row(arg[5], B, index, "presence", a.presence, a.presence_all);
  per_row(arg[6], B, index, "frequency", a.frequency, a.frequency_all);
  TORCH_CHECK_VALUE(a.repetition_all > 0.f, "repetition must be above 0, got ", a.repetition_all);
  TORCH_CHECK_VALUE(given(arg[7]) == given(arg[8]), "bias and bias_ids come together");
  if (given(arg[7])) {
    const Tensor &ids = tensor(arg[7], "bias_ids"), &bias = tensor(arg[8], "bias");
    TORCH_CHECK_VALUE(ids.dim() >= 1, "bias_ids must have a last dimension");
    const int64_t n = ids.size(-1);
    a.bias_ids_ld = by_row(ids, B, n, at::kLong, index, "bias_ids");
    a.bias_ld = by_row(bias, B, n, at::kFloat, index, "bias");
    a.bias_ids = static_cast<const int64_t*>(ids.data_ptr());
    a.bias = static_cast<const float*>(bias.data_ptr());
    a.num_bias = small(n, "bias_ids");
  }
  if (given(arg[9])) {
    const Tensor& allowed = tensor(arg[9], "allowed");
    a.allowed_ld = by_row(allowed, B, (V + 31) / 32, at::kInt, index, "allowed");
    a.allowed = static_cast<const int32_t*>(allowed.data_ptr());
  }
  c10::cuda::CUDAGuard guard(index);
  Tensor out;
  if (given(arg[10])) {
    out = tensor(arg[10], "out");
    on(out, index, "out");
    TORCH_CHECK_VALUE(out.dim() == 2 && out.size(0) == B && out.size(1) == V && (V <= 1 || out.stride(1) == 1),
                      "out must be [", B, ", ", V, "] with unit column stride");
    apart(out, x, true, "out", "logits");
  } else {
    out = at::empty({B, V}, x.options().dtype(at::kFloat));
  }
  a.logits = x.data_ptr(), a.out = out.data_ptr(), a.ld = x.stride(0), a.ld_out = out.stride(0);
  a.B = small(B, "B"), a.V = small(V, "V"), a.dtype = dtype_code(x, "logits"), a.out_dtype = dtype_code(out, "out");
  check(tread_adjust_logits(&a, stream_of(index)), "tread_adjust_logits");
  if (given(arg[10])) return Py_NewRef(arg[10]);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"paged_append", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(paged_append)), METH_FASTCALL, nullptr},
    {"paged_attn", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(paged_attn)), METH_FASTCALL, nullptr},
    {"adjust_logits", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(adjust_logits)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "tread_decode", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit_tread_decode(void) { return PyModule_Create(&module); }
