// Python binding of the rotary, paged, norm and 8-bit operators: checks of
// arguments, output tensors and workspace, and the C entry points of mrsa.h.
//
// A decode step is a chain of launches of a few microseconds each.  Checked and
// packed in Python, one such call took 11 to 15 us of host time, more than
// its kernels; here it is five to ten.  One function per operator, with
// positional arguments; the public functions with their defaults and
// documentation are in rotary.py, paged_cache.py, dense.py and int8.py.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/mrsa.h"

namespace {

using at::Tensor;

PyObject* g_check = nullptr;   // mrsa_b200._lib.check(code, name)

// An argument tensor, or an undefined one for None.
const Tensor& tensor(PyObject* o, const char* name) {
  static const Tensor none;
  if (o == Py_None) return none;
  if (!THPVariable_Check(o)) {
    TORCH_CHECK_TYPE(false, name, " must be a tensor");
  }
  return THPVariable_Unpack(o);
}

bool finish(int rc, const char* name) {
  if (rc == 0) return true;
  PyObject* r = PyObject_CallFunction(g_check, "is", rc, name);
  if (r != nullptr) {
    Py_DECREF(r);
    PyErr_SetString(PyExc_RuntimeError, name);
  }
  return false;
}

bool truth(PyObject* o) {
  const int r = PyObject_IsTrue(o);
  if (r < 0) throw python_error();
  return r != 0;
}

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

// No operator here has a forward-mode derivative: a tangent is an error, not lost.
void no_tangent(const char* op, std::initializer_list<const Tensor*> inputs) {
  for (const Tensor* x : inputs)
    TORCH_CHECK_NOT_IMPLEMENTED(!x->defined() || !x->_fw_grad(/*level=*/0).defined(), op, " has no forward-mode derivative");
}

// The frequencies are constants of a model: no gradient of theirs is recorded.
void fixed_frequencies(const Tensor& inv) {
  TORCH_CHECK_NOT_IMPLEMENTED(!c10::GradMode::is_enabled() || !inv.defined() || !inv.requires_grad(),
                              "the gradient of inv_freq is not recorded");
}

Tensor inner_contiguous(const Tensor& x) { return x.stride(-1) == 1 || x.size(-1) == 1 ? x : x.contiguous(); }

Tensor aligned(const Tensor& x) {
  Tensor y = x.contiguous();
  return reinterpret_cast<uintptr_t>(y.const_data_ptr()) % 16 == 0 ? y : y.clone();
}

template <typename T> const T* in(const Tensor& t) {
  return t.defined() ? static_cast<const T*>(t.const_data_ptr()) : nullptr;
}
template <typename T> T* out(const Tensor& t) { return t.defined() ? static_cast<T*>(t.mutable_data_ptr()) : nullptr; }

int type_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return MRSA_BF16;
    case at::kHalf: return MRSA_F16;
    case at::kFloat: return MRSA_F32;
    default: return -1;
  }
}

int layout_of(PyObject* o) {
  if (PyUnicode_Check(o)) {
    if (PyUnicode_CompareWithASCIIString(o, "half") == 0) return 0;
    if (PyUnicode_CompareWithASCIIString(o, "interleaved") == 0) return 1;
  }
  TORCH_CHECK_VALUE(false, "layout must be one of ('half', 'interleaved')");
}

void check_heads(const Tensor& x, const char* name) {
  TORCH_CHECK_VALUE(x.defined() && x.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK_VALUE(x.dim() == 4, name, " must be (B, L, H, D)");
}
void check_like(const Tensor& x, const char* name, const Tensor& like) {
  check_heads(x, name);
  TORCH_CHECK_VALUE(x.scalar_type() == like.scalar_type() && x.device() == like.device() && x.size(0) == like.size(0) &&
                        x.size(1) == like.size(1) && x.size(3) == like.size(3),
                    name, " must share type, device, (B, L) and D with the other heads");
}

// Frequencies and positions of a rotation; `inv` and `pos` keep what is passed on.
int64_t check_rotation(Tensor& inv, Tensor& pos, const Tensor& like) {
  const int64_t d = like.size(3), pairs = inv.dim() == 1 ? inv.size(0) : -1;
  TORCH_CHECK_VALUE(pairs >= 1 && pairs <= 128 && 2 * pairs <= d,
                    "inv_freq must be [n] with 2 n <= D and n <= 128, got ", inv.sizes(), ", D=", d);
  TORCH_CHECK_VALUE(!pos.defined() || (pos.dim() == 2 && pos.size(0) == like.size(0) && pos.size(1) == like.size(1) &&
                                       pos.scalar_type() == at::kLong && pos.device() == like.device()),
                    "position_ids must be int64 (B, L) on the tensors' device");
  if (inv.scalar_type() != at::kFloat || inv.device() != like.device()) inv = inv.to(like.device(), at::kFloat);
  if (!inv.is_contiguous()) inv = inv.contiguous();
  if (pos.defined() && !pos.is_contiguous()) pos = pos.contiguous();
  return pairs;
}

Tensor heads_like(const Tensor& x) { return at::empty(x.sizes(), x.options(), at::MemoryFormat::Contiguous); }

void set_q(mrsa_rotary_args& a, const Tensor& q, const Tensor& qo) {
  a.q = q.const_data_ptr();
  a.q_out = qo.mutable_data_ptr();
  a.q_batch_stride = q.stride(0);
  a.q_token_stride = q.stride(1);
  a.q_head_stride = q.stride(2);
  a.q_heads = q.size(2);
}
void set_k(mrsa_rotary_args& a, const Tensor& k) {
  a.k = k.const_data_ptr();
  a.k_batch_stride = k.stride(0);
  a.k_token_stride = k.stride(1);
  a.k_head_stride = k.stride(2);
  a.k_heads = k.size(2);
}

// (q', k') of checked arguments; k may be undefined.
std::pair<Tensor, Tensor> rotate(Tensor q, Tensor k, Tensor pos, Tensor inv, double factor, bool interleaved, bool inverse) {
  mrsa_rotary_args a = {};
  a.dtype = type_of(q);
  TORCH_CHECK_VALUE(a.dtype >= 0, "q must be BF16, FP16 or FP32, got ", q.scalar_type());
  if (k.defined()) check_like(k, "k", q);
  a.pairs = check_rotation(inv, pos, q);
  TORCH_CHECK_VALUE(!interleaved || q.size(3) % 2 == 0, "the interleaved layout needs an even head dim");
  q = inner_contiguous(q);
  Tensor qo = heads_like(q), ko;
  set_q(a, q, qo);
  if (k.defined()) {
    k = inner_contiguous(k);
    ko = heads_like(k);
    set_k(a, k);
    a.k_out = ko.mutable_data_ptr();
  }
  a.position_ids = in<int64_t>(pos);
  a.inv_freq = in<float>(inv);
  a.batch = q.size(0);
  a.len = q.size(1);
  a.head_dim = q.size(3);
  a.attention_factor = static_cast<float>(factor);
  a.interleaved = interleaved;
  a.inverse = inverse;
  const int rc = mrsa_rotary(&a, stream_of(q));
  TORCH_CHECK_VALUE(rc != MRSA_ERR_SHAPE && rc != MRSA_ERR_ARG && rc != MRSA_ERR_NULL && rc != MRSA_ERR_ALIGN,
                    "mrsa_rotary: ", mrsa_strerror(rc));
  TORCH_CHECK(rc == 0, "mrsa_rotary: ", mrsa_strerror(rc), " [", mrsa_last_error(), "]");
  return {std::move(qo), std::move(ko)};
}

// The gradient of a rotation is the rotation by minus the angle.
struct Rotary : torch::autograd::Function<Rotary> {
  using List = torch::autograd::variable_list;
  static List forward(torch::autograd::AutogradContext* ctx, const Tensor& q, const std::optional<Tensor>& k,
                      const Tensor& pos, const Tensor& inv, double factor, bool interleaved) {
    ctx->save_for_backward({pos, inv});
    ctx->saved_data["factor"] = factor;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["pair"] = k.has_value();
    auto [qo, ko] = rotate(q, k ? *k : Tensor(), pos, inv, factor, interleaved, false);
    return k ? List{qo, ko} : List{qo};
  }
  static List backward(torch::autograd::AutogradContext* ctx, const List& g) {
    TORCH_CHECK_NOT_IMPLEMENTED(!c10::GradMode::is_enabled(), "rotary_embedding: the gradient of its gradient is not recorded");
    const auto saved = ctx->get_saved_variables();
    auto [dq, dk] = rotate(g[0], ctx->saved_data["pair"].toBool() ? g[1] : Tensor(), saved[0], saved[1],
                           ctx->saved_data["factor"].toDouble(), ctx->saved_data["interleaved"].toBool(), true);
    return {dq, dk, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

// rotary(q, k, position_ids, inv_freq, attention_factor, layout)
PyObject* rotary(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 6, "rotary takes 6 arguments");
  const Tensor &q = tensor(o[0], "q"), &k = tensor(o[1], "k"), &pos = tensor(o[2], "position_ids"),
               &inv = tensor(o[3], "inv_freq");
  const double factor = PyFloat_AsDouble(o[4]);
  if (PyErr_Occurred()) return nullptr;
  const bool interleaved = layout_of(o[5]) == 1;
  check_heads(q, "q");
  TORCH_CHECK_VALUE(pos.defined() && inv.defined(), "position_ids must be int64 (B, L) and inv_freq fp32 [n]");
  no_tangent("rotary_embedding", {&q, &k, &inv});
  fixed_frequencies(inv);
  Tensor qo, ko;
  if (c10::GradMode::is_enabled() && (q.requires_grad() || (k.defined() && k.requires_grad()))) {
    const std::optional<Tensor> pair = k.defined() ? std::optional<Tensor>(k) : std::nullopt;
    auto r = Rotary::apply(q, pair, pos, inv, factor, interleaved);
    qo = std::move(r[0]);
    if (r.size() > 1) ko = std::move(r[1]);
  } else {
    std::tie(qo, ko) = rotate(q, k, pos, inv, factor, interleaved, false);
  }
  PyObject* r = PyTuple_New(2);
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(qo)));
  if (ko.defined()) {
    PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(ko)));
  } else {
    Py_INCREF(Py_None);
    PyTuple_SET_ITEM(r, 1, Py_None);
  }
  return r;
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------- pages
Tensor ints(const Tensor& x, const char* name, int64_t dim, const Tensor& like) {
  TORCH_CHECK_VALUE(x.defined() && x.scalar_type() == at::kInt && x.dim() == dim && x.is_cuda(), name,
                    " must be an int32 CUDA tensor with ", dim, dim > 1 ? " dimensions" : " dimension");
  TORCH_CHECK_VALUE(x.device() == like.device(), name, " must be on the table's device");
  return x.is_contiguous() ? x : x.contiguous();
}

// The state tensors are written, so they have to be contiguous.
mrsa_page_table page_table(const Tensor& table, const Tensor& lengths, const Tensor& refcount, const Tensor& status,
                           int64_t pages, int64_t page_size) {
  TORCH_CHECK_VALUE(table.defined() && table.scalar_type() == at::kInt && table.dim() == 2 && table.is_cuda() &&
                        table.is_contiguous(),
                    "table must be a contiguous int32 CUDA tensor [sequences, max_pages]");
  TORCH_CHECK_VALUE(lengths.defined() && lengths.scalar_type() == at::kInt && lengths.dim() == 1 &&
                        lengths.size(0) == table.size(0) && lengths.device() == table.device() && lengths.is_contiguous(),
                    "lengths must be contiguous int32 [sequences] on the table's device");
  if (refcount.defined()) {
    TORCH_CHECK_VALUE(refcount.scalar_type() == at::kInt && refcount.dim() == 1 && refcount.device() == table.device() &&
                          refcount.is_contiguous(),
                      "refcount must be contiguous int32 [pages] on the table's device");
    if (pages < 0) pages = refcount.size(0);
    TORCH_CHECK_VALUE(refcount.size(0) == pages, "refcount has ", refcount.size(0), " pages, the pool ", pages);
  }
  TORCH_CHECK_VALUE(page_size >= 16 && page_size <= 256 && (page_size & (page_size - 1)) == 0,
                    "page_size must be one of (16, 32, 64, 128, 256), got ", page_size);
  TORCH_CHECK_VALUE(!status.defined() || (status.scalar_type() == at::kInt && status.numel() == 1 &&
                                          status.device() == table.device()),
                    "status must be one int32 on the table's device");
  mrsa_page_table t = {};
  t.table = out<int32_t>(table);
  t.lengths = out<int32_t>(lengths);
  t.refcount = out<int32_t>(refcount);
  t.status = out<int32_t>(status);
  t.max_seqs = table.size(0);
  t.max_pages = table.size(1);
  t.pages = pages;
  t.page_size = page_size;
  return t;
}

// Memory that is written must not stand for several elements (an expanded tensor).
void check_written(const Tensor& x, const char* name) {
  TORCH_CHECK_VALUE(at::has_internal_overlap(x) != at::MemOverlap::Yes, name, " is written: its elements must not share memory");
}

mrsa_page_pool page_pool(const Tensor& pool, const Tensor& like) {
  TORCH_CHECK_VALUE(pool.defined() && pool.dim() == 6 && pool.size(1) == 2 && pool.device() == like.device(),
                    "pool must be [layers, 2, pages, page_size, kv_heads, D] on the table's device");
  check_written(pool, "pool");
  const auto s = pool.strides();
  const int64_t ps = pool.size(3), heads = pool.size(4), d = pool.size(5), e = pool.element_size();
  TORCH_CHECK_VALUE(s[5] == 1 && ((s[3] == heads * d && s[4] == d) || (s[3] == d && s[4] == ps * d)),
                    "each page of the pool must be one contiguous block, tokens or heads outside");
  mrsa_page_pool p = {};
  p.data = pool.mutable_data_ptr();
  p.layers = pool.size(0);
  p.layer_stride = s[0] * e;
  p.kv_stride = s[1] * e;
  p.page_stride = s[2] * e;
  p.token_stride = s[3] * e;
  p.head_stride = s[4] * e;
  p.heads = heads;
  p.row_bytes = d * e;
  return p;
}

Tensor bytes_on(const Tensor& like, size_t n) {
  return at::empty({static_cast<int64_t>(n)}, like.options().dtype(at::kByte));
}

int64_t count_of(const Tensor& x, const char* name) {
  TORCH_CHECK_VALUE(x.size(0) <= MRSA_PAGE_MAX_SEQS, name, ": at most ", MRSA_PAGE_MAX_SEQS, " sequences per call, got ",
                    x.size(0));
  return x.size(0);
}

// free(table, lengths, refcount, seqs, status)
PyObject* page_free(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 5, "free takes 5 arguments");
  const Tensor &table = tensor(o[0], "table"), &lengths = tensor(o[1], "lengths"), &refcount = tensor(o[2], "refcount");
  const mrsa_page_table t = page_table(table, lengths, refcount, tensor(o[4], "status"), -1, 16);
  const Tensor seqs = ints(tensor(o[3], "seqs"), "seqs", 1, table);
  if (!finish(mrsa_page_free(&t, in<int32_t>(seqs), count_of(seqs, "seqs"), stream_of(table)), "mrsa_page_free"))
    return nullptr;
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// extend(table, lengths, refcount, seqs, tokens, page_size, status)
PyObject* page_extend(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 7, "extend takes 7 arguments");
  const Tensor &table = tensor(o[0], "table"), &lengths = tensor(o[1], "lengths"), &refcount = tensor(o[2], "refcount");
  const int64_t page_size = PyLong_AsLongLong(o[5]);
  if (PyErr_Occurred()) return nullptr;
  const mrsa_page_table t = page_table(table, lengths, refcount, tensor(o[6], "status"), -1, page_size);
  const Tensor seqs = ints(tensor(o[3], "seqs"), "seqs", 1, table);
  const int64_t count = count_of(seqs, "seqs");
  Tensor each;
  int64_t all = 0;
  if (THPVariable_Check(o[4])) {
    each = ints(THPVariable_Unpack(o[4]), "tokens", 1, table);
    TORCH_CHECK_VALUE(each.size(0) == count, "tokens must hold one number per sequence");
  } else {
    all = PyLong_AsLongLong(o[4]);
    if (PyErr_Occurred()) return nullptr;
    TORCH_CHECK_VALUE(all >= 0, "a sequence cannot grow by a negative number of tokens");
  }
  if (count > 0) {
    const size_t size = mrsa_page_workspace(&t, count);
    const Tensor ws = bytes_on(table, size);
    if (!finish(mrsa_page_extend(&t, in<int32_t>(seqs), in<int32_t>(each), all, count, ws.mutable_data_ptr(), size,
                                 stream_of(table)), "mrsa_page_extend"))
      return nullptr;
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// fork(pool, table, lengths, refcount, src, dst, share, status)
PyObject* page_fork(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 8, "fork takes 8 arguments");
  const Tensor &pool = tensor(o[0], "pool"), &table = tensor(o[1], "table"), &lengths = tensor(o[2], "lengths"),
               &refcount = tensor(o[3], "refcount");
  Tensor share = tensor(o[6], "share");
  const mrsa_page_pool p = page_pool(pool, table);
  const mrsa_page_table t = page_table(table, lengths, refcount, tensor(o[7], "status"), pool.size(2), pool.size(3));
  const Tensor src = ints(tensor(o[4], "src"), "src", 1, table), dst = ints(tensor(o[5], "dst"), "dst", 1, table);
  const int64_t count = count_of(dst, "dst");
  if (share.defined()) share = ints(share, "share", 1, table);
  TORCH_CHECK_VALUE(src.size(0) == count && (!share.defined() || share.size(0) == count),
                    "src, dst and share must have one entry per fork");
  if (count > 0) {
    const size_t size = mrsa_page_workspace(&t, count);
    const Tensor ws = bytes_on(table, size);
    if (!finish(mrsa_page_fork(&t, &p, in<int32_t>(src), in<int32_t>(dst), in<int32_t>(share), count,
                               ws.mutable_data_ptr(), size, stream_of(table)), "mrsa_page_fork"))
      return nullptr;
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// compact(pool, table, lengths, refcount, seqs, keep, status)
PyObject* page_compact(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 7, "compact takes 7 arguments");
  const Tensor &pool = tensor(o[0], "pool"), &table = tensor(o[1], "table"), &lengths = tensor(o[2], "lengths"),
               &refcount = tensor(o[3], "refcount");
  Tensor keep = tensor(o[5], "keep");
  const mrsa_page_pool p = page_pool(pool, table);
  const mrsa_page_table t = page_table(table, lengths, refcount, tensor(o[6], "status"), pool.size(2), pool.size(3));
  const Tensor seqs = ints(tensor(o[4], "seqs"), "seqs", 1, table);
  const int64_t count = count_of(seqs, "seqs");
  TORCH_CHECK_VALUE(keep.defined() && keep.scalar_type() == at::kBool && keep.dim() == 2 && keep.size(0) == count &&
                        keep.size(1) == t.max_pages * t.page_size && keep.device() == table.device(),
                    "keep must be bool (", count, ", ", t.max_pages * t.page_size, ") on the table's device");
  if (count > 0) {
    keep = aligned(keep);
    const size_t size = mrsa_page_workspace(&t, count);
    const Tensor ws = bytes_on(table, size);
    if (!finish(mrsa_page_compact(&t, &p, in<int32_t>(seqs), in<uint8_t>(keep), count, ws.mutable_data_ptr(), size,
                                  stream_of(table)), "mrsa_page_compact"))
      return nullptr;
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// copy(pool, src, dst, status)
PyObject* page_copy(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 4, "copy takes 4 arguments");
  const Tensor& pool = tensor(o[0], "pool");
  TORCH_CHECK_VALUE(pool.defined() && pool.is_cuda(), "pool must be a CUDA tensor");
  const mrsa_page_pool p = page_pool(pool, pool);
  const Tensor src = ints(tensor(o[1], "src"), "src", 1, pool), dst = ints(tensor(o[2], "dst"), "dst", 1, pool);
  TORCH_CHECK_VALUE(src.size(0) == dst.size(0), "src and dst must have one entry per page");
  TORCH_CHECK_VALUE(src.size(0) <= pool.size(2), src.size(0), " copies into ", pool.size(2), " pages");
  if (src.size(0) > 0) {
    // a copy reads no table: one row of one page stands for it
    const mrsa_page_table t = page_table(src.slice(0, 0, 1).view({1, 1}), src.slice(0, 0, 1), Tensor(),
                                         tensor(o[3], "status"), pool.size(2), pool.size(3));
    const size_t size = src.size(0) > 1 ? mrsa_page_copy_workspace(&t) : 0;
    const Tensor ws = bytes_on(pool, size);
    if (!finish(mrsa_page_copy_checked(&t, &p, in<int32_t>(src), in<int32_t>(dst), src.size(0), ws.mutable_data_ptr(),
                                       size, stream_of(pool)), "mrsa_page_copy"))
      return nullptr;
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// An operator without a backward pass raises rather than lose a gradient.
void forward_only(const char* op, std::initializer_list<const Tensor*> inputs) {
  if (!c10::GradMode::is_enabled()) return;
  for (const Tensor* x : inputs)
    TORCH_CHECK_NOT_IMPLEMENTED(!x->defined() || !x->requires_grad(), op, " is forward-only");
}

// A layer's pages.
void check_pages(const Tensor& k, const Tensor& v) {
  TORCH_CHECK_VALUE(k.defined() && v.defined() && k.dim() == 4 && v.sizes() == k.sizes(),
                    "k_pages and v_pages must share a [pages, page_size, kv_heads, D] shape");
  TORCH_CHECK_VALUE(v.scalar_type() == k.scalar_type() && v.device() == k.device() && k.is_cuda(),
                    "k_pages and v_pages must share type and CUDA device");
  TORCH_CHECK_VALUE(k.stride(3) == 1 && v.stride(3) == 1,
                    "the last dimension of k_pages and v_pages must be contiguous");
}

// append(k_pages, v_pages, table, lengths, seqs, k, v, q, position_ids, inv_freq, attention_factor, layout, start,
//        refcount, status)
PyObject* append(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 15, "append takes 15 arguments");
  const Tensor &kp = tensor(o[0], "k_pages"), &vp = tensor(o[1], "v_pages"), &table = tensor(o[2], "table"),
               &lengths = tensor(o[3], "lengths"), &refcount = tensor(o[13], "refcount");
  Tensor k = tensor(o[5], "k"), v = tensor(o[6], "v"), q = tensor(o[7], "q"), pos = tensor(o[8], "position_ids"),
         inv = tensor(o[9], "inv_freq"), start = tensor(o[12], "start");
  const double factor = PyFloat_AsDouble(o[10]);
  if (PyErr_Occurred()) return nullptr;
  mrsa_rotary_args a = {};
  a.interleaved = layout_of(o[11]);
  check_heads(k, "k");
  check_like(v, "v", k);
  TORCH_CHECK_VALUE(v.size(2) == k.size(2), "v must have k's shape");
  check_pages(kp, vp);
  check_written(kp, "k_pages");
  check_written(vp, "v_pages");
  TORCH_CHECK_VALUE(kp.const_data_ptr() != vp.const_data_ptr() || kp.numel() == 0,
                    "k_pages and v_pages are written: they must not be the same memory");
  a.dtype = type_of(k);
  TORCH_CHECK_VALUE(a.dtype >= 0 && kp.scalar_type() == k.scalar_type() && kp.device() == k.device(),
                    "k, v and the pages must share a type (BF16, FP16 or FP32) and a device");
  TORCH_CHECK_VALUE(kp.size(2) == k.size(2) && kp.size(3) == k.size(3), "the pages hold heads of (", kp.size(2), ", ",
                    kp.size(3), "), k has (", k.size(2), ", ", k.size(3), ")");
  const mrsa_page_table t = page_table(table, lengths, refcount, tensor(o[14], "status"), kp.size(0), kp.size(1));
  TORCH_CHECK_VALUE(table.device() == k.device(), "the table must be on the tensors' device");
  const Tensor seqs = ints(tensor(o[4], "seqs"), "seqs", 1, table);
  TORCH_CHECK_VALUE(seqs.size(0) == k.size(0), "seqs must name one sequence per batch row");
  forward_only("paged_append", {&q, &k, &v, &kp, &vp});
  no_tangent("paged_append", {&q, &k, &v, &kp, &vp, &inv});
  fixed_frequencies(inv);
  if (inv.defined()) {
    a.pairs = check_rotation(inv, pos, k);
    a.inv_freq = in<float>(inv);
    a.position_ids = in<int64_t>(pos);
  }
  if (start.defined()) {
    start = ints(start, "start", 1, table);
    TORCH_CHECK_VALUE(start.size(0) == k.size(0), "start must hold one position per sequence");
  }
  TORCH_CHECK_VALUE(!a.interleaved || k.size(3) % 2 == 0, "the interleaved layout needs an even head dim");
  k = inner_contiguous(k);
  v = inner_contiguous(v);
  Tensor qo;
  if (q.defined()) {
    check_like(q, "q", k);
    q = inner_contiguous(q);
    qo = heads_like(q);
    set_q(a, q, qo);
  }
  set_k(a, k);
  a.batch = k.size(0);
  a.len = k.size(1);
  a.head_dim = k.size(3);
  a.attention_factor = static_cast<float>(factor);
  mrsa_paged_append_args p = {};
  p.k_pages = kp.mutable_data_ptr();
  p.v_pages = vp.mutable_data_ptr();
  p.v = v.const_data_ptr();
  p.seqs = in<int32_t>(seqs);
  p.start = in<int32_t>(start);
  p.k_page_stride = kp.stride(0);
  p.k_slot_stride = kp.stride(1);
  p.k_head_stride = kp.stride(2);
  p.v_page_stride = vp.stride(0);
  p.v_slot_stride = vp.stride(1);
  p.vp_head_stride = vp.stride(2);
  p.v_batch_stride = v.stride(0);
  p.v_token_stride = v.stride(1);
  p.v_head_stride = v.stride(2);
  p.check_shared = refcount.defined();
  if (!finish(mrsa_paged_append(&a, &t, &p, stream_of(k)), "mrsa_paged_append")) return nullptr;
  if (!qo.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(qo));
  END_HANDLE_TH_ERRORS
}

// attend(q, k_pages, v_pages, table, lengths, seqs, causal, key_valid, scale, return_lse, status)
PyObject* attend(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 11, "attend takes 11 arguments");
  Tensor q = tensor(o[0], "q"), valid = tensor(o[7], "key_valid");
  const Tensor &kp = tensor(o[1], "k_pages"), &vp = tensor(o[2], "v_pages"), &table = tensor(o[3], "table"),
               &lengths = tensor(o[4], "lengths");
  check_heads(q, "q");
  check_pages(kp, vp);
  const int64_t b = q.size(0), l = q.size(1), hq = q.size(2), d = q.size(3), hkv = kp.size(2);
  mrsa_paged_attention_args a = {};
  a.dtype = type_of(q);
  TORCH_CHECK_VALUE((a.dtype == MRSA_BF16 || a.dtype == MRSA_F16) && kp.scalar_type() == q.scalar_type() &&
                        kp.device() == q.device(),
                    "q and the pages must share a type (BF16 or FP16) and a device");
  TORCH_CHECK_VALUE((d == 64 || d == 128) && kp.size(3) == d && hkv >= 1 && hq >= hkv && hq % hkv == 0,
                    "heads must be of 64 or 128 dims, Hq a multiple of Hkv; got q ", q.sizes(), ", pages ", kp.sizes());
  forward_only("paged_attention", {&q, &kp, &vp});
  no_tangent("paged_attention", {&q, &kp, &vp});
  const mrsa_page_table t = page_table(table, lengths, Tensor(), tensor(o[10], "status"), kp.size(0), kp.size(1));
  TORCH_CHECK_VALUE(table.device() == q.device(), "the table must be on the tensors' device");
  const Tensor seqs = ints(tensor(o[5], "seqs"), "seqs", 1, table);
  TORCH_CHECK_VALUE(seqs.size(0) == b, "seqs must name one sequence per batch row");
  a.causal = truth(o[6]);
  double scale = d == 64 ? 0.125 : 0.08838834764831845;
  if (o[8] != Py_None) {
    scale = PyFloat_AsDouble(o[8]);
    if (PyErr_Occurred()) return nullptr;
    TORCH_CHECK_VALUE(scale > 0, "scale must be positive");
  }
  a.scale = static_cast<float>(scale);
  if (valid.defined()) {
    TORCH_CHECK_VALUE(valid.scalar_type() == at::kBool && valid.dim() == 2 && valid.size(0) == b &&
                          valid.size(1) == t.max_pages * t.page_size && valid.device() == q.device(),
                      "key_valid must be bool (", b, ", ", t.max_pages * t.page_size, ") on the tensors' device");
    valid = aligned(valid);
    a.key_valid = in<uint8_t>(valid);
  }
  if (q.stride(3) != 1 || q.stride(0) <= 0 || q.stride(1) <= 0 || q.stride(2) <= 0 || ((q.stride(0) | q.stride(1) | q.stride(2)) & 7) ||
      (reinterpret_cast<uintptr_t>(q.const_data_ptr()) & 15))
    q = aligned(q);
  Tensor out = heads_like(q), lse;
  if (truth(o[9])) {
    lse = at::empty({b, l, hq}, q.options().dtype(at::kFloat));
    a.lse = lse.mutable_data_ptr<float>();
  }
  a.q = q.const_data_ptr();
  a.k_pages = kp.const_data_ptr();
  a.v_pages = vp.const_data_ptr();
  a.out = out.mutable_data_ptr();
  a.seqs = in<int32_t>(seqs);
  a.q_batch_stride = q.stride(0);
  a.q_token_stride = q.stride(1);
  a.q_head_stride = q.stride(2);
  a.k_page_stride = kp.stride(0);
  a.k_slot_stride = kp.stride(1);
  a.k_head_stride = kp.stride(2);
  a.v_page_stride = vp.stride(0);
  a.v_slot_stride = vp.stride(1);
  a.v_head_stride = vp.stride(2);
  a.batch = b;
  a.len = l;
  a.q_heads = hq;
  a.kv_heads = hkv;
  a.head_dim = d;
  const size_t size = mrsa_paged_attention_workspace(&a);
  const Tensor ws = bytes_on(q, size);
  if (!finish(mrsa_paged_attention(&a, &t, ws.mutable_data_ptr(), size, stream_of(q)), "mrsa_paged_attention"))
    return nullptr;
  if (!lse.defined()) return THPVariable_Wrap(std::move(out));
  PyObject* r = PyTuple_New(2);
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(out)));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(lse)));
  return r;
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------- norms and 8 bits
int float_type(const Tensor& t, const char* name) {
  const int type = type_of(t);
  TORCH_CHECK_VALUE(type >= 0, name, " must be BF16, FP16 or FP32, got ", t.scalar_type());
  return type;
}

// [..., D] as [rows, D], the last dimension contiguous.
Tensor as_rows(const Tensor& x, const char* name) {
  TORCH_CHECK_VALUE(x.defined() && x.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, name, " must be (..., D) with D at least 1, got ", x.sizes());
  const Tensor y = x.dim() == 2 ? x : x.reshape({x.numel() / x.size(-1), x.size(-1)});
  return inner_contiguous(y);
}

int64_t pitch_of(int64_t n) { return (n + 15) / 16 * 16; }

// 8-bit rows like x's, 16 bytes times a whole number apart, and their scales.
std::pair<Tensor, Tensor> whole_like(const Tensor& x) {
  const int64_t k = x.size(-1);
  std::vector<int64_t> strides(x.dim(), 1);
  for (int64_t i = x.dim() - 2, step = pitch_of(k); i >= 0; --i) {
    strides[i] = step;
    step *= x.size(i);
  }
  return {at::empty_strided(x.sizes(), strides, x.options().dtype(at::kChar)),
          at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat))};
}

// The checked arguments of a norm: x, residual (or none) and weight as the C entry takes them.
struct Norm {
  Tensor x, residual, weight;
  mrsa_norm_args a = {};
  Norm(const Tensor& x_in, const Tensor& r_in, const Tensor& w_in, double eps) {
    x = as_rows(x_in, "x");
    a.dtype = float_type(x, "x");
    a.rows = x.size(0);
    a.dim = x.size(1);
    TORCH_CHECK_VALUE(w_in.defined() && w_in.dim() == 1 && w_in.size(0) == a.dim && w_in.scalar_type() == x.scalar_type() &&
                          w_in.device() == x.device(),
                      "weight must be (", a.dim, ") of x's type and device");
    weight = w_in.contiguous();
    if (r_in.defined()) {
      TORCH_CHECK_VALUE(r_in.sizes() == x_in.sizes() && r_in.scalar_type() == x.scalar_type() && r_in.device() == x.device(),
                        "residual must share x's shape, type and device");
      residual = as_rows(r_in, "residual");
      a.residual = residual.const_data_ptr();
      a.residual_stride = residual.stride(0);
    }
    TORCH_CHECK_VALUE(eps >= MRSA_NORM_MIN_EPS && eps <= 3.4028234663852886e38, "eps must be at least 1e-12, got ", eps);
    a.eps = static_cast<float>(eps);
    a.x = x.const_data_ptr();
    a.weight = weight.const_data_ptr();
    a.x_stride = x.stride(0);
  }
};

void checked(int rc, const char* name) {
  TORCH_CHECK_VALUE(rc != MRSA_ERR_SHAPE && rc != MRSA_ERR_ARG && rc != MRSA_ERR_NULL && rc != MRSA_ERR_ALIGN, name, ": ",
                    mrsa_strerror(rc));
  TORCH_CHECK(rc == 0, name, ": ", mrsa_strerror(rc), " [", mrsa_last_error(), "]");
}

// y, with a residual h, and with `keep` 1 / rms of each row.
struct Normed {
  Tensor y, h, rstd;
};
Normed add_norm(const Tensor& x, const Tensor& residual, const Tensor& weight, double eps, bool keep) {
  Norm n(x, residual, weight, eps);
  Normed r;
  r.y = heads_like(x);
  n.a.y = r.y.mutable_data_ptr();
  if (residual.defined()) {
    r.h = heads_like(x);
    n.a.h = r.h.mutable_data_ptr();
  }
  if (keep) {
    r.rstd = at::empty({n.a.rows}, x.options().dtype(at::kFloat));
    n.a.rstd = r.rstd.mutable_data_ptr<float>();
  }
  if (n.a.rows > 0) checked(mrsa_add_rms_norm(&n.a, stream_of(x)), "mrsa_add_rms_norm");
  return r;
}

struct AddRmsNorm : torch::autograd::Function<AddRmsNorm> {
  using List = torch::autograd::variable_list;
  static List forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& residual,
                      const Tensor& weight, double eps) {
    ctx->set_materialize_grads(false);
    const Normed r = add_norm(x, residual ? *residual : Tensor(), weight, eps, true);
    ctx->saved_data["add"] = residual.has_value();
    ctx->save_for_backward({residual ? r.h : x, weight, r.rstd});
    return residual ? List{r.y, r.h} : List{r.y};
  }
  static List backward(torch::autograd::AutogradContext* ctx, const List& g) {
    TORCH_CHECK_NOT_IMPLEMENTED(!c10::GradMode::is_enabled(), "add_rms_norm: the gradient of its gradient is not recorded");
    const bool add = ctx->saved_data["add"].toBool();
    const Tensor gh = add ? g[1] : Tensor();
    if (!g[0].defined()) return {gh, add ? gh : Tensor(), Tensor(), Tensor()};
    const auto saved = ctx->get_saved_variables();
    const Tensor gy = as_rows(g[0], "the gradient"), h = as_rows(saved[0], "h"), weight = saved[1].contiguous();
    mrsa_norm_backward_args a = {};
    a.rows = h.size(0);
    a.dim = h.size(1);
    Tensor dx = heads_like(saved[0]), dw, ws, gh2;
    const bool want_w = ctx->needs_input_grad(add ? 2 : 1);
    if (a.rows == 0) return {dx, add ? dx : Tensor(), want_w ? at::zeros_like(weight) : Tensor(), Tensor()};
    size_t size = 0;
    if (want_w) {
      dw = at::empty_like(weight);
      size = mrsa_add_rms_norm_backward_workspace(a.rows, a.dim);
      ws = bytes_on(h, size);
      a.dweight = dw.mutable_data_ptr();
    }
    if (gh.defined()) {
      gh2 = as_rows(gh, "the gradient");
      a.grad_h = gh2.const_data_ptr();
      a.grad_h_stride = gh2.stride(0);
    }
    a.grad_y = gy.const_data_ptr();
    a.grad_y_stride = gy.stride(0);
    a.h = h.const_data_ptr();
    a.h_stride = h.stride(0);
    a.weight = weight.const_data_ptr();
    a.rstd = saved[2].const_data_ptr<float>();
    a.dx = dx.mutable_data_ptr();
    a.dtype = type_of(h);
    checked(mrsa_add_rms_norm_backward(&a, want_w ? ws.mutable_data_ptr() : nullptr, size, stream_of(h)),
            "mrsa_add_rms_norm_backward");
    return {dx, add ? dx : Tensor(), dw, Tensor()};
  }
};

PyObject* tuple_of(std::initializer_list<Tensor> all) {
  PyObject* r = PyTuple_New(static_cast<Py_ssize_t>(all.size()));
  Py_ssize_t i = 0;
  for (const Tensor& t : all) PyTuple_SET_ITEM(r, i++, THPVariable_Wrap(t));
  return r;
}

// add_rms_norm(x, residual, weight, eps) -> (y, h)
PyObject* add_rms_norm(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 4, "add_rms_norm takes 4 arguments");
  const Tensor &x = tensor(o[0], "x"), &residual = tensor(o[1], "residual"), &weight = tensor(o[2], "weight");
  const double eps = PyFloat_AsDouble(o[3]);
  if (PyErr_Occurred()) return nullptr;
  no_tangent("add_rms_norm", {&x, &residual, &weight});
  TORCH_CHECK_VALUE(x.defined() && weight.defined(), "x and weight must be tensors");
  if (c10::GradMode::is_enabled() &&
      (x.requires_grad() || weight.requires_grad() || (residual.defined() && residual.requires_grad()))) {
    const std::optional<Tensor> add = residual.defined() ? std::optional<Tensor>(residual) : std::nullopt;
    const auto r = AddRmsNorm::apply(x, add, weight, eps);
    return tuple_of({r[0], r.size() > 1 ? r[1] : x});
  }
  const Normed r = add_norm(x, residual, weight, eps, false);
  return tuple_of({r.y, r.h.defined() ? r.h : x});
  END_HANDLE_TH_ERRORS
}

// add_rms_norm_int8(x, residual, weight, eps) -> (q, scale, h)
PyObject* add_rms_norm_int8(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 4, "add_rms_norm_int8 takes 4 arguments");
  const Tensor &x = tensor(o[0], "x"), &residual = tensor(o[1], "residual"), &weight = tensor(o[2], "weight");
  const double eps = PyFloat_AsDouble(o[3]);
  if (PyErr_Occurred()) return nullptr;
  forward_only("add_rms_norm_int8", {&x, &residual, &weight});
  no_tangent("add_rms_norm_int8", {&x, &residual, &weight});
  Norm c(x, residual, weight, eps);
  auto [q, scale] = whole_like(x);
  Tensor h = x;
  if (residual.defined()) {
    h = heads_like(x);
    c.a.h = h.mutable_data_ptr();
  }
  c.a.q = q.mutable_data_ptr<int8_t>();
  c.a.q_stride = pitch_of(c.a.dim);
  c.a.scale = scale.mutable_data_ptr<float>();
  if (c.a.rows > 0 && !finish(mrsa_add_rms_norm(&c.a, stream_of(x)), "mrsa_add_rms_norm")) return nullptr;
  return tuple_of({q, scale, h});
  END_HANDLE_TH_ERRORS
}

// quantize_int8(x) -> (q, scale)
PyObject* quantize_int8(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 1, "quantize_int8 takes 1 argument");
  const Tensor& x = tensor(o[0], "x");
  forward_only("quantize_int8", {&x});
  no_tangent("quantize_int8", {&x});
  const Tensor rows = as_rows(x, "x");
  const int type = float_type(x, "x");
  auto [q, scale] = whole_like(x);
  if (!finish(mrsa_quantize_int8(rows.const_data_ptr(), rows.stride(0), q.mutable_data_ptr<int8_t>(), pitch_of(rows.size(1)),
                                 scale.mutable_data_ptr<float>(), rows.size(0), rows.size(1), type, stream_of(x)),
              "mrsa_quantize_int8"))
    return nullptr;
  return tuple_of({q, scale});
  END_HANDLE_TH_ERRORS
}

// 8-bit rows as the products read them: on 16-byte boundaries, or copied to such rows.
Tensor whole_rows(const Tensor& x, const char* name) {
  TORCH_CHECK_VALUE(x.defined() && x.scalar_type() == at::kChar, name, " must be INT8");
  Tensor y = as_rows(x, name);
  const int64_t k = y.size(1);
  const bool fit = reinterpret_cast<uintptr_t>(y.const_data_ptr()) % 16 == 0 &&
                   (y.size(0) <= 1 || (y.stride(0) % 16 == 0 && y.stride(0) >= k));
  if (fit) return y;
  TORCH_CHECK_VALUE(k <= MRSA_INT8_MAX_K, name, " must have at most ", MRSA_INT8_MAX_K, " columns (sums of 32 bits)");
  Tensor z = at::empty({y.size(0), pitch_of(k)}, y.options());
  checked(mrsa_align_rows_int8(y.const_data_ptr<int8_t>(), y.stride(0), z.mutable_data_ptr<int8_t>(), pitch_of(k), y.size(0), k,
                               stream_of(y)), "mrsa_align_rows_int8");
  return z.narrow(1, 0, k);
}
int64_t row_pitch(const Tensor& x) { return x.size(0) > 1 ? x.stride(0) : pitch_of(x.size(1)); }

Tensor scales(const Tensor& x, const char* name, at::IntArrayRef sizes, const Tensor& like) {
  TORCH_CHECK_VALUE(x.defined() && x.scalar_type() == at::kFloat && x.sizes() == sizes && x.device() == like.device(), name,
                    " must be FP32 ", sizes, " on the tensors' device");
  return x.contiguous();
}

// linear_int8(q, scale, weight, weight_scale, bias, dtype, gated)
PyObject* linear_int8(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 7, "linear_int8 takes 7 arguments");
  const Tensor &q = tensor(o[0], "q"), &weight = tensor(o[2], "weight");
  Tensor bias = tensor(o[4], "bias");
  TORCH_CHECK_TYPE(THPDtype_Check(o[5]), "dtype must be a torch.dtype");
  const at::ScalarType type = reinterpret_cast<THPDtype*>(o[5])->scalar_type;
  const bool gated = truth(o[6]);
  forward_only("linear_int8", {&tensor(o[1], "scale"), &tensor(o[3], "weight_scale"), &bias});
  no_tangent("linear_int8", {&tensor(o[1], "scale"), &tensor(o[3], "weight_scale"), &bias});
  TORCH_CHECK_VALUE(weight.defined() && weight.dim() == 2, "weight must be (N, K)");
  const Tensor a = whole_rows(q, "q"), b = whole_rows(weight, "weight");
  TORCH_CHECK_VALUE(a.device() == b.device() && a.size(1) == b.size(1), "q and weight must share a device and K, got ",
                    q.sizes(), " and ", weight.sizes());
  TORCH_CHECK_VALUE(b.size(0) >= 1 && a.size(1) <= MRSA_INT8_MAX_K, "weight must have rows, and at most ", MRSA_INT8_MAX_K,
                    " columns (sums of 32 bits)");
  TORCH_CHECK_VALUE(!gated || b.size(0) % 256 == 0, "the gated product takes weights in blocks of 256 rows, got ", b.size(0));
  const Tensor sa = scales(tensor(o[1], "scale"), "scale", q.sizes().slice(0, q.dim() - 1), a),
               sb = scales(tensor(o[3], "weight_scale"), "weight_scale", {b.size(0)}, a);
  std::vector<int64_t> sizes = q.sizes().vec();
  sizes.back() = gated ? b.size(0) / 2 : b.size(0);
  Tensor out = at::empty(sizes, a.options().dtype(type));
  mrsa_gemm_int8_args p = {};
  p.dtype = type_of(out);
  TORCH_CHECK_VALUE(p.dtype >= 0, "dtype must be BF16, FP16 or FP32, got ", type);
  if (bias.defined()) {
    TORCH_CHECK_VALUE(bias.dim() == 1 && bias.size(0) == b.size(0) && bias.device() == a.device(),
                      "bias must be (", b.size(0), ") on the tensors' device");
    p.bias_dtype = float_type(bias, "bias");
    bias = bias.contiguous();
    p.bias = bias.const_data_ptr();
  }
  p.a = a.const_data_ptr<int8_t>();
  p.b = b.const_data_ptr<int8_t>();
  p.a_scale = sa.const_data_ptr<float>();
  p.b_scale = sb.const_data_ptr<float>();
  p.c = out.mutable_data_ptr();
  p.m = a.size(0);
  p.n = b.size(0);
  p.k = a.size(1);
  p.a_stride = row_pitch(a);
  p.b_stride = row_pitch(b);
  p.epilogue = gated ? MRSA_GEMM_SWIGLU : MRSA_GEMM_PLAIN;
  if (!finish(mrsa_gemm_int8(&p, stream_of(a)), "mrsa_gemm_int8")) return nullptr;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// set_check(callable): what turns a negative code of the library into an exception
PyObject* set_check(PyObject*, PyObject* f) {
  Py_INCREF(f);
  Py_XDECREF(g_check);
  g_check = f;
  Py_RETURN_NONE;
}

#define FAST(name, f) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {FAST("rotary", rotary), FAST("free", page_free), FAST("extend", page_extend),
                          FAST("fork", page_fork), FAST("compact", page_compact), FAST("copy", page_copy),
                          FAST("append", append), FAST("attend", attend),
                          FAST("add_rms_norm", add_rms_norm), FAST("add_rms_norm_int8", add_rms_norm_int8),
                          FAST("quantize_int8", quantize_int8), FAST("linear_int8", linear_int8),
                          {"set_check", set_check, METH_O, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "mrsa_b200_ext", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_mrsa_b200_ext(void) { return PyModule_Create(&kModule); }
