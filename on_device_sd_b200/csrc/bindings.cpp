// Python entry of the step operators: on_device_sd_b200/_step.so, called by attention.py and speculative.py.
//
// A draft step's kernels take a few microseconds, and checking a dozen tensors, filling the argument struct and
// allocating from Python takes 8-10 (measured with ctypes; a whole call from here, launches included, is 4.3 us for the cache
// write, 5 for verification, 4.5 for attention and 8 where it is cut, with a workspace and a second launch).  So these
// functions take the tensors themselves: they check devices, types, shapes and strides, allocate the outputs and the
// workspace from torch's allocator, and call the C ABI (include/b200moe.h) on the current stream of the tensors' device.  No
// arithmetic happens here.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <string>

#include "../../include/b200moe.h"
#include "overlap.h"

// What this file was compiled against; build.py and _lib.py read it from the file before they load it.
#ifndef B200MOE_STEP_TAG
#error "compile with build.py, which names the torch and the Python that this is built against"
#endif
extern "C" __attribute__((used, visibility("default"))) const char b200moe_step_tag[] = "b200moe_step built for <" B200MOE_STEP_TAG ">";

namespace {

struct Refusal {                     // becomes a Python exception
  PyObject* type;
  std::string text;
};
[[noreturn]] void refuse(PyObject* type, std::string text) { throw Refusal{type, std::move(text)}; }

std::string shape_text(at::IntArrayRef s) {
  std::string t = "(";
  for (size_t i = 0; i < s.size(); ++i) t += (i ? ", " : "") + std::to_string(s[i]);
  return t + ")";
}
const char* type_text(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return "torch.float32";
    case at::kHalf: return "torch.float16";
    case at::kBFloat16: return "torch.bfloat16";
    case at::kInt: return "torch.int32";
    case at::kLong: return "torch.int64";
    default: return c10::toString(t);
  }
}

// --- arguments --------------------------------------------------------------------------------
const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) refuse(PyExc_TypeError, std::string(name) + " must be a tensor, got " + Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}
const at::Tensor* maybe_tensor(PyObject* o, const char* name) { return o == Py_None ? nullptr : &tensor(o, name); }
int64_t integer(PyObject* o, const char* name) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse(PyExc_TypeError, std::string(name) + " must be an integer of at most 64 bits");
  }
  return v;
}
double number(PyObject* o, const char* name) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse(PyExc_TypeError, std::string(name) + " must be a number");
  }
  return v;
}
int int32(int64_t v, const char* name) {
  if (v > INT32_MAX || v < INT32_MIN) refuse(PyExc_ValueError, std::string(name) + " does not fit 32 bits: " + std::to_string(v));
  return (int)v;
}

// The stride of a dimension; of one with a single entry it says nothing and may be anything.
int64_t step(const at::Tensor& t, int64_t dim) { return t.size(dim) > 1 ? t.stride(dim) : 0; }

// A tensor that is written has a place of its own for every entry (expanded dimensions do not).
void own_places(const at::Tensor& t, const char* name) {
  for (int64_t d = 0; d < t.dim(); ++d)
    if (t.size(d) > 1 && t.stride(d) == 0) refuse(PyExc_ValueError, std::string(name) + " is written and must not be an expanded tensor, got strides " + shape_text(t.strides()));
}

// --- shared memory ----------------------------------------------------------------------------
// The rows (last dimension) of a tensor of 3 or 4 dimensions.
b200moe::StridedRows rows_of(const at::Tensor& t) {
  b200moe::StridedRows r;
  const int64_t e = (int64_t)t.element_size(), last = t.dim() - 1;
  r.base = (uintptr_t)t.data_ptr();
  r.width = t.size(last) * e;
  for (int64_t d = 0; d < last; ++d) r.axis(t.size(d), t.stride(d) * e);
  return r;
}
// A kernel reads some rows after it has written others: what is written may not partly cover what is read.
void apart(const b200moe::StridedRows& out, const char* out_name, const at::Tensor& t, const char* name, bool may_be_same) {
  const b200moe::StridedRows r = rows_of(t);
  if (may_be_same && out.same(r)) return;
  if (b200moe::rows_meet(out, r))
    refuse(PyExc_ValueError, std::string(out_name) + " shares memory with " + name + (may_be_same ? "; it may be the same tensor or a separate one, nothing between" : ""));
}

// --- checks -----------------------------------------------------------------------------------
int dtype_tag(const at::Tensor& t, const char* name) {
  int tag = -1;
  switch (t.scalar_type()) {
    case at::kFloat: tag = B200MOE_F32; break;
    case at::kHalf: tag = B200MOE_F16; break;
    case at::kBFloat16: tag = B200MOE_BF16; break;
    default: refuse(PyExc_TypeError, std::string("unsupported dtype ") + type_text(t.scalar_type()) + " of " + name + "; float32, float16 or bfloat16");
  }
  if (!t.is_cuda()) refuse(PyExc_ValueError, std::string(name) + " must live on a CUDA device, got " + t.device().str() + " (this package has no CPU path)");
  return tag;
}
void need(const at::Tensor& t, const char* name, c10::Device dev, at::ScalarType dtype, int64_t dims) {
  if (t.device() != dev)
    refuse(PyExc_ValueError, std::string(name) + " must live on " + dev.str() + ", got " + t.device().str() + " (this package has no CPU path)");
  if (t.scalar_type() != dtype) refuse(PyExc_TypeError, std::string(name) + " must be " + type_text(dtype) + ", got " + type_text(t.scalar_type()));
  if (t.dim() != dims) refuse(PyExc_ValueError, std::string(name) + " must have " + std::to_string(dims) + " dimensions, got " + shape_text(t.sizes()));
}
// a vector of the given length without gaps
void* vec(const at::Tensor& t, const char* name, c10::Device dev, at::ScalarType dtype, int64_t length) {
  need(t, name, dev, dtype, 1);
  if (t.size(0) != length || (length > 1 && t.stride(0) != 1))
    refuse(PyExc_ValueError, std::string(name) + " must be contiguous of length " + std::to_string(length) + ", got " + shape_text(t.sizes()));
  return t.data_ptr();
}
// an index vector, int64 or int32
void* index(const at::Tensor& t, const char* name, c10::Device dev, int64_t length, int32_t* is64) {
  const at::ScalarType s = t.scalar_type();
  if (s != at::kLong && s != at::kInt) refuse(PyExc_TypeError, std::string(name) + " must be int64 or int32, got " + type_text(s));
  *is64 = s == at::kLong;
  return vec(t, name, dev, s, length);
}
int32_t* status_ptr(PyObject* o, c10::Device dev) {
  const at::Tensor* t = maybe_tensor(o, "status");
  if (!t) return nullptr;
  if (t->device() != dev || t->scalar_type() != at::kInt || t->numel() != 1)
    refuse(PyExc_ValueError, "status must be an int32 tensor of one element on " + dev.str());
  return (int32_t*)t->data_ptr();
}
void heads_contiguous(const at::Tensor& t, const char* name) {
  if (t.stride(2) != 1 && t.size(2) > 1) refuse(PyExc_ValueError, std::string("heads must be contiguous, but ") + name + " has strides " + shape_text(t.strides()));
}
void cache_pair(const at::Tensor& k, const at::Tensor& v, c10::Device dev, at::ScalarType dtype, int64_t head_dim) {
  need(k, "k_cache", dev, dtype, 4);
  need(v, "v_cache", dev, dtype, 4);
  if (k.sizes() != v.sizes() || step(k, 0) != step(v, 0) || step(k, 1) != step(v, 1) || step(k, 2) != step(v, 2) || k.stride(3) != v.stride(3))
    refuse(PyExc_ValueError, "k_cache and v_cache must have the same shape and strides");
  if (k.size(3) != head_dim || k.stride(3) != 1)
    refuse(PyExc_ValueError, "the caches must be [blocks, block_size, kv_heads, " + std::to_string(head_dim) + "] with contiguous heads, got " + shape_text(k.sizes()));
  if (k.size(1) == 0) refuse(PyExc_ValueError, "the caches need a block size of at least one slot");
}
// torch.empty without the way through the dispatcher
at::Tensor empty(c10::Device dev, at::ScalarType dtype, at::IntArrayRef shape) { return at::detail::empty_cuda(shape, dtype, dev, std::nullopt); }
at::Tensor output(PyObject* o, c10::Device dev, at::ScalarType dtype, at::IntArrayRef shape) {
  if (o == Py_None) return empty(dev, dtype, shape);
  const at::Tensor& t = tensor(o, "out");
  need(t, "out", dev, dtype, 3);
  if (t.sizes() != shape || (t.stride(2) != 1 && shape[2] > 1))
    refuse(PyExc_ValueError, "out must be " + shape_text(shape) + " with contiguous heads, got " + shape_text(t.sizes()));
  own_places(t, "out");
  return t;
}

// --- calls ------------------------------------------------------------------------------------
PyObject* g_error = nullptr;         // on_device_sd_b200._lib.B200MoEError

struct Failure { int code; };
void check(int code) {
  if (code != B200MOE_OK) throw Failure{code};
}
template <typename F> PyObject* guarded(F&& f) {
  try {
    return f();
  } catch (const Refusal& r) {
    PyErr_SetString(r.type, r.text.c_str());
  } catch (const Failure& e) {
    PyObject* args = Py_BuildValue("(is)", e.code, b200moe_last_error(nullptr));
    if (args) {
      PyObject* exc = PyObject_CallObject(g_error, args);
      Py_DECREF(args);
      if (exc) {
        PyErr_SetObject(g_error, exc);
        Py_DECREF(exc);
      }
    }
  } catch (const std::exception& e) {   // torch's allocator among others
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}
bool arity(Py_ssize_t n, Py_ssize_t want) {
  if (n == want) return true;
  PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, n);
  return false;
}

// (query | None, key, value, positions | None, cos_sin | None, k_cache, v_cache, slot_mapping, q_norm_weight | None,
//  k_norm_weight | None, eps, out | None, status | None) -> out | None
PyObject* store_kv(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arity(n, 13)) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor &key = tensor(a[1], "key"), &value = tensor(a[2], "value"), &kc = tensor(a[5], "k_cache"), &vc = tensor(a[6], "v_cache");
    const at::Tensor *query = maybe_tensor(a[0], "query"), *table = maybe_tensor(a[4], "cos_sin");
    b200moe_store_kv_args s = {};
    s.dtype = dtype_tag(key, "key");
    const c10::Device dev = key.device();
    const at::ScalarType dt = key.scalar_type();
    need(key, "key", dev, dt, 3);
    need(value, "value", dev, dt, 3);
    if (key.sizes() != value.sizes())
      refuse(PyExc_ValueError, "key and value must have the same shape, got " + shape_text(key.sizes()) + " and " + shape_text(value.sizes()));
    const int64_t T = key.size(0), hk = key.size(1), D = key.size(2);
    cache_pair(kc, vc, dev, dt, D);
    if (kc.size(2) != hk) refuse(PyExc_ValueError, "the caches hold " + std::to_string(kc.size(2)) + " key-value heads, key and value " + std::to_string(hk));
    own_places(kc, "k_cache");
    own_places(vc, "v_cache");
    apart(rows_of(kc), "k_cache", vc, "v_cache", false);
    heads_contiguous(key, "key");
    heads_contiguous(value, "value");
    s.slots = index(tensor(a[7], "slot_mapping"), "slot_mapping", dev, T, &s.slots_are_int64);
    s.key = key.data_ptr(); s.value = value.data_ptr(); s.k_cache = kc.data_ptr(); s.v_cache = vc.data_ptr();
    s.k_token_stride = step(key, 0); s.k_head_stride = step(key, 1); s.v_token_stride = step(value, 0); s.v_head_stride = step(value, 1);
    s.cache_block_stride = step(kc, 0); s.cache_slot_stride = step(kc, 1); s.cache_head_stride = step(kc, 2);
    s.num_tokens = int32(T, "the number of tokens"); s.num_kv_heads = int32(hk, "kv_heads"); s.head_dim = int32(D, "head_dim");
    s.num_blocks = int32(kc.size(0), "the number of blocks"); s.block_size = int32(kc.size(1), "the block size");
    at::Tensor out;
    if (query) {
      need(*query, "query", dev, dt, 3);
      if (query->size(0) != T || query->size(2) != D)
        refuse(PyExc_ValueError, "query must be [" + std::to_string(T) + ", heads, " + std::to_string(D) + "], got " + shape_text(query->sizes()));
      heads_contiguous(*query, "query");
      out = output(a[11], dev, dt, query->sizes());
      if (a[11] != Py_None) {
        const b200moe::StridedRows o = rows_of(out);
        apart(o, "out", *query, "query", true);
        apart(o, "out", key, "key", false);
        apart(o, "out", value, "value", false);
        apart(o, "out", kc, "k_cache", false);
        apart(o, "out", vc, "v_cache", false);
      }
      s.query = query->data_ptr(); s.query_out = out.data_ptr(); s.num_heads = int32(query->size(1), "heads");
      s.q_token_stride = step(*query, 0); s.q_head_stride = step(*query, 1); s.o_token_stride = step(out, 0); s.o_head_stride = step(out, 1);
    }
    if (table) {
      need(*table, "cos_sin", dev, at::kFloat, 2);
      if (table->size(1) != D || !table->is_contiguous())
        refuse(PyExc_ValueError, "cos_sin must be a contiguous [positions, " + std::to_string(D) + "], got " + shape_text(table->sizes()));
      s.positions = index(tensor(a[3], "positions"), "positions", dev, T, &s.positions_are_int64);
      s.cos_sin = (const float*)table->data_ptr(); s.max_position = int32(table->size(0), "the number of positions");
    }
    if (const at::Tensor* w = maybe_tensor(a[8], "q_norm_weight")) s.q_norm_weight = vec(*w, "q_norm_weight", dev, dt, D);
    if (const at::Tensor* w = maybe_tensor(a[9], "k_norm_weight")) s.k_norm_weight = vec(*w, "k_norm_weight", dev, dt, D);
    s.eps = (float)number(a[10], "eps");
    s.status = status_ptr(a[12], dev);
    const c10::cuda::CUDAGuard guard(dev);
    check(b200moe_store_kv(&s, c10::cuda::getCurrentCUDAStream(dev.index()).stream()));
    if (!query) Py_RETURN_NONE;
    return a[11] == Py_None ? THPVariable_Wrap(std::move(out)) : Py_NewRef(a[11]);
  });
}

// (query, k_cache, v_cache, block_tables, context_lens, query_start | None, max_query_len | None, scale | None, out | None,
//  return_lse, status | None) -> out | (out, lse)
PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arity(n, 11)) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor &query = tensor(a[0], "query"), &kc = tensor(a[1], "k_cache"), &vc = tensor(a[2], "v_cache");
    const at::Tensor &tables = tensor(a[3], "block_tables"), &lens = tensor(a[4], "context_lens");
    b200moe_paged_attention_args s = {};
    s.dtype = dtype_tag(query, "query");
    const c10::Device dev = query.device();
    const at::ScalarType dt = query.scalar_type();
    need(query, "query", dev, dt, 3);
    const int64_t T = query.size(0), hq = query.size(1), D = query.size(2);
    cache_pair(kc, vc, dev, dt, D);
    heads_contiguous(query, "query");
    need(tables, "block_tables", dev, at::kInt, 2);
    const int64_t B = tables.size(0), width = tables.size(1);
    if (width > 1 && tables.stride(1) != 1) refuse(PyExc_ValueError, "the rows of block_tables must be contiguous");
    s.context_lens = (const int32_t*)vec(lens, "context_lens", dev, at::kInt, B);
    int64_t span = 1;
    if (const at::Tensor* start = maybe_tensor(a[5], "query_start")) {
      s.query_start = (const int32_t*)vec(*start, "query_start", dev, at::kInt, B + 1);
      span = a[6] == Py_None ? T : integer(a[6], "max_query_len");
      if (span < 0) refuse(PyExc_ValueError, "max_query_len must not be negative");
      if (span > T) span = T;
    } else if (T != B) {
      refuse(PyExc_ValueError, "without query_start there is one token per sequence, got " + std::to_string(T) + " tokens for " + std::to_string(B) + " sequences");
    }
    const double scale = a[7] == Py_None ? 1.0 / std::sqrt((double)D) : number(a[7], "scale");
    const int with_lse = PyObject_IsTrue(a[9]);
    if (with_lse < 0) return nullptr;
    s.status = status_ptr(a[10], dev);
    s.query = query.data_ptr(); s.k_cache = kc.data_ptr(); s.v_cache = vc.data_ptr(); s.block_tables = (const int32_t*)tables.data_ptr();
    s.q_token_stride = step(query, 0); s.q_head_stride = step(query, 1);
    s.cache_block_stride = step(kc, 0); s.cache_slot_stride = step(kc, 1); s.cache_head_stride = step(kc, 2); s.block_table_stride = step(tables, 0);
    s.num_tokens = int32(T, "the number of tokens"); s.num_seqs = int32(B, "the number of sequences");
    s.num_heads = int32(hq, "heads"); s.num_kv_heads = int32(kc.size(2), "kv_heads"); s.head_dim = int32(D, "head_dim");
    s.num_blocks = int32(kc.size(0), "the number of blocks"); s.block_size = int32(kc.size(1), "the block size");
    s.max_blocks_per_seq = int32(width, "the width of block_tables"); s.max_query_len = (int32_t)span;
    s.scale = (float)scale;
    const c10::cuda::CUDAGuard guard(dev);
    at::Tensor out = output(a[8], dev, dt, query.sizes()), lse, ws;
    if (a[8] != Py_None) {
      const b200moe::StridedRows o = rows_of(out);
      apart(o, "out", query, "query", true);
      apart(o, "out", kc, "k_cache", false);
      apart(o, "out", vc, "v_cache", false);
    }
    s.out = out.data_ptr(); s.o_token_stride = step(out, 0); s.o_head_stride = step(out, 1);
    if (with_lse) {
      lse = empty(dev, at::kFloat, {T, hq});
      s.lse_out = (float*)lse.data_ptr();
    }
    // the workspace belongs to this call: calls on several streams and captured graphs do not share one
    if (T > 0 && B > 0)
      check(b200moe_paged_attention_workspace(s.dtype, s.num_seqs, s.num_heads, s.num_kv_heads, s.head_dim, s.max_query_len, s.max_blocks_per_seq,
                                              s.block_size, &s.workspace_bytes));
    if (s.workspace_bytes) {
      ws = empty(dev, at::kByte, {s.workspace_bytes});
      s.workspace = ws.data_ptr();
    }
    check(b200moe_paged_attention(&s, c10::cuda::getCurrentCUDAStream(dev.index()).stream()));
    PyObject* o = a[8] == Py_None ? THPVariable_Wrap(std::move(out)) : Py_NewRef(a[8]);
    if (!o || !with_lse) return o;
    PyObject* l = THPVariable_Wrap(std::move(lse));
    PyObject* pair = l ? PyTuple_Pack(2, o, l) : nullptr;
    Py_DECREF(o);
    Py_XDECREF(l);
    return pair;
  });
}

// (draft_tokens, target_probs, draft_probs | None, accept_uniform, sample_uniform, draft_start, max_draft_len, status | None)
// -> (tokens, accepted)
PyObject* verify(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arity(n, 8)) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor &tokens = tensor(a[0], "draft_tokens"), &target = tensor(a[1], "target_probs");
    const at::Tensor &accept = tensor(a[3], "accept_uniform"), &sample = tensor(a[4], "sample_uniform"), &start = tensor(a[5], "draft_start");
    const at::Tensor* draft = maybe_tensor(a[2], "draft_probs");
    b200moe_verify_draft_args s = {};
    s.dtype = dtype_tag(target, "target_probs");
    const c10::Device dev = target.device();
    const at::ScalarType dt = target.scalar_type();
    need(target, "target_probs", dev, dt, 2);
    need(tokens, "draft_tokens", dev, at::kLong, 1);
    need(sample, "sample_uniform", dev, at::kFloat, 1);
    const int64_t drafts = tokens.size(0), B = sample.size(0), vocab = target.size(1), longest = integer(a[6], "max_draft_len");
    if (longest < 0) refuse(PyExc_ValueError, "max_draft_len must not be negative");
    if (vocab == 0) refuse(PyExc_ValueError, "the vocabulary is empty");
    if (target.size(0) < B)   // the drafts' own rows depend on draft_start, which the kernel reads: drafts behind its end need none
      refuse(PyExc_ValueError, "target_probs must have a row for every draft and one more per sequence, got " + std::to_string(target.size(0)) + " rows for " + std::to_string(B) + " sequences");
    s.draft_tokens = (const int64_t*)vec(tokens, "draft_tokens", dev, at::kLong, drafts);
    s.sample_uniform = (const float*)vec(sample, "sample_uniform", dev, at::kFloat, B);
    s.accept_uniform = (const float*)vec(accept, "accept_uniform", dev, at::kFloat, drafts);
    s.draft_start = (const int32_t*)vec(start, "draft_start", dev, at::kInt, B + 1);
    if (target.stride(1) != 1 && vocab > 1) refuse(PyExc_ValueError, "the rows of target_probs must be contiguous");
    if (draft) {
      need(*draft, "draft_probs", dev, dt, 2);
      if (draft->size(0) != drafts || draft->size(1) != vocab || (draft->stride(1) != 1 && vocab > 1))
        refuse(PyExc_ValueError, "draft_probs must be [" + std::to_string(drafts) + ", " + std::to_string(vocab) + "] with contiguous rows, got " + shape_text(draft->sizes()));
      // without drafts there is no row to point at, but the rule is the sampled one all the same
      s.draft_probs = draft->data_ptr() ? draft->data_ptr() : target.data_ptr();
      s.draft_stride = draft->stride(0);
    }
    s.status = status_ptr(a[7], dev);
    s.target_probs = target.data_ptr(); s.target_stride = target.stride(0);
    s.num_seqs = int32(B, "the number of sequences"); s.vocab_size = int32(vocab, "the vocabulary"); s.max_draft_len = int32(longest, "max_draft_len");
    s.num_draft_tokens = int32(drafts, "the number of drafts"); s.num_target_rows = int32(target.size(0), "the number of target rows");
    const c10::cuda::CUDAGuard guard(dev);
    at::Tensor out = empty(dev, at::kLong, {B, longest + 1});
    at::Tensor count = empty(dev, at::kInt, {B});
    s.tokens_out = (int64_t*)out.data_ptr(); s.accepted_out = (int32_t*)count.data_ptr();
    check(b200moe_verify_draft(&s, c10::cuda::getCurrentCUDAStream(dev.index()).stream()));
    PyObject *o = THPVariable_Wrap(std::move(out)), *c = THPVariable_Wrap(std::move(count));
    PyObject* pair = o && c ? PyTuple_Pack(2, o, c) : nullptr;
    Py_XDECREF(o);
    Py_XDECREF(c);
    return pair;
  });
}

PyMethodDef kMethods[] = {
    {"store_kv", (PyCFunction)(void (*)(void))store_kv, METH_FASTCALL, "b200moe_store_kv on tensors"},
    {"paged_attention", (PyCFunction)(void (*)(void))attention, METH_FASTCALL, "b200moe_paged_attention on tensors"},
    {"verify_draft", (PyCFunction)(void (*)(void))verify, METH_FASTCALL, "b200moe_verify_draft on tensors"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_step", "tensor entry points of the step operators", -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__step(void) {
  PyObject* lib = PyImport_ImportModule("on_device_sd_b200._lib");
  if (!lib) return nullptr;
  g_error = PyObject_GetAttrString(lib, "B200MoEError");
  Py_DECREF(lib);
  if (!g_error) return nullptr;
  return PyModule_Create(&kModule);
}
