// The host side of the drafted-step operators (tilejax_b200/ops.py: rpa_plan, qk_norm_rope, rpa_norm_rope_write,
// rpa_tree_attention, rpa_commit) as a CPython module: arguments checked, outputs and scratch allocated, the C ABI called
// on the tensors' device and its current stream. Their kernels take 3 to 11 us on a small step, and checking the arguments
// from Python, a query at a time, and passing them through ctypes took 11 to 18.
//
// The library's entry points come as addresses (`bind`), from the library that _lib.py has loaded; a negative return
// code goes back to _lib.check. Arguments come in ops.py's order, all of them, None where there is none.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <string>
#include <vector>

#include "../../include/tilejax_b200.h"

namespace {

decltype(&tjx_rpa_plan) plan_fn = nullptr;
decltype(&tjx_norm_rope_bf16) norm_rope_fn = nullptr;
decltype(&tjx_rpa_tree_attention_workspace_bytes) tree_bytes_fn = nullptr;
decltype(&tjx_rpa_tree_attention_bf16) tree_fn = nullptr;
decltype(&tjx_rpa_commit_bf16) commit_fn = nullptr;
PyObject* check_fn = nullptr;  // _lib.check

struct BadValue {  // becomes a Python ValueError
  std::string text;
};
struct PythonError {};  // one is set already
void require(bool fine, const char* text) {
  if (!fine) throw BadValue{text};
}

// The call's arguments by position.
struct Args {
  PyObject* const* at;
  Args(PyObject* const* args, Py_ssize_t n, Py_ssize_t want) : at(args) {
    if (n != want) throw BadValue{"wrong number of arguments"};
  }
  const at::Tensor& tensor(int i, const char* name) const {
    if (!THPVariable_Check(at[i])) {
      PyErr_Format(PyExc_TypeError, "%s must be a tensor", name);
      throw PythonError{};
    }
    return THPVariable_Unpack(at[i]);
  }
  bool none(int i) const { return at[i] == Py_None; }
  const at::Tensor* optional(int i, const char* name) const { return none(i) ? nullptr : &tensor(i, name); }
  long long integer(int i) const {
    const long long v = PyLong_AsLongLong(at[i]);
    if (v == -1 && PyErr_Occurred()) throw PythonError{};
    return v;
  }
  double number(int i) const {
    const double v = PyFloat_AsDouble(at[i]);
    if (v == -1.0 && PyErr_Occurred()) throw PythonError{};
    return v;
  }
  bool truth(int i) const {
    const int v = PyObject_IsTrue(at[i]);
    if (v < 0) throw PythonError{};
    return v != 0;
  }
};

int to_int(long long v) {  // (sizes past an int are past what the library takes)
  require(v >= -2147483647ll && v <= 2147483647ll, "a size does not fit in int32");
  return static_cast<int>(v);
}

// All tensors on one CUDA device and dense; the device.
class Device {
 public:
  void add(const at::Tensor& t) {
    place(t);
    require(t.is_contiguous(), "tensors must be contiguous (row-major)");
  }
  void place(const at::Tensor& t) {  // any strides
    require(t.is_cuda(), "tilejax_b200 operators take CUDA tensors (there is no CPU path)");
    if (!seen_) seen_ = true, device_ = t.device();
    require(t.device() == device_, "all tensors must be on the same device");
  }
  c10::Device get() const { return device_; }

 private:
  bool seen_ = false;
  c10::Device device_{c10::kCUDA, 0};
};

const int32_t* ints(const at::Tensor& t) { return static_cast<const int32_t*>(t.data_ptr()); }
int32_t* ints_out(const at::Tensor& t) { return static_cast<int32_t*>(t.data_ptr()); }
uintptr_t address(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()); }
bool is_vector(const at::Tensor& t) { return t.scalar_type() == at::kInt && t.dim() == 1; }
bool is_vector(const at::Tensor& t, int64_t n) { return is_vector(t) && t.size(0) == n; }

uintptr_t end_of(const at::Tensor& t) {  // the address behind the last element
  int64_t last = 1;
  for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
  return address(t) + last * t.element_size();
}
bool overlap(const at::Tensor& a, const at::Tensor& b) {  // from the first to the last element
  return a.numel() > 0 && b.numel() > 0 && address(a) < end_of(b) && address(b) < end_of(a);
}
bool same(const at::Tensor& a, const at::Tensor& b) {
  return address(a) == address(b) && a.sizes() == b.sizes() && a.strides() == b.strides();
}

at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, c10::Device device) {
  return at::empty(sizes, at::TensorOptions().dtype(type).device(device));
}

tjx_stream_t stream_of(c10::Device device) { return c10::cuda::getCurrentCUDAStream(device.index()).stream(); }

void check(int code) {
  if (code == 0) return;
  PyObject* r = PyObject_CallFunction(check_fn, "i", code);
  Py_XDECREF(r);
  if (r != nullptr) PyErr_SetString(PyExc_RuntimeError, "the library reported an error that _lib.check passed");
  throw PythonError{};
}

// The sizes of a ragged paged cache and its tables.
struct Cache {
  int pages, page_size, kv_heads, D, seqs, pages_per_seq;
  Cache(const at::Tensor& kv_cache, const at::Tensor& kv_lens, const at::Tensor& page_indices) {
    require(kv_cache.dim() == 5 && kv_cache.size(3) == 2 && kv_cache.scalar_type() == at::kBFloat16,
            "the cache is (pages, page_size, Hkv, 2, D) bfloat16: each head's key and value side by side");
    pages = to_int(kv_cache.size(0)), page_size = to_int(kv_cache.size(1)), kv_heads = to_int(kv_cache.size(2));
    D = to_int(kv_cache.size(4));
    require(kv_lens.scalar_type() == at::kInt && page_indices.scalar_type() == at::kInt, "kv_lens and page_indices must be int32");
    require(kv_lens.dim() == 1 && kv_lens.size(0) > 0 && page_indices.dim() == 1 && page_indices.size(0) % kv_lens.size(0) == 0,
            "page_indices is (S * pages_per_seq,), sequence s's pages at s * pages_per_seq");
    seqs = to_int(kv_lens.size(0)), pages_per_seq = to_int(page_indices.size(0) / seqs);
  }
};

// ------------------------------------------------------------------------------------------ rpa_plan

PyObject* plan(Args a) {
  const at::Tensor* in[7];
  static const char* names[7] = {"ctx_lens", "q_lens", "page_indices", "free_pages", "n_free", "pages_held", "depths"};
  for (int i = 0; i < 5; ++i) {
    in[i] = &a.tensor(i, names[i]);
    if (!is_vector(*in[i])) throw BadValue{std::string(names[i]) + " must be an int32 vector"};
  }
  const long long page_size = a.integer(5), T = a.integer(6);
  in[5] = a.optional(7, names[5]), in[6] = a.optional(8, names[6]);
  const int64_t S = in[0]->size(0), entries = in[2]->size(0);
  require(S > 0 && in[1]->size(0) == S && entries > 0 && entries % S == 0,
          "ctx_lens and q_lens are (S,), page_indices (S * pages_per_seq,)");
  require(in[4]->size(0) >= 1, "n_free holds the number of free pages");
  require(in[5] == nullptr || is_vector(*in[5], S), "pages_held is int32 (S,)");
  require(T >= 0 && page_size > 0, "page_size must be positive and tokens not negative");
  require(in[6] == nullptr || is_vector(*in[6], T), "depths is int32 (tokens,)");
  Device device;
  for (const at::Tensor* t : in)
    if (t != nullptr) device.add(*t);
  for (const at::Tensor* t : in) require(t == nullptr || t == in[2] || !overlap(*t, *in[2]), "page_indices overlaps another input");
  const int64_t sizes[6] = {S, S + 1, T, T, S, 2};
  at::Tensor out[6];
  if (a.none(9)) {
    at::Tensor block = fresh({3 * S + 3 + 2 * T}, at::kInt, device.get());
    int64_t at = 0;
    for (int i = 0; i < 6; at += sizes[i++]) {  // pieces of one allocation, one behind the other
      out[i] = at::detail::make_tensor<at::TensorImpl>(c10::Storage(block.storage()), block.key_set(), block.dtype());
      out[i].unsafeGetTensorImpl()->set_storage_offset(at);
      out[i].unsafeGetTensorImpl()->set_sizes_contiguous({sizes[i]});
    }
  } else {
    require(PyTuple_Check(a.at[9]) && PyTuple_GET_SIZE(a.at[9]) == 6, "out is a step");
    for (int i = 0; i < 6; ++i) {
      PyObject* o = PyTuple_GET_ITEM(a.at[9], i);
      require(THPVariable_Check(o), "out is a step of tensors");
      out[i] = THPVariable_Unpack(o);
      require(is_vector(out[i], sizes[i]), "out is a step of other sizes");
      device.add(out[i]);
      for (const at::Tensor* t : in) require(t == nullptr || !overlap(out[i], *t), "out overlaps an input");
      for (int j = 0; j < i; ++j) require(!overlap(out[i], out[j]), "out's tensors overlap");
    }
  }
  {
    const c10::cuda::CUDAGuard guard(device.get());
    check(plan_fn(ints(*in[0]), ints(*in[1]), in[5] ? ints(*in[5]) : nullptr, in[6] ? ints(*in[6]) : nullptr, ints_out(*in[2]),
                  ints(*in[3]), ints(*in[4]), to_int(in[3]->size(0)), to_int(S), to_int(T), to_int(entries / S), to_int(page_size),
                  ints_out(out[0]), ints_out(out[1]), ints_out(out[2]), ints_out(out[3]), ints_out(out[4]), ints_out(out[5]),
                  stream_of(device.get())));
  }
  PyObject* result = PyTuple_New(6);
  if (result == nullptr) throw PythonError{};
  for (int i = 0; i < 6; ++i) PyTuple_SET_ITEM(result, i, THPVariable_Wrap(out[i]));
  return result;
}

// ------------------------------------------------------------------------------------------ norm, rotation, write

// A (tokens, heads, D) operand of any token and head strides.
struct Heads {
  int64_t heads, token, head;
  Heads(const char* name, const at::Tensor& t, int64_t tokens, int64_t D) {
    if (t.dim() != 3 || t.scalar_type() != at::kBFloat16 || t.size(0) != tokens || t.size(2) != D)
      throw BadValue{std::string(name) + " must be bfloat16 (" + std::to_string(tokens) + ", heads, " + std::to_string(D) + ")"};
    heads = t.size(1), token = t.stride(0), head = t.stride(1);
    if (t.stride(2) != 1 || token % 4 != 0 || head % 4 != 0 || address(t) % 8 != 0)
      throw BadValue{std::string(name) + "'s last dimension must be dense, its strides multiples of 4 elements, its data 8-byte aligned"};
  }
};
// No two elements of an output in one place.
bool distinct(const at::Tensor& t) {
  const int64_t tokens = t.size(0), heads = t.size(1), D = t.size(2), token = t.stride(0), head = t.stride(1);
  auto nested = [D](int64_t n, int64_t inner, int64_t m, int64_t outer) {
    return (n <= 1 || inner >= D) && (m <= 1 || outer >= (n - 1) * inner + D);
  };
  return t.numel() == 0 || nested(heads, head, tokens, token) || nested(tokens, token, heads, head);
}
// Two operands without an element in common: apart, or views of one projection's output that share its token stride (side
// by side within a token, or head by head).
bool apart(const at::Tensor& a, const at::Tensor& b) {
  if (!overlap(a, b)) return true;
  if (a.stride(0) != b.stride(0) || a.stride(0) <= 0) return false;
  const int64_t difference = (static_cast<int64_t>(address(b)) - static_cast<int64_t>(address(a))) / 2;
  auto side_by_side = [&](int64_t period, int64_t span_a, int64_t span_b) {
    const int64_t d = (difference % period + period) % period;
    return d >= span_a && d + span_b <= period;
  };
  const int64_t token = a.stride(0), head = a.stride(1), D = a.size(2);
  if (side_by_side(token, (a.size(1) - 1) * head + D, (b.size(1) - 1) * b.stride(1) + D)) return true;
  return head > 0 && b.stride(1) == head && token % head == 0 && side_by_side(head, D, D);
}

// (q, k, v, q_gamma, k_gamma, positions, cos_sin, kv_cache, slots, eps, interleaved, q_out, k_out) -> (q_out, k_out); v,
// kv_cache and slots go together.
PyObject* norm_rope(Args a) {
  const at::Tensor &q = a.tensor(0, "q"), &k = a.tensor(1, "k"), &positions = a.tensor(5, "positions"), &cos_sin = a.tensor(6, "cos_sin");
  const at::Tensor *v = a.optional(2, "v"), *q_gamma = a.optional(3, "q_gamma"), *k_gamma = a.optional(4, "k_gamma");
  const at::Tensor *cache = a.optional(7, "kv_cache"), *slots = a.optional(8, "slots");
  require(q.dim() == 3, "q is (T, H, D)");
  const int64_t T = q.size(0), H = q.size(1), D = q.size(2);
  if (cache != nullptr) {
    require(cache->dim() == 5 && cache->size(3) == 2 && cache->scalar_type() == at::kBFloat16 && cache->numel() > 0,
            "the cache is (pages, page_size, Hkv, 2, D) bfloat16: each head's key and value side by side");
    require(v != nullptr && k.sizes() == at::IntArrayRef({T, cache->size(2), cache->size(4)}) && v->sizes() == k.sizes(),
            "q is (T, H, D), k and v (T, Hkv, D) with the cache's Hkv and D");
    require(cache->size(0) * cache->size(1) < (1ll << 31), "the cache's rows must fit in int32");
    require(slots != nullptr && is_vector(*slots, T), "slots is int32 (T,)");
  }
  const Heads hq("q", q, T, D), hk("k", k, T, D);
  require((q_gamma == nullptr) == (k_gamma == nullptr), "q_gamma and k_gamma are given together or not at all");
  for (const at::Tensor* g : {q_gamma, k_gamma})
    if (g != nullptr && (g->dim() != 1 || g->size(0) != D || g->scalar_type() != at::kBFloat16 || address(*g) % 8 != 0))
      throw BadValue{"the gammas are bfloat16 (" + std::to_string(D) + ",), 8-byte aligned"};
  require(is_vector(positions, T), "positions is int32 (T,)");
  require(cos_sin.dim() == 2 && cos_sin.scalar_type() == at::kFloat && cos_sin.size(1) <= D && cos_sin.size(1) % 8 == 0 &&
              cos_sin.size(0) > 0 && address(cos_sin) % 16 == 0,
          "cos_sin is float32 (max_positions, rot), rot a multiple of 8 up to the head dimension, 16-byte aligned");
  // Every warp reads these while others write. (q, k and v, which a row's own warp reads, below.)
  for (const at::Tensor* written : {a.optional(11, "out"), cache == nullptr ? a.optional(12, "out") : cache})
    for (const at::Tensor* read : {q_gamma, k_gamma, &positions, &cos_sin, slots})
      require(written == nullptr || read == nullptr || !overlap(*written, *read),
              "an output, or the cache, overlaps the gammas, positions, cos_sin or slots");
  int64_t strides[10] = {hq.token, hq.head, hk.token, hk.head, 0, 0, 0, 0, 0, 0};
  Device device;
  device.add(positions), device.add(cos_sin), device.place(q), device.place(k);
  for (const at::Tensor* g : {q_gamma, k_gamma})
    if (g != nullptr) device.add(*g);
  if (cache != nullptr) {
    const Heads hv("v", *v, T, D);
    strides[4] = hv.token, strides[5] = hv.head;
    device.place(*v), device.add(*slots), device.add(*cache);
  }
  at::Tensor q_out, k_out;
  if (a.none(11)) {
    q_out = fresh({T, H, D}, at::kBFloat16, device.get());
  } else {
    q_out = a.tensor(11, "out");
    const Heads ho("the queries' output", q_out, T, D);
    require(ho.heads == H && q_out.device() == device.get() && (same(q_out, q) || apart(q_out, q)) && apart(q_out, k) &&
                (v == nullptr || apart(q_out, *v)) && distinct(q_out),
            "the queries' output is q itself or memory of its own, like q");
  }
  strides[6] = q_out.stride(0), strides[7] = q_out.stride(1);
  if (cache != nullptr) {
    require(!overlap(*cache, q) && !overlap(*cache, k) && !overlap(*cache, *v) && !overlap(*cache, q_out), "the cache overlaps an operand");
  } else {
    if (a.none(12)) {
      k_out = fresh({T, hk.heads, D}, at::kBFloat16, device.get());
    } else {
      k_out = a.tensor(12, "out");
      const Heads ho("the keys' output", k_out, T, D);
      require(ho.heads == hk.heads && k_out.device() == device.get() && (same(k_out, k) || apart(k_out, k)) &&
                  apart(k_out, q) && apart(k_out, q_out) && distinct(k_out),
              "the keys' output is k itself or memory of its own, like k");
    }
    strides[8] = k_out.stride(0), strides[9] = k_out.stride(1);
  }
  if (T > 0) {
    const c10::cuda::CUDAGuard guard(device.get());
    check(norm_rope_fn(q.data_ptr(), k.data_ptr(), v ? v->data_ptr() : nullptr, strides, q_gamma ? q_gamma->data_ptr() : nullptr,
                       k_gamma ? k_gamma->data_ptr() : nullptr, ints(positions), static_cast<const float*>(cos_sin.data_ptr()),
                       slots ? ints(*slots) : nullptr, q_out.data_ptr(), cache ? nullptr : k_out.data_ptr(),
                       cache ? cache->data_ptr() : nullptr, to_int(T), to_int(H), to_int(hk.heads), to_int(D),
                       to_int(cos_sin.size(1)), to_int(cos_sin.size(0)), a.truth(10) ? 1 : 0,
                       cache ? to_int(cache->size(0) * cache->size(1)) : 0, static_cast<float>(a.number(9)), stream_of(device.get())));
  }
  PyObject* result = PyTuple_New(2);
  if (result == nullptr) throw PythonError{};
  PyTuple_SET_ITEM(result, 0, THPVariable_Wrap(q_out));
  PyTuple_SET_ITEM(result, 1, cache != nullptr ? Py_NewRef(Py_None) : THPVariable_Wrap(k_out));
  return result;
}

// ------------------------------------------------------------------------------------------ tree attention, commit

PyObject* tree_attention(Args a) {
  const at::Tensor &q = a.tensor(0, "q"), &kv_cache = a.tensor(1, "kv_cache"), &kv_lens = a.tensor(2, "kv_lens");
  const at::Tensor &page_indices = a.tensor(3, "page_indices"), &cu_q_lens = a.tensor(4, "cu_q_lens");
  const at::Tensor &tree_mask = a.tensor(5, "tree_mask"), &distribution = a.tensor(6, "distribution");
  const Cache c(kv_cache, kv_lens, page_indices);
  require(q.dim() == 3 && q.size(2) == c.D && q.scalar_type() == at::kBFloat16, "q is (T, H, D) bfloat16");
  const int T = to_int(q.size(0)), H = to_int(q.size(1));
  require(is_vector(cu_q_lens, c.seqs + 1) && is_vector(distribution, 3), "cu_q_lens is int32 (S + 1,), distribution int32 (3,)");
  require(tree_mask.dim() == 2 && tree_mask.size(0) == T && tree_mask.size(1) > 0 && tree_mask.scalar_type() == at::kInt,
          "tree_mask is int32 (T, words), 32 new tokens a word");
  Device device;
  for (const at::Tensor* t : {&q, &kv_cache, &kv_lens, &page_indices, &cu_q_lens, &tree_mask, &distribution}) device.add(*t);
  at::Tensor out;
  if (a.none(8)) {
    out = fresh({T, H, c.D}, at::kBFloat16, device.get());
  } else {
    out = a.tensor(8, "out");
    require(out.sizes() == q.sizes() && out.scalar_type() == at::kBFloat16 && out.is_contiguous() && out.device() == q.device(),
            "out must look like q");
    require(address(out) == address(q) || !overlap(out, q), "out is q itself or memory of its own");
    for (const at::Tensor* t : {&kv_cache, &kv_lens, &page_indices, &cu_q_lens, &tree_mask, &distribution})
      require(!overlap(out, *t), "out overlaps an input");
  }
  if (T > 0) {
    const c10::cuda::CUDAGuard guard(device.get());
    // Scratch of the stream it is used on, which no other gets while the kernels may still run.
    const size_t need = tree_bytes_fn(T, c.seqs, H, c.kv_heads);
    const at::Tensor scratch = fresh({static_cast<int64_t>(need) + 256}, at::kByte, device.get());
    const uintptr_t at = (address(scratch) + 255) & ~static_cast<uintptr_t>(255);
    check(tree_fn(q.data_ptr(), out.data_ptr(), kv_cache.data_ptr(), ints(kv_lens), ints(page_indices), ints(cu_q_lens),
                  ints(tree_mask), ints(distribution), T, c.seqs, H, c.kv_heads, c.D, to_int(tree_mask.size(1)), c.page_size,
                  c.pages_per_seq, c.pages, static_cast<float>(a.number(7)), reinterpret_cast<void*>(at), need,
                  stream_of(device.get())));
  }
  return a.none(8) ? THPVariable_Wrap(out) : Py_NewRef(a.at[8]);
}

PyObject* commit(Args a) {
  const at::Tensor &kv_cache = a.tensor(0, "kv_cache"), &kv_lens = a.tensor(1, "kv_lens"), &page_indices = a.tensor(2, "page_indices");
  const at::Tensor &cu_q_lens = a.tensor(3, "cu_q_lens"), &paths = a.tensor(4, "paths"), &n_accepted = a.tensor(5, "n_accepted");
  const Cache c(kv_cache, kv_lens, page_indices);
  require(is_vector(cu_q_lens, c.seqs + 1), "cu_q_lens is int32 (S + 1,)");
  require(paths.dim() == 2 && paths.size(0) == c.seqs && paths.size(1) > 0 && paths.scalar_type() == at::kInt &&
              is_vector(n_accepted, c.seqs),
          "paths is int32 (S, P), n_accepted int32 (S,)");
  for (const at::Tensor* t : {&kv_lens, &page_indices, &cu_q_lens, &paths, &n_accepted})
    require(!overlap(kv_cache, *t), "the cache overlaps kv_lens, page_indices, cu_q_lens, paths or n_accepted");
  Device device;
  for (const at::Tensor* t : {&kv_cache, &kv_lens, &page_indices, &cu_q_lens, &paths, &n_accepted}) device.add(*t);
  at::Tensor out;
  if (a.none(6)) {
    out = fresh({c.seqs}, at::kInt, device.get());
  } else {
    out = a.tensor(6, "out");
    require(is_vector(out, c.seqs) && out.is_contiguous() && out.device() == device.get(), "out is int32 (S,), on the cache's device");
    for (const at::Tensor* t : {&kv_cache, &kv_lens, &page_indices, &cu_q_lens, &paths, &n_accepted})
      require(!overlap(out, *t), "out overlaps an input");
  }
  const c10::cuda::CUDAGuard guard(device.get());
  check(commit_fn(kv_cache.data_ptr(), ints(kv_lens), ints(page_indices), ints(cu_q_lens), ints(paths), ints(n_accepted),
                  ints_out(out), c.seqs, to_int(paths.size(1)), c.kv_heads, c.D, c.page_size, c.pages_per_seq, c.pages,
                  stream_of(device.get())));
  return a.none(6) ? THPVariable_Wrap(out) : Py_NewRef(a.at[6]);
}

// ------------------------------------------------------------------------------------------ the module

template <PyObject* (*F)(Args), int N>
PyObject* method(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  try {
    if (check_fn == nullptr) throw BadValue{"the binding has not been given the library's entry points"};
    return F(Args(args, n, N));
  } catch (const BadValue& e) {
    PyErr_SetString(PyExc_ValueError, e.text.c_str());
  } catch (const PythonError&) {
  }
  return nullptr;
  END_HANDLE_TH_ERRORS
}

// bind(addresses of the five entry points in the order above, _lib.check)
PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long f[5];
  PyObject* check;
  if (!PyArg_ParseTuple(args, "KKKKKO", f, f + 1, f + 2, f + 3, f + 4, &check)) return nullptr;
  plan_fn = reinterpret_cast<decltype(plan_fn)>(f[0]), norm_rope_fn = reinterpret_cast<decltype(norm_rope_fn)>(f[1]);
  tree_bytes_fn = reinterpret_cast<decltype(tree_bytes_fn)>(f[2]), tree_fn = reinterpret_cast<decltype(tree_fn)>(f[3]);
  commit_fn = reinterpret_cast<decltype(commit_fn)>(f[4]);
  Py_INCREF(check);
  Py_XDECREF(check_fn);
  check_fn = check;
  Py_RETURN_NONE;
}

template <PyObject* (*F)(Args), int N>
PyMethodDef entry(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&method<F, N>)), METH_FASTCALL, nullptr};
}

PyMethodDef methods[] = {entry<plan, 10>("rpa_plan"), entry<norm_rope, 13>("norm_rope"), entry<tree_attention, 9>("rpa_tree_attention"),
                         entry<commit, 7>("rpa_commit"), {"bind", bind, METH_VARARGS, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, methods};

}  // namespace

// `built_for`: the Python and torch whose headers this was compiled against (build.py's binding_key).
PyMODINIT_FUNC PyInit__binding(void) {
  PyObject* m = PyModule_Create(&module);
  if (m != nullptr && PyModule_AddStringConstant(m, "built_for", TJX_BUILT_FOR) != 0) Py_CLEAR(m);
  return m;
}
