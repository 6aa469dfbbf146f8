// The Python calls of the operators on device memory (qd_operators.py): reads torch
// tensors, checks their types, shapes, devices and layouts, and calls the C ABI
// (include/qd/qd_operators.h). A small call takes the device 3 us; looking at its
// nine tensors from Python took 5 us on the host, from here 0.2.
//
// A call returns None, the library's status (its text is in qd_last_error()), or a
// text: what is wrong with an argument.
#include <torch/csrc/autograd/python_variable.h>

#include <climits>
#include <initializer_list>
#include <string>
#include <type_traits>

#include "qd/qd_operators.h"

namespace {

// The library's entry points, which Python hands over once.
struct {
  decltype(&qd_paged_append_at) append;
  decltype(&qd_paged_attention) attention;
  decltype(&qd_pages_fork) fork;
  decltype(&qd_beam_select) select;
  decltype(&qd_tree_attention) tree_attention;
  decltype(&qd_tree_accept) tree_accept;
  decltype(&qd_tree_commit) tree_commit;
  decltype(&qd_page_bounds) page_bounds;
  decltype(&qd_sparse_attention) sparse_attention;
} g_calls;

struct Refusal {
  std::string text;
};
[[noreturn]] void refuse(const std::string &text) { throw Refusal{text}; }

std::string words(at::IntArrayRef v) {
  std::string s = "(";
  for (size_t i = 0; i < v.size(); ++i) s += (i ? ", " : "") + std::to_string(v[i]);
  return s + ")";
}

bool missing(PyObject *o) { return o == Py_None; }

const at::Tensor &tensor(const char *name, PyObject *o) {
  if (missing(o)) refuse(std::string(name) + " is missing");
  if (!THPVariable_Check(o)) refuse(std::string(name) + " is no tensor");
  return THPVariable_Unpack(o);
}
const at::Tensor &tensor(const char *name, PyObject *o, int64_t dims) {
  const at::Tensor &t = tensor(name, o);
  if (t.dim() != dims) refuse(std::string(name) + " needs " + std::to_string(dims) + " dimensions");
  return t;
}

enum class Lies { kRows, kHeads, kTogether };  // contiguous: the last dimension, the last two, all

// The tensors that a call writes: torch copies their storage first where a lazy clone
// shares it, and counts the change, by which autograd knows that a tensor it keeps is not
// what it was. What a call writes is looked at before what it reads: both may be views of
// one storage.
constexpr int kMostTensors = 8;  // of a cache or a pool
class Written {
 public:
  void *at(const at::Tensor &t) {
    add(t);
    return t.mutable_data_ptr();
  }
  void add(const at::Tensor &t) { all_[n_++] = &t; }
  void changed() const {
    for (int i = 0; i < n_; ++i)
      if (!all_[i]->is_inference()) all_[i]->unsafeGetTensorImpl()->bump_version();
  }

 private:
  const at::Tensor *all_[kMostTensors + 4];
  int n_ = 0;
};

struct View {
  void *at;
  const int64_t *strides;
};
// A tensor of this type, shape, device and layout.
View view(const char *name, PyObject *o, at::ScalarType type, std::initializer_list<int64_t> shape, int device, Lies lies,
          Written *written = nullptr) {
  const at::Tensor &t = tensor(name, o);
  const at::IntArrayRef want(shape), sizes = t.sizes(), s = t.strides();
  if (sizes != want) refuse(std::string(name) + " has shape " + words(sizes) + ", not " + words(want));
  if (t.scalar_type() != type)
    refuse(std::string(name) + " has type " + c10::toString(t.scalar_type()) + ", not " + c10::toString(type));
  if (t.get_device() != device) refuse(std::string(name) + " is on " + t.device().str() + ", not on device " + std::to_string(device));
  const size_t n = sizes.size();
  bool good = true;
  if (lies == Lies::kTogether)
    good = t.is_contiguous();
  else
    good = (s[n - 1] == 1 || sizes[n - 1] <= 1) && (lies == Lies::kRows || s[n - 2] == sizes[n - 1] || sizes[n - 2] == 1);
  if (!good) refuse(std::string(name) + " is not contiguous where it has to be (strides " + words(s) + ")");
  return {written ? written->at(t) : const_cast<void *>(t.const_data_ptr()), s.data()};
}
template <typename T>
T *flat(const char *name, PyObject *o, at::ScalarType type, std::initializer_list<int64_t> shape, int device) {
  static_assert(std::is_const_v<T>, "results are Written");
  return static_cast<T *>(view(name, o, type, shape, device, Lies::kTogether).at);
}
template <typename T>
T *flat_or_null(const char *name, PyObject *o, at::ScalarType type, std::initializer_list<int64_t> shape, int device) {
  return missing(o) ? nullptr : flat<T>(name, o, type, shape, device);
}
template <typename T>
T *flat(const char *name, PyObject *o, at::ScalarType type, std::initializer_list<int64_t> shape, int device, Written &written) {
  return static_cast<T *>(view(name, o, type, shape, device, Lies::kTogether, &written).at);
}
// Of a tuple of tensors or None, whose addresses the call has already, those from `first` to `last`.
void add_some(Written &written, const char *name, PyObject *tensors, Py_ssize_t first, Py_ssize_t last) {
  if (!PyTuple_Check(tensors) || PyTuple_GET_SIZE(tensors) > kMostTensors) refuse(std::string(name) + " has no such tensors");
  for (Py_ssize_t i = first; i <= last && i < PyTuple_GET_SIZE(tensors); ++i) {
    PyObject *const t = PyTuple_GET_ITEM(tensors, i);
    if (THPVariable_Check(t)) written.add(THPVariable_Unpack(t));
  }
}

int64_t whole(const char *name, PyObject *o, int64_t low, int64_t high) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse(std::string(name) + " is no number that fits");
  }
  if (v < low || v > high) refuse(std::string(name) + " " + std::to_string(v) + " is out of range");
  return v;
}
void *address(const char *name, PyObject *o) {
  void *p = PyLong_AsVoidPtr(o);
  if (!p && PyErr_Occurred()) {
    PyErr_Clear();
    refuse(std::string(name) + " is no address");
  }
  return p;
}

float number(const char *name, PyObject *o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse(std::string(name) + " is no number");
  }
  return static_cast<float>(v);
}
// None: 1 / sqrt(head_dim)
float scale_of(PyObject *o, int64_t dim) { return !missing(o) ? number("scale", o) : dim == 64 ? 0.125f : 0.08838834764831845f; }

at::ScalarType type_of(uint32_t dtype) {
  return dtype == QD_DTYPE_F32 ? at::kFloat : dtype == QD_DTYPE_BF16 ? at::kBFloat16 : at::kHalf;
}

// Other threads may run while the library queues.
template <typename... A>
qd_status queue(const Written &written, qd_status (*call)(A...), A... args) {
  if (!call) refuse("the library is not loaded");
  PyThreadState *const state = PyEval_SaveThread();
  const qd_status status = call(args...);
  PyEval_RestoreThread(state);
  if (status == QD_SUCCESS) written.changed();
  return status;
}

// Runs one call: its refusals and errors become what Python is told.
template <typename F>
PyObject *answer(Py_ssize_t given, Py_ssize_t wanted, F &&call) noexcept {
  try {
    if (given != wanted) refuse("the call takes " + std::to_string(wanted) + " arguments");
    const qd_status status = call();
    if (status == QD_SUCCESS) Py_RETURN_NONE;
    return PyLong_FromLong(status);
  } catch (const Refusal &r) {
    return PyUnicode_FromString(r.text.c_str());
  } catch (const std::exception &e) {
    return PyUnicode_FromString(e.what());
  }
}

// (append, attention, fork, select, tree_attention, tree_accept, tree_commit, page_bounds, sparse_attention):
// the entry points' addresses
PyObject *call_bind(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return answer(n, 9, [&] {
    g_calls.append = reinterpret_cast<decltype(g_calls.append)>(address("append", a[0]));
    g_calls.attention = reinterpret_cast<decltype(g_calls.attention)>(address("attention", a[1]));
    g_calls.fork = reinterpret_cast<decltype(g_calls.fork)>(address("fork", a[2]));
    g_calls.select = reinterpret_cast<decltype(g_calls.select)>(address("select", a[3]));
    g_calls.tree_attention = reinterpret_cast<decltype(g_calls.tree_attention)>(address("tree_attention", a[4]));
    g_calls.tree_accept = reinterpret_cast<decltype(g_calls.tree_accept)>(address("tree_accept", a[5]));
    g_calls.tree_commit = reinterpret_cast<decltype(g_calls.tree_commit)>(address("tree_commit", a[6]));
    g_calls.page_bounds = reinterpret_cast<decltype(g_calls.page_bounds)>(address("page_bounds", a[7]));
    g_calls.sparse_attention = reinterpret_cast<decltype(g_calls.sparse_attention)>(address("sparse_attention", a[8]));
    return QD_SUCCESS;
  });
}

// (cache, q_out, q, k, v, positions, rows, cos, sin, interleaved, position_bias, stream, the cache's tensors, slots)
PyObject *call_append(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return answer(n, 14, [&] {
    const auto *c = static_cast<const qd_paged_cache *>(address("cache", a[0]));
    const int device = c->device;
    const at::ScalarType type = type_of(c->dtype);
    const int64_t tokens = tensor("k", a[3], 3).size(0), dim = c->head_dim, kv_heads = c->kv_heads;
    if (tokens > UINT32_MAX) refuse("too many tokens");
    qd_append_args g{};
    Written written;
    add_some(written, "cache", a[12], 0, 1);
    add_some(written, "cache", a[12], 4, 4);  // errors
    // Strides from token to token; that of a single one is not used and may be anything.
    const auto rows = [&](const char *name, PyObject *o, int64_t heads, int64_t &stride, Written *result = nullptr) {
      const View x = view(name, o, type, {tokens, heads, dim}, device, Lies::kHeads, result);
      stride = tokens > 1 ? x.strides[0] : heads * dim;
      return x.at;
    };
    if (missing(a[1]) != missing(a[2])) refuse("q and q_out go together");
    if (!missing(a[2])) {
      const int64_t heads = tensor("q", a[2], 3).size(1);
      if (heads > INT_MAX) refuse("too many heads");
      g.heads = static_cast<uint32_t>(heads);
      g.q_out = rows("q_out", a[1], heads, g.q_out_stride, &written);
      g.q = rows("q", a[2], heads, g.q_stride);
    }
    g.k = rows("k", a[3], kv_heads, g.k_stride);
    g.v = rows("v", a[4], kv_heads, g.v_stride);
    if (missing(a[7]) != missing(a[8])) refuse("cos and sin go together");
    if (!missing(a[7])) {
      const at::IntArrayRef s = tensor("cos", a[7], 2).sizes();
      if (s[0] > UINT32_MAX || s[1] > INT_MAX) refuse("cos is too large");
      g.cos_table = flat<const float>("cos", a[7], at::kFloat, {s[0], s[1]}, device);
      g.sin_table = flat<const float>("sin", a[8], at::kFloat, {s[0], s[1]}, device);
      g.table_positions = static_cast<uint32_t>(s[0]);
      g.rotary_dim = static_cast<uint32_t>(2 * s[1]);
    }
    g.positions = flat<const int32_t>("positions", a[5], at::kInt, {tokens}, device);
    g.rows = flat_or_null<const int32_t>("rows", a[6], at::kInt, {tokens}, device);
    const int32_t *const slots = flat_or_null<const int32_t>("slots", a[13], at::kInt, {tokens}, device);
    const int interleaved = PyObject_IsTrue(a[9]);
    if (interleaved < 0) {
      PyErr_Clear();
      refuse("interleaved is neither true nor false");
    }
    g.interleaved = static_cast<uint32_t>(interleaved);
    g.position_bias = static_cast<int32_t>(whole("position_bias", a[10], INT32_MIN, INT32_MAX));
    g.tokens = static_cast<uint32_t>(tokens);
    return queue<const qd_paged_cache *, const qd_append_args *, const int32_t *, void *>(written, g_calls.append, c, &g, slots,
                                                                                          address("stream", a[11]));
  });
}

// (cache, out, q, workspace, scale or None, stream, the cache's tensors)
PyObject *call_attention(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return answer(n, 7, [&] {
    const auto *c = static_cast<const qd_paged_cache *>(address("cache", a[0]));
    const at::ScalarType type = type_of(c->dtype);
    const int64_t rows = c->rows, heads = tensor("q", a[2], 3).size(1), dim = c->head_dim;
    if (heads > INT_MAX) refuse("too many heads");
    Written written;
    add_some(written, "cache", a[6], 4, 4);  // errors
    const View q = view("q", a[2], type, {rows, heads, dim}, c->device, Lies::kRows);
    const View out = view("out", a[1], type, {rows, heads, dim}, c->device, Lies::kRows, &written);
    qd_attention_args g{};
    g.q = tensor("q", a[2]).const_data_ptr();  // (where it lies now)
    g.out = out.at;
    // (The stride of a dimension of one element is not used and may be anything.)
    g.q_stride = rows > 1 ? q.strides[0] : heads * dim;
    g.out_stride = rows > 1 ? out.strides[0] : heads * dim;
    g.q_head_stride = heads > 1 ? q.strides[1] : dim;
    g.out_head_stride = heads > 1 ? out.strides[1] : dim;
    g.heads = static_cast<uint32_t>(heads);
    g.scale = scale_of(a[4], dim);
    return queue<const qd_paged_cache *, const qd_attention_args *, qd_workspace *, void *>(
        written, g_calls.attention, c, &g, static_cast<qd_workspace *>(address("workspace", a[3])), address("stream", a[5]));
  });
}

// (refs, page_size, memories, memory_count, table, lengths, parents, append, table_out, lengths_out, workspace,
// errors, stream, the memories' tensors)
PyObject *call_fork(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return answer(n, 14, [&] {
    const at::Tensor &refs = tensor("refs", a[0], 1), &table = tensor("table", a[4], 2);
    const int device = static_cast<int>(refs.get_device());
    const int64_t rows = table.size(0), width = table.size(1), pages = refs.size(0);
    if (rows > INT_MAX || width > INT_MAX || pages > INT_MAX) refuse("the table or the pool is too large");
    qd_fork_args g{};
    Written written;
    add_some(written, "pool", a[13], 0, kMostTensors);
    const View to = view("table_out", a[8], at::kInt, {rows, width}, device, Lies::kRows, &written);
    g.lengths_out = flat<int32_t>("lengths_out", a[9], at::kInt, {rows}, device, written);
    g.refs = flat<int32_t>("refs", a[0], at::kInt, {pages}, device, written);
    if (!missing(a[11])) g.errors = flat<uint32_t>("errors", a[11], at::kInt, {1}, device, written);
    const View from = view("table", a[4], at::kInt, {rows, width}, device, Lies::kRows);
    g.table = static_cast<const int32_t *>(from.at);
    g.table_out = static_cast<int32_t *>(to.at);
    g.table_stride = rows > 1 ? from.strides[0] : width;
    g.table_out_stride = rows > 1 ? to.strides[0] : width;
    g.lengths = flat<const int32_t>("lengths", a[5], at::kInt, {rows}, device);
    g.parents = flat_or_null<const int32_t>("parents", a[6], at::kInt, {rows}, device);
    g.memories = static_cast<const qd_page_memory *>(address("memories", a[2]));
    g.memory_count = static_cast<uint32_t>(whole("memories", a[3], 0, UINT32_MAX));
    g.rows = static_cast<uint32_t>(rows);
    g.table_width = static_cast<uint32_t>(width);
    g.pages = static_cast<uint32_t>(pages);
    g.page_size = static_cast<uint32_t>(whole("page_size", a[1], 0, UINT32_MAX));
    g.append = static_cast<uint32_t>(whole("append", a[7], 0, UINT32_MAX));
    g.device = device;
    return queue<const qd_fork_args *, qd_workspace *, void *>(
        written, g_calls.fork, &g, static_cast<qd_workspace *>(address("workspace", a[10])), address("stream", a[12]));
  });
}

// (logits, scores, scores_out, parents, tokens, workspace, done, done_out, eos, stream)
PyObject *call_select(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return answer(n, 10, [&] {
    const at::Tensor &logits = tensor("logits", a[0], 3);
    const at::ScalarType type = logits.scalar_type();
    if (type != at::kFloat && type != at::kBFloat16 && type != at::kHalf)
      refuse(std::string("logits of type ") + c10::toString(type));
    const int device = static_cast<int>(logits.get_device());
    const int64_t groups = logits.size(0), beams = logits.size(1), vocab = logits.size(2);
    const int64_t k = tensor("scores_out", a[2], 2).size(1);
    if (groups > INT_MAX || beams > INT_MAX || vocab > INT_MAX || k > INT_MAX) refuse("logits are too large");
    qd_select_args g{};
    Written written;
    g.scores_out = flat<float>("scores_out", a[2], at::kFloat, {groups, k}, device, written);
    g.parents = flat<int32_t>("parents", a[3], at::kInt, {groups, k}, device, written);
    g.tokens = flat<int32_t>("tokens", a[4], at::kInt, {groups, k}, device, written);
    if (missing(a[6]) != missing(a[7]) || (!missing(a[6]) && missing(a[8]))) refuse("done, done_out and eos go together");
    if (!missing(a[6])) g.done_out = flat<uint8_t>("done_out", a[7], at::kByte, {groups, k}, device, written);
    const View x = view("logits", a[0], type, {groups, beams, vocab}, device, Lies::kRows);
    g.logits = x.at;
    g.group_stride = x.strides[0];
    g.beam_stride = x.strides[1];
    g.scores = flat<const float>("scores", a[1], at::kFloat, {groups, beams}, device);
    if (!missing(a[6])) {
      g.done = flat<const uint8_t>("done", a[6], at::kByte, {groups, beams}, device);
      g.eos = static_cast<uint32_t>(whole("eos", a[8], 0, UINT32_MAX));
    }
    g.dtype = type == at::kFloat ? QD_DTYPE_F32 : type == at::kBFloat16 ? QD_DTYPE_BF16 : QD_DTYPE_F16;
    g.groups = static_cast<uint32_t>(groups);
    g.beams = static_cast<uint32_t>(beams);
    g.vocab = static_cast<uint32_t>(vocab);
    g.k = static_cast<uint32_t>(k);
    g.device = device;
    return queue<const qd_select_args *, qd_workspace *, void *>(
        written, g_calls.select, &g, static_cast<qd_workspace *>(address("workspace", a[5])), address("stream", a[9]));
  });
}

// (cache, out, q, parents, workspace, scale or None, stream, the cache's tensors)
PyObject *call_tree_attention(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return answer(n, 8, [&] {
    const auto *c = static_cast<const qd_paged_cache *>(address("cache", a[0]));
    const at::ScalarType type = type_of(c->dtype);
    const at::Tensor &first = tensor("q", a[2], 4);
    const int64_t rows = c->rows, nodes = first.size(1), heads = first.size(2), dim = c->head_dim;
    if (heads > INT_MAX || nodes > INT_MAX) refuse("too many heads or nodes");
    Written written;
    add_some(written, "cache", a[7], 4, 4);  // errors
    const View out = view("out", a[1], type, {rows, nodes, heads, dim}, c->device, Lies::kRows, &written);
    const View q = view("q", a[2], type, {rows, nodes, heads, dim}, c->device, Lies::kRows);
    qd_tree_attention_args g{};
    g.q = q.at;
    g.out = out.at;
    // (The stride of a dimension of one element is not used and may be anything.)
    g.q_stride = rows > 1 ? q.strides[0] : nodes * heads * dim;
    g.out_stride = rows > 1 ? out.strides[0] : nodes * heads * dim;
    g.q_node_stride = nodes > 1 ? q.strides[1] : heads * dim;
    g.out_node_stride = nodes > 1 ? out.strides[1] : heads * dim;
    g.q_head_stride = heads > 1 ? q.strides[2] : dim;
    g.out_head_stride = heads > 1 ? out.strides[2] : dim;
    g.parents = flat<const int32_t>("parents", a[3], at::kInt, {rows, nodes}, c->device);
    g.nodes = static_cast<uint32_t>(nodes);
    g.heads = static_cast<uint32_t>(heads);
    g.scale = scale_of(a[5], dim);
    return queue<const qd_paged_cache *, const qd_tree_attention_args *, qd_workspace *, void *>(
        written, g_calls.tree_attention, c, &g, static_cast<qd_workspace *>(address("workspace", a[4])), address("stream", a[6]));
  });
}

// (logits, tokens, parents, path, counts, next_tokens, workspace, draws or None, temperature, errors or None, stream)
PyObject *call_tree_accept(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return answer(n, 11, [&] {
    const at::Tensor &logits = tensor("logits", a[0], 3);
    const at::ScalarType type = logits.scalar_type();
    if (type != at::kFloat && type != at::kBFloat16 && type != at::kHalf)
      refuse(std::string("logits of type ") + c10::toString(type));
    const int device = static_cast<int>(logits.get_device());
    const int64_t rows = logits.size(0), nodes = logits.size(1), vocab = logits.size(2);
    if (rows > INT_MAX || nodes > INT_MAX || vocab > INT_MAX) refuse("logits are too large");
    qd_accept_args g{};
    Written written;
    g.path = flat<int32_t>("path", a[3], at::kInt, {rows, nodes}, device, written);
    g.counts = flat<int32_t>("counts", a[4], at::kInt, {rows}, device, written);
    g.next_tokens = flat<int32_t>("next_tokens", a[5], at::kInt, {rows}, device, written);
    if (!missing(a[9])) g.errors = flat<uint32_t>("errors", a[9], at::kInt, {1}, device, written);
    const View x = view("logits", a[0], type, {rows, nodes, vocab}, device, Lies::kRows);
    g.logits = x.at;
    g.row_stride = rows > 1 ? x.strides[0] : 0;
    g.node_stride = nodes > 1 ? x.strides[1] : 0;
    g.tokens = flat<const int32_t>("tokens", a[1], at::kInt, {rows, nodes}, device);
    g.parents = flat<const int32_t>("parents", a[2], at::kInt, {rows, nodes}, device);
    g.draws = flat_or_null<const float>("draws", a[7], at::kFloat, {rows, nodes}, device);
    g.temperature = number("temperature", a[8]);
    g.dtype = type == at::kFloat ? QD_DTYPE_F32 : type == at::kBFloat16 ? QD_DTYPE_BF16 : QD_DTYPE_F16;
    g.rows = static_cast<uint32_t>(rows);
    g.nodes = static_cast<uint32_t>(nodes);
    g.vocab = static_cast<uint32_t>(vocab);
    g.device = device;
    return queue<const qd_accept_args *, qd_workspace *, void *>(
        written, g_calls.tree_accept, &g, static_cast<qd_workspace *>(address("workspace", a[6])), address("stream", a[10]));
  });
}

// (page_size, pages, device, memories, memory_count, table, lengths, path, counts, lengths_out, errors or None, stream,
// the memories' tensors)
PyObject *call_tree_commit(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return answer(n, 13, [&] {
    const at::Tensor &table = tensor("table", a[5], 2), &path = tensor("path", a[7], 2);
    const int device = static_cast<int>(whole("device", a[2], -1, INT_MAX));
    const int64_t rows = table.size(0), width = table.size(1), nodes = path.size(1);
    if (rows > INT_MAX || width > INT_MAX || nodes > INT_MAX) refuse("the table or the tree is too large");
    qd_commit_args g{};
    Written written;
    add_some(written, "memory", a[12], 0, kMostTensors);
    g.lengths_out = flat<int32_t>("lengths_out", a[9], at::kInt, {rows}, device, written);
    if (!missing(a[10])) g.errors = flat<uint32_t>("errors", a[10], at::kInt, {1}, device, written);
    const View t = view("table", a[5], at::kInt, {rows, width}, device, Lies::kRows);
    g.table = static_cast<const int32_t *>(t.at);
    g.table_stride = rows > 1 ? t.strides[0] : width;
    g.lengths = flat<const int32_t>("lengths", a[6], at::kInt, {rows}, device);
    g.path = flat<const int32_t>("path", a[7], at::kInt, {rows, nodes}, device);
    g.counts = flat<const int32_t>("counts", a[8], at::kInt, {rows}, device);
    g.memories = static_cast<const qd_token_memory *>(address("memories", a[3]));
    g.memory_count = static_cast<uint32_t>(whole("memories", a[4], 0, UINT32_MAX));
    g.rows = static_cast<uint32_t>(rows);
    g.nodes = static_cast<uint32_t>(nodes);
    g.table_width = static_cast<uint32_t>(width);
    g.pages = static_cast<uint32_t>(whole("pages", a[1], 0, UINT32_MAX));
    g.page_size = static_cast<uint32_t>(whole("page_size", a[0], 0, UINT32_MAX));
    g.device = device;
    return queue<const qd_commit_args *, void *>(written, g_calls.tree_commit, &g, address("stream", a[11]));
  });
}

// (cache, bounds, recent, stream, the cache's tensors)
PyObject *call_page_bounds(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return answer(n, 5, [&] {
    const auto *c = static_cast<const qd_paged_cache *>(address("cache", a[0]));
    Written written;
    add_some(written, "cache", a[4], 4, 4);  // errors
    const View bounds = view("bounds", a[1], type_of(c->dtype), {c->pages, c->kv_heads, 2, c->head_dim}, c->device, Lies::kTogether, &written);
    return queue<const qd_paged_cache *, void *, uint32_t, void *>(
        written, g_calls.page_bounds, c, bounds.at, static_cast<uint32_t>(whole("recent", a[2], 0, UINT32_MAX)), address("stream", a[3]));
  });
}

// (cache, bounds, out, q, workspace, budget, first, last, chosen or None, scale or None, stream, the cache's tensors)
PyObject *call_sparse_attention(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return answer(n, 12, [&] {
    const auto *c = static_cast<const qd_paged_cache *>(address("cache", a[0]));
    const at::ScalarType type = type_of(c->dtype);
    const int64_t rows = c->rows, heads = tensor("q", a[3], 3).size(1), dim = c->head_dim;
    if (heads > INT_MAX) refuse("too many heads");
    qd_sparse_args g{};
    Written written;
    add_some(written, "cache", a[11], 4, 4);  // errors
    g.budget = static_cast<uint32_t>(whole("budget", a[5], 0, UINT32_MAX));
    g.first = static_cast<uint32_t>(whole("first", a[6], 0, UINT32_MAX));
    g.last = static_cast<uint32_t>(whole("last", a[7], 0, UINT32_MAX));
    const View out = view("out", a[2], type, {rows, heads, dim}, c->device, Lies::kRows, &written);
    if (!missing(a[8])) g.chosen = flat<int32_t>("chosen", a[8], at::kInt, {rows, c->kv_heads, g.budget}, c->device, written);
    const View q = view("q", a[3], type, {rows, heads, dim}, c->device, Lies::kRows);
    g.bounds = view("bounds", a[1], type, {c->pages, c->kv_heads, 2, dim}, c->device, Lies::kTogether).at;
    g.q = q.at;
    g.out = out.at;
    g.q_stride = rows > 1 ? q.strides[0] : heads * dim;
    g.out_stride = rows > 1 ? out.strides[0] : heads * dim;
    g.q_head_stride = heads > 1 ? q.strides[1] : dim;
    g.out_head_stride = heads > 1 ? out.strides[1] : dim;
    g.heads = static_cast<uint32_t>(heads);
    g.scale = scale_of(a[9], dim);
    return queue<const qd_paged_cache *, const qd_sparse_args *, qd_workspace *, void *>(
        written, g_calls.sparse_attention, c, &g, static_cast<qd_workspace *>(address("workspace", a[4])), address("stream", a[10]));
  });
}

#define QD_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(call_##name)), METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {QD_METHOD(bind), QD_METHOD(append), QD_METHOD(attention), QD_METHOD(fork), QD_METHOD(select),
                           QD_METHOD(tree_attention), QD_METHOD(tree_accept), QD_METHOD(tree_commit), QD_METHOD(page_bounds),
                           QD_METHOD(sparse_attention), {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_qd_tensors", nullptr, -1, g_methods};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject *PyInit__qd_tensors() { return PyModule_Create(&g_module); }
