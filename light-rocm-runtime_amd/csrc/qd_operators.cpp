// C ABI of the operators on the caller's device memory
// (include/qd/qd_operators.h): argument checks, the workspace, and the rotary
// tables. Nothing here throws; every refusal happens before any device work.
#include "qd/qd_operators.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <initializer_list>
#include <new>

#include "qd_operators.hpp"

namespace qd {
// Defined in qd_engine.cpp: keep the text for qd_last_error().
qd_status report(qd_status status, const char *text) noexcept;
qd_status report_hip(hipError_t e, const char *what) noexcept;
}  // namespace qd

struct qd_workspace {
  int32_t device;
  char *base;     // counters, then scratch
  size_t bytes;   // of scratch
};

namespace {

qd_status refuse(qd_status s, const char *fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  std::vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return qd::report(s, buf);
}
qd_status invalid(const char *what) { return refuse(QD_ERROR_INVALID_ARGUMENT, "%s", what); }

#define QD_TRY(call)                      \
  do {                                    \
    const qd_status try_status = (call);  \
    if (try_status != QD_SUCCESS) return try_status; \
  } while (0)

uint32_t element_bytes(uint32_t dtype) { return dtype == QD_DTYPE_F32 ? 4 : 2; }

qd_status check_dtype(uint32_t dtype) {
  if (dtype != QD_DTYPE_F32 && dtype != QD_DTYPE_BF16 && dtype != QD_DTYPE_F16)
    return refuse(QD_ERROR_INVALID_ARGUMENT, "dtype %u is none of QD_DTYPE_F32, QD_DTYPE_BF16 and QD_DTYPE_F16", dtype);
  return QD_SUCCESS;
}

bool aligned16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// A stride in elements, a multiple of 16 bytes, of at least `least` elements.
qd_status check_stride(int64_t stride, int64_t least, uint32_t bytes, const char *name) {
  if (stride < least || stride > (int64_t(1) << 40) || stride * bytes % 16 != 0)
    return refuse(QD_ERROR_INVALID_ARGUMENT, "%s %lld: at least %lld and a multiple of 16 bytes are needed", name,
                  static_cast<long long>(stride), static_cast<long long>(least));
  return QD_SUCCESS;
}

// Whether two arrays of so many 32-bit words share some; `b` may be rows, `stride` words apart.
bool overlap(const void *a, uint64_t a_words, const void *b, uint64_t b_words, uint64_t rows = 1, uint64_t stride = 0) {
  if (!a || !b || a_words == 0 || b_words == 0 || rows == 0) return false;
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  if (x < y) return (y - x) / 4 < a_words;
  const uint64_t in = (x - y) / 4, row = stride ? std::min(in / stride, rows - 1) : 0, at = in - row * stride;
  return at < b_words || (row + 1 < rows && at + a_words > stride);
}

qd_status check_page_size(uint32_t n) {
  if (n < qd::kPageSizeLeast || n > qd::kPageSizeMost || (n & (n - 1)) != 0)
    return refuse(QD_ERROR_NOT_SUPPORTED, "page_size %u: a power of two from %u to %u is needed", n, qd::kPageSizeLeast,
                  qd::kPageSizeMost);
  return QD_SUCCESS;
}

qd_status check_cache(const qd_paged_cache *c) {
  if (!c) return invalid("null cache");
  QD_TRY(check_dtype(c->dtype));
  QD_TRY(check_page_size(c->page_size));
  if (c->head_dim != 64 && c->head_dim != 128)
    return refuse(QD_ERROR_NOT_SUPPORTED, "head_dim %u: the kernels take 64 and 128", c->head_dim);
  if (c->kv_heads == 0 || c->kv_heads > 4096) return refuse(QD_ERROR_INVALID_ARGUMENT, "kv_heads %u", c->kv_heads);
  if (c->rows > (1u << 20) || c->pages > 0x7fffffffu) return invalid("too many rows or pages");
  const uint64_t positions = static_cast<uint64_t>(c->table_width) * c->page_size;
  if (positions > (1u << 30) || positions * c->rows > (uint64_t(1) << 35))
    return refuse(QD_ERROR_NOT_SUPPORTED, "tables of more than 2^30 positions per row or 2^35 in all");
  if (c->rows && (!c->table || !c->lengths)) return invalid("null table or lengths");
  if (c->table_stride < static_cast<int64_t>(c->table_width) || c->table_stride > (int64_t(1) << 40))
    return invalid("table_stride is less than table_width");
  if (c->pages && (!c->k || !c->v)) return invalid("null pages");
  if (!aligned16(c->k) || !aligned16(c->v)) return invalid("k and v need 16-byte aligned addresses");
  const uint32_t e = element_bytes(c->dtype);
  QD_TRY(check_stride(c->page_stride, 0, e, "page_stride"));
  QD_TRY(check_stride(c->token_stride, c->head_dim, e, "token_stride"));
  QD_TRY(check_stride(c->head_stride, c->kv_heads > 1 ? c->head_dim : 0, e, "head_stride"));
  if (c->token_stride * e * 16 > 0x7fffffff) return refuse(QD_ERROR_NOT_SUPPORTED, "token_stride past 2^27 bytes");
  return QD_SUCCESS;
}

// Makes `device` current while it lives.
class Device {
 public:
  qd_status enter(int32_t device) {
    static std::atomic<int> count{0};  // a process's devices do not change
    int n = count.load(std::memory_order_relaxed);
    if (n == 0) {
      if (hipGetDeviceCount(&n) != hipSuccess || n <= 0) {
        (void)hipGetLastError();
        return refuse(QD_ERROR_NOT_SUPPORTED, "no HIP device visible");
      }
      count.store(n, std::memory_order_relaxed);
    }
    if (device < 0 || device >= n) return refuse(QD_ERROR_INVALID_ARGUMENT, "device %d out of range (%d visible)", device, n);
    hipError_t e = hipGetDevice(&before_);
    if (e == hipSuccess && before_ != device) {
      e = hipSetDevice(device);
      moved_ = e == hipSuccess;
    }
    return e == hipSuccess ? QD_SUCCESS : qd::report_hip(e, "hipSetDevice");
  }
  ~Device() {
    if (moved_) (void)hipSetDevice(before_);
  }

 private:
  int before_ = 0;
  bool moved_ = false;
};

qd_status launched(hipError_t e, const char *what) {
  if (e == hipSuccess) return QD_SUCCESS;
  (void)hipGetLastError();  // not the next launch's error
  return qd::report_hip(e, what);
}

qd_status check_workspace(const qd_workspace *w, int32_t device, size_t bytes, qd::OpScratch *out) {
  if (!w) return invalid("null workspace");
  if (w->device != device)
    return refuse(QD_ERROR_INVALID_ARGUMENT, "the workspace is on device %d, the call on device %d", w->device, device);
  if (w->bytes < bytes)
    return refuse(QD_ERROR_INVALID_ARGUMENT, "the workspace has %zu bytes, the call needs %zu", w->bytes, bytes);
  out->counters = reinterpret_cast<uint32_t *>(w->base);
  out->scratch = w->base + qd::kOpCounterBytes;
  return QD_SUCCESS;
}

qd_status check_heads(uint32_t heads, uint32_t kv_heads) {
  if (heads == 0 || kv_heads == 0 || heads % kv_heads != 0 || heads > 65536)
    return refuse(QD_ERROR_INVALID_ARGUMENT, "heads %u: a multiple of kv_heads %u is needed", heads, kv_heads);
  return QD_SUCCESS;
}

qd_status check_select(uint32_t groups, uint32_t beams, uint32_t k, uint32_t vocab) {
  if (beams == 0 || vocab == 0 || k == 0) return invalid("beams, vocab and k must be positive");
  if (beams > qd::kSelectBeams || k > qd::kSelectK)
    return refuse(QD_ERROR_NOT_SUPPORTED, "%u beams, k %u: up to %u and %u", beams, k, qd::kSelectBeams, qd::kSelectK);
  if (k > static_cast<uint64_t>(beams) * vocab) return refuse(QD_ERROR_INVALID_ARGUMENT, "k %u of %u x %u", k, beams, vocab);
  if (vocab > qd::kSelectVocab) return refuse(QD_ERROR_NOT_SUPPORTED, "vocab %u: up to %u", vocab, qd::kSelectVocab);
  if (static_cast<uint64_t>(groups) * (beams + 1) > 65535)
    return refuse(QD_ERROR_NOT_SUPPORTED, "%u groups of %u beams: up to 65535 groups and beams together", groups, beams);
  return QD_SUCCESS;
}

qd_status check_nodes(uint32_t nodes) {
  if (nodes == 0 || nodes > qd::kTreeNodes) return refuse(QD_ERROR_NOT_SUPPORTED, "%u nodes: from 1 to %u", nodes, qd::kTreeNodes);
  return QD_SUCCESS;
}

// (An arrival counter for every node and every row; a grid's second dimension.)
qd_status check_accept(uint32_t rows, uint32_t nodes, uint32_t vocab) {
  QD_TRY(check_nodes(nodes));
  if (vocab == 0) return invalid("vocab must be positive");
  if (vocab > qd::kSelectVocab) return refuse(QD_ERROR_NOT_SUPPORTED, "vocab %u: up to %u", vocab, qd::kSelectVocab);
  if (static_cast<uint64_t>(rows) * (nodes + 1) > 65535)
    return refuse(QD_ERROR_NOT_SUPPORTED, "%u rows of %u nodes: up to 65535 rows and nodes together", rows, nodes);
  return QD_SUCCESS;
}

qd_status check_head_dim(uint32_t head_dim) {
  if (head_dim != 64 && head_dim != 128) return refuse(QD_ERROR_NOT_SUPPORTED, "head_dim %u: the kernels take 64 and 128", head_dim);
  return QD_SUCCESS;
}

// Queries and outputs of `rows` rows of heads.
qd_status check_rows_of_heads(const qd_paged_cache *c, const void *q, const void *out, int64_t q_stride, int64_t q_head_stride,
                              int64_t out_stride, int64_t out_head_stride, uint32_t heads) {
  const uint32_t e = element_bytes(c->dtype);
  if (!q || !out) return invalid("null tensor");
  if (!aligned16(q) || !aligned16(out)) return invalid("q and out need 16-byte aligned addresses");
  QD_TRY(check_stride(q_stride, 0, e, "q_stride"));
  QD_TRY(check_stride(q_head_stride, 0, e, "q_head_stride"));
  QD_TRY(check_stride(out_stride, c->rows > 1 ? c->head_dim : 0, e, "out_stride"));
  QD_TRY(check_stride(out_head_stride, heads > 1 ? c->head_dim : 0, e, "out_head_stride"));
  if (out == q && ((c->rows > 1 && out_stride != q_stride) || (heads > 1 && out_head_stride != q_head_stride)))
    return invalid("q in place needs one stride");
  return QD_SUCCESS;
}

qd_status check_attention_size(const qd_paged_cache *c, uint32_t heads, uint64_t positions) {
  const uint64_t parts = static_cast<uint64_t>(c->kv_heads) * ((heads / c->kv_heads + 15) / 16);
  // Tiles are counted in 31 bits, and a grid has fewer than 2^32 threads.
  if (c->rows * parts * (positions / 32 + 1) > 0x7f000000u || c->rows * parts > 0xffff00u)
    return refuse(QD_ERROR_NOT_SUPPORTED, "%u rows of up to %llu positions and %u heads are too much for one call", c->rows,
                  static_cast<unsigned long long>(positions), heads);
  return QD_SUCCESS;
}

// (An arrival counter for every row and KV head; a grid's second dimension.)
qd_status check_sparse(uint32_t rows, uint32_t heads, uint32_t kv_heads, uint32_t head_dim, uint32_t budget) {
  QD_TRY(check_heads(heads, kv_heads));
  QD_TRY(check_head_dim(head_dim));
  if (static_cast<uint64_t>(rows) * kv_heads > 65535)
    return refuse(QD_ERROR_NOT_SUPPORTED, "%u rows of %u KV heads: up to 65535 together", rows, kv_heads);
  if (budget == 0 || budget > (1u << 20)) return refuse(QD_ERROR_INVALID_ARGUMENT, "budget %u: from 1 to 2^20 pages", budget);
  return QD_SUCCESS;
}

}  // namespace

extern "C" {

qd_status qd_workspace_create(int32_t device, size_t bytes, qd_workspace **out) {
  if (!out) return invalid("null argument");
  *out = nullptr;
  if (bytes > (size_t(1) << 40)) return refuse(QD_ERROR_INVALID_ARGUMENT, "a workspace of %zu bytes", bytes);
  Device on;
  QD_TRY(on.enter(device));
  qd_workspace *w = new (std::nothrow) qd_workspace{device, nullptr, bytes};
  if (!w) return refuse(QD_ERROR_RUNTIME, "host allocation failed");
  void *p = nullptr;
  hipError_t e = hipMalloc(&p, qd::kOpCounterBytes + bytes);
  if (e == hipSuccess) {
    w->base = static_cast<char *>(p);
    e = qd::launch_op_clear(nullptr, static_cast<uint32_t *>(p), qd::kOpCounters);
    if (e == hipSuccess) e = hipStreamSynchronize(nullptr);
  }
  if (e != hipSuccess) {
    (void)hipGetLastError();
    if (p) (void)hipFree(p);
    delete w;
    return qd::report_hip(e, "workspace");
  }
  *out = w;
  return QD_SUCCESS;
}

qd_status qd_workspace_destroy(qd_workspace *w) {
  if (!w) return QD_SUCCESS;
  Device on;
  QD_TRY(on.enter(w->device));
  const hipError_t e = hipFree(w->base);
  delete w;
  return e == hipSuccess ? QD_SUCCESS : qd::report_hip(e, "hipFree");
}

qd_status qd_rope_table(double theta, uint32_t rotary_dim, uint32_t positions, double stretch, uint32_t original,
                        double fast, double slow, float *cos_table, float *sin_table) {
  if (!(theta > 0.0) || std::isinf(theta) || rotary_dim == 0 || rotary_dim % 2 != 0 || rotary_dim > 65536)
    return invalid("a positive theta and an even rotary_dim are needed");
  if (!(stretch >= 1.0) || std::isinf(stretch)) return invalid("stretch must be 1 or more");
  if (stretch > 1.0 && (original == 0 || !(fast > slow) || !(slow > 0.0)))
    return invalid("a stretched table needs the original length and fast > slow > 0");
  if (positions && (!cos_table || !sin_table)) return invalid("null table");
  const uint32_t half = rotary_dim / 2;
  const double two_pi = 6.283185307179586476925;
  const double size = stretch > 1.0 ? 0.1 * std::log(stretch) + 1.0 : 1.0;
  for (uint32_t i = 0; i < half; ++i) {
    double f = std::pow(theta, -2.0 * i / rotary_dim);
    if (stretch > 1.0) {
      const double turns = original * f / two_pi;
      const double keep = turns >= fast ? 1.0 : turns <= slow ? 0.0 : std::log(turns / slow) / std::log(fast / slow);
      f *= keep + (1.0 - keep) / stretch;
    }
    for (uint32_t p = 0; p < positions; ++p) {
      cos_table[static_cast<size_t>(p) * half + i] = static_cast<float>(std::cos(p * f) * size);
      sin_table[static_cast<size_t>(p) * half + i] = static_cast<float>(std::sin(p * f) * size);
    }
  }
  return QD_SUCCESS;
}

qd_status qd_paged_append(const qd_paged_cache *c, const qd_append_args *a, void *stream) {
  return qd_paged_append_at(c, a, nullptr, stream);
}

qd_status qd_paged_append_at(const qd_paged_cache *c, const qd_append_args *a, const int32_t *slots, void *stream) {
  QD_TRY(check_cache(c));
  if (!a) return invalid("null argument");
  const uint32_t e = element_bytes(c->dtype), dim = c->head_dim;
  if (a->q) QD_TRY(check_heads(a->heads, c->kv_heads));
  if (a->rotary_dim % 8 != 0 || a->rotary_dim > dim)
    return refuse(QD_ERROR_INVALID_ARGUMENT, "rotary_dim %u: a multiple of 8 up to head_dim %u is needed", a->rotary_dim, dim);
  // A grid has fewer than 2^32 threads: whole waves for each token, eight elements a lane.
  const uint64_t lanes = ((static_cast<uint64_t>(a->q ? a->heads : 0) + 2 * c->kv_heads) * (dim / 8) + 63) / 64 * 64;
  if (lanes * a->tokens > 0xffff0000ull) return refuse(QD_ERROR_NOT_SUPPORTED, "%u tokens are too many for one call", a->tokens);
  if (a->tokens) {
    if (!a->k || !a->v || !a->positions || (a->q && !a->q_out)) return invalid("null tensor");
    if (!aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) || !aligned16(a->q_out))
      return invalid("q, k, v and q_out need 16-byte aligned addresses");
    if (a->rotary_dim && (!a->cos_table || !a->sin_table || !aligned16(a->cos_table) || !aligned16(a->sin_table)))
      return invalid("rotary tables are needed, at 16-byte aligned addresses");
    if (a->q) {
      QD_TRY(check_stride(a->q_stride, 0, e, "q_stride"));
      QD_TRY(check_stride(a->q_out_stride, a->tokens > 1 ? static_cast<int64_t>(a->heads) * dim : 0, e, "q_out_stride"));
      if (a->q_out == a->q && a->tokens > 1 && a->q_out_stride != a->q_stride) return invalid("q in place needs one stride");
    }
    QD_TRY(check_stride(a->k_stride, 0, e, "k_stride"));
    QD_TRY(check_stride(a->v_stride, 0, e, "v_stride"));
  }
  Device on;
  QD_TRY(on.enter(c->device));
  return launched(qd::launch_paged_append(static_cast<hipStream_t>(stream), *c, *a, slots), "append launch");
}

qd_status qd_paged_attention_workspace(uint32_t rows, uint32_t heads, uint32_t kv_heads, uint32_t head_dim, size_t *bytes) {
  if (!bytes) return invalid("null argument");
  QD_TRY(check_heads(heads, kv_heads));
  if (head_dim != 64 && head_dim != 128) return refuse(QD_ERROR_NOT_SUPPORTED, "head_dim %u: the kernels take 64 and 128", head_dim);
  if (rows > (1u << 20)) return invalid("too many rows");
  *bytes = qd::paged_attention_scratch_most(rows, heads, kv_heads, head_dim);
  return QD_SUCCESS;
}

qd_status qd_paged_attention(const qd_paged_cache *c, const qd_attention_args *a, qd_workspace *w, void *stream) {
  QD_TRY(check_cache(c));
  if (!a) return invalid("null argument");
  QD_TRY(check_heads(a->heads, c->kv_heads));
  if (!std::isfinite(a->scale)) return invalid("scale must be finite");
  if (c->rows)
    QD_TRY(check_rows_of_heads(c, a->q, a->out, a->q_stride, a->q_head_stride, a->out_stride, a->out_head_stride, a->heads));
  QD_TRY(check_attention_size(c, a->heads, static_cast<uint64_t>(c->table_width) * c->page_size));
  qd::OpScratch scratch{};
  QD_TRY(check_workspace(w, c->device, qd::paged_attention_scratch(c->rows, a->heads, c->kv_heads, c->head_dim), &scratch));
  Device on;
  QD_TRY(on.enter(c->device));
  return launched(qd::launch_paged_attention(static_cast<hipStream_t>(stream), *c, *a, scratch), "attention launch");
}

qd_status qd_pages_fork_workspace(uint32_t rows, uint32_t pages, size_t *bytes) {
  if (!bytes) return invalid("null argument");
  if (rows > qd::kForkRows) return refuse(QD_ERROR_NOT_SUPPORTED, "%u rows: up to %u", rows, qd::kForkRows);
  *bytes = qd::pages_fork_scratch(rows, pages);
  return QD_SUCCESS;
}

qd_status qd_pages_fork(const qd_fork_args *a, qd_workspace *w, void *stream) {
  if (!a) return invalid("null argument");
  QD_TRY(check_page_size(a->page_size));
  if (a->rows > qd::kForkRows) return refuse(QD_ERROR_NOT_SUPPORTED, "%u rows: up to %u", a->rows, qd::kForkRows);
  if (a->pages > 0x7ffffff0u) return invalid("too many pages");
  if (a->append > (1u << 30) || static_cast<uint64_t>(a->table_width) * a->page_size > (1u << 30))
    return refuse(QD_ERROR_NOT_SUPPORTED, "rows of more than 2^30 positions");
  if (a->rows) {
    if (!a->table || !a->lengths || !a->table_out || !a->lengths_out || (a->pages && !a->refs)) return invalid("null tensor");
    if (a->table == a->table_out || a->lengths == a->lengths_out)
      return invalid("table_out and lengths_out must not be table and lengths");
    const int64_t width = a->table_width;
    if (a->table_stride < width || a->table_out_stride < width || a->table_stride > (int64_t(1) << 40) ||
        a->table_out_stride > (int64_t(1) << 40))
      return invalid("a table's stride is less than table_width");
  }
  if (a->memory_count > qd::kForkMemories || (a->memory_count && !a->memories))
    return refuse(QD_ERROR_INVALID_ARGUMENT, "up to %u memories", qd::kForkMemories);
  uint64_t pieces = 0;
  for (uint32_t m = 0; m < a->memory_count; ++m) {
    const qd_page_memory &p = a->memories[m];
    if (p.planes == 0 || p.bytes == 0) return invalid("a memory without planes or bytes");
    if (!p.base || !aligned16(p.base)) return invalid("a memory needs a 16-byte aligned address");
    if (p.bytes % 16 != 0 || p.page_stride % 16 != 0 || p.plane_stride % 16 != 0 || p.bytes > (uint64_t(1) << 40) ||
        p.page_stride < static_cast<int64_t>(p.bytes) || p.page_stride > (int64_t(1) << 40) || p.plane_stride < 0 ||
        p.plane_stride > (int64_t(1) << 45) || (p.planes > 1 && p.plane_stride < static_cast<int64_t>(p.bytes)))
      return invalid("a memory's bytes and strides: multiples of 16, strides of at least the bytes");
    pieces += (p.bytes / 16384 + 1) * p.planes;
  }
  if (pieces > 0x7fffffffu) return refuse(QD_ERROR_NOT_SUPPORTED, "pages of more than 2^31 pieces of 16 KiB");
  qd::OpScratch scratch{};
  QD_TRY(check_workspace(w, a->device, qd::pages_fork_scratch(a->rows, a->pages), &scratch));
  Device on;
  QD_TRY(on.enter(a->device));
  return launched(qd::launch_pages_fork(static_cast<hipStream_t>(stream), *a, scratch), "fork launch");
}

qd_status qd_beam_select_workspace(uint32_t groups, uint32_t beams, uint32_t k, uint32_t vocab, size_t *bytes) {
  if (!bytes) return invalid("null argument");
  QD_TRY(check_select(groups, beams, k, vocab));
  *bytes = qd::beam_select_scratch_most(groups, beams, k, vocab);
  return QD_SUCCESS;
}

qd_status qd_beam_select(const qd_select_args *a, qd_workspace *w, void *stream) {
  if (!a) return invalid("null argument");
  QD_TRY(check_dtype(a->dtype));
  QD_TRY(check_select(a->groups, a->beams, a->k, a->vocab));
  if (a->groups) {
    if (!a->logits || !a->scores || !a->scores_out || !a->parents || !a->tokens || (a->done && !a->done_out))
      return invalid("null tensor");
    if (a->scores_out == a->scores || (a->done && a->done_out == a->done))
      return invalid("scores_out and done_out must not be scores and done");
    if (reinterpret_cast<uintptr_t>(a->logits) % element_bytes(a->dtype) != 0) return invalid("misaligned logits");
    if (a->done && a->eos >= a->vocab) return refuse(QD_ERROR_INVALID_ARGUMENT, "eos %u >= vocab %u", a->eos, a->vocab);
    const int64_t most = int64_t(1) << 40;
    if (a->beam_stride < 0 || a->group_stride < 0 || a->beam_stride > most || a->group_stride > most)
      return invalid("the logits' strides must not be negative");
  }
  qd::OpScratch scratch{};
  QD_TRY(check_workspace(w, a->device, qd::beam_select_scratch(a->groups, a->beams, a->k, a->vocab), &scratch));
  Device on;
  QD_TRY(on.enter(a->device));
  return launched(qd::launch_beam_select(static_cast<hipStream_t>(stream), *a, scratch), "select launch");
}

qd_status qd_tree_attention_workspace(uint32_t rows, uint32_t nodes, uint32_t heads, uint32_t kv_heads, uint32_t head_dim,
                                      size_t *bytes) {
  if (!bytes) return invalid("null argument");
  QD_TRY(check_nodes(nodes));
  QD_TRY(check_heads(heads, kv_heads));
  QD_TRY(check_head_dim(head_dim));
  if (rows > (1u << 20)) return invalid("too many rows");
  *bytes = qd::tree_attention_scratch_most(rows, nodes, heads, kv_heads, head_dim);
  return QD_SUCCESS;
}

qd_status qd_tree_attention(const qd_paged_cache *c, const qd_tree_attention_args *a, qd_workspace *w, void *stream) {
  QD_TRY(check_cache(c));
  if (!a) return invalid("null argument");
  QD_TRY(check_nodes(a->nodes));
  QD_TRY(check_heads(a->heads, c->kv_heads));
  if (!std::isfinite(a->scale)) return invalid("scale must be finite");
  if (c->rows) {
    QD_TRY(check_rows_of_heads(c, a->q, a->out, a->q_stride, a->q_head_stride, a->out_stride, a->out_head_stride, a->heads));
    const uint32_t e = element_bytes(c->dtype);
    QD_TRY(check_stride(a->q_node_stride, 0, e, "q_node_stride"));
    QD_TRY(check_stride(a->out_node_stride, a->nodes > 1 ? c->head_dim : 0, e, "out_node_stride"));
    if (a->out == a->q && a->nodes > 1 && a->out_node_stride != a->q_node_stride) return invalid("q in place needs one stride");
    if (!a->parents) return invalid("null parents");
  }
  // A grid has fewer than 2^32 threads, 512 of a workgroup; a block has 16 columns or more.
  const uint64_t parts = static_cast<uint64_t>(c->kv_heads) * ((static_cast<uint64_t>(a->heads / c->kv_heads) * a->nodes + 63) / 64);
  if (c->rows * parts > 0x3f0000u)
    return refuse(QD_ERROR_NOT_SUPPORTED, "%u rows of %u nodes and %u heads are too much for one call", c->rows, a->nodes, a->heads);
  qd::OpScratch scratch{};
  QD_TRY(check_workspace(w, c->device, qd::tree_attention_scratch(c->dtype, c->rows, a->nodes, a->heads, c->kv_heads, c->head_dim), &scratch));
  Device on;
  QD_TRY(on.enter(c->device));
  return launched(qd::launch_tree_attention(static_cast<hipStream_t>(stream), *c, *a, scratch), "tree attention launch");
}

qd_status qd_tree_accept_workspace(uint32_t rows, uint32_t nodes, uint32_t vocab, size_t *bytes) {
  if (!bytes) return invalid("null argument");
  QD_TRY(check_accept(rows, nodes, vocab));
  *bytes = qd::tree_accept_scratch(rows, nodes);
  return QD_SUCCESS;
}

qd_status qd_tree_accept(const qd_accept_args *a, qd_workspace *w, void *stream) {
  if (!a) return invalid("null argument");
  QD_TRY(check_dtype(a->dtype));
  QD_TRY(check_accept(a->rows, a->nodes, a->vocab));
  if (a->rows) {
    if (!a->logits || !a->tokens || !a->parents || !a->path || !a->counts || !a->next_tokens) return invalid("null tensor");
    // (Rows that are done write theirs while others still read.)
    const uint64_t rows = a->rows, all = rows * a->nodes;
    for (const void *read : {static_cast<const void *>(a->tokens), static_cast<const void *>(a->parents), static_cast<const void *>(a->draws)}) {
      if (overlap(a->path, all, read, all)) return invalid("path must not be tokens or parents or draws, nor overlap them");
      // (Of trees of one node a row's token is read where the next one is written.)
      const bool own = a->nodes == 1 && read == a->tokens && a->next_tokens == a->tokens;
      if (overlap(a->counts, rows, read, all) || (!own && overlap(a->next_tokens, rows, read, all)))
        return invalid("counts and next_tokens must not overlap tokens, parents or draws");
    }
    if (overlap(a->path, all, a->counts, rows) || overlap(a->path, all, a->next_tokens, rows) || overlap(a->counts, rows, a->next_tokens, rows))
      return invalid("path, counts and next_tokens must not overlap");
    if (reinterpret_cast<uintptr_t>(a->logits) % element_bytes(a->dtype) != 0) return invalid("misaligned logits");
    const int64_t most = int64_t(1) << 40;
    if (a->row_stride < 0 || a->node_stride < 0 || a->row_stride > most || a->node_stride > most)
      return invalid("the logits' strides must not be negative");
    if (a->draws && !(a->temperature >= 1e-6f && a->temperature <= 1e6f)) return invalid("a temperature from 1e-6 to 1e6 is needed");
  }
  qd::OpScratch scratch{};
  QD_TRY(check_workspace(w, a->device, qd::tree_accept_scratch(a->rows, a->nodes), &scratch));
  Device on;
  QD_TRY(on.enter(a->device));
  return launched(qd::launch_tree_accept(static_cast<hipStream_t>(stream), *a, scratch), "accept launch");
}

qd_status qd_tree_commit(const qd_commit_args *a, void *stream) {
  if (!a) return invalid("null argument");
  QD_TRY(check_page_size(a->page_size));
  QD_TRY(check_nodes(a->nodes));
  if (a->rows > 65535) return refuse(QD_ERROR_NOT_SUPPORTED, "%u rows: up to 65535", a->rows);
  if (a->pages > 0x7fffffffu) return invalid("too many pages");
  if (static_cast<uint64_t>(a->table_width) * a->page_size > (1u << 30))
    return refuse(QD_ERROR_NOT_SUPPORTED, "rows of more than 2^30 positions");
  if (a->rows) {
    if (!a->table || !a->lengths || !a->path || !a->counts || !a->lengths_out) return invalid("null tensor");
    if (a->table_stride < static_cast<int64_t>(a->table_width) || a->table_stride > (int64_t(1) << 40))
      return invalid("table_stride is less than table_width");
  }
  if (a->memory_count > qd::kForkMemories || (a->memory_count && !a->memories))
    return refuse(QD_ERROR_INVALID_ARGUMENT, "up to %u memories", qd::kForkMemories);
  uint64_t columns = 0;
  for (uint32_t m = 0; m < a->memory_count; ++m) {
    const qd_token_memory &p = a->memories[m];
    const int64_t most = int64_t(1) << 45;
    if (p.planes == 0 || p.pieces == 0 || p.piece_bytes == 0) return invalid("a memory without planes, pieces or bytes");
    if (!p.base || !aligned16(p.base)) return invalid("a memory needs a 16-byte aligned address");
    if (p.piece_bytes % 16 != 0 || p.plane_stride % 16 != 0 || p.page_stride % 16 != 0 || p.token_stride % 16 != 0 ||
        p.piece_stride % 16 != 0 || p.plane_stride < 0 || p.plane_stride > most || p.page_stride < 0 || p.page_stride > most ||
        p.token_stride < static_cast<int64_t>(p.piece_bytes) || p.token_stride > most || p.piece_stride < 0 || p.piece_stride > most ||
        (p.pieces > 1 && p.piece_stride < static_cast<int64_t>(p.piece_bytes)) ||
        (a->pages > 1 && p.page_stride < static_cast<int64_t>(p.piece_bytes)) ||
        (p.planes > 1 && p.plane_stride < static_cast<int64_t>(p.piece_bytes)))
      return invalid("a memory's bytes and strides: multiples of 16, strides of at least the bytes");
    const uint64_t row = static_cast<uint64_t>(p.piece_bytes / 16) * p.pieces;
    if (row > 0x7fffffffu || row * p.planes > 0x7fffffffu) return refuse(QD_ERROR_NOT_SUPPORTED, "positions of more than 2^35 bytes");
    columns += row * p.planes;
  }
  // A grid has fewer than 2^32 threads, 256 for 64 columns.
  if ((columns / 64 + 1) * a->rows > 0xff0000u) return refuse(QD_ERROR_NOT_SUPPORTED, "%u rows are too much for one call", a->rows);
  // (A row's first workgroup writes its length while the others still read the rest.)
  if (overlap(a->lengths_out, a->rows, a->lengths, a->rows) || overlap(a->lengths_out, a->rows, a->counts, a->rows) ||
      overlap(a->lengths_out, a->rows, a->path, static_cast<uint64_t>(a->rows) * a->nodes) ||
      overlap(a->lengths_out, a->rows, a->table, a->table_width, a->rows, a->table_stride))
    return invalid("lengths_out must not be lengths, counts, path or table, nor overlap them");
  Device on;
  QD_TRY(on.enter(a->device));
  return launched(qd::launch_tree_commit(static_cast<hipStream_t>(stream), *a), "commit launch");
}

qd_status qd_page_bounds(const qd_paged_cache *c, void *bounds, uint32_t recent, void *stream) {
  QD_TRY(check_cache(c));
  if (c->rows && c->pages && (!bounds || !aligned16(bounds))) return invalid("bounds need a 16-byte aligned address");
  const uint64_t each = std::min<uint64_t>(c->table_width, (static_cast<uint64_t>(recent) + c->page_size - 2) / c->page_size + 1);
  // A grid has fewer than 2^32 threads, 256 for a page.
  if (each * c->rows > 0xff0000u || each * c->rows * c->kv_heads > 0xff0000u)
    return refuse(QD_ERROR_NOT_SUPPORTED, "%u rows of %llu pages are too much for one call", c->rows, static_cast<unsigned long long>(each));
  Device on;
  QD_TRY(on.enter(c->device));
  return launched(qd::launch_page_bounds(static_cast<hipStream_t>(stream), *c, bounds, recent), "bounds launch");
}

qd_status qd_sparse_attention_workspace(uint32_t rows, uint32_t heads, uint32_t kv_heads, uint32_t head_dim, uint32_t table_width,
                                        uint32_t budget, size_t *bytes) {
  if (!bytes) return invalid("null argument");
  QD_TRY(check_sparse(rows, heads, kv_heads, head_dim, budget));
  if (table_width > (1u << 26)) return invalid("too wide a table");
  *bytes = qd::sparse_attention_scratch_most(rows, heads, kv_heads, head_dim, table_width, budget);
  return QD_SUCCESS;
}

qd_status qd_sparse_attention(const qd_paged_cache *c, const qd_sparse_args *a, qd_workspace *w, void *stream) {
  QD_TRY(check_cache(c));
  if (!a) return invalid("null argument");
  QD_TRY(check_sparse(c->rows, a->heads, c->kv_heads, c->head_dim, a->budget));
  if (a->last == 0 || a->first > a->budget || a->last > a->budget - a->first)
    return refuse(QD_ERROR_INVALID_ARGUMENT, "first %u and last %u (1 at least): up to the budget, %u", a->first, a->last, a->budget);
  if (!std::isfinite(a->scale)) return invalid("scale must be finite");
  if (c->rows) {
    QD_TRY(check_rows_of_heads(c, a->q, a->out, a->q_stride, a->q_head_stride, a->out_stride, a->out_head_stride, a->heads));
    if (c->pages && (!a->bounds || !aligned16(a->bounds))) return invalid("bounds need a 16-byte aligned address");
    // (One row's list is written while another's table is read.)
    const uint64_t listed = static_cast<uint64_t>(c->rows) * c->kv_heads * a->budget;
    if (overlap(a->chosen, listed, c->table, c->table_width, c->rows, c->table_stride) || overlap(a->chosen, listed, c->lengths, c->rows))
      return invalid("chosen must not overlap the table or the lengths");
  }
  const uint64_t positions = static_cast<uint64_t>(a->budget) * c->page_size;
  if (positions > (1u << 30)) return refuse(QD_ERROR_NOT_SUPPORTED, "a budget of more than 2^30 positions");
  QD_TRY(check_attention_size(c, a->heads, positions));
  qd::OpScratch scratch{};
  QD_TRY(check_workspace(w, c->device, qd::sparse_attention_scratch(c->rows, a->heads, c->kv_heads, c->head_dim, c->table_width, a->budget),
                         &scratch));
  Device on;
  QD_TRY(on.enter(c->device));
  return launched(qd::launch_sparse_attention(static_cast<hipStream_t>(stream), *c, *a, scratch), "sparse attention launch");
}

}  // extern "C"
