// C ABI of the operators on the caller's device memory
// (include/qd/qd_operators.h): argument checks, the workspace, and the rotary
// tables. Nothing here throws; every refusal happens before any device work.
#include "qd/qd_operators.h"

#include <hip/hip_runtime.h>

#include <atomic>
#include <cmath>
#include <cstdarg>
#include <cstdio>
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
  return launched(qd::launch_paged_append(static_cast<hipStream_t>(stream), *c, *a), "append launch");
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
  const uint32_t e = element_bytes(c->dtype);
  if (c->rows) {
    if (!a->q || !a->out) return invalid("null tensor");
    if (!aligned16(a->q) || !aligned16(a->out)) return invalid("q and out need 16-byte aligned addresses");
    QD_TRY(check_stride(a->q_stride, 0, e, "q_stride"));
    QD_TRY(check_stride(a->q_head_stride, 0, e, "q_head_stride"));
    QD_TRY(check_stride(a->out_stride, c->rows > 1 ? c->head_dim : 0, e, "out_stride"));
    QD_TRY(check_stride(a->out_head_stride, a->heads > 1 ? c->head_dim : 0, e, "out_head_stride"));
    if (a->out == a->q && ((c->rows > 1 && a->out_stride != a->q_stride) ||
                           (a->heads > 1 && a->out_head_stride != a->q_head_stride)))
      return invalid("q in place needs one stride");
  }
  const uint64_t parts = static_cast<uint64_t>(c->kv_heads) * ((a->heads / c->kv_heads + 15) / 16);
  // Tiles are counted in 31 bits, and a grid has fewer than 2^32 threads.
  if (c->rows * parts * (static_cast<uint64_t>(c->table_width) * c->page_size / 32 + 1) > 0x7f000000u ||
      c->rows * parts > 0xffff00u)
    return refuse(QD_ERROR_NOT_SUPPORTED, "%u rows of up to %llu positions and %u heads are too much for one call", c->rows,
                  static_cast<unsigned long long>(static_cast<uint64_t>(c->table_width) * c->page_size), a->heads);
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

}  // extern "C"
