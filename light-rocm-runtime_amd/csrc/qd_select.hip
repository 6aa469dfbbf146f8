// Beam selection for gfx950: the best k of beams x vocabulary. Declared in
// include/qd/qd_operators.h.
//
// A workgroup takes a slice of a row's logits into registers in one pass and
// leaves its maximum, its sum of exponentials and its best k as sorted keys; the
// last slice of a row to arrive joins them into the row's best k with their
// scores; the last row of a group to arrive chooses among its beams'. Bound by
// reading the logits for many rows, by the two hand-overs for few.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "qd_attention.hpp"
#include "qd_device.hpp"
#include "qd_device_math.hpp"
#include "qd_operators.hpp"

namespace qd {
namespace {

using namespace dev;

constexpr int kT = kBlock;
constexpr int kJoin = 2048;   // keys that one row's slices, or one group's rows, hand over at most
constexpr int kShort = 1024;  // keys that are put in order; beyond, the slower ways below
constexpr uint32_t kLowest = 0x00800000u;  // the order of the lowest finite number

struct SelectLaunch {
  qd_select_args a;
  uint32_t slices;      // of a row
  uint64_t *keys;       // [rows][slices][k]
  double *sums;         // [rows][slices]
  float *maxima;        // [rows][slices]
  double *row_score;    // [rows][k]
  uint32_t *row_token;  // [rows][k]
  uint32_t *row_count;  // arrivals [rows]
  uint32_t *group_count;
};

// A key orders a row's continuations: the higher logit first, then the lower
// token. The high word is the logit's bits, monotone; 0 is no key.
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint64_t key) {
  const uint32_t u = static_cast<uint32_t>(key >> 32);
  return __uint_as_float(u & 0x80000000u ? u & 0x7FFFFFFFu : ~u);
}
__device__ __forceinline__ uint64_t key_of(float x, uint32_t token) {
  return static_cast<uint64_t>(order_of(x)) << 32 | ~token;
}
__device__ __forceinline__ uint32_t token_of(uint64_t key) { return ~static_cast<uint32_t>(key); }

__device__ __forceinline__ void wait_vm_stores() { __builtin_amdgcn_s_waitcnt(0x0F70); }

__device__ __forceinline__ uint64_t load64(const Coherent &c, uint32_t i) {
  return c.ldu(2 * i) | static_cast<uint64_t>(c.ldu(2 * i + 1)) << 32;
}
__device__ __forceinline__ void store64(const Coherent &c, uint32_t i, uint64_t v) {
  c.stu(2 * i, static_cast<uint32_t>(v));
  c.stu(2 * i + 1, static_cast<uint32_t>(v >> 32));
}

// Logits' types: FP32, or 16 bits whose values are FP32 ones.
template <typename E>
__device__ __forceinline__ float widen(uint32_t bits) {
  if constexpr (std::is_same_v<E, float>)
    return __uint_as_float(bits);
  else if constexpr (std::is_same_v<E, Bf16>)
    return __uint_as_float(bits << 16);
  else
    return half_lo(bits);
}
// 16 bytes at any element's address.
typedef uint32_t Words4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t Words2 __attribute__((ext_vector_type(4), aligned(2)));
template <typename E>
struct Piece {
  static constexpr int kElems = 16 / sizeof(E);
  using words = std::conditional_t<sizeof(E) == 4, Words4, Words2>;
};

struct Shared {
  uint64_t list[kJoin];
  uint64_t shorter[kShort];
  double sum[kWavesPerBlock];
  float top[kWavesPerBlock];
  uint32_t bound[kWavesPerBlock];
  uint32_t n, last;
};

// A lower bound of the order of the workgroup's k-th best, from each thread's
// best: the k-th best lane of a wave has k as good before or at it. (The last 12
// bits are left zero.) Between barriers.
__device__ __forceinline__ uint32_t wave_bound(uint32_t best, uint32_t k) {
  uint32_t t = 0;
#pragma unroll
  for (int bit = 31; bit >= 12; --bit) {
    const uint32_t with = t | 1u << bit;
    if (static_cast<uint32_t>(__popcll(__ballot(best >= with))) >= k) t = with;
  }
  return t;
}

// The best k of n keys in `from`, in order, through put(rank, key).
template <typename Put>
__device__ __forceinline__ void put_in_order(const uint64_t *from, uint32_t n, uint32_t k, Put put) {
  for (uint32_t i = threadIdx.x; i < n; i += kT) {
    const uint64_t key = from[i];
    uint32_t rank = 0;
    for (uint32_t j = 0; j < n; ++j) rank += from[j] > key;
    if (rank < k) put(rank, key);
  }
}

// Chooses among a group's rows; called by the workgroup that arrives last.
__device__ void choose(const SelectLaunch &p, uint32_t group, Shared &sh) {
  const uint32_t k = p.a.k, n = p.a.beams * k;
  const uint32_t row0 = group * p.a.beams;
  const Coherent scores(p.row_score + static_cast<size_t>(row0) * k, n * 8);
  const Coherent tokens(p.row_token + static_cast<size_t>(row0) * k, n * 4);
  double *list = reinterpret_cast<double *>(sh.list);
  __shared__ uint32_t flat_beam[kSelectK], flat_token[kSelectK];
  __shared__ uint8_t taken[2 * kSelectK];
  if (threadIdx.x == 0) sh.n = 0;
  __syncthreads();
  uint32_t mine = 0;
  for (uint32_t i = threadIdx.x; i < n; i += kT) {
    list[i] = __longlong_as_double(static_cast<long long>(load64(scores, i)));
    mine += list[i] != -INFINITY;
  }
  if (mine) atomicAdd(&sh.n, mine);
  __syncthreads();
  const uint32_t found = min(sh.n, k);
  auto put = [&](uint32_t i, double score, uint32_t beam, uint32_t token) {
    const size_t at = static_cast<size_t>(group) * k + i;
    p.a.scores_out[at] = static_cast<float>(score);
    p.a.parents[at] = static_cast<int32_t>(row0 + beam);
    p.a.tokens[at] = static_cast<int32_t>(token);
    if (p.a.done) p.a.done_out[at] = p.a.done[row0 + beam] != 0 || token == p.a.eos;
  };
  for (uint32_t i = threadIdx.x; i < n; i += kT) {
    const double s = list[i];
    if (s == -INFINITY) continue;
    uint32_t rank = 0;
    for (uint32_t j = 0; j < n; ++j) rank += list[j] > s || (list[j] == s && j < i);
    if (rank >= k) continue;
    const uint32_t token = tokens.ldu(i);
    put(rank, s, i / k, token);
    flat_beam[rank] = i / k;
    flat_token[rank] = token;
  }
  if (found == k) return;
  // The places left go to the lowest (beam, token) that have none.
  __syncthreads();
  const uint64_t all = static_cast<uint64_t>(p.a.beams) * p.a.vocab;
  const uint32_t t = threadIdx.x;
  if (t < 2 * kSelectK) {
    bool is = t >= all;
    for (uint32_t j = 0; j < found; ++j) is |= flat_beam[j] == t / p.a.vocab && flat_token[j] == t % p.a.vocab;
    taken[t] = is;
  }
  __syncthreads();
  if (t < 2 * kSelectK && !taken[t]) {
    uint32_t at = found;
    for (uint32_t j = 0; j < t; ++j) at += !taken[j];
    if (at < k) put(at, -INFINITY, t / p.a.vocab, t % p.a.vocab);
  }
}

// Joins a row's slices; called by the workgroup that arrives last.
__device__ void join_row(const SelectLaunch &p, uint32_t row, Shared &sh) {
  const uint32_t k = p.a.k, n = p.slices * k;
  const Coherent keys(p.keys + static_cast<size_t>(row) * n, n * 8);
  const Coherent sums(p.sums + static_cast<size_t>(row) * p.slices, p.slices * 8);
  const Coherent maxima(p.maxima + static_cast<size_t>(row) * p.slices, p.slices * 4);
  const Coherent scores(p.row_score + static_cast<size_t>(row) * k, k * 8);
  const Coherent tokens(p.row_token + static_cast<size_t>(row) * k, k * 4);
  float m = -INFINITY;
  for (uint32_t s = threadIdx.x; s < p.slices; s += kT) m = fmaxf(m, maxima.ld(s));
  m = wave_max(m);
  uint32_t best = 0;
  for (uint32_t i = threadIdx.x; i < n; i += kT) {
    sh.list[i] = load64(keys, i);
    best = max(best, static_cast<uint32_t>(sh.list[i] >> 32));
  }
  const uint32_t bound = wave_bound(best, k);
  if (lane_id() == 0) {
    sh.top[wave_id()] = m;
    sh.bound[wave_id()] = bound;
  }
  if (threadIdx.x == 0) sh.n = 0;
  __syncthreads();
  uint32_t least = kLowest;
#pragma unroll
  for (int w = 0; w < kWavesPerBlock; ++w) {
    m = fmaxf(m, sh.top[w]);
    least = max(least, sh.bound[w]);
  }
  double sum = 0.0;
  for (uint32_t s = threadIdx.x; s < p.slices; s += kT) {
    const float top = maxima.ld(s);
    const double part = __longlong_as_double(static_cast<long long>(load64(sums, s)));
    sum += top == m ? part : top == -INFINITY ? 0.0 : part * exp(static_cast<double>(top) - m);
  }
#pragma unroll
  for (int o = kWave / 2; o > 0; o >>= 1) sum += __shfl_xor(sum, o, kWave);
  if (lane_id() == 0) sh.sum[wave_id()] = sum;
  for (uint32_t i = threadIdx.x; i < n; i += kT)
    if (static_cast<uint32_t>(sh.list[i] >> 32) >= least) {
      const uint32_t at = atomicAdd(&sh.n, 1u);
      if (at < kShort) sh.shorter[at] = sh.list[i];
    }
  __syncthreads();
  const double total = (sh.sum[0] + sh.sum[1]) + (sh.sum[2] + sh.sum[3]);
  const double base = static_cast<double>(p.a.scores[row]), log_total = log(total);
  auto put = [&](uint32_t rank, uint64_t key) {
    const float x = logit_of(key);
    // (An infinite maximum leaves the others nothing.)
    const double s = key == 0 ? -INFINITY : base + ((x == m ? 0.0 : static_cast<double>(x) - m) - log_total);
    store64(scores, rank, static_cast<uint64_t>(__double_as_longlong(s)));
    tokens.stu(rank, token_of(key));
  };
  const uint32_t count = sh.n;
  if (count <= static_cast<uint32_t>(kShort)) {
    put_in_order(sh.shorter, count, k, put);
    for (uint32_t i = count + threadIdx.x; i < k; i += kT) put(i, 0);
  } else {
    put_in_order(sh.list, n, k, put);  // more than k keys are there: every place is filled
  }
}

// What is left of a row's way once its scores are stored.
__device__ __forceinline__ void row_done(const SelectLaunch &p, uint32_t row, Shared &sh) {
  const uint32_t group = row / p.a.beams;
  wait_vm_stores();
  __syncthreads();
  if (threadIdx.x == 0) {
    sh.last = p.a.beams == 1 || atomicAdd(p.group_count + group, 1u) == p.a.beams - 1;
    if (sh.last && p.a.beams > 1) p.group_count[group] = 0u;
  }
  __syncthreads();
  if (sh.last) choose(p, group, sh);
}

template <typename E, int kEach>
__global__ __launch_bounds__(kT) void select_kernel(SelectLaunch p) {
  using P = Piece<E>;
  constexpr int kPieces = kEach / P::kElems;
  __shared__ Shared sh;
  const uint32_t row = blockIdx.y, slice = blockIdx.x, k = p.a.k;
  const float score = p.a.scores[row];
  const bool live = fabsf(score) < INFINITY;
  const bool done = p.a.done && p.a.done[row];
  if (!live || done) {
    // No logits are read: one continuation, or none.
    if (slice) return;
    const Coherent scores(p.row_score + static_cast<size_t>(row) * k, k * 8);
    const Coherent tokens(p.row_token + static_cast<size_t>(row) * k, k * 4);
    for (uint32_t i = threadIdx.x; i < k; i += kT) {
      const double s = live && i == 0 ? static_cast<double>(score) : -INFINITY;
      store64(scores, i, static_cast<uint64_t>(__double_as_longlong(s)));
      tokens.stu(i, p.a.eos);
    }
    row_done(p, row, sh);
    return;
  }
  const E *logits = static_cast<const E *>(p.a.logits) + static_cast<int64_t>(row / p.a.beams) * p.a.group_stride +
                    static_cast<int64_t>(row % p.a.beams) * p.a.beam_stride;
  const uint32_t first = slice * (kT * kEach) + threadIdx.x * P::kElems;
  float x[kEach];
#pragma unroll
  for (int j = 0; j < kPieces; ++j) {
    const uint32_t at = first + j * (kT * P::kElems);
    typename P::words v = {0u, 0u, 0u, 0u};
    const bool whole = at + P::kElems <= p.a.vocab;
    if (whole) v = *reinterpret_cast<const typename P::words *>(logits + at);
#pragma unroll
    for (int c = 0; c < P::kElems; ++c) {
      uint32_t bits;
      if constexpr (sizeof(E) == 4)
        bits = v[c];
      else
        bits = c & 1 ? v[c >> 1] >> 16 : v[c >> 1] & 0xFFFFu;
      float y = widen<E>(bits);
      if (!whole) {
        y = -INFINITY;
        if (at + c < p.a.vocab) {
          if constexpr (sizeof(E) == 4)
            y = reinterpret_cast<const float *>(logits)[at + c];
          else
            y = widen<E>(reinterpret_cast<const uint16_t *>(logits)[at + c]);
        }
      }
      x[j * P::kElems + c] = y != y ? -INFINITY : y + 0.f;  // (+0 for -0, which is no lower)
    }
  }
  float top = x[0];
#pragma unroll
  for (int i = 1; i < kEach; ++i) top = fmaxf(top, x[i]);
  const uint32_t bound = wave_bound(order_of(top), k);
  const float wave_top = wave_max(top);
  if (lane_id() == 0) {
    sh.top[wave_id()] = wave_top;
    sh.bound[wave_id()] = bound;
  }
  if (threadIdx.x == 0) sh.n = 0;
  __syncthreads();
  float m = sh.top[0];
  uint32_t least = max(kLowest, sh.bound[0]);
#pragma unroll
  for (int w = 1; w < kWavesPerBlock; ++w) {
    m = fmaxf(m, sh.top[w]);
    least = max(least, sh.bound[w]);
  }
  // Sum of exp(x - m): FP32 within a thread, 64 bits beyond. The difference is
  // exact to half a step, so the sum has no error common to its terms.
  float part = 0.f;
  if (fabsf(m) < INFINITY) {
#pragma unroll
    for (int i = 0; i < kEach; ++i) part += exp2_fast((x[i] - m) * 1.44269504088896340736f);
  } else if (m > 0) {
#pragma unroll
    for (int i = 0; i < kEach; ++i) part += x[i] == m ? 1.f : 0.f;
  }
  double sum = part;
#pragma unroll
  for (int o = kWave / 2; o > 0; o >>= 1) sum += __shfl_xor(sum, o, kWave);
  if (lane_id() == 0) sh.sum[wave_id()] = sum;
  if (order_of(top) >= least) {
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      if (order_of(x[i]) >= least) {
        const uint32_t at = atomicAdd(&sh.n, 1u);
        if (at < kShort)
          sh.shorter[at] = key_of(x[i], first + (i / P::kElems) * (kT * P::kElems) + i % P::kElems);
      }
  }
  __syncthreads();
  const uint32_t n = p.slices * k;
  const Coherent keys(p.keys + static_cast<size_t>(row) * n, n * 8);
  const uint32_t count = sh.n;
  auto put = [&](uint32_t rank, uint64_t key) { store64(keys, slice * k + rank, key); };
  if (count <= static_cast<uint32_t>(kShort)) {
    put_in_order(sh.shorter, count, k, put);
    for (uint32_t i = count + threadIdx.x; i < k; i += kT) put(i, 0);
  } else {
    // Many equal or nearly equal logits: one after the other.
    uint64_t before = ~0ull;
    for (uint32_t rank = 0; rank < k; ++rank) {
      uint64_t best = 0;
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const uint64_t key =
            x[i] == -INFINITY ? 0 : key_of(x[i], first + (i / P::kElems) * (kT * P::kElems) + i % P::kElems);
        if (key < before && key > best) best = key;
      }
#pragma unroll
      for (int o = kWave / 2; o > 0; o >>= 1) {
        const uint64_t other = __shfl_xor(static_cast<unsigned long long>(best), o, kWave);
        best = other > best ? other : best;
      }
      if (lane_id() == 0) sh.list[wave_id()] = best;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kWavesPerBlock; ++w) best = sh.list[w] > best ? sh.list[w] : best;
      __syncthreads();
      if (threadIdx.x == 0) put(rank, best);
      before = best;
    }
  }
  if (threadIdx.x == 0) {
    const Coherent sums(p.sums + static_cast<size_t>(row) * p.slices, p.slices * 8);
    const Coherent maxima(p.maxima + static_cast<size_t>(row) * p.slices, p.slices * 4);
    store64(sums, slice, static_cast<uint64_t>(__double_as_longlong((sh.sum[0] + sh.sum[1]) + (sh.sum[2] + sh.sum[3]))));
    maxima.st(slice, m);
  }
  wait_vm_stores();
  __syncthreads();
  if (threadIdx.x == 0) {
    sh.last = p.slices == 1 || atomicAdd(p.row_count + row, 1u) == p.slices - 1;
    if (sh.last && p.slices > 1) p.row_count[row] = 0u;
  }
  __syncthreads();
  if (!sh.last) return;
  join_row(p, row, sh);
  row_done(p, row, sh);
}

// Logits of a thread: 32 where slices of that size give every CU two or more,
// else 8, as long as the slices' candidates fit the join.
constexpr uint32_t kWideSlice = kT * 32, kNarrowSlice = kT * 8;
uint32_t slices_of(uint32_t vocab, uint32_t slice) { return (vocab + slice - 1) / slice; }
bool wide_slices(uint32_t rows, uint32_t k, uint32_t vocab) {
  return static_cast<uint64_t>(slices_of(vocab, kWideSlice)) * rows >= 512 ||
         static_cast<uint64_t>(slices_of(vocab, kNarrowSlice)) * k > kJoin;
}

template <typename... A>
hipError_t launch(void (*kernel)(A...), dim3 grid, dim3 block, hipStream_t s, A... args) {
  void *packed[] = {&args...};
  return hipLaunchKernel(reinterpret_cast<const void *>(kernel), grid, block, packed, 0, s);
}

size_t round256(size_t n) { return (n + 255) / 256 * 256; }

// The scratch regions from `base` on (nullptr: the size only).
size_t carve(SelectLaunch &p, char *base, uint32_t rows, uint32_t k) {
  size_t used = 0;
  auto take = [&](size_t bytes) {
    char *r = base ? base + used : nullptr;
    used += round256(bytes);
    return r;
  };
  const size_t parts = static_cast<size_t>(rows) * p.slices;
  p.keys = reinterpret_cast<uint64_t *>(take(parts * k * 8));
  p.sums = reinterpret_cast<double *>(take(parts * 8));
  p.maxima = reinterpret_cast<float *>(take(parts * 4));
  p.row_score = reinterpret_cast<double *>(take(static_cast<size_t>(rows) * k * 8));
  p.row_token = reinterpret_cast<uint32_t *>(take(static_cast<size_t>(rows) * k * 4));
  return used;
}

}  // namespace

bool beam_select_fits(uint32_t k, uint32_t vocab) {
  return static_cast<uint64_t>(slices_of(vocab, kWideSlice)) * k <= kJoin;
}

size_t beam_select_scratch(uint32_t groups, uint32_t beams, uint32_t k, uint32_t vocab) {
  const uint32_t rows = groups * beams;
  SelectLaunch p{};
  p.slices = slices_of(vocab, wide_slices(rows, k, vocab) ? kWideSlice : kNarrowSlice);
  return carve(p, nullptr, rows, k);
}

hipError_t launch_beam_select(hipStream_t s, const qd_select_args &a, const OpScratch &w) {
  const uint32_t rows = a.groups * a.beams;
  if (rows == 0) return hipSuccess;
  const bool wide = wide_slices(rows, a.k, a.vocab);
  SelectLaunch p{};
  p.a = a;
  p.slices = slices_of(a.vocab, wide ? kWideSlice : kNarrowSlice);
  carve(p, w.scratch, rows, a.k);
  p.row_count = w.counters;
  p.group_count = w.counters + rows;
  const dim3 grid(p.slices, rows), block(kT);
  switch (a.dtype) {
    case QD_DTYPE_F32: return launch(wide ? select_kernel<float, 32> : select_kernel<float, 8>, grid, block, s, p);
    case QD_DTYPE_BF16: return launch(wide ? select_kernel<Bf16, 32> : select_kernel<Bf16, 8>, grid, block, s, p);
    default: return launch(wide ? select_kernel<F16, 32> : select_kernel<F16, 8>, grid, block, s, p);
  }
}

}  // namespace qd
