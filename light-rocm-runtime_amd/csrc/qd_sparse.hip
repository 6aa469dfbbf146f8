// Attention over chosen pages for gfx950: bounds of the keys in each page, the choice
// by them, and the attention of qd_paged.hip over what was chosen. Declared in
// include/qd/qd_operators.h.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "qd_device.hpp"
#include "qd_device_math.hpp"
#include "qd_operators.hpp"
#include "qd_paged.hpp"

namespace qd {
namespace {

using namespace dev;

// Values of 16 bytes.
template <typename E>
constexpr int kPer = std::is_same_v<E, float> ? 4 : 8;
template <typename E>
__device__ __forceinline__ void widen(const u4v &v, float (&y)[kPer<E>]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t word = v[i];
    if constexpr (std::is_same_v<E, float>) {
      y[i] = __uint_as_float(word);
    } else {
      y[2 * i] = E::lo(word);
      y[2 * i + 1] = E::hi(word);
    }
  }
}
__device__ __forceinline__ float from_lane(float v, int lane) {
  return __builtin_bit_cast(float, __builtin_amdgcn_ds_bpermute(lane << 2, __builtin_bit_cast(int, v)));
}

// ---- bounds -------------------------------------------------------------------------
// kWaves waves take one page of one KV head: a lane 16 bytes of a key, the lanes of a wave
// 1 KB of keys at a time, the waves every so many keys; the lanes at one element together at
// the end. The least and largest values are keys' own elements: nothing is rounded. Bound by memory
// for prompts (7 of 9,001 to 20,000, 2 heads of 64 in FP32, pages of 16, 58 MB, 10.3 us: 5.6 TB/s), by
// the chain length, page, keys for a step (64 rows, 8 heads of 128 in BF16, pages of 64, 4.2 us).
constexpr int kBoundsT = 256;
struct BoundsLaunch {
  qd_paged_cache c;
  void *bounds;
  uint32_t recent;
  uint32_t page_shift;
  uint32_t each;   // pages of a row in the grid
  uint32_t units;  // rows x each x KV heads
};

template <typename E, int D, int kWaves>
__global__ __launch_bounds__(kBoundsT) void bounds_kernel(BoundsLaunch p) {
  constexpr int kP = kPer<E>, kLanes = D / kP, kKeys = kWave / kLanes, kAhead = 4;
  __shared__ float4 part[kWaves > 1 ? kBoundsT / kWave : 1][2][kLanes][kP / 4];
  const int lane = lane_id(), w = __builtin_amdgcn_readfirstlane(wave_id());
  const uint32_t unit = kWaves > 1 ? blockIdx.x : blockIdx.x * (kBoundsT / kWave) + w;
  if (unit >= p.units) return;
  const uint32_t head = unit % p.c.kv_heads, in = unit / p.c.kv_heads, row = in / p.each, j = in % p.each;
  const int32_t length = load_uniform(p.c.lengths + row);
  const int64_t most = static_cast<int64_t>(p.c.table_width) << p.page_shift;
  const bool says = head == 0 && lane == 0 && (kWaves == 1 || w == 0);
  if (length < 0 || length > most) {
    if (says && j == 0) raise_error(p.c.errors, QD_PAGED_BAD_LENGTH);
    return;
  }
  const uint32_t n = static_cast<uint32_t>(length);
  const uint32_t column = ((n > p.recent ? n - p.recent : 0u) >> p.page_shift) + j;
  const int64_t begin = static_cast<int64_t>(column) << p.page_shift;
  if (p.recent == 0 || begin >= length) return;
  const int32_t page = load_uniform(p.c.table + row * p.c.table_stride + column);
  if (page < 0 || static_cast<uint32_t>(page) >= p.c.pages) {
    if (says) raise_error(p.c.errors, QD_PAGED_BAD_PAGE);
    return;
  }
  const int keys = static_cast<int>(min<int64_t>(p.c.page_size, length - begin));
  const char *k = static_cast<const char *>(p.c.k) +
                  (page * p.c.page_stride + head * p.c.head_stride) * static_cast<int64_t>(16 / kP) + (lane % kLanes) * 16;
  const int64_t stride = p.c.token_stride * (16 / kP);
  float low[kP], high[kP];
#pragma unroll
  for (int i = 0; i < kP; ++i) {
    low[i] = INFINITY;
    high[i] = -INFINITY;
  }
  for (int at = lane / kLanes + (kWaves > 1 ? w * kKeys : 0); at < keys; at += kAhead * kWaves * kKeys) {
    u4v v[kAhead];
    // (Past the last key: the last one again.)
#pragma unroll
    for (int u = 0; u < kAhead; ++u) v[u] = *reinterpret_cast<const u4v *>(k + min(at + u * kWaves * kKeys, keys - 1) * stride);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      float y[kP];
      widen<E>(v[u], y);
#pragma unroll
      for (int i = 0; i < kP; ++i) {
        low[i] = fminf(low[i], y[i]);
        high[i] = fmaxf(high[i], y[i]);
      }
    }
  }
#pragma unroll
  for (int step = kLanes; step < kWave; step <<= 1)
#pragma unroll
    for (int i = 0; i < kP; ++i) {
      low[i] = fminf(low[i], from_lane(low[i], lane ^ step));
      high[i] = fmaxf(high[i], from_lane(high[i], lane ^ step));
    }
  if constexpr (kWaves > 1) {
    if (lane < kLanes)
#pragma unroll
      for (int i = 0; i < kP; i += 4) {
        part[w][0][lane][i / 4] = make_float4(low[i], low[i + 1], low[i + 2], low[i + 3]);
        part[w][1][lane][i / 4] = make_float4(high[i], high[i + 1], high[i + 2], high[i + 3]);
      }
    __syncthreads();
    if (w != 0) return;
    if (lane < kLanes)
      for (int u = 1; u < kWaves; ++u)
#pragma unroll
        for (int i = 0; i < kP; i += 4) {
          const float4 a = part[u][0][lane][i / 4], b = part[u][1][lane][i / 4];
          low[i] = fminf(low[i], a.x), low[i + 1] = fminf(low[i + 1], a.y), low[i + 2] = fminf(low[i + 2], a.z), low[i + 3] = fminf(low[i + 3], a.w);
          high[i] = fmaxf(high[i], b.x), high[i + 1] = fmaxf(high[i + 1], b.y), high[i + 2] = fmaxf(high[i + 2], b.z), high[i + 3] = fmaxf(high[i + 3], b.w);
        }
  }
  if (lane >= kLanes) return;
  const int64_t to = (static_cast<int64_t>(page) * p.c.kv_heads + head) * 2 * D + lane * kP;
#pragma unroll
  for (int i = 0; i < kP; i += 4) {
    store4<E>(p.bounds, to + i, make_float4(low[i], low[i + 1], low[i + 2], low[i + 3]));
    store4<E>(p.bounds, to + D + i, make_float4(high[i], high[i + 1], high[i + 2], high[i + 3]));
  }
}

// ---- the choice ---------------------------------------------------------------------
// The score is linear in a page's bounds: sum_d (sum_h min(q_h, 0)) low_d + (sum_h max(q_h, 0))
// high_d, one product of 2 D in 64 bits whatever the number of query heads, if all are finite: an
// infinite bound, one without a number or a query without makes the product infinite or NaN, and the
// score is then summed as it is defined. Four lanes take a
// page, a quarter of its bounds each; a workgroup takes a share of the pages of one row and KV
// head. Scores go out as whole numbers in their order; the last share of a row's head to
// arrive finds the least chosen one by counting keys into bins between the least and the
// largest, finer in each pass, and lists the chosen pages in order. 24 rows of 0 to 60,000 with 8
// heads of 128 in BF16, pages of 64, 64 of them: 29 us, of which 5 are the launch and the arrivals,
// 11 the scores (46 MB), 13 the choice, which all heads come to at about one time; 16 rows of 2,001 to
// 8,192 with 2 heads of 64 in FP32, pages of 16, 32 of them: 11 us. Attention over them takes
// 75 and 8.7.
constexpr int kChooseT = 256;
constexpr uint32_t kChooseLeast = 64;    // pages of a share at least
// (512: 33 us instead of 29, 4,096 28 to 33)
constexpr uint32_t kChooseAim = 1024;    // shares in all
constexpr uint32_t kBins = 2048;
constexpr uint32_t kKept = 4096;         // keys kept in LDS

struct ChooseLaunch {
  qd_paged_cache c;
  qd_sparse_args a;
  uint64_t *keys;      // [rows * kv_heads][table_width]
  int32_t *table;      // [rows * kv_heads][budget] what attention reads
  int32_t *lengths;    // [rows]
  uint32_t *counters;  // [rows * kv_heads]
  uint32_t group;
  uint32_t page_shift;
  uint32_t share;      // pages
};

// One element, or a bound, as it is held.
template <typename E>
__device__ __forceinline__ double element(const void *base, int64_t i) {
  if constexpr (std::is_same_v<E, float>)
    return static_cast<const float *>(base)[i];
  else
    return E::lo(static_cast<const uint16_t *>(base)[i]);
}
// The terms of dimensions [from, from + n) as they are defined: bounds from element `at`, queries from `q` on.
template <typename E, int D>
__device__ __forceinline__ double defined_score(const ChooseLaunch &p, int64_t at, int64_t q, int from, int n) {
  double s = 0.0;
#pragma unroll 1
  for (int d = from; d < from + n; ++d) {
    const double low = element<E>(p.a.bounds, at + d), high = element<E>(p.a.bounds, at + D + d);
#pragma unroll 1
    for (uint32_t h = 0; h < p.group; ++h) {
      const double x = element<E>(p.a.q, q + h * p.a.q_head_stride + d), a = x * low, b = x * high;
      s += a != a || b != b ? __builtin_nan("") : a > b ? a : b;
    }
  }
  return s;
}

// Whole numbers in the order of the scores; NaN as +inf.
__device__ __forceinline__ uint64_t key_of(double s) {
  const uint64_t x = __builtin_bit_cast(uint64_t, s + 0.0);  // (-0 as 0)
  if (s != s) return 0xFFF0000000000000ull;
  return x >> 63 ? ~x : x | 1ull << 63;
}

// Sum over the threads before this one.
__device__ __forceinline__ uint32_t threads_before(uint32_t v, uint32_t *waves, uint32_t &total) {
  const uint32_t upto = lanes_upto(v);
  __syncthreads();
  if (lane_id() == kWave - 1) waves[wave_id()] = upto;
  __syncthreads();
  uint32_t before = 0;
  total = 0;
#pragma unroll
  for (int u = 0; u < kChooseT / kWave; ++u) {
    if (u < wave_id()) before += waves[u];
    total += waves[u];
  }
  return before + upto - v;
}

template <typename E, int D>
__global__ __launch_bounds__(kChooseT) void choose_kernel(ChooseLaunch p) {
  constexpr int kP = kPer<E>, kQuarter = 2 * D / 4, kW = kChooseT / kWave;
  __shared__ __attribute__((aligned(16))) double weight[2 * D + 8];  // quarters two apart: no shared banks
  __shared__ uint64_t kept[kKept];
  __shared__ uint32_t bins[kBins], waves[kW], last, bin, above;
  __shared__ uint64_t ends[2][kW];
  const uint32_t unit = blockIdx.y, row = unit / p.c.kv_heads, head = unit % p.c.kv_heads;
  const int lane = lane_id(), w = wave_id();
  const int32_t length = load_uniform(p.c.lengths + row);
  const int64_t most = static_cast<int64_t>(p.c.table_width) << p.page_shift;
  const bool bad = length < 0 || length > most;
  const uint32_t pages = bad ? 0u : (static_cast<uint32_t>(length) + p.c.page_size - 1) >> p.page_shift;
  const int32_t *table = p.c.table + row * p.c.table_stride;
  int32_t *list = p.table + static_cast<size_t>(unit) * p.a.budget;
  int32_t *chosen = p.a.chosen ? p.a.chosen + static_cast<size_t>(unit) * p.a.budget : nullptr;
  const uint32_t fixed = p.a.first + p.a.last, wanted = p.a.budget - fixed;
  const bool few = pages <= p.a.budget;
  if (blockIdx.x == 0 && head == 0 && threadIdx.x == 0) {
    const int32_t n = static_cast<int32_t>(few ? pages : p.a.budget);
    p.lengths[row] = bad ? -1 : n == 0 ? 0 : length - static_cast<int32_t>((pages - n) << p.page_shift);
  }
  if (few || wanted == 0) {
    if (blockIdx.x > 0) return;
    for (uint32_t i = threadIdx.x; i < p.a.budget; i += kChooseT) {
      const uint32_t column = few ? i : i < p.a.first ? i : pages - p.a.budget + i;
      const bool in = column < pages;
      list[i] = in ? table[column] : -1;
      if (chosen) chosen[i] = in ? static_cast<int32_t>(column) : -1;
    }
    return;
  }
  // The pages between the first and the last ones: all that is scored.
  const uint32_t middle = pages - fixed, from = blockIdx.x * p.share, to = min(middle, from + p.share);
  if (from >= middle) return;
  const int64_t queries = row * p.a.q_stride + static_cast<int64_t>(head) * p.group * p.a.q_head_stride;
  for (int d = threadIdx.x; d < D; d += kChooseT) {
    double low = 0.0, high = 0.0;
    for (uint32_t h = 0; h < p.group; ++h) {
      const double q = element<E>(p.a.q, queries + h * p.a.q_head_stride + d);
      low += q < 0.0 ? q : q > 0.0 ? 0.0 : q;  // (NaN stays)
      high += q > 0.0 ? q : q < 0.0 ? 0.0 : q;
    }
    weight[d + d / kQuarter * 2] = low;
    weight[D + d + (D + d) / kQuarter * 2] = high;
  }
  __syncthreads();
  uint64_t *keys = p.keys + static_cast<size_t>(unit) * p.c.table_width;
  const int quarter = lane & 3;
  for (uint32_t i = from + threadIdx.x / 4; i < to; i += kChooseT / 4) {
    const int32_t page = table[p.a.first + i];
    const bool there = page >= 0 && static_cast<uint32_t>(page) < p.c.pages;
    const int64_t first = (static_cast<int64_t>(page) * p.c.kv_heads + head) * 2 * D;
    double s = 0.0;
    if (there) {
      const char *at = static_cast<const char *>(p.a.bounds) + (first + quarter * kQuarter) * (16 / kP);
      u4v v[kQuarter / kP];
#pragma unroll
      for (int u = 0; u < kQuarter / kP; ++u) v[u] = *reinterpret_cast<const u4v *>(at + 16 * u);
      const double *mine = weight + quarter * (kQuarter + 2);
#pragma unroll
      for (int u = 0; u < kQuarter / kP; ++u) {
        float y[kP];
        widen<E>(v[u], y);
#pragma unroll
        for (int c = 0; c < kP; ++c) s = fma(mine[u * kP + c], static_cast<double>(y[c]), s);
      }
    }
    s += lane_of(s, lane ^ 1);
    s += lane_of(s, lane ^ 2);
    if (!(fabs(s) < INFINITY)) {  // (all four lanes)
      s = defined_score<E, D>(p, first, queries, quarter * (D / 4), D / 4);
      s += lane_of(s, lane ^ 1);
      s += lane_of(s, lane ^ 2);
    }
    // A page that does not exist comes first: attention then says so.
    if (quarter == 0) __hip_atomic_store(keys + i, there ? key_of(s) : UINT64_MAX, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  wait_vm_stores();
  __syncthreads();
  if (threadIdx.x == 0) {
    last = atomicAdd(p.counters + unit, 1u) == (middle + p.share - 1) / p.share - 1;
    if (last) p.counters[unit] = 0u;
  }
  __syncthreads();
  if (!__builtin_amdgcn_readfirstlane(last)) return;
  const bool keep = middle <= kKept;
  const auto load = [&](uint32_t i) {
    return __hip_atomic_load(keys + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  };
  const auto key = [&](uint32_t i) { return keep ? kept[i] : load(i); };
  uint64_t low = UINT64_MAX, high = 0;
  for (uint32_t i = threadIdx.x; i < middle; i += kChooseT) {
    const uint64_t x = load(i);
    if (keep) kept[i] = x;
    low = x < low ? x : low;
    high = x > high ? x : high;
  }
#pragma unroll
  for (int step = 32; step > 0; step >>= 1) {
    const uint64_t a = lane_of(low, lane ^ step), b = lane_of(high, lane ^ step);
    low = a < low ? a : low;
    high = b > high ? b : high;
  }
  if (lane == 0) {
    ends[0][w] = low;
    ends[1][w] = high;
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < kW; ++u) {
    low = ends[0][u] < low ? ends[0][u] : low;
    high = ends[1][u] > high ? ends[1][u] : high;
  }
  // `need` of the keys from `low` to `high` are chosen besides those above `high`. Each pass
  // takes the range down to one bin of 2^shift keys; when that is one key, its places go to the
  // lowest pages.
  uint32_t need = wanted, equal = 0;
  bool ties = false;
  for (;;) {
    const uint64_t span = high - low;
    const int bits = span == 0 ? 0 : 64 - __clzll(static_cast<long long>(span));
    const int shift = max(0, bits - 11);
    for (uint32_t b = threadIdx.x; b < kBins; b += kChooseT) bins[b] = 0;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < middle; i += kChooseT) {
      const uint64_t x = key(i);
      if (x >= low && x <= high) atomicAdd(&bins[(x - low) >> shift], 1u);
    }
    __syncthreads();
    // Thread t has bins of the 8 t-th from the top on.
    constexpr uint32_t kEach = kBins / kChooseT;
    uint32_t mine = 0, total;
#pragma unroll
    for (uint32_t u = 0; u < kEach; ++u) mine += bins[kBins - 1 - (threadIdx.x * kEach + u)];
    uint32_t before = threads_before(mine, waves, total);
    if (before < need && before + mine >= need) {
      for (uint32_t u = 0; u < kEach; ++u) {
        const uint32_t b = kBins - 1 - (threadIdx.x * kEach + u);
        if (before + bins[b] >= need) {
          bin = b;
          above = before;
          break;
        }
        before += bins[b];
      }
    }
    __syncthreads();
    const uint32_t at = bin, inside = bins[at];
    need -= above;
    low += static_cast<uint64_t>(at) << shift;
    const uint64_t rest = high - low, whole = (uint64_t(1) << shift) - 1;
    high = low + (whole < rest ? whole : rest);
    __syncthreads();
    if (inside == need) break;   // all of the bin
    if (shift == 0) {            // equal keys, more than places
      ties = true;
      equal = need;
      break;
    }
  }
  // Chosen: keys from `low` on, of those equal to it where there are ties the first `equal`.
  const uint32_t each = (middle + kChooseT - 1) / kChooseT;
  const uint32_t a = min(middle, threadIdx.x * each), b = min(middle, a + each);
  uint32_t total, same = 0, taken = 0;
  for (uint32_t i = a; i < b; ++i) {
    const uint64_t x = key(i);
    same += x == low;
    taken += ties ? x > low : x >= low;
  }
  uint32_t same_before = 0;
  if (ties) {
    same_before = threads_before(same, waves, total);
    taken += min(same_before + same, equal) - min(same_before, equal);
  }
  uint32_t to_place = p.a.first + threads_before(taken, waves, total);
  const auto put = [&](uint32_t place, uint32_t column) {
    list[place] = table[column];
    if (chosen) chosen[place] = static_cast<int32_t>(column);
  };
  for (uint32_t i = a; i < b; ++i) {
    const uint64_t x = key(i);
    bool in = x > low || (!ties && x == low);
    if (ties && x == low) in = same_before++ < equal;
    if (in) put(to_place++, p.a.first + i);
  }
  for (uint32_t i = threadIdx.x; i < fixed; i += kChooseT) {
    if (i < p.a.first)
      put(i, i);
    else
      put(p.a.budget - fixed + i, pages - fixed + i);
  }
}

uint32_t choose_share(uint32_t units, uint32_t width) {
  const uint32_t most = (width + kChooseLeast - 1) / kChooseLeast;
  const uint32_t shares = std::max(1u, std::min(most, (kChooseAim + units - 1) / std::max(units, 1u)));
  return std::max(kChooseLeast, ((width + shares - 1) / shares + kChooseLeast - 1) / kChooseLeast * kChooseLeast);
}

size_t choose_scratch(uint32_t rows, uint32_t kv_heads, uint32_t width, uint32_t budget) {
  const size_t units = static_cast<size_t>(rows) * kv_heads;
  return round256(units * width * sizeof(uint64_t)) + round256(units * budget * sizeof(int32_t)) + round256(rows * sizeof(int32_t));
}

}  // namespace

hipError_t launch_page_bounds(hipStream_t s, const qd_paged_cache &c, void *bounds, uint32_t recent) {
  BoundsLaunch p{};
  p.c = c;
  p.bounds = bounds;
  p.recent = recent;
  p.page_shift = log2_of(c.page_size);
  // The last `recent` positions touch so many pages at most.
  p.each = recent == 0 ? 0u : static_cast<uint32_t>(std::min<uint64_t>(c.table_width, (static_cast<uint64_t>(recent) + c.page_size - 2) / c.page_size + 1));
  const uint64_t units = static_cast<uint64_t>(c.rows) * p.each * c.kv_heads;
  if (units == 0) return hipSuccess;
  p.units = static_cast<uint32_t>(units);
  const auto run = [&](auto one, auto four) {
    // Pages of more than 64 positions by four waves (a step of 64 BF16 rows of 8 heads of 128: pages of 64 by
    // one or four 4.2 us, of 128 by one 6.1, by four 5.0, of 1,024 38 and 17).
    return c.page_size > 64 ? launch(four, dim3(p.units), dim3(kBoundsT), s, p)
                            : launch(one, dim3((p.units + 3) / 4), dim3(kBoundsT), s, p);
  };
  const bool wide = c.head_dim == 128;
  switch (c.dtype) {
    case QD_DTYPE_F32: return wide ? run(bounds_kernel<float, 128, 1>, bounds_kernel<float, 128, 4>) : run(bounds_kernel<float, 64, 1>, bounds_kernel<float, 64, 4>);
    case QD_DTYPE_BF16: return wide ? run(bounds_kernel<Brain, 128, 1>, bounds_kernel<Brain, 128, 4>) : run(bounds_kernel<Brain, 64, 1>, bounds_kernel<Brain, 64, 4>);
    default: return wide ? run(bounds_kernel<Half, 128, 1>, bounds_kernel<Half, 128, 4>) : run(bounds_kernel<Half, 64, 1>, bounds_kernel<Half, 64, 4>);
  }
}

size_t sparse_attention_scratch(uint32_t rows, uint32_t heads, uint32_t kv_heads, uint32_t head_dim, uint32_t width, uint32_t budget) {
  return choose_scratch(rows, kv_heads, width, budget) + paged_attention_scratch(rows, heads, kv_heads, head_dim);
}
size_t sparse_attention_scratch_most(uint32_t rows, uint32_t heads, uint32_t kv_heads, uint32_t head_dim, uint32_t width,
                                     uint32_t budget) {
  return choose_scratch(rows, kv_heads, width, budget) + paged_attention_scratch_most(rows, heads, kv_heads, head_dim);
}

hipError_t launch_sparse_attention(hipStream_t s, const qd_paged_cache &c, const qd_sparse_args &a, const OpScratch &w) {
  if (c.rows == 0) return hipSuccess;
  ChooseLaunch p{};
  p.c = c;
  p.a = a;
  const size_t units = static_cast<size_t>(c.rows) * c.kv_heads;
  char *at = w.scratch;
  const auto take = [&](size_t bytes) {
    char *r = at;
    at += round256(bytes);
    return r;
  };
  p.keys = reinterpret_cast<uint64_t *>(take(units * c.table_width * sizeof(uint64_t)));
  p.table = reinterpret_cast<int32_t *>(take(units * a.budget * sizeof(int32_t)));
  p.lengths = reinterpret_cast<int32_t *>(take(c.rows * sizeof(int32_t)));
  p.counters = w.counters;
  p.group = a.heads / c.kv_heads;
  p.page_shift = log2_of(c.page_size);
  p.share = choose_share(static_cast<uint32_t>(units), c.table_width);
  const uint32_t shares = c.table_width <= a.budget ? 1u : std::max(1u, (c.table_width + p.share - 1) / p.share);
  const dim3 grid(shares, static_cast<uint32_t>(units)), block(kChooseT);
  const auto run = [&](auto kernel) { return launch(kernel, grid, block, s, p); };
  const bool wide = c.head_dim == 128;
  hipError_t err;
  switch (c.dtype) {
    case QD_DTYPE_F32: err = wide ? run(choose_kernel<float, 128>) : run(choose_kernel<float, 64>); break;
    case QD_DTYPE_BF16: err = wide ? run(choose_kernel<Brain, 128>) : run(choose_kernel<Brain, 64>); break;
    default: err = wide ? run(choose_kernel<Half, 128>) : run(choose_kernel<Half, 64>); break;
  }
  if (err != hipSuccess) return err;
  qd_paged_cache chosen = c;
  chosen.table = p.table;
  chosen.table_stride = static_cast<int64_t>(a.budget) * c.kv_heads;
  chosen.table_width = a.budget;
  chosen.lengths = p.lengths;
  qd_attention_args args{};
  args.q = a.q;
  args.out = a.out;
  args.q_stride = a.q_stride;
  args.q_head_stride = a.q_head_stride;
  args.out_stride = a.out_stride;
  args.out_head_stride = a.out_head_stride;
  args.heads = a.heads;
  args.scale = a.scale;
  return launch_paged_attention(s, chosen, args, OpScratch{w.counters, at}, a.budget);
}

}  // namespace qd
