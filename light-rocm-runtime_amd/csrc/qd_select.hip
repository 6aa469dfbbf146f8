// Beam selection for gfx950: the best k of beams x vocabulary. Declared in
// include/qd/qd_operators.h.
//
// A workgroup takes a run of a row's logits, tile after tile with the next one's
// loads under way; each wave keeps, without a barrier, a running maximum and sum
// per lane and the keys at or above a bound that only rises, and hands over its
// best k. The last run of a row to arrive joins the row's best k with their
// scores; the last row of a group to arrive chooses among its beams'. Bound by
// the logits' bandwidth for many rows (32 groups of 8 beams x 151,936 in FP32, 156 MB,
// 40 us, of which 26 stream at 6.0 TB/s), by the hand-overs for few: 16 beams 14.4
// us, one 8.5, of which the logits take 3.
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
constexpr int kEach = 16, kTile = kT * kEach;  // logits of a thread and of a workgroup at once
constexpr int kJoin = 2048;  // keys that one row's runs, or one group's rows, hand over at most
constexpr int kOwn = 640;    // keys of a wave: k from before, and a piece of 64 x 8
constexpr int kOwnStride = kOwn + 8;  // and zeros behind them
constexpr uint32_t kLowest = 0x00800000u;  // the order of the lowest finite number
constexpr float kLog2e = 1.44269504088896340736f;

struct SelectLaunch {
  qd_select_args a;
  uint32_t runs;        // of a row
  uint32_t tiles;       // of a run
  uint64_t *keys;       // [rows][runs][k]
  double *sums;         // [rows][runs]
  float *maxima;        // [rows][runs]
  double *row_score;    // [rows][k]
  uint32_t *row_token;  // [rows][k]
  uint32_t *row_count;  // arrivals [rows * apart]
  uint32_t *group_count;
  uint32_t apart;       // words between two counters
};

// A key orders a row's continuations: the higher logit first, then the lower
// token. The high word is the logit's bits, monotone (those of 0 for -0, which is
// no lower); 0 is no key.
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint64_t key) {
  const uint32_t u = static_cast<uint32_t>(key >> 32);
  return __uint_as_float(u & 0x80000000u ? u & 0x7FFFFFFFu : ~u);
}
__device__ __forceinline__ uint64_t key_of(float x, uint32_t token) {
  return static_cast<uint64_t>(order_of(x + 0.f)) << 32 | ~token;
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
// (Under-aligned types: the compiler's loads take any address.)
typedef uint32_t Words4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t Words2 __attribute__((ext_vector_type(4), aligned(2)));
template <typename E>
struct Piece {
  static constexpr int kElems = 16 / sizeof(E);
  using words = std::conditional_t<sizeof(E) == 4, Words4, Words2>;
};

constexpr int kFew = 512;  // keys of a run that are ranked from one list

struct Shared {
  uint64_t own[kWavesPerBlock][kOwnStride];  // the waves' keys
  uint64_t best[kWavesPerBlock][kSelectK];
  uint64_t few[kFew];
  double sum[kWavesPerBlock];
  float top[kWavesPerBlock];
  uint32_t bound[kWavesPerBlock], count[kWavesPerBlock];
  uint32_t n, last, found;
};
// The joins' keys and their places, where the waves' keys were.
static_assert(sizeof(Shared::own) + sizeof(Shared::best) >= kJoin * (sizeof(uint64_t) + sizeof(uint16_t)), "the joins' lists");

// Sum over the wave in 64 bits, in wave_sum's order.
template <int kCtrl>
__device__ __forceinline__ double dpp64(double v) {
  const uint64_t u = static_cast<uint64_t>(__double_as_longlong(v));
  const uint32_t lo = __float_as_uint(dpp<kCtrl>(__uint_as_float(static_cast<uint32_t>(u))));
  const uint32_t hi = __float_as_uint(dpp<kCtrl>(__uint_as_float(static_cast<uint32_t>(u >> 32))));
  return __longlong_as_double(static_cast<long long>(static_cast<uint64_t>(hi) << 32 | lo));
}
__device__ __forceinline__ double read_lane64(double v, int lane) {
  const uint64_t u = static_cast<uint64_t>(__double_as_longlong(v));
  const uint32_t lo = __float_as_uint(read_lane(__uint_as_float(static_cast<uint32_t>(u)), lane));
  const uint32_t hi = __float_as_uint(read_lane(__uint_as_float(static_cast<uint32_t>(u >> 32)), lane));
  return __longlong_as_double(static_cast<long long>(static_cast<uint64_t>(hi) << 32 | lo));
}
__device__ __forceinline__ double wave_sum64(double v) {
  v += dpp64<kDppXor1>(v);
  v += dpp64<kDppXor2>(v);
  v += dpp64<kDppHalfMirror>(v);
  v += dpp64<kDppMirror>(v);
  return (read_lane64(v, 0) + read_lane64(v, 16)) + (read_lane64(v, 32) + read_lane64(v, 48));
}

// A lower bound of the order of the wave's k-th best, from each lane's best: the
// k-th best lane has k as good before or at it. (The last 12 bits are left zero.)
__device__ __forceinline__ uint32_t wave_bound(uint32_t best, uint32_t k) {
  uint32_t t = 0;
#pragma unroll
  for (int bit = 31; bit >= 12; --bit) {
    const uint32_t with = t | 1u << bit;
    if (static_cast<uint32_t>(__popcll(__ballot(best >= with))) >= k) t = with;
  }
  return t;
}

// Sum over the four lanes of a quad.
__device__ __forceinline__ uint32_t quad_sum_u(uint32_t v) {
  v += __builtin_amdgcn_update_dpp(0, static_cast<int>(v), kDppXor1, 0xf, 0xf, false);
  return v + __builtin_amdgcn_update_dpp(0, static_cast<int>(v), kDppXor2, 0xf, 0xf, false);
}

// How many of the n keys are greater. The list is read eight at a time: the
// caller has zeroed up to seven places behind it.
__device__ __forceinline__ uint32_t rank_of(uint64_t key, const uint64_t *list, uint32_t n) {
  uint32_t rank = 0;
  for (uint32_t j = 0; j < n; j += 8) {
    ulonglong2 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = reinterpret_cast<const ulonglong2 *>(list + j)[u];
#pragma unroll
    for (int u = 0; u < 4; ++u) rank += (v[u].x > key) + (v[u].y > key);
  }
  return rank;
}

// The same, of the list's first n keys, by the four lanes of a quad together.
__device__ __forceinline__ uint32_t quad_rank(uint64_t key, const uint64_t *list, uint32_t n) {
  uint32_t rank = 0;
  for (uint32_t j = 8 * (lane_id() & 3); j < n; j += 32) {
    ulonglong2 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = reinterpret_cast<const ulonglong2 *>(list + j)[u];
#pragma unroll
    for (int u = 0; u < 4; ++u) rank += (j + 2 * u < n && v[u].x > key) + (j + 2 * u + 1 < n && v[u].y > key);
  }
  return quad_sum_u(rank);
}

// Leaves the best k of the wave's n keys, in order, at the start of its list;
// returns how many there are. `best` has room for k. (A wave's LDS operations take
// place in their order; the barriers hold the compiler to it.)
__device__ __forceinline__ uint32_t wave_best(uint64_t *list, uint32_t n, uint32_t k, uint64_t *best) {
  const uint32_t lane = lane_id();
  if (lane < 8) list[n + lane] = 0;
  __builtin_amdgcn_wave_barrier();
  for (uint32_t i = lane; i < n; i += kWave) {
    const uint64_t key = list[i];
    const uint32_t rank = rank_of(key, list, n);
    if (rank < k) best[rank] = key;
  }
  __builtin_amdgcn_wave_barrier();
  const uint32_t left = min(n, k);
  if (lane < left) list[lane] = best[lane];
  __builtin_amdgcn_wave_barrier();
  return left;
}

// What a group's results say: places of its best continuations found so far, for
// those that go to others.
struct Places {
  uint32_t beam[kSelectK], token[kSelectK];
  uint8_t taken[2 * kSelectK];
};
__device__ __forceinline__ void put_result(const SelectLaunch &p, uint32_t group, uint32_t i, double score, uint32_t beam,
                                           uint32_t token, bool was_done) {
  const size_t at = static_cast<size_t>(group) * p.a.k + i;
  p.a.scores_out[at] = static_cast<float>(score);
  p.a.parents[at] = static_cast<int32_t>(group * p.a.beams + beam);
  p.a.tokens[at] = static_cast<int32_t>(token);
  if (p.a.done) p.a.done_out[at] = was_done || token == p.a.eos;
}
// The places behind the first `found` go to the lowest (beam, token) that have none.
template <typename Done>
__device__ void fill_places(const SelectLaunch &p, uint32_t group, uint32_t found, Places &sh, Done was_done) {
  __syncthreads();
  const uint64_t all = static_cast<uint64_t>(p.a.beams) * p.a.vocab;
  const uint32_t t = threadIdx.x;
  if (t < 2 * kSelectK) {
    bool is = t >= all;
    for (uint32_t j = 0; j < found; ++j) is |= sh.beam[j] == t / p.a.vocab && sh.token[j] == t % p.a.vocab;
    sh.taken[t] = is;
  }
  __syncthreads();
  if (t < 2 * kSelectK && !sh.taken[t]) {
    uint32_t at = found;
    for (uint32_t j = 0; j < t; ++j) at += !sh.taken[j];
    if (at < p.a.k) put_result(p, group, at, -INFINITY, t / p.a.vocab, t % p.a.vocab, was_done(t / p.a.vocab));
  }
}

// f(u) for the N shares of n things that a thread has, `step` of them in each: most
// calls have no more than the first, and code that is not run is not fetched either.
template <int N, typename F>
__device__ __forceinline__ void for_shares(uint32_t n, uint32_t step, F &&f) {
#pragma unroll
  for (int u = 0; u < N; ++u) {
    if (u && n <= u * step) return;
    f(u);
  }
}

// Chooses among a group's rows; called by the workgroup that arrives last.
__device__ void choose(const SelectLaunch &p, uint32_t group, Shared &sh, Places &places) {
  constexpr int kMine = kSelectBeams * kSelectK / kT;
  const uint32_t k = p.a.k, n = p.a.beams * k;
  const uint32_t row0 = group * p.a.beams;
  const Coherent scores(p.row_score + static_cast<size_t>(row0) * k, n * 8);
  const Coherent tokens(p.row_token + static_cast<size_t>(row0) * k, n * 4);
  uint64_t *list = &sh.own[0][0];
  uint16_t *place = reinterpret_cast<uint16_t *>(list + kJoin);
  __shared__ uint8_t was_done[kSelectBeams];
  __shared__ uint32_t held[kSelectBeams * kSelectK];  // the entries' tokens
  if (p.a.done && threadIdx.x < p.a.beams) was_done[threadIdx.x] = p.a.done[row0 + threadIdx.x] != 0;
  // A score's key: its 64 bits, monotone; 0 where there is none.
  uint64_t key[kMine];
  uint32_t token[kMine];
  for_shares<kMine>(n, kT, [&](int u) {  // (past the end the descriptors give zeros)
    key[u] = load64(scores, u * kT + threadIdx.x);
    token[u] = tokens.ldu(u * kT + threadIdx.x);
  });
  uint32_t best = 0;
  for_shares<kMine>(n, kT, [&](int u) {
    held[u * kT + threadIdx.x] = token[u];
    const double s = __longlong_as_double(static_cast<long long>(key[u]));
    if (u * kT + threadIdx.x >= n || s == -INFINITY)
      key[u] = 0;
    else
      key[u] = key[u] >> 63 ? ~key[u] : key[u] | 1ull << 63;
    best = max(best, static_cast<uint32_t>(key[u] >> 32));
  });
  const uint32_t bound = wave_bound(best, k);
  if (threadIdx.x == 0) sh.n = 0;
  if (lane_id() == 0) sh.bound[wave_id()] = bound;
  __syncthreads();
  uint32_t least = max(1u, sh.bound[0]);
#pragma unroll
  for (int w = 1; w < kWavesPerBlock; ++w) least = max(least, sh.bound[w]);
  uint32_t mine = 0;
  for_shares<kMine>(n, kT, [&](int u) { mine += static_cast<uint32_t>(key[u] >> 32) >= least; });
  if (mine) {
    uint32_t at = atomicAdd(&sh.n, mine);
    for_shares<kMine>(n, kT, [&](int u) {
      if (static_cast<uint32_t>(key[u] >> 32) >= least) {
        list[at] = key[u];
        place[at++] = static_cast<uint16_t>(u * kT + threadIdx.x);
      }
    });
  }
  __syncthreads();
  const uint32_t count = sh.n, found = min(count, k);
  // Four lanes find an entry's rank: higher scores, and equal ones of lower places.
  for (uint32_t i = threadIdx.x / 4; i < count; i += kT / 4) {
    const uint64_t it = list[i];
    const uint32_t at = place[i];
    uint32_t rank = 0;
    for (uint32_t j = 8 * (threadIdx.x & 3); j < count; j += 32) {
      ulonglong2 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = reinterpret_cast<const ulonglong2 *>(list + j)[u];
      const uint4 pl = *reinterpret_cast<const uint4 *>(place + j);
      const uint32_t pw[4] = {pl.x, pl.y, pl.z, pl.w};
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        rank += j + 2 * u < count && (v[u].x > it || (v[u].x == it && (pw[u] & 0xFFFFu) < at));
        rank += j + 2 * u + 1 < count && (v[u].y > it || (v[u].y == it && pw[u] >> 16 < at));
      }
    }
    rank = quad_sum_u(rank);
    if (rank >= k || (threadIdx.x & 3)) continue;
    const uint64_t bits = it >> 63 ? it & ~(1ull << 63) : ~it;
    const uint32_t tok = held[at];
    put_result(p, group, rank, __longlong_as_double(static_cast<long long>(bits)), at / k, tok, p.a.done && was_done[at / k]);
    places.beam[rank] = at / k;
    places.token[rank] = tok;
  }
  if (found < k) fill_places(p, group, found, places, [&](uint32_t beam) { return p.a.done && was_done[beam]; });
}

// Joins a row's runs; called by the workgroup that arrives last. The row of a group
// of one is the group's result.
__device__ void join_row(const SelectLaunch &p, uint32_t row, Shared &sh, Places &places) {
  constexpr int kMine = kJoin / 2 / kT;
  const uint32_t k = p.a.k, n = p.runs * k;
  const Coherent keys(p.keys + static_cast<size_t>(row) * (n + (n & 1)), (n + (n & 1)) * 8);
  const Coherent sums(p.sums + static_cast<size_t>(row) * p.runs, p.runs * 8);
  const Coherent maxima(p.maxima + static_cast<size_t>(row) * p.runs, p.runs * 4);
  const Coherent scores(p.row_score + static_cast<size_t>(row) * k, k * 8);
  const Coherent tokens(p.row_token + static_cast<size_t>(row) * k, k * 4);
  // Two keys a load, all of them on their way before the first is used. (An even k:
  // the runs' best pairs first, so that the first wave's bound is a near one.)
  const uint32_t depth = k & 1 ? 1 : k / 2, across = k & 1 ? (n + 1) / 2 : p.runs;
  const float per = __builtin_amdgcn_rcpf(static_cast<float>(across));  // (below 1,024: exact where it is rounded down)
  uint64_t key[2 * kMine];
  for_shares<kMine>(n, 2 * kT, [&](int u) {
    const uint32_t i = u * kT + threadIdx.x, down = static_cast<uint32_t>((static_cast<float>(i) + 0.5f) * per);
    const float4 v = keys.ld4((i - down * across) * depth + down);  // (past the end: zeros)
    const uint2 a = {__float_as_uint(v.x), __float_as_uint(v.y)}, b = {__float_as_uint(v.z), __float_as_uint(v.w)};
    key[2 * u] = a.x | static_cast<uint64_t>(a.y) << 32;
    key[2 * u + 1] = b.x | static_cast<uint64_t>(b.y) << 32;
  });
  float m = -INFINITY;
  double sum = 0.0;
  for (uint32_t s = threadIdx.x; s < p.runs; s += kT) {
    const float top = maxima.ld(s);
    const double part = __longlong_as_double(static_cast<long long>(load64(sums, s)));
    if (top > m) {
      sum = m == -INFINITY ? part : part + sum * exp2_fast((m - top) * kLog2e);
      m = top;
    } else if (top > -INFINITY) {
      sum += top == m ? part : part * exp2_fast((top - m) * kLog2e);
    }
  }
  uint32_t best = 0;
  for_shares<kMine>(n, 2 * kT, [&](int u) {
#pragma unroll
    for (int v = 2 * u; v < 2 * u + 2; ++v) {
      // (Indexes past the end come to others' pairs, and an odd number of keys ends
      // with half of a load.)
      if (2 * (u * kT + threadIdx.x) + (v & 1) >= n) key[v] = 0;
      best = max(best, static_cast<uint32_t>(key[v] >> 32));
    }
  });
  const uint32_t bound = wave_bound(best, k);
  const float wave_m = wave_max(m);
  if (lane_id() == 0) {
    sh.top[wave_id()] = wave_m;
    sh.bound[wave_id()] = bound;
  }
  if (threadIdx.x == 0) sh.n = sh.found = 0;
  __syncthreads();
  float top = sh.top[0];
  uint32_t least = max(kLowest, sh.bound[0]);
#pragma unroll
  for (int w = 1; w < kWavesPerBlock; ++w) {
    top = fmaxf(top, sh.top[w]);
    least = max(least, sh.bound[w]);
  }
  sum = m == top ? sum : m == -INFINITY ? 0.0 : sum * exp2_fast((m - top) * kLog2e);
  sum = wave_sum64(sum);
  if (lane_id() == 0) sh.sum[wave_id()] = sum;
  uint64_t *list = &sh.own[0][0];
  uint32_t mine = 0;
  for_shares<kMine>(n, 2 * kT, [&](int u) {
    mine += (static_cast<uint32_t>(key[2 * u] >> 32) >= least) + (static_cast<uint32_t>(key[2 * u + 1] >> 32) >= least);
  });
  if (mine) {
    uint32_t at = atomicAdd(&sh.n, mine);
    for_shares<kMine>(n, 2 * kT, [&](int u) {
#pragma unroll
      for (int v = 2 * u; v < 2 * u + 2; ++v)
        if (static_cast<uint32_t>(key[v] >> 32) >= least) list[at++] = key[v];
    });
  }
  __syncthreads();
  const uint32_t count = sh.n;
  const double log_total = log((sh.sum[0] + sh.sum[1]) + (sh.sum[2] + sh.sum[3]));
  const double base = static_cast<double>(p.a.scores[row]);
  const bool alone = p.a.beams == 1;
  for (uint32_t i = threadIdx.x / 4; i < max(count, k); i += kT / 4) {
    const uint64_t it = i < count ? list[i] : 0;
    const uint32_t rank = i < count ? quad_rank(it, list, count) : i;
    if (rank >= k || (threadIdx.x & 3)) continue;
    const float x = logit_of(it);
    // (An infinite maximum leaves the others nothing.)
    const double s =
        i >= count ? -INFINITY : base + ((x == top ? 0.0 : static_cast<double>(x) - top) - log_total);
    if (!alone) {
      store64(scores, rank, static_cast<uint64_t>(__double_as_longlong(s)));
      tokens.stu(rank, token_of(it));
    } else if (s > -INFINITY) {
      put_result(p, row, rank, s, 0, token_of(it), false);
      places.beam[rank] = 0;
      places.token[rank] = token_of(it);
      atomicAdd(&sh.found, 1u);
    }
  }
  if (!alone) return;
  __syncthreads();
  if (sh.found < k) fill_places(p, row, sh.found, places, [](uint32_t) { return false; });
}

// What is left of a row's way once its scores are stored.
__device__ __forceinline__ void row_done(const SelectLaunch &p, uint32_t row, Shared &sh, Places &places) {
  const uint32_t group = row / p.a.beams;
  wait_vm_stores();
  __syncthreads();
  if (threadIdx.x == 0) {
    sh.last = p.a.beams == 1 || atomicAdd(p.group_count + group * p.apart, 1u) == p.a.beams - 1;
    if (sh.last && p.a.beams > 1) p.group_count[group * p.apart] = 0u;
  }
  __syncthreads();
  if (sh.last) choose(p, group, sh, places);
}

template <typename E>
__global__ __launch_bounds__(kT) void select_kernel(SelectLaunch p) {
  using P = Piece<E>;
  constexpr int kPieces = kEach / P::kElems;
  static_assert(kOwn >= static_cast<int>(kSelectK) + kWave * P::kElems, "a piece fits behind k keys");
  __shared__ __attribute__((aligned(16))) Shared sh;
  __shared__ Places places;
  const uint32_t row = blockIdx.y, run = blockIdx.x, k = p.a.k;
  const E *logits = static_cast<const E *>(p.a.logits) + static_cast<int64_t>(row / p.a.beams) * p.a.group_stride +
                    static_cast<int64_t>(row % p.a.beams) * p.a.beam_stride;
  const uint32_t lane = lane_id(), w = wave_id();
  const uint32_t begin = run * p.tiles * kTile, end = min(p.a.vocab, begin + p.tiles * kTile);
  // Piece j of a tile: P::kElems logits of each thread, one after the other.
  typename P::words next[kPieces];
  auto fetch = [&](uint32_t tile) {
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      const uint32_t at = tile + (j * kT + threadIdx.x) * P::kElems;
      if (at + P::kElems <= end)
        next[j] = *reinterpret_cast<const typename P::words *>(logits + at);
      else
        next[j] = typename P::words{0u, 0u, 0u, 0u};
    }
  };
  fetch(begin);  // on its way while the row's score is looked at
  const float score = p.a.scores[row];
  const bool live = fabsf(score) < INFINITY;
  const bool done = p.a.done && p.a.done[row];
  if (__builtin_expect(!live || done, 0)) {
    // The logits do not matter: one continuation, or none.
    if (run) return;
    const Coherent scores(p.row_score + static_cast<size_t>(row) * k, k * 8);
    const Coherent tokens(p.row_token + static_cast<size_t>(row) * k, k * 4);
    for (uint32_t i = threadIdx.x; i < k; i += kT) {
      const double s = live && i == 0 ? static_cast<double>(score) + 0.0 : -INFINITY;  // (-0 is no lower than 0)
      store64(scores, i, static_cast<uint64_t>(__double_as_longlong(s)));
      tokens.stu(i, p.a.eos);
    }
    row_done(p, row, sh, places);
    return;
  }
  uint64_t *own = sh.own[w];
  uint32_t count = 0;
  float least = logit_of(static_cast<uint64_t>(kLowest) << 32);  // keys at or above it are kept
  float m = -INFINITY, base = -INFINITY;
  double sum = 0.0;
  for (uint32_t tile = begin; tile < end; tile += kTile) {
    float x[kEach];
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      const uint32_t at = tile + (j * kT + threadIdx.x) * P::kElems;
#pragma unroll
      for (int c = 0; c < P::kElems; ++c) {
        uint32_t bits;
        if constexpr (sizeof(E) == 4)
          bits = next[j][c];
        else
          bits = c & 1 ? next[j][c >> 1] >> 16 : next[j][c >> 1] & 0xFFFFu;
        x[j * P::kElems + c] = widen<E>(bits);
      }
      if (__builtin_expect(at + P::kElems > end, 0)) {  // the row's end: one by one
#pragma unroll
        for (int c = 0; c < P::kElems; ++c) {
          float y = -INFINITY;
          if (at + c < end) {
            if constexpr (sizeof(E) == 4)
              y = reinterpret_cast<const float *>(logits)[at + c];
            else
              y = widen<E>(reinterpret_cast<const uint16_t *>(logits)[at + c]);
          }
          x[j * P::kElems + c] = y;
        }
      }
    }
    if (tile + kTile < end) fetch(tile + kTile);
    float top = -INFINITY;
    // (NaN is no maximum and at or above no bound; of its exponential, fmaxf makes 0.)
#pragma unroll
    for (int i = 0; i < kEach; ++i) top = fmaxf(top, x[i]);
    // Sum of exp(x - base), 16 terms in FP32 and 64 bits beyond. The base follows the
    // lane's maximum by steps of 1 and more: the differences that count are exact to
    // half a step, and a new base's factor is soon outweighed.
    m = fmaxf(m, top);
    if (top > base + 1.f) {
      if (base > -INFINITY) sum *= exp2_fast((base - top) * kLog2e);
      base = top;
    }
    const float from = base == -INFINITY ? 0.f : base;
    float part = 0.f;
    if (__builtin_expect(!__any(base == INFINITY), 1)) {
#pragma unroll
      for (int i = 0; i < kEach; ++i) part += fmaxf(exp2_fast((x[i] - from) * kLog2e), 0.f);
    } else {
#pragma unroll
      for (int i = 0; i < kEach; ++i) part += x[i] == from ? 1.f : fmaxf(exp2_fast((x[i] - from) * kLog2e), 0.f);
    }
    sum += part;
    // The bound rises with the lanes' maxima, after 1, 2, 4, ... tiles, and when
    // the wave's list is full.
    if (const uint32_t seen = (tile - begin) / kTile + 1; (seen & (seen - 1)) == 0)
      least = fmaxf(least, logit_of(static_cast<uint64_t>(max(kLowest, wave_bound(order_of(m), k))) << 32));
    if (__any(top >= least)) {
#pragma unroll
      for (int j = 0; j < kPieces; ++j) {
        if (__builtin_expect(count + kWave * P::kElems > kOwn, 0)) {
          count = wave_best(own, count, k, sh.best[w]);
          // Later tokens are higher: only greater logits count. (A bound of
          // infinity keeps the infinite ones, of which enough are there.)
          if (count == k) {
            const uint32_t above = static_cast<uint32_t>(own[k - 1] >> 32) + 1;
            least = fmaxf(least, logit_of(static_cast<uint64_t>(min(above, order_of(INFINITY))) << 32));
          }
        }
        const uint32_t first = tile + (j * kT + threadIdx.x) * P::kElems;
#pragma unroll
        for (int c = 0; c < P::kElems; ++c) {
          const bool in = x[j * P::kElems + c] >= least;
          const uint64_t mask = __ballot(in);
          if (mask == 0) continue;
          if (in) own[count + __popcll(mask & ((1ull << lane) - 1))] = key_of(x[j * P::kElems + c], first + c);
          count += __popcll(mask);
        }
      }
    }
  }
  const float wave_m = wave_max(m);
  const uint32_t bound = wave_bound(order_of(m), k);
  if (lane == 0) {
    sh.top[w] = wave_m;
    sh.bound[w] = bound;
    sh.count[w] = count;
  }
  if (threadIdx.x == 0) sh.n = 0;
  if (lane < 8) own[count + lane] = 0;
  __syncthreads();
  float top = sh.top[0];
  uint32_t all_least = max(kLowest, sh.bound[0]);
#pragma unroll
  for (int u = 1; u < kWavesPerBlock; ++u) {
    top = fmaxf(top, sh.top[u]);
    all_least = max(all_least, sh.bound[u]);
  }
  // Its keys at or above the highest bound, mostly few, go to one list.
  for (uint32_t i = 0; i < count; i += kWave) {
    const uint64_t key = i + lane < count ? own[i + lane] : 0;
    const bool in = static_cast<uint32_t>(key >> 32) >= all_least;
    const uint64_t mask = __ballot(in);
    uint32_t at = 0;
    if (lane == 0) at = atomicAdd(&sh.n, static_cast<uint32_t>(__popcll(mask)));
    at = __builtin_amdgcn_readfirstlane(at) + __popcll(mask & ((1ull << lane) - 1));
    if (in && at < static_cast<uint32_t>(kFew)) sh.few[at] = key;
  }
  const double total = wave_sum64(base == top ? sum : base == -INFINITY ? 0.0 : sum * exp2_fast((base - top) * kLog2e));
  if (lane == 0) sh.sum[w] = total;
  __syncthreads();
  const uint32_t n = p.runs * k;
  const Coherent keys(p.keys + static_cast<size_t>(row) * (n + (n & 1)), (n + (n & 1)) * 8);
  uint32_t all = sh.n;
  if (__builtin_expect(all <= static_cast<uint32_t>(kFew), 1)) {
    for (uint32_t i = threadIdx.x / 4; i < all; i += kT / 4) {
      const uint64_t key = sh.few[i];
      const uint32_t rank = quad_rank(key, sh.few, all);
      if (rank < k && (threadIdx.x & 3) == 0) store64(keys, run * k + rank, key);
    }
  } else {
    // Crowded near the top: a key's place is the sum of its places in the four lists.
    for (uint32_t i = lane; i < count; i += kWave) {
      const uint64_t key = own[i];
      uint32_t rank = 0;
#pragma unroll
      for (int u = 0; u < kWavesPerBlock; ++u) rank += rank_of(key, sh.own[u], sh.count[u]);
      if (rank < k) store64(keys, run * k + rank, key);
    }
  }
  for (uint32_t i = all + threadIdx.x; i < k; i += kT) store64(keys, run * k + i, 0);
  if (threadIdx.x == 0) {
    const Coherent sums(p.sums + static_cast<size_t>(row) * p.runs, p.runs * 8);
    const Coherent maxima(p.maxima + static_cast<size_t>(row) * p.runs, p.runs * 4);
    store64(sums, run, static_cast<uint64_t>(__double_as_longlong((sh.sum[0] + sh.sum[1]) + (sh.sum[2] + sh.sum[3]))));
    maxima.st(run, top);
  }
  wait_vm_stores();
  __syncthreads();
  if (threadIdx.x == 0) {
    sh.last = p.runs == 1 || atomicAdd(p.row_count + row * p.apart, 1u) == p.runs - 1;
    if (sh.last && p.runs > 1) p.row_count[row * p.apart] = 0u;
  }
  __syncthreads();
  if (!sh.last) return;
  join_row(p, row, sh, places);
  if (p.a.beams > 1) row_done(p, row, sh, places);
}

// A row's runs: as many as make kAim workgroups (four fit a CU; 256 rows of 151,936
// 40.9 us, with 512 of them 48.8, with 2,048 48.0), no more than it has tiles and the
// join takes.
constexpr uint32_t kAim = 1024;
uint32_t tiles_of(uint32_t vocab) { return (vocab + kTile - 1) / kTile; }
void split_rows(SelectLaunch &p, uint32_t rows, uint32_t k, uint32_t vocab) {
  const uint32_t tiles = tiles_of(vocab);
  const uint32_t runs = std::max(1u, std::min({tiles, kAim / std::max(1u, rows), kJoin / k}));
  p.tiles = (tiles + runs - 1) / runs;
  p.runs = (tiles + p.tiles - 1) / p.tiles;
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
  const size_t parts = static_cast<size_t>(rows) * p.runs, keys = p.runs * k;
  p.keys = reinterpret_cast<uint64_t *>(take(rows * (keys + (keys & 1)) * 8));
  p.sums = reinterpret_cast<double *>(take(parts * 8));
  p.maxima = reinterpret_cast<float *>(take(parts * 4));
  p.row_score = reinterpret_cast<double *>(take(static_cast<size_t>(rows) * k * 8));
  p.row_token = reinterpret_cast<uint32_t *>(take(static_cast<size_t>(rows) * k * 4));
  return used;
}

}  // namespace

size_t beam_select_scratch(uint32_t groups, uint32_t beams, uint32_t k, uint32_t vocab) {
  const uint32_t rows = groups * beams;
  SelectLaunch p{};
  split_rows(p, rows, k, vocab);
  return carve(p, nullptr, rows, k);
}

// Whatever the rows, they are in no more parts than tiles, and than kAim or one each;
// fewer rows, places or tokens can be in more parts than more of them.
size_t beam_select_scratch_most(uint32_t groups, uint32_t beams, uint32_t k, uint32_t vocab) {
  const size_t rows = static_cast<size_t>(groups) * beams;
  const size_t parts = std::min<size_t>(rows * tiles_of(vocab), std::max<size_t>(rows, kAim));
  const size_t keys = std::min(parts * k, rows * kJoin) + rows;  // (an odd row's rest of a pair)
  return round256(keys * 8) + round256(parts * 8) + round256(parts * 4) + round256(rows * k * 8) + round256(rows * k * 4);
}

hipError_t launch_beam_select(hipStream_t s, const qd_select_args &a, const OpScratch &w) {
  const uint32_t rows = a.groups * a.beams;
  if (rows == 0) return hipSuccess;
  SelectLaunch p{};
  p.a = a;
  split_rows(p, rows, a.k, a.vocab);
  carve(p, w.scratch, rows, a.k);
  // Counters in lines of their own where there is room: 608 arrivals at 16 counters
  // of one line took 6 us, at lines of their own 1.1.
  p.apart = 32;
  while (static_cast<uint64_t>(rows + a.groups) * p.apart > kOpCounters) p.apart /= 2;
  p.row_count = w.counters;
  p.group_count = w.counters + static_cast<size_t>(rows) * p.apart;
  const dim3 grid(p.runs, rows), block(kT);
  return launch(a.dtype == QD_DTYPE_F32    ? select_kernel<float>
                : a.dtype == QD_DTYPE_BF16 ? select_kernel<Bf16>
                                           : select_kernel<F16>,
                grid, block, s, p);
}

}  // namespace qd
