// Operators on trees of drafted tokens for gfx950: their attention over a paged
// cache, the answer to them, and the move of what stands. Declared in
// include/qd/qd_operators.h.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "qd_attention.hpp"
#include "qd_device.hpp"
#include "qd_device_math.hpp"
#include "qd_operators.hpp"
#include "qd_paged.hpp"

namespace qd {
namespace {

using namespace dev;

constexpr uint32_t kNan = 0x7FC00000u;

// ---- the tree -------------------------------------------------------------------
// A node's mask: itself and the nodes above it, each lane its own node's, by
// doubling (after s steps a lane knows 2^s nodes of its chain). 0: not there.
__device__ __forceinline__ uint64_t ancestors(const int32_t *parents, uint32_t nodes, bool &bad) {
  const int lane = lane_id();
  int up = static_cast<uint32_t>(lane) < nodes ? parents[lane] : -2;
  const uint64_t there = __ballot(up >= -1);
  // A parent comes before its child, and is there.
  const bool wrong = up >= lane || (up >= 0 && !(there >> up & 1));
  bad = __any(wrong);
  if (wrong) up = -2;
  uint64_t mask = up >= -1 ? 1ull << lane : 0ull;
#pragma unroll
  for (int s = 0; s < 6; ++s) {
    const int from = up < 0 ? lane : up;
    const uint64_t more = lane_of(mask, from);
    const int next = __builtin_amdgcn_ds_bpermute(from << 2, up);
    if (up >= 0) {
      mask |= more;
      up = next;
    }
  }
  return mask;
}

// ---- attention --------------------------------------------------------------------
// A row's queries of one KV head, its columns, are all pairs of a node and one of the
// head's query heads. A workgroup takes a block of 16 NB WC columns over a run of the
// row's positions, in stages of 32 WP: K and V of a stage go to LDS without passing
// registers, the next stages' on their way, and are read from there by WC x WP waves,
// each for 16 NB columns and 32 positions of the stage:
//   S^T = K Q^T    lane l: column l % 16, positions 4 (l / 16) + r of each 16
//   O^T += V^T P^T with the lane's own probabilities as the operand; V is read in the
//                  operand's layout, 16-bit types by transposing reads.
// Positions before the tree are seen by every node; in the tree a bit of the node's
// mask says so. What does not is hidden from the sum by its score, and by zeros in V's
// place where V is not finite: the outputs that do see such a value become NaN.
// Few rows are cut into runs that fill the card, which the last one joins in order.
// 64 BF16 rows of 0 to 8,192 with 8 nodes of 4 heads on 8 KV heads of 128 take 212 us, 1,087 MB at
// 5.1 TB/s, bound by memory and by what ends a piece (187 us without results and joins); two FP16 rows of
// 30,001 to 40,001 with 63 nodes of 7 on 4 KV heads 140 us, 63 GFLOP at 0.45 PFLOP/s, bound by the
// sum of products and the exponentials' vector work, which overlap little (without K's half of a stage
// 96 us, without V's 100, without either 77; without the second number of a weight 117). 16 FP32 rows
// of 576 with 16 nodes of 7 on 2 heads of 64 19 us, one of 129 with 8 12.4: a chain of latencies.
constexpr int kStep = 32;                // positions of a wave's step
constexpr uint32_t kTreePieces = 64;     // of an item at most
// (128: one row of 129 with 8 nodes 15.0 us instead of 12.5, 16 of 576 with 16 19.3 and 19.1)
constexpr uint32_t kTreeLeast = 64;      // positions of a piece at least
constexpr uint32_t kTreeCus = 256, kTreePerCu = 3, kXcds = 8;
constexpr uint32_t kLds = 160 * 1024;
// A maximum is taken up once it passes the one in use by so many powers of two, as in the
// attention of one token (qd_paged.hip).
template <typename E>
constexpr float kLazy = 8.f;
template <>
constexpr float kLazy<Half> = 1.f;
// FP16 takes 2^14 times a probability (at most 2 before it is rounded), and what rounding
// that left: off by 2^-22 of it, or, at the end of FP16's range, 2^-39 of the largest. Sums
// have the same factor, which the division takes out.
template <typename E>
constexpr float kUnit = 0.f;
template <>
constexpr float kUnit<Half> = 14.f;

struct TreeLaunch {
  qd_paged_cache c;
  qd_tree_attention_args a;
  float *records;      // [pieces][kv_heads * blocks][columns of a block * (head_dim + 2)]
  uint32_t *counters;  // [rows][kv_heads * blocks]
  uint32_t apart;      // words between two counters
  uint32_t group;      // query heads of a KV head
  uint32_t columns;    // nodes * group
  uint32_t blocks;     // of columns
  uint32_t page_shift;
  uint32_t parts;      // items of a row: KV heads x blocks
  uint32_t target;     // pieces of one item that the card holds at once; 0: rows are not cut
  uint32_t units;      // pieces in the grid, of all rows and one item each; 0: equal runs of all stages
  uint32_t least;      // (equal runs) stages on either side of a cut
};

// One 16-byte global -> LDS DMA per lane (lane l's bytes land at lds + 16 l), from
// inline assembly: the compiler would guard every later LDS read with a wait for it.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // m0 is reserved: set before each use, never saved
// (lds and base are the wave's: the compiler is told where it cannot see it, by a vector instruction
// that writes scalar registers. A transfer may read those five wait states later.)
__device__ __forceinline__ void dma_to_lds(const void *src, uint32_t lds) {
  lds = __builtin_amdgcn_readfirstlane(lds);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(src) : "memory", "m0");
}
__device__ __forceinline__ void dma_to_lds(const void *base, uint32_t off, uint32_t lds) {
  const uint64_t at = reinterpret_cast<uint64_t>(base);
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(at)), hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(at >> 32));
  base = reinterpret_cast<const void *>(static_cast<uint64_t>(hi) << 32 | lo);
  lds = __builtin_amdgcn_readfirstlane(lds);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2 nt" ::"s"(lds), "v"(off), "s"(base) : "memory", "m0");
}
#pragma clang diagnostic pop
// Waits until at most kEach x `left` of this wave's transfers are on their way.
template <int kLeft>
__device__ __forceinline__ void dma_wait() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kLeft) : "memory");
}
template <int kEach, int kMost>
__device__ __forceinline__ void dma_wait(uint32_t left) {
  if constexpr (kMost > 0)
    if (left < kMost) return dma_wait<kEach, kMost - 1>(left);
  dma_wait<kEach * kMost>();
}
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

typedef __attribute__((address_space(3))) char lds_char;
typedef short s4v __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4v lds_s4v;

// A piece of an item: wave-uniform.
struct Piece {
  uint32_t row, kv, block;
  int length, start;      // of the row, and where its tree begins
  uint32_t first, last;   // stages
  uint32_t index, pieces; // of the row
  uint32_t number;        // of the row's first among all
  bool bad;               // the length
};

template <typename E, int D, int NB, int WC, int WP>
struct TreeShape {
  static constexpr bool kWide = std::is_same_v<E, float>;
  static constexpr int kElem = kWide ? 4 : 2;
  static constexpr int kWaves = WC * WP, kThreads = kWaves * kWave;
  static constexpr int kStage = kStep * WP;
  static constexpr int kRowBytes = D * kElem;
  static constexpr int kHalf = kStage * kRowBytes;  // K or V of a stage
  // So many of them in LDS. Up to 64 columns they are waited for one by one and all but one are
  // on their way, to three workgroups of a CU (five halves of 8 KB; nine and two workgroups: 64
  // rows of 0 to 8,192 with 8 nodes 227 us instead of 212); where products bound a stage, by
  // stages, three of them on their way.
  static constexpr bool kWhole = WP > 1;
  static constexpr bool kByHalves = !kWhole;
  static constexpr int kHalves = kWhole ? 8 : kRowBytes == 512 ? 4 : kRowBytes == 256 ? 5 : 9;
  static constexpr int kColumns = 16 * NB * WC;
  static constexpr int kRowsPerDma = 1024 / kRowBytes, kLanesPerRow = kRowBytes / 16;
  static constexpr int kRows = kStage / kWaves;                // of a half, that a wave transfers
  static constexpr int kDmas = kRows / kRowsPerDma;
  static constexpr int kIds = (kRows + 15) / 16;               // groups of 16 of them
  static constexpr int kAcc = D / 16;
  static constexpr int kMerge = WP > 1 ? WC * NB * (kAcc * 1024 + 512) : 0;
  static constexpr int kBytes = std::max(kHalves * kHalf, kMerge);
  static constexpr uint32_t kRecord = kColumns * (D + 2);  // floats
  // Workgroups of a CU that pieces are made for (four: 16 FP16 rows of 513 to 4,000 with 9 nodes of 7
  // heads of 64 34.2 us, three 28.3).
  static constexpr int kPerCu = std::min(kWhole ? 1 : 3, static_cast<int>(kLds) / (kBytes + 2048));
  static_assert(WP <= 2 && kDmas >= 1 && kDmas * kRowsPerDma * kWaves == kStage, "whole transfers");
  static_assert((kHalves - 2) * kDmas < 64, "the wait's count");
  static_assert(kBytes + 2048 <= static_cast<int>(kLds) && kPerCu <= static_cast<int>(kTreePerCu), "LDS");
};

template <typename S>
struct TreeShared {
  __attribute__((aligned(1024))) char stage[S::kBytes];
  uint64_t mask[64];     // of each node
  uint64_t poison[128];  // nodes that see a value that is not finite, by dimension
  uint32_t errors, last;
};

// Where 16-byte chunk c of row r of a stage lies in its row: so that neither rows
// at one chunk (K) nor 4 x 4 rows at one pair of chunks (V) share banks.
template <int kRowBytes, bool kWide>
__device__ __forceinline__ uint32_t swizzle(uint32_t r) {
  if constexpr (kWide) return r & 7;
  return kRowBytes == 256 ? 2 * (r & 7) : 2 * (r >> 1 & 3);
}

template <typename E, int D, int NB, int WC, int WP>
struct TreeAttention {
  using S = TreeShape<E, D, NB, WC, WP>;
  using Shared = TreeShared<S>;
  static constexpr bool kWide = S::kWide;
  static constexpr int kStage = S::kStage, kRows = S::kRows;
  static constexpr int kQ = D * S::kElem / 64;  // 16-byte pieces of a query per lane

  const TreeLaunch &p;
  Shared &sh;
  Piece it;
  const int w, lane, col, quad, wc, wp;
  const float scale;  // of the sizes of scores, in powers of two: the queries have its sign
  const uint32_t token_bytes;
  u4v q[NB][kQ];
  f4v o[NB][S::kAcc];
  float m[NB], ms[NB], l[NB];
  uint32_t errors = 0;
  uint32_t lane_off[S::kDmas / S::kIds];  // of a lane's bytes in a group of 16 rows

  __device__ __forceinline__ TreeAttention(const TreeLaunch &launch, Shared &shared)
      : p(launch),
        sh(shared),
        w(__builtin_amdgcn_readfirstlane(wave_id())),
        lane(lane_id()),
        col(lane & 15),
        quad(lane >> 4),
        wc(w % WC),
        wp(w / WC),
        scale(fabsf(p.a.scale) * 1.44269504088896340736f),
        token_bytes(static_cast<uint32_t>(p.c.token_stride) * S::kElem) {
#pragma unroll
    for (int n = 0; n < S::kDmas / S::kIds; ++n) {
      const uint32_t row = n * S::kRowsPerDma + lane / S::kLanesPerRow;
      lane_off[n] = row * token_bytes + 16 * ((lane % S::kLanesPerRow) ^ swizzle<S::kRowBytes, kWide>(w * kRows + row));
    }
  }

  // A wave transfers rows of its own of each half.
  struct Ids {
    int32_t id[S::kIds];
  };
  // Their pages. (Past the length: the last position's.)
  __device__ __forceinline__ Ids pages_of(uint32_t stage) const {
    Ids x{};
    if (stage >= it.last) return x;
#pragma unroll
    for (int n = 0; n < S::kIds; ++n) {
      const uint32_t pos = min(stage * kStage + w * kRows + 16 * n, static_cast<uint32_t>(it.length - 1));
      x.id[n] = load_uniform(p.c.table + it.row * p.c.table_stride + (pos >> p.page_shift));
    }
    return x;
  }
  // K (0) or V (1) of a stage. Positions past the length read the last one: nothing behind it is
  // touched. (A group of 16 rows lies in one page: its address is the wave's, and a lane's share of it
  // is the same in every full group.)
  template <int kOf>
  __device__ __forceinline__ void load(uint32_t stage, const Ids &pages) {
    const uint32_t lds = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_char *)sh.stage)) +
                         (2 * (stage - it.first) + kOf) % S::kHalves * S::kHalf + w * kRows * S::kRowBytes;
    const int64_t head = static_cast<int64_t>(it.kv) * p.c.head_stride;
    constexpr int kPerGroup = S::kDmas / S::kIds;
#pragma unroll
    for (int g = 0; g < S::kIds; ++g) {
      const int32_t id = pages.id[g];
      const uint32_t first = stage * kStage + w * kRows + 16 * g;
      if (id < 0 || static_cast<uint32_t>(id) >= p.c.pages) {
        errors |= QD_PAGED_BAD_PAGE;
        continue;
      }
      const char *base = static_cast<const char *>(kOf ? p.c.v : p.c.k) + (id * p.c.page_stride + head) * S::kElem;
      if (first + std::min(kRows, 16) <= static_cast<uint32_t>(it.length)) {
        const char *group = base + static_cast<uint64_t>(first & (p.c.page_size - 1)) * token_bytes;
#pragma unroll
        for (int n = 0; n < kPerGroup; ++n) dma_to_lds(group, lane_off[n], lds + (g * kPerGroup + n) * 1024);
      } else {
#pragma unroll
        for (int n = 0; n < kPerGroup; ++n) {
          const uint32_t row = n * S::kRowsPerDma + lane / S::kLanesPerRow;
          const uint32_t pos = min(first + row, static_cast<uint32_t>(it.length - 1)) & (p.c.page_size - 1);
          dma_to_lds(base + (static_cast<uint64_t>(pos) * token_bytes + lane_off[n] - row * token_bytes), lds + (g * kPerGroup + n) * 1024);
        }
      }
    }
  }
  __device__ __forceinline__ const char *half(uint32_t stage, int of) const {
    return sh.stage + (2 * (stage - it.first) + of) % S::kHalves * S::kHalf;
  }
  __device__ __forceinline__ uint32_t column(int nb) const { return it.block * S::kColumns + (wc * NB + nb) * 16 + col; }
  __device__ __forceinline__ void load_queries() {
    const uint32_t sign = p.a.scale < 0.f ? kWide ? 0x80000000u : 0x80008000u : 0u;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const uint32_t c = column(nb);
      if (c < p.columns) {
        const uint32_t node = c / p.group, head = it.kv * p.group + c % p.group;
        const char *at = static_cast<const char *>(p.a.q) +
                         (it.row * p.a.q_stride + node * p.a.q_node_stride + head * p.a.q_head_stride) * S::kElem + 16 * quad;
#pragma unroll
        for (int s = 0; s < kQ; ++s) q[nb][s] = *reinterpret_cast<const u4v *>(at + 64 * s) ^ sign;
      } else {
#pragma unroll
        for (int s = 0; s < kQ; ++s) q[nb][s] = u4v{0u, 0u, 0u, 0u};
      }
    }
  }
  // Positions of the tree in a stage, and those past it: V's values that are not finite
  // make way for zeros, and the nodes that see them are marked.
  __device__ __forceinline__ void clean(uint32_t stage) {
    char *v = const_cast<char *>(half(stage, 1));
    const int base = stage * kStage;
    for (int i = threadIdx.x; i < kStage * S::kLanesPerRow; i += S::kThreads) {
      const int row = i / S::kLanesPerRow, node = base + row - it.start;
      if (node < 0) continue;
      u4v *at = reinterpret_cast<u4v *>(v + i * 16);
      u4v x = *at;
      bool found = false;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if constexpr (kWide) {
          found |= (x[c] & 0x7F800000u) == 0x7F800000u;
        } else {
          constexpr uint32_t e = std::is_same_v<E, Half> ? 0x7C00u : 0x7F80u;
          found |= (x[c] & e) == e || (x[c] >> 16 & e) == e;
        }
      }
      if (!found) continue;
      if (node >= static_cast<int>(p.a.nodes)) {
        *at = u4v{0u, 0u, 0u, 0u};
        continue;
      }
      uint64_t seen = 0;  // by these nodes
      for (uint32_t n = 0; n < p.a.nodes; ++n) seen |= (sh.mask[n] >> node & 1) << n;
      const uint32_t chunk = i % S::kLanesPerRow ^ swizzle<S::kRowBytes, kWide>(row);
      uint32_t y[4] = {x[0], x[1], x[2], x[3]};
      for (int d = 0; d < 16 / S::kElem; ++d) {
        if constexpr (kWide) {
          if ((y[d] & 0x7F800000u) != 0x7F800000u) continue;
          y[d] = 0u;
        } else {
          constexpr uint32_t e = std::is_same_v<E, Half> ? 0x7C00u : 0x7F80u;
          if ((y[d / 2] >> 16 * (d & 1) & e) != e) continue;
          y[d / 2] &= d & 1 ? 0xFFFFu : 0xFFFF0000u;
        }
        atomicOr(reinterpret_cast<unsigned long long *>(&sh.poison[chunk * (16 / S::kElem) + d]), static_cast<unsigned long long>(seen));
      }
      *at = u4v{y[0], y[1], y[2], y[3]};
    }
  }
  // The probabilities of this wave's half of a stage: pr[nb][s][r] of its position 16 s + 4 quad + r.
  template <bool kTree>
  __device__ __forceinline__ void weigh(uint32_t stage, float (&pr)[NB][2][4]) {
    const char *k = half(stage, 0) + wp * kStep * S::kRowBytes;
    const int base = stage * kStage + wp * kStep;
    f4v s[2][NB];
#pragma unroll
    for (int sub = 0; sub < 2; ++sub)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) s[sub][nb] = f4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int sub = 0; sub < 2; ++sub)
#pragma unroll
      for (int t = 0; t < kQ; ++t) {
        const uint32_t chunk = (4 * t + quad) ^ swizzle<S::kRowBytes, kWide>(col);
        const u4v a = *reinterpret_cast<const u4v *>(k + (16 * sub + col) * S::kRowBytes + 16 * chunk);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          if constexpr (kWide) {
            const f4v x = __builtin_bit_cast(f4v, a), y = __builtin_bit_cast(f4v, q[nb][t]);
#pragma unroll
            for (int c = 0; c < 4; ++c) s[sub][nb] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[c], y[c], s[sub][nb], 0, 0, 0);
          } else {
            s[sub][nb] = E::mfma(a, q[nb][t], s[sub][nb]);
          }
        }
      }
    float top[NB];
    bool rises = false;
    bool hidden[kTree ? NB : 1][2][4];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      if constexpr (kTree) {
        const uint32_t c = column(nb);
        const uint64_t mask = c < p.columns ? sh.mask[c / p.group] : 0ull;
#pragma unroll
        for (int sub = 0; sub < 2; ++sub)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int node = base + 16 * sub + 4 * quad + r - it.start;
            hidden[nb][sub][r] = node >= 0 && (node >= static_cast<int>(p.a.nodes) || !(mask >> node & 1));
            if (hidden[nb][sub][r]) s[sub][nb][r] = -INFINITY;
          }
      }
      float x = s[0][nb][0];
#pragma unroll
      for (int i = 1; i < 8; ++i) x = fmaxf(x, s[i >> 2][nb][i & 3]);
      top[nb] = kTree && x == -INFINITY ? x : x * scale;
      rises |= top[nb] > m[nb] + kLazy<E>;
    }
    if (__any(rises)) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const float n = fmaxf(m[nb], quarters_max(top[nb]));
        const float f = n == m[nb] ? 1.f : exp2_fast(m[nb] - n);
        m[nb] = n;
        ms[nb] = n == -INFINITY ? -kUnit<E> : n - kUnit<E>;
        l[nb] *= f;
#pragma unroll
        for (int j = 0; j < S::kAcc; ++j) o[nb][j] *= f;
      }
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      float sum = 0.f;
#pragma unroll
      for (int sub = 0; sub < 2; ++sub)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float x = exp2_fast(fmaf(s[sub][nb][r], scale, -ms[nb]));
          if constexpr (kTree)
            if (hidden[nb][sub][r]) x = 0.f;
          pr[nb][sub][r] = x;
          sum += x;
        }
      l[nb] += sum;
    }
  }
  __device__ __forceinline__ void accumulate(uint32_t stage, const float (&pr)[NB][2][4]) {
    const char *v = half(stage, 1) + wp * kStep * S::kRowBytes;
    if constexpr (kWide) {
#pragma unroll
      for (int sub = 0; sub < 2; ++sub)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const uint32_t row = 16 * sub + 4 * quad + r;
#pragma unroll
          for (int n = 0; n < D / 64; ++n) {
            const uint32_t chunk = (16 * n + col) ^ swizzle<S::kRowBytes, kWide>(row);
            const f4v a = *reinterpret_cast<const f4v *>(v + row * S::kRowBytes + 16 * chunk);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
              for (int c = 0; c < 4; ++c)
                o[nb][4 * n + c] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[c], pr[nb][sub][r], o[nb][4 * n + c], 0, 0, 0);
          }
        }
    } else {
      // Probabilities as two numbers of the type, rounded and what that left, as in the
      // attention of one token.
      u4v b[NB], rest[NB];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x = pr[nb][i >> 1][2 * (i & 1)], y = pr[nb][i >> 1][2 * (i & 1) + 1];
          b[nb][i] = E::pack(x, y);
          rest[nb][i] = E::pack(x - E::lo(b[nb][i]), y - E::hi(b[nb][i]));
        }
#pragma unroll
      for (int j = 0; j < S::kAcc; ++j) {
        u4v a;
#pragma unroll
        for (int sub = 0; sub < 2; ++sub) {
          const uint32_t row = 16 * sub + 4 * quad + (col >> 2);
          const uint32_t chunk = (2 * j + (col >> 1 & 1)) ^ swizzle<S::kRowBytes, kWide>(row);
          const s4v x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4v *)(v + row * S::kRowBytes + 16 * chunk + 8 * (col & 1)));
          const u2v y = __builtin_bit_cast(u2v, x);
          a[2 * sub] = y[0];
          a[2 * sub + 1] = y[1];
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          o[nb][j] = E::mfma(a, rest[nb], o[nb][j]);
          o[nb][j] = E::mfma(a, b[nb], o[nb][j]);
        }
      }
    }
  }
  // All but one half (a stage) of what LDS holds is on its way when this returns.
  static constexpr int kFirst = S::kHalves / 2 - !S::kByHalves;  // stages
  Ids ahead;  // the pages of the stage that is loaded next
  __device__ __forceinline__ void begin() {
    if (it.length == 0) return;
    Ids early[kFirst];
#pragma unroll
    for (int i = 0; i < kFirst; ++i) early[i] = pages_of(it.first + i);
#pragma unroll
    for (int i = 0; i < kFirst; ++i) {
      if (it.first + i >= it.last) break;
      load<0>(it.first + i, early[i]);
      if (!S::kByHalves || S::kHalves % 2 || i + 1 < kFirst) load<1>(it.first + i, early[i]);
    }
    ahead = S::kByHalves && S::kHalves % 2 == 0 ? early[kFirst - 1] : pages_of(it.first + kFirst);
  }
  template <bool kTree>
  __device__ __forceinline__ void stage_through(uint32_t stage) {
    // (The last stage's second half may lie behind the row.)
    const bool some = WP == 1 || static_cast<int>(stage * kStage + wp * kStep) < it.length;
    const uint32_t more = it.last - 1 - stage;  // stages behind this one
    float pr[NB][2][4];
    if constexpr (S::kByHalves) {
      // A half that is read makes room for the one kHalves - 1 behind it.
      dma_wait<S::kDmas, S::kHalves - 2>(1 + 2 * more);
      lds_barrier();
      if constexpr (S::kHalves % 2) {
        if (more >= kFirst) load<0>(stage + kFirst, ahead);
      } else if (more >= kFirst - 1) {
        load<1>(stage + kFirst - 1, ahead);
        ahead = pages_of(stage + kFirst);
      }
      weigh<kTree>(stage, pr);
      dma_wait<S::kDmas, S::kHalves - 2>(2 * more);
      lds_barrier();
      if (more >= kFirst) {
        if constexpr (S::kHalves % 2) {
          load<1>(stage + kFirst, ahead);
          ahead = pages_of(stage + kFirst + 1);
        } else {
          load<0>(stage + kFirst, ahead);
        }
      }
    } else {
      dma_wait<2 * S::kDmas, kFirst - 1>(more);
      lds_barrier();
      if (more >= kFirst) {
        load<0>(stage + kFirst, ahead);
        load<1>(stage + kFirst, ahead);
        ahead = pages_of(stage + kFirst + 1);
      }
      if (some) weigh<kTree>(stage, pr);
    }
    if constexpr (kTree) {
      clean(stage);
      lds_barrier();
    }
    if (some) accumulate(stage, pr);
  }
  __device__ __forceinline__ void run() {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      m[nb] = -INFINITY;
      ms[nb] = -kUnit<E>;
      l[nb] = 0.f;
#pragma unroll
      for (int j = 0; j < S::kAcc; ++j) o[nb][j] = f4v{0.f, 0.f, 0.f, 0.f};
    }
    if (it.length) {
      uint32_t stage = it.first;
      const uint32_t plain = min(it.last, static_cast<uint32_t>(it.start) / kStage);  // stages before the tree
      for (; stage < plain; ++stage) stage_through<false>(stage);
      for (; stage < it.last; ++stage) stage_through<true>(stage);
    }
    lds_barrier();
  }
  // First dimension of this lane's i-th four of an accumulator.
  static __device__ __forceinline__ int dim_of(int i) {
    const int quad = lane_id() >> 4;
    return kWide ? 64 * (i >> 2) + 4 * (4 * quad + (i & 3)) : 16 * i + 4 * quad;
  }
  __device__ __forceinline__ float4 four(int nb, int i) const {
    if constexpr (kWide)
      return make_float4(o[nb][i & ~3][i & 3], o[nb][(i & ~3) + 1][i & 3], o[nb][(i & ~3) + 2][i & 3], o[nb][(i & ~3) + 3][i & 3]);
    else
      return make_float4(o[nb][i][0], o[nb][i][1], o[nb][i][2], o[nb][i][3]);
  }
  // The sums of a stage's two waves together, in the first WC waves.
  __device__ __forceinline__ void merge() {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) l[nb] = quarters_sum(l[nb]);
    if constexpr (WP == 1) {
      __syncthreads();
      return;
    }
    constexpr int kShare = NB * (S::kAcc * 1024 + 512);
    char *at = sh.stage + wc * kShare;
    if (wp > 0) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int j = 0; j < S::kAcc; ++j) *reinterpret_cast<f4v *>(at + (nb * S::kAcc + j) * 1024 + lane * 16) = o[nb][j];
        *reinterpret_cast<float2 *>(at + NB * S::kAcc * 1024 + nb * 512 + lane * 8) = make_float2(m[nb], l[nb]);
      }
    }
    __syncthreads();
    if (wp > 0) return;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const float2 x = *reinterpret_cast<const float2 *>(at + NB * S::kAcc * 1024 + nb * 512 + lane * 8);
      const float top = fmaxf(m[nb], x.x);
      const float f = m[nb] == top ? 1.f : exp2_fast(m[nb] - top), g = x.x == top ? 1.f : exp2_fast(x.x - top);
      l[nb] = fmaf(g, x.y, l[nb] * f);
#pragma unroll
      for (int j = 0; j < S::kAcc; ++j) {
        const f4v y = *reinterpret_cast<const f4v *>(at + (nb * S::kAcc + j) * 1024 + lane * 16);
#pragma unroll
        for (int c = 0; c < 4; ++c) o[nb][j][c] = fmaf(g, y[c], o[nb][j][c] * f);
      }
      m[nb] = top;
    }
  }
  // Column c's four outputs from dimension d on.
  __device__ __forceinline__ void emit(uint32_t c, int d, float4 acc, float sum, float poison) const {
    const uint32_t node = c / p.group, head = it.kv * p.group + c % p.group;
    const bool there = !it.bad && it.length > 0 && sh.mask[node] != 0;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (there) {
      const float inv = 1.f / sum;
      x = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
    }
    if (poison != 0.f) x = make_float4(poison, poison, poison, poison);  // NaN
    store4<E>(p.a.out, it.row * p.a.out_stride + node * p.a.out_node_stride + head * p.a.out_head_stride + d, x);
  }
  // A record is as the lanes hold it, whole lines at a time: [block of 16 columns][four][lane] float4,
  // then each column's maximum and sum.
  static constexpr uint32_t kFours = S::kAcc * kWave, kRecord = S::kRecord;  // float4 of 16 columns
  __device__ __forceinline__ uint32_t record_four(int nb, int i) const { return (wc * NB + nb) * kFours + i * kWave + lane; }
  __device__ __forceinline__ uint32_t record_sums(int nb) const { return S::kColumns * D + ((wc * NB + nb) * 16 + col) * 2; }
  // The piece's result, out or to its record.
  __device__ __forceinline__ void put(float *record) {
    const float nan = __uint_as_float(kNan);
    const bool spoilt = sh.errors != 0, whole = it.pieces == 1;
    const bool tree = static_cast<int>(it.last * kStage) > it.start && it.length > 0;
    if (threadIdx.x == 0 && spoilt) raise_error(p.c.errors, sh.errors);
    if (wp > 0) return;
    const Coherent rec(record, kRecord * static_cast<uint32_t>(sizeof(float)));
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const uint32_t c = column(nb);
      const uint32_t node = min(c / p.group, p.a.nodes - 1);
#pragma unroll
      for (int i = 0; i < S::kAcc; ++i) {
        const int d = dim_of(i);
        float4 x = four(nb, i);
        if (tree) {
          if (sh.poison[d] >> node & 1) x.x = nan;
          if (sh.poison[d + 1] >> node & 1) x.y = nan;
          if (sh.poison[d + 2] >> node & 1) x.z = nan;
          if (sh.poison[d + 3] >> node & 1) x.w = nan;
        }
        if (!whole)
          rec.st4(record_four(nb, i), x);
        else if (c < p.columns)
          emit(c, d, x, l[nb], spoilt ? nan : 0.f);
      }
      if (!whole && quad == 0) {
        rec.st(record_sums(nb), spoilt ? nan : m[nb]);
        rec.st(record_sums(nb) + 1, l[nb]);
      }
    }
  }
  // Counts the piece in; true in the workgroup whose piece came last.
  __device__ __forceinline__ bool arrive() {
    wait_vm_stores();
    __syncthreads();
    uint32_t *cnt = p.counters + (static_cast<size_t>(it.row) * p.parts + it.kv * p.blocks + it.block) * p.apart;
    if (threadIdx.x == 0) {
      sh.last = atomicAdd(cnt, 1u) == it.pieces - 1;
      if (sh.last) *cnt = 0u;
    }
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(sh.last);
  }
  // Joins the pieces in their order, each wave its columns (of two waves at the same ones each half of the
  // dimensions).
  __device__ __forceinline__ void join(const float *first, uint32_t second, uint32_t stride) {
    constexpr int kMine = S::kAcc / WP, kAhead = 4;  // fours of a lane; pieces on their way
    const uint32_t n = it.pieces;
    const Coherent rec(first, (second + (n - 2) * stride + kRecord) * static_cast<uint32_t>(sizeof(float)));
    const float nan = __uint_as_float(kNan);
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      float4 acc[kMine];
      float top = -INFINITY, sum = 0.f;
      bool spoilt = false;
#pragma unroll
      for (int i = 0; i < kMine; ++i) acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      for (uint32_t u0 = 0; u0 < n; u0 += kAhead) {
        float mu[kAhead], lu[kAhead];
        float4 x[kAhead][kMine];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
          const uint32_t u = min(u0 + a, n - 1), at = u == 0 ? 0u : second + (u - 1) * stride;
          mu[a] = rec.ld(at + record_sums(nb));
          lu[a] = rec.ld(at + record_sums(nb) + 1);
#pragma unroll
          for (int i = 0; i < kMine; ++i) x[a][i] = rec.ld4(at / 4 + record_four(nb, wp * kMine + i));
        }
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
          if (u0 + a >= n) break;
          spoilt |= mu[a] != mu[a];
          const float t = fmaxf(top, mu[a]);
          const float g = top == t ? 1.f : exp2_fast(top - t), f = mu[a] == t ? 1.f : exp2_fast(mu[a] - t);
          top = t;
          sum = fmaf(f, lu[a], sum * g);
#pragma unroll
          for (int i = 0; i < kMine; ++i) {
            acc[i].x = fmaf(f, x[a][i].x, acc[i].x * g);
            acc[i].y = fmaf(f, x[a][i].y, acc[i].y * g);
            acc[i].z = fmaf(f, x[a][i].z, acc[i].z * g);
            acc[i].w = fmaf(f, x[a][i].w, acc[i].w * g);
          }
        }
      }
      const uint32_t c = column(nb);
      if (c >= p.columns) continue;
#pragma unroll
      for (int i = 0; i < kMine; ++i) emit(c, dim_of(wp * kMine + i), acc[i], sum, spoilt ? nan : 0.f);
    }
  }
};

// The row of a piece, of length n.
__device__ __forceinline__ void set_row(const TreeLaunch &p, Piece &it, uint32_t row, int32_t n) {
  it.row = row;
  it.bad = n != 0 && (n < static_cast<int32_t>(p.a.nodes) || n > static_cast<int64_t>(p.c.table_width) << p.page_shift);
  it.length = it.bad ? 0 : n;
  it.start = it.length - static_cast<int>(p.a.nodes);
}

// The one piece that a workgroup takes: rows are cut into pieces of `size` stages, as few as let
// all of them be on the card at once (p.target of one item); where rows alone are a quarter of
// that, four times as many, since each place takes several of them then.
template <int kStage>
__device__ __forceinline__ bool find_piece(const TreeLaunch &p, Piece &it) {
  // Consecutive workgroups go to consecutive XCDs: the heads and blocks of a piece come to one.
  const uint32_t xcd = blockIdx.x % kXcds, idx = blockIdx.x / kXcds;
  const uint32_t x = idx / p.parts * kXcds + xcd;
  if (x >= p.units) return false;
  it.block = idx % p.blocks;
  it.kv = idx / p.blocks % p.c.kv_heads;
  const int lane = lane_id();
  const int64_t most = static_cast<int64_t>(p.c.table_width) << p.page_shift;
  const auto stages_of = [&](int32_t n) { return tiles_of<kStage>(p, n, most); };
  uint32_t size = 0x7fffffffu, row = x;
  int32_t n = 0;
  it.number = x;
  it.pieces = 1;
  if (p.target) {
    uint32_t total = 0, longest = 0;
    for (uint32_t r = lane; r < p.c.rows; r += kWave) {
      n = p.c.lengths[r];
      total += stages_of(n);
      longest = max(longest, stages_of(n));
    }
    total = __builtin_amdgcn_readlane(lanes_upto(total), kWave - 1);
    const bool once = p.c.rows <= kWave, few = 4 * p.c.rows <= p.target;
    const uint32_t aim = few ? p.target : 4 * p.target;
    size = max(max(kTreeLeast / kStage, (total + aim - 1) / aim), (lanes_max(longest) + kTreePieces - 1) / kTreePieces);
    const auto pieces_of = [&](uint32_t r, int32_t length) { return r < p.c.rows ? (stages_of(length) + size - 1) / size : 0u; };
    if (few && once)  // (a size of total / (target - rows) will do)
      while (__builtin_amdgcn_readlane(lanes_upto(pieces_of(lane, n)), kWave - 1) > p.target) size += max(1u, size / 16);
    uint32_t base = 0, upto, mine;
    it.number = 0;
    uint64_t past;
    for (;; base += kWave) {
      if (base >= p.c.rows) return false;
      if (!once) n = base + lane < p.c.rows ? p.c.lengths[base + lane] : 0;
      mine = pieces_of(base + lane, n);
      upto = lanes_upto(mine);
      past = __ballot(it.number + upto > x);
      if (past) break;
      it.number += __builtin_amdgcn_readlane(upto, kWave - 1);
    }
    const int at = __ffsll(static_cast<unsigned long long>(past)) - 1;
    row = base + at;
    it.number += __builtin_amdgcn_readlane(upto - mine, at);
    n = __builtin_amdgcn_readlane(n, at);
    it.pieces = __builtin_amdgcn_readlane(mine, at);
  } else {
    n = load_uniform(p.c.lengths + row);
  }
  set_row(p, it, row, n);
  it.index = x - it.number;
  const uint32_t stages = stages_of(n);
  it.first = it.pieces == 1 ? 0 : it.index * size;
  it.last = it.pieces == 1 ? stages : min(stages, it.first + size);
  return true;
}

template <typename E, int D, int NB, int WC, int WP>
__global__ __launch_bounds__(WC *WP *kWave) void tree_attention_kernel(TreeLaunch p) {
  using S = TreeShape<E, D, NB, WC, WP>;
  __shared__ TreeShared<S> sh;
  constexpr uint32_t kRecord = S::kRecord;
  TreeAttention<E, D, NB, WC, WP> a(p, sh);
  // (Told to the compiler: all lanes have the same.)
  const auto same = [](auto v) __attribute__((always_inline)) { return __builtin_amdgcn_readfirstlane(v); };
  const auto piece_of = [&](const Item &item) __attribute__((always_inline)) {
    Piece x;
    set_row(p, x, same(item.row), same(item.bad ? -1 : item.length));
    x.kv = same(item.part) / p.blocks;
    x.block = same(item.part) % p.blocks;
    x.first = same(item.first);
    x.last = same(item.last);
    x.pieces = same(item.pieces);
    x.number = same(item.home);
    x.index = x.pieces > 1 ? blockIdx.x - x.number : 0;
    return x;
  };
  // (A stage of two waves has no runs: its columns are so many that products bound it.)
  const bool single = S::kWhole || p.units;
  Deal deal{};
  Item item{};
  if (single) {
    if (!find_piece<S::kStage>(p, a.it)) return;
  } else {
    if (!same(first_item<S::kStage>(p, blockIdx.x, gridDim.x, deal, item) ? 1 : 0)) return;
    a.it = piece_of(item);
  }
  a.begin();
  for (;;) {
    a.load_queries();
    if (threadIdx.x == 0) sh.errors = 0;
    for (int i = threadIdx.x; i < 128; i += S::kThreads) sh.poison[i] = 0;
    if (a.w == 0) {
      bool bad;
      const uint64_t mask = ancestors(p.a.parents + static_cast<size_t>(a.it.row) * p.a.nodes, p.a.nodes, bad);
      sh.mask[a.lane] = mask;
      if (bad && (a.it.length || a.it.bad)) a.errors |= QD_TREE_BAD_PARENT;  // (a row of nothing may have any)
    }
    if (a.it.bad) a.errors |= QD_PAGED_BAD_LENGTH;
    a.run();
    if (a.errors && a.lane == 0) atomicOr(&sh.errors, a.errors);
    a.merge();
    // The next piece's loads are under way while this one's results are put together.
    const Piece now = a.it;
    Item next{};
    const bool more = !single && same(next_item<S::kStage>(p, deal, blockIdx.x, item, next) ? 1 : 0);
    uint32_t errors = 0;
    if (more) {
      a.it = piece_of(next);
      a.errors = 0;
      a.begin();
      errors = a.errors;
    }
    const Piece then = a.it;
    a.it = now;
    // Records: of pieces of an item one after the other; or (equal runs) a workgroup's first where a
    // piece begins inside its item, else the second.
    float *first;
    uint32_t second, stride;
    if (single) {
      first = p.records + (static_cast<size_t>(now.number) * p.parts + now.kv * p.blocks + now.block) * kRecord;
      second = stride = p.parts * kRecord;
    } else {
      first = p.records + (2 * static_cast<size_t>(now.number) + 1) * kRecord;
      second = kRecord;
      stride = 2 * kRecord;
    }
    a.put(first + (now.index ? second + static_cast<size_t>(now.index - 1) * stride : 0));
    if (now.pieces > 1 && a.arrive()) a.join(first, second, stride);
    if (!more) break;
    a.it = then;
    a.errors = errors;
    item = next;
    __syncthreads();  // the masks and marks are written again
  }
}

struct TreePlan {
  uint32_t group, columns, blocks, apart, target, records;
  bool few;  // rows, for pieces of one item that the card holds at once
};

// Calls f with the shape and kernel for so many columns. A wave of 32 columns has 340 registers and
// its SIMD to itself, which only more than 64 columns make up for (64 BF16 rows of 0 to 8,192, 8 KV heads
// of 128: 64 columns by four waves of 16 253 us, by two of 32 319, by the eight of 128 columns 294; 128
// columns by those 312, as two blocks of four waves 410; two rows of 1,000: 64 columns 18.5, 31 and 26,
// 128 28 and 21.5). Up to 32 columns two waves (16 columns by one wave 203 us and 18.0, by these
// 212 and 17.3; FP32, 16 rows of 513 to 4,000 with 14 columns 31.7 and 28.9; 28 columns by four 30.1,
// by two 29.0).
template <typename E, int D, typename F>
auto with_shape(uint32_t columns, F &&f) {
  const auto shape = [&](auto nb, auto wc, auto wp) {
    constexpr int NB = decltype(nb)::value, WC = decltype(wc)::value, WP = decltype(wp)::value;
    return f(TreeShape<E, D, NB, WC, WP>{}, tree_attention_kernel<E, D, NB, WC, WP>);
  };
  std::integral_constant<int, 1> one;
  std::integral_constant<int, 2> two;
  std::integral_constant<int, 4> four;
  if (columns <= 32) return shape(one, two, one);
  if constexpr (std::is_same_v<E, float>) {
    return shape(one, four, one);
  } else {
    return columns <= 64 ? shape(one, four, one) : shape(two, four, two);
  }
}
template <typename F>
auto with_type(uint32_t dtype, uint32_t head_dim, uint32_t columns, F &&f) {
  const bool wide = head_dim == 128;
  switch (dtype) {
    case QD_DTYPE_F32: return wide ? with_shape<float, 128>(columns, f) : with_shape<float, 64>(columns, f);
    case QD_DTYPE_BF16: return wide ? with_shape<Brain, 128>(columns, f) : with_shape<Brain, 64>(columns, f);
    default: return wide ? with_shape<Half, 128>(columns, f) : with_shape<Half, 64>(columns, f);
  }
}

// What a launch of shape S does, and the records that it can write: no more pieces than one of each row and `target`
// more, four times as many where rows are not few, or two of each workgroup that equal runs go to.
template <typename S>
TreePlan tree_plan(uint32_t rows, uint32_t nodes, uint32_t heads, uint32_t kv_heads) {
  TreePlan s{};
  s.group = heads / kv_heads;
  s.columns = nodes * s.group;
  s.blocks = (s.columns + S::kColumns - 1) / S::kColumns;
  const uint32_t parts = kv_heads * s.blocks;
  const uint64_t items = static_cast<uint64_t>(rows) * parts;
  if (items > kOpCounters) return s;
  for (s.apart = 32; items * s.apart > kOpCounters;) s.apart /= 2;
  // FP32's products bound it: no more pieces than CUs (16 rows of 576 with 16 nodes 19.1 us, as
  // many as the card holds 22.9).
  constexpr uint32_t kAim = S::kWide ? 1 : S::kPerCu;
  const uint32_t target = std::max(1u, std::max(1u, kTreePerCu * kTreeCus / parts) * kAim / kTreePerCu);
  // A join's offsets and its buffer have 32 bits: rows of so many items that they would not do stay whole.
  if (std::min(kTreePieces, 1 + 4 * target) * (parts * S::kRecord * sizeof(float)) > UINT32_MAX) return s;
  s.target = target;
  s.few = 4ull * rows <= target;
  s.records = (s.few ? rows + target : rows + 4 * target) * parts;
  if (S::kByHalves && s.blocks == 1 && !s.few) s.records = std::max(s.records, 2 * kTreeCus * S::kPerCu);
  return s;
}

// ---- accept ------------------------------------------------------------------------
// A workgroup takes a share of one node's logits, a quarter of it each wave: the largest, or
// (draws) each wave's sum of exp(x / T) in 64 bits, relative to a power of two above its largest. Greedy, the last
// share of a row to arrive finds each node's largest and walks the tree; with draws the last
// share of a node finds the quarter in which the running sum passes the draw, reads that one
// again and picks the token, and the last node of a row walks. Bound by memory for large
// batches (16 drawn trees of 16 over 151,936 tokens in FP32, 130 MB, 37 us; arithmetic left out
// changed nothing; in BF16 28 us), by the chain of hand-overs for small ones (a tree of 8 6.5 us).
constexpr int kAcceptT = 256, kAcceptWaves = kAcceptT / kWave;
constexpr uint32_t kAcceptShares = 64;    // of a node at most: a lane each
// (1,024: 16 drawn trees of 16 41 us instead of 38, 4,096 44)
constexpr uint32_t kAcceptAim = 2048;     // shares in all
// (4,096: one tree of 8 9.1 us instead of 6.5, 8,192 6.9, 32,768 7.3: arrivals at one counter)
constexpr uint32_t kAcceptLeast = 16384;  // logits of a share at least
constexpr float kHuge = 1e30f;            // logits past it are not exponentiated
// Where the largest logit's x c is past this either way, sums are relative to that logit, not to a whole number.
constexpr float kFar = 0x1p22f;

struct AcceptShare {
  double sum[kAcceptWaves];  // each wave's, of 2^(x c - r), r the whole number above the x c of
  float top[kAcceptWaves];   // its largest logit. Greedy: the share's largest, and its token's bits
};
struct AcceptLaunch {
  qd_accept_args a;
  AcceptShare *share;   // [rows * nodes][shares]
  int32_t *picks;       // [rows * nodes]
  uint32_t *counters;   // [rows * nodes] nodes, then [rows] rows
  uint32_t apart;       // words between two counters
  uint32_t shares;
  float c_hi, c_lo;     // log2(e) / temperature
  float most;           // 2 kFar / c
};

// A row's logit i as FP32.
template <typename E>
__device__ __forceinline__ float logit(const void *row, uint32_t i) {
  if constexpr (std::is_same_v<E, float>) {
    return static_cast<const float *>(row)[i];
  } else {
    const uint32_t v = static_cast<const uint16_t *>(row)[i];
    return E::lo(v);
  }
}
// The whole number above x c, of a sum whose largest logit is x. Logits count as +-2 kFar / c where they are past it, -inf
// and NaN too: x c is at least kFar below the largest then, and the number has FP32's 24 bits.
__device__ __forceinline__ float whole_above(const AcceptLaunch &p, float x) {
  return ceilf(fminf(fmaxf(x, -p.most), p.most) * p.c_hi);
}
// 2^(x c - r), x no larger than the logit that r stands above. Two roundings of an exponent -d, 2^-24 of it each, and the
// exponential's 2^-23: off by (1.4 d + 4) 2^-24 of itself. (r is subtracted inside: a product that is rounded first can be
// contracted with what follows, and is then corrected twice.)
__device__ __forceinline__ float power(const AcceptLaunch &p, float x, float r) {
  x = fmaxf(x, -p.most);
  return exp2_fast(fmaf(x, p.c_lo, fmaf(x, p.c_hi, -r)));
}
// The same relative to the largest logit itself: where x c is past kFar, differences of logits are what is exact. Off by
// (1.8 d + 2) 2^-24 of itself: the difference, c and their product.
__device__ __forceinline__ float power_far(const AcceptLaunch &p, float x, float top) { return exp2_fast((fmaxf(x, -INFINITY) - top) * p.c_hi); }
__device__ __forceinline__ double scaled(double s, float by) { return ldexp(s, static_cast<int>(fmaxf(by, -4000.f))); }
// Sum over the lanes up to this one.
__device__ __forceinline__ double lanes_upto(double v) {
#pragma unroll
  for (int step = 1; step < kWave; step <<= 1) {
    const double x = lane_of(v, max(lane_id() - step, 0));
    if (lane_id() >= step) v += x;
  }
  return v;
}

// One row's logits in 16-byte pieces, shares of them and quarters of shares. The row may start
// anywhere: the first quarter has what lies before the first piece too, the last one what lies
// behind the last.
template <typename E>
struct Logits {
  static constexpr int kPer = std::is_same_v<E, float> ? 4 : 8;
  const char *x;
  uint32_t vocab, head, pieces, each;
  __device__ __forceinline__ Logits(const char *at, uint32_t n, uint32_t quarters) : x(at), vocab(n) {
    const uint32_t skew = static_cast<uint32_t>(-(reinterpret_cast<uintptr_t>(x) / (16 / kPer))) % kPer;
    head = min(skew, vocab);
    pieces = (vocab - head) / kPer;
    each = (pieces + quarters - 1) / quarters;
  }
  __device__ __forceinline__ uint32_t first(uint32_t quarter) const { return min(pieces, quarter * each); }
  __device__ __forceinline__ uint32_t token(uint32_t piece) const { return head + piece * kPer; }
  __device__ __forceinline__ u4v load(uint32_t piece) const { return reinterpret_cast<const u4v *>(x + head * (16 / kPer))[piece]; }
  static __device__ __forceinline__ void values(const u4v &v, float (&y)[kPer]) {
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
};

template <typename E, bool kSampled>
__global__ __launch_bounds__(kAcceptT) void accept_kernel(AcceptLaunch p) {
  using Row = Logits<E>;
  constexpr int kPer = Row::kPer, kAhead = 4;
  __shared__ double sums[kAcceptWaves];
  __shared__ float tops[kAcceptWaves];
  __shared__ uint32_t ids[kAcceptWaves], last;
  __shared__ int32_t picks[64];
  const uint32_t node = blockIdx.y % p.a.nodes, row = blockIdx.y / p.a.nodes, share = blockIdx.x;
  const int lane = lane_id(), w = __builtin_amdgcn_readfirstlane(wave_id());
  const size_t at = static_cast<size_t>(row) * p.a.nodes;
  const int32_t parent = static_cast<uint32_t>(lane) < p.a.nodes ? p.a.parents[at + lane] : -2;
  const Row x(static_cast<const char *>(p.a.logits) + (row * p.a.row_stride + node * p.a.node_stride) * static_cast<int64_t>(16 / kPer),
              p.a.vocab, p.shares * kAcceptWaves);
  const uint32_t quarter = share * kAcceptWaves + w, from = x.first(quarter), to = x.first(quarter + 1);
  // (On their way before the tree is looked at.)
  u4v v[kAhead];
  const auto fetch = [&](uint32_t j) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) v[u] = x.load(min(j + u * kWave, to - 1));
  };
  if (from < to) fetch(from + lane);
  const uint64_t there = __ballot(parent >= -1);
  const bool bad = __any(parent >= lane || (parent >= 0 && !(there >> parent & 1)));
  if (bad || !(there & 1)) {
    if (node == 0 && share == 0) {
      if (bad && threadIdx.x == 0) raise_error(p.a.errors, QD_TREE_BAD_PARENT);
      if (threadIdx.x < p.a.nodes) p.a.path[at + threadIdx.x] = -1;
      if (threadIdx.x == 0) {
        p.a.counts[row] = 0;
        p.a.next_tokens[row] = -1;
      }
    }
    return;
  }
  if (!(there >> node & 1)) return;
  const uint32_t present = __popcll(there);
  float top = -INFINITY;
  uint32_t best = UINT32_MAX;
  double sum = 0.0;
  float r = kSampled ? whole_above(p, -INFINITY) : 0.f;
  const auto take = [&](float y, uint32_t i) {
    if (y > top) {
      top = y;
      best = i;
    }
  };
  // Raises r to the largest logit so far.
  const auto raise = [&](float most) {
    if (most > top) {
      top = most;
      const float up = whole_above(p, most);
      if (up > r) {
        sum = scaled(sum, r - up);
        r = up;
      }
    }
  };
  const auto single = [&](uint32_t i) {
    const float y = logit<E>(x.x, i);
    if constexpr (kSampled) {
      raise(y);
      sum += power(p, y, r);
    } else {
      take(y, i);
    }
  };
  if (quarter == 0 && static_cast<uint32_t>(lane) < x.head) single(lane);
  for (uint32_t j = from + lane; j < to; j += kAhead * kWave) {
    u4v now[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) now[u] = v[u];
    if (j + kAhead * kWave < to) fetch(j + kAhead * kWave);
    if constexpr (kSampled) {
      float most = -INFINITY;
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        float y[kPer];
        Row::values(now[u], y);
#pragma unroll
        for (int i = 0; i < kPer; ++i) most = fmaxf(most, y[i]);  // (a piece past the end is the last one again)
      }
      raise(most);
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (j + u * kWave >= to) break;
        float y[kPer];
        Row::values(now[u], y);
        // In pairs: three roundings at most.
#pragma unroll
        for (int i = 0; i < kPer; ++i) y[i] = power(p, y[i], r);
#pragma unroll
        for (int step = 1; step < kPer; step *= 2)
#pragma unroll
          for (int i = 0; i < kPer; i += 2 * step) y[i] += y[i + step];
        sum += y[0];
      }
    } else {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const uint32_t k = j + u * kWave;
        if (k >= to) break;
        float y[kPer];
        Row::values(now[u], y);
#pragma unroll
        for (int i = 0; i < kPer; ++i) take(y[i], x.token(k) + i);
      }
    }
  }
  if (quarter + 1 == p.shares * kAcceptWaves && x.token(x.pieces) + lane < p.a.vocab) single(x.token(x.pieces) + lane);
  // The workgroup's share.
  constexpr uint32_t kWords = sizeof(AcceptShare) / 4;
  const Coherent shares(p.share + at * p.shares, static_cast<uint32_t>(p.a.nodes * p.shares * sizeof(AcceptShare)));
  const auto word = [&](uint32_t n, uint32_t s) { return (n * p.shares + s) * kWords; };
  const uint32_t mine = word(node, share);
  if constexpr (kSampled) {
    const float wave_top = wave_max(top);
    double s = scaled(sum, r - whole_above(p, wave_top));
#pragma unroll
    for (int step = 32; step > 0; step >>= 1) s += lane_of(s, lane ^ step);
    if (lane == 0) {
      const uint64_t bits = __builtin_bit_cast(uint64_t, s);
      shares.stu(mine + 2 * w, static_cast<uint32_t>(bits));
      shares.stu(mine + 2 * w + 1, static_cast<uint32_t>(bits >> 32));
      shares.st(mine + 2 * kAcceptWaves + w, wave_top);
    }
  } else {
    const float wave_top = wave_max(top);
    // The lowest token of those that reach it.
    best = top == wave_top ? best : UINT32_MAX;
#pragma unroll
    for (int step = 32; step > 0; step >>= 1) best = min(best, static_cast<uint32_t>(__builtin_amdgcn_ds_bpermute((lane ^ step) << 2, static_cast<int>(best))));
    if (lane == 0) {
      tops[w] = wave_top;
      ids[w] = best;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      float all = tops[0];
      best = ids[0];
#pragma unroll
      for (int u = 1; u < kAcceptWaves; ++u)
        if (better(tops[u], ids[u], all, best)) {
          all = tops[u];
          best = ids[u];
        }
      shares.st(mine + 2 * kAcceptWaves, all);
      shares.stu(mine + 2 * kAcceptWaves + 1, best);
    }
  }
  const auto arrive = [&](uint32_t *counter, uint32_t of) {
    wait_vm_stores();
    __syncthreads();
    if (threadIdx.x == 0) {
      last = atomicAdd(counter, 1u) == of - 1;
      if (last) *counter = 0u;
    }
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(last) != 0;
  };
  uint32_t *row_counter = p.counters + (static_cast<size_t>(p.a.rows) * p.a.nodes + row) * p.apart;
  if constexpr (!kSampled) {
    if (!arrive(row_counter, present * p.shares)) return;
    // A group of lanes takes a node, a lane a share.
    const uint32_t lanes = p.shares <= 1 ? 1u : 1u << (32 - __builtin_clz(p.shares - 1));
    for (uint32_t n = threadIdx.x / lanes; n < (p.a.nodes + kAcceptT / lanes - 1) / (kAcceptT / lanes) * (kAcceptT / lanes); n += kAcceptT / lanes) {
      const uint32_t s = threadIdx.x % lanes;
      float y = -INFINITY;
      uint32_t i = UINT32_MAX;
      if (n < p.a.nodes && there >> n & 1 && s < p.shares) {
        y = shares.ld(word(n, s) + 2 * kAcceptWaves);
        i = shares.ldu(word(n, s) + 2 * kAcceptWaves + 1);
      }
      for (uint32_t step = lanes / 2; step > 0; step >>= 1) {
        const float z = __builtin_bit_cast(float, __builtin_amdgcn_ds_bpermute((lane ^ step) << 2, __builtin_bit_cast(int, y)));
        const uint32_t k = __builtin_amdgcn_ds_bpermute((lane ^ step) << 2, static_cast<int>(i));
        if (better(z, k, y, i)) {
          y = z;
          i = k;
        }
      }
      if (s == 0 && n < p.a.nodes) picks[n] = i == UINT32_MAX ? 0 : static_cast<int32_t>(i);  // (nothing above -inf)
    }
    __syncthreads();
    if (w != 0) return;
  } else {
    if (!arrive(p.counters + (at + node) * p.apart, p.shares)) return;
    // Every wave: all shares, a lane each.
    float largest[kAcceptWaves], most = -INFINITY;
    double part[kAcceptWaves] = {}, s = 0.0;
#pragma unroll
    for (int u = 0; u < kAcceptWaves; ++u) largest[u] = -INFINITY;
    if (static_cast<uint32_t>(lane) < p.shares) {
#pragma unroll
      for (int u = 0; u < kAcceptWaves; ++u) {
        largest[u] = shares.ld(word(node, lane) + 2 * kAcceptWaves + u);
        const uint64_t lo = shares.ldu(word(node, lane) + 2 * u), hi = shares.ldu(word(node, lane) + 2 * u + 1);
        part[u] = __builtin_bit_cast(double, hi << 32 | lo);
      }
    }
#pragma unroll
    for (int u = 0; u < kAcceptWaves; ++u) most = fmaxf(most, largest[u]);
    const float all = wave_max(most);
    if (!(fabsf(all) < kHuge)) {
      // The largest logit, read again by the whole workgroup.
      top = -INFINITY;
      best = UINT32_MAX;
      for (uint32_t i = threadIdx.x; i < p.a.vocab; i += kAcceptT) take(logit<E>(x.x, i), i);
      const float wave_top = wave_max(top);
      __syncthreads();
      if (lane == 0) tops[w] = wave_top;
      if (threadIdx.x == 0) ids[0] = UINT32_MAX;
      __syncthreads();
      const float m = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
      if (top == m && best != UINT32_MAX) atomicMin(&ids[0], best);
      __syncthreads();
      if (threadIdx.x == 0) picks[0] = ids[0] == UINT32_MAX ? 0 : static_cast<int32_t>(ids[0]);
    } else {
      const bool far = fabsf(all) * p.c_hi >= kFar;  // (then all of the node's logits are read again)
      const float up = whole_above(p, all);
#pragma unroll
      for (int u = 0; u < kAcceptWaves; ++u) {
        part[u] = scaled(part[u], whole_above(p, largest[u]) - up);
        s += part[u];
      }
      const double upto = lanes_upto(s), draw = fmaxf(p.a.draws[at + node], 0.f);
      // A draw of 1 or more passes nothing: the last share with a token, and there the last quarter and token.
      const auto aim_at = [&](double total) { return draw < 1.0 ? draw * total : static_cast<double>(INFINITY); };
      double aim = aim_at(lane_of(upto, kWave - 1));
      // (Lanes add in orders of their own: behind the last share sums may be larger by a rounding.)
      const uint64_t some = __ballot(s > 0.0), past = __ballot(upto > aim) & some;
      const int in = past ? __ffsll(static_cast<unsigned long long>(past)) - 1 : 63 - __clzll(static_cast<long long>(some));
      // Its quarter: the first that passes, or the last with a token.
      double before = lane_of(upto - s, in), begins = before, ends = before;
      int which = -1;
      float own = all;  // its largest logit
#pragma unroll
      for (int u = 0; u < kAcceptWaves; ++u) {
        const double y = lane_of(part[u], in);
        if (y > 0.0 && (which < 0 || !(ends > aim))) {
          which = u;
          begins = before;
          ends = before + y;
          own = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, largest[u]), in));
        }
        before += y;
      }
      // The rest is relative to the quarter's own whole number: to the node's, FP32 may have nothing of it.
      const float r_own = whole_above(p, own);
      aim = ldexp(aim - begins, static_cast<int>(up - r_own));
      const uint32_t q = in * kAcceptWaves + which, a0 = far ? 0 : x.first(q), b0 = far ? x.pieces : x.first(q + 1);
      // Its logits again, a run of pieces each thread; what lies before and behind the pieces with the first and last thread.
      const uint32_t n = (b0 - a0 + kAcceptT - 1) / kAcceptT, a = min(b0, a0 + threadIdx.x * n), b = min(b0, a + n);
      const uint32_t begin = (far || q == 0) && threadIdx.x == 0 ? 0 : x.token(a);
      const uint32_t end = (far || q + 1 == p.shares * kAcceptWaves) && threadIdx.x == kAcceptT - 1 ? p.a.vocab : x.token(b);
      const auto weight = [&](float y) { return far ? power_far(p, y, all) : power(p, y, r_own); };
      const auto each = [&](auto f) {  // f(token, probability), until it says so
        for (uint32_t i = begin; i < x.token(a) && i < end; ++i)
          if (f(i, weight(logit<E>(x.x, i)))) return;
        for (uint32_t k = a; k < b; ++k) {
          float y[kPer];
          Row::values(x.load(k), y);
#pragma unroll
          for (int i = 0; i < kPer; ++i)
            if (f(x.token(k) + i, weight(y[i]))) return;
        }
        for (uint32_t i = x.token(b); i < end; ++i)
          if (f(i, weight(logit<E>(x.x, i)))) return;
      };
      double run = 0.0;
      each([&](uint32_t, float y) {
        run += y;
        return false;
      });
      const double wave_upto = lanes_upto(run);
      __syncthreads();
      if (lane == kWave - 1) sums[w] = wave_upto;
      __syncthreads();
      if (far) aim = aim_at((sums[0] + sums[1]) + (sums[2] + sums[3]));
      double mine_before = wave_upto - run;
      for (int u = 0; u < w; ++u) mine_before += sums[u];
      // The first thread whose run passes the draw, or the last with a token.
      const uint64_t passes = __ballot(run > 0.0 && mine_before + run > aim), any = __ballot(run > 0.0);
      if (lane == 0) {
        ids[w] = passes ? w * kWave + __ffsll(static_cast<unsigned long long>(passes)) - 1 : UINT32_MAX;
        tops[w] = any ? static_cast<float>(w * kWave + 63 - __clzll(static_cast<long long>(any))) : -1.f;
      }
      __syncthreads();
      uint32_t who = min(min(ids[0], ids[1]), min(ids[2], ids[3]));
      if (who == UINT32_MAX) who = static_cast<uint32_t>(fmaxf(0.f, fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]))));
      if (threadIdx.x == who) {
        uint32_t found = begin;
        each([&](uint32_t i, float y) {
          if (y > 0.f) found = i;
          mine_before += y;
          return y > 0.f && mine_before > aim;
        });
        picks[0] = static_cast<int32_t>(found);
      }
    }
    __syncthreads();
    const Coherent out(p.picks + at, static_cast<uint32_t>(p.a.nodes * sizeof(int32_t)));
    if (threadIdx.x == 0) out.stu(node, static_cast<uint32_t>(picks[0]));
    if (!arrive(row_counter, present)) return;
    if (w != 0) return;
    if (there >> lane & 1) picks[lane] = static_cast<int32_t>(out.ldu(lane));
  }
  // The walk: lane n is node n.
  const int32_t token = static_cast<uint32_t>(lane) < p.a.nodes ? p.a.tokens[at + lane] : -1;
  const int32_t pick = there >> lane & 1 ? picks[lane] : -1;
  const int32_t wanted = __builtin_amdgcn_ds_bpermute(max(parent, 0) << 2, pick);
  const bool fits = parent >= 0 && token == wanted;
  int32_t here = 0, path = -1;
  uint32_t count = 0;
  for (;;) {
    if (static_cast<uint32_t>(lane) == count) path = here;
    ++count;
    const uint64_t next = __ballot(fits && parent == here);
    if (!next) break;
    here = __ffsll(static_cast<unsigned long long>(next)) - 1;
  }
  if (static_cast<uint32_t>(lane) < p.a.nodes) p.a.path[at + lane] = path;
  const int32_t following = __builtin_amdgcn_readlane(pick, here);
  if (lane == 0) {
    p.a.counts[row] = static_cast<int32_t>(count);
    p.a.next_tokens[row] = following;
  }
}

// ---- commit --------------------------------------------------------------------------
// Lane n of every wave looks up node n's move; a workgroup takes 64 columns of 16 bytes of
// one row, its waves every fourth move, and stores when all of them are loaded: a move's
// target is an earlier move's source. Bound by memory for large trees (64 of 63 nodes, 8 layers of 8 heads
// of 128 in BF16, 70 MB read and written, 16.7 us: 4.2 TB/s), else by the chain length, path, page,
// load, store (16 of 16, 24 layers of 2 of 64 in FP32, 4.9 us).
constexpr int kCommitT = 256;
constexpr int kMovesPerWave = 64 / (kCommitT / kWave);
struct CommitLaunch {
  qd_commit_args a;         // (a.memories is not for the device)
  qd_token_memory memory[kForkMemories];
  uint32_t columns[kForkMemories];  // of 16 bytes in all planes
  uint32_t page_shift;
};

__global__ __launch_bounds__(kCommitT) void commit_kernel(CommitLaunch p) {
  const uint32_t row = blockIdx.y, lane = lane_id(), w = wave_id();
  const int32_t length = p.a.lengths[row], nodes = static_cast<int32_t>(p.a.nodes);
  const bool first = blockIdx.x == 0 && threadIdx.x == 0;
  if (length == 0) {
    if (first) p.a.lengths_out[row] = 0;
    return;
  }
  const int64_t room = static_cast<int64_t>(p.a.table_width) << p.page_shift;
  uint32_t bad = length < nodes || length > room ? QD_PAGED_BAD_LENGTH : 0;
  const int32_t count = p.a.counts[row], start = length - nodes;
  if (count < 0 || count > nodes) bad |= QD_TREE_BAD_PATH;
  int32_t from = -1, from_page = -1, to_page = -1;
  const bool mine = !bad && static_cast<int32_t>(lane) < count;
  if (mine) from = p.a.path[static_cast<size_t>(row) * p.a.nodes + lane];
  const int32_t before = __builtin_amdgcn_ds_bpermute((static_cast<int>(lane) - 1) << 2, from);
  if (__any(mine && (from < 0 || from >= nodes || (lane > 0 && from <= before)))) bad |= QD_TREE_BAD_PATH;
  const bool moves = mine && !bad && from != static_cast<int32_t>(lane);
  if (moves) {
    const int32_t *table = p.a.table + row * p.a.table_stride;
    from_page = table[(start + from) >> p.page_shift];
    to_page = table[(start + static_cast<int32_t>(lane)) >> p.page_shift];
  }
  if (__any(moves && (from_page < 0 || static_cast<uint32_t>(from_page) >= p.a.pages || to_page < 0 ||
                      static_cast<uint32_t>(to_page) >= p.a.pages)))
    bad |= QD_PAGED_BAD_PAGE;
  if (first) {
    p.a.lengths_out[row] = bad ? length : start + count;
    if (bad) raise_error(p.a.errors, bad);
  }
  if (bad) return;
  const uint64_t moving = __ballot(moves);
  if (!moving) return;
  // This lane's column.
  uint32_t column = blockIdx.x * kWave + lane;
  char *base = nullptr;
  int64_t page_stride = 0, token_stride = 0;
#pragma unroll
  for (uint32_t m = 0; m < kForkMemories; ++m) {
    if (m >= p.a.memory_count || base) continue;
    if (column >= p.columns[m]) {
      column -= p.columns[m];
      continue;
    }
    const uint32_t per_piece = p.memory[m].piece_bytes / 16, piece = column / per_piece;
    base = static_cast<char *>(p.memory[m].base) + piece / p.memory[m].pieces * p.memory[m].plane_stride +
           piece % p.memory[m].pieces * p.memory[m].piece_stride + column % per_piece * 16;
    page_stride = p.memory[m].page_stride;
    token_stride = p.memory[m].token_stride;
  }
  const int32_t mask = static_cast<int32_t>(p.a.page_size) - 1;
  u4v x[kMovesPerWave];
#pragma unroll
  for (int u = 0; u < kMovesPerWave; ++u) {
    const int i = __builtin_amdgcn_readfirstlane(w) + u * (kCommitT / kWave);
    if (!(moving >> i & 1)) continue;
    const int32_t pos = start + __builtin_amdgcn_readlane(from, i), page = __builtin_amdgcn_readlane(from_page, i);
    if (base) x[u] = *reinterpret_cast<const u4v *>(base + page * page_stride + (pos & mask) * token_stride);
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < kMovesPerWave; ++u) {
    const int i = __builtin_amdgcn_readfirstlane(w) + u * (kCommitT / kWave);
    if (!(moving >> i & 1)) continue;
    const int32_t pos = start + i, page = __builtin_amdgcn_readlane(to_page, i);
    if (base) *reinterpret_cast<u4v *>(base + page * page_stride + (pos & mask) * token_stride) = x[u];
  }
}

uint32_t accept_shares(uint32_t rows, uint32_t nodes, uint32_t vocab) {
  const uint64_t all = static_cast<uint64_t>(rows) * nodes;
  const uint64_t want = (kAcceptAim + all - 1) / std::max<uint64_t>(all, 1);
  return static_cast<uint32_t>(std::max<uint64_t>(1, std::min({want, static_cast<uint64_t>(kAcceptShares),
                                                                static_cast<uint64_t>((vocab + kAcceptLeast - 1) / kAcceptLeast)})));
}

}  // namespace

size_t tree_attention_scratch(uint32_t dtype, uint32_t rows, uint32_t nodes, uint32_t heads, uint32_t kv_heads, uint32_t head_dim) {
  return with_type(dtype, head_dim, nodes * (heads / kv_heads), [&](auto shape, auto) {
    using S = decltype(shape);
    return static_cast<size_t>(tree_plan<S>(rows, nodes, heads, kv_heads).records) * S::kRecord * sizeof(float);
  });
}

size_t tree_attention_scratch_most(uint32_t rows, uint32_t nodes, uint32_t heads, uint32_t kv_heads, uint32_t head_dim) {
  size_t most = 0;
  // (More rows than there are counters for are not cut and keep nothing; fewer are. A
  // few nodes less may take narrower blocks.)
  for (const uint32_t dtype : {QD_DTYPE_F32, QD_DTYPE_BF16})
    for (uint32_t n = 1; n <= nodes; ++n)
      with_type(dtype, head_dim, n * (heads / kv_heads), [&](auto shape, auto) {
        const uint32_t parts = kv_heads * tree_plan<decltype(shape)>(0, n, heads, kv_heads).blocks;
        most = std::max(most, tree_attention_scratch(dtype, std::min(rows, static_cast<uint32_t>(kOpCounters / parts)), n, heads, kv_heads, head_dim));
      });
  return most;
}

hipError_t launch_tree_attention(hipStream_t s, const qd_paged_cache &c, const qd_tree_attention_args &a, const OpScratch &w) {
  if (c.rows == 0 || a.nodes == 0) return hipSuccess;
  TreeLaunch p{};
  p.c = c;
  p.a = a;
  p.records = reinterpret_cast<float *>(w.scratch);
  p.counters = w.counters;
  p.page_shift = log2_of(c.page_size);
  return with_type(c.dtype, c.head_dim, a.nodes * (a.heads / c.kv_heads), [&](auto shape, auto kernel) {
    using S = decltype(shape);
    const TreePlan plan = tree_plan<S>(c.rows, a.nodes, a.heads, c.kv_heads);
    p.apart = plan.apart;
    p.group = plan.group;
    p.columns = plan.columns;
    p.blocks = plan.blocks;
    p.parts = c.kv_heads * plan.blocks;
    const uint64_t most = ((static_cast<uint64_t>(c.table_width) << p.page_shift) + kTreeLeast - 1) / kTreeLeast;
    p.target = most <= 1 ? 0 : plan.target;
    uint64_t x = c.rows;
    if (p.target) x = std::min<uint64_t>(plan.few ? x + p.target : x + 4 * p.target, x * most);
    p.units = static_cast<uint32_t>(x);
    uint32_t grid = (p.units + kXcds - 1) / kXcds * kXcds * p.parts;
    // Many rows whose items read nothing twice: equal runs (64 BF16 rows of 0 to 8,192 with 16 columns
    // 203 us, in pieces 229, with 32 212 and 234; for few rows their two halves of a record cost more
    // than they even out: two of 1,000 24.5 us, in pieces 17.4, 16 FP32 of 513 to 4,000 33 and 29).
    // (Stages are counted in 31 bits.)
    const uint64_t stages = ((static_cast<uint64_t>(c.table_width) << p.page_shift) + S::kStage - 1) / S::kStage;
    if (S::kByHalves && p.target && p.blocks == 1 && !plan.few && c.rows * p.parts * (stages + kEdge) <= 0x7f000000u) {
      p.units = 0;
      p.least = kTreeLeast / S::kStage;
      grid = kTreeCus * S::kPerCu;
    }
    return launch(kernel, dim3(grid), dim3(S::kThreads), s, p);
  });
}

// (As many shares of a node as kAcceptAim asks for: all of them are fewer than that and
// one more of each node.)
size_t tree_accept_scratch(uint32_t rows, uint32_t nodes) {
  const size_t all = static_cast<size_t>(rows) * nodes;
  return round256(std::min(all * kAcceptShares, all + kAcceptAim) * sizeof(AcceptShare)) + round256(all * sizeof(int32_t));
}

hipError_t launch_tree_accept(hipStream_t s, const qd_accept_args &a, const OpScratch &w) {
  if (a.rows == 0 || a.nodes == 0) return hipSuccess;
  AcceptLaunch p{};
  p.a = a;
  p.shares = accept_shares(a.rows, a.nodes, a.vocab);
  const size_t all = static_cast<size_t>(a.rows) * a.nodes;
  p.share = reinterpret_cast<AcceptShare *>(w.scratch);
  p.picks = reinterpret_cast<int32_t *>(w.scratch + round256(std::min(all * kAcceptShares, all + kAcceptAim) * sizeof(AcceptShare)));
  p.counters = w.counters;
  for (p.apart = 32; (all + a.rows) * p.apart > kOpCounters;) p.apart /= 2;
  if (a.draws) {
    const double c = 1.4426950408889634074 / a.temperature;
    p.c_hi = static_cast<float>(c);
    p.c_lo = static_cast<float>(c - p.c_hi);
    p.most = static_cast<float>(2.0 * kFar / c);
  }
  const dim3 grid(p.shares, static_cast<uint32_t>(all)), block(kAcceptT);
  const auto run = [&](auto greedy, auto sampled) { return launch(a.draws ? sampled : greedy, grid, block, s, p); };
  switch (a.dtype) {
    case QD_DTYPE_F32: return run(accept_kernel<float, false>, accept_kernel<float, true>);
    case QD_DTYPE_BF16: return run(accept_kernel<Brain, false>, accept_kernel<Brain, true>);
    default: return run(accept_kernel<Half, false>, accept_kernel<Half, true>);
  }
}

hipError_t launch_tree_commit(hipStream_t s, const qd_commit_args &a) {
  if (a.rows == 0) return hipSuccess;
  CommitLaunch p{};
  p.a = a;
  p.a.memories = nullptr;
  uint64_t columns = 0;
  for (uint32_t m = 0; m < a.memory_count; ++m) {
    p.memory[m] = a.memories[m];
    p.columns[m] = a.memories[m].piece_bytes / 16 * a.memories[m].pieces * a.memories[m].planes;
    columns += p.columns[m];
  }
  p.page_shift = log2_of(a.page_size);
  const uint32_t x = static_cast<uint32_t>(std::max<uint64_t>(1, (columns + kWave - 1) / kWave));
  return launch(commit_kernel, dim3(x, a.rows), dim3(kCommitT), s, p);
}

}  // namespace qd
