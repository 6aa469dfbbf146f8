// Operators on a paged key-value cache for gfx950: writing rotated rows into
// pages, attention of one new token per row, and the fork of rows that share
// pages. Declared in include/qd/qd_operators.h.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "qd_attention.hpp"
#include "qd_device.hpp"
#include "qd_device_math.hpp"
#include "qd_operators.hpp"

namespace qd {
namespace {

using namespace dev;

typedef float f4v __attribute__((ext_vector_type(4)));
typedef uint32_t u4v __attribute__((ext_vector_type(4)));
typedef uint32_t u2v __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
// Lengths, tables and positions are written before the kernel starts: they may
// be read through the scalar cache.
typedef const __attribute__((address_space(4))) int32_t const_i32;

__device__ __forceinline__ int32_t load_uniform(const int32_t *p) { return *(const_i32 *)p; }

__device__ __forceinline__ void raise_error(uint32_t *errors, uint32_t bit) {
  if (errors) atomicOr(errors, bit);
}

// Waits until this thread's vector memory operations have completed.
__device__ __forceinline__ void wait_vm_stores() { __builtin_amdgcn_s_waitcnt(0x0F70); }

// The storage types' conversions; two values share a 32-bit register, low half first.
struct Half {
  static __device__ __forceinline__ float lo(uint32_t v) { return half_lo(v); }
  static __device__ __forceinline__ float hi(uint32_t v) { return half_hi(v); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const f16x2 v = {static_cast<_Float16>(a), static_cast<_Float16>(b)};  // to nearest even
    return __builtin_bit_cast(uint32_t, v);
  }
  static __device__ __forceinline__ f4v mfma(u4v a, u4v b, f4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};
struct Brain {
  static __device__ __forceinline__ float lo(uint32_t v) { return __uint_as_float(v << 16); }
  static __device__ __forceinline__ float hi(uint32_t v) { return __uint_as_float(v & 0xFFFF0000u); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const bf16x2 v = {static_cast<__bf16>(a), static_cast<__bf16>(b)};  // to nearest even
    return __builtin_bit_cast(uint32_t, v);
  }
  static __device__ __forceinline__ f4v mfma(u4v a, u4v b, f4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};

// Four consecutive elements as FP32, and back.
template <typename E>
__device__ __forceinline__ float4 load4(const void *base, int64_t i) {
  if constexpr (std::is_same_v<E, float>) {
    return *reinterpret_cast<const float4 *>(static_cast<const float *>(base) + i);
  } else {
    const uint2 v = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(base) + i);
    return make_float4(E::lo(v.x), E::hi(v.x), E::lo(v.y), E::hi(v.y));
  }
}
template <typename E>
__device__ __forceinline__ void store4(void *base, int64_t i, float4 v) {
  if constexpr (std::is_same_v<E, float>)
    *reinterpret_cast<float4 *>(static_cast<float *>(base) + i) = v;
  else
    *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(base) + i) = make_uint2(E::pack(v.x, v.y), E::pack(v.z, v.w));
}

// ---- append -------------------------------------------------------------------
// (a, b) -> (a c - b s, b c + a s) for the rotated pairs, a copy for the rest. A
// wave takes rows of one token, so that its position, page and angles are looked up
// once and through the scalar cache; each group of head_dim / 8 lanes takes a head,
// eight elements a lane. Bound by memory for prompts (6,000 tokens of 48 heads of 128
// in BF16, 149 MB, 28.7 us: 5.2 TB/s, what a copy reaches), by the chain position ->
// page -> store for a few tokens (16 of 18 heads of 64 in FP32 3.0 us).
struct AppendLaunch {
  qd_paged_cache c;
  qd_append_args a;
  uint32_t page_shift;
  uint32_t lanes_shift;  // of a head: log2(head_dim / 8)
  uint32_t waves;        // of a token
};

// Eight consecutive elements.
template <typename E>
struct Eight {
  float4 lo, hi;
};
template <typename E>
__device__ __forceinline__ Eight<E> load8(const void *base, int64_t i) {
  if constexpr (std::is_same_v<E, float>) {
    return {load4<E>(base, i), load4<E>(base, i + 4)};
  } else {
    const uint4 v = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(base) + i);
    return {make_float4(E::lo(v.x), E::hi(v.x), E::lo(v.y), E::hi(v.y)),
            make_float4(E::lo(v.z), E::hi(v.z), E::lo(v.w), E::hi(v.w))};
  }
}
// Past the caches: what is appended is read by other kernels, mostly on other XCDs.
// (6,000 tokens of 48 heads of 128 in BF16 28.7 us, with ordinary stores 34.1; 500 4.5
// and 5.2, 16 of 18 heads of 64 in FP32 3.05 and 3.03.)
template <typename E>
__device__ __forceinline__ void store8(void *base, int64_t i, const Eight<E> &v) {
  if constexpr (std::is_same_v<E, float>) {
    f4v *to = reinterpret_cast<f4v *>(static_cast<float *>(base) + i);
    __builtin_nontemporal_store(f4v{v.lo.x, v.lo.y, v.lo.z, v.lo.w}, to);
    __builtin_nontemporal_store(f4v{v.hi.x, v.hi.y, v.hi.z, v.hi.w}, to + 1);
  } else {
    __builtin_nontemporal_store(
        u4v{E::pack(v.lo.x, v.lo.y), E::pack(v.lo.z, v.lo.w), E::pack(v.hi.x, v.hi.y), E::pack(v.hi.z, v.hi.w)},
        reinterpret_cast<u4v *>(static_cast<uint16_t *>(base) + i));
  }
}

// Four elements x of one half of their pairs with the others' y: x c + sign y s.
__device__ __forceinline__ float4 turn4(float4 x, float4 y, float4 c, float4 s, bool second) {
  float4 a, b;
  if (second) {
    rope_rotate(y.x, x.x, c.x, s.x, a.x, b.x);
    rope_rotate(y.y, x.y, c.y, s.y, a.y, b.y);
    rope_rotate(y.z, x.z, c.z, s.z, a.z, b.z);
    rope_rotate(y.w, x.w, c.w, s.w, a.w, b.w);
    return b;
  }
  rope_rotate(x.x, y.x, c.x, s.x, a.x, b.x);
  rope_rotate(x.y, y.y, c.y, s.y, a.y, b.y);
  rope_rotate(x.z, y.z, c.z, s.z, a.z, b.z);
  rope_rotate(x.w, y.w, c.w, s.w, a.w, b.w);
  return a;
}

template <typename E>
__global__ __launch_bounds__(kBlock) void append_kernel(AppendLaunch p) {
  const uint32_t id = blockIdx.x * kWavesPerBlock + __builtin_amdgcn_readfirstlane(wave_id());
  const uint32_t token = id / p.waves;
  if (token >= p.a.tokens) return;
  const int64_t position = static_cast<int64_t>(load_uniform(p.a.positions + token)) + p.a.position_bias;
  if (position < 0) return;
  const uint32_t dim = p.c.head_dim, lane = lane_id();
  const uint32_t heads = p.a.q ? p.a.heads : 0, all = heads + 2 * p.c.kv_heads;  // queries, then keys, then values
  const uint32_t j = (id - token * p.waves) * (kWave >> p.lanes_shift) + (lane >> p.lanes_shift);  // this lane's row
  if (j >= all) return;
  const uint32_t e = 8 * (lane & ((1u << p.lanes_shift) - 1));  // this lane's first element of a head
  const uint32_t rotary = p.a.rotary_dim, half = rotary / 2;

  const int32_t row = p.a.rows ? load_uniform(p.a.rows + token) : static_cast<int32_t>(token);
  const uint64_t column = static_cast<uint64_t>(position) >> p.page_shift;
  uint32_t bad = 0;
  int64_t page = 0;
  if (row < 0 || static_cast<uint32_t>(row) >= p.c.rows) {
    bad = QD_PAGED_BAD_ROW;
  } else if (column >= p.c.table_width || (rotary && static_cast<uint64_t>(position) >= p.a.table_positions)) {
    bad = QD_PAGED_BAD_POSITION;
  } else {
    page = load_uniform(p.c.table + row * p.c.table_stride + static_cast<int64_t>(column));
    if (page < 0 || page >= p.c.pages) bad = QD_PAGED_BAD_PAGE;
  }
  if (bad) {
    const float n = __uint_as_float(0x7FC00000u);
    const float4 nans = make_float4(n, n, n, n);
    if (j < heads) store8<E>(p.a.q_out, token * p.a.q_out_stride + j * dim + e, {nans, nans});
    if (id == token * p.waves && lane == 0) raise_error(p.c.errors, bad);
    return;
  }
  // Four elements of a lane never lie on both sides of half or rotary (multiples of 4 and 8).
  const bool turned = e < rotary, lo_second = e >= half, hi_second = e + 4 >= half;
  float4 c[2], s[2];
  if (turned) {
    const float *cos_row = p.a.cos_table + position * half, *sin_row = p.a.sin_table + position * half;
    if (p.a.interleaved) {
      c[0] = *reinterpret_cast<const float4 *>(cos_row + e / 2);
      s[0] = *reinterpret_cast<const float4 *>(sin_row + e / 2);
    } else {
      const uint32_t lo = lo_second ? e - half : e, hi = hi_second ? e + 4 - half : e + 4;
      c[0] = *reinterpret_cast<const float4 *>(cos_row + lo);
      s[0] = *reinterpret_cast<const float4 *>(sin_row + lo);
      c[1] = *reinterpret_cast<const float4 *>(cos_row + hi);
      s[1] = *reinterpret_cast<const float4 *>(sin_row + hi);
    }
  }
  const bool query = j < heads, value = j >= heads + p.c.kv_heads;
  const uint32_t h = query ? j : value ? j - heads - p.c.kv_heads : j - heads;
  const void *src = query ? p.a.q : value ? p.a.v : p.a.k;
  const int64_t from = token * (query ? p.a.q_stride : value ? p.a.v_stride : p.a.k_stride) + h * dim;
  Eight<E> x = load8<E>(src, from + e);
  if (turned && !value) {
    if (p.a.interleaved) {
      const Eight<E> z = x;
      rope_rotate(z.lo.x, z.lo.y, c[0].x, s[0].x, x.lo.x, x.lo.y);
      rope_rotate(z.lo.z, z.lo.w, c[0].y, s[0].y, x.lo.z, x.lo.w);
      rope_rotate(z.hi.x, z.hi.y, c[0].z, s[0].z, x.hi.x, x.hi.y);
      rope_rotate(z.hi.z, z.hi.w, c[0].w, s[0].w, x.hi.z, x.hi.w);
    } else {
      // The other elements of the pairs, which other lanes of this wave turn. (In
      // place too: a wave loads before it stores.)
      const float4 lo = load4<E>(src, from + (lo_second ? e - half : e + half));
      const float4 hi = load4<E>(src, from + (hi_second ? e + 4 - half : e + 4 + half));
      x.lo = turn4(x.lo, lo, c[0], s[0], lo_second);
      x.hi = turn4(x.hi, hi, c[1], s[1], hi_second);
    }
  }
  void *dst = query ? p.a.q_out : value ? p.c.v : p.c.k;
  const int64_t to = query ? token * p.a.q_out_stride + h * dim
                           : page * p.c.page_stride + (position & (p.c.page_size - 1)) * p.c.token_stride + h * p.c.head_stride;
  store8<E>(dst, to + e, x);
}

// ---- attention ------------------------------------------------------------------
// The work is cut into tiles of 32 positions of one (row, KV head, up to 16 of its
// query heads), here an item, and dealt to the workgroups in equal runs, so that
// all are done at about the same time whatever the rows' lengths; a cut near an
// item's ends moves there. A workgroup's waves take an item's tiles in turn, each
// with a running maximum and sum. Everything stays in the registers of the matrix
// instructions:
//   S^T = K Q^T   lane l: head l % 16, positions 4 (l / 16) + r of each half tile
//   O^T += V^T P^T the same lane's probabilities are the operand as they are, and
//                 its share of O is of its own head, so a new maximum rescales
//                 with one factor per lane.
// K is read in the operand's layout (16 bytes of a row per lane). V's operand
// holds positions along the registers: FP32 takes one position per instruction,
// so float4 loads along the head serve four of them; 16-bit rows are loaded 8 at
// a time and turned with byte permutes.
// Bound by the memory for long rows: 64 rows of 0 to 8,192 with 8 KV heads of 128 in
// BF16, 1,086 MB, 182 us (6.0 TB/s; a streaming read reaches 6.6), two of about
// 105,000 with 4 in FP16, 431 MB, 85 us. Short ones wait: for the launch, length,
// page, K, the other waves, the other pieces, each near 1 us (one row of 129 6.75 us,
// 16 beams at 576 8.5).
constexpr int kTile = 32, kSub = 16;
constexpr uint32_t kMostPieces = 256;  // of an item
constexpr int kWaves = 4;              // of a workgroup
// Tiles that an item's results cost the long kernel as much time as: 128 rows of 0 to
// 4,000 took 171 us, counted as none 177, as one 176, as four 173.
constexpr uint32_t kEdge = 2;
// The short kernel: tiles of a piece at least, of an item that stays whole (one row of
// 129 positions 7.4 us, with items of 5 tiles cut 8.6; 8 rows of 448 8.8, with items
// of 14 whole 11.6), and pieces of an item at most (one row of 30,000 18.9 us, in up
// to 256 pieces 25.3; all before V was loaded with K).
constexpr uint32_t kShortLeast = 4, kShortWhole = 8, kShortPieces = 64;
// A maximum is only taken up when it passes the one in use by this many powers of
// two: until then probabilities grow to at most 2^8. (Taken up at once, 64 rows of 0 to
// 8,192 took 193 us instead of 192.) FP16's range is needed at the other end.
template <typename E>
constexpr float kLazyMax = 8.f;
template <>
constexpr float kLazyMax<Half> = 1.f;
// What FP16 takes of a probability p, at most 2 before it is rounded: kWeight p, up to
// 2^15, and kRest times the remainder, up to 2^3. Half of the least step, 2^-25, is then
// 2^-51 of the largest probability (as they are, without these factors, 2^-25: all
// that lay more than 17 below the largest score counted in the sum, but in no output).
constexpr float kWeight = 0x1p14f, kRest = 0x1p12f;

struct AttnLaunch {
  qd_paged_cache c;
  qd_attention_args a;
  float *records;       // [workgroups][2][rec_floats]: acc [rec_heads][head_dim], maxima, sums
  uint32_t *counters;   // [rows][parts * apart]
  uint32_t apart;       // words between two counters
  uint32_t parts;       // items of a row: KV heads x blocks of query heads
  uint32_t page_shift;
  uint32_t group;       // query heads of a KV head
  uint32_t blocks;      // of up to 16 of them
  uint32_t rec_heads;   // the most of a block
  uint32_t rec_floats;
  uint32_t least;       // tiles on either side of a cut; 0: items are not cut
  uint32_t target;      // pieces aimed at besides one of each item (the short kernel)
};

// Values of lanes l and l ^ 32 in a and b (any order).
__device__ __forceinline__ void half_swap(float v, float &a, float &b) {
  unsigned x = __builtin_bit_cast(unsigned, v), y = x;
  asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(x), "+v"(y));
  a = __builtin_bit_cast(float, x);
  b = __builtin_bit_cast(float, y);
}
// Over lanes l, l ^ 16, l ^ 32, l ^ 48.
__device__ __forceinline__ float quarters_max(float v) {
  float a, b;
  v = row_pair_max(v);
  half_swap(v, a, b);
  return fmaxf(a, b);
}
__device__ __forceinline__ float quarters_sum(float v) {
  float a, b;
  v = row_pair_sum(v);
  half_swap(v, a, b);
  return a + b;
}

// 16 positions of a page through a descriptor that ends with the last valid one:
// loads past it give zeros and touch no memory.
template <int kPolicy>
struct PageRows {
  __amdgpu_buffer_rsrc_t r;
  __device__ __forceinline__ u4v ld16(uint32_t byte) const {
    return __builtin_bit_cast(u4v, __builtin_amdgcn_raw_buffer_load_b128(r, byte, 0, kPolicy));
  }
  __device__ __forceinline__ u2v ld8(uint32_t byte) const {
    return __builtin_bit_cast(u2v, __builtin_amdgcn_raw_buffer_load_b64(r, byte, 0, kPolicy));
  }
};

// An item and the run of its tiles that a workgroup takes: wave-uniform.
struct Item {
  int row, length;
  uint32_t part;
  uint32_t at, tiles;        // its first tile among all in the deal, and how many it has (one at least)
  uint32_t first, last;      // the run
  uint32_t home, pieces;     // the workgroup of its first piece, and how many there are
  bool bad;                  // the row's length
};

// The runs of all workgroups: run i is [i share, (i + 1) share) of all tiles, but
// for the cuts that move. Before its tiles each item has kEdge more that stand for
// the time that its results take.
struct Deal {
  uint32_t share, total;
};

__device__ __forceinline__ uint32_t tiles_of(const AttnLaunch &p, int32_t n, int64_t most) {
  return n <= 0 || n > most ? 1u : (static_cast<uint32_t>(n) + kTile - 1) / kTile;
}

// Inclusive sum over the lanes up to this one.
__device__ __forceinline__ uint32_t lanes_upto(uint32_t v) {
  int x = static_cast<int>(v);
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr:1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row 0 to 1, 2 to 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row 1 to 2 and 3
  return static_cast<uint32_t>(x);
}

// How a cut `off` tiles into an item of n moves: 0 to its start, 1 not, 2 to its end.
__device__ __forceinline__ int cut_of(const AttnLaunch &p, uint32_t off, uint32_t n) {
  if (p.least && n >= 2 * p.least) return off < p.least ? 0 : n - off < p.least ? 2 : 1;
  return 2 * off < n ? 0 : 2;
}

__device__ __forceinline__ void set_item(const AttnLaunch &p, const Deal &d, Item &it, uint32_t row, uint32_t part,
                                         uint32_t at, int32_t n, int64_t most) {
  it.row = static_cast<int>(row);
  it.part = part;
  it.at = at + kEdge;
  it.bad = n < 0 || n > most;
  it.length = it.bad ? 0 : n;
  it.tiles = tiles_of(p, n, most);
  it.first = 0;
  it.last = it.tiles;
  it.home = 0;
  it.pieces = 1;
  if (p.least && it.tiles >= 2 * p.least) {
    const uint32_t lo = (it.at + p.least + d.share - 1) / d.share, hi = (it.at + it.tiles - p.least) / d.share;
    if (hi >= lo) {
      it.pieces = hi - lo + 2;
      it.home = lo - 1;
    }
  }
}

// Ends the run of `it` where workgroup i's does; false: the item is the next one's.
__device__ __forceinline__ bool end_run(const AttnLaunch &p, const Deal &d, uint32_t i, Item &it) {
  const uint32_t end = (i + 1) * d.share;
  if (it.at + it.tiles <= end || end >= d.total) return true;
  if (end <= it.at) return false;
  const int cut = cut_of(p, end - it.at, it.tiles);
  if (cut == 1) it.last = end - it.at;
  return cut != 0;
}

// Maximum over the wave of numbers below 2^31.
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
  int x = static_cast<int>(v);
  x = max(x, __builtin_amdgcn_update_dpp(0, x, kDppXor1, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, kDppXor2, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, kDppHalfMirror, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, kDppMirror, 0xf, 0xf, false));
  return static_cast<uint32_t>(max(max(__builtin_amdgcn_readlane(x, 0), __builtin_amdgcn_readlane(x, 16)),
                                   max(__builtin_amdgcn_readlane(x, 32), __builtin_amdgcn_readlane(x, 48))));
}

// Workgroup i's first item; false if it has none. Lane l looks at rows l, l + 64, ...
__device__ __forceinline__ bool first_item(const AttnLaunch &p, uint32_t i, uint32_t groups, Deal &d, Item &it) {
  const int lane = lane_id();
  const int64_t most = static_cast<int64_t>(p.c.table_width) << p.page_shift;
  uint32_t total = 0, longest = 0;
  int32_t n = 0;  // of the row looked at last
  for (uint32_t r = lane; r < p.c.rows; r += kWave) {
    n = p.c.lengths[r];
    const uint32_t tiles = tiles_of(p, n, most) + kEdge;
    total += tiles;
    longest = max(longest, tiles);
  }
  uint32_t upto = lanes_upto(total);
  total = __builtin_amdgcn_readlane(upto, kWave - 1) * p.parts;
  longest = lanes_max(longest);
  d.total = total;
  d.share = max((total + groups - 1) / groups, (longest + kMostPieces - 3) / (kMostPieces - 2));
  const uint32_t begin = i * d.share;
  if (static_cast<uint64_t>(i) * d.share >= total) return false;
  // The row in which the run begins.
  uint32_t before = 0, base = 0;
  const bool once = p.c.rows <= kWave;
  uint64_t past;
  for (;;) {
    if (!once) {
      n = base + lane < p.c.rows ? p.c.lengths[base + lane] : 0;
      upto = lanes_upto(base + lane < p.c.rows ? tiles_of(p, n, most) + kEdge : 0u);
    }
    past = __ballot(before + upto * p.parts > begin);
    if (past) break;
    before += __builtin_amdgcn_readlane(upto, kWave - 1) * p.parts;
    base += kWave;
  }
  const int at = __ffsll(static_cast<unsigned long long>(past)) - 1;
  const int32_t length = __builtin_amdgcn_readlane(n, at);
  const uint32_t tiles = tiles_of(p, length, most), each = tiles + kEdge, row = base + at;
  before += (__builtin_amdgcn_readlane(upto, at) - each) * p.parts;
  const uint32_t part = (begin - before) / each, in = begin - before - part * each;
  const int cut = in > kEdge ? cut_of(p, in - kEdge, tiles) : 0;
  if (cut < 2) {
    set_item(p, d, it, row, part, before + part * each, length, most);
    if (cut == 1) it.first = in - kEdge;
  } else if (part + 1 < p.parts) {  // from the next item on
    set_item(p, d, it, row, part + 1, before + (part + 1) * each, length, most);
  } else {
    if (row + 1 >= p.c.rows) return false;
    set_item(p, d, it, row + 1, 0, before + (part + 1) * each, load_uniform(p.c.lengths + row + 1), most);
  }
  return end_run(p, d, i, it);
}

// The short kernel's pieces: a row of n tiles has max(1, ceil(n / size)) of each
// item, where size makes about `target` of them. Piece x of all rows' (counted for
// one part); it.home is its number within the row, `begin` the number of its
// row's first.
__device__ __forceinline__ bool find_piece(const AttnLaunch &p, uint32_t x, uint32_t part, Item &it, uint32_t &begin) {
  const int lane = lane_id();
  const int64_t most = static_cast<int64_t>(p.c.table_width) << p.page_shift;
  uint32_t size = 0x7fffffffu, row = x;
  int32_t n = 0;
  begin = x;
  if (p.target) {
    uint32_t total = 0, longest = 0;
    for (uint32_t r = lane; r < p.c.rows; r += kWave) {
      n = p.c.lengths[r];
      const uint32_t tiles = tiles_of(p, n, most);
      total += tiles;
      longest = max(longest, tiles);
    }
    total = __builtin_amdgcn_readlane(lanes_upto(total), kWave - 1);
    size = max(max(kShortLeast, (total + p.target - 1) / p.target), (lanes_max(longest) + kShortPieces - 1) / kShortPieces);
    const auto pieces_of = [&](uint32_t tiles) { return tiles <= kShortWhole ? 1u : (tiles + size - 1) / size; };
    const bool once = p.c.rows <= kWave;
    uint32_t base = 0, upto, mine;
    begin = 0;
    uint64_t past;
    for (;; base += kWave) {
      if (base >= p.c.rows) return false;
      if (!once) n = base + lane < p.c.rows ? p.c.lengths[base + lane] : 0;
      mine = base + lane < p.c.rows ? pieces_of(tiles_of(p, n, most)) : 0u;
      upto = lanes_upto(mine);
      past = __ballot(begin + upto > x);
      if (past) break;
      begin += __builtin_amdgcn_readlane(upto, kWave - 1);
    }
    const int at = __ffsll(static_cast<unsigned long long>(past)) - 1;
    row = base + at;
    begin += __builtin_amdgcn_readlane(upto - mine, at);
    n = __builtin_amdgcn_readlane(n, at);
    it.pieces = __builtin_amdgcn_readlane(mine, at);
  } else {
    n = load_uniform(p.c.lengths + row);
    it.pieces = 1;
  }
  it.row = static_cast<int>(row);
  it.part = part;
  it.bad = n < 0 || n > most;
  it.length = it.bad ? 0 : n;
  it.at = 0;
  it.tiles = tiles_of(p, n, most);
  it.home = x - begin;
  it.first = it.pieces == 1 ? 0 : it.home * size;
  it.last = it.pieces == 1 ? it.tiles : min(it.tiles, it.first + size);
  return true;
}

// The item behind `it` in workgroup i's run; false at its end.
__device__ __forceinline__ bool next_item(const AttnLaunch &p, const Deal &d, uint32_t i, const Item &it, Item &next) {
  const int64_t most = static_cast<int64_t>(p.c.table_width) << p.page_shift;
  const uint32_t at = it.at + it.tiles;
  if (it.last < it.tiles || at >= d.total || at >= (i + 1) * d.share) return false;
  if (it.part + 1 < p.parts) {
    set_item(p, d, next, it.row, it.part + 1, at, it.bad ? -1 : it.length, most);
  } else {
    set_item(p, d, next, it.row + 1, 0, at, load_uniform(p.c.lengths + it.row + 1), most);
  }
  return end_run(p, d, i, next);
}

// kStages tiles are loaded ahead. kEarly (one stage): the next tile's V comes with its
// K, into registers of its own. In the short kernel, heads of 64: one row of 129
// positions 6.7 us instead of 7.2, one of 30,000 17.6 instead of 18.4. Heads of 128 do
// without (8 rows of 1,000 to 2,000, 8 KV heads, BF16 16.8 us, with it 17.2; FP32 has
// not the registers), and so does the long kernel, which has loads enough (64 rows of
// 1,000 to 4,000, 8 KV heads of 128, FP32 217 us, with it 248).
template <typename E, int D, int kStages, bool kEarly>
struct WaveTiles {
  static constexpr bool kWide = std::is_same_v<E, float>;
  static constexpr int kElem = kWide ? 4 : 2;
  static constexpr int kPieces = D * kElem / 64;  // 16-byte loads of K per lane and half tile
  static constexpr int kAcc = D / 16;
  static constexpr bool kScaled = std::is_same_v<E, Half>;  // o holds kWeight times the sum
  u4v q[kPieces];
  u4v k[kStages][2][kPieces];
  u4v v[kStages][2][4][kWide ? D / 64 : 1];  // rows 4 (l / 16) + j; 16-bit rows of 64 use half of a register quad
  u4v v_next[2][4][kWide ? D / 64 : 1];      // (kEarly)
  f4v o[kAcc];
  float m, ms, l;

  template <typename R>
  __device__ __forceinline__ void load_k(const R &r, int st, int sub, uint32_t off) {
#pragma unroll
    for (int s = 0; s < kPieces; ++s) k[st][sub][s] = r.ld16(off + 64 * s);
  }
  template <typename R>
  static __device__ __forceinline__ void load_v(const R &r, u4v (&to)[4][kWide ? D / 64 : 1], const uint32_t (&off)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (kWide) {
#pragma unroll
        for (int n = 0; n < D / 64; ++n) to[j][n] = r.ld16(off[j] + 256 * n);
      } else if constexpr (D == 128) {
        to[j][0] = r.ld16(off[j]);
      } else {
        const u2v x = r.ld8(off[j]);
        to[j][0] = u4v{x[0], x[1], 0u, 0u};
      }
    }
  }
  // Scores of half tile `sub`, in units of the query's scale.
  __device__ __forceinline__ f4v scores(int st, int sub) const {
    f4v acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < kPieces; ++s) {
      if constexpr (kWide) {
        const f4v a = __builtin_bit_cast(f4v, k[st][sub][s]), b = __builtin_bit_cast(f4v, q[s]);
#pragma unroll
        for (int c = 0; c < 4; ++c) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[c], b[c], acc, 0, 0, 0);
      } else {
        acc = E::mfma(k[st][sub][s], q[s], acc);
      }
    }
    return acc;
  }
  // o += V^T P^T; returns the sum of the probabilities.
  __device__ __forceinline__ float accumulate(int st, const float (&pr)[2][4]) {
    float sum = 0.f;
    if constexpr (kWide) {
#pragma unroll
      for (int sub = 0; sub < 2; ++sub)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          sum += pr[sub][j];
#pragma unroll
          for (int n = 0; n < D / 64; ++n) {
            const f4v a = __builtin_bit_cast(f4v, v[st][sub][j][n]);
#pragma unroll
            for (int c = 0; c < 4; ++c)
              o[4 * n + c] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[c], pr[sub][j], o[4 * n + c], 0, 0, 0);
          }
        }
    } else {
      // A probability goes to the matrix instruction as two numbers of the cache's
      // type, rounded and what that left, so that its rounding adds little to the
      // output's own (alone it made that 1.4 times as large): 2^-16 of it in BF16, whose
      // range is FP32's, in FP16 2^-22 of it or 2^-51 of the largest. The second
      // product costs no time that the loads do not take.
      u4v b, rest;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = pr[i >> 1][2 * (i & 1)], y = pr[i >> 1][2 * (i & 1) + 1];
        if constexpr (kScaled) {
          b[i] = E::pack(x * kWeight, y * kWeight);
          rest[i] = E::pack(fmaf(x, kWeight, -E::lo(b[i])) * kRest, fmaf(y, kWeight, -E::hi(b[i])) * kRest);
        } else {
          b[i] = E::pack(x, y);
          rest[i] = E::pack(x - E::lo(b[i]), y - E::hi(b[i]));
        }
        sum += x + y;
      }
      uint32_t low = 0x05040100u, high = 0x07060302u;  // the pairs' halves
#pragma unroll
      for (int j = 0; j < kAcc; ++j) {
        u4v a;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          a[i] = __builtin_amdgcn_perm(v[st][i >> 1][2 * (i & 1) + 1][0][j >> 1], v[st][i >> 1][2 * (i & 1)][0][j >> 1],
                                       j & 1 ? high : low);
        if constexpr (kScaled) {
          const f4v r = E::mfma(a, rest, f4v{0.f, 0.f, 0.f, 0.f});
          o[j] = E::mfma(a, b, o[j]);
#pragma unroll
          for (int c = 0; c < 4; ++c) o[j][c] = fmaf(r[c], 1.f / kRest, o[j][c]);
          // Four at a time: with all eight on their way FP16 heads of 128 take the registers
          // of two workgroups a CU, not three (8 rows of 1,000 to 2,000 with 8 KV heads 17.6
          // us, so 16.6; two of 90,001 to 120,001 with 4 85.4 and 85.3).
          if ((j & 3) == 3) asm volatile("" : "+s"(low), "+s"(high), "+v"(o[j - 3]), "+v"(o[j - 2]), "+v"(o[j - 1]), "+v"(o[j]));
        } else {
          o[j] = E::mfma(a, rest, o[j]);
          o[j] = E::mfma(a, b, o[j]);
        }
      }
    }
    return sum;
  }
  // First dimension of piece n (four dimensions) of accumulator row r.
  static __device__ __forceinline__ int dim_of(int r, int n) {
    const int row = 4 * (lane_id() >> 4) + r;
    return kWide ? 64 * n + 4 * row : kAcc * row + 4 * n;
  }
};

// What both kernels do with an item: its tiles, the waves' partial results, and
// the join of its pieces.
template <typename E, int D, int kStages>
struct AttnShared {
  __attribute__((aligned(16))) float wo[kWaves][16][D + 4];
  float wm[kWaves][16], wl[kWaves][16];
  uint32_t spoilt, last;
};

template <typename E, int D, int kStages, int kPolicy, bool kEarly>
struct Attention {
  static_assert(!kEarly || kStages == 1, "one stage");
  using Tiles = WaveTiles<E, D, kStages, kEarly>;
  using Shared = AttnShared<E, D, kStages>;
  static constexpr int kT = kWaves * kWave, kQuads = D / 4;
  const AttnLaunch &p;
  Shared &sh;
  const int w, lane, col, quad;
  const float scale;  // scores in powers of two
  const uint32_t token_bytes, k_off, rec_m, rec_l;
  uint32_t v_off[4];
  Tiles t;
  uint32_t tile;
  int ahead[2];  // the pages of the tile that is loaded next

  __device__ __forceinline__ Attention(const AttnLaunch &launch, Shared &shared)
      : p(launch),
        sh(shared),
        w(__builtin_amdgcn_readfirstlane(wave_id())),
        lane(lane_id()),
        col(lane & 15),
        quad(lane >> 4),
        scale(p.a.scale * 1.44269504088896340736f),
        token_bytes(static_cast<uint32_t>(p.c.token_stride) * Tiles::kElem),
        k_off(col * token_bytes + 16 * quad),
        rec_m(p.rec_heads * D),
        rec_l(rec_m + p.rec_heads) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v_off[j] = (4 * quad + j) * token_bytes + col * (Tiles::kWide ? 16 : D / 16 * 2);
  }
  __device__ __forceinline__ uint32_t first_head(const Item &x) const {
    return (x.part / p.blocks) * p.group + 16 * (x.part % p.blocks);
  }
  __device__ __forceinline__ int heads_of(const Item &x) const {
    return min(16, static_cast<int>(p.group - 16 * (x.part % p.blocks)));
  }
  // The 16 positions from `pos` on, in page `id`, of K or V.
  template <int kOf>
  __device__ __forceinline__ PageRows<kOf> rows_at(const Item &x, const void *base, uint32_t pos, int id, bool &bad) const {
    const int n = min(max(x.length - static_cast<int>(pos), 0), kSub);
    const bool in = id >= 0 && static_cast<uint32_t>(id) < p.c.pages;
    if (n > 0 && !in) bad = true;
    const int64_t at = (in ? id * p.c.page_stride : 0) + static_cast<int64_t>(pos & (p.c.page_size - 1)) * p.c.token_stride +
                       static_cast<int64_t>(x.part / p.blocks) * p.c.head_stride;
    const uint32_t bytes = n > 0 && in ? (n - 1) * token_bytes + D * Tiles::kElem : 0u;
    char *ptr = const_cast<char *>(static_cast<const char *>(base)) + at * Tiles::kElem;
    return PageRows<kOf>{__builtin_amdgcn_make_buffer_rsrc(ptr, 0, static_cast<int>(bytes), kRsrcWord3)};
  }
  // K stays in the caches, a stream or not: a load takes half of each line, and the
  // next one, the other half, found it gone (64 rows of 0 to 8,192 192 us, so 182).
  __device__ __forceinline__ void load_k(const Item &x, int st, uint32_t at, const int (&id)[2], bool &bad) {
#pragma unroll
    for (int s = 0; s < 2; ++s) t.load_k(rows_at<0>(x, p.c.k, at * kTile + s * kSub, id[s], bad), st, s, k_off);
  }
  __device__ __forceinline__ void load_v(const Item &x, u4v (&to)[2][4][Tiles::kWide ? D / 64 : 1], uint32_t at,
                                         const int (&id)[2], bool &bad) {
#pragma unroll
    for (int s = 0; s < 2; ++s) Tiles::load_v(rows_at<kPolicy>(x, p.c.v, at * kTile + s * kSub, id[s], bad), to[s], v_off);
  }
  // The pages of a wave's tile `at`, -1 past its run.
  __device__ __forceinline__ void pages_of(const Item &x, uint32_t at, int (&id)[2]) const {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const uint32_t pos = at * kTile + s * kSub;
      id[s] = at < x.last && pos < static_cast<uint32_t>(x.length)
                  ? load_uniform(p.c.table + x.row * p.c.table_stride + (pos >> p.page_shift))
                  : -1;
    }
  }
  // The queries and the first tiles of a run are on their way when this returns.
  __device__ __forceinline__ void begin(const Item &x, bool &bad) {
    tile = x.first + w;
    int id[kStages][2];
#pragma unroll
    for (int st = 0; st < kStages; ++st) pages_of(x, tile + st * kWaves, id[st]);
#pragma unroll
    for (int s = 0; s < Tiles::kPieces; ++s) t.q[s] = u4v{0u, 0u, 0u, 0u};
    if (col < heads_of(x)) {
      const char *q = static_cast<const char *>(p.a.q) +
                      (x.row * p.a.q_stride + (first_head(x) + col) * p.a.q_head_stride) * Tiles::kElem + 16 * quad;
#pragma unroll
      for (int s = 0; s < Tiles::kPieces; ++s) t.q[s] = *reinterpret_cast<const u4v *>(q + 64 * s);
    }
#pragma unroll
    for (int st = 0; st < kStages; ++st) {
      if (tile + st * kWaves >= x.last) continue;
      load_k(x, st, tile + st * kWaves, id[st], bad);
      load_v(x, t.v[st], tile + st * kWaves, id[st], bad);
    }
    pages_of(x, tile + kStages * kWaves, ahead);
  }
  __device__ __forceinline__ void tile_through(const Item &it, int st, bool &bad) {
    const bool more = tile + kStages * kWaves < it.last;
    float s[2][4];
#pragma unroll
    for (int sub = 0; sub < 2; ++sub) {
      const f4v x = t.scores(st, sub);
#pragma unroll
      for (int r = 0; r < 4; ++r) s[sub][r] = x[r] * scale;
    }
    if (more) {
      load_k(it, st, tile + kStages * kWaves, ahead, bad);
      if constexpr (kEarly) load_v(it, t.v_next, tile + kWaves, ahead, bad);
    }
    if (static_cast<int>((tile + 1) * kTile) > it.length)
#pragma unroll
      for (int sub = 0; sub < 2; ++sub)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (static_cast<int>(tile * kTile + sub * kSub + 4 * quad + r) >= it.length) s[sub][r] = -INFINITY;
    float top = s[0][0];
#pragma unroll
    for (int i = 1; i < 8; ++i) top = fmaxf(top, s[i >> 2][i & 3]);
    if (__any(top > t.m + kLazyMax<E>)) {
      const float m = fmaxf(t.m, quarters_max(top));
      const float f = m == t.m ? 1.f : exp2_fast(t.m - m);
      t.m = m;
      t.ms = m == -INFINITY ? 0.f : m;
      t.l *= f;
#pragma unroll
      for (int j = 0; j < Tiles::kAcc; ++j) t.o[j] *= f;
    }
    float pr[2][4];
#pragma unroll
    for (int sub = 0; sub < 2; ++sub)
#pragma unroll
      for (int r = 0; r < 4; ++r) pr[sub][r] = exp2_fast(s[sub][r] - t.ms);
    t.l += t.accumulate(st, pr);
    if (more) {
      if constexpr (kEarly) {
#pragma unroll
        for (int sub = 0; sub < 2; ++sub)
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int n = 0; n < (Tiles::kWide ? D / 64 : 1); ++n) t.v[0][sub][j][n] = t.v_next[sub][j][n];
      } else {
        load_v(it, t.v[st], tile + kStages * kWaves, ahead, bad);
      }
    }
    tile += kWaves;
    pages_of(it, tile + kStages * kWaves, ahead);
  }
  __device__ __forceinline__ void run(const Item &it, bool &bad) {
#pragma unroll
    for (int j = 0; j < Tiles::kAcc; ++j) t.o[j] = f4v{0.f, 0.f, 0.f, 0.f};
    t.m = -INFINITY;
    t.ms = 0.f;
    t.l = 0.f;
    static_assert(kStages <= 2, "the loop's two steps");
    for (;;) {
      if (tile >= it.last) break;
      tile_through(it, 0, bad);
      if constexpr (kStages > 1) {
        if (tile >= it.last) break;
        tile_through(it, 1, bad);
      }
    }
  }
  __device__ __forceinline__ void emit(const Item &x, int h, int d, float4 acc, float sum, float poison) const {
    // A row without positions: zeros.
    const float inv = x.length == 0 ? 0.f : 1.f / sum;
    const int64_t at = x.row * p.a.out_stride + (first_head(x) + h) * p.a.out_head_stride + d;
    store4<E>(p.a.out, at,
              make_float4(acc.x * inv + poison, acc.y * inv + poison, acc.z * inv + poison, acc.w * inv + poison));
  }
  // The waves' partial results to LDS. A barrier before the next ones.
  __device__ __forceinline__ void put_partials() {
    constexpr float unit = Tiles::kScaled ? 1.f / kWeight : 1.f;
    const float l = quarters_sum(t.l);
    if (quad == 0) {
      sh.wm[w][col] = t.m;
      sh.wl[w][col] = l;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int n = 0; n < D / 64; ++n)
        *reinterpret_cast<float4 *>(&sh.wo[w][col][Tiles::dim_of(r, n)]) =
            make_float4(t.o[4 * n][r] * unit, t.o[4 * n + 1][r] * unit, t.o[4 * n + 2][r] * unit, t.o[4 * n + 3][r] * unit);
  }
  // The piece's result, out or to its record. sh.spoilt is zero, and is again.
  __device__ __forceinline__ void put_piece(const Item &it, bool bad, float *record) {
    if (bad || it.bad) sh.spoilt = 1u;
    __syncthreads();
    const bool spoilt = sh.spoilt;
    const float poison = spoilt ? __uint_as_float(0x7FC00000u) : 0.f;
    const int heads = heads_of(it);
    const bool whole = it.pieces == 1;
    const Coherent rec(record, p.rec_floats * static_cast<uint32_t>(sizeof(float)));
    for (int i = threadIdx.x; i < heads * kQuads; i += kT) {
      const int h = i / kQuads, d = 4 * (i % kQuads);
      float mx = -INFINITY;
#pragma unroll
      for (int u = 0; u < kWaves; ++u) mx = fmaxf(mx, sh.wm[u][h]);
      float sum = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int u = 0; u < kWaves; ++u) {
        const float f = sh.wm[u][h] == mx ? 1.f : exp2_fast(sh.wm[u][h] - mx);
        const float4 x = *reinterpret_cast<const float4 *>(&sh.wo[u][h][d]);
        sum = fmaf(f, sh.wl[u][h], sum);
        acc.x = fmaf(f, x.x, acc.x);
        acc.y = fmaf(f, x.y, acc.y);
        acc.z = fmaf(f, x.z, acc.z);
        acc.w = fmaf(f, x.w, acc.w);
      }
      if (whole) {
        emit(it, h, d, acc, sum, poison);
      } else {
        rec.st4((h * D + d) / 4, make_float4(acc.x + poison, acc.y + poison, acc.z + poison, acc.w + poison));
        if (d == 0) {
          rec.st(rec_m + h, mx);
          rec.st(rec_l + h, sum);
        }
      }
    }
    if (spoilt) {
      if (threadIdx.x == 0) raise_error(p.c.errors, it.bad ? QD_PAGED_BAD_LENGTH : QD_PAGED_BAD_PAGE);
      __syncthreads();
      sh.spoilt = 0u;
    }
  }
  // Counts the piece in; true in the workgroup whose piece came last.
  __device__ __forceinline__ bool arrive(const Item &it) {
    wait_vm_stores();
    __syncthreads();
    uint32_t *cnt = p.counters + (static_cast<size_t>(it.row) * p.parts + it.part) * p.apart;
    if (threadIdx.x == 0) {
      sh.last = atomicAdd(cnt, 1u) == it.pieces - 1;
      if (sh.last) *cnt = 0u;
    }
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(sh.last);
  }
  // Joins an item's pieces in their order: each head's weights of the pieces, by a
  // wave per head with every maximum and sum on its way at once, then the weighted
  // sums, shared out among the threads. Piece c > 0 is `second` + (c - 1) * stride
  // floats behind piece 0.
  template <uint32_t kMost>  // pieces
  __device__ __forceinline__ void join(const Item &x, const float *records, uint32_t second, uint32_t stride) {
    float(*weight)[kMost] = reinterpret_cast<float(*)[kMost]>(&sh.wo[0][0][0]);
    static_assert(sizeof(float) * 16 * kMost <= sizeof(sh.wo), "a weight per head and piece");
    const int heads = heads_of(x);
    const uint32_t of = x.pieces;
    const Coherent recs(records, (second + (of - 2) * stride + p.rec_floats) * static_cast<uint32_t>(sizeof(float)));
    auto at_piece = [&](uint32_t c) { return c == 0 ? 0u : second + (c - 1) * stride; };
    const int items = heads * kQuads, shares = max(1, kT / items);
    const int i0 = static_cast<int>(threadIdx.x) % min(items, kT), share = threadIdx.x / min(items, kT);
    constexpr int kAhead = 8;
    float4 next[kAhead];
    auto fetch = [&](int i, uint32_t c) {
      const int h = i / kQuads, d = 4 * (i % kQuads);
#pragma unroll
      for (int u = 0; u < kAhead; ++u) next[u] = recs.ld4((at_piece(min(c + u * shares, of - 1)) + h * D + d) / 4);
    };
    // A wave's heads' maxima and sums: all on their way at once where the pieces are no
    // more than lanes (16 beams at 576 8.5 us, head after head 8.95).
    constexpr int kPer = kMost / kWave, kSlots = kPer == 1 ? 16 / kWaves : 1;
    float cm[kSlots][kPer], cl[kSlots][kPer];
    auto load_head = [&](int h, int slot) {
#pragma unroll
      for (int u = 0; u < kPer; ++u) {
        const uint32_t c = u * kWave + lane;
        cm[slot][u] = -INFINITY;
        cl[slot][u] = 0.f;
        if (h < heads && u * kWave < of && c < of) {
          cm[slot][u] = recs.ld(at_piece(c) + rec_m + h);
          cl[slot][u] = recs.ld(at_piece(c) + rec_l + h);
        }
      }
    };
    auto weigh_head = [&](int h, int slot) {
      if (h >= heads) return;
      float m = -INFINITY, sum = 0.f;
#pragma unroll
      for (int u = 0; u < kPer; ++u) m = fmaxf(m, cm[slot][u]);
      m = wave_max(m);
#pragma unroll
      for (int u = 0; u < kPer; ++u) {
        const uint32_t c = u * kWave + lane;
        if (c >= of) continue;
        const float f = cm[slot][u] == m ? 1.f : exp2_fast(cm[slot][u] - m);
        weight[h][c] = f;
        sum = fmaf(f, cl[slot][u], sum);
      }
      sum = wave_sum(sum);
      if (lane == 0) sh.wl[0][h] = sum;
    };
    if constexpr (kSlots > 1) {
#pragma unroll
      for (int i = 0; i < kSlots; ++i) load_head(w + i * kWaves, i);
    }
    fetch(min(i0, items - 1), min(static_cast<uint32_t>(share), of - 1));
    __syncthreads();  // the partial results have been read
    if constexpr (kSlots > 1) {
#pragma unroll
      for (int i = 0; i < kSlots; ++i) weigh_head(w + i * kWaves, i);
    } else {
      for (int h = w; h < heads; h += kWaves) {
        load_head(h, 0);
        weigh_head(h, 0);
      }
    }
    __syncthreads();
    for (int base = 0; base < items; base += kT) {
      const int i = base + i0, h = i / kQuads, d = 4 * (i % kQuads);
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      if (share < shares && i < items) {
        for (uint32_t c = share; c < of; c += kAhead * shares) {
          if (base > 0 || c != static_cast<uint32_t>(share)) fetch(i, c);
#pragma unroll
          for (int u = 0; u < kAhead; ++u) {
            if (c + u * shares >= of) continue;
            const float f = weight[h][c + u * shares];
            acc.x = fmaf(f, next[u].x, acc.x);
            acc.y = fmaf(f, next[u].y, acc.y);
            acc.z = fmaf(f, next[u].z, acc.z);
            acc.w = fmaf(f, next[u].w, acc.w);
          }
        }
      }
      if (shares > 1) {  // (then there is one pass: the weights are read no more)
        float4 *sums = reinterpret_cast<float4 *>(&sh.wo[0][0][0]);
        __syncthreads();
        sums[threadIdx.x] = acc;
        __syncthreads();
        if (share == 0)
          for (int u = 1; u < shares; ++u) {
            const float4 y = sums[threadIdx.x + u * items];
            acc = make_float4(acc.x + y.x, acc.y + y.y, acc.z + y.z, acc.w + y.w);
          }
      }
      if (share == 0 && i < items) emit(x, h, d, acc, sh.wl[0][h], 0.f);
    }
  }
};

// Workgroups of the short kernel that a CU holds, which its pieces are made for (16
// beams at 576 positions in pieces of 4 tiles or more 8.9 us, of 8 10.8, before the
// join took its loads at once; 4 rows of 3,000 with 8 KV heads of 128 in about 512
// pieces 15.5 us, in 768 18.6; 64 rows to 2,000 with 2 of 64 21.9 in 512, 20.4 in 768)
// and its registers: FP32 heads of 128 in as many as they like, one a CU, 4 rows of
// 2,000 to 4,000 with 4 heads 23.8 us, in those of two 20.3.
constexpr uint32_t short_per_cu(uint32_t head_dim) { return head_dim == 128 ? 2 : 3; }

// Few positions in all: a workgroup per piece, no more than `target` pieces
// besides one for each item. Short code and one dependent load less, because each
// step of such a call waits for the one before it.
template <typename E, int D>
__global__ __launch_bounds__(kWaves *kWave, short_per_cu(D)) void attention_short_kernel(AttnLaunch p) {
  __shared__ AttnShared<E, D, 1> sh;
  Item it;
  const uint32_t part = blockIdx.x % p.parts;
  uint32_t begin;
  if (!find_piece(p, blockIdx.x / p.parts, part, it, begin)) return;
  if (threadIdx.x == 0) sh.spoilt = 0u;
  Attention<E, D, 1, 0, D == 64> a(p, sh);
  bool bad = false;
  a.begin(it, bad);
  a.run(it, bad);
  a.put_partials();
  const uint32_t stride = p.parts * p.rec_floats;
  float *first = p.records + (static_cast<size_t>(begin) * p.parts + part) * p.rec_floats;
  __syncthreads();
  a.put_piece(it, bad, first + static_cast<size_t>(it.home) * stride);
  if (it.pieces == 1) return;
  if (a.arrive(it)) a.template join<kShortPieces>(it, first, stride, stride);
}

// Many: equal runs of all tiles, one for each workgroup that the card holds. V is read
// as a stream, as so much is not read again before others have taken its place: 16 rows
// of 2,000 to 4,000 of one layer after the other 45.6 us, by the caches 48.6 (of one
// layer again and again, 208 MB, 40.0 and 38.6), 64 of 0 to 8,192 182 and 202.
template <typename E, int D, int kStages>
__global__ __launch_bounds__(kWaves *kWave) void attention_long_kernel(AttnLaunch p) {
  __shared__ AttnShared<E, D, kStages> sh;
  const uint32_t group_id = blockIdx.x;
  Deal deal;
  Item it;
  if (!first_item(p, group_id, gridDim.x, deal, it)) return;
  if (threadIdx.x == 0) sh.spoilt = 0u;
  Attention<E, D, kStages, kPolicyNt, false> a(p, sh);
  // The record of an item's piece: its workgroup's first if it begins inside the item, else the second.
  auto record_of = [&](const Item &x, uint32_t piece) {
    return p.records + (2 * static_cast<size_t>(x.home + piece) + (piece == 0)) * p.rec_floats;
  };
  // At most the first and the last item of a run have other pieces.
  Item join[2];
  int to_join = 0;
  bool bad = false;
  a.begin(it, bad);
  for (;;) {
    a.run(it, bad);
    a.put_partials();
    // The next item's loads are under way while this one's results are put together.
    Item next;
    const bool more = next_item(p, deal, group_id, it, next);
    bool next_bad = false;
    if (more) a.begin(next, next_bad);
    __syncthreads();
    const bool whole = it.pieces == 1;
    a.put_piece(it, bad, record_of(it, whole ? 0 : group_id - it.home));
    if (!whole && a.arrive(it)) {
      join[1] = join[0];
      join[0] = it;
      ++to_join;
    }
    if (!more) break;
    __syncthreads();  // LDS is written again
    it = next;
    bad = next_bad;
  }
  for (; to_join > 0; --to_join, join[0] = join[1]) {
    if (join[0].pieces <= kShortPieces)
      a.template join<kShortPieces>(join[0], record_of(join[0], 0), p.rec_floats, 2 * p.rec_floats);
    else
      a.template join<kMostPieces>(join[0], record_of(join[0], 0), p.rec_floats, 2 * p.rec_floats);
    __syncthreads();
  }
}

// ---- fork -----------------------------------------------------------------------
// The first kernel, one workgroup, counts references, decides which rows copy
// their last page and deals out free pages; the second writes the new table and
// copies pages. The first is bound by latency, a few dependent passes over tables
// and counts (16 beams over pages of 24 layers: 4.5 of 8.8 us); the copies stream (64
// rows that copy about 22 pages of 2 x 8 layers x 128 KB, 91 MB, 23.5 us in all).
constexpr int kForkT = 1024, kForkWaves = kForkT / kWave;
constexpr int kForkScan = 8;   // counts that a thread looks at for free pages per pass
// Rows of a wave that are on their way (256 rows of 4 beams 24.0 us, two at a time
// 24.6, eight 23.4, but then 8 x 8 beams 23.8 instead of 23.5).
constexpr int kForkEarly = 4;

struct ForkRow {
  int32_t parent;   // -1: released
  int32_t held;     // pages taken over
  int32_t source;   // the page to copy, or -1
  uint32_t begin;   // its fresh pages in the free list, the copy's first
  int32_t fresh;
  int32_t length;
};
struct ForkPlan {
  uint32_t ok, copies;
};
struct ForkLaunch {
  qd_fork_args a;        // (a.memories is not for the device)
  qd_page_memory memory[kForkMemories];
  uint32_t page_shift;
  ForkPlan *plan;
  ForkRow *row;          // [rows]
  int32_t *copy_source;  // [rows] page pairs to copy
  int32_t *copy_to;
  int32_t *free_pages;   // [pages]
  uint32_t blocks;       // 16 KiB pieces of one page in all memories and planes
};

__device__ __forceinline__ int32_t load_count(int32_t *p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Sum over the lanes before this one, and over all waves before.
__device__ __forceinline__ uint32_t block_before(uint32_t v, uint32_t *waves, uint32_t &total) {
  const uint32_t upto = lanes_upto(v);
  __syncthreads();
  if (lane_id() == kWave - 1) waves[wave_id()] = upto;
  __syncthreads();
  uint32_t before = 0;
  total = 0;
#pragma unroll
  for (int u = 0; u < kForkWaves; ++u) {
    if (u < wave_id()) before += waves[u];
    total += waves[u];
  }
  return before + upto - v;
}

// The first columns of a row, a lane each.
__device__ __forceinline__ int32_t first_columns(const ForkLaunch &p, uint32_t r) {
  const uint32_t lane = lane_id();
  return r < p.a.rows && lane < p.a.table_width ? p.a.table[r * p.a.table_stride + lane] : -1;
}

// Adds `sign` times what the fork changes: a page that an old row takes over to
// c children counts c - 1 more, one behind its length one less. `early` holds the
// first columns of each wave's first rows; those of later ones are asked for as many
// rows ahead.
__device__ __forceinline__ void count_references(const ForkLaunch &p, const int *children, const int *lengths, int sign,
                                                 const int32_t (&early)[kForkEarly], uint32_t *bad) {
  const int lane = lane_id();
  int32_t columns[kForkEarly];
#pragma unroll
  for (int u = 0; u < kForkEarly; ++u) columns[u] = early[u];
  for (uint32_t r = wave_id(); r < p.a.rows; r += kForkWaves) {
    const int32_t first = columns[0];
#pragma unroll
    for (int u = 0; u + 1 < kForkEarly; ++u) columns[u] = columns[u + 1];
    columns[kForkEarly - 1] = first_columns(p, r + kForkEarly * kForkWaves);
    const int32_t *table = p.a.table + r * p.a.table_stride;
    const uint32_t held = (static_cast<uint32_t>(lengths[r]) + p.a.page_size - 1) >> p.page_shift;
    const int change = children[r] - 1;
    for (uint32_t base = 0;; base += kWave) {
      const uint32_t j = base + lane;
      const int32_t id = base == 0 ? first : j < p.a.table_width ? table[j] : -1;
      // Entries behind the first negative one, or the last column, are none.
      const uint64_t ends = __ballot(id < 0);
      if ((ends & ((1ull << lane) - 1)) == 0 && id >= 0) {
        if (static_cast<uint32_t>(id) >= p.a.pages)
          atomicOr(bad, QD_PAGED_BAD_PAGE);
        else if (j >= held)
          atomicAdd(p.a.refs + id, -sign);
        else if (change)
          atomicAdd(p.a.refs + id, sign * change);
      }
      if (ends) {
        // A row that ends before its length lacks a page.
        const uint32_t end = base + __ffsll(static_cast<unsigned long long>(ends)) - 1;
        if (end < held && lane == 0) atomicOr(bad, QD_PAGED_BAD_PAGE);
        break;
      }
    }
  }
}

__global__ __launch_bounds__(kForkT) void fork_plan_kernel(ForkLaunch p) {
  constexpr int kList = 1024;  // free pages kept in LDS too
  __shared__ __attribute__((aligned(16))) int last[kForkRows];  // -1 behind the rows
  __shared__ int children[kForkRows], lengths[kForkRows], list[kList];
  __shared__ uint32_t waves[kForkWaves], bad, copies;
  const uint32_t r = threadIdx.x;  // one thread per row where rows are meant
  static_assert(kForkT == kForkRows, "a thread per row");
  const int64_t room = static_cast<int64_t>(p.a.table_width) << p.page_shift;
  // Nothing here waits for another: the wave's first rows, the lengths and parents.
  int32_t early[kForkEarly];
#pragma unroll
  for (int u = 0; u < kForkEarly; ++u) early[u] = first_columns(p, wave_id() + u * kForkWaves);
  ForkRow row{-1, 0, -1, 0u, 0, 0};
  if (r < p.a.rows) {
    children[r] = 0;
    lengths[r] = p.a.lengths[r];
    row.parent = p.a.parents ? p.a.parents[r] : static_cast<int32_t>(r);
  }
  if (r == 0) bad = copies = 0;
  __syncthreads();
  int32_t id = -1;  // the page in which the row goes on
  if (r < p.a.rows) {
    if (lengths[r] < 0 || lengths[r] > room) atomicOr(&bad, QD_PAGED_BAD_LENGTH);
    if (row.parent < -1 || row.parent >= static_cast<int32_t>(p.a.rows)) {
      atomicOr(&bad, QD_PAGED_BAD_ROW);
      row.parent = -1;
    }
    if (row.parent >= 0) {
      row.length = lengths[row.parent];
      if (row.length < 0 || row.length + static_cast<int64_t>(p.a.append) > room) {
        atomicOr(&bad, QD_PAGED_BAD_LENGTH);
      } else {
        row.held = (row.length + p.a.page_size - 1) >> p.page_shift;
        if (p.a.append && (row.length & (p.a.page_size - 1)))
          id = p.a.table[row.parent * p.a.table_stride + row.held - 1];
      }
      atomicAdd(&children[row.parent], 1);
    }
  }
  last[r] = id;
  __syncthreads();
  const bool fits = bad == 0;
  __syncthreads();
  if (fits) count_references(p, children, lengths, 1, early, &bad);
  wait_vm_stores();  // the counts stand in L2 before any of them is read
  __syncthreads();
  const bool sound = bad == 0;
  uint32_t wanted = 0, found = 0;
  if (sound) {
    // The counts of the row's page and of the first pages, for the free ones.
    const int held_by = id >= 0 ? load_count(p.a.refs + id) : 0;
    int32_t n[kForkScan];
    auto look = [&](uint32_t base) {
#pragma unroll
      for (int u = 0; u < kForkScan; ++u) {
        const uint32_t page = base + r * kForkScan + u;
        n[u] = page < p.a.pages ? load_count(p.a.refs + page) : 1;
      }
    };
    look(0);
    if (id >= 0) {
      int holders = 0, lowest = kForkRows;
      for (int u = 0; u < static_cast<int>(p.a.rows); u += 8) {
        const int4 a = *reinterpret_cast<const int4 *>(last + u), b = *reinterpret_cast<const int4 *>(last + u + 4);
        const int ids[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (int v = 7; v >= 0; --v)
          if (ids[v] == id) {
            ++holders;
            lowest = min(lowest, u + v);
          }
      }
      if (held_by != holders || lowest != static_cast<int>(r)) row.source = id;
    }
    if (row.parent >= 0) {
      const uint32_t need = (static_cast<uint32_t>(row.length) + p.a.append + p.a.page_size - 1) >> p.page_shift;
      row.fresh = static_cast<int>(need) - row.held + (row.source >= 0);
    }
    row.begin = block_before(row.fresh, waves, wanted);
    // A row takes no more pages than the table has columns. Where all rows' may pass 32
    // bits, they are counted by 256 first: more of those than the pool has are too many,
    // and with no more the sum is below 2^31 + 2^18. (A table of 16 GB or more: the
    // others do without the second sum.)
    if (static_cast<uint64_t>(p.a.rows) * p.a.table_width >> 32) {
      uint32_t parts;
      block_before(static_cast<uint32_t>(row.fresh) >> 8, waves, parts);
      if (parts > p.a.pages >> 8) wanted = UINT32_MAX;
    }
    // The free pages of the lowest ids.
    for (uint32_t base = 0; base < p.a.pages && found < wanted; base += kForkT * kForkScan) {
      if (base) look(base);
      uint32_t mine = 0, here = 0;
#pragma unroll
      for (int u = 0; u < kForkScan; ++u) mine += n[u] == 0;
      uint32_t at = found + block_before(mine, waves, here);
#pragma unroll
      for (int u = 0; u < kForkScan; ++u)
        if (n[u] == 0) {
          const int32_t page = static_cast<int32_t>(base + r * kForkScan + u);
          if (at < wanted) p.free_pages[at] = page;
          if (at < static_cast<uint32_t>(kList)) list[at] = page;
          ++at;
        }
      found += here;
    }
    if (wanted > kList) wait_vm_stores();  // the rest is read back below
  }
  __syncthreads();
  if (!sound || found < wanted) {
    const uint32_t error = sound ? static_cast<uint32_t>(QD_PAGED_EXHAUSTED) : bad;
    __syncthreads();
    if (fits) count_references(p, children, lengths, -1, early, &bad);
    if (r == 0) {
      raise_error(p.a.errors, error);
      p.plan->ok = 0;
      p.plan->copies = 0;
    }
    return;
  }
  if (r < p.a.rows) {
    for (int u = 0; u < row.fresh; ++u) {
      const uint32_t at = row.begin + u;
      const int32_t page = at < static_cast<uint32_t>(kList) ? list[at] : p.free_pages[at];
      p.a.refs[page] = 1;
      if (u == 0 && row.source >= 0) {
        atomicSub(p.a.refs + row.source, 1);
        const uint32_t to = atomicAdd(&copies, 1u);
        p.copy_source[to] = row.source;
        p.copy_to[to] = page;
      }
    }
    p.row[r] = row;
  }
  __syncthreads();
  if (r == 0) {
    p.plan->ok = 1;
    p.plan->copies = copies;
  }
}

constexpr uint32_t kCopyPiece = 16384;

__global__ __launch_bounds__(kBlock) void fork_copy_kernel(ForkLaunch p) {
  const ForkPlan plan = *p.plan;
  if (blockIdx.x < p.a.rows) {
    const uint32_t r = blockIdx.x;
    const ForkRow row = plan.ok ? p.row[r] : ForkRow{};
    const int32_t *from = p.a.table + (plan.ok ? max(row.parent, 0) : static_cast<int32_t>(r)) * p.a.table_stride;
    int32_t *to = p.a.table_out + r * p.a.table_out_stride;
    const int copied = row.source >= 0;
    for (uint32_t j = threadIdx.x; j < p.a.table_width; j += kBlock) {
      int32_t id = -1;
      if (!plan.ok) {
        id = from[j];
      } else if (static_cast<int>(j) < row.held) {
        id = copied && static_cast<int>(j) == row.held - 1 ? p.free_pages[row.begin] : from[j];
      } else if (static_cast<int>(j) < row.held + row.fresh - copied) {
        id = p.free_pages[row.begin + copied + j - row.held];
      }
      to[j] = id;
    }
    if (threadIdx.x == 0)
      p.a.lengths_out[r] = !plan.ok ? p.a.lengths[r] : row.parent < 0 ? 0 : row.length + static_cast<int32_t>(p.a.append);
  }
  const uint64_t work = static_cast<uint64_t>(plan.copies) * p.blocks;
  for (uint64_t unit = blockIdx.x; unit < work; unit += gridDim.x) {
    const uint32_t copy = unit / p.blocks;
    uint32_t piece = unit % p.blocks;
    int64_t page_stride = 0;
    uint64_t bytes = 0;
    char *base = nullptr;
    // (A loop over a constant number of memories: no indexed copy of them in scratch.)
#pragma unroll
    for (uint32_t m = 0; m < kForkMemories; ++m) {
      if (m >= p.a.memory_count || base) continue;
      const uint32_t per_plane = (p.memory[m].bytes + kCopyPiece - 1) / kCopyPiece, all = per_plane * p.memory[m].planes;
      if (piece >= all) {
        piece -= all;
        continue;
      }
      base = static_cast<char *>(p.memory[m].base) + (piece / per_plane) * p.memory[m].plane_stride;
      page_stride = p.memory[m].page_stride;
      bytes = p.memory[m].bytes;
      piece %= per_plane;
    }
    if (!base) continue;
    const uint64_t begin = static_cast<uint64_t>(piece) * kCopyPiece;
    const uint32_t n = min(static_cast<uint64_t>(kCopyPiece), bytes - begin);
    const u4v *src = reinterpret_cast<const u4v *>(base + p.copy_source[copy] * page_stride + begin);
    u4v *dst = reinterpret_cast<u4v *>(base + p.copy_to[copy] * page_stride + begin);
    u4v x[kCopyPiece / 16 / kBlock];
#pragma unroll
    for (uint32_t u = 0; u < kCopyPiece / 16 / kBlock; ++u)
      if ((threadIdx.x + u * kBlock) * 16 < n) x[u] = src[threadIdx.x + u * kBlock];
#pragma unroll
    for (uint32_t u = 0; u < kCopyPiece / 16 / kBlock; ++u)
      if ((threadIdx.x + u * kBlock) * 16 < n) dst[threadIdx.x + u * kBlock] = x[u];
  }
}

__global__ void clear_kernel(uint32_t *p, size_t n) {
  for (size_t i = blockIdx.x * static_cast<size_t>(blockDim.x) + threadIdx.x; i < n; i += static_cast<size_t>(gridDim.x) * blockDim.x) p[i] = 0u;
}

uint32_t log2_of(uint32_t v) { return static_cast<uint32_t>(__builtin_ctz(v)); }

template <typename... A>
hipError_t launch(void (*kernel)(A...), dim3 grid, dim3 block, hipStream_t s, A... args) {
  void *packed[] = {&args...};
  return hipLaunchKernel(reinterpret_cast<const void *>(kernel), grid, block, packed, 0, s);
}

// How attention cuts its work. The long kernel's cuts keep eight tiles from an item's
// ends (as many as two 128 rows of 0 to 4,000 171 us too, 32 183).
constexpr uint32_t kAttnLeast = 8, kCus = 256, kMostPerCu = 2;
// Which kernel, by the bytes of all positions that the tables, or the pool, can
// hold: their real number is on the device. Where rows fill what they can hold, the
// kernels cross between 65 and 120 MB, by type, heads and raggedness: 65 MB of 8 heads of
// 128 in BF16 short 24.8 us, long 22.5; 74 of 4 in FP32 26.7 and 29.1; 98 of 8 in BF16, rows
// of one length, 25.7 and 28.3; 99 of 4 in FP16 32.7 and 30.4; 123 of 2 of 64 in FP32 42.7
// and 39.3. Short rows in a large pool get the long kernel all the same (in pages of 2 GB
// and tables of 32,768 positions, and in a pool of their size: 16 rows of 576 with 2 heads
// of 64 in FP32 13.5 us and 8.5, 8 of 448 with 8 of 128 in BF16 12.2 and 8.0, one of 129 7.1
// and 6.7, one of 3,000 9.2 and 9.2).
constexpr uint64_t kShortBytes = 96ull << 20;
struct AttnShape {
  uint32_t group, blocks, parts, rec_heads, rec_floats, apart, least, target, records;
};
AttnShape attention_shape(uint32_t rows, uint32_t heads, uint32_t kv_heads, uint32_t head_dim) {
  AttnShape s{};
  s.group = heads / kv_heads;
  s.blocks = (s.group + 15) / 16;
  s.parts = kv_heads * s.blocks;
  s.rec_heads = std::min(s.group, 16u);
  s.rec_floats = (s.rec_heads * (head_dim + 2) + 3) / 4 * 4;
  const uint64_t items = static_cast<uint64_t>(rows) * s.parts;
  if (items <= kOpCounters) {
    s.least = kAttnLeast;
    s.target = std::max(1u, kCus * short_per_cu(head_dim) / s.parts);
    s.records = std::max((rows + s.target) * s.parts, 2 * kCus * kMostPerCu);
    // Counters in lines of their own where there is room.
    for (s.apart = 32; items * s.apart > kOpCounters;) s.apart /= 2;
  }
  return s;
}

size_t round256(size_t n) { return (n + 255) / 256 * 256; }

}  // namespace

hipError_t launch_op_clear(hipStream_t s, uint32_t *counters, size_t n) {
  return launch(clear_kernel, dim3(64), dim3(kBlock), s, counters, n);
}

hipError_t launch_paged_append(hipStream_t s, const qd_paged_cache &c, const qd_append_args &a) {
  if (a.tokens == 0) return hipSuccess;
  AppendLaunch p{c, a, log2_of(c.page_size), c.head_dim == 128 ? 4u : 3u, 0};
  // (A wave that holds four rows of a token at a time was no faster: 6,000 tokens of
  // 48 heads of 128 in BF16 36.4 us against 35.3.)
  const uint32_t rows = (a.q ? a.heads : 0) + 2 * c.kv_heads, at_once = kWave >> p.lanes_shift;
  p.waves = (rows + at_once - 1) / at_once;
  const dim3 grid((static_cast<uint64_t>(a.tokens) * p.waves + kWavesPerBlock - 1) / kWavesPerBlock);
  const dim3 block(kBlock);
  switch (c.dtype) {
    case QD_DTYPE_F32: return launch(append_kernel<float>, grid, block, s, p);
    case QD_DTYPE_BF16: return launch(append_kernel<Brain>, grid, block, s, p);
    default: return launch(append_kernel<Half>, grid, block, s, p);
  }
}

size_t paged_attention_scratch(uint32_t rows, uint32_t heads, uint32_t kv_heads, uint32_t head_dim) {
  const AttnShape sh = attention_shape(rows, heads, kv_heads, head_dim);
  return static_cast<size_t>(sh.records) * sh.rec_floats * sizeof(float);
}

// (More rows than there are counters for are not cut and keep nothing; fewer are.)
size_t paged_attention_scratch_most(uint32_t rows, uint32_t heads, uint32_t kv_heads, uint32_t head_dim) {
  const uint32_t parts = attention_shape(0, heads, kv_heads, head_dim).parts;
  return paged_attention_scratch(std::min(rows, static_cast<uint32_t>(kOpCounters / parts)), heads, kv_heads, head_dim);
}

// The long kernel's tiles ahead and workgroups on a CU, by type and head_dim: with 64
// to 128 KB on their way to each CU, more only queue. Measured on 430 to 680 MB, tiles
// x workgroups: FP32 of 128 1 x 1 66.9 us, 2 x 1 68.6, 1 x 2 71.6; FP32 of 64 2 x 1 47.8,
// 1 x 2 48.4, 3 x 1 48.9; 16 bits of 128 2 x 1 66.1, 3 x 1 67.1, 1 x 2 69.2; 16 bits of
// 64 1 x 2 61.4, 1 x 3 65.7, 2 x 2 64.6, 2 x 1 66.5.
template <typename E, int D, int kStages, int per_cu>
static hipError_t launch_attention(hipStream_t s, AttnLaunch &p) {
  static_assert(per_cu <= static_cast<int>(kMostPerCu), "records");
  const uint64_t most = ((static_cast<uint64_t>(p.c.table_width) << p.page_shift) + kTile - 1) / kTile;
  const uint64_t position = 2ull * p.c.kv_heads * D * (std::is_same_v<E, float> ? 4 : 2);
  const uint64_t pool = static_cast<uint64_t>(p.c.pages) * p.c.page_size;
  const uint64_t positions = std::min<uint64_t>(static_cast<uint64_t>(p.c.rows) * p.c.table_width << p.page_shift, pool);
  const dim3 block(kWaves * kWave);
  if (positions * position <= kShortBytes || p.least == 0) {
    if (most <= kShortWhole) p.target = 0;
    uint64_t x = p.c.rows;
    if (p.target) x = std::min<uint64_t>(x + p.target, x * ((most + kShortLeast - 1) / kShortLeast));
    return launch(attention_short_kernel<E, D>, dim3(static_cast<uint32_t>(x * p.parts)), block, s, p);
  }
  return launch(attention_long_kernel<E, D, kStages>, dim3(kCus * per_cu), block, s, p);
}

hipError_t launch_paged_attention(hipStream_t s, const qd_paged_cache &c, const qd_attention_args &a, const OpScratch &w) {
  if (c.rows == 0) return hipSuccess;
  const AttnShape sh = attention_shape(c.rows, a.heads, c.kv_heads, c.head_dim);
  AttnLaunch p{};
  p.c = c;
  p.a = a;
  p.records = reinterpret_cast<float *>(w.scratch);
  p.counters = w.counters;
  p.page_shift = log2_of(c.page_size);
  p.group = sh.group;
  p.blocks = sh.blocks;
  p.rec_heads = sh.rec_heads;
  p.rec_floats = sh.rec_floats;
  p.apart = sh.apart;
  p.parts = sh.parts;
  p.least = sh.least;
  p.target = sh.target;
  const bool wide = c.head_dim == 128;
  switch (c.dtype) {
    case QD_DTYPE_F32: return wide ? launch_attention<float, 128, 1, 1>(s, p) : launch_attention<float, 64, 2, 1>(s, p);
    case QD_DTYPE_BF16: return wide ? launch_attention<Brain, 128, 2, 1>(s, p) : launch_attention<Brain, 64, 1, 2>(s, p);
    default: return wide ? launch_attention<Half, 128, 2, 1>(s, p) : launch_attention<Half, 64, 1, 2>(s, p);
  }
}

size_t pages_fork_scratch(uint32_t rows, uint32_t pages) {
  return round256(sizeof(ForkPlan)) + round256(rows * sizeof(ForkRow)) + 2 * round256(rows * sizeof(int32_t)) +
         round256(static_cast<size_t>(pages) * sizeof(int32_t));
}

hipError_t launch_pages_fork(hipStream_t s, const qd_fork_args &a, const OpScratch &w) {
  if (a.rows == 0) return hipSuccess;
  ForkLaunch p{};
  p.a = a;
  p.a.memories = nullptr;
  uint64_t blocks = 0;
  for (uint32_t m = 0; m < a.memory_count; ++m) {
    p.memory[m] = a.memories[m];
    blocks += (p.memory[m].bytes + kCopyPiece - 1) / kCopyPiece * p.memory[m].planes;
  }
  p.page_shift = log2_of(a.page_size);
  p.blocks = static_cast<uint32_t>(blocks);
  char *at = w.scratch;
  auto take = [&](size_t bytes) {
    char *r = at;
    at += round256(bytes);
    return r;
  };
  p.plan = reinterpret_cast<ForkPlan *>(take(sizeof(ForkPlan)));
  p.row = reinterpret_cast<ForkRow *>(take(a.rows * sizeof(ForkRow)));
  p.copy_source = reinterpret_cast<int32_t *>(take(a.rows * sizeof(int32_t)));
  p.copy_to = reinterpret_cast<int32_t *>(take(a.rows * sizeof(int32_t)));
  p.free_pages = reinterpret_cast<int32_t *>(take(static_cast<size_t>(a.pages) * sizeof(int32_t)));
  const hipError_t err = launch(fork_plan_kernel, dim3(1), dim3(kForkT), s, p);
  if (err != hipSuccess) return err;
  const uint64_t most = std::max<uint64_t>(a.rows, std::min<uint64_t>(a.rows * blocks, 2048));
  return launch(fork_copy_kernel, dim3(static_cast<uint32_t>(most)), dim3(kBlock), s, p);
}

}  // namespace qd
