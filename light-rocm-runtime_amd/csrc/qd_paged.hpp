// Device helpers of the operators on paged caches (qd_paged.hip, qd_tree.hip,
// qd_sparse.hip): the storage types, moves between lanes, and the launch.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>
#include <type_traits>

#include "qd_device.hpp"
#include "qd_device_math.hpp"

namespace qd {
namespace dev {

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

// Lane `from`'s value.
__device__ __forceinline__ uint64_t lane_of(uint64_t v, int from) {
  const uint32_t lo = __builtin_amdgcn_ds_bpermute(from << 2, static_cast<int>(v));
  const uint32_t hi = __builtin_amdgcn_ds_bpermute(from << 2, static_cast<int>(v >> 32));
  return static_cast<uint64_t>(hi) << 32 | lo;
}
__device__ __forceinline__ double lane_of(double v, int from) {
  return __builtin_bit_cast(double, lane_of(__builtin_bit_cast(uint64_t, v), from));
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


// ---- equal runs ----------------------------------------------------------------
// A launch's rows have `parts` items each, of tiles of kTile positions (one at least), which are
// dealt to the workgroups in equal runs. L is the launch: c (rows, lengths, table_width), page_shift,
// parts and least, the tiles on either side of a cut; 0: items are not cut.
constexpr uint32_t kMostPieces = 256;  // of an item
// Tiles that an item's results cost the long kernel as much time as: 128 rows of 0 to
// 4,000 took 171 us, counted as none 177, as one 176, as four 173.
constexpr uint32_t kEdge = 2;

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

template <int kTile, typename L>
__device__ __forceinline__ uint32_t tiles_of(const L &p, int32_t n, int64_t most) {
  return n <= 0 || n > most ? 1u : (static_cast<uint32_t>(n) + kTile - 1) / kTile;
}

// How a cut `off` tiles into an item of n moves: 0 to its start, 1 not, 2 to its end.
template <typename L>
__device__ __forceinline__ int cut_of(const L &p, uint32_t off, uint32_t n) {
  if (p.least && n >= 2 * p.least) return off < p.least ? 0 : n - off < p.least ? 2 : 1;
  return 2 * off < n ? 0 : 2;
}

template <int kTile, typename L>
__device__ __forceinline__ void set_item(const L &p, const Deal &d, Item &it, uint32_t row, uint32_t part,
                                         uint32_t at, int32_t n, int64_t most) {
  it.row = static_cast<int>(row);
  it.part = part;
  it.at = at + kEdge;
  it.bad = n < 0 || n > most;
  it.length = it.bad ? 0 : n;
  it.tiles = tiles_of<kTile>(p, n, most);
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
template <int kTile, typename L>
__device__ __forceinline__ bool end_run(const L &p, const Deal &d, uint32_t i, Item &it) {
  const uint32_t end = (i + 1) * d.share;
  if (it.at + it.tiles <= end || end >= d.total) return true;
  if (end <= it.at) return false;
  const int cut = cut_of(p, end - it.at, it.tiles);
  if (cut == 1) it.last = end - it.at;
  return cut != 0;
}

// Workgroup i's first item; false if it has none. Lane l looks at rows l, l + 64, ...
template <int kTile, typename L>
__device__ __forceinline__ bool first_item(const L &p, uint32_t i, uint32_t groups, Deal &d, Item &it) {
  const int lane = lane_id();
  const int64_t most = static_cast<int64_t>(p.c.table_width) << p.page_shift;
  uint32_t total = 0, longest = 0;
  int32_t n = 0;  // of the row looked at last
  for (uint32_t r = lane; r < p.c.rows; r += kWave) {
    n = p.c.lengths[r];
    const uint32_t tiles = tiles_of<kTile>(p, n, most) + kEdge;
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
      upto = lanes_upto(base + lane < p.c.rows ? tiles_of<kTile>(p, n, most) + kEdge : 0u);
    }
    past = __ballot(before + upto * p.parts > begin);
    if (past) break;
    before += __builtin_amdgcn_readlane(upto, kWave - 1) * p.parts;
    base += kWave;
  }
  const int at = __ffsll(static_cast<unsigned long long>(past)) - 1;
  const int32_t length = __builtin_amdgcn_readlane(n, at);
  const uint32_t tiles = tiles_of<kTile>(p, length, most), each = tiles + kEdge, row = base + at;
  before += (__builtin_amdgcn_readlane(upto, at) - each) * p.parts;
  const uint32_t part = (begin - before) / each, in = begin - before - part * each;
  const int cut = in > kEdge ? cut_of(p, in - kEdge, tiles) : 0;
  if (cut < 2) {
    set_item<kTile>(p, d, it, row, part, before + part * each, length, most);
    if (cut == 1) it.first = in - kEdge;
  } else if (part + 1 < p.parts) {  // from the next item on
    set_item<kTile>(p, d, it, row, part + 1, before + (part + 1) * each, length, most);
  } else {
    if (row + 1 >= p.c.rows) return false;
    set_item<kTile>(p, d, it, row + 1, 0, before + (part + 1) * each, load_uniform(p.c.lengths + row + 1), most);
  }
  return end_run<kTile>(p, d, i, it);
}

// The item behind `it` in workgroup i's run; false at its end.
template <int kTile, typename L>
__device__ __forceinline__ bool next_item(const L &p, const Deal &d, uint32_t i, const Item &it, Item &next) {
  const int64_t most = static_cast<int64_t>(p.c.table_width) << p.page_shift;
  const uint32_t at = it.at + it.tiles;
  if (it.last < it.tiles || at >= d.total || at >= (i + 1) * d.share) return false;
  if (it.part + 1 < p.parts) {
    set_item<kTile>(p, d, next, it.row, it.part + 1, at, it.bad ? -1 : it.length, most);
  } else {
    set_item<kTile>(p, d, next, it.row + 1, 0, at, load_uniform(p.c.lengths + it.row + 1), most);
  }
  return end_run<kTile>(p, d, i, next);
}

}  // namespace dev

inline uint32_t log2_of(uint32_t v) { return static_cast<uint32_t>(__builtin_ctz(v)); }

template <typename... A>
hipError_t launch(void (*kernel)(A...), dim3 grid, dim3 block, hipStream_t s, A... args) {
  void *packed[] = {&args...};
  return hipLaunchKernel(reinterpret_cast<const void *>(kernel), grid, block, packed, 0, s);
}

inline size_t round256(size_t n) { return (n + 255) / 256 * 256; }

}  // namespace qd
