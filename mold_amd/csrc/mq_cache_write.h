// mq_cache_write.h — rows of keys and values into the paged cache's tiles, quantized on the way
// where its type is a block type: what the kernels that write it share.
//
// The blocks are those of mq_quantize (mq_quant.hip), taken along the head, every step
// one f32 rounding; what differs is where the bytes go (mq_cache.h).
#pragma once

#include "mq_cache.h"

#pragma clang fp contract(off)

namespace mq {
namespace {

constexpr int kRows = kTileTokens;  // rows of a workgroup

template <int N>
__device__ __forceinline__ void load_row(const __bf16 *p, float *x) {
  typedef uint32_t words __attribute__((ext_vector_type(N / 2)));
  uint32_t w[N / 2];
  if constexpr (N == 2) {
    w[0] = *reinterpret_cast<const uint32_t *>(p);
  } else {
    const words u = *reinterpret_cast<const words *>(p);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) w[i] = u[i];
  }
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
template <int N>
__device__ __forceinline__ void load_row(const float *p, float *x) {
  typedef float vec __attribute__((ext_vector_type(N < 4 ? N : 4)));
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    const vec u = *reinterpret_cast<const vec *>(p + i);
#pragma unroll
    for (int k = 0; k < (N < 4 ? N : 4); ++k) x[i + k] = u[k];
  }
}
template <int N>
__device__ __forceinline__ void store_row(__bf16 *p, const float *x) {
  if constexpr (N == 2) {
    *reinterpret_cast<uint32_t *>(p) = pack2(x[0], x[1]);
  } else {
    typedef uint32_t words __attribute__((ext_vector_type(N / 2)));
    words u;
#pragma unroll
    for (int i = 0; i < N / 2; ++i) u[i] = pack2(x[2 * i], x[2 * i + 1]);
    *reinterpret_cast<words *>(p) = u;
  }
}
template <int N>
__device__ __forceinline__ void store_row(float *p, const float *x) {
  typedef float vec __attribute__((ext_vector_type(N < 4 ? N : 4)));
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    vec u;
#pragma unroll
    for (int k = 0; k < (N < 4 ? N : 4); ++k) u[k] = x[i + k];
    *reinterpret_cast<vec *>(p + i) = u;
  }
}

// Element `col` of a workgroup's row `in` (below 32), rows `step` (below 2^24) elements
// apart: a scalar base and a 32-bit offset.  Whole groups pass the lanes' part of the
// row and, in `more`, the part that all share, which then costs no vector operation.
template <typename X>
__device__ __forceinline__ X *at_row(X *base, int in, int more, int step, int col) {
  const uint32_t off = (__umul24(in, step) + col) * (uint32_t)sizeof(X);
  return reinterpret_cast<X *>(reinterpret_cast<uintptr_t>(base + (int64_t)more * step) + off);
}

// Where a workgroup's rows lie: lane i (and i + 32) of each wave knows row i's tile
// and token; `tile` is the one tile that all of them fill in order, if they do.
template <int T, int D>
struct Rows {
  int64_t at;  // the row's tile, in bytes from the cache's start; -1 outside the cache
  int token;
  uint8_t *tile, *data;

  __device__ Rows(const CacheView &c, int head, int64_t row0, const int64_t *slots, int64_t count) : at(-1), token(0), tile(nullptr), data(c.data) {
    const int i = threadIdx.x & 31;
    const int64_t row = row0 + i, slot = row < count ? slots[row] : -1;
    const int64_t first = ((int64_t)__builtin_amdgcn_readfirstlane((int)(slot >> 32)) << 32) |
                          (uint32_t)__builtin_amdgcn_readfirstlane((int)slot);
    if (__all((uint64_t)slot - (uint64_t)first == (uint64_t)i) && first >= 0 && first <= c.slots - kRows && first % kTileTokens == 0) {
      int t;
      tile = data + place(c, head, first, t);
    } else if (slot >= 0 && slot < c.slots) {
      at = place(c, head, slot, token);
    }
  }
  // A slot's tile and its token in it.
  __device__ static int64_t place(const CacheView &c, int head, int64_t slot, int &t) {
    const int64_t page = c.slots >> 32 ? slot / c.page_tokens : (uint32_t)slot / (uint32_t)c.page_tokens;
    const int in = (int)(slot - page * c.page_tokens);
    t = in % kTileTokens;
    return ((page * c.kv_heads + head) * (c.page_tokens / kTileTokens) + in / kTileTokens) * CacheTile<T, D>::kBytes;
  }
  // The tile and token of row i; NULL for a slot outside the cache.  All lanes join.
  __device__ uint8_t *of(int i, int &t) const {
    if (tile) {
      t = i;
      return tile;
    }
    const int64_t place = __shfl(at, i);
    t = __shfl(token, i);
    return place < 0 ? nullptr : data + place;
  }
};

template <int kCtrl>
__device__ __forceinline__ uint32_t dpp(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, kCtrl, 0xf, 0xf, false);
}

// The largest over the lanes r, r + 16, r + 32, r + 48.
__device__ __forceinline__ uint32_t column_max(uint32_t x) {
  const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = max(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return max(b[0], b[1]);
}
// The largest of each x[j] over the 16 lanes of a row, x[j]'s in lanes 2 j and
// 2 j + 1: at each step half of them go to the mirrored lane for the other half.
__device__ __forceinline__ uint32_t row_max8(const uint32_t *x) {
  const int r = threadIdx.x & 15;
  uint32_t a[4], b[2];
#pragma unroll
  for (int j = 0; j < 4; ++j) a[j] = max(r & 8 ? x[j + 4] : x[j], dpp<0x140>(r & 8 ? x[j] : x[j + 4]));  // row_mirror
#pragma unroll
  for (int j = 0; j < 2; ++j) b[j] = max(r & 4 ? a[j + 2] : a[j], dpp<0x141>(r & 4 ? a[j] : a[j + 2]));  // row_half_mirror
  const uint32_t c = max(r & 2 ? b[1] : b[0], dpp<0x4E>(r & 2 ? b[0] : b[1]));                           // quad_perm 2 3 0 1
  return max(c, dpp<0xB1>(c));                                                                            // quad_perm 1 0 3 2
}

// What a block's scale is made of: of Q8_0 the largest magnitude, whose bits order
// as its value (a NaN's above all); of Q4_0 also the sign of the first value that has
// it, the one with the highest rank: 2 (32 - its place in the block) + its sign.
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }
__device__ __forceinline__ uint32_t rank_of(float x, int place) { return 2 * (32 - place) + (__float_as_uint(x) >> 31); }

// Both in one for a value that came from bf16, whose magnitude is 15 bits.
__device__ __forceinline__ uint32_t key_of(float x, int place) {
  const uint32_t u = __float_as_uint(x);
  return ((u >> 9 & 0x3FFF80u) | (uint32_t)(2 * (32 - place))) + (u >> 31);
}
__device__ __forceinline__ uint32_t key_magnitude(uint32_t key) { return (key & 0x3FFF80u) << 9; }

// v if `yes`, else 0, without the branch that the compiler makes of it
__device__ __forceinline__ uint32_t only_if(bool yes, uint32_t v) {
  uint32_t mask = yes ? ~0u : 0u;
  asm("" : "+v"(mask));
  return v & mask;
}

struct Scale {
  float d, id;
};
// A block that holds a value that is not finite gets a scale that is not, and so
// reads as no number.
template <int T>
__device__ __forceinline__ Scale scale_of(uint32_t top, uint32_t rank) {
  const float d = T == Q8_0 ? __uint_as_float(top) / 127.f : __uint_as_float(top | (top ? rank << 31 : 0)) / -8.f;
  return {d, d != 0.f ? 1.f / d : 0.f};
}

// Truncated to a whole number; defined for every f32 (NaN gives 0, others saturate).
__device__ __forceinline__ int to_int(float y) {
  int q;
  asm("v_cvt_i32_f32 %0, %1" : "=v"(q) : "v"(y));
  return q;
}
template <int T>
__device__ __forceinline__ int quantize(float x, float id) {
  const float y = x * id;
  // halves away from zero: the largest f32 below 0.5 added, which takes 0.5 to 1 and nothing below it there
  if constexpr (T == Q8_0) return to_int(y + __builtin_copysignf(0.49999997f, y));
  return max(0, min(15, to_int(y + 8.5f)));
}

// the low bytes of four whole numbers
__device__ __forceinline__ uint32_t bytes4(const int *q) {
  return __builtin_amdgcn_perm((uint32_t)q[1], (uint32_t)q[0], 0x0C0C0400u) | __builtin_amdgcn_perm((uint32_t)q[3], (uint32_t)q[2], 0x04000C0Cu);
}

// Which of its eight values of a key block lane group g holds in place i.
template <int T>
__device__ __forceinline__ int key_place(int g, int i) {
  return T == Q4_0 ? (i < 4 ? 4 * g + i : 12 + 4 * g + i) : 8 * g + i;
}

// Block b of the keys of a workgroup's rows, by one wave: x[u][i] is value key_place(g, i)
// of the block of row 16 u + r (g = lane / 16, r = lane % 16).  kNarrow: values that came
// from bf16.
template <int T, int D, bool kNarrow>
__device__ __forceinline__ void put_keys(const Rows<T, D> &to, int b, int lane, const float (&x)[2][8]) {
  using L = CacheTile<T, D>;
  const int g = lane >> 4, r = lane & 15;
  Scale of[2]{};
  if constexpr (L::kQuant) {
    uint32_t top[2], rank[2] = {0, 0};
    constexpr bool kOne = T == Q4_0 && kNarrow;  // magnitude and rank in one key
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      top[u] = 0;
      if constexpr (kOne) {
#pragma unroll
        for (int i = 0; i < 8; ++i) top[u] = max(top[u], key_of(x[u][i], key_place<T>(g, i)));
        rank[u] = column_max(top[u]);
        top[u] = key_magnitude(rank[u]);
        continue;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) top[u] = max(top[u], magnitude(x[u][i]));
      top[u] = column_max(top[u]);
      if constexpr (T == Q4_0) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          rank[u] = max(rank[u], only_if(magnitude(x[u][i]) == top[u], rank_of(x[u][i], key_place<T>(g, i))));
        rank[u] = column_max(rank[u]);
      }
    }
    // even lane groups divide for the first row, odd ones for the second
    const Scale mine = scale_of<T>(g & 1 ? top[1] : top[0], g & 1 ? rank[1] : rank[0]);
    const uint32_t d = __float_as_uint(mine.d), id = __float_as_uint(mine.id);
    const auto ds = __builtin_amdgcn_permlane16_swap(d, d, false, false), ids = __builtin_amdgcn_permlane16_swap(id, id, false, false);
#pragma unroll
    for (int u = 0; u < 2; ++u) of[u] = {__uint_as_float(ds[u]), __uint_as_float(ids[u])};
  }
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    int t = 0, q[8];
    uint8_t *tile = to.of(16 * u + r, t);
    if constexpr (T == BF16) {
      if (tile) store_row<8>(reinterpret_cast<__bf16 *>(tile + L::key(t, b, g, 0)), x[u]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) q[i] = quantize<T>(x[u][i], of[u].id);
      if (tile) {
        if constexpr (T == Q8_0)
          *reinterpret_cast<uint2 *>(tile + L::key(t, b, g, 0)) = make_uint2(bytes4(q), bytes4(q + 4));
        else
          *reinterpret_cast<uint32_t *>(tile + L::key(t, b, g, 0)) = bytes4(q) | bytes4(q + 4) << 4;
        if (g == 0) *reinterpret_cast<_Float16 *>(tile + L::key_scale(t, b)) = (_Float16)of[u].d;
      }
    }
  }
}

// Block b of the values of a workgroup's rows, by one wave: x[j][i] is value 2 r + i of the
// block of row value_row(g, j).
__device__ __forceinline__ int value_row(int g, int j) { return 16 * (j >> 2) + 4 * g + (j & 3); }
template <int T, int D, bool kNarrow>
__device__ __forceinline__ void put_values(const Rows<T, D> &to, int b, int lane, const float (&x)[8][2]) {
  using L = CacheTile<T, D>;
  const int g = lane >> 4, r = lane & 15;
  int q[2][8];
  if constexpr (L::kQuant) {
    uint32_t top[8], rank[8];
    constexpr bool kOne = T == Q4_0 && kNarrow;  // magnitude and rank in one key
#pragma unroll
    for (int j = 0; j < 8; ++j)
      top[j] = kOne ? max(key_of(x[j][0], 2 * r), key_of(x[j][1], 2 * r + 1)) : max(magnitude(x[j][0]), magnitude(x[j][1]));
    uint32_t most = row_max8(top), first = most;  // of row r / 2 of the eight
    if constexpr (kOne) most = key_magnitude(most);
    auto each = [&](uint32_t v, auto f) {      // f(j, row j's v)
      f(0, dpp<0x150>(v)); f(1, dpp<0x152>(v)); f(2, dpp<0x154>(v)); f(3, dpp<0x156>(v));  // row_newbcast 0, 2, ..
      f(4, dpp<0x158>(v)); f(5, dpp<0x15A>(v)); f(6, dpp<0x15C>(v)); f(7, dpp<0x15E>(v));
    };
    if constexpr (T == Q4_0 && !kOne) {
      each(most, [&](int j, uint32_t m) {
        rank[j] = max(only_if(magnitude(x[j][0]) == m, rank_of(x[j][0], 2 * r)),
                      only_if(magnitude(x[j][1]) == m, rank_of(x[j][1], 2 * r + 1)));
      });
      first = row_max8(rank);
    }
    const Scale mine = scale_of<T>(most, first);
    each(__float_as_uint(mine.id), [&](int j, uint32_t id) {
#pragma unroll
      for (int i = 0; i < 2; ++i) q[i][j] = quantize<T>(x[j][i], __uint_as_float(id));
    });
    int t = 0;
    uint8_t *tile = to.of(value_row(g, r >> 1), t);
    if (tile && !(r & 1)) *reinterpret_cast<_Float16 *>(tile + L::value_scale(t, b)) = (_Float16)mine.d;
  }
  if (to.tile) {
    uint8_t *const plane = to.tile + L::kPlane + lane * 16;
    if constexpr (T == BF16) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        *reinterpret_cast<uint4 *>(plane + (2 * b + i) * 1024) =
            make_uint4(pack2(x[0][i], x[1][i]), pack2(x[2][i], x[3][i]), pack2(x[4][i], x[5][i]), pack2(x[6][i], x[7][i]));
    } else {
      if constexpr (T == Q8_0)
        *reinterpret_cast<uint4 *>(plane + b * 1024) = make_uint4(bytes4(q[0]), bytes4(q[0] + 4), bytes4(q[1]), bytes4(q[1] + 4));
      else
        *reinterpret_cast<uint2 *>(plane + (b >> 1) * 1024 + (b & 1) * 8) =
            make_uint2(bytes4(q[0]) | bytes4(q[1]) << 4, bytes4(q[0] + 4) | bytes4(q[1] + 4) << 4);
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    int t = 0;
    uint8_t *tile = to.of(value_row(g, j), t);
    if (!tile) continue;
#pragma unroll
    for (int i = 0; i < (T == Q4_0 ? 1 : 2); ++i) {
      uint8_t *p = tile + L::value(t, 32 * b + 2 * r + i);
      if constexpr (T == BF16) *reinterpret_cast<__bf16 *>(p) = (__bf16)x[j][i];
      else *p = (uint8_t)(T == Q8_0 ? q[i][j] : q[0][j] | q[1][j] << 4);
    }
  }
}

// The same of rows base .. base + last * step (of all kRows of them, or fewer at the end).
template <int T, int D, typename X>
__device__ __forceinline__ void append_values(const Rows<T, D> &to, int b, int lane, const X *base, int step, int last) {
  const int g = lane >> 4, r = lane & 15;
  float x[8][2];
  if (last == kRows - 1) {
#pragma unroll
    for (int j = 0; j < 8; ++j) load_row<2>(at_row(base, 4 * g, value_row(g, j) - 4 * g, step, 32 * b + 2 * r), x[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) load_row<2>(at_row(base, min(value_row(g, j), last), 0, step, 32 * b + 2 * r), x[j]);
  }
  put_values<T, D, sizeof(X) == 2>(to, b, lane, x);
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

CacheView view(const mq_kv_cache *c) {
  return {static_cast<uint8_t *>(c->data), c->pages * c->page_tokens, c->page_tokens, c->kv_heads};
}

}  // namespace
}  // namespace mq
