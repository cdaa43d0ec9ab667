// mq_cache.hip — writing keys and values into the paged cache, quantized on the
// way where its type is a block type, and reading them back.
//
// The blocks follow ggml's quantize_row_q8_0_ref / quantize_row_q4_0_ref along the
// head (oracle/ggml_oracle.c), every step one f32 rounding, so that they equal
// those of mq_quantize; what differs is where the bytes go (mq_cache.h).
//
// Both passes are bound by HBM: a value is read and written once.  A workgroup takes
// 32 consecutive rows of one head, K or V, a wave one block of 32 of their values,
// each lane what it would hold of them as an operand of the attention: eight values
// of a key for each of two keys, two values of eight tokens.  Rows whose slots fill
// one tile in order, as a prompt's do, are then stored and read in whole pieces; the
// others value by value, through the same registers.
#include "../../include/moldq.h"
#include "mq_cache.h"

#pragma clang fp contract(off)

namespace mq {
int set_error(int code, const char *msg);
}

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

// Where a workgroup's rows lie: lane i (and i + 32) of each wave knows row i's tile
// and token; `tile` is the one tile that all of them fill in order, if they do.
template <int T, int D>
struct Rows {
  int64_t at;  // the row's tile, in bytes from the cache's start; -1 outside the cache
  int token;
  uint8_t *tile, *data;

  __device__ Rows(const CacheView &c, int head, const int64_t *slots, int64_t count) : at(-1), token(0), tile(nullptr), data(c.data) {
    const int i = threadIdx.x & 31;
    const int64_t row = (int64_t)blockIdx.x * kRows + i, slot = row < count ? slots[row] : -1;
    if (slot >= 0 && slot < c.slots) {
      const int64_t page = c.slots >> 32 ? slot / c.page_tokens : (uint32_t)slot / (uint32_t)c.page_tokens;
      const int in = (int)(slot - page * c.page_tokens);
      at = ((page * c.kv_heads + head) * (c.page_tokens / kTileTokens) + in / kTileTokens) * CacheTile<T, D>::kBytes;
      token = in % kTileTokens;
    }
    const int64_t first = __shfl(at, 0);
    if (__all(at == first && token == i) && first >= 0) tile = data + first;
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

// The largest of a block's values: kOver 16 of the lanes 16 g .. + 15, or 4 of the
// lanes r, r + 16, r + 32, r + 48.
template <int kOver>
__device__ __forceinline__ uint32_t block_max(uint32_t x) {
  if constexpr (kOver == 16) {
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x128, 0xf, 0xf, false));  // row_ror 8, 4, 2, 1
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x124, 0xf, 0xf, false));
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x122, 0xf, 0xf, false));
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x121, 0xf, 0xf, false));
  } else {
    const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = max(a[0], a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    x = max(b[0], b[1]);
  }
  return x;
}

// The scale of the block that kOver lanes hold, N values each (value i of it has
// place at(i) in the block), and this lane's whole numbers (Q4_0: 0..15).  A block
// that holds a value that is not finite gets an infinite or NaN scale and zeros, and
// so reads as NaN.
template <int T, int kOver, int N, typename Place>
__device__ __forceinline__ float quantize(const float *x, int *q, Place at) {
  uint32_t top = 0;  // |x|'s bits order as its value, a NaN's above all
#pragma unroll
  for (int i = 0; i < N; ++i) top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
  top = block_max<kOver>(top);
  if constexpr (T == Q8_0) {
    const float d = __uint_as_float(top) / 127.f, id = d != 0.f ? 1.f / d : 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float y = __builtin_roundf(x[i] * id);  // halves away from zero
      q[i] = y == y ? (int)__builtin_fmaxf(-127.f, __builtin_fminf(127.f, y)) : 0;
    }
    return d;
  } else {
    // the first value of the largest magnitude, for its sign: the one of the highest 2 (32 - place) + sign
    uint32_t first = 0;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if ((__float_as_uint(x[i]) & 0x7FFFFFFFu) == top) first = max(first, (uint32_t)(2 * (32 - at(i))) + (__float_as_uint(x[i]) >> 31));
    first = top ? block_max<kOver>(first) : 0;
    const float d = __uint_as_float(top | first << 31) / -8.f, id = d != 0.f ? 1.f / d : 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float y = x[i] * id + 8.5f;
      q[i] = y == y ? (int)__builtin_fmaxf(0.f, __builtin_fminf(15.f, y)) : 8;
    }
    return d;
  }
}

__device__ __forceinline__ uint32_t bytes4(const int *q) {
  return (uint32_t)(q[0] & 0xFF) | (uint32_t)(q[1] & 0xFF) << 8 | (uint32_t)(q[2] & 0xFF) << 16 | (uint32_t)q[3] << 24;
}

// Which of its eight values of a key block lane group g holds in place i.
template <int T>
__device__ __forceinline__ int key_place(int g, int i) {
  return T == Q4_0 ? (i < 4 ? 4 * g + i : 12 + 4 * g + i) : 8 * g + i;
}

// rows of K (blockIdx.z 0) or V into the slots' places
template <int T, int D, typename X>
__global__ __launch_bounds__(2 * D) void append_kernel(CacheView c, const X *k, const X *v, int64_t rows, int64_t sk,
                                                       int64_t hk, int64_t sv, int64_t hv, const int64_t *slots) {
  using L = CacheTile<T, D>;
  const int head = blockIdx.y, b = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
  const int64_t row0 = (int64_t)blockIdx.x * kRows, last = rows - 1;
  const Rows<T, D> to(c, head, slots, rows);
  if (blockIdx.z == 0) {
    float x[2][8];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const X *p = k + head * hk + min(row0 + 16 * u + r, last) * sk + 32 * b;
      if constexpr (T == Q4_0) {
        load_row<4>(p + 4 * g, x[u]);
        load_row<4>(p + 16 + 4 * g, x[u] + 4);
      } else {
        load_row<8>(p + 8 * g, x[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      int t = 0, q[8];
      uint8_t *tile = to.of(16 * u + r, t);
      if constexpr (T == BF16) {
        if (tile) store_row<8>(reinterpret_cast<__bf16 *>(tile + L::key(t, b, g, 0)), x[u]);
      } else {
        const _Float16 d = (_Float16)quantize<T, 4, 8>(x[u], q, [&](int i) { return key_place<T>(g, i); });
        if (tile) {
          if constexpr (T == Q8_0)
            *reinterpret_cast<uint2 *>(tile + L::key(t, b, g, 0)) = make_uint2(bytes4(q), bytes4(q + 4));
          else
            *reinterpret_cast<uint32_t *>(tile + L::key(t, b, g, 0)) = bytes4(q) | bytes4(q + 4) << 4;
          if (g == 0) *reinterpret_cast<_Float16 *>(tile + L::key_scale(t, b)) = d;
        }
      }
    }
    return;
  }
  float x[8][2];
  auto row_of = [&](int j) { return 16 * (j >> 2) + 4 * g + (j & 3); };
#pragma unroll
  for (int j = 0; j < 8; ++j) load_row<2>(v + head * hv + min(row0 + row_of(j), last) * sv + 32 * b + 2 * r, x[j]);
  int q[2][8];
  _Float16 d[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    int two[2] = {0, 0};
    if constexpr (L::kQuant) d[j] = (_Float16)quantize<T, 16, 2>(x[j], two, [&](int i) { return 2 * r + i; });
    q[0][j] = two[0];
    q[1][j] = two[1];
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
      if (r == 0) {
        uint4 s;
        __builtin_memcpy(&s, d, 16);
        *reinterpret_cast<uint4 *>(to.tile + L::value_scale(4 * g, b)) = s;
      }
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    int t = 0;
    uint8_t *tile = to.of(row_of(j), t);
    if (!tile) continue;
#pragma unroll
    for (int i = 0; i < (T == Q4_0 ? 1 : 2); ++i) {
      uint8_t *p = tile + L::value(t, 32 * b + 2 * r + i);
      if constexpr (T == BF16) *reinterpret_cast<__bf16 *>(p) = (__bf16)x[j][i];
      else *p = (uint8_t)(T == Q8_0 ? q[i][j] : q[0][j] | q[1][j] << 4);
    }
    if (L::kQuant && r == 0) *reinterpret_cast<_Float16 *>(tile + L::value_scale(t, b)) = d[j];
  }
}

// the slots' keys (blockIdx.z 0) or values as rows [count, kv_heads, D]; zeros for a slot outside the cache
template <int T, int D, typename X>
__global__ __launch_bounds__(2 * D) void read_kernel(CacheView c, const int64_t *slots, int64_t count, X *k, X *v) {
  using L = CacheTile<T, D>;
  const int head = blockIdx.y, b = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
  const int64_t row0 = (int64_t)blockIdx.x * kRows;
  const Rows<T, D> from(c, head, slots, count);
  auto out = [&](X *p, int row) { return p + ((row0 + row) * c.kv_heads + head) * D + 32 * b; };
  if (blockIdx.z == 0) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int row = 16 * u + r;
      float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      int t = 0;
      const uint8_t *tile = from.of(row, t);
      if (tile) {
        const uint8_t *p = tile + L::key(t, b, g, 0);
        if constexpr (T == BF16) {
          load_row<8>(reinterpret_cast<const __bf16 *>(p), x);
        } else {
          const float d = (float)*reinterpret_cast<const _Float16 *>(tile + L::key_scale(t, b));
          if constexpr (T == Q8_0) {
            const uint2 w = *reinterpret_cast<const uint2 *>(p);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = (float)(int8_t)((i < 4 ? w.x : w.y) >> (8 * (i & 3))) * d;
          } else {
            const uint32_t w = *reinterpret_cast<const uint32_t *>(p);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = (float)((int)(w >> (8 * (i & 3) + 4 * (i >> 2)) & 15) - 8) * d;
          }
        }
      }
      if (row0 + row < count) {
        if constexpr (T == Q4_0) {
          store_row<4>(out(k, row) + 4 * g, x);
          store_row<4>(out(k, row) + 16 + 4 * g, x + 4);
        } else {
          store_row<8>(out(k, row) + 8 * g, x);
        }
      }
    }
    return;
  }
  float x[8][2];
  if (from.tile) {
    const uint8_t *const plane = from.tile + L::kPlane + lane * 16;
    if constexpr (T == BF16) {
      float y[2][8];
#pragma unroll
      for (int i = 0; i < 2; ++i) load_row<8>(reinterpret_cast<const __bf16 *>(plane + (2 * b + i) * 1024), y[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[j][0] = y[0][j];
        x[j][1] = y[1][j];
      }
    } else {
      const uint4 s = *reinterpret_cast<const uint4 *>(from.tile + L::value_scale(4 * g, b));
      _Float16 d[8];
      __builtin_memcpy(d, &s, 16);
      uint4 w{};
      if constexpr (T == Q8_0) {
        w = *reinterpret_cast<const uint4 *>(plane + b * 1024);
      } else {
        const uint2 n = *reinterpret_cast<const uint2 *>(plane + (b >> 1) * 1024 + (b & 1) * 8);
        w.x = n.x;
        w.y = n.y;
      }
      const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          x[j][i] = (T == Q8_0 ? (float)(int8_t)(u[2 * i + (j >> 2)] >> (8 * (j & 3)))
                               : (float)((int)(u[j >> 2] >> (8 * (j & 3) + 4 * i) & 15) - 8)) * (float)d[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      int t = 0;
      const uint8_t *tile = from.of(16 * (j >> 2) + 4 * g + (j & 3), t);
      x[j][0] = x[j][1] = 0.f;
      if (!tile) continue;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint8_t *p = tile + L::value(t, 32 * b + 2 * r + (T == Q4_0 ? 0 : i));
        if constexpr (T == BF16) {
          x[j][i] = (float)*reinterpret_cast<const __bf16 *>(p);
        } else {
          const float d = (float)*reinterpret_cast<const _Float16 *>(tile + L::value_scale(t, b));
          x[j][i] = (float)(T == Q8_0 ? (int)(int8_t)*p : (*p >> (4 * i) & 15) - 8) * d;
        }
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int row = 16 * (j >> 2) + 4 * g + (j & 3);
    if (row0 + row < count) store_row<2>(out(v, row) + 2 * r, x[j]);
  }
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
int invalid(const char *msg) { return set_error(MQ_E_INVALID, msg); }

CacheView view(const mq_kv_cache *c) {
  return {static_cast<uint8_t *>(c->data), c->pages * c->page_tokens, c->page_tokens, c->kv_heads};
}

}  // namespace
}  // namespace mq

extern "C" size_t mq_kv_cache_size(const mq_kv_cache *c) {
  using namespace mq;
  if (cache_fault(c)) return 0;
  return (size_t)c->pages * c->kv_heads * (c->page_tokens / kTileTokens) * cache_tile_bytes(c->dtype, c->head_dim);
}

extern "C" int mq_kv_cache_append(const mq_kv_cache *c, const void *k, int64_t k_token_stride, int64_t k_head_stride,
                                  const void *v, int64_t v_token_stride, int64_t v_head_stride, int x_dtype,
                                  int64_t tokens, const int64_t *slots, void *stream) {
  using namespace mq;
  if (const char *fault = cache_fault(c)) return invalid(fault);
  if (x_dtype != MQ_F32 && x_dtype != MQ_BF16) return invalid("mq_kv_cache_append: k and v are F32 or BF16");
  if (tokens < 0 || tokens >= (int64_t(1) << 31)) return invalid("mq_kv_cache_append: tokens outside 0 .. 2^31");
  if (tokens == 0 || c->pages == 0) return MQ_OK;
  if (!c->data || !k || !v || !slots) return invalid("mq_kv_cache_append: NULL pointer");
  const int64_t unit = x_dtype == MQ_F32 ? 4 : 8;
  for (int64_t s : {k_token_stride, k_head_stride, v_token_stride, v_head_stride})
    if (s < 0 || s % unit) return invalid("mq_kv_cache_append: strides must be multiples of 16 bytes, none negative");
  if (!aligned16(c->data) || !aligned16(k) || !aligned16(v) || (reinterpret_cast<uintptr_t>(slots) & 7))
    return invalid("mq_kv_cache_append: buffers must be 16-byte aligned");
  const dim3 grid((unsigned)((tokens + kRows - 1) / kRows), (unsigned)c->kv_heads, 2);
  with_cache_type(c, [&]<int T, int D>() {
    if (x_dtype == MQ_F32)
      hipLaunchKernelGGL((append_kernel<T, D, float>), grid, dim3(2 * D), 0, static_cast<hipStream_t>(stream), view(c),
                         static_cast<const float *>(k), static_cast<const float *>(v), tokens, k_token_stride,
                         k_head_stride, v_token_stride, v_head_stride, slots);
    else
      hipLaunchKernelGGL((append_kernel<T, D, __bf16>), grid, dim3(2 * D), 0, static_cast<hipStream_t>(stream), view(c),
                         static_cast<const __bf16 *>(k), static_cast<const __bf16 *>(v), tokens, k_token_stride,
                         k_head_stride, v_token_stride, v_head_stride, slots);
  });
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MQ_OK : set_error(MQ_E_HIP, hipGetErrorString(e));
}

extern "C" int mq_kv_cache_read(const mq_kv_cache *c, const int64_t *slots, int64_t count, void *k, void *v,
                                int out_dtype, void *stream) {
  using namespace mq;
  if (const char *fault = cache_fault(c)) return invalid(fault);
  if (out_dtype != MQ_F32 && out_dtype != MQ_BF16) return invalid("mq_kv_cache_read: k and v are F32 or BF16");
  if (count < 0 || count >= (int64_t(1) << 31)) return invalid("mq_kv_cache_read: count outside 0 .. 2^31");
  if (count == 0) return MQ_OK;
  if ((c->pages && !c->data) || !slots || !k || !v) return invalid("mq_kv_cache_read: NULL pointer");
  if (!aligned16(c->data) || !aligned16(k) || !aligned16(v) || (reinterpret_cast<uintptr_t>(slots) & 7))
    return invalid("mq_kv_cache_read: buffers must be 16-byte aligned");
  const dim3 grid((unsigned)((count + kRows - 1) / kRows), (unsigned)c->kv_heads, 2);
  with_cache_type(c, [&]<int T, int D>() {
    if (out_dtype == MQ_F32)
      hipLaunchKernelGGL((read_kernel<T, D, float>), grid, dim3(2 * D), 0, static_cast<hipStream_t>(stream), view(c),
                         slots, count, static_cast<float *>(k), static_cast<float *>(v));
    else
      hipLaunchKernelGGL((read_kernel<T, D, __bf16>), grid, dim3(2 * D), 0, static_cast<hipStream_t>(stream), view(c),
                         slots, count, static_cast<__bf16 *>(k), static_cast<__bf16 *>(v));
  });
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MQ_OK : set_error(MQ_E_HIP, hipGetErrorString(e));
}
