// mq_cache.hip — writing keys and values into the paged cache, quantized on the
// way where its type is a block type, and reading them back.
//
// The blocks follow ggml's quantize_row_q8_0_ref / quantize_row_q4_0_ref along the
// head (oracle/ggml_oracle.c), every step one f32 rounding, so that they equal
// those of mq_quantize; what differs is where the bytes go (mq_cache.h).
//
// Both passes are bound by HBM: a value is read and written once.  Four lanes take
// a block of 32, eight values each; a workgroup takes 32 consecutive rows of one
// head, K or V, so that where these fill one tile every line of it is completed by
// one XCD's L2, although the values' bytes are stored one by one.
#include "../../include/moldq.h"
#include "mq_cache.h"

#pragma clang fp contract(off)

namespace mq {
int set_error(int code, const char *msg);
}

namespace mq {
namespace {

constexpr int kRows = 32;  // rows of a workgroup

__device__ __forceinline__ void load8(const __bf16 *p, float *x) {
  const uint4 u = *reinterpret_cast<const uint4 *>(p);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ void load8(const float *p, float *x) {
  const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
  x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}

// The tile of a slot and its token in it; false for a slot outside the cache.
template <int T, int D>
__device__ __forceinline__ bool find(const CacheView &c, int64_t slot, int head, uint8_t *&tile, int &t) {
  if (slot < 0 || slot >= c.slots) return false;
  const int64_t page = slot / c.page_tokens;
  const int at = (int)(slot - page * c.page_tokens);
  tile = c.data + ((page * c.kv_heads + head) * (c.page_tokens / kTileTokens) + at / kTileTokens) * CacheTile<T, D>::kBytes;
  t = at % kTileTokens;
  return true;
}

// The scale of the block that four lanes hold (eight values each) and this
// lane's whole numbers (Q4_0: 0..15).  A block that holds a value that is not
// finite gets an infinite or NaN scale and zeros, and so reads as NaN.
template <int T>
__device__ __forceinline__ float quantize8(const float *x, int *q) {
  uint32_t top = 0;  // |x|'s bits order as its value, a NaN's above all
  float first = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t u = __float_as_uint(x[i]) & 0x7FFFFFFFu;
    if (u > top) {
      top = u;
      first = x[i];
    }
  }
  if (T == Q8_0) {
    top = max(top, (uint32_t)__shfl_xor((int)top, 1));
    top = max(top, (uint32_t)__shfl_xor((int)top, 2));
    const float d = __uint_as_float(top) / 127.f, id = d != 0.f ? 1.f / d : 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float y = __builtin_roundf(x[i] * id);  // halves away from zero
      q[i] = y == y ? (int)__builtin_fmaxf(-127.f, __builtin_fminf(127.f, y)) : 0;
    }
    return d;
  }
  // the first value of the largest magnitude, its sign with it
#pragma unroll
  for (int off = 1; off <= 2; off <<= 1) {
    const uint32_t u = (uint32_t)__shfl_xor((int)top, off);
    const float f = __shfl_xor(first, off);
    if (u > top || (u == top && (threadIdx.x & off))) {
      top = u;
      first = f;
    }
  }
  const float d = first / -8.f, id = d != 0.f ? 1.f / d : 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float y = x[i] * id + 8.5f;
    q[i] = y == y ? (int)__builtin_fmaxf(0.f, __builtin_fminf(15.f, y)) : 8;
  }
  return d;
}

// rows of K (blockIdx.z 0) or V into the slots' places
template <int T, int D, typename X>
__global__ __launch_bounds__(256) void append_kernel(CacheView c, const X *k, const X *v, int64_t rows, int64_t sk,
                                                     int64_t hk, int64_t sv, int64_t hv, const int64_t *slots) {
  using L = CacheTile<T, D>;
  constexpr int kLanes = D / 8, kPass = 256 / kLanes;  // lanes of a row, rows at a time
  const int head = blockIdx.y, sub = threadIdx.x & 3;
  const int b = (threadIdx.x % kLanes) >> 2;
  const bool values = blockIdx.z;
  const X *src = values ? v + head * hv : k + head * hk;
  const int64_t step = values ? sv : sk;
  const int64_t row0 = (int64_t)blockIdx.x * kRows + threadIdx.x / kLanes;
  float x[kRows / kPass][8];
  int64_t slot[kRows / kPass];
#pragma unroll
  for (int p = 0; p < kRows / kPass; ++p) {
    const int64_t row = row0 + p * kPass;
    slot[p] = row < rows ? slots[row] : -1;
    load8(src + (row < rows ? row : rows - 1) * step + 32 * b + 8 * sub, x[p]);
  }
#pragma unroll
  for (int p = 0; p < kRows / kPass; ++p) {
    uint8_t *tile = nullptr;
    int t = 0;
    const bool stored = find<T, D>(c, slot[p], head, tile, t);
    if constexpr (T == BF16) {
      uint32_t u[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) u[i] = pack2(x[p][2 * i], x[p][2 * i + 1]);
      if (!stored) continue;
      if (!values) {
        *reinterpret_cast<uint4 *>(tile + L::key(t, b, sub, 0)) = make_uint4(u[0], u[1], u[2], u[3]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          *reinterpret_cast<uint16_t *>(tile + L::value(t, 32 * b + 8 * sub + i)) = (uint16_t)(u[i >> 1] >> (16 * (i & 1)));
      }
    } else {
      int q[8];
      const _Float16 d = (_Float16)quantize8<T>(x[p], q);
      if constexpr (T == Q8_0) {
        if (!stored) continue;
        if (!values) {
          uint32_t w[2] = {0, 0};
#pragma unroll
          for (int i = 0; i < 8; ++i) w[i >> 2] |= (uint32_t)(q[i] & 0xFF) << (8 * (i & 3));
          *reinterpret_cast<uint2 *>(tile + L::key(t, b, sub, 0)) = make_uint2(w[0], w[1]);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) tile[L::value(t, 32 * b + 8 * sub + i)] = (uint8_t)q[i];
        }
      } else {
        // lanes 0 and 1 hold bytes 0..7 and 8..15's low halves, 2 and 3 the high
        // ones; each pair's lower lane then stores the first four, its upper the rest
        uint32_t mine[2] = {0, 0}, byte[2];
#pragma unroll
        for (int i = 0; i < 8; ++i) mine[i >> 2] |= (uint32_t)q[i] << (8 * (i & 3));
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t other = (uint32_t)__shfl_xor((int)mine[i], 2);
          byte[i] = sub < 2 ? mine[i] | other << 4 : other | mine[i] << 4;
        }
        if (!stored) continue;
        const int half = sub >> 1, g = 2 * (sub & 1) + half;
        const uint32_t w = half ? byte[1] : byte[0];
        if (!values) {
          *reinterpret_cast<uint32_t *>(tile + L::key(t, b, g, 0)) = w;
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) tile[L::value(t, 32 * b + 4 * g + i)] = (uint8_t)(w >> (8 * i));
        }
      }
      if (sub == 0) *reinterpret_cast<_Float16 *>(tile + (values ? L::value_scale(t, b) : L::key_scale(t, b))) = d;
    }
  }
}

__device__ __forceinline__ void store8(__bf16 *p, const float *x) {
  *reinterpret_cast<uint4 *>(p) = make_uint4(pack2(x[0], x[1]), pack2(x[2], x[3]), pack2(x[4], x[5]), pack2(x[6], x[7]));
}
__device__ __forceinline__ void store8(float *p, const float *x) {
  reinterpret_cast<float4 *>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
  reinterpret_cast<float4 *>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}

// the slots' keys (blockIdx.z 0) or values as rows [count, kv_heads, D]; zeros for a slot outside the cache
template <int T, int D, typename X>
__global__ __launch_bounds__(256) void read_kernel(CacheView c, const int64_t *slots, int64_t count, X *k, X *v) {
  using L = CacheTile<T, D>;
  constexpr int kLanes = D / 8, kPass = 256 / kLanes;
  const int head = blockIdx.y, sub = threadIdx.x & 3, b = (threadIdx.x % kLanes) >> 2;
  const bool values = blockIdx.z;
  X *dst = values ? v : k;
#pragma unroll
  for (int p = 0; p < kRows / kPass; ++p) {
    const int64_t row = (int64_t)blockIdx.x * kRows + p * kPass + threadIdx.x / kLanes;
    if (row >= count) return;
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    uint8_t *tile = nullptr;
    int t = 0;
    if (find<T, D>(c, slots[row], head, tile, t)) {
      if constexpr (T == BF16) {
        if (!values) load8(reinterpret_cast<const __bf16 *>(tile + L::key(t, b, sub, 0)), x);
        else
#pragma unroll
          for (int i = 0; i < 8; ++i)
            x[i] = __uint_as_float((uint32_t)*reinterpret_cast<const uint16_t *>(tile + L::value(t, 32 * b + 8 * sub + i)) << 16);
      } else {
        const float d = (float)*reinterpret_cast<const _Float16 *>(tile + (values ? L::value_scale(t, b) : L::key_scale(t, b)));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if constexpr (T == Q8_0) {
            x[i] = (float)(int8_t)tile[values ? L::value(t, 32 * b + 8 * sub + i) : L::key(t, b, sub, i)] * d;
          } else {
            const int j = (8 * sub + i) & 15;
            const uint8_t two = tile[values ? L::value(t, 32 * b + j) : L::key(t, b, j >> 2, j & 3)];
            x[i] = (float)((int)(sub < 2 ? two & 15 : two >> 4) - 8) * d;
          }
        }
      }
    }
    store8(dst + (row * c.kv_heads + head) * D + 32 * b + 8 * sub, x);
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
      hipLaunchKernelGGL((append_kernel<T, D, float>), grid, dim3(256), 0, static_cast<hipStream_t>(stream), view(c),
                         static_cast<const float *>(k), static_cast<const float *>(v), tokens, k_token_stride,
                         k_head_stride, v_token_stride, v_head_stride, slots);
    else
      hipLaunchKernelGGL((append_kernel<T, D, __bf16>), grid, dim3(256), 0, static_cast<hipStream_t>(stream), view(c),
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
      hipLaunchKernelGGL((read_kernel<T, D, float>), grid, dim3(256), 0, static_cast<hipStream_t>(stream), view(c),
                         slots, count, static_cast<float *>(k), static_cast<float *>(v));
    else
      hipLaunchKernelGGL((read_kernel<T, D, __bf16>), grid, dim3(256), 0, static_cast<hipStream_t>(stream), view(c),
                         slots, count, static_cast<__bf16 *>(k), static_cast<__bf16 *>(v));
  });
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MQ_OK : set_error(MQ_E_HIP, hipGetErrorString(e));
}
