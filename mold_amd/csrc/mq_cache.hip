// mq_cache.hip — writing keys and values into the paged cache, quantized on the
// way where its type is a block type, and reading them back.
//
// The blocks are those of mq_quantize (mq_quant.hip), taken along the head, every step
// one f32 rounding; what differs is where the bytes go (mq_cache.h).
//
// A value is read and written once: the bound is HBM, which BF16 rows reach (32768
// tokens of 8 heads of 128: written in 50 to 57 us, read in 46 to 49, 4.7 to 5.8 TB/s).
// Quantizing writes less but spends 330 vector instructions a wave, which is what Q4_0
// runs at (53 us of writing); there and back it takes 92.  A workgroup takes
// 32 consecutive rows of one head, K or V, a wave one block of 32 of their values,
// each lane what it would hold of them as an operand of the attention: eight values
// of a key for each of two keys, two values of eight tokens.  Rows whose slots fill
// one tile in order, as a prompt's do, are then stored and read in whole pieces; the
// others value by value, through the same registers.
#include "../../include/moldq.h"
#include "mq_cache_write.h"

#pragma clang fp contract(off)

namespace mq {
int set_error(int code, const char *msg);
}

namespace mq {
namespace {

// What a workgroup does.  Writing, the heads of one group of rows follow each other,
// keys and then values, so that workgroups that run together take in whole rows;
// reading, the groups of one head do, so that they take in whole pages.  32768 tokens
// of 8 heads, there and back: BF16 107 us, 117 if reading went by rows too; f32 rows and
// Q8_0 116 and 124; bf16 rows and Q4_0 93 and 92, Q8_0 95 and 86.
struct Part {
  int head;
  bool values;
  int64_t row0;

  __device__ Part(const CacheView &c, bool by_rows) {
    const uint32_t heads = (uint32_t)c.kv_heads, groups = gridDim.x / (2 * heads);
    const uint32_t i = blockIdx.x, in = by_rows ? i % (2 * heads) : i / groups, group = by_rows ? i / (2 * heads) : i % groups;
    values = in >= heads;
    head = (int)(values ? in - heads : in);
    row0 = (int64_t)group * kRows;
  }
};

// rows of K or V into the slots' places
template <int T, int D, typename X>
__global__ __launch_bounds__(2 * D) void append_kernel(CacheView c, const X *k, const X *v, int64_t rows, int64_t sk,
                                                       int64_t hk, int64_t sv, int64_t hv, const int64_t *slots) {
  const Part part(c, true);
  const int head = part.head, b = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
  const int64_t row0 = part.row0;
  const int last = (int)min(rows - row0, (int64_t)kRows) - 1;
  const Rows<T, D> to(c, head, row0, slots, rows);
  if (!part.values) {
    float x[2][8];
    const X *const base = k + row0 * sk + head * hk;
    auto load = [&](int u, int in, int more) {
      if constexpr (T == Q4_0) {
        load_row<4>(at_row(base, in, more, (int)sk, 32 * b + 4 * g), x[u]);
        load_row<4>(at_row(base, in, more, (int)sk, 32 * b + 16 + 4 * g), x[u] + 4);
      } else {
        load_row<8>(at_row(base, in, more, (int)sk, 32 * b + 8 * g), x[u]);
      }
    };
    if (last == kRows - 1) {
#pragma unroll
      for (int u = 0; u < 2; ++u) load(u, r, 16 * u);
    } else {
#pragma unroll
      for (int u = 0; u < 2; ++u) load(u, min(16 * u + r, last), 0);
    }
    put_keys<T, D, sizeof(X) == 2>(to, b, lane, x);
    return;
  }
  append_values<T, D>(to, b, lane, v + row0 * sv + head * hv, (int)sv, last);
}

// the slots' keys or values as rows [count, kv_heads, D]; zeros for a slot outside the cache
template <int T, int D, typename X>
__global__ __launch_bounds__(2 * D) void read_kernel(CacheView c, const int64_t *slots, int64_t count, X *k, X *v) {
  using L = CacheTile<T, D>;
  const Part part(c, false);
  const int head = part.head, b = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
  const int64_t row0 = part.row0;
  const Rows<T, D> from(c, head, row0, slots, count);
  const int step = c.kv_heads * D, left = (int)min(count - row0, (int64_t)kRows);
  if (!part.values) {
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
      X *const base = k + row0 * step + head * D;
      if (row < left) {
        if constexpr (T == Q4_0) {
          store_row<4>(at_row(base, r, 16 * u, step, 32 * b + 4 * g), x);
          store_row<4>(at_row(base, r, 16 * u, step, 32 * b + 16 + 4 * g), x + 4);
        } else {
          store_row<8>(at_row(base, r, 16 * u, step, 32 * b + 8 * g), x);
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
  X *const base = v + row0 * step + head * D;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int row = 16 * (j >> 2) + 4 * g + (j & 3);
    if (row < left) store_row<2>(at_row(base, 4 * g, row - 4 * g, step, 32 * b + 2 * r), x[j]);
  }
}

int invalid(const char *msg) { return set_error(MQ_E_INVALID, msg); }

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
    if (s < 0 || s % unit || s >= (int64_t(1) << 24))
      return invalid("mq_kv_cache_append: strides must be multiples of 16 bytes, 0 to 2^24 elements");
  if (!aligned16(c->data) || !aligned16(k) || !aligned16(v) || (reinterpret_cast<uintptr_t>(slots) & 7))
    return invalid("mq_kv_cache_append: buffers must be 16-byte aligned");
  const int64_t parts = (tokens + kRows - 1) / kRows * 2 * c->kv_heads;
  if (parts >= (int64_t(1) << 31)) return invalid("mq_kv_cache_append: too many tokens for the heads");
  const dim3 grid((unsigned)parts);
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
  const int64_t parts = (count + kRows - 1) / kRows * 2 * c->kv_heads;
  if (parts >= (int64_t(1) << 31)) return invalid("mq_kv_cache_read: too many tokens for the heads");
  const dim3 grid((unsigned)parts);
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
