// mq_heads.hip — what a text model does to q and k between their projections and the
// attention: each head RmsNormed with a weight (where the model has one) and its halves
// rotated by the token's position, and the same with k and v going on into the paged cache.
//
//   y = x rsqrt(mean(x^2) + eps) w,   a_i = position * inv_freq_i,
//   out_i = y_i cos a_i - y_(i+D/2) sin a_i,   out_(i+D/2) = y_(i+D/2) cos a_i + y_i sin a_i
//
// in f32, rounded once to bf16.  The angle is taken in 64 bits as turns, of which the whole
// ones are dropped, so that far positions keep their fraction (three roundings: within 2^-23 turns at
// 2^31), and its sine and cosine are within 0.53 and 0.51 of f32's last place: with v_sin_f32 and
// v_cos_f32, 2^-22.9 off, 4100 tokens took half a microsecond less, but half again as many results
// rounded to a neighbour of the right one.
//
// A value is read and written once; the bound is HBM, the launch for a step's few tokens.
// D / 8 lanes hold a head, each four values of its lower half and the four that they are
// rotated with, so that only the sum of squares crosses lanes, and a wave takes four heads
// of 128 (eight of 64) of one token at a time.  A lane's four angles serve all heads of the
// token that the wave takes: one pass of heads while tokens are few, the more the more waves
// there are to fill the chip anyway.  4100 tokens of 16 / 8 heads of 128 in bf16, 50 MB: 10.5 us;
// 14.1 with the wave's place in a vector register, which had every lane compute addresses and
// conditions.  7305 tokens of 20 / 20 heads of 64 from f32, 112 MB: 20 us (5.6 TB/s, part of it from
// the caches).
//
// Into the cache, a workgroup of 2 D threads takes 32 tokens of one k head through LDS
// (as bf16, what the attention of the prompt itself reads) into the shape in which
// mq_cache_write.h stores tiles; workgroups of v's and of q's share the launch.  32768
// tokens of 32 / 8 heads of 128 from bf16 into Q8_0, 809 MB read and written: 157 us (5.15 TB/s),
// 175 with all of q's workgroups behind the writing ones, whose vector work is half of the time.
#include "../../include/moldq.h"
#include "mq_cache_write.h"

namespace mq {
int set_error(int code, const char *msg);
}

namespace mq {
namespace {

struct HeadRows {
  const void *x;
  uint32_t token, head;  // strides in elements
  int heads;
  const float *weight;  // NULL: no norm
  __bf16 *out;          // contiguous [tokens, heads, D]; NULL: not wanted
};

struct HeadArgs {
  HeadRows q, k;
  const int64_t *positions;
  const float *inv_freq;
  float eps;
  int64_t tokens;
  int parts, passes;  // waves of a token, and of how many passes each
};

// The wave's place in its workgroup, in a scalar register, so that what follows from it is not
// computed in every lane.
__device__ __forceinline__ uint32_t wave_index() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// What one lane holds of a head.
template <typename X>
struct Piece;
template <>
struct Piece<__bf16> {
  uint2 u[2];
  __device__ void load(const __bf16 *p, int half) {
    u[0] = *reinterpret_cast<const uint2 *>(p);
    u[1] = *reinterpret_cast<const uint2 *>(p + half);
  }
  __device__ float get(int i, int j) const {
    const uint32_t w = j < 2 ? u[i].x : u[i].y;
    return __uint_as_float(j & 1 ? w & 0xFFFF0000u : w << 16);
  }
};
template <>
struct Piece<float> {
  float4 u[2];
  __device__ void load(const float *p, int half) {
    u[0] = *reinterpret_cast<const float4 *>(p);
    u[1] = *reinterpret_cast<const float4 *>(p + half);
  }
  __device__ float get(int i, int j) const { return j == 0 ? u[i].x : j == 1 ? u[i].y : j == 2 ? u[i].z : u[i].w; }
};

template <int kCtrl>
__device__ __forceinline__ float plus_lane(float v) {
  return v + __uint_as_float(dpp<kCtrl>(__float_as_uint(v)));
}
// The sum over the D / 8 lanes that hold a head.
template <int D>
__device__ __forceinline__ float head_sum(float v) {
  v = plus_lane<0xB1>(v);   // quad_perm 1 0 3 2
  v = plus_lane<0x4E>(v);   // quad_perm 2 3 0 1
  v = plus_lane<0x141>(v);  // row_half_mirror
  return D == 128 ? plus_lane<0x140>(v) : v;  // row_mirror
}

// A lane's part of the rotation: its four frequencies in turns, and a position's angles.
struct Turns {
  double freq[4];
  float c[4], s[4];
  __device__ void frequencies(const float *inv_freq) {
    const float4 f = *reinterpret_cast<const float4 *>(inv_freq);
    const float v[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) freq[i] = (double)v[i] * 0.15915494309189535;  // 1 / (2 pi)
  }
  // Of a = n / 4 + r turns, n the nearest whole number: sine and cosine of 2 pi r by their series
  // (what is left out is below 2^-29 of the sine, 2^-32 of the cosine, for |r| <= 1/8), in 64 bits
  // and rounded once, then by quarter.
  __device__ void at(int64_t position) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const double a = (double)position * freq[i], f = a - __builtin_rint(a);
      const float quarter = __builtin_rintf(4.f * (float)f);
      const int n = (int)quarter;
      const double r = __builtin_fma((double)quarter, -0.25, f), z = r * r;
      double x = __builtin_fma(z, 42.05869394489765, -76.70585975306136);
      x = __builtin_fma(z, x, 81.60524927607504);
      x = __builtin_fma(z, x, -41.341702240399755);
      x = __builtin_fma(z, x, 6.283185307179586);
      double y = __builtin_fma(z, -26.42625678337438, 60.24464137187666);
      y = __builtin_fma(z, y, -85.45681720669373);
      y = __builtin_fma(z, y, 64.93939402266829);
      y = __builtin_fma(z, y, -19.739208802178716);
      const float sine = (float)(r * x), cosine = (float)__builtin_fma(z, y, 1.);
      const float u = n & 1 ? cosine : sine, v = n & 1 ? sine : cosine;
      s[i] = n & 2 ? -u : u;
      c[i] = (n + 1) & 2 ? -v : v;
    }
  }
};

struct Weights {
  float w[2][4];
  bool norm;
  template <int D>
  __device__ void load(const float *weight, int sub) {
    norm = weight != nullptr;
    if (!norm) return;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float4 v = *reinterpret_cast<const float4 *>(weight + 4 * sub + i * (D / 2));
      w[i][0] = v.x, w[i][1] = v.y, w[i][2] = v.z, w[i][3] = v.w;
    }
  }
};

// The lane's eight results, packed: four of the lower half, four of the upper.
template <int D, typename X>
__device__ __forceinline__ void turn(const Piece<X> &p, const Weights &w, const Turns &t, float eps, uint2 (&out)[2]) {
  float x[2][4];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) x[i][j] = p.get(i, j);
  if (w.norm) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) sum = __builtin_fmaf(x[i][j], x[i][j], sum);
    const float r = rsqrtf(head_sum<D>(sum) * (1.f / D) + eps);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) x[i][j] = x[i][j] * r * w.w[i][j];
  }
  float a[4], b[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    a[j] = __builtin_fmaf(x[0][j], t.c[j], -(x[1][j] * t.s[j]));
    b[j] = __builtin_fmaf(x[1][j], t.c[j], x[0][j] * t.s[j]);
  }
  out[0] = make_uint2(pack2(a[0], a[1]), pack2(a[2], a[3]));
  out[1] = make_uint2(pack2(b[0], b[1]), pack2(b[2], b[3]));
}

// Part `part` of a token's q heads and, with kKeys, k heads, by one wave: passes of
// 64 / (D / 8) heads, q's first, `passes` of them from part * passes on.
template <int D, typename X, bool kKeys>
__device__ __forceinline__ void rotate_part(const HeadArgs &a, uint32_t token, uint32_t part) {
  constexpr int kLanes = D / 8, kHeads = 64 / kLanes;
  const int lane = threadIdx.x & 63, sub = lane & (kLanes - 1), in = lane / kLanes;
  const int q_passes = (a.q.heads + kHeads - 1) / kHeads, all = q_passes + (kKeys ? (a.k.heads + kHeads - 1) / kHeads : 0);
  int pass = (int)part * a.passes;
  const int end = min(all, pass + a.passes);
  if (pass >= end) return;
  const X *const q = static_cast<const X *>(a.q.x) + (uint64_t)token * a.q.token + 4 * sub;
  const X *const k = kKeys ? static_cast<const X *>(a.k.x) + (uint64_t)token * a.k.token + 4 * sub : nullptr;
  Piece<X> next;
  auto load = [&](int p) {
    if (!kKeys || p < q_passes) next.load(q + (uint64_t)min(p * kHeads + in, a.q.heads - 1) * a.q.head, D / 2);
    else next.load(k + (uint64_t)min((p - q_passes) * kHeads + in, a.k.heads - 1) * a.k.head, D / 2);
  };
  load(pass);
  const int64_t position = a.positions[token];
  Turns t;
  t.frequencies(a.inv_freq + 4 * sub);
  Weights w;
  w.load<D>(!kKeys || pass < q_passes ? a.q.weight : a.k.weight, sub);
  t.at(position);
  for (;;) {
    const Piece<X> x = next;
    const int now = pass++;
    if (pass < end) load(pass);
    uint2 out[2];
    turn<D, X>(x, w, t, a.eps, out);
    const bool of_q = !kKeys || now < q_passes;
    const int head = (of_q ? now : now - q_passes) * kHeads + in, heads = of_q ? a.q.heads : a.k.heads;
    if (head < heads) {
      __bf16 *const p = (of_q ? a.q.out : a.k.out) + ((int64_t)token * heads + head) * D + 4 * sub;
      *reinterpret_cast<uint2 *>(p) = out[0];
      *reinterpret_cast<uint2 *>(p + D / 2) = out[1];
    }
    if (pass >= end) return;
    if (kKeys && pass == q_passes) w.load<D>(a.k.weight, sub);
  }
}

template <int D, typename X>
__global__ __launch_bounds__(256) void rotate_kernel(HeadArgs a) {
  const uint32_t item = blockIdx.x * 4 + wave_index(), token = item / (uint32_t)a.parts;
  if (token < a.tokens) rotate_part<D, X, true>(a, token, item - token * (uint32_t)a.parts);
}

struct ValueRows {
  const void *x;
  uint32_t token, head;
};

// A group of 32 tokens has a workgroup for each of its k heads, then of its v heads, which
// write the cache, then `rotators` that rotate its q: neighbours, so that the vector work of the
// first and the bytes of the last overlap.
template <int T, int D, typename X>
__global__ __launch_bounds__(2 * D) void append_rotated_kernel(CacheView c, HeadArgs a, ValueRows v, const int64_t *slots, uint32_t rotators) {
  constexpr int kLanes = D / 8, kPitch = D + 8;  // rows 16 bytes apart beyond their size: a column of 16 rows in all banks
  __shared__ __attribute__((aligned(16))) __bf16 rows[kRows * kPitch];
  const uint32_t heads = (uint32_t)c.kv_heads, each = 2 * heads + rotators, group = blockIdx.x / each, in = blockIdx.x - group * each;
  if (in >= 2 * heads) {
    const uint32_t item = (in - 2 * heads) * (D / 32) + wave_index(), row = item / (uint32_t)a.parts, token = group * kRows + row;
    if (token < a.tokens) rotate_part<D, X, false>(a, token, item - row * (uint32_t)a.parts);
    return;
  }
  const int64_t row0 = (int64_t)group * kRows;
  const int last = (int)min(a.tokens - row0, (int64_t)kRows) - 1, b = (int)wave_index(), lane = threadIdx.x & 63;
  const int head = (int)(in >= heads ? in - heads : in);
  const Rows<T, D> to(c, head, row0, slots, a.tokens);
  if (in >= heads) {
    append_values<T, D>(to, b, lane, static_cast<const X *>(v.x) + row0 * v.token + (uint64_t)head * v.head, (int)v.token, last);
    return;
  }
  const int sub = threadIdx.x & (kLanes - 1), at = threadIdx.x / kLanes;  // 16 rows at a time
  const X *const base = static_cast<const X *>(a.k.x) + row0 * a.k.token + (uint64_t)head * a.k.head + 4 * sub;
  Piece<X> p[2];
  int64_t position[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int row = min(16 * u + at, last);
    p[u].load(base + (uint64_t)row * a.k.token, D / 2);
    position[u] = a.positions[row0 + row];
  }
  Turns t;
  t.frequencies(a.inv_freq + 4 * sub);
  Weights w;
  w.load<D>(a.k.weight, sub);
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int row = 16 * u + at;
    t.at(position[u]);
    uint2 out[2];
    turn<D, X>(p[u], w, t, a.eps, out);
#pragma unroll
    for (int i = 0; i < 2; ++i) *reinterpret_cast<uint2 *>(rows + row * kPitch + 4 * sub + i * (D / 2)) = out[i];
    if (a.k.out && row <= last) {
      __bf16 *const to_out = a.k.out + ((row0 + row) * heads + head) * D + 4 * sub;
      *reinterpret_cast<uint2 *>(to_out) = out[0];
      *reinterpret_cast<uint2 *>(to_out + D / 2) = out[1];
    }
  }
  __syncthreads();
  float x[2][8];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const __bf16 *const row = rows + (16 * u + (lane & 15)) * kPitch + 32 * b;
    const int g = lane >> 4;
    if constexpr (T == Q4_0) {
      load_row<4>(row + 4 * g, x[u]);
      load_row<4>(row + 16 + 4 * g, x[u] + 4);
    } else {
      load_row<8>(row + 8 * g, x[u]);
    }
  }
  put_keys<T, D, true>(to, b, lane, x);
}

int invalid(const char *msg) { return set_error(MQ_E_INVALID, msg); }

// What is wrong with the rows of q, k (and v), or NULL.
const char *rows_fault(int x_dtype, int head_dim, int64_t tokens, int heads, int kv_heads, std::initializer_list<int64_t> strides, float eps) {
  if (x_dtype != MQ_F32 && x_dtype != MQ_BF16) return "rotated heads: q, k and v are F32 or BF16";
  if (head_dim != 64 && head_dim != 128) return "rotated heads: head_dim is 64 or 128";
  if (tokens < 0 || tokens >= (int64_t(1) << 31)) return "rotated heads: tokens outside 0 .. 2^31";
  if (heads < 1 || heads > 65536 || kv_heads < 1 || kv_heads > 65536) return "rotated heads: 1 to 65536 heads";
  const int64_t unit = x_dtype == MQ_F32 ? 4 : 8;
  for (int64_t s : strides)
    if (s < 0 || s % unit || s >= (int64_t(1) << 24)) return "rotated heads: strides must be multiples of 16 bytes, 0 to 2^24 elements";
  if (!(eps >= 0.f && eps <= __FLT_MAX__)) return "rotated heads: eps is not negative and finite";
  return nullptr;
}

// How a token's passes are shared: a wave each while the waves do not fill the chip (256
// CUs, 32 waves), then as many passes a wave as leave it so.  -> the waves.
int64_t share(HeadArgs &a, int passes) {
  const int64_t waves = a.tokens * passes, each = waves / 8192 < 1 ? 1 : waves / 8192 < passes ? waves / 8192 : passes;
  a.parts = (int)((passes + each - 1) / each);
  a.passes = (passes + a.parts - 1) / a.parts;
  return a.tokens * a.parts;
}

// Workgroups of so many threads that a launch takes: its threads are counted in 32 bits.
bool takes_grid(int64_t groups, int threads) { return groups < (int64_t(1) << 32) / threads; }

}  // namespace
}  // namespace mq

extern "C" int mq_rotate_heads(const void *q, int64_t q_token_stride, int64_t q_head_stride, int heads, const void *k,
                               int64_t k_token_stride, int64_t k_head_stride, int kv_heads, int x_dtype, int head_dim,
                               int64_t tokens, const int64_t *positions, const float *inv_freq, const float *q_weight,
                               const float *k_weight, float eps, void *q_out, void *k_out, void *stream) {
  using namespace mq;
  if (const char *fault = rows_fault(x_dtype, head_dim, tokens, heads, kv_heads, {q_token_stride, q_head_stride, k_token_stride, k_head_stride}, eps))
    return invalid(fault);
  if (tokens == 0) return MQ_OK;
  if (!q || !k || !positions || !inv_freq || !q_out || !k_out) return invalid("mq_rotate_heads: NULL pointer");
  if (!aligned16(q) || !aligned16(k) || !aligned16(q_out) || !aligned16(k_out) || !aligned16(inv_freq) || !aligned16(q_weight) ||
      !aligned16(k_weight) || (reinterpret_cast<uintptr_t>(positions) & 7))
    return invalid("mq_rotate_heads: buffers must be 16-byte aligned");
  HeadArgs a{{q, (uint32_t)q_token_stride, (uint32_t)q_head_stride, heads, q_weight, static_cast<__bf16 *>(q_out)},
             {k, (uint32_t)k_token_stride, (uint32_t)k_head_stride, kv_heads, k_weight, static_cast<__bf16 *>(k_out)},
             positions, inv_freq, eps, tokens, 0, 0};
  const int each = 64 / (head_dim / 8);
  const int64_t groups = (share(a, (heads + each - 1) / each + (kv_heads + each - 1) / each) + 3) / 4;
  // of 8192 tokens and more a wave takes one whole, and a workgroup four
  if (!takes_grid(groups, 256)) return invalid("mq_rotate_heads: up to 2^26 - 4 tokens");
  const dim3 grid((unsigned)groups);
  auto launch = [&]<int D>() {
    if (x_dtype == MQ_F32) hipLaunchKernelGGL((rotate_kernel<D, float>), grid, dim3(256), 0, static_cast<hipStream_t>(stream), a);
    else hipLaunchKernelGGL((rotate_kernel<D, __bf16>), grid, dim3(256), 0, static_cast<hipStream_t>(stream), a);
  };
  if (head_dim == 128) launch.operator()<128>();
  else launch.operator()<64>();
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MQ_OK : set_error(MQ_E_HIP, hipGetErrorString(e));
}

extern "C" int mq_kv_cache_append_rotated(const mq_kv_cache *c, const int64_t *slots, const void *q, int64_t q_token_stride,
                                          int64_t q_head_stride, int heads, const void *k, int64_t k_token_stride,
                                          int64_t k_head_stride, const void *v, int64_t v_token_stride, int64_t v_head_stride,
                                          int x_dtype, int64_t tokens, const int64_t *positions, const float *inv_freq,
                                          const float *q_weight, const float *k_weight, float eps, void *q_out, void *k_out,
                                          void *stream) {
  using namespace mq;
  if (const char *fault = cache_fault(c)) return invalid(fault);
  if (const char *fault = rows_fault(x_dtype, c->head_dim, tokens, heads, c->kv_heads,
                                     {q_token_stride, q_head_stride, k_token_stride, k_head_stride, v_token_stride, v_head_stride}, eps))
    return invalid(fault);
  if (tokens == 0) return MQ_OK;
  if ((c->pages && !c->data) || !slots || !q || !k || !v || !positions || !inv_freq || !q_out)
    return invalid("mq_kv_cache_append_rotated: NULL pointer");
  if (!aligned16(c->data) || !aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(q_out) || !aligned16(k_out) || !aligned16(inv_freq) ||
      !aligned16(q_weight) || !aligned16(k_weight) || ((reinterpret_cast<uintptr_t>(positions) | reinterpret_cast<uintptr_t>(slots)) & 7))
    return invalid("mq_kv_cache_append_rotated: buffers must be 16-byte aligned");
  HeadArgs a{{q, (uint32_t)q_token_stride, (uint32_t)q_head_stride, heads, q_weight, static_cast<__bf16 *>(q_out)},
             {k, (uint32_t)k_token_stride, (uint32_t)k_head_stride, c->kv_heads, k_weight, static_cast<__bf16 *>(k_out)},
             positions, inv_freq, eps, tokens, 0, 0};
  const int each = 64 / (c->head_dim / 8);
  share(a, (heads + each - 1) / each);
  const int64_t rotators = (int64_t)kRows * a.parts / (c->head_dim / 32), groups = (tokens + kRows - 1) / kRows * (2 * c->kv_heads + rotators);
  if (!takes_grid(groups, 2 * c->head_dim)) return invalid("mq_kv_cache_append_rotated: tokens * (kv_heads + 512 / head_dim) below 2^35 / head_dim");
  const dim3 grid((unsigned)groups);
  const ValueRows rows{v, (uint32_t)v_token_stride, (uint32_t)v_head_stride};
  with_cache_type(c, [&]<int T, int D>() {
    if (x_dtype == MQ_F32)
      hipLaunchKernelGGL((append_rotated_kernel<T, D, float>), grid, dim3(2 * D), 0, static_cast<hipStream_t>(stream), view(c), a, rows, slots,
                         (uint32_t)rotators);
    else
      hipLaunchKernelGGL((append_rotated_kernel<T, D, __bf16>), grid, dim3(2 * D), 0, static_cast<hipStream_t>(stream), view(c), a, rows, slots,
                         (uint32_t)rotators);
  });
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MQ_OK : set_error(MQ_E_HIP, hipGetErrorString(e));
}
