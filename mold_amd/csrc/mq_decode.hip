// mq_decode.hip — attention of one new token per sequence over the paged cache:
//   out[b, h] = sum_{t < len_b} p_t v[t, g],  p = softmax_t(scale q[b, h] . k[t, g]),
// g = h / (heads / kv_heads), in one pass over the cache (the decode step of the
// prompt-expansion model, crates/mold-inference/src/expand.rs:200-203).
//
// What bounds it: reading the cache once.  The products of a group's heads (up to
// 16, the other columns of the matrix instruction are zeros) with a tile of 32
// tokens are 16 MFMAs, far from their rate, also after a block type's bytes have
// been widened.  So the kernel is laid out for the loads:
//   * the work of the whole batch is one line of (sequence, k/v head, tile of 32
//     tokens), cut into equal runs, one a wave, whatever the lengths are; the
//     lengths stay on the device (each wave adds them up), so the host neither
//     waits nor plans;
//   * a tile is read in the order of the matrix operands (mq_cache.h), 1 KiB a
//     load instruction; a wave has one tile in flight, the next one's keys
//     requested when this one's scores are made and its values when these are
//     added, and 8 or 12 waves a CU together keep HBM busy;
//   * the scores are computed transposed, S^T = K Q^T, so that a lane's eight
//     probabilities are its B operand of O^T = V^T P^T, as they stand;
//   * the block types' whole numbers enter the products as they are: a key block's
//     scale multiplies its 32 values' dot product in f32, a value block's the
//     probabilities, so that neither K nor V is rounded at all;
//   * the probabilities enter as two bf16 numbers, one near them and what it
//     lacks (relative 2^-16 together): the second product costs matrix time that
//     the loads leave free, and a step of a few tokens, whose roundings do not
//     average out, is as exact as its output's type.
// The waves of a workgroup that lie within one (sequence, head unit) join in LDS.
// What holds a whole one stores its result; the others store f32 sums, which
// join_kernel adds in the order of the line.  Where page tables are short a
// workgroup takes a whole (sequence, head unit), and there is no second launch.
// Reached (32 / 8 heads of 128, us a call, TB/s of the cache's bytes): 64 sequences
// of 8192 tokens BF16 358 (6.0), one of 65001 54 (4.9), 40 ragged ones up to 6000
// in Q8_0 51 (3.9: launch, the line and the join are some 10 us of it).
#include "../../include/moldq.h"
#include "mq_cache.h"

namespace mq {
int set_error(int code, const char *msg);
}

namespace mq {
namespace {

constexpr int kWaves = 4;           // of a workgroup whose waves take runs of the line
constexpr int kHeads = 16;          // columns of the matrix instruction

struct DecodeArgs {
  CacheView cache;
  int64_t pages;
  const __bf16 *q;
  __bf16 *out;
  int64_t sq, hq, so, ho;      // batch and head strides
  const int32_t *table, *lengths;
  int64_t table_stride;
  int max_pages, batch, heads, group, chunks;  // chunks of 16 heads of a group
  int waves;
  float scale;                 // times log2(e)
  float least;                 // what the running maximum starts at (least_score)
  float *partial;
};

__device__ __forceinline__ int lane_of(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }

// A value that is the same in all lanes, as the scalar that the compiler does not
// make of a division's result (or of what follows from it) by itself.
__device__ __forceinline__ int scalar(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Sums over lanes 0 .. lane.
__device__ __forceinline__ int scan64(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast 15 into rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast 31 into rows 2 and 3
  return x;
}

// The line of work: sequence by sequence, in it head unit by head unit (k/v head
// and chunk of its group), in it tile by tile.  Lane i of a wave holds sequence
// c0 + i; every wave sees the same line.
struct Line {
  int c0, before;      // first sequence of the 64 at hand, tiles of those before
  int n, tiles, upto;  // this lane's: its length, its tiles, the tiles of c0 .. its own
  int total, heads;    // tiles of all sequences, head units
  int runs, base, rest;  // runs, their least length, how many are one longer

  // The tiles of a sequence of n tokens, as far as its table reaches.
  __device__ static int tiles_of(const DecodeArgs &a, int n) {
    return n > 0 ? (min(n, a.max_pages * a.cache.page_tokens) + kTileTokens - 1) / kTileTokens : 0;
  }
  __device__ void load(const DecodeArgs &a, int lane) {
    const int b = c0 + lane, len = a.lengths[min(b, a.batch - 1)];
    n = b < a.batch ? len : 0;
    tiles = tiles_of(a, n);
    upto = scan64(tiles);
  }
  __device__ void make(const DecodeArgs &a, int lane) {
    c0 = before = total = 0;
    heads = a.cache.kv_heads * a.chunks;
    for (int c = (a.batch - 1) & ~63; c >= 0; c -= 64) {  // the first 64 last: they stay
      c0 = c;
      load(a, lane);
      total += lane_of(upto, 63);
    }
    const int units = total * heads;
    runs = max(min(a.waves, units), 1);
    base = scalar(units / runs);
    rest = units - base * runs;
  }
  __device__ int start(int run) const { return run * base + min(run, rest); }
  __device__ int run_of(int unit) const {
    const int longer = rest * (base + 1);
    return unit < longer ? unit / (base + 1) : rest + (unit - longer) / base;
  }
  // Whether the runs of `run`'s workgroup are all within the units u0 .. u1 - 1 of
  // one (sequence, head unit): then their sums are one record, at the first's place.
  __device__ bool together(int run, int u0, int u1) const {
    const int r0 = run & -kWaves;
    return r0 + kWaves <= runs && start(r0) >= u0 && start(r0 + kWaves) <= u1;
  }
  // The lane of the sequence that holds `unit`, after its 64 have been loaded.
  __device__ int seek(const DecodeArgs &a, int lane, int unit) {
    while ((before + lane_of(upto, 63)) * heads <= unit) {
      before += lane_of(upto, 63);
      c0 += 64;
      load(a, lane);
    }
    return __builtin_ctzll(__ballot((before + upto) * heads > unit));
  }
};

template <int T, int D>
struct Tile {
  using L = CacheTile<T, D>;
  static constexpr int kKeyWords = L::kKeyLane / 4, kScaleWords = L::kQuant ? 4 * L::kBlocks : 0;
  uint32_t k[2][kKeyWords], v[2 * kKeyWords], ks[kScaleWords + 1], vs[kScaleWords + 1];

  // Buffer loads: the tile's address is in scalar registers, a lane adds only its
  // place in a piece, so that no load needs vector registers for an address.
  __device__ __forceinline__ static void get16(uint32_t *to, __amdgpu_buffer_rsrc_t tile, int lane_at, int at) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    const u32x4 u = __builtin_amdgcn_raw_buffer_load_b128(tile, lane_at, at, 0);
    to[0] = u.x; to[1] = u.y; to[2] = u.z; to[3] = u.w;
  }
  __device__ __forceinline__ static __amdgpu_buffer_rsrc_t at(const uint8_t *tile) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(tile), 0, L::kBytes, 0x00027000);
  }
  __device__ __forceinline__ static int scale_lane(int lane) { return (lane >> 4) * (16 * L::kBlocks); }
  __device__ __forceinline__ void load_keys(__amdgpu_buffer_rsrc_t tile, int lane) {
    if constexpr (L::kKeyPiece == 16) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < kKeyWords; i += 4) get16(&k[u][i], tile, lane * 16, u * 64 * L::kKeyLane + i * 256);
    } else {
      typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const u32x2 w = __builtin_amdgcn_raw_buffer_load_b64(tile, lane * 8, u * 64 * L::kKeyLane, 0);
        k[u][0] = w.x;
        k[u][1] = w.y;
      }
    }
    if constexpr (L::kQuant)
#pragma unroll
      for (int i = 0; i < kScaleWords; i += 4) get16(&ks[i], tile, scale_lane(lane), 2 * L::kPlane + 4 * i);
  }
  __device__ __forceinline__ void load_values(__amdgpu_buffer_rsrc_t tile, int lane) {
#pragma unroll
    for (int i = 0; i < 2 * kKeyWords; i += 4) get16(&v[i], tile, lane * 16, L::kPlane + i * 256);
    if constexpr (L::kQuant)
#pragma unroll
      for (int i = 0; i < kScaleWords; i += 4) get16(&vs[i], tile, scale_lane(lane), 2 * L::kPlane + L::kScales + 4 * i);
  }
};

__device__ __forceinline__ bf16x8 operand(const uint32_t *w) {
  bf16x8 x;
  __builtin_memcpy(&x, w, 16);
  return x;
}
__device__ __forceinline__ float half_of(const uint32_t *w, int i) {
  return h2f((uint16_t)(w[i >> 1] >> (16 * (i & 1))));
}
// eight signed bytes as whole numbers, exact in bf16
__device__ __forceinline__ bf16x8 bytes8(const uint32_t *w) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    u[i] = pack2((float)(int8_t)(w[i >> 1] >> (16 * (i & 1))), (float)(int8_t)(w[i >> 1] >> (16 * (i & 1) + 8)));
  return operand(u);
}
// A nibble n, stored + 8, as n + 128 in bf16: the bit pattern 0x4300 | n.  One
// operation makes two values where the way through f32 takes seven; the 136 that
// are too many leave again as a product with a constant operand.  (Bytes as u + 1024
// in f16, with q in f16 too, made the Q8_0 kernel no faster: it waits for memory.)
constexpr uint32_t kMinus136 = 0xC308C308u;
// the low nibbles of w's bytes 0, 2, 1, 3; above: 0x43004300 in a register (an
// instruction takes one constant that is not in one, and that is the mask)
__device__ __forceinline__ void nibbles4_above(uint32_t w, uint32_t above, uint32_t *u) {
  u[0] = (w & 0x000F000Fu) | above;
  u[1] = ((w >> 8) & 0x000F000Fu) | above;
}
__device__ __forceinline__ bf16x8 four_of(uint32_t two) {
  const uint32_t u[4] = {two, two, two, two};
  return operand(u);
}

// p as two operands, hi + lo
struct Split {
  bf16x8 hi, lo;
};
// For whole numbers: hi rounded, lo what it lacks.
__device__ __forceinline__ Split split8(const float *p) {
  uint32_t hi[4], lo[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    hi[i] = pack2(p[2 * i], p[2 * i + 1]);
    lo[i] = pack2(p[2 * i] - __uint_as_float(hi[i] << 16), p[2 * i + 1] - __uint_as_float(hi[i] & 0xFFFF0000u));
  }
  return {operand(hi), operand(lo)};
}
// For values that may be infinite, p >= 0: hi the next bf16 below p, so that lo
// is positive too and neither product of an infinity is a NaN.
__device__ __forceinline__ Split split8_below(const float *p) {
  uint32_t hi[4], lo[4], b[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) b[j] = __builtin_elementwise_sub_sat(__float_as_uint(p[j]), 1u) & 0xFFFF0000u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    hi[i] = b[2 * i] >> 16 | b[2 * i + 1];
    lo[i] = pack2(p[2 * i] - __uint_as_float(b[2 * i]), p[2 * i + 1] - __uint_as_float(b[2 * i + 1]));
  }
  return {operand(hi), operand(lo)};
}

// The value combined with that of the other lanes of its column (lane % 16).
__device__ __forceinline__ float column_max(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return half_max(__builtin_fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float column_add(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return half_add(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// A lane's eight columns of a block, in order, from its two operands' results.
__device__ __forceinline__ void put8(float *p, const f32x4 *x) {
  reinterpret_cast<f32x4 *>(p)[0] = f32x4{x[0][0], x[1][0], x[0][1], x[1][1]};
  reinterpret_cast<f32x4 *>(p)[1] = f32x4{x[0][2], x[1][2], x[0][3], x[1][3]};
}

// Shares of one (sequence, head unit) that the waves of a workgroup hold, added
// in the order of the waves, each relative to its own maximum.
template <int D, int W>
struct Shares {
  float o[W][kHeads][D + 4], m[W][kHeads], l[W][kHeads];

  __device__ __forceinline__ void put(int wave, int lane, const f32x4 *x, float ms, float sum) {
    const int g = lane >> 4, r = lane & 15;
#pragma unroll
    for (int b = 0; b < D / 32; ++b) put8(&o[wave][r][32 * b + 8 * g], x + 2 * b);
    if (g == 0) {
      m[wave][r] = ms;
      l[wave][r] = sum;
    }
  }
  // head r's sums of columns 4 col .. + 3, relative to 2^top
  __device__ __forceinline__ f32x4 add(int r, int col, float &top, float &sum) const {
    top = m[0][r];
#pragma unroll
    for (int w = 1; w < W; ++w) top = __builtin_fmaxf(top, m[w][r]);
    f32x4 x{0.f, 0.f, 0.f, 0.f};
    sum = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float e = m[w][r] == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(m[w][r] - top);
      sum = __builtin_fmaf(e, l[w][r], sum);
      const f32x4 v = *reinterpret_cast<const f32x4 *>(&o[w][r][4 * col]);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = __builtin_fmaf(e, v[i], x[i]);
    }
    return x;
  }
};

__device__ __forceinline__ void store4(__bf16 *p, const f32x4 &x, float inv) {
  *reinterpret_cast<uint2 *>(p) = make_uint2(pack2(x[0] * inv, x[1] * inv), pack2(x[2] * inv, x[3] * inv));
}

// P > 0: a workgroup of P waves takes a (sequence, head unit), its waves equal shares
// of its tiles, and stores the result.  P = 0: a wave takes a run of the line.
template <int T, int D, int P>
__global__ __launch_bounds__(64 * (P ? P : kWaves), P == 8 ? 2 : D == 128 ? 3 : 4) void decode_kernel(const DecodeArgs a) {
  using L = CacheTile<T, D>;
  constexpr bool kPair = P > 0;
  constexpr int kB = L::kBlocks, kC = D / 16, kW = kPair ? P : kWaves;
  __shared__ Shares<D, kW> shares;
  const int lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int run = blockIdx.x * kW + wave;
  const int tpp = scalar(a.cache.page_tokens / kTileTokens), nh = min(a.group, kHeads);

  // The sequence's page numbers page0 .. page0 + 63, one a lane, and the place of
  // the tile that is fetched next.
  int page0, page, in_page, numbers;
  // What the wave works on: tiles t .. t + count - 1 of a sequence, for one head unit.
  int b, n, tiles, kv, chunk, t;  // sequence, its length, its tiles, k/v head, chunk of its heads
  Line line;
  int at, end;              // this wave's units
  int idx = 0;              // the lane of sequence b
  bool together = kPair;    // the workgroup's waves hold shares of one (sequence, head unit)
  bool whole = kPair;       // and no other wave does
  if constexpr (kPair) {
    const int units = a.cache.kv_heads * a.chunks, head = blockIdx.x % units;
    b = blockIdx.x / units;
    kv = head / a.chunks;
    chunk = head - kv * a.chunks;
    page0 = numbers = 0;  // its table has up to 64 pages, or none; it and the length are read together
    if (a.max_pages > 0) numbers = a.table[b * a.table_stride + min(lane, a.max_pages - 1)];
    n = a.lengths[b];
    tiles = Line::tiles_of(a, n);
    if (tiles == 0) {
      const uint32_t v = n > 0 ? 0x7FC07FC0u : 0u;  // tokens, but a table without pages: NaN
      const int count = min(a.group - chunk * kHeads, kHeads);
      for (int i = threadIdx.x; i < count * (D / 4); i += 64 * kW)
        *reinterpret_cast<uint2 *>(a.out + b * a.so + (int64_t)(kv * a.group + chunk * kHeads + i / (D / 4)) * a.ho +
                                   4 * (i % (D / 4))) = make_uint2(v, v);
      return;
    }
    at = t = tiles * wave / kW;
    end = tiles * (wave + 1) / kW;
  } else {
    line.make(a, lane);
    if (line.total == 0 || run >= line.runs) return;
    at = line.start(run);
    end = line.start(run + 1);
    idx = line.seek(a, lane, at);
    b = line.c0 + idx;
    n = lane_of(line.n, idx);
    tiles = lane_of(line.tiles, idx);
    const int in = at - (line.before + lane_of(line.upto, idx) - tiles) * line.heads, head = scalar(in / tiles);
    t = in - head * tiles;
    kv = scalar(head / a.chunks);
    chunk = head - kv * a.chunks;
    const int u0 = at - t, u1 = u0 + tiles;
    together = line.together(run, u0, u1);
    whole = together && line.start(run & -kWaves) == u0 && line.start((run & -kWaves) + kWaves) == u1;
  }
  const int first = at;

  bool bad;  // a page is not one of the cache's, or the sequence is longer than its table
  auto number_pages = [&]() {
    numbers = a.table[b * a.table_stride + min(page0 + lane, a.max_pages - 1)];  // no branch: what follows stays uniform
    asm volatile("" : "+v"(numbers));  // used here, so that the wait for it is here and not in every tile
  };
  auto place = [&]() {  // the tile's address
    const uint32_t id = (uint32_t)lane_of(numbers, page - page0);
    const bool ok = id < a.pages;
    bad |= !ok;
    return Tile<T, D>::at(a.cache.data + (((int64_t)(ok ? id : 0) * a.cache.kv_heads + kv) * tpp + in_page) * L::kBytes);
  };
  auto advance = [&]() {
    if (++in_page == tpp) {
      in_page = 0;
      if (++page == page0 + 64) {
        page0 = page;
        number_pages();
      }
    }
  };

  bf16x8 qf[kB];  // q, the scores' B operand
  f32x4 o[kC];  // O^T: this lane's head, columns 32 b + 8 g + 2 i + c in o[2 b + c][i]
  float m, l;
  auto begin = [&]() {
    const int in = chunk * kHeads + r;
    const __bf16 *p = a.q + b * a.sq + (int64_t)(kv * a.group + (in < a.group ? in : 0)) * a.hq;
    const uint32_t mine = in < a.group ? ~0u : 0u;  // a column past the group's heads: zeros
    uint32_t w[kB][4];
#pragma unroll
    for (int b = 0; b < kB; ++b) {
      if constexpr (T == Q4_0) {  // the values of a key lane's low, then high nibbles, each in the order 0, 2, 1, 3
        const uint2 lo = *reinterpret_cast<const uint2 *>(p + 32 * b + 4 * g), hi = *reinterpret_cast<const uint2 *>(p + 32 * b + 16 + 4 * g);
        w[b][0] = __builtin_amdgcn_perm(lo.y, lo.x, 0x05040100u);
        w[b][1] = __builtin_amdgcn_perm(lo.y, lo.x, 0x07060302u);
        w[b][2] = __builtin_amdgcn_perm(hi.y, hi.x, 0x05040100u);
        w[b][3] = __builtin_amdgcn_perm(hi.y, hi.x, 0x07060302u);
      } else {
        const uint4 x = *reinterpret_cast<const uint4 *>(p + 32 * b + 8 * g);
        w[b][0] = x.x; w[b][1] = x.y; w[b][2] = x.z; w[b][3] = x.w;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) w[b][i] &= mine;
    }
#pragma unroll
    for (int b = 0; b < kB; ++b) qf[b] = operand(w[b]);
#pragma unroll
    for (int c = 0; c < kC; ++c) o[c] = f32x4{0.f, 0.f, 0.f, 0.f};
    m = a.least;
    l = 0.f;
    bad = n > a.max_pages * a.cache.page_tokens;
  };

  Tile<T, D> x;
  f32x4 s[2];
  uint32_t above = 0x43004300u;
  if constexpr (T == Q4_0) asm volatile("" : "+v"(above));
  bf16x8 offset = four_of(kMinus136);
  auto scores = [&]() {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      s[h] = f32x4{0.f, 0.f, 0.f, 0.f};
      // a product with the offset every time: kept from one tile to the next it would
      // take 16 registers, and copies of them
      if constexpr (T == Q4_0) asm volatile("" : "+v"(offset));
      if constexpr (T == BF16) {
#pragma unroll
        for (int b = 0; b < kB; ++b) s[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(operand(&x.k[h][4 * b]), qf[b], s[h], 0, 0, 0);
      } else {
#pragma unroll
        for (int b = 0; b < kB; ++b) {
          f32x4 dot{0.f, 0.f, 0.f, 0.f};
          if constexpr (T == Q8_0) {
            dot = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bytes8(&x.k[h][2 * b]), qf[b], dot, 0, 0, 0);
          } else {
            uint32_t w[4];
            nibbles4_above(x.k[h][b], above, w);
            nibbles4_above(x.k[h][b] >> 4, above, w + 2);
            dot = __builtin_amdgcn_mfma_f32_16x16x32_bf16(offset, qf[b], dot, 0, 0, 0);
            dot = __builtin_amdgcn_mfma_f32_16x16x32_bf16(operand(w), qf[b], dot, 0, 0, 0);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) s[h][i] = __builtin_fmaf(half_of(x.ks, (h * kB + b) * 4 + i), dot[i], s[h][i]);
        }
      }
    }
  };
  auto take_in = [&](int tile) {
    if (tile + 1 == tiles) {  // tokens past the sequence's last: no weight, and no value or scale that could make 0 x NaN
      int over = n - (tiles - 1) * kTileTokens;
      asm volatile("" : "+s"(over));  // its masks are made here, not kept through every tile
      uint32_t keep[4] = {0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (16 * (j >> 2) + 4 * g + (j & 3) < over) keep[j >> 1] |= 0xFFFFu << (16 * (j & 1));
        else s[j >> 2][j & 3] = -__builtin_inff();
      }
      if constexpr (T == BF16) {
#pragma unroll
        for (int i = 0; i < 4 * kC; ++i) x.v[i] &= keep[i & 3];
      } else {
#pragma unroll
        for (int i = 0; i < 4 * kB; ++i) x.vs[i] &= keep[i & 3];
      }
    }
    float mx = __builtin_fmaxf(__builtin_fmaxf(__builtin_fmaxf(s[0][0], s[0][1]), __builtin_fmaxf(s[0][2], s[0][3])),
                               __builtin_fmaxf(__builtin_fmaxf(s[1][0], s[1][1]), __builtin_fmaxf(s[1][2], s[1][3])));
    mx = column_max(mx);
    if (__any(mx > m)) {
      const float mn = __builtin_fmaxf(m, mx), f = __builtin_amdgcn_exp2f((m - mn) * a.scale);
      m = mn;
      l *= f;
#pragma unroll
      for (int c = 0; c < kC; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[c][i] *= f;
    }
    const float ms = m * a.scale;
    float p[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      p[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j >> 2][j & 3], a.scale, -ms));
      l += p[j];
    }
    // O^T += V^T P^T over one operand of V
    auto add = [&](f32x4 &to, const bf16x8 &v, const Split &w) {
      to = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, w.lo, to, 0, 0, 0);
      to = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, w.hi, to, 0, 0, 0);
    };
    if constexpr (T == BF16) {
      const Split w = split8_below(p);
#pragma unroll
      for (int c = 0; c < kC; ++c) add(o[c], operand(&x.v[4 * c]), w);
    } else {
#pragma unroll
      for (int b = 0; b < kB; ++b) {
        // a token's probability times its block's scale (as a fused f16 operand: + 0
        // keeps the compiler from a conversion and a product), for Q4_0 in the order
        // 0, 2, 1, 3 of each four tokens, which its operands come in
        float pd[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int k = T == Q4_0 ? (j & 4) | (j & 1) << 1 | (j >> 1 & 1) : j;
          pd[j] = __builtin_fmaf(p[k], half_of(&x.vs[4 * b], k), 0.f);
        }
        const Split w = split8(pd);
        if constexpr (T == Q8_0) {
#pragma unroll
          for (int c = 0; c < 2; ++c) add(o[2 * b + c], bytes8(&x.v[4 * b + 2 * c]), w);
        } else {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t v[4];
            nibbles4_above(x.v[2 * b] >> (4 * c), above, v);
            nibbles4_above(x.v[2 * b + 1] >> (4 * c), above, v + 2);
            add(o[2 * b + c], four_of(kMinus136), w);
            add(o[2 * b + c], operand(v), w);
          }
        }
      }
    }
  };
  // the tiles at hand are done: their sums, or the result if they were all
  auto finish = [&](int from, int count) {
    if (bad) l = __builtin_nanf("");
    l = column_add(l);
    const int in = chunk * kHeads + r;
    if (together) {
      shares.put(wave, lane, o, m * a.scale, l);
    } else if (count == tiles) {
      const float inv = 1.f / l;
      __bf16 *p = a.out + b * a.so + (int64_t)(kv * a.group + in) * a.ho + 8 * g;
      if (in < a.group)
#pragma unroll
        for (int i = 0; i < kB; ++i) {
          const f32x4 &x = o[2 * i], &y = o[2 * i + 1];
          *reinterpret_cast<uint4 *>(p + 32 * i) = make_uint4(pack2(x[0] * inv, y[0] * inv), pack2(x[1] * inv, y[1] * inv),
                                                              pack2(x[2] * inv, y[2] * inv), pack2(x[3] * inv, y[3] * inv));
        }
    } else {
      float *rec = a.partial + (int64_t)(2 * run + (from != first)) * nh * (D + 4);
      if (in < a.group) {
#pragma unroll
        for (int i = 0; i < kB; ++i) put8(rec + r * D + 32 * i + 8 * g, o + 2 * i);
        if (g == 0) *reinterpret_cast<float2 *>(rec + nh * D + 2 * r) = make_float2(m * a.scale, l);
      }
    }
  };

  while (at < end) {
    const int count = min(tiles - t, end - at);
    page = scalar(t / tpp);
    if (!kPair) page0 = page;
    in_page = t - page * tpp;
    begin();
    if (!kPair) number_pages();
    __amdgpu_buffer_rsrc_t tile = place();
    x.load_keys(tile, lane);
    x.load_values(tile, lane);
#pragma unroll
    for (int b = 0; b < kB; ++b) asm volatile("" : "+v"(qf[b]));  // waited for here, not in every tile
    // The next tile's keys are requested as soon as this one's scores are made, its
    // values as soon as these are added.  Past the last the keys are requested once
    // more (a branch there would make the values' wait one for all loads).
    for (int i = 0;;) {
      scores();
      const bool last = i + 1 == count;
      if (!last) {
        advance();
        tile = place();
      }
      __builtin_amdgcn_sched_barrier(0);
      x.load_keys(tile, lane);
      __builtin_amdgcn_sched_barrier(0);
      take_in(t + i);
      if (last) break;
      ++i;
      __builtin_amdgcn_sched_barrier(0);
      x.load_values(tile, lane);
      __builtin_amdgcn_sched_barrier(0);
    }
    finish(at, count);
    at += count;
    if constexpr (!kPair) {
      if (at < end) {  // the sequence's next head unit, or the next sequence with tokens
        t = 0;
        if (++chunk == a.chunks) {
          chunk = 0;
          ++kv;
        }
        if (kv == a.cache.kv_heads) {
          kv = 0;
          uint64_t more = __ballot(line.tiles > 0) & ~((2ull << idx) - 1);
          while (more == 0) {
            line.before += lane_of(line.upto, 63);
            line.c0 += 64;
            line.load(a, lane);
            more = __ballot(line.tiles > 0);
          }
          idx = __builtin_ctzll(more);
          b = line.c0 + idx;
          n = lane_of(line.n, idx);
          tiles = lane_of(line.tiles, idx);
        }
      }
    }
  }
  if constexpr (kPair)
    if (first == end) {  // a share without tiles
#pragma unroll
      for (int c = 0; c < kC; ++c) o[c] = f32x4{0.f, 0.f, 0.f, 0.f};
      shares.put(wave, lane, o, -__builtin_inff(), 0.f);
    }
  if (!together) return;
  __syncthreads();
  const int count = min(a.group - chunk * kHeads, kHeads);
  for (int i = threadIdx.x; i < count * (D / 4); i += 64 * kW) {
    const int head = i / (D / 4), col = i - head * (D / 4);
    float top, sum;
    const f32x4 x = shares.add(head, col, top, sum);
    if (whole) {
      store4(a.out + b * a.so + (int64_t)(kv * a.group + chunk * kHeads + head) * a.ho + 4 * col, x, 1.f / sum);
    } else {
      float *rec = a.partial + (int64_t)(2 * (run & -kWaves)) * nh * (D + 4);
      *reinterpret_cast<f32x4 *>(rec + head * D + 4 * col) = x;
      if (col == 0) *reinterpret_cast<float2 *>(rec + nh * D + 2 * head) = make_float2(top, sum);
    }
  }
}

// A row's shares, added in the order of the line, each relative to its own
// maximum; zeros for a sequence without tokens.  A workgroup a row: D / 4 threads
// take 4 columns of every kLanes-th share, kBatch loads in flight.
template <int D>
__global__ __launch_bounds__(256) void join_kernel(const DecodeArgs a) {
  constexpr int kCols = D / 4, kLanes = 256 / kCols, kBatch = 4;
  __shared__ float red[kLanes][D + 2];
  const int lane = threadIdx.x & 63;
  const int b = blockIdx.x / a.heads, head = blockIdx.x - b * a.heads;
  const int col = threadIdx.x % kCols, part = threadIdx.x / kCols;
  __bf16 *out = a.out + b * a.so + (int64_t)head * a.ho;
  Line line;
  line.make(a, lane);
  const int n = a.lengths[b], tiles = Line::tiles_of(a, n);
  if (tiles == 0) {
    const uint32_t v = n > 0 ? 0x7FC07FC0u : 0u;  // tokens, but a table without pages: NaN
    if (part == 0) *reinterpret_cast<uint2 *>(out + 4 * col) = make_uint2(v, v);
    return;
  }
  while (line.c0 + 64 <= b) {
    line.before += lane_of(line.upto, 63);
    line.c0 += 64;
    line.load(a, lane);
  }
  const int kv = head / a.group, in = head - kv * a.group, nh = min(a.group, kHeads);
  const int u0 = (line.before + lane_of(line.upto, b - line.c0) - tiles) * line.heads + (kv * a.chunks + in / kHeads) * tiles;
  const int u1 = u0 + tiles, run0 = line.run_of(u0), run1 = line.run_of(u1 - 1);
  if (run0 == run1) return;  // stored whole
  // Its records: those of the runs before the first workgroup that is within it,
  // of each such workgroup, and of the runs after.
  int w0 = (run0 + (line.start(run0) < u0) + kWaves - 1) / kWaves;
  int w1 = min(line.runs, run1 + (line.start(run1 + 1) <= u1)) / kWaves;
  if (w1 < w0) w0 = w1 = run1 / kWaves + 1;
  const int before = min(w0 * kWaves, run1 + 1) - run0, groups = w1 - w0;
  const int count = before + groups + max(0, run1 + 1 - max(w1 * kWaves, run0 + before));
  if (groups == 1 && count == 1) return;  // stored whole by that workgroup
  const int64_t stride = (int64_t)nh * (D + 4);
  auto record = [&](int i) {
    const int run = i < before ? run0 + i : i < before + groups ? (w0 + i - before) * kWaves : w1 * kWaves + i - before - groups;
    return a.partial + (2 * run + (line.start(run) < u0)) * stride;
  };
  const int row = in % kHeads;
  float m = -__builtin_inff(), l = 0.f;
  f32x4 o{0.f, 0.f, 0.f, 0.f};
  for (int i = part; i < count; i += kLanes * kBatch) {
    f32x4 v[kBatch];
    float2 ml[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const float *rec = record(min(i + k * kLanes, count - 1));
      v[k] = *reinterpret_cast<const f32x4 *>(rec + row * D + 4 * col);
      ml[k] = *reinterpret_cast<const float2 *>(rec + nh * D + 2 * row);
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      if (i + k * kLanes >= count) break;
      const float top = __builtin_fmaxf(m, ml[k].x);
      const float f = m == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(m - top);
      const float e = ml[k].x == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(ml[k].x - top);
      m = top;
      l = l * f + ml[k].y * e;
#pragma unroll
      for (int c = 0; c < 4; ++c) o[c] = o[c] * f + v[k][c] * e;
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) red[part][4 * col + i] = o[i];
  if (col == 0) {
    red[part][D] = m;
    red[part][D + 1] = l;
  }
  __syncthreads();
  if (threadIdx.x >= D) return;
  float top = -__builtin_inff();
#pragma unroll
  for (int p = 0; p < kLanes; ++p) top = __builtin_fmaxf(top, red[p][D]);
  float z = 0.f, x = 0.f;
#pragma unroll
  for (int p = 0; p < kLanes; ++p) {
    const float e = red[p][D] == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(red[p][D] - top);
    z += e * red[p][D + 1];
    x += e * red[p][threadIdx.x];
  }
  out[threadIdx.x] = (__bf16)(x / z);
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
int invalid(const char *msg) { return set_error(MQ_E_INVALID, msg); }

int chunks_of(int heads, int kv_heads) { return (heads / kv_heads + kHeads - 1) / kHeads; }

// (sequence, head unit) pairs.
int64_t pairs_of(const mq_kv_cache *c, int64_t batch, int heads) { return batch * c->kv_heads * chunks_of(heads, c->kv_heads); }

// Waves of a workgroup that takes a whole pair, 0 where waves take runs of the line: by
// the tiles that a page table can hold, which is all the host knows of the lengths.  One
// launch, but the longest pair sets its end, so up to 32 tiles, and 64 where many pairs
// follow each other on every CU.  us, line and pairs, 32 / 8 heads of 128, up to 1900
// tokens: 256 sequences 203, 185 (Q8_0, equal), 148, 135 (BF16, ragged); 128 112, 100
// and 79, 81; 64 57.9, 52.3 and 26.3, 32.3 (Q8_0, ragged).  Eight waves a pair while a
// CU has not more than two pairs, then four, of which three fit: us with 8 and 4, up to
// 900 tokens, 16 sequences 12.6, 14.0; 64 30.9, 28.0; 256 112, 97.
int pair_waves(const mq_kv_cache *c, int64_t pairs, int64_t max_pages) {
  if (max_pages * (c->page_tokens / kTileTokens) > (pairs < 1024 ? 32 : 64)) return 0;
  return pairs < 512 ? 8 : 4;
}

// Waves of the largest launch: what the registers allow, 16 a CU with heads of 64 and 12
// with 128, or 8 where each has over 8 KiB in flight.  us with 8, 12 and 16 a CU: 64 x
// 8192 tokens, 32 / 8 heads of 128 in BF16 358, 371, Q8_0 210, 219, Q4_0 147, 143; heads
// of 64, 32 x 8192 x 32 in Q8_0 206, 208, 201, Q4_0 181, 158, 148, BF16 373, 382, 383; 16
// ragged ones up to 3500 x 20 in Q4_0 17.0, 16.2, 15.6, BF16 23.6, 22.4, 22.1.
int most_waves(const mq_kv_cache *c) {
  return c->head_dim == 64 ? 4096 : cache_tile_bytes(c->dtype, c->head_dim) > 8192 ? 2048 : 3072;
}

// Waves of a launch over `batch` sequences of up to `max_pages` pages: a run each, and no
// more than the tiles there can be.
int waves_of(const mq_kv_cache *c, int64_t batch, int chunks, int64_t max_pages) {
  const int64_t units = batch * c->kv_heads * chunks * (max_pages * (c->page_tokens / kTileTokens));
  const int64_t w = (units + kWaves - 1) / kWaves * kWaves, most = most_waves(c);
  return (int)(w < most ? w : most);
}

}  // namespace
}  // namespace mq

extern "C" size_t mq_cache_attention_scratch_size(const mq_kv_cache *c, int64_t batch, int heads, int64_t max_pages) {
  using namespace mq;
  if (cache_fault(c) || batch <= 0 || heads < 1 || heads % c->kv_heads || max_pages <= 0 ||
      pair_waves(c, pairs_of(c, batch, heads), max_pages))
    return 0;
  const int group = heads / c->kv_heads;
  return (size_t)2 * waves_of(c, batch, chunks_of(heads, c->kv_heads), max_pages) *
         (group < kHeads ? group : kHeads) * (c->head_dim + 4) * sizeof(float);
}

extern "C" int mq_cache_attention(const mq_kv_cache *c, const void *q, int64_t q_batch_stride, int64_t q_head_stride,
                                  int64_t batch, int heads, const int32_t *page_table, int64_t table_stride,
                                  int64_t max_pages, const int32_t *lengths, float scale, void *out,
                                  int64_t out_batch_stride, int64_t out_head_stride, void *scratch, size_t scratch_bytes,
                                  void *stream) {
  using namespace mq;
  if (const char *fault = cache_fault(c)) return invalid(fault);
  if (batch < 0 || heads < 1 || heads > 65536 || heads % c->kv_heads)
    return invalid("mq_cache_attention: negative batch, or heads not a multiple of the cache's");
  if (!takes_scale(scale)) return invalid("mq_cache_attention: scale must be positive, and finite times log2(e)");
  if (max_pages < 0 || max_pages >= (int64_t(1) << 31) || max_pages * c->page_tokens >= (int64_t(1) << 31))
    return invalid("mq_cache_attention: a page table of 0 to 2^31 tokens");
  if (batch == 0) return MQ_OK;
  if (!q || !out || !lengths || (max_pages && (!page_table || !c->data || c->pages == 0)))
    return invalid("mq_cache_attention: NULL pointer, or a cache without pages");
  const int chunks = chunks_of(heads, c->kv_heads);
  if (batch >= (int64_t(1) << 31) / heads ||
      batch * c->kv_heads * chunks >= (int64_t(1) << 31) / (max_pages * (c->page_tokens / kTileTokens) + 1))
    return invalid("mq_cache_attention: 2^31 rows or tiles");
  for (int64_t s : {q_batch_stride, q_head_stride, out_batch_stride, out_head_stride})
    if (s < 0 || s % 8) return invalid("mq_cache_attention: strides must be multiples of 8 elements, none negative");
  if (table_stride < 0 || (batch > 1 && table_stride < max_pages))
    return invalid("mq_cache_attention: table_stride below max_pages");
  if (!aligned16(c->data) || !aligned16(q) || !aligned16(out) || !aligned16(scratch) ||
      (reinterpret_cast<uintptr_t>(page_table) & 3) || (reinterpret_cast<uintptr_t>(lengths) & 3))
    return invalid("mq_cache_attention: buffers must be 16-byte aligned");
  const int dim = c->head_dim;
  if ((heads > 1 && out_head_stride < dim) ||
      (batch > 1 && (out_batch_stride < dim || (heads > 1 && out_batch_stride < (heads - 1) * out_head_stride + dim &&
                                                out_head_stride < (batch - 1) * out_batch_stride + dim))))
    return invalid("mq_cache_attention: rows or heads of out overlap");
  const uintptr_t q0 = reinterpret_cast<uintptr_t>(q), o0 = reinterpret_cast<uintptr_t>(out);
  const uintptr_t q1 = q0 + 2 * (uintptr_t)((batch - 1) * q_batch_stride + (heads - 1) * q_head_stride + dim);
  const uintptr_t o1 = o0 + 2 * (uintptr_t)((batch - 1) * out_batch_stride + (heads - 1) * out_head_stride + dim);
  if (q0 < o1 && o0 < q1) return invalid("mq_cache_attention: out lies over q");
  const size_t need = mq_cache_attention_scratch_size(c, batch, heads, max_pages);
  if (need && (!scratch || scratch_bytes < need))
    return invalid("mq_cache_attention: scratch below mq_cache_attention_scratch_size");
  const int waves = waves_of(c, batch, chunks, max_pages);
  const DecodeArgs a{{static_cast<uint8_t *>(c->data), c->pages * c->page_tokens, c->page_tokens, c->kv_heads}, c->pages,
                     static_cast<const __bf16 *>(q), static_cast<__bf16 *>(out), q_batch_stride, q_head_stride,
                     out_batch_stride, out_head_stride, page_table, lengths, table_stride, (int)max_pages, (int)batch,
                     heads, heads / c->kv_heads, chunks, waves, scale * kLog2e, least_score(scale), static_cast<float *>(scratch)};
  hipStream_t s = static_cast<hipStream_t>(stream);
  with_cache_type(c, [&]<int T, int D>() {
    const int64_t pairs = pairs_of(c, batch, heads);
    if (const int w = pair_waves(c, pairs, max_pages)) {
      if (w == 8) hipLaunchKernelGGL((decode_kernel<T, D, 8>), dim3((unsigned)pairs), dim3(64 * 8), 0, s, a);
      else hipLaunchKernelGGL((decode_kernel<T, D, 4>), dim3((unsigned)pairs), dim3(64 * 4), 0, s, a);
    } else {
      hipLaunchKernelGGL((decode_kernel<T, D, 0>), dim3((unsigned)(waves / kWaves)), dim3(64 * kWaves), 0, s, a);
      hipLaunchKernelGGL(join_kernel<D>, dim3((unsigned)(batch * heads)), dim3(256), 0, s, a);
    }
  });
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MQ_OK : set_error(MQ_E_HIP, hipGetErrorString(e));
}
