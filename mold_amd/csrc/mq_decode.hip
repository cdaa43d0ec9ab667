// mq_decode.hip — attention of one new token per sequence over the paged cache:
//   out[b, h] = sum_{t < len_b} p_t v[t, g],  p = softmax_t(scale q[b, h] . k[t, g]),
// g = h / (heads / kv_heads), in one pass over the cache (the decode step of the
// prompt-expansion model, crates/mold-inference/src/expand.rs:200-203).
//
// What bounds it: reading the cache once.  The products of a group's heads (up to
// 16, the other columns of the matrix instruction are zeros) with a tile of 32
// tokens are 16 MFMAs, far from their rate, also after a block type's bytes have
// been widened.  So the kernel is laid out for the loads:
//   * every wave is on its own: no LDS, no barrier.  The work of the whole batch
//     is one line of (sequence, k/v head, tile of 32 tokens), cut into equal runs,
//     one a wave, whatever the lengths are; the lengths stay on the device (each
//     wave adds them up), so the host neither waits nor plans;
//   * a tile is read in the order of the matrix operands (mq_cache.h), 1 KiB a
//     load instruction, two tiles in flight a wave, eight waves a CU;
//   * the scores are computed transposed, S^T = K Q^T, so that a lane's eight
//     probabilities are its B operand of O^T = V^T P^T, as they stand;
//   * whole numbers of the block types are exact in bf16: a key block's scale
//     multiplies its 32 values' dot product in f32, a value block's the
//     probabilities, so that neither K nor V is rounded at all;
//   * the probabilities enter as two bf16 numbers, one near them and what it
//     lacks (relative 2^-16 together): the second product costs matrix time that
//     the loads leave free, and a step of a few tokens, whose roundings do not
//     average out, is as exact as its output's type.
// A run that holds a whole (sequence, head) stores its result; the others store
// f32 sums, which join_kernel adds in the order of the line.
#include "../../include/moldq.h"
#include "mq_cache.h"

namespace mq {
int set_error(int code, const char *msg);
}

namespace mq {
namespace {

constexpr int kWaves = 4;           // of a workgroup
constexpr int kMaxWaves = 2048;     // of a launch: 8 a CU
constexpr int kMinTiles = 1;        // of a run
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
  float *partial;
};

__device__ __forceinline__ int lane_of(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }

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
  int tiles, upto;     // this lane's: its tiles, the tiles of c0 .. its own
  int total, heads;    // tiles of all sequences, head units
  int runs, base, rest;  // runs, their least length, how many are one longer

  __device__ static int tiles_of(const DecodeArgs &a, int b) {
    if (b >= a.batch) return 0;
    const int64_t cap = (int64_t)a.max_pages * a.cache.page_tokens;
    const int64_t n = a.lengths[b];
    return n <= 0 ? 0 : (int)(((n < cap ? n : cap) + kTileTokens - 1) / kTileTokens);
  }
  __device__ void load(const DecodeArgs &a, int lane) {
    tiles = tiles_of(a, c0 + lane);
    upto = scan64(tiles);
  }
  __device__ Line(const DecodeArgs &a, int lane) : c0(0), before(0), total(0), heads(a.cache.kv_heads * a.chunks) {
    for (int c = (a.batch - 1) & ~63; c >= 0; c -= 64) {  // the first 64 last: they stay
      c0 = c;
      load(a, lane);
      total += lane_of(upto, 63);
    }
    const int units = total * heads;
    runs = min(a.waves, units / kMinTiles);
    runs = max(runs, 1);
    base = units / runs;
    rest = units - base * runs;
  }
  __device__ int start(int run) const { return run * base + min(run, rest); }
  __device__ int run_of(int unit) const {
    const int longer = rest * (base + 1);
    return unit < longer ? unit / (base + 1) : rest + (unit - longer) / base;
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

  __device__ __forceinline__ static void get16(uint32_t *to, const uint8_t *p) {
    const uint4 u = *reinterpret_cast<const uint4 *>(p);
    to[0] = u.x; to[1] = u.y; to[2] = u.z; to[3] = u.w;
  }
  __device__ __forceinline__ void load(const uint8_t *tile, int lane) {
    if constexpr (L::kKeyPiece == 16) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < kKeyWords; i += 4) get16(&k[u][i], tile + u * 64 * L::kKeyLane + i * 256 + lane * 16);
    } else {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint2 w = *reinterpret_cast<const uint2 *>(tile + u * 64 * L::kKeyLane + lane * 8);
        k[u][0] = w.x;
        k[u][1] = w.y;
      }
    }
#pragma unroll
    for (int i = 0; i < 2 * kKeyWords; i += 4) get16(&v[i], tile + L::kPlane + i * 256 + lane * 16);
    if constexpr (L::kQuant) {
      const uint8_t *s = tile + 2 * L::kPlane + (lane >> 4) * (16 * L::kBlocks);
#pragma unroll
      for (int i = 0; i < kScaleWords; i += 4) {
        get16(&ks[i], s + 4 * i);
        get16(&vs[i], s + L::kScales + 4 * i);
      }
    }
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
// eight bytes as signed whole numbers, exact in bf16
__device__ __forceinline__ bf16x8 bytes8(const uint32_t *w) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    u[i] = pack2((float)(int8_t)(w[i >> 1] >> (16 * (i & 1))), (float)(int8_t)(w[i >> 1] >> (16 * (i & 1) + 8)));
  return operand(u);
}
// the low or high nibbles of bytes as whole numbers -8 .. 7, two a word of the operand
__device__ __forceinline__ void nibbles4(uint32_t w, uint32_t *u) {
  const uint32_t n = w & 0x0F0F0F0Fu;
  u[0] = pack2((float)(n & 0xFF) - 8.f, (float)((n >> 8) & 0xFF) - 8.f);
  u[1] = pack2((float)((n >> 16) & 0xFF) - 8.f, (float)(n >> 24) - 8.f);
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

template <int T, int D>
__global__ __launch_bounds__(64 * kWaves, 2) void decode_kernel(const DecodeArgs a) {
  using L = CacheTile<T, D>;
  constexpr int kB = L::kBlocks, kC = D / 16;
  const int lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
  const int run = __builtin_amdgcn_readfirstlane(blockIdx.x * kWaves + (threadIdx.x >> 6));
  Line line(a, lane);
  if (line.total == 0 || run >= line.runs) return;
  const int first = line.start(run), end = line.start(run + 1);
  const int tpp = a.cache.page_tokens / kTileTokens;

  // The unit whose tile is loaded next.
  struct Unit {
    int at, b, kv, chunk, t, tiles;  // place on the line, sequence, k/v head, chunk of its heads, tile of the sequence's tiles
    bool bad;                   // its page is not one of the cache's
  };
  int idx = line.seek(a, lane, first);  // its sequence's lane
  Unit nx;
  {
    const int tiles = lane_of(line.tiles, idx), in = first - (line.before + lane_of(line.upto, idx) - tiles) * line.heads;
    const int head = in / tiles;
    nx = Unit{first, line.c0 + idx, head / a.chunks, head % a.chunks, in - head * tiles, tiles, false};
  }
  // its sequence's page numbers page0 .. page0 + 63, one a lane
  int page0 = nx.t / tpp, page = page0, in_page = nx.t % tpp, numbers = 0;
  auto number_pages = [&]() {
    numbers = page0 + lane < a.max_pages ? a.table[nx.b * a.table_stride + page0 + lane] : 0;
  };
  number_pages();
  auto fetch = [&](Tile<T, D> &to) {
    const uint32_t id = (uint32_t)lane_of(numbers, page - page0);
    nx.bad = id >= a.pages;
    const int64_t at = ((int64_t)(nx.bad ? 0 : id) * a.cache.kv_heads + nx.kv) * tpp + in_page;
    to.load(a.cache.data + at * L::kBytes, lane);
  };
  auto advance = [&]() {  // to the run's next unit; past its last the tile stays where it is
    if (nx.at + 1 >= end) return;
    ++nx.at;
    if (++nx.t < nx.tiles) {
      if (++in_page == tpp) {
        in_page = 0;
        if (++page == page0 + 64) {
          page0 = page;
          number_pages();
        }
      }
      return;
    }
    nx.t = 0;
    if (++nx.chunk == a.chunks) {
      nx.chunk = 0;
      ++nx.kv;
    }
    if (nx.kv == a.cache.kv_heads) {
      nx.kv = 0;
      uint64_t more = __ballot(line.tiles > 0) & ~((2ull << idx) - 1);
      while (more == 0) {
        line.before += lane_of(line.upto, 63);
        line.c0 += 64;
        line.load(a, lane);
        more = __ballot(line.tiles > 0);
      }
      idx = __builtin_ctzll(more);
      nx.b = line.c0 + idx;
      nx.tiles = lane_of(line.tiles, idx);
    }
    page0 = page = in_page = 0;
    number_pages();
  };

  bf16x8 qf[kB];
  f32x4 o[kC];  // O^T: this lane's head, columns 16 c + 4 g + 0..3
  float m, l;
  bool bad = false;
  auto begin = [&](const Unit &u) {
    const int in = u.chunk * kHeads + r;
    const __bf16 *p = a.q + u.b * a.sq + (int64_t)(u.kv * a.group + (in < a.group ? in : 0)) * a.hq;
#pragma unroll
    for (int b = 0; b < kB; ++b) {
      uint32_t w[4];
      if constexpr (T == Q4_0) {
        const uint2 lo = *reinterpret_cast<const uint2 *>(p + 32 * b + 4 * g), hi = *reinterpret_cast<const uint2 *>(p + 32 * b + 16 + 4 * g);
        w[0] = lo.x; w[1] = lo.y; w[2] = hi.x; w[3] = hi.y;
      } else {
        const uint4 x = *reinterpret_cast<const uint4 *>(p + 32 * b + 8 * g);
        w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = in < a.group ? w[i] : 0u;
      qf[b] = operand(w);
    }
#pragma unroll
    for (int c = 0; c < kC; ++c) o[c] = f32x4{0.f, 0.f, 0.f, 0.f};
    m = -__FLT_MAX__;
    l = 0.f;
    bad = false;
  };

  auto compute = [&](Tile<T, D> &x, const Unit &u) {
    f32x4 s[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      s[h] = f32x4{0.f, 0.f, 0.f, 0.f};
      if constexpr (T == BF16) {
#pragma unroll
        for (int b = 0; b < kB; ++b) s[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(operand(&x.k[h][4 * b]), qf[b], s[h], 0, 0, 0);
      } else {
#pragma unroll
        for (int b = 0; b < kB; ++b) {
          bf16x8 k;
          if constexpr (T == Q8_0) {
            k = bytes8(&x.k[h][2 * b]);
          } else {
            uint32_t w[4];
            nibbles4(x.k[h][b], w);
            nibbles4(x.k[h][b] >> 4, w + 2);
            k = operand(w);
          }
          const f32x4 dot = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, qf[b], f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
          for (int i = 0; i < 4; ++i) s[h][i] = __builtin_fmaf(half_of(x.ks, (h * kB + b) * 4 + i), dot[i], s[h][i]);
        }
      }
    }
    if (u.t + 1 == u.tiles) {  // tokens past the sequence's last: no weight, and no value or scale that could make 0 x NaN
      const int over = min(a.lengths[u.b], a.max_pages * a.cache.page_tokens) - (u.tiles - 1) * kTileTokens;
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
        float pd[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) pd[j] = p[j] * half_of(&x.vs[4 * b], j);
        const Split w = split8(pd);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if constexpr (T == Q8_0) {
            add(o[2 * b + c], bytes8(&x.v[4 * b + 2 * c]), w);
          } else {
            uint32_t v[4];
            nibbles4(x.v[2 * b] >> (4 * c), v);
            nibbles4(x.v[2 * b + 1] >> (4 * c), v + 2);
            add(o[2 * b + c], operand(v), w);
          }
        }
      }
    }
    bad |= u.bad;
  };
  // the end of the run or of a (sequence, head)
  const int nh = min(a.group, kHeads);
  auto finish = [&](const Unit &u, int from) {
    if (bad || a.lengths[u.b] > (int64_t)a.max_pages * a.cache.page_tokens) l = __builtin_nanf("");
    l = column_add(l);
    const int in = u.chunk * kHeads + r;
    if (in >= a.group) return;
    if (u.t + 1 == u.tiles && u.at - from + 1 == u.tiles) {
      const float inv = 1.f / l;
      __bf16 *p = a.out + u.b * a.so + (int64_t)(u.kv * a.group + in) * a.ho + 4 * g;
#pragma unroll
      for (int c = 0; c < kC; ++c)
        *reinterpret_cast<uint2 *>(p + 16 * c) = make_uint2(pack2(o[c][0] * inv, o[c][1] * inv), pack2(o[c][2] * inv, o[c][3] * inv));
      return;
    }
    float *rec = a.partial + (int64_t)(2 * run + (from != first)) * nh * (D + 4);
#pragma unroll
    for (int c = 0; c < kC; ++c)
      *reinterpret_cast<f32x4 *>(rec + r * D + 16 * c + 4 * g) = o[c];
    if (g == 0) *reinterpret_cast<float2 *>(rec + nh * D + 2 * r) = make_float2(m * a.scale, l);
  };

  int from = first;  // where the (sequence, head) at hand began in this run
  Unit cu = nx;
  Tile<T, D> t0, t1;
  fetch(t0);
  cu.bad = nx.bad;
  begin(cu);
  // one unit: the next one's tile is requested, this one's taken in
  auto step = [&](Tile<T, D> &now, Tile<T, D> &then) {
    advance();
    fetch(then);
    compute(now, cu);
    const bool over = cu.at + 1 == end;
    if (over || cu.t + 1 == cu.tiles) {
      finish(cu, from);
      if (over) return false;
      from = nx.at;
      cu = nx;
      begin(cu);
    } else {
      cu = nx;
    }
    return true;
  };
  while (step(t0, t1) && step(t1, t0)) {
  }
}

// A row's shares, added in the order of the line, each relative to its own
// maximum; zeros for a sequence without tokens.  A workgroup a row: D / 4 threads
// take 4 columns of every kLanes-th share.
template <int D>
__global__ __launch_bounds__(256) void join_kernel(const DecodeArgs a) {
  constexpr int kCols = D / 4, kLanes = 256 / kCols;
  __shared__ float red[kLanes][D + 2];
  const int lane = threadIdx.x & 63;
  const int b = blockIdx.x / a.heads, head = blockIdx.x - b * a.heads;
  const int col = threadIdx.x % kCols, part = threadIdx.x / kCols;
  __bf16 *out = a.out + b * a.so + (int64_t)head * a.ho;
  Line line(a, lane);
  const int tiles = Line::tiles_of(a, b);
  if (tiles == 0) {
    const uint32_t v = a.lengths[b] > 0 ? 0x7FC07FC0u : 0u;  // tokens, but a table without pages
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
  const int run0 = line.run_of(u0), run1 = line.run_of(u0 + tiles - 1);
  if (run0 == run1) return;  // stored whole
  const int64_t stride = (int64_t)nh * (D + 4);
  auto record = [&](int run) { return a.partial + (2 * run + (line.start(run) < u0)) * stride; };
  const int row = in % kHeads;
  float m = -__builtin_inff(), l = 0.f;
  f32x4 o{0.f, 0.f, 0.f, 0.f};
  for (int run = run0 + part; run <= run1; run += kLanes) {
    const float *rec = record(run);
    const f32x4 v = *reinterpret_cast<const f32x4 *>(rec + row * D + 4 * col);
    const float2 ml = *reinterpret_cast<const float2 *>(rec + nh * D + 2 * row);
    const float top = __builtin_fmaxf(m, ml.x);
    const float f = m == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(m - top);
    const float e = ml.x == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(ml.x - top);
    m = top;
    l = l * f + ml.y * e;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = o[i] * f + v[i] * e;
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

// Waves of a launch over `batch` sequences of up to `tokens` tokens: a run each, and no more than the tiles there can be.
int waves_of(int64_t batch, int kv_heads, int chunks, int64_t tokens) {
  const int64_t units = batch * kv_heads * chunks * ((tokens + kTileTokens - 1) / kTileTokens);
  const int64_t w = (units + kWaves - 1) / kWaves * kWaves;
  return (int)(w < kMaxWaves ? w : kMaxWaves);
}

}  // namespace
}  // namespace mq

extern "C" size_t mq_cache_attention_scratch_size(const mq_kv_cache *c, int64_t batch, int heads, int64_t max_pages) {
  using namespace mq;
  if (cache_fault(c) || batch <= 0 || heads < 1 || heads % c->kv_heads || max_pages <= 0) return 0;
  const int group = heads / c->kv_heads;
  return (size_t)2 * waves_of(batch, c->kv_heads, chunks_of(heads, c->kv_heads), max_pages * c->page_tokens) *
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
  if (!(scale > 0.f) || scale > 3e38f) return invalid("mq_cache_attention: scale must be positive and finite");
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
  if (scratch_bytes < mq_cache_attention_scratch_size(c, batch, heads, max_pages) || (max_pages && !scratch))
    return invalid("mq_cache_attention: scratch below mq_cache_attention_scratch_size");
  const int waves = waves_of(batch, c->kv_heads, chunks, max_pages * c->page_tokens);
  const DecodeArgs a{{static_cast<uint8_t *>(c->data), c->pages * c->page_tokens, c->page_tokens, c->kv_heads}, c->pages,
                     static_cast<const __bf16 *>(q), static_cast<__bf16 *>(out), q_batch_stride, q_head_stride,
                     out_batch_stride, out_head_stride, page_table, lengths, table_stride, (int)max_pages, (int)batch,
                     heads, heads / c->kv_heads, chunks, waves, scale * 1.44269504f, static_cast<float *>(scratch)};
  hipStream_t s = static_cast<hipStream_t>(stream);
  with_cache_type(c, [&]<int T, int D>() {
    if (waves) hipLaunchKernelGGL((decode_kernel<T, D>), dim3((unsigned)(waves / kWaves)), dim3(64 * kWaves), 0, s, a);
    hipLaunchKernelGGL(join_kernel<D>, dim3((unsigned)(batch * heads)), dim3(256), 0, s, a);
  });
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MQ_OK : set_error(MQ_E_HIP, hipGetErrorString(e));
}
