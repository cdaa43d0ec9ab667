// mq_prompt.hip — causal attention of whole prompts: packed sequences of
// different lengths, grouped heads, what a decoder's layer runs between its
// projections, or an encoder's that is one (the Qwen text encoders,
// crates/mold-inference/src/encoders/qwen3_gguf.rs and qwen2_text_gguf.rs, and the
// prompt-expansion model, src/expand.rs:200-203; T5 attends both ways, with a bias).
//
//   out[i, h] = sum_{j <= i} p_ij v[j, g],  p_i = softmax_j(scale q[i, h] . k[j, g]),
//
// i, j inside one prompt and g = h / (heads / kv_heads), in one pass over the
// keys with a running maximum and sum of the softmax (f32).
//
// The wave's inner loop is the joint attention's: transposed scores S^T = K Q^T
// (v_mfma_f32_32x32x16, a lane holds 16 keys of one query), probabilities as the
// B operand of O^T = V^T P^T in place, K and V blocks of 64 keys by LDS DMA one
// block ahead, V read transposed from LDS, the scores half a block ahead of the
// softmax.  What is different here:
//   * a workgroup's waves take 32 tokens of several heads of one group where the
//     group has them (4 heads x 32 tokens; 2 x 64; 1 x 128), so that they share
//     the K and V blocks and end at the same diagonal: with 128 tokens of one
//     head the first wave would wait through three half blocks of 32 keys that
//     it masks whole;
//   * a wave computes the 32-key halves up to its own diagonal and no further,
//     and masks the diagonal one alone;
//   * tiles run longest first (the list the host makes of the packed prompts),
//     so that the short ones fill the launch's end;
//   * a key that a row does not see must not reach it even as 0 x NaN: the
//     diagonal half, the only one that mixes seen and unseen keys, looks for
//     non-finite values among its V and, if there are any, adds them row by row
//     (accumulate_seen).  Rows past a prompt's end are clamped to its last row,
//     so no neighbour in the pack is ever read;
//   * few tiles are split over the keys, two waves a tile (split_tiles below).
// Bound by the matrix cores and the softmax at the clock that the power limit leaves
// where prompts are long (32 / 8 heads of 128: one of 8192 tokens 499 to 544 us by box,
// 1010 to 1102 TFLOP/s of the pairs i >= j, the matrix cores 0.57 busy at 1.8 GHz); by the
// tiles' own costs where they are short: 24 ragged prompts, 7305 tokens, take 62 to 70 us
// (538 to 607), of which storing rows is 13 and reading q 8, as the waves that could hide them are
// few (two a SIMD: O, q and two blocks of scores fill the registers, K and V half the
// LDS).  Workgroups that go on to further tiles with the next one's K, V and q
// requested ahead were 4% slower.
#include "../../include/moldq.h"
#include "mq_attn.h"

#include <algorithm>

namespace mq {
int set_error(int code, const char *msg);
}

namespace mq {
namespace {

constexpr int kKeys = 64;  // keys per block

struct PromptArgs {
  const __bf16 *q, *k, *v;
  __bf16 *out;
  int64_t sq, sk, sv, so;  // token strides
  int64_t hq, hk, hv, ho;  // head strides
  const int4 *tiles;       // first row of the prompt, its length, first token of the tile, 0
  int64_t total;           // rows of q
  int units, group, log_heads;  // head units (of 1 << log_heads heads), heads per k/v head
  float scale;             // times log2(e)
  float least;             // what the running maximum starts at (least_score)
};

template <int S>
struct Slot {
  static constexpr int v = S;
};

// The largest magnitudes, as bit patterns, of the even and of the odd values: from
// 0x7F80 on one is not finite.
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void raise_magnitudes(u16x2 &most, const uint4 &u) {
  for (const uint32_t two : {u.x, u.y, u.z, u.w}) {
    const uint32_t bits = two & 0x7FFF7FFFu;
    u16x2 x;
    __builtin_memcpy(&x, &bits, 4);
    most = __builtin_elementwise_max(most, x);
  }
}

// W waves of 32 queries each; with P = 2 two waves share their queries and take
// every other 32 keys each.
template <int D, int W, int P>
__global__ __launch_bounds__(64 * W, D == 128 ? 2 : 3) void prompt_kernel(const PromptArgs a) {
  constexpr int kRow = 2 * D;              // bytes of a row in LDS
  constexpr int kBlock = kKeys * kRow;     // of a block
  constexpr int kChunks = kRow / 16;       // 16-byte chunks of a row
  constexpr int kDmaRows = 1024 / kRow;    // rows a wave's DMA instruction fills
  constexpr int kDmas = kKeys / kDmaRows / W;
  __shared__ uint4 lds[5 * kBlock / 16];  // K blocks 0 and 1, V blocks 0 to 2
  uint4 *const lds_k = lds, *const lds_v = lds + 2 * kBlock / 16;

  const int4 tile = a.tiles[blockIdx.x / a.units];
  const int unit = blockIdx.x % a.units;
  const int len = tile.y, first = tile.z;
  // a list that does not belong to these rows: nothing is read or stored
  if (tile.x < 0 || len <= 0 || first < 0 || first >= len || (int64_t)tile.x + len > a.total) return;

  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int slot = wave / P, part = P == 1 ? 0 : wave % P;  // which 32 queries, which keys of theirs
  const int head = (unit << a.log_heads) + (slot & ((1 << a.log_heads) - 1));
  const int tok0 = first + 32 * (slot >> a.log_heads);
  const int end = min(first + ((32 * W / P) >> a.log_heads), len);  // past the tile's last token
  const int nblk = (end + kKeys - 1) / kKeys;
  const int halves = tok0 < len ? tok0 / 32 + 1 : 0;  // 32-key halves these queries see; the last is their diagonal
  const int row = tok0 + l32;                         // this lane's query
  const int64_t kvhead = (unit << a.log_heads) / a.group;

  bf16x8 qf[D / 16];  // the B operand of the scores; rows past the prompt's end repeat its last and are not stored
  {
    const __bf16 *p = a.q + (tile.x + (int64_t)min(row, len - 1)) * a.sq + head * a.hq + 8 * h;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) qf[s] = *reinterpret_cast<const bf16x8 *>(p + 16 * s);
  }

  // DMA of a block: load j of a wave fills LDS rows kDmaRows (wave + W j) + 0 ..,
  // each lane fetching the chunk that the swizzle puts in its slot.  The swizzles
  // keep 16 rows' reads of one K chunk, and 4 rows' of one V segment, on
  // different banks.
  const int drow = kDmaRows * wave + lane / kChunks, dch = lane % kChunks;
  const int dk = D == 128 ? drow & 15 : (drow >> 1) & 7, dv = D == 128 ? drow & 3 : (drow >> 1) & 1;
  const uint32_t kch = (uint32_t)((dch ^ dk) << 4), vch = (uint32_t)((dch ^ (dv << 2)) << 4);
  const uint32_t lkw = (uint32_t)(uintptr_t)(lds_k) + 1024 * wave;
  const uint32_t lvw = (uint32_t)(uintptr_t)(lds_v) + 1024 * wave;
  const char *kbase = reinterpret_cast<const char *>(a.k + tile.x * a.sk + kvhead * a.hk);
  const char *vbase = reinterpret_cast<const char *>(a.v + tile.x * a.sv + kvhead * a.hv);
  const uint32_t kstep = (uint32_t)(2 * a.sk), vstep = (uint32_t)(2 * a.sv);
  auto dma = [&](int blk, int kslot, int vslot) {
    const char *kb = kbase + (int64_t)blk * (2 * kKeys) * a.sk, *vb = vbase + (int64_t)blk * (2 * kKeys) * a.sv;
    const int top = len - 1 - blk * kKeys;
#pragma unroll
    for (int j = 0; j < kDmas; ++j) {
      const uint32_t r = (uint32_t)min(drow + kDmaRows * W * j, top);
      dma16(kb, r * kstep + kch, __builtin_amdgcn_readfirstlane(lkw + kslot * kBlock + 1024 * W * j));
      dma16(vb, r * vstep + vch, __builtin_amdgcn_readfirstlane(lvw + vslot * kBlock + 1024 * W * j));
    }
  };

  f32x16 o[D / 32];  // O^T: this lane's query, columns 32 d + 8 (e / 4) + 4 h + e % 4
#pragma unroll
  for (int d = 0; d < D / 32; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
  float m = a.least, bar = m, l = 0.f;  // running maximum (both halves) and this half's sum

  const int i16 = lane & 15;
  lds_char *ka[D / 16], *va[D / 32];
  {
    const int fk = D == 128 ? l32 & 15 : (l32 >> 1) & 7, fv = D == 128 ? i16 >> 2 : i16 >> 3;
#pragma unroll
    for (int s = 0; s < D / 16; ++s)
      ka[s] = (lds_char *)lds_k + (uint32_t)((32 * part + l32) * kRow + (((2 * s + h) ^ fk) << 4));
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
      va[d] = (lds_char *)lds_v +
              (uint32_t)((32 * part + 4 * h + (i16 >> 2)) * kRow + ((d ^ fv) << 6) + 32 * ((lane >> 4) & 1) + 8 * (i16 & 3));
  }

  // scores of keys 32 kb .. + 31 of the block in K slot `slot`: lane l32's
  // query, keys 8 (e / 4) + 4 h + e % 4
  auto scores = [&](int slot, int kb, f32x16 &s) {
#pragma unroll
    for (int e = 0; e < 16; ++e) s[e] = 0.f;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      const bf16x8 x = *(__attribute__((address_space(3))) bf16x8 *)(ka[i] + slot * kBlock + kb * (kBlock / 2));
      s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, qf[i], s, 0, 0, 0);
    }
  };
  // a half of which row l32 sees the keys 0 .. seen (l32 on the diagonal, 31 of any
  // half before it)
  auto mask = [&](f32x16 &s, int seen) {
#pragma unroll
    for (int e = 0; e < 16; ++e)
      if (8 * (e >> 2) + 4 * h + (e & 3) > seen) s[e] = -__builtin_inff();
  };
  auto max16 = [&](const f32x16 &s) {
    float r = s[0];
#pragma unroll
    for (int e = 1; e < 16; ++e) r = __builtin_fmaxf(r, s[e]);
    return r;
  };
  // The maximum follows only where a score passes it by 2^8 and more, row by row (what a
  // row adds up does not depend on the others): O is then rescaled in few of the halves.
  // Probabilities reach 2^8 instead of 1, whose bf16 rounding is as large relative to them;
  // only the largest is no longer exact.  Distance to 64 bits 0.0018 to 0.0019 with every
  // step followed, 0.0018 to 0.0022 so (the result's own rounding alone is 0.0016); 8192
  // tokens 549 -> 511 us, 24 ragged prompts 67.1 -> 64.5, 8 x 1000 x 12 heads of 64 26.9 -> 24.6.
  auto raise_max = [&](float mx) {
    if (__any(mx > bar)) {  // mx: this half's; the row's is looked up only here
      mx = half_max(mx);
      const float mn = mx > bar ? mx : m;
      const float f = __builtin_amdgcn_exp2f((m - mn) * a.scale);
      m = mn;
      bar = mn + 8.f / a.scale;
      l *= f;
#pragma unroll
      for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] *= f;
    }
  };
  // probabilities 2^(scale (s - m)): summed in f32, rounded once to bf16, the
  // matrix operand's type, in its order (relative 2^-9 each, independent from
  // key to key)
  auto probs = [&](const f32x16 &s, bf16x8 *p) {
    const float ms = m * a.scale;
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      uint32_t u[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[8 * t + 2 * i], a.scale, -ms));
        const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[8 * t + 2 * i + 1], a.scale, -ms));
        sum[t] += x + y;
        u[i] = pack2(x, y);
      }
      __builtin_memcpy(&p[t], u, 16);
    }
    l += sum[0] + sum[1];
  };
  // V^T of keys 32 kb + 16 t .. + 15, columns 32 d .. + 31: the A operand, its
  // key order the probabilities' (4 h + 0..3 and 8 + 4 h + 0..3 of each 16)
  auto values = [&](int slot, int kb, int t, int d) {
    s16x4 x[2];
#pragma unroll
    for (int j = 0; j < 2; ++j)
      x[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) s16x4 *)(va[d] + slot * kBlock + (2 * kb + t) * (16 * kRow) + j * (8 * kRow)));
    uint4 u;
    __builtin_memcpy(&u, x, 16);
    return u;
  };
  auto as_bf16 = [](const uint4 &u) {
    bf16x8 x;
    __builtin_memcpy(&x, &u, 16);
    return x;
  };
  auto accumulate = [&](int slot, int kb, const bf16x8 *p) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int d = 0; d < D / 32; ++d)
        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16(values(slot, kb, t, d)), p[t], o[d], 0, 0, 0);
  };
  // The diagonal half, whose V holds a value that is not finite: the finite
  // values by their probabilities as ever, and for each row the infinities and
  // NaN (which count as both) that it sees, counted by products with its mask.
  auto accumulate_seen = [&](int slot, int kb, int last, const bf16x8 *p) {
    bf16x8 seen[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      uint32_t u[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = 16 * t + 8 * (i >> 1) + 4 * h + 2 * (i & 1);
        u[i] = (key <= last ? 0x3F80u : 0u) | (key + 1 <= last ? 0x3F800000u : 0u);
      }
      __builtin_memcpy(&seen[t], u, 16);
    }
    // pass by pass and one tile of columns at a time, each reading V anew: together
    // they would spill
    auto classes = [&](int t, int d, auto pick) {
      asm volatile("" ::: "memory");
      const uint4 v4 = values(slot, kb, t, d);
      const uint32_t w[4] = {v4.x, v4.y, v4.z, v4.w};
      uint32_t u[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) u[i] = pick(w[i] & 0xFFFFu) | pick(w[i] >> 16) << 16;
      return as_bf16(make_uint4(u[0], u[1], u[2], u[3]));
    };
    auto finite = [](uint32_t x) { return (x & 0x7F80u) != 0x7F80u; };
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int t = 0; t < 2; ++t)
        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(classes(t, d, [&](uint32_t x) { return finite(x) ? x : 0u; }), p[t], o[d], 0, 0, 0);
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (uint32_t sign = 0; sign <= 0x8000u; sign += 0x8000u) {
        f32x16 count;
#pragma unroll
        for (int e = 0; e < 16; ++e) count[e] = 0.f;
#pragma unroll
        for (int t = 0; t < 2; ++t)
          count = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
              classes(t, d, [&](uint32_t x) { return !finite(x) && ((x & 0x7Fu) || (x & 0x8000u) == sign) ? 0x3F80u : 0u; }), seen[t], count,
              0, 0, 0);
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (count[e] > 0.f) o[d][e] += sign ? -__builtin_inff() : __builtin_inff();
        __builtin_amdgcn_sched_barrier(0);
      }
  };
  auto diagonal = [&](int slot, int kb, int last, f32x16 &s) {
    bf16x8 p[2];
    mask(s, last);
    raise_max(max16(s));
    probs(s, p);
    u16x2 most{0, 0};
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int d = 0; d < D / 32; ++d) raise_magnitudes(most, values(slot, kb, t, d));
    if (__any(max(most[0], most[1]) >= 0x7F80)) accumulate_seen(slot, kb, last, p);
    else accumulate(slot, kb, p);
  };

  dma(0, 0, 0);
  block_barrier();
  if (nblk > 1) dma(1, 1, 1);
  f32x16 s0, s1;
  if (halves > part) scores(0, 0, s0);
  int vs = 0;  // V slot of block i
  // The barrier in the middle of block i says that block i + 1 has landed and
  // that every wave has read all of K(i) and V(i - 1), whose slots block i + 2
  // then takes.  Waves pass it wherever they are: past their diagonal they only
  // fetch for the others.
  auto turn = [&](int i, int ks) {
    if (i + 1 < nblk) {
      block_barrier();
      if (i + 2 < nblk) dma(i + 2, ks, vs == 0 ? 2 : vs - 1);
    }
  };
  int i = 0;
  if constexpr (P == 1) {
    // a block whose keys are all seen and that is not the wave's last; its first half's scores are in s0
    auto full = [&](int i, auto kslot) {
      constexpr int ks = decltype(kslot)::v;
      bf16x8 p[2];
      raise_max(max16(s0));
      scores(ks, 1, s1);
      probs(s0, p);
      accumulate(vs, 0, p);
      const float mx = max16(s1);
      turn(i, ks);
      raise_max(mx);
      scores(ks ^ 1, 0, s0);
      probs(s1, p);
      accumulate(vs, 1, p);
      vs = vs == 2 ? 0 : vs + 1;
    };
    for (; 2 * i + 4 < halves; i += 2) {
      full(i, Slot<0>{});
      full(i + 1, Slot<1>{});
    }
    if (2 * i + 2 < halves) full(i++, Slot<0>{});
    if (halves) {
      const int ks = i & 1, kb = (halves - 1) & 1;
      if (kb) {
        bf16x8 p[2];
        raise_max(max16(s0));
        scores(ks, 1, s1);
        probs(s0, p);
        accumulate(vs, 0, p);
        s0 = s1;
      }
      turn(i, ks);
      diagonal(vs, kb, l32, s0);
      vs = vs == 2 ? 0 : vs + 1;
      ++i;
    }
  } else {
    // one half of each block, its scores in `now`; the next block's, made after the barrier, in `then`
    auto half = [&](int i, auto kslot, f32x16 &now, f32x16 &then) {
      constexpr int ks = decltype(kslot)::v;
      bf16x8 p[2];
      const float mx = max16(now);
      turn(i, ks);
      raise_max(mx);
      scores(ks ^ 1, 0, then);
      probs(now, p);
      accumulate(vs, 0, p);
      vs = vs == 2 ? 0 : vs + 1;
    };
    const int mine = (halves + 1 - part) / 2;  // blocks of which this wave has a half
    for (; i + 2 < mine; i += 2) {
      half(i, Slot<0>{}, s0, s1);
      half(i + 1, Slot<1>{}, s1, s0);
    }
    if (i + 1 < mine) {
      half(i, Slot<0>{}, s0, s1);
      s0 = s1;
      ++i;
    }
    if (mine) {
      turn(i, i & 1);
      diagonal(vs, 0, ((halves - 1) & 1) == part ? l32 : 31, s0);  // the diagonal is one of the two waves'
      vs = vs == 2 ? 0 : vs + 1;
      ++i;
    }
  }
  for (; i < nblk; ++i) {
    turn(i, i & 1);
    vs = vs == 2 ? 0 : vs + 1;
  }

  l = half_add(l);
  constexpr int kKept = D / 32 / P;  // 32-column tiles of O that this wave stores
  if constexpr (P == 2) {
    // the two waves' sums: each gives the other half of its columns, the maximum and the sum
    float *const shared = reinterpret_cast<float *>(lds);
    constexpr int kWave = 64 * (16 * kKept + 2);
    static_assert(W * kWave * 4 <= 5 * kBlock);
    block_barrier();  // every wave has read its last K and V
    float *const give = shared + wave * kWave + lane;
#pragma unroll
    for (int d = 0; d < kKept; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) give[64 * (16 * d + e)] = part ? o[d][e] : o[kKept + d][e];
    give[64 * 16 * kKept] = m;
    give[64 * (16 * kKept + 1)] = l;
    __syncthreads();
    const float *const take = shared + (wave ^ 1) * kWave + lane;
    const float m2 = take[64 * 16 * kKept], top = __builtin_fmaxf(m, m2);
    const float f = __builtin_amdgcn_exp2f((m - top) * a.scale), f2 = __builtin_amdgcn_exp2f((m2 - top) * a.scale);
    l = l * f + take[64 * (16 * kKept + 1)] * f2;
#pragma unroll
    for (int d = 0; d < kKept; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[d][e] = (part ? o[kKept + d][e] : o[d][e]) * f + take[64 * (16 * d + e)] * f2;
  }
  const float inv = 1.f / l;
  const bool stored = row < len;
  __bf16 *orow = a.out + (tile.x + (int64_t)row) * a.so + head * a.ho + 32 * kKept * part;
#pragma unroll
  for (int d = 0; d < kKept; ++d)
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      // columns 32 d + 16 g + 0..15 of this query sit in lanes l32 and l32 + 32
      // by fours; exchanged so that lane half h stores columns 8 h .. 8 h + 7
      const f32x16 &t = o[d];
      const uint32_t a0 = pack2(t[8 * g] * inv, t[8 * g + 1] * inv), a1 = pack2(t[8 * g + 2] * inv, t[8 * g + 3] * inv);
      const uint32_t c0 = pack2(t[8 * g + 4] * inv, t[8 * g + 5] * inv),
                     c1 = pack2(t[8 * g + 6] * inv, t[8 * g + 7] * inv);
      const auto x = __builtin_amdgcn_permlane32_swap(a0, c0, false, false);
      const auto y = __builtin_amdgcn_permlane32_swap(a1, c1, false, false);
      if (stored) *reinterpret_cast<uint4 *>(orow + 32 * d + 16 * g + 8 * h) = make_uint4(x[0], y[0], x[1], y[1]);
    }
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
int invalid(const char *msg) { return set_error(MQ_E_INVALID, msg); }

constexpr int kWaves = 4;

// Heads that a workgroup of `waves` waves takes together: the largest power of
// two that divides the group.
int unit_log(int group, int waves) {
  int n = 0;
  while ((2 << n) <= waves && group % (2 << n) == 0) ++n;
  return n;
}

int tile_tokens(int group, int parts) { return (32 * kWaves / parts) >> unit_log(group, kWaves / parts); }

constexpr int64_t kCus = 256;
// Workgroups that the chip holds at once: two a CU, three with heads of 64.
int64_t places(int head_dim) { return head_dim == 128 ? 2 * kCus : 3 * kCus; }
// Up to how many whole tiles they are split over the keys: a wave's half tile runs
// 0.8 us on its CU alone, so that few long tiles leave the chip waiting for the
// longest, while split ones fetch each key for half as many queries.  us, whole and
// split, by tiles and whatever the lengths are.  Heads of 128, 32 / 8: 56 (200 tokens) 9.4,
// 9.5; 64 (500, 16 / 8) 12.1, 10.1; 256 (1000) 22.0, 18.2; 264 (three of up to 600) 16.3,
// 14.1; 376 (1500) 31.0, 31.4; 512 (2048) 44.0, 47.8; 512 (4096, 16 / 8) 81.0, 85.5; 1936
// (24 of up to 1000) 62, 87.  Heads of 64: 144 (four of up to 600, 12 / 12) 10.1, 9.6; 228
// (eight) 10.7, 9.7; 580 (eight of up to 1500, 20 / 20) 21.1, 18.9; 632 (2500, 32 / 8) 39.1,
// 38.5; 640 (4000, 20 / 20) 60.8, 57.5; 640 (2 x 2000) 33.8, 32.5; 768 (8 x 1000, 12 / 12)
// 22.3, 23.9; 768 (16 x 512) 16.0, 17.9; 768 (64 x 77) 9.5, 11.7; 1024 (4096, 32 / 8) 83.1,
// 89.1; 1280 (32 x 200, 20 / 20) 18.0, 23.6.
int64_t split_tiles(int head_dim) { return head_dim == 128 ? 320 : 700; }

// The bytes from a view's first element to past its last.
struct Span {
  uintptr_t lo, hi;
};
Span span(const void *p, int64_t rows, int64_t row_stride, int64_t heads, int64_t head_stride, int64_t dim) {
  const uintptr_t lo = reinterpret_cast<uintptr_t>(p);
  return {lo, lo + 2 * (uintptr_t)((rows - 1) * row_stride + (heads - 1) * head_stride + dim)};
}

}  // namespace
}  // namespace mq

extern "C" int mq_prompt_plan_make(const int64_t *lengths, int64_t count, int heads, int kv_heads, int head_dim,
                                   mq_prompt_plan *plan, int32_t *tiles, int64_t capacity) {
  using namespace mq;
  if (!plan || (count > 0 && !lengths)) return invalid("mq_prompt_plan_make: NULL pointer");
  if (head_dim != 64 && head_dim != 128) return invalid("mq_prompt_plan_make: head_dim must be 64 or 128");
  if (count < 0 || heads < 1 || heads > 65536 || kv_heads < 1 || heads % kv_heads)
    return invalid("mq_prompt_plan_make: negative count, or heads not a multiple of kv_heads");
  int64_t total = 0;
  for (int64_t s = 0; s < count; ++s) {
    if (lengths[s] < 0 || lengths[s] >= (int64_t(1) << 31) || (total += lengths[s]) >= (int64_t(1) << 31))
      return invalid("mq_prompt_plan_make: a negative length, or 2^31 tokens or more");
  }
  // parts 2 where whole tiles would leave the chip's places empty or be few enough
  // that the longest sets the time
  int64_t n = 0, longest = 0;
  int tile = 0, parts = 1;
  for (;;) {
    tile = tile_tokens(heads / kv_heads, parts);
    n = 0;
    for (int64_t s = 0; s < count; ++s) {
      n += (lengths[s] + tile - 1) / tile;
      longest = std::max(longest, lengths[s]);
    }
    if (parts == 2 || n * (heads >> unit_log(heads / kv_heads, kWaves)) > split_tiles(head_dim)) break;
    parts = 2;
  }
  *plan = mq_prompt_plan{total, n, heads, kv_heads, head_dim, tile, parts};
  if (!tiles) return MQ_OK;
  if (capacity < n) return invalid("mq_prompt_plan_make: tiles holds fewer than the plan's tiles");
  // longest first: the tiles at one distance from their prompts' starts, the furthest
  // first.  Where all run at once, those after the first of each CU are taken from
  // the other end, so that a long tile shares its CU with a short one.
  const int64_t units = heads >> unit_log(heads / kv_heads, kWaves / parts);
  const int64_t turn = n * units <= places(head_dim) ? std::max<int64_t>(1, kCus / units) : n;
  int64_t at = 0;
  for (int64_t first = (longest - 1) / tile * tile; longest > 0 && first >= 0; first -= tile) {
    int64_t start = 0;
    for (int64_t s = 0; s < count; start += lengths[s++])
      if (lengths[s] > first) {
        int32_t *t = tiles + 4 * (at < turn ? at : n - 1 - (at - turn));
        ++at;
        t[0] = (int32_t)start;
        t[1] = (int32_t)lengths[s];
        t[2] = (int32_t)first;
        t[3] = 0;
      }
  }
  return MQ_OK;
}

extern "C" int mq_prompt_attention(const mq_prompt_plan *plan, const int32_t *tiles, const void *q, int64_t q_token_stride,
                                   int64_t q_head_stride, const void *k, int64_t k_token_stride, int64_t k_head_stride,
                                   const void *v, int64_t v_token_stride, int64_t v_head_stride, float scale, void *out,
                                   int64_t out_token_stride, int64_t out_head_stride, void *stream) {
  using namespace mq;
  if (!plan) return invalid("mq_prompt_attention: NULL plan");
  const int heads = plan->heads, kv = plan->kv_heads, dim = plan->head_dim;
  if ((dim != 64 && dim != 128) || heads < 1 || heads > 65536 || kv < 1 || heads % kv || plan->tokens < 0 ||
      plan->tokens >= (int64_t(1) << 31) || plan->tiles < 0 || plan->tiles > plan->tokens || (plan->parts != 1 && plan->parts != 2) ||
      plan->tile_tokens != tile_tokens(heads / kv, plan->parts))
    return invalid("mq_prompt_attention: not a plan of mq_prompt_plan_make");
  if (!takes_scale(scale)) return invalid("mq_prompt_attention: scale must be positive, and finite times log2(e)");
  if (plan->tokens == 0 || plan->tiles == 0) return MQ_OK;
  if (!tiles || !q || !k || !v || !out) return invalid("mq_prompt_attention: NULL pointer");
  if (!aligned16(tiles) || !aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out))
    return invalid("mq_prompt_attention: buffers must be 16-byte aligned");
  for (int64_t s : {q_token_stride, q_head_stride, k_token_stride, k_head_stride, v_token_stride, v_head_stride,
                    out_token_stride, out_head_stride})
    if (s < 0 || s % 8 || s >= (int64_t(1) << 24))
      return invalid("mq_prompt_attention: strides must be multiples of 8 elements, 0 to 2^24");
  // rows and heads of out apart from each other; the stride of a single one may be anything
  const bool rows = plan->tokens > 1, several = heads > 1;
  if ((rows && out_token_stride < dim) || (several && out_head_stride < dim) ||
      (rows && several && out_token_stride < (heads - 1) * out_head_stride + dim &&
       out_head_stride < (plan->tokens - 1) * out_token_stride + dim))
    return invalid("mq_prompt_attention: rows or heads of out overlap");
  const Span o = span(out, plan->tokens, out_token_stride, heads, out_head_stride, dim);
  for (const Span &in : {span(q, plan->tokens, q_token_stride, heads, q_head_stride, dim),
                         span(k, plan->tokens, k_token_stride, kv, k_head_stride, dim),
                         span(v, plan->tokens, v_token_stride, kv, v_head_stride, dim)})
    if (o.lo < in.hi && in.lo < o.hi) return invalid("mq_prompt_attention: out lies over q, k or v");
  const int log_heads = unit_log(heads / kv, kWaves / plan->parts), units = heads >> log_heads;
  const int64_t grid = plan->tiles * units;
  if (grid >= (int64_t(1) << 31)) return invalid("mq_prompt_attention: 2^31 tiles or more");
  const PromptArgs a{static_cast<const __bf16 *>(q), static_cast<const __bf16 *>(k), static_cast<const __bf16 *>(v),
                     static_cast<__bf16 *>(out), q_token_stride, k_token_stride, v_token_stride, out_token_stride,
                     q_head_stride, k_head_stride, v_head_stride, out_head_stride, reinterpret_cast<const int4 *>(tiles),
                     plan->tokens, units, heads / kv, log_heads, scale * kLog2e, least_score(scale)};
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto launch = [&]<int D, int P>() {
    hipLaunchKernelGGL((prompt_kernel<D, kWaves, P>), dim3((unsigned)grid), dim3(64 * kWaves), 0, s, a);
  };
  if (dim == 128) plan->parts == 1 ? launch.template operator()<128, 1>() : launch.template operator()<128, 2>();
  else plan->parts == 1 ? launch.template operator()<64, 1>() : launch.template operator()<64, 2>();
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MQ_OK : set_error(MQ_E_HIP, hipGetErrorString(e));
}
