// mq_cache.h — the device layout of the paged key/value cache.
//
// A page holds page_tokens tokens (a multiple of 32) of every k/v head, and is
// made of tiles of 32 tokens of one head, keys and values together:
//   data + ((page * kv_heads + head) * (page_tokens / 32) + token / 32) * kTile.
// Inside a tile the bytes stand in the order in which the attention's matrix
// instructions (v_mfma_f32_16x16x32_bf16) take them, so that a wave reads each
// 16-byte piece of an operand as one run of 1 KiB, with no transposition:
//   keys    plane of 2 x (D / 32) operands, S^T = K Q^T: lane 16 g + r holds token
//           16 u + r and, of each block b of 32 of the head, eight values.  In BF16
//           and Q8_0 these are 32 b + 8 g + 0..7; in Q4_0, whose byte j of a block
//           is ggml's (values j and j + 16), bytes 4 g + 0..3.
//   values  plane of D / 16 operands, O^T = V^T P^T, two a block: lane 16 g + r holds
//           value 32 b + 2 r + c of the eight tokens 16 (j / 4) + 4 g + j % 4 (j =
//           0..7), which are the ones whose scores S^T leaves in that lane; c = 0 in
//           the first operand, 1 in the second, so that a lane's eight results of a
//           block lie next to each other.  A Q4_0 byte is the pair, c = 0 its low half.
//   scales  of the block types, f16: the keys' as [g][u][b][token 4 g + 0..3 of
//           u], the values' as [g][b][j].
// A lane's bytes of one plane are split into pieces of 16 (8 for the keys of Q4_0
// heads of 64), a piece of all 64 lanes together.
#pragma once

#include "mq_attn.h"

namespace mq {
namespace {

constexpr int kTileTokens = 32;

template <int T, int D>
struct CacheTile {
  static constexpr bool kQuant = T != BF16;
  static constexpr int kBlocks = D / 32;
  static constexpr int kKeyLane = kBlocks * (T == BF16 ? 16 : T == Q8_0 ? 8 : 4);  // bytes of a lane, one u
  static constexpr int kKeyPiece = kKeyLane < 16 ? kKeyLane : 16;
  static constexpr int kValueLane = 2 * kKeyLane;
  static constexpr int kPlane = 128 * kKeyLane;  // of keys, and of values
  static constexpr int kScales = kQuant ? 64 * kBlocks : 0;
  static constexpr int kBytes = 2 * kPlane + 2 * kScales;

  // Byte `i` of the eight values of block b of token t (of 32) in lane group g.
  __device__ static int key(int t, int b, int g, int i) {
    const int at = b * (kKeyLane / kBlocks) + i;
    return (t >> 4) * (64 * kKeyLane) + at / kKeyPiece * (64 * kKeyPiece) + (16 * g + (t & 15)) * kKeyPiece + at % kKeyPiece;
  }
  // Value d of token t: its first byte (Q4_0: of the pair, d even).
  __device__ static int value(int t, int d) {
    const int j = 4 * (t >> 4) + (t & 3), c = 2 * (d >> 5) + (d & 1);
    const int at = T == BF16 ? c * 16 + 2 * j : T == Q8_0 ? c * 8 + j : (d >> 5) * 8 + j;
    return kPlane + at / 16 * 1024 + (16 * ((t >> 2) & 3) + ((d >> 1) & 15)) * 16 + at % 16;
  }
  __device__ static int key_scale(int t, int b) {
    return 2 * kPlane + 2 * ((((((t >> 2) & 3) * 2 + (t >> 4)) * kBlocks) + b) * 4 + (t & 3));
  }
  __device__ static int value_scale(int t, int b) {
    return 2 * kPlane + kScales + 2 * (((((t >> 2) & 3) * kBlocks) + b) * 8 + 4 * (t >> 4) + (t & 3));
  }
};

struct CacheView {
  uint8_t *data;
  int64_t slots;     // pages * page_tokens
  int page_tokens, kv_heads;
};

inline int64_t cache_tile_bytes(int dtype, int head_dim) {
  return dtype == BF16 ? 128 * head_dim : dtype == Q8_0 ? 68 * head_dim : 36 * head_dim;
}
static_assert(CacheTile<BF16, 128>::kBytes == 128 * 128 && CacheTile<Q8_0, 64>::kBytes == 68 * 64 &&
              CacheTile<Q4_0, 128>::kBytes == 36 * 128);

// What is wrong with a cache's description, or NULL.
inline const char *cache_fault(const mq_kv_cache *c) {
  if (!c) return "NULL cache";
  if (c->dtype != MQ_BF16 && c->dtype != MQ_Q8_0 && c->dtype != MQ_Q4_0) return "a cache is BF16, Q8_0 or Q4_0";
  if (c->head_dim != 64 && c->head_dim != 128) return "a cache's head_dim is 64 or 128";
  if (c->kv_heads < 1 || c->kv_heads > 4096) return "a cache has 1 to 4096 k/v heads";
  if (c->page_tokens < kTileTokens || c->page_tokens % kTileTokens || c->page_tokens > 65536)
    return "a cache's pages hold a multiple of 32 tokens, up to 65536";
  if (c->pages < 0 || c->pages >= (int64_t(1) << 31)) return "a cache has 0 to 2^31 pages";
  int64_t size;  // a page alone is below 2^38
  if (__builtin_mul_overflow(c->pages, c->kv_heads * (c->page_tokens / kTileTokens) * cache_tile_bytes(c->dtype, c->head_dim), &size))
    return "a cache has less than 2^63 bytes";
  return nullptr;
}

// Calls f<type, head_dim>() for a cache without a fault.
template <typename F>
void with_cache_type(const mq_kv_cache *c, F f) {
  const bool wide = c->head_dim == 128;
  if (c->dtype == MQ_BF16) wide ? f.template operator()<BF16, 128>() : f.template operator()<BF16, 64>();
  else if (c->dtype == MQ_Q8_0) wide ? f.template operator()<Q8_0, 128>() : f.template operator()<Q8_0, 64>();
  else wide ? f.template operator()<Q4_0, 128>() : f.template operator()<Q4_0, 64>();
}

}  // namespace
}  // namespace mq
