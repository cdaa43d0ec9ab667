// mq_beams.hip — beam search over a decoder's logits and paged caches.
//
// mq_beam_select: of all continuations (beam b, token t) of a request the `count` with the
// largest score_b + log softmax(x_b)_t = score_b + (x - m) - log sum exp(x - m), ties to the lowest
// (b, t); a beam that has ended has one, its stop token, at its score as it is.
//   The logits are read once: the bound is HBM for a batch, two launches for a request or
// two.  scan_kernel cuts each row into runs of a workgroup, and a wave keeps of its part the
// sum of exponentials and the `count` largest logits, one a lane, sorted.  The sum needs no
// second pass: it is relative to a reference that follows the logits only where one passes
// it by more than 1, and the same comparison finds what may enter the list, so that a group
// of logits costs its exponentials, its maximum and one comparison with the smaller of the
// two.  merge_kernel joins a request's runs, takes the totals in 64 bits, in which beams
// whose totals lie close compare as their logits say, and ranks them.
//   Exponentials are f32 (v_exp_f32 of differences, whose error shrinks with the term's weight),
// sums of a group f32, of a lane and beyond f64.
//
// mq_beam_reorder: beam j of a request goes on from beam parents[j].  Whole pages are shared: a
// row of the page table takes its parent's entries.  The last, partial page goes to one child
// of each parent (to the parent's own row if it is one, else the first); every other child
// takes the page of a row without children, as many as there are, and has the tokens so far
// copied into it, in every layer's cache.  plan_kernel does the tables, copy_kernel moves the
// bytes: those of the used tiles (32 tokens) and no others, which bound it.
#include "../../include/moldq.h"
#include "mq_cache_write.h"

namespace mq {
int set_error(int code, const char *msg);
}

namespace mq {
namespace {

constexpr int kScanThreads = 256, kScanWaves = kScanThreads / 64;
constexpr int kMergeThreads = 256, kMergeWaves = kMergeThreads / 64;

// A logit and its token as one key: larger logits first, of equal ones the lower token.  0 is
// none.  Adding 0 makes the two zeros one.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u ^ (uint32_t)(((int)u >> 31) | (int)0x80000000);
}
__device__ __forceinline__ uint64_t key_of_logit(float x, uint32_t token) { return ((uint64_t)ordered(x) << 32) | (0xFFFFFFFFu - token); }
__device__ __forceinline__ float logit_of(uint64_t key) {
  const uint32_t u = (uint32_t)(key >> 32);
  return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u);
}
__device__ __forceinline__ uint32_t token_of(uint64_t key) { return 0xFFFFFFFFu - (uint32_t)key; }

__device__ __forceinline__ uint64_t xor_lane(uint64_t v, int with) {
  return ((uint64_t)__shfl_xor((uint32_t)(v >> 32), with) << 32) | __shfl_xor((uint32_t)v, with);
}
__device__ __forceinline__ uint64_t lane_of(uint64_t v, int lane) {
  return ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32) | (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}
// Lane i takes the larger (where `high`) or the smaller of its own and lane i ^ with's.
template <typename K>
__device__ __forceinline__ K exchange(K v, int with, bool high) {
  K other;
  if constexpr (sizeof(K) == 8) other = xor_lane(v, with);
  else other = __shfl_xor(v, with);
  return high == (v > other) ? v : other;
}
// Sorted over the wave, the largest in lane 0.
template <typename K>
__device__ __forceinline__ K sorted(K v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int size = 2; size <= 64; size <<= 1)
#pragma unroll
    for (int with = size >> 1; with; with >>= 1) v = exchange(v, with, ((lane & size) == 0) == ((lane & with) == 0));
  return v;
}

// The largest keys that a wave has seen, one a lane, the largest in lane 0.
struct Largest {
  uint64_t key, least;  // `least`: the count-th, below which nothing enters
  int count;

  __device__ explicit Largest(int n) : key(0), least(0), count(n) {}
  // A key of each lane, or 0.  All lanes join.
  __device__ void offer(uint64_t k) {
    uint64_t in = __ballot(k > least);
    if (!in) return;
    if (__popcll(in) <= 6) {
      const int lane = threadIdx.x & 63;
      do {
        const int from = __builtin_ctzll(in);
        in &= in - 1;
        const uint64_t one = lane_of(k, from);
        const int at = __popcll(__ballot(key > one));
        const uint64_t before = ((uint64_t)__shfl_up((uint32_t)(key >> 32), 1) << 32) | __shfl_up((uint32_t)key, 1);
        key = lane < at ? key : lane == at ? one : before;
      } while (in);
    } else {
      k = sorted(k > least ? k : 0);
      const uint64_t turned = xor_lane(k, 63);  // ascending: with the list one bitonic sequence
      key = key > turned ? key : turned;
#pragma unroll
      for (int with = 32; with; with >>= 1) key = exchange(key, with, (threadIdx.x & with) == 0);
    }
    const uint64_t last = lane_of(key, count - 1);
    if (last > least) least = last;
  }
};

// 16 bytes of a row, which may start at any element: how its logits are grouped, and so their
// sum to the last bit, goes by their places in the row alone, and rows alike give the same.
template <typename X>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int kN = 4;
  typedef float raw __attribute__((ext_vector_type(4), aligned(4)));
  __device__ static void get(const raw &r, float *x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = r[i];
  }
};
template <>
struct Vec<__bf16> {
  static constexpr int kN = 8;
  typedef uint32_t raw __attribute__((ext_vector_type(4), aligned(2)));
  __device__ static void get(const raw &r, float *x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(r[i] << 16), x[2 * i + 1] = __uint_as_float(r[i] & 0xFFFF0000u);
  }
};

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int off = 32; off; off >>= 1) v = fmaxf(v, __shfl_xor(v, off));
  return v;
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int off = 32; off; off >>= 1) v += __shfl_xor(v, off);
  return v;
}

// What a wave, and then a workgroup, keeps of a run of logits.
struct Run {
  double sum;  // of exp(x - ref); NaN where a logit is NaN or plus infinity
  float ref;
};

struct SelectArgs {
  const void *logits;
  int64_t request, beam;  // strides in elements
  int64_t vocab, n;
  const float *scores;    // [n, beams]
  const int64_t *last;    // [n, beams], NULL: no beam has ended
  int64_t stop;
  int beams, count, splits;
  Run *runs;              // [n, beams, splits]
  uint64_t *keys;         // [n, beams, splits, count]
  float *out_scores;
  int32_t *parents;
  int64_t *tokens;
};

__device__ __forceinline__ bool ended(const SelectArgs &a, int64_t row) { return a.last && a.last[row] == a.stop; }

// Reads part `part` of `parts` of a row by one wave.
template <typename X>
struct Scan {
  Largest top;
  double sum;
  float ref, enter;  // `enter`: what a logit has to reach to enter the list or to move the reference

  __device__ explicit Scan(int count) : top(count), sum(0.), ref(-__FLT_MAX__), enter(-__FLT_MAX__) {}

  // The reference follows the largest of the lanes' logits; the sums so far with it.
  __device__ void follow(float most) {
    const float to = wave_max(most);
    if (!(to > ref + 1.f)) return;  // also where `to` is the lowest value, and NaN
    sum *= (double)__builtin_amdgcn_exp2f((ref - to) * kLog2e);
    ref = to;
  }
  __device__ void bounds() {
    const float least = top.least ? logit_of(top.least) : -__FLT_MAX__;
    enter = fminf(least, ref + 1.f);
  }
  template <int N>
  __device__ void add(const float *x) {
    float s[N];
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = __builtin_amdgcn_exp2f((x[i] - ref) * kLog2e);
#pragma unroll
    for (int w = N / 2; w; w >>= 1)
#pragma unroll
      for (int i = 0; i < w; ++i) s[i] += s[i + w];
    sum += (double)s[0];
  }
  template <int N>
  __device__ static float most_of(const float *x) {
    float m = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) m = fmaxf(m, x[i]);
    return m;
  }
  // N logits of each lane, tokens token .. token + N - 1; minus infinity for none.
  template <int N>
  __device__ void take(const float *x, uint32_t token) {
    const float most = most_of<N>(x);
    if (__any(most >= enter)) {
      follow(most);
#pragma unroll
      for (int i = 0; i < N; ++i) top.offer(x[i] >= -__FLT_MAX__ ? key_of_logit(x[i], token + i) : 0);
      bounds();
    }
    add<N>(x);
  }

  __device__ void row(const X *p, int64_t vocab, int64_t part, int64_t parts) {
    constexpr int N = Vec<X>::kN;
    typedef typename Vec<X>::raw raw;
    const int lane = threadIdx.x & 63;
    const int64_t vectors = vocab / N, rest = vocab - vectors * N;
    const raw *const body = reinterpret_cast<const raw *>(p);
    const int64_t from = vectors * part / parts, to = vectors * (part + 1) / parts;
    constexpr int U = 4;
    for (int64_t v = from; v < to; v += 64 * U) {
      float x[U][N];
      raw r[U];
#pragma unroll
      for (int u = 0; u < U; ++u) r[u] = body[min(v + 64 * u + lane, to - 1)];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        Vec<X>::get(r[u], x[u]);
        if (v + 64 * u + lane >= to) {
#pragma unroll
          for (int i = 0; i < N; ++i) x[u][i] = -__builtin_inff();
        }
      }
      if (v == from) {  // the count-th largest of the lanes' maxima: as many logits reach it, so what lies below need not enter
        float most = most_of<N>(x[0]);
#pragma unroll
        for (int u = 1; u < U; ++u) most = fmaxf(most, most_of<N>(x[u]));
        follow(most);
        most = most >= -__FLT_MAX__ ? most : -__FLT_MAX__;
        const uint32_t least = __builtin_amdgcn_readlane((int)sorted(ordered(most)), top.count - 1);
        // a key that every logit of that value passes, and none below it
        top.least = least > ordered(-__FLT_MAX__) ? ((uint64_t)least << 32) - 1 : 0;
        enter = fminf(logit_of((uint64_t)least << 32), ref + 1.f);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (v + 64 * u < to) take<N>(x[u], (uint32_t)((v + 64 * u + lane) * N));
    }
    if (part == parts - 1 && rest) {
      const int64_t at = vectors * N + lane;
      const float x = lane < rest ? (float)p[at] : -__builtin_inff();
      take<1>(&x, (uint32_t)at);
    }
  }
};

template <typename X>
__global__ __launch_bounds__(kScanThreads) void scan_kernel(SelectArgs a) {
  __shared__ Run runs[kScanWaves];
  __shared__ uint64_t lists[kScanWaves][64];
  const int64_t row = blockIdx.x / (uint32_t)a.splits, split = blockIdx.x - row * a.splits;
  if (ended(a, row) || !(fabsf(a.scores[row]) <= __FLT_MAX__)) return;  // has no logits to look at
  const int64_t n = row / a.beams;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  Scan<X> scan(a.count);
  scan.row(static_cast<const X *>(a.logits) + n * a.request + (row - n * a.beams) * a.beam, a.vocab, split * kScanWaves + wave,
           (int64_t)a.splits * kScanWaves);
  const double sum = wave_sum(scan.sum);
  if (lane == 0) runs[wave] = {sum, scan.ref};
  lists[wave][lane] = scan.top.key;
  __syncthreads();
  if (wave) return;
  Largest top = scan.top;
  top.least = lane_of(top.key, a.count - 1);
  for (int first = a.count; first < kScanWaves * a.count; first += 64) {
    const int at = first + lane;
    top.offer(at < kScanWaves * a.count ? lists[at / a.count][at % a.count] : 0);
  }
  Run all = runs[0];
#pragma unroll
  for (int i = 1; i < kScanWaves; ++i) all.ref = fmaxf(all.ref, runs[i].ref);
  all.sum = 0.;
#pragma unroll
  for (int i = 0; i < kScanWaves; ++i) all.sum += runs[i].sum * exp((double)runs[i].ref - (double)all.ref);
  if (lane == 0) a.runs[row * a.splits + split] = all;
  if (lane < a.count) a.keys[(row * a.splits + split) * a.count + lane] = top.key;
}

// A continuation of a request: its total as an ordered f64, 0 for none.
struct Candidate {
  uint64_t total;
  int64_t token;
};
__device__ __forceinline__ uint64_t ordered64(double x) {
  const int64_t u = __double_as_longlong(x + 0.);
  return (uint64_t)u ^ ((uint64_t)(u >> 63) | 0x8000000000000000ull);
}
__device__ __forceinline__ double total_of(uint64_t u) {
  return __longlong_as_double((int64_t)(u >> 63 ? u ^ 0x8000000000000000ull : ~u));
}

// A workgroup a request: a wave joins a beam's runs at a time, then every candidate counts
// those over it: of its own beam the ones before it, of a lower beam those of no smaller
// total, of a higher one those of a larger.
__global__ __launch_bounds__(kMergeThreads) void merge_kernel(SelectArgs a) {
  extern __shared__ Candidate found[];  // [beams, count], each beam's sorted
  const int64_t n = blockIdx.x;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  for (int b = wave; b < a.beams; b += kMergeWaves) {
    const int64_t row = n * a.beams + b;
    const float score = a.scores[row];
    Candidate mine{0, -1};
    if (!(fabsf(score) <= __FLT_MAX__)) {
    } else if (ended(a, row)) {
      if (lane == 0) mine = {ordered64(score), a.stop};
    } else {
      Run run{0., -__FLT_MAX__};
      if (lane < a.splits) run = a.runs[row * a.splits + lane];
      const float ref = wave_max(run.ref);
      const double sum = wave_sum(run.sum * exp((double)run.ref - (double)ref));
      Largest top(a.count);
      const uint64_t *const keys = a.keys + row * a.splits * a.count;
      for (int first = 0; first < a.splits * a.count; first += 64) top.offer(first + lane < a.splits * a.count ? keys[first + lane] : 0);
      if (sum > 0. && sum <= __DBL_MAX__ && top.key)
        mine = {ordered64((double)score + (((double)logit_of(top.key) - (double)ref) - log(sum))), (int64_t)token_of(top.key)};
    }
    if (lane < a.count) found[b * a.count + lane] = mine;
  }
  __syncthreads();
  // how many of beam b's are over `total`, or level with it too: they stand first
  auto over = [&](int b, uint64_t total, bool level) {
    int lo = 0, hi = a.count;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      const uint64_t t = found[b * a.count + mid].total;
      if (t > total || (level && t == total)) lo = mid + 1;
      else hi = mid;
    }
    return lo;
  };
  for (int i = threadIdx.x; i < a.beams * a.count; i += kMergeThreads) {
    const Candidate mine = found[i];
    if (!mine.total) continue;
    const int of = i / a.count;
    int rank = i - of * a.count;
    for (int b = 0; b < a.beams && rank < a.count; ++b)
      if (b != of) rank += over(b, mine.total, b < of);
    if (rank >= a.count) continue;
    const int64_t to = n * a.count + rank;
    a.out_scores[to] = (float)total_of(mine.total);
    a.parents[to] = of;
    a.tokens[to] = mine.token;
  }
  int have = 0;
  for (int b = 0; b < a.beams && have < a.count; ++b) have += over(b, 0, false);
  for (int i = have + threadIdx.x; i < a.count; i += kMergeThreads) {
    const int64_t to = n * a.count + i;
    a.out_scores[to] = -__builtin_inff();
    a.parents[to] = 0;
    a.tokens[to] = -1;
  }
}

// ------------------------------------------------------------------ reordering

struct Copy {
  int32_t from, to, tiles, pad;  // pages, and how many tiles of each head; from -1: nothing
};

struct ReorderArgs {
  int32_t *table;
  int64_t stride, width, pages;
  const int32_t *lengths;  // [requests, beams], the first of a request read
  const int32_t *parents;  // [requests, beams]
  Copy *plan;              // [requests, beams]
  int beams, page;
};

constexpr int kPlanThreads = 256, kPlanColumns = 64;

// A workgroup a request.  Lane j of its first wave is beam j.
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(ReorderArgs a) {
  __shared__ int32_t entries[MQ_MAX_BEAMS * kPlanColumns];
  __shared__ int parent[MQ_MAX_BEAMS], taken[MQ_MAX_BEAMS], dead[MQ_MAX_BEAMS], moves;
  const int64_t row0 = (int64_t)blockIdx.x * a.beams;
  const int length = max(a.lengths[row0], 0), full = length / a.page, tail = length - full * a.page;
  if (threadIdx.x < 64) {
    const int j = threadIdx.x;
    const bool is = j < a.beams;
    int p = is ? a.parents[row0 + j] : j;
    if (p < 0 || p >= a.beams) p = j;  // no parent: goes on as it is
    uint64_t children = 0;  // of beam j
    for (int q = 0; q < a.beams; ++q) {
      const uint64_t of = __ballot(is && p == q);
      if (q == j) children = of;
    }
    const int keeper = children ? (children >> j & 1 ? j : __builtin_ctzll(children)) : -1;
    const uint64_t deads = __ballot(is && !children);
    const bool keeps = __shfl(keeper, p) == j;
    const uint64_t copies = __ballot(is && !keeps), below = ((uint64_t)1 << j) - 1;
    if (is && !children) dead[__popcll(deads & below)] = j;
    __builtin_amdgcn_wave_barrier();
    __threadfence_block();
    if (is) {
      parent[j] = p;
      taken[j] = keeps ? p : dead[__popcll(copies & below)];
    }
    const bool moved = __any(is && p != j);
    if (j == 0) moves = moved;
  }
  __syncthreads();
  // the partial page: which each row has now, and what is copied into it
  if (threadIdx.x < a.beams) {
    const int j = threadIdx.x;
    Copy copy{-1, -1, 0, 0};
    if (tail && full < a.width && moves) {
      const int from = a.table[(row0 + parent[j]) * a.stride + full], to = a.table[(row0 + taken[j]) * a.stride + full];
      if (taken[j] != parent[j] && from >= 0 && from < a.pages && to >= 0 && to < a.pages) copy = {from, to, (tail + kTileTokens - 1) / kTileTokens, 0};
      entries[j] = to;
    }
    a.plan[row0 + j] = copy;
  }
  if (!moves) return;
  __syncthreads();
  if (tail && full < a.width && threadIdx.x < a.beams) a.table[(row0 + threadIdx.x) * a.stride + full] = entries[threadIdx.x];
  const int64_t columns = min((int64_t)full, a.width);
  for (int64_t c0 = 0; c0 < columns; c0 += kPlanColumns) {
    const int here = (int)min(columns - c0, (int64_t)kPlanColumns);
    __syncthreads();
    for (int i = threadIdx.x; i < a.beams * kPlanColumns; i += kPlanThreads) {
      const int c = i % kPlanColumns, j = i / kPlanColumns;
      if (c < here) entries[i] = a.table[(row0 + j) * a.stride + c0 + c];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < a.beams * kPlanColumns; i += kPlanThreads) {
      const int c = i % kPlanColumns, j = i / kPlanColumns;
      if (c < here && parent[j] != j) a.table[(row0 + j) * a.stride + c0 + c] = entries[parent[j] * kPlanColumns + c];
    }
  }
}

constexpr int kMaxCaches = 64, kCopyThreads = 256, kCopyTiles = 4;
struct CacheList {
  uint8_t *data[kMaxCaches];
};

// A workgroup a (request, run of kCopyTiles tiles, head, cache): its beams' copies in turn.
__global__ __launch_bounds__(kCopyThreads) void copy_kernel(CacheList caches, const Copy *plan, int beams, uint32_t tile_units, int tiles, int runs) {
  const uint32_t request = blockIdx.x / (uint32_t)runs, first = (blockIdx.x - request * runs) * kCopyTiles;
  const int64_t head = blockIdx.y, heads = gridDim.y;
  uint4 *const data = reinterpret_cast<uint4 *>(caches.data[blockIdx.z]);
  const int lane = threadIdx.x & 63;
  Copy mine{-1, -1, 0, 0};
  if (lane < beams) mine = plan[(int64_t)request * beams + lane];
  for (uint64_t some = __ballot(mine.from >= 0 && mine.tiles > (int)first); some; some &= some - 1) {
    const int j = __builtin_ctzll(some);
    const int64_t page_from = __builtin_amdgcn_readlane(mine.from, j), page_to = __builtin_amdgcn_readlane(mine.to, j);
    const int count = min(__builtin_amdgcn_readlane(mine.tiles, j) - (int)first, kCopyTiles);
    const int64_t in = first * (int64_t)tile_units;
    const uint4 *const from = data + (page_from * heads + head) * tiles * tile_units + in;
    uint4 *const to = data + (page_to * heads + head) * tiles * tile_units + in;
    const uint32_t units = count * tile_units;
    uint32_t i = threadIdx.x;
    for (; i + 3 * kCopyThreads < units; i += 4 * kCopyThreads) {
      uint4 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = from[i + u * kCopyThreads];
#pragma unroll
      for (int u = 0; u < 4; ++u) to[i + u * kCopyThreads] = v[u];
    }
    for (; i < units; i += kCopyThreads) to[i] = from[i];
  }
}

int invalid(const char *msg) { return set_error(MQ_E_INVALID, msg); }
bool aligned_to(const void *p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// Runs of a row: enough workgroups for eight on each of 256 CUs, none below 4096 logits (16 a
// thread), 64 at most (a lane each when they are joined).
int splits_of(int64_t rows, int64_t vocab) {
  const int64_t want = (2048 + rows - 1) / rows, most = vocab / 4096;
  const int64_t s = want < most ? want : most;
  return (int)(s < 1 ? 1 : s > 64 ? 64 : s);
}

const char *select_fault(int64_t n, int beams, int64_t vocab, int count) {
  if (n < 0 || n > (int64_t(1) << 20)) return "mq_beam_select: 0 to 2^20 requests";
  if (beams < 1 || beams > MQ_MAX_BEAMS || count < 1 || count > MQ_MAX_BEAMS) return "mq_beam_select: 1 to 64 beams and continuations";
  if (vocab < 1 || vocab >= (int64_t(1) << 31)) return "mq_beam_select: a vocabulary of 1 to 2^31 tokens";
  return nullptr;
}

}  // namespace
}  // namespace mq

extern "C" size_t mq_beam_select_scratch_size(int64_t requests, int beams, int64_t vocab, int count) {
  using namespace mq;
  if (requests == 0 || select_fault(requests, beams, vocab, count)) return 0;
  const int64_t rows = requests * beams;
  return (size_t)rows * splits_of(rows, vocab) * (sizeof(Run) + 8 * (size_t)count);
}

extern "C" int mq_beam_select(const void *logits, int dtype, int64_t requests, int beams, int64_t vocab, int64_t request_stride,
                              int64_t beam_stride, const float *scores, const int64_t *last, int64_t stop, int count, float *out_scores,
                              int32_t *parents, int64_t *tokens, void *scratch, size_t scratch_bytes, void *stream) {
  using namespace mq;
  if (const char *fault = select_fault(requests, beams, vocab, count)) return invalid(fault);
  if (dtype != MQ_F32 && dtype != MQ_BF16) return invalid("mq_beam_select: logits are F32 or BF16");
  if (last && (stop < 0 || stop >= vocab)) return invalid("mq_beam_select: the stop token is one of the vocabulary");
  if (requests == 0) return MQ_OK;
  for (int64_t s : {request_stride, beam_stride})
    if (s < 0 || s >= (int64_t(1) << 40)) return invalid("mq_beam_select: strides outside 0 .. 2^40");
  if (!logits || !scores || !out_scores || !parents || !tokens || !scratch) return invalid("mq_beam_select: NULL pointer");
  if (scratch_bytes < mq_beam_select_scratch_size(requests, beams, vocab, count)) return invalid("mq_beam_select: too little scratch");
  if (!aligned_to(logits, dtype == MQ_F32 ? 4 : 2) || !aligned_to(scores, 4) || !aligned_to(out_scores, 4) || !aligned_to(parents, 4) ||
      !aligned_to(last, 8) || !aligned_to(tokens, 8) || !aligned_to(scratch, 16))
    return invalid("mq_beam_select: misaligned buffer");
  const int64_t rows = requests * beams;
  const int splits = splits_of(rows, vocab);
  if (rows * splits >= (int64_t(1) << 24)) return invalid("mq_beam_select: too many requests");
  Run *const runs = static_cast<Run *>(scratch);
  const SelectArgs a{logits, request_stride, beam_stride, vocab, requests, scores, last, stop, beams, count, splits, runs,
                     reinterpret_cast<uint64_t *>(runs + rows * splits), out_scores, parents, tokens};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)(rows * splits));
  if (dtype == MQ_F32) hipLaunchKernelGGL(scan_kernel<float>, grid, dim3(kScanThreads), 0, s, a);
  else hipLaunchKernelGGL(scan_kernel<__bf16>, grid, dim3(kScanThreads), 0, s, a);
  hipLaunchKernelGGL(merge_kernel, dim3((unsigned)requests), dim3(kMergeThreads), sizeof(Candidate) * beams * count, s, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MQ_OK : set_error(MQ_E_HIP, hipGetErrorString(e));
}

extern "C" size_t mq_beam_reorder_scratch_size(int64_t requests, int beams) {
  if (requests < 0 || requests > (int64_t(1) << 20) || beams < 1 || beams > MQ_MAX_BEAMS) return 0;
  return (size_t)requests * beams * sizeof(mq::Copy);
}

extern "C" int mq_beam_reorder(const mq_kv_cache *caches, int count, int32_t *table, int64_t table_stride, int64_t max_pages,
                               const int32_t *lengths, const int32_t *parents, int64_t requests, int beams, void *scratch,
                               size_t scratch_bytes, void *stream) {
  using namespace mq;
  if (!caches || count < 1) return invalid("mq_beam_reorder: no caches");
  for (int i = 0; i < count; ++i) {
    if (const char *fault = cache_fault(caches + i)) return invalid(fault);
    if (caches[i].dtype != caches[0].dtype || caches[i].pages != caches[0].pages || caches[i].kv_heads != caches[0].kv_heads ||
        caches[i].head_dim != caches[0].head_dim || caches[i].page_tokens != caches[0].page_tokens)
      return invalid("mq_beam_reorder: the caches of a model's layers are alike");
    if ((caches[i].pages && !caches[i].data) || !aligned16(caches[i].data)) return invalid("mq_beam_reorder: a cache's data is NULL or misaligned");
  }
  if (requests < 0 || requests > (int64_t(1) << 20) || beams < 1 || beams > MQ_MAX_BEAMS) return invalid("mq_beam_reorder: 0 to 2^20 requests, 1 to 64 beams");
  if (max_pages < 0 || max_pages >= (int64_t(1) << 31) || table_stride < max_pages || table_stride >= (int64_t(1) << 40))
    return invalid("mq_beam_reorder: a table's rows are apart, of 0 to 2^31 pages");
  if (requests == 0 || beams == 1) return MQ_OK;
  if ((!table && max_pages) || !lengths || !parents || !scratch) return invalid("mq_beam_reorder: NULL pointer");
  if (scratch_bytes < mq_beam_reorder_scratch_size(requests, beams)) return invalid("mq_beam_reorder: too little scratch");
  if (!aligned_to(table, 4) || !aligned_to(lengths, 4) || !aligned_to(parents, 4) || !aligned_to(scratch, 16))
    return invalid("mq_beam_reorder: misaligned buffer");
  const mq_kv_cache &c = caches[0];
  const int tiles = c.page_tokens / kTileTokens, runs = (tiles + kCopyTiles - 1) / kCopyTiles;
  if (requests * runs >= (int64_t(1) << 24)) return invalid("mq_beam_reorder: too many requests");
  const hipStream_t s = static_cast<hipStream_t>(stream);
  Copy *const plan = static_cast<Copy *>(scratch);
  hipLaunchKernelGGL(plan_kernel, dim3((unsigned)requests), dim3(kPlanThreads), 0, s,
                     ReorderArgs{table, table_stride, max_pages, c.pages, lengths, parents, plan, beams, c.page_tokens});
  for (int from = 0; from < count; from += kMaxCaches) {
    CacheList list{};
    const int here = count - from < kMaxCaches ? count - from : kMaxCaches;
    for (int i = 0; i < here; ++i) list.data[i] = static_cast<uint8_t *>(caches[from + i].data);
    hipLaunchKernelGGL(copy_kernel, dim3((unsigned)(requests * runs), (unsigned)c.kv_heads, (unsigned)here), dim3(kCopyThreads), 0, s, list, plan, beams,
                       (uint32_t)(cache_tile_bytes(c.dtype, c.head_dim) / 16), tiles, runs);
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MQ_OK : set_error(MQ_E_HIP, hipGetErrorString(e));
}
