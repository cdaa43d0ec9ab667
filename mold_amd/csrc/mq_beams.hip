// mq_beams.hip — beam search over a decoder's logits and paged caches.
//
// mq_beam_select: of all continuations (beam b, token t) of a request the `count` with the
// largest score_b + log softmax(x_b)_t = score_b + (x - m) - log sum exp(x - m); within a beam
// logits decide, then the lower token, between beams the totals, then the lower beam; a beam
// that has ended has one, its stop token, at its score as it is.
//   The logits are read once: the bound is HBM for a batch, two launches for a request or
// two.  scan_kernel cuts each row into runs of a workgroup.  A wave keeps of its part the sum
// of exponentials, relative to a reference that follows the logits only where one passes it
// by more than 1, and those logits that reach a bar: the count-th largest of its lanes' maxima,
// which as many logits reach.  One comparison with the lower of the two finds what needs more
// than its exponential.  merge_kernel joins a request's runs, takes the totals in 64 bits,
// in which beams whose totals lie close compare as their logits say, and ranks them.  Where a
// request's logits are few, or the requests as many as the CUs, whole_kernel does all of it
// (takes_whole).
//   Exponentials are f32 (v_exp_f32 of differences, whose error shrinks with the term's weight),
// sums of 16 bytes of logits f32, of a lane and beyond f64: totals are good to some 2^-22.
//   512 rows of 128000 in f32, a fifth of them of ended beams, 210 MB: 49 us and 5.9 of joining;
// 80 rows of 151111 in bf16: 14.4 and 4.8, of which reading alone takes 8.6, exponentials 0.9, the
// bars 2, putting down and sorting 3; one request of 4 x 32000: 6.7 and 4.1, chains of dependent
// instructions behind one load.
//
// mq_beam_reorder: beam j of a request goes on from beam parents[j].  Whole pages are shared: a
// row of the page table takes its parent's entries.  The last, partial page goes to one child
// of each parent (to the parent's own row if it is one, else the first); every other child
// takes the page of a row without children, as many as there are, and has the tokens so far
// copied into it, in every layer's cache.  plan_kernel does the tables, copy_kernel moves the
// bytes, which bound it: those of the tiles (32 tokens) that the tokens reach, and no others.
// 64 x 8 beams in BF16, 28 layers, 1585 MB read and written: 300 us (5.3 TB/s) and 4.8 of
// planning; 8 x 4 beams in Q8_0, 51 MB: 11.6 and 4.1.
#include "../../include/moldq.h"
#include "mq_cache.h"

namespace mq {
int set_error(int code, const char *msg);
}

namespace mq {
namespace {

constexpr int kScanThreads = 256, kScanWaves = kScanThreads / 64;
constexpr int kMergeThreads = 512, kMergeWaves = kMergeThreads / 64;

// The wave's place in its workgroup, in a scalar register, so that what follows from it is not
// computed in every lane.
__device__ __forceinline__ int wave_index() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

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

// A permutation that gives every lane a value, so that no old one need be kept for it.
template <int kCtrl>
__device__ __forceinline__ uint32_t permuted(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, kCtrl, 0xf, 0xf, true);
}
// Lane i ^ kWith's value, by vector instructions alone (an LDS permutation takes ten times as long).
template <int kWith>
__device__ __forceinline__ uint32_t lane_xor(uint32_t x) {
  if constexpr (kWith == 1) return permuted<0xB1>(x);                 // quad_perm 1 0 3 2
  else if constexpr (kWith == 2) return permuted<0x4E>(x);            // quad_perm 2 3 0 1
  else if constexpr (kWith == 4) return permuted<0x1B>(permuted<0x141>(x));  // row_half_mirror, quad_perm 3 2 1 0
  else if constexpr (kWith == 8) return permuted<0x128>(x);           // row_ror 8
  else if constexpr (kWith == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return threadIdx.x & 16 ? r[0] : r[1];
  } else {
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return threadIdx.x & 32 ? r[0] : r[1];
  }
}
template <int kWith>
__device__ __forceinline__ uint64_t lane_xor(uint64_t v) {
  return ((uint64_t)lane_xor<kWith>((uint32_t)(v >> 32)) << 32) | lane_xor<kWith>((uint32_t)v);
}
template <int kWith>
__device__ __forceinline__ float lane_xor(float v) {
  return __uint_as_float(lane_xor<kWith>(__float_as_uint(v)));
}
template <int kWith>
__device__ __forceinline__ double lane_xor(double v) {
  return __longlong_as_double((int64_t)lane_xor<kWith>((uint64_t)__double_as_longlong(v)));
}
// The lane before's; 0 in lane 0.
__device__ __forceinline__ uint64_t lane_before(uint64_t v) {
  return ((uint64_t)permuted<0x138>((uint32_t)(v >> 32)) << 32) | permuted<0x138>((uint32_t)v);  // wave_shr 1
}
__device__ __forceinline__ uint64_t lane_of(uint64_t v, int lane) {
  return ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32) | (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}
// Lane i takes the larger (where `high`) or the smaller of its own and lane i ^ kWith's.
template <int kWith, typename K>
__device__ __forceinline__ K exchange(K v, bool high) {
  const K other = lane_xor<kWith>(v);
  return high == (v > other) ? v : other;
}
template <int kWith>
__device__ __forceinline__ uint32_t exchange(uint32_t v, bool high) {
  const uint32_t other = lane_xor<kWith>(v), most = max(v, other), least = min(v, other);
  return high ? most : least;
}
// A bitonic sequence sorted over runs of 2 kWith lanes, the largest first where `down`.
template <int kWith, typename K>
__device__ __forceinline__ K merged(K v, bool down) {
  v = exchange<kWith>(v, down == !(threadIdx.x & kWith));
  if constexpr (kWith > 1) return merged<kWith / 2>(v, down);
  return v;
}
// Sorted over the wave, the largest in lane 0.
template <typename K>
__device__ __forceinline__ K sorted(K v) {
  v = merged<1>(v, !(threadIdx.x & 2));
  v = merged<2>(v, !(threadIdx.x & 4));
  v = merged<4>(v, !(threadIdx.x & 8));
  v = merged<8>(v, !(threadIdx.x & 16));
  v = merged<16>(v, !(threadIdx.x & 32));
  return merged<32>(v, true);
}

// The largest keys that a wave has seen, one a lane, the largest in lane 0.
struct Largest {
  uint64_t key, least;  // `least`: nothing of it and below enters
  int count;
  bool any;

  __device__ __forceinline__ explicit Largest(int n) : key(0), least(0), count(n), any(false) {}
  // A key of each lane, or 0.  All lanes join.
  __device__ __forceinline__ void offer(uint64_t k) {
    uint64_t in = __ballot(k > least);
    if (!in) return;
    if (any && __popcll(in) <= 4) {
      const int lane = threadIdx.x & 63;
      do {
        const int from = __builtin_ctzll(in);
        in &= in - 1;
        const uint64_t one = lane_of(k, from);
        const int at = __popcll(__ballot(key > one));
        const uint64_t before = lane_before(key);
        key = lane < at ? key : lane == at ? one : before;
      } while (in);
      bound();
    } else {
      take(k > least ? k : 0);
    }
  }
  // The same however many enter.
  __device__ __forceinline__ void take(uint64_t k) {
    k = sorted(k);
    if (any) {
      // ascending, so that with the list it makes one bitonic sequence
      k = lane_xor<32>(lane_xor<16>(((uint64_t)permuted<0x140>((uint32_t)(k >> 32)) << 32) | permuted<0x140>((uint32_t)k)));  // row_mirror
      k = merged<32>(key > k ? key : k, true);
    }
    key = k;
    any = true;
    bound();
  }
  __device__ __forceinline__ void bound() {
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
  __device__ __forceinline__ static void get(const raw &r, float *x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = r[i];
  }
};
template <>
struct Vec<__bf16> {
  static constexpr int kN = 8;
  typedef uint32_t raw __attribute__((ext_vector_type(4), aligned(2)));
  __device__ __forceinline__ static void get(const raw &r, float *x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(r[i] << 16), x[2 * i + 1] = __uint_as_float(r[i] & 0xFFFF0000u);
  }
};

template <int kWith = 32>
__device__ __forceinline__ float wave_max(float v) {
  v = fmaxf(v, lane_xor<kWith>(v));
  if constexpr (kWith > 1) return wave_max<kWith / 2>(v);
  return v;
}
template <int kWith = 32>
__device__ __forceinline__ double wave_sum(double v) {
  v += lane_xor<kWith>(v);
  if constexpr (kWith > 1) return wave_sum<kWith / 2>(v);
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

// Keys that a wave may put down before they are sorted: those of one vector a lane beside 63.
template <typename X>
constexpr int kBuffer = 64 + 64 * Vec<X>::kN;

// What a wave keeps of the logits that it has seen.  Those that may be among the largest are
// put down in `buffer` and sorted 64 at a time, most often only once, with the other waves'
// at the end: putting each in its place at once is a chain of some 15 instructions that
// depend on each other (80 rows of 151111, the ten largest: 30 us, 22 now).  One place a vector
// sorts them, not one a logit, so that the code stays within the instruction cache.
struct Scan {
  Largest top;
  uint64_t *buffer;
  int held;            // in the buffer
  double sum;
  float ref, least;  // `least`: what a logit has to reach to be put down
  float enter;       // ..: for that or to move the reference
  float lane_most;

  __device__ __forceinline__ Scan(int count, uint64_t *b)
      : top(count), buffer(b), held(0), sum(0.), ref(-__FLT_MAX__), least(-__FLT_MAX__), enter(-__FLT_MAX__), lane_most(-__FLT_MAX__) {}

  // A logit of each lane.
  __device__ __forceinline__ void put(float x, uint32_t token) {
    const uint64_t k = x >= -__FLT_MAX__ ? key_of_logit(x, token) : 0, in = __ballot(k > top.least);
    if (!in) return;
    if (k > top.least) buffer[held + __builtin_amdgcn_mbcnt_hi((uint32_t)(in >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)in, 0))] = k;
    held += (int)__popcll(in);
  }
  // The reference follows the largest of the lanes' logits where that passes it by more than 1;
  // the sums so far with it.
  __device__ __forceinline__ void follow(float most) {
    if (!__any(most > ref + 1.f)) return;  // also where all are the lowest value, or NaN
    const float to = wave_max(most);
    sum *= (double)__builtin_amdgcn_exp2f((ref - to) * kLog2e);
    ref = to;
  }
  __device__ __forceinline__ void bounds() {
    least = top.least ? logit_of(top.least + 1) : -__FLT_MAX__;  // the least logit of a larger key
    enter = fminf(least, ref + 1.f);
  }
  // The lanes' maxima so far in the order of ordered(), the largest in lane 0.
  __device__ __forceinline__ uint32_t maxima() const { return sorted(ordered(lane_most >= -__FLT_MAX__ ? lane_most : -__FLT_MAX__)); }
  // The bar below which a logit need not enter: the count-th of them, which as many logits reach.
  __device__ __forceinline__ uint32_t bar(uint32_t of) const { return __builtin_amdgcn_readlane((int)of, top.count - 1); }
  __device__ __forceinline__ void raise(uint32_t to) {
    const uint64_t below = to > ordered(-__FLT_MAX__) ? ((uint64_t)to << 32) - 1 : 0;  // the key that all of it pass
    if (below > top.least) top.least = below;
    bounds();
  }
  template <int N>
  __device__ __forceinline__ static float most_of(const float *x) {
    float m = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) m = fmaxf(m, x[i]);
    return m;
  }
  // N logits of each lane, the largest of them `most`, tokens token .. token + N - 1; minus
  // infinity for none.
  template <int N>
  __device__ __forceinline__ void take(const float *x, float most, uint32_t token) {
    if (__any(most >= enter)) {
      follow(most);
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (__any(x[i] >= least)) put(x[i], token + i);
      if (held >= 64) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        do {
          held -= 64;
          top.take(buffer[held + (threadIdx.x & 63)]);
        } while (held >= 64);
      }
      bounds();
    }
    float s[N];
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = __builtin_amdgcn_exp2f((x[i] - ref) * kLog2e);
#pragma unroll
    for (int w = N / 2; w; w >>= 1)
#pragma unroll
      for (int i = 0; i < w; ++i) s[i] += s[i + w];
    sum += (double)s[0];
  }
};

// Part `part` of `parts` of a row, read by one wave.
template <typename X>
struct Reader {
  static constexpr int N = Vec<X>::kN, U = 4;
  typedef typename Vec<X>::raw raw;
  const X *row;
  int64_t v, to;  // in vectors
  int rest, held;
  raw next[U];
  float x[U][N], most[U];
  Scan scan;

  __device__ __forceinline__ Reader(const X *p, int64_t vocab, int64_t part, int64_t parts, int count, uint64_t *buffer) : row(p), scan(count, buffer) {
    const int64_t vectors = vocab / N;
    v = vectors * part / parts, to = vectors * (part + 1) / parts;
    rest = part == parts - 1 ? (int)(vocab - vectors * N) : 0;
    if (v < to) fetch(v);
  }
  __device__ __forceinline__ void fetch(int64_t at) {
    const raw *const body = reinterpret_cast<const raw *>(row);
#pragma unroll
    for (int u = 0; u < U; ++u) next[u] = body[min(at + 64 * u + (int)(threadIdx.x & 63), to - 1)];
  }
  __device__ __forceinline__ void unpack() {  // and what comes after it on its way
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int u = 0; u < U; ++u) Vec<X>::get(next[u], x[u]);
    if (v + 64 * U < to) {
      fetch(v + 64 * U);
    } else if (v + 64 * U > to) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < N; ++i) x[u][i] = v + 64 * u + lane < to ? x[u][i] : -__builtin_inff();
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      most[u] = Scan::most_of<N>(x[u]);
      scan.lane_most = fmaxf(scan.lane_most, most[u]);
    }
  }
  // The bar of the first logits; of several waves' that read one row the highest serves all.
  __device__ __forceinline__ uint32_t first() {
    if (v >= to) return 0;
    unpack();
    const uint32_t maxima = scan.maxima();
    scan.ref = logit_of((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)maxima) << 32);
    return scan.bar(maxima);
  }
  // Everything, given that bar: what is large is in the buffer then, `held` keys.
  __device__ __forceinline__ Run read(uint32_t bar) {
    const int lane = threadIdx.x & 63;
    scan.raise(bar);
    const int64_t tail = to;
    for (uint32_t turn = 1; v < to; ++turn) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (v + 64 * u < to) scan.take<N>(x[u], most[u], (uint32_t)((v + 64 * u + lane) * N));
      v += 64 * U;
      if (v >= to) break;
      unpack();
      // at each doubling: what enters between two is about the same; sooner the bar of all the waves serves
      if (turn > 1 && (turn & (turn - 1)) == 0) scan.raise(scan.bar(scan.maxima()));
    }
    if (rest) {
      const int64_t at = tail * N + lane;
      const float y = lane < rest ? (float)row[at] : -__builtin_inff();
      scan.take<1>(&y, y, (uint32_t)at);
    }
    held = scan.held;
    if (scan.top.any) {
      if (lane < scan.top.count) scan.buffer[held + lane] = scan.top.key;
      held += scan.top.count;
    }
    return {wave_sum(scan.sum), scan.ref};
  }
};

// What `waves` waves (up to 16) have put down, joined by one.
__device__ __forceinline__ Largest join(const uint64_t *buffers, int stride, const uint32_t *helds, int waves, int count) {
  const int lane = threadIdx.x & 63;
  Largest top(count);
  const int mine = lane < waves ? (int)helds[lane] : 0;
  int total = 0;
  for (int i = 0; i < waves; ++i) total += __builtin_amdgcn_readlane(mine, i);
  for (int first = 0; first < total; first += 64) {
    const int at = first + lane;
    int of = 0, from = 0, next = 0;
    for (int i = 1; i < waves; ++i) {
      next += __builtin_amdgcn_readlane(mine, i - 1);
      if (at >= next) of = i, from = next;
    }
    top.offer(at < total ? buffers[of * stride + at - from] : 0);
  }
  return top;
}

// One run of those that the lanes hold; a lane without one has sum 0 and the lowest reference.
__device__ __forceinline__ Run join(const Run &mine) {
  const float ref = wave_max(mine.ref);
  return {wave_sum(mine.sum * exp((double)mine.ref - (double)ref)), ref};
}

template <typename X>
__device__ __forceinline__ const X *row_of(const SelectArgs &a, int64_t n, int64_t beam) {
  return static_cast<const X *>(a.logits) + n * a.request + beam * a.beam;
}
// Whether a beam's logits matter.
__device__ __forceinline__ bool goes_on(const SelectArgs &a, int64_t row) { return !ended(a, row) && fabsf(a.scores[row]) <= __FLT_MAX__; }

// A workgroup a run of a row.
template <typename X>
__global__ __launch_bounds__(kScanThreads) void scan_kernel(SelectArgs a) {
  __shared__ Run runs[kScanWaves];
  __shared__ uint64_t buffers[kScanWaves][kBuffer<X>];
  __shared__ uint32_t bars[kScanWaves], helds[kScanWaves];
  const int64_t row = blockIdx.x / (uint32_t)a.splits, split = blockIdx.x - row * a.splits, n = row / a.beams;
  const int wave = wave_index(), lane = threadIdx.x & 63;
  Reader<X> reader(row_of<X>(a, n, row - n * a.beams), a.vocab, split * kScanWaves + wave, (int64_t)a.splits * kScanWaves, a.count, buffers[wave]);
  if (!goes_on(a, row)) return;
  uint32_t bar = reader.first();
  if (lane == 0) bars[wave] = bar;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kScanWaves; ++i) bar = max(bar, bars[i]);
  const Run run = reader.read(bar);
  if (lane == 0) runs[wave] = run, helds[wave] = reader.held;
  __syncthreads();
  if (wave) return;
  const Largest top = join(buffers[0], kBuffer<X>, helds, kScanWaves, a.count);
  const Run all = join(lane < kScanWaves ? runs[lane] : Run{0., -__FLT_MAX__});
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

// A request's candidates in LDS, [beams, count] and each beam's sorted.
struct Found {
  Candidate *all;
  int *ranks, *have;

  __device__ __forceinline__ Found(Candidate *lds, const SelectArgs &a) : all(lds), ranks(reinterpret_cast<int *>(lds + a.beams * a.count)), have(ranks + a.beams * a.count) {}
  // Beam b's, by one wave: `top` and `run` of its logits, which do not matter if it has ended.
  __device__ __forceinline__ void put(const SelectArgs &a, int64_t row, int b, const Largest &top, const Run &run) {
    const int lane = threadIdx.x & 63;
    const float score = a.scores[row];
    Candidate mine{0, -1};
    if (!(fabsf(score) <= __FLT_MAX__)) {
    } else if (ended(a, row)) {
      if (lane == 0) mine = {ordered64(score), a.stop};
    } else if (run.sum > 0. && run.sum <= __DBL_MAX__ && top.key) {
      mine = {ordered64((double)score + (((double)logit_of(top.key) - (double)run.ref) - log(run.sum))), (int64_t)token_of(top.key)};
    }
    if (lane < a.count) {
      all[b * a.count + lane] = mine;
      ranks[b * a.count + lane] = lane;
    }
    const uint64_t some = __ballot(lane < a.count && mine.total);
    if (lane == 0 && some) atomicAdd(have, (int)__popcll(some));
  }
  // The whole workgroup: every candidate counts those over it, of its own beam the ones before
  // it, of a lower beam those of no smaller total, of a higher one those of a larger.
  __device__ __forceinline__ void rank(const SelectArgs &a, int64_t n) {
    const int total = a.beams * a.count;
    for (int i = threadIdx.x; i < total * a.beams; i += blockDim.x) {  // a candidate, another beam
      const int b = i / total, c = i - b * total, of = c / a.count;
      const uint64_t mine = all[c].total;
      if (!mine || b == of) continue;
      int lo = 0, hi = a.count;  // how many of beam b's are over it
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        const uint64_t t = all[b * a.count + mid].total;
        if (t > mine || (b < of && t == mine)) lo = mid + 1;
        else hi = mid;
      }
      if (lo) atomicAdd(ranks + c, lo);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < total; i += blockDim.x) {
      const Candidate mine = all[i];
      if (!mine.total || ranks[i] >= a.count) continue;
      const int64_t to = n * a.count + ranks[i];
      a.out_scores[to] = (float)total_of(mine.total);
      a.parents[to] = i / a.count;
      a.tokens[to] = mine.token;
    }
    for (int i = *have + threadIdx.x; i < a.count; i += blockDim.x) {
      const int64_t to = n * a.count + i;
      a.out_scores[to] = -__builtin_inff();
      a.parents[to] = 0;
      a.tokens[to] = -1;
    }
  }
};
size_t found_bytes(int beams, int count) { return (sizeof(Candidate) + sizeof(int)) * beams * count + sizeof(int); }

// A workgroup a request: a wave joins a beam's runs at a time.
__global__ __launch_bounds__(kMergeThreads) void merge_kernel(SelectArgs a) {
  extern __shared__ Candidate lds[];
  Found found(lds, a);
  const int64_t n = blockIdx.x;
  const int wave = wave_index(), lane = threadIdx.x & 63;
  if (threadIdx.x == 0) *found.have = 0;
  __syncthreads();
  for (int b = wave; b < a.beams; b += kMergeWaves) {
    const int64_t row = n * a.beams + b;
    const uint64_t *const keys = a.keys + row * a.splits * a.count;
    auto key_at = [&](int at) -> uint64_t {  // the runs' largest first, then their second ones, ..: what comes later seldom enters
      const int rank = at / a.splits;
      return rank < a.count ? keys[(at - rank * a.splits) * a.count + rank] : 0;
    };
    const uint64_t first_key = key_at(lane);
    Run run{0., -__FLT_MAX__};
    if (lane < a.splits) run = a.runs[row * a.splits + lane];
    Largest top(a.count);
    if (goes_on(a, row)) {
      top.offer(first_key);
      for (int first = 64; first < a.splits * a.count; first += 64) top.offer(key_at(first + lane));
      run = join(run);
    }
    found.put(a, row, b, top, run);
  }
  __syncthreads();
  found.rank(a, n);
}

// A workgroup a request that does all of it, `each` waves a beam.
constexpr int kWholeThreads = 512, kWholeWaves = kWholeThreads / 64;
template <typename X>
__global__ __launch_bounds__(kWholeThreads) void whole_kernel(SelectArgs a, int each) {
  extern __shared__ Candidate lds[];
  __shared__ Run runs[kWholeWaves];
  __shared__ uint64_t buffers[kWholeWaves][kBuffer<X>];
  __shared__ uint32_t bars[kWholeWaves], helds[kWholeWaves];
  Found found(lds, a);
  const int64_t n = blockIdx.x;
  const int wave = wave_index(), lane = threadIdx.x & 63, b = wave / each, part = wave - b * each;
  const int64_t row = n * a.beams + b;
  const bool is = b < a.beams, reads = is && goes_on(a, row);
  if (threadIdx.x == 0) *found.have = 0;
  Reader<X> reader(row_of<X>(a, n, is ? b : 0), reads ? a.vocab : 0, part, each, a.count, buffers[wave]);
  uint32_t bar = reader.first();
  if (lane == 0) bars[wave] = bar;
  __syncthreads();
  if (reads) {
    for (int i = 0; i < each; ++i) bar = max(bar, bars[wave - part + i]);
    const Run run = reader.read(bar);
    if (lane == 0) runs[wave] = run, helds[wave] = reader.held;
  }
  __syncthreads();
  if (is && part == 0) {
    Largest top(a.count);
    Run run{0., -__FLT_MAX__};
    if (reads) {
      top = join(buffers[wave], kBuffer<X>, helds + wave, each, a.count);
      if (lane < each) run = runs[wave + lane];
      run = join(run);
    }
    found.put(a, row, b, top, run);
  }
  __syncthreads();
  found.rank(a, n);
}

// ------------------------------------------------------------------ reordering

constexpr int kMaxCaches = 256, kMaxRequests = 1024;  // of a launch of copy_kernel
struct Copy {
  int32_t from, to;  // pages
};
struct Copies {
  int32_t count, tiles;  // of a request, and how many tiles of each page and head
};
struct CacheList {
  uint8_t *data[kMaxCaches];
};
// What plan_kernel leaves to copy_kernel.  The caches' addresses are there too: read from the
// launch's arguments, host memory, by every workgroup they cost more than the copies of a few
// requests.
struct Plan {
  CacheList *caches;
  Copies *requests;
  Copy *copies;  // [requests, beams], the first `count` of each
};

struct ReorderArgs {
  int32_t *table;
  int64_t stride, width, pages;
  const int32_t *lengths;  // [requests, beams], the first of a request read
  const int32_t *parents;  // [requests, beams]
  Plan plan;
  int beams, page;
};

constexpr int kPlanThreads = 256, kPlanColumns = 64;
static_assert(kPlanThreads >= kMaxCaches);  // a thread passes on each address

// Workgroups (request, y): the first of a request's plans, all take every gridDim.y-th part of its
// columns of whole pages.  Lane j of a workgroup's first wave is beam j.
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(ReorderArgs a, CacheList caches, int count) {
  if (blockIdx.x == 0 && blockIdx.y == 0 && (int)threadIdx.x < count) a.plan.caches->data[threadIdx.x] = caches.data[threadIdx.x];
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
  if (blockIdx.y == 0 && threadIdx.x < 64) {
    const int j = threadIdx.x;
    bool copied = false;
    int from = 0, to = 0;
    if (j < a.beams && tail && full < a.width && moves) {
      from = a.table[(row0 + parent[j]) * a.stride + full];
      to = a.table[(row0 + taken[j]) * a.stride + full];
      copied = taken[j] != parent[j] && from >= 0 && from < a.pages && to >= 0 && to < a.pages;
      entries[j] = to;
    }
    const uint64_t all = __ballot(copied);
    if (copied) a.plan.copies[row0 + __popcll(all & (((uint64_t)1 << j) - 1))] = {from, to};
    if (j == 0) a.plan.requests[blockIdx.x] = {(int32_t)__popcll(all), (tail + kTileTokens - 1) / kTileTokens};
  }
  if (!moves) return;
  __syncthreads();
  if (blockIdx.y == 0 && tail && full < a.width && threadIdx.x < a.beams) a.table[(row0 + threadIdx.x) * a.stride + full] = entries[threadIdx.x];
  const int64_t columns = min((int64_t)full, a.width);
  for (int64_t c0 = (int64_t)blockIdx.y * kPlanColumns; c0 < columns; c0 += (int64_t)gridDim.y * kPlanColumns) {
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

// Workgroups (x, cache), as many as fill the chip whatever the requests' shares are, each every
// gridDim.x-th tile of what is copied in the cache.  64 x 8 beams: 305 us, 366 with a workgroup a
// (request, head, cache), 365 with all heads of a page copied on one XCD; of a quarter as many
// workgroups 323, of twice as many 302.  Its loads stand behind no branch: with one 8 x 4 beams
// took 27 us instead of 16.
constexpr int kCopyThreads = 256;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
template <int T, int D>
__global__ __launch_bounds__(kCopyThreads) void copy_kernel(Plan plan, int requests, int beams, int kv_heads, int tiles) {
  constexpr int kUnits = CacheTile<T, D>::kBytes / 16, kPer = kMaxRequests / kCopyThreads, U = (kUnits + kCopyThreads - 1) / kCopyThreads;
  __shared__ uint32_t before[kMaxRequests], sums[kCopyThreads / 64];
  u32x4 *const data = reinterpret_cast<u32x4 *>(plan.caches->data[blockIdx.y]);
  const int tid = threadIdx.x, wave = wave_index(), lane = tid & 63;
  uint32_t mine[kPer], sum = 0;  // the tiles, of one head, of the requests before
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int r = tid * kPer + i;
    mine[i] = sum;
    if (r < requests) {
      const Copies c = plan.requests[r];
      sum += c.count * c.tiles;
    }
  }
  uint32_t upto = sum;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint32_t u = __shfl_up(upto, off);
    if (lane >= off) upto += u;
  }
  if (lane == 63) sums[wave] = upto;
  __syncthreads();
  uint32_t start = upto - sum, all = 0;
#pragma unroll
  for (int i = 0; i < kCopyThreads / 64; ++i) {
    if (i < wave) start += sums[i];
    all += sums[i];
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) before[tid * kPer + i] = start + mine[i];
  __syncthreads();
  const uint64_t units = (uint64_t)all * kv_heads;
  for (uint64_t unit = blockIdx.x; unit < units; unit += gridDim.x) {
    const uint32_t t = units >> 32 ? (uint32_t)(unit / kv_heads) : (uint32_t)unit / (uint32_t)kv_heads, head = (uint32_t)(unit - (uint64_t)t * kv_heads);
    // the last request that starts at or before t (those without copies start where the next does)
    const int row = __popcll(__ballot(lane < kMaxRequests / 64 && before[(lane & (kMaxRequests / 64 - 1)) * 64] <= t)) - 1;
    const int r = row * 64 + __popcll(__ballot(before[row * 64 + lane] <= t)) - 1;
    const uint32_t of = (uint32_t)plan.requests[r].tiles, in = t - before[r], c = in / of, tile = in - c * of;
    const Copy copy = plan.copies[(int64_t)r * beams + c];
    const u32x4 *const from = data + (((int64_t)copy.from * kv_heads + head) * tiles + tile) * kUnits;
    u32x4 *const to = data + (((int64_t)copy.to * kv_heads + head) * tiles + tile) * kUnits;
    u32x4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = from[min(u * kCopyThreads + tid, kUnits - 1)];  // none behind a branch, which would wait for the one before
#pragma unroll
    for (int u = 0; u < U; ++u)
      if ((u + 1) * kCopyThreads <= kUnits || u * kCopyThreads + tid < kUnits) to[u * kCopyThreads + tid] = v[u];
  }
}

int invalid(const char *msg) { return set_error(MQ_E_INVALID, msg); }
bool aligned_to(const void *p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// Runs of a row: no more workgroups than four on each of 256 CUs, as many as can be there at once in
// bf16 (registers); none of fewer than 4096 logits (16 a thread), 64 at most (a lane each when
// they are joined).  In a graph, with joining: 80 rows of 151111 in bf16 18.3 us with 960 workgroups, 20.0
// with 1040, whose last start when others end, 19.3 with 1600, 18.6 with 480; 512 rows of 128000
// in f32 59.6 with 1024, 63.3 with 2048, 63.6 with 512.
int splits_of(int64_t rows, int64_t vocab) {
  const int64_t want = 1024 / rows, most = vocab / 4096, s = want < most ? want : most;
  return (int)(s < 1 ? 1 : s > 64 ? 64 : s);
}

// Whether a workgroup a request reads all its logits, which spares a launch and the scratch:
// where a wave has 16 KB of them at most, or where the requests are as many as the CUs and no wave
// is left over.  Against two launches, 4 beams in f32: 1 to 384 requests of 1000 to 4000 tokens
// 12 to 15 us against 16, of 8000 12 to 20 against 16 to 21, one of 16000 17 against 16; 5000 of 1000
// 58 against 84; 256 to 2048 of 32000 35 to 186 against 37 to 199.  With 5 beams, three of eight waves
// idle, 256 of 32000 53 against 42.
bool takes_whole(int64_t requests, int beams, int64_t vocab, int dtype) {
  if (beams > kWholeWaves) return false;
  return vocab * (dtype == MQ_F32 ? 4 : 2) <= (16 << 10) * (kWholeWaves / beams) || (requests >= 256 && kWholeWaves % beams == 0);
}

const char *select_fault(int64_t n, int beams, int64_t vocab, int count) {
  if (n < 0 || n > (int64_t(1) << 20)) return "mq_beam_select: 0 to 2^20 requests";
  if (beams < 1 || beams > MQ_MAX_BEAMS || count < 1 || count > MQ_MAX_BEAMS) return "mq_beam_select: 1 to 64 beams and continuations";
  // a launch's threads are counted in 32 bits, and where there are more than 1024 rows a workgroup of 256 takes one
  if (n * beams >= (int64_t(1) << 24)) return "mq_beam_select: fewer than 2^24 rows of logits (requests * beams)";
  if (vocab < 1 || vocab >= (int64_t(1) << 31)) return "mq_beam_select: a vocabulary of 1 to 2^31 tokens";
  return nullptr;
}

}  // namespace
}  // namespace mq

extern "C" size_t mq_beam_select_scratch_size(int64_t requests, int beams, int64_t vocab, int count, int dtype) {
  using namespace mq;
  if (requests == 0 || select_fault(requests, beams, vocab, count) || (dtype != MQ_F32 && dtype != MQ_BF16)) return 0;
  const int64_t rows = requests * beams;
  if (takes_whole(requests, beams, vocab, dtype)) return 0;
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
  const size_t need = mq_beam_select_scratch_size(requests, beams, vocab, count, dtype);
  if (!logits || !scores || !out_scores || !parents || !tokens || (need && !scratch)) return invalid("mq_beam_select: NULL pointer");
  if (scratch_bytes < need) return invalid("mq_beam_select: too little scratch");
  if (!aligned_to(logits, dtype == MQ_F32 ? 4 : 2) || !aligned_to(scores, 4) || !aligned_to(out_scores, 4) || !aligned_to(parents, 4) ||
      !aligned_to(last, 8) || !aligned_to(tokens, 8) || !aligned_to(scratch, 16))
    return invalid("mq_beam_select: misaligned buffer");
  const int64_t rows = requests * beams;
  const int splits = need ? splits_of(rows, vocab) : 1;
  Run *const runs = static_cast<Run *>(scratch);
  const SelectArgs a{logits, request_stride, beam_stride, vocab, requests, scores, last, stop, beams, count, splits, runs,
                     reinterpret_cast<uint64_t *>(runs + rows * splits), out_scores, parents, tokens};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const size_t lds = found_bytes(beams, count);
  auto launch = [&]<typename X>() {
    if (need) {
      hipLaunchKernelGGL(scan_kernel<X>, dim3((unsigned)(rows * splits)), dim3(kScanThreads), 0, s, a);
      hipLaunchKernelGGL(merge_kernel, dim3((unsigned)requests), dim3(kMergeThreads), lds, s, a);
    } else {
      hipLaunchKernelGGL(whole_kernel<X>, dim3((unsigned)requests), dim3(kWholeThreads), lds, s, a, kWholeWaves / beams);
    }
  };
  if (dtype == MQ_F32) launch.operator()<float>();
  else launch.operator()<__bf16>();
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MQ_OK : set_error(MQ_E_HIP, hipGetErrorString(e));
}

extern "C" size_t mq_beam_reorder_scratch_size(int64_t requests, int beams) {
  using namespace mq;
  if (requests < 0 || requests > (int64_t(1) << 20) || beams < 1 || beams > MQ_MAX_BEAMS) return 0;
  return sizeof(CacheList) + (size_t)requests * (sizeof(Copies) + beams * sizeof(Copy));
}

extern "C" int mq_beam_reorder(const mq_kv_cache *caches, int count, int32_t *table, int64_t table_stride, int64_t max_pages,
                               const int32_t *lengths, const int32_t *parents, int64_t requests, int beams, void *scratch,
                               size_t scratch_bytes, void *stream) {
  using namespace mq;
  if (!caches || count < 1 || count > kMaxCaches) return invalid("mq_beam_reorder: 1 to 256 caches");
  CacheList list{};
  for (int i = 0; i < count; ++i) {
    if (const char *fault = cache_fault(caches + i)) return invalid(fault);
    if (caches[i].dtype != caches[0].dtype || caches[i].pages != caches[0].pages || caches[i].kv_heads != caches[0].kv_heads ||
        caches[i].head_dim != caches[0].head_dim || caches[i].page_tokens != caches[0].page_tokens)
      return invalid("mq_beam_reorder: the caches of a model's layers are alike");
    if ((caches[i].pages && !caches[i].data) || !aligned_to(caches[i].data, 16)) return invalid("mq_beam_reorder: a cache's data is NULL or misaligned");
    list.data[i] = static_cast<uint8_t *>(caches[i].data);
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
  const int tiles = c.page_tokens / kTileTokens;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  Copies *const of = reinterpret_cast<Copies *>(static_cast<CacheList *>(scratch) + 1);
  const Plan plan{static_cast<CacheList *>(scratch), of, reinterpret_cast<Copy *>(of + requests)};
  // a workgroup for each kPlanColumns columns, while there are fewer than fill the chip.  4 requests of 64 beams
  // over 31 250 whole pages: a call of 21 us, 3190 with a workgroup a request.
  const int64_t parts = (max_pages + kPlanColumns - 1) / kPlanColumns, most_parts = 2048 / requests;
  const unsigned part = (unsigned)(parts < most_parts ? (parts ? parts : 1) : most_parts ? most_parts : 1);
  hipLaunchKernelGGL(plan_kernel, dim3((unsigned)requests, part), dim3(kPlanThreads), 0, s,
                     ReorderArgs{table, table_stride, max_pages, c.pages, lengths, parents, plan, beams, c.page_tokens}, list, count);
  for (int64_t first = 0; first < requests; first += kMaxRequests) {
    const int here = (int)(requests - first < kMaxRequests ? requests - first : kMaxRequests);
    // sixteen workgroups for each of 256 CUs, or as many as there can be tiles to copy
    const int64_t most = (int64_t)here * (beams - 1) * tiles * c.kv_heads, fill = (4096 + count - 1) / count;
    with_cache_type(&c, [&]<int T, int D>() {
      hipLaunchKernelGGL((copy_kernel<T, D>), dim3((unsigned)(most < fill ? most : fill), (unsigned)count), dim3(kCopyThreads), 0, s,
                         Plan{plan.caches, plan.requests + first, plan.copies + first * beams}, here, beams, c.kv_heads, tiles);
    });
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MQ_OK : set_error(MQ_E_HIP, hipGetErrorString(e));
}
