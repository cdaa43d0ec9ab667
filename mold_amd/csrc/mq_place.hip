// mq_place.hip — page tables, slots and positions of packed sequences, made on the GPU from
// their lengths: mq_cache_place for prompts that start, mq_cache_extend for sequences
// that go on over the pages they have.
//
//   shared_i = beams > 1 ? floor(count_i / page) : 0       pages of i that all its beams read
//   columns_i = min(ceil((count_i + room) / page), width)  pages of each beam
//   need_i = shared_i + beams (columns_i - shared_i)        first_i = need_0 + .. + need_(i-1)
//   table[i beams + j, c] = pages[first_i + (c < shared_i ? c : shared_i + j (columns_i - shared_i) + c - shared_i)]
//   token at offset p of i: position p, slot table[i beams, p / page] page + p % page
//
// There is next to nothing to move (16 bytes a token, 4 a table entry) and nothing to
// compute but two prefix sums over the sequences, so the launch is the cost, and there is
// one: every workgroup takes the sums over all sequences itself (a window of 1024 at a
// time, of which a batch has one), rather than wait for another launch or workgroup that
// did.  Where that is many windows (summed), a launch before takes each one's sums, which wait in
// entries of `lengths` that a launch after sets.  A slot comes from the formula and not from
// the table, which is being written.
// 24 prompts (7305 tokens) take 6.0 us, 256 with four beams (163 000 tokens, 38 000 table
// entries) 6.7, one token each of 200 sequences 3.5, of which a launch of nothing is 2.
#include "../../include/moldq.h"
#include "mq_cache.h"

namespace mq {
int set_error(int code, const char *msg);
}

namespace mq {
namespace {

constexpr int kPlaceThreads = 256, kPer = 4, kWindow = kPlaceThreads * kPer;
constexpr int kBlockTokens = 1024;  // tokens of a workgroup
constexpr int kBlockEntries = 4096; // table entries of a workgroup
// Windows of more than these are summed beforehand.  In a graph, prompts of 20 tokens: 2048 of them 8.4 us, 12.1
// with the sums; 4096 14.0 and 14.2; 8192 29.8 and 18.4; 65536 233 and 25.  Sequences that go on, which need
// the tokens' sums alone: 9.4 and 11.4, 14.6 and 12.3, 103 and 18.  A call for 2^20 prompts 43, 190 000.
constexpr int kSummed = 4;
constexpr uint32_t kMost = 0x7FFFFFFFu;

struct PlaceArgs {
  const int32_t *counts, *held;  // counts NULL: one token each; held NULL: prompts that start
  const int32_t *pages;          // NULL: 0, 1, ..
  int32_t *table;
  int64_t n, tokens, width, stride, page_count, cache_pages;
  int64_t *slots, *positions, *last;
  int32_t *lengths;
  uint32_t room, page;
  int beams;
  uint32_t per, slices;  // sequences whose table rows are shared by workgroups, and by how many
  bool summed;
};

// Sums stop at kMost, so that counts that mean nothing cannot wrap them.
__device__ __forceinline__ uint32_t add_capped(uint32_t a, uint32_t b) { return min(a + b, kMost); }

struct Need {
  uint32_t count, shared, columns, pages;
  __device__ Need(const PlaceArgs &a, int64_t i) : count(0), shared(0), columns(0), pages(0) {
    if (i >= a.n) return;
    count = a.counts ? (uint32_t)max(a.counts[i], 0) : 1;
    if (a.held) return;
    const uint32_t most = (uint32_t)min(a.width, (int64_t)kMost);
    columns = min((count + a.room) / a.page + ((count + a.room) % a.page != 0), most);
    shared = a.beams > 1 ? min(count / a.page, columns) : 0;
    const uint64_t need = shared + (uint64_t)a.beams * (columns - shared);
    pages = (uint32_t)min(need, (uint64_t)kMost);
  }
};

// Before each sequence of the window that starts at `from`: the tokens and pages of all
// sequences before it, given those before the window; after it those of the window's too.
struct Window {
  uint32_t tokens[kWindow + 1], pages[kWindow];
};
template <typename F>  // of(i): tokens and pages of the window's i-th
__device__ __forceinline__ void scan(const F &of, uint32_t &tokens, uint32_t &pages, Window &w, uint32_t (*sums)[2]) {
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  uint32_t t[kPer], p[kPer], at = 0, ap = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const uint2 need = of(tid * kPer + i);
    t[i] = at, p[i] = ap;
    at = add_capped(at, need.x), ap = add_capped(ap, need.y);
  }
  uint32_t st = at, sp = ap;  // over the lanes up to this one
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint32_t ut = __shfl_up(st, off), up = __shfl_up(sp, off);
    if (lane >= off) st = add_capped(st, ut), sp = add_capped(sp, up);
  }
  __syncthreads();  // the window before has been read
  if (lane == 63) sums[wave][0] = st, sums[wave][1] = sp;
  uint32_t bt = __shfl_up(st, 1), bp = __shfl_up(sp, 1);
  if (lane == 0) bt = bp = 0;
  __syncthreads();
  uint32_t all_t = tokens, all_p = pages;
  bt = add_capped(tokens, bt), bp = add_capped(pages, bp);
#pragma unroll
  for (int i = 0; i < kPlaceThreads / 64; ++i) {
    if (i < wave) bt = add_capped(bt, sums[i][0]), bp = add_capped(bp, sums[i][1]);
    all_t = add_capped(all_t, sums[i][0]), all_p = add_capped(all_p, sums[i][1]);
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    w.tokens[tid * kPer + i] = add_capped(bt, t[i]);
    w.pages[tid * kPer + i] = add_capped(bp, p[i]);
  }
  if (tid == 0) w.tokens[kWindow] = all_t;
  tokens = all_t, pages = all_p;
  __syncthreads();
}
__device__ __forceinline__ void scan_window(const PlaceArgs &a, int64_t from, uint32_t &tokens, uint32_t &pages, Window &w, uint32_t (*sums)[2]) {
  scan([&](int i) {
    const Need need(a, from + i);
    return make_uint2(need.count, need.pages);
  }, tokens, pages, w, sums);
}
// The last of the window's (below 1024) that starts at or before t and, if t is inside, holds it.
__device__ __forceinline__ int holder(const Window &w, int64_t t) {
  int at = 0;
#pragma unroll
  for (int step = kWindow / 2; step; step >>= 1)
    if (w.tokens[at + step] <= t) at += step;
  return at;
}

// Where a window's sums wait, of all windows but the last: the first two entries of its
// sequences' lengths.
__device__ __forceinline__ int64_t sums_at(const PlaceArgs &a, int64_t window) { return window * kWindow * a.beams; }
__device__ __forceinline__ int64_t last_window(const PlaceArgs &a) { return (a.n - 1) / kWindow; }
__device__ __forceinline__ int32_t length_of(const PlaceArgs &a, int64_t i, uint32_t count) {
  return (int32_t)(a.held ? min((int64_t)a.held[i] + count, (int64_t)kMost) : count);
}
// A workgroup a window but the last.
__global__ __launch_bounds__(kPlaceThreads) void sum_windows(PlaceArgs a) {
  __shared__ uint32_t sums[kPlaceThreads / 64][2];
  const int tid = threadIdx.x;
  uint32_t t = 0, p = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const Need need(a, (int64_t)blockIdx.x * kWindow + i * kPlaceThreads + tid);
    t = add_capped(t, need.count), p = add_capped(p, need.pages);
  }
#pragma unroll
  for (int off = 32; off; off >>= 1) t = add_capped(t, __shfl_xor(t, off)), p = add_capped(p, __shfl_xor(p, off));
  if ((tid & 63) == 0) sums[tid >> 6][0] = t, sums[tid >> 6][1] = p;
  __syncthreads();
  if (tid >= 2) return;
  uint32_t all = 0;
#pragma unroll
  for (int i = 0; i < kPlaceThreads / 64; ++i) all = add_capped(all, sums[i][tid]);
  a.lengths[sums_at(a, blockIdx.x) + tid] = (int32_t)all;
}
// The lengths where the sums were.
__global__ __launch_bounds__(kPlaceThreads) void put_lengths(PlaceArgs a) {
  const int64_t e = (int64_t)blockIdx.x * kPlaceThreads + threadIdx.x, at = sums_at(a, e >> 1) + (e & 1), i = at / a.beams;
  if (e >> 1 < last_window(a)) a.lengths[at] = length_of(a, i, Need(a, i).count);
}

// Page `at` of those to take, or -1.
__device__ __forceinline__ int32_t page_at(const PlaceArgs &a, int64_t at) {
  if (at >= a.page_count) return -1;
  const int32_t page = a.pages ? a.pages[at] : (int32_t)at;
  return page >= 0 && page < a.cache_pages ? page : -1;
}

// A token's slot and position: offset `in` of sequence i, whose first page is `first`.
__device__ __forceinline__ void put_token(const PlaceArgs &a, int64_t t, int64_t i, uint32_t in, uint32_t first) {
  const int64_t position = in + (a.held ? (int64_t)a.held[i] : 0);  // below 2^32
  const uint32_t column = (uint32_t)position / a.page;
  int32_t page = -1;
  if (position >= 0 && column < a.width) {
    page = a.held ? a.table[i * a.stride + column] : page_at(a, (int64_t)first + column);  // beam 0's, whose own pages follow the shared ones
    if (page >= a.cache_pages) page = -1;
  }
  a.positions[t] = position;
  a.slots[t] = page < 0 ? -1 : (int64_t)page * a.page + ((uint32_t)position - column * a.page);
}

// Workgroups 0 .. rows - 1 write table rows, every `slices` of them those of `per` sequences, and the
// first of these their lengths and last rows; the others write kBlockTokens tokens' slots and positions.
__global__ __launch_bounds__(kPlaceThreads) void place_kernel(PlaceArgs a, uint32_t rows) {
  __shared__ Window w;
  __shared__ uint32_t sums[kPlaceThreads / 64][2];
  const int tid = threadIdx.x;
  uint32_t tokens = 0, pages = 0;
  int64_t from = 0;
  // the sums before the window in which to start, given as one that the windows' sums are known of
  auto start = [&](auto window_of) {
    if (!a.summed) return;
    const int64_t last = last_window(a);
    scan([&](int i) { return i < last ? make_uint2((uint32_t)a.lengths[sums_at(a, i)], (uint32_t)a.lengths[sums_at(a, i) + 1]) : make_uint2(0, 0); },
         tokens, pages, w, sums);
    const int window = (int)min(window_of(), last);
    from = (int64_t)window * kWindow, tokens = w.tokens[window], pages = w.pages[window];
  };
  if (blockIdx.x < rows) {
    const uint32_t group = blockIdx.x / a.slices, slice = blockIdx.x - group * a.slices;
    const int64_t first = (int64_t)group * a.per, end = min(a.n, first + a.per);
    if (!a.held) {
      start([&] { return first / kWindow; });
      for (;; from += kWindow) {  // kWindow is a multiple of a.per: the sequences lie in one window
        scan_window(a, from, tokens, pages, w, sums);
        if (first < from + kWindow) break;
      }
    }
    if (slice == 0)
      for (int64_t i = first + tid; i < end; i += kPlaceThreads) {
        const Need need(a, i);
        const int32_t length = length_of(a, i, need.count);
        const int64_t kept = a.summed && i / kWindow < last_window(a) ? sums_at(a, i / kWindow) + 2 : 0;  // before it sums wait
        for (int j = 0; j < a.beams; ++j)
          if (i * a.beams + j >= kept) a.lengths[i * a.beams + j] = length;
        if (!a.held) {
          const int64_t at = (int64_t)w.tokens[i - from] + need.count - 1;
          a.last[i] = need.count == 0 || at >= a.tokens ? -1 : at;
        }
      }
    if (a.held || a.width == 0) return;
    const uint32_t width = (uint32_t)a.width, beams = (uint32_t)a.beams;
    const uint64_t entries = (uint64_t)(end - first) * beams * width;
#pragma unroll 4
    for (uint64_t e = slice * kPlaceThreads + tid; e < entries; e += a.slices * kPlaceThreads) {
      const uint32_t row = entries >> 32 ? (uint32_t)(e / width) : (uint32_t)e / width, c = (uint32_t)(e - (uint64_t)row * width);
      const uint32_t i = row / beams, j = row - i * beams;
      const Need need(a, first + i);
      const int64_t own = need.columns - need.shared;
      a.table[((first + i) * beams + j) * a.stride + c] =
          c < need.columns ? page_at(a, w.pages[first + i - from] + (c < need.shared ? c : c + j * own)) : -1;
    }
    return;
  }
  const int64_t t0 = (int64_t)(blockIdx.x - rows) * kBlockTokens, t1 = min(a.tokens, t0 + kBlockTokens);
  if (!a.counts) {  // a token each
    for (int64_t t = t0 + tid; t < t1; t += kPlaceThreads) {
      if (t < a.n) put_token(a, t, t, 0, 0);
      else a.slots[t] = -1, a.positions[t] = 0;
    }
    return;
  }
  start([&] { return (int64_t)holder(w, t0); });
  for (; from < a.n; from += kWindow) {
    const uint32_t before = tokens;
    scan_window(a, from, tokens, pages, w, sums);
    const int64_t lo = max(t0, (int64_t)before), hi = min(t1, (int64_t)tokens);
    for (int64_t t = lo + tid; t < hi; t += kPlaceThreads) {
      const int at = holder(w, t);
      put_token(a, t, from + at, (uint32_t)(t - w.tokens[at]), w.pages[at]);
    }
    if (tokens >= t1) return;
  }
  for (int64_t t = max(t0, (int64_t)tokens) + tid; t < t1; t += kPlaceThreads) a.slots[t] = -1, a.positions[t] = 0;
}

int invalid(const char *msg) { return set_error(MQ_E_INVALID, msg); }
bool aligned_to(const void *p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// 4 prompts with 64 beams of 2004 pages, 513 000 table entries: a call of 13.7 us, 905 with one workgroup
// for every four sequences' rows, however many entries these have.
int launch_place(PlaceArgs a, void *stream) {
  const hipStream_t s = static_cast<hipStream_t>(stream);
  for (a.per = 4; a.per < kWindow && a.n > (int64_t)a.per * 2048;) a.per *= 2;
  const int64_t groups = (a.n + a.per - 1) / a.per, entries = a.held ? 0 : min(a.n, (int64_t)a.per) * a.beams * a.width;
  const int64_t slices = (entries + kBlockEntries - 1) / kBlockEntries, most = groups ? (int64_t(1) << 20) / groups : 1;  // a launch has so many workgroups at most
  a.slices = (uint32_t)(slices < 1 ? 1 : slices < most ? slices : most);
  const int64_t rows = groups * a.slices, blocks = rows + (a.tokens + kBlockTokens - 1) / kBlockTokens;
  if (blocks == 0) return MQ_OK;
  const int64_t windows = (a.n + kWindow - 1) / kWindow;
  a.summed = a.counts && windows > kSummed;
  if (a.summed) hipLaunchKernelGGL(sum_windows, dim3((unsigned)windows - 1), dim3(kPlaceThreads), 0, s, a);
  hipLaunchKernelGGL(place_kernel, dim3((unsigned)blocks), dim3(kPlaceThreads), 0, s, a, (uint32_t)rows);
  if (a.summed) hipLaunchKernelGGL(put_lengths, dim3((unsigned)((2 * (windows - 1) + kPlaceThreads - 1) / kPlaceThreads)), dim3(kPlaceThreads), 0, s, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MQ_OK : set_error(MQ_E_HIP, hipGetErrorString(e));
}

const char *place_fault(const mq_kv_cache *c, int64_t n, int64_t tokens, int64_t width, int64_t stride, int64_t rows) {
  if (const char *fault = cache_fault(c)) return fault;
  if (n < 0 || n > (int64_t(1) << 20)) return "placing tokens: 0 to 2^20 sequences";
  if (tokens < 0 || tokens >= (int64_t(1) << 31)) return "placing tokens: tokens outside 0 .. 2^31";
  if (width < 0 || width >= (int64_t(1) << 31) || stride < (rows > 1 ? width : 0) || stride >= (int64_t(1) << 40))
    return "placing tokens: a table's rows are apart, of 0 to 2^31 pages";
  return nullptr;
}

}  // namespace
}  // namespace mq

extern "C" int mq_cache_place(const mq_kv_cache *c, const int32_t *counts, int64_t sequences, int beams, int64_t room,
                              const int32_t *pages, int64_t page_count, int32_t *table, int64_t table_stride, int64_t max_pages,
                              int64_t tokens, int64_t *slots, int64_t *positions, int32_t *lengths, int64_t *last, void *stream) {
  using namespace mq;
  if (beams < 1 || beams > MQ_MAX_BEAMS) return invalid("mq_cache_place: 1 to 64 beams");
  if (const char *fault = place_fault(c, sequences, tokens, max_pages, table_stride, sequences * beams)) return invalid(fault);
  if (room < 0 || room >= (int64_t(1) << 31)) return invalid("mq_cache_place: room outside 0 .. 2^31");
  if (page_count < 0 || page_count >= (int64_t(1) << 31)) return invalid("mq_cache_place: 0 to 2^31 pages");
  if ((sequences && (!counts || !lengths || !last || (!table && max_pages))) || (tokens && (!slots || !positions)))
    return invalid("mq_cache_place: NULL pointer");
  if (!aligned_to(counts, 4) || !aligned_to(pages, 4) || !aligned_to(table, 4) || !aligned_to(lengths, 4) || !aligned_to(slots, 8) ||
      !aligned_to(positions, 8) || !aligned_to(last, 8))
    return invalid("mq_cache_place: misaligned buffer");
  return launch_place({counts, nullptr, pages, table, sequences, tokens, max_pages, table_stride, page_count, c->pages, slots,
                       positions, last, lengths, (uint32_t)room, (uint32_t)c->page_tokens, beams, 4, 1, false},
                      stream);
}

extern "C" int mq_cache_extend(const mq_kv_cache *c, const int32_t *held, const int32_t *counts, int64_t sequences, const int32_t *table,
                               int64_t table_stride, int64_t max_pages, int64_t tokens, int64_t *slots, int64_t *positions, int32_t *lengths,
                               void *stream) {
  using namespace mq;
  if (const char *fault = place_fault(c, sequences, tokens, max_pages, table_stride, sequences)) return invalid(fault);
  if ((sequences && (!held || !lengths || (!table && max_pages))) || (tokens && (!slots || !positions)))
    return invalid("mq_cache_extend: NULL pointer");
  if (!aligned_to(counts, 4) || !aligned_to(held, 4) || !aligned_to(table, 4) || !aligned_to(lengths, 4) || !aligned_to(slots, 8) ||
      !aligned_to(positions, 8))
    return invalid("mq_cache_extend: misaligned buffer");
  return launch_place({counts, held, nullptr, const_cast<int32_t *>(table), sequences, tokens, max_pages, table_stride, 0, c->pages, slots,
                       positions, nullptr, lengths, 0, (uint32_t)c->page_tokens, 1, 4, 1, false},
                      stream);
}
