// Pages of a cache between sequences: sequences that go on from chosen ones (pages shared, copied, released), and pages that move to the
// front of their pools.
//
// Both make a plan and carry it out: in one launch where every workgroup can make the plan for itself, in two with a plan in memory otherwise.  Holders
// of a page are counted in LDS (integer sums, so the order of the atomics changes nothing), places in lists come from running sums over sequences or
// pages, so that every result is the same from run to run.  Nothing is written that the plan is made from, so a call can be repeated, and a
// captured one replayed, on the same inputs.
//
// A server's step is bound by latency (loads that wait for each other), a move of many pages by HBM.
#include <algorithm>

#include "tpa_common.h"

namespace tpa {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kThreads = 256;
constexpr int kRange = 8192;       // pages whose holders a workgroup counts
constexpr int kChunk = 16384;      // bytes of a page that a workgroup copies at a time

struct Move { int32_t src, dst, tokens, unused; };
// what the plan leaves for the second launch
struct Meta {
  int32_t moves;        // entries of the list of moves
  int32_t taken, start;  // fork: pages taken from the free list, and from where on
  int32_t used;         // compact: pages in use
};
constexpr int kMetaInts = 16;

// sum over the threads before this one and, in `total`, over all; `red` = an int per wave
__device__ __forceinline__ int sum_before(int x, int* red, int& total) {
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  int upto = x;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int y = __shfl_up(upto, d);
    if (lane >= d) upto += y;
  }
  if (lane == 63) red[w] = upto;
  __syncthreads();
  int before = 0;
  total = 0;
  for (int i = 0; i < (int)(blockDim.x >> 6); ++i) {
    if (i < w) before += red[i];
    total += red[i];
  }
  __syncthreads();
  return before + upto - x;
}

// ------------------------------------------------------------------------------------------------ contents of pages
struct Pool { char* ptr; int64_t stride; int32_t token_bytes, unit; };  // unit: bytes of a load, 16, 4 or 1
struct Pools {
  Pool pool[TPA_MAX_POOLS];
  int n, chunks;  // chunks of kChunk bytes in a page, at most
};

constexpr int kCopyThreads = 256;  // that copy a chunk: four loads each in flight
// Past the caches, which hold none of it when it is read next: 500 MB read and written take 100.5 us (5.0 TB/s), through them 109.7.
template <typename T>
__device__ __forceinline__ void copy_chunk(char* to, const char* from, int64_t bytes, int thread) {
  T* const t = reinterpret_cast<T*>(to);
  const T* const f = reinterpret_cast<const T*>(from);
  const int n = (int)(bytes / (int64_t)sizeof(T));
  for (int i = thread; i < n; i += 4 * kCopyThreads) {
    T x[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (i + u * kCopyThreads < n) x[u] = __builtin_nontemporal_load(f + i + u * kCopyThreads);
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (i + u * kCopyThreads < n) __builtin_nontemporal_store(x[u], t + i + u * kCopyThreads);
  }
}
// `group` of `groups` groups of threads that share out the moves' chunks
template <typename MoveAt>
__device__ __forceinline__ void copy_pages(const Pools& pools, int moves, MoveAt move_at, int64_t group, int64_t groups) {
  const int per_move = pools.n * pools.chunks, thread = threadIdx.x % kCopyThreads;
  const int64_t items = (int64_t)moves * per_move;
  for (int64_t item = group; item < items; item += groups) {
    const int m = (int)(item / per_move), rest = (int)(item - (int64_t)m * per_move), chunk = rest / pools.n;
    const Move move = move_at(m);
    const Pool& pool = pools.pool[rest - chunk * pools.n];
    const int64_t first = (int64_t)chunk * kChunk, bytes = min((int64_t)move.tokens * pool.token_bytes - first, (int64_t)kChunk);
    if (bytes <= 0) continue;
    char* const to = pool.ptr + move.dst * pool.stride + first;
    const char* const from = pool.ptr + move.src * pool.stride + first;
    if (pool.unit == 16) copy_chunk<u32x4>(to, from, bytes, thread);
    else if (pool.unit == 4) copy_chunk<uint32_t>(to, from, bytes, thread);
    else copy_chunk<uint8_t>(to, from, bytes, thread);
  }
}

// ------------------------------------------------------------------------------------------------ fork
struct ForkParams {
  const int32_t *table, *lengths, *parents, *shares, *free_pages, *free_start;
  int32_t *new_table, *new_lengths, *new_shares, *new_free, *new_start;
  Meta* meta;
  int32_t* released_count;  // [ranges]
  int32_t* released;        // [pages]: those of range r from r * kRange on
  int32_t* fresh;           // [M]: the page that a new sequence got for its copy, or -1
  Move* moves;              // [M]
  int B, M, P, page, N, F;
};

__device__ __forceinline__ int clamped_length(const int32_t* lengths, int s, int cap) { return max(0, min(lengths[s], cap)); }

__device__ __forceinline__ int shares_of(const ForkParams& p, int page) { return max(p.shares[page], 0); }
__device__ __forceinline__ int start_of(const int32_t* free_start, int F) { return free_start ? max(0, min(free_start[0], F)) : 0; }

// in LDS: lengths of the old sequences, how many new ones each has and the first of them
__device__ __forceinline__ void find_children(const ForkParams& p, int32_t* children, int32_t* first, int32_t* length) {
  const int cap = p.P * p.page;
  for (int s = threadIdx.x; s < p.B; s += kPlanThreads) {
    children[s] = 0;
    first[s] = INT32_MAX;
    length[s] = clamped_length(p.lengths, s, cap);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < p.M; i += kPlanThreads) {
    const int s = p.parents[i];
    if (s >= 0 && s < p.B) {
      atomicAdd(&children[s], 1);
      atomicMin(&first[s], i);
    }
  }
  __syncthreads();
}
// this thread's new sequences, side by side: found(i, page that it got for its copy or -1, length), moved(rank, move) for those that need one.
// Returns the pages taken, and how many need one in `moves`.
template <typename Found, typename Moved>
__device__ __forceinline__ int deal_pages(const ForkParams& p, const int32_t* first, const int32_t* length, int start, int* red, int& moves, Found found, Moved moved) {
  const int each = (p.M + kPlanThreads - 1) / kPlanThreads, i0 = min((int)threadIdx.x * each, p.M), i1 = min(i0 + each, p.M);
  auto needs = [&](int i, int& s, int& last) {
    s = p.parents[i];
    if (s < 0 || s >= p.B) { s = -1; return false; }
    if (length[s] % p.page == 0) return false;
    last = p.table[(int64_t)s * p.P + length[s] / p.page];
    if (last < 0 || last >= p.N) return false;
    return first[s] != i || shares_of(p, last) != 0;
  };
  int count = 0, s, last = 0;
  for (int i = i0; i < i1; ++i) count += needs(i, s, last);
  const bool again = each > 1;
  bool copies = count > 0;  // of the one sequence, if there is no other
  int rank = sum_before(count, red, moves);
  for (int i = i0; i < i1; ++i) {
    if (again) copies = needs(i, s, last);
    int fresh = -1, len = s < 0 ? 0 : length[s];
    if (copies) {
      if (rank < p.F - start) fresh = p.free_pages[start + rank];
      if (fresh < 0 || fresh >= p.N) {
        fresh = -1;
        len = len / p.page * p.page;
      }
      moved(rank, Move{last, max(fresh, 0), fresh < 0 ? 0 : len % p.page, 0});
      ++rank;
    }
    found(i, fresh, len);
  }
  return min(moves, p.F - start);
}
// in LDS: holders that pages lo .. lo + n - 1 gain or lose.  A wave takes eight sequences at a time, a lane a page of each: sequences that go on once have
// nothing to count but the last page.
__device__ __forceinline__ void count_holders(const ForkParams& p, const int32_t* children, const int32_t* length, int32_t* change, int lo, int n) {
  // last pages: lost unless a new sequence keeps it
  for (int s = threadIdx.x; s < p.B; s += kPlanThreads)
    if (length[s] % p.page != 0) {
      const int page = p.table[(int64_t)s * p.P + length[s] / p.page];
      if (page >= lo && page < lo + n && (children[s] == 0 || shares_of(p, page) != 0)) atomicAdd(&change[page - lo], -1);
    }
  constexpr int kTogether = 8;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int s0 = wave * kTogether; s0 < p.B; s0 += kPlanThreads / 64 * kTogether) {
    int most = 0, full[kTogether], by[kTogether];
#pragma unroll
    for (int u = 0; u < kTogether; ++u) {
      const int s = min(s0 + u, p.B - 1);
      full[u] = length[s] / p.page;
      by[u] = s0 + u < p.B ? children[s] - 1 : 0;
      most = max(most, (by[u] ? full[u] : 0));
    }
    for (int e = lane; e < most; e += 64) {
      int page[kTogether];
#pragma unroll
      for (int u = 0; u < kTogether; ++u) {
        page[u] = -1;
        if (by[u] != 0 && e < full[u]) page[u] = p.table[(int64_t)(s0 + u) * p.P + e];
      }
#pragma unroll
      for (int u = 0; u < kTogether; ++u)
        if (page[u] >= lo && page[u] < lo + n) atomicAdd(&change[page[u] - lo], by[u]);
    }
  }
}
// Counts of pages lo .. lo + n - 1 after the step, page j * kPlanThreads + i of them by thread i; put(rank, how many there are, page) for those that are released,
// in rising order.  Returns how many.  `slabs` = kSlabs ints
constexpr int kEach = kRange / kPlanThreads, kSlabs = kEach * (kPlanThreads / 64);
template <typename Put>
__device__ __forceinline__ int settle_counts(const ForkParams& p, const int32_t* change, int lo, int n, int* slabs, Put put) {
  static_assert(kSlabs == 128, "two of them a lane");
  const int tid = threadIdx.x, lane = tid & 63, w = scalar(tid >> 6);
  int before[kEach];
#pragma unroll
  for (int j = 0; j < kEach; ++j) before[j] = shares_of(p, lo + min(j * kPlanThreads + tid, n - 1));  // all on their way together
  uint64_t gone[kEach];
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const int i = j * kPlanThreads + tid, now = i < n ? before[j] + change[i] : 0;
    if (i < n) p.new_shares[lo + i] = max(now, 0);
    gone[j] = __ballot(now < 0);
    if (lane == 0) slabs[j * (kPlanThreads / 64) + w] = __popcll(gone[j]);
  }
  __syncthreads();
  // every wave: released pages before each slab of 64
  const int first = slabs[2 * lane], both = first + slabs[2 * lane + 1];
  int upto = both;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int y = __shfl_up(upto, d);
    if (lane >= d) upto += y;
  }
  const int total = __builtin_amdgcn_readlane(upto, 63);
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const int slab = j * (kPlanThreads / 64) + w;
    const int base = __builtin_amdgcn_readlane(upto - both, slab >> 1) + (slab & 1 ? __builtin_amdgcn_readlane(first, slab >> 1) : 0);
    if (gone[j] >> lane & 1) put(base + __popcll(gone[j] & ((1ull << lane) - 1)), total, lo + j * kPlanThreads + tid);
  }
  return total;
}

// ---- one launch, for pages of one range and no more than kSmall sequences: the first workgroup counts holders and makes the list, every other one makes the plan for
// itself and carries out its share (a second launch costs the host 3.5 us; with it, 256 sequences over 4170 pages and 14 MB read and written took 16.4 + 5.4 us, with one
// 17.8; 12.3 since the first workgroup, which is the last to end, reads the last pages, the counts and the table's rows in as few rounds of waiting as there
// are).  One of these workgroups fits a compute unit (76 registers; at 64, for two, 60 bytes go to scratch memory: 15.9 us).
constexpr int kSmall = 2048;
__global__ __launch_bounds__(kPlanThreads) void fork_small_kernel(ForkParams p, Pools pools) {
  extern __shared__ int32_t smem[];
  __shared__ int red[kPlanThreads / 64], slabs[kSlabs];
  int32_t* const children = smem;
  int32_t* const first = children + p.B;
  int32_t* const length = first + p.B;
  int32_t* const rest = length + p.B;  // [N] changes, or [M] pages got, [M] lengths, [M] moves of three numbers
  const int tid = threadIdx.x, start = start_of(p.free_start, p.F);
  const bool counts = blockIdx.x == 0;
  if (counts)
    for (int i = tid; i < p.N; i += kPlanThreads) rest[i] = 0;
  find_children(p, children, first, length);
  int moves;
  if (counts) {
    const int taken = deal_pages(p, first, length, start, red, moves, [&](int i, int, int len) { p.new_lengths[i] = len; }, [](int, Move) {});
    count_holders(p, children, length, rest, 0, p.N);
    __syncthreads();
    const int end = start + taken;
    const int begin = end - settle_counts(p, rest, 0, p.N, slabs, [&](int rank, int released, int page) {
      if (end - released + rank >= 0) p.new_free[end - released + rank] = page;
    });
    for (int j = tid; j < p.F; j += kPlanThreads)
      if (j < begin || j >= end) p.new_free[j] = p.free_pages[j];
    if (tid == 0) p.new_start[0] = max(begin, 0);
    return;
  }
  int32_t *const got = rest, *const len = rest + p.M, *const move = len + p.M;
  deal_pages(p, first, length, start, red, moves, [&](int i, int fresh, int l) { got[i] = fresh; len[i] = l; },
             [&](int rank, Move m) { move[3 * rank] = m.src; move[3 * rank + 1] = m.dst; move[3 * rank + 2] = m.tokens; });
  __syncthreads();
  constexpr int kGroups = kPlanThreads / kCopyThreads;
  const int block = blockIdx.x - 1, blocks = gridDim.x - 1;
  copy_pages(pools, moves, [&](int m) { return Move{move[3 * m], move[3 * m + 1], move[3 * m + 2], 0}; }, (int64_t)(tid / kCopyThreads) * blocks + block,
             (int64_t)kGroups * blocks);
  // the table from the last groups on, which have the fewest chunks
  for (int64_t at = ((int64_t)(kGroups - 1 - tid / kCopyThreads) * blocks + block) * kCopyThreads + tid % kCopyThreads; at < (int64_t)p.M * p.P; at += (int64_t)blocks * kPlanThreads) {
    const int i = (int)(at / p.P), e = (int)(at - (int64_t)i * p.P);
    int page = 0;
    if ((int64_t)e * p.page < len[i]) {
      const int s = p.parents[i];
      page = got[i] >= 0 && e == length[s] / p.page ? got[i] : p.table[(int64_t)s * p.P + e];
    }
    p.new_table[at] = page;
  }
}

// ---- two launches
__global__ __launch_bounds__(kPlanThreads) void fork_plan_kernel(ForkParams p) {
  extern __shared__ int32_t smem[];
  __shared__ int red[kPlanThreads / 64], slabs[kSlabs];
  int32_t* const children = smem;
  int32_t* const first = children + p.B;
  int32_t* const length = first + p.B;
  int32_t* const change = length + p.B;
  const int lo = blockIdx.x * kRange, n = min(kRange, p.N - lo);
  for (int i = threadIdx.x; i < n; i += kPlanThreads) change[i] = 0;
  find_children(p, children, first, length);
  if (blockIdx.x == 0) {
    const int start = start_of(p.free_start, p.F);
    int moves;
    const int taken = deal_pages(p, first, length, start, red, moves, [&](int i, int fresh, int len) { p.fresh[i] = fresh; p.new_lengths[i] = len; },
                                 [&](int rank, Move m) { p.moves[rank] = m; });
    if (threadIdx.x == 0) *p.meta = Meta{moves, taken, start, 0};
  }
  count_holders(p, children, length, change, lo, n);
  __syncthreads();
  const int total = settle_counts(p, change, lo, n, slabs, [&](int rank, int, int page) { p.released[lo + rank] = page; });
  if (threadIdx.x == 0) p.released_count[blockIdx.x] = total;
}

// sum of counts[0 .. n) over the workgroup
__device__ __forceinline__ int sum_of(const int32_t* counts, int n, int* red) {
  int x = 0, total;
  for (int i = threadIdx.x; i < n; i += kThreads) x += counts[i];
  (void)sum_before(x, red, total);
  return total;
}

__global__ __launch_bounds__(kThreads) void fork_kernel(ForkParams p, Pools pools, int contents_only) {
  __shared__ int red[kThreads / 64];
  copy_pages(pools, p.meta->moves, [&](int m) { return p.moves[m]; }, blockIdx.x, gridDim.x);
  if (contents_only) return;

  const int64_t id = (int64_t)blockIdx.x * kThreads + threadIdx.x, all = (int64_t)gridDim.x * kThreads;
  const int cap = p.P * p.page;
  for (int64_t at = id; at < (int64_t)p.M * p.P; at += all) {
    const int i = (int)(at / p.P), e = (int)(at - (int64_t)i * p.P), len = p.new_lengths[i], s = p.parents[i];
    int page = 0;
    if ((int64_t)e * p.page < len) {  // (then s is a sequence)
      const int fresh = p.fresh[i];
      page = fresh >= 0 && e == clamped_length(p.lengths, s, cap) / p.page ? fresh : p.table[(int64_t)s * p.P + e];
    }
    p.new_table[at] = page;
  }

  const int ranges = (p.N + kRange - 1) / kRange;
  const int released = sum_of(p.released_count, ranges, red);
  const int end = p.meta->start + p.meta->taken;
  const int64_t begin = (int64_t)end - released;
  for (int64_t j = id; j < p.F; j += all)
    if (j < begin || j >= end) p.new_free[j] = p.free_pages[j];
  for (int r = blockIdx.x; r < ranges; r += gridDim.x) {
    const int64_t to = begin + sum_of(p.released_count, r, red);
    for (int k = threadIdx.x; k < p.released_count[r]; k += kThreads)
      if (to + k >= 0) p.new_free[to + k] = p.released[(int64_t)r * kRange + k];
  }
  if (id == 0) p.new_start[0] = (int)max(begin, (int64_t)0);
}

// ------------------------------------------------------------------------------------------------ compact
struct CompactParams {
  const int32_t *table, *lengths, *shares, *free_pages, *free_start;
  int32_t *new_table, *new_shares, *new_free, *new_start, *moved;
  Meta* meta;
  int32_t* map;             // [N]: page p stays (p), is a hole (kHole + p), is number r of the pages that move (-1 - r)
  int32_t *holes, *movers;  // [N]
  int B, P, page, N, F;
};
constexpr int32_t kHole = INT32_MIN;

// in LDS: a bit for every page that is free, and how many are free before those of each thread's words
struct FreeBits {
  uint32_t* bits;
  int* before;
  int each, total;
  __device__ __forceinline__ void find(const CompactParams& p, int* red) {
    const int tid = threadIdx.x, words = (p.N + 31) / 32;
    each = (words + kPlanThreads - 1) / kPlanThreads;
    for (int w = tid; w < words; w += kPlanThreads) bits[w] = 0;
    __syncthreads();
    for (int j = start_of(p.free_start, p.F) + tid; j < p.F; j += kPlanThreads) {
      const int page = p.free_pages[j];
      if (page >= 0 && page < p.N) atomicOr(&bits[page >> 5], 1u << (page & 31));
    }
    __syncthreads();
    int count = 0;
    for (int w = tid * each; w < min((tid + 1) * each, words); ++w) count += __popc(bits[w]);
    before[tid] = sum_before(count, red, total);
    __syncthreads();
  }
  __device__ __forceinline__ bool free(int page) const { return bits[page >> 5] >> (page & 31) & 1; }
  __device__ __forceinline__ int free_before(int page) const {
    const int w = page >> 5, t = w / each;
    int r = before[t] + __popc(bits[w] & ((1u << (page & 31)) - 1));
    for (int v = t * each; v < w; ++v) r += __popc(bits[v]);
    return r;
  }
};

// What is written beside the contents: place(page) = where it is now, is_free(page).  `id` of `all` threads.
template <typename Place, typename IsFree>
__device__ __forceinline__ void write_compacted(const CompactParams& p, int used, Place place, IsFree is_free, int64_t id, int64_t all) {
  for (int64_t page = id; page < p.N; page += all) {
    const int at = place((int)page);
    p.moved[page] = at;
    if (page >= used) p.new_shares[page] = 0;
    if (!is_free((int)page)) p.new_shares[at] = p.shares[page];
  }
  const int cap = p.P * p.page, first_free = p.F - (p.N - used);
  for (int64_t i = id; i < (int64_t)p.B * p.P; i += all) {
    const int b = (int)(i / p.P), e = (int)(i - (int64_t)b * p.P);
    int page = 0;
    if ((int64_t)e * p.page < clamped_length(p.lengths, b, cap)) {
      page = p.table[i];
      if (page >= 0 && page < p.N) page = place(page);
    }
    p.new_table[i] = page;
  }
  for (int64_t j = id; j < p.F; j += all) p.new_free[j] = j < first_free ? p.free_pages[j] : used + (int)(j - first_free);
  if (id == 0) p.new_start[0] = first_free;
}

// ---- one launch, for pools of no more than kRange pages: every workgroup makes the plan for itself and carries out its share
__global__ __launch_bounds__(kPlanThreads) void compact_small_kernel(CompactParams p, Pools pools) {
  __shared__ uint32_t bits[kRange / 32];
  __shared__ int red[kPlanThreads / 64], before[kPlanThreads];
  __shared__ uint16_t holes[kRange / 2], movers[kRange / 2];
  static_assert(kRange <= 65536, "pages as 16 bits");
  FreeBits f{bits, before};
  f.find(p, red);
  const int tid = threadIdx.x, used = p.N - f.total, moves = used < p.N ? f.free_before(used) : f.total;
  auto rank_of = [&](int page) { return (page - used) - (f.free_before(page) - moves); };  // of a page that moves
  for (int page = tid; page < p.N; page += kPlanThreads) {
    const bool free = f.free(page);
    if (free && page < used) holes[f.free_before(page)] = page;
    else if (!free && page >= used) movers[rank_of(page)] = page;
  }
  __syncthreads();
  constexpr int kGroups = kPlanThreads / kCopyThreads;
  copy_pages(pools, moves, [&](int m) { return Move{movers[m], holes[m], p.page, 0}; }, (int64_t)(tid / kCopyThreads) * gridDim.x + blockIdx.x, (int64_t)kGroups * gridDim.x);
  write_compacted(p, used, [&](int page) { return page < used || f.free(page) ? page : holes[rank_of(page)]; }, [&](int page) { return f.free(page); },
                  (int64_t)blockIdx.x * kPlanThreads + tid, (int64_t)gridDim.x * kPlanThreads);
}

// ---- two launches
__global__ __launch_bounds__(kPlanThreads) void compact_plan_kernel(CompactParams p) {
  extern __shared__ uint32_t bits_of_all[];
  __shared__ int red[kPlanThreads / 64], before[kPlanThreads];
  FreeBits f{bits_of_all, before};
  f.find(p, red);
  const int tid = threadIdx.x, used = p.N - f.total, holes = used < p.N ? f.free_before(used) : f.total;
  for (int page = blockIdx.x * kPlanThreads + tid; page < p.N; page += gridDim.x * kPlanThreads) {
    const bool free = f.free(page);
    int to = page;
    if (free && page < used) {
      p.holes[f.free_before(page)] = page;
      to = kHole + page;
    } else if (!free && page >= used) {
      const int r = (page - used) - (f.free_before(page) - holes);
      p.movers[r] = page;
      to = -1 - r;
    }
    p.map[page] = to;
  }
  if (blockIdx.x == 0 && tid == 0) *p.meta = Meta{holes, 0, 0, used};
}

__global__ __launch_bounds__(kThreads) void compact_kernel(CompactParams p, Pools pools, int contents_only) {
  copy_pages(pools, p.meta->moves, [&](int m) { return Move{p.movers[m], p.holes[m], p.page, 0}; }, blockIdx.x, gridDim.x);
  if (contents_only) return;
  const int used = p.meta->used;
  auto place = [&](int page) {
    const int to = p.map[page];
    return to >= 0 ? to : to < -p.N ? to - kHole : p.holes[-1 - to];
  };
  write_compacted(p, used, place, [&](int page) { return p.map[page] < -p.N || (page >= used && p.map[page] >= 0); }, (int64_t)blockIdx.x * kThreads + threadIdx.x,
                  (int64_t)gridDim.x * kThreads);
}

// ------------------------------------------------------------------------------------------------ host side
struct Layout { size_t counts, released, second, third, fresh, moves, bytes; };
Layout layout_of(int64_t M, int64_t N) {
  auto up = [](size_t x) { return (x + 15) / 16 * 16; };
  Layout l;
  l.counts = 4 * kMetaInts;
  l.released = l.counts + up(4 * ((N + kRange - 1) / kRange));
  l.second = l.released + up(4 * N);
  l.third = l.second + (M ? 0 : up(4 * N));
  l.fresh = l.third + (M ? 0 : up(4 * N));
  l.moves = l.fresh + up(4 * M);
  l.bytes = l.moves + sizeof(Move) * M;
  return l;
}

bool overlap(const void* a, int64_t na, const void* b, int64_t nb) {
  const char *x = static_cast<const char*>(a), *y = static_cast<const char*>(b);
  return a && b && na > 0 && nb > 0 && x < y + 4 * nb && y < x + 4 * na;
}
struct Ints { const int32_t* ptr; int64_t n; };
template <int NI, int NO>
bool outputs_apart(const Ints (&in)[NI], const Ints (&out)[NO]) {
  for (int o = 0; o < NO; ++o) {
    for (const Ints& i : in)
      if (overlap(i.ptr, i.n, out[o].ptr, out[o].n)) return false;
    for (int q = 0; q < o; ++q)
      if (overlap(out[q].ptr, out[q].n, out[o].ptr, out[o].n)) return false;
  }
  return true;
}

int check_pools(const TpaPool* pools, int n, int page_size) {
  if (n < 0) return TPA_ERR_SHAPE;
  if (n && !pools) return TPA_ERR_NULL;
  for (int i = 0; i < n; ++i) {
    if (!pools[i].ptr) return TPA_ERR_NULL;
    if (pools[i].token_bytes <= 0 || pools[i].token_bytes > INT32_MAX || pools[i].token_bytes * page_size > INT32_MAX) return TPA_ERR_SHAPE;
    if (pools[i].page_stride < pools[i].token_bytes * page_size) return TPA_ERR_UNSUPPORTED;  // pages that overlap
  }
  return TPA_OK;
}
Pools pools_of(const TpaPool* pools, int n, int page_size) {
  Pools p{};
  p.n = n;
  p.chunks = 1;
  for (int i = 0; i < n; ++i) {
    const uintptr_t all = reinterpret_cast<uintptr_t>(pools[i].ptr) | (uintptr_t)pools[i].page_stride | (uintptr_t)pools[i].token_bytes;
    p.pool[i] = Pool{static_cast<char*>(pools[i].ptr), pools[i].page_stride, (int32_t)pools[i].token_bytes, all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 1};
    p.chunks = std::max(p.chunks, (int)((pools[i].token_bytes * page_size + kChunk - 1) / kChunk));
  }
  return p;
}

// the second launch, and one for every further TPA_MAX_POOLS pools
template <typename Params, typename Kernel>
int carry_out(Kernel kern, const Params& p, const TpaPool* pools, int num_pools, int page_size, int64_t most_moves, int64_t numbers, hipStream_t stream) {
  for (int at = 0; at == 0 || at < num_pools; at += TPA_MAX_POOLS) {
    const Pools these = pools_of(pools + at, std::min(num_pools - at, TPA_MAX_POOLS), page_size);
    const int64_t items = std::max(most_moves * these.n * these.chunks, at ? 0 : (numbers + kThreads - 1) / kThreads);
    hipLaunchKernelGGL(kern, dim3((unsigned)std::max<int64_t>(1, std::min<int64_t>(items, 2048))), dim3(kThreads), 0, stream, p, these, at > 0);
    if (hipGetLastError() != hipSuccess) return TPA_ERR_LAUNCH;
  }
  return TPA_OK;
}

// workgroups of one launch that does all: two on a compute unit, fewer where there are fewer chunks (four at a time) and numbers
constexpr int kMostBlocks = 512;
int blocks_for(int64_t chunks, int64_t numbers) {
  const int64_t want = std::max((chunks + 3) / 4, (numbers + kPlanThreads - 1) / kPlanThreads);
  return (int)std::max<int64_t>(1, std::min<int64_t>(want, kMostBlocks));
}

template <typename Args>
int check_pages(const Args* a) {
  if (a->B < 0 || a->B > TPA_PAGE_TABLES_MAX_REQUESTS || a->pages_per_seq <= 0 || a->page_size <= 0 || a->num_pages <= 0 || a->num_free < 0) return TPA_ERR_SHAPE;
  if ((int64_t)a->pages_per_seq * a->page_size > INT32_MAX || (int64_t)a->num_pages * a->page_size > INT32_MAX) return TPA_ERR_SHAPE;
  if (a->B && (!a->page_table || !a->kv_lengths)) return TPA_ERR_NULL;
  if (!a->page_shares || !a->new_page_shares || !a->new_free_start) return TPA_ERR_NULL;
  if (a->num_free && (!a->free_pages || !a->new_free_pages)) return TPA_ERR_NULL;
  return check_pools(a->pools, a->num_pools, a->page_size);
}
bool in_one_launch(int B, int M, int num_pages, int num_pools) {
  return num_pages <= kRange && (M == 0 || (B <= kSmall && M <= kSmall)) && num_pools <= TPA_MAX_POOLS;
}
template <typename Args>
int check_workspace(const Args* a, size_t need) {
  if (!a->workspace || a->workspace_bytes < need) return TPA_ERR_WORKSPACE;
  return reinterpret_cast<uintptr_t>(a->workspace) % 16 ? TPA_ERR_ALIGN : TPA_OK;
}

}  // namespace
}  // namespace tpa

extern "C" size_t tpa_pages_workspace_bytes(int32_t B, int32_t M, int32_t num_pages, int32_t num_pools) {
  return M >= 0 && num_pages > 0 && !tpa::in_one_launch(B, M, num_pages, num_pools) ? tpa::layout_of(M, num_pages).bytes : 0;
}

extern "C" int tpa_pages_fork(const TpaPagesForkArgs* a, void* stream) {
  using namespace tpa;
  if (!a) return TPA_ERR_NULL;
  if (int rc = check_pages(a); rc != TPA_OK) return rc;
  if (a->M < 0 || a->M > TPA_PAGE_TABLES_MAX_REQUESTS) return TPA_ERR_SHAPE;
  if (a->M && (!a->parents || !a->new_page_table || !a->new_kv_lengths)) return TPA_ERR_NULL;
  const int64_t P = a->pages_per_seq;
  const Ints in[] = {{a->page_table, a->B * P}, {a->kv_lengths, a->B}, {a->parents, a->M}, {a->page_shares, a->num_pages}, {a->free_pages, a->num_free}, {a->free_start, 1}};
  const Ints out[] = {{a->new_page_table, a->M * P}, {a->new_kv_lengths, a->M}, {a->new_page_shares, a->num_pages}, {a->new_free_pages, a->num_free}, {a->new_free_start, 1}};
  if (!outputs_apart(in, out)) return TPA_ERR_UNSUPPORTED;
  ForkParams p{};
  p.table = a->page_table; p.lengths = a->kv_lengths; p.parents = a->parents; p.shares = a->page_shares; p.free_pages = a->free_pages; p.free_start = a->free_start;
  p.new_table = a->new_page_table; p.new_lengths = a->new_kv_lengths; p.new_shares = a->new_page_shares; p.new_free = a->new_free_pages; p.new_start = a->new_free_start;
  p.B = a->B; p.M = a->M; p.P = a->pages_per_seq; p.page = a->page_size; p.N = a->num_pages; p.F = a->num_free;
  if (in_one_launch(a->B, a->M, a->num_pages, a->num_pools)) {
    const Pools pools = pools_of(a->pools, a->num_pools, a->page_size);
    const size_t lds = 4 * ((size_t)3 * a->B + std::max(a->num_pages, 5 * a->M));
    static bool configured[kMaxDevices] = {};
    if (int rc = raise_lds_limit(configured, reinterpret_cast<const void*>(fork_small_kernel), 4 * (3 * TPA_PAGE_TABLES_MAX_REQUESTS + std::max(kRange, 5 * kSmall))); rc != TPA_OK) return rc;
    const int groups = std::min(blocks_for((int64_t)a->M * pools.n * pools.chunks, a->M * P), 255);
    hipLaunchKernelGGL(fork_small_kernel, dim3(1 + groups), dim3(kPlanThreads), lds, static_cast<hipStream_t>(stream), p, pools);
    return hipGetLastError() == hipSuccess ? TPA_OK : TPA_ERR_LAUNCH;
  }
  const Layout l = layout_of(a->M, a->num_pages);
  if (int rc = check_workspace(a, l.bytes); rc != TPA_OK) return rc;
  char* const ws = static_cast<char*>(a->workspace);
  p.meta = reinterpret_cast<Meta*>(ws);
  p.released_count = reinterpret_cast<int32_t*>(ws + l.counts); p.released = reinterpret_cast<int32_t*>(ws + l.released);
  p.fresh = reinterpret_cast<int32_t*>(ws + l.fresh); p.moves = reinterpret_cast<Move*>(ws + l.moves);
  const int ranges = (a->num_pages + kRange - 1) / kRange;
  const size_t lds = 4 * ((size_t)3 * a->B + std::min(a->num_pages, kRange));
  static bool configured[kMaxDevices] = {};
  if (int rc = raise_lds_limit(configured, reinterpret_cast<const void*>(fork_plan_kernel), 4 * (3 * TPA_PAGE_TABLES_MAX_REQUESTS + kRange)); rc != TPA_OK) return rc;
  hipLaunchKernelGGL(fork_plan_kernel, dim3(ranges), dim3(kPlanThreads), lds, static_cast<hipStream_t>(stream), p);
  if (hipGetLastError() != hipSuccess) return TPA_ERR_LAUNCH;
  return carry_out(fork_kernel, p, a->pools, a->num_pools, a->page_size, a->M, a->M * P + a->num_free, static_cast<hipStream_t>(stream));
}

extern "C" int tpa_pages_compact(const TpaPagesCompactArgs* a, void* stream) {
  using namespace tpa;
  if (!a) return TPA_ERR_NULL;
  if (int rc = check_pages(a); rc != TPA_OK) return rc;
  if (a->num_pages > TPA_COMPACT_MAX_PAGES) return TPA_ERR_SHAPE;
  if ((a->B && !a->new_page_table) || !a->moved) return TPA_ERR_NULL;
  const int64_t P = a->pages_per_seq;
  const Ints in[] = {{a->page_table, a->B * P}, {a->kv_lengths, a->B}, {a->page_shares, a->num_pages}, {a->free_pages, a->num_free}, {a->free_start, 1}};
  const Ints out[] = {{a->new_page_table, a->B * P}, {a->moved, a->num_pages}, {a->new_page_shares, a->num_pages}, {a->new_free_pages, a->num_free}, {a->new_free_start, 1}};
  if (!outputs_apart(in, out)) return TPA_ERR_UNSUPPORTED;
  CompactParams p{};
  p.table = a->page_table; p.lengths = a->kv_lengths; p.shares = a->page_shares; p.free_pages = a->free_pages; p.free_start = a->free_start;
  p.new_table = a->new_page_table; p.new_shares = a->new_page_shares; p.new_free = a->new_free_pages; p.new_start = a->new_free_start; p.moved = a->moved;
  p.B = a->B; p.P = a->pages_per_seq; p.page = a->page_size; p.N = a->num_pages; p.F = a->num_free;
  const int64_t most = std::min<int64_t>(a->num_free, a->num_pages / 2), numbers = std::max<int64_t>({a->num_pages, a->B * P, a->num_free});
  if (in_one_launch(a->B, 0, a->num_pages, a->num_pools)) {
    const Pools pools = pools_of(a->pools, a->num_pools, a->page_size);
    hipLaunchKernelGGL(compact_small_kernel, dim3(blocks_for(most * pools.n * pools.chunks, numbers)), dim3(kPlanThreads), 0, static_cast<hipStream_t>(stream), p, pools);
    return hipGetLastError() == hipSuccess ? TPA_OK : TPA_ERR_LAUNCH;
  }
  const Layout l = layout_of(0, a->num_pages);
  if (int rc = check_workspace(a, l.bytes); rc != TPA_OK) return rc;
  char* const ws = static_cast<char*>(a->workspace);
  p.meta = reinterpret_cast<Meta*>(ws);
  p.map = reinterpret_cast<int32_t*>(ws + l.released); p.holes = reinterpret_cast<int32_t*>(ws + l.second); p.movers = reinterpret_cast<int32_t*>(ws + l.third);
  static bool configured[kMaxDevices] = {};
  if (int rc = raise_lds_limit(configured, reinterpret_cast<const void*>(compact_plan_kernel), TPA_COMPACT_MAX_PAGES / 8); rc != TPA_OK) return rc;
  const size_t lds = 4 * (size_t)((a->num_pages + 31) / 32);
  const int groups = std::min(64, (a->num_pages + kPlanThreads - 1) / kPlanThreads);
  hipLaunchKernelGGL(compact_plan_kernel, dim3(groups), dim3(kPlanThreads), lds, static_cast<hipStream_t>(stream), p);
  if (hipGetLastError() != hipSuccess) return TPA_ERR_LAUNCH;
  return carry_out(compact_kernel, p, a->pools, a->num_pools, a->page_size, most, numbers, static_cast<hipStream_t>(stream));
}
