// Pages of a cache between sequences: sequences that go on from chosen ones (pages shared, copied, released), and pages that move to the
// front of their pools.
//
// Both take two launches.  The first makes the plan: who holds which page is counted in LDS by a workgroup for every 8192 pages (integer sums, so
// the order of the atomics changes nothing), places in lists come from running sums over sequences or pages, so that every result is the same from run to
// run.  The second carries it out with the whole card: contents of pages, tables, the free list.  Nothing is written that the first one reads,
// so a call can be repeated, and a captured one replayed, on the same inputs.
//
// A server's step is bound by latency (two launches, four loads that wait for each other), a move of many pages by HBM.
#include <algorithm>

#include "tpa_common.h"

namespace tpa {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kThreads = 256;
constexpr int kRange = 8192;       // pages that a workgroup of the plan counts
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

template <typename T>
__device__ __forceinline__ void copy_chunk(char* to, const char* from, int64_t bytes) {
  T* const t = reinterpret_cast<T*>(to);
  const T* const f = reinterpret_cast<const T*>(from);
  const int n = (int)(bytes / (int64_t)sizeof(T));
  int i = threadIdx.x;
  for (; i + 3 * kThreads < n; i += 4 * kThreads) {  // four loads in flight
    const T a = f[i], b = f[i + kThreads], c = f[i + 2 * kThreads], d = f[i + 3 * kThreads];
    t[i] = a; t[i + kThreads] = b; t[i + 2 * kThreads] = c; t[i + 3 * kThreads] = d;
  }
  for (; i < n; i += kThreads) t[i] = f[i];
}
template <typename MoveAt>
__device__ __forceinline__ void copy_pages(const Pools& pools, int moves, MoveAt move_at) {
  const int per_move = pools.n * pools.chunks;
  const int64_t items = (int64_t)moves * per_move;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int m = (int)(item / per_move), rest = (int)(item - (int64_t)m * per_move), chunk = rest / pools.n;
    const Move move = move_at(m);
    const Pool& pool = pools.pool[rest - chunk * pools.n];
    const int64_t first = (int64_t)chunk * kChunk, bytes = min((int64_t)move.tokens * pool.token_bytes - first, (int64_t)kChunk);
    if (bytes <= 0) continue;
    char* const to = pool.ptr + move.dst * pool.stride + first;
    const char* const from = pool.ptr + move.src * pool.stride + first;
    if (pool.unit == 16) copy_chunk<u32x4>(to, from, bytes);
    else if (pool.unit == 4) copy_chunk<uint32_t>(to, from, bytes);
    else copy_chunk<uint8_t>(to, from, bytes);
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

__global__ __launch_bounds__(kPlanThreads) void fork_plan_kernel(ForkParams p) {
  extern __shared__ int32_t smem[];
  __shared__ int red[kPlanThreads / 64];
  int32_t* const children = smem;         // [B] new sequences of an old one
  int32_t* const first = smem + p.B;      // [B] the first of them
  int32_t* const length = smem + 2 * p.B;  // [B]
  int32_t* const change = smem + 3 * p.B;  // [pages of the range]
  const int tid = threadIdx.x;
  const int lo = blockIdx.x * kRange, n = min(kRange, p.N - lo), cap = p.P * p.page;
  for (int s = tid; s < p.B; s += kPlanThreads) {
    children[s] = 0;
    first[s] = INT32_MAX;
    length[s] = clamped_length(p.lengths, s, cap);
  }
  for (int i = tid; i < n; i += kPlanThreads) change[i] = 0;
  __syncthreads();
  for (int i = tid; i < p.M; i += kPlanThreads) {
    const int s = p.parents[i];
    if (s >= 0 && s < p.B) {
      atomicAdd(&children[s], 1);
      atomicMin(&first[s], i);
    }
  }
  __syncthreads();

  auto shares_of = [&](int page) { return max(p.shares[page], 0); };
  if (blockIdx.x == 0) {
    // this thread's new sequences, side by side: whether they need a page of their own, the place of that page in the list
    const int start = p.free_start ? max(0, min(p.free_start[0], p.F)) : 0;
    const int each = (p.M + kPlanThreads - 1) / kPlanThreads, i0 = min(tid * each, p.M), i1 = min(i0 + each, p.M);
    auto needs = [&](int i, int& s, int& last) {
      s = p.parents[i];
      if (s < 0 || s >= p.B) { s = -1; return false; }
      const int tail = length[s] % p.page;
      if (!tail) return false;
      last = p.table[(int64_t)s * p.P + length[s] / p.page];
      if (last < 0 || last >= p.N) return false;
      return first[s] != i || shares_of(last) != 0;
    };
    int count = 0, s, last;
    for (int i = i0; i < i1; ++i) count += needs(i, s, last);
    int total;
    int rank = sum_before(count, red, total);
    for (int i = i0; i < i1; ++i) {
      const bool copies = needs(i, s, last);
      int fresh = -1, len = s < 0 ? 0 : length[s];
      if (copies) {
        if (rank < p.F - start) fresh = p.free_pages[start + rank];
        if (fresh < 0 || fresh >= p.N) {
          fresh = -1;
          len = len / p.page * p.page;
        }
        p.moves[rank] = Move{last, max(fresh, 0), fresh < 0 ? 0 : len % p.page, 0};
        ++rank;
      }
      p.fresh[i] = fresh;
      p.new_lengths[i] = len;
    }
    if (tid == 0) {
      p.meta->moves = total;
      p.meta->taken = min(total, p.F - start);
      p.meta->start = start;
    }
  }

  // holders that the pages of this range gain and lose, four table entries asked for at a time
  const int64_t entries = (int64_t)p.B * p.P;
  for (int64_t at0 = tid; at0 < entries; at0 += 4 * kPlanThreads) {
    int page[4], by[4];
    bool tail[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t at = at0 + u * kPlanThreads;
      by[u] = 0;
      tail[u] = false;
      page[u] = -1;
      if (at < entries) {
        const int s = (int)(at / p.P), e = (int)(at - (int64_t)s * p.P), full = length[s] / p.page;
        tail[u] = e == full && length[s] % p.page != 0;
        by[u] = e < full ? children[s] - 1 : tail[u] ? -1 : 0;
        if (tail[u] && children[s] > 0) by[u] = 1;  // kept where nobody else holds it
        if (by[u] != 0) page[u] = p.table[at];
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (page[u] < lo || page[u] >= lo + n) continue;
      if (tail[u] && by[u] > 0) by[u] = shares_of(page[u]) != 0 ? -1 : 0;
      if (by[u]) atomicAdd(&change[page[u] - lo], by[u]);
    }
  }
  __syncthreads();

  constexpr int kEach = kRange / kPlanThreads;
  int count = 0;
  uint32_t gone = 0;
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const int i = tid * kEach + j;
    if (i >= n) break;
    const int now = shares_of(lo + i) + change[i];
    p.new_shares[lo + i] = max(now, 0);
    if (now < 0) { gone |= 1u << j; ++count; }
  }
  int total;
  int at = sum_before(count, red, total);
#pragma unroll
  for (int j = 0; j < kEach; ++j)
    if (gone >> j & 1) p.released[lo + at++] = lo + tid * kEach + j;
  if (tid == 0) p.released_count[blockIdx.x] = total;
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
  copy_pages(pools, p.meta->moves, [&](int m) { return p.moves[m]; });
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

__global__ __launch_bounds__(kPlanThreads) void compact_plan_kernel(CompactParams p) {
  extern __shared__ uint32_t is_free[];  // a bit for every page
  __shared__ int red[kPlanThreads / 64];
  __shared__ int before[kPlanThreads];  // free pages before those of a thread's words
  const int tid = threadIdx.x, words = (p.N + 31) / 32, each = (words + kPlanThreads - 1) / kPlanThreads;
  for (int w = tid; w < words; w += kPlanThreads) is_free[w] = 0;
  __syncthreads();
  const int start = p.free_start ? max(0, min(p.free_start[0], p.F)) : 0;
  for (int j = start + tid; j < p.F; j += kPlanThreads) {
    const int page = p.free_pages[j];
    if (page >= 0 && page < p.N) atomicOr(&is_free[page >> 5], 1u << (page & 31));
  }
  __syncthreads();
  int count = 0, total;
  for (int w = tid * each; w < min((tid + 1) * each, words); ++w) count += __popc(is_free[w]);
  before[tid] = sum_before(count, red, total);
  __syncthreads();
  auto free_before = [&](int page) {
    const int w = page >> 5, t = w / each;
    int r = before[t] + __popc(is_free[w] & ((1u << (page & 31)) - 1));
    for (int v = t * each; v < w; ++v) r += __popc(is_free[v]);
    return r;
  };
  const int used = p.N - total, holes = used < p.N ? free_before(used) : total;
  for (int page = blockIdx.x * kPlanThreads + tid; page < p.N; page += gridDim.x * kPlanThreads) {
    const bool free = is_free[page >> 5] >> (page & 31) & 1;
    int to = page;
    if (free && page < used) {
      p.holes[free_before(page)] = page;
      to = kHole + page;
    } else if (!free && page >= used) {
      const int r = (page - used) - (free_before(page) - holes);
      p.movers[r] = page;
      to = -1 - r;
    }
    p.map[page] = to;
  }
  if (blockIdx.x == 0 && tid == 0) {
    p.meta->moves = holes;
    p.meta->used = used;
  }
}

__global__ __launch_bounds__(kThreads) void compact_kernel(CompactParams p, Pools pools, int contents_only) {
  copy_pages(pools, p.meta->moves, [&](int m) { return Move{p.movers[m], p.holes[m], p.page, 0}; });
  if (contents_only) return;
  const int used = p.meta->used, first_free = p.F - (p.N - used);
  const int64_t id = (int64_t)blockIdx.x * kThreads + threadIdx.x, all = (int64_t)gridDim.x * kThreads;
  auto place = [&](int to) { return to >= 0 ? to : to < -p.N ? to - kHole : p.holes[-1 - to]; };
  for (int64_t page = id; page < p.N; page += all) {
    const int to = p.map[page], at = place(to);
    p.moved[page] = at;
    if (page >= used) p.new_shares[page] = 0;
    if (at < used && to >= -p.N) p.new_shares[at] = p.shares[page];  // (a page that is not free)
  }
  const int cap = p.P * p.page;
  for (int64_t i = id; i < (int64_t)p.B * p.P; i += all) {
    const int b = (int)(i / p.P), e = (int)(i - (int64_t)b * p.P);
    int page = 0;
    if ((int64_t)e * p.page < clamped_length(p.lengths, b, cap)) {
      page = p.table[i];
      if (page >= 0 && page < p.N) page = place(p.map[page]);
    }
    p.new_table[i] = page;
  }
  for (int64_t j = id; j < p.F; j += all) p.new_free[j] = j < first_free ? p.free_pages[j] : used + (int)(j - first_free);
  if (id == 0) p.new_start[0] = first_free;
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

template <typename Args>
int check_pages(const Args* a) {
  if (a->B < 0 || a->B > TPA_PAGE_TABLES_MAX_REQUESTS || a->pages_per_seq <= 0 || a->page_size <= 0 || a->num_pages <= 0 || a->num_free < 0) return TPA_ERR_SHAPE;
  if ((int64_t)a->pages_per_seq * a->page_size > INT32_MAX || (int64_t)a->num_pages * a->page_size > INT32_MAX) return TPA_ERR_SHAPE;
  if (a->B && (!a->page_table || !a->kv_lengths)) return TPA_ERR_NULL;
  if (!a->page_shares || !a->new_page_shares || !a->new_free_start) return TPA_ERR_NULL;
  if (a->num_free && (!a->free_pages || !a->new_free_pages)) return TPA_ERR_NULL;
  return check_pools(a->pools, a->num_pools, a->page_size);
}
template <typename Args>
int check_workspace(const Args* a, size_t need) {
  if (!a->workspace || a->workspace_bytes < need) return TPA_ERR_WORKSPACE;
  return reinterpret_cast<uintptr_t>(a->workspace) % 16 ? TPA_ERR_ALIGN : TPA_OK;
}

}  // namespace
}  // namespace tpa

extern "C" size_t tpa_pages_workspace_bytes(int32_t M, int32_t num_pages) {
  return M >= 0 && num_pages > 0 ? tpa::layout_of(M, num_pages).bytes : 0;
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
  const Layout l = layout_of(a->M, a->num_pages);
  if (int rc = check_workspace(a, l.bytes); rc != TPA_OK) return rc;
  char* const ws = static_cast<char*>(a->workspace);
  ForkParams p{};
  p.table = a->page_table; p.lengths = a->kv_lengths; p.parents = a->parents; p.shares = a->page_shares; p.free_pages = a->free_pages; p.free_start = a->free_start;
  p.new_table = a->new_page_table; p.new_lengths = a->new_kv_lengths; p.new_shares = a->new_page_shares; p.new_free = a->new_free_pages; p.new_start = a->new_free_start;
  p.meta = reinterpret_cast<Meta*>(ws);
  p.released_count = reinterpret_cast<int32_t*>(ws + l.counts); p.released = reinterpret_cast<int32_t*>(ws + l.released);
  p.fresh = reinterpret_cast<int32_t*>(ws + l.fresh); p.moves = reinterpret_cast<Move*>(ws + l.moves);
  p.B = a->B; p.M = a->M; p.P = a->pages_per_seq; p.page = a->page_size; p.N = a->num_pages; p.F = a->num_free;
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
  const Layout l = layout_of(0, a->num_pages);
  if (int rc = check_workspace(a, l.bytes); rc != TPA_OK) return rc;
  char* const ws = static_cast<char*>(a->workspace);
  CompactParams p{};
  p.table = a->page_table; p.lengths = a->kv_lengths; p.shares = a->page_shares; p.free_pages = a->free_pages; p.free_start = a->free_start;
  p.new_table = a->new_page_table; p.new_shares = a->new_page_shares; p.new_free = a->new_free_pages; p.new_start = a->new_free_start; p.moved = a->moved;
  p.meta = reinterpret_cast<Meta*>(ws);
  p.map = reinterpret_cast<int32_t*>(ws + l.released); p.holes = reinterpret_cast<int32_t*>(ws + l.second); p.movers = reinterpret_cast<int32_t*>(ws + l.third);
  p.B = a->B; p.P = a->pages_per_seq; p.page = a->page_size; p.N = a->num_pages; p.F = a->num_free;
  static bool configured[kMaxDevices] = {};
  if (int rc = raise_lds_limit(configured, reinterpret_cast<const void*>(compact_plan_kernel), TPA_COMPACT_MAX_PAGES / 8); rc != TPA_OK) return rc;
  const size_t lds = 4 * (size_t)((a->num_pages + 31) / 32);
  const int groups = std::min(64, (a->num_pages + kPlanThreads - 1) / kPlanThreads);
  hipLaunchKernelGGL(compact_plan_kernel, dim3(groups), dim3(kPlanThreads), lds, static_cast<hipStream_t>(stream), p);
  if (hipGetLastError() != hipSuccess) return TPA_ERR_LAUNCH;
  const int64_t most = std::min<int64_t>(a->num_free, a->num_pages / 2);
  return carry_out(compact_kernel, p, a->pools, a->num_pools, a->page_size, most, std::max<int64_t>({a->num_pages, a->B * P, a->num_free}), static_cast<hipStream_t>(stream));
}
