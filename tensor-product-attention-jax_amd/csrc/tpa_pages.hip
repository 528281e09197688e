// Page tables, slots and positions of a serving step's new tokens, from the requests' lengths, in one launch.
//
// A step's tokens are packed request after request, so what a token needs is its request (from the running sum of the new tokens)
// and, where it opens a page, that page's place in the free list (from the running sum of the pages that the requests before it
// open).  Both sums run over the requests only, a few thousand at most: every workgroup makes them for itself, from cached
// reads, and then serves its own tokens from LDS.  Nothing passes between workgroups, and nothing depends on their order: a token
// that reads the table reads entries below ceil(length / page size), one that writes it writes those above.
//
// Latency bounds it: the requests' lengths, two sums over the workgroup, a search, a table entry.  3.4 us for a token of each of 64 requests, 5.6 us for 384
// requests with up to 512 tokens each (0.3 MB read and written, 0.06 us at the rate of a copy); the host's call takes 7.
#include "tpa_common.h"

namespace tpa {
namespace {

constexpr int kThreads = 256;

struct PageTablesParams {
  const int32_t *kv_lengths, *new_tokens, *free_pages, *free_start;
  int32_t *page_table, *slots, *positions, *starts, *new_kv_lengths, *new_free_start;
  int B, pages_per_seq, page_size, num_free, num_tokens, rows_per_group;
};

// Sums that stop at `most` (below 2^31): associative on numbers that are not negative, and they cannot overflow, whatever the counts are
__device__ __forceinline__ uint32_t stop_at(uint32_t a, uint32_t b, uint32_t most) { return min(a + b, most); }
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t sum_from(uint32_t x, uint32_t most) {
  return stop_at(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false), most);
}
__device__ __forceinline__ uint32_t wave_running_sum(uint32_t x, uint32_t most) {  // lane i: sum of lanes 0 .. i
  x = sum_from<0x111, 0xf>(x, most);  // row_shr 1, 2, 4, 8: inside rows of 16 lanes
  x = sum_from<0x112, 0xf>(x, most);
  x = sum_from<0x114, 0xf>(x, most);
  x = sum_from<0x118, 0xf>(x, most);
  x = sum_from<0x142, 0xa>(x, most);    // row_bcast 15: the last lane of rows 0 and 2 to rows 1 and 3
  return sum_from<0x143, 0xc>(x, most);  // row_bcast 31: lane 31 to rows 2 and 3
}
// sum over the threads before this one; `red` = an int per wave
__device__ __forceinline__ uint32_t sum_before(uint32_t x, uint32_t most, uint32_t* red) {
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const uint32_t upto = wave_running_sum(x, most);
  if (lane == 63) red[w] = upto;
  __syncthreads();
  uint32_t before = 0;
  for (int i = 0; i < w; ++i) before = stop_at(before, red[i], most);
  __syncthreads();
  const uint32_t mine = (uint32_t)__shfl_up((int)upto, 1);
  return stop_at(before, lane ? mine : 0, most);
}

__global__ __launch_bounds__(kThreads) void page_tables_kernel(PageTablesParams p) {
  extern __shared__ int32_t smem[];
  __shared__ uint32_t red[kThreads / 64];
  int32_t* const ends = smem;         // row behind request b's tokens
  int32_t* const firsts = smem + p.B;  // index of request b's first new page in the free list
  const int tid = threadIdx.x;
  const int cap = p.pages_per_seq * p.page_size;
  const int free0 = p.free_start ? max(0, min(p.free_start[0], p.num_free)) : 0;

  // this thread's requests, side by side: their tokens, then the pages that these open, then both in LDS
  const int each = (p.B + kThreads - 1) / kThreads, b0 = min(tid * each, p.B), b1 = min(b0 + each, p.B);
  auto pages_of = [&](int tokens) { return (int)(((uint32_t)tokens + (uint32_t)p.page_size - 1) / (uint32_t)p.page_size); };  // (both below 2^31)
  auto length_of = [&](int b) { return max(0, min(p.kv_lengths[b], cap)); };
  uint32_t tokens = 0;
  for (int b = b0; b < b1; ++b) tokens = stop_at(tokens, (uint32_t)max(p.new_tokens[b], 0), p.num_tokens);
  const uint32_t row0 = sum_before(tokens, p.num_tokens, red);
  // tokens of request b that the table has room for, and the pages that they open
  auto place = [&](int b, uint32_t& row, int& len, int& end, int& have) {
    const uint32_t next = stop_at(row, (uint32_t)max(p.new_tokens[b], 0), p.num_tokens);
    len = length_of(b);
    end = min((int)(next - row), cap - len) + len;
    have = pages_of(len);
    row = next;
    return pages_of(end) - have;
  };
  uint32_t pages = 0, row = row0;
  for (int b = b0, len, end, have; b < b1; ++b) pages = stop_at(pages, place(b, row, len, end, have), p.num_free);
  uint32_t taken = sum_before(pages, p.num_free, red);
  row = row0;
  const bool writes = blockIdx.x == 0;
  for (int b = b0; b < b1; ++b) {
    int len, end, have;
    if (writes) p.starts[b] = row;
    const int want = place(b, row, len, end, have);
    ends[b] = row;
    firsts[b] = free0 + (int)min(taken, (uint32_t)(p.num_free - free0));
    const int got = min(want, p.num_free - firsts[b]);
    if (writes) p.new_kv_lengths[b] = got == want ? end : (have + got) * p.page_size;
    taken = stop_at(taken, want, p.num_free);
    if (b == p.B - 1 && writes) {
      p.starts[p.B] = row;
      p.new_free_start[0] = firsts[b] + got;
    }
  }
  __syncthreads();

  const uint32_t begin = blockIdx.x * (uint32_t)p.rows_per_group, stop = min(begin + (uint32_t)p.rows_per_group, (uint32_t)p.num_tokens);
  for (uint32_t next = begin + tid; next < stop; next += kThreads) {  // (behind the last row up to 2^31 + 255)
    const int r = (int)next;
    if (r >= ends[p.B - 1]) {
      p.slots[r] = -1;
      p.positions[r] = 0;
      continue;
    }
    int lo = 0, hi = p.B - 1;  // the first request whose tokens end behind this row
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (ends[mid] > r) hi = mid;
      else lo = mid + 1;
    }
    const int len = length_of(lo), have = pages_of(len);
    const int64_t pos = (int64_t)len + r - (lo ? ends[lo - 1] : 0);
    int slot = -1;
    if (pos < cap) {
      const int nth = (int)pos / p.page_size, in_page = (int)pos - nth * p.page_size;
      int32_t* const entry = p.page_table + (int64_t)lo * p.pages_per_seq + nth;
      // of a page that 31 bits do not number, or none: no slot
      auto slot_of = [&](int page) {
        const int64_t at = (int64_t)page * p.page_size + in_page;
        return page >= 0 && at <= INT32_MAX ? (int)at : -1;
      };
      if (nth < have) {
        slot = slot_of(*entry);
      } else if (const int64_t at = (int64_t)firsts[lo] + nth - have; at < p.num_free) {
        const int page = p.free_pages[at];
        slot = slot_of(page);
        if (in_page == 0) *entry = page;  // the token that opens a page
      }
    }
    p.slots[r] = slot;
    p.positions[r] = (int)min(pos, (int64_t)INT32_MAX);
  }
}

bool overlap(const int32_t* a, const int32_t* b, int n) { return a < b + n && b < a + n; }

}  // namespace
}  // namespace tpa

extern "C" int tpa_page_tables(const TpaPageTablesArgs* a, void* stream) {
  using namespace tpa;
  if (!a) return TPA_ERR_NULL;
  if (a->B <= 0 || a->B > TPA_PAGE_TABLES_MAX_REQUESTS || a->pages_per_seq <= 0 || a->page_size <= 0 || a->num_free < 0 || a->num_tokens < 0)
    return TPA_ERR_SHAPE;
  if ((int64_t)a->pages_per_seq * a->page_size > INT32_MAX) return TPA_ERR_SHAPE;
  if (!a->kv_lengths || !a->new_tokens || !a->page_table || !a->starts || !a->new_kv_lengths || !a->new_free_start) return TPA_ERR_NULL;
  if ((!a->free_pages && a->num_free) || (a->num_tokens && (!a->slots || !a->positions))) return TPA_ERR_NULL;
  if (overlap(a->kv_lengths, a->new_kv_lengths, a->B) || a->free_start == a->new_free_start) return TPA_ERR_UNSUPPORTED;
  PageTablesParams p{};
  p.kv_lengths = a->kv_lengths; p.new_tokens = a->new_tokens; p.free_pages = a->free_pages; p.free_start = a->free_start;
  p.page_table = a->page_table; p.slots = a->slots; p.positions = a->positions; p.starts = a->starts;
  p.new_kv_lengths = a->new_kv_lengths; p.new_free_start = a->new_free_start;
  p.B = a->B; p.pages_per_seq = a->pages_per_seq; p.page_size = a->page_size; p.num_free = a->num_free; p.num_tokens = a->num_tokens;
  // a row per thread until every compute unit has two workgroups
  const int64_t rounds = ((int64_t)a->num_tokens + 512 * kThreads - 1) / (512 * kThreads);
  const int64_t per = (rounds > 1 ? rounds : 1) * kThreads;
  p.rows_per_group = (int)per;
  const int groups = (int)((a->num_tokens + per - 1) / per);
  hipLaunchKernelGGL(page_tables_kernel, dim3(groups > 0 ? groups : 1), dim3(kThreads), 2 * sizeof(int32_t) * a->B, static_cast<hipStream_t>(stream), p);
  return hipGetLastError() == hipSuccess ? TPA_OK : TPA_ERR_LAUNCH;
}
