// Decode of a batch whose sequences share their first tokens: the shared prefix is read once for all of them.
//
// A query row attends to the keys of the prefix, which are entry 0's, and to the keys behind it, which are its own sequence's; the
// parts are joined by the running maximum and sum of the softmax.
//
// What bounds it: over a long prefix the matrix cores, at the power that the chip has for them - a tile of 4 blocks (64 tokens of rank 2, 256 columns of
// 128) takes 5.8 us, of which its 768 matrix instructions are 3.7 by themselves and LDS 3.0 - and the way in and out: 6 us to a
// first tile, 2 to 3 for the parts, 4 to 9 for the merge.  64 sequences over 8192 + 700 tokens, 32 heads: 50.6 us; 32 over 32768 + 300: 76.2; 4 over
// 1500 + 120, 16 heads: 15.2, as long as the host's call.
#include <algorithm>
#include <cmath>

#include "tpa_common.h"

namespace tpa {
namespace {

struct SharedParams {
  TpaFactor qa, qb, ka, kb, va, vb;
  void* o;
  float* lse;                // [B, H, lq] or null
  const int32_t* kvlen;      // [B] keys of each entry, the prefix's among them, or null (= lk)
  const int32_t* page_table;  // [B, pages_per_seq] or null
  int page_size, pages_per_seq;
  int B, lq, lk, H, dk, dv, rq, rk;
  int prefix;
  int causal, coff;          // as in the decode: with the mask, row i sees its first i + coff + 1 keys (bottom right: + keys - lq)
  float scale;               // sm_scale * log2 e
};

// keys that query row `row` of an entry of `length` keys sees
__device__ __forceinline__ int keys_seen(const SharedParams& p, int length, int row) {
  const int len = max(0, min(length, p.lk));
  if (!p.causal) return len;
  const int64_t last = (int64_t)row + p.coff + 1 + (p.causal == TPA_CAUSAL_BOTTOM_RIGHT ? len - p.lq : 0);
  return (int)max((int64_t)0, min((int64_t)len, last));
}
// element offsets (batch or page, token) of key t of entry b
__device__ __forceinline__ void place_of(const SharedParams& p, int b, int t, int64_t& page, int64_t& at) {
  if (t < p.prefix) b = 0;
  if (p.page_table) {
    const int nth = t / p.page_size;
    page = p.page_table[(int64_t)b * p.pages_per_seq + nth];
    at = t - nth * p.page_size;
  } else {
    page = b;
    at = t;
  }
}

// ---------------------------------------------------------------------------------------------- any shape
// A workgroup per query row and head: 256 keys at a time, a thread's key by itself, then a thread's output column over the keys.
constexpr int kAnyThreads = 256;
template <typename T>
__global__ __launch_bounds__(kAnyThreads) void shared_any_kernel(SharedParams p) {
  __shared__ float q[256], weight[kAnyThreads], red[2][kAnyThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int h = blockIdx.x % p.H;
  const int64_t row_of_all = blockIdx.x / p.H;
  const int b = (int)(row_of_all / p.lq), row = (int)(row_of_all - (int64_t)b * p.lq);
  const T* const qa = static_cast<const T*>(p.qa.ptr) + b * p.qa.stride_b + row * p.qa.stride_l + h;
  const T* const qb = static_cast<const T*>(p.qb.ptr) + b * p.qb.stride_b + row * p.qb.stride_l;
  if (tid < p.dk) {
    float sum = 0.f;
    for (int r = 0; r < p.rq; ++r) sum += load_as_f32(qa + r * p.qa.stride_r) * load_as_f32(qb + r * p.qb.stride_r + tid);
    q[tid] = sum * (p.scale / ((float)p.rq * p.rk));
  }
  __syncthreads();
  const int keys = keys_seen(p, p.kvlen ? p.kvlen[b] : p.lk, row);
  float most = -INFINITY, total = 0.f, out = 0.f;  // the same in all threads; out: of column tid
  for (int t0 = 0; t0 < keys; t0 += kAnyThreads) {
    float x = -INFINITY;
    if (t0 + tid < keys) {
      int64_t page, at;
      place_of(p, b, t0 + tid, page, at);
      const T* const ka = static_cast<const T*>(p.ka.ptr) + page * p.ka.stride_b + at * p.ka.stride_l + h;
      const T* const kb = static_cast<const T*>(p.kb.ptr) + page * p.kb.stride_b + at * p.kb.stride_l;
      x = 0.f;
      for (int r = 0; r < p.rk; ++r) {
        float dot = 0.f;
        for (int d = 0; d < p.dk; ++d) dot += q[d] * load_as_f32(kb + r * p.kb.stride_r + d);
        x += dot * load_as_f32(ka + r * p.ka.stride_r);
      }
    }
    float m = x;
    bool nan = x != x;
#pragma unroll
    for (int s = 32; s; s >>= 1) m = fmaxf(m, __shfl_xor(m, s));
    if (__ballot(nan)) m = NAN;
    if (lane == 0) red[0][w] = m;
    __syncthreads();
    for (int i = 0; i < kAnyThreads / 64; ++i) m = red[0][i] != red[0][i] || m != m ? NAN : fmaxf(m, red[0][i]);
    m = m != m || most != most ? NAN : fmaxf(m, most);
    const float base = m == -INFINITY ? 0.f : m;  // every logit so far -inf: weights of zero
    const float e = exp2f(x - base);
    weight[tid] = t0 + tid < keys ? e : 0.f;
    float sum = weight[tid];
#pragma unroll
    for (int s = 32; s; s >>= 1) sum += __shfl_xor(sum, s);
    if (lane == 0) red[1][w] = sum;
    __syncthreads();
    const float keep = exp2f(most - base);
    total *= keep;
    for (int i = 0; i < kAnyThreads / 64; ++i) total += red[1][i];
    out *= keep;
    most = m;
    if (tid < p.dv) {
      const int n = min(kAnyThreads, keys - t0);
      for (int i = 0; i < n; ++i) {
        int64_t page, at;
        place_of(p, b, t0 + i, page, at);
        const T* const va = static_cast<const T*>(p.va.ptr) + page * p.va.stride_b + at * p.va.stride_l + h;
        const T* const vb = static_cast<const T*>(p.vb.ptr) + page * p.vb.stride_b + at * p.vb.stride_l + tid;
        float v = 0.f;
        for (int r = 0; r < p.rk; ++r) v += load_as_f32(va + r * p.va.stride_r) * load_as_f32(vb + r * p.vb.stride_r);
        out += weight[i] * v;
      }
    }
    __syncthreads();  // the next keys' weights go where these are
  }
  const bool empty = total == 0.f;
  if (tid < p.dv) store_from_f32(static_cast<T*>(p.o) + (row_of_all * p.H + h) * p.dv + tid, empty ? NAN : out / total / (float)p.rk);
  if (tid == 0 && p.lse) p.lse[((int64_t)b * p.H + h) * p.lq + row] = empty ? -INFINITY : (most + log2f(total)) * kLn2;
}

// ---------------------------------------------------------------------------------------------- matrix cores
// As in the split-key decode nothing is expanded to dense keys or values: with Qm[c, :] = (scale / (Rq R)) sum_i qa_i qb_i of column c = (row,
// head) the logits are s[c, t] = sum_r ka[t, r, h] (Qm[c, :] . kb[t, r, :]), the output (1 / R) sum_t sum_r (p[c, t] va[t, r, h]) vb[t, r, :], two
// products of the rows (t, r) with the columns.  The rows serve every column, so a workgroup takes a tile of 4 blocks of 32 rows
// once for up to 256 columns: the columns of the prefix are those of all sequences, 32 to a wave; where there are fewer (a sequence's
// own keys, few sequences) waves share the tile's blocks and are joined at the end.  Tiles go from memory straight to LDS, two
// buffers.  (Dense keys would halve the matrix work at rank 2, but every wave would have to build them: 32 columns a head use a key
// once.  By count only; sets of 32 query rows of one head, which would use a key 32 times, were not built either.)
// Qm is kept as two bf16 numbers, 2^-17 of it off: with one the logits carry the rounding of Qm, 2^-9 each, and the output's error
// grows by half; the second costs 8 of 24 matrix instructions a block.  The weights p va are rounded to bf16 once, sums are fp32.
// In fp32 nothing is rounded, a tile has 2 blocks, and what a product takes is read as it lies: over d the halves of a wave take d = 8 m + 4 g + e
// in turn (16 bytes of a row feed four products), over a block's rows the row that their logits' register belongs to, and row i of
// block db of the output is d = (D / 32) i + db, so that one read of a v row serves all blocks.
constexpr int kRows = 32;           // rows (token, rank) of a block
constexpr int kWaves = 8;
constexpr int kRsrcFlags = 0x00020000;  // raw 32-bit data format
constexpr int64_t kFarthestRow = 1 << 26;  // bytes between neighbouring rows, at most: 31 of them in 32-bit byte offsets
constexpr int blocks_of_tile(int bytes) { return bytes == 2 ? 4 : 2; }  // of numbers of so many bytes

template <typename T, int D>
struct SharedLds {
  static constexpr int kBlocks = blocks_of_tile(sizeof(T));
  static constexpr int kB = kRows * D * sizeof(T), kA = kRows * 32 * sizeof(T);  // bytes of a block's b rows, a rows (32 heads)
  static constexpr int kBuffer = kBlocks * 2 * (kB + kA);                     // kb, vb, ka, va of a tile
  static constexpr int kPart = 32 * D * 4 + 2 * 64 * 4;                       // a wave's sums of a set of columns on their way to others
  static constexpr size_t kBytes = 2 * kBuffer;
  static_assert(kWaves * kPart <= 2 * kBuffer, "what all waves hand over fits the buffers");
};

// Columns come in sets of 32: the heads of a block of heads (8, 16, 24 or 32) for as many query rows as fit, so that all sets have the same head
// factors.
struct SharedPart {        // the prefix, or the sequences' own keys
  int waves, side;         // waves side by side over the columns, waves that share the blocks of each
  int groups;              // workgroups for all columns of a block of heads
  int ranges, blocks;      // key ranges, blocks of a range
  int grid;                // workgroups
};
struct SharedPlan {
  int hb, nhb;             // heads of a block of heads, blocks of heads
  SharedPart prefix, own;
  int64_t rows;            // B lq
};
struct SharedMfmaParams {
  SharedParams c;
  SharedPlan plan;
  float *part_o, *part_m, *part_l;  // [range][B lq][H][D], [range][B lq][H]: the prefix's ranges, then the own keys'
  float qscale;
  int page_shift;  // log2 of the rows of a page, or -1
};

// Where a lane's pieces of a block of rows of D lie in LDS (elements): 16-byte chunk c of row r at chunk c ^ f(r), so that neither the reads of
// one chunk of 16 rows nor the transposed ones of 4 chunks of 4 rows meet a bank twice
template <typename T, int D>
struct BlockAt;
template <int D>
struct BlockAt<uint16_t, D> {
  static constexpr int CPR = D / 8;
  __device__ __forceinline__ static int f(int r) { return CPR == 16 ? (r & 3) << 2 | (r >> 2 & 3) : (r >> 1 & 1) << 2 | (r >> 2 & 3); }
  int row, tr;
  __device__ __forceinline__ explicit BlockAt(int l) {
    const int i = l & 31, g = l >> 5, lp = l & 15, dhalf = (l >> 4) & 1, r = 4 * g + (lp >> 2);
    row = i * D + 8 * (g ^ f(i));
    tr = r * D + 8 * ((2 * dhalf + ((lp & 3) >> 1)) ^ f(r)) + 4 * (lp & 1);
  }
  __device__ __forceinline__ int read(int ks) const { return row ^ (16 * ks); }  // row i, chunk 2 ks + g
  // transposed: rows 16 kk + 8 hi + 4 g + 0..3, columns 32 db + 0..31
  __device__ __forceinline__ int read_tr(int kk, int hi, int db) const { return (tr ^ (32 * db) ^ (16 * hi)) + (16 * kk + 8 * hi) * D; }
};
template <int D>
struct BlockAt<float, D> {
  __device__ __forceinline__ static int f(int r) { return r & 15; }
  int l, row;
  __device__ __forceinline__ explicit BlockAt(int lane) : l(lane), row((lane & 31) * D + 4 * ((lane >> 5) ^ f(lane & 31))) {}
  __device__ __forceinline__ int read(int m) const { return row ^ (8 * m); }  // row i, chunk 2 m + g
  // columns D / 32 i and following of the row of register v
  __device__ __forceinline__ int read_v(int v) const {
    const int i = l & 31, r = 8 * (v >> 2) + 4 * (l >> 5) + (v & 3), at = D / 32 * i;
    return r * D + (at ^ (4 * f(r)));
  }
};
typedef s16x4 __attribute__((address_space(3))) lds_s16x4;
template <int D>
__device__ __forceinline__ bf16x8 block_tr(const uint16_t* block, const BlockAt<uint16_t, D>& at, int kk, int db) {
  const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(block + at.read_tr(kk, 0, db)));
  const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(block + at.read_tr(kk, 1, db)));
  return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

template <typename T, int D, int RK, bool PAGED>
__device__ __forceinline__ void shared_part(const SharedMfmaParams& p, const SharedPart& part, bool own, int id, unsigned char* mem) {
  using Lds = SharedLds<T, D>;
  using At = BlockAt<T, D>;
  constexpr bool F32 = sizeof(T) == 4;
  constexpr int kBlocks = Lds::kBlocks, kSize = sizeof(T), kPer = 16 / kSize;  // kPer: numbers of a load of 16 bytes
  constexpr int WPB = kWaves / kBlocks, RPW = kRows / WPB;                     // waves that bring a block, rows of each
  constexpr int NKS = D / 16, NDB = D / 32, CPR = D / kPer, RPI = 64 / CPR, NI = RPW / RPI;  // NI: load instructions of a wave's b rows
  constexpr int TPB = kRows / RK;                                                           // tokens of a block
  constexpr int NTOK = RK <= 4 ? 16 / RK : 32 / RK;  // tokens whose rows this lane holds, per block
  constexpr int NV = RK <= 4 ? RK : RK / 2;          // rows of one token held by this half of the wave
  const SharedParams& c = p.c;
  const SharedPlan& plan = p.plan;
  const int tid = threadIdx.x, w = scalar(tid >> 6), l = tid & 63, i = l & 31, g = l >> 5, lp = l & 15, dhalf = (l >> 4) & 1;

  // ---- which keys and columns: workgroups that read the same keys sit on one XCD (ids are dealt to the eight in turn)
  const int sharing = plan.nhb * part.groups;
  const int unit = id / (8 * sharing) * 8 + (id & 7), member = id / 8 % sharing;
  if (unit >= (own ? c.B * part.ranges : part.ranges)) return;
  const int b_own = own ? unit / part.ranges : 0, range = own ? unit - b_own * part.ranges : unit;
  const int h0 = member % plan.nhb * plan.hb, rps = plan.hb >= 24 ? 1 : plan.hb == 16 ? 2 : 4;  // rows of a set
  const int cwaves = part.waves, kwaves = part.side, cw = w & (cwaves - 1), kw = w >> __builtin_ctz(cwaves);
  const int n_rows = own ? c.lq : (int)plan.rows, wave_row = (member / plan.nhb * cwaves + cw) * rps;  // this wave's first row
  const bool works = kw < kwaves && wave_row < n_rows;
  auto in_block = [&](int x) __attribute__((always_inline)) { return plan.hb == 24 ? (x >= 24 ? x - 24 : x) : x & (plan.hb - 1); };  // x % hb, x < 32
  const int in_set = rps == 1 ? 0 : i >> __builtin_ctz(plan.hb), head = h0 + in_block(i);  // lanes behind the last whole row of a set repeat it
  const bool stored = wave_row + in_set < n_rows && i < rps * plan.hb;
  const int row = (own ? b_own * c.lq : 0) + min(wave_row + in_set, n_rows - 1);  // this lane's query row among all
  const int b = c.lq == 1 ? row : row / c.lq, row_in_b = row - b * c.lq;

  // ---- keys of this part that a column sees: those below `mine`; the workgroup's range ends with the last that any of them sees
  auto row_among_all = [&](int of) __attribute__((always_inline)) { return (own ? b_own * c.lq : 0) + min(of, n_rows - 1); };  // row `of` of this part's
  const int row_of[2] = {row, row_among_all(member / plan.nhb * cwaves * rps + min(l, cwaves * rps - 1))};
  const int entry_of[2] = {b, c.lq == 1 ? row_of[1] : row_of[1] / c.lq};
  int length_of[2] = {c.lk, c.lk};
  if (c.kvlen) {  // (nothing but the loads here, which would be waited for one by one)
    length_of[0] = c.kvlen[entry_of[0]];
    length_of[1] = c.kvlen[entry_of[1]];
  }
  // ---- the range's rows (token, rank), in blocks from a block's border on
  const int origin = own ? c.prefix / TPB * TPB : 0;
  const int begin = origin + range * part.blocks * TPB;
  const int rpp = PAGED ? c.page_size * RK : 1;
  auto block_row = [&](int tile) __attribute__((always_inline)) { return begin * RK + (tile * kBlocks + w / WPB) * kRows; };
  auto page_of = [&](int row0) __attribute__((always_inline)) { return p.page_shift >= 0 ? row0 >> p.page_shift : row0 / rpp; };
  auto lookup = [&](int tile, int rows) __attribute__((always_inline)) -> int {  // of a cache of so many rows
    if constexpr (!PAGED) return 0;
    return c.page_table[(int64_t)b_own * c.pages_per_seq + page_of(min(block_row(tile), rows - 1) / kRows * kRows)];
  };
  const int first_page = lookup(0, c.lk * RK);  // asked for before it is known whether there are keys

  // ---- Qm^T[d, c] = sum_r qb[r, d] qa[r, c] by the matrix cores in bf16, 16 ranks a step, a set's rows one after the other with the other rows'
  // columns zero; qb's rows go by LDS (the second buffer, a part for each wave), which transposes them.  Asked for here, two steps in flight, finished while
  // the first tile is on its way.
  constexpr int QRPI = F32 ? 1 : 64 / (D / 8), QL = 16 / QRPI;  // rows of a load instruction, loads of 16 rows
  struct QIn { uint16_t a[8]; u32x4 b[QL]; };
  [[maybe_unused]] QIn q_in[2];
  // (steps in order: the ranks of a row, the next row)
  struct QStep { int in_row, r0; };
  [[maybe_unused]] auto after = [&](const QStep& n) __attribute__((always_inline)) { return n.r0 + 16 < c.rq ? QStep{n.in_row, n.r0 + 16} : QStep{n.in_row + 1, 0}; };
  [[maybe_unused]] auto request_q = [&](QIn& in, const QStep& n) __attribute__((always_inline)) {
    const auto [in_row, r0] = n;
    const int of = (own ? b_own * c.lq : 0) + min(wave_row + in_row, n_rows - 1), ob = c.lq == 1 ? of : of / c.lq;
    const uint16_t* const qa = static_cast<const uint16_t*>(c.qa.ptr) + ob * c.qa.stride_b + (of - ob * c.lq) * c.qa.stride_l + head;
    const uint16_t* const qb = static_cast<const uint16_t*>(c.qb.ptr) + ob * c.qb.stride_b + (of - ob * c.lq) * c.qb.stride_l + 8 * (l % (D / 8));
#pragma unroll
    for (int x = 0; x < QL; ++x) in.b[x] = *reinterpret_cast<const u32x4*>(qb + min(r0 + x * QRPI + l / (D / 8), c.rq - 1) * c.qb.stride_r);
#pragma unroll
    for (int j = 0; j < 8; ++j) in.a[j] = qa[min(r0 + 8 * (j / 4) + 4 * g + j % 4, c.rq - 1) * c.qa.stride_r];
  };
  if constexpr (!F32) request_q(q_in[0], QStep{0, 0});  // (in no branch, behind which the keys would be waited for together with it)

  auto keys_of = [&](int x) __attribute__((always_inline)) {
    const int seen = keys_seen(c, length_of[x], row_of[x] - entry_of[x] * c.lq);
    return own ? seen : min(seen, c.prefix);
  };
  const int mine = keys_of(0), least = scalar(wave_min(mine)), end = scalar(wave_max(keys_of(1)));
  const int stop = min(end, begin + part.blocks * TPB);
  const int64_t slot = ((own ? plan.prefix.ranges : 0) + range) * plan.rows;
  if (stop <= begin || stop <= (own ? c.prefix : 0)) {  // no key of this range is seen
    if (works && kw == 0 && g == 0 && stored) p.part_m[(slot + row) * c.H + head] = -INFINITY;
    return;
  }
  const int n_tiles = (stop - begin + kBlocks * TPB - 1) / (kBlocks * TPB);
  const int row_end = stop * RK;  // rows from here on read as zeros

  // ---- loads: wave w brings RPW rows of block w / WPB of a tile; a lane's chunk is the one that belongs where it lands
  typedef uint32_t Resource __attribute__((ext_vector_type(4)));
  const int64_t boff = PAGED ? 0 : b_own;
  const T* const base[4] = {static_cast<const T*>(c.kb.ptr) + boff * c.kb.stride_b, static_cast<const T*>(c.vb.ptr) + boff * c.vb.stride_b,
                            static_cast<const T*>(c.ka.ptr) + boff * c.ka.stride_b + h0, static_cast<const T*>(c.va.ptr) + boff * c.va.stride_b + h0};
  const int64_t page_stride[4] = {c.kb.stride_b, c.vb.stride_b, c.ka.stride_b, c.va.stride_b};
  const int sr[4] = {kSize * (int)c.kb.stride_r, kSize * (int)c.vb.stride_r, kSize * (int)c.ka.stride_r, kSize * (int)c.va.stride_r};
  constexpr int ACH = 32 / kPer;  // 16-byte chunks of a row of 32 heads
  const int a_row = RPW * (w % WPB) + l / ACH, b_row = RPW * (w % WPB) + l / CPR;
  const int a_chunk = 16 * min(l % ACH, plan.hb / kPer - 1), b_chunk = 16 * ((l % CPR) ^ At::f(b_row));  // and of row b_row + n RPI: f differs by f(n RPI)
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)mem;
  auto load = [&](uint32_t to, int at, const Resource& rs) __attribute__((always_inline)) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(to), "v"(at), "s"(rs) : "memory");
  };
  auto issue = [&](int tile, int buffer, int page) __attribute__((always_inline)) {
    // rows behind the last key and, in a sequence's own first block, those of the prefix are outside the resource and read as zeros (a
    // lane's offset below it is one of nearly 2^32)
    const int row0 = block_row(tile), skip = own ? max(0, c.prefix * RK - row0) : 0, rows = min(kRows, row_end - row0) - skip;
    const int64_t first = (PAGED ? row0 - page_of(row0) * rpp : row0) + skip;
    const uint32_t to = lds0 + buffer * Lds::kBuffer;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const uintptr_t at = reinterpret_cast<uintptr_t>(base[x] + (PAGED ? (int64_t)page * page_stride[x] : 0) + first * (sr[x] / kSize));
      const int width = kSize * (x < 2 ? D : plan.hb);
      const Resource rs = {(uint32_t)scalar((int)(uint32_t)at), (uint32_t)scalar((int)((uint32_t)(at >> 32) & 0xffff)), (uint32_t)scalar(rows > 0 ? (rows - 1) * sr[x] + width : 0),
                           (uint32_t)kRsrcFlags};
      if (x < 2) {
#pragma unroll
        for (int n = 0; n < NI; ++n)
          load((uint32_t)scalar(to + (x * kBlocks + w / WPB) * Lds::kB + (NI * (w % WPB) + n) * 1024), (b_row + n * RPI - skip) * sr[x] + (b_chunk ^ (16 * At::f(n * RPI))), rs);
      } else {
        load((uint32_t)scalar(to + 2 * kBlocks * Lds::kB + ((x - 2) * kBlocks + w / WPB) * Lds::kA + (w % WPB) * 1024), (a_row - skip) * sr[x] + a_chunk, rs);
      }
    }
  };
  issue(0, 0, block_row(0) < row_end ? scalar(first_page) : 0);
  int page_ahead = lookup(1, row_end);

  // ---- Qm of this lane's column as the operand of its products: in bf16 d = 16 ks + 8 g + 0..7, in two parts, in fp32 d = 8 m + 4 g + e
  [[maybe_unused]] bf16x8 q_hi[NKS], q_lo[NKS];
  [[maybe_unused]] float qf[D / 2];
  f32x16 o[NDB];
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int v = 0; v < 16; ++v) o[db][v] = 0.f;
  if constexpr (F32) {
    if (works) {
      const T* const qa = static_cast<const T*>(c.qa.ptr) + b * c.qa.stride_b + row_in_b * c.qa.stride_l + head;
      const T* const qb = static_cast<const T*>(c.qb.ptr) + b * c.qb.stride_b + row_in_b * c.qb.stride_l + 4 * g;
#pragma unroll
      for (int x = 0; x < D / 2; ++x) qf[x] = 0.f;
      for (int r = 0; r < c.rq; ++r) {
        const float a = qa[r * c.qa.stride_r];
#pragma unroll
        for (int mm = 0; mm < D / 8; ++mm) {
          const f32x4 x = *reinterpret_cast<const f32x4*>(qb + r * c.qb.stride_r + 8 * mm);
#pragma unroll
          for (int e = 0; e < 4; ++e) qf[4 * mm + e] = fmaf(a, x[e], qf[4 * mm + e]);
        }
      }
#pragma unroll
      for (int x = 0; x < D / 2; ++x) qf[x] *= p.qscale;
    }
  } else {
    const BlockAt<uint16_t, D> q_at(l);
    uint16_t* const rows_at = reinterpret_cast<uint16_t*>(mem + Lds::kBuffer + w * (16 * D * 2));
    f32x16 sum[NDB];
    auto use_q = [&](const QIn& in, const QStep& n) __attribute__((always_inline)) {
      const auto [in_row, r0] = n;
#pragma unroll
      for (int x = 0; x < QL; ++x) {
        const int r = x * QRPI + l / (D / 8);
        *reinterpret_cast<u32x4*>(rows_at + r * D + 8 * (l % (D / 8) ^ BlockAt<uint16_t, D>::f(r))) = r0 + r < c.rq ? in.b[x] : u32x4{0, 0, 0, 0};
      }
      u32x4 a;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = r0 + 8 * (j / 2) + 4 * g + 2 * j % 4;
        const uint32_t lo = r < c.rq ? 0xffffu : 0u, hi = r + 1 < c.rq ? 0xffff0000u : 0u;
        a[j] = in_set == in_row ? (((uint32_t)in.a[2 * j + 1] << 16 | in.a[2 * j]) & (lo | hi)) : 0u;
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (r0 == 0)
#pragma unroll
        for (int db = 0; db < NDB; ++db)
#pragma unroll
          for (int v = 0; v < 16; ++v) sum[db][v] = 0.f;
#pragma unroll
      for (int db = 0; db < NDB; ++db) sum[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(block_tr<D>(rows_at, q_at, 0, db), __builtin_bit_cast(bf16x8, a), sum[db], 0, 0, 0);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (r0 + 16 >= c.rq)  // the row's own columns: another row's infinities stay with it
#pragma unroll
        for (int db = 0; db < NDB; ++db)
#pragma unroll
          for (int v = 0; v < 16; ++v) o[db][v] = in_set == in_row ? sum[db][v] : o[db][v];
    };
    if (works) {
      QStep now = {0, 0}, then = after(now);
      if (then.in_row < rps) request_q(q_in[1], then);
      for (;;) {
        use_q(q_in[0], now);
        if (then.in_row >= rps) break;
        now = after(then);
        if (now.in_row < rps) request_q(q_in[0], now);
        use_q(q_in[1], then);
        if (now.in_row >= rps) break;
        then = after(now);
        if (then.in_row < rps) request_q(q_in[1], then);
      }
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks) {
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float q0 = o[ks / 2][8 * (ks & 1) + 2 * j] * p.qscale, q1 = o[ks / 2][8 * (ks & 1) + 2 * j + 1] * p.qscale;
          hi[j] = pack_bf16(q0, q1);
          lo[j] = pack_bf16(q0 - bf16lo_to_f32(hi[j]), q1 - bf16hi_to_f32(hi[j]));
        }
        // a result column has d = 8 q + 4 g + e of its block: the halves exchange for the operand's order
        auto order = [&](const uint32_t (&x)[4]) __attribute__((always_inline)) {
          const auto even = __builtin_amdgcn_permlane32_swap(x[0], x[2], false, false), odd = __builtin_amdgcn_permlane32_swap(x[1], x[3], false, false);
          return __builtin_bit_cast(bf16x8, u32x4{even[0], odd[0], even[1], odd[1]});
        };
        q_hi[ks] = order(hi);
        q_lo[ks] = order(lo);
      }
    }
  }
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int v = 0; v < 16; ++v) o[db][v] = 0.f;
  float m = -INFINITY, lsum = 0.f;
  const At at(l);
  [[maybe_unused]] const int a_head = in_block(16 * dhalf + 4 * (lp & 3));  // of the four columns whose a's this lane helps to transpose
  const int row_first = own ? c.prefix * RK : 0;

  struct Block { const T *kb, *vb, *ka, *va; int row0; };
  auto block_of = [&](int tile, int blk) __attribute__((always_inline)) {
    const unsigned char* const buf = mem + (tile & 1) * Lds::kBuffer;
    const T* const ka = reinterpret_cast<const T*>(buf + 2 * kBlocks * Lds::kB + blk * Lds::kA);
    return Block{reinterpret_cast<const T*>(buf + blk * Lds::kB), reinterpret_cast<const T*>(buf + (kBlocks + blk) * Lds::kB), ka, ka + kBlocks * Lds::kA / kSize,
                 begin * RK + (tile * kBlocks + blk) * kRows};
  };
  auto step = [&](const Block& x) __attribute__((always_inline)) {
    // S'^T[row, c] = kb[row, :] . Qm[c, :]
    f32x16 sp;
#pragma unroll
    for (int v = 0; v < 16; ++v) sp[v] = 0.f;
    float ak[16], av[16];
    if constexpr (F32) {
      f32x16 odd;  // a second chain of sums
#pragma unroll
      for (int v = 0; v < 16; ++v) odd[v] = 0.f;
#pragma unroll
      for (int mm = 0; mm < D / 8; ++mm) {
        const f32x4 kf = *reinterpret_cast<const f32x4*>(x.kb + at.read(mm));
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          sp = __builtin_amdgcn_mfma_f32_32x32x2f32(kf[e], qf[4 * mm + e], sp, 0, 0, 0);
          odd = __builtin_amdgcn_mfma_f32_32x32x2f32(kf[e + 1], qf[4 * mm + e + 1], odd, 0, 0, 0);
        }
      }
      const int a_at = 4 * g * 32 + head - h0;
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        sp[v] += odd[v];
        ak[v] = x.ka[a_at + (8 * (v >> 2) + (v & 3)) * 32];
        av[v] = x.va[a_at + (8 * (v >> 2) + (v & 3)) * 32];
      }
    } else {
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks) {
        const bf16x8 kf = *reinterpret_cast<const bf16x8*>(x.kb + at.read(ks));
        sp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, q_lo[ks], sp, 0, 0, 0);
        sp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, q_hi[ks], sp, 0, 0, 0);
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int a_at = (8 * q + 4 * g + (lp >> 2)) * 32 + a_head;
        const s16x4 tk = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(x.ka + a_at));
        const s16x4 tv = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(x.va + a_at));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          ak[4 * q + j] = bf16bits_to_f32((uint16_t)tk[j]);
          av[4 * q + j] = bf16bits_to_f32((uint16_t)tv[j]);
        }
      }
    }
    // logits per token (log2 domain); a token's rows are registers v0 .. v0 + NV - 1, at rank 8 in both halves of the wave
    float st[NTOK];
#pragma unroll
    for (int t = 0; t < NTOK; ++t) {
      float acc = 0.f;
#pragma unroll
      for (int j = 0; j < NV; ++j) acc = fmaf(ak[t * NV + j], sp[t * NV + j], acc);
      if constexpr (RK >= 8) acc = halves_sum(acc);
      st[t] = acc;
    }
    if (x.row0 + kRows > least * RK || x.row0 < row_first) {
#pragma unroll
      for (int t = 0; t < NTOK; ++t) {
        const int at_row = RK >= 8 ? x.row0 + RK * t : x.row0 + 8 * (t * NV >> 2) + 4 * g + (t * NV & 3);  // the token's first row
        if (at_row >= mine * RK || at_row < row_first) st[t] = -INFINITY;
      }
    }
    float tmax = st[0];
#pragma unroll
    for (int t = 1; t < NTOK; ++t) tmax = fmaxf(tmax, st[t]);
    tmax = halves_max(tmax);
    // the reference is the largest logit when it was set, and set again where one more than twice as heavy comes: what weighs most by far then
    // has the weight 1, whose product with va needs no rounding, and the sums are rescaled seldom
    const float m_new = tmax > m + 1.f ? tmax : m;
    const float m_use = m_new == -INFINITY ? 0.f : m_new;
    if (__any(m_new > m)) {
      const float alpha = __builtin_amdgcn_exp2f(m - m_use);
      lsum *= alpha;
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[db][v] *= alpha;
      m = m_new;
    }
    float pp[16];
#pragma unroll
    for (int t = 0; t < NTOK; ++t) {
      const float pt = __builtin_amdgcn_exp2f(st[t] - m_use);
      lsum += RK >= 8 ? 0.5f * pt : pt;  // at rank 8 both halves hold the token: each adds half of it
#pragma unroll
      for (int j = 0; j < NV; ++j) pp[t * NV + j] = pt * av[t * NV + j];
    }
    // O^T[d, c] += sum_row vb[row, d] P'[row, c]; in bf16 slot (g, j) = row 16 kk + 8 (j / 4) + 4 g + j % 4
    if constexpr (F32) {
      typedef float Values __attribute__((ext_vector_type(NDB)));
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        const Values vf = *reinterpret_cast<const Values*>(x.vb + at.read_v(v));
#pragma unroll
        for (int db = 0; db < NDB; ++db) o[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(vf[db], pp[v], o[db], 0, 0, 0);
      }
    } else {
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        u32x4 pk;
#pragma unroll
        for (int j = 0; j < 4; ++j) pk[j] = pack_bf16(pp[8 * kk + 2 * j], pp[8 * kk + 2 * j + 1]);
#pragma unroll
        for (int db = 0; db < NDB; ++db)
          o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(block_tr<D>(x.vb, at, kk, db), __builtin_bit_cast(bf16x8, pk), o[db], 0, 0, 0);
      }
    }
  };

  for (int t = 0; t < n_tiles; ++t) {
    // this wave's part of tile t has landed and nobody reads the other buffer any more; behind the barrier everyone's has
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (t + 1 < n_tiles) {
      issue(t + 1, (t + 1) & 1, scalar(page_ahead));
      page_ahead = lookup(t + 2, row_end);
    }
    if (works)
      for (int blk = kw; blk < kBlocks; blk += kwaves) {
        const Block x = block_of(t, blk);
        if (x.row0 < row_end) step(x);
      }
  }

  // ---- results: in pieces of four neighbouring d, 16 bytes a lane
  constexpr int NP = NDB * 4;
  auto piece = [&](int x) __attribute__((always_inline)) {
    f32x4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = F32 ? o[e % NDB][x * 4 / NDB + e / NDB] : o[x / 4][4 * (x % 4) + e];
    return y;
  };
  const int64_t to = (slot + row) * c.H + head;
  // (not for this XCD's cache, where the kernel's end would wait for its way out: 12 sequences of 4 tokens over 4096, 64 heads of 64: 45.5 -> 44.0 us)
  auto store = [&](int x, const f32x4& y) __attribute__((always_inline)) {
    const int v = x * 4 / NDB, d = F32 ? NDB * (8 * (v >> 2) + 4 * g + (v & 3)) : 32 * (x / 4) + 8 * (x % 4) + 4 * g;
    __builtin_nontemporal_store(y, reinterpret_cast<f32x4*>(p.part_o + to * D + d));
  };
  lsum = halves_sum(lsum);
  if (kwaves == 1) {
    if (!works || !stored) return;
#pragma unroll
    for (int x = 0; x < NP; ++x) store(x, piece(x));
  } else {  // the waves that shared the blocks are joined: each puts all it has into LDS and adds up its share of the pieces
    float* const parts = reinterpret_cast<float*>(mem + cw * Lds::kPart);
    const int next = cwaves * Lds::kPart / 4;
    __syncthreads();  // the tiles have been read
    if (works) {
      float* const mine_of = parts + kw * next;
#pragma unroll
      for (int x = 0; x < NP; ++x) *reinterpret_cast<f32x4*>(mine_of + 256 * x + 4 * l) = piece(x);
      mine_of[32 * D + l] = m;
      mine_of[32 * D + 64 + l] = lsum;
    }
    __syncthreads();
    if (!works || !stored) return;
    float weight[kBlocks];
    m = -INFINITY;
#pragma unroll
    for (int k = 0; k < kBlocks; ++k) {
      weight[k] = k < kwaves ? parts[k * next + 32 * D + l] : -INFINITY;
      m = fmaxf(m, weight[k]);
    }
    const float base_m = m == -INFINITY ? 0.f : m;
    lsum = 0.f;
#pragma unroll
    for (int k = 0; k < kBlocks; ++k) {
      weight[k] = __builtin_amdgcn_exp2f(weight[k] - base_m);
      if (k < kwaves) lsum += weight[k] * parts[k * next + 32 * D + 64 + l];
    }
#pragma unroll 2
    for (int x = kw * (NP / kwaves); x < (kw + 1) * (NP / kwaves); ++x) {
      f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < kBlocks; ++k)
        if (k < kwaves) sum += weight[k] * *reinterpret_cast<const f32x4*>(parts + k * next + 256 * x + 4 * l);
      store(x, sum);
    }
    if (kw) return;
  }
  if (g == 0) {
    // (a range in which all logits are NaN has not moved m, and -inf would say that it has no keys)
    p.part_m[to] = lsum != lsum ? NAN : m;
    p.part_l[to] = lsum;
  }
}

template <typename T, int D, int RK, bool PAGED>
__global__ __launch_bounds__(kWaves * 64, 2) void shared_mfma_kernel(SharedMfmaParams p) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char shared_mem[];
  const bool own = (int)blockIdx.x >= p.plan.prefix.grid;
  const SharedPart& part = own ? p.plan.own : p.plan.prefix;
  const int id = (int)blockIdx.x - (own ? p.plan.prefix.grid : 0);
  shared_part<T, D, RK, PAGED>(p, part, own, id, shared_mem);
}

// Joins the ranges' parts: W waves per query row and head.  A wave's lanes take a range each for the weights; then groups of D / 4 lanes, 16
// bytes a lane, walk the ranges side by side with several loads on their way, and are added up.
template <typename T, int D, int W>
__global__ __launch_bounds__(256) void shared_merge_kernel(SharedMfmaParams p) {
  constexpr int TPR = D / 4, GROUPS = 64 / TPR * W, AHEAD = 8;
  __shared__ f32x4 from_wave[W == 1 ? 1 : W - 1][TPR];
  const SharedParams& c = p.c;
  const int w = scalar(threadIdx.x >> 6), lane = threadIdx.x & 63, grp = lane / TPR + (W == 1 ? 0 : w * (64 / TPR)), d = 4 * (lane % TPR);
  const int ranges = p.plan.prefix.ranges + p.plan.own.ranges;
  const int64_t n = p.plan.rows * c.H, at = W == 1 ? (int64_t)blockIdx.x * 4 + w : blockIdx.x;
  if (at >= n) return;
  float most = -INFINITY, total = 0.f;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f}, part[AHEAD];
  auto request = [&](int first, int count) __attribute__((always_inline)) {  // ranges first .. first + count - 1
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
      if (u * GROUPS < count) part[u] = *reinterpret_cast<const f32x4*>(p.part_o + ((first + min(u * GROUPS + grp, count - 1)) * n + at) * D + d);
  };
  for (int x0 = 0; x0 < ranges; x0 += 64) {
    const bool there = x0 + lane < ranges;
    const int count = min(64, ranges - x0);
    request(x0, min(count, GROUPS * AHEAD));  // beside the maxima; a range without keys has left here what was there
    const float m = there ? p.part_m[(x0 + lane) * n + at] : -INFINITY, l = there ? p.part_l[(x0 + lane) * n + at] : 0.f;
    float m_new = m;
#pragma unroll
    for (int s = 32; s; s >>= 1) m_new = fmaxf(m_new, __shfl_xor(m_new, s));
    m_new = fmaxf(m_new, most);
    const float base = m_new == -INFINITY ? 0.f : m_new, keep = __builtin_amdgcn_exp2f(most - base);
    const float f = __builtin_amdgcn_exp2f(m - base);
    total = total * keep + (m == -INFINITY ? 0.f : f * l);  // a range without keys has written nothing but its maximum
    sum *= keep;
    most = m_new;
    for (int x = 0; x < count; x += GROUPS * AHEAD) {
      if (x) request(x0 + x, min(count - x, GROUPS * AHEAD));
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int mine = x + u * GROUPS + grp;
        const float g = __shfl(f, min(mine, 63)), gm = __shfl(m, min(mine, 63));
        if (mine < count && gm != -INFINITY) sum += g * part[u];
      }
    }
  }
#pragma unroll
  for (int s = 32; s; s >>= 1) total += __shfl_xor(total, s);
#pragma unroll
  for (int s = 32; s >= TPR; s >>= 1)
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[e] += __shfl_xor(sum[e], s);
  if constexpr (W > 1) {
    if (w && lane < TPR) from_wave[w - 1][lane] = sum;
    __syncthreads();
    if (w) return;
#pragma unroll
    for (int x = 0; x < W - 1; ++x) sum += from_wave[x][lane % TPR];
  }
  const bool empty = most == -INFINITY && total == 0.f;  // (the maxima above pass over NaN, the sums do not)
  const float inv = empty ? NAN : 1.f / (total * c.rk);
  T* const out = static_cast<T*>(c.o) + at * D + d;
  if (lane < TPR) {
    if constexpr (sizeof(T) == 2) *reinterpret_cast<u32x2*>(out) = u32x2{pack_bf16(sum[0] * inv, sum[1] * inv), pack_bf16(sum[2] * inv, sum[3] * inv)};
    else *reinterpret_cast<f32x4*>(out) = f32x4{sum[0] * inv, sum[1] * inv, sum[2] * inv, sum[3] * inv};
  }
  if (lane == 0 && c.lse) {
    const int64_t row = at / c.H;
    const int h = (int)(at - row * c.H), b = (int)(row / c.lq);
    c.lse[((int64_t)b * c.H + h) * c.lq + (row - (int64_t)b * c.lq)] = empty ? -INFINITY : (most + __log2f(total)) * kLn2;
  }
}

// Below so many rows and heads four waves share one: the chip has 1024 SIMDs.  (us of the call with one / four waves: 64 rows and heads 18.7 / 14.8,
// 512 57.5 / 54.1, 1024 77.9 / 78.0, 2048 54.7 / 56.3.)
constexpr int64_t kMergeWaves = 1024;

bool aligned16(const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15) == 0; }
int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

bool mfma_takes(const TpaFwdArgs* a) {
  if (a->kernel == TPA_KERNEL_GENERIC) return false;
  const int size = a->dtype == TPA_DTYPE_BF16 ? 2 : 4, per = 16 / size;
  if (a->dk != a->dv || (a->dk != 64 && a->dk != 128)) return false;
  if (a->rk != 1 && a->rk != 2 && a->rk != 4 && a->rk != 8) return false;
  if (a->H % 8) return false;
  // rows (token, rank) are uniformly strided and lie where 32-bit offsets reach; 16-byte loads
  const TpaFactor* fs[4] = {&a->ka, &a->kb, &a->va, &a->vb};
  for (const TpaFactor* f : fs) {
    if (f->stride_l != (int64_t)a->rk * f->stride_r || f->stride_r < 0 || f->stride_r > kFarthestRow / size) return false;
    if (!aligned16(f->ptr) || f->stride_r % per || f->stride_b % per) return false;
  }
  if (!aligned16(a->qb.ptr) || a->qb.stride_r % per || a->qb.stride_l % per || a->qb.stride_b % per) return false;
  if (a->page_table && (a->page_size * (int64_t)a->rk % kRows || a->page_size * (int64_t)a->rk >= (1 << 30))) return false;
  return (int64_t)a->lk * a->rk < (1 << 30);
}

// What the plan reckons with, ns.  In bf16 the columns' waves take kBlockNs for a block at head size 128 and 64 (5.8 and 3.5 us for a tile of four by
// eight waves), or kOwnTileNs for a tile of a sequence's own keys, which memory brings; in fp32 the matrix cores decide (kBlockF32Ns).  Half the
// waves or fewer have the unit to themselves and are faster (kFewWaves).  Data of a first tile arrives at kLandNs for a KiB: what a compute unit
// gets by itself.  A workgroup's way to its first load and behind its last block; a number of a range's results, written and read again;
// a range's turn in the merge; a workgroup that finds no keys.
constexpr double kBlockNs128 = 1450, kBlockNs64 = 875, kOwnTileNs = 3000, kBlockF32Ns = 7000, kFewWaves = .7, kLandNs = 45, kFixedNs = 7500, kPartNs = 8. / 5e3, kMergeNs = 30, kEmptyNs = 3000;
constexpr double kUnits = 256;  // compute units
SharedPlan plan_of(const TpaFwdArgs* a, int prefix) {
  SharedPlan s{};
  s.hb = a->H % 32 == 0 ? 32 : a->H % 24 == 0 ? 24 : a->H % 16 == 0 ? 16 : 8;
  s.nhb = a->H / s.hb;
  s.rows = (int64_t)a->B * a->lq;
  const bool bf16 = a->dtype == TPA_DTYPE_BF16;
  const int in_tile = blocks_of_tile(bf16 ? 2 : 4), tpb = kRows / a->rk, rps = 32 / s.hb;
  auto columns = [&](SharedPart& x, int64_t rows) {
    const int sets = ceil_div(rows, rps);
    x.waves = 1;
    while (x.waves < kWaves && x.waves < sets) x.waves *= 2;
    x.groups = ceil_div(sets, x.waves);
  };
  columns(s.prefix, s.rows);
  columns(s.own, a->lq);
  const int all_p = ceil_div(prefix, tpb), all_s = ceil_div(a->lk - prefix / tpb * tpb, tpb);
  // waves that share the blocks of a range of so many
  auto side = [&](const SharedPart& x, int blocks) {
    int n = std::min(kWaves / x.waves, in_tile);
    while (n / 2 >= blocks) n /= 2;
    return n;
  };
  const double block_ns = bf16 ? (a->dk == 128 ? kBlockNs128 : kBlockNs64) : kBlockF32Ns * a->dk / 128;
  const double land_ns = kLandNs * kRows * 2 * (a->dk + s.hb) * (bf16 ? 2 : 4) / 1024, own_ns = bf16 ? kOwnTileNs * a->dk / 128 : 0.;
  auto each = [&](const SharedPart& x, int blocks) {  // a workgroup of a range of so many blocks, 1, 2 or whole tiles
    const int n = side(x, blocks), first = std::min(blocks, in_tile);
    double tile = block_ns * ((first + n - 1) / n) * (n * x.waves <= kWaves / 2 ? kFewWaves : 1.);
    if (&x == &s.own && blocks >= in_tile) tile = std::max(tile, own_ns);
    return kFixedNs + land_ns * first + tile * ((blocks + in_tile - 1) / in_tile);
  };
  auto longer = [&](int blocks) { return blocks < in_tile ? 2 * blocks : in_tile * std::max(blocks / in_tile + 1, blocks / in_tile * 9 / 8); };
  // One workgroup is resident on a compute unit and the prefix's start first: their rounds of 256, then the own keys' where a round leaves units
  // free and behind them (own lengths differ: on average half of their ranges have no keys).  For every length of the prefix's ranges - 1, 2
  // blocks, whole tiles, from those on that make two rounds - the own keys' that last as long and half as long are tried; the shortest
  // launch wins.
  const double share_p = (double)s.nhb * s.prefix.groups, share_s = (double)s.nhb * s.own.groups;
  double best = 0;
  // ranges of p and o blocks (0: there are none), whose workgroups last each_p and each_s
  auto consider = [&](int p, int o, double each_p, double each_s) {
    const int ranges_p = p ? (all_p + p - 1) / p : 0, ranges_s = o ? (all_s + o - 1) / o : 0;
    // an XCD takes whole ranges: what counts is the one that has most of them, as if all had
    const double groups_p = (ranges_p + 7) / 8 * 8 * share_p, groups_s = std::ceil(ranges_s * (double)a->B / 8) * 8 * share_s;
    const double mean_s = o ? (.5 * (ranges_s + 1) * each_s + .5 * (ranges_s - 1) * kEmptyNs) / ranges_s : 0.;
    const double rounds = std::floor(groups_p / kUnits), last = groups_p - rounds * kUnits;
    const double beside = last && o ? (kUnits - last) * std::max(1., std::floor(each_p / mean_s)) : 0.;
    double cost = rounds * each_p + (last ? std::max(each_p, each_s) : 0.);
    if (groups_s > beside) cost += std::max(std::ceil((groups_s - beside) / kUnits) * mean_s, last ? 0. : each_s);
    cost += (ranges_p + ranges_s) * (kMergeNs + kPartNs * (double)s.rows * a->H * a->dv);
    if (best != 0 && cost >= best) return;
    best = cost;
    s.prefix.blocks = p; s.own.blocks = o; s.prefix.ranges = ranges_p; s.own.ranges = ranges_s;
  };
  int p = prefix > 0, o = prefix < a->lk;
  while (p && p < all_p && ceil_div(all_p, p) * share_p > 2 * kUnits) p = std::min(longer(p), all_p);
  while (o && o < all_s && ceil_div(all_s, o) * share_s * a->B > 4 * kUnits) o = std::min(longer(o), all_s);
  double each_p = p ? each(s.prefix, p) : 0., each_s = o ? each(s.own, o) : 0.;
  for (;;) {
    consider(p, o, each_p, each_s);
    if (o > in_tile) {
      const int half = (o / 2 + in_tile - 1) / in_tile * in_tile;
      consider(p, half, each_p, each(s.own, half));
    }
    const bool more_p = p && p < all_p, more_o = o && o < all_s;
    if (std::max(each_p, each_s) > 2 * best || !(more_p || more_o)) break;
    // the part whose workgroups would still be the shorter ones gets longer ranges
    const int next_p = std::min(longer(p), all_p), next_o = std::min(longer(o), all_s);
    const double then_p = more_p ? each(s.prefix, next_p) : 0., then_s = more_o ? each(s.own, next_o) : 0.;
    if (more_p && (!more_o || then_p <= then_s)) {
      p = next_p;
      each_p = then_p;
    } else {
      o = next_o;
      each_s = then_s;
    }
  }
  s.prefix.side = side(s.prefix, std::max(1, s.prefix.blocks));
  s.own.side = side(s.own, std::max(1, s.own.blocks));
  s.prefix.grid = (int)((s.prefix.ranges + 7) / 8 * 8 * share_p);
  s.own.grid = (int)(ceil_div((int64_t)s.own.ranges * a->B, 8) * 8 * share_s);
  return s;
}
int ranges_of(const SharedPlan& s) { return s.prefix.ranges + s.own.ranges; }
size_t plan_bytes(const SharedPlan& s, int H, int D) { return (size_t)ranges_of(s) * s.rows * H * (D + 2) * sizeof(float); }

template <typename T, int D, int RK, bool PAGED>
int launch_mfma_t(const SharedMfmaParams& p, hipStream_t s) {
  auto kern = shared_mfma_kernel<T, D, RK, PAGED>;
  constexpr size_t bytes = SharedLds<T, D>::kBytes;
  static bool done[kMaxDevices] = {};
  if (const int rc = raise_lds_limit(done, reinterpret_cast<const void*>(kern), bytes); rc != TPA_OK) return rc;
  hipLaunchKernelGGL(kern, dim3(p.plan.prefix.grid + p.plan.own.grid), dim3(kWaves * 64), bytes, s, p);
  if (hipGetLastError() != hipSuccess) return TPA_ERR_LAUNCH;
  const int64_t n = p.plan.rows * p.c.H;
  if (n < kMergeWaves) hipLaunchKernelGGL((shared_merge_kernel<T, D, 4>), dim3(n), dim3(256), 0, s, p);
  else hipLaunchKernelGGL((shared_merge_kernel<T, D, 1>), dim3(ceil_div(n, 4)), dim3(256), 0, s, p);
  return hipGetLastError() == hipSuccess ? TPA_OK : TPA_ERR_LAUNCH;
}
template <typename T, int D, int RK>
int launch_mfma_p(const SharedMfmaParams& p, hipStream_t s) {
  return p.c.page_table ? launch_mfma_t<T, D, RK, true>(p, s) : launch_mfma_t<T, D, RK, false>(p, s);
}
template <typename T, int D>
int launch_mfma(const SharedMfmaParams& p, hipStream_t s) {
  switch (p.c.rk) {
    case 1: return launch_mfma_p<T, D, 1>(p, s);
    case 2: return launch_mfma_p<T, D, 2>(p, s);
    case 4: return launch_mfma_p<T, D, 4>(p, s);
    default: return launch_mfma_p<T, D, 8>(p, s);
  }
}

SharedParams shared_params(const TpaFwdArgs* a, int prefix) {
  SharedParams p{};
  p.qa = a->qa; p.qb = a->qb; p.ka = a->ka; p.kb = a->kb; p.va = a->va; p.vb = a->vb;
  p.o = a->o; p.lse = a->lse; p.kvlen = a->kv_lengths; p.page_table = a->page_table;
  p.page_size = a->page_size; p.pages_per_seq = a->pages_per_seq;
  p.B = a->B; p.lq = a->lq; p.lk = a->lk; p.H = a->H; p.dk = a->dk; p.dv = a->dv; p.rq = a->rq; p.rk = a->rk;
  p.prefix = prefix; p.causal = a->causal; p.coff = causal_offset_of(a);
  p.scale = a->sm_scale * kLog2e;
  return p;
}

// what tpa_decode_shared checks; the outputs are the launch's own matter
int validate(const TpaFwdArgs* a, int prefix) {
  if (!a) return TPA_ERR_NULL;
  TpaFwdArgs b = *a;
  if (!b.o) b.o = &b;  // only its being there is looked at
  if (const int rc = tpa_validate_fwd_args(&b); rc != TPA_OK) return rc;
  if (a->q_segment_ids || a->nomat || a->num_splits) return TPA_ERR_UNSUPPORTED;
  if (prefix < 0 || prefix > a->lk) return TPA_ERR_SHAPE;
  if (a->page_table && (a->page_size <= 0 || a->pages_per_seq <= 0 || (int64_t)a->pages_per_seq * a->page_size < a->lk)) return TPA_ERR_SHAPE;
  if ((int64_t)a->B * a->lq * a->H >= 1 << 24) return TPA_ERR_SHAPE;  // workgroups of 256 threads, 2^32 threads a launch
  return TPA_OK;
}

}  // namespace
}  // namespace tpa

extern "C" size_t tpa_decode_shared_workspace_bytes(const TpaFwdArgs* a, int32_t prefix) {
  using namespace tpa;
  if (validate(a, prefix) != TPA_OK || !mfma_takes(a)) return 0;
  return plan_bytes(plan_of(a, prefix), a->H, a->dv);
}

extern "C" int tpa_decode_shared(const TpaFwdArgs* a, int32_t prefix, void* stream) {
  using namespace tpa;
  if (const int rc = validate(a, prefix); rc != TPA_OK) return rc;
  if (!a->o) return TPA_ERR_NULL;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const SharedParams p = shared_params(a, prefix);
  if (mfma_takes(a)) {
    SharedMfmaParams m{p, plan_of(a, prefix)};
    if (!a->workspace || a->workspace_bytes < plan_bytes(m.plan, a->H, a->dv)) return TPA_ERR_WORKSPACE;
    if (reinterpret_cast<uintptr_t>(a->workspace) & 255) return TPA_ERR_ALIGN;
    const size_t parts = (size_t)ranges_of(m.plan) * m.plan.rows * a->H;
    m.part_o = static_cast<float*>(a->workspace);
    m.part_m = m.part_o + parts * a->dv;
    m.part_l = m.part_m + parts;
    m.qscale = p.scale / ((float)a->rq * a->rk);
    m.page_shift = -1;
    if (a->page_table) {
      const int rows = a->page_size * a->rk;
      if (!(rows & (rows - 1))) m.page_shift = __builtin_ctz(rows);
    }
    if (a->dtype == TPA_DTYPE_BF16) return a->dk == 128 ? launch_mfma<uint16_t, 128>(m, s) : launch_mfma<uint16_t, 64>(m, s);
    return a->dk == 128 ? launch_mfma<float, 128>(m, s) : launch_mfma<float, 64>(m, s);
  }
  if (a->kernel == TPA_KERNEL_MFMA) return TPA_ERR_UNSUPPORTED;
  const dim3 grid((unsigned)(a->B * a->lq * a->H));
  if (a->dtype == TPA_DTYPE_BF16) hipLaunchKernelGGL(shared_any_kernel<uint16_t>, grid, dim3(kAnyThreads), 0, s, p);
  else hipLaunchKernelGGL(shared_any_kernel<float>, grid, dim3(kAnyThreads), 0, s, p);
  return hipGetLastError() == hipSuccess ? TPA_OK : TPA_ERR_LAUNCH;
}
