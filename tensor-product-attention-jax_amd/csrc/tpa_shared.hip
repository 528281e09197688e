// Decode of a batch whose sequences share their first tokens: the shared prefix is read once for all of them.
//
// A query row attends to the keys of the prefix, which are entry 0's, and to the keys behind it, which are its own sequence's; the
// parts are joined by the running maximum and sum of the softmax.
#include <algorithm>

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

// keys that query row `row` of entry b sees
__device__ __forceinline__ int keys_seen(const SharedParams& p, int b, int row) {
  const int len = p.kvlen ? max(0, min(p.kvlen[b], p.lk)) : p.lk;
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
  const int keys = keys_seen(p, b, row);
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

// ---------------------------------------------------------------------------------------------- bf16, matrix cores
// As in the split-key decode nothing is expanded to dense keys or values: with Qm[c, :] = (scale / (Rq R)) sum_i qa_i qb_i of column c = (row,
// head) the logits are s[c, t] = sum_r ka[t, r, h] (Qm[c, :] . kb[t, r, :]), the output (1 / R) sum_t sum_r (p[c, t] va[t, r, h]) vb[t, r, :], two
// products of the rows (t, r) with the columns.  The rows serve every column, so a workgroup takes a tile of 4 blocks of 32 rows
// once for up to 256 columns: the columns of the prefix are those of all sequences, 32 to a wave; where there are fewer (a sequence's
// own keys, few sequences) groups of waves share the tile's blocks and are joined at the end.  Tiles go from memory straight to LDS,
// two buffers, one barrier a tile.
// Qm is kept as two bf16 numbers, 2^-17 of it off: with one the logits carry the rounding of Qm, 2^-9 each, and the output's error
// grows by half; the second costs 8 of 24 matrix instructions a block.  The weights p va are rounded to bf16 once, sums are fp32.
constexpr int kRows = 32;           // rows (token, rank) of a block
constexpr int kBlocks = 4;          // blocks of a tile
constexpr int kWaves = 8;
constexpr int kRsrcFlags = 0x00020000;  // raw 32-bit data format
constexpr int64_t kFarthestRow = 1 << 25;  // elements between neighbouring rows, at most: 31 of them in 32-bit byte offsets

template <int D>
struct SharedLds {
  static constexpr int kB = kRows * D * 2, kA = kRows * 32 * 2;              // bytes of a block's b rows, a rows (32 heads)
  static constexpr int kBuffer = kBlocks * 2 * (kB + kA);                     // kb, vb, ka, va of a tile
  static constexpr int kPart = 32 * D * 4 + 2 * 64 * 4;                       // a wave's sums on their way to another
  static constexpr size_t kBytes = 2 * kBuffer > 4 * kPart ? 2 * kBuffer : 4 * kPart;
};

struct SharedPlan {
  int hb, nhb;             // heads of a block of heads, blocks of heads
  int waves_p, waves_s;    // waves side by side over the columns, of the prefix and of a sequence's own keys
  int groups_p, groups_s;  // groups of as many columns
  int ranges_p, ranges_s;  // key ranges
  int tiles_p, tiles_s;    // tiles of a range
  int grid_p, grid_s;      // workgroups
  int64_t rows;            // B lq
};
struct SharedMfmaParams {
  SharedParams c;
  SharedPlan plan;
  float *part_o, *part_m, *part_l;  // [range][B lq][H][D], [range][B lq][H]: the prefix's ranges, then the own keys'
  float qscale;
  int page_shift;  // log2 of the rows of a page, or -1
};

// Where a lane's pieces of a block of rows of D lie in LDS (elements): 16-byte chunk c of row r at chunk c ^ (r mod chunks)
template <int D>
struct BlockAt {
  static constexpr int CPR = D / 8;
  int row, tr;
  __device__ __forceinline__ explicit BlockAt(int l) {
    const int i = l & 31, g = l >> 5, lp = l & 15, dhalf = (l >> 4) & 1, r = 4 * g + (lp >> 2);
    row = i * D + 8 * (g ^ (i & (CPR - 1)));
    tr = r * D + 8 * ((2 * dhalf + ((lp & 3) >> 1)) ^ r) + 4 * (lp & 1);
  }
  __device__ __forceinline__ int read(int ks) const { return row ^ (16 * ks); }  // row i, chunk 2 ks + g
  // transposed: rows 16 kk + 8 hi + 4 g + 0..3, columns 32 db + 0..31
  __device__ __forceinline__ int read_tr(int kk, int hi, int db) const { return (tr ^ (32 * db) ^ (hi && CPR == 16 ? 64 : 0)) + (16 * kk + 8 * hi) * D; }
};
typedef s16x4 __attribute__((address_space(3))) lds_s16x4;
template <int D>
__device__ __forceinline__ bf16x8 block_tr(const uint16_t* block, const BlockAt<D>& at, int kk, int db) {
  const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(block + at.read_tr(kk, 0, db)));
  const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(block + at.read_tr(kk, 1, db)));
  return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

template <int D, int RK, bool PAGED>
__global__ __launch_bounds__(kWaves * 64, 2) void shared_mfma_kernel(SharedMfmaParams p) {
  using Lds = SharedLds<D>;
  constexpr int NKS = D / 16, NDB = D / 32, CPR = D / 8, RPI = 64 / CPR, NI = 16 / RPI;  // NI: load instructions of a wave for its 16 b rows
  constexpr int TPB = kRows / RK;                                                          // tokens of a block
  constexpr int NTOK = RK <= 4 ? 16 / RK : 32 / RK;  // tokens whose rows this lane holds, per block
  constexpr int NV = RK <= 4 ? RK : RK / 2;          // rows of one token held by this half of the wave
  extern __shared__ __attribute__((aligned(1024))) unsigned char shared_mem[];
  const SharedParams& c = p.c;
  const SharedPlan& plan = p.plan;
  const int tid = threadIdx.x, w = scalar(tid >> 6), l = tid & 63, i = l & 31, g = l >> 5, lp = l & 15, dhalf = (l >> 4) & 1;

  // ---- which keys and columns: workgroups that read the same keys sit on one XCD (ids are dealt to the eight in turn)
  const bool own = (int)blockIdx.x >= plan.grid_p;
  const int id = (int)blockIdx.x - (own ? plan.grid_p : 0);
  const int cwaves = own ? plan.waves_s : plan.waves_p, sharing = plan.nhb * (own ? plan.groups_s : plan.groups_p);
  const int unit = id / (8 * sharing) * 8 + (id & 7), member = id / 8 % sharing;
  if (unit >= (own ? c.B * plan.ranges_s : plan.ranges_p)) return;
  const int b_own = own ? unit / plan.ranges_s : 0, range = own ? unit - b_own * plan.ranges_s : unit;
  const int h0 = member % plan.nhb * plan.hb;
  const int kwaves = min(kWaves / cwaves, kBlocks), cw = w % cwaves, kw = w / cwaves;
  const int col0 = (member / plan.nhb * cwaves + cw) * 32;  // this wave's first column
  const int64_t row_base = own ? (int64_t)b_own * c.lq : 0;
  const int n_cols = (int)(own ? c.lq : plan.rows) * plan.hb;
  const int col = min(col0 + i, n_cols - 1);
  const int64_t row = row_base + col / plan.hb;  // this lane's query row among all, and its head
  const int head = h0 + col % plan.hb;
  const int b = (int)(row / c.lq), row_in_b = (int)(row - (int64_t)b * c.lq);
  const bool works = kw < kwaves && col0 < n_cols;

  // ---- the range's rows (token, rank): first .. end - 1 of those, in blocks from a block's border on
  const int tiles = own ? plan.tiles_s : plan.tiles_p;
  const int origin = own ? c.prefix / TPB * TPB : 0;
  const int seen = keys_seen(c, b, row_in_b);
  const int mine = own ? seen : min(seen, c.prefix);  // keys of this part that this lane's column sees: those below
  const int most = scalar(wave_max(mine)), least = scalar(wave_min(mine));
  int* const red = reinterpret_cast<int*>(shared_mem);
  if (l == 0) red[w] = most;
  __syncthreads();
  int end = 0;
#pragma unroll
  for (int x = 0; x < kWaves; ++x) end = max(end, red[x]);
  __syncthreads();
  end = scalar(end);
  const int begin = origin + range * tiles * kBlocks * TPB;
  const int stop = min(end, begin + tiles * kBlocks * TPB);
  const int64_t slot = ((own ? plan.ranges_p : 0) + range) * plan.rows;
  if (stop <= begin || stop <= (own ? c.prefix : 0)) {  // no key of this range is seen
    if (works && kw == 0 && g == 0 && col0 + i < n_cols) p.part_m[(slot + row) * c.H + head] = -INFINITY;
    return;
  }
  const int n_tiles = (stop - begin + kBlocks * TPB - 1) / (kBlocks * TPB);
  const int row_end = stop * RK;  // rows from here on read as zeros

  // ---- loads: wave w brings rows 16 (w & 1) .. + 15 of block w / 2 of a tile; a lane's chunk is the one that belongs where it lands
  typedef uint32_t Resource __attribute__((ext_vector_type(4)));
  const int64_t boff = PAGED ? 0 : b_own;
  const uint16_t* const base[4] = {static_cast<const uint16_t*>(c.kb.ptr) + boff * c.kb.stride_b, static_cast<const uint16_t*>(c.vb.ptr) + boff * c.vb.stride_b,
                                   static_cast<const uint16_t*>(c.ka.ptr) + boff * c.ka.stride_b + h0, static_cast<const uint16_t*>(c.va.ptr) + boff * c.va.stride_b + h0};
  const int64_t page_stride[4] = {c.kb.stride_b, c.vb.stride_b, c.ka.stride_b, c.va.stride_b};
  const int sr[4] = {2 * (int)c.kb.stride_r, 2 * (int)c.vb.stride_r, 2 * (int)c.ka.stride_r, 2 * (int)c.va.stride_r};
  const int a_chunk = min(l & 3, plan.hb / 8 - 1);
  const int chunk = 16 * ((l % CPR) ^ (l / CPR));
  const int b_row = 16 * (w & 1) + l / CPR, a_row = 16 * (w & 1) + (l >> 2);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)shared_mem;
  const int rpp = PAGED ? c.page_size * RK : 1;
  auto block_row = [&](int tile) __attribute__((always_inline)) { return begin * RK + (tile * kBlocks + (w >> 1)) * kRows; };
  auto page_of = [&](int row0) __attribute__((always_inline)) { return p.page_shift >= 0 ? row0 >> p.page_shift : row0 / rpp; };
  auto lookup = [&](int tile) __attribute__((always_inline)) -> int {
    if constexpr (!PAGED) return 0;
    return c.page_table[(int64_t)b_own * c.pages_per_seq + page_of(min(block_row(tile), row_end - 1) / kRows * kRows)];
  };
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
      const uintptr_t at = reinterpret_cast<uintptr_t>(base[x] + (PAGED ? (int64_t)page * page_stride[x] : 0) + first * (sr[x] / 2));
      const int width = x < 2 ? 2 * D : 2 * plan.hb;
      const Resource rs = {(uint32_t)scalar((int)(uint32_t)at), (uint32_t)scalar((int)((uint32_t)(at >> 32) & 0xffff)), (uint32_t)scalar(rows > 0 ? (rows - 1) * sr[x] + width : 0),
                           (uint32_t)kRsrcFlags};
      if (x < 2) {
#pragma unroll
        for (int n = 0; n < NI; ++n)
          load((uint32_t)scalar(to + x * kBlocks * Lds::kB + (w >> 1) * Lds::kB + (16 * (w & 1) + n * RPI) * 2 * D),
               (b_row + n * RPI - skip) * sr[x] + (chunk ^ (CPR == 16 ? 64 * n : 0)), rs);
      } else {
        load((uint32_t)scalar(to + 2 * kBlocks * Lds::kB + (x - 2) * kBlocks * Lds::kA + (w >> 1) * Lds::kA + 16 * (w & 1) * 64), (a_row - skip) * sr[x] + 16 * a_chunk, rs);
      }
    }
  };
  issue(0, 0, scalar(lookup(0)));
  int page_ahead = lookup(1);

  // ---- Qm of this lane's column, d = 16 ks + 8 g + 0..7, in two parts
  bf16x8 q_hi[NKS], q_lo[NKS];
  {
    const uint16_t* const qa = static_cast<const uint16_t*>(c.qa.ptr) + b * c.qa.stride_b + row_in_b * c.qa.stride_l + head;
    const uint16_t* const qb = static_cast<const uint16_t*>(c.qb.ptr) + b * c.qb.stride_b + row_in_b * c.qb.stride_l + 8 * g;
    float q[NKS][8];
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks)
#pragma unroll
      for (int e = 0; e < 8; ++e) q[ks][e] = 0.f;
    for (int r = 0; r < c.rq; ++r) {
      const float a = bf16bits_to_f32(qa[r * c.qa.stride_r]) * p.qscale;
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks) {
        const u32x4 x = *reinterpret_cast<const u32x4*>(qb + r * c.qb.stride_r + 16 * ks);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          q[ks][2 * e] = fmaf(a, bf16lo_to_f32(x[e]), q[ks][2 * e]);
          q[ks][2 * e + 1] = fmaf(a, bf16hi_to_f32(x[e]), q[ks][2 * e + 1]);
        }
      }
    }
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) {
      u32x4 hi, lo;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        hi[e] = pack_bf16(q[ks][2 * e], q[ks][2 * e + 1]);
        lo[e] = pack_bf16(q[ks][2 * e] - bf16lo_to_f32(hi[e]), q[ks][2 * e + 1] - bf16hi_to_f32(hi[e]));
      }
      q_hi[ks] = __builtin_bit_cast(bf16x8, hi);
      q_lo[ks] = __builtin_bit_cast(bf16x8, lo);
    }
  }

  f32x16 o[NDB];
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int v = 0; v < 16; ++v) o[db][v] = 0.f;
  float m = -INFINITY, lsum = 0.f;
  const BlockAt<D> at(l);
  const int a_head = ((col0 + 16 * dhalf + 4 * (lp & 3)) % plan.hb);  // of the four columns whose a's this lane helps to transpose
  const int row_last = mine * RK - 1, row_first = own ? c.prefix * RK : 0;

  auto compute = [&](int tile, int buffer, int blk) __attribute__((always_inline)) {
    const int row0 = begin * RK + (tile * kBlocks + blk) * kRows;
    if (row0 >= row_end) return;
    const unsigned char* const buf = shared_mem + buffer * Lds::kBuffer;
    const uint16_t* const kb = reinterpret_cast<const uint16_t*>(buf + blk * Lds::kB);
    const uint16_t* const vb = reinterpret_cast<const uint16_t*>(buf + (kBlocks + blk) * Lds::kB);
    const uint16_t* const ka = reinterpret_cast<const uint16_t*>(buf + 2 * kBlocks * Lds::kB + blk * Lds::kA);
    const uint16_t* const va = ka + kBlocks * Lds::kA / 2;
    // S'^T[row, c] = kb[row, :] . Qm[c, :]
    f32x16 sp;
#pragma unroll
    for (int v = 0; v < 16; ++v) sp[v] = 0.f;
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) {
      const bf16x8 kf = *reinterpret_cast<const bf16x8*>(kb + at.read(ks));
      sp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, q_lo[ks], sp, 0, 0, 0);
      sp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, q_hi[ks], sp, 0, 0, 0);
    }
    float ak[16], av[16];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int a_at = (8 * q + 4 * g + (lp >> 2)) * 32 + a_head;
      const s16x4 tk = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(ka + a_at));
      const s16x4 tv = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(va + a_at));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        ak[4 * q + j] = bf16bits_to_f32((uint16_t)tk[j]);
        av[4 * q + j] = bf16bits_to_f32((uint16_t)tv[j]);
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
    if (row0 + kRows > least * RK || row0 < row_first) {
#pragma unroll
      for (int t = 0; t < NTOK; ++t) {
        const int at_row = RK >= 8 ? row0 + RK * t : row0 + 8 * (t * NV >> 2) + 4 * g + (t * NV & 3);  // the token's first row
        if (at_row > row_last || at_row < row_first) st[t] = -INFINITY;
      }
    }
    float tmax = st[0];
#pragma unroll
    for (int t = 1; t < NTOK; ++t) tmax = fmaxf(tmax, st[t]);
    tmax = halves_max(tmax);
    // the reference is a whole number (the running maximum rounded up): the rounding of p va does not depend on how the keys are
    // split, and every rescaling factor is an exact power of two
    const float m_new = fmaxf(m, __builtin_ceilf(tmax));
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
    // O^T[d, c] += sum_row vb[row, d] P'[row, c]; slot (g, j) = row 16 kk + 8 (j / 4) + 4 g + j % 4
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      u32x4 pk;
#pragma unroll
      for (int j = 0; j < 4; ++j) pk[j] = pack_bf16(pp[8 * kk + 2 * j], pp[8 * kk + 2 * j + 1]);
#pragma unroll
      for (int db = 0; db < NDB; ++db)
        o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(block_tr<D>(vb, at, kk, db), __builtin_bit_cast(bf16x8, pk), o[db], 0, 0, 0);
    }
  };

  for (int t = 0; t < n_tiles; ++t) {
    // this wave's part of tile t has landed and nobody reads the other buffer any more; behind the barrier everyone's has
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (t + 1 < n_tiles) {
      issue(t + 1, (t + 1) & 1, scalar(page_ahead));
      page_ahead = lookup(t + 2);
    }
    if (works)
      for (int blk = kw; blk < kBlocks; blk += kwaves) compute(t, t & 1, blk);
  }

  // ---- the groups of waves that shared the blocks are joined, half of them handing their sums to the other half at a time
  lsum = halves_sum(lsum);
  for (int half = kwaves / 2; half; half /= 2) {
    float* const part = reinterpret_cast<float*>(shared_mem + (cw + cwaves * (kw % half)) * Lds::kPart);
    __syncthreads();  // the tiles, or what was handed over before, have been read
    if (works && kw >= half && kw < 2 * half) {
#pragma unroll
      for (int x = 0; x < NDB * 4; ++x)
        *reinterpret_cast<f32x4*>(part + 256 * x + 4 * l) = f32x4{o[x / 4][4 * (x % 4)], o[x / 4][4 * (x % 4) + 1], o[x / 4][4 * (x % 4) + 2], o[x / 4][4 * (x % 4) + 3]};
      part[32 * D + l] = m;
      part[32 * D + 64 + l] = lsum;
    }
    __syncthreads();
    if (works && kw < half) {
      const float m2 = part[32 * D + l], m_new = fmaxf(m, m2), m_use = m_new == -INFINITY ? 0.f : m_new;
      const float f1 = __builtin_amdgcn_exp2f(m - m_use), f2 = __builtin_amdgcn_exp2f(m2 - m_use);
      lsum = lsum * f1 + part[32 * D + 64 + l] * f2;
      m = m_new;
#pragma unroll
      for (int x = 0; x < NDB * 4; ++x) {
        const f32x4 other = *reinterpret_cast<const f32x4*>(part + 256 * x + 4 * l);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[x / 4][4 * (x % 4) + e] = o[x / 4][4 * (x % 4) + e] * f1 + other[e] * f2;
      }
    }
  }
  if (!works || kw || col0 + i >= n_cols) return;
  const int64_t to = (slot + row) * c.H + head;
#pragma unroll
  for (int x = 0; x < NDB * 4; ++x)
    *reinterpret_cast<f32x4*>(p.part_o + to * D + 32 * (x / 4) + 8 * (x % 4) + 4 * g) = f32x4{o[x / 4][4 * (x % 4)], o[x / 4][4 * (x % 4) + 1], o[x / 4][4 * (x % 4) + 2], o[x / 4][4 * (x % 4) + 3]};
  if (g == 0) {
    p.part_m[to] = m;
    p.part_l[to] = lsum;
  }
}

// Joins the ranges' parts of a row and head: a thread per four columns of the output
template <typename T, int D>
__global__ __launch_bounds__(256) void shared_merge_kernel(SharedMfmaParams p) {
  constexpr int TPR = D / 4;
  const SharedParams& c = p.c;
  const int64_t n = p.plan.rows * c.H, at = (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
  if (at >= n) return;
  const int d = 4 * (threadIdx.x % TPR), ranges = p.plan.ranges_p + p.plan.ranges_s;
  float most = -INFINITY;
  for (int x = 0; x < ranges; ++x) most = fmaxf(most, p.part_m[x * n + at]);
  float total = 0.f;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int x = 0; x < ranges; ++x) {
    const float m = p.part_m[x * n + at];
    if (m == -INFINITY) continue;  // nothing else was written
    const float f = __builtin_amdgcn_exp2f(m - most);
    total += f * p.part_l[x * n + at];
    sum += f * *reinterpret_cast<const f32x4*>(p.part_o + (x * n + at) * D + d);
  }
  const bool empty = most == -INFINITY;
  const float inv = empty ? NAN : 1.f / (total * c.rk);
  T* const out = static_cast<T*>(c.o) + at * D + d;
  if constexpr (sizeof(T) == 2) {
    *reinterpret_cast<u32x2*>(out) = u32x2{pack_bf16(sum[0] * inv, sum[1] * inv), pack_bf16(sum[2] * inv, sum[3] * inv)};
  } else {
    *reinterpret_cast<f32x4*>(out) = f32x4{sum[0] * inv, sum[1] * inv, sum[2] * inv, sum[3] * inv};
  }
  if (d == 0 && c.lse) {
    const int64_t row = at / c.H;
    const int h = (int)(at - row * c.H), b = (int)(row / c.lq);
    c.lse[((int64_t)b * c.H + h) * c.lq + (row - (int64_t)b * c.lq)] = empty ? -INFINITY : (most + __log2f(total)) * kLn2;
  }
}

bool aligned16(const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15) == 0; }
int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

bool mfma_takes(const TpaFwdArgs* a) {
  if (a->dtype != TPA_DTYPE_BF16 || a->kernel == TPA_KERNEL_GENERIC) return false;
  if (a->dk != a->dv || (a->dk != 64 && a->dk != 128)) return false;
  if (a->rk != 1 && a->rk != 2 && a->rk != 4 && a->rk != 8) return false;
  if (a->H % 8) return false;
  // rows (token, rank) are uniformly strided and lie where 32-bit offsets reach; 16-byte loads
  const TpaFactor* fs[4] = {&a->ka, &a->kb, &a->va, &a->vb};
  for (const TpaFactor* f : fs) {
    if (f->stride_l != (int64_t)a->rk * f->stride_r || f->stride_r < 0 || f->stride_r > kFarthestRow) return false;
    if (!aligned16(f->ptr) || f->stride_r % 8 || f->stride_b % 8) return false;
  }
  if (!aligned16(a->qb.ptr) || a->qb.stride_r % 8 || a->qb.stride_l % 8 || a->qb.stride_b % 8) return false;
  if (a->page_table && a->page_size * (int64_t)a->rk % kRows) return false;
  return (int64_t)a->lk * a->rk < (1 << 30);
}

SharedPlan plan_of(const TpaFwdArgs* a, int prefix) {
  SharedPlan s{};
  s.hb = a->H % 32 == 0 ? 32 : a->H % 24 == 0 ? 24 : a->H % 16 == 0 ? 16 : 8;
  s.nhb = a->H / s.hb;
  s.rows = (int64_t)a->B * a->lq;
  auto waves = [&](int64_t cols) { int n = 1; while (n < kWaves && 32 * n < cols) n *= 2; return n; };
  s.waves_p = waves(s.rows * s.hb);
  s.waves_s = waves((int64_t)a->lq * s.hb);
  s.groups_p = ceil_div(s.rows * s.hb, 32 * s.waves_p);
  s.groups_s = ceil_div((int64_t)a->lq * s.hb, 32 * s.waves_s);
  const int tpb = kRows / a->rk, tpt = tpb * kBlocks;
  const int all_p = ceil_div(prefix, tpt), all_s = ceil_div(a->lk - prefix / tpb * tpb, tpt);
  const int share_p = s.nhb * s.groups_p, share_s = s.nhb * s.groups_s;
  // as many tiles to a workgroup as give every compute unit one
  const int64_t work = (int64_t)all_p * share_p + (prefix < a->lk ? (int64_t)all_s * share_s * a->B : 0);
  const int each = std::max(1, ceil_div(work, 256));
  if (prefix) {
    s.ranges_p = std::max(1, ceil_div(all_p, each));
    s.tiles_p = ceil_div(all_p, s.ranges_p);
    s.ranges_p = ceil_div(all_p, s.tiles_p);
  }
  if (prefix < a->lk) {
    s.ranges_s = std::max(1, ceil_div(all_s, each));
    s.tiles_s = ceil_div(all_s, s.ranges_s);
    s.ranges_s = ceil_div(all_s, s.tiles_s);
  }
  s.grid_p = ceil_div(s.ranges_p, 8) * 8 * share_p;
  s.grid_s = ceil_div((int64_t)s.ranges_s * a->B, 8) * 8 * share_s;
  return s;
}
size_t plan_bytes(const SharedPlan& s, int H, int D) { return (size_t)(s.ranges_p + s.ranges_s) * s.rows * H * (D + 2) * sizeof(float); }

template <int D, int RK, bool PAGED>
int launch_mfma_t(const SharedMfmaParams& p, hipStream_t s) {
  auto kern = shared_mfma_kernel<D, RK, PAGED>;
  static bool done[kMaxDevices] = {};
  if (const int rc = raise_lds_limit(done, reinterpret_cast<const void*>(kern), SharedLds<D>::kBytes); rc != TPA_OK) return rc;
  hipLaunchKernelGGL(kern, dim3(p.plan.grid_p + p.plan.grid_s), dim3(kWaves * 64), SharedLds<D>::kBytes, s, p);
  if (hipGetLastError() != hipSuccess) return TPA_ERR_LAUNCH;
  hipLaunchKernelGGL((shared_merge_kernel<uint16_t, D>), dim3(ceil_div(p.plan.rows * p.c.H, 256 / (D / 4))), dim3(256), 0, s, p);
  return hipGetLastError() == hipSuccess ? TPA_OK : TPA_ERR_LAUNCH;
}
template <int D, int RK>
int launch_mfma_p(const SharedMfmaParams& p, hipStream_t s) {
  return p.c.page_table ? launch_mfma_t<D, RK, true>(p, s) : launch_mfma_t<D, RK, false>(p, s);
}
template <int D>
int launch_mfma(const SharedMfmaParams& p, hipStream_t s) {
  switch (p.c.rk) {
    case 1: return launch_mfma_p<D, 1>(p, s);
    case 2: return launch_mfma_p<D, 2>(p, s);
    case 4: return launch_mfma_p<D, 4>(p, s);
    default: return launch_mfma_p<D, 8>(p, s);
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
  if ((int64_t)a->B * a->lq * a->H > INT32_MAX) return TPA_ERR_SHAPE;
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
    const size_t parts = (size_t)(m.plan.ranges_p + m.plan.ranges_s) * m.plan.rows * a->H;
    m.part_o = static_cast<float*>(a->workspace);
    m.part_m = m.part_o + parts * a->dv;
    m.part_l = m.part_m + parts;
    m.qscale = p.scale / ((float)a->rq * a->rk);
    m.page_shift = -1;
    if (a->page_table) {
      const int rows = a->page_size * a->rk;
      if (!(rows & (rows - 1))) m.page_shift = __builtin_ctz(rows);
    }
    return a->dk == 128 ? launch_mfma<128>(m, s) : launch_mfma<64>(m, s);
  }
  if (a->kernel == TPA_KERNEL_MFMA) return TPA_ERR_UNSUPPORTED;
  const dim3 grid((unsigned)(a->B * a->lq * a->H));
  if (a->dtype == TPA_DTYPE_BF16) hipLaunchKernelGGL(shared_any_kernel<uint16_t>, grid, dim3(kAnyThreads), 0, s, p);
  else hipLaunchKernelGGL(shared_any_kernel<float>, grid, dim3(kAnyThreads), 0, s, p);
  return hipGetLastError() == hipSuccess ? TPA_OK : TPA_ERR_LAUNCH;
}
