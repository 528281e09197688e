// Decode over the factored KV cache in 4 bits: a few query tokens against a long cache.
//
// As in the decode over 16-bit factors, K and V are never formed: with Qm[c, :] = (scale / (Rq Rk)) sum_i qa[i, h] qb[i, :] for every column c = (query row,
// head) the logits are s[c, t] = sum_j a_k[t, j, h] (Qm[c, :] . b_k[t, j, :]), and o[c, :] = (1/Rk) sum_t sum_j (p[c, t] a_v[t, j, h]) b_v[t, j, :]: two
// products of the matrix cores with the rows of a block of 32 (token, rank) rows and 32 columns.
//
// A lane reads half a row, 32 bytes of codes for 128 numbers.  The product with Q sums over the numbers in any order, so Q takes the order in which they lie in
// that half and the codes go from memory to the matrix cores through the registers: four conversions a word, exact in bf16, the block's scale within them.
// V is contracted over the rows: its numbers go through LDS as bf16 and come back transposed, and so do the head factors of both.
//
// The blocks of all sequences, one behind the other, are dealt to the workgroups in equal shares (of whole rounds of four blocks, one for each wave), whatever
// the lengths are; a workgroup that meets several sequences leaves a part for each, and a second launch joins the parts of a sequence by maximum and sum.
#include <algorithm>

#include "tpa_fp4.h"

namespace tpa {
namespace {

constexpr int kWaves = 4, kThreads = 64 * kWaves;
constexpr int kRows = 32;  // (token, rank) rows of a block
constexpr int kMostGroups = 512;                 // workgroups that share out the rounds: two on a compute unit
constexpr int64_t kNarrow = (1ll << 31) / kMostGroups;  // rounds up to which their shares are quotients of 32 bits (of 64 they take a microsecond)

// x / d and the rest of small numbers (below 2^24), inv = 1 / d rounded: off by one at most, which the rest shows
__device__ __forceinline__ int small_quotient(int x, int d, float inv, int& rest) {
  int q = (int)((float)x * inv);
  rest = x - q * d;
  if (rest < 0) { --q; rest += d; }
  if (rest >= d) { ++q; rest -= d; }
  return q;
}

struct Fp4Params {
  TpaFactor qa, qb, kc, vc;
  void* o;
  float* lse;
  const int32_t *kvlen, *table;
  float *part_o, *part_m, *part_l;  // [slot, column, D], [slot, column], [slot, column]
  int32_t* plan;                    // [B + 1] rounds before each sequence (rounds_of)
  int page_size, page_shift, pages_per_seq, num_pages;
  int B, lq, lk, H, dk, dv, rq, rk, cols;
  int causal, coff;
  int groups;   // workgroups that share out the rounds, at most
  float inv_h;  // 1 / H
  float scale;  // of Q: sm_scale log2(e) / (rq rk); of the vector-unit kernel: sm_scale
};

// keys that query row `row` of a sequence of `length` keys sees
__device__ __forceinline__ int keys_seen(const Fp4Params& p, int length, int row) {
  const int len = max(0, min(length, p.lk));
  if (!p.causal) return len;
  const int64_t last = (int64_t)row + p.coff + 1 + (p.causal == TPA_CAUSAL_BOTTOM_RIGHT ? len - p.lq : 0);
  return (int)max((int64_t)0, min((int64_t)len, last));
}
__device__ __forceinline__ int length_of(const Fp4Params& p, int b) { return p.kvlen ? p.kvlen[b] : p.lk; }
// Rounds of blocks of a sequence, those of the last row, which sees the most, and kStart more that stand for what it costs to begin one: Q's fragments, the first block's
// way, the part.  (Without them workgroups that met two sequences ended last, 101 us after the start where the median was at 88.)
constexpr int kStart = 3;
template <int RK>
__device__ __forceinline__ int rounds_of(const Fp4Params& p, int b) {
  const int n = (int)(((int64_t)keys_seen(p, length_of(p, b), p.lq - 1) * RK + kRows * kWaves - 1) / (kRows * kWaves));
  return n ? n + kStart : 0;
}

template <int CTRL, int ROWS>
__device__ __forceinline__ int add_from(int x) { return x + __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false); }
__device__ __forceinline__ int wave_prefix_sum(int x) {  // lane i: sum of lanes 0 .. i
  x = add_from<0x111, 0xf>(x);  // row_shr 1, 2, 4, 8: inside rows of 16 lanes
  x = add_from<0x112, 0xf>(x);
  x = add_from<0x114, 0xf>(x);
  x = add_from<0x118, 0xf>(x);
  x = add_from<0x142, 0xa>(x);  // row_bcast 15: the last lane of rows 0 and 2 to rows 1 and 3
  return add_from<0x143, 0xc>(x);  // row_bcast 31: lane 31 to rows 2 and 3
}

enum { kRowsApart, kFewHeads, kWholeSets };  // LAYOUT of the kernel

// LDS: the tiles of the waves, the parts of Q that are not held in registers.  (Those that are held are made where the tiles will be.)
template <int D, int QS, int LAYOUT>
struct Fp4Lds {
  static constexpr int kV = kRows * D;                            // elements of V's tile
  static constexpr int kA = kRows * 32;                           // of the head factors of 32 columns
  static constexpr int kPerWave = kV + 2 * kA;                    // bf16 elements
  static constexpr int kHalf = D / 2, kRowStride = kHalf + 4;     // the waves are joined in two halves of D
  static_assert(4 * (32 * kRowStride + 64) <= 2 * kPerWave, "the join takes the room of the tiles");
  static constexpr int kPart = D / 16 * 64;                      // 16-byte words of a part of Q
  static constexpr int kHeld = QS > 2 ? 0 : D == 64 || LAYOUT != kRowsApart ? QS : 1;  // parts in registers: as far as they go there
  static_assert(16 * kHeld * kPart <= 2 * kPerWave * kWaves, "the held parts of Q take the room of the tiles");
  static constexpr size_t kBytes = 2 * (size_t)kPerWave * kWaves + 16 * (size_t)(QS - kHeld) * kPart;
};

// a [32][D] bf16 tile: 16-byte chunk c of row r at chunk c ^ turn(r).  The 16 lanes of a transposed read take two neighbouring chunks of four rows, those of a
// write one chunk of sixteen rows: turn() sends both to places of their own among the 16 of a line of banks (with r mod chunks, under which two
// rows have the same two places, and the head factors' tile as it comes, 202 of a block's 500 LDS cycles were conflicts).
template <int D>
__device__ __forceinline__ int turn(int row) {
  return D == 128 ? (row << 1 | (row >> 3 & 1)) & 15 : (row & 6) | (row >> 3 & 1);
}
template <int D>
__device__ __forceinline__ int tile_write_at(int row, int chunk) { return row * D + 8 * (chunk ^ turn<D>(row)); }
// a [32][32] bf16 tile of head factors: the same with four chunks
__device__ __forceinline__ int a_write_at(int row, int chunk) { return row * 32 + 8 * (chunk ^ (row >> 2 & 3)); }
// transposed read: lane (i, g) gets rows 16 kk + 8 hi + 4 g + 0..3 of column 32 db + i
template <int D>
__device__ __forceinline__ bf16x8 tile_tr(const uint16_t* tile, int l, int kk, int db) {
  const int g = l >> 5, lp = l & 15, dhalf = (l >> 4) & 1;
  auto at = [&](int hi) {
    const int r = 16 * kk + 8 * hi + 4 * g + (lp >> 2);
    return tile_write_at<D>(r, 4 * db + 2 * dhalf + ((lp & 3) >> 1)) + 4 * (lp & 1);
  };
  const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4 __attribute__((address_space(3)))*)(tile + at(0)));
  const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4 __attribute__((address_space(3)))*)(tile + at(1)));
  return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

// x as a sum of NS bf16 numbers (3: all 24 bits), two at a time
template <int NS>
__device__ __forceinline__ void split_pair(float x, float y, uint32_t (&out)[NS]) {
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    out[s] = pack_bf16(x, y);
    x -= bf16lo_to_f32(out[s]);
    y -= bf16hi_to_f32(out[s]);
  }
}

// eight numbers from a place that need not be aligned
struct Eight {
  typedef f32x4 __attribute__((aligned(4))) Raw;
  f32x4 w[2];
  __device__ __forceinline__ void load(const float* p) {
    w[0] = *reinterpret_cast<const Raw*>(p);
    w[1] = *reinterpret_cast<const Raw*>(p + 4);
  }
  __device__ __forceinline__ float get(int j) const { return w[j >> 2][j & 3]; }
};

// T: of the queries and the output.  QS, PS: bf16 numbers that stand for one of Q and of the weights p a_v: two for bf16 queries (with one, logits were off by up to 6e-3,
// and outputs by half as much again as their own rounding, up to 0.0026 of their norm where that is 0.0016; the second number of a weight makes
// 101 us of 94 for 128 sequences of 12 000 keys, in calls one behind the other, which the power limit slows down, 113 of 101), three for fp32.
// LAYOUT: kRowsApart: every lane finds its row by itself and loads 8 heads and a scale at a time.
// The others take blocks whose 32 rows lie one behind the other, all of them in memory (pages of whole blocks): a block has one address, a lane's place in it
// never changes, and the ends of K's rows come in one half of the wave, those of V's in the other.
// All columns have their head factors in one block of 32, so its scale goes into those of K's and V's numbers, and the codes themselves are transposed, to fp32 right from
// there (with scales of their own in the tile, as kRowsApart has them, 43.7 us for 41 with 64 heads of 64).
// kFewHeads: 8 or 16 heads.  kWholeSets: 32 or 64 heads, or 96 or 128 of 128 numbers, whose scales are all in the last words of a row.
// A workgroup has 32 columns.  (With two sets of them a block is unpacked once for 64, but one wave fits a SIMD with 128 numbers and no more with 64: from 46.8 us
// for one set's 45 with 64 heads of 64 to 98 for 56 with 64 heads of 128.)
// What bounds the kernel is the issue of instructions, vector and matrix ones half and half, by two waves a SIMD (three, of 168 registers, gain nothing):
//   128 sequences of 12 000 keys, 32 heads of 128, rank 2: 96 us, kRowsApart 115; 64 of 8192: 39, kRowsApart 46
//   12 sequences of 4500 keys, 4 query rows, 64 heads of 64, rank 4: 41, kRowsApart 50; 48 of 8192, one row, 64 heads of 128, rank 2: 51, kRowsApart 62
// (24 heads with one address a block and all else as for kRowsApart: 41.9 against 42.6, which is not worth a variant.)
// Where there are few blocks, what is done once counts: 8 us with a block for every wave, 0.8 of them to find the share, 1.5 until the block is asked for,
// 1.1 for Q, 2.1 for the block and 1.8 to join the waves.
template <typename T, int D, int RK, int QS, int PS, int LAYOUT>
__global__ __launch_bounds__(kThreads, 2) void decode_fp4_kernel(Fp4Params p) {
  using Lds = Fp4Lds<D, QS, LAYOUT>;
  constexpr int NKS = D / 16, NDB = D / 32, NW = D / 64;  // NW: 16-byte words of half a row's codes
  constexpr int NTOK = RK <= 4 ? 16 / RK : 32 / RK;       // tokens whose rows this lane has logits of
  constexpr int NV = RK <= 4 ? RK : RK / 2;               // rows of a token in this half of the wave
  extern __shared__ __attribute__((aligned(16))) uint16_t smem_fp4[];
  const int tid = threadIdx.x, w = scalar(tid >> 6), l = tid & 63, i = l & 31, g = l >> 5;
  const int c0 = blockIdx.y * 32;

  // ---- this workgroup's share of the rounds, which every wave finds for itself: a lane has neighbouring sequences
  const int each = (p.B + 63) / 64, e0 = min(l * each, p.B), e1 = min(e0 + each, p.B);
  int mine = 0;
  for (int b = e0; b < e1; ++b) mine += rounds_of<RK>(p, b);
  const int upto = wave_prefix_sum(mine), total = __builtin_amdgcn_readlane(upto, 63);
  const int groups = min(p.groups, total);
  const int64_t share = blockIdx.x;
  if (blockIdx.x == 0 && blockIdx.y == 0 && w == 0) {
    int before = upto - mine;
    for (int b = e0; b < e1; ++b) {
      p.plan[b] = before;
      before += rounds_of<RK>(p, b);
    }
    if (l == 0) p.plan[p.B] = total;
  }
  if (share >= groups) return;
  int r0, r1;
  if (total < kNarrow) {
    r0 = (int)((uint32_t)share * (uint32_t)total / (uint32_t)groups);
    r1 = (int)(((uint32_t)share + 1) * (uint32_t)total / (uint32_t)groups);
  } else {
    r0 = (int)(share * total / groups);
    r1 = (int)((share + 1) * total / groups);
  }
  int b = e0, first_round = upto - mine;
  if (r0 >= first_round && r0 < upto)
    for (int n; r0 >= first_round + (n = rounds_of<RK>(p, b)); ++b) first_round += n;
  const int there = __builtin_ctzll(__ballot(r0 >= upto - mine && r0 < upto));
  b = __builtin_amdgcn_readlane(b, there);
  first_round = __builtin_amdgcn_readlane(first_round, there);

  uint16_t* const lds_v = smem_fp4 + w * Lds::kPerWave;
  uint16_t* const lds_a = lds_v + Lds::kV;  // [K, V][32 rows][32 columns]
  u32x4* const lds_q = reinterpret_cast<u32x4*>(smem_fp4);  // parts in registers later
  u32x4* const lds_q_rest = reinterpret_cast<u32x4*>(smem_fp4 + kWaves * Lds::kPerWave);
  constexpr int kHeld = Lds::kHeld;

  const Fp4Row parts(p.H, D);
  // where the head factors of this lane's columns lie in a row: two chunks of 8
  int a_at[2], a_scale_at[2];  // (kWholeSets: 32 heads from a_at[0] on, their scale's place among the scales of a in a_scale_at[0])
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    int h;
    small_quotient(c0 + 16 * g + 8 * q, p.H, p.inv_h, h);
    a_at[q] = parts.a_codes + h / 2;
    a_scale_at[q] = parts.a_scales + h / 32;
    if constexpr (LAYOUT == kWholeSets) {
      a_at[q] -= 8 * g;
      a_scale_at[q] = h / 32;
    }
  }
  // this lane's row of a block: always the same rank
  const uint8_t* const k_base = static_cast<const uint8_t*>(p.kc.ptr) + (i % RK) * p.kc.stride_r;
  const uint8_t* const v_base = static_cast<const uint8_t*>(p.vc.ptr) + (i % RK) * p.vc.stride_r;
  int head;
  const int row_of_col = small_quotient(min(c0 + i, p.cols - 1), p.H, p.inv_h, head);  // query row of this lane's column (past the last: the last)

  while (r0 < r1) {
    const int rounds = rounds_of<RK>(p, b);
    if (r0 >= first_round + rounds) {  // (a sequence without keys, or one whose end is a share's)
      first_round += rounds;
      ++b;
      continue;
    }
    const int stop = min(r1, first_round + rounds), begin = max(r0 - first_round - kStart, 0), end = stop - first_round - kStart;
    r0 = stop;
    if (end <= begin) continue;  // nothing but a share of its start
    const int len = length_of(p, b);
    const int last_of = keys_seen(p, len, row_of_col) * RK - 1, least_last = scalar(last_of);  // (the first column's row sees the fewest keys)
    const int last_row = keys_seen(p, len, p.lq - 1) * RK - 1;  // not below 0 here
    const int blk_begin = begin * kWaves + w, blk_end = min(end * kWaves, last_row / kRows + 1);

    // ---- loads of a block; its page is looked up a block ahead
    typedef u32x4 __attribute__((aligned(4))) Word;
    typedef u32x2 __attribute__((aligned(4))) Pair;
    struct Raw {
      u32x4 k[NW], v[NW];
      uint32_t k_scales, v_scales;           // not kRowsApart: of b and of a, k_scales and v_scales the first and second word of K's row (g = 0) or V's
      uint32_t ka[2], va[2];                 // kRowsApart: 8 heads of K and of V twice; kFewHeads: ka the heads of K's row (g = 0) or V's
      uint8_t ka_scale[2], va_scale[2];      // (kRowsApart)
      u32x4 a;                               // kWholeSets: the 32 heads of K's row (g = 0) or V's, whose scale words are as for kFewHeads
    } raw;
    // this lane's half of K's row and of V's, and their ends
    auto take = [&](const uint8_t* k, const uint8_t* v) __attribute__((always_inline)) {
#pragma unroll
      for (int n = 0; n < NW; ++n) {
        raw.k[n] = *reinterpret_cast<const Word*>(k + g * (D / 4) + 16 * n);
        raw.v[n] = *reinterpret_cast<const Word*>(v + g * (D / 4) + 16 * n);
      }
      raw.k_scales = *reinterpret_cast<const uint32_t*>(k + parts.b_scales);
      raw.v_scales = *reinterpret_cast<const uint32_t*>(v + parts.b_scales);
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        raw.ka[q] = *reinterpret_cast<const uint32_t*>(k + a_at[q]);
        raw.va[q] = *reinterpret_cast<const uint32_t*>(v + a_at[q]);
        raw.ka_scale[q] = k[a_scale_at[q]];
        raw.va_scale[q] = v[a_scale_at[q]];
      }
    };
    // the same with the whole end of K's row in one half of the wave and of V's in the other (8 heads: what is read behind
    // them is not used)
    auto take_ends = [&](const uint8_t* k, const uint8_t* v, uint32_t at_k, uint32_t at_v) __attribute__((always_inline)) {
#pragma unroll
      for (int n = 0; n < NW; ++n) {
        raw.k[n] = *reinterpret_cast<const Word*>(k + (at_k + g * (D / 4)) + 16 * n);
        raw.v[n] = *reinterpret_cast<const Word*>(v + (at_v + g * (D / 4)) + 16 * n);
      }
      const uint8_t* const mine = g ? v + at_v : k + at_k;
      if constexpr (LAYOUT == kWholeSets) {
        raw.a = *reinterpret_cast<const Word*>(mine + a_at[0]);
      } else {
        const u32x2 codes = *reinterpret_cast<const Pair*>(mine + parts.a_codes);
        raw.ka[0] = codes[0]; raw.ka[1] = codes[1];
      }
      if constexpr (D == 128) {
        const u32x2 x = *reinterpret_cast<const Pair*>(mine + parts.b_scales);
        raw.k_scales = x[0];
        raw.v_scales = x[1];
      } else {
        raw.k_scales = *reinterpret_cast<const uint32_t*>(mine + parts.b_scales);
      }
    };
    auto page_of = [&](int token) __attribute__((always_inline)) { return p.page_shift >= 0 ? token >> p.page_shift : token / p.page_size; };
    const int last_token = last_row / RK;
    auto token_of = [&](int blk) __attribute__((always_inline)) {  // the block's first, or this lane's (of a row past the last: the last)
      return LAYOUT != kRowsApart ? min(blk, last_row / kRows) * (kRows / RK) : min(blk * (kRows / RK) + i / RK, last_token);
    };
    auto lookup = [&](int blk) __attribute__((always_inline)) { return p.table ? p.table[(int64_t)b * p.pages_per_seq + page_of(token_of(blk))] : b; };
    int page_ahead = lookup(blk_begin);
    auto issue = [&](int blk) __attribute__((always_inline)) {
      const int token = token_of(blk);
      int page = p.table ? max(0, min(page_ahead, p.num_pages - 1)) : b;
      const int in_page = p.table ? token - page_of(token) * p.page_size : token;
      if constexpr (LAYOUT != kRowsApart) {
        page = scalar(page);
        const int64_t k = page * p.kc.stride_b + in_page * p.kc.stride_l, v = page * p.vc.stride_b + in_page * p.vc.stride_l;
        const uint8_t *const k_block = static_cast<const uint8_t*>(p.kc.ptr) + k, *const v_block = static_cast<const uint8_t*>(p.vc.ptr) + v;
        take_ends(k_block, v_block, i * (uint32_t)p.kc.stride_r, i * (uint32_t)p.vc.stride_r);
      } else {
        take(k_base + page * p.kc.stride_b + in_page * p.kc.stride_l, v_base + page * p.vc.stride_b + in_page * p.vc.stride_l);
      }
      page_ahead = lookup(blk + kWaves);
    };
    issue(blk_begin);

    // ---- Q's fragments: lane (column, g) of step ks holds numbers g D/2 + 8 ks + 0..7
    __syncthreads();  // the sequence before has left LDS
    auto part_q = [&](int q) __attribute__((always_inline)) { return q < kHeld ? lds_q + q * Lds::kPart : lds_q_rest + (q - kHeld) * Lds::kPart; };
    auto place_q = [&](int col, int d) __attribute__((always_inline)) {  // of number d of a column in a part of Q
      const int half = d / (D / 2), ks = d % (D / 2) / 8;
      return ks * 64 + 32 * half + col;
    };
    if constexpr (sizeof(T) == 2) {
      // by the matrix cores, 32 numbers of 32 columns a wave: rows d, columns c, contraction over the ranks, whose loads are all on their way at once.
      // (On the vector units, eight numbers a thread, the loads waited for four times: 6100 of the 18 800 cycles of the shortest call.)
      for (int db = w; db < NDB; db += kWaves) {
        const uint16_t* const qa = static_cast<const uint16_t*>(p.qa.ptr) + b * p.qa.stride_b + row_of_col * p.qa.stride_l + head;
        // (the columns may be of several query rows: their b rows differ, so a product for each of these rows, of which a column takes its own)
        const int first_row = __builtin_amdgcn_readlane(row_of_col, 0), last = __builtin_amdgcn_readlane(row_of_col, 31);
        f32x16 x;
        for (int row = first_row; row <= last; ++row) {
          const uint16_t* const qb = static_cast<const uint16_t*>(p.qb.ptr) + b * p.qb.stride_b + row * p.qb.stride_l + 32 * db + i;
          f32x16 acc;
#pragma unroll
          for (int v = 0; v < 16; ++v) acc[v] = 0.f;
          for (int r0 = 0; r0 < p.rq; r0 += 16) {
            uint16_t av[8], bv[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const int r = min(r0 + 8 * g + j, p.rq - 1);
              av[j] = qa[r * p.qa.stride_r];
              bv[j] = qb[r * p.qb.stride_r];
            }
            u32x4 aw, bw;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int r = r0 + 8 * g + 2 * j;  // ranks past the last count as zero in both
              aw[j] = (r < p.rq ? (uint32_t)av[2 * j] : 0u) | (r + 1 < p.rq ? (uint32_t)av[2 * j + 1] << 16 : 0u);
              bw[j] = (r < p.rq ? (uint32_t)bv[2 * j] : 0u) | (r + 1 < p.rq ? (uint32_t)bv[2 * j + 1] << 16 : 0u);
            }
            acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, bw), __builtin_bit_cast(bf16x8, aw), acc, 0, 0, 0);
          }
#pragma unroll
          for (int v = 0; v < 16; ++v) x[v] = row == first_row || row == row_of_col ? acc[v] : x[v];
        }
#pragma unroll
        for (int n = 0; n < 4; ++n) {  // numbers 32 db + 8 n + 4 g + 0..3
          uint32_t lo[QS], hi[QS];
          split_pair<QS>(x[4 * n] * p.scale, x[4 * n + 1] * p.scale, lo);
          split_pair<QS>(x[4 * n + 2] * p.scale, x[4 * n + 3] * p.scale, hi);
#pragma unroll
          for (int q = 0; q < QS; ++q)
            reinterpret_cast<u32x2*>(part_q(q))[2 * place_q(i, 32 * db + 8 * n) + g] = u32x2{lo[q], hi[q]};
        }
      }
    } else {
      for (int item = tid; item < 32 * (D / 8); item += kThreads) {
        const int col = item / (D / 8), chunk = item % (D / 8);
        int h;
        const int qi = small_quotient(min(c0 + col, p.cols - 1), p.H, p.inv_h, h);
        const T* const qa = static_cast<const T*>(p.qa.ptr) + b * p.qa.stride_b + qi * p.qa.stride_l + h;
        const T* const qb = static_cast<const T*>(p.qb.ptr) + b * p.qb.stride_b + qi * p.qb.stride_l + 8 * chunk;
        float x[8] = {};
        for (int r0 = 0; r0 < p.rq; r0 += 6) {  // six ranks asked for together, those past the last again the last, which counts once
          float a[6];
          Eight row[6];
#pragma unroll
          for (int u = 0; u < 6; ++u) {
            const int r = min(r0 + u, p.rq - 1);
            a[u] = qa[r * p.qa.stride_r];
            row[u].load(qb + r * p.qb.stride_r);
          }
#pragma unroll
          for (int u = 0; u < 6; ++u)
            if (r0 + u < p.rq) {
#pragma unroll
              for (int j = 0; j < 8; ++j) x[j] = fmaf(a[u], row[u].get(j), x[j]);
            }
        }
        uint32_t words[4][QS];
#pragma unroll
        for (int j = 0; j < 4; ++j) split_pair<QS>(x[2 * j] * p.scale, x[2 * j + 1] * p.scale, words[j]);
#pragma unroll
        for (int q = 0; q < QS; ++q) part_q(q)[place_q(col, 8 * chunk)] = u32x4{words[0][q], words[1][q], words[2][q], words[3][q]};
      }
    }
    __syncthreads();
    bf16x8 qf[kHeld ? kHeld * NKS : 1];
    if constexpr (kHeld > 0) {
#pragma unroll
      for (int n = 0; n < kHeld * NKS; ++n) qf[n] = __builtin_bit_cast(bf16x8, lds_q[n * 64 + l]);
      __syncthreads();  // the tiles take their place
    }

    f32x16 o[NDB];
    float m = -INFINITY, sum = 0.f;
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int v = 0; v < 16; ++v) o[db][v] = 0.f;

    // products of the rows of K with Q; numbers of V and of the head factors to LDS
    auto unpack = [&](int blk, f32x16& sp) __attribute__((always_inline)) {
      uint32_t k_scales = raw.k_scales, v_scales = raw.v_scales;
      float ka_scale = 1.f, va_scale = 1.f;
      if constexpr (LAYOUT != kRowsApart) {
        const auto first = __builtin_amdgcn_permlane32_swap(raw.k_scales, raw.k_scales, false, false);
        k_scales = first[0];
        v_scales = first[1];
      }
      if constexpr (LAYOUT == kFewHeads && D == 128) {
        const auto second = __builtin_amdgcn_permlane32_swap(raw.v_scales, raw.v_scales, false, false);
        ka_scale = fp4_scale(second[0] & 255);
        va_scale = fp4_scale(second[1] & 255);
      } else if constexpr (LAYOUT == kFewHeads) {
        ka_scale = fp4_scale(k_scales >> 16 & 255);
        va_scale = fp4_scale(v_scales >> 16 & 255);
      } else if constexpr (LAYOUT == kWholeSets) {
        const uint32_t of_half = (D == 128 ? raw.v_scales : raw.k_scales >> 16) >> 8 * a_scale_at[0] & 255;
        const auto both = __builtin_amdgcn_permlane32_swap(of_half, of_half, false, false);
        ka_scale = fp4_scale(both[0]);
        va_scale = fp4_scale(both[1]);
      }
      if (LAYOUT != kRowsApart && blk * kRows + kRows - 1 > last_row && blk * kRows + i > last_row) {
        // behind the last token: whatever is there, numbers that a weight of 0 leaves at 0
        v_scales = 0;
        va_scale = 1.f;
      }
      float scale[2][NW];
#pragma unroll
      for (int n = 0; n < NW; ++n) {
        const int shift = 8 * (NW * g + n);
        scale[0][n] = fp4_scale((k_scales >> shift) & 255);
        scale[1][n] = fp4_scale((v_scales >> shift) & 255);
        if constexpr (LAYOUT != kRowsApart) {  // (a product past 2^127 is infinity, which the conversions make NaN of; one below 2^-127 counts as that)
          scale[0][n] *= ka_scale;
          scale[1][n] *= va_scale;
        }
      }
#pragma unroll
      for (int v = 0; v < 16; ++v) sp[v] = 0.f;
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks) {
        const bf16x8 kf = fp4_bf16x8(raw.k[ks / 4][ks % 4], scale[0][ks / 4]);
#pragma unroll
        for (int q = 0; q < QS; ++q) {
          const bf16x8 qv = q < kHeld ? qf[q < kHeld ? q * NKS + ks : 0] : __builtin_bit_cast(bf16x8, part_q(q)[ks * 64 + l]);
          sp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qv, sp, 0, 0, 0);
        }
        *reinterpret_cast<bf16x8*>(lds_v + tile_write_at<D>(i, NKS * g + ks)) = fp4_bf16x8(raw.v[ks / 4][ks % 4], scale[1][ks / 4]);
      }
      if constexpr (LAYOUT == kFewHeads) {
        const uint32_t odd = p.H == 8 ? raw.ka[0] : raw.ka[1];
        reinterpret_cast<u32x4*>(lds_a)[l] = u32x4{raw.ka[0], odd, raw.ka[0], odd};  // [K, V][32 rows][32 codes]
      } else if constexpr (LAYOUT == kWholeSets) {
        reinterpret_cast<u32x4*>(lds_a)[l] = raw.a;
      } else {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          uint16_t* const at = lds_a + a_write_at(i, 2 * g + q);
          *reinterpret_cast<bf16x8*>(at) = fp4_bf16x8(raw.ka[q], fp4_scale(raw.ka_scale[q]));
          *reinterpret_cast<bf16x8*>(at + Lds::kA) = fp4_bf16x8(raw.va[q], fp4_scale(raw.va_scale[q]));
        }
      }
    };
    auto consume = [&](int blk, const f32x16& sp) __attribute__((always_inline)) {
      const int lp = l & 15, dhalf = (l >> 4) & 1, row0 = blk * kRows;
      float ak[16], av[16];  // of this lane's column, rows 8q + 4g + 0..3
      if constexpr (LAYOUT != kRowsApart) {
        // lane lp of 16 names row 8 (lp / 4) + 4 g + lp % 4, and gets its own column's codes of the sixteen rows
        typedef int s32x2 __attribute__((ext_vector_type(2)));
        const int at = 8 * (2 * (8 * (lp >> 2) + 4 * g + (lp & 3)) + dhalf);
        const s32x2 tk = __builtin_amdgcn_ds_read_tr4_b64_v2i32((s32x2 __attribute__((address_space(3)))*)(reinterpret_cast<uint8_t*>(lds_a) + at));
        const s32x2 tv = __builtin_amdgcn_ds_read_tr4_b64_v2i32((s32x2 __attribute__((address_space(3)))*)(reinterpret_cast<uint8_t*>(lds_a) + 512 + at));
        float x[8];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          fp4_f32x8((uint32_t)tk[n], 1.f, x);
#pragma unroll
          for (int j = 0; j < 8; ++j) ak[8 * n + j] = x[j];
          fp4_f32x8((uint32_t)tv[n], 1.f, x);
#pragma unroll
          for (int j = 0; j < 8; ++j) av[8 * n + j] = x[j];
        }
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int at = a_write_at(8 * q + 4 * g + (lp >> 2), 2 * dhalf + ((lp & 3) >> 1)) + 4 * (lp & 1);
          const s16x4 tk = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4 __attribute__((address_space(3)))*)(lds_a + at));
          const s16x4 tv = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4 __attribute__((address_space(3)))*)(lds_a + Lds::kA + at));
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            ak[4 * q + j] = bf16bits_to_f32((uint16_t)tk[j]);
            av[4 * q + j] = bf16bits_to_f32((uint16_t)tv[j]);
          }
        }
      }
      // ---- logits per token (log2 domain); from rank 8 on a token's rows span both halves of the wave
      float st[NTOK], most = -INFINITY;
#pragma unroll
      for (int t = 0; t < NTOK; ++t) {
        const int v0 = t * NV;
        float acc = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) acc = fmaf(ak[v0 + j], sp[v0 + j], acc);
        if constexpr (RK >= 8) acc = halves_sum(acc);
        st[t] = acc;
      }
      if (row0 + kRows - 1 > least_last) {  // (the same in all lanes)
        asm volatile("");                      // a branch: it is taken for the last keys alone
#pragma unroll
        for (int t = 0; t < NTOK; ++t) {
          const int v0 = t * NV, row = RK >= 8 ? row0 + RK * t : row0 + 8 * (v0 >> 2) + 4 * g + (v0 & 3);  // the token's first row
          if (row > last_of) st[t] = -INFINITY;
        }
      }
#pragma unroll
      for (int t = 0; t < NTOK; ++t) most = fmaxf(most, st[t]);
      most = halves_max(most);
      // the reference is a whole number: a weight then has the same significand, and is rounded the same way, however the keys are dealt to
      // waves and workgroups, and every factor that joins them is a power of two
      const float m_new = fmaxf(m, __builtin_ceilf(most)), m_use = m_new == -INFINITY ? 0.f : m_new;
      if (__any(m_new > m)) {
        const float alpha = __builtin_amdgcn_exp2f(m - m_use);
        sum *= alpha;
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
        sum += RK >= 8 ? 0.5f * pt : pt;  // both halves hold the token: each adds half of it
#pragma unroll
        for (int j = 0; j < NV; ++j) pp[t * NV + j] = pt * av[t * NV + j];
      }
      // ---- O^T[d, column] += sum over the rows of V[row, d] P'[row, column]; slot (g, j) = row 16 kk + 8 (j / 4) + 4 g + j % 4
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        uint32_t words[4][PS];
#pragma unroll
        for (int j = 0; j < 4; ++j) split_pair<PS>(pp[8 * kk + 2 * j], pp[8 * kk + 2 * j + 1], words[j]);
#pragma unroll
        for (int db = 0; db < NDB; ++db) {
          const bf16x8 vf = tile_tr<D>(lds_v, l, kk, db);
#pragma unroll
          for (int q = 0; q < PS; ++q)
            o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, __builtin_bit_cast(bf16x8, u32x4{words[0][q], words[1][q], words[2][q], words[3][q]}), o[db], 0, 0, 0);
        }
      }
    };
    // The two waves of a SIMD come first block by block in turn: the older one, always first, ended its share at 25 us where the younger one took 42, half of it
    // alone (12 sequences of 4500 keys, 4 query rows, 64 heads of 64; the kernel 1 to 3 us shorter)
    int first = (blockIdx.x + blockIdx.y * gridDim.x) / (kMostGroups / 2);
    for (int blk = blk_begin; blk < blk_end; blk += kWaves) {
      if (first++ & 1) __builtin_amdgcn_s_setprio(1);
      else __builtin_amdgcn_s_setprio(0);
      f32x16 sp;
      unpack(blk, sp);
      issue(blk + kWaves);
      consume(blk, sp);
    }

    // ---- join the waves through LDS, half of D at a time, and leave the part
    const int64_t slot = (int64_t)share + b;
    float* const red_o = reinterpret_cast<float*>(lds_v);
    constexpr int RS = Lds::kRowStride, HB = NDB / 2;
    const int n_cols = min(32, p.cols - c0);
    const float all = halves_sum(sum);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      __syncthreads();
#pragma unroll
      for (int db = 0; db < HB; ++db)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const f32x16& x = o[half * HB + db];
          *reinterpret_cast<f32x4*>(red_o + i * RS + 32 * db + 8 * q + 4 * g) = f32x4{x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]};
        }
      if (g == 0) {
        red_o[32 * RS + i] = m;
        red_o[32 * RS + 32 + i] = all;
      }
      __syncthreads();
      const int64_t base = slot * p.cols + c0;
      for (int idx = tid; idx < n_cols * (D / 8); idx += kThreads) {
        const int c = idx / (D / 8), d = 4 * (idx % (D / 8));
        float mw[kWaves], lw[kWaves], most = -INFINITY;
#pragma unroll
        for (int ww = 0; ww < kWaves; ++ww) {
          const float* const from = reinterpret_cast<const float*>(smem_fp4 + ww * Lds::kPerWave);
          mw[ww] = from[32 * RS + c];
          lw[ww] = from[32 * RS + 32 + c];
          most = fmaxf(most, mw[ww]);
        }
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
        float lacc = 0.f;
#pragma unroll
        for (int ww = 0; ww < kWaves; ++ww) {
          const float* const from = reinterpret_cast<const float*>(smem_fp4 + ww * Lds::kPerWave);
          const float f = lw[ww] == 0.f ? 0.f : __builtin_amdgcn_exp2f(mw[ww] - most);  // 0: no key of this wave
          acc += f * *reinterpret_cast<const f32x4*>(from + c * RS + d);
          lacc += f * lw[ww];
        }
        *reinterpret_cast<f32x4*>(p.part_o + (base + c) * D + half * (D / 2) + d) = acc;
        if (half == 0 && d == 0) {
          p.part_m[base + c] = most;
          p.part_l[base + c] = lacc;
        }
      }
    }
  }
}

// The parts of a sequence's columns joined: D / 4 threads have a column, or SLICES times as many, which share out its parts where there are many (128 sequences of 12 000
// keys, five parts each: 7.5 us in eight slices).
template <typename T, int D, int SLICES>
__global__ __launch_bounds__(kThreads) void join_kernel(Fp4Params p) {
  constexpr int LANES = D / 4, COLS = kThreads / LANES / SLICES;
  __shared__ f32x4 part[SLICES > 1 ? kThreads : 1];
  __shared__ float part_m[SLICES > 1 ? COLS * SLICES : 1], part_l[SLICES > 1 ? COLS * SLICES : 1];
  const int at = threadIdx.x % LANES, slice = threadIdx.x / LANES % SLICES, mine = threadIdx.x / LANES / SLICES;
  const int64_t column = (int64_t)blockIdx.x * COLS + mine, last = (int64_t)p.B * p.cols - 1;
  const int b = (int)(min(column, last) / p.cols), c = (int)(min(column, last) - (int64_t)b * p.cols);
  const int64_t total = p.plan[p.B], first = p.plan[b] + kStart, rounds = p.plan[b + 1] - first, groups = min((int64_t)p.groups, total);
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, sum = 0.f;
  if (rounds > 0) {
    int from, to;
    if (total < kNarrow) {
      from = (int)((((uint32_t)first + 1) * (uint32_t)groups - 1) / (uint32_t)total);
      to = (int)((((uint32_t)first + (uint32_t)rounds) * (uint32_t)groups - 1) / (uint32_t)total);
    } else {
      from = (int)(((first + 1) * groups - 1) / total);
      to = (int)(((first + rounds) * groups - 1) / total);
    }
    constexpr int kTogether = 4;
    for (int share = from + slice; share <= to; share += kTogether * SLICES) {
      float ms[kTogether], ls[kTogether];
      f32x4 os[kTogether];
#pragma unroll
      for (int u = 0; u < kTogether; ++u) {
        const int64_t base = (int64_t)(min(share + u * SLICES, to) + b) * p.cols + c;
        ms[u] = p.part_m[base];
        ls[u] = share + u * SLICES <= to ? p.part_l[base] : 0.f;
        os[u] = *reinterpret_cast<const f32x4*>(p.part_o + base * D + 4 * at);
      }
#pragma unroll
      for (int u = 0; u < kTogether; ++u) {
        if (ls[u] == 0.f) continue;  // no key of this column
        const float most = fmaxf(m, ms[u]), use = most == -INFINITY ? 0.f : most;
        const float f = __builtin_amdgcn_exp2f(m - use), fs = __builtin_amdgcn_exp2f(ms[u] - use);
        acc = acc * f + os[u] * fs;
        sum = sum * f + ls[u] * fs;
        m = most;
      }
    }
  }
  if constexpr (SLICES > 1) {
    part[threadIdx.x] = acc;
    if (at == 0) { part_m[mine * SLICES + slice] = m; part_l[mine * SLICES + slice] = sum; }
    __syncthreads();
    if (slice) return;
    m = -INFINITY;
#pragma unroll
    for (int s = 0; s < SLICES; ++s) m = fmaxf(m, part_m[mine * SLICES + s]);
    const float use = m == -INFINITY ? 0.f : m;
    acc = f32x4{0.f, 0.f, 0.f, 0.f};
    sum = 0.f;
#pragma unroll
    for (int s = 0; s < SLICES; ++s) {
      if (part_l[mine * SLICES + s] == 0.f) continue;
      const float f = __builtin_amdgcn_exp2f(part_m[mine * SLICES + s] - use);
      acc += f * part[(mine * SLICES + s) * LANES + at];
      sum += f * part_l[mine * SLICES + s];
    }
  }
  if (column > last) return;
  const float inv = sum == 0.f ? NAN : 1.f / (sum * p.rk);
  T* const o = static_cast<T*>(p.o) + column * D + 4 * at;
  if constexpr (sizeof(T) == 2) *reinterpret_cast<u32x2*>(o) = u32x2{pack_bf16(acc[0] * inv, acc[1] * inv), pack_bf16(acc[2] * inv, acc[3] * inv)};
  else *reinterpret_cast<f32x4*>(o) = acc * inv;
  if (p.lse && at == 0) {
    const int qi = c / p.H, h = c - qi * p.H;
    p.lse[((int64_t)b * p.H + h) * p.lq + qi] = sum == 0.f ? -INFINITY : (m + log2f(sum)) * kLn2;
  }
}

// ------------------------------------------------------------------------------------------------ any shape
// A workgroup per query row and head, 256 keys at a time: a thread's key by itself, then the threads' output columns over the keys.
template <typename T>
__global__ __launch_bounds__(kThreads) void decode_fp4_any_kernel(Fp4Params p) {
  __shared__ float q[256], weight[kThreads], red[2][kWaves], out[kThreads];
  __shared__ int64_t v_row[kThreads];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int b = blockIdx.x / p.cols, c = blockIdx.x - b * p.cols, qi = c / p.H, h = c - qi * p.H;
  const Fp4Row k_parts(p.H, p.dk), v_parts(p.H, p.dv);
  for (int d = tid; d < p.dk; d += kThreads) {
    float x = 0.f;
    for (int r = 0; r < p.rq; ++r)
      x += load_as_f32(static_cast<const T*>(p.qa.ptr) + b * p.qa.stride_b + qi * p.qa.stride_l + r * p.qa.stride_r + h) *
           load_as_f32(static_cast<const T*>(p.qb.ptr) + b * p.qb.stride_b + qi * p.qb.stride_l + r * p.qb.stride_r + d);
    q[d] = x / p.rq;
  }
  const int keys = keys_seen(p, length_of(p, b), qi);
  const int columns = kThreads / p.dv, d = tid % p.dv, slice = tid / p.dv;  // (dv <= 256) threads past the last slice idle
  float m = -INFINITY, sum = 0.f, acc = 0.f;
  __syncthreads();
  for (int t0 = 0; t0 < keys; t0 += kThreads) {
    const int t = t0 + tid;
    float x = -INFINITY;
    if (t < keys) {
      int64_t page = b;
      int in_page = t;
      if (p.table) {
        const int nth = t / p.page_size;
        page = max(0, min(p.table[(int64_t)b * p.pages_per_seq + nth], p.num_pages - 1));
        in_page = t - nth * p.page_size;
      }
      v_row[tid] = page * p.vc.stride_b + in_page * p.vc.stride_l;
      const uint8_t* const k = static_cast<const uint8_t*>(p.kc.ptr) + page * p.kc.stride_b + in_page * p.kc.stride_l;
      x = 0.f;
      for (int r = 0; r < p.rk; ++r) {
        const uint8_t* const row = k + r * p.kc.stride_r;
        float dot = 0.f;
        for (int j = 0; j < p.dk; ++j) dot += q[j] * fp4_number(row, row + k_parts.b_scales, j);
        x += dot * fp4_number(row + k_parts.a_codes, row + k_parts.a_scales, h);
      }
      x *= p.scale / p.rk;
    }
    float most = x;
#pragma unroll
    for (int s = 32; s; s /= 2) most = fmaxf(most, __shfl_xor(most, s));
    if (lane == 0) red[0][w] = most;
    __syncthreads();
    most = m;
    for (int s = 0; s < kWaves; ++s) most = fmaxf(most, red[0][s]);
    const float use = most == -INFINITY ? 0.f : most, f = expf(m - use);
    m = most;
    float part = t < keys ? expf(x - use) : 0.f;
    weight[tid] = part;
#pragma unroll
    for (int s = 32; s; s /= 2) part += __shfl_xor(part, s);
    if (lane == 0) red[1][w] = part;
    __syncthreads();
    sum *= f;
    for (int s = 0; s < kWaves; ++s) sum += red[1][s];
    acc *= f;
    if (slice < columns)
      for (int u = slice; u < min(kThreads, keys - t0); u += columns) {
        const uint8_t* const v = static_cast<const uint8_t*>(p.vc.ptr) + v_row[u];
        float x = 0.f;
        for (int r = 0; r < p.rk; ++r) {
          const uint8_t* const row = v + r * p.vc.stride_r;
          x += fp4_number(row + v_parts.a_codes, row + v_parts.a_scales, h) * fp4_number(row, row + v_parts.b_scales, d);
        }
        acc += weight[u] * x;
      }
    __syncthreads();
  }
  out[tid] = acc;
  __syncthreads();
  if (tid < p.dv) {
    float x = 0.f;
    for (int s = 0; s < columns; ++s) x += out[s * p.dv + tid];
    store_from_f32(static_cast<T*>(p.o) + ((int64_t)b * p.cols + c) * p.dv + tid, sum == 0.f ? NAN : x / (sum * p.rk));
  }
  if (p.lse && tid == 0) p.lse[((int64_t)b * p.H + h) * p.lq + qi] = sum == 0.f ? -INFINITY : m + logf(sum);
}

// ------------------------------------------------------------------------------------------------ host side
bool mfma_takes(const TpaDecodeFp4Args* a) {
  if (a->dk != a->dv || (a->dk != 64 && a->dk != 128) || a->H % 8 || (a->rk != 1 && a->rk != 2 && a->rk != 4 && a->rk != 8)) return false;
  if ((int64_t)a->B * ((int64_t)a->lk * a->rk / (kRows * kWaves) + 1 + kStart) > INT32_MAX) return false;  // rounds
  if ((int64_t)a->lq * a->H > 32 * 65535) return false;  // sets of columns are the second dimension of the grid
  for (const TpaFactor* f : {&a->k_cache, &a->v_cache})
    if (reinterpret_cast<uintptr_t>(f->ptr) % 4 || f->stride_b % 4 || f->stride_l % 4 || f->stride_r % 4) return false;
  return true;
}

// whether rows lie one behind the other and blocks of 32 of them are inside a page (a block is then less than 2^31 bytes)
bool dense_rows(const TpaDecodeFp4Args* a) {
  for (const TpaFactor* f : {&a->k_cache, &a->v_cache})
    if (f->stride_r < 0 || f->stride_r > 1 << 20 || f->stride_l != a->rk * f->stride_r) return false;
  return (a->page_table ? (int64_t)a->page_size * a->rk : (int64_t)a->lk * a->rk) % kRows == 0;
}

struct Plan { int col_groups, groups; bool dense; int64_t slots; size_t plan_bytes, bytes; };
Plan plan_of(const TpaDecodeFp4Args* a) {
  Plan p;
  const int64_t cols = (int64_t)a->lq * a->H;
  p.col_groups = (int)((cols + 31) / 32);
  const int64_t rounds = a->B * (((int64_t)a->lk * a->rk + kRows * kWaves - 1) / (kRows * kWaves) + kStart);
  p.groups = (int)std::max<int64_t>(1, std::min<int64_t>(rounds, kMostGroups / p.col_groups));
  p.dense = dense_rows(a);
  p.slots = (int64_t)p.groups + a->B;
  p.plan_bytes = (4 * ((size_t)a->B + 1) + 255) / 256 * 256;
  p.bytes = p.plan_bytes + 4 * (size_t)p.slots * cols * (a->dv + 2);
  return p;
}

bool on_vector_units(const TpaDecodeFp4Args* a) { return a->kernel == TPA_KERNEL_GENERIC || !mfma_takes(a); }

int check_args(const TpaDecodeFp4Args* a) {
  if (!a) return TPA_ERR_NULL;
  if (a->dtype != TPA_DTYPE_F32 && a->dtype != TPA_DTYPE_BF16) return TPA_ERR_DTYPE;
  if (a->B <= 0 || a->lq <= 0 || a->lk <= 0 || a->H <= 0 || a->dk <= 0 || a->dv <= 0 || a->rq <= 0 || a->rk <= 0) return TPA_ERR_SHAPE;
  if (a->dk > 256 || a->dv > 256 || (int64_t)a->B * a->lq > 1 << 24 || (int64_t)a->B * a->lq * a->H > 1 << 24 || (int64_t)a->lk * a->rk > INT32_MAX / 2) return TPA_ERR_SHAPE;
  if (a->causal < TPA_CAUSAL_NONE || a->causal > TPA_CAUSAL_BOTTOM_RIGHT) return TPA_ERR_UNSUPPORTED;
  if (a->kernel != TPA_KERNEL_AUTO && a->kernel != TPA_KERNEL_GENERIC && a->kernel != TPA_KERNEL_MFMA) return TPA_ERR_UNSUPPORTED;
  for (const TpaFactor* f : {&a->qa, &a->qb, &a->k_cache, &a->v_cache})
    if (!f->ptr) return TPA_ERR_NULL;
  if (a->page_table && (a->page_size <= 0 || a->pages_per_seq <= 0 || a->num_pages <= 0 || (int64_t)a->page_size * a->pages_per_seq < a->lk)) return TPA_ERR_SHAPE;
  if (a->kernel == TPA_KERNEL_MFMA && !mfma_takes(a)) return TPA_ERR_UNSUPPORTED;
  // the vector-unit kernel's workgroups of 256 threads: a launch takes fewer than 2^32
  if (on_vector_units(a) && (int64_t)a->B * a->lq * a->H == 1 << 24) return TPA_ERR_SHAPE;
  return TPA_OK;
}

template <typename T, int D, int RK, int QS, int PS, int LAYOUT>
int launch(const Fp4Params& p, const Plan& plan, hipStream_t stream) {
  auto kern = decode_fp4_kernel<T, D, RK, QS, PS, LAYOUT>;
  constexpr size_t lds = Fp4Lds<D, QS, LAYOUT>::kBytes;
  static bool configured[kMaxDevices] = {};
  if (int rc = raise_lds_limit(configured, reinterpret_cast<const void*>(kern), lds); rc != TPA_OK) return rc;
  hipLaunchKernelGGL(kern, dim3(p.groups, plan.col_groups), dim3(kThreads), lds, stream, p);
  return hipGetLastError() == hipSuccess ? TPA_OK : TPA_ERR_LAUNCH;
}
template <typename T, int D, int SLICES>
int launch_join(const Fp4Params& p, hipStream_t stream) {
  constexpr int cols = kThreads / (D / 4) / SLICES;
  hipLaunchKernelGGL((join_kernel<T, D, SLICES>), dim3((unsigned)(((int64_t)p.B * p.cols + cols - 1) / cols)), dim3(kThreads), 0, stream, p);
  return hipGetLastError() == hipSuccess ? TPA_OK : TPA_ERR_LAUNCH;
}
template <typename T, int D, int RK>
int launch_layout(const Fp4Params& p, const Plan& plan, hipStream_t stream) {
  constexpr int QS = sizeof(T) == 2 ? 2 : 3, PS = QS;
  if (!plan.dense) return launch<T, D, RK, QS, PS, kRowsApart>(p, plan, stream);
  if (p.H == 8 || p.H == 16) return launch<T, D, RK, QS, PS, kFewHeads>(p, plan, stream);
  if (p.H % 32 == 0 && D / 32 + p.H / 32 <= D / 16) return launch<T, D, RK, QS, PS, kWholeSets>(p, plan, stream);
  return launch<T, D, RK, QS, PS, kRowsApart>(p, plan, stream);
}
template <typename T, int D>
int launch_both(const Fp4Params& p, const Plan& plan, hipStream_t stream) {
  int rc;
  switch (p.rk) {
    case 1: rc = launch_layout<T, D, 1>(p, plan, stream); break;
    case 2: rc = launch_layout<T, D, 2>(p, plan, stream); break;
    case 4: rc = launch_layout<T, D, 4>(p, plan, stream); break;
    default: rc = launch_layout<T, D, 8>(p, plan, stream);
  }
  if (rc != TPA_OK) return rc;
  return p.groups > 8 * (int64_t)p.B ? launch_join<T, D, 8>(p, stream) : launch_join<T, D, 1>(p, stream);
}

}  // namespace
}  // namespace tpa

extern "C" size_t tpa_decode_fp4_workspace_bytes(const TpaDecodeFp4Args* a) {
  using namespace tpa;
  if (check_args(a) != TPA_OK || on_vector_units(a)) return 0;
  return plan_of(a).bytes;
}

extern "C" int tpa_decode_fp4(const TpaDecodeFp4Args* a, void* stream) {
  using namespace tpa;
  if (int rc = check_args(a); rc != TPA_OK) return rc;
  if (!a->o) return TPA_ERR_NULL;
  Fp4Params p{};
  p.qa = a->qa; p.qb = a->qb; p.kc = a->k_cache; p.vc = a->v_cache;
  p.o = a->o; p.lse = a->lse; p.kvlen = a->kv_lengths; p.table = a->page_table;
  p.page_size = a->page_size > 0 ? a->page_size : 1; p.pages_per_seq = a->pages_per_seq; p.num_pages = a->num_pages;
  p.page_shift = (p.page_size & (p.page_size - 1)) == 0 ? __builtin_ctz(p.page_size) : -1;
  p.B = a->B; p.lq = a->lq; p.lk = a->lk; p.H = a->H; p.dk = a->dk; p.dv = a->dv; p.rq = a->rq; p.rk = a->rk; p.cols = a->lq * a->H;
  p.causal = a->causal;
  if (a->causal) {
    const int far = a->causal == TPA_CAUSAL_BOTTOM_RIGHT ? a->lq + a->lk : a->lk;
    p.coff = clamp_causal_offset(a->causal_offset, a->causal == TPA_CAUSAL_BOTTOM_RIGHT ? -far : -a->lq, far);
  }
  const hipStream_t on = static_cast<hipStream_t>(stream);
  if (on_vector_units(a)) {
    p.scale = a->sm_scale;
    const dim3 grid((unsigned)(p.B * p.cols));
    if (a->dtype == TPA_DTYPE_BF16) hipLaunchKernelGGL(decode_fp4_any_kernel<uint16_t>, grid, dim3(kThreads), 0, on, p);
    else hipLaunchKernelGGL(decode_fp4_any_kernel<float>, grid, dim3(kThreads), 0, on, p);
    return hipGetLastError() == hipSuccess ? TPA_OK : TPA_ERR_LAUNCH;
  }
  const Plan plan = plan_of(a);
  if (!a->workspace || a->workspace_bytes < plan.bytes) return TPA_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(a->workspace) % 256 || reinterpret_cast<uintptr_t>(a->o) % 16) return TPA_ERR_ALIGN;
  p.scale = a->sm_scale * kLog2e / ((float)a->rq * (float)a->rk);
  p.groups = plan.groups;
  p.inv_h = 1.f / (float)a->H;
  p.plan = static_cast<int32_t*>(a->workspace);
  p.part_o = reinterpret_cast<float*>(static_cast<char*>(a->workspace) + plan.plan_bytes);
  p.part_m = p.part_o + plan.slots * p.cols * p.dv;
  p.part_l = p.part_m + plan.slots * p.cols;
  if (a->dtype == TPA_DTYPE_BF16) return a->dk == 128 ? launch_both<uint16_t, 128>(p, plan, on) : launch_both<uint16_t, 64>(p, plan, on);
  return a->dk == 128 ? launch_both<float, 128>(p, plan, on) : launch_both<float, 64>(p, plan, on);
}
