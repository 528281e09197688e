// The continuations of a step of beam search: the largest values of score + logit - log sum exp over a request's beams and vocabulary.
//
// First launch: a wave holds a chunk of a beam's logits in its registers.  Every lane sums exponentials against a maximum of its own, a logit; the k-th largest of
// the lanes' maxima bounds the chunk's k largest logits from below, and what is above it is put into a list sorted over the lanes (lane r: the r-th).
// (Inside a beam the order of the values is that of the logits, where these differ enough for 64 bits.)
// Second launch: a workgroup for each request joins the sums and ranks the chunks' candidates, in 64 bits, behind a bound found in the same way.  It has
// 1024 threads where there are many lists: each sum's and each list's reading is a wait of about 1 us (16 beams, 16 continuations, 160 000 fp32 logits, one
// request: 15.8 us; when it took 15.3, 23.3 with 256 threads and 54 with all candidates read in place of each list's first ones), and 256 elsewhere (its barriers are
// cheaper).
// Equal values go to the lower index: logits are put in by rising index, behind their equals, the last step compares value and index, and where different logits can have the last
// place's value they are looked for once more.
//
// HBM bounds it where there are many beams (64 requests, 4 beams, 131 072 bf16 logits: 19.2 + 6.8 us, 67 MB at 3.5 TB/s in the first), the latency of two
// launches where there are few (one request, 4 beams, 50 021 fp32 logits: 5.3 + 6.6 us).
#include <algorithm>

#include "tpa_common.h"

namespace tpa {
namespace {

constexpr int kThreads = 256;
constexpr int kMostThreads = 1024;  // of the second launch, where a request has many lists
constexpr int kBatch = 512;      // logits that a wave looks at together, eight a lane
constexpr int kHeld = 4096;      // candidates that the second launch holds in LDS
constexpr int kListed = 512;     // candidates that it ranks among each other
// log2(e) in two parts: one alone is off by 1.3e-8 of itself, which a distance of 12 makes 2e-7 of a term
constexpr float kLog2eHigh = 1.44269502f, kLog2eLow = 1.92596299e-8f;
// exp(d) of a distance d <= 0 from a maximum.  The maximum itself is a logit: its own term is then 1, and no term more, however large the logits are.  (A maximum
// times log2(e) is rounded, and from logits of 3e9 on what it is off by makes infinities and zeros of the terms that stand at it.)
__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(fmaf(d, kLog2eHigh, d * kLog2eLow)); }

struct Sum { double s; float most; int unused; };  // sum of exp(x - most), most = the largest x; 0 and -inf: nothing but -inf
struct Candidate { float logit; int token; };    // token < 0: none

struct alignas(16) Ranked { double v; int flat, unused; };
// of a beam, `most` = its largest logit (one number for all three would lose the small ones beside a large `most`)
struct alignas(32) Beam {
  double score, most, log_sum, unused;
  __device__ __forceinline__ double value(float logit) const { return score + (((double)logit - most) - log_sum); }
};

struct BeamParams {
  const void* logits;
  int64_t stride_b, stride_n;
  const float* scores;
  const uint8_t* finished;
  float* new_scores;
  int32_t *parents, *tokens;
  uint8_t* new_finished;
  Sum* sums;              // [B, beams, chunks]
  Candidate* candidates;  // [B, beams, chunks, k]
  int B, n, vocab, k, eos, chunks;
  int chunk;              // logits of a chunk
  bool bf16;
};

__device__ __forceinline__ float max8(const float (&x)[8]) {
  return fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
}
// order of floats as that of ints
__device__ __forceinline__ int ordered(float x) {
  const int b = __float_as_int(x);
  return b ^ ((b >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float from_ordered(int b) { return __int_as_float(b ^ ((b >> 31) & 0x7fffffff)); }
__device__ __forceinline__ int lane_before(int x) { return __builtin_amdgcn_update_dpp(x, x, 0x138, 0xf, 0xf, false); }  // wave_shr 1
__device__ __forceinline__ float lane_value(float x, int lane) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), lane)); }

// eight logits from a place that need not be aligned
template <typename T>
struct Eight;
template <>
struct Eight<uint16_t> {
  typedef u32x4 __attribute__((aligned(2))) Raw;
  u32x4 w;
  __device__ __forceinline__ void load(const uint16_t* p) { w = *reinterpret_cast<const Raw*>(p); }
  __device__ __forceinline__ void get(float (&x)[8]) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[2 * j] = bf16lo_to_f32(w[j]);
      x[2 * j + 1] = bf16hi_to_f32(w[j]);
    }
  }
  __device__ __forceinline__ void load_part(const uint16_t* p, int n) {  // the first n of them, -inf behind
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = (2 * j < n ? (uint32_t)p[2 * j] : 0xff80u) | (2 * j + 1 < n ? (uint32_t)p[2 * j + 1] : 0xff80u) << 16;
  }
};
template <>
struct Eight<float> {
  typedef f32x4 __attribute__((aligned(4))) Raw;
  f32x4 lo, hi;
  __device__ __forceinline__ void load(const float* p) {
    lo = *reinterpret_cast<const Raw*>(p);
    hi = *reinterpret_cast<const Raw*>(p + 4);
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[j] = lo[j];
      x[4 + j] = hi[j];
    }
  }
  __device__ __forceinline__ void load_part(const float* p, int n) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      lo[j] = j < n ? p[j] : -INFINITY;
      hi[j] = 4 + j < n ? p[4 + j] : -INFINITY;
    }
  }
};

// NB: batches of a chunk.  The chunk stays in registers: all of it is asked for at once, and when the lanes' maxima are known, the k-th largest of
// them leaves hardly more than k logits to put in.
template <typename T, int NB>
__global__ __launch_bounds__(kThreads) void chunk_kernel(BeamParams p) {
  const int lane = threadIdx.x & 63;
  const int64_t id = (int64_t)blockIdx.x * (kThreads / 64) + scalar((int)(threadIdx.x >> 6));
  if (id >= (int64_t)p.B * p.n * p.chunks) return;
  const int row = (int)(id / p.chunks), chunk = (int)(id - (int64_t)row * p.chunks), b = row / p.n, beam = row - b * p.n;
  if (p.finished && p.finished[row]) return;  // its one candidate needs no logits
  const T* const logits = static_cast<const T*>(p.logits) + b * p.stride_b + beam * p.stride_n;
  const int begin = chunk * (NB * kBatch), end = begin + min(NB * kBatch, p.vocab - begin);

  Eight<T> held[NB];
  if (end - begin == NB * kBatch) {
#pragma unroll
    for (int n = 0; n < NB; ++n) held[n].load(logits + begin + n * kBatch + 8 * lane);
  } else {
#pragma unroll
    for (int n = 0; n < NB; ++n) held[n].load_part(logits + begin + n * kBatch + 8 * lane, end - begin - n * kBatch - 8 * lane);
  }

  float top = -INFINITY, s = 0.f;  // this lane's logits: the largest, sum of exp(x - top)
  float most[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    float x[8];
    held[n].get(x);
    most[n] = max8(x);
    const float now = fmaxf(top, most[n]), use = now == -INFINITY ? 0.f : now;
    float terms[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) terms[j] = exp_of(x[j] - use);
    s = fmaf(s, exp_of(top - use), ((terms[0] + terms[1]) + (terms[2] + terms[3])) + ((terms[4] + terms[5]) + (terms[6] + terms[7])));
    top = now;
  }

  // the k-th largest of the lanes' maxima: at least k logits are no smaller
  int key = ordered(top), at_key = 0;
  for (int i = 0; i < p.k; ++i) {
    at_key = wave_max(key);
    const uint64_t there = __ballot(key == at_key);
    if (lane == __builtin_ctzll(there)) key = INT32_MIN;
  }
  // what a logit has to beat: the number below that one, -inf for that of -inf (whose neighbour is a NaN), and no zero, which the zero on its
  // other side does not beat
  float least = fmaxf(from_ordered(max(at_key, INT32_MIN + 1) - 1), -INFINITY);
  if (least == 0.f) least = __uint_as_float(0x80000001u);
  float best = -INFINITY;  // lane i: the i-th largest logit so far
  int token = -1;
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    uint64_t lanes = __ballot(most[n] > least);
    if (!lanes) continue;
    float x[8];
    held[n].get(x);
    do {
      const int from = __builtin_ctzll(lanes);
      lanes &= lanes - 1;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float v = lane_value(x[j], from);
        if (v > least) {
          const int at = __popcll(__ballot(best >= v));  // behind its equals
          const float best_before = __int_as_float(lane_before(__float_as_int(best)));
          const int token_before = lane_before(token);
          best = lane > at ? best_before : lane == at ? v : best;
          token = lane > at ? token_before : lane == at ? begin + n * kBatch + 8 * from + j : token;
          least = fmaxf(least, lane_value(best, p.k - 1));
        }
      }
    } while (lanes);
  }

  const float all = from_ordered(wave_max(ordered(top))), use = all == -INFINITY ? 0.f : all;
  double sum = (double)s * (double)exp_of(top - use);
#pragma unroll
  for (int d = 32; d; d /= 2) sum += __shfl_xor(sum, d);
  if (lane == 0) p.sums[id] = Sum{sum, all, 0};
  if (lane < p.k) p.candidates[id * p.k + lane] = Candidate{best, token};
}

// Candidates of each list that the second launch copies to LDS first, in loads that do not wait for each other: all, if they fit, or the best one
__host__ __device__ inline int held_of_each(int lists, int k) { return (int64_t)lists * k <= kHeld ? k : lists <= kHeld ? 1 : 0; }

__global__ __launch_bounds__(kMostThreads) void select_kernel(BeamParams p) {
  extern __shared__ __attribute__((aligned(8))) char smem_beam[];
  __shared__ Beam beams[TPA_BEAM_MAX];
  __shared__ double red_value[kMostThreads / 64];
  __shared__ int red_flat[kMostThreads / 64];
  __shared__ double won_value[TPA_BEAM_MAX];
  __shared__ int won[TPA_BEAM_MAX], listed;
  __shared__ Ranked list[kListed];
  __shared__ int keys[kMostThreads];
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = tid >> 6, threads = blockDim.x, waves = threads / 64;
  const int lists = p.n * p.chunks;
  const Candidate* const all = p.candidates + (int64_t)b * lists * p.k;
  Candidate* const held = reinterpret_cast<Candidate*>(smem_beam);
  const int hold = held_of_each(lists, p.k);
  if (hold == 1)
    for (int i = tid; i < lists; i += threads) held[i] = all[i * p.k];
  else
    for (int i = tid; i < lists * hold; i += threads) held[i] = all[i];

  for (int j = w; j < p.n; j += waves) {
    const int row = b * p.n + j;
    double log_of = NAN;  // a finished beam's chunks have no candidates: nothing was written there
    float most = -INFINITY;
    if (!(p.finished && p.finished[row])) {
      for (int c = lane; c < p.chunks; c += 64) most = fmaxf(most, p.sums[(int64_t)row * p.chunks + c].most);
      most = from_ordered(wave_max(ordered(most)));
      double s = 0;
      for (int c = lane; c < p.chunks; c += 64) {
        const Sum x = p.sums[(int64_t)row * p.chunks + c];
        if (x.s != 0) s += x.s * exp((double)x.most - (double)most);  // (0: nothing but logits of -inf)
      }
#pragma unroll
      for (int d = 32; d; d /= 2) s += __shfl_xor(s, d);
      log_of = log(s);
    }
    if (lane == 0) beams[j] = Beam{(double)p.scores[row], (double)most, log_of, 0};
  }
  __syncthreads();

  // This thread's candidates, list by list, each list's best first; values that are no number, or infinite, are none.  `visit` says whether it wants
  // more of a list: of most lists only the first candidate is looked at, which is what keeps many beams with many continuations cheap.
  auto for_each = [&](auto visit) __attribute__((always_inline)) {
    for (int i = tid; i < lists; i += threads) {
      const int j = i / p.chunks;
      for (int r = 0; r < p.k; ++r) {
        const Candidate c = r < hold ? held[i * hold + r] : all[i * p.k + r];
        const double v = beams[j].value(c.logit);
        if (c.token < 0 || !(fabs(v) < INFINITY) || !visit(v, j * p.vocab + c.token)) break;
      }
    }
    if (p.finished && tid < p.n && p.finished[b * p.n + tid]) {
      const double v = (double)p.scores[b * p.n + tid];
      if (fabs(v) < INFINITY) visit(v, tid * p.vocab + p.eos);
    }
  };
  // A bound: the k-th largest of the threads' best candidates, as fp32 rounded down, leaves k candidates or hardly more (every wave looks for it)
  double most = -INFINITY;
  for_each([&](double v, int) { most = fmax(most, v); return false; });
  keys[tid] = ordered((float)most) - ((double)(float)most > most);
  if (tid == 0) listed = 0;
  __syncthreads();
  int key[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) key[j] = keys[64 * j + lane];
  for (int i = kThreads; i < threads; i += kThreads)
#pragma unroll
    for (int j = 0; j < 4; ++j) key[j] = max(key[j], keys[i + 64 * j + lane]);
  int at_key = 0;
  for (int i = 0; i < p.k; ++i) {
    const int of_lane = max(max(key[0], key[1]), max(key[2], key[3]));
    at_key = wave_max(of_lane);
    const uint64_t there = __ballot(of_lane == at_key);
    bool here = lane == __builtin_ctzll(there);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (here && key[j] == at_key) { key[j] = INT32_MIN; here = false; }
  }
  const float bound = from_ordered(max(at_key, ordered(-INFINITY)));
  for_each([&](double v, int f) {
    if (v < (double)bound) return false;
    const int at = atomicAdd(&listed, 1);
    if (at < kListed) list[at] = Ranked{v, f, 0};
    return true;
  });
  __syncthreads();
  int found = 0;
  if (listed <= kListed) {
    // in whatever order they stand: each one's place is the number of those that beat it
    found = min(listed, p.k);
    for (int i = tid; i < listed; i += threads) {
      const double v = list[i].v;
      const int f = list[i].flat;
      int place = 0;
#pragma unroll 8
      for (int j = 0; j < listed; ++j) place += list[j].v > v || (list[j].v == v && list[j].flat < f);
      if (place < p.k) { won_value[place] = v; won[place] = f; }
    }
  } else {
    // many that are alike: the best one behind the last, k times
    double best;
    int flat;
    auto best_behind = [&](double value, int after) {
      best = -INFINITY;
      flat = INT32_MAX;
      for_each([&](double v, int f) {
        if (v < best) return false;
        if ((v < value || (v == value && f > after)) && (v > best || f < flat)) { best = v; flat = f; }
        return true;
      });
    };
    best_behind(INFINITY, -1);
    for (; found < p.k; ++found) {
      double v = best;
      int f = flat;
#pragma unroll
      for (int d = 32; d; d /= 2) {
        const double ov = __shfl_xor(v, d);
        const int of = __shfl_xor(f, d);
        if (ov > v || (ov == v && of < f)) { v = ov; f = of; }
      }
      if (lane == 0) { red_value[w] = v; red_flat[w] = f; }
      __syncthreads();
      v = red_value[0];
      f = red_flat[0];
      for (int i = 1; i < waves; ++i)
        if (red_value[i] > v || (red_value[i] == v && red_flat[i] < f)) { v = red_value[i]; f = red_flat[i]; }
      if (f == INT32_MAX) break;  // no candidate is left (the same in every thread)
      if (tid == 0) { won_value[found] = v; won[found] = f; }
      if (f == flat) best_behind(v, f);
      __syncthreads();
    }
  }
  __syncthreads();
  // Logits that differ can have the same value: beside one of 1e30 all others are -1e30.  The lists go by logits, so of those with the last place's value they may lack some, and lower
  // indices than they hold.  Fp32 numbers are 2^-24 of themselves apart or more, the steps of the value's sums are 2^-51 of its largest number or less: such logits are no more than
  // 2^-27 of that one (2^-26: x is off by as little).  Then the logits with this value are looked for again, in the chunks that have one of them in their lists.
  if (found == p.k) {
    const double last = won_value[p.k - 1];
    bool alike = false;
    if (lane < p.n) {  // every wave all beams (x is no number, or infinite, for a beam that is finished or without candidates)
      const Beam of = beams[lane];
      const double x = ((last - of.score) + of.log_sum) + of.most;
      alike = fabs(x) < INFINITY && fabs(x) <= 0x1p-26 * fmax(fmax(fabs(last), fabs(of.score)), fmax(fabs(of.log_sum), fabs(of.most)));
    }
    if (__any(alike)) {
      int count = 0;  // places before, then those given again
      while (won_value[count] > last) ++count;
      for (int l0 = 0; l0 < lists && count < p.k; l0 += 64) {  // every wave the same lists
        const int mine = l0 + lane, j_of_mine = mine / p.chunks;
        bool has = false;
        if (mine < lists) {
          for (int r = 0; r < p.k && !has; ++r) {
            const Candidate c = all[(int64_t)mine * p.k + r];
            const double v = beams[j_of_mine].value(c.logit);
            if (c.token < 0 || !(v >= last)) break;
            has = v == last;
          }
          if (mine % p.chunks == 0 && p.finished && p.finished[b * p.n + j_of_mine]) has = beams[j_of_mine].score == last;
        }
        for (uint64_t those = __ballot(has); those && count < p.k; those &= those - 1) {
          const int i = l0 + __builtin_ctzll(those), j = i / p.chunks, begin = (i - j * p.chunks) * p.chunk, end = begin + min(p.chunk, p.vocab - begin);
          if (p.finished && p.finished[b * p.n + j]) {
            if (tid == 0) won[count] = j * p.vocab + p.eos;
            ++count;
            continue;
          }
          const int64_t row = b * p.stride_b + j * p.stride_n;
          for (int t0 = begin; t0 < end && count < p.k; t0 += threads) {
            const int t = t0 + tid;
            float x = -INFINITY;
            if (t < end) x = p.bf16 ? bf16bits_to_f32(static_cast<const uint16_t*>(p.logits)[row + t]) : static_cast<const float*>(p.logits)[row + t];
            const uint64_t here = __ballot(t < end && beams[j].value(x) == last);
            if (lane == 0) red_flat[w] = __popcll(here);
            __syncthreads();
            int place = count + __popcll(here & ((1ull << lane) - 1));
            for (int v = 0; v < waves; ++v) {
              if (v < w) place += red_flat[v];
              count += red_flat[v];
            }
            if ((here >> lane & 1) && place < p.k) won[place] = j * p.vocab + t;
            __syncthreads();
          }
        }
      }
      __syncthreads();
    }
  } else {
    // places without a candidate: values of -inf, the lowest indices that have not won
    if (tid == 0) {
      int next = 0;
      for (int i = found; i < p.k; ++next) {
        bool taken = false;
        for (int j = 0; j < found; ++j) taken = taken || won[j] == next;
        if (taken) continue;
        won_value[i] = -INFINITY;
        won[i++] = next;
      }
    }
    __syncthreads();
  }
  if (tid < p.k) {
    const int64_t to = (int64_t)b * p.k + tid;
    const int beam = won[tid] / p.vocab, token = won[tid] - beam * p.vocab, row = b * p.n + beam;
    p.new_scores[to] = (float)won_value[tid];
    p.parents[to] = row;
    p.tokens[to] = token;
    p.new_finished[to] = (p.finished && p.finished[row]) || token == p.eos;
  }
}

// Batches of a chunk: as many as leave about 4096 waves, as far as a chunk fits the registers
int batches_of(int64_t B, int64_t n, int64_t vocab, int dtype) {
  const int64_t logits = B * n * vocab;
  int batches = 2;
  while (batches < (dtype == TPA_DTYPE_BF16 ? 16 : 8) && logits > (int64_t)4096 * batches * kBatch) batches *= 2;
  return batches;
}
int64_t chunks_of(int64_t B, int64_t n, int64_t vocab, int dtype) {
  const int64_t chunk = (int64_t)batches_of(B, n, vocab, dtype) * kBatch;
  return (vocab + chunk - 1) / chunk;
}
// Workgroups of the first launch for sizes that a call takes, otherwise 0.  A launch takes fewer than 2^32 work-items.
int64_t groups_of(int64_t B, int64_t n, int64_t vocab, int64_t k, int dtype) {
  if (dtype != TPA_DTYPE_F32 && dtype != TPA_DTYPE_BF16) return 0;
  if (B <= 0 || n <= 0 || vocab <= 0 || k <= 0 || n > TPA_BEAM_MAX || k > TPA_BEAM_MAX || vocab > 1 << 30 || n * vocab > INT32_MAX || k > n * vocab || B * n > INT32_MAX) return 0;
  const int64_t chunks = chunks_of(B, n, vocab, dtype), groups = (B * n * chunks + kThreads / 64 - 1) / (kThreads / 64);
  // (the second launch has 1024 threads for more than 512 lists, of which the first has a wave for each: B is below 2^17 there)
  return std::max(groups, B) * kThreads > UINT32_MAX || n * chunks * k > INT32_MAX ? 0 : groups;
}

}  // namespace
}  // namespace tpa

extern "C" size_t tpa_beam_select_workspace_bytes(int32_t B, int32_t beams, int32_t vocab, int32_t num_out, int32_t dtype) {
  using namespace tpa;
  if (!groups_of(B, beams, vocab, num_out, dtype)) return 0;
  const size_t parts = (size_t)B * beams * chunks_of(B, beams, vocab, dtype);
  return parts * (sizeof(Sum) + num_out * sizeof(Candidate));
}

extern "C" int tpa_beam_select(const TpaBeamSelectArgs* a, void* stream) {
  using namespace tpa;
  if (!a) return TPA_ERR_NULL;
  if (a->dtype != TPA_DTYPE_F32 && a->dtype != TPA_DTYPE_BF16) return TPA_ERR_DTYPE;
  const int64_t groups = groups_of(a->B, a->beams, a->vocab, a->num_out, a->dtype);
  if (!groups) return TPA_ERR_SHAPE;
  if (a->eos_token < -1 || a->eos_token >= a->vocab) return TPA_ERR_SHAPE;
  if (!a->logits || !a->scores || !a->new_scores || !a->parents || !a->tokens || !a->new_finished) return TPA_ERR_NULL;
  if (a->finished && a->eos_token < 0) return TPA_ERR_UNSUPPORTED;
  BeamParams p{};
  p.chunks = (int)chunks_of(a->B, a->beams, a->vocab, a->dtype);
  const int64_t parts = (int64_t)a->B * a->beams * p.chunks;
  if (!a->workspace || a->workspace_bytes < tpa_beam_select_workspace_bytes(a->B, a->beams, a->vocab, a->num_out, a->dtype)) return TPA_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(a->workspace) % 16) return TPA_ERR_ALIGN;
  p.logits = a->logits; p.stride_b = a->stride_b; p.stride_n = a->stride_n; p.scores = a->scores; p.finished = a->finished;
  p.new_scores = a->new_scores; p.parents = a->parents; p.tokens = a->tokens; p.new_finished = a->new_finished;
  p.sums = static_cast<Sum*>(a->workspace);
  p.candidates = reinterpret_cast<Candidate*>(p.sums + parts);
  p.B = a->B; p.n = a->beams; p.vocab = a->vocab; p.k = a->num_out; p.eos = a->eos_token;
  p.chunk = batches_of(a->B, a->beams, a->vocab, a->dtype) * kBatch; p.bf16 = a->dtype == TPA_DTYPE_BF16;
  const hipStream_t on = static_cast<hipStream_t>(stream);
  void (*kern)(BeamParams) = nullptr;
  switch (batches_of(a->B, a->beams, a->vocab, a->dtype)) {
    case 2: kern = p.bf16 ? chunk_kernel<uint16_t, 2> : chunk_kernel<float, 2>; break;
    case 4: kern = p.bf16 ? chunk_kernel<uint16_t, 4> : chunk_kernel<float, 4>; break;
    case 8: kern = p.bf16 ? chunk_kernel<uint16_t, 8> : chunk_kernel<float, 8>; break;
    default: kern = chunk_kernel<uint16_t, 16>;
  }
  hipLaunchKernelGGL(kern, dim3((unsigned)groups), dim3(kThreads), 0, on, p);
  if (hipGetLastError() != hipSuccess) return TPA_ERR_LAUNCH;
  const int lists = p.n * p.chunks;
  static bool configured[kMaxDevices] = {};
  if (int rc = raise_lds_limit(configured, reinterpret_cast<const void*>(select_kernel), kHeld * sizeof(Candidate)); rc != TPA_OK) return rc;
  hipLaunchKernelGGL(select_kernel, dim3(a->B), dim3(lists > 2 * kThreads ? kMostThreads : kThreads), (size_t)lists * held_of_each(lists, p.k) * sizeof(Candidate), on, p);
  return hipGetLastError() == hipSuccess ? TPA_OK : TPA_ERR_LAUNCH;
}
