// The continuations of a step of beam search: the largest values of score + logit - log sum exp over a request's beams and vocabulary.
//
// First launch: a wave reads a chunk of a beam's logits once.  Every lane keeps a sum of exponentials against a maximum of its own; the largest logits of the
// chunk stand sorted in the lanes of the wave (lane r: the r-th), and a logit goes in only if it beats the last of them, which after the first few hundred
// hardly any does: num_out * ln(chunk / 512) on average.  (Inside a beam the order of the values is that of the logits.)
// Second launch: a workgroup for each request joins the sums and picks num_out times the largest of the chunks' candidates, in 64 bits.
// Equal values go to the lower index: logits are put in by rising index, behind their equals, and the last step compares value and index.
//
// HBM bounds it where there are many beams, the latency of two launches where there are few.
#include <algorithm>

#include "tpa_common.h"

namespace tpa {
namespace {

constexpr int kThreads = 256;
constexpr int kBatch = 512;      // logits that a wave looks at together, eight a lane
constexpr int kAhead = 4;        // batches asked for together
constexpr int kHeld = 8192;      // candidates that the second launch holds in LDS
// log2(e) in two parts: one alone is off by 1.3e-8 of itself, which a logit of 12 makes 2e-7 of every term
constexpr float kLog2eHigh = 1.44269502f, kLog2eLow = 1.92596299e-8f;

struct Sum { double s; float r; int unused; };  // sum of exp2(x log2 e - r)
struct Candidate { float logit; int token; };    // token < 0: none

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
  int B, n, vocab, k, eos, chunk, chunks;
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
};

template <typename T>
__global__ __launch_bounds__(kThreads) void chunk_kernel(BeamParams p) {
  const int lane = threadIdx.x & 63;
  const int64_t id = (int64_t)blockIdx.x * (kThreads / 64) + scalar((int)(threadIdx.x >> 6));
  if (id >= (int64_t)p.B * p.n * p.chunks) return;
  const int row = (int)(id / p.chunks), chunk = (int)(id - (int64_t)row * p.chunks), b = row / p.n, beam = row - b * p.n;
  if (p.finished && p.finished[row]) return;  // its one candidate needs no logits
  const T* const logits = static_cast<const T*>(p.logits) + b * p.stride_b + beam * p.stride_n;
  const int begin = chunk * p.chunk, end = begin + min(p.chunk, p.vocab - begin);

  float r = -INFINITY, s = 0.f;             // this lane's logits: sum of exp2(x log2 e - r)
  float best = -INFINITY;                   // lane i: the i-th largest logit so far
  int token = -1;
  float least = -INFINITY;                  // the k-th largest: what a logit has to beat
  auto look = [&](const float (&x)[8], int first, bool fill) __attribute__((always_inline)) {
    const float most = max8(x);
    const float rn = fmaxf(r, most * kLog2eHigh), ru = rn == -INFINITY ? 0.f : rn;
    float terms[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) terms[j] = __builtin_amdgcn_exp2f(fmaf(x[j], kLog2eLow, fmaf(x[j], kLog2eHigh, -ru)));
    s = fmaf(s, __builtin_amdgcn_exp2f(r - ru), ((terms[0] + terms[1]) + (terms[2] + terms[3])) + ((terms[4] + terms[5]) + (terms[6] + terms[7])));
    r = rn;
    if (fill) {
      // the k-th largest of the lanes' maxima: at least k logits of the first batch are no smaller
      int key = ordered(most), at = 0;
      for (int i = 0; i < p.k; ++i) {
        at = wave_max(key);
        const uint64_t there = __ballot(key == at);
        if (lane == __builtin_ctzll(there)) key = INT32_MIN;
      }
      // the number below it, for what is not below the maximum goes in: -inf for that of -inf (whose neighbour is a NaN), and no zero, which
      // the zero on its other side does not beat
      least = fmaxf(from_ordered(max(at, INT32_MIN + 1) - 1), -INFINITY);
      if (least == 0.f) least = __uint_as_float(0x80000001u);
    }
    uint64_t lanes = __ballot(most > least);
    while (lanes) {
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
          token = lane > at ? token_before : lane == at ? first + 8 * from + j : token;
          least = fmaxf(least, lane_value(best, p.k - 1));
        }
      }
    }
  };

  Eight<T> now[kAhead], next[kAhead];
  const int whole = (end - begin) / kBatch;  // batches without a missing logit
  auto request = [&](Eight<T>(&to)[kAhead], int batch) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) to[u].load(logits + begin + (int64_t)min(batch + u, whole - 1) * kBatch + 8 * lane);
  };
  if (whole > 0) request(now, 0);
  for (int batch = 0; batch < whole; batch += kAhead) {
    if (batch + kAhead < whole) request(next, batch + kAhead);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (batch + u >= whole) break;
      float x[8];
      now[u].get(x);
      look(x, begin + (batch + u) * kBatch, batch + u == 0);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) now[u] = next[u];
  }
  if (begin + whole * kBatch < end) {
    float x[8];
    const int first = begin + whole * kBatch;
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = first + 8 * lane + j < end ? load_as_f32(logits + first + 8 * lane + j) : -INFINITY;
    look(x, first, whole == 0);
  }

  const float rw = from_ordered(wave_max(ordered(r))), ru = rw == -INFINITY ? 0.f : rw;
  double sum = (double)s * (double)__builtin_amdgcn_exp2f(r - ru);
#pragma unroll
  for (int d = 32; d; d /= 2) sum += __shfl_xor(sum, d);
  if (lane == 0) p.sums[id] = Sum{sum, rw, 0};
  if (lane < p.k) p.candidates[id * p.k + lane] = Candidate{best, token};
}

__global__ __launch_bounds__(kThreads) void select_kernel(BeamParams p) {
  extern __shared__ __attribute__((aligned(8))) char smem_beam[];
  __shared__ double base[TPA_BEAM_MAX];  // of a beam: what is added to its logits
  __shared__ double red_value[kThreads / 64];
  __shared__ int red_flat[kThreads / 64];
  __shared__ double won_value[TPA_BEAM_MAX];
  __shared__ int won[TPA_BEAM_MAX];
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int per_beam = p.chunks * p.k, total = p.n * per_beam;
  const Candidate* const all = p.candidates + (int64_t)b * total;
  Candidate* const held = reinterpret_cast<Candidate*>(smem_beam);
  const bool hold = total <= kHeld;
  if (hold)
    for (int i = tid; i < total; i += kThreads) held[i] = all[i];

  for (int j = w; j < p.n; j += kThreads / 64) {
    const int row = b * p.n + j;
    double value = NAN;  // a finished beam's chunks have no candidates: nothing was written there
    if (!(p.finished && p.finished[row])) {
      float r = -INFINITY;
      for (int c = lane; c < p.chunks; c += 64) r = fmaxf(r, p.sums[(int64_t)row * p.chunks + c].r);
      r = from_ordered(wave_max(ordered(r)));
      double s = 0;
      for (int c = lane; c < p.chunks; c += 64) {
        const Sum x = p.sums[(int64_t)row * p.chunks + c];
        if (x.s != 0) s += x.s * exp2((double)x.r - (double)r);  // (0: nothing but logits of -inf)
      }
#pragma unroll
      for (int d = 32; d; d /= 2) s += __shfl_xor(s, d);
      value = (double)p.scores[row] - ((double)r + log2(s)) * 0.693147180559945309417;
    }
    if (lane == 0) base[j] = value;
  }
  __syncthreads();

  // the best candidate of this thread's behind (value, flat index); values that are no number, or infinite, are none
  auto best_behind = [&](double value, int flat, double& best, int& best_flat) {
    best = -INFINITY;
    best_flat = INT32_MAX;
    auto consider = [&](double v, int f) {
      if (!(fabs(v) < INFINITY)) return;
      if (!(v < value || (v == value && f > flat))) return;
      if (v > best || (v == best && f < best_flat)) { best = v; best_flat = f; }
    };
    for (int i = tid; i < total; i += kThreads) {
      const int j = i / per_beam;
      const Candidate c = hold ? held[i] : all[i];
      if (c.token >= 0) consider(base[j] + (double)c.logit, j * p.vocab + c.token);
    }
    if (p.finished && tid < p.n && p.finished[b * p.n + tid]) consider((double)p.scores[b * p.n + tid], tid * p.vocab + p.eos);
  };
  double best;
  int flat;
  best_behind(INFINITY, -1, best, flat);
  int found = 0;
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
#pragma unroll
    for (int i = 1; i < kThreads / 64; ++i)
      if (red_value[i] > v || (red_value[i] == v && red_flat[i] < f)) { v = red_value[i]; f = red_flat[i]; }
    if (f == INT32_MAX) break;  // no candidate is left (the same in every thread)
    if (tid == 0) { won_value[found] = v; won[found] = f; }
    if (f == flat) best_behind(v, f, best, flat);
    __syncthreads();
  }
  __syncthreads();
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
  if (tid < p.k) {
    const int64_t to = (int64_t)b * p.k + tid;
    const int beam = won[tid] / p.vocab, token = won[tid] - beam * p.vocab, row = b * p.n + beam;
    p.new_scores[to] = (float)won_value[tid];
    p.parents[to] = row;
    p.tokens[to] = token;
    p.new_finished[to] = (p.finished && p.finished[row]) || token == p.eos;
  }
}

// Logits of a wave: as many as leave about 4096 waves, between 2 and 32 batches.
int chunk_of(int64_t B, int64_t n, int64_t vocab) {
  const int64_t each = (B * n * vocab / 4096 + kBatch - 1) / kBatch * kBatch;
  return (int)std::max<int64_t>(2 * kBatch, std::min<int64_t>(each, 32 * kBatch));
}

}  // namespace
}  // namespace tpa

extern "C" size_t tpa_beam_select_workspace_bytes(int32_t B, int32_t beams, int32_t vocab, int32_t num_out, int32_t dtype) {
  using namespace tpa;
  if (B <= 0 || beams <= 0 || vocab <= 0 || num_out <= 0 || beams > TPA_BEAM_MAX || num_out > TPA_BEAM_MAX) return 0;
  (void)dtype;
  const int chunk = chunk_of(B, beams, vocab);
  const size_t parts = (size_t)B * beams * (((size_t)vocab + chunk - 1) / chunk);
  return parts * (sizeof(Sum) + num_out * sizeof(Candidate));
}

extern "C" int tpa_beam_select(const TpaBeamSelectArgs* a, void* stream) {
  using namespace tpa;
  if (!a) return TPA_ERR_NULL;
  if (a->dtype != TPA_DTYPE_F32 && a->dtype != TPA_DTYPE_BF16) return TPA_ERR_DTYPE;
  if (a->B <= 0 || a->beams <= 0 || a->vocab <= 0 || a->num_out <= 0 || a->beams > TPA_BEAM_MAX || a->num_out > TPA_BEAM_MAX || a->vocab > 1 << 30)
    return TPA_ERR_SHAPE;
  if ((int64_t)a->beams * a->vocab > INT32_MAX || a->num_out > (int64_t)a->beams * a->vocab || (int64_t)a->B * a->beams > INT32_MAX) return TPA_ERR_SHAPE;
  if (a->eos_token < -1 || a->eos_token >= a->vocab) return TPA_ERR_SHAPE;
  if (!a->logits || !a->scores || !a->new_scores || !a->parents || !a->tokens || !a->new_finished) return TPA_ERR_NULL;
  if (a->finished && a->eos_token < 0) return TPA_ERR_UNSUPPORTED;
  BeamParams p{};
  p.chunk = chunk_of(a->B, a->beams, a->vocab);
  p.chunks = (a->vocab + p.chunk - 1) / p.chunk;
  const int64_t parts = (int64_t)a->B * a->beams * p.chunks, groups = (parts + kThreads / 64 - 1) / (kThreads / 64);
  if (groups > INT32_MAX || (int64_t)a->beams * p.chunks * a->num_out > INT32_MAX) return TPA_ERR_SHAPE;
  if (!a->workspace || a->workspace_bytes < tpa_beam_select_workspace_bytes(a->B, a->beams, a->vocab, a->num_out, a->dtype)) return TPA_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(a->workspace) % 16) return TPA_ERR_ALIGN;
  p.logits = a->logits; p.stride_b = a->stride_b; p.stride_n = a->stride_n; p.scores = a->scores; p.finished = a->finished;
  p.new_scores = a->new_scores; p.parents = a->parents; p.tokens = a->tokens; p.new_finished = a->new_finished;
  p.sums = static_cast<Sum*>(a->workspace);
  p.candidates = reinterpret_cast<Candidate*>(p.sums + parts);
  p.B = a->B; p.n = a->beams; p.vocab = a->vocab; p.k = a->num_out; p.eos = a->eos_token;
  const hipStream_t on = static_cast<hipStream_t>(stream);
  if (a->dtype == TPA_DTYPE_BF16) hipLaunchKernelGGL(chunk_kernel<uint16_t>, dim3((unsigned)groups), dim3(kThreads), 0, on, p);
  else hipLaunchKernelGGL(chunk_kernel<float>, dim3((unsigned)groups), dim3(kThreads), 0, on, p);
  if (hipGetLastError() != hipSuccess) return TPA_ERR_LAUNCH;
  const int64_t total = (int64_t)p.n * p.chunks * p.k;
  static bool configured[kMaxDevices] = {};
  if (int rc = raise_lds_limit(configured, reinterpret_cast<const void*>(select_kernel), kHeld * sizeof(Candidate)); rc != TPA_OK) return rc;
  hipLaunchKernelGGL(select_kernel, dim3(a->B), dim3(kThreads), total <= kHeld ? total * sizeof(Candidate) : 0, on, p);
  return hipGetLastError() == hipSuccess ? TPA_OK : TPA_ERR_LAUNCH;
}
