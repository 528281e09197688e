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
  return 0;
}

extern "C" int tpa_decode_shared(const TpaFwdArgs* a, int32_t prefix, void* stream) {
  using namespace tpa;
  if (const int rc = validate(a, prefix); rc != TPA_OK) return rc;
  if (!a->o) return TPA_ERR_NULL;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a->kernel == TPA_KERNEL_MFMA) return TPA_ERR_UNSUPPORTED;
  const SharedParams p = shared_params(a, prefix);
  const dim3 grid((unsigned)(a->B * a->lq * a->H));
  if (a->dtype == TPA_DTYPE_BF16) hipLaunchKernelGGL(shared_any_kernel<uint16_t>, grid, dim3(kAnyThreads), 0, s, p);
  else hipLaunchKernelGGL(shared_any_kernel<float>, grid, dim3(kAnyThreads), 0, s, p);
  return hipGetLastError() == hipSuccess ? TPA_OK : TPA_ERR_LAUNCH;
}
