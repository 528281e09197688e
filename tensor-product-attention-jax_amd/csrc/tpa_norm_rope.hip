// Norms of queries and keys for each head and the rotation by position, on the rank factors, and their gradients.
//
// X_h = (1/R) sum_r a_r[h] b_r is never formed.  Its norm needs the R x R products G of the token's b rows only:
// |X_h|^2 = (1/R^2) a_h^T G a_h; the norm of a head is a factor of its a's, the weight and the rotation act on the b rows, so the
// result has the form that it came in, a cache of it stays factored, and a token costs its factors read once and written once.
// The gradient of |X_h|^2 is of the same kind: G a_h for the a's, and an R x R mixture of the b rows.
//
// G has signs, so |X_h|^2 may be far below the sum of its terms' sizes where ranks cancel.  It is summed in fp32 for bf16 factors,
// whose products are exact there, and in 64 bits for fp32 factors.
#include <type_traits>

#include "tpa_common.h"

namespace tpa {
namespace {

struct Rotation {
  const float *cos, *sin;
  const int32_t* positions;  // [tokens, axes] or null
  int n_axes, last_of[4];    // pairs below last_of[a] and not of an axis before it belong to axis a
  int rope_len;
};
struct Side {  // the queries or the keys
  TpaFactor a, b, a_out, b_out;
  const void* weight;
  int R;
};
struct NormRopeParams {
  Side side[2];
  TpaFactor va, vb, va_out, vb_out;
  const int32_t* slots;
  int page_size, num_slots;
  Rotation rot;
  int B, l, H, D;
  int weight_bf16, normalize;
  float eps;
};
struct BwdSide {
  TpaFactor a, b, da_out, db_out, da, db;
  const void* weight;
  void* d_weight;
  int R;
};
struct NormRopeBwdParams {
  BwdSide side[2];
  Rotation rot;
  int B, l, H, D;
  int weight_bf16, normalize;
  float eps;
  float* partial;  // [side][kPartials][D]
};
constexpr int kPartials = 768;  // partial sums of each weight's gradient, at most

__device__ __forceinline__ float weight_at(const void* w, int bf16, int d) {
  return !w ? 1.f : bf16 ? bf16bits_to_f32(static_cast<const uint16_t*>(w)[d]) : static_cast<const float*>(w)[d];
}
__device__ __forceinline__ int64_t row_of(const Rotation& rot, int64_t token, int i, int axis) {
  const int pos = rot.positions ? rot.positions[token * rot.n_axes + axis] : i;
  return max(0, min(pos, rot.rope_len - 1));
}
// cos and sin of pair j of a token; (1, 0) past the last section
__device__ __forceinline__ float2 turn_of(const Rotation& rot, int64_t token, int i, int j, int pairs) {
  int axis = 0;
  while (axis < rot.n_axes && j >= rot.last_of[axis]) ++axis;
  if (axis == rot.n_axes) return make_float2(1.f, 0.f);
  const int64_t at = row_of(rot, token, i, axis) * pairs + j;
  return make_float2(rot.cos[at], rot.sin[at]);
}
__device__ __forceinline__ float inverse_norm(double square, int D, float eps) {
  const double mean = square / D;
  return 1.f / sqrtf((float)((mean < 0 ? 0 : mean) + eps));  // NaN stays NaN
}

// ---------------------------------------------------------------------------------------------- any shape
// A workgroup serves the tokens of one side in turn, a token in LDS as fp32: a[R][H], b[R][D].  Latency of its steps bounds it.
constexpr int kAnyThreads = 256;
inline size_t any_lds(int R, int H, int D, bool bwd) {
  return (size_t)R * R * sizeof(double) + ((size_t)(bwd ? 2 : 1) * R * (H + D) + (bwd ? 2 : 1) * H + (bwd ? R * R : 0)) * sizeof(float);
}

// G and 1 / norms of the token in LDS
__device__ __forceinline__ void any_norms(const float* a, const float* b, double* G, float* s, int R, int H, int D, int normalize, float eps) {
  if (normalize) {
    for (int x = threadIdx.x; x < R * R; x += kAnyThreads) {
      const int r = x / R, t = x - r * R;
      double sum = 0;
      for (int d = 0; d < D; ++d) sum += (double)b[r * D + d] * (double)b[t * D + d];
      G[x] = sum;
    }
    __syncthreads();
    for (int h = threadIdx.x; h < H; h += kAnyThreads) {
      double sum = 0;
      for (int r = 0; r < R; ++r)
        for (int t = 0; t < R; ++t) sum += (double)a[r * H + h] * (double)a[t * H + h] * G[r * R + t];
      s[h] = inverse_norm(sum / ((double)R * R), D, eps);
    }
  } else {
    for (int h = threadIdx.x; h < H; h += kAnyThreads) s[h] = 1.f;
  }
  __syncthreads();
}
template <typename T>
__device__ __forceinline__ void any_load(float* to, const TpaFactor& f, int bi, int i, int R, int W) {
  const T* const from = static_cast<const T*>(f.ptr) + bi * f.stride_b + i * f.stride_l;
  for (int x = threadIdx.x; x < R * W; x += kAnyThreads) {
    const int r = x / W;
    to[x] = load_as_f32(from + r * f.stride_r + (x - r * W));
  }
}

template <typename T>
__global__ __launch_bounds__(kAnyThreads) void norm_rope_any_kernel(NormRopeParams p) {
  extern __shared__ __attribute__((aligned(16))) double any_smem[];
  const int which = blockIdx.y;  // queries, keys, with slots the values
  const Side& side = p.side[which < 2 ? which : 1];
  const int R = side.R, H = p.H, D = p.D;
  double* const G = any_smem;
  float *const a = reinterpret_cast<float*>(G + R * R), *const b = a + R * H, *const s = b + R * D;
  const int64_t tokens = (int64_t)p.B * p.l;
  for (int64_t token = blockIdx.x; token < tokens; token += gridDim.x) {
    const int bi = (int)(token / p.l), i = (int)(token - (int64_t)bi * p.l);
    int64_t out_b = bi, out_l = i;
    if (which && p.slots) {
      const int slot = p.slots[token];
      if (slot < 0 || slot >= p.num_slots) continue;
      out_b = slot / p.page_size;
      out_l = slot - out_b * p.page_size;
    }
    if (which == 2) {
      const T *const va = static_cast<const T*>(p.va.ptr) + bi * p.va.stride_b + i * p.va.stride_l, *const vb = static_cast<const T*>(p.vb.ptr) + bi * p.vb.stride_b + i * p.vb.stride_l;
      T* const oa = static_cast<T*>(const_cast<void*>(p.va_out.ptr)) + out_b * p.va_out.stride_b + out_l * p.va_out.stride_l;
      T* const ob = static_cast<T*>(const_cast<void*>(p.vb_out.ptr)) + out_b * p.vb_out.stride_b + out_l * p.vb_out.stride_l;
      for (int x = threadIdx.x; x < R * (H + D); x += kAnyThreads) {
        const int r = x / (H + D), c = x - r * (H + D);
        if (c < H) oa[r * p.va_out.stride_r + c] = va[r * p.va.stride_r + c];
        else ob[r * p.vb_out.stride_r + c - H] = vb[r * p.vb.stride_r + c - H];
      }
      continue;
    }
    any_load<T>(a, side.a, bi, i, R, H);
    any_load<T>(b, side.b, bi, i, R, D);
    __syncthreads();
    any_norms(a, b, G, s, R, H, D, p.normalize, p.eps);
    T* const oa = static_cast<T*>(const_cast<void*>(side.a_out.ptr)) + out_b * side.a_out.stride_b + out_l * side.a_out.stride_l;
    T* const ob = static_cast<T*>(const_cast<void*>(side.b_out.ptr)) + out_b * side.b_out.stride_b + out_l * side.b_out.stride_l;
    for (int x = threadIdx.x; x < R * H; x += kAnyThreads) {
      const int r = x / H, h = x - r * H;
      store_from_f32(oa + r * side.a_out.stride_r + h, a[x] * s[h]);
    }
    const int pairs = D / 2;
    for (int x = threadIdx.x; x < R * pairs; x += kAnyThreads) {
      const int r = x / pairs, j = x - r * pairs;
      const float2 t = turn_of(p.rot, token, i, j, pairs);
      const float y0 = b[r * D + 2 * j] * weight_at(side.weight, p.weight_bf16, 2 * j), y1 = b[r * D + 2 * j + 1] * weight_at(side.weight, p.weight_bf16, 2 * j + 1);
      store_from_f32(ob + r * side.b_out.stride_r + 2 * j, y0 * t.x - y1 * t.y);
      store_from_f32(ob + r * side.b_out.stride_r + 2 * j + 1, y1 * t.x + y0 * t.y);
    }
    __syncthreads();  // the next token's factors go where these are
  }
}

template <typename T>
__global__ __launch_bounds__(kAnyThreads) void norm_rope_bwd_any_kernel(NormRopeBwdParams p) {
  extern __shared__ __attribute__((aligned(16))) double any_smem[];
  const BwdSide& side = p.side[blockIdx.y];
  if (!side.da_out.ptr) return;
  const int R = side.R, H = p.H, D = p.D, pairs = D / 2, tid = threadIdx.x;
  double* const G = any_smem;
  float *const a = reinterpret_cast<float*>(G + R * R), *const b = a + R * H, *const da = b + R * D, *const e = da + R * H;
  float *const s = e + R * D, *const w = s + H, *const M = w + H;
  const int64_t tokens = (int64_t)p.B * p.l;
  float d_weight = 0.f;
  for (int64_t token = blockIdx.x; token < tokens; token += gridDim.x) {
    const int bi = (int)(token / p.l), i = (int)(token - (int64_t)bi * p.l);
    any_load<T>(a, side.a, bi, i, R, H);
    any_load<T>(b, side.b, bi, i, R, D);
    any_load<T>(da, side.da_out, bi, i, R, H);
    const T* const db = static_cast<const T*>(side.db_out.ptr) + bi * side.db_out.stride_b + i * side.db_out.stride_l;
    for (int x = tid; x < R * pairs; x += kAnyThreads) {
      const int r = x / pairs, j = x - r * pairs;
      const float2 t = turn_of(p.rot, token, i, j, pairs);
      const float y0 = load_as_f32(db + r * side.db_out.stride_r + 2 * j), y1 = load_as_f32(db + r * side.db_out.stride_r + 2 * j + 1);
      e[r * D + 2 * j] = y0 * t.x + y1 * t.y;
      e[r * D + 2 * j + 1] = y1 * t.x - y0 * t.y;
    }
    __syncthreads();
    any_norms(a, b, G, s, R, H, D, p.normalize, p.eps);
    T* const oa = static_cast<T*>(const_cast<void*>(side.da.ptr)) + bi * side.da.stride_b + i * side.da.stride_l;
    T* const ob = static_cast<T*>(const_cast<void*>(side.db.ptr)) + bi * side.db.stride_b + i * side.db.stride_l;
    for (int h = tid; h < H; h += kAnyThreads) {
      float u = 0.f;
      for (int r = 0; r < R; ++r) u += da[r * H + h] * a[r * H + h];
      w[h] = p.normalize ? -s[h] * s[h] * s[h] * u / ((float)D * R * R) : 0.f;
      for (int r = 0; r < R; ++r) {
        double y = 0;
        if (p.normalize)
          for (int t = 0; t < R; ++t) y += G[r * R + t] * (double)a[t * H + h];
        store_from_f32(oa + r * side.da.stride_r + h, p.normalize ? da[r * H + h] * s[h] + w[h] * (float)y : da[r * H + h]);
      }
    }
    __syncthreads();
    if (p.normalize) {
      for (int x = tid; x < R * R; x += kAnyThreads) {
        const int r = x / R, t = x - r * R;
        float sum = 0.f;
        for (int h = 0; h < H; ++h) sum += w[h] * a[r * H + h] * a[t * H + h];
        M[x] = sum;
      }
      __syncthreads();
    }
    for (int x = tid; x < R * D; x += kAnyThreads) {
      const int r = x / D, d = x - r * D;
      float sum = e[x] * weight_at(side.weight, p.weight_bf16, d);
      if (p.normalize)
        for (int t = 0; t < R; ++t) sum += M[r * R + t] * b[t * D + d];
      store_from_f32(ob + r * side.db.stride_r + d, sum);
    }
    if (side.d_weight && tid < D)
      for (int r = 0; r < R; ++r) d_weight += e[r * D + tid] * b[r * D + tid];
    __syncthreads();
  }
  if (side.d_weight && tid < D) p.partial[((int64_t)blockIdx.y * kPartials + blockIdx.x) * D + tid] = d_weight;
}

// The partial sums of a weight's gradient, in the order of their numbers: 32 columns a workgroup, each summed by 32 threads
struct SumParams {
  const float* partial;
  void* out[2];
  int count[2];
  int D, bf16;
};
__global__ __launch_bounds__(1024) void sum_partials_kernel(SumParams p) {
  __shared__ float red[32][33];
  const int which = blockIdx.y, col = threadIdx.x & 31, part = threadIdx.x >> 5, d = blockIdx.x * 32 + col;
  if (!p.out[which]) return;
  float sum = 0.f;
  if (d < p.D)
    for (int i = part; i < p.count[which]; i += 32) sum += p.partial[((int64_t)which * kPartials + i) * p.D + d];
  red[part][col] = sum;
  __syncthreads();
  if (part == 0 && d < p.D) {
    for (int i = 1; i < 32; ++i) sum += red[i][col];
    if (p.bf16) store_from_f32(static_cast<uint16_t*>(p.out[which]) + d, sum);
    else static_cast<float*>(p.out[which])[d] = sum;
  }
}

// ---------------------------------------------------------------------------------------------- checks
constexpr size_t kMostLds = 160 * 1024;
int check_sizes(int B, int l, int H, int D, int rq, int rk, int rope_len, int dtype, int weight_dtype, int kernel, int n_axes, const int32_t* sections) {
  if (dtype != TPA_DTYPE_F32 && dtype != TPA_DTYPE_BF16) return TPA_ERR_DTYPE;
  if (weight_dtype != TPA_DTYPE_F32 && weight_dtype != TPA_DTYPE_BF16) return TPA_ERR_DTYPE;
  if (B <= 0 || l <= 0 || H <= 0 || D <= 0 || D > 256 || D % 2 || rq <= 0 || rk <= 0 || rope_len <= 0) return TPA_ERR_SHAPE;
  if ((int64_t)B * l > INT32_MAX) return TPA_ERR_SHAPE;
  if (n_axes < 1 || n_axes > 4) return TPA_ERR_SHAPE;
  int64_t sum = 0;
  for (int i = 0; i < n_axes; ++i) {
    if (sections[i] < 0) return TPA_ERR_SHAPE;
    sum += sections[i];
  }
  if (sum > D / 2) return TPA_ERR_SHAPE;
  if (kernel != TPA_KERNEL_AUTO && kernel != TPA_KERNEL_GENERIC && kernel != TPA_KERNEL_MFMA) return TPA_ERR_UNSUPPORTED;
  return TPA_OK;
}
Rotation rotation_of(const float* cos, const float* sin, const int32_t* positions, int n_axes, const int32_t* sections, int rope_len) {
  Rotation r{};
  r.cos = cos; r.sin = sin; r.positions = positions; r.n_axes = n_axes; r.rope_len = rope_len;
  int last = 0;
  for (int i = 0; i < 4; ++i) r.last_of[i] = last += i < n_axes ? sections[i] : 0;
  return r;
}
template <typename K, typename P>
int launch_any(K kern, dim3 grid, size_t lds, bool (&done)[kMaxDevices], hipStream_t s, const P& p) {
  if (lds > 64 * 1024)
    if (const int rc = raise_lds_limit(done, reinterpret_cast<const void*>(kern), kMostLds); rc != TPA_OK) return rc;
  hipLaunchKernelGGL(kern, grid, dim3(kAnyThreads), lds, s, p);
  return hipGetLastError() == hipSuccess ? TPA_OK : TPA_ERR_LAUNCH;
}

}  // namespace
}  // namespace tpa

extern "C" int tpa_norm_rope(const TpaNormRopeArgs* a, void* stream) {
  using namespace tpa;
  if (!a) return TPA_ERR_NULL;
  if (const int rc = check_sizes(a->B, a->l, a->H, a->D, a->rq, a->rk, a->rope_len, a->dtype, a->weight_dtype, a->kernel, a->n_axes, a->sections); rc != TPA_OK) return rc;
  const TpaFactor* fs[12] = {&a->qa, &a->qb, &a->ka, &a->kb, &a->qa_out, &a->qb_out, &a->ka_out, &a->kb_out, &a->va, &a->vb, &a->va_out, &a->vb_out};
  for (int i = 0; i < (a->slots ? 12 : 8); ++i)
    if (!fs[i]->ptr) return TPA_ERR_NULL;
  if (!a->rope_cos || !a->rope_sin) return TPA_ERR_NULL;
  if (a->slots && (a->page_size <= 0 || a->num_slots <= 0 || a->num_slots % a->page_size)) return TPA_ERR_SHAPE;
  NormRopeParams p{};
  p.side[0] = {a->qa, a->qb, a->qa_out, a->qb_out, a->q_weight, a->rq};
  p.side[1] = {a->ka, a->kb, a->ka_out, a->kb_out, a->k_weight, a->rk};
  p.va = a->va; p.vb = a->vb; p.va_out = a->va_out; p.vb_out = a->vb_out;
  p.slots = a->slots; p.page_size = a->page_size; p.num_slots = a->num_slots;
  p.rot = rotation_of(a->rope_cos, a->rope_sin, a->positions, a->n_axes, a->sections, a->rope_len);
  p.B = a->B; p.l = a->l; p.H = a->H; p.D = a->D;
  p.weight_bf16 = a->weight_dtype == TPA_DTYPE_BF16; p.normalize = a->normalize != 0; p.eps = a->eps;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a->kernel == TPA_KERNEL_MFMA) return TPA_ERR_UNSUPPORTED;
  const size_t lds = any_lds(a->rq > a->rk ? a->rq : a->rk, a->H, a->D, false);
  if (lds > kMostLds) return TPA_ERR_SHAPE;
  const int64_t tokens = (int64_t)a->B * a->l;
  const dim3 grid((unsigned)(tokens < 4096 ? tokens : 4096), a->slots ? 3 : 2);
  static bool done[2][kMaxDevices] = {};
  if (a->dtype == TPA_DTYPE_BF16) return launch_any(norm_rope_any_kernel<uint16_t>, grid, lds, done[0], s, p);
  return launch_any(norm_rope_any_kernel<float>, grid, lds, done[1], s, p);
}

extern "C" size_t tpa_norm_rope_bwd_workspace_bytes(int32_t B, int32_t l, int32_t D) {
  if (B <= 0 || l <= 0 || D <= 0) return 0;
  return (size_t)2 * tpa::kPartials * D * sizeof(float);
}

extern "C" int tpa_norm_rope_bwd(const TpaNormRopeBwdArgs* a, void* stream) {
  using namespace tpa;
  if (!a) return TPA_ERR_NULL;
  if (const int rc = check_sizes(a->B, a->l, a->H, a->D, a->rq, a->rk, a->rope_len, a->dtype, a->weight_dtype, a->kernel, a->n_axes, a->sections); rc != TPA_OK) return rc;
  const TpaFactor* fs[2][6] = {{&a->qa, &a->qb, &a->dqa_out, &a->dqb_out, &a->dqa, &a->dqb}, {&a->ka, &a->kb, &a->dka_out, &a->dkb_out, &a->dka, &a->dkb}};
  for (auto& side : fs)
    for (const TpaFactor* f : side)
      if (side[2]->ptr && !f->ptr) return TPA_ERR_NULL;
  if (!a->rope_cos || !a->rope_sin) return TPA_ERR_NULL;
  NormRopeBwdParams p{};
  p.side[0] = {a->qa, a->qb, a->dqa_out, a->dqb_out, a->dqa, a->dqb, a->q_weight, a->dqa_out.ptr ? a->dq_weight : nullptr, a->rq};
  p.side[1] = {a->ka, a->kb, a->dka_out, a->dkb_out, a->dka, a->dkb, a->k_weight, a->dka_out.ptr ? a->dk_weight : nullptr, a->rk};
  const bool sums = p.side[0].d_weight || p.side[1].d_weight;
  if (sums && (!a->workspace || a->workspace_bytes < tpa_norm_rope_bwd_workspace_bytes(a->B, a->l, a->D))) return TPA_ERR_WORKSPACE;
  if (sums && (reinterpret_cast<uintptr_t>(a->workspace) & 15)) return TPA_ERR_ALIGN;
  p.rot = rotation_of(a->rope_cos, a->rope_sin, a->positions, a->n_axes, a->sections, a->rope_len);
  p.B = a->B; p.l = a->l; p.H = a->H; p.D = a->D;
  p.weight_bf16 = a->weight_dtype == TPA_DTYPE_BF16; p.normalize = a->normalize != 0; p.eps = a->eps;
  p.partial = static_cast<float*>(a->workspace);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a->kernel == TPA_KERNEL_MFMA) return TPA_ERR_UNSUPPORTED;
  const size_t lds = any_lds(a->rq > a->rk ? a->rq : a->rk, a->H, a->D, true);
  if (lds > kMostLds) return TPA_ERR_SHAPE;
  const int64_t tokens = (int64_t)a->B * a->l;
  const int groups = (int)(tokens < kPartials ? tokens : kPartials);
  SumParams sum{p.partial, {p.side[0].d_weight, p.side[1].d_weight}, {groups, groups}, a->D, p.weight_bf16};
  static bool done[2][kMaxDevices] = {};
  const int rc = a->dtype == TPA_DTYPE_BF16 ? launch_any(norm_rope_bwd_any_kernel<uint16_t>, dim3(groups, 2), lds, done[0], s, p)
                                            : launch_any(norm_rope_bwd_any_kernel<float>, dim3(groups, 2), lds, done[1], s, p);
  if (rc != TPA_OK || !sums) return rc;
  hipLaunchKernelGGL(sum_partials_kernel, dim3((a->D + 31) / 32, 2), dim3(1024), 0, s, sum);
  return hipGetLastError() == hipSuccess ? TPA_OK : TPA_ERR_LAUNCH;
}
