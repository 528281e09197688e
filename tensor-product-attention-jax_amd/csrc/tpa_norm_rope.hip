// Norms of queries and keys for each head and the rotation by position, on the rank factors, and their gradients.
//
// X_h = (1/R) sum_r a_r[h] b_r is never formed.  Its norm needs the R x R products G of the token's b rows only:
// |X_h|^2 = (1/R^2) a_h^T G a_h; the norm of a head is a factor of its a's, the weight and the rotation act on the b rows, so the
// result has the form that it came in, a cache of it stays factored, and a token costs its factors read once and written once.
// The gradient of |X_h|^2 is of the same kind: G a_h for the a's, and an R x R mixture of the b rows.
//
// G has signs, so |X_h|^2 may be far below the sum of its terms' sizes where ranks cancel.  It is summed in fp32 for bf16 factors,
// whose products are exact there, and in 64 bits for fp32 factors.
#include <algorithm>
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

// ---------------------------------------------------------------------------------------------- matrix cores
// A wave takes the rank rows of as many tokens of one side as fit the 16 rows of a matrix instruction, RM to a token: lane (i, g) holds
// row i's elements 32 s + 8 g + 0..7 of every chunk s, 16 bytes a load.  That is at once the layout of both operands of G = B B^T
// (no exchange between lanes) and whole pairs for the rotation.  A head's norm is a lane's: G through LDS, R^2 products.
// HBM bounds it: a token's factors come once and go once.
typedef __attribute__((ext_vector_type(4))) double f64x4;
constexpr int kNormWaves = 4;

template <typename T>
struct Chunk {  // eight elements as loaded
  u32x4 x[sizeof(T) / 2];
  __device__ __forceinline__ float operator[](int e) const {
    if constexpr (sizeof(T) == 2) return e & 1 ? bf16hi_to_f32(x[0][e / 2]) : bf16lo_to_f32(x[0][e / 2]);
    else return __uint_as_float(x[e / 4][e % 4]);
  }
};
template <typename T>
__device__ __forceinline__ Chunk<T> load_chunk(const T* from) {
  Chunk<T> c;
#pragma unroll
  for (int n = 0; n < (int)sizeof(T) / 2; ++n) c.x[n] = reinterpret_cast<const u32x4*>(from)[n];
  return c;
}
template <typename T>
__device__ __forceinline__ void store_chunk(T* to, const float (&y)[8]) {
  if constexpr (sizeof(T) == 2) {
    *reinterpret_cast<u32x4*>(to) = u32x4{pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]), pack_bf16(y[4], y[5]), pack_bf16(y[6], y[7])};
  } else {
    *reinterpret_cast<f32x4*>(to) = f32x4{y[0], y[1], y[2], y[3]};
    *reinterpret_cast<f32x4*>(to + 4) = f32x4{y[4], y[5], y[6], y[7]};
  }
}
// VH neighbouring head factors
template <typename T, int VH>
__device__ __forceinline__ void load_heads(const T* from, float (&a)[VH]) {
  if constexpr (VH == 1) {
    a[0] = load_as_f32(from);
  } else if constexpr (sizeof(T) == 2) {
    const uint32_t x = *reinterpret_cast<const uint32_t*>(from);
    a[0] = bf16lo_to_f32(x); a[1] = bf16hi_to_f32(x);
  } else {
    const float2 x = *reinterpret_cast<const float2*>(from);
    a[0] = x.x; a[1] = x.y;
  }
}
template <typename T, int VH>
__device__ __forceinline__ void store_heads(T* to, const float (&a)[VH]) {
  if constexpr (VH == 1) store_from_f32(to, a[0]);
  else if constexpr (sizeof(T) == 2) *reinterpret_cast<uint32_t*>(to) = pack_bf16(a[0], a[1]);
  else *reinterpret_cast<float2*>(to) = make_float2(a[0], a[1]);
}

// what a wave's tokens are: 16 / RM of them, lane i's row is rank i % RM of token i / RM
template <int RM>
struct Rows {
  static constexpr int P = 16 / RM;
  int token, bi, i;  // of this lane's row (clamped)
  int r;
  bool there;        // the row is a rank of a token
  int first;         // token of row 0
  __device__ __forceinline__ Rows(int group, int tokens, int l, int R, int lane) {
    const int row = lane & 15, tt = row / RM;
    first = group * P;
    r = row - tt * RM;
    there = tt < P && r < R && first + tt < tokens;
    token = min(first + min(tt, P - 1), tokens - 1);
    r = min(r, R - 1);
    bi = token / l;
    i = token - bi * l;
  }
};
// the sums of G and what is made from them: 32 bits for bf16 factors, 64 for fp32
template <typename T>
using Sum = std::conditional_t<sizeof(T) == 2, float, double>;

// G of the wave's tokens, token by token in LDS: row r of token tt at (tt RM + r) RMP
template <int RM>
constexpr int kGramStride = (RM + 3) / 4 * 4;
template <typename T, int D, int RM>
__device__ __forceinline__ bool gram_to_lds(const Chunk<T> (&x)[D / 32], Sum<T>* G, int lane) {
  const int i = lane & 15, g = lane >> 4;
  bool finite = true;
  auto put = [&](int row, Sum<T> v) __attribute__((always_inline)) {
    finite = finite && __builtin_fabs(v) <= 3.4028235e38;
    if (row / RM == i / RM && i / RM < 16 / RM) G[(i / RM * RM + row % RM) * kGramStride<RM> + i % RM] = v;
  };
  if constexpr (sizeof(T) == 2) {
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < D / 32; ++s) {
      const bf16x8 f = __builtin_bit_cast(bf16x8, x[s].x[0]);
      acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f, f, acc, 0, 0, 0);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) put(4 * g + e, acc[e]);
  } else {
    f64x4 acc = {0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < D / 32; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const double f = x[s][e];
        acc = __builtin_amdgcn_mfma_f64_16x16x4f64(f, f, acc, 0, 0, 0);
      }
#pragma unroll
    for (int e = 0; e < 4; ++e) put(4 * e + g, acc[e]);
  }
  return !__any(!finite);
}
// G a of a lane's heads; a^T G a comes back
template <typename T, int RM, int VH>
__device__ __forceinline__ void times_gram(const Sum<T>* G, int tt, const float (&a)[RM][VH], Sum<T> (&y)[RM][VH], Sum<T> (&square)[VH]) {
#pragma unroll
  for (int v = 0; v < VH; ++v) square[v] = 0;
#pragma unroll
  for (int r = 0; r < RM; ++r) {
    const Sum<T>* const row = G + (tt * RM + r) * kGramStride<RM>;
#pragma unroll
    for (int v = 0; v < VH; ++v) y[r][v] = 0;
#pragma unroll
    for (int t = 0; t < RM; ++t) {
      const Sum<T> x = row[t];
#pragma unroll
      for (int v = 0; v < VH; ++v) y[r][v] += x * (Sum<T>)a[t][v];
    }
#pragma unroll
    for (int v = 0; v < VH; ++v) square[v] += (Sum<T>)a[r][v] * y[r][v];
  }
}
template <typename S>
__device__ __forceinline__ float inverse_norm_of(S square, int R, int D, float eps) {
  const float mean = (float)(square / (S)(R * R * D));
  return rsqrtf((mean < 0 ? 0 : mean) + eps);  // NaN stays NaN
}

// cos and sin of a lane's four pairs of chunk s
template <int D, bool AXES>
struct Turns {
  f32x4 c[D / 32], s[D / 32];
  __device__ __forceinline__ Turns(const Rotation& rot, int token, int i, int g) {
    int64_t row = 0;
    if constexpr (!AXES) row = row_of(rot, token, i, 0) * (D / 2);
#pragma unroll
    for (int x = 0; x < D / 32; ++x) {
      const int j = 16 * x + 4 * g;
      if constexpr (AXES) {
        int axis = 0;
#pragma unroll
        for (int a = 0; a < 3; ++a) axis += j >= rot.last_of[a];
        row = row_of(rot, token, i, min(axis, rot.n_axes - 1)) * (D / 2);
      }
      c[x] = *reinterpret_cast<const f32x4*>(rot.cos + row + j);
      s[x] = *reinterpret_cast<const f32x4*>(rot.sin + row + j);
      if constexpr (AXES)
        if (j >= rot.last_of[3]) {
          c[x] = f32x4{1.f, 1.f, 1.f, 1.f};
          s[x] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
    }
  }
};
__device__ __forceinline__ void weights_at(const void* w, int bf16, int d, float (&out)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) out[e] = 1.f;
  if (!w) return;
  if (bf16) {
    const Chunk<uint16_t> c = load_chunk(static_cast<const uint16_t*>(w) + d);
#pragma unroll
    for (int e = 0; e < 8; ++e) out[e] = c[e];
  } else {
    const Chunk<float> c = load_chunk(static_cast<const float*>(w) + d);
#pragma unroll
    for (int e = 0; e < 8; ++e) out[e] = c[e];
  }
}
__device__ __forceinline__ void wave_lds_fence() {  // the wave's own writes have landed
  __builtin_amdgcn_s_waitcnt(0xc07f);
  __builtin_amdgcn_wave_barrier();
}

// calls f with the rows to a token that a rank of R takes
template <typename F>
__device__ __forceinline__ void with_rows(int R, F f) {
  if (R == 1) f(std::integral_constant<int, 1>{});
  else if (R == 2) f(std::integral_constant<int, 2>{});
  else if (R <= 4) f(std::integral_constant<int, 4>{});
  else if (R <= 6) f(std::integral_constant<int, 6>{});
  else if (R <= 8) f(std::integral_constant<int, 8>{});
  else f(std::integral_constant<int, 16>{});
}
__host__ __device__ inline int tokens_per_wave(int R) { return R == 1 ? 16 : R == 2 ? 8 : R <= 4 ? 4 : R <= 8 ? 2 : 1; }

constexpr int kGramElements = 16 * 16;  // of G of a wave's tokens, at most

// the place that a token's K and V factors go to: page and token in it, or the token's own
__device__ __forceinline__ bool place_of(const NormRopeParams& p, bool cached, int token, int bi, int i, int64_t& page, int64_t& at) {
  page = bi;
  at = i;
  if (!cached) return true;
  const int slot = p.slots[token];
  if (slot < 0 || slot >= p.num_slots) return false;
  page = slot / p.page_size;
  at = slot - page * p.page_size;
  return true;
}

template <typename T, int D, bool AXES, int RM>
__device__ __forceinline__ void norm_rope_rows(const NormRopeParams& p, const Side& side, bool cached, int group, int tokens, Sum<T>* G) {
  constexpr int P = 16 / RM, NS = D / 32;
  const int lane = threadIdx.x & 63, g = lane >> 4, R = side.R, H = p.H;
  const Rows<RM> me(group, tokens, p.l, R, lane);
  const T* const b = static_cast<const T*>(side.b.ptr) + me.bi * side.b.stride_b + me.i * side.b.stride_l + me.r * side.b.stride_r + 8 * g;
  Chunk<T> x[NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) x[s] = me.there ? load_chunk(b + 32 * s) : Chunk<T>{};
  const Turns<D, AXES> turn(p.rot, me.token, me.i, g);
  int64_t page, at;
  const bool stored = place_of(p, cached, me.token, me.bi, me.i, page, at) && me.there;
  if (p.normalize) {
    gram_to_lds<T, D, RM>(x, G, lane);
    wave_lds_fence();
  }
  // the b rows: weight, rotation
  T* const bo = static_cast<T*>(const_cast<void*>(side.b_out.ptr)) + page * side.b_out.stride_b + at * side.b_out.stride_l + me.r * side.b_out.stride_r + 8 * g;
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    float wt[8], y[8];
    weights_at(side.weight, p.weight_bf16, 32 * s + 8 * g, wt);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float y0 = x[s][2 * e] * wt[2 * e], y1 = x[s][2 * e + 1] * wt[2 * e + 1];
      y[2 * e] = y0 * turn.c[s][e] - y1 * turn.s[s][e];
      y[2 * e + 1] = y1 * turn.c[s][e] + y0 * turn.s[s][e];
    }
    if (stored) store_chunk(bo + 32 * s, y);
  }
  // the head factors
  auto heads = [&](auto vh_c) __attribute__((always_inline)) {
    constexpr int VH = decltype(vh_c)::value;
    for (int at_head = VH * lane; at_head < P * H; at_head += VH * 64) {
      const int tt = at_head / H, h = at_head - tt * H, token = me.first + tt;
      if (token >= tokens) continue;
      const int bi = token / p.l, i = token - bi * p.l;
      int64_t page, at;
      if (!place_of(p, cached, token, bi, i, page, at)) continue;
      const T* const from = static_cast<const T*>(side.a.ptr) + bi * side.a.stride_b + i * side.a.stride_l + h;
      T* const to = static_cast<T*>(const_cast<void*>(side.a_out.ptr)) + page * side.a_out.stride_b + at * side.a_out.stride_l + h;
      float a[RM][VH];
#pragma unroll
      for (int r = 0; r < RM; ++r) {
        if (r < R) load_heads<T, VH>(from + r * side.a.stride_r, a[r]);
        else
#pragma unroll
          for (int v = 0; v < VH; ++v) a[r][v] = 0.f;
      }
      float scale[VH];
#pragma unroll
      for (int v = 0; v < VH; ++v) scale[v] = 1.f;
      if (p.normalize) {
        Sum<T> y[RM][VH], square[VH];
        times_gram<T, RM, VH>(G, tt, a, y, square);
#pragma unroll
        for (int v = 0; v < VH; ++v) scale[v] = inverse_norm_of(square[v], R, D, p.eps);
      }
#pragma unroll
      for (int r = 0; r < RM; ++r) {
        float out[VH];
#pragma unroll
        for (int v = 0; v < VH; ++v) out[v] = a[r][v] * scale[v];
        if (r < R) store_heads<T, VH>(to + r * side.a_out.stride_r, out);
      }
    }
  };
  if (P * H <= 64) heads(std::integral_constant<int, 1>{});
  else heads(std::integral_constant<int, 2>{});
}

template <typename T, int D, bool AXES>
__global__ __launch_bounds__(kNormWaves * 64) void norm_rope_kernel(NormRopeParams p, int groups_q, int groups_k, int groups_v) {
  __shared__ Sum<T> gram[kNormWaves][kGramElements];
  const int w = scalar(threadIdx.x >> 6), tokens = p.B * p.l;
  int task = blockIdx.x * kNormWaves + w;
  if (task < groups_q + groups_k) {
    const bool keys = task >= groups_q;
    const Side& side = p.side[keys];
    with_rows(side.R, [&](auto rm) __attribute__((always_inline)) {
      norm_rope_rows<T, D, AXES, decltype(rm)::value>(p, side, keys && p.slots, keys ? task - groups_q : task, tokens, gram[w]);
    });
    return;
  }
  task -= groups_q + groups_k;
  if (task >= groups_v) return;
  // V factors into their slots, 16 bytes a lane: chunks of a row of ranks, head factors first
  constexpr int E = 16 / sizeof(T);
  const int R = p.side[1].R, lane = threadIdx.x & 63, per_rank = (p.H + D) / E, per_token = R * per_rank, P = tokens_per_wave(R);
  for (int x = lane; x < P * per_token; x += 64) {
    const int tt = x / per_token, token = task * P + tt, rest = x - tt * per_token, r = rest / per_rank, c = (rest - r * per_rank) * E;
    if (token >= tokens) break;
    const int bi = token / p.l, i = token - bi * p.l;
    int64_t page, at;
    if (!place_of(p, true, token, bi, i, page, at)) continue;
    const bool head = c < p.H;
    const TpaFactor &in = head ? p.va : p.vb, &out = head ? p.va_out : p.vb_out;
    const int col = head ? c : c - p.H;
    *reinterpret_cast<u32x4*>(static_cast<T*>(const_cast<void*>(out.ptr)) + page * out.stride_b + at * out.stride_l + r * out.stride_r + col) =
        *reinterpret_cast<const u32x4*>(static_cast<const T*>(in.ptr) + bi * in.stride_b + i * in.stride_l + r * in.stride_r + col);
  }
}

// ---- gradients.  The R x R sums M = A diag(w) A^T over the heads and the mixture M B of the b rows are products of the matrix cores
// too: M's result layout is that of the second product's operand, whose other one are the b rows read back transposed.  For bf16
// factors w a and M are kept as two bf16 numbers each.  The rows of a wave's tokens stand in one product, so the rows of the other
// tokens meet zeros: where a b row is not finite, 0 * inf would spread, and the tokens take turns instead.
template <typename T, int D>
struct BwdLds {
  static constexpr int kStride = sizeof(T) == 2 ? D : D + 4;              // of a b row (elements)
  static constexpr size_t kRows = 16 * kStride * sizeof(T), kGram = kGramElements * sizeof(Sum<T>);
  static size_t bytes(int most_pairs) { return kNormWaves * (kRows + kGram + (size_t)(most_pairs + 3) / 4 * 16); }
};

template <typename T, int D, bool AXES, int RM>
__device__ __forceinline__ void norm_rope_bwd_rows(const NormRopeBwdParams& p, const BwdSide& side, int group, int tokens, unsigned char* lds, float (&d_weight)[D / 4]) {
  constexpr int P = 16 / RM, NS = D / 32;
  using Lds = BwdLds<T, D>;
  T* const rows = reinterpret_cast<T*>(lds);
  Sum<T>* const G = reinterpret_cast<Sum<T>*>(lds + Lds::kRows);
  float* const W = reinterpret_cast<float*>(lds + Lds::kRows + Lds::kGram);  // [P][H]
  const int lane = threadIdx.x & 63, row = lane & 15, g = lane >> 4, R = side.R, H = p.H;
  const Rows<RM> me(group, tokens, p.l, R, lane);
  const T* const b = static_cast<const T*>(side.b.ptr) + me.bi * side.b.stride_b + me.i * side.b.stride_l + me.r * side.b.stride_r + 8 * g;
  const T* const db = static_cast<const T*>(side.db_out.ptr) + me.bi * side.db_out.stride_b + me.i * side.db_out.stride_l + me.r * side.db_out.stride_r + 8 * g;
  Chunk<T> x[NS], dy[NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    x[s] = me.there ? load_chunk(b + 32 * s) : Chunk<T>{};
    dy[s] = me.there ? load_chunk(db + 32 * s) : Chunk<T>{};
  }
  const Turns<D, AXES> turn(p.rot, me.token, me.i, g);
  bool finite = true;
  if (p.normalize) {
    finite = gram_to_lds<T, D, RM>(x, G, lane);
    if (finite)
#pragma unroll
      for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int n = 0; n < (int)sizeof(T) / 2; ++n) reinterpret_cast<u32x4*>(rows + row * Lds::kStride + 32 * s + 8 * g)[n] = x[s].x[n];
    wave_lds_fence();
  }
  // head factors: a lane's heads
  auto heads = [&](auto vh_c) __attribute__((always_inline)) {
    constexpr int VH = decltype(vh_c)::value;
    for (int at_head = VH * lane; at_head < P * H; at_head += VH * 64) {
      const int tt = at_head / H, h = at_head - tt * H, token = me.first + tt;
      float w[VH];
      if (token < tokens) {
        const int bi = token / p.l, i = token - bi * p.l;
        const T* const from = static_cast<const T*>(side.a.ptr) + bi * side.a.stride_b + i * side.a.stride_l + h;
        const T* const d_from = static_cast<const T*>(side.da_out.ptr) + bi * side.da_out.stride_b + i * side.da_out.stride_l + h;
        T* const to = static_cast<T*>(const_cast<void*>(side.da.ptr)) + bi * side.da.stride_b + i * side.da.stride_l + h;
        float a[RM][VH], da[RM][VH];
#pragma unroll
        for (int r = 0; r < RM; ++r) {
          if (r < R) {
            load_heads<T, VH>(from + r * side.a.stride_r, a[r]);
            load_heads<T, VH>(d_from + r * side.da_out.stride_r, da[r]);
          } else {
#pragma unroll
            for (int v = 0; v < VH; ++v) a[r][v] = da[r][v] = 0.f;
          }
        }
        if (p.normalize) {
          Sum<T> y[RM][VH], square[VH];
          times_gram<T, RM, VH>(G, tt, a, y, square);
#pragma unroll
          for (int v = 0; v < VH; ++v) {
            const float scale = inverse_norm_of(square[v], R, D, p.eps);
            float u = 0.f;
#pragma unroll
            for (int r = 0; r < RM; ++r) u = fmaf(da[r][v], a[r][v], u);
            w[v] = -scale * scale * scale * u / (float)(D * R * R);
#pragma unroll
            for (int r = 0; r < RM; ++r) da[r][v] = da[r][v] * scale + w[v] * (float)y[r][v];
          }
        }
#pragma unroll
        for (int r = 0; r < RM; ++r)
          if (r < R) store_heads<T, VH>(to + r * side.da.stride_r, da[r]);
      } else {
#pragma unroll
        for (int v = 0; v < VH; ++v) w[v] = 0.f;
      }
      if (p.normalize)
#pragma unroll
        for (int v = 0; v < VH; ++v) W[at_head + v] = w[v];
    }
  };
  if (P * H <= 64) heads(std::integral_constant<int, 1>{});
  else heads(std::integral_constant<int, 2>{});
  // M[4 g + e][row] of the token's rows
  f32x4 M = {0.f, 0.f, 0.f, 0.f};
  if (p.normalize) {
    wave_lds_fence();
    const T* const a = static_cast<const T*>(side.a.ptr) + me.bi * side.a.stride_b + me.i * side.a.stride_l + me.r * side.a.stride_r;
    const float* const w_of = W + min(row / RM, P - 1) * H;
    if constexpr (sizeof(T) == 2) {
      for (int h = 8 * g; h - 8 * g < H; h += 32) {
        const bool there = me.there && h < H;
        const Chunk<T> ac = there ? load_chunk(a + h) : Chunk<T>{};
        u32x4 hi, lo;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float w0 = there ? ac[2 * e] * w_of[h + 2 * e] : 0.f, w1 = there ? ac[2 * e + 1] * w_of[h + 2 * e + 1] : 0.f;
          hi[e] = pack_bf16(w0, w1);
          lo[e] = pack_bf16(w0 - bf16lo_to_f32(hi[e]), w1 - bf16hi_to_f32(hi[e]));
        }
        const bf16x8 f = __builtin_bit_cast(bf16x8, ac.x[0]);
        M = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f, __builtin_bit_cast(bf16x8, lo), M, 0, 0, 0);
        M = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f, __builtin_bit_cast(bf16x8, hi), M, 0, 0, 0);
      }
    } else {
      for (int h = 8 * g; h - 8 * g < H; h += 32) {
        const bool there = me.there && h < H;
        const Chunk<T> ac = there ? load_chunk(a + h) : Chunk<T>{};
#pragma unroll
        for (int e = 0; e < 8; ++e) M = __builtin_amdgcn_mfma_f32_16x16x4f32(ac[e], there ? ac[e] * w_of[h + e] : 0.f, M, 0, 0, 0);
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if ((4 * g + e) / RM != row / RM || row / RM >= P) M[e] = 0.f;
  }
  // mixture of the b rows: out[n][e] of this lane's row at d = 32 (n / 2) + 8 g + 4 (n % 2) + e
  f32x4 mixed[2 * NS];
#pragma unroll
  for (int n = 0; n < 2 * NS; ++n) mixed[n] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto mix = [&](f32x4 (&out)[2 * NS]) __attribute__((always_inline)) {
    if constexpr (sizeof(T) == 2) {
      const u32x2 hi = {pack_bf16(M[0], M[1]), pack_bf16(M[2], M[3])};
      const u32x2 lo = {pack_bf16(M[0] - bf16lo_to_f32(hi[0]), M[1] - bf16hi_to_f32(hi[0])), pack_bf16(M[2] - bf16lo_to_f32(hi[1]), M[3] - bf16hi_to_f32(hi[1]))};
#pragma unroll
      for (int n = 0; n < 2 * NS; ++n) {
        // rows 4 g + 0..3 of the column that this lane stands for: 16 lanes bring 4 rows x 16 columns and get them transposed
        const T* const from = rows + (4 * g + (row >> 2)) * Lds::kStride + 32 * (n / 2) + 8 * (row & 3) + 4 * (n % 2);
        const s16x4 f = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4 __attribute__((address_space(3)))*)from);
        out[n] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(f, __builtin_bit_cast(s16x4, lo), out[n], 0, 0, 0);
        out[n] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(f, __builtin_bit_cast(s16x4, hi), out[n], 0, 0, 0);
      }
    } else {
#pragma unroll
      for (int n = 0; n < 2 * NS; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          out[n] = __builtin_amdgcn_mfma_f32_16x16x4f32(rows[(4 * g + e) * Lds::kStride + 32 * (n / 2) + 8 * (row >> 2) + 4 * (n % 2) + (row & 3)], M[e], out[n], 0, 0, 0);
    }
  };
  if (p.normalize) {
    if (finite) {
      mix(mixed);
    } else {
      for (int tt = 0; tt < P; ++tt) {
        wave_lds_fence();
        const bool mine = row / RM == tt;
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
          for (int n = 0; n < (int)sizeof(T) / 2; ++n)
            reinterpret_cast<u32x4*>(rows + row * Lds::kStride + 32 * s + 8 * g)[n] = mine ? x[s].x[n] : u32x4{0, 0, 0, 0};
        wave_lds_fence();
        f32x4 one[2 * NS];
#pragma unroll
        for (int n = 0; n < 2 * NS; ++n) one[n] = f32x4{0.f, 0.f, 0.f, 0.f};
        mix(one);
#pragma unroll
        for (int n = 0; n < 2 * NS; ++n) mixed[n] = mine ? one[n] : mixed[n];
      }
    }
  }
  T* const bo = static_cast<T*>(const_cast<void*>(side.db.ptr)) + me.bi * side.db.stride_b + me.i * side.db.stride_l + me.r * side.db.stride_r + 8 * g;
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    float wt[8], y[8];
    weights_at(side.weight, p.weight_bf16, 32 * s + 8 * g, wt);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float y0 = dy[s][2 * e], y1 = dy[s][2 * e + 1];
      const float e0 = y0 * turn.c[s][e] + y1 * turn.s[s][e], e1 = y1 * turn.c[s][e] - y0 * turn.s[s][e];
      d_weight[8 * s + 2 * e] = fmaf(e0, x[s][2 * e], d_weight[8 * s + 2 * e]);
      d_weight[8 * s + 2 * e + 1] = fmaf(e1, x[s][2 * e + 1], d_weight[8 * s + 2 * e + 1]);
      y[2 * e] = fmaf(e0, wt[2 * e], mixed[2 * s + e / 2][2 * e % 4]);
      y[2 * e + 1] = fmaf(e1, wt[2 * e + 1], mixed[2 * s + e / 2][(2 * e + 1) % 4]);
    }
    if (me.there) store_chunk(bo + 32 * s, y);
  }
  wave_lds_fence();  // the next tokens' rows go where these are
}

// Workgroups 0 .. parts_q - 1 share out the queries' tokens, the others the keys'
template <typename T, int D, bool AXES>
__global__ __launch_bounds__(kNormWaves * 64) void norm_rope_bwd_kernel(NormRopeBwdParams p, int parts_q, int parts_k, int wave_bytes) {
  extern __shared__ __attribute__((aligned(16))) unsigned char bwd_mem[];
  const int w = scalar(threadIdx.x >> 6), lane = threadIdx.x & 63, tokens = p.B * p.l;
  const bool keys = (int)blockIdx.x >= parts_q;
  const BwdSide& side = p.side[keys];
  const int part = keys ? blockIdx.x - parts_q : blockIdx.x, parts = keys ? parts_k : parts_q;
  float d_weight[D / 4];  // of this lane's row: element 8 s + e is d = 32 s + 8 g + e
#pragma unroll
  for (int x = 0; x < D / 4; ++x) d_weight[x] = 0.f;
  with_rows(side.R, [&](auto rm) __attribute__((always_inline)) {
    constexpr int RM = decltype(rm)::value, P = 16 / RM;
    for (int group = part * kNormWaves + w; group < (tokens + P - 1) / P; group += parts * kNormWaves)
      norm_rope_bwd_rows<T, D, AXES, RM>(p, side, group, tokens, bwd_mem + w * wave_bytes, d_weight);
  });
  if (!side.d_weight) return;
  // over the rows of the wave, then over the waves
#pragma unroll
  for (int x = 0; x < D / 4; ++x) {
    float v = d_weight[x];
    v += __int_as_float(lanes_of<0xB1>(__float_as_int(v)));
    v += __int_as_float(lanes_of<0x4E>(__float_as_int(v)));
    v += __int_as_float(lanes_of<0x141>(__float_as_int(v)));
    v += __int_as_float(lanes_of<0x140>(__float_as_int(v)));
    d_weight[x] = v;
  }
  __syncthreads();
  float* const sums = reinterpret_cast<float*>(bwd_mem);
  if ((lane & 15) == 0)
#pragma unroll
    for (int x = 0; x < D / 4; ++x) sums[w * D + 32 * (x / 8) + 8 * (lane >> 4) + x % 8] = d_weight[x];
  __syncthreads();
  if (threadIdx.x < D) {
    float v = 0.f;
    for (int x = 0; x < kNormWaves; ++x) v += sums[x * D + threadIdx.x];
    p.partial[((int64_t)keys * kPartials + part) * D + threadIdx.x] = v;
  }
}

// ---------------------------------------------------------------------------------------------- checks
template <typename Args>
bool fast_takes(const Args* a, const TpaFactor* const* fs, int n) {
  if (a->kernel == TPA_KERNEL_GENERIC || (a->D != 64 && a->D != 128) || a->H % 8 || a->rq > 16 || a->rk > 16) return false;
  if ((int64_t)a->B * a->l > (1 << 30)) return false;
  for (int i = 0; i < a->n_axes; ++i)
    if (a->sections[i] % 4) return false;
  const int chunk = a->dtype == TPA_DTYPE_BF16 ? 8 : 4;
  for (int i = 0; i < n; ++i) {
    const TpaFactor& f = *fs[i];
    if ((reinterpret_cast<uintptr_t>(f.ptr) & 15) || f.stride_b % chunk || f.stride_l % chunk || f.stride_r % chunk) return false;
  }
  return !((reinterpret_cast<uintptr_t>(a->rope_cos) | reinterpret_cast<uintptr_t>(a->rope_sin) | reinterpret_cast<uintptr_t>(a->q_weight) | reinterpret_cast<uintptr_t>(a->k_weight)) & 15);
}
template <typename T, int D>
int launch_fast(const NormRopeParams& p, hipStream_t s) {
  const int64_t tokens = (int64_t)p.B * p.l;
  auto groups = [&](int R) { return (int)((tokens + tokens_per_wave(R) - 1) / tokens_per_wave(R)); };
  const int q = groups(p.side[0].R), k = groups(p.side[1].R), v = p.slots ? k : 0;
  const dim3 grid((unsigned)(((int64_t)q + k + v + kNormWaves - 1) / kNormWaves));
  const bool axes = p.rot.n_axes > 1 || p.rot.last_of[3] < D / 2;
  if (axes) hipLaunchKernelGGL((norm_rope_kernel<T, D, true>), grid, dim3(kNormWaves * 64), 0, s, p, q, k, v);
  else hipLaunchKernelGGL((norm_rope_kernel<T, D, false>), grid, dim3(kNormWaves * 64), 0, s, p, q, k, v);
  return hipGetLastError() == hipSuccess ? TPA_OK : TPA_ERR_LAUNCH;
}
inline int most_pairs(int rq, int rk, int H) { return (tokens_per_wave(rq) > tokens_per_wave(rk) ? tokens_per_wave(rq) : tokens_per_wave(rk)) * H; }
template <typename T, int D>
int launch_fast_bwd(const NormRopeBwdParams& p, int (&parts)[2], hipStream_t s) {
  const int64_t tokens = (int64_t)p.B * p.l;
  for (int x = 0; x < 2; ++x) {
    const int64_t groups = (tokens + tokens_per_wave(p.side[x].R) - 1) / tokens_per_wave(p.side[x].R);
    parts[x] = p.side[x].da_out.ptr ? (int)std::min<int64_t>((groups + kNormWaves - 1) / kNormWaves, kPartials) : 0;
  }
  const size_t lds = BwdLds<T, D>::bytes(most_pairs(p.side[0].R, p.side[1].R, p.H));
  const bool axes = p.rot.n_axes > 1 || p.rot.last_of[3] < D / 2;
  const dim3 grid(parts[0] + parts[1]);
  if (axes) hipLaunchKernelGGL((norm_rope_bwd_kernel<T, D, true>), grid, dim3(kNormWaves * 64), lds, s, p, parts[0], parts[1], (int)(lds / kNormWaves));
  else hipLaunchKernelGGL((norm_rope_bwd_kernel<T, D, false>), grid, dim3(kNormWaves * 64), lds, s, p, parts[0], parts[1], (int)(lds / kNormWaves));
  return hipGetLastError() == hipSuccess ? TPA_OK : TPA_ERR_LAUNCH;
}

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
  if (fast_takes(a, fs, a->slots ? 12 : 8)) {
    if (a->dtype == TPA_DTYPE_BF16) return a->D == 128 ? launch_fast<uint16_t, 128>(p, s) : launch_fast<uint16_t, 64>(p, s);
    return a->D == 128 ? launch_fast<float, 128>(p, s) : launch_fast<float, 64>(p, s);
  }
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
  SumParams sum{p.partial, {p.side[0].d_weight, p.side[1].d_weight}, {0, 0}, a->D, p.weight_bf16};
  int rc;
  if (fast_takes(a, &fs[0][0], 12) && (a->dtype == TPA_DTYPE_BF16 ? BwdLds<uint16_t, 128>::bytes(most_pairs(a->rq, a->rk, a->H))
                                                                  : BwdLds<float, 128>::bytes(most_pairs(a->rq, a->rk, a->H))) <= 64 * 1024) {
    if (a->dtype == TPA_DTYPE_BF16) rc = a->D == 128 ? launch_fast_bwd<uint16_t, 128>(p, sum.count, s) : launch_fast_bwd<uint16_t, 64>(p, sum.count, s);
    else rc = a->D == 128 ? launch_fast_bwd<float, 128>(p, sum.count, s) : launch_fast_bwd<float, 64>(p, sum.count, s);
  } else {
    if (a->kernel == TPA_KERNEL_MFMA) return TPA_ERR_UNSUPPORTED;
    const size_t lds = any_lds(a->rq > a->rk ? a->rq : a->rk, a->H, a->D, true);
    if (lds > kMostLds) return TPA_ERR_SHAPE;
    const int64_t tokens = (int64_t)a->B * a->l;
    const int groups = sum.count[0] = sum.count[1] = (int)(tokens < kPartials ? tokens : kPartials);
    static bool done[2][kMaxDevices] = {};
    rc = a->dtype == TPA_DTYPE_BF16 ? launch_any(norm_rope_bwd_any_kernel<uint16_t>, dim3(groups, 2), lds, done[0], s, p)
                                    : launch_any(norm_rope_bwd_any_kernel<float>, dim3(groups, 2), lds, done[1], s, p);
  }
  if (rc != TPA_OK || !sums) return rc;
  hipLaunchKernelGGL(sum_partials_kernel, dim3((a->D + 31) / 32, 2), dim3(1024), 0, s, sum);
  return hipGetLastError() == hipSuccess ? TPA_OK : TPA_ERR_LAUNCH;
}
