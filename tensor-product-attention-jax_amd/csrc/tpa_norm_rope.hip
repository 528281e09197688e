// Norms of queries and keys for each head and the rotation by position, on the rank factors, and their gradients.
//
// X_h = (1/R) sum_r a_r[h] b_r is never formed.  Its norm needs the R x R products G of the token's b rows only:
// |X_h|^2 = (1/R^2) a_h^T G a_h; the norm of a head is a factor of its a's, the weight and the rotation act on the b rows, so the
// result has the form that it came in, a cache of it stays factored, and a token costs its factors read once and written once.
// The gradient of |X_h|^2 is of the same kind: G a_h for the a's, and an R x R mixture of the b rows.
//
// G has signs, so |X_h|^2 may be far below the sum of its terms' sizes where ranks cancel.  It is summed in fp32 for bf16 factors,
// whose products are exact there - heads that cancel are summed anew from X_h itself, see squares_of_vectors() - and in 64 bits for fp32
// factors.
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
constexpr size_t kMostLds = 160 * 1024;
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
      w[h] = p.normalize ? -(s[h] * u) * (s[h] / ((float)D * R * R)) * s[h] : 0.f;  // (the cube alone may pass 2^128)
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
  if (d < p.D) {
    float v[kPartials / 32];  // all of them on their way at once
#pragma unroll
    for (int x = 0; x < kPartials / 32; ++x) v[x] = part + 32 * x < p.count[which] ? p.partial[((int64_t)which * kPartials + part + 32 * x) * p.D + d] : 0.f;
#pragma unroll
    for (int x = 0; x < kPartials / 32; ++x) sum += v[x];
  }
  red[part][col] = sum;
  __syncthreads();
  if (part == 0 && d < p.D) {
    for (int i = 1; i < 32; ++i) sum += red[i][col];
    if (p.bf16) store_from_f32(static_cast<uint16_t*>(p.out[which]) + d, sum);
    else static_cast<float*>(p.out[which])[d] = sum;
  }
}

// ---------------------------------------------------------------------------------------------- matrix cores
// A wave takes the rank rows of as many tokens of one side as fit the 16 rows of a matrix instruction, a power of two to a token.  Lane (i, g)
// holds row i's elements 32 s + 8 g + 0..7 of every chunk s, 16 bytes a load: at once the layout of both operands of G = B B^T and whole
// pairs for the rotation.  G's result layout - column i, four rows - is, G being symmetric, that of an operand of the next product Y = G A, 16
// heads a time; there lane (n, g) holds four rows of head n of Y and, as the other operand, the same four of A, so that |X_h|^2 = a_h . y_h is
// a sum over a lane's registers and a few lanes.  The b rows wait in LDS, which saves their registers while the heads go by (with them the kernel
// of 16 heads of 128 takes 33 us in place of 19).  For bf16 factors G goes into that product as three bf16
// numbers, 2^-27 of it off; for fp32 factors both are products in 64 bits.
// The rows of a wave's tokens stand in one product, so a token's rows meet zeros for the other tokens'; where those are not finite, 0 * inf
// would spread, and the tokens take turns.
// HBM bounds it: a token's factors come once and go once, forward at 3.9 to 4.8 TB/s in the cases below, backward, whose chain of products is longer, at
// 3.5 to 3.6, where a copy of 1 GiB has 5.15.  (With
// G through LDS and R^2 products a head on the vector units, 310 registers and 1300 vector instructions per 16 rows, their backward
// took 66 and 256 us.)
typedef __attribute__((ext_vector_type(4))) double f64x4;
constexpr int kNormWaves = 4;
// Waves of a SIMD that the registers are kept to.  More of them hide more of the loads until they cost much scratch memory: us of the backward of
// 4 x 4096 tokens, 16 heads of 128, at 2 / 3 waves 39.0 / 34.3, of 4099 tokens, 32 heads, three axes 20.7 / 24.5; of 8 x 2048, 64 heads of 64, ranks 16
// and 8, at 2 / 3 / 4 108 / 85 / 152; forward of the last at 3 / 4 / 5 / 6 waves 42.2 / 41.5 / 63.2 / 138.  (The factors of the next tokens asked for ahead take the registers of
// a wave, which costs more than it hides.)
constexpr int fwd_waves(int size, int d) { return size == 2 ? 4 : d == 64 ? 3 : 2; }
constexpr int bwd_waves(int size, int d, int heads_of_lane) { return size == 2 && (d == 64 || heads_of_lane == 1) ? 3 : 2; }

template <typename T>
struct Chunk {  // eight elements as loaded
  u32x4 x[sizeof(T) / 2];
  __device__ __forceinline__ void keep(bool there) {  // zeros otherwise
#pragma unroll
    for (int n = 0; n < (int)sizeof(T) / 2; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) x[n][j] = there ? x[n][j] : 0u;
  }
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
// VH neighbouring head factors as loaded
template <typename T, int VH>
struct Heads {
  using Word = std::conditional_t<sizeof(T) * VH == 2, uint16_t, std::conditional_t<sizeof(T) * VH == 4, uint32_t, u32x2>>;
  Word x;
  __device__ __forceinline__ void unpack(bool there, float (&a)[VH]) const {  // zeros where they are not there
#pragma unroll
    for (int v = 0; v < VH; ++v) {
      float y;
      if constexpr (sizeof(Word) == 2) y = bf16bits_to_f32(x);
      else if constexpr (sizeof(T) == 2) y = v ? bf16hi_to_f32(x) : bf16lo_to_f32(x);
      else if constexpr (VH == 1) y = __uint_as_float(x);
      else y = __uint_as_float(x[v]);
      a[v] = there ? y : 0.f;
    }
  }
};
template <typename T, int VH>
__device__ __forceinline__ Heads<T, VH> load_heads(const T* from) {
  return {*reinterpret_cast<const typename Heads<T, VH>::Word*>(from)};
}
template <typename T, int VH>
__device__ __forceinline__ void store_heads(T* to, const float (&a)[VH]) {
  if constexpr (VH == 1) store_from_f32(to, a[0]);
  else if constexpr (sizeof(T) == 2) *reinterpret_cast<uint32_t*>(to) = pack_bf16(a[0], a[1]);
  else *reinterpret_cast<float2*>(to) = make_float2(a[0], a[1]);
}
// two where 16 lanes still take whole rows of them (four of 64 heads: backward of the second case below 157 us, two 117)
template <typename F>
void with_heads(int H, F f) {
  if (H > 16) f(std::integral_constant<int, 2>{});
  else f(std::integral_constant<int, 1>{});
}
// log2 of the rows that a token of rank R takes
__host__ __device__ inline int rows_log2(int R) { return R <= 1 ? 0 : R <= 2 ? 1 : R <= 4 ? 2 : R <= 8 ? 3 : 4; }
__host__ __device__ inline int tokens_per_wave(int R) { return 16 >> rows_log2(R); }

// sums in 32 bits for bf16 factors, in 64 for fp32
template <typename T>
struct Sums {
  using S = float;
  using V = f32x4;
  __device__ __forceinline__ static int row(int g, int j) { return 4 * g + j; }  // of a lane's result register j
};
template <>
struct Sums<float> {
  using S = double;
  using V = f64x4;
  __device__ __forceinline__ static int row(int g, int j) { return 4 * j + g; }
};

__device__ __forceinline__ float with_lane(float x, int apart) {  // x + that of the lane 16 (32) apart
  const uint32_t u = __float_as_uint(x);
  const auto r = apart == 16 ? __builtin_amdgcn_permlane16_swap(u, u, false, false) : __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ double with_lane(double x, int apart) {
  const uint64_t u = (uint64_t)__double_as_longlong(x);
  const uint32_t lo = (uint32_t)u, hi = (uint32_t)(u >> 32);
  const auto rl = apart == 16 ? __builtin_amdgcn_permlane16_swap(lo, lo, false, false) : __builtin_amdgcn_permlane32_swap(lo, lo, false, false);
  const auto rh = apart == 16 ? __builtin_amdgcn_permlane16_swap(hi, hi, false, false) : __builtin_amdgcn_permlane32_swap(hi, hi, false, false);
  return __longlong_as_double((long long)((uint64_t)rh[0] << 32 | rl[0])) + __longlong_as_double((long long)((uint64_t)rh[1] << 32 | rl[1]));
}
// four rows' terms -> for each the sum over the 2^lg rows of its token (in scalars: arrays that a lambda or a branch writes went to scratch memory)
template <typename T, typename S>
__device__ __forceinline__ void over_token(S (&v)[4], int lg) {
  S a = v[0], b = v[1], c = v[2], d = v[3];
  if constexpr (sizeof(T) == 2) {  // rows 4 g + j
    if (lg >= 1) {
      a += b; b = a;
      c += d; d = c;
    }
    if (lg >= 2) {
      a += c;
      if (lg >= 3) a = with_lane(a, 16);
      if (lg >= 4) a = with_lane(a, 32);
      b = c = d = a;
    }
  } else {  // rows 4 j + g
    if (lg >= 1) {
      a = with_lane(a, 16); b = with_lane(b, 16); c = with_lane(c, 16); d = with_lane(d, 16);
    }
    if (lg >= 2) {
      a = with_lane(a, 32); b = with_lane(b, 32); c = with_lane(c, 32); d = with_lane(d, 32);
    }
    if (lg >= 3) {
      a += b; b = a;
      c += d; d = c;
    }
    if (lg >= 4) {
      a += c;
      b = c = d = a;
    }
  }
  v[0] = a; v[1] = b; v[2] = c; v[3] = d;
}
template <typename S>
__device__ __forceinline__ float inverse_norm_of(S square, S inv, float eps) {  // inv = 1 / (R R D)
  const float mean = (float)(square * inv);
  return __builtin_amdgcn_rsqf((mean < 0 ? 0 : mean) + eps);  // one unit in the last place; NaN stays NaN
}
// for four rows; rows of one token have one
template <typename T, typename S>
__device__ __forceinline__ void inverse_norms(const S (&square)[4], S inv, float eps, int lg, float (&scale)[4]) {
  const float a = inverse_norm_of(square[0], inv, eps);
  float b = a, c = a, d = a;
  if (lg < (sizeof(T) == 2 ? 2 : 4)) {
    b = inverse_norm_of(square[1], inv, eps);
    c = inverse_norm_of(square[2], inv, eps);
    d = inverse_norm_of(square[3], inv, eps);
  }
  scale[0] = a; scale[1] = b; scale[2] = c; scale[3] = d;
}

// positions by which a lane's pairs turn: asked for first, since the rows of cos and sin wait for them
template <int D, bool AXES>
struct TurnAt {
  int row[AXES ? D / 32 : 1];
  __device__ __forceinline__ TurnAt(const Rotation& rot, int token, int i, int g) {
    if constexpr (!AXES) {
      row[0] = (int)row_of(rot, token, i, 0);
    } else {
#pragma unroll
      for (int x = 0; x < D / 32; ++x) {
        int axis = 0;
#pragma unroll
        for (int a = 0; a < 3; ++a) axis += 16 * x + 4 * g >= rot.last_of[a];
        row[x] = (int)row_of(rot, token, i, min(axis, rot.n_axes - 1));
      }
    }
  }
};
// cos and sin of a lane's four pairs of chunk s
template <int D, bool AXES>
struct Turns {
  f32x4 c[D / 32], s[D / 32];
  __device__ __forceinline__ Turns(const Rotation& rot, const TurnAt<D, AXES>& at, int g) {
#pragma unroll
    for (int x = 0; x < D / 32; ++x) {
      const int j = 16 * x + 4 * g;
      const int64_t row = (int64_t)at.row[AXES ? x : 0] * (D / 2);
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
// a side's weights as fp32 in LDS, by the whole workgroup
template <int D>
__device__ __forceinline__ void weights_to_lds(const void* from, int bf16, float* to) {
  if (threadIdx.x < D) to[threadIdx.x] = weight_at(from, bf16, threadIdx.x);
  __syncthreads();
}
__device__ __forceinline__ void wave_lds_fence() {  // the wave's own writes have landed
  __builtin_amdgcn_s_waitcnt(0xc07f);
  __builtin_amdgcn_wave_barrier();
}

// A wave's tokens are of one batch entry: what its lanes add to the entry's base fits 32 bits
template <typename T>
__device__ __forceinline__ T* base_of(const TpaFactor& f, int bi, int first) {
  return static_cast<T*>(const_cast<void*>(f.ptr)) + bi * f.stride_b + first * f.stride_l;
}
__device__ __forceinline__ uint32_t offset_of(const TpaFactor& f, int tt, int r) { return (uint32_t)(tt * (int)f.stride_l + r * (int)f.stride_r); }
// page and place of a token's slot
__device__ __forceinline__ bool slot_of(const NormRopeParams& p, int bi, int i, int64_t& page, int64_t& at) {
  const int slot = p.slots[bi * p.l + i];
  page = slot / p.page_size;
  at = slot - page * p.page_size;
  return slot >= 0 && slot < p.num_slots;
}

// G of the wave's rows, the other tokens' columns zero; `finite`: whether all of its numbers are
template <typename T, int D>
__device__ __forceinline__ typename Sums<T>::V gram(const Chunk<T> (&x)[D / 32], int row, int g, int lg, bool& finite) {
  typename Sums<T>::V G = {0, 0, 0, 0};
#pragma unroll
  for (int s = 0; s < D / 32; ++s) {
    if constexpr (sizeof(T) == 2) {
      const bf16x8 f = __builtin_bit_cast(bf16x8, x[s].x[0]);
      G = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f, f, G, 0, 0, 0);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) G = __builtin_amdgcn_mfma_f64_16x16x4f64((double)x[s][e], (double)x[s][e], G, 0, 0, 0);
    }
  }
  bool fine = true;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    fine = fine && __builtin_fabsf((float)G[j]) <= 3.4028235e38f;
    if (Sums<T>::row(g, j) >> lg != row >> lg) G[j] = 0;
  }
  finite = !__any(!fine);
  return G;
}
// two pairs of numbers of bf16
__device__ __forceinline__ u32x2 packed(const float (&a)[4]) {
  return u32x2{__builtin_amdgcn_perm(__float_as_uint(a[1]), __float_as_uint(a[0]), 0x07060302), __builtin_amdgcn_perm(__float_as_uint(a[3]), __float_as_uint(a[2]), 0x07060302)};
}
// four numbers as three of bf16 each, the largest part first: 2^-27 of them off
__device__ __forceinline__ void in_three(f32x4 x, s16x4 (&part)[3]) {
#pragma unroll
  for (int n = 0; n < 3; ++n) {
    const u32x2 p = {pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3])};
    part[n] = __builtin_bit_cast(s16x4, p);
    x = f32x4{x[0] - bf16lo_to_f32(p[0]), x[1] - bf16hi_to_f32(p[0]), x[2] - bf16lo_to_f32(p[1]), x[3] - bf16hi_to_f32(p[1])};
  }
}
// G as the operand of Y = G A
template <typename T>
struct GramOperand;
template <>
struct GramOperand<uint16_t> {
  s16x4 part[3];
  __device__ __forceinline__ explicit GramOperand(f32x4 G) { in_three(G, part); }
  __device__ __forceinline__ f32x4 times(const float (&a)[4]) const {  // a: numbers of bf16
    const u32x2 p = packed(a);
    f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int n = 2; n >= 0; --n) y = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(part[n], __builtin_bit_cast(s16x4, p), y, 0, 0, 0);
    return y;
  }
};
template <>
struct GramOperand<float> {
  f64x4 G;
  __device__ __forceinline__ explicit GramOperand(f64x4 from) : G(from) {}
  __device__ __forceinline__ f64x4 times(const float (&a)[4]) const {
    f64x4 y = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 4; ++j) y = __builtin_amdgcn_mfma_f64_16x16x4f64(G[j], (double)a[j], y, 0, 0, 0);
    return y;
  }
};
// Y of 16 heads; where a number is not finite the tokens take turns
template <typename T>
__device__ __forceinline__ typename Sums<T>::V times_gram(const GramOperand<T>& G, const float (&a)[4], bool finite, int g, int lg) {
  bool fine = finite;
#pragma unroll
  for (int j = 0; j < 4; ++j) fine = fine && __builtin_fabsf(a[j]) <= 3.4028235e38f;
  if (lg == 4 || !__any(!fine)) return G.times(a);
  typename Sums<T>::V y = {0, 0, 0, 0};
  for (int tt = 0; tt < 16 >> lg; ++tt) {
    float one[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) one[j] = Sums<T>::row(g, j) >> lg == tt ? a[j] : 0.f;
    const typename Sums<T>::V yt = G.times(one);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (Sums<T>::row(g, j) >> lg == tt) y[j] = yt[j];
  }
  return y;
}

// b rows of a wave in LDS; the padding spreads the 16 rows that a transposing read meets over the banks
template <typename T, int D>
struct RowsInLds {
  static constexpr int kStride = sizeof(T) == 2 ? D + 8 : D + 4;  // elements
  static constexpr int kBytes = 16 * kStride * sizeof(T);
};
template <typename T, int D>
__device__ __forceinline__ void rows_to_lds(const Chunk<T>& x, int s, int row, int g, T* rows) {
#pragma unroll
  for (int n = 0; n < (int)sizeof(T) / 2; ++n) reinterpret_cast<u32x4*>(rows + row * RowsInLds<T, D>::kStride + 32 * s + 8 * g)[n] = x.x[n];
}
// rows 4 g + 0..3 of the column that this lane stands for: 16 lanes bring 4 rows x 4 columns from `column` on each and get them transposed
template <int D>
__device__ __forceinline__ s16x4 rows_transposed(const uint16_t* rows, int row, int g, int column) {
  const uint16_t* const from = rows + (4 * g + (row >> 2)) * RowsInLds<uint16_t, D>::kStride + column;
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4 __attribute__((address_space(3)))*)from);
}
// Where ranks cancel a^T G a is off by the square of (sum of the terms' sizes / sum) in units of 2^-24, the head vectors themselves by the first
// power.  The sum of the sizes is at most R^2 of the largest a_r^2 |b_r|^2: heads whose sum is less than 2^-10 of that, where the norm may be 2^-13 off,
// are summed anew from R X_h[d] = sum_r b_r[d] a_r[h], whose terms are exact, 16 elements of 16 heads an instruction, which keeps none of them.
// (4 x 4096 tokens, 16 heads of 128, ranks 6 and 2: forward 18.4 us with no such head, 25.5 with nothing else, backward 34.4 and 51.8; without the
// comparison 17.7 and 36.3.)
// A token's rows stand beside zeros for the other tokens', in the b rows too, which need not be finite.  `most`: |a_r| lengths_of(), of which the largest decides.
constexpr float kCancelled = 1.f / 32;
template <int D>
__device__ __forceinline__ void squares_of_vectors(const uint16_t* rows, const float (&a)[4], const float (&most)[4], int row, int g, int lg, float (&square)[4]) {
  float low[4];  // rows of the token that say so
#pragma unroll
  for (int j = 0; j < 4; ++j) low[j] = square[j] < most[j] * most[j] ? 1.f : 0.f;
  over_token<uint16_t>(low, lg);
  wave_lds_fence();
  const u32x2 p = packed(a);
#pragma unroll 1
  for (int tt = 0; tt < 16 >> lg; ++tt) {
    u32x2 keep;
#pragma unroll
    for (int n = 0; n < 2; ++n) keep[n] = ((4 * g + 2 * n) >> lg == tt ? 0xffffu : 0u) | ((4 * g + 2 * n + 1) >> lg == tt ? 0xffff0000u : 0u);
    const s16x4 of_token = __builtin_bit_cast(s16x4, p & keep);
    float sum = 0.f;
#pragma unroll 2
    for (int x = 0; x < D / 16; ++x) {
      const s16x4 f = __builtin_bit_cast(s16x4, __builtin_bit_cast(u32x2, rows_transposed<D>(rows, row, g, 16 * x + 4 * (row & 3))) & keep);
      const f32x4 y = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(f, of_token, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
      for (int e = 0; e < 4; ++e) sum = fmaf(y[e], y[e], sum);
    }
    sum = with_lane(with_lane(sum, 16), 32);
#pragma unroll
    for (int j = 0; j < 4; ++j) square[j] = low[j] != 0.f && (4 * g + j) >> lg == tt ? sum : square[j];
  }
}
// R / 32 of |b_r| of this lane's four rows, off the diagonal of G
__device__ __forceinline__ f32x4 lengths_of(const f32x4& G, int R, int g) {
  f32x4 length;
#pragma unroll
  for (int j = 0; j < 4; ++j) length[j] = kCancelled * R * __builtin_amdgcn_sqrtf(__shfl(G[j], 20 * g + j));
  return length;
}
// the sums of squares of 16 heads, `y` = G a; bf16 factors: `rows` has the b rows, `length` is lengths_of()
template <typename T, int D>
__device__ __forceinline__ void squares_of(const float (&a)[4], const typename Sums<T>::V& y, [[maybe_unused]] const f32x4& length, [[maybe_unused]] const T* rows, [[maybe_unused]] int row,
                                           [[maybe_unused]] int g, int lg, typename Sums<T>::S (&square)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) square[j] = a[j] * y[j];
  over_token<T>(square, lg);
  if constexpr (sizeof(T) == 2) {
    float most[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) most[j] = __builtin_fabsf(a[j] * length[j]);
    bool low;
    if (lg >= 2) {  // the four rows are one token's
      const float m = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
      low = square[0] < m * m;
    } else {
      low = lg && (square[0] < most[0] * most[0] || square[1] < most[1] * most[1] || square[2] < most[2] * most[2] || square[3] < most[3] * most[3]);
    }
    if (__any(low)) squares_of_vectors<D>(rows, a, most, row, g, lg, square);
  }
}

// a wave's tokens, and this lane's row of theirs
struct Rows {
  int bi, first;  // batch entry, its first token
  int tt, r, i;   // this lane's token among the wave's, its rank, the token in the entry (clamped)
  bool there;
  __device__ __forceinline__ Rows(int group, int l, int R, int lg, int lane) {
    const int P = 16 >> lg, per_entry = (l + P - 1) / P, row = lane & 15;
    bi = group / per_entry;
    first = (group - bi * per_entry) * P;
    tt = min(row >> lg, l - 1 - first);
    there = (row & ((1 << lg) - 1)) < R && row >> lg == tt;
    r = min(row & ((1 << lg) - 1), R - 1);
    i = first + tt;
  }
};

template <typename T, int D, bool AXES, int VH, bool CACHED>
__device__ __forceinline__ void norm_rope_rows(const NormRopeParams& p, const Side& side, int group, const float* wt, [[maybe_unused]] T* rows) {
  constexpr int NS = D / 32;
  const int lane = threadIdx.x & 63, row = lane & 15, g = lane >> 4, R = side.R, H = p.H, lg = rows_log2(R);
  const Rows me(group, p.l, R, lg, lane);
  const TurnAt<D, AXES> turn_at(p.rot, me.bi * p.l + me.i, me.i, g);
  const T* const b = base_of<const T>(side.b, me.bi, me.first) + (offset_of(side.b, me.tt, me.r) + 8 * g);
  Chunk<T> x[NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) x[s] = load_chunk(b + 32 * s);  // (rows that are not there repeat one: a load in a branch would be waited for there)
  // head factors: of four rows this lane has VH heads of every 16 VH
  const T* const a_base = base_of<const T>(side.a, me.bi, me.first);
  uint32_t a_in[4];
  T* a_out[4];  // CACHED: by slot
  uint32_t a_to[4];
  T* const a_out_base = CACHED ? nullptr : base_of<T>(side.a_out, me.bi, me.first);
  bool a_there[4], a_stored[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int rj = Sums<T>::row(g, j), tt = min(rj >> lg, p.l - 1 - me.first), r = min(rj & ((1 << lg) - 1), R - 1);
    a_there[j] = rj >> lg == tt && (rj & ((1 << lg) - 1)) < R;
    a_in[j] = offset_of(side.a, tt, r);
    a_stored[j] = a_there[j];
    if constexpr (CACHED) {
      int64_t page, at;
      a_stored[j] = slot_of(p, me.bi, me.first + tt, page, at) && a_there[j];
      a_out[j] = static_cast<T*>(const_cast<void*>(side.a_out.ptr)) + page * side.a_out.stride_b + at * side.a_out.stride_l + r * side.a_out.stride_r;
    } else {
      a_to[j] = offset_of(side.a_out, tt, r);
    }
  }
  Heads<T, VH> next[4];
  auto heads = [&](int h) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 4; ++j) next[j] = load_heads<T, VH>(a_base + (a_in[j] + min(h, H - VH)));
  };
  heads(VH * row);
  const Turns<D, AXES> turn(p.rot, turn_at, g);
  bool stored = me.there;
  T* bo;
  if constexpr (CACHED) {
    int64_t page, at;
    stored = slot_of(p, me.bi, me.i, page, at) && me.there;
    bo = static_cast<T*>(const_cast<void*>(side.b_out.ptr)) + page * side.b_out.stride_b + at * side.b_out.stride_l + me.r * side.b_out.stride_r + 8 * g;
  } else {
    bo = base_of<T>(side.b_out, me.bi, me.first) + (offset_of(side.b_out, me.tt, me.r) + 8 * g);
  }
#pragma unroll
  for (int s = 0; s < NS; ++s) x[s].keep(me.there);
  bool finite = true;
  typename Sums<T>::V G0 = {0, 0, 0, 0};
  if (p.normalize) G0 = gram<T, D>(x, row, g, lg, finite);
  const GramOperand<T> G(G0);
  f32x4 length = {0.f, 0.f, 0.f, 0.f};
  if constexpr (sizeof(T) == 2) {
    length = lengths_of(G0, R, g);
#pragma unroll
    for (int s = 0; s < NS; ++s) rows_to_lds<T, D>(x[s], s, row, g, rows);  // where they wait for the heads too
  }
  const typename Sums<T>::S inv = (typename Sums<T>::S)1 / (typename Sums<T>::S)(R * R * D);
  for (int h = VH * row; h - VH * row < H; h += 16 * VH) {
    float a[4][VH];
#pragma unroll
    for (int j = 0; j < 4; ++j) next[j].unpack(a_there[j] && h < H, a[j]);
    if (h - VH * row + 16 * VH < H) heads(h + 16 * VH);
    if (p.normalize) {
#pragma unroll
      for (int v = 0; v < VH; ++v) {
        const float av[4] = {a[0][v], a[1][v], a[2][v], a[3][v]};
        const typename Sums<T>::V y = times_gram<T>(G, av, finite, g, lg);
        typename Sums<T>::S square[4];
        squares_of<T, D>(av, y, length, rows, row, g, lg, square);
        float scale[4];
        inverse_norms<T>(square, inv, p.eps, lg, scale);
#pragma unroll
        for (int j = 0; j < 4; ++j) a[j][v] *= scale[j];
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (a_stored[j] && h < H) store_heads<T, VH>(CACHED ? a_out[j] + h : a_out_base + (a_to[j] + h), a[j]);
  }
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    float y[8];
    const Chunk<float> w = load_chunk(wt + 32 * s + 8 * g);
    if constexpr (sizeof(T) == 2) x[s] = load_chunk(rows + row * RowsInLds<T, D>::kStride + 32 * s + 8 * g);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float y0 = x[s][2 * e] * w[2 * e], y1 = x[s][2 * e + 1] * w[2 * e + 1];
      y[2 * e] = y0 * turn.c[s][e] - y1 * turn.s[s][e];
      y[2 * e + 1] = y1 * turn.c[s][e] + y0 * turn.s[s][e];
    }
    if (stored) store_chunk(bo + 32 * s, y);
  }
  if constexpr (sizeof(T) == 2) wave_lds_fence();  // the next tokens' rows go where these are
}

// V factors into their slots, 16 bytes a lane: chunks of a row of ranks, head factors first
template <typename T, int D>
__device__ __forceinline__ void copy_values(const NormRopeParams& p, int group) {
  constexpr int E = 16 / sizeof(T);
  const int R = p.side[1].R, lane = threadIdx.x & 63, per_rank = (p.H + D) / E, per_token = R * per_rank, P = tokens_per_wave(R);
  const int per_entry = (p.l + P - 1) / P, bi = group / per_entry, first = (group - bi * per_entry) * P;
  for (int x = lane; x < P * per_token; x += 64) {
    const int tt = x / per_token, i = first + tt, rest = x - tt * per_token, r = rest / per_rank, c = (rest - r * per_rank) * E;
    if (i >= p.l) break;
    int64_t page, at;
    if (!slot_of(p, bi, i, page, at)) continue;
    const bool head = c < p.H;
    const TpaFactor &in = head ? p.va : p.vb, &out = head ? p.va_out : p.vb_out;
    const int col = head ? c : c - p.H;
    *reinterpret_cast<u32x4*>(static_cast<T*>(const_cast<void*>(out.ptr)) + page * out.stride_b + at * out.stride_l + r * out.stride_r + col) =
        *reinterpret_cast<const u32x4*>(base_of<const T>(in, bi, first) + (offset_of(in, tt, r) + col));
  }
}

// Workgroups 0 .. parts_q - 1 share out the queries' tokens, the next parts_k the keys', the others the values'
template <typename T, int D, bool AXES, int VH, bool CACHED>
__global__ __launch_bounds__(kNormWaves * 64, fwd_waves(sizeof(T), D)) void norm_rope_kernel(NormRopeParams p, int parts_q, int parts_k, int parts_v) {
  __shared__ __attribute__((aligned(16))) float wt[D];
  __shared__ __attribute__((aligned(16))) unsigned char rows_mem[sizeof(T) == 2 ? kNormWaves * RowsInLds<T, D>::kBytes : 16];
  const int w = scalar(threadIdx.x >> 6), part = blockIdx.x;
  T* const rows = reinterpret_cast<T*>(rows_mem + (sizeof(T) == 2 ? w * RowsInLds<T, D>::kBytes : 0));
  auto groups = [&](int R) { return (p.l + tokens_per_wave(R) - 1) / tokens_per_wave(R) * p.B; };
  if (part < parts_q) {
    weights_to_lds<D>(p.side[0].weight, p.weight_bf16, wt);
    for (int group = part * kNormWaves + w; group < groups(p.side[0].R); group += parts_q * kNormWaves) norm_rope_rows<T, D, AXES, VH, false>(p, p.side[0], group, wt, rows);
  } else if (part < parts_q + parts_k) {
    weights_to_lds<D>(p.side[1].weight, p.weight_bf16, wt);
    for (int group = (part - parts_q) * kNormWaves + w; group < groups(p.side[1].R); group += parts_k * kNormWaves) norm_rope_rows<T, D, AXES, VH, CACHED>(p, p.side[1], group, wt, rows);
  } else if constexpr (CACHED) {
    for (int group = (part - parts_q - parts_k) * kNormWaves + w; group < groups(p.side[1].R); group += parts_v * kNormWaves) copy_values<T, D>(p, group);
  }
}

// ---- gradients.  The R x R sums M = A diag(w) A^T over the heads and the mixture M B of the b rows are products of the matrix cores
// too: M's result layout is that of the second product's operand, whose other one are the b rows read back transposed from LDS.  For bf16
// factors w a and M are kept as three bf16 numbers each (2^-27 off: where ranks cancel the mixture is off by that times sum of sizes / sum).
template <typename T, int D>
struct BwdLds {
  static constexpr int kStride = RowsInLds<T, D>::kStride;
  static constexpr size_t kRows = RowsInLds<T, D>::kBytes;
  static size_t wave_bytes(int most_pairs) { return kRows + (size_t)(most_pairs + 3) / 4 * 16; }
  static size_t bytes(int most_pairs) { return kNormWaves * wave_bytes(most_pairs) + D * sizeof(float); }
};

template <typename T, int D, bool AXES, int VH>
__device__ __forceinline__ void norm_rope_bwd_rows(const NormRopeBwdParams& p, const BwdSide& side, int group, unsigned char* lds, const float* wt, float (&d_weight)[D / 4]) {
  constexpr int NS = D / 32;
  using Lds = BwdLds<T, D>;
  T* const rows = reinterpret_cast<T*>(lds);
  float* const W = reinterpret_cast<float*>(lds + Lds::kRows);  // [token][H]
  const int lane = threadIdx.x & 63, row = lane & 15, g = lane >> 4, R = side.R, H = p.H, lg = rows_log2(R);
  const Rows me(group, p.l, R, lg, lane);
  const TurnAt<D, AXES> turn_at(p.rot, me.bi * p.l + me.i, me.i, g);
  const T* const b = base_of<const T>(side.b, me.bi, me.first) + (offset_of(side.b, me.tt, me.r) + 8 * g);
  const T* const db = base_of<const T>(side.db_out, me.bi, me.first) + (offset_of(side.db_out, me.tt, me.r) + 8 * g);
  Chunk<T> x[NS], dy[NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) x[s] = load_chunk(b + 32 * s);
  const T *const a_base = base_of<const T>(side.a, me.bi, me.first), *const da_base = base_of<const T>(side.da_out, me.bi, me.first);
  T* const out_base = base_of<T>(side.da, me.bi, me.first);
  uint32_t a_in[4], da_in[4], da_out[4];
  bool a_there[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int rj = Sums<T>::row(g, j), tt = min(rj >> lg, p.l - 1 - me.first), r = min(rj & ((1 << lg) - 1), R - 1);
    a_there[j] = rj >> lg == tt && (rj & ((1 << lg) - 1)) < R;
    a_in[j] = offset_of(side.a, tt, r);
    da_in[j] = offset_of(side.da_out, tt, r);
    da_out[j] = offset_of(side.da, tt, r);
  }
  Heads<T, VH> next[4], d_next[4];
  auto heads = [&](int h) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      next[j] = load_heads<T, VH>(a_base + (a_in[j] + min(h, H - VH)));
      d_next[j] = load_heads<T, VH>(da_base + (da_in[j] + min(h, H - VH)));
    }
  };
  heads(VH * row);
#pragma unroll
  for (int s = 0; s < NS; ++s) dy[s] = load_chunk(db + 32 * s);
#pragma unroll
  for (int s = 0; s < NS; ++s) x[s].keep(me.there);
  bool finite = true;
  typename Sums<T>::V G0 = {0, 0, 0, 0};
#pragma unroll
  for (int s = 0; s < NS; ++s) rows_to_lds<T, D>(x[s], s, row, g, rows);  // where they wait for the heads too
  if (p.normalize) G0 = gram<T, D>(x, row, g, lg, finite);
  const GramOperand<T> G(G0);
  f32x4 length = {0.f, 0.f, 0.f, 0.f};
  if constexpr (sizeof(T) == 2) length = lengths_of(G0, R, g);
  const typename Sums<T>::S inv = (typename Sums<T>::S)1 / (typename Sums<T>::S)(R * R * D);
  for (int h = VH * row; h - VH * row < H; h += 16 * VH) {
    float a[4][VH], da[4][VH];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      next[j].unpack(a_there[j] && h < H, a[j]);
      d_next[j].unpack(a_there[j] && h < H, da[j]);
    }
    if (h - VH * row + 16 * VH < H) heads(h + 16 * VH);
    if (p.normalize) {
#pragma unroll
      for (int v = 0; v < VH; ++v) {
        const float av[4] = {a[0][v], a[1][v], a[2][v], a[3][v]};
        const typename Sums<T>::V y = times_gram<T>(G, av, finite, g, lg);
        typename Sums<T>::S square[4];
        float u[4];
        squares_of<T, D>(av, y, length, rows, row, g, lg, square);
#pragma unroll
        for (int j = 0; j < 4; ++j) u[j] = da[j][v] * av[j];
        over_token<T>(u, lg);
        float scale[4];
        inverse_norms<T>(square, inv, p.eps, lg, scale);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float w = -(scale[j] * u[j]) * (scale[j] * (float)inv) * scale[j];  // (the cube alone may pass 2^128)
          da[j][v] = da[j][v] * scale[j] + w * (float)y[j];
          const int rj = Sums<T>::row(g, j);
          if ((rj & ((1 << lg) - 1)) == 0 && h < H) W[(rj >> lg) * H + h + v] = w;
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (a_there[j] && h < H) store_heads<T, VH>(out_base + (da_out[j] + h), da[j]);
  }
#pragma unroll
  for (int s = 0; s < NS; ++s) dy[s].keep(me.there);
  const T* const a_row = a_base + offset_of(side.a, me.tt, me.r);
  auto factors = [&](int h) __attribute__((always_inline)) { return load_chunk(a_row + min(h, H - 8)); };
  Chunk<T> ac = factors(8 * g);
  const Turns<D, AXES> turn(p.rot, turn_at, g);
  f32x4 M = {0.f, 0.f, 0.f, 0.f};  // M[4 g + e][row] of the token's rows
  [[maybe_unused]] s16x4 M_part[3] = {};
  wave_lds_fence();
  if (p.normalize) {
    const float* const w_of = W + (row >> lg) * H;
    for (int h = 8 * g; h - 8 * g < H; h += 32) {
      const bool there = me.there && h < H;
      ac.keep(there);
      const Chunk<T> next = factors(h + 32);
      float w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = there ? ac[e] * w_of[h + e] : 0.f;
      if constexpr (sizeof(T) == 2) {
        const bf16x8 f = __builtin_bit_cast(bf16x8, ac.x[0]);
#pragma unroll
        for (int n = 0; n < 3; ++n) {
          u32x4 part;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            part[e] = pack_bf16(w[2 * e], w[2 * e + 1]);
            w[2 * e] -= bf16lo_to_f32(part[e]);
            w[2 * e + 1] -= bf16hi_to_f32(part[e]);
          }
          M = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f, __builtin_bit_cast(bf16x8, part), M, 0, 0, 0);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) M = __builtin_amdgcn_mfma_f32_16x16x4f32(ac[e], w[e], M, 0, 0, 0);
      }
      ac = next;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if ((4 * g + e) >> lg != row >> lg) M[e] = 0.f;
    if constexpr (sizeof(T) == 2) in_three(M, M_part);
  }
  // the mixture of the b rows for this lane's row: element e of piece n is d = 32 (n / 2) + 8 g + 4 (n % 2) + e
  auto mix = [&](int n) __attribute__((always_inline)) {
    f32x4 out = {0.f, 0.f, 0.f, 0.f};
    if constexpr (sizeof(T) == 2) {
      const s16x4 f = rows_transposed<D>(rows, row, g, 32 * (n / 2) + 8 * (row & 3) + 4 * (n % 2));
#pragma unroll
      for (int x = 2; x >= 0; --x) out = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(f, M_part[x], out, 0, 0, 0);
      return out;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        out = __builtin_amdgcn_mfma_f32_16x16x4f32(rows[(4 * g + e) * Lds::kStride + 32 * (n / 2) + 8 * (row >> 2) + 4 * (n % 2) + (row & 3)], M[e], out, 0, 0, 0);
      return out;
    }
  };
  T* const bo = base_of<T>(side.db, me.bi, me.first) + (offset_of(side.db, me.tt, me.r) + 8 * g);
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    f32x4 mixed[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    const Chunk<T> xs = load_chunk(rows + row * Lds::kStride + 32 * s + 8 * g);
    if (p.normalize) {
      if (finite) {
        mixed[0] = mix(2 * s);
        mixed[1] = mix(2 * s + 1);
      } else {
        for (int tt = 0; tt < 16 >> lg; ++tt) {
          wave_lds_fence();
          const bool mine = row >> lg == tt;
          Chunk<T> one = xs;
          one.keep(mine);
          rows_to_lds<T, D>(one, s, row, g, rows);
          wave_lds_fence();
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const f32x4 by_token = mix(2 * s + n);
            mixed[n] = mine ? by_token : mixed[n];
          }
        }
      }
    }
    float y[8];
    const Chunk<float> w = load_chunk(wt + 32 * s + 8 * g);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float y0 = dy[s][2 * e], y1 = dy[s][2 * e + 1];
      const float e0 = y0 * turn.c[s][e] + y1 * turn.s[s][e], e1 = y1 * turn.c[s][e] - y0 * turn.s[s][e];
      d_weight[8 * s + 2 * e] = fmaf(e0, xs[2 * e], d_weight[8 * s + 2 * e]);
      d_weight[8 * s + 2 * e + 1] = fmaf(e1, xs[2 * e + 1], d_weight[8 * s + 2 * e + 1]);
      y[2 * e] = fmaf(e0, w[2 * e], mixed[e / 2][2 * e % 4]);
      y[2 * e + 1] = fmaf(e1, w[2 * e + 1], mixed[e / 2][(2 * e + 1) % 4]);
    }
    if (me.there) store_chunk(bo + 32 * s, y);
  }
  wave_lds_fence();  // the next tokens' rows go where these are
}

// Workgroups 0 .. parts_q - 1 share out the queries' tokens, the others the keys'
template <typename T, int D, bool AXES, int VH>
__global__ __launch_bounds__(kNormWaves * 64, bwd_waves(sizeof(T), D, VH)) void norm_rope_bwd_kernel(NormRopeBwdParams p, int parts_q, int parts_k, int wave_bytes) {
  extern __shared__ __attribute__((aligned(16))) unsigned char bwd_mem[];
  const int w = scalar(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const bool keys = (int)blockIdx.x >= parts_q;
  const int part = keys ? blockIdx.x - parts_q : blockIdx.x;
  float d_weight[D / 4];  // of this lane's row: element 8 s + e is d = 32 s + 8 g + e
#pragma unroll
  for (int x = 0; x < D / 4; ++x) d_weight[x] = 0.f;
  float* const wt = reinterpret_cast<float*>(bwd_mem + kNormWaves * wave_bytes);
  auto rows_of = [&](const BwdSide& side, int parts) __attribute__((always_inline)) {
    const int P = tokens_per_wave(side.R), groups = (p.l + P - 1) / P * p.B;
    weights_to_lds<D>(side.weight, p.weight_bf16, wt);
    for (int group = part * kNormWaves + w; group < groups; group += parts * kNormWaves)
      norm_rope_bwd_rows<T, D, AXES, VH>(p, side, group, bwd_mem + w * wave_bytes, wt, d_weight);
  };
  if (keys) rows_of(p.side[1], parts_k);
  else rows_of(p.side[0], parts_q);
  if (!(keys ? p.side[1].d_weight : p.side[0].d_weight)) return;
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
bool fast_takes(const Args* a, int rq, int rk, const TpaFactor* const* fs, int n) {
  if (a->kernel == TPA_KERNEL_GENERIC || (a->D != 64 && a->D != 128) || a->H % 8 || rq > 16 || rk > 16) return false;
  if ((int64_t)a->B * a->l > (1 << 26)) return false;  // groups of tokens of every entry in 32 bits
  for (int i = 0; i < a->n_axes; ++i)
    if (a->sections[i] % 4) return false;
  const int chunk = a->dtype == TPA_DTYPE_BF16 ? 8 : 4;
  for (int i = 0; i < n; ++i) {
    const TpaFactor& f = *fs[i];
    if ((reinterpret_cast<uintptr_t>(f.ptr) & 15) || f.stride_b % chunk || f.stride_l % chunk || f.stride_r % chunk) return false;
    if (f.stride_l < 0 || f.stride_r < 0 || f.stride_l > (1 << 25) || f.stride_r > (1 << 25)) return false;  // 16 tokens' offsets in 32 bits
  }
  return !((reinterpret_cast<uintptr_t>(a->rope_cos) | reinterpret_cast<uintptr_t>(a->rope_sin)) & 15);
}
// entries that follow one another in every array are one: what positions count from then has to be given
bool follows(const TpaFactor& f, int l) { return f.stride_b == f.stride_l * l; }
// workgroups for a side's tokens
int parts_of(int B, int l, int R, int most) {
  const int64_t groups = (int64_t)B * ((l + tokens_per_wave(R) - 1) / tokens_per_wave(R));
  return (int)std::min<int64_t>((groups + kNormWaves - 1) / kNormWaves, most);
}
template <typename T, int D>
int launch_fast(NormRopeParams p, hipStream_t s) {
  const int64_t tokens = (int64_t)p.B * p.l;
  bool one = p.rot.positions != nullptr;
  for (const Side& x : p.side) one = one && follows(x.a, p.l) && follows(x.b, p.l);
  for (int x = 0; x < (p.slots ? 1 : 2); ++x) one = one && follows(p.side[x].a_out, p.l) && follows(p.side[x].b_out, p.l);
  if (p.slots) one = one && follows(p.va, p.l) && follows(p.vb, p.l);
  if (one) {
    p.l = (int)tokens;
    p.B = 1;
  }
  const int q = parts_of(p.B, p.l, p.side[0].R, 4096), k = parts_of(p.B, p.l, p.side[1].R, 4096), v = p.slots ? k : 0;
  const bool axes = p.rot.n_axes > 1 || p.rot.last_of[3] < D / 2;
  with_heads(p.H, [&](auto vh) {
    constexpr int VH = decltype(vh)::value;
    auto kern = axes ? (p.slots ? norm_rope_kernel<T, D, true, VH, true> : norm_rope_kernel<T, D, true, VH, false>)
                     : (p.slots ? norm_rope_kernel<T, D, false, VH, true> : norm_rope_kernel<T, D, false, VH, false>);
    hipLaunchKernelGGL(kern, dim3(q + k + v), dim3(kNormWaves * 64), 0, s, p, q, k, v);
  });
  return hipGetLastError() == hipSuccess ? TPA_OK : TPA_ERR_LAUNCH;
}
inline int most_pairs(int rq, int rk, int H) { return (tokens_per_wave(rq) > tokens_per_wave(rk) ? tokens_per_wave(rq) : tokens_per_wave(rk)) * H; }
size_t bwd_lds(int dtype, int D, int pairs) {
  if (dtype == TPA_DTYPE_BF16) return D == 128 ? BwdLds<uint16_t, 128>::bytes(pairs) : BwdLds<uint16_t, 64>::bytes(pairs);
  return D == 128 ? BwdLds<float, 128>::bytes(pairs) : BwdLds<float, 64>::bytes(pairs);
}
template <typename T, int D>
int launch_fast_bwd(NormRopeBwdParams p, int (&parts)[2], hipStream_t s) {
  const int64_t tokens = (int64_t)p.B * p.l;
  bool one = p.rot.positions != nullptr;
  for (int x = 0; x < 2; ++x) {
    const BwdSide& side = p.side[x];
    if (side.da_out.ptr)
      for (const TpaFactor* f : {&side.a, &side.b, &side.da_out, &side.db_out, &side.da, &side.db}) one = one && follows(*f, p.l);
  }
  if (one) {
    p.l = (int)tokens;
    p.B = 1;
  }
  // All workgroups are resident at once, and their waves take the same number of tokens' groups: what a wave has to do behind its last one - the weights'
  // gradients - is done once.  (With up to 768 workgroups
  // a side / so, us: 4 x 4096 tokens, 16 heads of 128, three axes 42.1 / 40.3, 4 x 2048, 24 heads 29.3 / 27.0.)
  const int pairs = most_pairs(p.side[0].R, p.side[1].R, p.H), wave = (int)BwdLds<T, D>::wave_bytes(pairs);
  const size_t lds = BwdLds<T, D>::bytes(pairs);
  const int64_t resident = 256 * std::min<int64_t>(bwd_waves(sizeof(T), D, p.H > 16 ? 2 : 1), kMostLds / lds);
  int64_t groups[2];
  for (int x = 0; x < 2; ++x) groups[x] = p.side[x].da_out.ptr ? (int64_t)p.B * ((p.l + tokens_per_wave(p.side[x].R) - 1) / tokens_per_wave(p.side[x].R)) : 0;
  auto parts_for = [&](int x, int64_t each) { return (groups[x] + each * kNormWaves - 1) / (each * kNormWaves); };
  int64_t each = std::max<int64_t>(1, (groups[0] + groups[1]) / (kNormWaves * resident));
  while (parts_for(0, each) + parts_for(1, each) > resident) ++each;
  for (int x = 0; x < 2; ++x) parts[x] = (int)parts_for(x, each);
  const bool axes = p.rot.n_axes > 1 || p.rot.last_of[3] < D / 2;
  const dim3 grid(parts[0] + parts[1]);
  int rc = TPA_OK;
  with_heads(p.H, [&](auto vh) {
    constexpr int VH = decltype(vh)::value;
    auto kern = axes ? norm_rope_bwd_kernel<T, D, true, VH> : norm_rope_bwd_kernel<T, D, false, VH>;
    static bool done[2][kMaxDevices] = {};
    if (lds > 64 * 1024) rc = raise_lds_limit(done[axes], reinterpret_cast<const void*>(kern), kMostLds);
    if (rc == TPA_OK) hipLaunchKernelGGL(kern, grid, dim3(kNormWaves * 64), lds, s, p, parts[0], parts[1], wave);
  });
  if (rc != TPA_OK) return rc;
  return hipGetLastError() == hipSuccess ? TPA_OK : TPA_ERR_LAUNCH;
}

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
  if (fast_takes(a, a->rq, a->rk, fs, a->slots ? 12 : 8)) {
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
  // a side without a gradient is as if it had the other's: nothing of its own is looked at
  const bool q = a->dqa_out.ptr, k = a->dka_out.ptr;
  const int rq = q || !k ? a->rq : a->rk, rk = k || !q ? a->rk : a->rq;
  if (const int rc = check_sizes(a->B, a->l, a->H, a->D, q || k ? rq : 1, q || k ? rk : 1, a->rope_len, a->dtype, a->weight_dtype, a->kernel, a->n_axes, a->sections); rc != TPA_OK) return rc;
  if (!q && !k) return TPA_OK;
  const TpaFactor* fs[12] = {};
  int n = 0;
  if (q)
    for (const TpaFactor* f : {&a->qa, &a->qb, &a->dqa_out, &a->dqb_out, &a->dqa, &a->dqb}) fs[n++] = f;
  if (k)
    for (const TpaFactor* f : {&a->ka, &a->kb, &a->dka_out, &a->dkb_out, &a->dka, &a->dkb}) fs[n++] = f;
  for (int i = 0; i < n; ++i)
    if (!fs[i]->ptr) return TPA_ERR_NULL;
  if (!a->rope_cos || !a->rope_sin) return TPA_ERR_NULL;
  NormRopeBwdParams p{};
  if (q) p.side[0] = {a->qa, a->qb, a->dqa_out, a->dqb_out, a->dqa, a->dqb, a->q_weight, a->dq_weight, rq};
  if (k) p.side[1] = {a->ka, a->kb, a->dka_out, a->dkb_out, a->dka, a->dkb, a->k_weight, a->dk_weight, rk};
  p.side[0].R = rq;
  p.side[1].R = rk;
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
  if (fast_takes(a, rq, rk, fs, n) && bwd_lds(a->dtype, a->D, most_pairs(rq, rk, a->H)) <= kMostLds) {
    if (a->dtype == TPA_DTYPE_BF16) rc = a->D == 128 ? launch_fast_bwd<uint16_t, 128>(p, sum.count, s) : launch_fast_bwd<uint16_t, 64>(p, sum.count, s);
    else rc = a->D == 128 ? launch_fast_bwd<float, 128>(p, sum.count, s) : launch_fast_bwd<float, 64>(p, sum.count, s);
  } else {
    if (a->kernel == TPA_KERNEL_MFMA) return TPA_ERR_UNSUPPORTED;
    const size_t lds = any_lds(rq > rk ? rq : rk, a->H, a->D, true);
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
