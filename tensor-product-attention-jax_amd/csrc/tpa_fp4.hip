// K and V factors of new tokens into a paged cache in 4 bits, and the factors that its slots stand for.
//
// A block of 32 numbers shares a scale 2^e: e from the exponent of the largest magnitude (one up where its significand is over 7.25 / 4), the codes by
// the hardware's conversion (to the nearest, halves to even, at most 6), which is exact arithmetic: the bytes depend on nothing but the numbers.
// Four lanes hold a block, eight numbers each: 16 bytes read (bf16), two exchanges for the largest magnitude, a word of codes and every fourth lane a scale
// written; reading back is the same the other way round.
//
// A step's few tokens are bound by latency, a chunk of a prompt by HBM.
#include "tpa_fp4.h"

namespace tpa {
namespace {

constexpr int kThreads = 256;

struct RowsParams {
  TpaFactor ka, kb, va, vb, k_cache, v_cache;
  const int32_t* slots;
  int page_size, num_slots, l, H, dk, dv, rk;
  int lanes;              // of a row
  int tokens;             // B * l
};

// the part of a row that a lane works on: 8 numbers from `first` on of n numbers of a or b
struct Part {
  bool of_a;
  int n, first, codes, scale;  // bytes from the start of the row
};
__device__ __forceinline__ Part part_of(int lane, int H, int D) {
  const Fp4Row row(H, D);
  const int of_b = 4 * fp4_blocks(D);
  Part p;
  p.of_a = lane >= of_b;
  const int at = p.of_a ? lane - of_b : lane;
  p.n = p.of_a ? H : D;
  p.first = 8 * at;
  p.codes = (p.of_a ? row.a_codes : 0) + 4 * at;
  p.scale = (p.of_a ? row.a_scales : row.b_scales) + at / 4;
  return p;
}
// one of two field by field: through a pointer all of the arguments would be copied to scratch memory first (a chunk of 8195 tokens 61 us)
__device__ __forceinline__ TpaFactor pick(bool second, const TpaFactor& x, const TpaFactor& y) {
  return TpaFactor{second ? y.ptr : x.ptr, second ? y.stride_b : x.stride_b, second ? y.stride_l : x.stride_l, second ? y.stride_r : x.stride_r};
}
// (token, rank, lane of the row) of a thread, which has that lane of K's row and of V's: two loads on their way instead of one, half the waves
// (with a thread for each, write and read of 8195 tokens, 32 heads of 128, rank 2, 11.0 + 10.3 us)
struct Place {
  int token, rank, lane;
  int64_t b, i;     // of the factors
  int page, in_page;
  bool there;       // the slot is in the pools
};
__device__ __forceinline__ bool place_of(const RowsParams& p, Place& at) {
  const uint32_t id = blockIdx.x * kThreads + threadIdx.x, row = id / (uint32_t)p.lanes;
  at.lane = (int)(id - row * p.lanes);
  at.token = (int)(row / (uint32_t)p.rk);
  at.rank = (int)(row - (uint32_t)at.token * p.rk);
  if (at.token >= p.tokens) return false;
  const int slot = p.slots[at.token];
  at.there = slot >= 0 && slot < p.num_slots;
  at.page = (int)((uint32_t)slot / (uint32_t)p.page_size);
  at.in_page = slot - at.page * p.page_size;
  const int b = (int)((uint32_t)at.token / (uint32_t)p.l);
  at.b = b;
  at.i = at.token - b * p.l;
  return true;
}
__device__ __forceinline__ uint8_t* row_of(const TpaFactor& cache, const Place& at) {
  return static_cast<uint8_t*>(const_cast<void*>(cache.ptr)) + at.page * cache.stride_b + at.in_page * cache.stride_l + at.rank * cache.stride_r;
}
template <typename T>
__device__ __forceinline__ T* numbers_of(const TpaFactor& a, const TpaFactor& b, const Place& at, const Part& part) {
  const TpaFactor f = pick(part.of_a, b, a);
  return static_cast<T*>(const_cast<void*>(f.ptr)) + at.b * f.stride_b + at.i * f.stride_l + at.rank * f.stride_r + part.first;
}

// WHOLE: sizes that are multiples of 8, rows at multiples of 16 bytes (the cache's of 4)
template <typename T, bool WHOLE>
struct Numbers {  // eight of them, as bits of fp32
  uint32_t x[8];
  __device__ __forceinline__ void load(const T* from, int n) {
    if constexpr (WHOLE && sizeof(T) == 2) {
      const u32x4 w = n > 0 ? *reinterpret_cast<const u32x4*>(from) : u32x4{0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[2 * j] = w[j] << 16;
        x[2 * j + 1] = w[j] & 0xffff0000u;
      }
    } else if constexpr (WHOLE) {
      const u32x4 lo = n > 0 ? *reinterpret_cast<const u32x4*>(from) : u32x4{0, 0, 0, 0}, hi = n > 0 ? *reinterpret_cast<const u32x4*>(from + 4) : u32x4{0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[j] = lo[j];
        x[4 + j] = hi[j];
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = j < n ? __float_as_uint(load_as_f32(from + j)) : 0u;
    }
  }
};
template <typename T, bool WHOLE>
__device__ __forceinline__ void write_part(const uint32_t (&x)[8], int n, const Part& part, uint8_t* row) {
  // the bits of magnitudes are ordered as these are, those of infinity and NaN above all others
  uint32_t most = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) most = max(most, x[j] & 0x7fffffffu);
  most = max(most, (uint32_t)lanes_of<0xB1>((int)most));  // the four lanes of the block
  most = max(most, (uint32_t)lanes_of<0x4E>((int)most));
  if (n <= 0) return;
  const int exponent = (int)(most >> 23);
  const bool finite = exponent < 255;
  // floor(log2 m) - 2 + 127, one more where m > 7.25 * 2^e: a significand over 1.8125
  const uint32_t scale = finite ? (uint32_t)max(2, min(exponent - 2 + ((most & 0x7fffffu) > 0x680000u), 252)) : 255u;
  uint32_t codes = 0;
  if (finite) {
    const float s = fp4_scale(scale);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, __uint_as_float(x[0]), __uint_as_float(x[1]), s, 0);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, __uint_as_float(x[2]), __uint_as_float(x[3]), s, 1);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, __uint_as_float(x[4]), __uint_as_float(x[5]), s, 2);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, __uint_as_float(x[6]), __uint_as_float(x[7]), s, 3);
  }
  if constexpr (WHOLE) {
    *reinterpret_cast<uint32_t*>(row + part.codes) = codes;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (2 * j < n) row[part.codes + j] = (uint8_t)(codes >> (8 * j));
  }
  if (part.first % 32 == 0) row[part.scale] = (uint8_t)scale;
}

// numbers of its part that a lane has (none past the end of a short block, or of the shorter of K's and V's rows)
__device__ __forceinline__ int numbers_in(const Part& part) { return min(8, part.n - part.first); }

template <typename T, bool WHOLE>
__global__ __launch_bounds__(kThreads) void write_kernel(RowsParams p) {
  Place at;
  if (!place_of(p, at) || !at.there) return;
  const Part of_k = part_of(at.lane, p.H, p.dk), of_v = part_of(at.lane, p.H, p.dv);
  const int nk = numbers_in(of_k), nv = numbers_in(of_v);
  Numbers<T, WHOLE> k, v;
  k.load(numbers_of<const T>(p.ka, p.kb, at, of_k), nk);
  v.load(numbers_of<const T>(p.va, p.vb, at, of_v), nv);
  write_part<T, WHOLE>(k.x, nk, of_k, row_of(p.k_cache, at));
  write_part<T, WHOLE>(v.x, nv, of_v, row_of(p.v_cache, at));
}

template <typename T, bool WHOLE>
__device__ __forceinline__ void read_part(uint32_t codes, uint32_t scale, bool there, int n, T* to) {
  if (n <= 0) return;
  float x[8] = {};
  if (there) fp4_f32x8(codes, fp4_scale(scale), x);
  if constexpr (WHOLE && sizeof(T) == 2) {
    *reinterpret_cast<u32x4*>(to) = u32x4{pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7])};
  } else if constexpr (WHOLE) {
    *reinterpret_cast<f32x4*>(to) = f32x4{x[0], x[1], x[2], x[3]};
    *reinterpret_cast<f32x4*>(to + 4) = f32x4{x[4], x[5], x[6], x[7]};
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) store_from_f32(to + j, x[j]);
  }
}
template <bool WHOLE>
__device__ __forceinline__ uint32_t codes_of(const uint8_t* codes, int n) {
  if constexpr (WHOLE) return n > 0 ? *reinterpret_cast<const uint32_t*>(codes) : 0;
  uint32_t w = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (2 * j < n) w |= (uint32_t)codes[j] << (8 * j);
  return w;
}

template <typename T, bool WHOLE>
__global__ __launch_bounds__(kThreads) void read_kernel(RowsParams p) {
  Place at;
  if (!place_of(p, at)) return;
  const Part of_k = part_of(at.lane, p.H, p.dk), of_v = part_of(at.lane, p.H, p.dv);
  const int nk = numbers_in(of_k), nv = numbers_in(of_v);
  uint32_t k = 0, v = 0, k_scale = 0, v_scale = 0;
  if (at.there) {
    const uint8_t *const k_row = row_of(p.k_cache, at), *const v_row = row_of(p.v_cache, at);
    k = codes_of<WHOLE>(k_row + of_k.codes, nk);
    v = codes_of<WHOLE>(v_row + of_v.codes, nv);
    if (nk > 0) k_scale = k_row[of_k.scale];
    if (nv > 0) v_scale = v_row[of_v.scale];
  }
  read_part<T, WHOLE>(k, k_scale, at.there, nk, numbers_of<T>(p.ka, p.kb, at, of_k));
  read_part<T, WHOLE>(v, v_scale, at.there, nv, numbers_of<T>(p.va, p.vb, at, of_v));
}

int rows_call(const TpaFp4RowsArgs* a, void* stream, bool write) {
  if (!a) return TPA_ERR_NULL;
  if (a->dtype != TPA_DTYPE_F32 && a->dtype != TPA_DTYPE_BF16) return TPA_ERR_DTYPE;
  if (a->B <= 0 || a->l <= 0 || a->H <= 0 || a->dk <= 0 || a->dv <= 0 || a->rk <= 0 || a->page_size <= 0 || a->num_slots < 0) return TPA_ERR_SHAPE;
  if (a->num_slots % a->page_size || a->rk > 16384 || a->H > 8192 || a->dk > 8192 || a->dv > 8192) return TPA_ERR_SHAPE;
  const int64_t tokens = (int64_t)a->B * a->l;
  if (tokens > INT32_MAX) return TPA_ERR_SHAPE;
  if (!a->ka.ptr || !a->kb.ptr || !a->va.ptr || !a->vb.ptr || !a->slots) return TPA_ERR_NULL;
  if (a->num_slots && (!a->k_cache.ptr || !a->v_cache.ptr)) return TPA_ERR_NULL;
  RowsParams p{};
  p.ka = a->ka; p.kb = a->kb; p.va = a->va; p.vb = a->vb; p.k_cache = a->k_cache; p.v_cache = a->v_cache;
  p.slots = a->slots; p.page_size = a->page_size; p.num_slots = a->num_slots;
  p.l = a->l; p.H = a->H; p.dk = a->dk; p.dv = a->dv; p.rk = a->rk; p.tokens = (int)tokens;
  const int e = a->dtype == TPA_DTYPE_BF16 ? 8 : 4;  // elements of 16 bytes
  bool whole = a->H % 8 == 0 && a->dk % 8 == 0 && a->dv % 8 == 0;
  for (const TpaFactor* f : {&a->ka, &a->kb, &a->va, &a->vb})
    whole = whole && reinterpret_cast<uintptr_t>(f->ptr) % 16 == 0 && f->stride_b % e == 0 && f->stride_l % e == 0 && f->stride_r % e == 0;
  for (const TpaFactor* f : {&a->k_cache, &a->v_cache})
    whole = whole && reinterpret_cast<uintptr_t>(f->ptr) % 4 == 0 && f->stride_b % 4 == 0 && f->stride_l % 4 == 0 && f->stride_r % 4 == 0;
  p.lanes = 4 * (fp4_blocks(a->dk > a->dv ? a->dk : a->dv) + fp4_blocks(a->H));
  const int64_t groups = (tokens * a->rk * p.lanes + kThreads - 1) / kThreads;
  if (groups * kThreads > UINT32_MAX) return TPA_ERR_SHAPE;
  auto launch = [&](auto kern) {
    hipLaunchKernelGGL(kern, dim3((unsigned)groups), dim3(kThreads), 0, static_cast<hipStream_t>(stream), p);
    return hipGetLastError() == hipSuccess ? TPA_OK : TPA_ERR_LAUNCH;
  };
  if (a->dtype == TPA_DTYPE_BF16) {
    if (write) return whole ? launch(write_kernel<uint16_t, true>) : launch(write_kernel<uint16_t, false>);
    return whole ? launch(read_kernel<uint16_t, true>) : launch(read_kernel<uint16_t, false>);
  }
  if (write) return whole ? launch(write_kernel<float, true>) : launch(write_kernel<float, false>);
  return whole ? launch(read_kernel<float, true>) : launch(read_kernel<float, false>);
}

}  // namespace
}  // namespace tpa

extern "C" size_t tpa_fp4_row_bytes(int32_t H, int32_t D) { return H > 0 && D > 0 ? (size_t)tpa::fp4_row_bytes(H, D) : 0; }
extern "C" int tpa_cache_write_fp4(const TpaFp4RowsArgs* a, void* stream) { return tpa::rows_call(a, stream, true); }
extern "C" int tpa_cache_read_fp4(const TpaFp4RowsArgs* a, void* stream) { return tpa::rows_call(a, stream, false); }
