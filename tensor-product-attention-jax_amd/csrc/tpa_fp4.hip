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
  int64_t tokens;  // B * l
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
// (token, lane of its row) of a thread; blockIdx.y = rank, K's and then V's
struct Place {
  bool of_v;
  int rank, D, lane;
  int64_t token, slot;
  const TpaFactor *a, *b, *cache;
};
__device__ __forceinline__ bool place_of(const RowsParams& p, Place& at) {
  at.of_v = (int)blockIdx.y >= p.rk;
  at.rank = (int)blockIdx.y - (at.of_v ? p.rk : 0);
  at.D = at.of_v ? p.dv : p.dk;
  const int lanes = 4 * (fp4_blocks(at.D) + fp4_blocks(p.H));
  const int64_t id = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  at.token = id / lanes;
  at.lane = (int)(id - at.token * lanes);
  if (at.token >= p.tokens) return false;
  at.slot = p.slots[at.token];
  at.a = at.of_v ? &p.va : &p.ka;
  at.b = at.of_v ? &p.vb : &p.kb;
  at.cache = at.of_v ? &p.v_cache : &p.k_cache;
  return true;
}
__device__ __forceinline__ uint8_t* row_of(const RowsParams& p, const Place& at) {
  const int64_t page = at.slot / p.page_size, in_page = at.slot - page * p.page_size;
  return static_cast<uint8_t*>(const_cast<void*>(at.cache->ptr)) + page * at.cache->stride_b + in_page * at.cache->stride_l + at.rank * at.cache->stride_r;
}
template <typename T>
__device__ __forceinline__ T* numbers_of(const RowsParams& p, const Place& at, const Part& part) {
  const TpaFactor& f = part.of_a ? *at.a : *at.b;
  const int64_t b = at.token / p.l, i = at.token - b * p.l;
  return static_cast<T*>(const_cast<void*>(f.ptr)) + b * f.stride_b + i * f.stride_l + at.rank * f.stride_r + part.first;
}

// WHOLE: sizes that are multiples of 8, rows at multiples of 16 bytes (the cache's of 4)
template <typename T, bool WHOLE>
__global__ __launch_bounds__(kThreads) void write_kernel(RowsParams p) {
  Place at;
  if (!place_of(p, at) || at.slot < 0 || at.slot >= p.num_slots) return;
  const Part part = part_of(at.lane, p.H, at.D);
  const int n = min(8, part.n - part.first);  // none for lanes past the end of a short block
  uint32_t x[8] = {};                          // bits of fp32
  if (n > 0) {
    const T* from = numbers_of<const T>(p, at, part);
    if constexpr (WHOLE && sizeof(T) == 2) {
      const u32x4 w = *reinterpret_cast<const u32x4*>(from);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[2 * j] = w[j] << 16;
        x[2 * j + 1] = w[j] & 0xffff0000u;
      }
    } else if constexpr (WHOLE) {
      const u32x4 lo = *reinterpret_cast<const u32x4*>(from), hi = *reinterpret_cast<const u32x4*>(from + 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[j] = lo[j];
        x[4 + j] = hi[j];
      }
    } else {
      for (int j = 0; j < 8; ++j)
        if (j < n) x[j] = __float_as_uint(load_as_f32(from + j));
    }
  }
  // the bits of magnitudes are ordered as these are, those of infinity and NaN above all others
  uint32_t most = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) most = max(most, x[j] & 0x7fffffffu);
  most = max(most, (uint32_t)lanes_of<0xB1>((int)most));  // the four lanes of the block
  most = max(most, (uint32_t)lanes_of<0x4E>((int)most));
  const int exponent = (int)(most >> 23);
  const bool finite = exponent < 255;
  // floor(log2 m) - 2 + 127, one more where m > 7.25 * 2^e: a significand over 1.8125
  const uint32_t scale = finite ? (uint32_t)max(2, min(exponent - 2 + ((most & 0x7fffffu) > 0x680000u), 252)) : 255u;
  if (n <= 0) return;
  uint32_t codes = 0;
  if (finite) {
    const float s = fp4_scale(scale);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, __uint_as_float(x[0]), __uint_as_float(x[1]), s, 0);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, __uint_as_float(x[2]), __uint_as_float(x[3]), s, 1);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, __uint_as_float(x[4]), __uint_as_float(x[5]), s, 2);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, __uint_as_float(x[6]), __uint_as_float(x[7]), s, 3);
  }
  uint8_t* const row = row_of(p, at);
  if constexpr (WHOLE) {
    *reinterpret_cast<uint32_t*>(row + part.codes) = codes;
  } else {
    for (int j = 0; j < 4; ++j)
      if (2 * j < n) row[part.codes + j] = (uint8_t)(codes >> (8 * j));
  }
  if (part.first % 32 == 0) row[part.scale] = (uint8_t)scale;
}

template <typename T, bool WHOLE>
__global__ __launch_bounds__(kThreads) void read_kernel(RowsParams p) {
  Place at;
  if (!place_of(p, at)) return;
  const Part part = part_of(at.lane, p.H, at.D);
  const int n = min(8, part.n - part.first);
  if (n <= 0) return;
  float x[8] = {};
  if (at.slot >= 0 && at.slot < p.num_slots) {
    const uint8_t* const row = row_of(p, at);
    uint32_t codes = 0;
    if constexpr (WHOLE) {
      codes = *reinterpret_cast<const uint32_t*>(row + part.codes);
    } else {
      for (int j = 0; j < 4; ++j)
        if (2 * j < n) codes |= (uint32_t)row[part.codes + j] << (8 * j);
    }
    fp4_f32x8(codes, fp4_scale(row[part.scale]), x);
  }
  T* const to = numbers_of<T>(p, at, part);
  if constexpr (WHOLE && sizeof(T) == 2) {
    *reinterpret_cast<u32x4*>(to) = u32x4{pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7])};
  } else if constexpr (WHOLE) {
    *reinterpret_cast<f32x4*>(to) = f32x4{x[0], x[1], x[2], x[3]};
    *reinterpret_cast<f32x4*>(to + 4) = f32x4{x[4], x[5], x[6], x[7]};
  } else {
    for (int j = 0; j < 8; ++j)
      if (j < n) store_from_f32(to + j, x[j]);
  }
}

int rows_call(const TpaFp4RowsArgs* a, void* stream, bool write) {
  if (!a) return TPA_ERR_NULL;
  if (a->dtype != TPA_DTYPE_F32 && a->dtype != TPA_DTYPE_BF16) return TPA_ERR_DTYPE;
  if (a->B <= 0 || a->l <= 0 || a->H <= 0 || a->dk <= 0 || a->dv <= 0 || a->rk <= 0 || a->page_size <= 0 || a->num_slots < 0) return TPA_ERR_SHAPE;
  if (a->num_slots % a->page_size || a->rk > 16384 || a->H > 8192 || a->dk > 8192 || a->dv > 8192) return TPA_ERR_SHAPE;
  const int64_t tokens = (int64_t)a->B * a->l, lanes = 4 * (fp4_blocks(a->dk > a->dv ? a->dk : a->dv) + fp4_blocks(a->H));
  const int64_t groups = (tokens * lanes + kThreads - 1) / kThreads;
  if (tokens > INT32_MAX || groups > INT32_MAX) return TPA_ERR_SHAPE;
  if (!a->ka.ptr || !a->kb.ptr || !a->va.ptr || !a->vb.ptr || !a->slots) return TPA_ERR_NULL;
  if (a->num_slots && (!a->k_cache.ptr || !a->v_cache.ptr)) return TPA_ERR_NULL;
  RowsParams p{};
  p.ka = a->ka; p.kb = a->kb; p.va = a->va; p.vb = a->vb; p.k_cache = a->k_cache; p.v_cache = a->v_cache;
  p.slots = a->slots; p.page_size = a->page_size; p.num_slots = a->num_slots;
  p.l = a->l; p.H = a->H; p.dk = a->dk; p.dv = a->dv; p.rk = a->rk; p.tokens = tokens;
  const int e = a->dtype == TPA_DTYPE_BF16 ? 8 : 4;  // elements of 16 bytes
  bool whole = a->H % 8 == 0 && a->dk % 8 == 0 && a->dv % 8 == 0;
  for (const TpaFactor* f : {&a->ka, &a->kb, &a->va, &a->vb})
    whole = whole && reinterpret_cast<uintptr_t>(f->ptr) % 16 == 0 && f->stride_b % e == 0 && f->stride_l % e == 0 && f->stride_r % e == 0;
  for (const TpaFactor* f : {&a->k_cache, &a->v_cache})
    whole = whole && reinterpret_cast<uintptr_t>(f->ptr) % 4 == 0 && f->stride_b % 4 == 0 && f->stride_l % 4 == 0 && f->stride_r % 4 == 0;
  auto launch = [&](auto kern) {
    hipLaunchKernelGGL(kern, dim3((unsigned)groups, 2 * a->rk), dim3(kThreads), 0, static_cast<hipStream_t>(stream), p);
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
