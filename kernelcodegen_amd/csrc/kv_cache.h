// Host-side checks and the device form of a kcg_kv_cache, shared by the operators that use one.
#pragma once

#include "rows.h"

#include "kv_cache_index.h"

namespace kcg {

// T: uint16_t (bf16) or uint8_t (e4m3)
template <typename T>
struct KvCache {
  T *k, *v;
  uint8_t *k_exp, *v_exp;
  KvShape shape;
};

// 2^(x - 127)
__device__ __forceinline__ float exponent_to_scale(int x) { return __builtin_bit_cast(float, static_cast<unsigned>(x) << 23); }

// Eight elements of a cached row.
__device__ __forceinline__ void cache_load8(const uint16_t *from, const uint8_t *, float (&x)[8]) { load8<true>(from, x); }
__device__ __forceinline__ void cache_load8(const uint8_t *from, const uint8_t *exponent, float (&x)[8]) {
  const uint2_t q = *reinterpret_cast<const uint2_t *>(from);
  const float scale = exponent_to_scale(*exponent);
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const float2_t a = __builtin_amdgcn_cvt_pk_f32_fp8(q[w], false), b = __builtin_amdgcn_cvt_pk_f32_fp8(q[w], true);
    x[4 * w] = a[0] * scale;
    x[4 * w + 1] = a[1] * scale;
    x[4 * w + 2] = b[0] * scale;
    x[4 * w + 3] = b[1] * scale;
  }
}

template <typename T>
inline KvCache<T> make_cache(const kcg_kv_cache &c) {
  int log2_page = 4;
  while ((1 << log2_page) < c.page_size) ++log2_page;
  return {static_cast<T *>(c.k), static_cast<T *>(c.v), c.k_exp, c.v_exp, {c.pages, log2_page, c.heads}};
}

inline int check_cache(const kcg_kv_cache *c) {
  if (!c || !c->k || !c->v) return KCG_ERR_NULL_POINTER;
  if (c->dtype != KCG_BF16 && c->dtype != KCG_E4M3) return KCG_ERR_BAD_ARGUMENT;
  if (c->dtype == KCG_E4M3 && (!c->k_exp || !c->v_exp)) return KCG_ERR_NULL_POINTER;
  if (c->pages <= 0 || c->page_size <= 0 || c->heads <= 0 || c->dim <= 0) return KCG_ERR_BAD_SHAPE;
  if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1)) ||
      (c->dim != 64 && c->dim != 128))
    return KCG_ERR_UNSUPPORTED_SHAPE;
  // slots are 32-bit numbers; rows stay far inside 64 bits
  if (static_cast<int64_t>(c->pages) * c->page_size > 0x7fffffffLL || c->heads > (1 << 16))
    return KCG_ERR_UNSUPPORTED_SHAPE;
  if (!aligned16(c->k) || !aligned16(c->v) ||
      (c->dtype == KCG_E4M3 && (!aligned16(c->k_exp) || !aligned16(c->v_exp))))
    return KCG_ERR_BAD_ARGUMENT;
  return KCG_OK;
}

}  // namespace kcg
