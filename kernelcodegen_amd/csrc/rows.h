// Rows of D elements of strided tensors, eight elements to a lane: D / 8 lanes hold a row.
#pragma once

#include <math.h>

#include "kcg_common.h"

namespace kcg {

typedef unsigned int uint4_t __attribute__((ext_vector_type(4)));
typedef unsigned int uint2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16_pair_t __attribute__((ext_vector_type(2)));

// kcg_rows on the device
template <typename T>
struct Rows {
  T *data;
  int64_t stride_b, stride_s, stride_h;
  __device__ __forceinline__ T *at(int b, int s, int h) const {
    return data + b * stride_b + s * stride_s + h * stride_h;
  }
};

template <typename T>
inline Rows<T> make_rows(const kcg_rows &r) {
  return {static_cast<T *>(r.data), r.stride_b, r.stride_s, r.stride_h};
}

__device__ __forceinline__ float bf16_to_float(uint16_t x) { return __builtin_bit_cast(float, static_cast<unsigned>(x) << 16); }
__device__ __forceinline__ uint16_t float_to_bf16(float x) {
  return __builtin_bit_cast(uint16_t, static_cast<__bf16>(x));
}
__device__ __forceinline__ unsigned float_to_bf16_pair(float a, float b) {
  bf16_pair_t r;
  r[0] = static_cast<__bf16>(a);
  r[1] = static_cast<__bf16>(b);
  return __builtin_bit_cast(unsigned, r);
}

// Eight elements from p as fp32; VEC: p is 16-byte aligned.
template <bool VEC>
__device__ __forceinline__ void load8(const float *p, float (&x)[8]) {
  if (VEC) {
    const float4_t a = *reinterpret_cast<const float4_t *>(p), b = *reinterpret_cast<const float4_t *>(p + 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[j] = a[j];
      x[4 + j] = b[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = p[j];
  }
}
template <bool VEC>
__device__ __forceinline__ void load8(const uint16_t *p, float (&x)[8]) {
  if (VEC) {
    const uint4_t a = *reinterpret_cast<const uint4_t *>(p);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[2 * j] = __builtin_bit_cast(float, a[j] << 16);
      x[2 * j + 1] = __builtin_bit_cast(float, a[j] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = bf16_to_float(p[j]);
  }
}
// STREAM: past the caches, for outputs larger than those that would serve their reader
template <bool STREAM, typename V>
__device__ __forceinline__ void store_vector(V x, void *p) {
  if (STREAM) __builtin_nontemporal_store(x, static_cast<V *>(p));
  else *static_cast<V *>(p) = x;
}
template <bool VEC, bool STREAM = false>
__device__ __forceinline__ void store8(float *p, const float (&x)[8]) {
  if (VEC) {
    store_vector<STREAM>(float4_t{x[0], x[1], x[2], x[3]}, p);
    store_vector<STREAM>(float4_t{x[4], x[5], x[6], x[7]}, p + 4);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) p[j] = x[j];
  }
}
template <bool VEC, bool STREAM = false>
__device__ __forceinline__ void store8(uint16_t *p, const float (&x)[8]) {
  if (VEC) {
    uint4_t a;
#pragma unroll
    for (int j = 0; j < 4; ++j) a[j] = float_to_bf16_pair(x[2 * j], x[2 * j + 1]);
    store_vector<STREAM>(a, p);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) p[j] = float_to_bf16(x[j]);
  }
}

// x of another lane, in registers: lane ^ 1, lane ^ 2, 7 - lane of eight, 15 - lane of sixteen.
template <int CTRL, typename T>
__device__ __forceinline__ T from_lane(T x) {
  return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
constexpr int kXor1 = 0xb1, kXor2 = 0x4e, kMirror8 = 0x141, kMirror16 = 0x140;

// Sum (maximum) over the 8 or 16 lanes that hold a row; every lane gets it, in one order.
template <int LANES>
__device__ __forceinline__ float row_sum(float x) {
  static_assert(LANES == 8 || LANES == 16, "lanes of a row");
  x += from_lane<kXor1>(x);
  x += from_lane<kXor2>(x);
  x += from_lane<kMirror8>(x);
  if (LANES == 16) x += from_lane<kMirror16>(x);
  return x;
}
template <int LANES>
__device__ __forceinline__ unsigned row_max(unsigned x) {
  static_assert(LANES == 8 || LANES == 16, "lanes of a row");
  x = max(x, from_lane<kXor1>(x));
  x = max(x, from_lane<kXor2>(x));
  x = max(x, from_lane<kMirror8>(x));
  if (LANES == 16) x = max(x, from_lane<kMirror16>(x));
  return x;
}

// ---- checks on the host ----

inline int element_bytes(int dtype) { return dtype == KCG_F32 ? 4 : 2; }

// every row starts on a 16-byte boundary (a stride counts only where it is used)
inline bool rows_aligned16(const kcg_rows &r, int dtype, int B, int S, int H) {
  const int64_t n = 16 / element_bytes(dtype);
  return aligned16(r.data) && (B == 1 || r.stride_b % n == 0) && (S == 1 || r.stride_s % n == 0) &&
         (H == 1 || r.stride_h % n == 0);
}

// KCG_OK if `r` can be read as [B][S][H][D] of `dtype` or, `written`, also written.
inline int check_rows(const kcg_rows *r, int dtype, int B, int S, int H, int D, bool written) {
  if (!r || !r->data) return KCG_ERR_NULL_POINTER;
  if (reinterpret_cast<uintptr_t>(r->data) % element_bytes(dtype)) return KCG_ERR_BAD_ARGUMENT;
  if (r->stride_b < 0 || r->stride_s < 0 || r->stride_h < 0) return KCG_ERR_BAD_ARGUMENT;
  if (written) {
    // dimensions by growing stride: each step has to clear all that lies below it
    int64_t stride[3] = {r->stride_b, r->stride_s, r->stride_h};
    int extent[3] = {B, S, H};
    int64_t below = D;
    for (int k = 0; k < 3; ++k) {
      int least = -1;
      for (int i = 0; i < 3; ++i)
        if (extent[i] > 1 && (least < 0 || stride[i] < stride[least])) least = i;
      if (least < 0) break;
      if (stride[least] < below) return KCG_ERR_BAD_ARGUMENT;
      if (stride[least] > (int64_t{1} << 48) / (extent[least] - 1)) return KCG_ERR_BAD_ARGUMENT;  // (more than any memory)
      below += stride[least] * (extent[least] - 1);
      extent[least] = 1;
    }
  }
  return KCG_OK;
}

// The common refusals of [B][S][H][D] extents.
inline int check_extents(int64_t B, int64_t S, int64_t H, int64_t D) {
  if (B <= 0 || S <= 0 || H <= 0 || D <= 0) return KCG_ERR_BAD_SHAPE;
  if (D != 64 && D != 128) return KCG_ERR_UNSUPPORTED_SHAPE;
  if (B * S > 0x7fffffffLL || H > 0x7fffffffLL / D || B * S > 0x7fffffffLL / (H * D)) return KCG_ERR_UNSUPPORTED_SHAPE;
  return KCG_OK;
}

}  // namespace kcg
