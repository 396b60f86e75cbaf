// Writing keys and values into a paged cache, quantised to e4m3 where the cache is, and reading
// them back.
//
// e4m3 rows share one power of two, 2^(x - 127): a float type loses nothing to a power of two that
// it would not lose to any other scale (but the one binade at its small end), the scaling of a row
// is exact, and every dequantised value is a bf16 number.  Both kernels are bound by memory; a row
// is D / 8 lanes of eight elements, as everywhere.
#include "kv_cache.h"

namespace kcg {

template <typename T, typename C>
struct KvMoveArgs {
  Rows<T> k, v;
  KvCache<C> cache;
  const int32_t *slots;
  int S, tokens;
};

// The least x in [1, 254] with amax <= 448 * 2^(x - 127), for a finite amax: 448 is 1.75 * 2^8.
__device__ __forceinline__ int e4m3_exponent(float amax) {
  const unsigned bits = __builtin_bit_cast(unsigned, amax);
  const int x = static_cast<int>(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return x < 1 ? 1 : x;
}

// Eight elements of a row into the cache.
template <int LANES>
__device__ __forceinline__ void cache_store8(uint16_t *to, uint8_t *, const float (&x)[8], int) {
  store8<true>(to, x);
}
template <int LANES>
__device__ __forceinline__ void cache_store8(uint8_t *to, uint8_t *exponent, const float (&x)[8], int lane_in_row) {
  float amax = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float m = fabsf(x[j]);
    amax = m < INFINITY ? fmaxf(amax, m) : amax;
  }
  amax = row_max<LANES>(amax);
  const int e = e4m3_exponent(amax);
  const float inverse = exponent_to_scale(254 - e);
  uint2_t q;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    float y[4];
    unsigned nan = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool finite = fabsf(x[4 * w + j]) < INFINITY;
      y[j] = finite ? x[4 * w + j] * inverse : 0.0f;
      nan |= finite ? 0u : 0x7fu << (8 * j);
    }
    int p = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    p = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], p, true);
    q[w] = static_cast<unsigned>(p) | nan;
  }
  *reinterpret_cast<uint2_t *>(to) = q;
  if (lane_in_row == 0) *exponent = static_cast<uint8_t>(e);
}

// GROUP tokens to a workgroup, all their heads.  A token that names the same slot as a later one is
// left out, so that the last one is what the slot holds, whichever workgroup runs first: the
// workgroup compares its GROUP slots with all that follow.  That is 4 bytes read per following
// token and workgroup (tokens^2 / GROUP * 2 bytes from L2).
template <typename T, typename C, int D, bool VEC, int GROUP>
__global__ __launch_bounds__(256) void kv_cache_write_kernel(const KvMoveArgs<const T, C> a) {
  constexpr int LANES = D / 8, PER = 256 / LANES;
  __shared__ int later[GROUP];
  const int t0 = blockIdx.x * GROUP;
  int slot[GROUP];
#pragma unroll
  for (int g = 0; g < GROUP; ++g) slot[g] = t0 + g < a.tokens ? a.slots[t0 + g] : -1;
  if (threadIdx.x < GROUP) later[threadIdx.x] = 0;
  __syncthreads();
  for (int t = t0 + 1 + threadIdx.x; t < a.tokens; t += 256) {
    const int s = a.slots[t];
#pragma unroll
    for (int g = 0; g < GROUP; ++g)
      if (s == slot[g] && t > t0 + g) later[g] = 1;
  }
  __syncthreads();
  const int lane = threadIdx.x % LANES;
  const int rows = 2 * a.cache.shape.heads;  // of a token: keys, then values
  for (int i = threadIdx.x / LANES; i < GROUP * rows; i += PER) {
    const int g = i / rows, r = i - g * rows;
    const bool is_v = r >= a.cache.shape.heads;
    const int h = is_v ? r - a.cache.shape.heads : r;
    const int t = t0 + g;
    if (t >= a.tokens || later[g]) continue;
    const int64_t row = kv_slot_row(a.cache.shape, a.slots[t], h);
    if (row < 0) continue;
    const int b = t / a.S, s = t - b * a.S;
    float x[8];
    load8<VEC>((is_v ? a.v.at(b, s, h) : a.k.at(b, s, h)) + 8 * lane, x);
    cache_store8<LANES>((is_v ? a.cache.v : a.cache.k) + row * D + 8 * lane,
                        (is_v ? a.cache.v_exp : a.cache.k_exp) + row, x, lane);
  }
}

template <typename T, typename C, int D, bool VEC>
__global__ __launch_bounds__(256) void kv_cache_read_kernel(const KvMoveArgs<T, C> a) {
  constexpr int LANES = D / 8, PER = 256 / LANES;
  const int lane = threadIdx.x % LANES;
  const int rows = 2 * a.cache.shape.heads;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * PER + threadIdx.x / LANES;
  const int t = static_cast<int>(i / rows), r = static_cast<int>(i - static_cast<int64_t>(t) * rows);
  if (t >= a.tokens) return;
  const bool is_v = r >= a.cache.shape.heads;
  const int h = is_v ? r - a.cache.shape.heads : r;
  const int64_t row = kv_slot_row(a.cache.shape, a.slots[t], h);
  float x[8] = {};
  if (row >= 0)
    cache_load8((is_v ? a.cache.v : a.cache.k) + row * D + 8 * lane, (is_v ? a.cache.v_exp : a.cache.k_exp) + row, x);
  const int b = t / a.S, s = t - b * a.S;
  store8<VEC>((is_v ? a.v.at(b, s, h) : a.k.at(b, s, h)) + 8 * lane, x);
}

template <typename T, typename C, int D, bool VEC>
int run_write(const KvMoveArgs<const T, C> &a, hipStream_t stream) {
  // One token to a workgroup fills the chip soonest; from 4096 tokens on it is full anyway and the
  // comparison with the following slots is what grows.
  if (a.tokens < 4096)
    return launch(kv_cache_write_kernel<T, C, D, VEC, 1>, dim3(a.tokens), dim3(256), 0, stream, a);
  return launch(kv_cache_write_kernel<T, C, D, VEC, 16>, dim3((a.tokens + 15) / 16), dim3(256), 0, stream, a);
}

template <typename T, typename C, int D, bool VEC>
int run_read(const KvMoveArgs<T, C> &a, hipStream_t stream) {
  const int64_t rows = static_cast<int64_t>(a.tokens) * 2 * a.cache.shape.heads, per = 256 / (D / 8);
  return launch(kv_cache_read_kernel<T, C, D, VEC>, dim3(static_cast<unsigned>((rows + per - 1) / per)), dim3(256), 0,
                stream, a);
}

template <bool WRITE, typename T, typename C>
int move(const kcg_kv_cache &cache, const kcg_rows &k, const kcg_rows &v, int dtype, const int32_t *slots, int B, int S,
         hipStream_t stream) {
  const bool vec = rows_aligned16(k, dtype, B, S, cache.heads) && rows_aligned16(v, dtype, B, S, cache.heads);
  using U = std::conditional_t<WRITE, const T, T>;
  const KvMoveArgs<U, C> a = {make_rows<U>(k), make_rows<U>(v), make_cache<C>(cache), slots, S, B * S};
#define KCG_PICK(DD, V)                                         \
  if constexpr (WRITE) return run_write<T, C, DD, V>(a, stream); \
  else return run_read<T, C, DD, V>(a, stream)
  if (cache.dim == 64) {
    if (vec) { KCG_PICK(64, true); }
    KCG_PICK(64, false);
  }
  if (vec) { KCG_PICK(128, true); }
  KCG_PICK(128, false);
#undef KCG_PICK
}

template <bool WRITE>
int check_and_move(const kcg_kv_cache *cache, const kcg_rows *k, const kcg_rows *v, int dtype, const int32_t *slots,
                   int B, int S, hipStream_t stream) {
  if (const int e = check_cache(cache)) return e;
  if (!slots) return KCG_ERR_NULL_POINTER;
  if ((dtype != KCG_F32 && dtype != KCG_BF16) || reinterpret_cast<uintptr_t>(slots) % 4) return KCG_ERR_BAD_ARGUMENT;
  if (const int e = check_extents(B, S, cache->heads, cache->dim)) return e;
  if (const int e = check_rows(k, dtype, B, S, cache->heads, cache->dim, !WRITE)) return e;
  if (const int e = check_rows(v, dtype, B, S, cache->heads, cache->dim, !WRITE)) return e;
  if (dtype == KCG_F32)
    return cache->dtype == KCG_E4M3 ? move<WRITE, float, uint8_t>(*cache, *k, *v, dtype, slots, B, S, stream)
                                    : move<WRITE, float, uint16_t>(*cache, *k, *v, dtype, slots, B, S, stream);
  return cache->dtype == KCG_E4M3 ? move<WRITE, uint16_t, uint8_t>(*cache, *k, *v, dtype, slots, B, S, stream)
                                  : move<WRITE, uint16_t, uint16_t>(*cache, *k, *v, dtype, slots, B, S, stream);
}

}  // namespace kcg

extern "C" {

int kcg_kv_cache_write(const kcg_kv_cache *cache, const kcg_rows *k, const kcg_rows *v, int dtype, const int32_t *slots,
                       int32_t B, int32_t S, void *stream) {
  return kcg::check_and_move<true>(cache, k, v, dtype, slots, B, S, static_cast<hipStream_t>(stream));
}

int kcg_kv_cache_read(const kcg_kv_cache *cache, const int32_t *slots, const kcg_rows *k, const kcg_rows *v, int dtype,
                      int32_t B, int32_t S, void *stream) {
  return kcg::check_and_move<false>(cache, k, v, dtype, slots, B, S, static_cast<hipStream_t>(stream));
}

}  // extern "C"
