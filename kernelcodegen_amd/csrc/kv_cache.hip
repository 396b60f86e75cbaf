// Writing keys and values into a paged cache, quantised to e4m3 where the cache is, and reading
// them back.
//
// e4m3 rows share one power of two, 2^(x - 127): a float type loses nothing to a power of two that
// it would not lose to any other scale (but the one binade at its small end), the scaling of a row
// is exact, and every dequantised value is a bf16 number.  A row is D / 8 lanes of eight elements,
// as everywhere.
// Reading is bound by memory (32768 tokens, 8 heads of 128, e4m3 to bf16: 33 us, 202 MB, 6.1 TB/s);
// writing by its instructions and by the comparison of the slots (8191 tokens of the same: 14.5 us for
// 50 MB, 12.9 without the comparison, where a copy of as much takes 8.5; into a bf16 cache 16.2 us for 67 MB).  Of
// about 180 instructions for eight elements a third quantises; most others form addresses of rows and slots, and the
// slot is loaded once more for each row.
#include "kv_cache.h"

namespace kcg {

template <typename T, typename C>
struct KvMoveArgs {
  Rows<T> k, v;
  KvCache<C> cache;
  const int32_t *slots;
  int S, tokens;
  int first, end;  // writing: the tokens of this launch
};

// The least x in [1, 254] with amax <= 448 * 2^(x - 127), from the bits of a finite amax: 448 is 1.75 * 2^8.
__device__ __forceinline__ int e4m3_exponent(unsigned bits) {
  const int x = static_cast<int>(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return x < 1 ? 1 : x;
}

constexpr unsigned kInfBits = 0x7f800000u;

__device__ __forceinline__ unsigned magnitude_bits(float x) { return __builtin_bit_cast(unsigned, x) & 0x7fffffffu; }

// Eight elements of a row into the cache.
template <int LANES>
__device__ __forceinline__ void cache_store8(uint16_t *to, uint8_t *, float (&x)[8], int) {
  store8<true>(to, x);
}
template <int LANES>
__device__ __forceinline__ void cache_store8(uint8_t *to, uint8_t *exponent, float (&x)[8], int lane_in_row) {
  // magnitudes compare as their bits do; infinity and NaN are the largest
  unsigned top = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) top = max(top, magnitude_bits(x[j]));
  top = row_max<LANES>(top);
  unsigned nan[2] = {0, 0};
  if (top >= kInfBits) {  // rare: the row's largest finite magnitude, and which elements become NaN
    top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const bool finite = magnitude_bits(x[j]) < kInfBits;
      if (finite) top = max(top, magnitude_bits(x[j]));
      else nan[j / 4] |= 0x7fu << (8 * (j % 4));
      x[j] = finite ? x[j] : 0.0f;
    }
    top = row_max<LANES>(top);
  }
  const int e = e4m3_exponent(top);
  const float inverse = exponent_to_scale(254 - e);
  uint2_t q;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    int p = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * w] * inverse, x[4 * w + 1] * inverse, 0, false);
    p = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * w + 2] * inverse, x[4 * w + 3] * inverse, p, true);
    q[w] = static_cast<unsigned>(p) | nan[w];
  }
  *reinterpret_cast<uint2_t *>(to) = q;
  if (lane_in_row == 0) *exponent = static_cast<uint8_t>(e);
}

// GROUP tokens to a workgroup, all their heads.  A token that names the same slot as a later one is
// left out, so that the last one is what the slot holds, whichever workgroup runs first: the
// workgroup compares its GROUP slots with all that follow.  That is 4 bytes read per following
// token and workgroup (2 tokens^2 / GROUP bytes, from L2); the first rows are on their way meanwhile
// (later ones ahead of their turn gained nothing: the chip is full of waves).
template <typename T, typename C, int D, bool VEC, int GROUP>
__global__ __launch_bounds__(256) void kv_cache_write_kernel(const KvMoveArgs<const T, C> a) {
  constexpr int LANES = D / 8, PER = 256 / LANES;
  __shared__ int later[GROUP];
  const int t0 = a.first + blockIdx.x * GROUP, end = a.end;
  const int lane = threadIdx.x % LANES;
  const int heads = a.cache.shape.heads, rows = 2 * heads;  // of a token: keys, then values
  const int count = min(GROUP, end - t0);
  // this lane's rows: PER apart in the order (token, row)
  const int step_g = PER / rows, step_r = PER - step_g * rows;
  int g = threadIdx.x / LANES / rows, r = threadIdx.x / LANES - g * rows;
  auto load = [&](int g, int r, float(&x)[8]) {
    const int t = t0 + g, b = a.S == a.tokens ? 0 : t / a.S, s = t - b * a.S;
    load8<VEC>((r >= heads ? a.v.at(b, s, r - heads) : a.k.at(b, s, r)) + 8 * lane, x);
  };
  float x[8];
  if (g < count) load(g, r, x);
  int slot[GROUP];
#pragma unroll
  for (int g = 0; g < GROUP; ++g) slot[g] = t0 + g < end ? a.slots[t0 + g] : -1;
  if (threadIdx.x < GROUP) later[threadIdx.x] = 0;
  __syncthreads();
  auto compare = [&](int t, int s) {
    unsigned least = 0xffffffffu;  // 0 if s is one of the slots
#pragma unroll
    for (int g = 0; g < GROUP; ++g) least = min(least, static_cast<unsigned>(s ^ slot[g]));
    if (least == 0) {
#pragma unroll
      for (int g = 0; g < GROUP; ++g)
        if (s == slot[g] && t > t0 + g) later[g] = 1;
    }
  };
  int t = t0 + 1 + threadIdx.x;
  for (; t + 7 * 256 < end; t += 8 * 256) {  // eight loads under way
    int s[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) s[k] = a.slots[t + 256 * k];
#pragma unroll
    for (int k = 0; k < 8; ++k) compare(t + 256 * k, s[k]);
  }
  for (; t < end; t += 256) compare(t, a.slots[t]);
  __syncthreads();
  while (g < count) {
    const bool is_v = r >= heads;
    const int64_t row = later[g] ? -1 : kv_slot_row(a.cache.shape, a.slots[t0 + g], is_v ? r - heads : r);
    if (row >= 0)
      cache_store8<LANES>((is_v ? a.cache.v : a.cache.k) + row * D + 8 * lane,
                          (is_v ? a.cache.v_exp : a.cache.k_exp) + row, x, lane);
    g += step_g;
    r += step_r;
    if (r >= rows) {
      r -= rows;
      ++g;
    }
    if (g < count) load(g, r, x);
  }
}

// `group` tokens to a workgroup; up to ROWS rows of a lane are on their way at a time.  STREAM: outputs past the caches.
template <typename T, typename C, int D, bool VEC, int ROWS, bool STREAM>
__global__ __launch_bounds__(256) void kv_cache_read_kernel(const KvMoveArgs<T, C> a, int group) {
  constexpr int LANES = D / 8, PER = 256 / LANES;
  const int lane = threadIdx.x % LANES;
  const int heads = a.cache.shape.heads, rows = 2 * heads;
  const int t0 = blockIdx.x * group, count = min(group, a.tokens - t0);
  const int step_g = PER / rows, step_r = PER - step_g * rows;
  int g = threadIdx.x / LANES / rows, r = threadIdx.x / LANES - g * rows;
  while (g < count) {
    float x[ROWS][8];
    T *to[ROWS];
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
      to[k] = nullptr;
      if (g < count) {
        const int t = t0 + g, b = a.S == a.tokens ? 0 : t / a.S, s = t - b * a.S;
        const bool is_v = r >= heads;
        const int h = is_v ? r - heads : r;
        to[k] = (is_v ? a.v.at(b, s, h) : a.k.at(b, s, h)) + 8 * lane;
        const int64_t row = kv_slot_row(a.cache.shape, a.slots[t], h);
        if (row >= 0) {
          cache_load8((is_v ? a.cache.v : a.cache.k) + row * D + 8 * lane, (is_v ? a.cache.v_exp : a.cache.k_exp) + row,
                      x[k]);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) x[k][j] = 0.0f;
        }
      }
      g += step_g;
      r += step_r;
      if (r >= rows) {
        r -= rows;
        ++g;
      }
    }
#pragma unroll
    for (int k = 0; k < ROWS; ++k)
      if (to[k]) store8<VEC, STREAM>(to[k], x[k]);
  }
}

template <typename T, typename C, int D, bool VEC>
int run_write(const KvMoveArgs<const T, C> &a, hipStream_t stream) {
  // Launches of 8192 tokens at most: the comparison grows with their square (131072 tokens, 8 heads of 128:
  // 616 us in one launch, 314 so; 16384: 38 either way), and a later launch writes after an earlier one, as
  // its tokens have to.
  KvMoveArgs<const T, C> part = a;
  for (part.first = 0; part.first < a.tokens; part.first = part.end) {
    part.end = a.tokens - part.first > 8192 ? part.first + 8192 : a.tokens;
    const int n = part.end - part.first;
    // One token to a workgroup where that fills the chip less than once (64 tokens: 3.4 us, with four 5.3);
    // more where there are more workgroups than places (4096: 9.3 with two, 10.9 with four, 10.6 with one;
    // 8191: 15.2 with four, 16.3 with two, 19.8 with one).
    const int e = n < 2048 ? launch(kv_cache_write_kernel<T, C, D, VEC, 1>, dim3(n), dim3(256), 0, stream, part)
                  : n < 6144 ? launch(kv_cache_write_kernel<T, C, D, VEC, 2>, dim3((n + 1) / 2), dim3(256), 0, stream, part)
                             : launch(kv_cache_write_kernel<T, C, D, VEC, 4>, dim3((n + 3) / 4), dim3(256), 0, stream, part);
    if (e) return e;
  }
  return KCG_OK;
}

template <typename T, typename C, int D, bool VEC>
int run_read(const KvMoveArgs<T, C> &a, hipStream_t stream) {
  const int per = 256 / (D / 8), rows = 2 * a.cache.shape.heads;
  // two rows to a lane (8 heads of 128, e4m3 to bf16: 32768 tokens 39.0 us with one, 35.7 with two, 34.5 with four; 512
  // tokens 3.0, 3.4 and 4.3)
  int group = 2 * per / rows;
  if (group < 1) group = 1;
  const dim3 grid((a.tokens + group - 1) / group);
  // Outputs that the L2s hold (4 MiB on each of 8 XCDs) are left in them for the attention that reads them next: 1000
  // tokens and it take 36 us so, 41 past the caches, 8192 tokens (32 MiB) 178 and 212, alone 12.5 and 11.1.  With more
  // the two together take the same either way (12288 tokens: 365 and 362, 32768: 1873 and 1878), and the read alone
  // 29 and 20 with 16384, 52 and 35 with 32768.
  if (VEC && static_cast<int64_t>(a.tokens) * rows * D * static_cast<int64_t>(sizeof(T)) > int64_t{32} << 20)
    return launch(kv_cache_read_kernel<T, C, D, VEC, 2, VEC>, grid, dim3(256), 0, stream, a, group);
  return launch(kv_cache_read_kernel<T, C, D, VEC, 2, false>, grid, dim3(256), 0, stream, a, group);
}

template <bool WRITE, typename T, typename C>
int move(const kcg_kv_cache &cache, const kcg_rows &k, const kcg_rows &v, int dtype, const int32_t *slots, int B, int S,
         hipStream_t stream) {
  const bool vec = rows_aligned16(k, dtype, B, S, cache.heads) && rows_aligned16(v, dtype, B, S, cache.heads);
  using U = std::conditional_t<WRITE, const T, T>;
  const KvMoveArgs<U, C> a = {make_rows<U>(k), make_rows<U>(v), make_cache<C>(cache), slots, S, B * S, 0, 0};
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
  if (!WRITE && k->data == v->data) return KCG_ERR_BAD_ARGUMENT;
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
