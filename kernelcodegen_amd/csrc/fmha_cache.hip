// Attention of the newest tokens (one, a chain or a tree of drafts) over a paged cache.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q.k_j - m),  over the keys that the query sees.
#include "kv_cache.h"

namespace kcg {

template <typename C>
struct FmhaCacheArgs {
  Rows<const uint16_t> q;
  Rows<void> out;
  KvCache<C> cache;
  const int32_t *table, *context, *drafts;
  const uint64_t *tree;
  int B, N, Hq, width;
  float scale;
};

// One wave to a query head of a token: D / 8 lanes to a key, so 512 / D keys at a time, each with a
// running maximum, sum and output of its own that are joined at the end.
template <typename C, typename O, int D, bool VEC>
__global__ __launch_bounds__(256) void fmha_cache_kernel(const FmhaCacheArgs<C> a) {
  constexpr int LANES = D / 8, PER = 64 / LANES;
  const int lane = threadIdx.x & 63;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (item >= static_cast<int64_t>(a.B) * a.N * a.Hq) return;
  const int h = static_cast<int>(item % a.Hq), n = static_cast<int>(item / a.Hq % a.N);
  const int b = static_cast<int>(item / a.Hq / a.N);
  const int page = 1 << a.cache.shape.log2_page;
  const KvLens len = kv_lens(a.context[b], a.drafts ? a.drafts[b] : a.N, a.N, static_cast<int64_t>(a.width) * page);
  if (n >= len.queries) return;
  const uint64_t seen = kv_seen(a.tree, static_cast<int64_t>(b) * a.N + n, n, len.drafts);
  const int head = h / (a.Hq / a.cache.shape.heads);
  const int e0 = 8 * (lane % LANES);
  float q[8], acc[8] = {}, m = -INFINITY, l = 0.0f;
  load8<VEC>(a.q.at(b, n, h) + e0, q);
#pragma unroll
  for (int j = 0; j < 8; ++j) q[j] *= a.scale;
  for (int key = lane / LANES; key < len.context + len.drafts; key += PER) {
    if (key >= len.context && !((seen >> (key - len.context)) & 1)) continue;
    const int64_t row = kv_row(a.cache.shape, a.table[static_cast<int64_t>(b) * a.width + (key >> a.cache.shape.log2_page)],
                               head, key & (page - 1));
    if (row < 0) continue;
    float k[8], v[8], s = 0.0f;
    cache_load8(a.cache.k + row * D + e0, a.cache.k_exp + row, k);
    cache_load8(a.cache.v + row * D + e0, a.cache.v_exp + row, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) s = __builtin_fmaf(q[j], k[j], s);
    s = row_sum<LANES>(s);
    const float top = fmaxf(m, s);
    const float keep = top == -INFINITY ? 0.0f : expf(m - top);
    const float p = s == -INFINITY ? 0.0f : expf(s - top);
    l = l * keep + p;
    m = top;
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] = acc[j] * keep + p * v[j];
  }
#pragma unroll
  for (int step = LANES; step < 64; step *= 2) {
    const float m2 = __shfl_xor(m, step), l2 = __shfl_xor(l, step);
    const float top = fmaxf(m, m2);
    const float c1 = m == -INFINITY ? 0.0f : expf(m - top), c2 = m2 == -INFINITY ? 0.0f : expf(m2 - top);
    l = l * c1 + l2 * c2;
    m = top;
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] = acc[j] * c1 + __shfl_xor(acc[j], step) * c2;
  }
  if (lane < LANES) {
    const float r = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] *= r;
    O *to = static_cast<O *>(a.out.data) + b * a.out.stride_b + n * a.out.stride_s + h * a.out.stride_h;
    store8<VEC>(to + e0, acc);
  }
}

template <typename C>
int fmha_cache(const kcg_rows &q, const kcg_kv_cache &cache, const int32_t *table, int width, const int32_t *context,
               const int32_t *drafts, const uint64_t *tree, const kcg_rows &out, int o_dtype, int B, int N, int Hq,
               float scale, hipStream_t stream) {
  FmhaCacheArgs<C> a = {make_rows<const uint16_t>(q), make_rows<void>(out), make_cache<C>(cache), table, context, drafts, tree, B, N, Hq, width, scale};
  const bool vec = rows_aligned16(q, KCG_BF16, B, N, Hq) && rows_aligned16(out, o_dtype, B, N, Hq);
  const dim3 grid(static_cast<unsigned>((static_cast<int64_t>(B) * N * Hq + 3) / 4));
#define KCG_PICK(O, DD, V) return launch(fmha_cache_kernel<C, O, DD, V>, grid, dim3(256), 0, stream, a)
#define KCG_PICK2(O)                     \
  if (cache.dim == 64) {                 \
    if (vec) { KCG_PICK(O, 64, true); }  \
    KCG_PICK(O, 64, false);              \
  }                                      \
  if (vec) { KCG_PICK(O, 128, true); }   \
  KCG_PICK(O, 128, false)
  if (o_dtype == KCG_F32) { KCG_PICK2(float); }
  KCG_PICK2(uint16_t);
#undef KCG_PICK2
#undef KCG_PICK
}

// Shapes and types that both the call and its workspace query check.
inline int check_fmha_cache(const kcg_kv_cache *cache, int64_t width, int64_t B, int64_t N, int64_t Hq) {
  if (const int e = check_cache(cache)) return e;
  if (width <= 0 || B <= 0 || N <= 0 || Hq <= 0) return KCG_ERR_BAD_SHAPE;
  if (N > 64 || Hq % cache->heads) return KCG_ERR_UNSUPPORTED_SHAPE;
  if (width > 0x7fffffffLL / cache->page_size || B > 0x7fffffffLL / width) return KCG_ERR_UNSUPPORTED_SHAPE;
  return check_extents(B, N, Hq, cache->dim);
}

}  // namespace kcg

extern "C" {

int64_t kcg_fmha_cache_ws_bytes(const kcg_kv_cache *cache, int32_t table_width, int32_t B, int32_t N, int32_t Hq) {
  (void)cache, (void)table_width, (void)B, (void)N, (void)Hq;
  return 0;
}

int kcg_fmha_cache(const kcg_rows *q, const kcg_kv_cache *cache, const int32_t *block_table, int32_t table_width,
                   const int32_t *context_lens, const int32_t *draft_lens, const uint64_t *tree_mask,
                   const kcg_rows *out, int o_dtype, int32_t B, int32_t N, int32_t Hq, float scale, void *workspace,
                   int64_t workspace_bytes, void *stream) {
  if (const int e = kcg::check_fmha_cache(cache, table_width, B, N, Hq)) return e;
  if (!block_table || !context_lens) return KCG_ERR_NULL_POINTER;
  if (o_dtype != KCG_F32 && o_dtype != KCG_BF16) return KCG_ERR_BAD_ARGUMENT;
  if (const int e = kcg::check_rows(q, KCG_BF16, B, N, Hq, cache->dim, false)) return e;
  if (const int e = kcg::check_rows(out, o_dtype, B, N, Hq, cache->dim, true)) return e;
  if (!(fabsf(scale) < INFINITY) || reinterpret_cast<uintptr_t>(block_table) % 4 ||
      reinterpret_cast<uintptr_t>(context_lens) % 4 || reinterpret_cast<uintptr_t>(draft_lens) % 4 ||
      reinterpret_cast<uintptr_t>(tree_mask) % 8 || (workspace && !kcg::aligned16(workspace)) || workspace_bytes < 0)
    return KCG_ERR_BAD_ARGUMENT;
  hipStream_t st = static_cast<hipStream_t>(stream);
  return cache->dtype == KCG_E4M3
             ? kcg::fmha_cache<uint8_t>(*q, *cache, block_table, table_width, context_lens, draft_lens, tree_mask, *out,
                                        o_dtype, B, N, Hq, scale, st)
             : kcg::fmha_cache<uint16_t>(*q, *cache, block_table, table_width, context_lens, draft_lens, tree_mask, *out,
                                         o_dtype, B, N, Hq, scale, st);
}

}  // extern "C"
