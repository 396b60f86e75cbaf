// Per-head RMS norm and position rotation of queries and keys, and its gradient.
//
//   r = (mean x^2 + eps)^(-1/2),  y = w * x * r,  (a, b) -> (a cos t - b sin t, b cos t + a sin t)
//   gradient: g = rotation by -t of dy,  dw = sum g * x * r,  h = g * w,
//             dx = r (h - x r mean(h x r))
//
// Both are bound by memory: a row is read once, held in registers (eight elements to a lane,
// D / 8 lanes to a row) and written once.  A wave works on one token at a time, so the token's
// angles are computed once, one pair to a lane, and shared by all of its heads through LDS.
// The angle is a 64-bit product reduced to a fraction of a turn before it is rounded: position
// 10^6 times a frequency near 1 has only four bits behind the point in fp32.
// Measured on bf16 heads of 128: 16384 tokens of 64 heads 98 us (537 MB, 5.5 TB/s), the gradient for
// 8192 tokens of 40 heads 43 us (252 MB, 5.8 TB/s) and 5 us more for the sum of the weights' shares;
// 8 tokens 3.2 us.  fp32: 4096 tokens of 64 heads 63 us (268 MB, 4.3 TB/s), 8192 124 us, the gradient for 4096
// tokens of 40 heads 53 us with the sum (252 MB).  Requesting a row ahead of its turn made the gradient a
// quarter slower.
#include "rows.h"

namespace kcg {

template <typename T>
struct NormRopeArgs {
  Rows<const T> q, k;    // inputs of the forward pass
  Rows<const T> dq, dk;  // gradients of its outputs (backward)
  Rows<T> q_out, k_out;  // outputs, or gradients of the inputs
  const T *q_weight, *k_weight;
  const int32_t *positions;
  const float *inv_freq;
  float *partial;  // backward: [workgroup][2][D] sums of the weights' gradients
  int S, Hq, rows, rot, tokens;  // rows = Hq + Hk
  int units, unit_rows;          // a token's rows in `units` parts of unit_rows
  float eps;
};

constexpr int kNrWaves = 4;

// cos and sin of the token's angles for this lane's eight elements.  Half pairing: one angle per
// element; interleaved: one per two elements.  Elements that are not rotated get (1, 0), which is not used.
template <int D, bool INTERLEAVED, typename T>
__device__ __forceinline__ void load_turns(const NormRopeArgs<T> &a, int token, float *turns, int lane,
                                           float (&cs)[8], float (&sn)[8]) {
  const int pairs = a.rot / 2;
  __builtin_amdgcn_wave_barrier();
  if (lane < pairs) {
    double t = static_cast<double>(a.positions[token]) * static_cast<double>(a.inv_freq[lane]);
    t *= 0.15915494309189533576888;  // turns
    t -= rint(t);
    float s, c;
    sincospif(2.0f * static_cast<float>(t), &s, &c);
    turns[lane] = c;
    turns[64 + lane] = s;
  }
  // the wave's own LDS operations complete in order; this keeps the compiler from moving them
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  const int e0 = 8 * (lane % (D / 8));
  const bool rotated = e0 < a.rot;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int i = INTERLEAVED ? (e0 + j) / 2 : (e0 >= pairs ? e0 - pairs : e0) + j;
    cs[j] = rotated ? turns[i] : 1.0f;
    sn[j] = rotated ? turns[64 + i] : 0.0f;
  }
}

// Rotates the row by the angles (cs, sn).  Elements behind the rotated ones are left out, not turned by (1, 0),
// for which an infinity beside one would make it NaN.
template <int D, bool INTERLEAVED>
__device__ __forceinline__ void rotate(float (&y)[8], const float (&cs)[8], const float (&sn)[8], int rot, int lane) {
  const bool rotated = 8 * (lane % (D / 8)) < rot;
  if (INTERLEAVED) {
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const float a = y[j], b = y[j + 1];
      y[j] = rotated ? a * cs[j] - b * sn[j] : a;
      y[j + 1] = rotated ? b * cs[j] + a * sn[j] : b;
    }
  } else {
    // the other element of a pair is rot / 2 further on, or back, in lane +- rot / 16
    const int lane_in_row = lane % (D / 8), step = rot / 16;
    const bool first = lane_in_row < step;
    const int from = lane_in_row >= 2 * step ? lane : (first ? lane + step : lane - step);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float other = __shfl(y[j], from);
      const float turned = first ? y[j] * cs[j] - other * sn[j] : y[j] * cs[j] + other * sn[j];
      y[j] = rotated ? turned : y[j];
    }
  }
}

template <typename T, int D, bool VEC, bool INTERLEAVED, bool STREAM>
__global__ __launch_bounds__(64 * kNrWaves) void qk_norm_rope_kernel(const NormRopeArgs<T> a) {
  constexpr int LANES = D / 8, PER = 64 / LANES;  // rows that a wave holds at a time
  __shared__ float turns[kNrWaves][128];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int item = blockIdx.x * kNrWaves + wave;
  const int token = item / a.units, unit = item - token * a.units;
  if (token >= a.tokens) return;
  const int b = token / a.S, s = token - b * a.S;
  const int e0 = 8 * (lane % LANES);
  float cs[8], sn[8], wq[8], wk[8];
  load_turns<D, INTERLEAVED>(a, token, turns[wave], lane, cs, sn);
  load8<VEC>(a.q_weight + e0, wq);
  load8<VEC>(a.k_weight + e0, wk);
  const int end = min(a.rows, (unit + 1) * a.unit_rows);
  for (int row = unit * a.unit_rows + lane / LANES; row - lane / LANES < end; row += PER) {
    const bool live = row < end;
    const bool is_q = row < a.Hq;
    float x[8] = {};
    if (live) load8<VEC>(is_q ? a.q.at(b, s, row) + e0 : a.k.at(b, s, row - a.Hq) + e0, x);
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) sum = __builtin_fmaf(x[j], x[j], sum);
    const float r = __builtin_amdgcn_rsqf(row_sum<LANES>(sum) * (1.0f / D) + a.eps);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = x[j] * r * (is_q ? wq[j] : wk[j]);
    rotate<D, INTERLEAVED>(x, cs, sn, a.rot, lane);
    if (live) store8<VEC, STREAM>(is_q ? a.q_out.at(b, s, row) + e0 : a.k_out.at(b, s, row - a.Hq) + e0, x);
  }
}

// A workgroup takes every gridDim.x-th group of kNrWaves items and keeps its share of the weights'
// gradients in registers until it is done with all of them.
template <typename T, int D, bool VEC, bool INTERLEAVED>
__global__ __launch_bounds__(64 * kNrWaves) void qk_norm_rope_backward_kernel(const NormRopeArgs<T> a) {
  constexpr int LANES = D / 8, PER = 64 / LANES;
  __shared__ float turns[kNrWaves][128];
  __shared__ float sums[kNrWaves][2][D];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int e0 = 8 * (lane % LANES);
  float wq[8], wk[8], gq[8] = {}, gk[8] = {};
  load8<VEC>(a.q_weight + e0, wq);
  load8<VEC>(a.k_weight + e0, wk);
  const int items = a.tokens * a.units;
  for (int item = blockIdx.x * kNrWaves + wave; item < items; item += gridDim.x * kNrWaves) {
    const int token = item / a.units, unit = item - token * a.units;
    const int b = token / a.S, s = token - b * a.S;
    float cs[8], sn[8];
    load_turns<D, INTERLEAVED>(a, token, turns[wave], lane, cs, sn);
#pragma unroll
    for (int j = 0; j < 8; ++j) sn[j] = -sn[j];
    const int end = min(a.rows, (unit + 1) * a.unit_rows);
    for (int row = unit * a.unit_rows + lane / LANES; row - lane / LANES < end; row += PER) {
      const bool live = row < end;
      const bool is_q = row < a.Hq;
      const int h = is_q ? row : row - a.Hq;
      float x[8] = {}, g[8] = {};
      if (live) {
        load8<VEC>(is_q ? a.q.at(b, s, h) + e0 : a.k.at(b, s, h) + e0, x);
        load8<VEC>(is_q ? a.dq.at(b, s, h) + e0 : a.dk.at(b, s, h) + e0, g);
      }
      rotate<D, INTERLEAVED>(g, cs, sn, a.rot, lane);
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) sum = __builtin_fmaf(x[j], x[j], sum);
      const float r = __builtin_amdgcn_rsqf(row_sum<LANES>(sum) * (1.0f / D) + a.eps);
      float dot = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[j] *= r;
        const float gx = g[j] * x[j];
        if (live && is_q) gq[j] += gx;
        if (live && !is_q) gk[j] += gx;
        g[j] *= is_q ? wq[j] : wk[j];
        dot = __builtin_fmaf(g[j], x[j], dot);
      }
      const float mean = row_sum<LANES>(dot) * (1.0f / D);
#pragma unroll
      for (int j = 0; j < 8; ++j) g[j] = r * (g[j] - x[j] * mean);
      if (live) store8<VEC>(is_q ? a.q_out.at(b, s, h) + e0 : a.k_out.at(b, s, h) + e0, g);
    }
  }
  // rows of the wave, then waves of the workgroup, in a fixed order
#pragma unroll
  for (int j = 0; j < 8; ++j) {
#pragma unroll
    for (int m = LANES; m < 64; m *= 2) {
      gq[j] += __shfl_xor(gq[j], m);
      gk[j] += __shfl_xor(gk[j], m);
    }
    if (lane < LANES) {
      sums[wave][0][e0 + j] = gq[j];
      sums[wave][1][e0 + j] = gk[j];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * D; i += 64 * kNrWaves) {
    float t = 0.0f;
    for (int w = 0; w < kNrWaves; ++w) t += sums[w][i / D][i % D];
    a.partial[static_cast<int64_t>(blockIdx.x) * 2 * D + i] = t;
  }
}

// Adds the workgroups' shares: 16 columns to a workgroup, 64 threads to a column, so that the up to 16
// loads of a thread are under way together (1024 shares of 256 columns: 20 us with 16 threads to a
// column, 4 with 64).
template <typename T, int D>
__global__ __launch_bounds__(1024) void qk_norm_rope_weight_sum_kernel(const float *__restrict__ partial, int groups,
                                                                       T *__restrict__ gq, T *__restrict__ gk) {
  __shared__ float sums[64][17];
  const int c = threadIdx.x % 16, r = threadIdx.x / 16;
  const int column = blockIdx.x * 16 + c;
  float t = 0.0f;
#pragma unroll 8
  for (int i = r; i < groups; i += 64) t += partial[static_cast<int64_t>(i) * 2 * D + column];
  sums[r][c] = t;
  __syncthreads();
  if (r < 8) {
    t = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) t += sums[8 * i + r][c];
  }
  __syncthreads();
  if (r < 8) sums[r][c] = t;
  __syncthreads();
  if (r == 0) {
#pragma unroll
    for (int i = 1; i < 8; ++i) t += sums[i][c];
    T *to = column < D ? gq + column : gk + column - D;
    if constexpr (sizeof(T) == 4) *to = t;
    else *to = float_to_bf16(t);
  }
}

// Parts a token's rows are cut into: few tokens would not fill the chip with a wave each.
inline int norm_rope_units(int64_t tokens, int rows, int D) {
  const int per = 64 / (D / 8);
  const int most = (rows + per - 1) / per;
  int64_t units = 1;
  while (units < most && tokens * units < 4096) units *= 2;
  return static_cast<int>(units < most ? units : most);
}

inline int unit_rows(int rows, int units, int D) {
  const int per = 64 / (D / 8);
  return ((rows + units - 1) / units + per - 1) / per * per;
}

constexpr int kNrMaxGroups = 1024;

inline int backward_groups(int64_t items) {
  const int64_t g = (items + kNrWaves - 1) / kNrWaves;
  return static_cast<int>(g < kNrMaxGroups ? g : kNrMaxGroups);
}

template <typename T>
NormRopeArgs<T> norm_rope_args(int B, int S, int Hq, int Hk, int D, int rot, float eps) {
  NormRopeArgs<T> a = {};
  a.S = S;
  a.Hq = Hq;
  a.rows = Hq + Hk;
  a.rot = rot;
  a.tokens = B * S;
  a.eps = eps < 1.17549435e-38f ? 1.17549435e-38f : eps;  // (v_rsq_f32 takes no subnormal numbers)
  const int u = norm_rope_units(a.tokens, a.rows, D);
  a.unit_rows = unit_rows(a.rows, u, D);
  a.units = (a.rows + a.unit_rows - 1) / a.unit_rows;
  return a;
}

inline int check_norm_rope(const void *q_weight, const void *k_weight, const int32_t *positions,
                           const float *inv_freq, int dtype, int64_t B, int64_t S, int64_t Hq, int64_t Hk, int64_t D,
                           int rot, int interleaved, float eps) {
  if (!q_weight || !k_weight || !positions || !inv_freq) return KCG_ERR_NULL_POINTER;
  if (dtype != KCG_F32 && dtype != KCG_BF16) return KCG_ERR_BAD_ARGUMENT;
  if (Hq <= 0 || Hk <= 0) return KCG_ERR_BAD_SHAPE;
  if (const int e = check_extents(B, S, Hq + Hk, D)) return e;
  if (rot < 16 || rot > D || rot % 16) return KCG_ERR_UNSUPPORTED_SHAPE;
  if (interleaved != 0 && interleaved != 1) return KCG_ERR_BAD_ARGUMENT;
  if (!(eps >= 0.0f) || isinf(eps)) return KCG_ERR_BAD_ARGUMENT;
  if (reinterpret_cast<uintptr_t>(positions) % 4 || reinterpret_cast<uintptr_t>(inv_freq) % 4 ||
      reinterpret_cast<uintptr_t>(q_weight) % element_bytes(dtype) ||
      reinterpret_cast<uintptr_t>(k_weight) % element_bytes(dtype))
    return KCG_ERR_BAD_ARGUMENT;
  return KCG_OK;
}

template <typename T, int D, bool VEC, bool INTERLEAVED>
int run_norm_rope(const NormRopeArgs<T> &a, T *gq, T *gk, hipStream_t stream) {
  const int64_t items = static_cast<int64_t>(a.tokens) * a.units;
  if (!a.partial) {
    const unsigned grid = static_cast<unsigned>((items + kNrWaves - 1) / kNrWaves);
    // Outputs of the last-level cache's size (256 MiB) and more go past it: 16384 tokens of 64 heads of 128 in
    // bf16 take 99 us so, 106 otherwise.  Smaller ones are left to their reader: 8192 tokens take 52 us past the
    // caches and 57 through them, 4096 24 and 31, but with a pass over the outputs behind 95 either way, and 52 past
    // them and 50 through them (16384: 193 and 187).
    if (VEC && static_cast<int64_t>(a.tokens) * a.rows * D * static_cast<int64_t>(sizeof(T)) >= int64_t{256} << 20)
      return launch(qk_norm_rope_kernel<T, D, VEC, INTERLEAVED, VEC>, dim3(grid), dim3(64 * kNrWaves), 0, stream, a);
    return launch(qk_norm_rope_kernel<T, D, VEC, INTERLEAVED, false>, dim3(grid), dim3(64 * kNrWaves), 0, stream, a);
  }
  const int groups = backward_groups(items);
  if (const int e = launch(qk_norm_rope_backward_kernel<T, D, VEC, INTERLEAVED>, dim3(groups), dim3(64 * kNrWaves), 0,
                           stream, a))
    return e;
  return launch(qk_norm_rope_weight_sum_kernel<T, D>, dim3(2 * D / 16), dim3(1024), 0, stream, a.partial, groups, gq, gk);
}

template <typename T>
int pick_norm_rope(const NormRopeArgs<T> &a, int D, bool vec, bool interleaved, T *gq, T *gk, hipStream_t stream) {
#define KCG_PICK(DD, V) \
  return interleaved ? run_norm_rope<T, DD, V, true>(a, gq, gk, stream) : run_norm_rope<T, DD, V, false>(a, gq, gk, stream)
  if (D == 64) {
    if (vec) KCG_PICK(64, true);
    KCG_PICK(64, false);
  }
  if (vec) KCG_PICK(128, true);
  KCG_PICK(128, false);
#undef KCG_PICK
}

template <typename T>
int norm_rope(const kcg_rows *q, const kcg_rows *k, const kcg_rows *dq, const kcg_rows *dk, const kcg_rows *q_out,
              const kcg_rows *k_out, const void *q_weight, const void *k_weight, void *gq, void *gk,
              const int32_t *positions, const float *inv_freq, int dtype, int B, int S, int Hq, int Hk, int D, int rot,
              int interleaved, float eps, void *workspace, hipStream_t stream) {
  NormRopeArgs<T> a = norm_rope_args<T>(B, S, Hq, Hk, D, rot, eps);
  a.q = make_rows<const T>(*q);
  a.k = make_rows<const T>(*k);
  a.q_out = make_rows<T>(*q_out);
  a.k_out = make_rows<T>(*k_out);
  a.q_weight = static_cast<const T *>(q_weight);
  a.k_weight = static_cast<const T *>(k_weight);
  a.positions = positions;
  a.inv_freq = inv_freq;
  bool vec = rows_aligned16(*q, dtype, B, S, Hq) && rows_aligned16(*k, dtype, B, S, Hk) &&
             rows_aligned16(*q_out, dtype, B, S, Hq) && rows_aligned16(*k_out, dtype, B, S, Hk) &&
             aligned16(q_weight) && aligned16(k_weight);
  if (workspace) {
    a.dq = make_rows<const T>(*dq);
    a.dk = make_rows<const T>(*dk);
    a.partial = static_cast<float *>(workspace);
    vec = vec && rows_aligned16(*dq, dtype, B, S, Hq) && rows_aligned16(*dk, dtype, B, S, Hk);
  }
  return pick_norm_rope<T>(a, D, vec, interleaved != 0, static_cast<T *>(gq), static_cast<T *>(gk), stream);
}

}  // namespace kcg

extern "C" {

int kcg_qk_norm_rope(const kcg_rows *q, const kcg_rows *k, const kcg_rows *q_out, const kcg_rows *k_out,
                     const void *q_weight, const void *k_weight, const int32_t *positions, const float *inv_freq,
                     int dtype, int32_t B, int32_t S, int32_t Hq, int32_t Hk, int32_t D, int32_t rot_dim,
                     int interleaved, float eps, void *stream) {
  if (const int e = kcg::check_norm_rope(q_weight, k_weight, positions, inv_freq, dtype, B, S, Hq, Hk, D, rot_dim,
                                         interleaved, eps))
    return e;
  if (const int e = kcg::check_rows(q, dtype, B, S, Hq, D, false)) return e;
  if (const int e = kcg::check_rows(k, dtype, B, S, Hk, D, false)) return e;
  if (const int e = kcg::check_rows(q_out, dtype, B, S, Hq, D, true)) return e;
  if (const int e = kcg::check_rows(k_out, dtype, B, S, Hk, D, true)) return e;
  if (q_out->data == k_out->data) return KCG_ERR_BAD_ARGUMENT;
  hipStream_t st = static_cast<hipStream_t>(stream);
  return dtype == KCG_F32
             ? kcg::norm_rope<float>(q, k, nullptr, nullptr, q_out, k_out, q_weight, k_weight, nullptr, nullptr,
                                     positions, inv_freq, dtype, B, S, Hq, Hk, D, rot_dim, interleaved, eps, nullptr, st)
             : kcg::norm_rope<uint16_t>(q, k, nullptr, nullptr, q_out, k_out, q_weight, k_weight, nullptr, nullptr,
                                        positions, inv_freq, dtype, B, S, Hq, Hk, D, rot_dim, interleaved, eps, nullptr,
                                        st);
}

int64_t kcg_qk_norm_rope_backward_ws_bytes(int32_t B, int32_t S, int32_t Hq, int32_t Hk, int32_t D) {
  if (Hq <= 0 || Hk <= 0 || kcg::check_extents(B, S, static_cast<int64_t>(Hq) + Hk, D)) return 0;
  const auto a = kcg::norm_rope_args<float>(B, S, Hq, Hk, D, 16, 0.0f);
  return int64_t{kcg::backward_groups(static_cast<int64_t>(a.tokens) * a.units)} * 2 * D * 4;
}

int kcg_qk_norm_rope_backward(const kcg_rows *dq, const kcg_rows *dk, const kcg_rows *q, const kcg_rows *k,
                              const kcg_rows *grad_q, const kcg_rows *grad_k, const void *q_weight,
                              const void *k_weight, void *grad_q_weight, void *grad_k_weight, const int32_t *positions,
                              const float *inv_freq, int dtype, int32_t B, int32_t S, int32_t Hq, int32_t Hk, int32_t D,
                              int32_t rot_dim, int interleaved, float eps, void *workspace, int64_t workspace_bytes,
                              void *stream) {
  if (const int e = kcg::check_norm_rope(q_weight, k_weight, positions, inv_freq, dtype, B, S, Hq, Hk, D, rot_dim,
                                         interleaved, eps))
    return e;
  for (const kcg_rows *r : {dq, q})
    if (const int e = kcg::check_rows(r, dtype, B, S, Hq, D, false)) return e;
  for (const kcg_rows *r : {dk, k})
    if (const int e = kcg::check_rows(r, dtype, B, S, Hk, D, false)) return e;
  if (const int e = kcg::check_rows(grad_q, dtype, B, S, Hq, D, true)) return e;
  if (const int e = kcg::check_rows(grad_k, dtype, B, S, Hk, D, true)) return e;
  if (!grad_q_weight || !grad_k_weight || !workspace) return KCG_ERR_NULL_POINTER;
  if (reinterpret_cast<uintptr_t>(grad_q_weight) % kcg::element_bytes(dtype) ||
      reinterpret_cast<uintptr_t>(grad_k_weight) % kcg::element_bytes(dtype) || !kcg::aligned16(workspace) ||
      workspace_bytes < kcg_qk_norm_rope_backward_ws_bytes(B, S, Hq, Hk, D) || grad_q->data == grad_k->data ||
      grad_q_weight == grad_k_weight)
    return KCG_ERR_BAD_ARGUMENT;
  hipStream_t st = static_cast<hipStream_t>(stream);
  return dtype == KCG_F32
             ? kcg::norm_rope<float>(q, k, dq, dk, grad_q, grad_k, q_weight, k_weight, grad_q_weight, grad_k_weight,
                                     positions, inv_freq, dtype, B, S, Hq, Hk, D, rot_dim, interleaved, eps, workspace,
                                     st)
             : kcg::norm_rope<uint16_t>(q, k, dq, dk, grad_q, grad_k, q_weight, k_weight, grad_q_weight, grad_k_weight,
                                        positions, inv_freq, dtype, B, S, Hq, Hk, D, rot_dim, interleaved, eps,
                                        workspace, st);
}

}  // extern "C"
