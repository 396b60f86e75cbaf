// Attention of the newest tokens (one, a chain or a tree of drafts) over a paged cache.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(c q.k_j - m),  c = scale log2(e), over the keys that
//   the query sees.
//
// Few queries read many keys, so the keys are what is split: into units of whole 32-key chunks, a unit
// to a workgroup, and inside it a contiguous range of chunks to each of the four waves.  The N * Hq /
// heads query rows that share a key head are the 32 or 64 columns of the wave's matrix products.
//
//  * Every wave streams its own chunks through LDS of its own, one buffer of K and one of V, with direct
//    global -> LDS loads: nothing is shared before the end, so there is no barrier in the loop and a wave
//    waits only for its own loads (vmcnt).  The next K is under way while weights and output are computed,
//    the next V while the scores are; the other workgroups of the CU cover the rest.  (A ring of two of each
//    took twice the LDS and the same time, and with bf16 pages of 128 left one workgroup to a CU: 96 us
//    against 72 for 8 x 16 drafts over 8192 keys.)  One variant has no registers left for the lanes' load offsets
//    and keeps them in scratch memory: with fp32 output, bf16 pages of 128 and two tiles a reload sits between
//    the requests of a chunk's K, each of which then waits for the one before.
//  * S^T = K . Q^T (v_mfma_f32_32x32x16_bf16): the A operand is K rows as ds_read_b128, e4m3 bytes
//    becoming bf16 with the row's power of two in the conversion itself; B is Q, in registers.  A lane
//    then holds one query and 16 of the 32 keys, which is the B operand of O^T += V^T . P^T as it
//    stands.  V^T comes from V's natural rows by the transposing LDS reads (b8 or b16); V's powers of
//    two go into P, where they cost nothing in precision.
//  * The sum over d may run in any order, so an e4m3 lane takes the 16 bytes of one ds_read_b128 as
//    two steps' worth of its row, and Q is loaded to match.
//  * LDS rows are unpadded (a direct load fills 1024 consecutive bytes); 16-byte pieces sit at
//    piece ^ swizzle(row), applied to the global address on loading and to the LDS address on
//    reading, so that 16 lanes of a read hit 16 different 16-byte columns of the banks.
//  * Only chunks that reach beyond the context, or touch a page that the cache does not have, look at
//    masks.  There, V rows that nobody sees are zeroed in LDS (their weight is 0, and 0 * NaN is not),
//    and values that are not finite are taken out of the product and added to the rows that see them.
//  * How many chunks make a unit follows from the lengths, which are on the device: every wave sums
//    them up and finds its unit (no host synchronisation, equal work for ragged batches); for more than 64
//    sequences a launch of one workgroup does that first.  A sequence that fits one unit is written at
//    once; the others leave normalised partial outputs and the logarithms of their sums in the
//    workspace, joined by a last launch.
// Measured: 64 single tokens over contexts to 8192, 32 query heads on 8 of 128, e4m3: 105 to 111 us by the lengths
// (542 MB, 4.9 to 5.15 TB/s: HBM); one token over 2048 keys: 8.0 us and 4.8 for joining, each a chain of dependent
// loads; a tree of 32 over 131072 keys: 106 to 111 us with the joining (9), 69 GFLOP, 0.65 PFLOP/s.  In the last
// neither unit is full: the vector units are busy 52 % of the time (conversions of e4m3, exponentials), the matrix
// units 35 %, both at once 13 %, and about a quarter of the time neither is.
#include "kv_cache.h"

namespace kcg {

typedef __bf16 bf16x8_v __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4_v __attribute__((ext_vector_type(4)));
typedef int int2_v __attribute__((ext_vector_type(2)));
typedef int int4_v __attribute__((ext_vector_type(4)));

constexpr int kFcWaves = 4;
constexpr int kFcChunk = 32;      // keys to a chunk
constexpr int kFcMinChunks = 4;   // of a unit: one to a wave
constexpr int kFcWhole = 24;      // where no sequence can have more, none is cut
constexpr float kFcTau = 8.0f;    // log2 by which a maximum may lag behind before the sums are rescaled

template <typename C>
struct FmhaCacheArgs {
  Rows<const uint16_t> q;
  Rows<void> out;
  KvCache<C> cache;
  const int32_t *table, *context, *drafts;
  const uint64_t *tree;
  float *partial;  // [slot][head][tile][rows][D], then the logarithms [slot][head][tile][rows]
  int64_t logs;    // where those begin, in floats
  int4_v *sequences;  // for more than 64 sequences: first unit, units and first slot of each,
  int32_t *unit_of;   // and the sequence of each unit, -1 behind the last one
  int B, N, Hq, width, group, tiles, rows, want_units, max_units;
  bool few;        // sequences, so that each may have many units
  bool stream;     // K and V past the caches
  float c;
  unsigned q_flip;  // sign bits of two bf16 numbers, or 0
  bool vec;
};

// Unit `index` of the `count` of sequence b.  A sequence of several units has slots of the workspace from
// `slot` on, one to a unit: units of sequences that are cut are at most twice the units wanted.
struct FcUnit {
  int b, index, count, slot;
  KvLens len;
};

template <typename C>
__device__ __forceinline__ KvLens fc_lens(const FmhaCacheArgs<C> &a, int b) {
  return kv_lens(a.context[b], a.drafts ? a.drafts[b] : a.N, a.N,
                 static_cast<int64_t>(a.width) << a.cache.shape.log2_page);
}

// Sum over the lanes up to and with this one, in registers (row shifts, then the rows' last lanes handed on).
__device__ __forceinline__ int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr:1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15 to rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31 to rows 2 and 3
  return x;
}

__device__ __forceinline__ int fc_chunks(const KvLens &l) { return (l.context + l.drafts + kFcChunk - 1) / kFcChunk; }

// Chunks to a unit, for `total` chunks of all sequences.
__device__ __forceinline__ int fc_chunks_per_unit(int64_t total, int want_units) {
  const int64_t per = (total + want_units - 1) / want_units;
  return static_cast<int>(per < kFcMinChunks ? kFcMinChunks : per > (1 << 28) ? 1 << 28 : per);  // (none has as many)
}

// Sequences without queries have no unit, the others at least one.  A sequence a little longer than a unit is
// left whole.
__device__ __forceinline__ int fc_units(const KvLens &l, int per) {
  const int chunks = fc_chunks(l);
  return !l.queries ? 0 : 4 * chunks < 5 * per ? 1 : (chunks + per - 1) / per;
}

// Finds unit `unit`, or with `unit` < 0 the units of sequence -1 - unit; false: there is no such unit.  Up
// to 64 sequences: every wave does it for itself, a sequence to a lane.
template <typename C>
__device__ __forceinline__ bool find_unit(const FmhaCacheArgs<C> &a, int unit, FcUnit &u) {
  const int lane = threadIdx.x & 63;
  if (!a.want_units) {  // every sequence is one unit
    u = {unit, 0, 1, 0, fc_lens(a, unit)};
    return u.len.queries > 0;
  }
  if (a.B > 64) {
    u.b = unit < 0 ? -1 - unit : a.unit_of[unit];
    if (u.b < 0) return false;
    const int4_v s = a.sequences[u.b];
    u.index = unit - s[0];
    u.count = s[1];
    u.slot = s[2];
    u.len = fc_lens(a, u.b);
    return true;
  }
  KvLens l = {0, 0, 0};
  if (lane < a.B) l = fc_lens(a, lane);
  const int per = fc_chunks_per_unit(__builtin_amdgcn_readlane(wave_scan(l.queries ? fc_chunks(l) : 0), 63), a.want_units);
  const int units = fc_units(l, per), upto = wave_scan(units), slots = wave_scan(units > 1 ? units : 0);
  const uint64_t found = __ballot(unit >= 0 ? unit >= upto - units && unit < upto : lane == -1 - unit);
  if (!found) return false;
  u.b = __builtin_ctzll(found);
  u.count = __builtin_amdgcn_readlane(units, u.b);
  u.index = unit - __builtin_amdgcn_readlane(upto, u.b) + u.count;
  u.slot = __builtin_amdgcn_readlane(slots, u.b) - u.count;
  u.len.context = __builtin_amdgcn_readlane(l.context, u.b);
  u.len.drafts = __builtin_amdgcn_readlane(l.drafts, u.b);
  u.len.queries = __builtin_amdgcn_readlane(l.queries, u.b);
  return true;
}

// One workgroup for more than 64 sequences, 1024 at a time.
template <typename C>
__global__ __launch_bounds__(1024) void fmha_cache_units_kernel(const FmhaCacheArgs<C> a) {
  __shared__ int sums[2][16];
  __shared__ unsigned long long total;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (threadIdx.x == 0) total = 0;
  __syncthreads();
  int64_t mine = 0;
  for (int b = threadIdx.x; b < a.B; b += 1024) {
    const KvLens l = fc_lens(a, b);
    if (l.queries) mine += fc_chunks(l);
  }
  if (mine) atomicAdd(&total, static_cast<unsigned long long>(mine));  // (whole numbers: any order)
  __syncthreads();
  const int per = fc_chunks_per_unit(static_cast<int64_t>(total), a.want_units);
  int units_before = 0, slots_before = 0;
  for (int b0 = 0; b0 < a.B; b0 += 1024) {
    const int b = b0 + threadIdx.x;
    int units = 0;
    if (b < a.B) units = fc_units(fc_lens(a, b), per);
    const int cut = units > 1 ? units : 0;
    int first = wave_scan(units), slot = wave_scan(cut);
    if (lane == 63) {
      sums[0][wave] = first;
      sums[1][wave] = slot;
    }
    __syncthreads();
    first += units_before - units;
    slot += slots_before - cut;
    for (int w = 0; w < 16; ++w) {
      if (w < wave) {
        first += sums[0][w];
        slot += sums[1][w];
      }
      units_before += sums[0][w];
      slots_before += sums[1][w];
    }
    if (b < a.B) {
      a.sequences[b] = int4_v{first, units, slot, 0};
      for (int i = 0; i < units; ++i) a.unit_of[first + i] = b;
    }
    __syncthreads();  // (sums are written again)
  }
  for (int i = units_before + threadIdx.x; i < a.max_units; i += 1024) a.unit_of[i] = -1;
}

// What a chunk looks like in LDS.  C: element of the cache; QT: 32-row tiles of queries to a wave.
template <typename C, int D, int QT>
struct FcTile {
  static constexpr int kRow = D * static_cast<int>(sizeof(C));  // bytes
  static constexpr int kPieces = kRow / 16;
  static constexpr int kRowsPer256 = 16 / kPieces;
  static constexpr int kRowsPerLoad = 64 / kPieces;             // one wave-wide direct load: 1024 bytes
  static constexpr int kLoads = kFcChunk / kRowsPerLoad;
  static constexpr int kBytes = kFcChunk * kRow;                // K, or V
  // LDS of a wave: a buffer of K, one of V, two of exponents (K's and V's)
  static constexpr int kExps = sizeof(C) == 1 ? 256 : 0;
  static constexpr int kWave = 2 * kBytes + 2 * kExps;
  static constexpr int kLoadsK = kLoads + (kExps ? 1 : 0), kLoadsV = kLoads;
  static constexpr int kJoinRow = 64 + 4;                       // floats; padded
  static constexpr int kJoin = kFcWaves * 32 * kJoinRow * 4;
  static constexpr int kStream = kFcWaves * kWave > kJoin ? kFcWaves * kWave : kJoin;
  // The last kQLds steps of Q are kept in LDS where the accumulators of two tiles leave no registers for them:
  // all of them, or as many as let two workgroups share a CU's 160 KiB.
  static constexpr int kQLds = D * QT < 256 ? 0 : sizeof(C) == 1 ? 8 : 5;
  static constexpr int kQ = QT * kQLds * 64 * 16;
  static constexpr int kStats = 2 * kFcWaves * 32 * QT * 4;
  static constexpr int kLds = kStream + kQ + kStats;
  static_assert(kRowsPerLoad <= 16, "a load stays inside a page");

  // K: 16 consecutive rows, one piece each
  static __device__ __forceinline__ int swizzle_k(int row) { return (row / kRowsPer256) % kPieces; }
  // V: b8 reads 32 lanes wide take rows {0-3, 8-11} (+ 4, + 16) of two neighbouring pieces, b16 reads four
  // rows of four
  static __device__ __forceinline__ int swizzle_v(int row) {
    if (sizeof(C) == 1) return kPieces == 8 ? 2 * ((row >> 1) & 1) + 4 * ((row >> 3) & 1) : 2 * ((row >> 3) & 1);
    return 4 * ((row / kRowsPer256) & (kPieces / 4 - 1));
  }
};

__device__ __forceinline__ unsigned lds_address(const void *p) {
  return static_cast<unsigned>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const void *)p));
}

// direct_load_16B past the caches, for what is not read again before they have been filled anew
__device__ __forceinline__ void direct_load_16B_stream(const void *base, unsigned off, unsigned lds_addr) {
#if defined(__HIP_DEVICE_COMPILE__)
  unsigned saved_m0;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %1\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %2, %3 nt\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(saved_m0)
      : "s"(lds_addr), "v"(off), "s"(base)
      : "memory");
#endif
}

// lane l's 4 bytes at `from` go to LDS byte address to + 4 * l
__device__ __forceinline__ void direct_load_4B(const void *from, unsigned to) {
#if defined(__HIP_DEVICE_COMPILE__)
  unsigned saved_m0;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %1\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dword %2, off\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(saved_m0)
      : "s"(to), "v"(from)
      : "memory");
#endif
}

// 8 e4m3 bytes times a power of two, as bf16.
__device__ __forceinline__ bf16x8_v to_bf16(unsigned lo, unsigned hi, float scale) {
  const bf16_pair_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false);
  const bf16_pair_t b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
  const bf16_pair_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false);
  const bf16_pair_t d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
  return bf16x8_v{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

__device__ __forceinline__ bool not_finite(uint8_t x) { return (x & 0x7f) == 0x7f; }
__device__ __forceinline__ bool not_finite(uint16_t x) { return (x & 0x7f80) == 0x7f80; }

// Q rows of the tile: 32 * QT columns of the products; TERMS: bf16 numbers that a weight is split over.
// Two waves to a SIMD; three (168 registers) with one tile, where that spills nothing.
template <typename C, int D, int QT, int TERMS>
__global__ __launch_bounds__(64 * kFcWaves, QT == 1 && (D == 64 || TERMS == 1) ? 3 : 2) void fmha_cache_kernel(const FmhaCacheArgs<C> a) {
  using T = FcTile<C, D, QT>;
  constexpr bool E8 = sizeof(C) == 1;
  constexpr int DT = D / 32, DS = D / 16;
  extern __shared__ __align__(16) uint8_t lds[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r32 = lane & 31, half = lane >> 5;

  // tiles of one (unit, head) share its keys: they go to one XCD (workgroup w runs on XCD w % 8)
  const int w = blockIdx.x;
  const int tile = (w / kNumXcd) % a.tiles;
  const int item = w / (kNumXcd * a.tiles) * kNumXcd + w % kNumXcd;
  const int heads = a.cache.shape.heads;
  const int unit = item / heads, head = item - unit * heads;
  FcUnit u;
  if (unit >= a.max_units || !find_unit(a, unit, u)) return;
  const int b = u.b;
  const int row0 = tile * 32 * QT;  // first query row; row = node * group + query head within the group
  if (row0 >= u.len.queries * a.group) return;

  // ---- this wave's chunks ----
  const int keys = u.len.context + u.len.drafts;
  const int chunks = (keys + kFcChunk - 1) / kFcChunk;
  const int per_unit = (chunks + u.count - 1) / u.count;  // a sequence's units are of one size
  const int unit_begin = min(chunks, u.index * per_unit), unit_end = min(chunks, unit_begin + per_unit);
  const int per_wave = (unit_end - unit_begin + kFcWaves - 1) / kFcWaves;
  const int begin = min(unit_end, unit_begin + wave * per_wave), end = min(unit_end, begin + per_wave);

  // ---- pages of this wave, 64 at a time in the lanes of a register ----
  const int log2_page = a.cache.shape.log2_page;
  const int32_t *table = a.table + static_cast<int64_t>(b) * a.width;
  int page_base = 0, pages = 0;
  auto load_pages = [&](int first) {
    page_base = first;
    pages = table[min(first + lane, a.width - 1)];
    // has it arrive here: a load that may still be under way at the next use would make every use wait
    // for all loads, those of the chunks ahead among them
    asm volatile("" ::"v"(pages));
  };
  load_pages((begin * kFcChunk) >> log2_page);
  // page of a key (not beyond the wave's last chunk), -1 if the cache does not have it
  auto page_of = [&](int key) {
    const int index = key >> log2_page;
    if (index >= a.width) return -1;
    if (index - page_base >= 64) load_pages(index);
    const int p = __builtin_amdgcn_readlane(pages, index - page_base);
    return p >= 0 && p < a.cache.shape.pages ? p : -1;
  };

  uint8_t *ring = lds + wave * T::kWave;
  const unsigned ring_at = __builtin_amdgcn_readfirstlane(lds_address(ring));
  constexpr int kV = T::kBytes, kX = 2 * kV;  // where V's buffer and the exponents' begin
  const int load_row = lane / T::kPieces, load_pos = lane % T::kPieces;
  // A chunk's rows: the cache rows of its first and its second 16 keys (of page 0 where the cache does not have
  // their page), and bit g: it has the page of keys 16 g .. 16 g + 15.
  int64_t base0 = 0, base1 = 0;
  int ok = 0, next_ok = 0;
  auto locate = [&](int chunk) {
    const int key0 = chunk * kFcChunk;
    const int p0 = page_of(key0), p1 = page_of(key0 + 16);
    const int in_page = (1 << log2_page) - 1;
    next_ok = (p0 >= 0 ? 1 : 0) | (p1 >= 0 ? 2 : 0);
    base0 = kv_row(a.cache.shape, max(p0, 0), head, key0 & in_page);
    base1 = kv_row(a.cache.shape, max(p1, 0), head, (key0 + 16) & in_page);
  };
  // Requests the K (V) of the chunk located last, number n of this wave.  Whatever was read from the buffer has
  // been used; the wait says so to the hardware as well.
  auto load = [&](int n, bool is_v) {
    const unsigned to = ring_at + (is_v ? kV : 0);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    auto request = [&](auto direct_load) {
#pragma unroll
      for (int j = 0; j < T::kLoads; ++j) {
        const int first = j * T::kRowsPerLoad;
        const int swizzle = is_v ? T::swizzle_v(first + load_row) : T::swizzle_k(first + load_row);
        direct_load((is_v ? a.cache.v : a.cache.k) + ((first < 16 ? base0 : base1) + first % 16) * D,
                    load_row * T::kRow + (load_pos ^ swizzle) * 16, to + j * 1024);
      }
    };
    if (a.stream) request([](const C *from, unsigned off, unsigned to) { direct_load_16B_stream(from, off, to); });
    else request([](const C *from, unsigned off, unsigned to) { direct_load_16B(from, off, to); });
    if (E8 && !is_v) {
      // dwords 0-7: K's exponents, 8-15: V's (the other lanes repeat them)
      const int i = lane & 7;
      direct_load_4B((lane & 8 ? a.cache.v_exp : a.cache.k_exp) + (i < 4 ? base0 : base1) + 4 * (i & 3),
                     ring_at + kX + (n & 1) * T::kExps);
    }
  };

  if (begin < end) {
    locate(begin);
    load(0, false);
    load(0, true);
  }

  // ---- Q ----
  constexpr int QL = T::kQLds;
  uint4_t *q_lds = reinterpret_cast<uint4_t *>(lds + T::kStream);  // [QT][QL][64]
  bf16x8_v q[QT][DS - QL ? DS - QL : 1];
  // Columns beyond the last row repeat it: what they compute is never stored.
  const int last_row = u.len.queries * a.group - 1;
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int row = min(row0 + 32 * t + r32, last_row);
    const int node = row / a.group, h = head * a.group + row - node * a.group;
    const uint16_t *from = a.q.at(b, node, h) + (E8 ? 16 : 8) * half;
    auto d_of = [](int s) { return E8 ? 32 * (s / 2) + 8 * (s % 2) : 16 * s; };
    uint4_t x[DS];
    if (a.vec) {
#pragma unroll
      for (int s = 0; s < DS; ++s) x[s] = *reinterpret_cast<const uint4_t *>(from + d_of(s));
    } else {
#pragma unroll
      for (int s = 0; s < DS; ++s)
#pragma unroll
        for (int j = 0; j < 4; ++j) x[s][j] = from[d_of(s) + 2 * j] | static_cast<unsigned>(from[d_of(s) + 2 * j + 1]) << 16;
    }
#pragma unroll
    for (int s = 0; s < DS; ++s) {
#pragma unroll
      for (int j = 0; j < 4; ++j) x[s][j] ^= a.q_flip;
      if (s < DS - QL) q[t][s] = __builtin_bit_cast(bf16x8_v, x[s]);
      else if (wave == (s - (DS - QL)) % kFcWaves) q_lds[(t * QL + s - (DS - QL)) * 64 + lane] = x[s];
    }
  }
  if (QL) __syncthreads();
  auto q_of = [&](int t, int s) {
    return s < DS - QL ? q[t][s < DS - QL ? s : 0] : __builtin_bit_cast(bf16x8_v, q_lds[(t * QL + s - (DS - QL)) * 64 + lane]);
  };

  float16_t acc[QT][DT];
  float m[QT], l[QT];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    m[t] = -INFINITY;
    l[t] = 0.0f;
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[t][i][e] = 0.0f;
  }

  // V: row and byte column of this lane's transposing reads, within 16 keys and 32 columns
  const int l16 = lane & 15, side = (lane >> 4) & 1;
  const int v_row = E8 ? 4 * half + ((l16 >> 1) & 3) + 8 * (l16 >> 3) : 4 * half + (l16 >> 2);
  const int v_piece = E8 ? side : 2 * side + ((l16 & 3) >> 1);
  const int v_at = v_row * T::kRow + (l16 & 1) * 8;

  for (int chunk = begin; chunk < end; ++chunk) {
    // Requests run K, V, K, V ...: while the scores of a chunk are computed its V is under way, while the weights
    // and the output are, the next K.
    const int n = chunk - begin;
    const bool more = chunk + 1 < end;
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(T::kLoadsV) : "memory");
    const uint8_t *ks = ring;
    uint8_t *vs = ring + kV;
    const uint8_t *xs = ring + kX + (n & 1) * T::kExps;
    ok = next_ok;
    // ---- S^T = K . Q^T ----
    float16_t s[QT];
#pragma unroll
    for (int t = 0; t < QT; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) s[t][e] = 0.0f;
    if constexpr (E8) {
      const float scale = exponent_to_scale(xs[r32]);
#pragma unroll
      for (int p = 0; p < D / 32; ++p) {
        const uint4_t x = *reinterpret_cast<const uint4_t *>(ks + r32 * T::kRow + ((2 * p + half) ^ T::swizzle_k(r32)) * 16);
        const bf16x8_v k0 = to_bf16(x[0], x[1], scale), k1 = to_bf16(x[2], x[3], scale);
#pragma unroll
        for (int t = 0; t < QT; ++t) {
          s[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k0, q_of(t, 2 * p), s[t], 0, 0, 0);
          s[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k1, q_of(t, 2 * p + 1), s[t], 0, 0, 0);
        }
      }
    } else {
#pragma unroll
      for (int p = 0; p < DS; ++p) {
        const uint4_t x = *reinterpret_cast<const uint4_t *>(ks + r32 * T::kRow + ((2 * p + half) ^ T::swizzle_k(r32)) * 16);
        const bf16x8_v k = __builtin_bit_cast(bf16x8_v, x);
#pragma unroll
        for (int t = 0; t < QT; ++t) s[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k, q_of(t, p), s[t], 0, 0, 0);
      }
    }

    if (more) {
      locate(chunk + 1);
      load(n + 1, false);
    }

    // ---- masks ----
    const int key0 = chunk * kFcChunk;
    const bool masked = key0 + kFcChunk > u.len.context || ok != 3;
    const unsigned there = (ok & 1 ? 0x0000ffffu : 0u) | (ok & 2 ? 0xffff0000u : 0u);
    unsigned vis[QT];  // of a masked chunk: the keys that this lane's query sees
    if (masked) {
      const int d0 = key0 - u.len.context;  // the first key's place among the drafts
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        const int node = min(row0 + 32 * t + r32, last_row) / a.group;
        const uint64_t seen = kv_seen(a.tree, static_cast<int64_t>(b) * a.N + node, node, u.len.drafts);
        unsigned v;
        if (d0 >= 0) v = d0 < 64 ? static_cast<unsigned>(seen >> d0) : 0u;
        else if (d0 > -32) v = static_cast<unsigned>(seen << -d0) | ((1u << -d0) - 1);
        else v = 0xffffffffu;
        vis[t] = v & there;
        const unsigned mine = vis[t] >> (4 * half);
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (!((mine >> (8 * (e / 4) + e % 4)) & 1)) s[t][e] = -INFINITY;
      }
    }

    // ---- maxima ----
    float neg[QT];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      // The first maximum is the compiler's: it knows how long a product's result takes, the assembly
      // of max3 does not, and each max3 needs the one before.
      float top = fmaxf(s[t][0], s[t][1]);
#pragma unroll
      for (int e = 2; e < 16; e += 2) top = max3(top, s[t][e], s[t][e + 1]);
      top *= a.c;
      top = max_across_halves(top);
      if (top > m[t] + kFcTau) {
        const float keep = __builtin_amdgcn_exp2f(m[t] - top);  // 0 the first time
        m[t] = top;
        l[t] *= keep;
#pragma unroll
        for (int i = 0; i < DT; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[t][i][e] *= keep;
      }
      neg[t] = m[t] == -INFINITY ? 0.0f : -m[t];
    }

    // ---- weights of 16 keys ----
    unsigned p[QT][2][TERMS][4];  // bf16 pairs
    auto weigh = [&](int kb) {
      unsigned x[2] = {};
      if constexpr (E8) {
#pragma unroll
        for (int g = 0; g < 2; ++g)  // V's exponents of the keys 16 kb + 8 g + 4 half .. + 3, less 128
          x[g] = *reinterpret_cast<const unsigned *>(xs + 32 + 16 * kb + 8 * g + 4 * half) ^ 0x80808080u;
      }
#pragma unroll
      for (int t = 0; t < QT; ++t)
#pragma unroll
        for (int w2 = 0; w2 < 4; ++w2) {
          float y[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) y[k] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][8 * kb + 2 * w2 + k], a.c, neg[t]));
          if (TERMS == 1) {
            // the sum of the weights as they are rounded: what rounding does to one key alone cancels
            const bf16_pair_t ones = {static_cast<__bf16>(1.0f), static_cast<__bf16>(1.0f)};
            l[t] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16_pair_t, float_to_bf16_pair(y[0], y[1])), ones,
                                                   l[t], false);
          } else {
            l[t] += y[0] + y[1];
          }
          if constexpr (E8) {
#pragma unroll
            for (int k = 0; k < 2; ++k)
              y[k] = __builtin_ldexpf(y[k], static_cast<int>(x[w2 / 2] << (24 - 8 * (2 * (w2 % 2) + k))) >> 24);
          }
          if constexpr (TERMS == 1) {
            p[t][kb][0][w2] = float_to_bf16_pair(y[0], y[1]);
          } else {
            // Terms cut off after eight bits each, which hold all 24 of a weight.  None of a weight's is negative, or,
            // against values that may be infinite (e4m3 has no infinity), zero: those would make NaN of an infinity.
            const float least[2] = {E8 ? 0.0f : y[0] * 0x1p-30f, E8 ? 0.0f : y[1] * 0x1p-30f};
#pragma unroll
            for (int z = 0; z < TERMS; ++z) {
              if (!E8 && z) {
#pragma unroll
                for (int k = 0; k < 2; ++k) y[k] = fmaxf(y[k], least[k]);
              }
              const unsigned a = __builtin_bit_cast(unsigned, y[0]), b = __builtin_bit_cast(unsigned, y[1]);
              p[t][kb][z][w2] = __builtin_amdgcn_perm(b, a, 0x07060302u);
              y[0] -= __builtin_bit_cast(float, a & 0xffff0000u);
              y[1] -= __builtin_bit_cast(float, b & 0xffff0000u);
            }
          }
        }
    };
    weigh(0);

    // ---- V ----
    if (more) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(T::kLoadsK) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (masked) {
      // keys that some query may see; the rows of the others are zeroed
      const int left = keys - key0;
      const unsigned some = (left >= 32 ? 0xffffffffu : (1u << left) - 1) & there;
      unsigned bad = 0;  // rows with values that are not finite
#pragma unroll 1
      for (int j = 0; j < T::kLoads; ++j) {
        const int row = j * T::kRowsPerLoad + load_row;
        uint4_t *piece = reinterpret_cast<uint4_t *>(vs + j * 1024 + lane * 16);
        uint4_t x = *piece;
        bool any = false;
        if (!((some >> row) & 1)) {
          *piece = uint4_t{0, 0, 0, 0};
        } else {
#pragma unroll
          for (int i = 0; i < static_cast<int>(16 / sizeof(C)); ++i)
            any |= not_finite(static_cast<C>(x[i * sizeof(C) / 4] >> (8 * (i * sizeof(C) % 4))));
        }
        uint64_t where = __ballot(any);
        while (where) {
          const int at = __builtin_ctzll(where);
          bad |= 1u << (j * T::kRowsPerLoad + at / T::kPieces);
          where &= where - 1;
        }
      }
      if (bad) {  // (uniform)
        for (unsigned left_over = bad; left_over; left_over &= left_over - 1) {
          const int row = __builtin_ctz(left_over);
#pragma unroll
          for (int i = 0; i < DT; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const int byte = (32 * i + 8 * (e / 4) + 4 * half + e % 4) * static_cast<int>(sizeof(C));
              const C x = *reinterpret_cast<const C *>(vs + row * T::kRow + ((byte / 16) ^ T::swizzle_v(row)) * 16 + byte % 16);
              if (not_finite(x)) {
                const float y = E8 ? NAN : bf16_to_float(static_cast<uint16_t>(x));
#pragma unroll
                for (int t = 0; t < QT; ++t)
                  if ((vis[t] >> row) & 1) acc[t][i][e] += y;
              }
            }
        }
#pragma unroll 1
        for (int j = 0; j < T::kLoads; ++j) {
          C *piece = reinterpret_cast<C *>(vs + j * 1024 + lane * 16);
#pragma unroll 1
          for (int i = 0; i < static_cast<int>(16 / sizeof(C)); ++i)
            if (not_finite(piece[i])) piece[i] = 0;
        }
      }
    }

    // all its reads before the first product: one takes longer than the products between two
    constexpr int kWords = E8 ? 2 : 4;
    unsigned v_raw[2][DT][kWords];
    auto read_v = [&](int kb) {
#pragma unroll
      for (int i = 0; i < DT; ++i) {
        // rows 16 apart have one swizzle, and with b16 reads rows 8 apart
        const int piece = ((E8 ? 2 : 4) * i + v_piece) ^ T::swizzle_v(v_row);
        const uint8_t *from = vs + kb * 16 * T::kRow + v_at + piece * 16;
        if constexpr (E8) {
          const int2_v x = __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) int2_v *)from);
          v_raw[kb][i][0] = static_cast<unsigned>(x[0]);
          v_raw[kb][i][1] = static_cast<unsigned>(x[1]);
        } else {
          const uint2_t lo = __builtin_bit_cast(
              uint2_t, __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) bf16x4_v *)from));
          const uint2_t hi = __builtin_bit_cast(
              uint2_t, __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) bf16x4_v *)(from + 8 * T::kRow)));
          v_raw[kb][i][0] = lo[0];
          v_raw[kb][i][1] = lo[1];
          v_raw[kb][i][2] = hi[0];
          v_raw[kb][i][3] = hi[1];
        }
      }
    };
    read_v(0);
    read_v(1);
    asm volatile("" ::: "memory");  // (or the compiler moves the reads down to their uses)

    // ---- O^T += V^T . P^T; the other weights are computed between the products of the first 16 keys ----
    auto multiply = [&](int kb) {
#pragma unroll
      for (int i = 0; i < DT; ++i) {
        bf16x8_v v;
        if constexpr (E8) v = to_bf16(v_raw[kb][i][0], v_raw[kb][i][1], 1.0f);
        else v = __builtin_bit_cast(bf16x8_v, uint4_t{v_raw[kb][i][0], v_raw[kb][i][1], v_raw[kb][i][2], v_raw[kb][i][3]});
#pragma unroll
        for (int t = 0; t < QT; ++t)
#pragma unroll
          for (int z = 0; z < TERMS; ++z) {
            const uint4_t y = {p[t][kb][z][0], p[t][kb][z][1], p[t][kb][z][2], p[t][kb][z][3]};
            acc[t][i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, __builtin_bit_cast(bf16x8_v, y), acc[t][i], 0, 0, 0);
          }
      }
    };
    multiply(0);
    weigh(1);
    multiply(1);
    if (more) load(n + 1, true);
  }

  // ---- join the waves: 64 columns of 32 rows at a time ----
  float *join = reinterpret_cast<float *>(lds);
  float *stats_m = reinterpret_cast<float *>(lds + T::kStream + T::kQ);  // [waves][32 * QT]
  float *stats_l = stats_m + kFcWaves * 32 * QT;
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    l[t] += __shfl_xor(l[t], 32);
    if (half == 0) {
      stats_m[wave * 32 * QT + 32 * t + r32] = m[t];
      stats_l[wave * 32 * QT + 32 * t + r32] = l[t];
    }
  }
  const bool whole = u.count == 1;
  const int64_t slot = (static_cast<int64_t>(u.slot + u.index) * heads + head) * a.tiles + tile;
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    float norm = 0.0f;
#pragma unroll
    for (int part = 0; part < D / 64; ++part) {
      __syncthreads();  // statistics are there; ring buffers and the last round's outputs are done with
      if (part == 0) {
        const int row = 32 * t + r32;
        float top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int k = 0; k < kFcWaves; ++k) top = fmaxf(top, stats_m[k * 32 * QT + row]);
        const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll
        for (int k = 0; k < kFcWaves; ++k)
          sum += stats_l[k * 32 * QT + row] * __builtin_amdgcn_exp2f(stats_m[k * 32 * QT + row] - ref);
        // (e4m3: the weights were 2^-1 of what they stand for)
        norm = (sum == 0.0f ? 0.0f : (E8 ? 2.0f : 1.0f) / sum) * __builtin_amdgcn_exp2f(m[t] - ref);
        if (!whole && wave == 0 && half == 0 && row < a.rows)
          a.partial[a.logs + slot * a.rows + row] = sum == 0.0f ? -INFINITY : ref + __builtin_amdgcn_logf(sum);
      }
      float *mine = join + (wave * 32 + r32) * T::kJoinRow + 4 * half;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float16_t &x = acc[t][2 * part + i];
          *reinterpret_cast<float4_t *>(mine + 32 * i + 8 * g) =
              float4_t{x[4 * g] * norm, x[4 * g + 1] * norm, x[4 * g + 2] * norm, x[4 * g + 3] * norm};
        }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = 16 * i + threadIdx.x / 16, column = 4 * (threadIdx.x % 16), d = 64 * part + column;
        const int row = row0 + 32 * t + r, node = row / a.group, h = head * a.group + row - node * a.group;
        if (node >= u.len.queries) break;
        float4_t y = {};
#pragma unroll
        for (int k = 0; k < kFcWaves; ++k) y += *reinterpret_cast<const float4_t *>(join + (k * 32 + r) * T::kJoinRow + column);
        if (!whole) {
          *reinterpret_cast<float4_t *>(a.partial + (slot * a.rows + 32 * t + r) * D + d) = y;
        } else if constexpr (TERMS == 1) {
          uint16_t *to = static_cast<uint16_t *>(a.out.data) + b * a.out.stride_b + node * a.out.stride_s + h * a.out.stride_h + d;
          const uint2_t z = {float_to_bf16_pair(y[0], y[1]), float_to_bf16_pair(y[2], y[3])};
          if (a.vec) *reinterpret_cast<uint2_t *>(to) = z;
          else
            for (int j = 0; j < 4; ++j) to[j] = float_to_bf16(y[j]);
        } else {
          float *to = static_cast<float *>(a.out.data) + b * a.out.stride_b + node * a.out.stride_s + h * a.out.stride_h + d;
          if (a.vec) *reinterpret_cast<float4_t *>(to) = y;
          else
            for (int j = 0; j < 4; ++j) to[j] = y[j];
        }
      }
    }
  }
}

// Joins the units of the sequences that have several, D / 4 lanes of float4 to a unit's share of a row.  Few
// sequences: a workgroup to a row, 1024 / D units under way at a time.  Many: a workgroup to 1024 / D rows of
// a sequence, since each has few units if any, and finding them takes longer than joining them.
template <typename C, int D, typename O>
__global__ __launch_bounds__(256) void fmha_cache_join_kernel(const FmhaCacheArgs<C> a) {
  constexpr int LANES = D / 4, GROUPS = 256 / LANES;
  __shared__ float4_t shares[GROUPS][LANES];
  __shared__ float sums[GROUPS];
  const int per_sequence = a.N * a.Hq, parts = a.few ? per_sequence : (per_sequence + GROUPS - 1) / GROUPS;
  const int b = blockIdx.x / parts, part = blockIdx.x - b * parts;
  FcUnit u;
  if (!find_unit(a, -1 - b, u) || u.count < 2) return;
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES, d = 4 * lane;
  const int at = a.few ? part : part * GROUPS + group;  // row of the sequence
  const int node = at / a.Hq, h = at - node * a.Hq;
  const bool live = node < u.len.queries && at < per_sequence;
  if (a.few && !live) return;
  const int head = h / a.group, row = node * a.group + h - head * a.group;
  const int tile = row / 64, r = row - tile * 64;  // (one tile holds at most 64 rows)
  const int64_t step = static_cast<int64_t>(a.cache.shape.heads) * a.tiles * a.rows;
  const int64_t first = (static_cast<int64_t>(u.slot) * a.cache.shape.heads + head) * a.tiles * a.rows +
                        static_cast<int64_t>(tile) * a.rows + r;
  const float *logs = a.partial + a.logs + first, *share = a.partial + first * D + d;
  float top = -INFINITY, sum = 0.0f;
  float4_t y = {};
  if (live)
#pragma unroll 4
    for (int i = 0; i < u.count; ++i) top = fmaxf(top, logs[i * step]);
  const float ref = top == -INFINITY ? 0.0f : top;
  auto add = [&](int i) {
    const float weight = __builtin_amdgcn_exp2f(logs[i * step] - ref);
    const float4_t x = *reinterpret_cast<const float4_t *>(share + i * step * D);
    sum += weight;
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = __builtin_fmaf(weight, x[j], y[j]);
  };
  if (!a.few) {
    if (!live) return;
#pragma unroll 4
    for (int i = 0; i < u.count; ++i) add(i);
  } else {
#pragma unroll 4
    for (int i = group; i < u.count; i += GROUPS) add(i);
    shares[group][lane] = y;
    if (lane == 0) sums[group] = sum;
    __syncthreads();
    if (group) return;
    for (int k = 1; k < GROUPS; ++k) {  // (in a fixed order)
      y += shares[k][lane];
      sum += sums[k];
    }
  }
  y *= sum == 0.0f ? 0.0f : 1.0f / sum;
  O *to = static_cast<O *>(a.out.data) + b * a.out.stride_b + node * a.out.stride_s + h * a.out.stride_h + d;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (sizeof(O) == 2) to[j] = float_to_bf16(y[j]);
    else to[j] = y[j];
  }
}

// How a call is split; the query and the call agree on it.
struct FcPlan {
  int group, qt, tiles, rows;  // rows: of a tile that are stored
  int want_units, max_units;   // want_units 0: one unit to a sequence, nothing is stored between
  bool few;
  int64_t logs, sequences, unit_of, bytes;  // where the parts of the workspace begin, and its size
};

inline FcPlan plan_fmha_cache(const kcg_kv_cache &c, int width, int B, int N, int Hq, int64_t workspace_bytes) {
  FcPlan p = {};
  p.group = Hq / c.heads;
  const int rows = N * p.group;
  p.qt = rows <= 32 ? 1 : 2;
  p.tiles = (rows + 32 * p.qt - 1) / (32 * p.qt);
  p.rows = p.tiles > 1 ? 64 : rows;
  p.max_units = B;
  const int64_t per_unit = static_cast<int64_t>(c.heads) * p.tiles;
  const int64_t round = 2 * kNumCu / per_unit;  // units that run at once, two workgroups to a CU
  // A few sequences: one round, less the unit that each one's remainder may add (a tree of 32 over 131072
  // keys: 111 us, with two rounds 121, with four 142; 8 single tokens over 4000: 22, 25 and 29, whole 40).  Many:
  // one and a half (64 single tokens over contexts to 8192: 111 us, with one round 113, with two 106; 24 over 4000:
  // 45, 51 and 50).  That pays where lengths differ or the chip is not full (32 query heads on 8 of 128, e4m3, cut
  // and whole): 64 to 8192 111 and 115, 32 64 and 79, 16 39 and 73, 12 x 8 drafts to 20000 62 and 169.  It costs
  // where whole sequences fill the chip evenly, or where the third launch weighs: 64 over 4096 97 and 92, 32 x 4
  // drafts over 4000 54 and 49, 24 over 1000 and 16 x 4 over 1000 19 and 16, 128 over 2000 95 and 88, 128 to 2000 65
  // and 56.  A call with a workspace of no bytes cuts nothing.
  p.few = 8 * static_cast<int64_t>(B) <= round;
  int64_t want = p.few ? round - B : 3 * round / 2;
  const int64_t chunks = (static_cast<int64_t>(width) * c.page_size + kFcChunk - 1) / kFcChunk;
  // (1 x 4 drafts over 500 keys, e4m3: 10.1 us whole, 11.0 cut; 750: 12.3 and 11.6; 24 single tokens over 1000: 15.6, 18.6)
  if (chunks <= kFcWhole) return p;
  for (; want > 0; want /= 2) {  // (less, where the workspace does not hold what is preferred)
    const int64_t slots = B < want ? want + B : 2 * want;  // see FcUnit
    p.logs = slots * per_unit * p.rows * c.dim;
    p.sequences = ((p.logs + slots * per_unit * p.rows) * 4 + 15) / 16 * 16;
    p.unit_of = p.sequences + (B > 64 ? static_cast<int64_t>(B) * 16 : 0);
    p.bytes = p.unit_of + (B > 64 ? (want + B) * 4 : 0);
    if (workspace_bytes >= 0 && p.bytes > workspace_bytes) continue;
    p.want_units = static_cast<int>(want);
    p.max_units = static_cast<int>(want + B);
    return p;
  }
  p.bytes = 0;
  return p;
}

template <typename C, int D, int QT, int TERMS>
int run_fmha_cache(const FmhaCacheArgs<C> &a, hipStream_t stream) {
  const auto kernel = fmha_cache_kernel<C, D, QT, TERMS>;
  const int lds = FcTile<C, D, QT>::kLds;
  if (!allow_lds(kernel, lds)) return KCG_ERR_LAUNCH;
  const int64_t items = static_cast<int64_t>(a.max_units) * a.cache.shape.heads;
  const int64_t grid = (items + kNumXcd - 1) / kNumXcd * kNumXcd * a.tiles;
  if (grid > 0x7fffffffLL) return KCG_ERR_UNSUPPORTED_SHAPE;
  if (a.want_units && a.B > 64)
    if (const int e = launch(fmha_cache_units_kernel<C>, dim3(1), dim3(1024), 0, stream, a)) return e;
  if (const int e = launch(kernel, dim3(static_cast<unsigned>(grid)), dim3(64 * kFcWaves), lds, stream, a)) return e;
  if (!a.want_units) return KCG_OK;
  const int64_t rows = static_cast<int64_t>(a.N) * a.Hq, groups = a.few ? 1 : 1024 / D;
  using O = std::conditional_t<TERMS == 1, uint16_t, float>;
  return launch(fmha_cache_join_kernel<C, D, O>, dim3(static_cast<unsigned>(a.B * ((rows + groups - 1) / groups))), dim3(256),
                0, stream, a);
}

template <typename C>
int fmha_cache(const kcg_rows &q, const kcg_kv_cache &cache, const int32_t *table, int width, const int32_t *context,
               const int32_t *drafts, const uint64_t *tree, const kcg_rows &out, int o_dtype, int B, int N, int Hq,
               float scale, void *workspace, int64_t workspace_bytes, hipStream_t stream) {
  const FcPlan p = plan_fmha_cache(cache, width, B, N, Hq, workspace ? workspace_bytes : 0);
  FmhaCacheArgs<C> a = {};
  a.q = make_rows<const uint16_t>(q);
  a.out = make_rows<void>(out);
  a.cache = make_cache<C>(cache);
  a.table = table;
  a.context = context;
  a.drafts = drafts;
  a.tree = tree;
  a.partial = static_cast<float *>(workspace);
  a.logs = p.logs;
  if (p.want_units && B > 64) {
    a.sequences = reinterpret_cast<int4_v *>(static_cast<char *>(workspace) + p.sequences);
    a.unit_of = reinterpret_cast<int32_t *>(static_cast<char *>(workspace) + p.unit_of);
  }
  a.B = B;
  a.N = N;
  a.Hq = Hq;
  a.width = width;
  a.group = p.group;
  a.tiles = p.tiles;
  a.rows = p.rows;
  a.want_units = p.want_units;
  a.max_units = p.max_units;
  a.few = p.few;
  // The scale's sign goes into Q, so that the maximum of the scores is that of the products.  For a scale
  // of 0 the smallest normal number stands: its products vanish beside 1, and -inf stays -inf under it.
  a.q_flip = scale < 0.0f ? 0x80008000u : 0u;
  a.c = scale == 0.0f ? 1.17549435e-38f : fabsf(scale) * 1.44269504088896340736f;
  // Past the caches where the table has room for more than most of the last-level cache (256 MiB): 64 single
  // tokens over contexts to 8192 (1 GiB of room) 111 us so, 122 otherwise, 8 over 4000 (64 MiB) 22.6 and 22.0.
  a.stream = static_cast<int64_t>(B) * width * cache.page_size * cache.heads * cache.dim * 2 * static_cast<int64_t>(sizeof(C)) >
             (int64_t{192} << 20);
  a.vec = rows_aligned16(q, KCG_BF16, B, N, Hq) && rows_aligned16(out, o_dtype, B, N, Hq);
#define KCG_PICK(DD, QQ) \
  return o_dtype == KCG_F32 ? run_fmha_cache<C, DD, QQ, 3>(a, stream) : run_fmha_cache<C, DD, QQ, 1>(a, stream)
  if (cache.dim == 64) {
    if (p.qt == 1) { KCG_PICK(64, 1); }
    KCG_PICK(64, 2);
  }
  if (p.qt == 1) { KCG_PICK(128, 1); }
  KCG_PICK(128, 2);
#undef KCG_PICK
}

// Shapes and types that both the call and its workspace query check.
inline int check_fmha_cache(const kcg_kv_cache *cache, int64_t width, int64_t B, int64_t N, int64_t Hq) {
  if (const int e = check_cache(cache)) return e;
  if (width <= 0 || B <= 0 || N <= 0 || Hq <= 0) return KCG_ERR_BAD_SHAPE;
  if (N > 64 || Hq % cache->heads) return KCG_ERR_UNSUPPORTED_SHAPE;
  if (width > 0x7fffff00LL / cache->page_size || B > 0x7fffffffLL / width) return KCG_ERR_UNSUPPORTED_SHAPE;
  // (the chunks of all sequences are summed in 32 bits, and lengths may say that every table is full)
  if (B * width > (int64_t{1} << 35) / cache->page_size) return KCG_ERR_UNSUPPORTED_SHAPE;
  return check_extents(B, N, Hq, cache->dim);
}

}  // namespace kcg

extern "C" {

int64_t kcg_fmha_cache_ws_bytes(const kcg_kv_cache *cache, int32_t table_width, int32_t B, int32_t N, int32_t Hq) {
  if (kcg::check_fmha_cache(cache, table_width, B, N, Hq)) return 0;
  return kcg::plan_fmha_cache(*cache, table_width, B, N, Hq, -1).bytes;
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
                                        o_dtype, B, N, Hq, scale, workspace, workspace_bytes, st)
             : kcg::fmha_cache<uint16_t>(*q, *cache, block_table, table_width, context_lens, draft_lens, tree_mask, *out,
                                         o_dtype, B, N, Hq, scale, workspace, workspace_bytes, st);
}

}  // extern "C"
