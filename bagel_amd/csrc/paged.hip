// A paged key-value cache (gfx950): append of new keys and values with the q/k norm and the rotation on the way, and one
// new token's attention over it.
//
// The cache is a pool of pages of page_size slots, element (page, slot, kv head, d) at
// page * page_stride + slot * slot_stride + head * head_stride + d, in bf16 or in OCP e4m3 with one fp32 scale per kv
// head (a stored unit stands for `scale`).  A sequence owns pages in any order; its page table row lists them.  Rows of a
// head are contiguous, whichever of slots and heads comes first, and nothing about a sequence's length or place is fixed:
// sequences grow page by page, finish and hand their pages on without a copy.
#include "common.h"
#include <algorithm>
#include "qk_rope.h"
#include "../../include/bagel_hip.h"

namespace {

constexpr float E4M3_MAX = 448.f;

typedef __attribute__((ext_vector_type(4))) unsigned u32x4;
typedef __attribute__((ext_vector_type(2))) unsigned u32x2;

struct Pool {          // one of the two pools, strides in BYTES
  char* base;
  long page, slot, head;
  const float* scale;  // per kv head, null for bf16
};

// fp32 -> four e4m3 in a dword, round to nearest even, clamped to the largest finite value (a NaN stays one: the clamp is
// written so that it passes).
__device__ __forceinline__ unsigned pack_e4m3(float a, float b, float c, float d) {
  auto clamp = [](float x) { return x > E4M3_MAX ? E4M3_MAX : x < -E4M3_MAX ? -E4M3_MAX : x; };
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(clamp(a), clamp(b), 0, false);
  return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(clamp(c), clamp(d), r, true);
}

// ---------------------------------------------------------------------------------------------------------------------
// Append.  Row r of qkv holds Hq query heads, Hkv key heads and Hkv value heads of D; D / 8 lanes hold a head (16 bytes
// each), so a head's norm and its rotation partner stay inside those lanes.  Everything is one pass, bound by memory: each projected
// element is read once and each result written once.  A thread takes G neighbouring heads of its row, whose loads are in
// flight together and which share the row's slot and rotation; G = 1 where there are too few rows (launch_append).
// Many rows (G = 4) pass the caches by: 32768 rows of 36 heads of 128, 621 MB, take 107 us = 5.8 TB/s (121 us through the
// caches, 138 us with one head per thread; a large copy reaches 4.9 TB/s); the same into e4m3 pages, 587 MB, 146 us.
// ---------------------------------------------------------------------------------------------------------------------
struct AppendParams {
  const bf16* qkv;
  long ld;
  const bf16 *q_w, *k_w, *cos_t, *sin_t;   // norm weights [D], rotation rows [*][D]; null: that step is left out
  const int *row_cs, *row_slot;
  bf16* Q;                                 // null where Hq is 0
  long ldq;
  Pool k, v;
  long capacity;                           // slots in the pool
  int rows, Hq, Hkv, page_shift, cs_rows, und_rounding;
  float eps;
};

template <int D, bool F8, int G>
__global__ __launch_bounds__(256) void paged_append_kernel(AppendParams p) {
  constexpr int LPH = D / 8;
  const int heads = p.Hq + 2 * p.Hkv, groups = (heads + G - 1) / G;
  const unsigned item = blockIdx.x * (256 / LPH) + threadIdx.x / LPH;
  const int row = item / groups, first = (item - row * groups) * G;
  if (row >= p.rows) return;                     // a head's lanes leave together
  const int j = threadIdx.x % LPH;
  const bf16* src = p.qkv + row * p.ld + (long)first * D + 8 * j;
  bf16x8 x[G];
#pragma unroll
  for (int g = 0; g < G; ++g)
    if (first + g < heads) x[g] = G > 1 ? __builtin_nontemporal_load((const bf16x8*)(src + g * D)) : *(const bf16x8*)(src + g * D);
  const int slot = p.row_slot[row], cs = p.cos_t ? p.row_cs[row] : 0;
  if (slot < 0) return;                          // padding: the cache and the row's queries are left as they are
  bf16* q = p.Q + row * p.ldq + (long)first * D + 8 * j;
  if (slot >= p.capacity || (p.cos_t && (cs < 0 || cs >= p.cs_rows))) {
    // a slot or rotation row that does not exist: nothing is stored, and the row's queries say so
#pragma unroll
    for (int g = 0; g < G; ++g)
      if (first + g < p.Hq) {
        bf16x8 nan;
#pragma unroll
        for (int e = 0; e < 8; ++e) nan[e] = (bf16)__builtin_nanf("");
        *(bf16x8*)(q + g * D) = nan;
      }
    return;
  }
  const int keys = p.Hq, values = p.Hq + p.Hkv;  // first heads of either
  bf16x8 c{}, s{}, qw{}, kw{};
  if (first < values) {
    if (p.cos_t) c = *(const bf16x8*)(p.cos_t + (long)cs * D + 8 * j), s = *(const bf16x8*)(p.sin_t + (long)cs * D + 8 * j);
    if (p.q_w) qw = *(const bf16x8*)(p.q_w + 8 * j);
    if (p.k_w) kw = *(const bf16x8*)(p.k_w + 8 * j);
  }
  const long page = slot >> p.page_shift, at = slot & ((1 << p.page_shift) - 1);
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const int head = first + g;
    if (head >= heads) continue;
    float y[8];
    if (head >= values) {
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = (float)x[g][e];
    } else {
      const bool is_q = head < keys;
      norm_rope_lane<D>(x[g], j, is_q ? p.q_w : p.k_w, is_q ? qw : kw, p.cos_t, c, s, p.eps, p.und_rounding, y);
    }
    bf16x8 o;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = (bf16)y[e];
    if (head < keys) {
      if constexpr (G > 1) __builtin_nontemporal_store(o, (bf16x8*)(q + g * D));
      else *(bf16x8*)(q + g * D) = o;
      continue;
    }
    const Pool& pool = head >= values ? p.v : p.k;
    const int h = head >= values ? head - values : head - keys;
    char* dst = pool.base + page * pool.page + at * pool.slot + h * pool.head;
    if constexpr (F8) {
      const float u = pool.scale[h];
      *(u32x2*)(dst + 8 * j) = u32x2{pack_e4m3(y[0] / u, y[1] / u, y[2] / u, y[3] / u), pack_e4m3(y[4] / u, y[5] / u, y[6] / u, y[7] / u)};
    } else {
      *(bf16x8*)(dst + 16 * j) = o;
    }
  }
}

template <int D, bool F8>
int launch_append(const AppendParams& p, hipStream_t st) {
  constexpr int LPH = D / 8, PER_BLOCK = 256 / LPH;
  const int heads = p.Hq + 2 * p.Hkv;
  // Four heads per thread once that still gives every CU four workgroups; in e4m3, whose divisions take longer by the thread, only
  // where the rows no longer fit the caches that the four-heads form passes by.  Measured (us, one and four heads per thread):
  //   28 / 4 heads of 128, bf16   1500 rows 9.2 9.9    1820 (four workgroups per CU) 10.7 10.1   2400 13.1 11.5   32768 138 107
  //   24 / 1 of 128, bf16         1820 rows 8.4 8.8    2400 (four) 10.2 9.6                      6553 22.2 19.2   32768 104 79
  //   14 / 2 of 64, bf16          4500 rows 8.4 9.1    6553 (four) 10.2 10.1                     8192 12.5 11.1   20000 24.3 23.0
  //   28 / 4 of 128, e4m3         2400 rows 14.2 16.5  8192 (18) 35.1 41.0                       20000 (44) 97 92   32768 154 146
  //   32 / 8 of 128, e4m3         8192 rows 44.9 48.5  20000 (59) 127 107                        32768 201 171
  //   16 / 16 of 64               bf16 8192 rows (12) 22.7 25.2, the worst of the rule, 32768 94 76;   e4m3 20000 rows (29) 60 73, 32768 (48) 115 115
  const int g = (long)p.rows * ((heads + 3) / 4) >= (F8 ? 40L : 4L) * bagel_cu_count() * PER_BLOCK ? 4 : 1;
  const long blocks = ((long)p.rows * ((heads + g - 1) / g) + PER_BLOCK - 1) / PER_BLOCK;
  BAGEL_CHECK(blocks * PER_BLOCK <= 0x7fffffffL, "bagel_paged_kv_append_bf16: %d rows are too many for one launch", p.rows);
  if (g == 4) hipLaunchKernelGGL((paged_append_kernel<D, F8, 4>), dim3((unsigned)blocks), dim3(256), 0, st, p);
  else hipLaunchKernelGGL((paged_append_kernel<D, F8, 1>), dim3((unsigned)blocks), dim3(256), 0, st, p);
  BAGEL_LAUNCH_CHECK();
  return 0;
}

// ---------------------------------------------------------------------------------------------------------------------
// Attention of one new token per row.
//
// The keys and values of a (row, kv head) are read once for all the query heads that share them, up to 16 per workgroup,
// so that the matrix instruction's 16 columns are heads:
//   S^T[key][head] = K . Q^T      and      O^T[d][head] += V^T . P^T
// with 32 keys as the contraction of the second product.
//   - Key rows go to LDS whole, without passing a register, and a lane of S^T's operand reads 16 bytes of ONE key row
//     (lane & 15 = row, lane >> 4 = part of the contraction).
//   - Row m of key tile t is key 8 (m / 4) + 4 t + m % 4 of the 32, so that the results a lane gets - rows 4 g + i of both
//     tiles, g = lane >> 4 - are keys 8 g ... 8 g + 7 of its head: exactly what the second product wants of P^T from it.
//   - V rows go to registers (16 lanes x D / 16 elements, 8 keys per lane group).  The operand wants 8 KEYS of one d per
//     lane; the lane has D / 16 d's of those 8 keys, so byte permutes turn one into the other inside the lane, and
//     row r of product dd is d = (D / 16) r + dd.
// The softmax is the running form: one maximum and sum per head and wave, scores and sums in fp32.  The matrix product takes P as the
// sum of two bf16 parts: the next bf16 number below the weight, and what that leaves, which is positive (a value of infinity
// times a part of zero would be NaN).  e4m3 has no infinity, so there the first part is the weight rounded, in fewer instructions.
// Together they are within 2^-15 of each weight, so the output's rounding is the only one to bf16 that shows; one rounded part alone
// is off by up to 2^-8, as much as the output's rounding, and by far more where values cancel.  What the second part costs (us, one
// part and two): 64 rows of up to 8192 bf16 keys, slots first, 121.0 and 121.5, 200 rows of e4m3 94.6 and 95.4, one row of 131072 53.7 and 53.4.
// An e4m3 value is a bf16 value: keys and values are widened exactly, the scales enter in fp32.
//
// One workgroup = four waves that take turns at the chunk's tiles, each with its own running softmax.  A row with more keys
// than one chunk is split over workgroups; each leaves an unnormalised partial (sums in fp32) and the last one to finish
// joins them in chunk order, JOIN at a time: more chunks than that are joined in groups first.
//
// Bound by the reads of the cache.  28 query and 4 kv heads of 128: 64 rows of up to 8192 keys, 561 MB of bf16, 110 us =
// 5.1 TB/s; one row of 131072, 268 MB, 55 us = 4.9 TB/s, joins included; e4m3, 200 rows of up to 4096, 476 MB, 94 us = 5.1 TB/s.
// (Reads of random 16 KB pages alone reach 6.9 TB/s past the caches, 6.0 through them; a large copy 4.9.)
// Keys straight to registers, 16 bytes of each of 16 rows per lane, took 128 us for the first and 115 for the last of these where
// keys through LDS took 108 and 93.
// ---------------------------------------------------------------------------------------------------------------------
constexpr int WAVES = 4;
constexpr int JOIN = 16;             // partials that are joined at once
constexpr int MAX_SPLITS = 8 * JOIN;
constexpr long MAX_KEYS = 1L << 30;  // of a row
constexpr int SHORT = 512;           // keys that take as long as a level of joins
constexpr int TICKETS = 16;          // per (row, kv head, head block): one for all chunks or groups of them, eight for the groups

// Blocks of 32 keys per tile: 8 KB of keys and as much of values, half of that for the shortest rows.
template <int D, bool F8>
constexpr int tile_blocks() {
  return D * (F8 ? 1 : 2) == 256 ? 1 : 2;
}

struct AttendParams {
  const bf16* Q;
  long ldq;
  Pool k, v;
  const int* table;      // [rows][table_width] page ids
  long table_stride;
  int table_width, num_pages, page_shift;
  const int* kv_lens;
  bf16* O;
  long ldo;
  float* part;           // [rows][Hkv][head blocks][splits][heads in the block][D] sums
  float2* stats;         // [rows][Hkv][head blocks][splits][heads in the block] maximum, weight
  unsigned* tickets;     // [rows][Hkv][head blocks][TICKETS], zero on entry, left zero
  int Hq, Hkv, chunk;
  float scale_log2;
};

__device__ __forceinline__ bf16x8 widen8(unsigned a, unsigned b) {   // eight e4m3 -> eight bf16
  const bf16x2 x0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, false), x1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, true);
  const bf16x2 x2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, false), x3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, true);
  return bf16x8{x0[0], x0[1], x1[0], x1[1], x2[0], x2[1], x3[0], x3[1]};
}

// maximum / sum over the four lanes that hold one head's column
__device__ __forceinline__ float column_max(float v) {
  const u32x2 a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const u32x2 b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float column_sum(float v) {
  const u32x2 a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const u32x2 b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Three waves per SIMD: at most 168 registers, and the compiler takes 167 (bf16 at D = 128) without being held to it; held to it, it
// spills two of them.
template <int D, bool F8>
__global__ __launch_bounds__(64 * WAVES, 2) void paged_attention_kernel(AttendParams p) {
  constexpr int ITEM = F8 ? 1 : 2;
  constexpr int SUB = tile_blocks<D, F8>();    // blocks of 32 keys per tile
  constexpr int TK = 32 * SUB;                 // keys per tile
  constexpr int CH = D * ITEM / 16;            // 16-byte pieces of a key row
  constexpr int RPI = 64 / CH;                 // key rows that one load instruction of a wave covers, whole
  constexpr int LOADS = TK / RPI;              // such instructions per tile
  constexpr int KM = D / 32;                   // matrix instructions per 16 keys of S^T
  constexpr int ND = D / 16;                   // d's per lane of a value row
  constexpr int VW = ND * ITEM / 4;            // dwords per lane of a value row
  const int row = blockIdx.z, kvh = blockIdx.y % p.Hkv, hb = blockIdx.y / p.Hkv, c = blockIdx.x;
  const int rep = p.Hq / p.Hkv, h0 = hb * 16, nh = min(16, rep - h0);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, g = lane >> 4;
  int len = p.kv_lens[row];
  const long head0 = (long)kvh * rep + h0;     // first query head of this workgroup
  bf16* orow = p.O + row * p.ldo + head0 * D;
  if (len <= 0) {                              // a free slot of the batch: zeros
    if (c == 0)
      for (int i = tid; i < nh * D / 8; i += 64 * WAVES) *(u32x4*)(orow + 8 * i) = u32x4{0, 0, 0, 0};
    return;
  }
  bool bad = len > p.table_width << p.page_shift;   // more keys than the row's table has pages for
  if (bad) len = p.table_width << p.page_shift;
  // at most as many chunks as the grid has: a bound on the lengths that was too small costs time, not keys
  const int splits_max = (int)gridDim.x;
  const int chunk = max(p.chunk, ((len + splits_max - 1) / splits_max + TK - 1) / TK * TK);
  const int nsplit = (len + chunk - 1) / chunk;
  if (c >= nsplit) return;
  const int begin = c * chunk, end = min(len - begin, chunk) + begin;

  union Shared {
    u32x4 keys[WAVES][LOADS * 64];             // each wave's tile of keys
    float o[WAVES][16][D + 4];
  };
  __shared__ Shared lds;
  __shared__ float m_s[WAVES][16], l_s[WAVES][16];
  __shared__ unsigned ticket_s;

  const int* table = p.table + row * p.table_stride;
  const int mask = (1 << p.page_shift) - 1;
  const int last_page = (len - 1) >> p.page_shift;
  // Whole rows of 128 bytes and more pass the caches by (each is read once); two rows of 64 share a line.
  constexpr bool PAST = CH >= 8;
  const char* kbase = p.k.base + kvh * p.k.head + (long)(lane / CH) * p.k.slot;
  const char* vbase = p.v.base + kvh * p.v.head + n * (ND * ITEM);
  u32x4* keys = lds.keys[wave];

  // Pieces of a key row lie in LDS exchanged by XOR with `turn` of the row, so that the eight lanes that read the same piece
  // of eight rows at once (keys 0 ... 3 and 8 ... 11, or 4 more) find them in eight different places of 128 bytes.
  auto turn = [](int key) {
    const int r = 4 * ((key >> 3) & 1) + (key & 3);
    return CH == 4 ? r >> 1 : r;
  };

  struct Tile {
    unsigned v[SUB][8][VW];
  };
  // Page ids of the tile at key k0, one per lane group and block of 32: that of keys 8 g ... 8 g + 7, which share a
  // page.  A page id outside the pool is not followed: the row's output says so instead.
  auto load_ids = [&](int (&ids)[SUB], int k0) {
#pragma unroll
    for (int s = 0; s < SUB; ++s) ids[s] = table[min((k0 + 32 * s + 8 * g) >> p.page_shift, last_page)];
  };
  auto check_ids = [&](int (&ids)[SUB]) {
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      const bool none = (unsigned)ids[s] >= (unsigned)p.num_pages;
      bad |= none;
      ids[s] = none ? 0 : ids[s];
    }
  };
  // Keys go to LDS without passing a register, in whole rows.
  auto load_keys = [&](const int (&ids)[SUB], int k0) {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");       // the tile before has been read
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      // the groups of eight keys of this instruction's rows: one, or two with 16 rows
      auto row0 = [&](int group) {
        const long page = __builtin_amdgcn_readlane(ids[group / 4], 16 * (group % 4));
        return page * p.k.page + (long)((k0 + 8 * group) & mask) * p.k.slot;
      };
      const int first = i * RPI;                              // of the tile
      long at = row0(first / 8) + (long)(first % 8) * p.k.slot;
      if constexpr (RPI == 16) at = lane < 32 ? at : row0(first / 8 + 1) - 8 * p.k.slot;      // kbase counts rows from the first
      const char* src = kbase + at + 16 * ((lane % CH) ^ turn(first + lane / CH));
      __builtin_amdgcn_global_load_lds(GLOBAL_PTR(src), LDS_PTR(keys + 64 * i), 16, 0, PAST ? 2 : 0);
    }
  };
  auto load_values = [&](Tile& x, const int (&ids)[SUB], int k0) {
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      const char* vp = vbase + (long)ids[s] * p.v.page + (long)((k0 + 32 * s + 8 * g) & mask) * p.v.slot;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if constexpr (VW == 4) {
          const u32x4 w = __builtin_nontemporal_load((const u32x4*)(vp + e * p.v.slot));
#pragma unroll
          for (int i = 0; i < 4; ++i) x.v[s][e][i] = w[i];
        } else if constexpr (VW == 2) {
          const u32x2 w = __builtin_nontemporal_load((const u32x2*)(vp + e * p.v.slot));
          x.v[s][e][0] = w[0];
          x.v[s][e][1] = w[1];
        } else {
          x.v[s][e][0] = *(const unsigned*)(vp + e * p.v.slot);
        }
      }
    }
  };

  // queries: column n of the operand is head n; element e of lane group g is d = 32 j + 8 g + e (bf16 keys) or
  // 64 (j / 2) + 16 g + 8 (j % 2) + e (e4m3: a 16-byte load of keys feeds two instructions)
  bf16x8 q[KM];
#pragma unroll
  for (int j = 0; j < KM; ++j) {
    const int d = F8 ? 64 * (j / 2) + 16 * g + 8 * (j % 2) : 32 * j + 8 * g;
    q[j] = *(const bf16x8*)(p.Q + row * p.ldq + (head0 + min(n, nh - 1)) * D + d);
  }
  const float scale = p.scale_log2 * (F8 ? p.k.scale[kvh] : 1.0f);

  f32x4 acc[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  // The maximum starts at the lowest number and not at -inf: scores of -inf (keys that hold infinities) weigh nothing even
  // where a wave or a chunk has no others.
  float m_run = -3.402823466e38f, l_run = 0.f; // l_run: this lane's keys only

  typedef float Scores[SUB][8];
  auto scores = [&](Scores& s) {
#pragma unroll
    for (int b = 0; b < SUB; ++b)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        f32x4 a = f32x4{0.f, 0.f, 0.f, 0.f};
        const int key = 32 * b + 8 * (n >> 2) + 4 * t + (n & 3);      // this lane's row
#pragma unroll
        for (int c = 0; c < CH / 4; ++c) {
          const u32x4 w = keys[key * CH + ((4 * c + g) ^ turn(key))];
          if constexpr (F8) {
            a = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen8(w[0], w[1]), q[2 * c], a, 0, 0, 0);
            a = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen8(w[2], w[3]), q[2 * c + 1], a, 0, 0, 0);
          } else {
            a = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w), q[c], a, 0, 0, 0);
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) s[b][4 * t + i] = a[i] * scale;
      }
  };
  auto add_values = [&](const Tile& x, Scores& s) {
    float mx = s[0][0];
#pragma unroll
    for (int b = 0; b < SUB; ++b)
#pragma unroll
      for (int e = 0; e < 8; ++e) mx = fmaxf(mx, s[b][e]);
    const float m_new = fmaxf(m_run, column_max(mx));
    const float alpha = __builtin_amdgcn_exp2f(m_run - m_new);
    m_run = m_new;
    l_run *= alpha;
#pragma unroll
    for (int i = 0; i < ND; ++i) acc[i] *= alpha;
#pragma unroll
    for (int b = 0; b < SUB; ++b) {
      u32x4 most;
      bf16x8 rest;
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        float w[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          w[i] = __builtin_amdgcn_exp2f(s[b][e + i] - m_new);
          l_run += w[i];
        }
        if constexpr (F8) {
          const bf16x2 r = {(bf16)w[0], (bf16)w[1]};
          most[e / 2] = __builtin_bit_cast(unsigned, r);
          rest[e] = (bf16)(w[0] - __uint_as_float(most[e / 2] << 16));
          rest[e + 1] = (bf16)(w[1] - __uint_as_float(most[e / 2] & 0xffff0000u));
        } else {
          unsigned below[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            below[i] = __builtin_elementwise_sub_sat(__float_as_uint(w[i]), 1u);
            rest[e + i] = (bf16)(w[i] - __uint_as_float(below[i] & 0xffff0000u));      // exact before its rounding
          }
          most[e / 2] = __builtin_amdgcn_perm(below[1], below[0], 0x07060302u);
        }
      }
#pragma unroll
      for (int dd = 0; dd < ND; ++dd) {
        u32x4 a;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (F8) {
            const unsigned w = __builtin_amdgcn_perm(x.v[b][2 * i + 1][dd / 4], x.v[b][2 * i][dd / 4], dd % 4 < 2 ? 0x05010400u : 0x07030602u);
            const bf16x2 two = dd % 2 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true)
                                      : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false);
            a[i] = __builtin_bit_cast(unsigned, two);
          } else {
            a[i] = __builtin_amdgcn_perm(x.v[b][2 * i + 1][dd / 2], x.v[b][2 * i][dd / 2], dd % 2 ? 0x07060302u : 0x05040100u);
          }
        }
        acc[dd] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), rest, acc[dd], 0, 0, 0);
        acc[dd] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, most), acc[dd], 0, 0, 0);
      }
    }
  };

  // A wave's next keys are requested as soon as its scores are there, its next values after their product; the other waves
  // of the SIMD compute meanwhile.  No load of the loop is conditional: the waits are counted, and a load that may have been
  // left out would have to be waited for as if it were.
  constexpr int STEP = WAVES * TK;
  int k0 = begin + wave * TK;
  if (k0 < end) {
    int ids[SUB], next[SUB];
    Tile x;
    Scores s;
    load_ids(ids, k0);
    load_ids(next, k0 + STEP);
    check_ids(ids);
    load_keys(ids, k0);
    load_values(x, ids, k0);
    for (; k0 + STEP < end; k0 += STEP) {
      check_ids(next);
#pragma unroll
      for (int b = 0; b < SUB; ++b) ids[b] = next[b];
      load_ids(next, k0 + 2 * STEP);
      scores(s);
      load_keys(ids, k0 + STEP);
      add_values(x, s);
      load_values(x, ids, k0 + STEP);
    }
    scores(s);
    // keys behind the end: their scores are replaced, and their values cleared (0 x NaN is NaN)
#pragma unroll
    for (int b = 0; b < SUB; ++b)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (k0 + 32 * b + 8 * g + e >= end) {
          s[b][e] = -INFINITY;
#pragma unroll
          for (int i = 0; i < VW; ++i) x.v[b][e][i] = 0;
        }
    add_values(x, s);
  }

  // ---- join the waves
  l_run = column_sum(l_run);
  if (__any(bad)) l_run = __builtin_nanf("");
  __syncthreads();                             // the last keys have been read everywhere
  if (g == 0) {
    m_s[wave][n] = m_run;
    l_s[wave][n] = l_run;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int dd = 0; dd < ND; ++dd) lds.o[wave][n][ND * (4 * g + i) + dd] = acc[dd][i];
  __syncthreads();
  const float vscale = F8 ? p.v.scale[kvh] : 1.0f;
  // two neighbouring d's of a head per thread
  auto finish = [&](int i, float o0, float o1, float l) {
    const bf16x2 o = {(bf16)(o0 / l * vscale), (bf16)(o1 / l * vscale)};
    *(bf16x2*)(orow + 2 * i) = o;
  };
  const long pair = ((long)row * p.Hkv + kvh) * ((rep + 15) / 16) + hb;
  // partials of all head blocks of a (row, kv head) lie together: rep heads of `splits_max` chunks
  const long block = (((long)row * p.Hkv + kvh) * rep + h0) * splits_max;
  unsigned long long* part = (unsigned long long*)(p.part + block * D);
  unsigned long long* stats = (unsigned long long*)(p.stats + block);
  // Partials pass between workgroups on different XCDs by the same forms as in decode_attention.hip: agent-scope stores and
  // loads (written through, read past the CU's cache), every store complete before the ticket is taken.
  auto put = [&](unsigned long long* at, float a, float b) {
    __hip_atomic_store(at, ((unsigned long long)__float_as_uint(b) << 32) | __float_as_uint(a), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  };
  auto get = [&](const unsigned long long* at) { return __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
  auto low = [](unsigned long long v) { return __uint_as_float((unsigned)v); };
  auto high = [](unsigned long long v) { return __uint_as_float((unsigned)(v >> 32)); };
  for (int i = tid; i < nh * D / 2; i += 64 * WAVES) {
    const int h = i / (D / 2), d = 2 * (i % (D / 2));
    float mx = m_s[0][h];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) mx = fmaxf(mx, m_s[w][h]);
    float o0 = 0.f, o1 = 0.f, l = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float f = __builtin_amdgcn_exp2f(m_s[w][h] - mx);
      o0 += lds.o[w][h][d] * f;
      o1 += lds.o[w][h][d + 1] * f;
      l += l_s[w][h] * f;
    }
    if (nsplit == 1) {
      finish(i, o0, o1, l);
    } else {
      put(part + (long)c * nh * (D / 2) + i, o0, o1);
      if (d == 0) put(stats + (long)c * nh + h, mx, l);
    }
  }
  if (nsplit == 1) return;

  // whether this workgroup is the last of `count` to come here
  auto last_of = [&](unsigned* ticket, int count) {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tid == 0) {
      ticket_s = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      if (ticket_s == (unsigned)(count - 1)) __hip_atomic_store(ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);   // for the next launch
    }
    __syncthreads();
    return ticket_s == (unsigned)(count - 1);
  };
  // the partials first, first + step, ... of at most JOIN chunks, all loads in flight together: to the output, or in the first's place
  __shared__ float2 stats_s[JOIN][16];
  auto join = [&](int first, int step, int count, bool output) {
    for (int i = tid; i < count * nh; i += 64 * WAVES) {
      const unsigned long long v = get(stats + (long)(first + i / nh * step) * nh + i % nh);
      stats_s[i / nh][i % nh] = float2{low(v), high(v)};
    }
    __syncthreads();
    // two columns per thread at a time: 32 loads in flight
    for (int i0 = tid; i0 < nh * D / 2; i0 += 128 * WAVES) {
      unsigned long long v[2][JOIN];
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int u = 0; u < JOIN; ++u)
          if (u < count && i0 + 64 * WAVES * e < nh * D / 2) v[e][u] = get(part + (long)(first + u * step) * nh * (D / 2) + i0 + 64 * WAVES * e);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int i = i0 + 64 * WAVES * e, h = i / (D / 2);
        if (i >= nh * D / 2) break;
        float mx = stats_s[0][h].x, o0 = 0.f, o1 = 0.f, l = 0.f;
        for (int u = 1; u < count; ++u) mx = fmaxf(mx, stats_s[u][h].x);
#pragma unroll
        for (int u = 0; u < JOIN; ++u)
          if (u < count) {
            const float f = __builtin_amdgcn_exp2f(stats_s[u][h].x - mx);
            l += stats_s[u][h].y * f;
            o0 += low(v[e][u]) * f;
            o1 += high(v[e][u]) * f;
          }
        if (output) {
          finish(i, o0, o1, l);
        } else {
          put(part + (long)first * nh * (D / 2) + i, o0, o1);
          if (i % (D / 2) == 0) put(stats + (long)first * nh + h, mx, l);
        }
      }
    }
  };
  unsigned* tickets = p.tickets + pair * TICKETS;
  if (nsplit <= JOIN) {
    if (last_of(tickets, nsplit)) join(0, 1, nsplit, true);
    return;
  }
  // groups of chunks first, then the groups
  const int group = c / JOIN, groups = (nsplit + JOIN - 1) / JOIN, mine = min(JOIN, nsplit - group * JOIN);
  if (!last_of(tickets + 1 + group, mine)) return;
  join(group * JOIN, 1, mine, false);
  if (last_of(tickets, groups)) join(0, JOIN, groups, true);
}

// What both entry points ask of a cache; 0 when it is sound.
int check_cache(const bagel_paged_cache* c, const char* who) {
  BAGEL_CHECK(c && c->k && c->v, "%s: null cache", who);
  BAGEL_CHECK(c->head_dim == 128 || c->head_dim == 64, "%s: head_dim %d not supported (128 or 64)", who, c->head_dim);
  BAGEL_CHECK(c->num_kv_heads > 0 && c->num_pages > 0, "%s: %d kv heads, %d pages", who, c->num_kv_heads, c->num_pages);
  BAGEL_CHECK(c->page_size >= 8 && (c->page_size & (c->page_size - 1)) == 0, "%s: page_size %d is not a power of two of at least 8", who,
              c->page_size);
  BAGEL_CHECK((long)c->num_pages * c->page_size <= 0x7fffffffL, "%s: %d pages of %d slots: slots are numbered in 32 bits", who, c->num_pages,
              c->page_size);
  BAGEL_CHECK(c->e4m3 == 0 || c->e4m3 == 1, "%s: e4m3=%d", who, c->e4m3);
  BAGEL_CHECK(!c->e4m3 || (c->k_scale && c->v_scale), "%s: an e4m3 cache needs k_scale and v_scale", who);
  const long step = c->e4m3 ? 16 : 8;   // elements in 16 bytes
  BAGEL_CHECK(((uintptr_t)c->k | (uintptr_t)c->v) % 16 == 0 &&
                  (c->k_page_stride | c->k_slot_stride | c->k_head_stride | c->v_page_stride | c->v_slot_stride | c->v_head_stride) % step == 0,
              "%s: pages, slots and heads of the cache must start on 16-byte boundaries", who);
  BAGEL_CHECK(c->k_slot_stride >= c->head_dim && c->v_slot_stride >= c->head_dim && c->k_page_stride >= c->head_dim &&
                  c->v_page_stride >= c->head_dim && c->k_head_stride >= c->head_dim && c->v_head_stride >= c->head_dim,
              "%s: a stride of the cache is below head_dim", who);
  return 0;
}

Pool pool_of(void* base, long page, long slot, long head, const void* scale, int e4m3) {
  const long item = e4m3 ? 1 : 2;
  return Pool{(char*)base, page * item, slot * item, head * item, e4m3 ? (const float*)scale : nullptr};
}
Pool k_pool(const bagel_paged_cache* c) { return pool_of(c->k, c->k_page_stride, c->k_slot_stride, c->k_head_stride, c->k_scale, c->e4m3); }
Pool v_pool(const bagel_paged_cache* c) { return pool_of(c->v, c->v_page_stride, c->v_slot_stride, c->v_head_stride, c->v_scale, c->e4m3); }

// Chunks that rows are split into where none has more than max_kv_len keys: whole rounds of the waves' tiles, two workgroups
// per CU.  A level of joins takes 3 to 4 us, about as long as a workgroup takes for 512 keys: rows up to there are not split, and
// rows of up to JOIN times as many into no more chunks than one level joins.  One row of 28 / 4 heads of 128 in bf16, so and with a
// chunk per round: 500 keys 6.4 and 7.6 us, 3000 9.2 and 12.3, 8192 13.1 and 13.6 (four rows: 17.9 and 22.0).
// Batches that fill the chip are not split, however long a row may be: max_kv_len is all that is known here, and a workgroup for a chunk
// that its row turns out not to have takes 16 ns to come and go.  Chunks of at most 8192 keys in every batch bring 100 rows of 500
// keys and one of 100000 from 1085 to 121 us, but 100 rows of 500 keys under a bound of 131072 from 26 to 133 us, and 1000 such rows from
// 184 to 1224 us (at most 4096: 101, 230 and 2190; at most 16384: 186, 94 and 827).
struct Split {
  int splits, chunk;
};
long head_blocks(int Hq, int Hkv) { return Hkv * (long)((Hq / Hkv + 15) / 16); }
long attend_round(int D, int e4m3) { return WAVES * 32 * (D * (e4m3 ? 1 : 2) == 256 ? 1 : 2); }
Split attend_split(long rows, int Hq, int Hkv, int D, int e4m3, long max_kv_len) {
  const long most = max_kv_len <= SHORT ? 1 : max_kv_len <= SHORT * JOIN ? JOIN : MAX_SPLITS;
  const long want = std::max(1L, std::min(most, 2L * bagel_cu_count() / (rows * head_blocks(Hq, Hkv))));
  const long round = attend_round(D, e4m3), rounds = std::max(1L, (max_kv_len + round - 1) / round);
  const long chunk = (rounds + want - 1) / want * round;
  return Split{(int)std::max(1L, (max_kv_len + chunk - 1) / chunk), (int)chunk};
}
// Only rows that are split take tickets, and then there are no more (row, kv head, head block) triples than CUs: the place of
// the tickets does not depend on the call, so that one workspace serves batches of every size.
long ticket_bytes() { return (long)bagel_cu_count() * TICKETS * 4; }
// Partials of the largest call with up to these rows and keys.
long most_partials(long rows, int Hq, int Hkv, int D, int e4m3, long max_kv_len) {
  const long round = attend_round(D, e4m3), rounds = std::max(1L, (max_kv_len + round - 1) / round);
  const long splits = std::min<long>(MAX_SPLITS, rounds);
  return splits > 1 ? std::min(rows * splits, 2L * bagel_cu_count() / head_blocks(Hq, Hkv)) * Hq : 0;
}

}  // namespace

extern "C" int bagel_paged_kv_append_bf16(const void* qkv, long ld, int rows, int Hq, const bagel_paged_cache* cache, const void* q_norm,
                                          const void* k_norm, const void* cos_table, const void* sin_table, int table_rows,
                                          const void* row_cs, const void* row_slot, void* Q, long ldq, float eps, int und_rounding,
                                          void* stream) {
  if (int rc = check_cache(cache, "bagel_paged_kv_append_bf16")) return rc;
  const int D = cache->head_dim, Hkv = cache->num_kv_heads;
  BAGEL_CHECK(rows >= 0 && Hq >= 0, "bagel_paged_kv_append_bf16: rows=%d Hq=%d", rows, Hq);
  if (rows == 0) return 0;
  BAGEL_CHECK(qkv && row_slot, "bagel_paged_kv_append_bf16: null operand");
  BAGEL_CHECK(!cos_table == !sin_table && !cos_table == !row_cs && (!cos_table || table_rows > 0),
              "bagel_paged_kv_append_bf16: the rotation needs cos_table, sin_table, table_rows and row_cs together");
  BAGEL_CHECK(ld % 8 == 0 && ld >= (long)(Hq + 2 * Hkv) * D, "bagel_paged_kv_append_bf16: bad leading dim");
  BAGEL_CHECK(!Q || (ldq % 8 == 0 && ldq >= (long)Hq * D), "bagel_paged_kv_append_bf16: bad leading dim of Q");
  BAGEL_CHECK(((uintptr_t)qkv | (uintptr_t)Q | (uintptr_t)q_norm | (uintptr_t)k_norm | (uintptr_t)cos_table | (uintptr_t)sin_table) % 16 == 0,
              "bagel_paged_kv_append_bf16: misaligned operand");
  if (!Q) {                                      // the heads from the keys on are all there is
    qkv = (const bf16*)qkv + (long)Hq * D;
    Hq = 0;
  }
  AppendParams p;
  p.qkv = (const bf16*)qkv; p.ld = ld; p.q_w = (const bf16*)q_norm; p.k_w = (const bf16*)k_norm;
  p.cos_t = (const bf16*)cos_table; p.sin_t = (const bf16*)sin_table;
  p.row_cs = (const int*)row_cs; p.row_slot = (const int*)row_slot; p.Q = (bf16*)Q; p.ldq = ldq;
  p.k = k_pool(cache); p.v = v_pool(cache);
  p.capacity = (long)cache->num_pages * cache->page_size;
  p.rows = rows; p.Hq = Hq; p.Hkv = Hkv; p.page_shift = __builtin_ctz(cache->page_size); p.cs_rows = table_rows;
  p.und_rounding = und_rounding; p.eps = eps;
  hipStream_t st = (hipStream_t)stream;
  if (D == 128) return cache->e4m3 ? launch_append<128, true>(p, st) : launch_append<128, false>(p, st);
  return cache->e4m3 ? launch_append<64, true>(p, st) : launch_append<64, false>(p, st);
}

extern "C" long bagel_paged_decode_attention_workspace_bytes(int rows, int Hq, int Hkv, int head_dim, long max_kv_len) {
  if (rows <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || head_dim <= 0 || max_kv_len < 0) return 0;
  if (max_kv_len == 0) max_kv_len = MAX_KEYS;
  return ticket_bytes() + std::max(most_partials(rows, Hq, Hkv, head_dim, 0, max_kv_len), most_partials(rows, Hq, Hkv, head_dim, 1, max_kv_len)) *
                              (head_dim + 2) * 4;
}

extern "C" int bagel_paged_decode_attention_bf16(const void* Q, long ldq, int rows, int Hq, const bagel_paged_cache* cache,
                                                 const void* page_table, long table_stride, int table_width, const void* kv_lens,
                                                 long max_kv_len, void* O, long ldo, float softmax_scale, void* workspace,
                                                 long workspace_bytes, void* stream) {
  if (int rc = check_cache(cache, "bagel_paged_decode_attention_bf16")) return rc;
  const int D = cache->head_dim, Hkv = cache->num_kv_heads;
  BAGEL_CHECK(rows >= 0 && rows <= 65535, "bagel_paged_decode_attention_bf16: rows=%d (at most 65535)", rows);
  BAGEL_CHECK(Hq > 0 && Hq % Hkv == 0, "bagel_paged_decode_attention_bf16: Hq=%d is not a multiple of the cache's %d kv heads", Hq, Hkv);
  if (rows == 0) return 0;
  BAGEL_CHECK(Q && O && page_table && kv_lens && workspace, "bagel_paged_decode_attention_bf16: null operand");
  BAGEL_CHECK(table_width > 0 && table_stride >= table_width, "bagel_paged_decode_attention_bf16: page table of %d pages, stride %ld",
              table_width, table_stride);
  BAGEL_CHECK(ldq % 8 == 0 && ldq >= (long)Hq * D && ldo % 8 == 0 && ldo >= (long)Hq * D,
              "bagel_paged_decode_attention_bf16: bad leading dim");
  BAGEL_CHECK(((uintptr_t)Q | (uintptr_t)O | (uintptr_t)workspace) % 16 == 0, "bagel_paged_decode_attention_bf16: misaligned operand");
  const int blocks = (Hq / Hkv + 15) / 16;
  BAGEL_CHECK((long)Hkv * blocks <= 65535, "bagel_paged_decode_attention_bf16: too many heads");
  const long room = (long)table_width * cache->page_size;
  BAGEL_CHECK(room <= MAX_KEYS, "bagel_paged_decode_attention_bf16: a page table of %d pages of %d slots (at most 2^30 keys a row)",
              table_width, cache->page_size);
  const long bound = max_kv_len > 0 ? std::min(max_kv_len, room) : room;
  const Split split = attend_split(rows, Hq, Hkv, D, cache->e4m3, bound);
  const long partials = split.splits > 1 ? (long)rows * Hq * split.splits : 0, need = ticket_bytes() + partials * (D + 2) * 4;
  BAGEL_CHECK(workspace_bytes >= need, "bagel_paged_decode_attention_bf16: workspace of %ld bytes, %ld needed", workspace_bytes, need);
  AttendParams p;
  p.Q = (const bf16*)Q; p.ldq = ldq; p.k = k_pool(cache); p.v = v_pool(cache);
  p.table = (const int*)page_table; p.table_stride = table_stride; p.table_width = table_width; p.num_pages = cache->num_pages;
  p.page_shift = __builtin_ctz(cache->page_size); p.kv_lens = (const int*)kv_lens; p.O = (bf16*)O; p.ldo = ldo;
  p.tickets = (unsigned*)workspace; p.part = (float*)((char*)workspace + ticket_bytes());
  p.Hq = Hq; p.Hkv = Hkv;
  p.chunk = split.chunk;
  p.stats = (float2*)(p.part + partials * D);
  p.scale_log2 = 1.4426950408889634f * (softmax_scale != 0.f ? softmax_scale : 1.0f / sqrtf((float)D));
  const dim3 grid(split.splits, Hkv * blocks, rows), block(64 * WAVES);
  hipStream_t st = (hipStream_t)stream;
  if (D == 128 && !cache->e4m3) hipLaunchKernelGGL((paged_attention_kernel<128, false>), grid, block, 0, st, p);
  else if (D == 128) hipLaunchKernelGGL((paged_attention_kernel<128, true>), grid, block, 0, st, p);
  else if (!cache->e4m3) hipLaunchKernelGGL((paged_attention_kernel<64, false>), grid, block, 0, st, p);
  else hipLaunchKernelGGL((paged_attention_kernel<64, true>), grid, block, 0, st, p);
  BAGEL_LAUNCH_CHECK();
  return 0;
}
