// Sampling of a row of logits (gfx950): temperature, top-k, top-p and min-p, from a random number that the caller gives.
//
// With the row's tokens ordered by descending logit, equal ones by ascending index, and w_i = exp((x_i - max) / T), every
// filter keeps a prefix of that order: top-k its first k, top-p the shortest prefix whose weights reach p of the weights
// that top-k left, min-p the tokens with w_i >= m.  The token drawn is the first whose running sum of weights exceeds
// u x (the kept weights).  A border of one of these sums decides a whole token, so sums have to be better than fp32 and
// must not depend on the order in which threads come by.
//
// No row is sorted.  Tokens are counted into bins of 1/32 octave of weight: with v = 32 log2(e) x / T, token x is in the
// bin of v's nearest whole number r, and weighs 2^((v - r) / 32), between 0.989 and 1.011, in that bin's unit, which is
// computed in 64 bits (to 2^-33) and counted as an integer in steps of 2^-32.  Integer sums are exact in any order, LDS
// atomics included, and bins and weights depend neither on the maximum nor on how a row is cut up: so the logits are read
// ONCE, in slices that know nothing of each other, and each slice's histogram reaches 44 octaves below its own maximum (what
// lies below weighs less than 2^-44 of the first token: nothing).  Where bins are added up, a bin's sum is brought to steps
// of 2^-42 of the first bin's unit.
//
// Two launches.  The first: a workgroup per slice, whose logits stay in registers: maximum, histogram, and a list of the
// slice's foremost tokens as (value, index) keys of 64 bits.  Bound by its vector instructions (busy 4/5 of the time), some
// forty a logit and thread: 14 for bin and weight, 10 where tokens are listed, the rest once per slice.  A bin's count and weight
// are the two parts of one 64-bit word, so that a logit is one LDS atomic.  Measured: 256 rows of 151936 32-bit logits, 156 MB,
// 48 us = 3.2 TB/s; 64 rows of 152064 bf16 ones, 19 MB, 15.8 us; a single such row 6.7 us.
// The second (7 us for a row whose borders are listed, 30 us and more where borders lie deep in some rows): one workgroup per row, in one
// of three ways:
//   - a top-k of a few: the lists hold it, whatever the row's weights are, so the first launch only counted tokens (without weights),
//     and the listed tokens are sorted;
//   - a top-p whose border lies among the listed tokens: they are sorted, and everything else is prefix sums over them;
//   - else each border is resolved by itself: its bin comes from the histogram, and the tokens of that bin alone, gathered from the
//     lists or, further down, from the row, are sorted.  A bin of too many tokens (equal or nearly equal logits) is first
//     narrowed by histograms over the key's bits, eleven at a time, which ends at a single token at the latest.
// Up to 64 tokens are sorted and summed by one wave in its registers.
#include "common.h"
#include <algorithm>
#include <type_traits>
#include "../../include/bagel_hip.h"

namespace {

typedef unsigned long long u64;

constexpr int OCTAVE = 32;           // bins per octave of weight
constexpr int BINS = 44 * OCTAVE;
constexpr int STEPS_LOG2 = 32;       // 2^32 steps to a bin's unit: 2^20 tokens of one bin stay below 2^53
constexpr int FINER = 10;            // bins are added up in steps of 2^-(32 + 10) of the first bin's unit
constexpr int COUNT_SHIFT = 48;      // a slice's bin: steps (2^15 tokens stay below 2^48), and the count above them
constexpr int SUB = 2048;            // bins of a narrowing histogram
constexpr int CAP = 4096;            // tokens that are sorted at once
constexpr int LIST = 512;            // tokens that a slice lists at most
constexpr int FEW = 512;             // a top-k up to here is looked for in the lists first
constexpr int THREADS = 1024;
constexpr int CHUNK = 8 * THREADS;   // logits that a workgroup loads at a time
constexpr int MAX_SLICES = 128;
constexpr int MAX_TOKENS = 1 << 20;

struct Slice {       // what the first launch says of a slice
  u64 best;          // the order key of its first maximum (where it is not greedy: of the maximum and no index)
  int listed, cut;   // tokens in its list; the last of its bins (from its own first) that the list holds
};

struct Params {
  const void* logits;
  long ld;
  int n, slices;
  const float *uniforms, *temperature, *top_p, *min_p;
  const int* top_k;
  int* tokens;
  float* logprobs;
  Slice* slice;                      // [rows][slices]
  u64* list;                         // [rows][slices][LIST], in no order
  u64* bins;                         // [rows][slices][BINS] count << COUNT_SHIFT | steps
};

// A NaN counts as a masked token: the maximum of a NaN and a number is the number.
__device__ __forceinline__ float clean(float x) { return fmaxf(x, -INFINITY); }

// Ascending in the order of the tokens: descending value (the two zeros are one), then ascending index.
__device__ __forceinline__ u64 order_key(float x, int i) {
  const unsigned b = __float_as_uint(x + 0.0f);
  return ((u64)((int)b < 0 ? b : b ^ 0x7fffffffu) << 32) | (unsigned)i;
}
__device__ __forceinline__ float key_value(u64 key) {
  const unsigned up = ~(unsigned)(key >> 32);
  return __uint_as_float(up ^ ((up >> 31) ? 0x80000000u : 0xffffffffu));
}

// The number of x's bin, and `part`, its v less that number: one fused multiply-add with 1.5 x 2^52 leaves the whole number
// nearest v in the sum's low bits (of x on a border the same one everywhere: nothing is rounded before).
constexpr double WHOLE = 6755399441055744.0;
__device__ __forceinline__ double bin_number(float x, double per, double& part) {
#pragma clang fp contract(off)
  const double v = (double)x * per;
  const bool small = __builtin_fabs(v) < 1125899906842624.0;      // 2^50
  const double near = __builtin_fma((double)x, per, WHOLE) - WHOLE, far = __builtin_rint(v);
  const double p = __builtin_fma((double)x, per, -near), q = v - far;
  part = small ? p : q;
  return small ? near : far;
}
__device__ __forceinline__ double bin_number(float x, double per) {
  double part;
  return bin_number(x, per, part);
}

// Bins counted down from that of a maximum `top`.
struct Scale {
  float top;
  double per;        // 32 log2(e) / T
  double inverse;    // of it, or nearly
  double base;       // number of the maximum's bin
};
constexpr double LN2 = 0.69314718055994530942;
__device__ __forceinline__ double per_unit(float t) { return OCTAVE / LN2 / (double)t; }
__device__ __forceinline__ Scale make_scale(float top, float t, double per) {
  return Scale{top, per, (double)t * (LN2 / OCTAVE), bin_number(top, per)};
}
__device__ __forceinline__ Scale make_scale(float top, float t) { return make_scale(top, t, per_unit(t)); }
// Token x's bin, BINS for one that weighs nothing, and `part`.  The maximum is in bin 0 even where v is no number (an
// infinite maximum, an infinite T).
__device__ __forceinline__ int bin_of(float x, const Scale& s, double& part) {
  const double d = s.base - bin_number(x, s.per, part);
  if (x == s.top) {
    part = part == part ? part : 0.0;
    return 0;
  }
  return d < (double)BINS ? (int)d : BINS;
}
__device__ __forceinline__ int bin_of(float x, const Scale& s) {
  double part;
  return bin_of(x, s, part);
}
// The next value, up or down, in the order of the values.
__device__ __forceinline__ float next(float x, int step) {
  const unsigned u = __float_as_uint(x), up = (u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u)) + step;
  return __uint_as_float(up ^ ((up >> 31) ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ float before(float x) { return next(x, -1); }
// The smallest value in a bin up to `b`: x is in one of them just when it is not below.  By a whole wave, whose lanes try the
// values around lowest / per; the quotient is within a step or two of it.
__device__ __forceinline__ float edge_of(int b, const Scale& s) {
#pragma clang fp contract(off)
  if (s.top == INFINITY) return s.top;
  if (!(s.per > 0.0)) return -3.402823466e38f;      // an infinite T: every value is in the maximum's bin
  const double lowest = s.base - b;
  const float x = next((float)((lowest - 0.5) * s.inverse), (int)(threadIdx.x & 63) - 32);
  const u64 inside = __ballot(bin_number(x, s.per) >= lowest);      // false for what lies below -inf in the bits' order: NaN
  return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), inside ? __ffsll(inside) - 1 : 63));
}
// 2^(part / 32) in steps: a cubic through its values at the four Chebyshev points of [-1/2, 1/2] (8e-11 of it off at most); a sum
// with 2^52 leaves the rounded steps in the low bits.
struct Cubic {
  double c3 = 1.693860906736419904e-06 * (1ull << STEPS_LOG2), c2 = 2.345984913507675400e-04 * (1ull << STEPS_LOG2);
  double c1 = 2.166084939218784396e-02 * (1ull << STEPS_LOG2), c0 = 9.999999999283390737e-01 * (1ull << STEPS_LOG2) + 4503599627370496.0;
  double whole = WHOLE;
  // kept in registers, only one of an instruction's two constants in scalar ones: otherwise every use copies them first
  __device__ __forceinline__ void settle() { asm volatile("" : "+v"(c3), "+s"(c2), "+s"(c1), "+s"(c0), "+v"(whole)); }
  // and `more` (a multiple of 2^32) on top
  __device__ __forceinline__ u64 steps(double part, u64 more = 0) const {
    double p = __builtin_fma(part, c3, c2);
    p = __builtin_fma(p, part, c1);
    p = __builtin_fma(p, part, c0);
    return (u64)__double_as_longlong(p) + (more - 0x4330000000000000ull);
  }
};
__device__ __forceinline__ u64 steps_of(double part) { return Cubic().steps(part); }
// Steps of bin b in the finer ones of bin 0; table: 2^(-j / 32).  Exact for b = 0: equal logits share out exactly.
__device__ __forceinline__ u64 scaled(u64 steps, int b, const double* table) {
  return (u64)__builtin_rint(__builtin_ldexp((double)steps * table[b % OCTAVE], FINER - b / OCTAVE));
}
// 2^(-j / 32) for j = 0 ... 31, by the exponential series.
struct Table {
  double at[OCTAVE];
  constexpr Table() : at() {
    for (int j = 0; j < OCTAVE; ++j) {
      double term = 1.0, sum = 1.0;
      for (int i = 1; i < 24; ++i) sum += term *= -LN2 * j / OCTAVE / i;
      at[j] = sum;
    }
  }
};
__constant__ const Table powers;

// The whole part of f x whole, 0 <= f <= 1, or with `up` the next whole number at or above it: exact, since tokens of
// equal weight put sums precisely on these borders.
__device__ __forceinline__ u64 part_of(float f, u64 whole, bool up) {
  if (!(f > 0.f)) return 0;
  int e;
  const u64 m = (u64)(frexpf(f, &e) * 16777216.f);       // f = m 2^(e - 24)
  const int sh = 24 - e;                                  // 23 for f = 1, up to 172
  const u64 low = m * whole, high = __umul64hi(m, whole);
  u64 part, rest;
  if (sh < 64) {
    part = (high << (64 - sh)) | (low >> sh);
    rest = low & ((1ull << sh) - 1);
  } else if (sh < 128) {
    part = sh == 64 ? high : high >> (sh - 64);
    rest = low | (sh == 64 ? 0 : high & ((1ull << (sh - 64)) - 1));
  } else {
    part = 0;
    rest = 1;
  }
  return part + (up && rest ? 1 : 0);
}

__device__ __forceinline__ u64 shfl_u64(u64 v, int from) {
  return ((u64)(unsigned)__shfl((int)(v >> 32), from) << 32) | (unsigned)__shfl((int)(unsigned)v, from);
}
// The smallest key of all lanes, in all of them.
__device__ __forceinline__ u64 wave_min(u64 v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = min(v, shfl_u64(v, (threadIdx.x & 63) ^ o));
  return v;
}

// The value of lane ^ W.
template <int W>
__device__ __forceinline__ unsigned xor_u32(unsigned v) {
  typedef __attribute__((ext_vector_type(2))) unsigned u32x2_;
  if constexpr (W < 16) return __float_as_uint(xor_lane<W>(__uint_as_float(v)));
  const u32x2_ a = W == 16 ? __builtin_amdgcn_permlane16_swap(v, v, false, false) : __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return threadIdx.x & W ? a[0] : a[1];
}
// One key per lane -> ascending over the wave: a bitonic network in registers.
template <int Q, int J>
__device__ __forceinline__ void wave_sort_step(u64& key) {
  const u64 other = ((u64)xor_u32<J>((unsigned)(key >> 32)) << 32) | xor_u32<J>((unsigned)key);
  const bool up = (threadIdx.x & Q) == 0 || Q == 64, lower = (threadIdx.x & J) == 0;
  key = (up == lower) == (other < key) ? other : key;
  if constexpr (J > 1) wave_sort_step<Q, J / 2>(key);
}
__device__ __forceinline__ void wave_sort(u64& key) {
  wave_sort_step<2, 1>(key);
  wave_sort_step<4, 2>(key);
  wave_sort_step<8, 4>(key);
  wave_sort_step<16, 8>(key);
  wave_sort_step<32, 16>(key);
  wave_sort_step<64, 32>(key);
}

typedef __attribute__((ext_vector_type(4))) unsigned u32x4_;
// Logits of a chunk as they are loaded.  settle(): what was made of them so far is not kept in registers.
template <typename T>
struct Raw;
template <>
struct Raw<bf16> {
  u32x4_ w;
  __device__ __forceinline__ float raw(int e) const { return __uint_as_float(e % 2 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16); }
  __device__ __forceinline__ float at(int e) const { return clean(raw(e)); }
  __device__ __forceinline__ void settle() { asm volatile("" : "+v"(w)); }
};
template <>
struct Raw<float> {
  f32x4 w[2];
  __device__ __forceinline__ float raw(int e) const { return w[e / 4][e % 4]; }
  __device__ __forceinline__ float at(int e) const { return clean(raw(e)); }
  __device__ __forceinline__ void settle() { asm volatile("" : "+v"(w[0]), "+v"(w[1])); }
};

// A row for loads of 16 bytes wherever it starts: places count from the boundary before it, `off` logits ahead of the first.
template <typename T>
struct Row {
  const T* x;        // place 0, which may be in front of the row
  int off, end;      // the row is at the places [off, end)
  __device__ __forceinline__ Row(const Params& p, int row) {
    const T* first = (const T*)p.logits + (long)row * p.ld;
    off = (int)((uintptr_t)first % 16 / sizeof(T));
    x = first - off;
    end = off + p.n;
  }
  // eight logits from place i on (a multiple of 8), -inf outside the row
  __device__ __forceinline__ Raw<T> load(int i) const {
    if (i >= off && i + 8 <= end) return *(const Raw<T>*)(x + i);
    T w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = i + e >= off && i + e < end ? x[i + e] : (T)-INFINITY;
    return __builtin_bit_cast(Raw<T>, w);
  }
};
// f(value, index) for this thread's share of a whole row's logits in [least, beyond) - a NaN for beyond: no upper end -, four
// loads in flight.
template <typename T, typename F>
__device__ __forceinline__ void for_range(const Params& p, int row, float least, float beyond, F f) {
  const Row<T> r(p, row);
  constexpr int N = 4;
  for (int i0 = 8 * (int)threadIdx.x; i0 < r.end; i0 += N * CHUNK) {
    Raw<T> v[N];
    if (i0 >= r.off && i0 + (N - 1) * CHUNK + 8 <= r.end) {
#pragma unroll
      for (int c = 0; c < N; ++c) v[c] = *(const Raw<T>*)(r.x + i0 + c * CHUNK);
    } else {
#pragma unroll
      for (int c = 0; c < N; ++c) v[c] = r.load(i0 + c * CHUNK);
    }
    // first which, then f: few lanes have one at the same place, and what f waits for is waited for once per round
    unsigned hits = 0;
#pragma unroll
    for (int c = 0; c < N; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) hits |= (unsigned)(v[c].raw(e) >= least && !(v[c].raw(e) >= beyond)) << (8 * c + e);
    for (; hits; hits &= hits - 1) {
      const int bit = __ffs(hits) - 1, i = i0 + bit / 8 * CHUNK + bit % 8;
      f((float)r.x[i], i - r.off);
    }
  }
}

struct Sums {
  u64 mass;
  unsigned count;
};
// Inclusive scans, over a wave by DPP row shifts and broadcasts, over the workgroup through the waves' totals.
template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned dpp_or_0(unsigned v) {
  return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}
template <typename V, typename F>
__device__ __forceinline__ V wave_scan(V v, F moved) {
  v += moved.template operator()<0x111, 0xf>(v);      // from the lane 1, 2, 4, 8 below in the row of 16
  v += moved.template operator()<0x112, 0xf>(v);
  v += moved.template operator()<0x114, 0xf>(v);
  v += moved.template operator()<0x118, 0xf>(v);
  v += moved.template operator()<0x142, 0xa>(v);      // the last lane of rows 0 and 2 to rows 1 and 3
  v += moved.template operator()<0x143, 0xc>(v);      // lane 31 to the upper half
  return v;
}
struct Move64 {
  template <int CTRL, int ROWS>
  __device__ __forceinline__ u64 operator()(u64 v) const {
    return ((u64)dpp_or_0<CTRL, ROWS>((unsigned)(v >> 32)) << 32) | dpp_or_0<CTRL, ROWS>((unsigned)v);
  }
};
struct Move32 {
  template <int CTRL, int ROWS>
  __device__ __forceinline__ unsigned operator()(unsigned v) const { return dpp_or_0<CTRL, ROWS>(v); }
};
__device__ __forceinline__ u64 wave_scan(u64 v) { return wave_scan(v, Move64{}); }
constexpr int WAVES = THREADS / 64;
// What the waves below hold, from the lanes' scan of the waves' totals.
static_assert(WAVES == 16, "a lane of a row per wave");
template <typename V, typename F>
__device__ __forceinline__ V row_scan(V v, F moved) {
  v += moved.template operator()<0x111, 0xf>(v);
  v += moved.template operator()<0x112, 0xf>(v);
  v += moved.template operator()<0x114, 0xf>(v);
  v += moved.template operator()<0x118, 0xf>(v);
  return v;
}
__device__ __forceinline__ unsigned below(unsigned total) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  return wave ? __builtin_amdgcn_readlane(row_scan(total, Move32{}), wave - 1) : 0;
}
__device__ __forceinline__ u64 below(u64 total) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const u64 v = row_scan(total, Move64{});
  return wave ? ((u64)(unsigned)__builtin_amdgcn_readlane((int)(v >> 32), wave - 1) << 32) | (unsigned)__builtin_amdgcn_readlane((int)v, wave - 1) : 0;
}
__device__ __forceinline__ u64 scan(u64 v, u64* per_wave, int stride) {
  v = wave_scan(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) per_wave[(threadIdx.x >> 6) * stride] = v;
  __syncthreads();
  return v + below(per_wave[(threadIdx.x & 15) * stride]);
}
__device__ __forceinline__ Sums scan(Sums v, Sums* per_wave) {
  v.mass = wave_scan(v.mass);
  v.count = wave_scan(v.count, Move32{});
  __syncthreads();
  if ((threadIdx.x & 63) == 63) per_wave[threadIdx.x >> 6] = v;
  __syncthreads();
  const Sums total = per_wave[threadIdx.x & 15];
  return Sums{v.mass + below(total.mass), v.count + below(total.count)};
}
// Bins -> sums up to and including them (two neighbours per thread).
template <int N>
__device__ __forceinline__ void prefix(u64* packed, Sums* per_wave) {
  static_assert(N <= 2 * THREADS && N % 2 == 0, "two bins per thread");
  const int t = threadIdx.x;
  u64 a = 0, b = 0;
  __syncthreads();
  if (2 * t < N) a = packed[2 * t], b = packed[2 * t + 1];
  const u64 v = scan(a + b, &per_wave->mass, sizeof(Sums) / 8);
  if (2 * t < N) packed[2 * t] = v - b, packed[2 * t + 1] = v;
  __syncthreads();
}
template <int N>
__device__ __forceinline__ void prefix(u64* mass, unsigned* count, Sums* per_wave) {
  static_assert(N <= 2 * THREADS && N % 2 == 0, "two bins per thread");
  const int t = threadIdx.x;
  Sums a{0, 0}, b{0, 0};
  __syncthreads();
  if (2 * t < N) a = Sums{mass[2 * t], count[2 * t]}, b = Sums{mass[2 * t + 1], count[2 * t + 1]};
  const Sums v = scan(Sums{a.mass + b.mass, a.count + b.count}, per_wave);
  if (2 * t < N) {
    mass[2 * t] = v.mass - b.mass, count[2 * t] = v.count - b.count;
    mass[2 * t + 1] = v.mass, count[2 * t + 1] = v.count;
  }
  __syncthreads();
}

__device__ __forceinline__ float row_temperature(const Params& p, int row) { return p.temperature ? p.temperature[row] : 1.0f; }
// A row's top-k: 0 where it leaves nothing out.
__device__ __forceinline__ int row_top_k(const Params& p, int row) {
  const int k = p.top_k ? p.top_k[row] : 0;
  return k >= 1 && k < p.n ? k : 0;
}

// ---- first launch: a workgroup per slice of C chunks
template <typename T, int C>
__global__ __launch_bounds__(THREADS, 8) void sample_slice_kernel(Params p) {
  const int row = blockIdx.y, slice = blockIdx.x, tid = threadIdx.x, wave = tid >> 6;
  __shared__ u64 bins[BINS];
  __shared__ unsigned count_s[THREADS / 64];
  __shared__ float top_s[THREADS / 64];
  __shared__ int first, reach, fits;
  __shared__ unsigned listed, reach_count, fits_count;
  const Row<T> r(p, row);
  const int place = slice * C * CHUNK + 8 * tid, from = place - r.off;      // in the row with what is ahead of it; in the row
  Raw<T> v[C];
  if (slice * C * CHUNK >= r.off && (slice + 1) * C * CHUNK <= r.end) {       // every load at once
#pragma unroll
    for (int c = 0; c < C; ++c) v[c] = *(const Raw<T>*)(r.x + place + c * CHUNK);
  } else {
#pragma unroll
    for (int c = 0; c < C; ++c) v[c] = r.load(place + c * CHUNK);
  }
  const float t = row_temperature(p, row);
  const int k = row_top_k(p, row);
  const bool few = k >= 1 && k <= FEW;
  const double per = per_unit(t);                      // while the logits are on their way
  for (int b = tid; b < BINS; b += THREADS) bins[b] = 0;
  if (tid == 0) first = 0x7fffffff, reach = BINS, fits = -1, listed = 0;
  float top = -INFINITY;
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) top = fmaxf(top, v[c].raw(e));      // passes over NaN
  top = wave_max(top);
  if ((tid & 63) == 0) top_s[wave] = top;
  __syncthreads();
  static_assert(THREADS / 64 == 16, "a lane per wave");
  top = row_reduce(top_s[tid & 15], [](float a, float b) { return fmaxf(a, b); });
  auto settle = [&] {
#pragma unroll
    for (int c = 0; c < C; ++c) v[c].settle();
  };
  settle();
  Slice* out = p.slice + (long)row * p.slices + slice;
  if (!(t > 0.f) || top == -INFINITY) {       // greedy, or nothing to choose from here: the first maximum
    int at = 0x7fffffff;
#pragma unroll
    for (int c = C - 1; c >= 0; --c)
#pragma unroll
      for (int e = 7; e >= 0; --e)
        if (v[c].at(e) == top) at = from + c * CHUNK + e;
    if (at != 0x7fffffff) atomicMin(&first, at);
    __syncthreads();
    if (tid == 0) *out = Slice{order_key(top, first), 0, BINS - 1};
    return;
  }
  const Scale s = make_scale(top, t, per);
  constexpr u64 ONE = 1ull << COUNT_SHIFT;
  static_assert(C * CHUNK <= 1 << 15, "a slice's sums fit their half of the word");
  const float low = before(edge_of(BINS - 1, s));
  if (s.base > -1e9 && s.base < 1e9 && low > -INFINITY) {
    // all but the strangest rows: bins as 32-bit integers, and `low`, which is just below the last bin, in place of all values
    // further down, masked ones and NaN among them: nothing here is infinite
    const int base = (int)s.base;
    Cubic cubic;
    cubic.settle();
    auto tally = [&](auto weights) {
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const double x = fmaxf(v[c].raw(e), low), whole = __builtin_fma(x, s.per, cubic.whole);
          const int b = base - (int)__double_as_longlong(whole);
          if (b < BINS) {
            if constexpr (weights.value) atomicAdd(&bins[b], cubic.steps(__builtin_fma(x, s.per, WHOLE - whole), ONE));
            else atomicAdd(&bins[b], ONE);
          }
        }
    };
    if (few) tally(std::false_type{});
    else tally(std::true_type{});
  } else {
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        double part;
        const int b = bin_of(v[c].at(e), s, part);
        if (b < BINS) atomicAdd(&bins[b], ONE + steps_of(part));
      }
  }
  __syncthreads();
  if (!few) {
    u64* at = p.bins + ((long)row * p.slices + slice) * BINS;
    for (int b = tid; b < BINS; b += THREADS) at[b] = bins[b];
  }
  // the list: the bins up to `cut`, the last that fits or, for a top-k of a few, the first that brings k tokens
  unsigned one = 0, two = 0, third = 0;                // tokens of this thread's two bins and of the next
  if (2 * tid < BINS) {
    one = bins[2 * tid] >> COUNT_SHIFT;
    two = bins[2 * tid + 1] >> COUNT_SHIFT;
    third = 2 * tid + 2 < BINS ? bins[2 * tid + 2] >> COUNT_SHIFT : LIST + 1;
  }
  unsigned upto = wave_scan(one + two, Move32{});
  if ((tid & 63) == 63) count_s[wave] = upto;
  __syncthreads();
  upto += below(count_s[tid & 15]);
  auto look = [&](int b, unsigned ahead, unsigned upto, unsigned after) {
    if (upto <= LIST && after > LIST) fits = b, fits_count = upto;
    if (few && upto >= (unsigned)k && ahead < (unsigned)k) reach = b, reach_count = upto;
  };
  if (2 * tid < BINS) {
    look(2 * tid, upto - two - one, upto - two, upto);
    look(2 * tid + 1, upto - two, upto, upto + third);
  }
  __syncthreads();
  const int cut = min(fits, reach);
  if (cut >= 0) {
    // places in the list by a scan over the lanes' numbers of tokens and one atomic per wave
    const float edge = edge_of(cut, s);
    settle();
    unsigned mine = 0;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) mine += v[c].raw(e) >= edge ? 1 : 0;
    const unsigned upto = wave_scan(mine, Move32{});
    unsigned base = 0;
    if ((tid & 63) == 63 && upto) base = atomicAdd(&listed, upto);
    base = __builtin_amdgcn_readlane(base, 63) + upto - mine;
    char* at = (char*)(p.list + ((long)row * p.slices + slice) * LIST);
    unsigned to = 8 * base;
    settle();
    if (mine && base + mine <= LIST)                  // always: cut is a bin that fits
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (v[c].raw(e) >= edge) {
            *(u64*)(at + to) = order_key(v[c].raw(e), from + c * CHUNK + e);
            to += 8;
          }
  }
  if (tid == 0) *out = Slice{order_key(top, 0), cut < 0 ? 0 : (int)(fits <= reach ? fits_count : reach_count), cut};
}

// ---- second launch: one workgroup per row finds the token
struct Hit {         // a token of the order, with the steps of bin 0 up to and including it
  u64 key, mass;
};

template <typename T>
__global__ __launch_bounds__(THREADS) void sample_pick_kernel(Params p) {
  const int row = blockIdx.x, tid = threadIdx.x;
  __shared__ u64 mass[BINS];                 // steps of bin 0 up to and including a bin
  __shared__ unsigned count[BINS];
  __shared__ u64 work[CAP];                  // the tokens being sorted, or the histogram of a narrowing step
  __shared__ double table[OCTAVE];
  __shared__ Sums per_wave[THREADS / 64];
  __shared__ int listed_s[MAX_SLICES];       // tokens in a slice's list
  __shared__ int down[MAX_SLICES];           // a slice's first bin, counted from the row's
  __shared__ int found, lowest_cut, enough;
  __shared__ unsigned gathered, inside_s;
  __shared__ u64 best_s, edge_s;
  __shared__ Hit hit_s;
  u64* sub_mass = work;                      // [SUB]
  unsigned* sub_count = (unsigned*)(work + SUB);

  // What other workgroups just wrote is two microseconds away, so the lists are on their way before anything is known of
  // them: half the workgroup per slice, the first ten slices at once.
  static_assert(2 * LIST == THREADS, "a thread per token of two lists");
  constexpr int AHEAD = 5;
  const int half = tid / LIST;
  const u64* list = p.list + (long)row * p.slices * LIST + tid % LIST;
  u64 ahead[AHEAD];
#pragma unroll
  for (int c = 0; c < AHEAD; ++c) ahead[c] = half + 2 * c < p.slices ? list[(long)(half + 2 * c) * LIST] : 0;
  Slice mine{~0ull, 0, BINS - 1};
  if (tid < p.slices) mine = p.slice[(long)row * p.slices + tid];
  const float t = row_temperature(p, row), top_p = p.top_p ? p.top_p[row] : 1.0f, min_p = p.min_p ? p.min_p[row] : 0.f, u = p.uniforms[row];
  const int k = row_top_k(p, row);
  const bool few = k >= 1 && k <= FEW;
  const double power = powers.at[tid % OCTAVE];
  if (tid == 0) best_s = ~0ull, lowest_cut = BINS, enough = 1, gathered = 0;
  __syncthreads();
  if (tid < OCTAVE) table[tid] = power;
  if (tid < MAX_SLICES) {
    const u64 m = wave_min(mine.best);
    if ((tid & 63) == 0) atomicMin(&best_s, m);
  }
  __syncthreads();
  const u64 best = best_s;
  const float top = key_value(best);
  if (!(t > 0.f) || top == -INFINITY) {
    if (tid == 0) {
      p.tokens[row] = top == -INFINITY ? 0 : (int)(unsigned)best;
      if (p.logprobs) p.logprobs[row] = top == -INFINITY ? -INFINITY : 0.f;
    }
    return;
  }
  const Scale s = make_scale(top, t);
  auto place = [&](u64 key, double& part) { return bin_of(key_value(key), s, part); };
  auto weight = [&](float x) { return x == top ? 1.0 : exp(((double)x - (double)top) / (double)t); };
  // a token's steps, in those of bin 0
  auto steps = [&](u64 key) {
    double part;
    const int b = place(key, part);
    return b < BINS ? scaled(steps_of(part), b, table) : 0ull;
  };
  double top_part;
  place(best, top_part);
  const u64 top_steps = steps_of(top_part) << FINER;        // scaled() for bin 0
  if (tid == 0) hit_s = Hit{best, top_steps};
  if (tid < MAX_SLICES) {
    const float their = key_value(mine.best);
    const double d = s.base - make_scale(their, t).base;
    const int off = tid >= p.slices || their == -INFINITY ? BINS : their == top ? 0 : d < (double)BINS ? (int)d : BINS;
    down[tid] = off;
    if (off < BINS && mine.cut < BINS - 1) atomicMin(&lowest_cut, mine.cut + off);
    if (mine.listed < k && mine.cut < BINS - 1) enough = 0;       // tokens of the top k may be missing
    listed_s[tid] = mine.listed;
  }
  __syncthreads();

  // f(key) of every listed token
  auto for_listed = [&](auto f) {
    for (int s0 = half; s0 < p.slices; s0 += 2 * AHEAD) {
      u64 key[AHEAD];
#pragma unroll
      for (int c = 0; c < AHEAD; ++c) {
        key[c] = ahead[c];
        if (s0 != half && s0 + 2 * c < p.slices) key[c] = list[(long)(s0 + 2 * c) * LIST];
      }
#pragma unroll
      for (int c = 0; c < AHEAD; ++c)
        if (s0 + 2 * c < p.slices && tid % LIST < listed_s[s0 + 2 * c]) f(key[c]);
    }
  };
  auto put = [&](u64 key) {
    const unsigned at = atomicAdd(&gathered, 1u);
    if (at < CAP) work[at] = key;
  };
  // work[0 ... len) ascending: a bitonic network whose steps inside 64 keys run in a wave's registers
  auto sort = [&](int len) {
    int size = 64;
    while (size < len) size *= 2;
    __syncthreads();
    for (int i = len + tid; i < size; i += THREADS) work[i] = ~0ull;
    __syncthreads();
    const int wave = tid >> 6, lane = tid & 63;
    for (int at = wave * 64; at < size; at += THREADS) {
      const u64 turned = at & 64 ? ~0ull : 0;                // descending: ascending in the complement
      u64 key = work[at + lane] ^ turned;
      wave_sort(key);
      work[at + lane] = key ^ turned;
    }
    for (int q = 128; q <= size; q *= 2) {
      for (int j = q / 2; j >= 64; j /= 2) {
        __syncthreads();
        for (int t = tid; t < size / 2; t += THREADS) {
          const int i = 2 * t - (t & (j - 1)), o = i + j;
          const u64 a = work[i], b = work[o];
          if ((a > b) == ((i & q) == 0)) work[i] = b, work[o] = a;
        }
      }
      __syncthreads();
      for (int at = wave * 64; at < size; at += THREADS) {
        const u64 turned = at & q ? ~0ull : 0;
        u64 key = work[at + lane] ^ turned;
        wave_sort_step<64, 32>(key);
        work[at + lane] = key ^ turned;
      }
    }
    __syncthreads();
  };
  constexpr int EACH = CAP / THREADS;        // neighbours per thread in the sorted order
  // f(key) of the sorted tokens as sums up to and including each of the thread's own, and up to the one before them
  auto sums_of = [&](int len, u64& before, u64 (&upto)[EACH], auto f) {
    u64 sum = 0;
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      const int i = tid * EACH + e;
      if (i < len) sum += f(work[i]);
      upto[e] = sum;
    }
    before = scan(sum, &per_wave->mass, sizeof(Sums) / 8) - sum;
#pragma unroll
    for (int e = 0; e < EACH; ++e) upto[e] += before;
  };
  auto answer = [&](u64 key, u64 kept) {               // by one thread
    p.tokens[row] = (int)(unsigned)key;
    if (p.logprobs) {
      const float x = key_value(key);
      p.logprobs[row] = (float)((x == top ? 0.0 : ((double)x - (double)top) / (double)t) - log((double)kept / (double)top_steps));
    }
  };
  auto p_target = [&](u64 whole) { return max((u64)1, part_of(top_p, whole, true)); };
  auto u_target = [&](u64 kept) { return 1 + min(part_of(u < 1.0f ? u : u >= 1.0f ? 1.0f : 0.f, kept, false), kept - 1); };

  // the token, from `len` tokens in work that hold everything the filters keep; whole: the weights that top_p is a share of
  // (of the first k of these where there is a top-k)
  auto finish = [&](int len, u64 whole) {
    if (len <= 64) {
      if (tid >= 64) return;
      u64 key = tid < len ? work[tid] : ~0ull;
      wave_sort(key);
      const u64 sum = wave_scan(tid < len ? steps(key) : 0);
      // the place at which the sums reach the target (the last one where roundings leave them short)
      auto place_at = [&](u64 target) {
        const u64 m = __ballot(tid < len && sum >= target);
        return m ? __ffsll(m) - 1 : len - 1;
      };
      u64 kept = whole;
      if (k) whole = kept = shfl_u64(sum, min(k, len) - 1);
      if (top_p < 1.0f) kept = shfl_u64(sum, place_at(p_target(whole)));
      if (min_p > 0.f) {
        const u64 m = __ballot(tid < len && sum <= kept && (tid == 0 || weight(key_value(key)) >= (double)min_p));
        kept = shfl_u64(sum, 63 - __clzll(m));
      }
      const int at = place_at(u_target(kept));
      if (tid == at) answer(key, kept);
      return;
    }
    sort(len);
    u64 before, upto[EACH];
    sums_of(len, before, upto, steps);
    // the token for which `is` holds, given its place in the order and the sums before and up to it
    auto token_where = [&](auto is) {
#pragma unroll
      for (int e = 0; e < EACH; ++e)
        if (tid * EACH + e < len && is(tid * EACH + e, e ? upto[e ? e - 1 : 0] : before, upto[e])) hit_s = Hit{work[tid * EACH + e], upto[e]};
      __syncthreads();
      const Hit h = hit_s;
      __syncthreads();
      return h;
    };
    // (the last token is taken where the roundings of single tokens and of whole bins leave the sum short)
    auto token_at = [&](u64 target) {
      return token_where([&](int i, u64 from, u64 to) { return from < target && (to >= target || i == len - 1); });
    };
    u64 kept = whole;
    if (k) whole = kept = token_where([&](int i, u64, u64) { return i == min(k, len) - 1; }).mass;
    if (top_p < 1.0f) kept = token_at(p_target(whole)).mass;
    if (min_p > 0.f) {
      // a prefix: the largest sum among those that stay
      if (tid == 0) edge_s = 0;
      __syncthreads();
#pragma unroll
      for (int e = 0; e < EACH; ++e) {
        const int i = tid * EACH + e;
        if (i < len && upto[e] <= kept && (i == 0 || weight(key_value(work[i])) >= (double)min_p)) atomicMax(&edge_s, upto[e]);
      }
      __syncthreads();
      kept = edge_s;
    }
    const Hit h = token_at(u_target(kept));
    if (tid == 0) answer(h.key, kept);
  };

  // the bin of N for which `is` holds, given the bin; N where there is none
  auto find = [&](int n, auto is) {
    if (tid == 0) found = n;
    __syncthreads();
    for (int b = 2 * tid; b < min(2 * tid + 2, n); ++b)
      if (is(b)) found = b;
    __syncthreads();
    const int b = found;
    __syncthreads();
    return b;
  };
  if (few && enough) {
    // of the slices' first k only those in the bins of the row's first k (or all, where that many weigh nothing)
    for (int b = tid; b < BINS; b += THREADS) count[b] = 0;
    if (tid == 0) found = BINS;
    __syncthreads();
    for_listed([&](u64 key) {
      const int b = bin_of(key_value(key), s);
      if (b < BINS) atomicAdd(&count[b], 1u);
    });
    __syncthreads();
    unsigned one = 0, two = 0;                           // tokens of this thread's two bins
    if (2 * tid < BINS) one = count[2 * tid], two = count[2 * tid + 1];
    unsigned upto = wave_scan(one + two, Move32{});
    if ((tid & 63) == 63) per_wave[tid >> 6].count = upto;
    __syncthreads();
    upto += below(per_wave[tid & 15].count);
    if (upto >= (unsigned)k && upto - two - one < (unsigned)k) {
      const bool first = upto - two >= (unsigned)k;
      found = first ? 2 * tid : 2 * tid + 1;
      inside_s = first ? upto - two : upto;
    } else if (tid == THREADS - 1 && upto < (unsigned)k) {
      inside_s = upto;
    }
    __syncthreads();
    const int b = min(found, BINS - 1);
    if (inside_s <= CAP) {
      const float edge = edge_of(b, s);
      for_listed([&](u64 key) {
        if (key_value(key) >= edge) put(key);
      });
      __syncthreads();
      finish((int)min(gathered, (unsigned)CAP), 0);
      return;
    }
    __syncthreads();
  }

  // the row's histogram: the slices' or, where the lists of a top-k did not do and weights were left out, made here
  if (few) {
    for (int b = tid; b < BINS; b += THREADS) mass[b] = 0, count[b] = 0;
    __syncthreads();
    for_range<T>(p, row, edge_of(BINS - 1, s), __builtin_nanf(""), [&](float x, int) {
      double part;
      const int b = bin_of(x, s, part);
      if (b < BINS) {
        atomicAdd(&count[b], 1u);
        atomicAdd(&mass[b], steps_of(part));
      }
    });
    __syncthreads();
    for (int b = tid; b < BINS; b += THREADS) mass[b] = scaled(mass[b], b, table);
  } else {
    constexpr int N = (BINS + THREADS - 1) / THREADS;
    u64 m[N] = {};
    unsigned c[N] = {};
    constexpr int B = 2 * AHEAD;
    for (int s0 = 0; s0 < p.slices; s0 += B) {         // twenty loads in flight
      u64 both[B][N];
#pragma unroll
      for (int i = 0; i < B; ++i) {
        const int sl = min(s0 + i, p.slices - 1), off = s0 + i < p.slices ? down[sl] : BINS;
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const int theirs = tid + e * THREADS - off;
          both[i][e] = theirs >= 0 && theirs < BINS ? p.bins[((long)row * p.slices + sl) * BINS + theirs] : 0;
        }
      }
#pragma unroll
      for (int i = 0; i < B; ++i)
#pragma unroll
        for (int e = 0; e < N; ++e) {
          m[e] += both[i][e] & ((1ull << COUNT_SHIFT) - 1);
          c[e] += (unsigned)(both[i][e] >> COUNT_SHIFT);
        }
    }
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (tid + e * THREADS < BINS) mass[tid + e * THREADS] = scaled(m[e], tid + e * THREADS, table), count[tid + e * THREADS] = c[e];
  }
  prefix<BINS>(mass, count, per_wave);
  const u64 total = mass[BINS - 1];

  auto bin_by_count = [&](u64 target) { return find(BINS, [&](int b) { return (b == 0 || count[b - 1] < target) && count[b] >= target; }); };
  auto bin_by_mass = [&](u64 target) { return find(BINS, [&](int b) { return (b == 0 || mass[b - 1] < target) && mass[b] >= target; }); };

  // the first token of the order at which the count / the steps reach the target, somewhere in `bin`
  auto resolve = [&](int bin, bool by_count, u64 target) {
    const Sums base{bin ? mass[bin - 1] : 0, bin ? count[bin - 1] : 0};      // before the bin
    Sums inner{0, 0};                                                        // in the bin before what is left of it, in its own steps
    unsigned inside = count[bin] - base.count;
    u64 low = 0, high = ~0ull;
    auto reached = [&](u64 m, unsigned c) {
      return by_count ? (u64)(base.count + inner.count + c) >= target : base.mass + scaled(inner.mass + m, bin, table) >= target;
    };
    const float least = edge_of(bin, s), beyond = bin ? edge_of(bin - 1, s) : __builtin_nanf("");
    auto part_steps = [&](u64 key) {
      double part;
      place(key, part);
      return steps_of(part);
    };
    for (int sh = 53; inside > CAP; sh = max(sh - 11, 0)) {
      __syncthreads();
      for (int b = tid; b < SUB; b += THREADS) sub_mass[b] = 0, sub_count[b] = 0;
      __syncthreads();
      for_range<T>(p, row, least, beyond, [&](float x, int i) {
        const u64 key = order_key(x, i);
        if (key < low || key > high) return;
        const int b = (int)((key - low) >> sh);
        atomicAdd(&sub_count[b], 1u);
        atomicAdd(&sub_mass[b], part_steps(key));
      });
      prefix<SUB>(sub_mass, sub_count, per_wave);
      const int b = min(find(SUB, [&](int b) { return (b == 0 || !reached(sub_mass[b - 1], sub_count[b - 1])) && reached(sub_mass[b], sub_count[b]); }), SUB - 1);
      const Sums before{b ? sub_mass[b - 1] : 0, b ? sub_count[b - 1] : 0};
      inside = sub_count[b] - before.count;
      inner.mass += before.mass;
      inner.count += before.count;
      low += (u64)b << sh;
      high = low + ((1ull << sh) - 1);
      __syncthreads();
    }
    __syncthreads();
    if (tid == 0) gathered = 0;
    __syncthreads();
    auto gather = [&](u64 key) {
      if (key >= low && key <= high) put(key);
    };
    if (bin <= lowest_cut) for_listed([&](u64 key) {
      if (key_value(key) >= least && !(key_value(key) >= beyond)) gather(key);
    });
    else for_range<T>(p, row, least, beyond, [&](float x, int i) { gather(order_key(x, i)); });
    __syncthreads();
    const int len = (int)min(gathered, (unsigned)CAP);
    sort(len);
    u64 before, upto[EACH];
    sums_of(len, before, upto, part_steps);
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      const int i = tid * EACH + e;
      if (i < len && (i == 0 || !reached(e ? upto[e ? e - 1 : 0] : before, (unsigned)i)) && (i == len - 1 || reached(upto[e], (unsigned)i + 1)))
        hit_s = Hit{work[i], base.mass + scaled(inner.mass + upto[e], bin, table)};
    }
    __syncthreads();
    const Hit h = hit_s;
    __syncthreads();
    return h;
  };

  const int k_bin = k ? bin_by_count((u64)k) : BINS;
  const bool has_k = k_bin < BINS;                     // further down there is no weight to cut off
  // everything that stays lies in the bins up to this one
  const int last_bin = has_k ? k_bin : top_p < 1.0f ? bin_by_mass(p_target(total)) : BINS;
  if (last_bin <= lowest_cut && last_bin < BINS && count[last_bin] <= CAP && (has_k || !k)) {
    const float edge = edge_of(last_bin, s);
    for_listed([&](u64 key) {
      if (key_value(key) >= edge) put(key);
    });
    __syncthreads();
    finish((int)min(gathered, (unsigned)CAP), total);
    return;
  }

  Hit border{~0ull, total};                            // the last token kept
  if (has_k) border = resolve(k_bin, true, (u64)k);
  if (top_p < 1.0f) {
    const u64 target = p_target(border.mass);
    const int bin = bin_by_mass(target);
    if (bin < BINS) border = resolve(bin, false, target);
  }
  u64 kept = border.mass;
  if (min_p > 0.f) {
    // the threshold's bin, and one to each side for the roundings at the bins' borders: only their tokens are looked at
    const double edge = -log((double)min_p) * (OCTAVE / LN2);
    constexpr int LOOK = 6;
    const int b0 = edge < 2.0 ? 0 : edge < BINS ? (int)edge - 2 : BINS, b1 = b0 + LOOK - 1;
    if (b0 < BINS && (border.key == ~0ull || bin_of(key_value(border.key), s) >= b0)) {
      // by bin, so that the sum of what stays is rounded as resolve() rounds it and a draw of all of it ends at its last token
      u64 sum[LOOK] = {};
      __syncthreads();
      if (tid < LOOK) work[tid] = 0;
      __syncthreads();
      const float least = edge_of(min(b1, BINS - 1), s), beyond = b0 ? edge_of(b0 - 1, s) : __builtin_nanf("");
      auto add = [&](u64 key) {
        if (!(key <= border.key && weight(key_value(key)) >= (double)min_p)) return;
        double part;
        const int b = place(key, part);
        const u64 mine = steps_of(part);
#pragma unroll
        for (int i = 0; i < LOOK; ++i) sum[i] += b == b0 + i ? mine : 0;
      };
      if (b1 <= lowest_cut) for_listed([&](u64 key) {
        if (key_value(key) >= least && !(key_value(key) >= beyond)) add(key);
      });
      else for_range<T>(p, row, least, beyond, [&](float x, int i) { add(order_key(x, i)); });
#pragma unroll
      for (int i = 0; i < LOOK; ++i) {
        const u64 all = wave_scan(sum[i]);
        if ((tid & 63) == 63 && all) atomicAdd(&work[i], all);
      }
      __syncthreads();
      int last = LOOK - 1;                               // the last bin with a token that stays; all of those before it do
      while (last > 0 && !work[last]) --last;
      const int b = b0 + last;
      kept = max((b ? mass[b - 1] : 0) + scaled(work[last], b, table), top_steps);     // the first token stays whatever min_p is
      __syncthreads();
    }
  }
  const u64 target = u_target(kept);
  const Hit h = resolve(min(bin_by_mass(target), BINS - 1), false, target);
  if (tid == 0) answer(h.key, kept);
}

// Chunks per slice.  A round of one workgroup per CU takes 1.3 us + 1.1 us a chunk, in both types (two share a CU, so a second
// one beside the first costs as much as one behind it), and whole rounds count; the second launch waits 2 us for every ten slices of a
// row.  Over 120 sizes, 1 to 600 rows of 5000 to 10^6 tokens, this picks the fastest of the four or one within 3 % of it.  Calls of
// 1, 2, 3 and 4 chunks (us, bf16; top-k 20): 32 rows of 152064 20.0 17.4 15.2 16.2; 64 of them 24.6 20.3 18.6 20.1; 128 of
// them 36.4 28.2 28.5 27.7; 128 of 32000 14.6 13.2 14.6 15.5; 32-bit logits, 64 rows of 152064 25.1 22.1 20.8 22.8.
int slices_of(int n, int chunks) { return (n + chunks * CHUNK - 1) / (chunks * CHUNK); }
int chunks_of(int rows, int n) {
  const int most = 4;                  // a slice's steps fit 48 bits, and two workgroups' registers a CU
  int best = most;
  long least = 0;
  for (int c = most; c >= 1 && slices_of(n, c) <= MAX_SLICES; --c) {
    const long rounds = ((long)rows * slices_of(n, c) + bagel_cu_count() - 1) / bagel_cu_count();
    const long time = rounds * (13 + 11 * c) + 20 * ((slices_of(n, c) + 9) / 10);        // in tenths of a microsecond
    if (c == most || time < least) best = c, least = time;
  }
  return best;
}
template <typename T>
int launch(const Params& p, int rows, int chunks, hipStream_t st) {
  const dim3 grid(p.slices, rows), block(THREADS);
  if (chunks == 4) hipLaunchKernelGGL((sample_slice_kernel<T, 4>), grid, block, 0, st, p);
  else if (chunks == 3) hipLaunchKernelGGL((sample_slice_kernel<T, 3>), grid, block, 0, st, p);
  else if (chunks == 2) hipLaunchKernelGGL((sample_slice_kernel<T, 2>), grid, block, 0, st, p);
  else hipLaunchKernelGGL((sample_slice_kernel<T, 1>), grid, block, 0, st, p);
  hipLaunchKernelGGL(sample_pick_kernel<T>, dim3(rows), block, 0, st, p);
  BAGEL_LAUNCH_CHECK();
  return 0;
}
// Rows that do not start on 16-byte boundaries reach up to seven places further.
int places_of(int n) { return n + 7; }
long workspace_of(int rows, int n) {
  return (long)rows * slices_of(places_of(n), chunks_of(rows, places_of(n))) * (sizeof(Slice) + LIST * 8 + BINS * 8);
}

}  // namespace

extern "C" long bagel_sample_rows_workspace_bytes(int rows, int n) {
  long most = 0;       // fewer rows can be cut into more slices altogether
  if (n > 0 && n <= MAX_TOKENS)
    for (int r = 1; r <= std::min(rows, 65535); ++r) most = std::max(most, workspace_of(r, n));
  return most;
}

extern "C" int bagel_sample_rows(const void* logits, long ld, int rows, int n, int logits_f32, const void* uniforms, const void* temperature,
                                 const void* top_k, const void* top_p, const void* min_p, void* tokens, void* logprobs,
                                 void* workspace, long workspace_bytes, void* stream) {
  BAGEL_CHECK(rows >= 0 && rows <= 65535, "bagel_sample_rows: rows=%d (at most 65535)", rows);
  BAGEL_CHECK(n > 0 && n <= MAX_TOKENS, "bagel_sample_rows: %d tokens (1 to 2^20)", n);
  BAGEL_CHECK(logits_f32 == 0 || logits_f32 == 1, "bagel_sample_rows: logits_f32=%d", logits_f32);
  if (rows == 0) return 0;
  BAGEL_CHECK(logits && uniforms && tokens && workspace, "bagel_sample_rows: null operand");
  BAGEL_CHECK(ld >= n || ld == 0, "bagel_sample_rows: leading dim %ld below %d tokens", ld, n);
  BAGEL_CHECK((uintptr_t)logits % (logits_f32 ? 4 : 2) == 0 && (uintptr_t)workspace % 16 == 0, "bagel_sample_rows: misaligned operand");
  const long need = workspace_of(rows, n);
  BAGEL_CHECK(workspace_bytes >= need, "bagel_sample_rows: workspace of %ld bytes, %ld needed", workspace_bytes, need);
  Params p;
  p.logits = logits; p.ld = ld; p.n = n;
  p.uniforms = (const float*)uniforms; p.temperature = (const float*)temperature; p.top_k = (const int*)top_k;
  p.top_p = (const float*)top_p; p.min_p = (const float*)min_p; p.tokens = (int*)tokens; p.logprobs = (float*)logprobs;
  const int c = chunks_of(rows, places_of(n));
  p.slices = slices_of(places_of(n), c);
  const long slices = (long)rows * p.slices;
  p.slice = (Slice*)workspace;
  p.list = (u64*)(p.slice + slices);
  p.bins = p.list + slices * LIST;
  hipStream_t st = (hipStream_t)stream;
  return logits_f32 ? launch<float>(p, rows, c, st) : launch<bf16>(p, rows, c, st);
}
