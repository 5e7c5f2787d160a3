// Sampling of a row of logits (gfx950): temperature, top-k, top-p and min-p, from a random number that the caller gives.
//
// With the row's tokens ordered by descending logit, equal ones by ascending index, and w_i = exp((x_i - max) / T), every
// filter keeps a prefix of that order: top-k its first k, top-p the shortest prefix whose weights reach p of the weights
// that top-k left, min-p the tokens with w_i >= m.  The token drawn is the first whose running sum of weights exceeds
// u x (the kept weights).  A border of one of these sums decides a whole token, so sums have to be better than fp32 and
// must not depend on the order in which threads come by: a weight is computed in 64 bits and then counted in whole units
// of 2^-44 (2^-43, 2^-42 beyond 2^18, 2^19 tokens, so that a row's sum stays below 2^63); integer sums are exact in any
// order, atomics included.  A token below half a unit (31 T under the maximum) has no weight.
//
// No row is sorted.  One histogram over the value - 2048 bins of equal width from the maximum down to where weights
// vanish, each with its count and its weight - finds the bin that holds a border; only that bin's tokens are gathered
// and sorted, by (value, index) as one 64-bit key.  A bin of too many tokens (equal or nearly equal logits) is first narrowed by histograms
// over that key's bits, eleven at a time, which ends at a single token at the latest.
#include "common.h"
#include <algorithm>
#include "../../include/bagel_hip.h"

namespace {

typedef unsigned long long u64;

constexpr int BINS = 2048;
constexpr int CAP = 4096;            // tokens that are sorted at once
constexpr int MAX_SLICES = 32;       // workgroups per row
constexpr int THREADS = 1024;
constexpr float WINDOW = 31.25f;     // exp(-31.25) < 2^-45: half a unit

struct Params {
  const void* logits;
  long ld;
  int n, slices, shift;              // shift: a unit of weight is 2^-shift
  bool vec;                          // rows start on 16-byte boundaries
  const float *uniforms, *temperature, *top_p, *min_p;
  const int* top_k;
  int* tokens;
  float* logprobs;
  u64* best;                         // [rows][MAX_SLICES] smallest order key of each slice
  u64* mass;                         // [rows][BINS]
  unsigned* count;                   // [rows][BINS]
};

// A NaN counts as a masked token; the two zeros are one value.
__device__ __forceinline__ float clean(float x) { return x != x ? -INFINITY : x + 0.0f; }

// Ascending in the order of the tokens: descending value, then ascending index.
__device__ __forceinline__ u64 order_key(float x, int i) {
  const unsigned b = __float_as_uint(x);
  const unsigned up = b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
  return ((u64)~up << 32) | (unsigned)i;
}
__device__ __forceinline__ float key_value(u64 key) {
  const unsigned up = ~(unsigned)(key >> 32);
  return __uint_as_float(up ^ ((up >> 31) ? 0x80000000u : 0xffffffffu));
}

struct Scale {       // of one row
  float top, per;    // maximum; bins per unit of value
  double inv_t;
  double unit;       // 2^shift
};
__device__ __forceinline__ Scale make_scale(float top, float t, int shift) {
  return Scale{top, (BINS - 1) / WINDOW / t, 1.0 / (double)t, __builtin_ldexp(1.0, shift)};
}

// Monotone in x; the last bin is that of the tokens without weight.
__device__ __forceinline__ int bin_of(float x, const Scale& s) {
#pragma clang fp contract(off)
  const float v = (s.top - x) * s.per;
  return x == s.top ? 0 : v < (float)(BINS - 1) ? (int)v : BINS - 1;
}

constexpr double LN2_HIGH = 2977044471.0 / 4294967296.0;   // floor(2^32 ln 2) / 2^32
constexpr double LN2_LOW = 1.90821492927058770002e-10;    // the rest of ln 2

// exp(z) for z <= 0 in 64 bits: 2^n exp(r), |r| <= ln 2 / 2, the exponential series to r^13 (its next term is below 2^-57).
__device__ __forceinline__ double exp64(double z) {
  const double n = __builtin_rint(z * 1.4426950408889634074);
  double r = __builtin_fma(n, -LN2_HIGH, z);          // exact: n and the 32 bits of the first part leave room
  r = __builtin_fma(n, -LN2_LOW, r);
  double p = 1.0 / 6227020800.0;
  p = __builtin_fma(p, r, 1.0 / 479001600.0);
  p = __builtin_fma(p, r, 1.0 / 39916800.0);
  p = __builtin_fma(p, r, 1.0 / 3628800.0);
  p = __builtin_fma(p, r, 1.0 / 362880.0);
  p = __builtin_fma(p, r, 1.0 / 40320.0);
  p = __builtin_fma(p, r, 1.0 / 5040.0);
  p = __builtin_fma(p, r, 1.0 / 720.0);
  p = __builtin_fma(p, r, 1.0 / 120.0);
  p = __builtin_fma(p, r, 1.0 / 24.0);
  p = __builtin_fma(p, r, 1.0 / 6.0);
  p = __builtin_fma(p, r, 0.5);
  p = __builtin_fma(p, r, 1.0);
  p = __builtin_fma(p, r, 1.0);
  return __builtin_ldexp(p, (int)n);
}
__device__ __forceinline__ double weight(float x, const Scale& s) {   // of a token that is not in the last bin
#pragma clang fp contract(off)
  return x == s.top ? 1.0 : exp64(((double)x - (double)s.top) * s.inv_t);
}
// The weight in units, rounded to nearest: a sum with 2^52 leaves it in the low bits.
__device__ __forceinline__ u64 units(double w, const Scale& s) {
  return (u64)__double_as_longlong(__builtin_fma(w, s.unit, 4503599627370496.0)) & ((1ull << 52) - 1);
}

// f(value, index) for this thread's share of tokens [from, to) of a row; from is a multiple of 8.
template <typename T, typename F>
__device__ __forceinline__ void for_each(const Params& p, int row, int from, int to, F f) {
  const T* x = (const T*)p.logits + (long)row * p.ld;
  for (int i = from + 8 * (int)threadIdx.x; i < to; i += 8 * THREADS) {
    float v[8];
    if (p.vec && i + 8 <= to) {
      if constexpr (sizeof(T) == 2) {
        const bf16x8 w = *(const bf16x8*)(x + i);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (float)w[e];
      } else {
        const f32x4 a = *(const f32x4*)(x + i), b = *(const f32x4*)(x + i + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] = a[e];
          v[4 + e] = b[e];
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = i + e < to ? (float)x[i + e] : 0.f;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (i + e < to) f(clean(v[e]), i + e);
  }
}

__device__ __forceinline__ u64 shfl_u64(u64 v, int from) {
  return ((u64)(unsigned)__shfl((int)(v >> 32), from) << 32) | (unsigned)__shfl((int)(unsigned)v, from);
}

// ---- first launch: the maximum of every slice (as the order key, so the first maximum), and an empty histogram
template <typename T>
__global__ __launch_bounds__(THREADS) void sample_top_kernel(Params p) {
  const int row = blockIdx.y, slice = blockIdx.x;
  const int per = ((p.n + p.slices - 1) / p.slices + 7) / 8 * 8;
  const int from = min(slice * per, p.n), to = min(from + per, p.n);
  for (int b = slice * THREADS + threadIdx.x; b < BINS; b += p.slices * THREADS) {
    p.mass[(long)row * BINS + b] = 0;
    p.count[(long)row * BINS + b] = 0;
  }
  u64 best = ~0ull;
  for_each<T>(p, row, from, to, [&](float x, int i) { best = min(best, order_key(x, i)); });
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) best = min(best, shfl_u64(best, (threadIdx.x & 63) ^ o));
  __shared__ u64 s[THREADS / 64];
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = best;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < THREADS / 64; ++w) best = min(best, s[w]);
    p.best[(long)row * MAX_SLICES + slice] = best;
  }
}

__device__ __forceinline__ u64 row_best(const Params& p, int row) {
  u64 best = ~0ull;
  for (int s = 0; s < p.slices; ++s) best = min(best, p.best[(long)row * MAX_SLICES + s]);
  return best;
}
__device__ __forceinline__ float row_temperature(const Params& p, int row) { return p.temperature ? p.temperature[row] : 1.0f; }

// ---- second launch: counts and weights of the bins
template <typename T>
__global__ __launch_bounds__(THREADS) void sample_histogram_kernel(Params p) {
  const int row = blockIdx.y, slice = blockIdx.x;
  const float t = row_temperature(p, row), top = key_value(row_best(p, row));
  if (!(t > 0.f) || top == -INFINITY) return;       // greedy, or nothing to choose from
  const Scale s = make_scale(top, t, p.shift);
  __shared__ u64 mass[BINS];
  __shared__ unsigned count[BINS];
  for (int b = threadIdx.x; b < BINS; b += THREADS) mass[b] = 0, count[b] = 0;
  __syncthreads();
  const int per = ((p.n + p.slices - 1) / p.slices + 7) / 8 * 8;
  const int from = min(slice * per, p.n), to = min(from + per, p.n);
  for_each<T>(p, row, from, to, [&](float x, int i) {
    const int b = bin_of(x, s);
    if (b < BINS - 1) {                              // those of the last bin are what is left
      atomicAdd(&count[b], 1u);
      atomicAdd(&mass[b], units(weight(x, s), s));
    }
  });
  __syncthreads();
  for (int b = threadIdx.x; b < BINS; b += THREADS)
    if (count[b]) {
      atomicAdd(p.count + (long)row * BINS + b, count[b]);
      atomicAdd(p.mass + (long)row * BINS + b, mass[b]);
    }
}

// ---- third launch: one workgroup per row finds the borders and the token
struct Sums {
  u64 mass;
  unsigned count;
};
struct Hit {         // a token of the order, with the sums up to and including it
  u64 key;
  Sums sums;
};

// Inclusive scan over the workgroup's threads.
__device__ __forceinline__ Sums scan(Sums v, Sums* per_wave) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const u64 m = shfl_u64(v.mass, max(lane - o, 0));
    const unsigned c = (unsigned)__shfl((int)v.count, max(lane - o, 0));
    if (lane >= o) {
      v.mass += m;
      v.count += c;
    }
  }
  __syncthreads();
  if (lane == 63) per_wave[wave] = v;
  __syncthreads();
  for (int w = 0; w < wave; ++w) {
    v.mass += per_wave[w].mass;
    v.count += per_wave[w].count;
  }
  return v;
}

template <typename T>
__global__ __launch_bounds__(THREADS) void sample_pick_kernel(Params p) {
  const int row = blockIdx.x, tid = threadIdx.x;
  const u64 best = row_best(p, row);
  const float t = row_temperature(p, row), top = key_value(best);
  if (!(t > 0.f) || top == -INFINITY) {
    if (tid == 0) {
      p.tokens[row] = top == -INFINITY ? 0 : (int)(unsigned)best;
      if (p.logprobs) p.logprobs[row] = top == -INFINITY ? -INFINITY : 0.f;
    }
    return;
  }
  const Scale s = make_scale(top, t, p.shift);
  __shared__ u64 mass[BINS];                 // sums up to and including a bin
  __shared__ unsigned count[BINS];
  __shared__ u64 work[CAP];                  // the tokens being sorted, or the histogram of a narrowing step
  __shared__ Sums per_wave[THREADS / 64];
  __shared__ int found;
  __shared__ unsigned listed;
  __shared__ Hit hit_s;
  u64* sub_mass = work;                      // [BINS]
  unsigned* sub_count = (unsigned*)(work + BINS);

  // two neighbouring bins per thread
  auto prefix = [&](u64* m, unsigned* c) {
    __syncthreads();
    const Sums a{m[2 * tid], c[2 * tid]}, b{m[2 * tid + 1], c[2 * tid + 1]};
    const Sums v = scan(Sums{a.mass + b.mass, a.count + b.count}, per_wave);
    m[2 * tid] = v.mass - b.mass, c[2 * tid] = v.count - b.count;
    m[2 * tid + 1] = v.mass, c[2 * tid + 1] = v.count;
    __syncthreads();
  };
  if (tid == 0) hit_s = Hit{best, Sums{(u64)s.unit, 1}};
  for (int b = tid; b < BINS; b += THREADS) mass[b] = p.mass[(long)row * BINS + b], count[b] = p.count[(long)row * BINS + b];
  prefix(mass, count);
  const u64 total = mass[BINS - 1];

  // the first bin whose sum, on top of `base`, reaches the target; BINS where none does
  auto find_bin = [&](const u64* m, const unsigned* c, const Sums base, bool by_count, u64 target) {
    if (tid == 0) found = BINS;
    __syncthreads();
    for (int b = 2 * tid; b < 2 * tid + 2; ++b) {
      const u64 upto = by_count ? (u64)base.count + c[b] : base.mass + m[b];
      const u64 before = b == 0 ? (by_count ? (u64)base.count : base.mass) : by_count ? (u64)base.count + c[b - 1] : base.mass + m[b - 1];
      if (before < target && upto >= target) found = b;
    }
    __syncthreads();
    const int b = found;
    __syncthreads();
    return b;
  };
  // the first token of the order at which the count / the weights reach the target, somewhere in `bin`
  auto resolve = [&](int bin, bool by_count, u64 target) {
    Sums base{bin ? mass[bin - 1] : 0, bin ? count[bin - 1] : 0};
    unsigned inside = count[bin] - base.count;
    u64 low = 0, high = ~0ull;
    for (int sh = 53; inside > CAP; sh = max(sh - 11, 0)) {
      __syncthreads();
      for (int b = tid; b < BINS; b += THREADS) sub_mass[b] = 0, sub_count[b] = 0;
      __syncthreads();
      for_each<T>(p, row, 0, p.n, [&](float x, int i) {
        if (bin_of(x, s) != bin) return;
        const u64 key = order_key(x, i);
        if (key < low || key > high) return;
        const int b = (int)((key - low) >> sh);
        atomicAdd(&sub_count[b], 1u);
        atomicAdd(&sub_mass[b], units(weight(x, s), s));
      });
      prefix(sub_mass, sub_count);
      const int b = min(find_bin(sub_mass, sub_count, base, by_count, target), BINS - 1);
      const Sums before{b ? sub_mass[b - 1] : 0, b ? sub_count[b - 1] : 0};
      inside = sub_count[b] - before.count;
      base.mass += before.mass;
      base.count += before.count;
      low += (u64)b << sh;
      high = low + ((1ull << sh) - 1);
      __syncthreads();
    }
    __syncthreads();
    if (tid == 0) listed = 0;
    __syncthreads();
    for_each<T>(p, row, 0, p.n, [&](float x, int i) {
      if (bin_of(x, s) != bin) return;
      const u64 key = order_key(x, i);
      if (key < low || key > high) return;
      const unsigned at = atomicAdd(&listed, 1u);
      if (at < CAP) work[at] = key;
    });
    __syncthreads();
    const int len = (int)min(listed, (unsigned)CAP);
    int size = 2;
    while (size < len) size *= 2;
    for (int i = len + tid; i < size; i += THREADS) work[i] = ~0ull;
    for (int k = 2; k <= size; k *= 2)
      for (int j = k / 2; j > 0; j /= 2) {
        __syncthreads();
        for (int i = tid; i < size; i += THREADS) {
          const int o = i ^ j;
          if (o > i) {
            const u64 a = work[i], b = work[o];
            if ((a > b) == ((i & k) == 0)) work[i] = b, work[o] = a;
          }
        }
      }
    __syncthreads();
    // four neighbours per thread
    Sums each[CAP / THREADS], sum{0, 0};
#pragma unroll
    for (int e = 0; e < CAP / THREADS; ++e) {
      const int i = tid * (CAP / THREADS) + e;
      if (i < len) {
        sum.mass += units(weight(key_value(work[i]), s), s);
        sum.count += 1;
      }
      each[e] = sum;
    }
    const Sums all = scan(sum, per_wave);
    base.mass += all.mass - sum.mass;
    base.count += all.count - sum.count;
#pragma unroll
    for (int e = 0; e < CAP / THREADS; ++e) {
      const int i = tid * (CAP / THREADS) + e;
      const Sums upto{base.mass + each[e].mass, base.count + each[e].count};
      const Sums before{e ? base.mass + each[e ? e - 1 : 0].mass : base.mass, e ? base.count + each[e ? e - 1 : 0].count : base.count};
      if (i < len && (by_count ? (before.count < target && upto.count >= target) : (before.mass < target && upto.mass >= target)))
        hit_s = Hit{work[i], upto};
    }
    __syncthreads();
    const Hit h = hit_s;
    __syncthreads();
    return h;
  };

  Hit border{~0ull, Sums{total, (unsigned)p.n}};      // the last token kept
  const int k = p.top_k ? p.top_k[row] : 0;
  if (k >= 1 && k < p.n) {
    const int bin = find_bin(mass, count, Sums{0, 0}, true, (u64)k);
    if (bin < BINS - 1) border = resolve(bin, true, (u64)k);      // further down there is no weight to cut off
  }
  const float top_p = p.top_p ? p.top_p[row] : 1.0f;
  if (top_p < 1.0f) {
    const u64 target = max((u64)1, (u64)__builtin_ceil((double)max(top_p, 0.f) * (double)border.sums.mass));
    const int bin = find_bin(mass, count, Sums{0, 0}, false, target);
    if (bin < BINS - 1) border = resolve(bin, false, target);
  }
  u64 kept = border.sums.mass;
  const float min_p = p.min_p ? p.min_p[row] : 0.f;
  if (min_p > 0.f) {
    // the bins that the threshold may lie in, one to each side for the roundings of the bins' borders
    const double edge = -log((double)min_p) * ((BINS - 1) / (double)WINDOW);
    const int b0 = edge < 1.0 ? 0 : edge < BINS ? (int)edge - 1 : BINS, b1 = b0 + 3;
    if (b0 < BINS - 1 && (border.key == ~0ull || bin_of(key_value(border.key), s) >= b0)) {
      u64 mine = 0;
      for_each<T>(p, row, 0, p.n, [&](float x, int i) {
        const int b = bin_of(x, s);
        if (b < b0 || b > b1 || b >= BINS - 1 || order_key(x, i) > border.key) return;
        const double w = weight(x, s);
        if (w >= (double)min_p) mine += units(w, s);
      });
      __syncthreads();
      const Sums v = scan(Sums{mine, 0}, per_wave);
      if (tid == THREADS - 1) hit_s.sums = v;
      __syncthreads();
      kept = (b0 ? mass[b0 - 1] : 0) + hit_s.sums.mass;
      __syncthreads();
      kept = max(kept, (u64)s.unit);                  // the first token stays whatever min_p is
    }
  }
  const float u = p.uniforms[row];
  const u64 target = 1 + min((u64)((u > 0.f ? min((double)u, 1.0) : 0.0) * (double)kept), kept - 1);
  const Hit h = resolve(min(find_bin(mass, count, Sums{0, 0}, false, target), BINS - 1), false, target);
  if (tid == 0) {
    p.tokens[row] = (int)(unsigned)h.key;
    if (p.logprobs) {
      const float x = key_value(h.key);
      p.logprobs[row] = (float)((x == top ? 0.0 : ((double)x - (double)top) * s.inv_t) - log((double)kept / s.unit));
    }
  }
}

long row_bytes() { return MAX_SLICES * 8 + BINS * 12; }

}  // namespace

extern "C" long bagel_sample_rows_workspace_bytes(int rows, int n) {
  return rows <= 0 || n <= 0 ? 0 : rows * row_bytes();
}

extern "C" int bagel_sample_rows(const void* logits, long ld, int rows, int n, int logits_f32, const void* uniforms, const void* temperature,
                                 const void* top_k, const void* top_p, const void* min_p, void* tokens, void* logprobs,
                                 void* workspace, long workspace_bytes, void* stream) {
  BAGEL_CHECK(rows >= 0 && rows <= 65535, "bagel_sample_rows: rows=%d (at most 65535)", rows);
  BAGEL_CHECK(n > 0 && n <= 1 << 20, "bagel_sample_rows: %d tokens (1 to 2^20)", n);
  BAGEL_CHECK(logits_f32 == 0 || logits_f32 == 1, "bagel_sample_rows: logits_f32=%d", logits_f32);
  if (rows == 0) return 0;
  BAGEL_CHECK(logits && uniforms && tokens && workspace, "bagel_sample_rows: null operand");
  BAGEL_CHECK(ld >= n || ld == 0, "bagel_sample_rows: leading dim %ld below %d tokens", ld, n);
  BAGEL_CHECK((uintptr_t)logits % (logits_f32 ? 4 : 2) == 0 && (uintptr_t)workspace % 16 == 0, "bagel_sample_rows: misaligned operand");
  BAGEL_CHECK(workspace_bytes >= bagel_sample_rows_workspace_bytes(rows, n), "bagel_sample_rows: workspace of %ld bytes, %ld needed",
              workspace_bytes, bagel_sample_rows_workspace_bytes(rows, n));
  Params p;
  p.logits = logits; p.ld = ld; p.n = n;
  p.vec = (uintptr_t)logits % 16 == 0 && ld % (logits_f32 ? 4 : 8) == 0;
  p.shift = n <= 1 << 18 ? 44 : n <= 1 << 19 ? 43 : 42;
  p.uniforms = (const float*)uniforms; p.temperature = (const float*)temperature; p.top_k = (const int*)top_k;
  p.top_p = (const float*)top_p; p.min_p = (const float*)min_p; p.tokens = (int*)tokens; p.logprobs = (float*)logprobs;
  p.mass = (u64*)workspace;
  p.best = p.mass + (long)rows * BINS;
  p.count = (unsigned*)(p.best + (long)rows * MAX_SLICES);
  // two workgroups per CU, each with at least 8192 tokens
  p.slices = std::max(1, std::min(std::min(MAX_SLICES, 2 * bagel_cu_count() / rows), n / 8192));
  const dim3 grid(p.slices, rows), block(THREADS);
  hipStream_t st = (hipStream_t)stream;
  if (logits_f32) {
    hipLaunchKernelGGL(sample_top_kernel<float>, grid, block, 0, st, p);
    hipLaunchKernelGGL(sample_histogram_kernel<float>, grid, block, 0, st, p);
    hipLaunchKernelGGL(sample_pick_kernel<float>, dim3(rows), block, 0, st, p);
  } else {
    hipLaunchKernelGGL(sample_top_kernel<bf16>, grid, block, 0, st, p);
    hipLaunchKernelGGL(sample_histogram_kernel<bf16>, grid, block, 0, st, p);
    hipLaunchKernelGGL(sample_pick_kernel<bf16>, dim3(rows), block, 0, st, p);
  }
  BAGEL_LAUNCH_CHECK();
  return 0;
}
