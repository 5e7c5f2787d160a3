// Per-head q/k RMSNorm followed by rotary embedding, as one lane's share of a head.
//
// PackedAttentionMoT.forward_inference (qwen2_navit.py:549-566): the norm is computed in fp32 from the bf16
// projection output; with und_rounding the norm output and every RoPE product are rounded to bf16 (the
// understanding-mode graph, :526-530), otherwise only the final sum is.
// D/8 lanes hold one head; lane j holds elements 8j..8j+7 and its rotate_half partner is lane j ^ (D/16).  All D/8
// lanes of a head must be active together.
#pragma once
#include "common.h"

// The value of lane ^ W inside a head's lanes, by DPP (no LDS): W = 4 is the half row's mirror image (lane ^ 7) in each four
// of it reversed (lane ^ 3).
template <int W>
__device__ __forceinline__ float head_xor(float v) {
  if constexpr (W == 4) return dpp_f32<0x1B>(dpp_f32<DPP_HALF_MIRROR>(v));
  return xor_lane<W>(v);
}
template <int W>
__device__ __forceinline__ float head_sum(float v) {   // over 2 W lanes: lane ^ W first
  v += head_xor<W>(v);
  if constexpr (W > 1) return head_sum<W / 2>(v);
  return v;
}

// The lane's eight results in fp32 (with und_rounding: bf16 values).  norm / rope: whether that step is taken; w, c, s: the lane's
// eight norm weights and elements of the rotation's rows.
template <int D>
__device__ __forceinline__ void norm_rope_lane(const bf16x8 v, int j, bool norm, const bf16x8 w, bool rope, const bf16x8 c, const bf16x8 s,
                                               float eps, int und_rounding, float (&o)[8]) {
  constexpr int LPH = D / 8;
  float y[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = (float)v[e];
  if (norm) {
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss += y[e] * y[e];
    const float rs = rsqrtf(head_sum<LPH / 2>(ss) / (float)D + eps);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float n = y[e] * rs;
      y[e] = und_rounding ? round_bf16((float)w[e] * round_bf16(n)) : (float)w[e] * n;
    }
  }
  if (!rope) {
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = y[e];
    return;
  }
  const float sign = j < LPH / 2 ? -1.f : 1.f;  // rotate_half: first half gets -x2, second half +x1
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float yr = sign * head_xor<LPH / 2>(y[e]), ce = (float)c[e], se = (float)s[e];
    if (und_rounding)
      o[e] = round_bf16(round_bf16(y[e] * ce) + round_bf16(yr * se));
    else
      o[e] = __fmul_rn(y[e], ce) + __fmul_rn(yr, se);
  }
}

template <int D>
__device__ __forceinline__ bf16x8 qk_norm_rope_lane(const bf16x8 v, int j, const bf16* __restrict__ w,
                                                    const bf16* __restrict__ cos_row, const bf16* __restrict__ sin_row,
                                                    float eps, int und_rounding) {
  float y[8];
  norm_rope_lane<D>(v, j, true, *(const bf16x8*)(w + 8 * j), true, *(const bf16x8*)(cos_row + 8 * j), *(const bf16x8*)(sin_row + 8 * j),
                    eps, und_rounding, y);
  bf16x8 o;
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = (bf16)y[e];
  return o;
}
