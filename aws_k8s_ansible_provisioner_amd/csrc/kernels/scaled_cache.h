// The scaled 8-bit cache (--kv-cache-dtype fp8_scaled): e4m3 codes in the page layouts of the other
// caches (K in MFMA-fragment order, V in 8-token groups, see common.h and rope_cache.hip) and for each
// page and kv head one power of two that its codes are multiplied with, keys' and values' apart.
//
//   need(A) = the least 2^e, -100 <= e <= 100, with every finite |x| of A <= 448 * 2^e
//   scale   = need(new entries) where the page's first token is among them, else max(scale, need)
//   code    = e4m3(clamp(x / scale, -448, 448)), to nearest even; of a NaN 0
//
// A power of two, because every product with it is exact: a code times its scale is a bf16 number (the
// exponents are kept to +-100 for that), the hardware's scaled conversions take it for nothing, and codes
// that move to a larger scale lose nothing but what falls below the smallest normal code, 2^-6.
#pragma once

#include "common.h"

namespace akap {

constexpr float kCodeMax = 448.f;   // the largest e4m3 number, 1.75 * 2^8

// what counts towards the scale: finite magnitudes
__device__ __forceinline__ float scale_mag(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.f;
}

// exponent e of need() for the largest magnitude: most = m 2^E, 1 <= m < 2, is <= 1.75 * 2^(8 + e) from
// e = E - 8 on where m <= 1.75, else from E - 7 on
__device__ __forceinline__ int scale_exp(float most) {
  const uint32_t b = __float_as_uint(most);
  const int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffff) > 0x600000 ? 1 : 0);
  return max(-100, min(100, e));    // (zero and what is no normal number: far below, so -100)
}
__device__ __forceinline__ float exp_scale(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
// exponent of a stored scale (a power of two between 2^-100 and 2^100; anything else is taken as the nearest
// bound or the power below, so that what is derived from it stays finite)
__device__ __forceinline__ int stored_exp(float s) {
  return max(-100, min(100, (int)((__float_as_uint(s) >> 23) & 0xff) - 127));
}

__device__ __forceinline__ float code_clamp(float x) {
  return x != x ? 0.f : __builtin_amdgcn_fmed3f(x, -kCodeMax, kCodeMax);
}
// x times inv (the scale's inverse, a power of two) as four codes, the first in the lowest byte
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d, float inv) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(code_clamp(a * inv), code_clamp(b * inv), 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(code_clamp(c * inv), code_clamp(d * inv), w, true);
  return (uint32_t)w;
}

// four codes as they are rounded for a larger scale: ratio = old scale / new one
__device__ __forceinline__ uint32_t codes_again(uint32_t w, float ratio) {
  const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(w, false);
  const auto b = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
  return codes4(a[0], a[1], b[0], b[1], ratio);
}

// 8 codes -> 8 bf16, times a power of two (exact)
__device__ __forceinline__ bf16x8 codes_wide(uint32_t lo, uint32_t hi, float scale) {
  const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false);
  const bf16x2_t b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
  const bf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false);
  const bf16x2_t d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Head rows in 16 lanes, dims 8 li .. + 7 to a lane.
__device__ __forceinline__ float pair_half(float v) {    // row_ror:8: lane ^ 8, which holds the other half's dims
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x128, 0xf, 0xf, false));
}
__device__ __forceinline__ float squares(const float (&x)[8]) {
#pragma clang fp contract(off)
  return (((x[0] * x[0] + x[1] * x[1]) + x[2] * x[2]) + x[3] * x[3]) +
         (((x[4] * x[4] + x[5] * x[5]) + x[6] * x[6]) + x[7] * x[7]);
}
// 1 / sqrt(m) to the nearest: a Newton step from the instruction's, whose error is up to one unit in the last place
__device__ __forceinline__ float inv_sqrt(float m) {
  const float y = rsqrtf(m), r = m * y;
  const float e = fmaf(-fmaf(m, y, -r), y, fmaf(-r, y, 1.f));
  return m > 0.f && m < INFINITY ? fmaf(0.5f * e, y, y) : y;
}
// Norm (optional), then the rotation (optional) of dims d and d + 64 by c and s, in fp32 throughout.  Every product and
// sum is rounded by itself, squares are added by fours and those in pairs, as whole tensors' arithmetic does it: an
// entry that lies between two codes would fall to the other side of that form's once in a million, half a code away.
__device__ __forceinline__ void norm_rotate(float (&x)[8], bool norm, const bf16x8& w, bool rotate, const f32x4 (&c)[2],
                                            const f32x4 (&s)[2], int li, float eps) {
#pragma clang fp contract(off)
  if (norm) {
    float ss = squares(x);
    ss += dpp_mov<0xB1>(ss);
    ss += dpp_mov<0x4E>(ss);
    ss += dpp_mov<0x141>(ss);
    ss += dpp_mov<0x140>(ss);
    const float inv = inv_sqrt(ss * (1.f / 128) + eps);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = x[e] * inv * bf2f(w[e]);
  }
  if (rotate) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float t = pair_half(x[e]) * s[e >> 2][e & 3];
      x[e] = x[e] * c[e >> 2][e & 3] + (li < 8 ? -t : t);
    }
  }
}

// A page and head's codes rounded anew for a scale 2^-down times theirs, by N threads.
template <int N>
__device__ __forceinline__ void codes_grow(uint8_t* codes, int down, int BS) {
  const float ratio = exp_scale(max(down, -126));      // (126 halvings leave no code but 0)
  u32x4* at = reinterpret_cast<u32x4*>(codes);
  for (int i = threadIdx.x & (N - 1); i < BS * 8; i += N) {
    u32x4 w = at[i];
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = codes_again(w[k], ratio);
    at[i] = w;
  }
}

// The new exponent of a page and head, by N threads that hold the largest magnitude `most` of its new entries, which
// begin at token `off`; where a page that was begun before needs a larger one its codes are rounded anew, and waited
// for.
template <int N>
__device__ __forceinline__ int page_exp(float most, float* scale, uint8_t* codes, int off, int BS) {
  int e = scale_exp(most);
  if (off > 0) {
    const int was = stored_exp(*scale);
    if (e > was) {
      codes_grow<N>(codes, was - e, BS);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    e = max(e, was);
  }
  if ((threadIdx.x & (N - 1)) == 0) *scale = exp_scale(e);
  return e;
}

}  // namespace akap
