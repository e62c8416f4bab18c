// Steps shared by the sampler, the judging of drafted tokens and the attention of drafted trees.
#pragma once
#include "exact_common.h"

namespace exact {

__device__ __forceinline__ int64_t wave_incl_scan64(int64_t v, int lane) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t w = __shfl_up(v, o, 64);
    if (lane >= o) v = (int64_t)((uint64_t)v + (uint64_t)w);
  }
  return v;
}

// lut_exp in 32 bits for a distance d kept against the maximum of a part (at most EXP_FAR, from where exponentials are 0, or EXP_UNSEEN
// for a value left out), where that maximum lies gap (exp_gap) below the row's. The last table entries read are 10240 and 10241, and
// a - shr((a - b) fr, 8) lies between a and b.
#define EXP_FAR (40U << EXACT_F)
#define EXP_UNSEEN 0xffffffU
__device__ __forceinline__ uint32_t exp_gap(int64_t mx, int64_t part) {
  const uint64_t g = (uint64_t)mx - (uint64_t)part;
  return g < EXP_FAR ? (uint32_t)g : EXP_FAR;
}
__device__ __forceinline__ int32_t lut_exp_kept(const int32_t* T, uint32_t gap, uint32_t d) {
  const uint32_t x = min(gap + d, EXP_FAR);
  const int fr = x & 255, a = T[x >> 8], b = T[(x >> 8) + 1];
  const int e = a - (int)(((int64_t)a * fr - (int64_t)b * fr + 128) >> 8);
  return x < EXP_FAR ? e : 0;
}

// floor(e 2^20 / es) for e below 2^31 and es < 2^51, at least 0: with es20 = max(es, 1) 2^-20 and rb = (1 - 2^-45) / es20 the estimate
// is p or p - 1, and its remainder, exact in one fma, tells which. e <= es gives at most 2^20; more (of an exp table with negative
// entries, whose sum may be small) goes through the division and counts as PROB_NONE from there on.
//
// A row whose p sum to PROB_NONE or more counts as one without probability (p = 0): below it the products of judging, u q P, p Q 2^20 and
// u W, stay under 2^63. Only tables with negative entries give sums above 2^20.
#define PROB_NONE ((int64_t)1 << 23)
__device__ __forceinline__ int64_t prob20(int32_t e, int64_t es, double es20, double rb) {
  if (e <= 0 || es <= 0) return 0;
  if (e > es) {
    const int64_t p = floordiv_pos(shl64(e, 20), es);
    return p < PROB_NONE ? p : PROB_NONE;   // 2^30 of them sum up in 64 bits
  }
  const double p = __builtin_floor((double)e * rb);
  return (int64_t)(uint32_t)p + (__builtin_fma(-p, es20, (double)e) >= es20);
}
__device__ __forceinline__ double sum20(int64_t es) { return (double)max64(es, 1) * 0x1p-20; }
__device__ __forceinline__ double sum20_rcp(double es20) { return (1.0 - 0x1p-45) / es20; }

// A token of probabilities p of P (target) and q of Q (draft) is accepted for the random number u (its low 20 bits)
__device__ __forceinline__ bool verify_accepts(int32_t u, int64_t p, int64_t P, int64_t q, int64_t Q) {
  return (int64_t)(u & 0xFFFFF) * q * P < shl64(p * Q, 20);
}

// ... and what a rejection leaves of it: max(p / P - q / Q, 0) in units of 1 / (P Q)
__device__ __forceinline__ int64_t verify_rest(int64_t p, int64_t P, int64_t q, int64_t Q) { return max64(p * Q - q * P, 0); }

// the first prefix sum above it is the token's, of weights that sum to W < 2^43
__device__ __forceinline__ int64_t verify_target(int32_t u, int64_t W) { return ((int64_t)(u & 0xFFFFF) * W) >> 20; }

}  // namespace exact
