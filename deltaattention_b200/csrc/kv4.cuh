// The 4-bit form of K / V rows, shared by its kernels.
//
// A row of D elements is cut into NG = D / 32 groups of 32. Per group, in fp32:
//   zero  = min rounded down to bf16           (never above any element, so codes are >= 0)
//   scale = (max - zero) * (1 / 15, as fp32) rounded to bf16
//   code  = clamp(rint((x - zero) / scale), 0, 15), 0 where scale is 0
//   value = zero + scale * code
// A group with an element that is not finite has scale = zero = NaN and reads back as NaN.
// Two bf16 numbers per group for every input type: their exponent range covers bf16 and fp16
// values, and the codes are taken against the rounded pair, so its rounding costs no more than
// half a step anywhere.
//
// Codes: word t * NG + g of the row's D / 8 words holds elements 32 g + 8 t + i in bits 4 i.. (i
// = 0..7, t = 0..3). So the 4 NG bytes of t hold an eighth of every group: the lanes of a matrix
// fragment that share t read them as one piece, and each word stays within one group.
// Scales: NG scales, then NG zeros.
#pragma once
#include "common.cuh"

namespace dab {

struct Kv4Hist {
  uint8_t* k_codes; uint8_t* v_codes;               // [B, H, cap, D / 2], rows contiguous
  __nv_bfloat16* k_scales; __nv_bfloat16* v_scales; // [B, H, cap, D / 16]
  int64_t cb, ch;                                   // code strides over batch, head (bytes)
  int64_t sb, sh;                                   // scale strides over batch, head (elements)
};

// single-token cache update; strides in elements, rows contiguous
struct Kv4Update {
  const void* k_new; const void* v_new;
  int64_t kb, kh, kd, vb, vh, vd;
  Kv4Hist hist;
  int32_t* counts; int32_t* times; float* mass;  // [B, H, cap], mass may be null
  int64_t mb, mh;
  int32_t* lengths; int64_t lb, lh;              // [B, H]
  void* last_key; int64_t lkb, lkh;              // [B, H, D]
  void* k_exact; void* v_exact;                  // [B, H, W, D]
  int64_t eb, eh, en;
  float* exact_mass; int64_t emb, emh;           // [B, H, W], may be null
  const int64_t* state;                          // (exact, total) lengths
  int* err;
  float threshold;                               // squared distance, or cosine
  int B, H, cap, W;
};

// single-token attention
struct Kv4Attn {
  const void* q; int64_t qb, qh;                 // [B, Hq, D]
  void* out; int64_t ob, oh;
  Kv4Hist hist;
  const int32_t* counts; float* mass; int64_t mb, mh;
  const int32_t* lengths; int64_t lb, lh;
  const void* k_exact; const void* v_exact; int64_t eb, eh, en;
  float* exact_mass; int64_t emb, emh;
  int64_t* state; int lag;                       // device lengths (or null); lag: one step behind, advanced after use
  int exact_len;                                 // without state
  float scale_log2;                              // sm_scale * log2(e)
  int B, H, G, cap, W;                           // G q-heads per kv-head
  // workspace: per 8 q-heads (first part, last piece); per q-head row of an unsplit head (max,
  // 1 / sum); per part and q-head (max, sum) and the unscaled output; per row the scores of history
  // and window (null without mass)
  int2* info; float2* row_stats; float2* stats; float* part; float* scores;
  int* used;                                     // with state: the window length this call attends with
  int64_t sstride; int wcol;                     // columns of a row of scores, the window's first
  int splits, pieces;                            // per head, or in all
};

// x rounded down (towards -inf) to bf16, as fp32
__device__ __forceinline__ float floor_bf16(float x) {
  const uint32_t i = __float_as_uint(x);
  return __uint_as_float((i + ((i >> 31) ? 0xFFFFu : 0u)) & 0xFFFF0000u);
}

// (scale, zero) of a group from its minimum and maximum; NaN for both when either is not finite. Without
// ANY a range past fp32's largest number gives an infinite scale.
template <bool ANY>
__device__ __forceinline__ void kv4_scale_zero(float mn, float mx, float& scale, float& zero) {
  zero = floor_bf16(mn);
  const float range = __fsub_rn(mx, zero);
  float x = __fmul_rn(range, 1.f / 15.f);
  if (ANY && range == INFINITY) x = 2.f * __fmul_rn(__fsub_rn(0.5f * mx, 0.5f * zero), 1.f / 15.f);
  scale = round_as<__nv_bfloat16>(x);
  // an infinity or NaN in either makes the scale one
  if (ANY && !(scale < INFINITY)) scale = zero = __int_as_float(0x7FC00000);
}

// Differences past fp32's largest number are taken by halves: scales from 2^100 on have room for that.
__device__ __forceinline__ uint32_t kv4_code(float x, float scale, float zero) {
  const float f = scale < 0x1p100f ? 1.f : 0.5f;
  const float q = rintf(__fdiv_rn(__fsub_rn(x * f, zero * f), scale * f));
  // NaN (scale 0 or NaN) compares false and gives 0
  return q > 0.f && scale > 0.f ? static_cast<uint32_t>(fminf(q, 15.f)) : 0u;
}

// minimum / maximum that keep a NaN of either operand (one instruction)
__device__ __forceinline__ float fmin_nan(float a, float b) {
  float d;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float fmax_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// One row by one warp: lane l holds elements 32 g + l in x[g]. Writes the row's codes (4-byte
// aligned) and scales.
template <int NG>
__device__ __forceinline__ void kv4_quantize_row(const float* x, uint32_t* codes, __nv_bfloat16* scales, int lane) {
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    float mn = x[g], mx = x[g];
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      mn = fmin_nan(mn, __shfl_xor_sync(0xFFFFFFFFu, mn, o));
      mx = fmax_nan(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, o));
    }
    float scale, zero;
    kv4_scale_zero<true>(mn, mx, scale, zero);
    uint32_t w = kv4_code(x[g], scale, zero) << (4 * (lane & 7));
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) w |= __shfl_xor_sync(0xFFFFFFFFu, w, o);
    if ((lane & 7) == 0) codes[(lane >> 3) * NG + g] = w;
    if (lane == 0) {
      scales[g] = __float2bfloat16_rn(scale);
      scales[NG + g] = __float2bfloat16_rn(zero);
    }
  }
}

}  // namespace dab
