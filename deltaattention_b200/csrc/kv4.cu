// A decode history in 4 bits (format in kv4.cuh): quantisation of packed K / V rows, reading
// back, and the single-token cache update.
#include <cfloat>
#include <type_traits>

#include "kv4.cuh"

namespace dab {

// ------------------------------------------------------------------- quantise / read back
// Both are bound by memory when every element costs few instructions: K and V rows of 2 D bytes
// against 5 D / 8 bytes of codes and scales. To quantise, a lane takes 16 neighbouring elements (two
// 16-byte pieces, two code words); the 2 lanes of a group exchange minimum and maximum once, and
// the pieces of KV4_QROWS rows are in flight. To read back, a lane takes 8 elements of KV4_ROWS rows.
// 16 x 8 heads x 8191 rows of 128, K and V, in bf16 (705 MB each way): quantising 128 us (8 elements a lane: 189,
// the group's scale and reciprocal are found four times), reading back 116 us, 6.1 TB/s.
constexpr int KV4_ROWS = 4, KV4_QROWS = 4;

template <typename T> struct Pair;
template <> struct Pair<__nv_bfloat16> {
  using V = __nv_bfloat162;
  static __device__ __forceinline__ float2 f32(V v) { return __bfloat1622float2(v); }
};
template <> struct Pair<__half> {
  using V = __half2;
  static __device__ __forceinline__ float2 f32(V v) { return __half22float2(v); }
};

// Codes of 8 elements x (pairs of T) against scale s > 0 with reciprocal r, and zero. The quotient
// a / s is corrected from a r by one step with the exact remainder (Markstein, IBM J. Res. Dev. 34,
// 1990), so it rounds as a division does; adding 1.5 * 2^23 rounds it to an integer, half to even,
// in the number's lowest bits. s is at least KV4_FAST: its reciprocal and the remainders are fp32
// numbers, and as it is rounded by 2^-9 at most, 0 <= a <= 15.06 s and codes need no clamp.
constexpr float KV4_FAST = 0x1p-100f;
template <typename T>
__device__ __forceinline__ uint32_t kv4_code8(const typename Pair<T>::V* x, float s, float r, float zero) {
  uint32_t w = 0u;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 f = Pair<T>::f32(x[i >> 1]);
    const float a = __fsub_rn(i & 1 ? f.y : f.x, zero);
    const float q = a * r;
    const float c = fmaf(fmaf(-q, s, a), r, q);
    w += __float_as_uint(__fadd_rn(c, 12582912.f)) << (4 * i);  // 0x4B400000 + code
  }
  // less the constant's own contributions, 0x4B400000 << 4 i, i = 0..7 (those past bit 31 are gone)
  return w - (0x4B400000u + 0xB4000000u + 0x40000000u);
}
// 16 elements of a group with minimum mn and maximum mx, whatever its scale: (codes, codes, scale, zero).
// Scales down to bf16's subnormals (groups within 2^-96 of one value) are rounded by up to a third, so
// that quotients pass 15, and have no reciprocal: divided, and cut. So are very large ones, whose
// elements may lie further apart than fp32's largest number.
template <typename T>
__device__ __noinline__ uint4 kv4_code16_any(uint4 a, uint4 b, float mn, float mx) {
  using V = typename Pair<T>::V;
  float s, zero;
  kv4_scale_zero<true>(mn, mx, s, zero);
  uint32_t w[2] = {0u, 0u};
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float2 f = Pair<T>::f32(reinterpret_cast<const V*>(i < 8 ? &a : &b)[(i & 7) >> 1]);
    w[i >> 3] |= kv4_code(i & 1 ? f.y : f.x, s, zero) << (4 * (i & 7));
  }
  return make_uint4(w[0], w[1], __float_as_uint(s), __float_as_uint(zero));
}

template <typename T, int D>
__global__ void __launch_bounds__(256) kv4_quantize_kernel(const T* __restrict__ k, const T* __restrict__ v, int64_t kb,
                                                           int64_t kh, int64_t kn, int64_t vb, int64_t vh, int64_t vn,
                                                           Kv4Hist out, int H, int64_t N) {
  constexpr int NG = D / 32, LPR = D / 16, RPI = 256 / LPR;  // lanes per row, rows per CTA and step
  using V = typename Pair<T>::V;
  const int j = threadIdx.x % LPR, g = j >> 1, t = (j & 1) * 2;  // words t and t + 1 of group g
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * (RPI * KV4_QROWS) + threadIdx.x / LPR;
  const int b = blockIdx.y / H, h = blockIdx.y - b * H;
  const bool is_v = blockIdx.z != 0;
  const T* x = (is_v ? v + b * vb + h * vh : k + b * kb + h * kh) + 16 * j;
  const int64_t sn = is_v ? vn : kn;
  uint4 raw[KV4_QROWS][2];
#pragma unroll
  for (int i = 0; i < KV4_QROWS; ++i) {
    const int64_t n = n0 + i * RPI;
    if (n < N) {
      raw[i][0] = *reinterpret_cast<const uint4*>(x + n * sn);
      raw[i][1] = *reinterpret_cast<const uint4*>(x + n * sn + 8);
    }
  }
  uint32_t* c = reinterpret_cast<uint32_t*>((is_v ? out.v_codes : out.k_codes) + b * out.cb + h * out.ch) + t * NG + g;
  __nv_bfloat16* s = (is_v ? out.v_scales : out.k_scales) + b * out.sb + h * out.sh + (t == 0 ? g : NG + g);
#pragma unroll
  for (int i = 0; i < KV4_QROWS; ++i) {
    const int64_t n = n0 + i * RPI;
    const V* e = reinterpret_cast<const V*>(&raw[i][0]);
    V lo = __hmin2_nan(__hmin2_nan(__hmin2_nan(e[0], e[1]), __hmin2_nan(e[2], e[3])),
                       __hmin2_nan(__hmin2_nan(e[4], e[5]), __hmin2_nan(e[6], e[7])));
    V hi = __hmax2_nan(__hmax2_nan(__hmax2_nan(e[0], e[1]), __hmax2_nan(e[2], e[3])),
                       __hmax2_nan(__hmax2_nan(e[4], e[5]), __hmax2_nan(e[6], e[7])));
    lo = __hmin2_nan(lo, __shfl_xor_sync(0xFFFFFFFFu, lo, 1));
    hi = __hmax2_nan(hi, __shfl_xor_sync(0xFFFFFFFFu, hi, 1));
    const float2 l2 = Pair<T>::f32(lo), h2 = Pair<T>::f32(hi);
    float scale, zero;
    const float mn = fmin_nan(l2.x, l2.y), mx = fmax_nan(h2.x, h2.y);
    kv4_scale_zero<false>(mn, mx, scale, zero);
    const bool fast = scale >= KV4_FAST && scale < 0x1p100f;
    const float step = fast ? scale : 1.f, r = __frcp_rn(step);
    uint32_t w0 = kv4_code8<T>(e, step, r, zero), w1 = kv4_code8<T>(e + 4, step, r, zero);
    if (!fast) {
      w0 = w1 = 0u;
      if (mx - mn != 0.f) {  // not a constant group (NaN and infinities give NaN)
        if constexpr (TypeOf<T>::value == BF16) {
          const uint4 any = kv4_code16_any<T>(raw[i][0], raw[i][1], mn, mx);
          w0 = any.x;
          w1 = any.y;
          scale = __uint_as_float(any.z);
          zero = __uint_as_float(any.w);
        } else {  // fp16 has no other steps
          scale = zero = __int_as_float(0x7FC00000);
        }
      }
    }
    if (n < N) {
      c[n * (D / 8)] = w0;
      c[n * (D / 8) + NG] = w1;
      s[n * (2 * NG)] = __float2bfloat16_rn(t == 0 ? scale : zero);
    }
  }
}

// Any strides: one warp per row.
template <typename T, int D>
__global__ void __launch_bounds__(256) kv4_quantize_any_kernel(const T* __restrict__ k, const T* __restrict__ v,
                                                               int64_t kb, int64_t kh, int64_t kn, int64_t kd,
                                                               int64_t vb, int64_t vh, int64_t vn, int64_t vd,
                                                               Kv4Hist out, int H, int64_t N) {
  constexpr int NG = D / 32;
  const int lane = threadIdx.x & 31;
  const int64_t n = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (n >= N) return;
  const int b = blockIdx.y / H, h = blockIdx.y - b * H;
  const bool is_v = blockIdx.z != 0;
  const T* x = is_v ? v + b * vb + h * vh + n * vn : k + b * kb + h * kh + n * kn;
  const int64_t sd = is_v ? vd : kd;
  float r[NG];
#pragma unroll
  for (int g = 0; g < NG; ++g) r[g] = to_f32(x[(32 * g + lane) * sd]);
  uint8_t* c = (is_v ? out.v_codes : out.k_codes) + b * out.cb + h * out.ch + n * (D / 2);
  __nv_bfloat16* s = (is_v ? out.v_scales : out.k_scales) + b * out.sb + h * out.sh + n * (2 * NG);
  kv4_quantize_row<NG>(r, reinterpret_cast<uint32_t*>(c), s, lane);
}

// Two values rounded to T, those past its largest numbers cut to them: the zero and 15 steps of a group at the
// type's limits may lie outside them, and a finite group reads back finite. NaN stays.
template <typename T>
__device__ __forceinline__ uint32_t pack_cut(float lo, float hi) {
  uint32_t d;
  if constexpr (TypeOf<T>::value == BF16) asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  else asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}

template <typename T, int D>
__global__ void __launch_bounds__(256) kv4_dequantize_kernel(Kv4Hist in, T* __restrict__ k, T* __restrict__ v,
                                                             int64_t ob, int64_t oh, int64_t on, int H, int64_t N) {
  constexpr int NG = D / 32, LPR = D / 8, RPI = 256 / LPR;
  const int j = threadIdx.x % LPR, g = j >> 2, t = j & 3;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * (RPI * KV4_ROWS) + threadIdx.x / LPR;
  const int b = blockIdx.y / H, h = blockIdx.y - b * H;
  const bool is_v = blockIdx.z != 0;
  const uint32_t* c = reinterpret_cast<const uint32_t*>((is_v ? in.v_codes : in.k_codes) + b * in.cb + h * in.ch) + t * NG + g;
  const __nv_bfloat16* s = (is_v ? in.v_scales : in.k_scales) + b * in.sb + h * in.sh + g;
  T* dst = (is_v ? v : k) + b * ob + h * oh + 8 * j;
  uint32_t w[KV4_ROWS];
  __nv_bfloat16 sc[KV4_ROWS], ze[KV4_ROWS];
#pragma unroll
  for (int i = 0; i < KV4_ROWS; ++i) {
    const int64_t n = n0 + i * RPI;
    if (n < N) {
      w[i] = c[n * LPR];
      sc[i] = s[n * (2 * NG)];
      ze[i] = s[n * (2 * NG) + NG];
    }
  }
#pragma unroll
  for (int i = 0; i < KV4_ROWS; ++i) {
    const int64_t n = n0 + i * RPI;
    if (n >= N) return;
    const float scale = to_f32(sc[i]), zero = to_f32(ze[i]);
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)  // 2^23 + code, less 2^23
      x[e] = fmaf(scale, __uint_as_float(((w[i] >> (4 * e)) & 15u) | 0x4B000000u) - 8388608.f, zero);
    T* o = dst + n * on;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = fmin_nan(x[e], FLT_MAX);
      __stcs(reinterpret_cast<float4*>(o), make_float4(x[0], x[1], x[2], x[3]));
      __stcs(reinterpret_cast<float4*>(o) + 1, make_float4(x[4], x[5], x[6], x[7]));
    } else {
      __stcs(reinterpret_cast<uint4*>(o),
             make_uint4(pack_cut<T>(x[0], x[1]), pack_cut<T>(x[2], x[3]), pack_cut<T>(x[4], x[5]), pack_cut<T>(x[6], x[7])));
    }
  }
}

cudaError_t launch_kv4_quantize(int dtype, const void* k, const int64_t* ks, const void* v, const int64_t* vs,
                                const Kv4Hist& out, int64_t B, int64_t H, int64_t N, int64_t D, cudaStream_t st) {
  if (B * H * N == 0) return cudaSuccess;
  // 16-byte pieces: contiguous rows on 16-byte boundaries; anything else goes one warp per row
  const bool rows16 = ks[3] == 1 && vs[3] == 1 &&
                      ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0 &&
                      ((ks[0] | ks[1] | ks[2] | vs[0] | vs[1] | vs[2]) & 7) == 0;
  auto run = [&](auto tag, auto dd) -> cudaError_t {
    using T = decltype(tag);
    constexpr int DD = decltype(dd)::value;
    const T* kp = static_cast<const T*>(k);
    const T* vp = static_cast<const T*>(v);
    const int64_t per = rows16 ? 256 / (DD / 16) * KV4_QROWS : 8;
    dim3 grid(static_cast<unsigned>((N + per - 1) / per), static_cast<unsigned>(B * H), 2);
    if (rows16)
      kv4_quantize_kernel<T, DD><<<grid, 256, 0, st>>>(kp, vp, ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], out,
                                                       static_cast<int>(H), N);
    else
      kv4_quantize_any_kernel<T, DD><<<grid, 256, 0, st>>>(kp, vp, ks[0], ks[1], ks[2], ks[3], vs[0], vs[1], vs[2],
                                                           vs[3], out, static_cast<int>(H), N);
    return cudaGetLastError();
  };
  using I64 = std::integral_constant<int, 64>;
  using I128 = std::integral_constant<int, 128>;
  if (dtype == BF16) return D == 64 ? run(__nv_bfloat16{}, I64{}) : run(__nv_bfloat16{}, I128{});
  return D == 64 ? run(__half{}, I64{}) : run(__half{}, I128{});
}

cudaError_t launch_kv4_dequantize(int dtype, const Kv4Hist& in, void* k, void* v, const int64_t* os, int64_t B,
                                  int64_t H, int64_t N, int64_t D, cudaStream_t st) {
  if (B * H * N == 0) return cudaSuccess;
  const int64_t per = 256 / (D / 8) * KV4_ROWS;
  dim3 grid(static_cast<unsigned>((N + per - 1) / per), static_cast<unsigned>(B * H), 2);
#define DAB_DQ(TY, DD)                                                                                          \
  kv4_dequantize_kernel<TY, DD><<<grid, 256, 0, st>>>(in, static_cast<TY*>(k), static_cast<TY*>(v), os[0], os[1], \
                                                      os[2], static_cast<int>(H), N);                            \
  return cudaGetLastError();
#define DAB_DQ_D(TY) if (D == 64) { DAB_DQ(TY, 64) } DAB_DQ(TY, 128)
  switch (dtype) {
    case F32: DAB_DQ_D(float)
    case F16: DAB_DQ_D(__half)
    case BF16: DAB_DQ_D(__nv_bfloat16)
    default: return cudaErrorInvalidValue;
  }
#undef DAB_DQ
#undef DAB_DQ_D
}

// -------------------------------------------------------------------------------- update
// One warp per (batch, kv-head): the token that leaves the full exact ring is merged into the
// last anchor (count + 1) or appended in 4 bits, then the new token takes its slot
// (deltaDecoding.py:9-104 with a 4-bit history). The comparison is with `last_key`, the last
// anchor's key in 16 bits, in the reduction order of decode_update_kernel, so decisions are those
// of the 16-bit cache. The slot's attention mass goes with the token. One row a head is read and
// written; what counts is the chain state, row, comparison, write: 5 us for 1 sequence and for 64.
template <typename T, int D, bool COS>
__global__ void __launch_bounds__(128) kv4_update_kernel(Kv4Update p) {
  constexpr int NG = D / 32, PER = D / 8;
  const int lane = threadIdx.x & 31, g8 = lane & 7;
  const int64_t pid = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (pid >= static_cast<int64_t>(p.B) * p.H) return;
  const int b = static_cast<int>(pid) / p.H, h = static_cast<int>(pid) - b * p.H;
  const int64_t e = p.state[0], total = p.state[1];
  const int64_t slot = e % p.W;
  T* ek = static_cast<T*>(p.k_exact) + b * p.eb + h * p.eh + slot * p.en;
  T* ev = static_cast<T*>(p.v_exact) + b * p.eb + h * p.eh + slot * p.en;
  T* lk = static_cast<T*>(p.last_key) + b * p.lkb + h * p.lkh;
  int32_t* len = p.lengths + b * p.lb + h * p.lh;
  float* em = p.exact_mass ? p.exact_mass + b * p.emb + h * p.emh + slot : nullptr;
  const int32_t n = *len;
  const T* sk = static_cast<const T*>(p.k_new) + b * p.kb + h * p.kh;
  const T* sv = static_cast<const T*>(p.v_new) + b * p.vb + h * p.vh;
  T nk[NG], nv[NG];
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    nk[g] = sk[(32 * g + lane) * p.kd];
    nv[g] = sv[(32 * g + lane) * p.vd];
  }
  if (e >= p.W) {
    float xk[NG], xv[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      xk[g] = to_f32(ek[32 * g + lane]);
      xv[g] = to_f32(ev[32 * g + lane]);
    }
    const float m = em ? *em : 0.f;
    const int64_t meta = b * p.mb + h * p.mh;
    bool merge = false;
    if (n > 0 && n <= p.cap) {
      auto tree = [](float v) {
        v = __fadd_rn(v, __shfl_xor_sync(0xFFFFFFFFu, v, 1));
        v = __fadd_rn(v, __shfl_xor_sync(0xFFFFFFFFu, v, 2));
        return __fadd_rn(v, __shfl_xor_sync(0xFFFFFFFFu, v, 4));
      };
      float a0 = 0.f, a1 = 0.f, a2 = 0.f;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const float x = to_f32(ek[g8 + 8 * j]), y = to_f32(lk[g8 + 8 * j]);
        if constexpr (COS) {
          const float xy = __fmul_rn(x, y), xx = __fmul_rn(x, x), yy = __fmul_rn(y, y);
          a0 = j ? __fadd_rn(a0, xy) : xy;
          a1 = j ? __fadd_rn(a1, xx) : xx;
          a2 = j ? __fadd_rn(a2, yy) : yy;
        } else {
          const float d = __fsub_rn(x, y), dd = __fmul_rn(d, d);
          a0 = j ? __fadd_rn(a0, dd) : dd;
        }
      }
      a0 = tree(a0);
      if constexpr (COS) {
        const float ne = __fsqrt_rn(__fadd_rn(tree(a1), 1e-8f)), nl = __fsqrt_rn(__fadd_rn(tree(a2), 1e-8f));
        merge = __fdiv_rn(a0, __fmul_rn(ne, nl)) >= p.threshold;
      } else {
        merge = a0 <= p.threshold;
      }
    }
    if (merge) {
      if (lane == 0) {
        p.counts[meta + n - 1] += 1;
        if (p.mass) p.mass[meta + n - 1] += m;
      }
    } else if (n >= 0 && n < p.cap) {
      kv4_quantize_row<NG>(xk, reinterpret_cast<uint32_t*>(p.hist.k_codes + b * p.hist.cb + h * p.hist.ch + static_cast<int64_t>(n) * (D / 2)),
                           p.hist.k_scales + b * p.hist.sb + h * p.hist.sh + static_cast<int64_t>(n) * (2 * NG), lane);
      kv4_quantize_row<NG>(xv, reinterpret_cast<uint32_t*>(p.hist.v_codes + b * p.hist.cb + h * p.hist.ch + static_cast<int64_t>(n) * (D / 2)),
                           p.hist.v_scales + b * p.hist.sb + h * p.hist.sh + static_cast<int64_t>(n) * (2 * NG), lane);
      __syncwarp();  // every lane has read the last key before it changes
#pragma unroll
      for (int g = 0; g < NG; ++g) lk[32 * g + lane] = ek[32 * g + lane];
      if (lane == 0) {
        p.counts[meta + n] = 1;
        p.times[meta + n] = static_cast<int32_t>(total - p.W);
        if (p.mass) p.mass[meta + n] = m;
        *len = n + 1;
      }
    } else if (lane == 0 && p.err) {
      atomicCAS(p.err, 0, 0x201);  // history full: evict first
    }
  }
  __syncwarp();  // the leaving row has been read by every lane before it is overwritten
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    ek[32 * g + lane] = nk[g];
    ev[32 * g + lane] = nv[g];
  }
  if (lane == 0 && em) *em = 0.f;
}

cudaError_t launch_kv4_update(int dtype, int64_t D, bool cosine, const Kv4Update& p, cudaStream_t st) {
  const int64_t heads = static_cast<int64_t>(p.B) * p.H;
  if (heads == 0) return cudaSuccess;
  const unsigned blocks = static_cast<unsigned>((heads + 3) / 4);
#define DAB_U(TY, DD)                                                     \
  if (cosine) kv4_update_kernel<TY, DD, true><<<blocks, 128, 0, st>>>(p); \
  else kv4_update_kernel<TY, DD, false><<<blocks, 128, 0, st>>>(p);       \
  return cudaGetLastError();
  if (dtype == BF16) { if (D == 64) { DAB_U(__nv_bfloat16, 64) } DAB_U(__nv_bfloat16, 128) }
  if (D == 64) { DAB_U(__half, 64) }
  DAB_U(__half, 128)
#undef DAB_U
}

}  // namespace dab
