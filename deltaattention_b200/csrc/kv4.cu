// A decode history in 4 bits (format in kv4.cuh): quantisation of packed K / V rows, reading
// back, and the single-token cache update.
#include "kv4.cuh"

namespace dab {

// ------------------------------------------------------------------- quantise / read back
// One warp per row; blockIdx.y: batch * head, blockIdx.z: K or V.
template <typename T, int D>
__global__ void __launch_bounds__(256) kv4_quantize_kernel(const T* __restrict__ k, const T* __restrict__ v, int64_t kb,
                                                           int64_t kh, int64_t kn, int64_t kd, int64_t vb, int64_t vh,
                                                           int64_t vn, int64_t vd, Kv4Hist out, int H, int64_t N) {
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

// One thread per code word (8 elements).
template <typename T, int D>
__global__ void __launch_bounds__(256) kv4_dequantize_kernel(Kv4Hist in, T* __restrict__ k, T* __restrict__ v,
                                                             int64_t ob, int64_t oh, int64_t on, int H, int64_t N) {
  constexpr int NG = D / 32, NWORD = D / 8;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t n = i / NWORD;
  if (n >= N) return;
  const int w = static_cast<int>(i % NWORD), t = w / NG, g = w % NG;
  const int b = blockIdx.y / H, h = blockIdx.y - b * H;
  const bool is_v = blockIdx.z != 0;
  const uint8_t* c = (is_v ? in.v_codes : in.k_codes) + b * in.cb + h * in.ch + n * (D / 2);
  const __nv_bfloat16* s = (is_v ? in.v_scales : in.k_scales) + b * in.sb + h * in.sh + n * (2 * NG);
  const uint32_t word = reinterpret_cast<const uint32_t*>(c)[w];
  const float scale = to_f32(s[g]), zero = to_f32(s[NG + g]);
  T* dst = (is_v ? v : k) + b * ob + h * oh + n * on + 32 * g + 8 * t;
#pragma unroll
  for (int e = 0; e < 8; ++e)
    dst[e] = from_f32<T>(fmaf(scale, static_cast<float>((word >> (4 * e)) & 15u), zero));
}

cudaError_t launch_kv4_quantize(int dtype, const void* k, const int64_t* ks, const void* v, const int64_t* vs,
                                const Kv4Hist& out, int64_t B, int64_t H, int64_t N, int64_t D, cudaStream_t st) {
  if (B * H * N == 0) return cudaSuccess;
  dim3 grid(static_cast<unsigned>((N + 7) / 8), static_cast<unsigned>(B * H), 2);
#define DAB_Q(TY, DD)                                                                                             \
  kv4_quantize_kernel<TY, DD><<<grid, 256, 0, st>>>(static_cast<const TY*>(k), static_cast<const TY*>(v), ks[0],    \
                                                    ks[1], ks[2], ks[3], vs[0], vs[1], vs[2], vs[3], out,           \
                                                    static_cast<int>(H), N);                                       \
  return cudaGetLastError();
  if (dtype == BF16) { if (D == 64) { DAB_Q(__nv_bfloat16, 64) } DAB_Q(__nv_bfloat16, 128) }
  if (D == 64) { DAB_Q(__half, 64) }
  DAB_Q(__half, 128)
#undef DAB_Q
}

cudaError_t launch_kv4_dequantize(int dtype, const Kv4Hist& in, void* k, void* v, const int64_t* os, int64_t B,
                                  int64_t H, int64_t N, int64_t D, cudaStream_t st) {
  if (B * H * N == 0) return cudaSuccess;
  dim3 grid(static_cast<unsigned>((N * (D / 8) + 255) / 256), static_cast<unsigned>(B * H), 2);
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
// of the 16-bit cache. The slot's attention mass goes with the token.
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
