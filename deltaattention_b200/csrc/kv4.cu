// A decode history in 4 bits (format in kv4.cuh): quantisation of packed K / V rows, reading
// back, the single-token cache update and single-token attention.
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

// ----------------------------------------------------------------------------- attention
// Split over the keys: a CTA scores 128 keys (history, then exact window) for up to 8 q-heads of
// one kv-head, one key per thread, then sums the values one column per thread. Scores are kept in
// log2 units without the count, which weights the exponential: p = count * 2^(z - max). A second
// kernel joins the parts; with `mass` a third adds every key's share, from the scores that the
// first one left in the workspace.
constexpr int KV4_CHUNK = 128;

template <typename T, int D>
__global__ void __launch_bounds__(128) kv4_attn_kernel(Kv4Attn p) {
  constexpr int NG = D / 32;
  __shared__ float sq[8][D];
  __shared__ float sp[8][KV4_CHUNK];
  __shared__ float red[4][8];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int bh = blockIdx.y, b = bh / p.H, h = bh - b * p.H;
  const int g0 = blockIdx.z * 8, ng = min(8, p.G - g0);
  int64_t elen = p.exact_len;
  if (p.state) elen = min(static_cast<int64_t>(p.W), p.state[0] + p.lag);
  const int64_t n = max(0, min(p.lengths[b * p.lb + h * p.lh], p.cap));
  const int64_t total = n + elen, k0 = static_cast<int64_t>(blockIdx.x) * KV4_CHUNK;
  float* part = p.part + ((static_cast<int64_t>(bh) * p.G + g0) * p.nsplit + blockIdx.x) * (D + 2);
  if (k0 >= total) {
    if (tid < ng) {
      part[static_cast<int64_t>(tid) * p.nsplit * (D + 2)] = -INFINITY;
      part[static_cast<int64_t>(tid) * p.nsplit * (D + 2) + 1] = 0.f;
    }
    return;
  }
  const T* q = static_cast<const T*>(p.q) + b * p.qb + (static_cast<int64_t>(h) * p.G + g0) * p.qh;
  for (int i = tid; i < 8 * D; i += 128) {
    const int g = i / D, d = i - g * D;
    sq[g][d] = g < ng ? to_f32(q[g * p.qh + d]) * p.scale_log2 : 0.f;
  }
  __syncthreads();
  const int64_t key = k0 + tid;
  const bool old = key < n;
  float c = key < total ? 1.f : 0.f;
  if (old) c = static_cast<float>(max(0, p.counts[b * p.mb + h * p.mh + key]));
  float z[8];
#pragma unroll
  for (int g = 0; g < 8; ++g) z[g] = 0.f;
  if (c > 0.f) {
    if (old) {
      const uint32_t* w = reinterpret_cast<const uint32_t*>(p.hist.k_codes + b * p.hist.cb + h * p.hist.ch + key * (D / 2));
      const __nv_bfloat16* s = p.hist.k_scales + b * p.hist.sb + h * p.hist.sh + key * (2 * NG);
      for (int i = 0; i < D / 8; ++i) {
        const int t = i / NG, gr = i - t * NG;
        const uint32_t word = w[i];
        const float sc = to_f32(s[gr]), ze = to_f32(s[NG + gr]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = fmaf(sc, static_cast<float>((word >> (4 * e)) & 15u), ze);
#pragma unroll
          for (int g = 0; g < 8; ++g) z[g] = fmaf(sq[g][32 * gr + 8 * t + e], x, z[g]);
        }
      }
    } else {
      const T* row = static_cast<const T*>(p.k_exact) + b * p.eb + h * p.eh + (key - n) * p.en;
      for (int d = 0; d < D; ++d) {
        const float x = to_f32(row[d]);
#pragma unroll
        for (int g = 0; g < 8; ++g) z[g] = fmaf(sq[g][d], x, z[g]);
      }
    }
  }
#pragma unroll
  for (int g = 0; g < 8; ++g) {
    if (!(c > 0.f)) z[g] = -INFINITY;
    float m = z[g];
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
    if (lane == 0) red[warp][g] = m;
    if (p.scores && g < ng && key < total)
      p.scores[(static_cast<int64_t>(bh) * p.G + g0 + g) * p.sstride + key] = z[g];
  }
  __syncthreads();
  float mx[8];
#pragma unroll
  for (int g = 0; g < 8; ++g) mx[g] = fmaxf(fmaxf(red[0][g], red[1][g]), fmaxf(red[2][g], red[3][g]));
  __syncthreads();
#pragma unroll
  for (int g = 0; g < 8; ++g) {
    const float pr = c > 0.f ? c * ex2(z[g] - (mx[g] == -INFINITY ? 0.f : mx[g])) : 0.f;
    sp[g][tid] = pr;
    float l = pr;
#pragma unroll
    for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(0xFFFFFFFFu, l, o);
    if (lane == 0) red[warp][g] = l;
  }
  __syncthreads();
  const int kend = static_cast<int>(min(static_cast<int64_t>(KV4_CHUNK), total - k0));
  if (tid < D) {
    float acc[8];
#pragma unroll
    for (int g = 0; g < 8; ++g) acc[g] = 0.f;
    const int gr = tid / 32, t = (tid / 8) & 3, e = tid & 7;
    for (int j = 0; j < kend; ++j) {
      const int64_t kk = k0 + j;
      float x;
      if (kk < n) {
        if (p.counts[b * p.mb + h * p.mh + kk] <= 0) continue;
        const uint32_t word = reinterpret_cast<const uint32_t*>(p.hist.v_codes + b * p.hist.cb + h * p.hist.ch + kk * (D / 2))[t * NG + gr];
        const __nv_bfloat16* s = p.hist.v_scales + b * p.hist.sb + h * p.hist.sh + kk * (2 * NG);
        x = fmaf(to_f32(s[gr]), static_cast<float>((word >> (4 * e)) & 15u), to_f32(s[NG + gr]));
      } else {
        x = to_f32(static_cast<const T*>(p.v_exact)[b * p.eb + h * p.eh + (kk - n) * p.en + tid]);
      }
#pragma unroll
      for (int g = 0; g < 8; ++g) acc[g] = fmaf(sp[g][j], x, acc[g]);
    }
    for (int g = 0; g < ng; ++g) part[static_cast<int64_t>(g) * p.nsplit * (D + 2) + 2 + tid] = acc[g];
  }
  if (tid < ng) {
    part[static_cast<int64_t>(tid) * p.nsplit * (D + 2)] = mx[tid];
    part[static_cast<int64_t>(tid) * p.nsplit * (D + 2) + 1] = (red[0][tid] + red[1][tid]) + (red[2][tid] + red[3][tid]);
  }
}

// One CTA of D threads per q-head: out = sum of the parts' accumulators over their sums, 0 where
// nothing is left; (max, 1 / sum) of the whole row for the mass.
template <typename T, int D>
__global__ void __launch_bounds__(D) kv4_join_kernel(Kv4Attn p) {
  const int row = blockIdx.x;  // batch * q-heads
  const float* part = p.part + static_cast<int64_t>(row) * p.nsplit * (D + 2);
  float m = -INFINITY;
  for (int s = 0; s < p.nsplit; ++s) m = fmaxf(m, part[static_cast<int64_t>(s) * (D + 2)]);
  const float ref = m == -INFINITY ? 0.f : m;
  float l = 0.f, acc = 0.f;
  for (int s = 0; s < p.nsplit; ++s) {
    const float* ps = part + static_cast<int64_t>(s) * (D + 2);
    if (ps[0] == -INFINITY) continue;  // a part without keys has no accumulators
    const float f = ex2(ps[0] - ref);
    l = fmaf(ps[1], f, l);
    acc = fmaf(ps[2 + threadIdx.x], f, acc);
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int hq = p.H * p.G, b = row / hq, h = row - b * hq;
  static_cast<T*>(p.out)[b * p.ob + h * p.oh + threadIdx.x] = from_f32<T>(l == 0.f ? 0.f : acc * inv);
  if (threadIdx.x == 0) {
    p.stats[2 * row] = ref;
    p.stats[2 * row + 1] = inv;
    if (p.lag && row == 0) {  // the step's length advance, after the state's last reader
      p.state[0] += 1;
      p.state[1] += 1;
    }
  }
}

__global__ void __launch_bounds__(256) kv4_mass_kernel(Kv4Attn p) {
  const int bh = blockIdx.y, b = bh / p.H, h = bh - b * p.H;
  int64_t elen = p.exact_len;
  if (p.state) elen = min(static_cast<int64_t>(p.W), p.state[0]);  // the join has advanced it
  const int64_t n = max(0, min(p.lengths[b * p.lb + h * p.lh], p.cap));
  const int64_t key = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (key >= n + elen) return;
  const float c = key < n ? static_cast<float>(max(0, p.counts[b * p.mb + h * p.mh + key])) : 1.f;
  if (!(c > 0.f)) return;
  float w = 0.f;
  for (int g = 0; g < p.G; ++g) {
    const int64_t row = static_cast<int64_t>(bh) * p.G + g;
    w = fmaf(ex2(p.scores[row * p.sstride + key] - p.stats[2 * row]), p.stats[2 * row + 1], w);
  }
  float* dst = key < n ? p.mass + b * p.mb + h * p.mh + key : p.exact_mass + b * p.emb + h * p.emh + (key - n);
  *dst += c * w;
}

namespace {
struct Kv4Ws {
  int nsplit;
  int64_t sstride, part, scores, stats, total;  // offsets in bytes
};
Kv4Ws kv4_ws(int64_t B, int64_t Hq, int64_t D, int64_t cap, int64_t W, bool mass) {
  auto up = [](int64_t x) { return (x + 255) & ~int64_t{255}; };
  Kv4Ws w;
  w.nsplit = static_cast<int>((cap + W + KV4_CHUNK - 1) / KV4_CHUNK);
  if (w.nsplit < 1) w.nsplit = 1;
  w.sstride = cap + W;
  w.part = 256;
  w.stats = w.part + up(B * Hq * w.nsplit * (D + 2) * 4);
  w.scores = w.stats + up(B * Hq * 2 * 4);
  w.total = w.scores + (mass ? up(B * Hq * w.sstride * 4) : 0);
  return w;
}
}  // namespace

size_t kv4_attn_workspace(int64_t B, int64_t Hq, int64_t D, int64_t cap, int64_t W, bool mass) {
  return static_cast<size_t>(kv4_ws(B, Hq, D, cap, W, mass).total);
}

cudaError_t launch_kv4_attn(int dtype, int64_t D, Kv4Attn p, uint8_t* ws, cudaStream_t st) {
  const int64_t Hq = static_cast<int64_t>(p.H) * p.G;
  if (p.B * Hq == 0) return cudaSuccess;
  const Kv4Ws w = kv4_ws(p.B, Hq, D, p.cap, p.W, p.mass != nullptr);
  p.nsplit = w.nsplit;
  p.sstride = w.sstride;
  p.part = reinterpret_cast<float*>(ws + w.part);
  p.stats = reinterpret_cast<float*>(ws + w.stats);
  p.scores = p.mass ? reinterpret_cast<float*>(ws + w.scores) : nullptr;
  dim3 grid(static_cast<unsigned>(w.nsplit), static_cast<unsigned>(p.B * p.H), static_cast<unsigned>((p.G + 7) / 8));
#define DAB_A(TY, DD)                                                                    \
  kv4_attn_kernel<TY, DD><<<grid, 128, 0, st>>>(p);                                       \
  kv4_join_kernel<TY, DD><<<static_cast<unsigned>(p.B * Hq), DD, 0, st>>>(p);
  if (dtype == BF16 && D == 64) { DAB_A(__nv_bfloat16, 64) }
  else if (dtype == BF16) { DAB_A(__nv_bfloat16, 128) }
  else if (D == 64) { DAB_A(__half, 64) }
  else { DAB_A(__half, 128) }
#undef DAB_A
  if (p.mass) {
    dim3 gm(static_cast<unsigned>((p.cap + p.W + 255) / 256), static_cast<unsigned>(p.B * p.H));
    kv4_mass_kernel<<<gm, 256, 0, st>>>(p);
  }
  return cudaGetLastError();
}

}  // namespace dab
