// New K / V rows into a paged cache, with the rotation of K and of the tokens' queries on the way.
//
// A token at position p of its sequence goes to row p % page_size of the page table[b][p / page_size]:
//   K' = K cos[p] + turned(K) sin[p], turned(x) = (-x[D/2:], x[:D/2]);  V' = V;  Q' = Q cos[p] + turned(Q) sin[p]
// in fp32 and rounded once (ops.rope rounds its products as eager bf16 does; here nothing is compared
// with those bits, and one rounding is nearer to the formula).
//
// Nothing is read twice but the tables' rows, so bytes or, for a step's few tokens, latency bound it. A
// warp takes one slice of one token's heads: D / 16 lanes hold a row's piece and its partner half a row
// away, 16 bytes each, so a rotation needs no exchange, and the token's sines and cosines stay in
// registers over all heads of the slice. 56000 tokens of 32 + 2 x 8 heads of 128 (1.35 GB): 220 us, 6.1 TB/s.
// Loads that are not kept (the rows are read once) took it there from 250 us, four blocks on an SM with two rows a
// lane in flight instead of three with four from 262; stores that are not kept cost 7 us. One token: 3 us.
#include "paged.cuh"

namespace dab {

template <typename T> __device__ __forceinline__ void unpack8(const uint4& w, float* x) {
  const T* t = reinterpret_cast<const T*>(&w);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = to_f32(t[i]);
}
template <typename T> __device__ __forceinline__ uint4 pack8(const float* x) {
  uint4 w;
  T* t = reinterpret_cast<T*>(&w);
#pragma unroll
  for (int i = 0; i < 8; ++i) t[i] = from_f32<T>(x[i]);
  return w;
}
template <typename TT> __device__ __forceinline__ void load_table8(const void* base, int64_t off, float* x) {
  const TT* t = static_cast<const TT*>(base) + off;
  if constexpr (sizeof(TT) == 4) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(t)), b = __ldg(reinterpret_cast<const float4*>(t) + 1);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  } else {
    unpack8<TT>(__ldg(reinterpret_cast<const uint4*>(t)), x);
  }
}

template <int D, typename T, typename TT>
__global__ void __launch_bounds__(256, 4) paged_append_kernel(const PagedAppend p, int slices) {
  constexpr int LR = D / 16;        // lanes of a rotated row
  constexpr int RW = 32 / LR;       // rotated rows a warp has at once
  const int64_t item = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int t = static_cast<int>(item / slices), slice = static_cast<int>(item % slices), lane = lane_id();
  if (t >= p.T) return;
  int b = t, left = 1;  // tokens of the sequence from this one on
  if (p.cu) {
    b = paged_sequence(p.cu, p.B, t);
    if (b < 0) return;
    left = p.cu[b + 1] - t;
  }
  const int pos = p.lengths[b] - left;
  if (pos < 0) return;  // an idle place of the batch
  const int page_at = pos >> p.ps_shift;
  if (page_at >= p.max_pages) {
    if (lane == 0) paged_error(p.err, ERR_LENGTH);
    return;
  }
  const int page = p.table[b * p.table_stride + page_at];
  const bool rotate = p.cos != nullptr;
  if (rotate && pos >= p.table_rows) {
    if (lane == 0) paged_error(p.err, ERR_POSITION);
    return;
  }
  const bool stored = page >= 0 && page < p.num_pages;
  if (!stored && lane == 0) paged_error(p.err, ERR_PAGE);
  const int64_t row = page * p.p_p + (pos & ((1 << p.ps_shift) - 1)) * p.p_r;
  const int rl = lane / LR, at = (lane % LR) * 8;

  if (rotate) {
    float c0[8], c1[8], s0[8], s1[8];
    load_table8<TT>(p.cos, pos * p.cs_r + at, c0);
    load_table8<TT>(p.cos, pos * p.cs_r + D / 2 + at, c1);
    load_table8<TT>(p.sin, pos * p.cs_r + at, s0);
    load_table8<TT>(p.sin, pos * p.cs_r + D / 2 + at, s1);
    const int rows = p.H + p.Hq;
#pragma unroll 2
    for (int h = slice * RW + rl; h < rows; h += slices * RW) {
      const T* src;
      T* dst;
      if (h < p.H) {
        src = static_cast<const T*>(p.k) + t * p.k_t + h * p.k_h;
        dst = stored ? static_cast<T*>(p.kp) + row + h * p.p_h : nullptr;
      } else {
        src = static_cast<const T*>(p.q) + t * p.q_t + (h - p.H) * p.q_h;
        dst = static_cast<T*>(p.q_out) + t * p.qo_t + (h - p.H) * p.qo_h;
      }
      float a[8], c[8], x[8], y[8];
      unpack8<T>(__ldcs(reinterpret_cast<const uint4*>(src + at)), a);
      unpack8<T>(__ldcs(reinterpret_cast<const uint4*>(src + D / 2 + at)), c);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = a[i] * c0[i] - c[i] * s0[i];
        y[i] = c[i] * c1[i] + a[i] * s1[i];
      }
      if (dst) {
        *reinterpret_cast<uint4*>(dst + at) = pack8<T>(x);
        *reinterpret_cast<uint4*>(dst + D / 2 + at) = pack8<T>(y);
      }
    }
  }
  if (!stored) return;
  // rows that go in as they are: V, and K without tables
  const int rows = rotate ? p.H : 2 * p.H;
#pragma unroll 2
  for (int h = slice * RW + rl; h < rows; h += slices * RW) {
    const bool is_v = h < p.H;
    const int hh = is_v ? h : h - p.H;
    const T* src = is_v ? static_cast<const T*>(p.v) + t * p.v_t + hh * p.v_h
                        : static_cast<const T*>(p.k) + t * p.k_t + hh * p.k_h;
    T* dst = static_cast<T*>(is_v ? p.vp : p.kp) + row + hh * p.p_h;
    const uint4 w0 = __ldcs(reinterpret_cast<const uint4*>(src + at)), w1 = __ldcs(reinterpret_cast<const uint4*>(src + D / 2 + at));
    *reinterpret_cast<uint4*>(dst + at) = w0;
    *reinterpret_cast<uint4*>(dst + D / 2 + at) = w1;
  }
}

template <int D, typename T, typename TT>
static cudaError_t launch_append_t(const PagedAppend& p, int num_sms, cudaStream_t st) {
  constexpr int RW = 512 / D;
  // Few tokens: a row of heads to every warp, the latency of one pass. Many: slices merge until the
  // tables' values are read once for a token.
  const int most = (p.H + p.Hq + RW - 1) / RW;
  int slices = most;
  while (slices > 1 && static_cast<int64_t>(p.T) * slices > static_cast<int64_t>(num_sms) * 64) slices = (slices + 1) / 2;
  const int64_t warps = static_cast<int64_t>(p.T) * slices;
  const int per = warps >= static_cast<int64_t>(num_sms) * 8 ? 8 : 2;
  paged_append_kernel<D, T, TT><<<static_cast<unsigned>((warps + per - 1) / per), per * 32, 0, st>>>(p, slices);
  return cudaGetLastError();
}

cudaError_t launch_paged_append(int dtype, bool table_f32, int head_dim, const PagedAppend& p, int num_sms,
                                cudaStream_t st) {
  if (p.T == 0) return cudaSuccess;
#define GO(D, T) \
  return table_f32 ? launch_append_t<D, T, float>(p, num_sms, st) : launch_append_t<D, T, T>(p, num_sms, st)
  if (dtype == BF16) {
    if (head_dim == 64) GO(64, __nv_bfloat16);
    if (head_dim == 128) GO(128, __nv_bfloat16);
  } else if (dtype == F16) {
    if (head_dim == 64) GO(64, __half);
    if (head_dim == 128) GO(128, __half);
  }
#undef GO
  return cudaErrorInvalidValue;
}

}  // namespace dab
