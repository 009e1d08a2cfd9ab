// Attention of packed prompts, of prompts over a paged cache, and of one token per sequence over it.
//
// out_i = sum_{j < limit_i} softmax_j(scale q_i . k_j) v_j, limit_i = the query's position + 1 (causal) or
// the sequence's length; q-head h reads K / V head h / G. A row that sees nothing gives 0.
//
// One block of 128 threads per (query, q-head): 128 keys at a time, a score per thread, the running
// maximum and sum in fp32, then an output element per thread.
#include "paged.cuh"

namespace dab {

template <int D, typename T>
__global__ void __launch_bounds__(128) paged_attn_kernel(const PagedAttn p) {
  __shared__ float sq[D], sp[128], red[4];
  __shared__ int sb;
  const int t = blockIdx.x, hq = blockIdx.y, h = hq / p.G, tid = threadIdx.x;
  if (tid < 32) {
    const int b = p.cu ? paged_sequence(p.cu, p.B, t) : t;
    if (tid == 0) sb = b;
  }
  if (tid < D) sq[tid] = to_f32(static_cast<const T*>(p.q)[t * p.q_t + hq * p.q_h + tid]) * p.scale_log2;
  __syncthreads();
  const int b = sb;
  if (b < 0) return;
  int c0, c1;
  paged_tokens(p.cu, b, p.T, p.err, c0, c1);
  const int n = c1 - c0;
  const int len = p.table ? paged_length(p.lengths[b], p.max_pages, p.ps_shift, p.err) : n;
  const int limit = p.causal ? len - n + (t - c0) + 1 : len;
  float m = -INFINITY, l = 0.f, o = 0.f;
  auto row_of = [&](int j, int64_t& ko, int64_t& vo) {
    if (!p.table) {
      ko = static_cast<int64_t>(c0 + j) * p.k_r + h * p.k_h;
      vo = static_cast<int64_t>(c0 + j) * p.v_r + h * p.v_h;
      return true;
    }
    const int page = p.table[b * p.table_stride + (j >> p.ps_shift)], r = j & ((1 << p.ps_shift) - 1);
    if (page < 0 || page >= p.num_pages) {
      paged_error(p.err, ERR_PAGE);
      return false;
    }
    ko = page * p.k_p + h * p.k_h + r * p.k_r;
    vo = page * p.v_p + h * p.v_h + r * p.v_r;
    return true;
  };
  for (int j0 = 0; j0 < limit; j0 += 128) {
    const int j = j0 + tid;
    float s = -INFINITY;
    int64_t ko, vo;
    if (j < limit) {
      s = 0.f;
      if (row_of(j, ko, vo))
        for (int d = 0; d < D; ++d) s += sq[d] * to_f32(static_cast<const T*>(p.k)[ko + d]);
    }
    float mx = s;
    for (int o2 = 16; o2; o2 >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, o2));
    if ((tid & 31) == 0) red[tid >> 5] = mx;
    __syncthreads();
    const float mn = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
    const float base = mn == -INFINITY ? 0.f : mn, f = ex2(m - base);
    sp[tid] = ex2(s - base);
    m = mn;
    __syncthreads();
    l *= f;
    o *= f;
    for (int i = 0; i < 128 && j0 + i < limit; ++i) {
      l += sp[i];
      if (tid < D && row_of(j0 + i, ko, vo)) o += sp[i] * to_f32(static_cast<const T*>(p.v)[vo + tid]);
    }
    __syncthreads();
  }
  if (tid < D) static_cast<T*>(p.out)[t * p.o_t + hq * p.o_h + tid] = from_f32<T>(limit > 0 ? o / l : 0.f);
}

size_t paged_attn_workspace(int64_t, int64_t, int64_t, int64_t, int64_t, int64_t) { return 256; }

cudaError_t launch_paged_attn(int dtype, int head_dim, const PagedAttn& p, uint8_t*, int, cudaStream_t st) {
  if (p.T == 0) return cudaSuccess;
  const dim3 grid(p.T, p.H * p.G);
  if (dtype == BF16 && head_dim == 64) paged_attn_kernel<64, __nv_bfloat16><<<grid, 128, 0, st>>>(p);
  else if (dtype == BF16 && head_dim == 128) paged_attn_kernel<128, __nv_bfloat16><<<grid, 128, 0, st>>>(p);
  else if (dtype == F16 && head_dim == 64) paged_attn_kernel<64, __half><<<grid, 128, 0, st>>>(p);
  else if (dtype == F16 && head_dim == 128) paged_attn_kernel<128, __half><<<grid, 128, 0, st>>>(p);
  else return cudaErrorInvalidValue;
  return cudaGetLastError();
}

}  // namespace dab
