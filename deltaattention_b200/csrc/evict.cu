// Eviction from a decode cache by accumulated attention weight.
//
// A head longer than `trigger` is cut to `budget` entries: its first `first`, its last `recent`,
// and of the entries between the k = budget - first - recent heaviest, ties to the lowest index.
// Entries keep their order, and every row buffer is compacted in place with the mass.
//
//  * evict_select: the k-th largest weight of the middle entries by radix selection over 4 digits
//    of 8 bits, and how many entries that equal it are kept.
//  * evict_move: kept entries move to the front. An entry's destination is never behind its
//    source, so tiles taken in order overwrite only entries that have been read.
#include "evict.cuh"

namespace dab {

// Unsigned key of a weight in the order of floats: NaN below everything, -0 equal to +0.
__device__ __forceinline__ uint32_t mass_key(float x) {
  if (x != x) return 0u;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u ^ ((u >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}

__global__ void __launch_bounds__(1024) evict_select_kernel(EvictParams p) {
  __shared__ uint32_t hist[256];
  __shared__ uint32_t s_prefix, s_k;
  const int bh = blockIdx.x, b = bh / p.H, h = bh - b * p.H;
  const int n = min(p.lengths[b * p.lb + h * p.lh], p.cap);
  if (n <= p.trigger) return;
  const float* mass = p.mass + b * p.mb + h * p.mh;
  const int lo = p.first, hi = n - p.recent;
  uint32_t k = p.budget - p.first - p.recent;
  if (k == 0) {  // nothing between the protected ends stays
    if (threadIdx.x == 0) p.cut[bh] = make_uint2(0xFFFFFFFFu, 0u);
    return;
  }
  uint32_t prefix = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256; i += blockDim.x) hist[i] = 0;
    __syncthreads();
    const uint32_t mask = shift == 24 ? 0u : 0xFFFFFFFFu << (shift + 8);
    for (int i = lo + threadIdx.x; i < hi; i += blockDim.x) {
      const uint32_t key = mass_key(mass[i]);
      if ((key & mask) == prefix) atomicAdd(&hist[(key >> shift) & 255u], 1u);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      uint32_t left = k;
      int d = 255;
      for (; d > 0 && hist[d] < left; --d) left -= hist[d];
      s_prefix = prefix | (static_cast<uint32_t>(d) << shift);
      s_k = left;
    }
    __syncthreads();
    prefix = s_prefix;
    k = s_k;
    __syncthreads();
  }
  if (threadIdx.x == 0) p.cut[bh] = make_uint2(prefix, k);
}

template <typename U>
__device__ __forceinline__ void move_rows(uint8_t* base, int bytes, const int* src, int dst0, int kept) {
  const int upr = bytes / static_cast<int>(sizeof(U));
  const int total = kept * upr;
  for (int u0 = 0; u0 < total; u0 += blockDim.x) {
    const int u = u0 + threadIdx.x;
    const int r = u / upr, c = u - r * upr;
    U v;
    if (u < total) v = reinterpret_cast<const U*>(base + static_cast<int64_t>(src[r]) * bytes)[c];
    __syncthreads();
    if (u < total) reinterpret_cast<U*>(base + static_cast<int64_t>(dst0 + r) * bytes)[c] = v;
    __syncthreads();
  }
}

__global__ void __launch_bounds__(256) evict_move_kernel(EvictParams p) {
  __shared__ int src[256];
  __shared__ int w_tie[8], w_keep[8];
  const int bh = blockIdx.x, b = bh / p.H, h = bh - b * p.H;
  int32_t* len = p.lengths + b * p.lb + h * p.lh;
  const int n = min(*len, p.cap);
  if (n <= p.trigger) return;
  const uint2 cut = p.cut[bh];
  float* mass = p.mass + b * p.mb + h * p.mh;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t below = (1u << lane) - 1u;
  int ties = 0, dst = 0;
  for (int i0 = 0; i0 < n; i0 += 256) {
    const int i = i0 + threadIdx.x;
    const float m = i < n ? mass[i] : 0.f;
    const bool mid = i >= p.first && i < n - p.recent;
    const uint32_t key = mass_key(m);
    const bool tie = mid && key == cut.x;
    bool keep = i < n && (!mid || key > cut.x);
    const uint32_t tb = __ballot_sync(0xFFFFFFFFu, tie);
    if (lane == 0) w_tie[warp] = __popc(tb);
    __syncthreads();
    int before = ties + __popc(tb & below), tt = 0;
    for (int w = 0; w < 8; ++w) {
      if (w < warp) before += w_tie[w];
      tt += w_tie[w];
    }
    ties += tt;
    if (tie && before < static_cast<int>(cut.y)) keep = true;
    const uint32_t kb = __ballot_sync(0xFFFFFFFFu, keep);
    if (lane == 0) w_keep[warp] = __popc(kb);
    __syncthreads();
    int pos = __popc(kb & below), kept = 0;
    for (int w = 0; w < 8; ++w) {
      if (w < warp) pos += w_keep[w];
      kept += w_keep[w];
    }
    if (keep) {
      src[pos] = i;
      mass[dst + pos] = m;  // the tile's weights have all been read
    }
    __syncthreads();
    for (int r = 0; r < p.n_rows; ++r) {
      uint8_t* base = p.row[r] + b * p.rb[r] + h * p.rh[r];
      if (p.unit[r] == 16) move_rows<uint4>(base, p.bytes[r], src, dst, kept);
      else if (p.unit[r] == 8) move_rows<uint2>(base, p.bytes[r], src, dst, kept);
      else move_rows<uint32_t>(base, p.bytes[r], src, dst, kept);
    }
    dst += kept;
    __syncthreads();
  }
  if (threadIdx.x == 0) *len = p.budget;
}

size_t evict_workspace(int64_t B, int64_t H, int64_t cap) {
  (void)cap;
  return static_cast<size_t>(256 + B * H * 8);
}

cudaError_t launch_evict(EvictParams p, uint8_t* ws, cudaStream_t st) {
  if (p.B * p.H == 0 || p.cap == 0) return cudaSuccess;
  p.cut = reinterpret_cast<uint2*>(ws + 256);
  evict_select_kernel<<<p.B * p.H, 1024, 0, st>>>(p);
  evict_move_kernel<<<p.B * p.H, 256, 0, st>>>(p);
  return cudaGetLastError();
}

}  // namespace dab
