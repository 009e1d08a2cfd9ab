// Eviction from a decode cache by accumulated attention weight.
//
// A head longer than `trigger` is cut to `budget` entries: its first `first`, its last `recent`,
// and of the entries between the k = budget - first - recent heaviest, ties to the lowest index.
// Entries keep their order, and every row buffer is compacted in place with the mass.
//
//  * evict_select: one cluster per head finds the k-th largest weight of the middle entries by
//    radix selection, digits of 11, 11 and 10 bits. Every CTA keeps the keys of its slice in
//    registers, 16 a thread, and counts a pass's digits in shared memory. The counts are summed
//    over the cluster in two steps, 256 sums of 8 bins and then the 8 bins of the one where the
//    count reaches k (8 CTAs reading all 2048 bins from each other took 5000 cycles a pass). Then
//    it writes for every tile how many entries are kept before it and how many of the ties come
//    before it.
//  * evict_move: one CTA per tile reads its kept rows into shared memory, says so, waits for the
//    (at most two) tiles on whose rows its own will land to have said so too, and writes. Tiles are
//    handed out in order by a ticket per head and nothing is waited for before a tile has read
//    its rows, so the tiles waited for are running and never wait themselves. Every kept row is
//    read and written once, with no second buffer.
#include <cooperative_groups.h>

#include "evict.cuh"

namespace dab {

namespace cg = cooperative_groups;

constexpr int SEL_THREADS = 1024, SEL_MAX_CTAS = 8;  // of a cluster
constexpr int SEL_KEYS = 16;                         // a thread's keys in registers; longer slices are read again
constexpr int SEL_BINS = 2048;
constexpr int SEL_CHUNK = SEL_THREADS * SEL_KEYS;
constexpr int MOVE_THREADS = 128;
enum { ERR_EVICT_WAIT = 0x501 };

// Unsigned key of a weight in the order of floats: NaN below everything, -0 equal to +0.
__device__ __forceinline__ uint32_t mass_key(float x) {
  if (x != x) return 0u;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u ^ ((u >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
constexpr uint32_t KEY_ZERO = 0x80000000u;  // weights of 0, which may be many

__device__ __forceinline__ void grid_next() { asm volatile("griddepcontrol.launch_dependents;"); }

__global__ void __launch_bounds__(SEL_THREADS) evict_select_kernel(const __grid_constant__ EvictParams p) {
  cg::cluster_group cl = cg::this_cluster();
  __shared__ __align__(16) uint32_t hist[3][SEL_BINS];
  __shared__ uint32_t coarse[3][256];
  __shared__ uint32_t cnt[SEL_CHUNK / 32];  // of a chunk's 32 entries each: surely kept, ties << 16
  __shared__ uint32_t wsum[8], s_bin, s_prefix, s_k;
  __shared__ __align__(8) uint32_t s_tot[2];
  __shared__ uint2 wcnt[SEL_CHUNK / 1024];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int C = static_cast<int>(cl.num_blocks()), rank = static_cast<int>(cl.block_rank());
  const int bh = blockIdx.y, b = bh / p.H, h = bh - b * p.H;
  int32_t* len = p.lengths + b * p.lb + h * p.lh;
  const int n = min(*len, p.cap);
  if (n <= p.trigger) {  // for the whole cluster
    if (rank == 0 && tid == 0) p.cut[bh] = make_uint4(0u, 0u, 0u, 0u);
    return;
  }
  const float* mass = p.mass + b * p.mb + h * p.mh;
  // this CTA's slice: whole tiles
  const int tiles = (n + p.tile - 1) / p.tile;
  const int t0 = static_cast<int>(static_cast<int64_t>(tiles) * rank / C);
  const int t1 = static_cast<int>(static_cast<int64_t>(tiles) * (rank + 1) / C);
  const int i0 = t0 * p.tile, i1 = min(n, t1 * p.tile);
  const int lo = p.first, hi = n - p.recent;  // the entries that compete
  uint32_t key[SEL_KEYS];
  auto load = [&](int base) {
#pragma unroll
    for (int j = 0; j < SEL_KEYS; ++j) {
      const int e = base + j * SEL_THREADS + tid;
      key[j] = __float_as_uint(mass[min(e, i1 - 1)]);  // all loads in flight
    }
#pragma unroll
    for (int j = 0; j < SEL_KEYS; ++j) key[j] = mass_key(__uint_as_float(key[j]));
  };
  load(i0);
  const bool one = i1 - i0 <= SEL_CHUNK;
  for (int i = tid; i < 3 * SEL_BINS; i += SEL_THREADS) (&hist[0][0])[i] = 0;
  for (int t = t0 + tid; t < t1; t += SEL_THREADS) p.loaded[static_cast<int64_t>(bh) * p.max_tiles + t] = 0u;
  uint32_t k = p.budget - p.first - p.recent, prefix = k ? 0u : 0xFFFFFFFFu;
  __syncthreads();
  if (k) {
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
      const uint32_t above = pass == 0 ? 0u : pass == 1 ? 0xFFE00000u : 0xFFFFFC00u;
      const uint32_t digits = pass == 2 ? 1023u : 2047u;
      uint32_t* hp = hist[pass];
      uint32_t zeros = 0;  // many weights may be 0: one addition a warp
      for (int base = i0; base < i1; base += SEL_CHUNK) {
        if (!one) load(base);
#pragma unroll
        for (int j = 0; j < SEL_KEYS; ++j) {
          const int e = base + j * SEL_THREADS + tid;
          if (base + j * SEL_THREADS >= i1) break;
          if (e >= lo && e < hi && e < i1 && (key[j] & above) == prefix) {
            if (key[j] == KEY_ZERO) ++zeros;
            else atomicAdd(&hp[(key[j] >> shift) & digits], 1u);
          }
        }
      }
      zeros = __reduce_add_sync(0xFFFFFFFFu, zeros);
      if (lane == 0 && zeros) atomicAdd(&hp[(KEY_ZERO >> shift) & digits], zeros);
      __syncthreads();
      if (tid < 256) {
        const uint4 x = reinterpret_cast<const uint4*>(hp)[2 * tid], y = reinterpret_cast<const uint4*>(hp)[2 * tid + 1];
        coarse[pass][tid] = (x.x + x.y) + (x.z + x.w) + (y.x + y.y) + (y.z + y.w);
      }
      if (C > 1) cl.sync();
      else __syncthreads();
      // thread i: sum 255 - i over the cluster; the digit is where the count from the top reaches k
      uint32_t c = 0, incl = 0;
      if (tid < 256) {
        if (C == 1) c = coarse[pass][255 - tid];
        else
#pragma unroll
          for (int r = 0; r < SEL_MAX_CTAS; ++r) {  // all loads in flight
            const uint32_t v = cl.map_shared_rank(&coarse[pass][0], min(r, C - 1))[255 - tid];
            c += r < C ? v : 0u;
          }
        incl = c;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, incl, o);
          if (lane >= o) incl += v;
        }
        if (lane == 31) wsum[warp] = incl;
      }
      __syncthreads();
      if (tid < 256) {
        uint32_t before = incl - c;
#pragma unroll
        for (int w = 0; w < 7; ++w)
          if (w < warp) before += wsum[w];
        if (before < k && k <= before + c) {
          s_bin = 255 - tid;
          s_k = k - before;
        }
      }
      __syncthreads();
      if (warp == 0) {  // lane i: bin 7 - i of the eight
        const uint32_t bin = 8 * s_bin + 7 - (lane & 7);
        c = 0;
        if (C == 1) c = hp[bin];
        else
#pragma unroll
          for (int r = 0; r < SEL_MAX_CTAS; ++r) {
            const uint32_t v = cl.map_shared_rank(hp, min(r, C - 1))[bin];
            c += r < C ? v : 0u;
          }
        incl = c;
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) {
          const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, incl, o, 8);
          if ((lane & 7) >= o) incl += v;
        }
        const uint32_t want = s_k;
        __syncwarp();
        if (lane < 8 && incl - c < want && want <= incl) {
          s_prefix = prefix | (bin << shift);
          s_k = want - (incl - c);
        }
      }
      __syncthreads();
      prefix = s_prefix;
      k = s_k;
    }
  }
  // per tile: entries surely kept, and ties
  uint2* before = p.before + static_cast<int64_t>(bh) * p.max_tiles;
  uint32_t run_s = 0, run_t = 0;  // of this CTA's entries so far
  for (int base = i0; base < i1; base += SEL_CHUNK) {
    if (!one) load(base);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < SEL_KEYS; ++j) {
      const int e = base + j * SEL_THREADS + tid;
      const bool mid = e >= lo && e < hi;
      const uint32_t sb = __ballot_sync(0xFFFFFFFFu, e < i1 && (!mid || key[j] > prefix));
      const uint32_t tb = __ballot_sync(0xFFFFFFFFu, e < i1 && mid && key[j] == prefix);
      if (lane == 0) cnt[j * (SEL_THREADS / 32) + warp] = __popc(sb) | __popc(tb) << 16;
    }
    __syncthreads();
    uint2 v = make_uint2(0u, 0u), x = v;  // exclusive sums: thread i, entries [32 i, 32 i + 32) of the chunk
    if (tid < SEL_CHUNK / 32) {
      v = x = make_uint2(cnt[tid] & 0xFFFFu, cnt[tid] >> 16);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t a = __shfl_up_sync(0xFFFFFFFFu, x.x, o), q = __shfl_up_sync(0xFFFFFFFFu, x.y, o);
        if (lane >= o) { x.x += a; x.y += q; }
      }
      if (lane == 31) wcnt[warp] = x;
    }
    __syncthreads();
    uint32_t add_s = run_s, add_t = run_t;
#pragma unroll
    for (int w = 0; w < SEL_CHUNK / 1024; ++w) {
      const uint2 y = wcnt[w];
      if (w < warp) { add_s += y.x; add_t += y.y; }
      run_s += y.x;
      run_t += y.y;
    }
    const int o = tid * 32;
    if (tid < SEL_CHUNK / 32 && (o & (p.tile - 1)) == 0 && base + o < i1)
      before[(base + o) >> p.tile_shift] = make_uint2(add_s + x.x - v.x, add_t + x.y - v.y);
  }
  if (tid == 0) {
    s_tot[0] = run_s;
    s_tot[1] = run_t;
  }
  __syncthreads();
  if (C > 1) cl.sync();
  uint32_t base_s = 0, base_t = 0;
  if (C > 1) {
#pragma unroll
    for (int r = 0; r < SEL_MAX_CTAS - 1; ++r) {
      const uint2 v = *reinterpret_cast<const uint2*>(cl.map_shared_rank(s_tot, min(r, C - 1)));
      if (r < rank) { base_s += v.x; base_t += v.y; }
    }
  }
  for (int t = t0 + tid; t < t1; t += SEL_THREADS) {
    const uint2 v = before[t];
    const uint32_t ties = base_t + v.y;
    before[t] = make_uint2(base_s + v.x + min(ties, k), ties);
  }
  if (rank == 0 && tid == 0) {
    p.cut[bh] = make_uint4(prefix, k, static_cast<uint32_t>(n), 0u);
    *len = p.budget;  // every CTA of the cluster has read it
  }
  grid_next();
  if (C > 1) cl.sync();  // no CTA leaves while its counts are read
}

// Kernels launched after one another with programmatic dependent launch
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// The kept rows of one buffer into shared memory, U bytes a copy; a row has 2^shift of them, or any
// number (shift < 0).
template <int U>
__device__ __forceinline__ void move_rows(uint32_t dst, const uint8_t* base, int bytes, int shift, const int* src, int kept) {
  const int upr = bytes / U, total = kept * upr;
#pragma unroll 4
  for (int u = threadIdx.x; u < total; u += MOVE_THREADS) {
    const int e = shift >= 0 ? u >> shift : u / upr;
    const uint8_t* from = base + static_cast<int64_t>(src[e]) * bytes + (u - e * upr) * U;
    if constexpr (U == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + u * U), "l"(from) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst + u * U), "l"(from), "n"(U) : "memory");
  }
}

__global__ void __launch_bounds__(MOVE_THREADS) evict_move_kernel(const __grid_constant__ EvictParams p) {
  extern __shared__ __align__(16) uint8_t mv_smem[];  // src[tile] and mass[tile], then the rows of each buffer
  __shared__ int w_tie[MOVE_THREADS / 32], w_keep[MOVE_THREADS / 32], s_tile;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int bh = blockIdx.y, b = bh / p.H, h = bh - b * p.H;
  grid_wait();
  const int n = static_cast<int>(p.cut[bh].z);
  if (n == 0 || static_cast<int>(blockIdx.x) * p.tile >= n) return;
  if (tid == 0) s_tile = static_cast<int>(atomicAdd(&p.cut[bh].w, 1u));
  const uint32_t thr = p.cut[bh].x;
  const int need = static_cast<int>(p.cut[bh].y);
  __syncthreads();
  const int tile = s_tile, i0 = tile * p.tile;
  const uint2 bf = p.before[static_cast<int64_t>(bh) * p.max_tiles + tile];
  const int dst0 = static_cast<int>(bf.x);
  int* src = reinterpret_cast<int*>(mv_smem);
  float* kept_mass = reinterpret_cast<float*>(src + p.tile);
  uint8_t* rows = reinterpret_cast<uint8_t*>(kept_mass + p.tile);
  float* mass = p.mass + b * p.mb + h * p.mh;
  // which entries stay, and where they go (tiles have at most MOVE_THREADS entries)
  const int i = i0 + tid;
  const bool live = tid < p.tile && i < n;
  const float m = live ? mass[i] : 0.f;
  const bool mid = i >= p.first && i < n - p.recent;
  const uint32_t key = mass_key(m), below = (1u << lane) - 1u;
  const bool tie = live && mid && key == thr;
  bool keep = live && (!mid || key > thr);
  const uint32_t tb = __ballot_sync(0xFFFFFFFFu, tie);
  if (lane == 0) w_tie[warp] = __popc(tb);
  __syncthreads();
  int ties = static_cast<int>(bf.y) + __popc(tb & below);
  for (int w = 0; w < warp; ++w) ties += w_tie[w];
  keep = keep || (tie && ties < need);
  const uint32_t kb = __ballot_sync(0xFFFFFFFFu, keep);
  if (lane == 0) w_keep[warp] = __popc(kb);
  __syncthreads();
  int pos = __popc(kb & below), kept = 0;
  for (int w = 0; w < MOVE_THREADS / 32; ++w) {
    if (w < warp) pos += w_keep[w];
    kept += w_keep[w];
  }
  const bool still = dst0 == i0 && kept == min(p.tile, n - i0);  // nothing before or in the tile goes
  if (keep && !still) {
    src[pos] = i;
    kept_mass[pos] = m;
  }
  __syncthreads();
  if (!still && kept) {
    uint8_t* at = rows;
    for (int r = 0; r < p.n_rows; ++r) {
      const uint8_t* base = p.row[r] + b * p.rb[r] + h * p.rh[r];
      const uint32_t dst = smem_u32(at);
      if (p.unit[r] == 16) move_rows<16>(dst, base, p.bytes[r], p.shift[r], src, kept);
      else if (p.unit[r] == 8) move_rows<8>(dst, base, p.bytes[r], p.shift[r], src, kept);
      else move_rows<4>(dst, base, p.bytes[r], p.shift[r], src, kept);
      at += (p.tile * p.bytes[r] + 15) & ~15;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
  __syncthreads();
  uint32_t* loaded = p.loaded + static_cast<int64_t>(bh) * p.max_tiles;
  if (tid == 0) {
    // this tile's rows have been read (the barrier comes after everybody's copies): others may land on them
    asm volatile("st.release.gpu.global.u32 [%0], %1;" ::"l"(loaded + tile), "r"(1u) : "memory");
  }
  if (still || !kept) return;
  if (tid < 2) {  // rows land on one tile, or two
    const int on = (tid == 0 ? dst0 : dst0 + kept - 1) >> p.tile_shift;
    uint32_t v = 1u;
    if (on != tile) {
      const uint64_t began = globaltimer();
      while (true) {
        asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(loaded + on) : "memory");
        if (v) break;
        if (globaltimer() - began > DAB_WAIT_TIMEOUT_NS) {
          atomicCAS(p.err, 0, static_cast<int>(ERR_EVICT_WAIT));
          break;
        }
      }
    }
    w_keep[tid] = static_cast<int>(v);
  }
  __syncthreads();
  if (!w_keep[0] || !w_keep[1]) return;  // timed out: the error word says that the cache is not valid
  uint8_t* at = rows;
  for (int r = 0; r < p.n_rows; ++r) {
    uint8_t* base = p.row[r] + b * p.rb[r] + h * p.rh[r] + static_cast<int64_t>(dst0) * p.bytes[r];
    const int total = kept * p.bytes[r];
    if (p.unit[r] == 16) {
      for (int u = tid * 16; u < total; u += MOVE_THREADS * 16)
        *reinterpret_cast<uint4*>(base + u) = *reinterpret_cast<const uint4*>(at + u);
    } else if (p.unit[r] == 8) {
      for (int u = tid * 8; u < total; u += MOVE_THREADS * 8)
        *reinterpret_cast<uint2*>(base + u) = *reinterpret_cast<const uint2*>(at + u);
    } else {
      for (int u = tid * 4; u < total; u += MOVE_THREADS * 4)
        *reinterpret_cast<uint32_t*>(base + u) = *reinterpret_cast<const uint32_t*>(at + u);
    }
    at += (p.tile * p.bytes[r] + 15) & ~15;
  }
  if (tid < kept) mass[dst0 + tid] = kept_mass[tid];
}

namespace {
int64_t evict_up(int64_t x) { return (x + 255) & ~int64_t{255}; }
}  // namespace

size_t evict_workspace(int64_t B, int64_t H, int64_t cap) {
  const int64_t tiles = (cap + EVICT_MIN_TILE - 1) / EVICT_MIN_TILE;
  return static_cast<size_t>(256 + evict_up(B * H * 16) + evict_up(B * H * tiles * 8) + evict_up(B * H * tiles * 4));
}

cudaError_t launch_evict(EvictParams p, uint8_t* ws, cudaStream_t st) {
  if (p.B * p.H == 0 || p.cap == 0) return cudaSuccess;
  // tiles of up to 128 entries and 80 KB of rows
  int bytes = 0;
  for (int r = 0; r < p.n_rows; ++r) bytes += p.bytes[r];
  p.tile = 128;
  while (p.tile > EVICT_MIN_TILE && p.tile * bytes > 80 * 1024) p.tile >>= 1;
  p.max_tiles = (p.cap + p.tile - 1) / p.tile;
  p.tile_shift = __builtin_ctz(static_cast<unsigned>(p.tile));
  const int64_t heads = static_cast<int64_t>(p.B) * p.H;
  p.err = reinterpret_cast<int*>(ws);
  p.cut = reinterpret_cast<uint4*>(ws + 256);
  p.before = reinterpret_cast<uint2*>(ws + 256 + evict_up(heads * 16));
  p.loaded = reinterpret_cast<uint32_t*>(ws + 256 + evict_up(heads * 16) + evict_up(heads * p.max_tiles * 8));
  // 4096 entries a CTA keep a pass near its latency, as long as all CTAs run at once (one an SM)
  int C = 1;
  while (C < SEL_MAX_CTAS && p.cap > C * 4096 && heads * C * 2 <= 148) C <<= 1;
  int move_smem = p.tile * 8;
  for (int r = 0; r < p.n_rows; ++r) {
    const int upr = p.bytes[r] / p.unit[r];
    p.shift[r] = (upr & (upr - 1)) == 0 ? __builtin_ctz(static_cast<unsigned>(upr)) : -1;
    move_smem += (p.tile * p.bytes[r] + 15) & ~15;
  }
  cudaError_t e = cudaSuccess;
  if (move_smem > 48 * 1024)
    e = cudaFuncSetAttribute(evict_move_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, move_smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(C), static_cast<unsigned>(heads));
  cfg.blockDim = dim3(SEL_THREADS);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = static_cast<unsigned>(C);
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, evict_select_kernel, p);
  if (e != cudaSuccess) return e;
  cfg.gridDim = dim3(static_cast<unsigned>(p.max_tiles), static_cast<unsigned>(heads));
  cfg.blockDim = dim3(MOVE_THREADS);
  cfg.dynamicSmemBytes = static_cast<size_t>(move_smem);
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  return cudaLaunchKernelEx(&cfg, evict_move_kernel, p);
}

}  // namespace dab
