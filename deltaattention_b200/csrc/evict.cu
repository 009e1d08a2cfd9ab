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
//    it writes which entries are kept for sure and which are ties, how many of both come before
//    every tile, and in which tile the entries of every tile of the result begin.
//  * evict_move: one CTA per tile of the result gathers its rows into shared memory, says so, waits
//    for the (at most two) tiles of the result that come from the entries it is about to overwrite
//    to have said so too, and writes. Tiles are handed out in order by a ticket per head, an entry
//    never moves back, and nothing is waited for before a tile's rows have been read: the tiles
//    waited for have smaller tickets, so they are running and never wait for this one. Every kept
//    row is read and written once, with no second buffer. The chain of dependent reads of a tile
//    (ticket, place, entries, rows, flag) takes about 7 us, so what counts is how many kept rows the
//    tiles in an SM's shared memory hold: tiles of the result hold nothing else. 8 heads of 131072
//    16-bit entries cut to half take 93 us, 5.9 TB/s; tiles of the source, half of them evicted, took
//    130 us.
#include <cooperative_groups.h>

#include <atomic>

#include "evict.cuh"

namespace dab {

namespace cg = cooperative_groups;

constexpr int SEL_THREADS = 1024, SEL_MAX_CTAS = 8;  // of a cluster
constexpr int SEL_KEYS = 16;                         // a thread's keys in registers; longer slices are read again
constexpr int SEL_BINS = 2048;
constexpr int SEL_CHUNK = SEL_THREADS * SEL_KEYS;
constexpr int MOVE_THREADS = 256;
constexpr int MOVE_BYTES = 80 * 1024;  // of a tile's rows, where it has more than EVICT_MIN_TILE entries
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
  if (i0 < i1) load(i0);  // a head of fewer tiles than CTAs leaves some without entries
  const bool one = i1 - i0 <= SEL_CHUNK;
  for (int i = tid; i < 3 * SEL_BINS; i += SEL_THREADS) (&hist[0][0])[i] = 0;
  const int out_tiles = (p.budget + p.tile - 1) >> p.tile_shift;
  for (int t = rank * SEL_THREADS + tid; t < out_tiles; t += C * SEL_THREADS)
    p.loaded[static_cast<int64_t>(bh) * p.max_tiles + t] = 0u;
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
      if (lane == 0) {
        cnt[j * (SEL_THREADS / 32) + warp] = __popc(sb) | __popc(tb) << 16;
        if (e < i1) p.words[static_cast<int64_t>(bh) * p.max_words + (e >> 5)] = make_uint2(sb, tb);
      }
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
  uint4* begins = p.begins + static_cast<int64_t>(bh) * p.max_tiles;
  for (int t = t0; t < t1; t += SEL_THREADS) {  // kept and ties before every tile; where result tiles begin
    const int u = t + tid;
    uint2 v = make_uint2(0u, 0u), w = make_uint2(run_s, run_t);
    if (u < t1) v = before[u];
    if (u + 1 < t1) w = before[u + 1];
    __syncthreads();
    if (u < t1) {
      const uint32_t at = base_s + v.x + min(base_t + v.y, k), end = base_s + w.x + min(base_t + w.y, k);
      before[u] = make_uint2(at, base_t + v.y);
      for (uint32_t d = (at + p.tile - 1) >> p.tile_shift; (d << p.tile_shift) < end; ++d)
        begins[d] = make_uint4(u, at, base_t + v.y, 0u);
    }
    __syncthreads();
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
  extern __shared__ __align__(16) uint8_t mv_smem[];  // src[tile], then the rows of mass and each buffer
  __shared__ uint2 wsum[MOVE_THREADS / 32];
  __shared__ int s_tile, s_ok[2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int bh = blockIdx.y, b = bh / p.H, h = bh - b * p.H;
  grid_wait();
  if (tid == 0) s_tile = static_cast<int>(atomicAdd(&p.cut[bh].w, 1u));
  const uint32_t need = p.cut[bh].y;
  const int n = static_cast<int>(p.cut[bh].z);
  __syncthreads();
  if (n == 0) return;  // left alone
  const int tile = s_tile, d0 = tile << p.tile_shift, rows_n = min(p.tile, p.budget - d0);
  const uint2* before = p.before + static_cast<int64_t>(bh) * p.max_tiles;
  const uint4 f = p.begins[static_cast<int64_t>(bh) * p.max_tiles + tile];
  const int from = static_cast<int>(f.x);
  // the tiles of the result that come from the entries this one overwrites: from the `on`th to `upto`
  const int on = static_cast<int>(before[tile].x) >> p.tile_shift;
  const int next = tile + 1 < (n + p.tile - 1) >> p.tile_shift ? static_cast<int>(before[tile + 1].x) : p.budget;
  const int upto = max(static_cast<int>(before[tile].x), next - 1) >> p.tile_shift;
  // the kept entries d0, d0 + 1, .. of the result, from words of 32 source entries
  static_assert(MOVE_THREADS == 256, "eight warps");
  int* src = reinterpret_cast<int*>(mv_smem);
  uint2 at = make_uint2(f.y, f.z);  // kept entries of both kinds before the first word of a round
  const uint2* words = p.words + static_cast<int64_t>(bh) * p.max_words;
  const int nw = (n + 31) / 32;
  int w0 = (from << p.tile_shift) / 32;
  auto word = [&](int i) { return i < nw ? words[i] : make_uint2(0u, 0u); };
  auto sums = [&](uint2 x) {  // up to and with this lane's
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t s = __shfl_up_sync(0xFFFFFFFFu, x.x, o), q = __shfl_up_sync(0xFFFFFFFFu, x.y, o);
      if (lane >= o) { x.x += s; x.y += q; }
    }
    return x;
  };
  // word `base` + lane, with `pre` (surely kept, ties) before it in the round; `mine`: words to write out
  auto place = [&](uint2 w, uint2 pre, int base, uint32_t mine) {
    // of its ties the lowest are kept, as long as fewer than `need` came before
    const uint32_t ties = __popc(w.y), t0 = at.y + pre.y;
    const uint32_t keep = min(t0 + ties, need) - min(t0, need);
    const uint32_t bits = w.x | (keep == ties ? w.y : keep == 0 ? 0u : w.y & ((1u << __fns(w.y, 0, keep + 1)) - 1u));
    const int pos = static_cast<int>(at.x + pre.x + min(t0, need) - min(at.y, need)) - d0;
    uint32_t some = __ballot_sync(0xFFFFFFFFu, bits && pos < rows_n && pos + __popc(bits) > 0);
#pragma unroll 1
    for (some &= mine; some; some &= some - 1) {  // a lane a bit
      const int l = __ffs(some) - 1;
      const uint32_t wb = __shfl_sync(0xFFFFFFFFu, bits, l);
      const int wp = __shfl_sync(0xFFFFFFFFu, pos, l) + __popc(wb & ((1u << lane) - 1u));
      if ((wb >> lane & 1u) && wp >= 0 && wp < rows_n) src[wp] = (base + l) * 32 + lane;
    }
  };
  auto pass = [&](uint2 all) {
    at.x += all.x + min(at.y + all.y, need) - min(at.y, need);
    at.y += all.y;
  };
  auto more = [&] { return static_cast<int>(at.x) < d0 + rows_n && w0 < nw; };
  // Two rounds of 32 words, by every warp alike and without a barrier, are enough where one entry in
  // eight or more is kept; after them 256 words a round.
  uint2 w = word(w0 + lane), ahead = word(w0 + 32 + lane);
#pragma unroll 1
  for (int round = 0; round < 2 && more(); ++round, w0 += 32, w = ahead) {
    const uint2 own = make_uint2(__popc(w.x), __popc(w.y)), x = sums(own);
    place(w, make_uint2(x.x - own.x, x.y - own.y), w0, 0x01010101u << warp);
    pass(make_uint2(__shfl_sync(0xFFFFFFFFu, x.x, 31), __shfl_sync(0xFFFFFFFFu, x.y, 31)));
  }
#pragma unroll 1
  for (; more(); w0 += MOVE_THREADS) {
    w = word(w0 + tid);
    const uint2 own = make_uint2(__popc(w.x), __popc(w.y)), x = sums(own);
    __syncthreads();
    if (lane == 31) wsum[warp] = x;
    __syncthreads();
    uint2 pre = make_uint2(x.x - own.x, x.y - own.y), all = make_uint2(0u, 0u);
#pragma unroll
    for (int v = 0; v < MOVE_THREADS / 32; ++v) {
      const uint2 y = wsum[v];
      if (v < warp) { pre.x += y.x; pre.y += y.y; }
      all.x += y.x;
      all.y += y.y;
    }
    place(w, pre, w0 + warp * 32, 0xFFFFFFFFu);
    pass(all);
  }
  __syncthreads();
  const bool still = src[0] == d0 && src[rows_n - 1] == d0 + rows_n - 1;  // nothing moves
  uint8_t* rows = mv_smem + p.tile * 4;
  if (!still) {
    uint8_t* to = rows;
    for (int r = 0; r < p.n_rows; ++r) {
      const uint8_t* base = p.row[r] + b * p.rb[r] + h * p.rh[r];
      const uint32_t dst = smem_u32(to);
      if (p.unit[r] == 16) move_rows<16>(dst, base, p.bytes[r], p.shift[r], src, rows_n);
      else if (p.unit[r] == 8) move_rows<8>(dst, base, p.bytes[r], p.shift[r], src, rows_n);
      else move_rows<4>(dst, base, p.bytes[r], p.shift[r], src, rows_n);
      to += (p.tile * p.bytes[r] + 15) & ~15;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
  __syncthreads();
  uint32_t* loaded = p.loaded + static_cast<int64_t>(bh) * p.max_tiles;
  if (tid == 0) {
    // this tile's rows have been read (the barrier comes after everybody's copies): others may land on them
    asm volatile("st.release.gpu.global.u32 [%0], %1;" ::"l"(loaded + tile), "r"(1u) : "memory");
  }
  if (still) return;
  if (tid < 2) {
    const int wait = tid == 0 ? on : upto;
    uint32_t v = 1u;
    if (wait != tile) {
      const uint64_t began = globaltimer();
      while (true) {
        asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(loaded + wait) : "memory");
        if (v) break;
        if (globaltimer() - began > DAB_WAIT_TIMEOUT_NS) {
          atomicCAS(p.err, 0, static_cast<int>(ERR_EVICT_WAIT));
          break;
        }
      }
    }
    s_ok[tid] = static_cast<int>(v);
  }
  __syncthreads();
  if (!s_ok[0] || !s_ok[1]) return;  // timed out: the error word says that the cache is not valid
  const uint8_t* out = rows;
  for (int r = 0; r < p.n_rows; ++r) {
    uint8_t* base = p.row[r] + b * p.rb[r] + h * p.rh[r] + static_cast<int64_t>(d0) * p.bytes[r];
    const int total = rows_n * p.bytes[r];
    if (p.unit[r] == 16) {
#pragma unroll 4
      for (int u = tid * 16; u < total; u += MOVE_THREADS * 16)
        *reinterpret_cast<uint4*>(base + u) = *reinterpret_cast<const uint4*>(out + u);
    } else if (p.unit[r] == 8) {
      for (int u = tid * 8; u < total; u += MOVE_THREADS * 8)
        *reinterpret_cast<uint2*>(base + u) = *reinterpret_cast<const uint2*>(out + u);
    } else {
      for (int u = tid * 4; u < total; u += MOVE_THREADS * 4)
        *reinterpret_cast<uint32_t*>(base + u) = *reinterpret_cast<const uint32_t*>(out + u);
    }
    out += (p.tile * p.bytes[r] + 15) & ~15;
  }
}

namespace {
// The kernel's shared-memory limit, raised once per device to the most that any call takes (the
// smallest tile of the widest entries): it is one for all threads of the process.
cudaError_t move_smem_limit() {
  constexpr int MOST = EVICT_MIN_TILE * (4 + EVICT_MAX_BYTES + 4);
  static_assert(MOST >= MOVE_THREADS * 4 + MOVE_BYTES, "larger tiles take no more");
  static std::atomic<uint64_t> set{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = 1ull << (dev & 63);
  if (set.load() & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(evict_move_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MOST);
  if (e == cudaSuccess) set.fetch_or(bit);
  return e;
}
int64_t evict_up(int64_t x) { return (x + 255) & ~int64_t{255}; }
}  // namespace

size_t evict_workspace(int64_t B, int64_t H, int64_t cap) {
  const int64_t tiles = (cap + EVICT_MIN_TILE - 1) / EVICT_MIN_TILE, heads = B * H;
  return static_cast<size_t>(256 + evict_up(heads * 16) + evict_up(heads * tiles * 8) + evict_up(heads * tiles * 4) +
                             evict_up(heads * tiles * 16) +
                             evict_up(heads * ((cap + 31) / 32) * 8));
}

cudaError_t launch_evict(EvictParams p, uint8_t* ws, cudaStream_t st) {
  if (p.B * p.H == 0 || p.cap == 0) return cudaSuccess;
  // tiles of up to 256 entries and MOVE_BYTES of rows
  int bytes = 0;
  for (int r = 0; r < p.n_rows; ++r) bytes += p.bytes[r];
  p.tile = MOVE_THREADS;
  while (p.tile > EVICT_MIN_TILE && p.tile * bytes > MOVE_BYTES) p.tile >>= 1;
  p.tile_shift = __builtin_ctz(static_cast<unsigned>(p.tile));
  p.max_tiles = (p.cap + p.tile - 1) / p.tile;
  p.max_words = (p.cap + 31) / 32;
  const int64_t heads = static_cast<int64_t>(p.B) * p.H;
  uint8_t* at = ws + 256;
  auto take = [&](int64_t n) {
    uint8_t* x = at;
    at += evict_up(n);
    return x;
  };
  p.err = reinterpret_cast<int*>(ws);
  p.cut = reinterpret_cast<uint4*>(take(heads * 16));
  p.before = reinterpret_cast<uint2*>(take(heads * p.max_tiles * 8));
  p.loaded = reinterpret_cast<uint32_t*>(take(heads * p.max_tiles * 4));
  p.begins = reinterpret_cast<uint4*>(take(heads * p.max_tiles * 16));
  p.words = reinterpret_cast<uint2*>(take(heads * p.max_words * 8));
  // 4096 entries a CTA keep a pass near its latency, as long as all CTAs run at once (one an SM)
  int C = 1;
  while (C < SEL_MAX_CTAS && p.cap > C * 4096 && heads * C * 2 <= 148) C <<= 1;
  int move_smem = p.tile * 4;
  for (int r = 0; r < p.n_rows; ++r) {
    const int upr = p.bytes[r] / p.unit[r];
    p.shift[r] = (upr & (upr - 1)) == 0 ? __builtin_ctz(static_cast<unsigned>(upr)) : -1;
    move_smem += (p.tile * p.bytes[r] + 15) & ~15;
  }
  cudaError_t e = move_smem_limit();
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(C), static_cast<unsigned>(heads));
  cfg.blockDim = dim3(SEL_THREADS);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(C);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, evict_select_kernel, p);
  if (e != cudaSuccess) return e;
  cfg.gridDim = dim3(static_cast<unsigned>((p.budget + p.tile - 1) / p.tile), static_cast<unsigned>(heads));
  cfg.blockDim = dim3(MOVE_THREADS);
  cfg.dynamicSmemBytes = static_cast<size_t>(move_smem);
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  return cudaLaunchKernelEx(&cfg, evict_move_kernel, p);
}

}  // namespace dab
