// Attention of packed prompts, of prompts over a paged cache, and of one token per sequence over it, on
// tcgen05 tensor cores.
//
//   out_i = sum_{j < limit_i} softmax_j(scale q_i . k_j) v_j,
// limit_i = the query's position + 1 (causal) or the sequence's length; q-head h reads K / V head h / G.
//
// Rows of a 128-row query tile are (token, q-head of one K / V head) pairs, 128 / G tokens by G heads, so
// that every K / V head's rows are loaded once for all of its q-heads. A unit is two such tiles over the
// same keys, a piece a range of a unit's 128-key tiles. Three kinds of units:
//   prompts   2 * (128 / G) consecutive tokens of a sequence; causal tiles end at their last row's limit;
//   prefixes  as many sequences of a group that shares its first pages, one token each: these pages are
//             read once for all of them;
//   own       one token of one sequence over the rows behind its prefix: G rows. Bytes bound it. Up to 8 rows are
//             computed transposed (thin): S^T = K Q^T has a key per row and 8 columns, which takes a warp a tenth
//             of the time of 128 columns; the two tiles take every other key tile, two chains at a time.
// A decode step's prefixes are cut into even ranges of cost, one for each of the first CTAs, its own units into ranges for
// the others, so that a CTA's pieces are all of one kind: thin ones or pairs. Prompts take pieces
// from a counter, heavy ones first; where whole units would leave SMs idle they are cut into chunks of key tiles, the
// units of one chunk next to each other so that they find its keys in L2. Pieces of cut units leave fp32
// partial sums with their maxima, joined by a second kernel that is launched early (programmatic dependent launch).
//
// One persistent CTA per SM, 384 threads: warp 0 fetches pieces, publishes them to all other warps and
// loads Q and K; warp 3 loads V; warps 1 and 2 issue the products of the two tiles; warps 4-7 and 8-11 are
// the tiles' softmax, a row per thread. The loads are TMA boxes of a page (or of 128 packed rows), scores
// and weights live in TMEM, weights in the rows' 16-bit type: an error of half a step per weight, as large as
// that of the rounded output. The running maximum moves only when a row outgrows it by 2^8.
//
// Measured (device time, 32 q-heads on 8 K / V heads of 128, bf16; floors at 6550 GB/s and 1680 TFLOP/s):
//   prompt of 32768 tokens            7.8 ms, 1120 TFLOP/s (floor 5.24): a pair of tiles over 128 keys takes 3300 cycles at
//     the 1.5 GHz that the power limit leaves. Its products take 2050 of the tensor pipe (64 each, measured alone) and its
//     exponentials 2050 of their units, but neither is what it waits for: that is each tile's chain of scores, softmax (1700
//     cycles), P V of the last 64 keys and two hand-overs; two chains alternate. Tried: one area of scores for both tiles and
//     one of weights for each, so that scores are computed a tile ahead (the softmax then holds 128 scores in registers and
//     takes 2700: 18 % slower); a tile scored in two halves (13 %; products of N = 64 take 60 cycles); exponentials in part
//     as polynomials (4 %); turns of the products' warps that end before the scores (9 %) or none (12 %); one election for
//     a batch of products (no gain); a single lane for the products' role (12 %)
//   16 sequences of 32000 rows        310 us, 6.8 TB/s (floor 320); 48 of 500 to 12000: 200 us (floor 185)
//   64 sequences, 32000 rows shared and up to 1000 own: 85 us (floor 40). Neither bytes (38 % of nominal) nor products (19 %)
//     fill it: the prefix's CTAs are bound by the chain above, and the join ends 8 us after the last piece
//   1 sequence of 1900 rows (d 64)    17 us: two launches, each a chain of reads, code that is fetched, one key tile
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "paged.cuh"

namespace dab {

constexpr int PT_THREADS = 384;
constexpr int PT_BN = 128;   // keys of a tile
constexpr int PT_RING = 4;   // pieces published ahead
constexpr int PT_ROWS = 256; // partial rows between the pieces of neighbouring CTAs
constexpr int PT_THIN = 8;   // most rows of a thin piece (its products are computed for 16)
constexpr int PT_CHUNKS = 16;   // most chunks that a prompt's mean unit is cut into, of PT_MIN_CHUNK key tiles at least
constexpr int PT_MIN_CHUNK = 2;
constexpr int PT_FILL = 7;      // most chunks per SM: they bound the workspace
constexpr int PT_PIECE = 5;     // what beginning and ending a piece costs, in key tiles of a pair
constexpr int PT_JOIN = 3;      // and the joining kernel, with 3 / 100 for every piece

// A CTA's part of a decode step: costs [begin, end), its place among the CTAs in their order, its first item and what
// lies before that. Of prompts only `item` is used, the key tiles of a chunk.
struct Range {
  int64_t begin, end, base_t, base_r;
  int place, item;
};

struct Piece {
  int end;         // no more pieces
  int tok0, ntok;  // first token, tokens
  int h;           // K / V head
  int trow;        // row of the page table; first row of the sequence for packed rows
  int kb;          // first key of key tile 0
  int kend;        // keys that exist: rows from here on are not read
  int j0, nt0, nt1;  // key tiles: from j0 up to nt0 for tile 0, nt1 for tile 1
  int thin;        // at most PT_THIN rows: both tiles hold them and take every other key tile (by the parity of its
                   // fill), and scores and output are computed transposed
  int lim0, lim_step;  // keys that token tok0 + i sees: lim0 + i * lim_step ..
  int by_length;   // .. and no more than the token's sequence has
  int before;      // prompts: tokens at negative positions, which see nothing
  int split;       // partial results to rows orow0 / orow1 (thin: orow0), else the output
  int q1;          // one token: the query box of one token
  int64_t orow0, orow1;
  __device__ __forceinline__ int jend() const { return max(nt0, nt1); }
  // query tiles it needs: tiles that hold the same rows share one
  __device__ __forceinline__ int q_tiles(int tpt) const { return !thin && ntok > tpt ? 2 : 1; }
};

template <int D> struct PtCfg {
  static constexpr int QBYTES = 128 * D * 2;
  static constexpr int KVBYTES = PT_BN * D * 2;
  static constexpr int NK = (D == 128) ? 2 : 4;
  static constexpr int NV = (D == 128) ? 2 : 4;
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_K = 2 * QBYTES;
  static constexpr int OFF_V = OFF_K + NK * KVBYTES;
  static constexpr int EPI_PITCH = 80;  // 64 bytes of a row's output and 16 more against bank conflicts
  static constexpr int OFF_EPI = OFF_V + NV * KVBYTES;
  // weights of thin pieces, [2][16 rows x 128 keys], rows from PT_THIN on unused
  static constexpr int OFF_P = OFF_EPI + 8 * 32 * EPI_PITCH;
  static constexpr int PBYTES = 16 * PT_BN * 2;
  static constexpr int OFF_VOTE = OFF_P + 2 * PBYTES;  // [2 tiles][2][4 warps][PT_THIN] maxima, then flags
  static constexpr int OFF_X = OFF_VOTE + 2 * 2 * 4 * (PT_THIN + 1) * 4;  // thin: tile 1's O^T, maxima and sums
  static constexpr int OFF_PIECE = OFF_X + PT_THIN * (D + 2) * 4;
  static constexpr int OFF_BAR = OFF_PIECE + PT_RING * static_cast<int>(sizeof(Piece));
  static constexpr int NBAR = 4 + 2 * NK + 2 * NV + 2 * PT_RING + 2 * 6 + 1 + 2 + 2;
  static constexpr int OFF_MISC = OFF_BAR + NBAR * 8;
  static constexpr int SMEM = OFF_MISC + 256 + 1024;  // and slack for alignment
};

// ------------------------------------------------------------------------------------ the work
__device__ __forceinline__ int64_t shfl64(int64_t v, int src) { return __shfl_sync(0xFFFFFFFFu, v, src); }

// a / b of non-negative numbers, mostly below 2^32
__device__ __noinline__ int64_t quotient(int64_t a, int64_t b) {
  if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
  return a / b;
}

// Whether the groups of sequences rise inside the batch; the whole block calls it.
__device__ __forceinline__ bool groups_ok(const PagedAttn& p) {
  if (!p.groups) return true;
  bool bad = false;
  for (int g = threadIdx.x; g < p.groups; g += blockDim.x)
    bad |= p.prefix_cu[g + 1] < p.prefix_cu[g] || p.prefix_cu[g] < 0 || p.prefix_cu[g + 1] > p.B;
  const bool any = __syncthreads_or(bad);
  if (any && threadIdx.x == 0) paged_error(p.err, ERR_STARTS);
  return !any;
}

// Rows of group g's prefix that are read for all: whole pages.
__device__ __forceinline__ int prefix_rows(const PagedAttn& p, int g) {
  const int64_t most = static_cast<int64_t>(p.max_pages) << p.ps_shift;
  const int n = static_cast<int>(min(static_cast<int64_t>(max(p.prefix_len[g], 0)), most));
  return n >> p.ps_shift << p.ps_shift;
}
// The group of sequence b, or -1.
__device__ __forceinline__ int group_of(const PagedAttn& p, int groups, int b) {
  if (!groups || b < p.prefix_cu[0] || b >= p.prefix_cu[groups]) return -1;
  int lo = 0, hi = groups;  // cu[lo] <= b < cu[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (p.prefix_cu[mid] <= b) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Items of a decode step: the groups, then the sequences. Every item has `units` units for each K / V head, of
// `tiles` key tiles each, and `rows` partial rows for each head.
struct Item {
  int first, count;  // sequences
  int start, len;    // rows [start, len) of the sequences
  int tiles, units, rows, thin;
  // what a unit and the item cost: a start for each unit, and its key tiles
  __device__ __forceinline__ int tile_cost(const PagedAttn& p) const { return thin ? p.w_thin : p.w_pair; }
  __device__ __forceinline__ int64_t unit_cost(const PagedAttn& p) const {
    return tiles ? p.w_start + static_cast<int64_t>(tiles) * tile_cost(p) : 0;
  }
  __device__ __forceinline__ int64_t cost(const PagedAttn& p) const { return static_cast<int64_t>(p.H) * units * unit_cost(p); }
};
// The CTAs of a decode step: the first n[0] share the prefixes' costs, n[1] after them the own rows'. In each part the
// dearest key tile at least for every CTA, so that one whose range lies inside a unit has one of its tiles. The first
// part is even: products bound the prefixes of many sequences and bytes the own rows, and two neighbouring CTAs
// (two SMs that share a path to memory) that do one each both run at a third of their speed. 64 sequences over 32000
// shared rows: 155 us where all neighbours were mixed, 120 us where one pair was, 95 us without.
__device__ __forceinline__ Ctas decode_ctas(const PagedAttn& p, int64_t prefixes, int64_t total) {
  Ctas c;
  c.cost[0] = prefixes;
  c.cost[1] = total - prefixes;
  int first = 0;
  if (prefixes) {
    first = static_cast<int>(quotient((prefixes + 1) / 2 * p.num_ctas, (total + 1) / 2));
    first = (first + 1) & ~1;
    if (c.cost[1]) first = min(max(first, 2), p.num_ctas - 2);
    first = min(first, p.num_ctas);
  }
  c.from[0] = 0;
  c.from[1] = first;
  const int64_t w = max(p.w_thin, p.w_pair);
  for (int k = 0; k < 2; ++k) {
    const int most = k ? p.num_ctas - first : first;
    c.n[k] = c.cost[k] ? static_cast<int>(min(max(quotient(c.cost[k], w), int64_t{1}), static_cast<int64_t>(most))) : 0;
  }
  return c;
}
// (Not inlined, like prompt_seq: a launch's first pass through code waits for instructions, and the copies of
// these on the way to the first load cost more than the calls.)
__device__ __noinline__ Item decode_item(const PagedAttn& p, int groups, int tpt, int i) {
  Item it;
  if (i < groups) {
    it.first = p.prefix_cu[i];
    it.count = p.prefix_cu[i + 1] - it.first;
    it.start = 0;
    it.len = it.count ? prefix_rows(p, i) : 0;
    it.units = (it.count + 2 * tpt - 1) / (2 * tpt);
    it.thin = 0;
  } else {
    const int b = i - groups;
    const int g = group_of(p, groups, b);
    it.first = b;
    it.count = 1;
    it.len = paged_length(p.lengths[b], p.max_pages, p.ps_shift, p.err);
    it.start = g < 0 ? 0 : min(prefix_rows(p, g), it.len);
    it.units = 1;
    it.thin = p.G <= PT_THIN;
  }
  it.tiles = (it.len - it.start + PT_BN - 1) / PT_BN;
  it.rows = it.count * p.G;
  return it;
}

// Exclusive sums over the block's threads of two numbers; returns the totals.
__device__ __noinline__ void block_scan2(int64_t& a, int64_t& b, int64_t* smem, int64_t& ta, int64_t& tb) {
  const int lane = lane_id(), warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  int64_t sa = a, sb = b;
#pragma unroll 1
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t ua = __shfl_up_sync(0xFFFFFFFFu, sa, o), ub = __shfl_up_sync(0xFFFFFFFFu, sb, o);
    if (lane >= o) {
      sa += ua;
      sb += ub;
    }
  }
  if (lane == 31) {
    smem[warp] = sa;
    smem[nw + warp] = sb;
  }
  __syncthreads();
  int64_t pa = 0, pb = 0;
  ta = tb = 0;
#pragma unroll 1
  for (int w = 0; w < nw; ++w) {
    if (w == warp) {
      pa = ta;
      pb = tb;
    }
    ta += smem[w];
    tb += smem[nw + w];
  }
  __syncthreads();
  a = pa + sa - a;
  b = pb + sb - b;
}

// A prompt's sequence: queries [c0, c1), `len` keys, `nq` units of 2 * tpt tokens and `mt` key tiles.
struct Seq {
  int c0, n, len, nq, mt;
  bool falls;  // its start lies behind its end
};
__device__ __noinline__ Seq prompt_seq(const PagedAttn& p, int utok, int b) {
  Seq s;
  int c1;
  s.falls = paged_tokens(p.cu, b, p.T, p.err, s.c0, c1);
  s.n = c1 - s.c0;
  s.len = s.n == 0 ? 0 : p.table ? paged_length(p.lengths[b], p.max_pages, p.ps_shift, p.err) : s.n;
  s.nq = (s.n + utok - 1) / utok;
  s.mt = max(1, (s.len + PT_BN - 1) / PT_BN);
  return s;
}
// Key tiles of a chunk, or 0 where units stay whole: of the ways to cut the mean unit into 1 to 16 chunks, the one
// with the least rounds of pieces times their length, joining counted.
__device__ __forceinline__ int chunk_tiles(const PagedAttn& p, int64_t units, int64_t tiles) {
  if (!p.may_split || units == 0 || units >= 2 * static_cast<int64_t>(p.num_ctas)) return 0;
  const unsigned n = static_cast<unsigned>(units), mean = static_cast<unsigned>(quotient(tiles + units - 1, units));
  const unsigned ctas = static_cast<unsigned>(p.num_ctas);
  unsigned best = 0, least = 0xFFFFFFFFu;
#pragma unroll 1
  for (unsigned k = 1; k <= PT_CHUNKS && (k == 1 || (mean >= PT_MIN_CHUNK * k && n * k <= PT_FILL * ctas)); ++k) {
    const unsigned len = (mean + k - 1) / k;
    const unsigned cost = (n * k + ctas - 1) / ctas * (len + PT_PIECE) + (k > 1 ? PT_JOIN + n * k * 3 / 100 : 0);
    if (cost < least) {
      least = cost;
      best = k == 1 ? 0 : len;
    }
  }
  return static_cast<int>(best);
}
__device__ __forceinline__ int64_t prompt_pieces(const PagedAttn& p, const Seq& s, int chunk) {
  return static_cast<int64_t>(p.H) * s.nq * (chunk ? (s.mt + chunk - 1) / chunk : 1);
}

// every lane of the warp waits; the outcome is warp-uniform
__device__ __forceinline__ bool pt_wait(uint64_t* bar, uint32_t par, const Abort& ab, int code) {
  const bool ok = mbar_wait(bar, par, ab, code);
  return __all_sync(0xFFFFFFFFu, ok);
}
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// ------------------------------------------------------------------------------------ pieces
// The pieces of one CTA, in order. All lanes of warp 0 call it and hold an item (a group or sequence of a decode step,
// a prompt's sequence) each; the lane whose item is next works the piece out and writes it to `to`.
// (Code that is rarely run waits for its instructions each time, so there is little of it.)
template <bool DEC> struct Sched {
  int64_t pos, end;             // decode: the range of costs left
  int i0, n;                    // items i0 .. i0 + 31 of n are in the lanes
  int64_t base_t, base_r;       // costs (pieces) and partial rows before item i0
  int64_t before_t, inc_t, before_r, inc_r;  // the lane's item: sums of costs and rows before and with it
  typename std::conditional<DEC, Item, Seq>::type item;
  int groups, tpt, chunk;
  int place;                    // decode: of the CTA's range in the order of costs
  bool loaded;

  __device__ __forceinline__ void load(const PagedAttn& p) {
    // lanes past the last item look at it too: a warp that runs apart is slow from here on
    const bool has = i0 + lane_id() < n;
    const int i = min(i0 + lane_id(), n - 1);
    int64_t t, r = 0;
    if constexpr (DEC) {
      item = decode_item(p, groups, tpt, i);
      t = item.cost(p);
      r = static_cast<int64_t>(p.H) * item.rows;
    } else {
      item = prompt_seq(p, 2 * tpt, i);
      t = prompt_pieces(p, item, chunk);
    }
    inc_t = has ? t : 0;
    inc_r = has ? r : 0;
    before_t = inc_t;
    before_r = inc_r;
#pragma unroll 1
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t a = __shfl_up_sync(0xFFFFFFFFu, inc_t, o), b = DEC ? __shfl_up_sync(0xFFFFFFFFu, inc_r, o) : 0;
      if (lane_id() >= o) {
        inc_t += a;
        inc_r += b;
      }
    }
    before_t = inc_t - before_t;
    before_r = inc_r - before_r;
  }
  // the lane whose item has place `at`; -1 past the last item
  __device__ __forceinline__ int find(const PagedAttn& p, int64_t at) {
    while (true) {
      if (!loaded) {
        if (i0 >= n) return -1;
        load(p);
        loaded = true;
      }
      const int64_t past = base_t + shfl64(inc_t, 31);
      if (at < past) break;
      base_t = past;
      if (DEC) base_r += shfl64(inc_r, 31);
      i0 += 32;
      loaded = false;
    }
    return __ffs(__ballot_sync(0xFFFFFFFFu, at < base_t + inc_t)) - 1;
  }

  __device__ __forceinline__ void next(const PagedAttn& p, Piece* to) {
    const int lane = lane_id();
    Piece pc;
    int src = -1;
    bool shared = false;
    while (true) {
      if constexpr (DEC) {
        src = pos < end ? find(p, pos) : -1;
        if (src < 0) break;
        const int w = item.tile_cost(p), each = static_cast<int>(max(item.unit_cost(p), int64_t{1}));
        const int64_t off = max(pos - base_t - before_t, int64_t{0});
        const int64_t u = quotient(off, each);
        // the place within the unit, and where the range ends in it; tile t begins at w_start + t * w
        const int at = static_cast<int>(off - u * each);
        const int stop = static_cast<int>(min(static_cast<int64_t>(each), at + end - pos));
        pc.j0 = (max(at - p.w_start, 0) + w - 1) / w;
        pc.nt0 = min((max(stop - p.w_start, 0) + w - 1) / w, item.tiles);
        const bool any = __shfl_sync(0xFFFFFFFFu, pc.j0 < pc.nt0, src);
        pos += __shfl_sync(0xFFFFFFFFu, stop - at, src);
        if (!any) continue;
        const int h = static_cast<int>(u) / max(item.units, 1), up = static_cast<int>(u) - h * item.units;
        shared = i0 + src < groups;
        pc.h = h;
        pc.tok0 = item.first + up * 2 * tpt;
        pc.ntok = min(2 * tpt, item.count - up * 2 * tpt);
        pc.kb = item.start;
        pc.kend = item.len;
        pc.trow = item.first;
        pc.q1 = !shared;
        pc.thin = item.thin;
        pc.nt1 = item.thin || pc.ntok > tpt ? pc.nt0 : 0;
        pc.lim0 = item.len;
        pc.lim_step = 0;
        pc.by_length = shared;
        pc.before = 0;
        pc.split = 1;
        pc.orow0 = base_r + before_r + static_cast<int64_t>(h) * item.rows + static_cast<int64_t>(up) * 2 * tpt * p.G +
                   static_cast<int64_t>(place) * PT_ROWS;
        pc.orow1 = pc.orow0 + tpt * p.G;
        break;
      } else {
        unsigned id = 0;
        if (lane == 0) id = atomicAdd(p.counter, 1u);
        __syncwarp();
        id = __shfl_sync(0xFFFFFFFFu, id, 0);
        src = find(p, id);
        if (src < 0) break;
        const int64_t off = max(static_cast<int64_t>(id) - base_t - before_t, int64_t{0});
        const int nq = max(item.nq, 1), utok = 2 * tpt;
        const int nch = chunk ? (item.mt + chunk - 1) / chunk : 1;
        // whole units: the heads of one place next to each other; cut ones: the places of one chunk
        const int inner = nch == 1 ? p.H : nq;
        const int64_t outer = quotient(off, inner);
        const int in = static_cast<int>(off - outer * inner);
        int place = static_cast<int>(outer), ch = 0;
        pc.h = in;
        if (nch > 1) {
          place = in;
          pc.h = static_cast<int>(outer) / nch;
          ch = static_cast<int>(outer) - pc.h * nch;
        }
        const int q = nq - 1 - place;  // later tokens, which see more, first
        pc.tok0 = item.c0 + q * utok;
        pc.ntok = min(utok, item.n - q * utok);
        const int pos0 = item.len - item.n + q * utok;  // position of the first token
        const int l0 = p.causal ? pos0 + min(tpt, pc.ntok) : item.len;
        const int l1 = pc.ntok <= tpt ? 0 : p.causal ? pos0 + pc.ntok : item.len;
        pc.nt0 = (max(l0, 0) + PT_BN - 1) / PT_BN;
        pc.nt1 = (max(l1, 0) + PT_BN - 1) / PT_BN;
        pc.j0 = ch * chunk;
        const bool none = ch > 0 && max(pc.nt0, pc.nt1) <= pc.j0;  // nothing to see in this chunk
        if (__shfl_sync(0xFFFFFFFFu, none, src)) continue;
        if (nch > 1) {
          pc.nt0 = min(pc.nt0, pc.j0 + chunk);
          pc.nt1 = min(pc.nt1, pc.j0 + chunk);
        }
        pc.kb = 0;
        pc.kend = item.len;
        pc.trow = p.table ? i0 + lane : item.c0;
        pc.q1 = pc.thin = pc.by_length = 0;
        pc.lim0 = p.causal ? pos0 + 1 : item.len;
        pc.lim_step = p.causal ? 1 : 0;
        pc.before = max(-pos0, 0);
        pc.split = nch > 1;
        pc.orow0 = static_cast<int64_t>(id) * PT_ROWS;
        pc.orow1 = pc.orow0 + 128;
        break;
      }
    }
    if constexpr (DEC) if (shared) {
      // the prefix is read through the first member that has all of it, or else through a longest one
      const int first = __shfl_sync(0xFFFFFFFFu, item.first, src), count = __shfl_sync(0xFFFFFFFFu, item.count, src);
      const int len = __shfl_sync(0xFFFFFFFFu, item.len, src);
      int best = 0, best_len = 0;
      for (int m0 = 0; m0 < count && best_len < len; m0 += 32) {
        const int l = m0 + lane < count ? min(p.lengths[first + m0 + lane], len) : 0;
        const int most = __reduce_max_sync(0xFFFFFFFFu, l);
        if (most > best_len) {
          best_len = most;
          best = m0 + __ffs(__ballot_sync(0xFFFFFFFFu, l == most)) - 1;
        }
      }
      pc.trow = first + best;
      pc.kend = pc.lim0 = best_len;
    }
    pc.end = src < 0;
    if (src < 0 ? lane == 0 : lane == src) *to = pc;
    __syncwarp();
  }
};

// One key tile by the calling warp: lanes look pages up a batch of tiles ahead and load their own.
struct TileLoader {
  int npt, box;          // pages of a tile, rows of a box
  int batch, page, ahead;  // the batch whose pages the lanes hold, and the next one's
  __device__ __forceinline__ void init(const PagedAttn& p) {
    box = min(1 << p.ps_shift, PT_BN);
    npt = PT_BN / box;
    batch = -1;
    page = ahead = 0;
  }
  __device__ __forceinline__ int batch_of(int j) const { return j / (32 / npt); }
  __device__ __forceinline__ int look(const PagedAttn& p, const Piece& pc, int bt) {
    const int key = pc.kb + bt * 32 * box + lane_id() * box;
    if (key >= pc.kend) return 0;
    const int pg = __ldg(p.table + pc.trow * p.table_stride + (key >> p.ps_shift));
    if (pg >= 0 && pg < p.num_pages) return pg;
    paged_error(p.err, ERR_PAGE);
    return p.num_pages;  // past the map: zeros
  }
  __device__ __forceinline__ void load(const PagedAttn& p, const Piece& pc, const CUtensorMap* map, int j, int D,
                                       uint8_t* dst, uint64_t* bar) {
    const int lane = lane_id();
    if (!p.table) {
      if (lane == 0) {
        mbar_arrive_expect_tx(bar, PT_BN * D * 2);
        for (int x = 0; x < D / 64; ++x)
          tma_load_4d(dst + x * (PT_BN * 128), map, bar, x * 64, pc.trow + j * PT_BN, pc.h, 0);
      }
      return;
    }
    const int per = 32 / npt;  // tiles of a batch
    const int bt = j / per;
    if (bt != batch) {
      page = batch >= 0 && bt == batch + 1 ? ahead : look(p, pc, bt);
      ahead = look(p, pc, bt + 1);
      batch = bt;
    }
    const int i = lane - (j - bt * per) * npt;  // the lane's page of this tile
    const int key = pc.kb + j * PT_BN + i * box;
    const bool mine = i >= 0 && i < npt && key < pc.kend;
    const int n = __popc(__ballot_sync(0xFFFFFFFFu, mine));
    if (lane == 0) mbar_arrive_expect_tx(bar, n * box * D * 2);
    __syncwarp();
    if (mine) {
      const int row = key & ((1 << p.ps_shift) - 1);
      for (int x = 0; x < D / 64; ++x)
        tma_load_4d(dst + x * (PT_BN * 128) + i * box * 128, map, bar, x * 64, row, pc.h, page);
    }
    __syncwarp();
  }
};

// ------------------------------------------------------------------------------------ the kernel
template <int D, bool BF16, bool DEC>
__global__ void __launch_bounds__(PT_THREADS, 1) paged_attn_kernel(const __grid_constant__ PagedAttn p) {
  using C = PtCfg<D>;
  constexpr int NK = C::NK, NV = C::NV;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t* q_full = bars;              // [2] a tile of queries each
  uint64_t* q_empty = bars + 2;         // [2]
  uint64_t* k_full = bars + 4;          // [NK]
  uint64_t* k_empty = k_full + NK;      // [NK]
  uint64_t* v_full = k_empty + NK;      // [NV]
  uint64_t* v_empty = v_full + NV;      // [NV]
  uint64_t* w_full = v_empty + NV;      // [PT_RING] a piece is published
  uint64_t* w_empty = w_full + PT_RING; // [PT_RING] and has been read by all
  uint64_t* s_full = w_empty + PT_RING; // [2]
  uint64_t* p_lo = s_full + 2;          // [2] weights of keys 0..63 stored
  uint64_t* p_full = p_lo + 2;          // [2] all weights stored
  uint64_t* o_full = p_full + 2;        // [2]
  uint64_t* tile_free = o_full + 2;     // [2]
  uint64_t* vote = tile_free + 2;       // [2] thin pieces: the tile's warps have looked at their scores
  uint64_t* mma_done = vote + 2;
  uint64_t* turn = mma_done + 1;        // [2]
  uint64_t* xfer = turn + 2;            // [2] thin: tile 1's result is there, and has been read
  Piece* pieces = reinterpret_cast<Piece*>(smem + C::OFF_PIECE);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::OFF_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::OFF_MISC + 8);
  Range* range = reinterpret_cast<Range*>(smem + C::OFF_MISC + 16);
  int64_t* scan = reinterpret_cast<int64_t*>(smem + C::OFF_EPI);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < NK; ++s) {
      mbar_init(k_full + s, 1);
      mbar_init(k_empty + s, 2);
    }
    for (int s = 0; s < NV; ++s) {
      mbar_init(v_full + s, 1);
      mbar_init(v_empty + s, 2);
    }
    for (int s = 0; s < PT_RING; ++s) {
      mbar_init(w_full + s, 1);
      mbar_init(w_empty + s, 11);
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(q_full + x, 1);
      mbar_init(q_empty + x, 2);
      mbar_init(s_full + x, 1);
      mbar_init(p_lo + x, 4);
      mbar_init(p_full + x, 4);
      mbar_init(o_full + x, 1);
      mbar_init(tile_free + x, 4);
      mbar_init(vote + x, 4);
      mbar_init(turn + x, 1);
      mbar_init(xfer + x, 4);
    }
    mbar_init(mma_done, 2);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 3 && lane == 0) {
    tma_prefetch_desc(&p.tm_q);
    tma_prefetch_desc(&p.tm_q1);
    tma_prefetch_desc(&p.tm_k);
    tma_prefetch_desc(&p.tm_v);
  }
  if (warp == 2) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  // ---------------------------------------------------------------- where this CTA's work begins
  const int tpt = 128 / p.G;
  int groups = 0;
  if constexpr (DEC) groups = groups_ok(p) ? p.groups : 0;
  const int n = DEC ? groups + p.B : p.B;
  // Where a start falls sequences overlap, and there may be more units than the scratch was made for: there are none then.
  bool rising = true;
  if (!DEC && !p.may_split) {
    bool bad = false;
    for (int b = threadIdx.x; b < p.B; b += PT_THREADS) bad |= p.cu[b + 1] < p.cu[b];
    rising = !__syncthreads_or(bad);
    if (!rising && threadIdx.x == 0) paged_error(p.err, ERR_STARTS);
  }
  if (DEC || p.may_split) {
    // `per` items in a row for every thread; all threads take all turns, since a warp that parts here
    // does not come together again, and runs apart through everything below
    const int per = (n + PT_THREADS - 1) / PT_THREADS;
    const int first = static_cast<int>(threadIdx.x) * per;
    int64_t c = 0, r = 0, tc, tr;
    bool bad = false;
    Item it;
#pragma unroll 1
    for (int k = 0; k < per; ++k) {
      const int i = min(first + k, n - 1);
      const bool has = first + k < n;
      if constexpr (DEC) {
        it = decode_item(p, groups, tpt, i);
        c += has ? it.cost(p) : 0;
        r += has ? static_cast<int64_t>(p.H) * it.rows : 0;
      } else {
        const Seq s = prompt_seq(p, 2 * tpt, i);
        bad |= s.falls;
        c += has ? static_cast<int64_t>(p.H) * s.nq * s.mt : 0;
        r += has ? static_cast<int64_t>(p.H) * s.nq : 0;
      }
    }
    block_scan2(c, r, scan, tc, tr);
    if constexpr (DEC) {
      int64_t prefixes = 0;
      if (groups) {
        // the prefixes' costs end where the first sequence's begin
        int64_t at = c;
#pragma unroll 1
        for (int k = 0; k < per; ++k) {
          if (per > 1) it = decode_item(p, groups, tpt, min(first + k, n - 1));
          if (first + k == groups) range->base_t = at;
          at += it.cost(p);
        }
        __syncthreads();
        prefixes = range->base_t;
        __syncthreads();
      }
      const Ctas ct = decode_ctas(p, prefixes, tc);
      const int bid = static_cast<int>(blockIdx.x), list = bid >= ct.from[1], nc = list ? ct.n[1] : ct.n[0];
      int at = bid - (list ? ct.from[1] : 0);
      int64_t pos = 0, pos_end = 0;
      if (at < nc) {
        // neighbours on the chip take ranges far from each other (64 sequences of 1000 rows: 69 -> 65 us)
        at = at & 1 ? (nc + 1) / 2 + at / 2 : at / 2;
        const int64_t total = list ? ct.cost[1] : prefixes, from = list ? prefixes : 0;
        pos = from + quotient(total * at, nc);
        pos_end = from + quotient(total * (at + 1), nc);
      }
      if (threadIdx.x == 0) {
        range->begin = pos;
        range->end = pos_end;
        range->place = at + (list ? ct.from[1] : 0);
        if (bid == 0) *p.rec_ctas = ct;
      }
#pragma unroll 1
      for (int k = 0; k < per; ++k) {
        const int i = min(first + k, n - 1);
        const bool has = first + k < n;
        if (per > 1) it = decode_item(p, groups, tpt, i);
        const int64_t ci = has ? it.cost(p) : 0;
        if (c <= pos && pos < c + ci) {
          range->item = i;
          range->base_t = c;
          range->base_r = r;
        }
        if (bid == 0 && has) {
          p.rec_cost[i] = c;
          p.rec_row[i] = r;
        }
        c += ci;
        r += static_cast<int64_t>(p.H) * it.rows;
      }
    } else {
      rising = !__syncthreads_or(bad);  // (prompt_seq has reported it)
      const int chunk = rising ? chunk_tiles(p, tr, tc) : 0;
      if (threadIdx.x == 0) range->item = chunk;
      if (blockIdx.x == 0 && chunk) {
        // the sequences' first pieces, for the joining kernel
        int64_t zero = 0, tz;
        c = 0;
#pragma unroll 1
        for (int k = 0; k < per; ++k)
          c += first + k < n ? prompt_pieces(p, prompt_seq(p, 2 * tpt, min(first + k, n - 1)), chunk) : 0;
        block_scan2(c, zero, scan, tc, tz);
#pragma unroll 1
        for (int k = 0; k < per; ++k) {
          const Seq s = prompt_seq(p, 2 * tpt, min(first + k, n - 1));
          if (first + k < n) p.rec_cost[first + k] = c;
          c += prompt_pieces(p, s, chunk);
        }
      }
      if (blockIdx.x == 0 && threadIdx.x == 0) p.rec_cost[p.B] = chunk;
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t tmem = *tmem_slot;
  const Abort ab{abort_flag, p.err};

  // the next published piece, for all warps but warp 0
  int wpos = 0;
  auto take = [&](Piece& pc, int code) -> bool {
    const int s = wpos % PT_RING;
    if (!pt_wait(w_full + s, (wpos / PT_RING) & 1, ab, code)) return false;
    pc = pieces[s];
    __syncwarp();
    if (lane == 0) mbar_arrive(w_empty + s);
    ++wpos;
    return !pc.end;
  };

  if (warp == 0) {
    // ================================================================ pieces, Q and K
    Sched<DEC> sc;
    sc.groups = groups;
    sc.tpt = tpt;
    sc.n = rising ? n : 0;
    sc.chunk = !DEC && p.may_split ? range->item : 0;
    sc.i0 = sc.place = 0;
    sc.base_t = sc.base_r = sc.pos = sc.end = 0;
    if constexpr (DEC) {
      sc.pos = range->begin;
      sc.end = range->end;
      if (sc.pos < sc.end) {
        sc.place = range->place;
        sc.i0 = range->item;
        sc.base_t = range->base_t;
        sc.base_r = range->base_r;
      }
    }
    sc.loaded = false;
    int published = 0;
    TileLoader ld;
    ld.init(p);
    Piece nx, pc;
    int kpos = 0, qpos = 0, j = 0, je = 0;
    int pg0 = 0, pg1 = 0;  // the next piece's first pages, looked up early
    bool want = true, have = false, ok = true;
    while (true) {
      if (want) {
        // the next piece, while this one's first tiles are on their way
        const int s = published % PT_RING;
        ok = pt_wait(w_empty + s, ((published / PT_RING) & 1) ^ 1, ab, ERR_TIMEOUT_PRODUCER);
        if (!ok) break;
        sc.next(p, pieces + s);
        if (lane == 0) mbar_arrive(w_full + s);
        nx = pieces[s];
        __syncwarp();
        ++published;
        if (p.table && !nx.end) {
          pg0 = ld.look(p, nx, ld.batch_of(nx.j0));
          pg1 = ld.look(p, nx, ld.batch_of(nx.j0) + 1);
        }
        want = false;
        have = true;
      }
      if (j >= je) {
        if (!have) {
          want = true;
          continue;
        }
        if (nx.end) break;
        pc = nx;
        have = false;
        j = pc.j0;
        je = pc.jend();
        ld.batch = ld.batch_of(j);
        ld.page = pg0;
        ld.ahead = pg1;
        for (int x = 0; ok && x < pc.q_tiles(tpt); ++x, ++qpos) {
          const int slot = qpos & 1;
          ok = pt_wait(q_empty + slot, ((qpos >> 1) & 1) ^ 1, ab, ERR_TIMEOUT_PRODUCER);
          if (!ok) break;
          if (lane == 0) {
            mbar_arrive_expect_tx(q_full + slot, (pc.q1 ? 1 : tpt) * p.G * 128 * (D / 64));
            for (int d = 0; d < D / 64; ++d)
              tma_load_4d(smem + C::OFF_Q + slot * C::QBYTES + d * (128 * 128), pc.q1 ? &p.tm_q1 : &p.tm_q,
                          q_full + slot, d * 64, pc.h * p.G, pc.tok0 + x * tpt, 0);
          }
          __syncwarp();
        }
        if (!ok) break;
        if (j >= je) continue;
      }
      const int slot = kpos % NK;
      ok = pt_wait(k_empty + slot, ((kpos / NK) & 1) ^ 1, ab, ERR_TIMEOUT_PRODUCER);
      if (!ok) break;
      ld.load(p, pc, &p.tm_k, j, D, smem + C::OFF_K + slot * C::KVBYTES, k_full + slot);
      ++kpos;
      ++j;
      if (!have && j - pc.j0 == NK) want = true;
    }
    __syncwarp();
    if (lane == 0) {
      // copies in flight must land before the CTA exits
      bool drained = true;
      for (int f = (kpos > NK ? kpos - NK : 0); f < kpos && drained; ++f)
        drained = mbar_drain(k_full + f % NK, (f / NK) & 1, p.err);
      for (int f = (qpos > 2 ? qpos - 2 : 0); f < qpos && drained; ++f)
        drained = mbar_drain(q_full + (f & 1), (f >> 1) & 1, p.err);
      // the last CTA leaves the counter as it found it
      if (!DEC && atomicAdd(p.counter + 1, 1u) == gridDim.x - 1) {
        p.counter[0] = 0;
        p.counter[1] = 0;
      }
    }
  } else if (warp == 3) {
    // ================================================================ V
    TileLoader ld;
    ld.init(p);
    Piece pc;
    int vpos = 0;
    bool ok = true;
    while (ok && take(pc, ERR_TIMEOUT_PRODUCER)) {
      ld.batch = -1;
      const int je = pc.jend();
      for (int j = pc.j0; j < je; ++j) {
        const int slot = vpos % NV;
        ok = pt_wait(v_empty + slot, ((vpos / NV) & 1) ^ 1, ab, ERR_TIMEOUT_PRODUCER);
        if (!ok) break;
        ld.load(p, pc, &p.tm_v, j, D, smem + C::OFF_V + slot * C::KVBYTES, v_full + slot);
        ++vpos;
      }
    }
    __syncwarp();
    if (lane == 0) {
      bool drained = true;
      for (int f = (vpos > NV ? vpos - NV : 0); f < vpos && drained; ++f)
        drained = mbar_drain(v_full + f % NV, (f / NV) & 1, p.err);
    }
  } else if (warp == 1 || warp == 2) {
    // ================================================================ products of tile x
    // The warp runs converged and one elected lane issues. Tiles of a pair walk the same key tiles; both
    // warps wait for every fill, in order, and release it, so a slot's two arrivals are of one fill. They issue
    // their batches (a tile's P V and the next one's Q K^T) in turn, tile 0 first, which keeps the two
    // softmax passes half a period apart; a tile on its own takes no turns (16 x 32 tokens over 4000 rows: 83 -> 77 us).
    // The two of a thin piece go apart: fills of even number are
    // tile 0's, of odd number tile 1's, and their warp releases them with both arrivals. As the slots of a
    // parity stay with a warp, it sees all of their phases: no CTA has a pair's piece beside a thin one.
    const int x = warp - 1;
    constexpr uint32_t IDESC_S = umma_idesc_f16(128, PT_BN, BF16, false);
    constexpr uint32_t IDESC_PV = umma_idesc_f16(128, D, BF16, true);
    constexpr uint32_t IDESC_T = umma_idesc_f16(128, 16, BF16, false);  // thin: keys by rows
    constexpr uint32_t IDESC_TV = IDESC_T | (1u << 15);  // thin: channels (V transposed: MN-major A) by rows
    const uint32_t tS = tmem + 128 * x;
    const uint32_t tO = tmem + 256 + D * x;
    const uint64_t qdesc0 = umma_desc_sw128(smem_u32(smem + C::OFF_Q), 16, 1024);
    const uint64_t kdesc0 = umma_desc_sw128(smem_u32(smem + C::OFF_K), 16, 1024);
    const uint64_t pdesc = umma_desc_sw128(smem_u32(smem + C::OFF_P + x * C::PBYTES), 16, 1024);
    const uint64_t vdesc0 = umma_desc_sw128(smem_u32(smem + C::OFF_V), PT_BN * 128, 1024);
    int fpos = 0, qpos = 0;  // fills of the K and V rings, of the query slots
    uint32_t free_par = 1, p_par = 0, nbatch = 0;
    Piece pc;
    bool ok = true;
    auto my_turn = [&]() -> bool {
      if (x == 1) return pt_wait(turn + 0, nbatch & 1, ab, ERR_TIMEOUT_MMA);
      return nbatch == 0 || pt_wait(turn + 1, (nbatch - 1) & 1, ab, ERR_TIMEOUT_MMA);
    };
    auto end_turn = [&]() {
      __syncwarp();
      if (lane == 0) mbar_arrive(turn + x);
      ++nbatch;
    };
    while (ok && take(pc, ERR_TIMEOUT_MMA)) {
      const int nq = pc.q_tiles(tpt), q0 = qpos;
      for (int f = q0; ok && f < q0 + nq; ++f) ok = pt_wait(q_full + (f & 1), (f >> 1) & 1, ab, ERR_TIMEOUT_MMA);
      if (!ok) break;
      qpos += nq;
      tc_fence_after();
      const uint64_t qdesc = qdesc0 + static_cast<uint64_t>(((q0 + (nq == 2 ? x : 0)) & 1) * (C::QBYTES >> 4));
      auto free_q = [&]() {  // once every score of this piece is issued
        for (int f = q0; f < q0 + nq; ++f) umma_commit(q_empty + (f & 1));
      };
      const int je = pc.jend();
      const bool pair = pc.ntok > tpt;  // (not of thin pieces)
      const bool mine = x == 0 || pc.thin || pair;
      bool freed = false, o_init = false;
      auto ensure_free = [&]() -> bool {
        if (freed) return true;
        if (!pt_wait(tile_free + x, free_par, ab, ERR_TIMEOUT_MMA)) return false;
        free_par ^= 1;
        tc_fence_after();
        freed = true;
        return true;
      };
      auto issue_S = [&](int f) {
        const uint64_t kb = kdesc0 + static_cast<uint64_t>((f % NK) * (C::KVBYTES >> 4));
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint64_t off = ((kk >> 2) * (128 * 128) + (kk & 3) * 32) >> 4;
          umma_ss(tS, qdesc + off, kb + off, IDESC_S, kk > 0);
        }
        umma_commit(s_full + x);
      };
      auto issue_St = [&](int f) {
        const uint64_t kb = kdesc0 + static_cast<uint64_t>((f % NK) * (C::KVBYTES >> 4));
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint64_t off = ((kk >> 2) * (128 * 128) + (kk & 3) * 32) >> 4;
          umma_ss(tS, kb + off, qdesc + off, IDESC_T, kk > 0);
        }
        umma_commit(s_full + x);
      };
      // O^T (+)= V^T P^T. With 64 channels the rows from 64 on are of whatever lies a tile behind, and not read.
      auto issue_thin = [&](int f) {
        const uint64_t vb = vdesc0 + static_cast<uint64_t>((f % NV) * (C::KVBYTES >> 4));
#pragma unroll
        for (int kk = 0; kk < PT_BN / 16; ++kk)
          umma_ss(tO, vb + static_cast<uint64_t>((kk * 2048) >> 4),
                  pdesc + static_cast<uint64_t>(((kk >> 2) * (16 * 128) + (kk & 3) * 32) >> 4), IDESC_TV,
                  (o_init || kk > 0) ? 1u : 0u);
        o_init = true;
      };
      auto issue_PV = [&](int f, int half) {
        const uint64_t vb = vdesc0 + static_cast<uint64_t>((f % NV) * (C::KVBYTES >> 4));
#pragma unroll
        for (int k4 = 0; k4 < PT_BN / 32; ++k4) {
          const int kk = half * (PT_BN / 32) + k4;
          umma_ts(tO, tS + kk * 8, vb + static_cast<uint64_t>((kk * 2048) >> 4), IDESC_PV, (o_init || kk > 0) ? 1u : 0u);
        }
        o_init = true;
      };
      auto weights = [&]() -> bool {  // the first half of them is there, and O may be written
        if (!pt_wait(p_lo + x, p_par, ab, ERR_TIMEOUT_MMA)) return false;
        tc_fence_after();
        return ensure_free();
      };
      auto weigh = [&](int f) -> bool {  // P V of the tile whose V is fill f
        if (DEC && pc.thin) {
          if (!pt_wait(p_full + x, p_par, ab, ERR_TIMEOUT_MMA)) return false;
          p_par ^= 1;
          tc_fence_after();
          issue_thin(f);
          return true;
        }
        issue_PV(f, 0);
        if (!pt_wait(p_full + x, p_par, ab, ERR_TIMEOUT_MMA)) return false;
        p_par ^= 1;
        tc_fence_after();
        issue_PV(f, 1);
        return true;
      };
      auto wait_k = [&](int f) -> bool {
        if (!pt_wait(k_full + f % NK, (f / NK) & 1, ab, ERR_TIMEOUT_MMA)) return false;
        tc_fence_after();
        return true;
      };
      auto wait_v = [&](int f) -> bool {
        if (!pt_wait(v_full + f % NV, (f / NV) & 1, ab, ERR_TIMEOUT_MMA)) return false;
        tc_fence_after();
        return true;
      };
      if (DEC && pc.thin) {
        const int n = je - pc.j0, first = (fpos ^ x) & 1;
        if (first >= n) free_q();
        for (int i = first; first < n; i += 2) {
          if (i > first) {
            const int f = fpos + i - 2;
            if (i >= n) free_q();
            ok = wait_v(f) && weights() && weigh(f);
            if (!ok) break;
            umma_commit(v_empty + f % NV);
            umma_commit(v_empty + f % NV);
            if (i >= n) break;
          }
          const int f = fpos + i;
          ok = wait_k(f);
          if (!ok) break;
          issue_St(f);
          umma_commit(k_empty + f % NK);
          umma_commit(k_empty + f % NK);
        }
        if (!ok) break;
        fpos += n;
      } else {
        auto uses = [&](int j) { return mine && j < (x ? pc.nt1 : pc.nt0); };
        if (pc.j0 >= je) free_q();
        // batch j: P V of tile j - 1, Q K^T of tile j
        for (int j = pc.j0; pc.j0 < je && j <= je; ++j, ++fpos) {
          const bool before = j > pc.j0, more = j < je;
          // nothing is waited for in a turn that could be before it
          ok = (!before || wait_v(fpos - 1)) && (!more || wait_k(fpos)) && (!before || !uses(j - 1) || weights());
          if (!ok) break;
          if (!more) free_q();
          ok = !pair || my_turn();
          if (!ok) break;
          if (before && uses(j - 1)) {
            ok = weigh(fpos - 1);
            if (!ok) break;
          }
          if (more && uses(j)) issue_S(fpos);
          if (pair) end_turn();
          if (before) umma_commit(v_empty + (fpos - 1) % NV);
          if (more) umma_commit(k_empty + fpos % NK);
        }
        if (!ok) break;
        if (pc.j0 < je) --fpos;
      }
      // The products' warp waits for the tile once a piece and always announces O; the epilogue always
      // waits for that before it gives the tile back, so the parities cannot run apart.
      if (mine) {
        ok = ensure_free();
        if (!ok) break;
        umma_commit(o_full + x);
      }
    }
    umma_commit(mma_done);
    if (lane == 0) mbar_drain(mma_done, 0, p.err);
    __syncwarp();
  } else {
    // ================================================================ softmax and epilogue of tile x
    const int x = (warp - 4) >> 2;
    const int wq = warp & 3;
    const int r = wq * 32 + lane;
    const uint32_t lane_base = static_cast<uint32_t>(wq * 32) << 16;
    const uint32_t tS = tmem + lane_base + 128 * x;
    const uint32_t tO = tmem + lane_base + 256 + D * x;
    const float sl2 = p.scale_log2;
    int vpos = 0;
    uint32_t s_par = 0, o_par = 0, votes = 0, xfers = 0;
    Piece pc;
    bool ok = true;
    while (ok && take(pc, ERR_TIMEOUT_SOFTMAX)) {
      if (!DEC) pc.by_length = 0;
      const int je = pc.jend();
      const bool valid = x == 0 || pc.ntok > tpt;  // (not of thin pieces)
      const int ntok = max(0, min(tpt, pc.ntok - x * tpt));
      const int nrows = ntok * p.G;
      const bool warp_live = wq * 32 < nrows;
      const bool live = r < nrows;
      const int ti = r / p.G;                               // token of this row within the tile
      const int tok = pc.tok0 + x * tpt + ti;
      int lim_row = 0;  // keys from kb on that this row sees
      if (live) {
        lim_row = pc.lim0 + (tok - pc.tok0) * pc.lim_step;
        if (!DEC && tok - pc.tok0 < pc.before) lim_row = 0;
        if (pc.by_length) lim_row = min(lim_row, p.lengths[tok]);
        lim_row -= pc.kb;
      }
      if (DEC && pc.thin) {
        // ------------ transposed: a key per thread, a query row per column. All of the tile's warps hold the
        // same references; a warp that finds a score more than 2^8 above one says so in the vote that
        // every key tile has, and O^T (a channel per thread) moves to the new references before the next product.
        float* vmax = reinterpret_cast<float*>(smem + C::OFF_VOTE) + x * 2 * 4 * PT_THIN;
        int* vflag = reinterpret_cast<int*>(smem + C::OFF_VOTE + 2 * 2 * 4 * PT_THIN * 4) + x * 2 * 4;
        uint8_t* ps = smem + C::OFF_P + x * C::PBYTES + (r >> 6) * (16 * 128) + (r & 7) * 2;
        float m[PT_THIN], ls[PT_THIN];
#pragma unroll
        for (int g = 0; g < PT_THIN; ++g) {
          m[g] = -INFINITY;
          ls[g] = 0.f;
        }
        bool has = false;
        // Column lane / 4's maximum or sum over the warp: the lanes halve the columns among themselves three times.
        auto reduce = [&](const float (&in)[PT_THIN], bool sum) -> float {
          float v[PT_THIN];
#pragma unroll
          for (int g = 0; g < PT_THIN; ++g) v[g] = in[g];
#pragma unroll
          for (int o = 16, n = PT_THIN / 2; o; o >>= 1, n >>= 1) {
            if (n) {
              const bool up = lane & o;
#pragma unroll
              for (int g = 0; g < n; ++g) {
                const float keep = up ? v[g + n] : v[g], give = up ? v[g] : v[g + n];
                const float got = __shfl_xor_sync(0xFFFFFFFFu, give, o);
                v[g] = sum ? keep + got : fmaxf(keep, got);
              }
            } else {
              const float got = __shfl_xor_sync(0xFFFFFFFFu, v[0], o);
              v[0] = sum ? v[0] + got : fmaxf(v[0], got);
            }
          }
          return v[0];
        };
        auto cast_vote = [&](float mine, bool put, bool flag) -> bool {
          const int at = (votes & 1) * 4 + wq;
          if (put && (lane & 3) == 0) vmax[at * PT_THIN + (lane >> 2)] = mine;
          if (lane == 0) vflag[at] = flag;
          __syncwarp();
          if (lane == 0) mbar_arrive(vote + x);
          const bool all = pt_wait(vote + x, votes & 1, ab, ERR_TIMEOUT_SOFTMAX);
          ++votes;
          return all;
        };
        for (int j = pc.j0 + ((vpos ^ x) & 1); j < je; j += 2) {
          const int f = vpos + (j - pc.j0);
          const int have = pc.kend - pc.kb - j * PT_BN;
          if (!pt_wait(s_full + x, s_par, ab, ERR_TIMEOUT_SOFTMAX)) { ok = false; break; }
          s_par ^= 1;
          tc_fence_after();
          uint32_t sc[PT_THIN];
          tmem_ld8(tS, sc);
          float s[PT_THIN];
          bool over = false;
#pragma unroll
          for (int g = 0; g < PT_THIN; ++g) {
            s[g] = g < p.G && r < have ? __uint_as_float(sc[g]) * sl2 : -INFINITY;
            over |= s[g] > m[g] + 8.f;
          }
          over = __any_sync(0xFFFFFFFFu, over);
          float mine = 0.f;
          if (over) mine = reduce(s, false);
          ok = cast_vote(mine, over, over);
          if (!ok) break;
          const int seen = (votes & 1) ^ 1;
          const int4 fl = *reinterpret_cast<const int4*>(vflag + seen * 4);
          if (fl.x | fl.y | fl.z | fl.w) {
            float mn[PT_THIN];
#pragma unroll
            for (int g = 0; g < PT_THIN; ++g) mn[g] = m[g];
#pragma unroll 1
            for (int w = 0; w < 4; ++w) {
              if (!vflag[seen * 4 + w]) continue;
              const float4* v = reinterpret_cast<const float4*>(vmax + (seen * 4 + w) * PT_THIN);
#pragma unroll
              for (int q = 0; q < PT_THIN / 4; ++q) {
                const float4 u = v[q];
                mn[4 * q] = fmaxf(mn[4 * q], u.x);
                mn[4 * q + 1] = fmaxf(mn[4 * q + 1], u.y);
                mn[4 * q + 2] = fmaxf(mn[4 * q + 2], u.z);
                mn[4 * q + 3] = fmaxf(mn[4 * q + 3], u.w);
              }
            }
            uint32_t o[PT_THIN];
            if (has) tmem_ld8(tO, o);
#pragma unroll
            for (int g = 0; g < PT_THIN; ++g) {
              const float fac = m[g] == -INFINITY ? 0.f : ex2(m[g] - mn[g]);
              m[g] = mn[g];
              ls[g] = fac == 0.f ? 0.f : ls[g] * fac;
              o[g] = !has || fac == 0.f ? 0u : __float_as_uint(__uint_as_float(o[g]) * fac);
            }
            if (has) {
              tmem_st8(tO, o);
              tmem_st_wait();
            }
          }
#pragma unroll
          for (int g = 0; g < PT_THIN; ++g) {
            const float w = g < p.G && r < have ? ex2(s[g] - m[g]) : 0.f;
            ls[g] += w;
            const int at = g * 128 + ((((r & 63) >> 3) ^ g) << 4);
            if (BF16) *reinterpret_cast<__nv_bfloat16*>(ps + at) = __float2bfloat16_rn(w);
            else *reinterpret_cast<__half*>(ps + at) = __float2half_rn(w);
          }
          if (have < PT_BN) {
            // V rows past the sequence hold anything: 0 in their place, before the products read them. (With this
            // tile's scores there, the slot's earlier fills have been read, so the wait is for this one.)
            if (!pt_wait(v_full + f % NV, (f / NV) & 1, ab, ERR_TIMEOUT_SOFTMAX)) { ok = false; break; }
            if (r >= have) {
              uint8_t* row = smem + C::OFF_V + (f % NV) * C::KVBYTES + r * 128;
#pragma unroll 1
              for (int c = 0; c < D / 64; ++c)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                  *reinterpret_cast<uint4*>(row + c * (PT_BN * 128) + e * 16) = make_uint4(0, 0, 0, 0);
            }
          }
          fence_async_smem();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(p_lo + x);
            mbar_arrive(p_full + x);
          }
          has = true;
        }
        if (!ok) break;
        vpos += je - pc.j0;
        // the sums over the tile's keys: the warp's, then the four warps' through the votes' memory
        if (!cast_vote(reduce(ls, true), true, false)) break;
        const float* sums = vmax + ((votes & 1) ^ 1) * 4 * PT_THIN;
        if (!pt_wait(o_full + x, o_par, ab, ERR_TIMEOUT_EPILOGUE)) break;
        o_par ^= 1;
        tc_fence_after();
        uint32_t o[PT_THIN];
        tmem_ld8(tO, o);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(tile_free + x);
        // tile 1 hands its O^T, maxima and sums over, tile 0 adds them to its own and stores the piece's
        float* xo = reinterpret_cast<float*>(smem + C::OFF_X);
        float* xm = xo + PT_THIN * D;
        float* xl = xm + PT_THIN;
        if (!pt_wait(xfer + (x ^ 1), (xfers & 1) ^ x, ab, ERR_TIMEOUT_EPILOGUE)) break;
        ++xfers;
        if (x) {
#pragma unroll
          for (int g = 0; g < PT_THIN; ++g) {
            if (r < D) xo[g * D + r] = __uint_as_float(o[g]);
            if (r == g) {
              xm[g] = m[g];
              xl[g] = has ? (sums[g] + sums[PT_THIN + g]) + (sums[2 * PT_THIN + g] + sums[3 * PT_THIN + g]) : 0.f;
            }
          }
        } else {
#pragma unroll
          for (int g = 0; g < PT_THIN; ++g) {
            if (g >= p.G) continue;
            const float l0 = has ? (sums[g] + sums[PT_THIN + g]) + (sums[2 * PT_THIN + g] + sums[3 * PT_THIN + g]) : 0.f;
            const float l1 = xl[g], m1 = xm[g];
            // a tile that has nothing for the row (sum 0; not NaN) takes no part
            const float mm = l0 == 0.f ? m1 : l1 == 0.f ? m[g] : fmaxf(m[g], m1);
            const float a0 = l0 == 0.f ? 0.f : ex2(m[g] - mm), a1 = l1 == 0.f ? 0.f : ex2(m1 - mm);
            if (r < D)
              p.part_o[(pc.orow0 + g) * D + r] = (l0 == 0.f ? 0.f : a0 * __uint_as_float(o[g])) + (l1 == 0.f ? 0.f : a1 * xo[g * D + r]);
            if (r == g) p.part_s[pc.orow0 + g] = make_float2(mm, (l0 == 0.f ? 0.f : a0 * l0) + (l1 == 0.f ? 0.f : a1 * l1));
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(xfer + x);
        continue;
      }
      // rows that do not exist get a reference no score exceeds, and weigh nothing
      float m_used = live ? -INFINITY : 1e30f, l = 0.f;
      bool o_has = false;
      const int my_end = x ? pc.nt1 : pc.nt0;
      for (int j = pc.j0; valid && j < my_end; ++j) {
        const int f = vpos + (j - pc.j0);
        const int n0 = j * PT_BN;
        const int have = pc.kend - pc.kb - n0;  // rows of this tile that exist
        const bool tail = have < PT_BN;
        const int lim = live ? lim_row - n0 : PT_BN;
        const bool masked = __any_sync(0xFFFFFFFFu, lim < PT_BN);
        if (!pt_wait(s_full + x, s_par, ab, ERR_TIMEOUT_SOFTMAX)) { ok = false; break; }
        s_par ^= 1;
        if (tail) {
          // V rows past the sequence hold anything: 0 in their place, before the products read them. (With this
          // tile's scores there, every fill before the previous one has landed, so the wait is for this one.)
          if (!pt_wait(v_full + f % NV, (f / NV) & 1, ab, ERR_TIMEOUT_SOFTMAX)) { ok = false; break; }
          if (r >= have) {
            uint8_t* row = smem + C::OFF_V + (f % NV) * C::KVBYTES + r * 128;
#pragma unroll
            for (int c = 0; c < D / 64; ++c)
#pragma unroll
              for (int e = 0; e < 8; ++e)
                *reinterpret_cast<uint4*>(row + c * (PT_BN * 128) + e * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_async_smem();
        }
        tc_fence_after();
        if (!warp_live) {  // no row of this warp exists: its weights go nowhere
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(p_lo + x);
            mbar_arrive(p_full + x);
          }
          o_has = true;
          continue;
        }
        if (masked) {
          // scores past the row's limit become -inf in TMEM
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            if (!__any_sync(0xFFFFFFFFu, lim < c * 32 + 32)) continue;
            uint32_t sc[32];
            tmem_ld32(tS + c * 32, sc);
#pragma unroll
            for (int e = 0; e < 32; ++e) sc[e] = (c * 32 + e < lim) ? sc[e] : 0xFF800000u;
            tmem_st32(tS + c * 32, sc);
          }
          tmem_st_wait();
        }
        auto chunk_max = [&](const uint32_t* sc) {  // the scale is positive
          float m0 = __uint_as_float(sc[0]), m1 = __uint_as_float(sc[1]);
#pragma unroll
          for (int e = 2; e < 32; e += 4) {
            m0 = fmax3(m0, __uint_as_float(sc[e]), __uint_as_float(sc[e + 1]));
            if (e + 2 < 32) m1 = fmax3(m1, __uint_as_float(sc[e + 2]), __uint_as_float(sc[e + 3]));
          }
          return fmaxf(m0, m1) * sl2;
        };
        float2 la = make_float2(0.f, 0.f), lb = la;
        auto half = [&](const uint32_t* sc, float nb, uint32_t* out) {
          const float2 s2 = make_float2(sl2, sl2), n2 = make_float2(nb, nb);
#pragma unroll
          for (int e = 0; e < 16; e += 4) {
            const float2 a01 = ffma2(make_float2(__uint_as_float(sc[e]), __uint_as_float(sc[e + 1])), s2, n2);
            const float2 a23 = ffma2(make_float2(__uint_as_float(sc[e + 2]), __uint_as_float(sc[e + 3])), s2, n2);
            float w[4];
            w[0] = ex2(a01.x); w[1] = ex2(a01.y); w[2] = ex2(a23.x); w[3] = ex2(a23.y);
            la = fadd2(la, make_float2(w[0], w[1]));
            lb = fadd2(lb, make_float2(w[2], w[3]));
            out[e / 2] = pack2(w[0], w[1], BF16);
            out[e / 2 + 1] = pack2(w[2], w[3], BF16);
          }
        };
        auto weights = [&](const uint32_t* sc, float nb, uint32_t* out) {
          half(sc, nb, out);
          half(sc + 16, nb, out + 8);
        };
        int stop = 0;          // first 32-column chunk that the stream did not finish
        bool lo_sent = false;  // weights of keys 0..63 are final and announced
        {
          // A chunk's maximum is taken among the exponentials of the chunk before it (prompts: 2 % with the waits before
          // the turns).
          uint32_t sa[32], sb[32], w[16];
          tmem_ld32_async(tS, sa);
          tmem_ld32_wait(sa);
          tmem_ld32_async(tS + 32, sb);
          const float m0 = chunk_max(sa);
          if (m_used == -INFINITY) m_used = m0 == -INFINITY ? 0.f : m0;
          const float nb = -m_used, most = m_used + 8.f;
          bool over = __any_sync(0xFFFFFFFFu, m0 > most);
          auto one = [&](int c, uint32_t(&cur)[32], uint32_t(&nxt)[32]) {  // weights of chunk c, maximum of the next
            half(cur, nb, w);
            tmem_ld32_wait(nxt);
            half(cur + 16, nb, w + 8);
            const float mn = chunk_max(nxt);
            tmem_st16(tS + c * 16, w);
            tmem_ld32_async(tS + (c + 2) * 32, cur);
            over = __any_sync(0xFFFFFFFFu, mn > most);
            stop = c + 1;
          };
          if (!over) one(0, sa, sb);
          if (!over) one(1, sb, sa);
          if (!over) {
            const float2 la0 = la, lb0 = lb;
            half(sa, nb, w);
            tmem_ld32_wait(sb);
            if (__any_sync(0xFFFFFFFFu, chunk_max(sb) > most)) {
              la = la0;
              lb = lb0;
            } else {
              // nothing stored will be rescaled: P V of keys 0..63 may begin
              tmem_st_wait();
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(p_lo + x);
              lo_sent = true;
              half(sa + 16, nb, w + 8);
              tmem_st16(tS + 32, w);
              weights(sb, nb, w);
              tmem_st16(tS + 48, w);
              stop = 4;
            }
          } else {
            tmem_ld32_wait(sa);
            tmem_ld32_wait(sb);
          }
        }
        if (stop < 4) {
          // some row outgrew its reference: the maximum of what is left, everything so far rescaled, by whole
          // octaves where weights of this tile are stored already, then the rest
          tmem_st_wait();
          float mt = -INFINITY;
#pragma unroll 1
          for (int c = stop; c < 4; ++c) {
            uint32_t sc[32];
            tmem_ld32(tS + c * 32, sc);
            mt = fmaxf(mt, chunk_max(sc));
          }
          const bool need = mt > m_used + 8.f;
          if (__any_sync(0xFFFFFFFFu, need)) {
            float m_new = m_used, fac = 1.f;
            if (need) {
              if (stop > 0) {
                const float k = ceilf(mt - m_used);
                m_new = m_used + k;
                fac = k < 127.f ? __int_as_float((127 - static_cast<int>(k)) << 23) : 0.f;
              } else {
                m_new = mt;
                fac = ex2(m_used - m_new);
              }
            }
            l *= fac;
            la.x *= fac; la.y *= fac; lb.x *= fac; lb.y *= fac;
            if (o_has) {
#pragma unroll 1
              for (int c = 0; c < D / 16; ++c) {
                uint32_t o[16];
                tmem_ld16(tO + c * 16, o);
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * fac);
                tmem_st16(tO + c * 16, o);
              }
            }
#pragma unroll 1
            for (int c = 0; c < stop; ++c) {
              uint32_t w[16];
              tmem_ld16(tS + c * 16, w);
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                float2 v;
                if (BF16) v = __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&w[e]));
                else v = __half22float2(*reinterpret_cast<__half2*>(&w[e]));
                w[e] = pack2(v.x * fac, v.y * fac, BF16);
              }
              tmem_st16(tS + c * 16, w);
            }
            m_used = m_new;
          }
#pragma unroll 1
          for (int c = stop; c < 4; ++c) {
            uint32_t sc[32], w[16];
            tmem_ld32(tS + c * 32, sc);
            weights(sc, -m_used, w);
            tmem_st16(tS + c * 16, w);
          }
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (!lo_sent) mbar_arrive(p_lo + x);
          mbar_arrive(p_full + x);
        }
        l += (la.x + la.y) + (lb.x + lb.y);
        o_has = true;
      }
      if (!ok) break;
      vpos += max(0, je - pc.j0);
      if (!valid) continue;
      // ---------------- epilogue
      if (!pt_wait(o_full + x, o_par, ab, ERR_TIMEOUT_EPILOGUE)) break;
      o_par ^= 1;
      tc_fence_after();
      if (warp_live) {
        uint8_t* stg = smem + C::OFF_EPI + (warp - 4) * 32 * C::EPI_PITCH;
        const int rr = lane >> 2, seg = lane & 3;  // the row and 16-byte piece this lane stores
        const int left = nrows - wq * 32;          // rows of this warp
        if (pc.split) {
          const int64_t row0 = (x ? pc.orow1 : pc.orow0) + wq * 32;
          if (live) p.part_s[row0 + lane] = make_float2(m_used, o_has ? l : 0.f);
          if (o_has && left <= 8) {
            // a few rows: every lane writes its own
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              uint32_t o[32];
              tmem_ld32(tO + c * 32, o);
              if (live) {
                uint4* to = reinterpret_cast<uint4*>(p.part_o + (row0 + lane) * D + c * 32);
#pragma unroll
                for (int e = 0; e < 8; ++e) to[e] = make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
              }
            }
          } else if (o_has) {
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              uint32_t o[32];
              tmem_ld32(tO + c * 32, o);
#pragma unroll
              for (int hf = 0; hf < 2; ++hf) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  *reinterpret_cast<uint4*>(stg + lane * C::EPI_PITCH + e * 16) = make_uint4(
                      o[hf * 16 + 4 * e], o[hf * 16 + 4 * e + 1], o[hf * 16 + 4 * e + 2], o[hf * 16 + 4 * e + 3]);
                __syncwarp();
#pragma unroll
                for (int q4 = 0; q4 < 4; ++q4) {
                  const int lr = q4 * 8 + rr;
                  if (lr < left)
                    *reinterpret_cast<uint4*>(p.part_o + (row0 + lr) * D + c * 32 + hf * 16 + seg * 4) =
                        *reinterpret_cast<const uint4*>(stg + lr * C::EPI_PITCH + seg * 16);
                }
                __syncwarp();
              }
            }
          }
        } else {
          using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
          const bool none = l == 0.f;  // a row that sees nothing gives 0, whatever 0 times V was
          const float inv = none ? 0.f : 1.f / l;
          const int64_t mine = live ? tok * p.o_t + (pc.h * p.G + r - ti * p.G) * p.o_h : 0;
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            if (o_has) tmem_ld32(tO + c * 32, o);
            if (!o_has || none) {
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = 0u;
            }
#pragma unroll
            for (int e = 0; e < 32; e += 8) {
              uint4 w;
              w.x = pack2(__uint_as_float(o[e]) * inv, __uint_as_float(o[e + 1]) * inv, BF16);
              w.y = pack2(__uint_as_float(o[e + 2]) * inv, __uint_as_float(o[e + 3]) * inv, BF16);
              w.z = pack2(__uint_as_float(o[e + 4]) * inv, __uint_as_float(o[e + 5]) * inv, BF16);
              w.w = pack2(__uint_as_float(o[e + 6]) * inv, __uint_as_float(o[e + 7]) * inv, BF16);
              *reinterpret_cast<uint4*>(stg + lane * C::EPI_PITCH + e * 2) = w;
            }
            __syncwarp();
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4) {
              const int lr = q4 * 8 + rr;
              const int64_t off = shfl64(mine, lr);
              if (lr < left)
                *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + off + c * 32 + seg * 8) =
                    *reinterpret_cast<const uint4*>(stg + lr * C::EPI_PITCH + seg * 16);
            }
            __syncwarp();
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(tile_free + x);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 2) tmem_dealloc(tmem, 512);
}

// ------------------------------------------------------------------------------------ joining
// Prompts, whose many rows have a few pieces each: one warp per output row, the maxima and sums of its pieces, then
// their weighted sum, D / 32 elements a lane. Pieces that hold nothing for the row (sum 0) are left out.
template <int D, typename T> struct Joiner {
  float acc[D / 32], m, l;
  __device__ __forceinline__ Joiner() : m(-INFINITY), l(0.f) {
#pragma unroll
    for (int i = 0; i < D / 32; ++i) acc[i] = 0.f;
  }
  // pieces i in [0, n) at partial row `row(i)`
  template <typename F> __device__ __forceinline__ void add(const PagedAttn& p, int n, F row) {
    const int lane = lane_id();
    for (int i0 = 0; i0 < n; i0 += 32) {
      float2 s = make_float2(-INFINITY, 0.f);
      if (i0 + lane < n) s = __ldcg(p.part_s + row(i0 + lane));
      const bool has = s.y != 0.f;  // NaN too
      float mx = has ? s.x : -INFINITY;
#pragma unroll
      for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, o));
      const unsigned any = __ballot_sync(0xFFFFFFFFu, has);
      if (!any) continue;
      const float mn = fmaxf(m, mx), f = m == -INFINITY ? 0.f : ex2(m - mn);
      m = mn;
      const float w = has ? ex2(s.x - mn) : 0.f;
      float sum = has ? w * s.y : 0.f;
#pragma unroll
      for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
      l = l * f + sum;
#pragma unroll
      for (int e = 0; e < D / 32; ++e) acc[e] *= f;
      const int most = min(32, n - i0);
      for (int i = 0; i < most; i += 8) {
        // eight pieces' rows on their way at once; a piece without a sum may hold anything
        float v[8][D / 32];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const bool live = i + k < most && (any >> (i + k) & 1);
          const float* src = p.part_o + row(i0 + (live ? i + k : 0)) * D + lane * (D / 32);
          if constexpr (D == 128) {
            const float4 f4 = live ? __ldcg(reinterpret_cast<const float4*>(src)) : make_float4(0.f, 0.f, 0.f, 0.f);
            v[k][0] = f4.x; v[k][1] = f4.y; v[k][2] = f4.z; v[k][3] = f4.w;
          } else {
            const float2 f2 = live ? __ldcg(reinterpret_cast<const float2*>(src)) : make_float2(0.f, 0.f);
            v[k][0] = f2.x; v[k][1] = f2.y;
          }
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float wk = __shfl_sync(0xFFFFFFFFu, w, (i + k) & 31);
#pragma unroll
          for (int e = 0; e < D / 32; ++e) acc[e] += (i + k < most ? wk : 0.f) * v[k][e];
        }
      }
    }
  }
  __device__ __forceinline__ void store(T* dst) {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T o[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) o[i] = from_f32<T>(acc[i] * inv);
    if constexpr (D == 128) *reinterpret_cast<uint2*>(dst + lane_id() * 4) = *reinterpret_cast<const uint2*>(o);
    else *reinterpret_cast<uint32_t*>(dst + lane_id() * 2) = *reinterpret_cast<const uint32_t*>(o);
  }
};

template <int D, typename T>
__global__ void __launch_bounds__(128) prompt_join_kernel(const __grid_constant__ PagedAttn p) {
  const int tpt = 128 / p.G, Hq = p.H * p.G;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (row >= static_cast<int64_t>(p.T) * Hq) return;  // (every block has rows, whose warps wait)
  const int t = static_cast<int>(row / Hq), hq = static_cast<int>(row % Hq), h = hq / p.G, rg = hq % p.G;
  // What goes by the inputs alone comes before the wait for the partial results. Warps that have nothing to join wait
  // too: a grid of which none did could end before the attention kernel, and the stream's next call begin on its scratch.
  const int b = paged_sequence(p.cu, p.B, t);
  if (b < 0) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    return;
  }
  const Seq s = prompt_seq(p, 2 * tpt, b);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int chunk = static_cast<int>(p.rec_cost[p.B]);
  if (!chunk) return;
  const int nch = (s.mt + chunk - 1) / chunk;
  if (nch == 1 || t < s.c0 || t >= s.c0 + s.n) return;
  const int q = (t - s.c0) / (2 * tpt), in = t - s.c0 - q * 2 * tpt, x = in / tpt;
  const int last = min(2 * tpt, s.n - q * 2 * tpt);  // tokens of the unit
  const int lim = p.causal ? max(0, s.len - s.n + q * 2 * tpt + last) : s.len;
  const int n = max(1, ((lim + PT_BN - 1) / PT_BN + chunk - 1) / chunk);
  const int64_t id0 = p.rec_cost[b] + static_cast<int64_t>(h) * nch * s.nq + (s.nq - 1 - q);
  const int64_t base = id0 * PT_ROWS + x * 128 + (in - x * tpt) * p.G + rg;
  const int64_t stride = static_cast<int64_t>(s.nq) * PT_ROWS;
  Joiner<D, T> jn;
  jn.add(p, n, [&](int k) { return base + k * stride; });
  jn.store(static_cast<T*>(p.out) + t * p.o_t + hq * p.o_h);
}

// Decoding, whose few rows have many pieces each (one for every CTA that had a part of the prefix or of the own rows):
// eight of them on their way at once. WPR warps share a row's pieces, and their sums meet in shared memory: four where a
// block per row fits the GPU at once, one for more rows (see launch_paged_t).
template <int D, typename T, int WPR>
__global__ void __launch_bounds__(128, 6) decode_join_kernel(const __grid_constant__ PagedAttn p) {
  constexpr int E = D / 32;
  __shared__ float acc_s[4][D];
  __shared__ float2 s_s[4];
  const int tpt = 128 / p.G, Hq = p.H * p.G, lane = lane_id(), warp = threadIdx.x >> 5;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (4 / WPR) + warp / WPR;
  const int groups = groups_ok(p) ? p.groups : 0;
  if (row >= static_cast<int64_t>(p.B) * Hq) return;  // (every block has rows, whose warps wait)
  const int b = static_cast<int>(row / Hq), hq = static_cast<int>(row % Hq), h = hq / p.G, rg = hq % p.G;
  const int g = group_of(p, groups, b);
  const Item own = decode_item(p, groups, tpt, groups + b);
  Item shared = own;
  if (g >= 0) shared = decode_item(p, groups, tpt, g);
  // everything above goes by the inputs alone
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Ctas ct = *p.rec_ctas;
  int n0 = 0, n1 = 0;
  int64_t base0 = 0, base1 = 0;
  // pieces of a unit: one in every CTA from that of its first key tile to that of its last
  if (own.tiles) {
    const int64_t u0 = p.rec_cost[groups + b] - ct.cost[0] + h * own.unit_cost(p) + p.w_start;
    const int c0 = static_cast<int>(quotient((u0 + 1) * ct.n[1] - 1, ct.cost[1]));
    n1 = static_cast<int>(quotient((u0 + static_cast<int64_t>(own.tiles - 1) * own.tile_cost(p) + 1) * ct.n[1] - 1, ct.cost[1])) - c0 + 1;
    base1 = p.rec_row[groups + b] + static_cast<int64_t>(h) * own.rows + static_cast<int64_t>(c0 + ct.from[1]) * PT_ROWS + rg;
  }
  if (g >= 0 && shared.tiles) {
    const int in = b - shared.first, up = in / (2 * tpt);
    const int64_t u0 = p.rec_cost[g] + (static_cast<int64_t>(h) * shared.units + up) * shared.unit_cost(p) + p.w_start;
    const int c0 = static_cast<int>(quotient((u0 + 1) * ct.n[0] - 1, ct.cost[0]));
    n0 = static_cast<int>(quotient((u0 + static_cast<int64_t>(shared.tiles - 1) * shared.tile_cost(p) + 1) * ct.n[0] - 1, ct.cost[0])) - c0 + 1;
    base0 = p.rec_row[g] + static_cast<int64_t>(h) * shared.rows + in * p.G + static_cast<int64_t>(c0) * PT_ROWS + rg;
  }
  const int n = n0 + n1;
  base1 -= static_cast<int64_t>(n0) * PT_ROWS;
  float acc[E], l = 0.f, m = -INFINITY;
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
#pragma unroll 1
  for (int i0 = warp % WPR; i0 < n; i0 += 8 * WPR) {
    float v[8][E];
    float2 st[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int i = min(i0 + WPR * k, n - 1);  // the last one again where there are fewer
      const int64_t at = (i < n0 ? base0 : base1) + static_cast<int64_t>(i) * PT_ROWS;
      st[k] = __ldcg(p.part_s + at);
      if constexpr (D == 128) {
        const float4 f4 = __ldcg(reinterpret_cast<const float4*>(p.part_o + at * D) + lane);
        v[k][0] = f4.x; v[k][1] = f4.y; v[k][2] = f4.z; v[k][3] = f4.w;
      } else {
        const float2 f2 = __ldcg(reinterpret_cast<const float2*>(p.part_o + at * D) + lane);
        v[k][0] = f2.x; v[k][1] = f2.y;
      }
    }
    // pieces that hold nothing for the row (sum 0; not NaN) take no part
    float mn = m;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (i0 + WPR * k >= n) st[k].y = 0.f;
      if (st[k].y != 0.f) mn = fmaxf(mn, st[k].x);
    }
    const float f = m == -INFINITY ? 0.f : ex2(m - mn);
    m = mn;
    l *= f;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] *= f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const bool has = st[k].y != 0.f;
      const float w = has ? ex2(st[k].x - m) : 0.f;
      l += has ? w * st[k].y : 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] += has ? w * v[k][e] : 0.f;
    }
  }
  T* dst = static_cast<T*>(p.out) + b * p.o_t + hq * p.o_h;
  if constexpr (WPR == 1) {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = from_f32<T>(acc[e] * inv);
    if constexpr (D == 128) *reinterpret_cast<uint2*>(dst + lane * E) = *reinterpret_cast<const uint2*>(o);
    else *reinterpret_cast<uint32_t*>(dst + lane * E) = *reinterpret_cast<const uint32_t*>(o);
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) acc_s[warp][lane * E + e] = acc[e];
    if (lane == 0) s_s[warp] = make_float2(m, l);
    __syncthreads();
    if (threadIdx.x < D) {
      const int d = threadIdx.x;
      float mn = -INFINITY, sum = 0.f, o = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w)
        if (s_s[w].y != 0.f) mn = fmaxf(mn, s_s[w].x);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        if (s_s[w].y == 0.f) continue;
        const float f = ex2(s_s[w].x - mn);
        sum += f * s_s[w].y;
        o += f * acc_s[w][d];
      }
      dst[d] = from_f32<T>(sum == 0.f ? 0.f : o / sum);
    }
  }
}

// ------------------------------------------------------------------------------------ launch
namespace {
struct Sizes {
  int64_t rows, recs;  // partial rows, records of items
  bool split;
};
Sizes sizes_of(int64_t T, int64_t B, int64_t H, int64_t G, int64_t groups, bool decode, int sms) {
  Sizes s;
  const int64_t utok = 2 * (128 / G);
  if (decode) {
    s.split = true;
    s.rows = 2 * B * H * G + PT_ROWS * static_cast<int64_t>(sms);
    s.recs = groups + B;
  } else {
    // whole units where the tokens alone make two for every SM
    s.split = H * (T / utok) < 2 * static_cast<int64_t>(sms);
    const int64_t units = H * ((T + utok - 1) / utok + B);
    // of fewer than 2 * sms units; the chunks in the mean, and one more of each unit
    const int64_t most = std::min<int64_t>(units, 2 * sms);
    const int64_t pieces = std::min(PT_CHUNKS * most, PT_FILL * static_cast<int64_t>(sms)) + most;
    s.rows = s.split ? pieces * PT_ROWS : 0;
    s.recs = s.split ? B + 1 : 0;
  }
  return s;
}
size_t up256(size_t x) { return (x + 255) & ~size_t(255); }
}  // namespace

// Scratch of one call. It rises with every size but a prompt's tokens: units stay whole from paged_attn_split_tokens
// on, and need none.
size_t paged_attn_workspace(int64_t T, int64_t B, int64_t H, int64_t G, int64_t D, int64_t groups, bool decode, int sms) {
  const Sizes s = sizes_of(T, B, H, G, groups, decode, sms);
  return 256 + 2 * up256(s.recs * 8) + up256(s.rows * 8) + up256(s.rows * D * 4);
}

// The most tokens of prompts whose units may be cut: the last T with H * (T / utok) < 2 * sms.
int64_t paged_attn_split_tokens(int64_t H, int64_t G, int sms) {
  const int64_t utok = 2 * (128 / G);
  return ((2 * static_cast<int64_t>(sms) - 1) / H + 1) * utok - 1;
}

template <int D, bool BF16, bool DEC>
static cudaError_t launch_paged_t(PagedAttn& p, uint8_t* ws, int sms, cudaStream_t st) {
  using C = PtCfg<D>;
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  const Sizes s = sizes_of(p.T, p.B, p.H, p.G, p.groups, p.decode, sms);
  p.counter = reinterpret_cast<unsigned*>(ws);
  p.rec_ctas = reinterpret_cast<Ctas*>(ws + 64);
  ws += 256;
  p.rec_cost = reinterpret_cast<int64_t*>(ws);
  ws += up256(s.recs * 8);
  p.rec_row = reinterpret_cast<int64_t*>(ws);
  ws += up256(s.recs * 8);
  p.part_s = reinterpret_cast<float2*>(ws);
  ws += up256(s.rows * 8);
  p.part_o = reinterpret_cast<float*>(ws);
  p.may_split = s.split;
  p.num_ctas = sms;
  // Sixteenths of a microsecond with all SMs at work, from traces: 2 to begin and end a unit; 2 for a pair of tiles over
  // 128 keys of 128 (of 64: 1.5); 1.5 (0.75) for 128 keys of one token, which bytes bound. 1 to 4 for the first and 1.6 to
  // 2.5 for the second were within 5 % over shared prefixes, or slower.
  p.w_start = 32;
  p.w_pair = D == 128 ? 32 : 24;
  p.w_thin = D == 128 ? 24 : 12;
  auto kfn = paged_attn_kernel<D, BF16, DEC>;
  // the limit is raised once per device: asking for it costs a microsecond
  static std::atomic<bool> raised[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev >= 64 || !raised[dev].load(std::memory_order_relaxed))) {
    e = cudaFuncSetAttribute(kfn, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    if (e == cudaSuccess && dev < 64) raised[dev].store(true, std::memory_order_relaxed);
  }
  if (e != cudaSuccess) return e;
  kfn<<<sms, PT_THREADS, C::SMEM, st>>>(p);
  e = cudaGetLastError();
  if (e != cudaSuccess || !s.split) return e;
  cudaLaunchConfig_t cfg = {};
  const int64_t rows = static_cast<int64_t>(p.T) * p.H * p.G;
  const bool wide = DEC && rows <= 6 * sms;
  cfg.gridDim = dim3(static_cast<unsigned>(wide ? rows : (rows + 3) / 4));
  cfg.blockDim = dim3(128);
  cfg.stream = st;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  if constexpr (DEC) return cudaLaunchKernelEx(&cfg, wide ? decode_join_kernel<D, T, 4> : decode_join_kernel<D, T, 1>, p);
  else return cudaLaunchKernelEx(&cfg, prompt_join_kernel<D, T>, p);
}

cudaError_t launch_paged_attn(int dtype, int head_dim, PagedAttn& p, uint8_t* ws, int sms, cudaStream_t st) {
  const bool b = dtype == BF16;
  if (head_dim == 128 && p.decode) return b ? launch_paged_t<128, true, true>(p, ws, sms, st) : launch_paged_t<128, false, true>(p, ws, sms, st);
  if (head_dim == 128) return b ? launch_paged_t<128, true, false>(p, ws, sms, st) : launch_paged_t<128, false, false>(p, ws, sms, st);
  if (p.decode) return b ? launch_paged_t<64, true, true>(p, ws, sms, st) : launch_paged_t<64, false, true>(p, ws, sms, st);
  return b ? launch_paged_t<64, true, false>(p, ws, sms, st) : launch_paged_t<64, false, false>(p, ws, sms, st);
}

}  // namespace dab
