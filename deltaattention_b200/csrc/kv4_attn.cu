// Single-token attention over a decode history in 4 bits and an exact window in 16 bits.
//
// z_hj = sm_scale * q_h . k_j, p_hj = count_j exp(z_hj - max_h), out_h = sum_j p_hj v_j / sum_j p_hj.
// With k_jd = zero_jg + scale_jg code_jd (g = d / 32) both products are sums over codes:
//   q . k_j  = sum_g scale_jg (sum_{d in g} q_d code_jd) + sum_g zero_jg qsum_g
//   sum_j p_j v_jd = sum_j (p_j scale_jg) code_jd + sum_j p_j zero_jg
// so the matrix instructions take the codes themselves, and nothing is dequantised.
//  * Scores: keys are the rows of the product, q-heads its 8 columns. A code alone in the low byte
//    of a half is an fp16 subnormal, code 2^-24 or code 2^-20: one shift and four ands give 8
//    operands, and nothing has to be taken off again. q goes in as fp16, scaled by a power of two so
//    that its largest element is in [2^13, 2^14), every second pair by 2^-4 of that: what is below
//    2^-26 of the largest is rounded, all else exact. One accumulator per group, multiplied by the
//    group's scale in fp32. The zeros are one more product: their coefficients, the sums of q, go in
//    as three bf16 parts (24 bits).
//    (16-bit numbers 256 + code and 16 + code, the offsets taken off with the zeros, took two shifts,
//    one product more and lost 4 bits of the sums; 8-bit float operands took a quarter longer: this
//    matrix path converts them to fp16 first.)
//  * Values: elements are the rows, q-heads the columns, in bf16, whose range the scales need. Up to
//    255 a byte is a bf16 number too, byte 2^-133, so again a shift and four ands give 8 operands.
//    The weights carry 2^64, which keeps products in fp32's normal range: scales from 2^-40 and values
//    below 2^50 have it all. p scale_g goes in as two bf16 parts, high and the rest (16 bits of every
//    weight); p alone, in two parts, times the stored (scales, zeros) gives the zeros' share.
//    (Numbers 16 + code took a shift for every operand.)
//    The zeros are added to the codes' sums after every tile. Over a long history of flat weights both
//    are hundreds of times larger than what is left of them, and a product rounds the sum it adds to
//    towards zero: added at the end, 100003 entries were 4e-6 of the terms off, all in one
//    direction, 25 times the rounding of an fp16 output. Tile by tile, 1e-9 (8 shuffles and 32 FMA a
//    tile, 3 us of the 73 below).
//    With up to 4 q-heads the columns 4 to 7 hold them again: the first parts go into columns 0 to 3,
//    the rest into 4 to 7, and one product does for two (73 us where 8 q-heads take 77, below).
#include <algorithm>
#include <atomic>
#include <cfloat>

#include "kv4.cuh"
#include "mma16.cuh"

namespace dab {

constexpr int KV4_NW = 4;      // warps per CTA, each with its own tiles and its own ring
constexpr int KV4_TILE = 32;   // keys per tile
constexpr int KV4_STAGES = 2;  // tiles in a warp's ring
constexpr int KV4_MAX_PIECES = 1024, KV4_MAX_HEADS = 2048;  // that are cut into pieces
// of a piece: two tiles a warp (8 heads of 8192: 10.5 us; pieces of 4: 12.6, of 12: 11.7)
constexpr int KV4_MIN_UNITS = 8;
// units that beginning and ending a head costs as much as (4 sequences of 65536 / 16 ragged ones with
// mass: 73.1 / 37.4 us; none: 74.9 / 38.6; 3: 74.4 / 37.9; 9: 72.7 / 36.9)
constexpr int KV4_START = 6;
constexpr int KV4_BIAS = 64;      // log2 of what history weights carry until they are joined with the window's
constexpr float KV4_SLACK = 8.f;  // log2 units a score may exceed the running maximum by before it moves

// one stage of a warp's ring
template <int D>
struct Kv4Stage {
  static constexpr int ROW = D / 2, SROW = D / 8;  // bytes of a row's codes, of its scales
  static constexpr int K = 0, V = KV4_TILE * ROW, KS = 2 * V, VS = KS + KV4_TILE * SROW, C = VS + KV4_TILE * SROW;
  static constexpr int BYTES = C + KV4_TILE * 4;
  // place of 16-byte piece c of row r: pieces are rotated so that the value loads, which take one
  // piece of every second row, meet different banks
  __device__ static int piece(int r, int c) { return r * ROW + ((D == 128 ? c ^ ((r >> 1) & 3) : c ^ ((r >> 2) & 1)) << 4); }
};

// copies of N bytes to shared memory, and of N or 0 (zeros are written)
template <int N>
__device__ __forceinline__ void cp_async(uint32_t dst, const void* src) {
  if constexpr (N == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(N) : "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_if(uint32_t dst, const void* src, bool valid) {
  if constexpr (N == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? N : 0) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(N), "r"(valid ? N : 0) : "memory");
}
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_next() { asm volatile("griddepcontrol.launch_dependents;"); }
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) { return __byte_perm(a, b, sel); }
__device__ __forceinline__ float lo_f32(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi_f32(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }
__device__ __forceinline__ uint32_t bmul2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t bfma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
__device__ __forceinline__ uint32_t bfms2(uint32_t a, uint32_t b, uint32_t c) {  // a b - c
  uint32_t d;
  asm("{\n\t.reg .b32 n;\n\tneg.bf16x2 n, %3;\n\tfma.rn.bf16x2 %0, %1, %2, n;\n\t}" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
// shared memory by 32-bit address
__device__ __forceinline__ uint32_t lds32(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t lds16(uint32_t at) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(at) : "memory");
  return v;
}
template <int N>
__device__ __forceinline__ void lds_words(uint32_t* w, uint32_t at) {
  if constexpr (N == 4)
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
  else if constexpr (N == 2)
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at) : "memory");
  else
    w[0] = lds32(at);
}
__device__ __forceinline__ void ldsm_x4_trans(uint32_t* r, uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void sts32(uint32_t at, uint32_t v) {
  asm volatile("st.shared.u32 [%0], %1;" ::"r"(at), "r"(v) : "memory");
}
__device__ __forceinline__ void sts16(uint32_t at, uint32_t v) {
  asm volatile("st.shared.u16 [%0], %1;" ::"r"(at), "h"(static_cast<uint16_t>(v)) : "memory");
}
__device__ __forceinline__ uint32_t movm(uint32_t x) {  // transpose of an 8 x 8 fragment of 16-bit numbers
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// x as a high T part and the rest, for two numbers
template <typename T>
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  hi = pack_t2<T>(x, y);
  float hx, hy;
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    hx = lo_f32(hi);
    hy = hi_f32(hi);
  } else {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    hx = f.x;
    hy = f.y;
  }
  lo = pack_t2<T>(x - hx, y - hy);
}

// What a warp keeps over its tiles: per lane the heads 2 t and 2 t + 1 (t = lane % 4).
template <int D>
struct Kv4Acc {
  float m[2], l[2];
  float o[D / 16][4];  // [2 g + i / 2]: element 32 g + 4 (lane / 4) + i in [2 (i % 2) + head]

  __device__ __forceinline__ void init() {
    m[0] = m[1] = -INFINITY;
    l[0] = l[1] = 0.f;
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
  }

  // Scores of 16 NT keys (lane: rows lane / 4 + 8 f of each 16, heads 2 t + e in [2 f + e]) to
  // weights. The maximum moves only when a score is KV4_SLACK above it: weights stay below
  // 2^KV4_SLACK, and the accumulators are hardly ever rescaled.
  template <int NT, int BIAS>
  __device__ __forceinline__ void weights(float (&z)[NT][4]) {
    float a = -INFINITY, b = -INFINITY;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      a = fmax3(a, z[i][0], z[i][2]);
      b = fmax3(b, z[i][1], z[i][3]);
    }
    if (__any_sync(0xFFFFFFFFu, a > m[0] + KV4_SLACK || b > m[1] + KV4_SLACK)) {
#pragma unroll
      for (int o_ = 4; o_ <= 16; o_ <<= 1) {
        a = fmaxf(a, __shfl_xor_sync(0xFFFFFFFFu, a, o_));
        b = fmaxf(b, __shfl_xor_sync(0xFFFFFFFFu, b, o_));
      }
      const float na = fmaxf(m[0], a), nb = fmaxf(m[1], b);
      const float fa = na == m[0] ? 1.f : ex2(m[0] - na), fb = nb == m[1] ? 1.f : ex2(m[1] - nb);
      m[0] = na;
      m[1] = nb;
      l[0] *= fa;
      l[1] *= fb;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        o[i][0] *= fa; o[i][1] *= fb;
        o[i][2] *= fa; o[i][3] *= fb;
      }
    }
    const float ra = (m[0] == -INFINITY ? 0.f : m[0]) - BIAS, rb = (m[1] == -INFINITY ? 0.f : m[1]) - BIAS;
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        z[i][e] = ex2(z[i][e] - (e & 1 ? rb : ra));
        l[e & 1] += z[i][e];
      }
  }
};

// q of up to 8 heads as column fragments of the score product, and the coefficients of the stored
// scales and zeros
template <typename T, int D, bool FOLD>
struct Kv4Query {
  static constexpr int NG = D / 32;
  uint32_t zc[2];        // coefficients of a row's zeros: sums of q in three parts
  float back[2];         // of heads 2 t, 2 t + 1: what takes the product to log2 units

  // `frag` gets the pairs (8 t + 2 half + {0, 1}, + 4) of every group, [group][lane][2 half + ..]
  __device__ __forceinline__ void load(const T* q, int64_t stride, int ng, float scale_log2, uint4* frag) {
    const int lane = threadIdx.x & 31, t = lane & 3, head = (lane >> 2) & (FOLD ? 3 : 7);
    uint4 w[NG];
    float top = 0.f;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      w[g] = make_uint4(0, 0, 0, 0);
      if (head < ng) w[g] = *reinterpret_cast<const uint4*>(q + head * stride + 32 * g + 8 * t);
      const T* e = reinterpret_cast<const T*>(&w[g]);
#pragma unroll
      for (int i = 0; i < 8; ++i) top = fmax_nan(top, fabsf(to_f32(e[i])));
    }
    top = fmax_nan(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
    top = fmax_nan(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
    // 2^k with top * 2^k in [2^13, 2^14); 1 for a row of zeros and one that is not finite
    const int ex = static_cast<int>(__float_as_uint(top) >> 23) - 127;
    const int k = top > 0.f && ex < 128 ? max(-126, min(126, 13 - ex)) : 0;
    const float f = __uint_as_float(static_cast<uint32_t>(k + 127) << 23);
    float qsum[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const T* e = reinterpret_cast<const T*>(&w[g]);
      float sum = 0.f;
      uint32_t b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // elements i, i + 4; odd i meet codes 2^4 higher
        const float u = i & 1 ? f * 0.0625f : f;
        const __half2 x = __floats2half2_rn(to_f32(e[i]) * u, to_f32(e[i + 4]) * u);
        const float2 y = __half22float2(x);
        b[i] = *reinterpret_cast<const uint32_t*>(&x);
        sum = fmaf(y.x + y.y, i & 1 ? 16.f : 1.f, sum);
      }
      if (threadIdx.x < 32) frag[g * 32 + lane] = make_uint4(b[0], b[1], b[2], b[3]);
#pragma unroll
      for (int o = 1; o <= 2; o <<= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
      qsum[g] = sum * 0x1p-24f;  // in units of the codes
    }
    // pairs of zeros; lane t takes pair t (NG = 4: pairs 0, 1, 0, 1; NG = 2: the only one)
    float x[2];
    const bool second = NG == 4 && (t & 1);
    x[0] = second ? qsum[NG - 2] : qsum[0];
    x[1] = second ? qsum[NG - 1] : qsum[1];
    uint32_t part[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      part[i] = pack_t2<__nv_bfloat16>(x[0], x[1]);
      x[0] -= lo_f32(part[i]);
      x[1] -= hi_f32(part[i]);
    }
    if constexpr (NG == 4) {
      zc[0] = t < 2 ? part[0] : part[1];
      zc[1] = t < 2 ? part[2] : 0u;
    } else {
      zc[0] = t == 0 ? part[0] : t == 1 ? part[1] : t == 2 ? part[2] : 0u;
      zc[1] = 0u;
    }
    // 2^24 2^-k; finite, so that a score of 0 stays one
    const float unit = scale_log2 * __uint_as_float(static_cast<uint32_t>(127 - k) << 23) * 0x1p24f;
    const float bk = fmaxf(fminf(unit, FLT_MAX), -FLT_MAX);
    back[0] = __shfl_sync(0xFFFFFFFFu, bk, 8 * t);
    back[1] = __shfl_sync(0xFFFFFFFFu, bk, 8 * t + 4);
  }
};

// Units of a head: tiles of 32 history entries, then tiles of 16 window rows; at least one, so that
// every head has a CTA that writes its output.
__device__ __forceinline__ int kv4_len(const Kv4Attn& p, int bh) {
  const int b = bh / p.H, h = bh - b * p.H;
  return max(0, min(p.lengths[b * p.lb + h * p.lh], p.cap));
}
__device__ __forceinline__ int kv4_units(int n, int elen) {
  return max(1, (n + KV4_TILE - 1) / KV4_TILE + (elen + 15) / 16);
}

// Units [u0, u1) of group z (8 q-heads) of head bh, by the whole CTA.
template <typename T, int D, bool MASS, bool FOLD>
__device__ __forceinline__ void kv4_segment(const Kv4Attn& p, uint8_t* smem, uint4* frag, int bh, int z, int n, int elen, int u0,
                                            int u1, int slot) {
  using St = Kv4Stage<D>;
  constexpr int NG = D / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t = lane & 3, gq = lane >> 2;
  const int b = bh / p.H, h = bh - b * p.H;
  const int h0 = z * 8, ng = min(8, p.G - h0);
  const int n4 = (n + KV4_TILE - 1) / KV4_TILE;
  const int64_t row0 = static_cast<int64_t>(bh) * p.G + h0;

  // Shared-memory addresses of this lane in the first stage of its warp's ring; rows 8 and 16 further
  // have the same rotation (Kv4Stage::piece).
  constexpr int PPR = St::ROW / 16;  // 16-byte pieces per row
  const uint32_t ring = smem_u32(smem) + warp * (KV4_STAGES * St::BYTES);
  const uint32_t k_at = ring + St::K + (NG == 4 ? St::piece(gq, t) : St::piece(gq, t >> 1) + 8 * (t & 1));
  const uint32_t v_at = ring + St::V + (NG == 4 ? St::piece(2 * t, gq >> 1) : St::piece(2 * t, gq >> 2) + 8 * ((gq >> 1) & 1));
  const uint32_t ks_at = ring + St::KS + gq * St::SROW, vs_at = ring + St::VS + 2 * t * St::SROW;
  const uint32_t vl_at = ring + St::VS + ((lane & 7) + ((lane >> 1) & 8)) * St::SROW;  // for ldmatrix
  const uint32_t zk_at = ks_at + 2 * NG + (NG == 4 ? 4 * (t & 1) : 0);  // a pair of zeros
  // A lane copies pieces lane + 32 i of a tile's codes (they are contiguous), its row's scales and
  // count.
  const int last = min(u1, n4);  // history tiles of this segment end here
  int next = u0 + warp;          // the next tile to copy
  const uint8_t *kp, *vp, *ksp, *vsp;
  const int32_t* cp;
  {
    const int64_t r = static_cast<int64_t>(next) * KV4_TILE;
    kp = p.hist.k_codes + b * p.hist.cb + h * p.hist.ch + r * St::ROW + lane * 16;
    vp = p.hist.v_codes + b * p.hist.cb + h * p.hist.ch + r * St::ROW + lane * 16;
    ksp = reinterpret_cast<const uint8_t*>(p.hist.k_scales + b * p.hist.sb + h * p.hist.sh) + (r + lane) * St::SROW;
    vsp = reinterpret_cast<const uint8_t*>(p.hist.v_scales + b * p.hist.sb + h * p.hist.sh) + (r + lane) * St::SROW;
    cp = p.counts + b * p.mb + h * p.mh + r + lane;
  }
  const uint32_t code_at = ring + St::piece(lane / PPR, lane % PPR), row_at = ring + lane * St::SROW;
  auto issue = [&](int stage) {
    if (next < last) {
      const int rem = n - next * KV4_TILE;
      const uint32_t code = code_at + stage * St::BYTES, row = row_at + stage * St::BYTES;
      if (rem >= KV4_TILE) {
#pragma unroll
        for (int i = 0; i < PPR; ++i) {
          cp_async<16>(code + St::K + 512 * i, kp + 512 * i);
          cp_async<16>(code + St::V + 512 * i, vp + 512 * i);
        }
        cp_async<St::SROW>(row + St::KS, ksp);
        cp_async<St::SROW>(row + St::VS, vsp);
        cp_async<4>(row - lane * (St::SROW - 4) + St::C, cp);
      } else {  // rows past the end are filled with zeros (count 0 masks them), read from the first row: nothing
#pragma unroll
        for (int i = 0; i < PPR; ++i) {
          const bool ok = lane / PPR + i * (32 / PPR) < rem;
          cp_async_if<16>(code + St::K + 512 * i, ok ? kp + 512 * i : kp - lane * 16, ok);
          cp_async_if<16>(code + St::V + 512 * i, ok ? vp + 512 * i : vp - lane * 16, ok);
        }
        const bool ok = lane < rem;
        cp_async_if<St::SROW>(row + St::KS, ok ? ksp : ksp - lane * St::SROW, ok);
        cp_async_if<St::SROW>(row + St::VS, ok ? vsp : vsp - lane * St::SROW, ok);
        cp_async_if<4>(row - lane * (St::SROW - 4) + St::C, ok ? cp : cp - lane, ok);
      }
      next += KV4_NW;
      kp += KV4_NW * KV4_TILE * St::ROW;
      vp += KV4_NW * KV4_TILE * St::ROW;
      ksp += KV4_NW * KV4_TILE * St::SROW;
      vsp += KV4_NW * KV4_TILE * St::SROW;
      cp += KV4_NW * KV4_TILE;
    }
    cp_commit();
  };
#pragma unroll
  for (int s = 0; s < KV4_STAGES - 1; ++s) issue(s);

  const T* qp = static_cast<const T*>(p.q) + b * p.qb + (static_cast<int64_t>(h) * p.G + h0) * p.qh;
  Kv4Query<T, D, FOLD> q;
  q.load(qp, p.qh, ng, p.scale_log2, frag);
  __syncthreads();  // the fragments are there
  Kv4Acc<D> acc;
  acc.init();
  float* sc0 = MASS ? p.scores + (row0 + 2 * t) * p.sstride + gq : nullptr;
  const uint32_t frag_at = smem_u32(frag + lane);
  // A tile's value scales by group, in the order in which lanes want them: a lane's keys 2 t, 2 t + 1,
  // 2 t + 8, 2 t + 9 of each 16 (the lane of a key writes them; 8 selections a lane and 16 keys saved)
  __shared__ __align__(16) uint8_t turned[KV4_NW * NG * 64];
  const uint32_t turn = smem_u32(turned) + warp * (NG * 64), turn_r = turn + 16 * t;
  const uint32_t turn_w = turn + 8 * (lane & 6) + 8 * (lane >> 4) + 4 * ((lane >> 3) & 1) + 2 * (lane & 1);
  const bool head0 = 2 * t < ng, head1 = 2 * t + 1 < ng;
  const bool second = FOLD && gq >= 4;  // this lane's column takes the second parts

  int unit = u0 + warp, stage = 0;
  for (; unit < last; unit += KV4_NW) {
    cp_wait<KV4_STAGES - 2>();
    __syncwarp();  // and every lane has read the tile before this one: its stage may be filled again
    issue(stage == 0 ? KV4_STAGES - 1 : stage - 1);
    const uint32_t su = stage * St::BYTES;  // the last term of addresses: the same for all lanes
    // log2 of the counts; entries that take no part have -inf, and their scales, which may be
    // anything, are set to 0
    const int32_t count = static_cast<int32_t>(lds32((ring + 4 * lane) + su + St::C));
    sts32((ring + 4 * lane) + su + St::C, __float_as_uint(count > 0 ? lg2(static_cast<float>(count)) : -INFINITY));
    uint32_t own[NG / 2];
    lds_words<NG / 2>(own, ring + lane * St::SROW + su + St::VS);
#pragma unroll
    for (int g = 0; g < NG; ++g) sts16(turn_w + g * 64, count > 0 ? (g & 1 ? own[g >> 1] >> 16 : own[g >> 1]) : 0u);
    if (count <= 0) {
#pragma unroll
      for (int i = 0; i < St::SROW / 4; ++i) {
        sts32((ring + lane * St::SROW) + su + St::KS + 4 * i, 0u);
        sts32((ring + lane * St::SROW) + su + St::VS + 4 * i, 0u);
      }
    }
    __syncwarp();
    // ---- scores
    float zs[2][4];
    {
      uint32_t w[2][2][NG], s2[2][2][NG / 2];  // codes (word g) and scale pairs of rows 16 i + 8 f + gq
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int f = 0; f < 2; ++f) {
          const int r = 16 * i + 8 * f;
          lds_words<NG>(w[i][f], k_at + su + r * St::ROW);
          lds_words<NG / 2>(s2[i][f], ks_at + su + r * St::SROW);
        }
        uint32_t zw[2];  // pairs of zeros of both rows, the same for every part
#pragma unroll
        for (int f = 0; f < 2; ++f) zw[f] = lds32(zk_at + su + (16 * i + 8 * f) * St::SROW);
        mma16816_set<__nv_bfloat16>(zs[i], zw[0], zw[1], zw[0], zw[1], q.zc[0], q.zc[1]);
      }
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        uint32_t qf[4];
        lds_words<4>(qf, frag_at + g * 512);
        float a[2][4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t x[2] = {w[i][0][g], w[i][1][g]};
          mma16816_set<__half>(a[i], x[0] & 0x000F000Fu, x[1] & 0x000F000Fu, x[0] & 0x00F000F0u, x[1] & 0x00F000F0u, qf[0], qf[1]);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t x[2] = {w[i][0][g] >> 8, w[i][1][g] >> 8};
          mma16816<__half>(a[i], x[0] & 0x000F000Fu, x[1] & 0x000F000Fu, x[0] & 0x00F000F0u, x[1] & 0x00F000F0u, qf[2], qf[3]);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float xa = g & 1 ? hi_f32(s2[i][0][g >> 1]) : lo_f32(s2[i][0][g >> 1]);
          const float xb = g & 1 ? hi_f32(s2[i][1][g >> 1]) : lo_f32(s2[i][1][g >> 1]);
          zs[i][0] = fmaf(xa, a[i][0], zs[i][0]);
          zs[i][1] = fmaf(xa, a[i][1], zs[i][1]);
          zs[i][2] = fmaf(xb, a[i][2], zs[i][2]);
          zs[i][3] = fmaf(xb, a[i][3], zs[i][3]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        const float lg = __uint_as_float(lds32((ring + 4 * gq) + su + St::C + 64 * i + 32 * f));
        zs[i][2 * f] = fmaf(zs[i][2 * f], q.back[0], lg);
        zs[i][2 * f + 1] = fmaf(zs[i][2 * f + 1], q.back[1], lg);
      }
      if constexpr (MASS) {  // the rows of the workspace have room for whole tiles
        float* o = sc0 + static_cast<int64_t>(unit) * KV4_TILE + 16 * i;
        if (head0) { o[0] = zs[i][0]; o[8] = zs[i][2]; }
        if (head1) { o[p.sstride] = zs[i][1]; o[p.sstride + 8] = zs[i][3]; }
      }
    }
    // value codes of keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9 and their scales in pairs; those of the first
    // 16 keys are loaded before the exponentials, which hide the latency
    uint32_t w[4][NG], s[NG][2];
    auto load_values = [&](int i) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int r = 16 * i + (k & 1) + 8 * (k >> 1);
        lds_words<NG>(w[k], v_at + su + r * St::ROW);
      }
#pragma unroll
      for (int g = 0; g < NG; ++g) lds_words<2>(s[g], turn_r + g * 64 + 8 * i);
    };
    load_values(0);
    acc.template weights<2, KV4_BIAS>(zs);
    // ---- values
    float sz[4] = {0.f, 0.f, 0.f, 0.f};  // the tile's sums of p zero_g: value lane / 4 of the stored row in [0], [1]
    uint32_t ph[2][2], pl[2][2];  // weights of keys 2 t, 2 t + 1 (+ 8) for head lane / 4, two parts
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        split2<__nv_bfloat16>(zs[i][2 * f], zs[i][2 * f + 1], ph[i][f], pl[i][f]);
        ph[i][f] = movm(ph[i][f]);
        pl[i][f] = movm(pl[i][f]);
      }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (i) load_values(1);
      // sums of p zero: rows are the stored values (and again, for whole operands)
      using B = __nv_bfloat16;
      uint32_t v[4];
      if constexpr (NG == 4) {
        ldsm_x4_trans(v, vl_at + su + 16 * i * St::SROW);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          v[k] = lds16(vs_at + su + 2 * (gq & 3) + (16 * i + (k & 1) + 8 * (k >> 1)) * St::SROW);
        v[0] = v[1] = prmt(v[0], v[1], 0x5410);
        v[2] = v[3] = prmt(v[2], v[3], 0x5410);
      }
      mma16816<B>(sz, v[0], v[1], v[2], v[3], second ? pl[i][0] : ph[i][0], second ? pl[i][1] : ph[i][1]);
      if constexpr (!FOLD) mma16816<B>(sz, v[0], v[1], v[2], v[3], pl[i][0], pl[i][1]);
      const uint32_t half = gq & 1 ? 0x7632u : 0x5410u;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        uint32_t wh[2], wl[2], x[2];
#pragma unroll
        for (int f = 0; f < 2; ++f) {
          const uint32_t sc = s[g][f];
          wh[f] = bmul2(ph[i][f], sc);
          wl[f] = bfma2(pl[i][f], sc, bfms2(ph[i][f], sc, wh[f]));
          if constexpr (FOLD) wh[f] = second ? wl[f] : wh[f];
          x[f] = prmt(w[2 * f][g], w[2 * f + 1][g], half);
        }
        const uint32_t y[2] = {x[0] >> 8, x[1] >> 8};
        const uint32_t a[4] = {x[0] & 0x000F000Fu, x[0] & 0x00F000F0u, x[1] & 0x000F000Fu, x[1] & 0x00F000F0u};
        const uint32_t d[4] = {y[0] & 0x000F000Fu, y[0] & 0x00F000F0u, y[1] & 0x000F000Fu, y[1] & 0x00F000F0u};
        mma16816<B>(acc.o[2 * g], a[0], a[1], a[2], a[3], wh[0], wh[1]);
        mma16816<B>(acc.o[2 * g + 1], d[0], d[1], d[2], d[3], wh[0], wh[1]);
        if constexpr (!FOLD) {
          mma16816<B>(acc.o[2 * g], a[0], a[1], a[2], a[3], wl[0], wl[1]);
          mma16816<B>(acc.o[2 * g + 1], d[0], d[1], d[2], d[3], wl[0], wl[1]);
        }
      }
    }
    // the zeros, in the units of the codes
    constexpr float EVEN = 0x1p-133f, ODD = 0x1p-129f;
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const float z = __shfl_sync(0xFFFFFFFFu, sz[e], 4 * (NG + g) + t);
        acc.o[2 * g][e] = fmaf(z, EVEN, acc.o[2 * g][e]);
        acc.o[2 * g][2 + e] = fmaf(z, ODD, acc.o[2 * g][2 + e]);
        acc.o[2 * g + 1][e] = fmaf(z, EVEN, acc.o[2 * g + 1][e]);
        acc.o[2 * g + 1][2 + e] = fmaf(z, ODD, acc.o[2 * g + 1][2 + e]);
      }
    stage = stage == KV4_STAGES - 1 ? 0 : stage + 1;
  }
  cp_wait<0>();

  // sums of codes to values: their units and the weights' bias
  static_assert(KV4_BIAS == 64, "2^(133 - 64), 2^(129 - 64), 2^-64");
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    acc.l[e] *= 0x1p-64f;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      acc.o[i][e] *= 0x1p69f;
      acc.o[i][2 + e] *= 0x1p65f;
    }
  }

  // ---- window rows, 16 at a time, straight from memory
  const T* ke = static_cast<const T*>(p.k_exact) + b * p.eb + h * p.eh;
  const T* ve = static_cast<const T*>(p.v_exact) + b * p.eb + h * p.eh;
  uint32_t qw[NG][2][2];  // pairs (8 t + 2 half + {0, 1}, + 4) of each group, as rows are read below
  if (unit < u1) {
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      uint4 w = make_uint4(0, 0, 0, 0);
      const int head = gq & (FOLD ? 3 : 7);
      if (head < ng) w = *reinterpret_cast<const uint4*>(qp + head * p.qh + 32 * g + 8 * t);
      qw[g][0][0] = prmt(w.x, w.z, 0x5410);
      qw[g][0][1] = prmt(w.x, w.z, 0x7632);
      qw[g][1][0] = prmt(w.y, w.w, 0x5410);
      qw[g][1][1] = prmt(w.y, w.w, 0x7632);
    }
  }
  for (; unit < u1; unit += KV4_NW) {
    const int j0 = (unit - n4) * 16;
    float zs[1][4];
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    const bool okr[2] = {j0 + gq < elen, j0 + gq + 8 < elen};
    uint4 ka[NG], kb[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      ka[g] = kb[g] = make_uint4(0, 0, 0, 0);
      if (okr[0]) ka[g] = *reinterpret_cast<const uint4*>(ke + static_cast<int64_t>(j0 + gq) * p.en + 32 * g + 8 * t);
      if (okr[1]) kb[g] = *reinterpret_cast<const uint4*>(ke + static_cast<int64_t>(j0 + gq + 8) * p.en + 32 * g + 8 * t);
    }
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      mma16816<T>(s, prmt(ka[g].x, ka[g].z, 0x5410), prmt(kb[g].x, kb[g].z, 0x5410), prmt(ka[g].x, ka[g].z, 0x7632),
                  prmt(kb[g].x, kb[g].z, 0x7632), qw[g][0][0], qw[g][0][1]);
      mma16816<T>(s, prmt(ka[g].y, ka[g].w, 0x5410), prmt(kb[g].y, kb[g].w, 0x5410), prmt(ka[g].y, ka[g].w, 0x7632),
                  prmt(kb[g].y, kb[g].w, 0x7632), qw[g][1][0], qw[g][1][1]);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool ok = okr[e >> 1];
      zs[0][e] = ok ? s[e] * p.scale_log2 : -INFINITY;
      if (MASS && (e & 1 ? head1 : head0) && ok) sc0[(e & 1) * p.sstride + p.wcol + j0 + 8 * (e >> 1)] = zs[0][e];
    }
    acc.template weights<1, 0>(zs);
    uint32_t ph[2], pl[2];
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      split2<T>(zs[0][2 * f], zs[0][2 * f + 1], ph[f], pl[f]);
      if constexpr (FOLD) {  // column 4 + j: the second part of head j
        ph[f] = movm(t < 2 ? ph[f] : pl[f]);
      } else {
        ph[f] = movm(ph[f]);
        pl[f] = movm(pl[f]);
      }
    }
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      uint2 x[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int j = j0 + 2 * t + (k & 1) + 8 * (k >> 1);
        x[k] = make_uint2(0u, 0u);
        if (j < elen) x[k] = *reinterpret_cast<const uint2*>(ve + static_cast<int64_t>(j) * p.en + 32 * g + 4 * gq);
      }
      const uint32_t a[4] = {prmt(x[0].x, x[1].x, 0x5410), prmt(x[0].x, x[1].x, 0x7632), prmt(x[2].x, x[3].x, 0x5410),
                             prmt(x[2].x, x[3].x, 0x7632)};
      const uint32_t d[4] = {prmt(x[0].y, x[1].y, 0x5410), prmt(x[0].y, x[1].y, 0x7632), prmt(x[2].y, x[3].y, 0x5410),
                             prmt(x[2].y, x[3].y, 0x7632)};
      mma16816<T>(acc.o[2 * g], a[0], a[1], a[2], a[3], ph[0], ph[1]);
      mma16816<T>(acc.o[2 * g + 1], d[0], d[1], d[2], d[3], ph[0], ph[1]);
      if constexpr (!FOLD) {
        mma16816<T>(acc.o[2 * g], a[0], a[1], a[2], a[3], pl[0], pl[1]);
        mma16816<T>(acc.o[2 * g + 1], d[0], d[1], d[2], d[3], pl[0], pl[1]);
      }
    }
  }
  if constexpr (FOLD) {
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc.o[i][e] += __shfl_xor_sync(0xFFFFFFFFu, acc.o[i][e], 2);
  }

  // ---- the warps' parts to one: common maximum, then sums through shared memory
  __shared__ float sm_m[KV4_NW][8], sm_l[KV4_NW][8];
#pragma unroll
  for (int o_ = 4; o_ <= 16; o_ <<= 1) {
    acc.l[0] += __shfl_xor_sync(0xFFFFFFFFu, acc.l[0], o_);
    acc.l[1] += __shfl_xor_sync(0xFFFFFFFFu, acc.l[1], o_);
  }
  if (gq == 0) {
    sm_m[warp][2 * t] = acc.m[0];
    sm_m[warp][2 * t + 1] = acc.m[1];
  }
  __syncthreads();  // and every warp is done with its ring
  float f[2], mm[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    float m = sm_m[0][2 * t + e];
#pragma unroll
    for (int w = 1; w < KV4_NW; ++w) m = fmaxf(m, sm_m[w][2 * t + e]);
    mm[e] = m;
    f[e] = acc.m[e] == m ? 1.f : ex2(acc.m[e] - m);  // a warp without keys has 0 accumulators
  }
  if (gq == 0) {
    sm_l[warp][2 * t] = acc.l[0] * f[0];
    sm_l[warp][2 * t + 1] = acc.l[1] * f[1];
  }
  // [head][element], rows padded against bank conflicts
  constexpr int OR = D + 4;
  float* so = reinterpret_cast<float*>(smem) + warp * 8 * OR;
#pragma unroll
  for (int g = 0; g < NG; ++g)
#pragma unroll
    for (int e = 0; e < 2; ++e)
      *reinterpret_cast<float4*>(so + (2 * t + e) * OR + 32 * g + 4 * gq) =
          make_float4(acc.o[2 * g][e] * f[e], acc.o[2 * g][2 + e] * f[e], acc.o[2 * g + 1][e] * f[e],
                      acc.o[2 * g + 1][2 + e] * f[e]);
  __syncthreads();
  const float* base = reinterpret_cast<const float*>(smem);
  for (int i = threadIdx.x; i < ng * (D / 4); i += KV4_NW * 32) {
    const int hd = i / (D / 4), d = (i - hd * (D / 4)) * 4;
    float4 a = *reinterpret_cast<const float4*>(base + hd * OR + d);
    float l = sm_l[0][hd];
#pragma unroll
    for (int w = 1; w < KV4_NW; ++w) {
      const float4 x = *reinterpret_cast<const float4*>(base + (w * 8 + hd) * OR + d);
      a.x += x.x; a.y += x.y; a.z += x.z; a.w += x.w;
      l += sm_l[w][hd];
    }
    if (slot < 0) {  // the whole head: its output
      const float inv = l == 0.f ? 0.f : 1.f / l;
      T* o = static_cast<T*>(p.out) + b * p.ob + (static_cast<int64_t>(h) * p.G + h0 + hd) * p.oh + d;
      o[0] = from_f32<T>(a.x * inv); o[1] = from_f32<T>(a.y * inv);
      o[2] = from_f32<T>(a.z * inv); o[3] = from_f32<T>(a.w * inv);
    } else {
      *reinterpret_cast<float4*>(p.part + (static_cast<int64_t>(slot) * 8 + hd) * D + d) = a;
    }
  }
  if (warp == 0 && gq == 0) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int hd = 2 * t + e;
      float l = sm_l[0][hd];
#pragma unroll
      for (int w = 1; w < KV4_NW; ++w) l += sm_l[w][hd];
      if (hd < ng) {
        if (slot < 0) p.row_stats[row0 + hd] = make_float2(mm[e] == -INFINITY ? 0.f : mm[e], l == 0.f ? 0.f : 1.f / l);
        else p.stats[slot * 8 + hd] = make_float2(mm[e], l);
      }
    }
  }
  __syncthreads();  // the ring may be filled again
}

// Bound by what the SMs issue: 16 keys take a warp about 335 instructions, 18 of them products, which
// hold up the other pipes too, so that 62 % of the issue slots are used. Copies are not what it waits
// for: with all tiles from one address an earlier form took 8 % less. 12 warps an SM of 168 registers;
// 16 of 128 registers spill and took 7 % longer, a ring of 3 tiles changed nothing. bf16, d = 128, 4
// q-heads per kv-head, device times with the join:
//   4 sequences of 65536 entries a head, 8 kv-heads (346 MB): 73 us, 4.7 TB/s
//   16 sequences of 1024 to 8192 entries, 8 kv-heads (108 MB): 32 us, with mass 37 us
//   1 sequence of 8192 entries: 10.5 us, most of it the latencies of two launches
//
// With `splits` every head is cut into that many pieces (as many as it has units). Otherwise the
// units of all heads in a row are cut into even pieces, one per CTA, whatever the heads' lengths: all
// CTAs run at once and end together, and a piece may begin and end inside a head. Heads in several
// pieces are joined from their parts (a CTA's first segment is its part 0, a later one its part 1), a
// head inside one piece is written here.
template <typename T, int D, bool MASS, bool FOLD>
__global__ void __launch_bounds__(KV4_NW * 32, D == 64 ? 4 : 3) kv4_attn_kernel(const __grid_constant__ Kv4Attn p) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint4 frag[D];  // q's fragments: D / 32 groups of 32 lanes
  __shared__ int64_t warp_sum[KV4_NW];
  __shared__ int lens[KV4_MAX_HEADS];
  __shared__ int s_bh, s_at;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, hg = (p.G + 7) / 8;
  grid_next();  // the joining CTAs take the places that ending CTAs leave, and wait there for the last
  int elen = p.exact_len;
  if (p.state) elen = static_cast<int>(max(int64_t{0}, min(static_cast<int64_t>(p.W), p.state[0] + p.lag)));
  if (p.state && blockIdx.x == 0 && tid == 0) *p.used = elen;
  // this piece: `left` units from unit `at` of head `bh` (all its groups of q-heads in a row)
  int bh, at, ns = 1, split = 0;
  int64_t left, start = 0, piece = 1;
  if (p.splits) {
    const int w = blockIdx.x / p.splits, z = w % hg;
    bh = w / hg;
    split = blockIdx.x - w * p.splits;
    const int un = kv4_units(kv4_len(p, bh), elen);
    ns = min(p.splits, un);
    if (split >= ns) return;
    const int u0 = static_cast<int>(static_cast<int64_t>(un) * split / ns);
    left = static_cast<int64_t>(un) * (split + 1) / ns - u0;
    at = z * un + u0;
  } else {
    // where it begins: the heads' units summed up, each thread a run of heads
    const int heads = p.B * p.H, per = (heads + KV4_NW * 32 - 1) / (KV4_NW * 32);
    for (int k = tid; k < heads; k += KV4_NW * 32) lens[k] = kv4_len(p, k);
    __syncthreads();
    int64_t mine = 0;
    for (int k = tid * per; k < min(heads, (tid + 1) * per); ++k) mine += kv4_units(lens[k], elen) + KV4_START;
    mine *= hg;
    int64_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t v = __shfl_up_sync(0xFFFFFFFFu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) warp_sum[warp] = incl;
    __syncthreads();
    int64_t first = incl - mine, total = 0;
#pragma unroll
    for (int w = 0; w < KV4_NW; ++w) {
      if (w < warp) first += warp_sum[w];
      total += warp_sum[w];
    }
    const int64_t up = total + p.pieces - 1;
    piece = up >> 32 ? up / p.pieces : static_cast<uint32_t>(up) / static_cast<uint32_t>(p.pieces);
    piece = max(piece, static_cast<int64_t>(KV4_MIN_UNITS));
    start = piece * blockIdx.x;
    if (start >= total) return;
    left = min(piece, total - start);
    if (first <= start && start < first + mine) {
      int k = tid * per;
      int64_t pos = first;
      while (true) {
        const int64_t u = static_cast<int64_t>(hg) * (kv4_units(lens[k], elen) + KV4_START);
        if (start < pos + u) break;
        pos += u;
        ++k;
      }
      s_bh = k;
      s_at = static_cast<int>(start - pos);
    }
    __syncthreads();
    bh = s_bh;
    at = s_at;
  }
  const int ahead = p.splits ? 0 : KV4_START;  // units before a head's first that stand for its cost
  for (int part = 0; left > 0;) {
    const int n = p.splits ? kv4_len(p, bh) : lens[bh], un = kv4_units(n, elen), z = at / (un + ahead);
    const int v0 = at - z * (un + ahead), v1 = static_cast<int>(min(static_cast<int64_t>(un + ahead), v0 + left));
    const int u0 = max(0, v0 - ahead), u1 = v1 - ahead;
    if (u0 < u1) {
      int slot = -1;
      if (u1 - u0 < un) slot = blockIdx.x * 2 + part;
      if (u0 == 0 && tid == 0) {
        // the head's first part and its last piece; -1: no parts
        int2 info = make_int2(-1, 0);
        if (slot >= 0) {
          info = make_int2(slot, p.splits ? static_cast<int>(blockIdx.x) + ns - 1
                                          : static_cast<int>((start - v0 + ahead + un - 1) / piece));
        }
        p.info[bh * hg + z] = info;
      }
      kv4_segment<T, D, MASS, FOLD>(p, smem, frag, bh, z, n, elen, u0, u1, slot);
      part = 1;
    }
    left -= v1 - v0;
    start += v1 - v0;
    at += v1 - v0;
    if (at == hg * (un + ahead)) {
      at = 0;
      ++bh;
    }
  }
}

// ---------------------------------------------------------------------------------- joining
// Launched while the attention kernel ends (programmatic dependent launch): grid_wait returns once
// that kernel's writes are there. Joining is a chain of dependent reads (the head's parts, their
// maxima and sums, their outputs), 5.3 us alone. The mass reads the scores again and adds 5 us for 16
// sequences of 1024 to 8192 entries: 4 G bytes a key written and read, where a key has 5 D / 4. Four
// q-heads at a time keep enough of its CTAs resident (eight at a time: 1.6 us more).
// blockIdx.y: kv-head. The first G CTAs join the parts of one q-head each and write its output;
// the others add the weights of 1024 entries each (history, then window) to their mass.
constexpr int KV4_MASS_KEYS = 1024;

// part k of a row whose first part and last piece are `info`: part 0 of piece after piece
__device__ __forceinline__ int64_t part_of(int2 info, int k) { return k == 0 ? info.x : (info.x / 2 + k) * int64_t{2}; }

// (max, 1 / sum) of a row, by one warp; 1 / sum is 0 where nothing is left. A lane has the loads of 8
// parts in flight.
__device__ __forceinline__ float2 row_stats(const Kv4Attn& p, int64_t row, int head, int2 info, int lane) {
  if (info.x < 0) return p.row_stats[row];
  const int parts = info.y - info.x / 2 + 1;
  float m = -INFINITY, l = 0.f;
  for (int k0 = 0; k0 < parts; k0 += 256) {
    float2 s[8];
    float top = m;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int k = k0 + 32 * j + lane;
      s[j] = make_float2(-INFINITY, 0.f);
      if (k < parts) s[j] = p.stats[part_of(info, k) * 8 + head];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) top = fmaxf(top, s[j].x);
    const float ref = top == -INFINITY ? 0.f : top;
    l *= ex2(m - ref);
#pragma unroll
    for (int j = 0; j < 8; ++j) l = fmaf(s[j].y, ex2(s[j].x - ref), l);
    m = top;
  }
  float all = m;
#pragma unroll
  for (int o = 16; o; o >>= 1) all = fmaxf(all, __shfl_xor_sync(0xFFFFFFFFu, all, o));
  const float ref = all == -INFINITY ? 0.f : all;
  l *= ex2(m - ref);
#pragma unroll
  for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(0xFFFFFFFFu, l, o);
  return make_float2(ref, l == 0.f ? 0.f : 1.f / l);
}

template <typename T, int D>
__global__ void __launch_bounds__(256) kv4_join_kernel(const __grid_constant__ Kv4Attn p) {
  __shared__ float2 st[4];
  __shared__ float4 red[256];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, hg = (p.G + 7) / 8;
  const int bh = blockIdx.y, b = bh / p.H, h = bh - b * p.H;
  if (static_cast<int>(blockIdx.x) < p.G) {
    grid_wait();
    if (p.lag && (blockIdx.x | blockIdx.y) == 0 && threadIdx.x == 0) {
      // the step's length advance: this kernel reads the length that was used from the workspace
      p.state[0] += 1;
      p.state[1] += 1;
    }
    const int2 info = p.info[bh * hg + blockIdx.x / 8];
    if (info.x < 0) return;  // written already
    // a part's row is read by D / 4 lanes, and every warp works out the row's maximum and sum
    constexpr int LANES = D / 4, ROWS = 256 / LANES;
    const int parts = info.y - info.x / 2 + 1, head = blockIdx.x & 7;
    const int d = threadIdx.x % LANES, first = threadIdx.x / LANES;
    const float2 r = row_stats(p, 0, head, info, lane);
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int k = first; k < parts; k += ROWS) {
      const int64_t at = part_of(info, k) * 8 + head;
      const float w = ex2(p.stats[at].x - r.x) * r.y;
      const float4 x = *reinterpret_cast<const float4*>(p.part + at * D + 4 * d);
      a.x = fmaf(x.x, w, a.x);
      a.y = fmaf(x.y, w, a.y);
      a.z = fmaf(x.z, w, a.z);
      a.w = fmaf(x.w, w, a.w);
    }
    red[threadIdx.x] = a;
    __syncthreads();
    if (threadIdx.x < D) {
      const float* e = reinterpret_cast<const float*>(red) + threadIdx.x;
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < ROWS; ++i) sum += e[i * D];
      static_cast<T*>(p.out)[b * p.ob + (static_cast<int64_t>(h) * p.G + blockIdx.x) * p.oh + threadIdx.x] = from_f32<T>(sum);
    }
    return;
  }
  // 4 neighbouring entries a thread: history [0, cap), window from column wcol on
  const int n = max(0, min(p.lengths[b * p.lb + h * p.lh], p.cap));
  const int k0 = (blockIdx.x - p.G) * KV4_MASS_KEYS, key = k0 + 4 * threadIdx.x;
  if (k0 >= n && k0 + KV4_MASS_KEYS <= p.wcol) return;  // past the history, before the window
  float* mp = p.mass + b * p.mb + h * p.mh + key;
  float m[4], w[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 4; ++i) m[i] = key + i < n ? mp[i] : 0.f;  // read while the attention kernel ends
  grid_wait();
  const int elen = p.state ? *p.used : p.exact_len, j = key - p.wcol;
  if (k0 >= max(n, p.wcol + elen)) return;
  const bool some = key < n || (j >= 0 && j < elen);
  for (int g0 = 0; g0 < p.G; g0 += 4) {
    const int ng = min(4, p.G - g0);
    const int64_t row = static_cast<int64_t>(bh) * p.G + g0;
    float4 sc[4];
#pragma unroll
    for (int g = 0; g < 4; ++g)
      if (g < ng && some) sc[g] = *reinterpret_cast<const float4*>(p.scores + (row + g) * p.sstride + key);
    if (g0) __syncthreads();
    if (warp < ng) {
      const float2 r = row_stats(p, row + warp, (g0 & 4) + warp, p.info[bh * hg + g0 / 8], lane);
      if (lane == 0) st[warp] = r;
    }
    __syncthreads();
#pragma unroll
    for (int g = 0; g < 4; ++g)
      if (g < ng && some) {
        w[0] = fmaf(ex2(sc[g].x - st[g].x), st[g].y, w[0]);
        w[1] = fmaf(ex2(sc[g].y - st[g].x), st[g].y, w[1]);
        w[2] = fmaf(ex2(sc[g].z - st[g].x), st[g].y, w[2]);
        w[3] = fmaf(ex2(sc[g].w - st[g].x), st[g].y, w[3]);
      }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (key + i < n) mp[i] = m[i] + w[i];
    if (j >= 0 && j + i < elen) p.exact_mass[b * p.emb + h * p.emh + j + i] += w[i];
  }
}

namespace {
struct Kv4Plan {
  int splits, pieces;                           // one of them is 0
  int wcol;                                     // first window column of a row of scores
  int64_t ctas, sstride, info, row_stats, stats, part, scores, total;  // offsets in bytes
};
Kv4Plan kv4_plan(int64_t B, int64_t H, int64_t G, int64_t D, int64_t cap, int64_t W, bool mass, int sms) {
  auto up = [](int64_t x) { return (x + 255) & ~int64_t{255}; };
  Kv4Plan w;
  const int64_t rows = B * H * G, heads = B * H * ((G + 7) / 8);
  const int64_t slots = std::min<int64_t>((D == 64 ? 4 : 3) * static_cast<int64_t>(sms), KV4_MAX_PIECES);
  const int64_t units = std::max<int64_t>(1, (cap + KV4_TILE - 1) / KV4_TILE + (W + 15) / 16);
  w.splits = w.pieces = 0;
  // Very many heads even out by themselves (2048 of 512: 73 us, as pieces 78; of 20 to 512: 63, 67).
  // Few units run at once, and where a piece begins needs no search (8 heads of 8192: 10.5 us, as
  // pieces 11.9; of 20000, above the limit: as pieces 16.2, cut alike 19.6).
  if (heads >= std::min<int64_t>(4 * slots, KV4_MAX_HEADS)) w.splits = 1;
  else if (heads * units <= slots * KV4_MIN_UNITS)
    w.splits = static_cast<int>((units + KV4_MIN_UNITS - 1) / KV4_MIN_UNITS);
  else w.pieces = static_cast<int>(slots);
  w.ctas = w.pieces ? w.pieces : heads * w.splits;
  w.wcol = static_cast<int>((cap + KV4_TILE - 1) / KV4_TILE * KV4_TILE);
  w.sstride = w.wcol + (W + 3) / 4 * 4;
  const int64_t slots2 = w.splits == 1 ? 0 : 2 * w.ctas;  // parts
  w.info = 256;
  w.row_stats = w.info + up(heads * 8);
  w.stats = w.row_stats + up(rows * 8);
  w.part = w.stats + up(slots2 * 8 * 8);
  w.scores = w.part + up(slots2 * 8 * D * 4);
  w.total = w.scores + (mass ? up(rows * w.sstride * 4) : 0);
  return w;
}
int kv4_sms() {
  int dev = 0, sms = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms > 0 ? sms : 148;
}
}  // namespace

size_t kv4_attn_workspace(int64_t B, int64_t H, int64_t G, int64_t D, int64_t cap, int64_t W, bool mass) {
  return static_cast<size_t>(kv4_plan(B, H, G, D, cap, W, mass, kv4_sms()).total);
}

template <typename T, int D, bool MASS, bool FOLD>
static cudaError_t kv4_start(const Kv4Attn& p, int64_t ctas, cudaStream_t st) {
  constexpr int RING = KV4_NW * KV4_STAGES * Kv4Stage<D>::BYTES, OUT = KV4_NW * 8 * (D + 4) * 4;
  constexpr int SMEM = RING > OUT ? RING : OUT;
  static std::atomic<uint64_t> set{0};  // the shared-memory limit is raised once per device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = 1ull << (dev & 63);
  if (!(set.load() & bit)) {
    e = cudaFuncSetAttribute(kv4_attn_kernel<T, D, MASS, FOLD>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
    if (e != cudaSuccess) return e;
    set.fetch_or(bit);
  }
  kv4_attn_kernel<T, D, MASS, FOLD><<<static_cast<unsigned>(ctas), KV4_NW * 32, SMEM, st>>>(p);
  return cudaGetLastError();
}

template <typename T, int D>
static cudaError_t kv4_run(const Kv4Attn& p, int64_t ctas, cudaStream_t st) {
  cudaError_t e;
  if (p.G <= 4) e = p.scores ? kv4_start<T, D, true, true>(p, ctas, st) : kv4_start<T, D, false, true>(p, ctas, st);
  else e = p.scores ? kv4_start<T, D, true, false>(p, ctas, st) : kv4_start<T, D, false, false>(p, ctas, st);
  if (e != cudaSuccess) return e;
  const int mass = p.scores ? static_cast<int>((p.sstride + KV4_MASS_KEYS - 1) / KV4_MASS_KEYS) : 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.G + mass), static_cast<unsigned>(p.B * p.H));
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kv4_join_kernel<T, D>, p);
}

cudaError_t launch_kv4_attn(int dtype, int64_t D, Kv4Attn p, uint8_t* ws, cudaStream_t st) {
  if (p.B * p.H == 0) return cudaSuccess;
  const bool mass = p.mass || p.exact_mass;
  const Kv4Plan w = kv4_plan(p.B, p.H, p.G, D, p.cap, p.W, mass, kv4_sms());
  p.splits = w.splits;
  p.pieces = w.pieces;
  p.sstride = w.sstride;
  p.wcol = w.wcol;
  p.info = reinterpret_cast<int2*>(ws + w.info);
  p.row_stats = reinterpret_cast<float2*>(ws + w.row_stats);
  p.stats = reinterpret_cast<float2*>(ws + w.stats);
  p.part = reinterpret_cast<float*>(ws + w.part);
  p.used = reinterpret_cast<int*>(ws);
  p.scores = mass ? reinterpret_cast<float*>(ws + w.scores) : nullptr;
  if (dtype == BF16) return D == 64 ? kv4_run<__nv_bfloat16, 64>(p, w.ctas, st) : kv4_run<__nv_bfloat16, 128>(p, w.ctas, st);
  return D == 64 ? kv4_run<__half, 64>(p, w.ctas, st) : kv4_run<__half, 128>(p, w.ctas, st);
}

}  // namespace dab
