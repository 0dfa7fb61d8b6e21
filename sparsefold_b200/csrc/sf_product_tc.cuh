// Matrix products of the linear layers with gradients on tcgen05: z = A B^T (bf16 in, fp32 accumulate) with
// the epilogues of Epi.  Either operand may be K-major or M/N-major in memory: the gradients read the
// same matrices as the forward along the other axis, so nothing is transposed.
//
// fp32 values arrive as three bf16 terms; their product is the sum of the six term products above 2^-24
// (smallest first), which are six passes of the same K loop over other planes of the tensor maps.
//
// Persistent, warp-specialised: one warp streams 64-deep A and B tiles by TMA through a ring, one thread of
// another issues tcgen05.mma (M 128, N = bn, K 16) into one of two TMEM accumulators of up to 256 columns; 8 or 16
// warps drain the other one (thread = row).  Few tiles and a deep K: the K loop is split over CTAs, fp32 partials
// summed in order by k_sums.  Waits that are long as a rule are suspended and the ring's slots counted
// without divisions: polling and dividing threads took 20 % of the products' time (16384 x 4096 x 4096: 454 -> 360 us).
#pragma once

#include "sf_linear_grad.cuh"
#include "sf_tc.cuh"

namespace sf {
namespace lg {
namespace pr {

constexpr int BM = 128, BK = 64, MAX_BN = 256, MAX_STAGES = 8;
// Epilogue warps: 8 of 32 columns at a time, or (staged) 16 of 16.  With K = 128 the epilogue is the kernel, and a
// warp issues an instruction every 8 or 9 cycles, so it takes more of them to fill the schedulers; staged stores
// need few enough registers for 16 (65536 x 128 -> 2 x 512, dz: 100 us with 8).
constexpr int epi_warps(bool staged) { return staged ? 16 : 8; }
constexpr int threads_of(bool staged) { return (epi_warps(staged) + 2) * 32; }
constexpr int A_SLOT = BM * BK * 2;                 // 16 KB
constexpr int SMEM_MAX = 227 * 1024, SMEM_REST = 1024 /* alignment */ + 512 /* barriers */;
constexpr int GROUP_M = 12;                         // row tiles that share B tiles in L2 before the next columns

// CTAS = 2: a cluster of two CTAs computes 256 x bn tiles with cta_group::2 MMAs.  Each CTA loads its 128 rows
// of A and half of B's rows, so a 256 x 256 tile moves 2 x 32 KB per 64-deep step instead of 2 x 48 KB: the L2
// reads and the shared-memory reads of B halve (16384 x 4096 x 4096 bf16: 430 us with single CTAs, 664 with both
// operands M/N-major; 353 and 385 us in pairs, where the library product takes 346 and 357; tensor pipe 90 % active).

// The six term products of two split fp32 operands, smallest first, as nibbles (a plane, b plane).
constexpr uint32_t kPairA = 0x001102u, kPairB = 0x010120u;   // (2,0) (0,2) (1,1) (1,0) (0,1) (0,0)

struct Params {
  int64_t m, n;              // output rows and features
  int mt, nt, items;         // tiles; tiles * splits
  int bn, part;              // product columns of a tile; of one part of it (bn / 2 when gated)
  int stages, a_slot, b_slot, tx;   // ring; bytes that land per stage
  int nkb, pairs;            // 64-deep blocks of K; passes over them
  int splits, kb_split;      // K blocks of a split
  int seg_kb;                // K blocks of a segment (see Segments)
  int accs, acc_stride;      // accumulators in TMEM, columns between them
  int two;                   // two threads issue a tile's MMAs (see issue_half)
  int a_mn, b_mn, a_boxes;
  int a_one, b_one;          // M/N-major operand in one load (its extent is a multiple of 64)
  int act;
  const float* bias;
  const void* aux;
  int64_t aux_sr;
  void* out;
  int64_t out_sr;
  float* saved;
  float* colpart;
  int vec_out, vec_aux, vec_saved, vec_bias;   // 16-byte accesses are aligned
  int slots, pool;           // staged epilogue: buffers of a warp, and of them the ones that outputs take in turn
  uint32_t* status;
};

// Segments.  The tensor cores cut what does not fit their accumulator, always towards zero, so a sum loses about
// 1.1e-9 of itself per unit of K (measured: 4.7e-7 at K = 512, 9e-6 at 8192).  Where the result has to be good to
// fp32 (split fp32 operands; pre-activations whose gradient is summed over the rows for dbias), and where it is very long,
// K is cut into segments: each starts a new accumulator, and the epilogue warps add it, rounding to nearest, to a sum
// that waits in TMEM (columns kTotal on) until the last one.
constexpr int kTotal = 256;
// An accumulator's place and the parity of its use `it`.
struct Acc {
  uint32_t off, slot, phase;
  __device__ __forceinline__ Acc(const Params& p, uint32_t it) {
    slot = p.accs == 2 ? it & 1 : 0;
    phase = (p.accs == 2 ? it >> 1 : it) & 1;
    off = slot * (uint32_t)p.acc_stride;
  }
};
// Whether a tile's values are the accumulator and the columns kTotal on of TMEM together.
__device__ __forceinline__ bool has_total(const Params& p, int segs) { return segs > 1 || p.two; }
__device__ __forceinline__ int split_blocks(const Params& p, int split) {
  return min(p.kb_split, p.nkb - split * p.kb_split);
}

// Row and column tile and K split of an item (32-bit: the launcher checks that the items fit).
__device__ __forceinline__ void tile_at(const Params& p, uint32_t w, uint32_t& mi, uint32_t& ni, int& split) {
  uint32_t t = w;
  split = 0;
  if (p.splits > 1) {
    t = w / (uint32_t)p.splits;
    split = (int)(w - t * (uint32_t)p.splits);
  }
  const uint32_t per = GROUP_M * (uint32_t)p.nt, g = t / per, in = t - g * per, left = (uint32_t)p.mt - g * GROUP_M;
  ni = left < GROUP_M ? in / left : in / GROUP_M;
  mi = g * GROUP_M + in - ni * (left < GROUP_M ? left : GROUP_M);
}

// ---- epilogue pieces: one row, 32 columns ---------------------------------------------------------
template <int OUT>
struct OutT { using T = float; };
template <>
struct OutT<kOutBf16> { using T = bf16; };

__device__ __forceinline__ void load8(const float* p, bool vec, int count, float (&v)[8]) {
  if (vec && count >= 8) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < count ? p[e] : 0.f;
  }
}
__device__ __forceinline__ void load8(const bf16* p, bool vec, int count, float (&v)[8]) {
  if (vec && count >= 8) {
    const uint4 q = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < count ? __bfloat162float(p[e]) : 0.f;
  }
}
__device__ __forceinline__ void store8(float* p, bool vec, int count, const float (&v)[8]) {
  if (vec && count >= 8) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < count) p[e] = v[e];
  }
}
__device__ __forceinline__ void store8(bf16* p, bool vec, int count, const float (&v)[8]) {
  if (vec && count >= 8) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < count) p[e] = __float2bfloat16_rn(v[e]);
  }
}
// Sum over the warp's 32 rows of each of the W (16 or 32) columns: lane c returns column c's sum.  Each step
// halves the columns a lane carries and exchanges the other half (31 shuffles for 32 columns instead of 160).
template <int W>
__device__ __forceinline__ float column_sums(float (&v)[W], int lane) {
  if constexpr (W == 16) {
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], 16);
  }
#pragma unroll
  for (int w = W / 2; w >= 1; w >>= 1) {
    const bool up = (lane & w) != 0;
#pragma unroll
    for (int i = 0; i < W / 2; ++i)
      if (i < w) {
        const float keep = up ? v[i + w] : v[i], give = up ? v[i] : v[i + w];
        v[i] = keep + __shfl_xor_sync(0xffffffffu, give, w);
      }
  }
  return v[0];
}

// Packed fp32 pairs, each lane IEEE as its scalar form.
typedef unsigned long long pair_t;
__device__ __forceinline__ pair_t pk(float a, float b) {
  pair_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ pair_t pk1(float a) { return pk(a, a); }
__device__ __forceinline__ void unpk(pair_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ pair_t mul2(pair_t a, pair_t b) {
  pair_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ pair_t add2(pair_t a, pair_t b) {
  pair_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ pair_t fma2(pair_t a, pair_t b, pair_t c) {
  pair_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ pair_t ex2_2(pair_t v) {
  float a, b;
  unpk(v, a, b);
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(a));
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(b));
  return pk(a, b);
}
__device__ __forceinline__ pair_t rcp2(pair_t v) {
  float a, b;
  unpk(v, a, b);
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(a));
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(b));
  return pk(a, b);
}
// sigmoid: 1 / (1 + 2^(-z log2 e)), relative error about 2^-21
__device__ __forceinline__ pair_t sigmoid2(pair_t z) {
  return rcp2(add2(ex2_2(mul2(z, pk1(-1.4426950408889634f))), pk1(1.0f)));
}
// Phi(z) and exp(-z^2 / 2) as normal_cdf<true>: q is chosen by the sign of z, not formed as 1 - (1 - q), which would
// lose it in the negative tail (4 % of gelu at z = -5, all of it at -6).  65536 x 128 -> 2 x 1024: forward 76 us, backward
// 239 (75 and 232 with five terms and that loss).
__device__ __forceinline__ void cdf2(pair_t z, pair_t& cdf, pair_t& e) {
  e = ex2_2(mul2(mul2(z, z), pk1(-0.72134752044448170f)));
  const pair_t t = rcp2(fma2(pk1(kTailC), z & 0x7FFFFFFF7FFFFFFFull, pk1(1.0f)));
  pair_t y = pk1(tail(7));
#pragma unroll
  for (int i = 6; i >= 0; --i) y = fma2(t, y, pk1(tail(i)));
  const pair_t q = mul2(mul2(t, y), e), r = fma2(q, pk1(-1.0f), pk1(1.0f));
  float z0, z1, q0, q1, r0, r1;
  unpk(z, z0, z1);
  unpk(q, q0, q1);
  unpk(r, r0, r1);
  cdf = pk(z0 < 0.f ? q0 : r0, z1 < 0.f ? q1 : r1);
}
// act(z), and with GRAD act'(z).
template <int ACT, bool GRAD>
__device__ __forceinline__ void act2(pair_t z, pair_t& a, pair_t& da) {
  if constexpr (ACT == SF_POST_SILU) {
    const pair_t s = sigmoid2(z);
    a = mul2(z, s);
    if (GRAD) da = fma2(a, fma2(s, pk1(-1.f), pk1(1.f)), s);
  } else if constexpr (ACT == SF_POST_GELU) {
    pair_t p, e;
    cdf2(z, p, e);
    a = mul2(z, p);
    if (GRAD) da = fma2(mul2(z, pk1(0.39894228040143268f)), e, p);
  } else if constexpr (ACT == SF_POST_SIGMOID) {
    a = sigmoid2(z);
    if (GRAD) da = mul2(a, fma2(a, pk1(-1.f), pk1(1.f)));
  } else if constexpr (ACT == SF_POST_RELU) {
    float z0, z1, a0, a1, d0, d1;
    unpk(z, z0, z1);
    act_grad<SF_POST_RELU, true>(z0, a0, d0);
    act_grad<SF_POST_RELU, true>(z1, a1, d1);
    a = pk(a0, a1);
    if (GRAD) da = pk(d0, d1);
  } else {
    a = z;
    if (GRAD) da = pk1(1.0f);
  }
}

// FAST (bf16 results): in pairs, with the approximations above.
template <int KIND, int ACT, bool FAST, int W>
__device__ __forceinline__ void act_row(float (&z)[W], const float (&u)[W]) {
  if constexpr (FAST) {
#pragma unroll
    for (int e = 0; e < W; e += 2) {
      pair_t a, da;
      act2<ACT, false>(pk(z[e], z[e + 1]), a, da);
      unpk(KIND == kGated ? mul2(a, pk(u[e], u[e + 1])) : a, z[e], z[e + 1]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < W; ++e) z[e] = KIND == kGated ? act_value<ACT, false>(z[e]) * u[e] : act_value<ACT, false>(z[e]);
  }
}
template <int KIND, int ACT, bool FAST, int W>
__device__ __forceinline__ void grad_row(const float (&x)[W], float (&z)[W], float (&u)[W]) {
  if constexpr (FAST) {
#pragma unroll
    for (int e = 0; e < W; e += 2) {
      const pair_t dy = pk(x[e], x[e + 1]);
      pair_t a, da;
      act2<ACT, true>(pk(z[e], z[e + 1]), a, da);
      if (KIND == kDGated) {
        unpk(mul2(mul2(dy, pk(u[e], u[e + 1])), da), z[e], z[e + 1]);
        unpk(mul2(dy, a), u[e], u[e + 1]);
      } else {
        unpk(mul2(dy, da), z[e], z[e + 1]);
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < W; ++e) {
      float a, da;
      act_grad<ACT, false>(z[e], a, da);
      if (KIND == kDGated) {
        z[e] = x[e] * u[e] * da;
        u[e] = x[e] * a;
      } else {
        z[e] = x[e] * da;
      }
    }
  }
}

// One row's 32 columns c .. c + 31 (`count` of them exist) of the tile, z (and u, the other half's).
template <int KIND, int OUT>
__device__ __forceinline__ void chunk(const Params& p, int64_t row, bool live, int64_t c, int count, int split,
                                      float (&z)[32], float (&u)[32], int lane) {
  constexpr bool GATED = KIND == kGated || KIND == kDGated;
  using T = typename OutT<OUT>::T;
  if (KIND == kLinear && p.splits > 1) {   // fp32 partial [split][m][n]
    if (live) {
      float* o = static_cast<float*>(p.out) + ((int64_t)split * p.m + row) * p.out_sr + c;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = z[g * 8 + e];
        store8(o + g * 8, p.vec_out, count - g * 8, v);
      }
    }
    return;
  }
  const int64_t wide = GATED ? 2 * p.n : p.n;
  if (p.bias) {
#pragma unroll
    for (int e = 0; e < 32; ++e)
      if (e < count) {
        z[e] += __ldg(p.bias + c + e);
        if (GATED) u[e] += __ldg(p.bias + p.n + c + e);
      }
  }
  if ((KIND == kLinear || KIND == kGated) && p.saved && live) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = z[g * 8 + e];
      store8(p.saved + row * wide + c + g * 8, p.vec_saved, count - g * 8, v);
      if (GATED) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = u[g * 8 + e];
        store8(p.saved + row * wide + p.n + c + g * 8, p.vec_saved, count - g * 8, v);
      }
    }
  }
  if constexpr (KIND == kLinear || KIND == kGated) {
    SF_ACT_SWITCH(p.act, (act_row<KIND, ACT, OUT == kOutBf16>(z, u)))
    if (!live) return;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      if (g * 8 >= count) break;
      float v[8], x[8];
      if (KIND == kLinear && p.aux) {
        load8(static_cast<const T*>(p.aux) + row * p.aux_sr + c + g * 8, p.vec_aux, count - g * 8, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = z[g * 8 + e] + x[e];
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = z[g * 8 + e];
      }
      store8(static_cast<T*>(p.out) + row * p.out_sr + c + g * 8, p.vec_out, count - g * 8, v);
    }
  } else {
    float x[32];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (live && g * 8 < count)
        load8(static_cast<const T*>(p.aux) + row * p.aux_sr + c + g * 8, p.vec_aux, count - g * 8, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[g * 8 + e] = v[e];
    }
    SF_ACT_SWITCH(p.act, (grad_row<KIND, ACT, OUT == kOutBf16>(x, z, u)))
    if (live) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        if (g * 8 >= count) break;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = z[g * 8 + e];
        store8(static_cast<T*>(p.out) + row * p.out_sr + c + g * 8, p.vec_out, count - g * 8, v);
        if (GATED) {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = u[g * 8 + e];
          store8(static_cast<T*>(p.out) + row * p.out_sr + p.n + c + g * 8, p.vec_out, count - g * 8, v);
        }
      }
    } else {   // a row behind the last one (its accumulator holds anything) adds nothing to the sums
#pragma unroll
      for (int e = 0; e < 32; ++e) z[e] = u[e] = 0.f;
    }
    if (p.colpart) {
      const int64_t blk = row / 32;   // rows of a warp start at a multiple of 32
      const float s = column_sums(z, lane);
      const bool in = blk * 32 < p.m && lane < count;
      if (in) p.colpart[blk * wide + c + lane] = s;
      if (GATED) {
        const float t = column_sums(u, lane);
        if (in) p.colpart[blk * wide + p.n + c + lane] = t;
      }
    }
  }
}

// A slot of the ring and the parity of its current use.
struct Ring {
  uint32_t slot = 0, phase = 0;
  __device__ __forceinline__ void next(int stages) {
    if (++slot == (uint32_t)stages) slot = 0, phase ^= 1;
  }
};

// A segment that is not the last: this lane's columns from `from` on, WIDE of every `every`, onto (or as) the sum.
template <bool GATED, int WIDE>
__device__ __forceinline__ void fold_segment(const Params& p, uint32_t d, uint32_t total, int from, int every, int cols,
                                             bool add) {
#pragma unroll 1
  for (int c = from; c < cols; c += every)
#pragma unroll 1
    for (int part = 0; part < (GATED ? 2 : 1); ++part)
#pragma unroll 1
      for (int h = 0; h < WIDE && c + h < p.part; h += 16) {   // part is a multiple of 16: no column twice
        const uint32_t at = (uint32_t)(part * p.part + c + h);
        float z[16];
        uint32_t bits[16];
        tc::tmem_ld16(d + at, z);
        if (add) {
          float t[16];
          tc::tmem_ld16(total + at, t);
#pragma unroll
          for (int e = 0; e < 16; ++e) z[e] += t[e];
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) bits[e] = __float_as_uint(z[e]);
        tc::tmem_st16(total + at, bits);
      }
  tc::tmem_wait_st();
}
template <int CTAS>
__device__ __forceinline__ void free_acc(uint64_t* acce, int lane) {
  tc::tc_fence_before();
  __syncwarp();
  if (lane == 0) {
    if (CTAS == 2) tc::mbar_arrive_cluster(tc::map_shared(acce, 0));
    else tc::mbar_arrive(acce);
  }
}

// ---- the staged epilogue --------------------------------------------------------------------------
// Stores straight from the accumulator's layout (a thread holds a row) reach the L2 as one request per row and 16
// bytes; with K = 128 those requests are the kernel's bound (65536 x 128 -> 1024, no activation: 69 us for 151
// MB).  So each warp puts 32 rows x 64 bytes (32 bf16 or 16 fp32 columns) into a 2 KB buffer (64-byte swizzle,
// conflict-free) and lane 0 hands it to a TMA store, which also cuts what lies behind the last row or column;
// dy or the residual arrives the same way, a chunk ahead.  A matrix whose rows do not start on 16 bytes goes between
// buffer and memory a row at a time, lane = column, which is still one request per row and not one per element.
// The activation is a template argument and the arithmetic works on packed fp32 pairs: with K = 128 a tile's
// products take 2.6k cycles and the epilogue has to keep up (with a switch and scalar arithmetic 37 us, 28 us so).
struct Maps {
  CUtensorMap a, b, b2;      // operands
  CUtensorMap out, out2;     // the output, and its second half (kDGated)
  CUtensorMap sav, sav2;     // the saved pre-activations, and their second half
  CUtensorMap aux;           // dy or residual
};

constexpr int SLOT = 2048, CW = 16;

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void sts16(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}

// Waits until at most `left` (0 or 1) of the warp's last stores still read their buffers.  One left over means the other
// buffer's only if every use of a buffer commits a group: warps without a row in a tile commit an empty one (without it
// they overwrote what the tile before still had to store, seen where the stores are the bound: 12346 x 8 -> 4072).
__device__ __forceinline__ void free_slot(int left, int lane) {
  if (lane == 0) {
    if (left == 0) tc::bulk_wait_read0();
    else tc::bulk_wait_read1();
  }
  __syncwarp();
}
// A warp's buffer to rows of a matrix (`rows` of 32, `cols` of 32 bf16 or 16 fp32 there) by plain accesses.
__device__ __forceinline__ void copy_out(uint32_t buf, bf16* dst, int64_t sr, int rows, int cols, int lane) {
  if (lane < cols)
#pragma unroll 8
    for (int r = 0; r < 32; ++r)
      if (r < rows) {
        uint16_t v;
        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(buf + tc::sw64_off(r, lane >> 3) + (lane & 7) * 2) : "memory");
        *reinterpret_cast<uint16_t*>(dst + r * sr + lane) = v;
      }
  __syncwarp();
}
__device__ __forceinline__ void copy_out(uint32_t buf, float* dst, int64_t sr, int rows, int cols, int lane) {
  const int e = lane & 15;
  if (e < cols)
#pragma unroll 8
    for (int r = lane >> 4; r < 32; r += 2)
      if (r < rows) {
        float v;
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(buf + tc::sw64_off(r, e >> 2) + (e & 3) * 4) : "memory");
        dst[r * sr + e] = v;
      }
  __syncwarp();
}
// Rows of a matrix into a warp's buffer, zero where there are none.
__device__ __forceinline__ void copy_in(uint32_t buf, const float* src, int64_t sr, int rows, int cols, int lane) {
  const int e = lane & 15;
#pragma unroll 8
  for (int r = lane >> 4; r < 32; r += 2) {
    const float v = r < rows && e < cols ? src[r * sr + e] : 0.f;
    asm volatile("st.shared.f32 [%0], %1;" ::"r"(buf + tc::sw64_off(r, e >> 2) + (e & 3) * 4), "f"(v) : "memory");
  }
  __syncwarp();
}
__device__ __forceinline__ void copy_in(uint32_t buf, const bf16* src, int64_t sr, int rows, int cols, int lane) {
#pragma unroll 8
  for (int r = 0; r < 32; ++r) {
    uint16_t v = 0;
    if (r < rows && lane < cols) v = *reinterpret_cast<const uint16_t*>(src + r * sr + lane);
    asm volatile("st.shared.u16 [%0], %1;" ::"r"(buf + tc::sw64_off(r, lane >> 3) + (lane & 7) * 2), "h"(v) : "memory");
  }
  __syncwarp();
}
// Sixteen fp32 values of a lane's row into the buffer, and from there to the matrix (by TMA, or plainly to `dst`).
__device__ __forceinline__ void store_f32(const CUtensorMap* map, float* dst, int64_t sr, bool tma, uint8_t* buf,
                                          const uint32_t (&at)[4], const float (&v)[CW], int c, int row0, int z, int rows,
                                          int cols, int lane) {
  const uint32_t to = tc::smem_u32(buf);
#pragma unroll
  for (int j = 0; j < 4; ++j)
    sts16(to + at[j], __float_as_uint(v[4 * j]), __float_as_uint(v[4 * j + 1]), __float_as_uint(v[4 * j + 2]),
          __float_as_uint(v[4 * j + 3]));
  if (tma) {
    tc::fence_proxy_async();
    __syncwarp();
    if (lane == 0) {
      if (rows > 0) tc::tma_store_3d(map, buf, c, row0, z);
      tc::bulk_commit();
    }
  } else {
    __syncwarp();
    copy_out(to, dst, sr, rows, cols, lane);
  }
}
// bias[0 .. 15] onto v, in fours where `vec` (`count` is then a multiple of four, the address 16-byte aligned).
__device__ __forceinline__ void add_bias(const float* bias, bool vec, int count, float (&v)[CW]) {
  if (vec) {
#pragma unroll
    for (int g = 0; g < CW; g += 4)
      if (g < count) {
        const float4 b = __ldg(reinterpret_cast<const float4*>(bias + g));
        v[g] += b.x, v[g + 1] += b.y, v[g + 2] += b.z, v[g + 3] += b.w;
      }
  } else {
#pragma unroll
    for (int e = 0; e < CW; ++e)
      if (e < count) v[e] += __ldg(bias + e);
  }
}

// LEAN: without bias, residual, saved pre-activations, column sums and segments, decided when compiled: what a transition's
// three products are, and worth 10 % of them at K = 128 (65536 x 128 -> 1024: 28 us against 32).
// The epilogue warps' part of the kernel: bf16 out (activation EACT), or fp32 out (EACT < 0: p.act decides; exact
// functions).
template <int KIND, int OUT, int EACT, bool LEAN, int CTAS, typename First>
__device__ __forceinline__ void staged_epilogue(const Params& p, const Maps& tm, uint8_t* area, uint64_t* aux_bar,
                                                uint64_t* accf, uint64_t* acce, uint32_t tbase, int first_item, int step,
                                                uint32_t rank, int warp, int lane, bool& aborted, First first) {
  constexpr bool GATED = KIND == kGated || KIND == kDGated, GRAD = KIND == kDLinear || KIND == kDGated;
  constexpr bool BF = OUT == kOutBf16;
  using T = typename OutT<OUT>::T;
  constexpr int CHUNK = BF ? 32 : 16;                      // columns of a 64-byte row
  const int quad = warp & 3, from = (warp >> 2) * CHUNK;   // this warp's rows, and its first chunk of every four
  const uint32_t lane_addr = tbase + ((uint32_t)(quad * 32) << 16);
  uint8_t* mine = area + warp * p.slots * SLOT;            // [aux][p.pool buffers][one more for out while saving]
  const bool with_aux = GRAD || (!LEAN && KIND == kLinear && p.aux), saving = !LEAN && !GRAD && p.saved;
  uint8_t* pool = mine + (with_aux ? SLOT : 0);
  uint32_t at[4];                                          // this lane's four pieces of a buffer
#pragma unroll
  for (int j = 0; j < 4; ++j) at[j] = tc::sw64_off(lane, j);
  const uint32_t aux_at = tc::smem_u32(mine);
  const int turns = p.pool - 1;                            // outputs alternate (1) or share one buffer (0)
  const int64_t wide = GATED ? 2 * p.n : p.n;
  uint64_t* bar = aux_bar + warp;
  uint32_t aux_phase = 0, turn = 0;
  auto tile_of = [&](int w, int& row0, int& c0, int& cols, int& split) {
    uint32_t mi, ni;
    tile_at(p, (uint32_t)w, mi, ni, split);
    row0 = (int)(mi * BM * CTAS + rank * BM) + quad * 32;
    c0 = (int)ni * p.part;
    cols = (int)(p.n - c0 < p.part ? p.n - c0 : p.part);
  };
  // asks for the aux chunk at column c of item w, or of the first item behind it that has one
  bool asked = false;      // one is on its way
  auto ask = [&](int w, int c) {
    for (; w < p.items; w += step, c = from) {
      int row0, c0, cols, split;
      tile_of(w, row0, c0, cols, split);
      if (c < cols) {
        if (lane == 0) {
          tc::mbar_expect_tx(bar, SLOT);
          tc::tma_load_3d(mine, &tm.aux, bar, c0 + c, row0, 0);
        }
        asked = true;
        return;
      }
    }
  };
  const bool ahead = with_aux && p.vec_aux;
  if (ahead) ask(first_item, from);
  if constexpr (!LEAN) first();
  uint32_t it = 0;
  for (int w = first_item; w < p.items; w += step, ++it) {
    int row0, c0, cols, split;
    tile_of(w, row0, c0, cols, split);
    const int64_t left = p.m - row0;
    const int rows = left < 0 ? 0 : left < 32 ? (int)left : 32;   // of this warp's 32
    int segs = 1;
    if constexpr (!LEAN) {
      segs = (split_blocks(p, split) + p.seg_kb - 1) / p.seg_kb;
      for (int s = 0; s + 1 < segs; ++s, ++it) {
        const Acc acc(p, it);
        tc::mbar_wait_long(&accf[acc.slot], acc.phase, p.status, aborted);
        tc::tc_fence_after();
        fold_segment<GATED, CHUNK>(p, lane_addr + acc.off, lane_addr + kTotal, from, 4 * CHUNK, cols, s > 0);
        free_acc<CTAS>(&acce[acc.slot], lane);
      }
    }
    const Acc acc(p, it);
    const uint32_t d = lane_addr + acc.off;
    tc::mbar_wait_long(&accf[acc.slot], acc.phase, p.status, aborted);
    tc::tc_fence_after();
#pragma unroll 1
    for (int c = from; c < cols; c += 4 * CHUNK) {
      uint4 xr[4];
      if (with_aux) {
        if (asked && __all_sync(0xffffffffu, tc::mbar_wait(bar, aux_phase, p.status, aborted))) {
          aux_phase ^= 1;
          asked = false;
        }
        if (!ahead)
          copy_in(aux_at, static_cast<const T*>(p.aux) + (int64_t)row0 * p.aux_sr + c0 + c, p.aux_sr, rows, cols - c, lane);
#pragma unroll
        for (int j = 0; j < 4; ++j) xr[j] = lds16(aux_at + at[j]);
        __syncwarp();
        // the buffer has been read: the next chunk's (nothing more once a wait has given up)
        if (ahead && !__any_sync(0xffffffffu, aborted) && !asked) ask(w, c + 4 * CHUNK);
      }
      // one buffer for the chunk (kDGated: one for each output), beside those that saved values take in turn
      uint8_t* out_buf = pool;
      if (KIND == kDGated || saving) {
        free_slot(0, lane);
        if (saving) out_buf = pool + p.pool * SLOT;
      } else {
        free_slot(turns, lane);
        out_buf = pool + (turn++ & turns) * SLOT;
      }
      const uint32_t out = tc::smem_u32(out_buf);
#pragma unroll
      for (int h = 0; h < CHUNK / CW; ++h) {
        float z[CW], u[CW];
        const int cc = c + h * CW, count = cols - cc;      // count may be 0 or less: the store cuts it
        if (GATED) tc::tmem_ld16x2(d + cc, d + p.part + cc, z, u);
        else tc::tmem_ld16(d + cc, z);
        if (!LEAN && has_total(p, segs)) {
          float t[CW];
          tc::tmem_ld16(lane_addr + kTotal + cc, t);
#pragma unroll
          for (int e = 0; e < CW; ++e) z[e] += t[e];
          if (GATED) {
            tc::tmem_ld16(lane_addr + kTotal + p.part + cc, t);
#pragma unroll
            for (int e = 0; e < CW; ++e) u[e] += t[e];
          }
        }
        if (!LEAN && p.bias) {
          add_bias(p.bias + c0 + cc, p.vec_bias, count, z);
          if (GATED) add_bias(p.bias + p.n + c0 + cc, p.vec_bias, count, u);
        }
        if (saving && count > 0) {
          free_slot(turns, lane);
          float* to = p.saved + (int64_t)row0 * wide + c0 + cc;
          store_f32(&tm.sav, to, wide, p.vec_saved, pool + (turn++ & turns) * SLOT, at, z, c0 + cc, row0, 0, rows, count, lane);
          if (GATED) {
            free_slot(turns, lane);
            store_f32(&tm.sav2, to + p.n, wide, p.vec_saved, pool + (turn++ & turns) * SLOT, at, u, c0 + cc, row0, 0, rows,
                      count, lane);
          }
        }
        if constexpr (!BF) {
          float x[CW];
          if (with_aux) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              x[4 * j] = __uint_as_float(xr[j].x), x[4 * j + 1] = __uint_as_float(xr[j].y),
              x[4 * j + 2] = __uint_as_float(xr[j].z), x[4 * j + 3] = __uint_as_float(xr[j].w);
          }
          if constexpr (GRAD) {
            SF_ACT_SWITCH(p.act, (grad_row<KIND, ACT, false>(x, z, u)))
          } else {
            SF_ACT_SWITCH(p.act, (act_row<KIND, ACT, false>(z, u)))
            if (with_aux)
#pragma unroll
              for (int e = 0; e < CW; ++e) z[e] += x[e];
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            sts16(out + at[j], __float_as_uint(z[4 * j]), __float_as_uint(z[4 * j + 1]), __float_as_uint(z[4 * j + 2]),
                  __float_as_uint(z[4 * j + 3]));
            if (KIND == kDGated)
              sts16(out + SLOT + at[j], __float_as_uint(u[4 * j]), __float_as_uint(u[4 * j + 1]), __float_as_uint(u[4 * j + 2]),
                    __float_as_uint(u[4 * j + 3]));
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            pair_t zz = pk(z[2 * i], z[2 * i + 1]), a, da;
            act2<EACT, GRAD>(zz, a, da);
            pair_t x = 0;
            if (with_aux) {
              const uint4& xx = xr[h * 2 + i / 4];
              const uint32_t xw = i % 4 == 0 ? xx.x : i % 4 == 1 ? xx.y : i % 4 == 2 ? xx.z : xx.w;
              x = pk(__uint_as_float(xw << 16), __uint_as_float(xw & 0xFFFF0000u));
            }
            if constexpr (KIND == kLinear) {
              unpk(with_aux ? add2(a, x) : a, z[2 * i], z[2 * i + 1]);
            } else if constexpr (KIND == kGated) {
              unpk(mul2(a, pk(u[2 * i], u[2 * i + 1])), z[2 * i], z[2 * i + 1]);
            } else if constexpr (KIND == kDLinear) {
              unpk(mul2(x, da), z[2 * i], z[2 * i + 1]);
            } else {
              unpk(mul2(mul2(x, pk(u[2 * i], u[2 * i + 1])), da), z[2 * i], z[2 * i + 1]);
              unpk(mul2(x, a), u[2 * i], u[2 * i + 1]);
            }
          }
          sts16(out + at[h * 2], pack2(z[0], z[1]), pack2(z[2], z[3]), pack2(z[4], z[5]), pack2(z[6], z[7]));
          sts16(out + at[h * 2 + 1], pack2(z[8], z[9]), pack2(z[10], z[11]), pack2(z[12], z[13]), pack2(z[14], z[15]));
          if constexpr (KIND == kDGated) {
            sts16(out + SLOT + at[h * 2], pack2(u[0], u[1]), pack2(u[2], u[3]), pack2(u[4], u[5]), pack2(u[6], u[7]));
            sts16(out + SLOT + at[h * 2 + 1], pack2(u[8], u[9]), pack2(u[10], u[11]), pack2(u[12], u[13]), pack2(u[14], u[15]));
          }
        }
        if (!LEAN && GRAD && p.colpart && count > 0) {
          if (row0 + lane >= p.m)   // a row behind the last one (its accumulator holds anything) adds nothing
#pragma unroll
            for (int e = 0; e < CW; ++e) z[e] = u[e] = 0.f;
          const bool in = rows > 0 && lane < CW && lane < count;
          float* part = p.colpart + (int64_t)(row0 / 32) * wide + c0 + cc + lane;
          const float s0 = column_sums(z, lane);
          if (in) part[0] = s0;
          if (KIND == kDGated) {
            const float s1 = column_sums(u, lane);
            if (in) part[p.n] = s1;
          }
        }
      }
      if (p.vec_out) {
        tc::fence_proxy_async();
        __syncwarp();
        if (lane == 0) {
          if (rows > 0) {
            tc::tma_store_3d(&tm.out, out_buf, c0 + c, row0, split);
            if (KIND == kDGated) tc::tma_store_3d(&tm.out2, out_buf + SLOT, c0 + c, row0, split);
          }
          tc::bulk_commit();
        }
      } else {
        __syncwarp();
        T* to = static_cast<T*>(p.out) + (int64_t)row0 * p.out_sr + c0 + c;   // (a split's partials have 16-byte rows)
        copy_out(out, to, p.out_sr, rows, cols - c, lane);
        if (KIND == kDGated) copy_out(out + SLOT, to + p.n, p.out_sr, rows, cols - c, lane);
      }
    }
    free_acc<CTAS>(&acce[acc.slot], lane);
  }
  if (asked) tc::mbar_wait_drain(bar, aux_phase, p.status);   // abort path only
  if (lane == 0) tc::bulk_wait0();   // stores done before the shared memory goes away
}

// Barriers and loads by shared-memory address, for the producer.
__device__ __forceinline__ bool wait_at(uint32_t bar, uint32_t parity, uint32_t* status, bool& aborted) {
  const uint32_t limit = aborted ? 1u : tc::kWaitLimit;
  for (uint32_t i = 0; i < limit; ++i) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity), "r"(0u)
        : "memory");
    if (ok) return true;
  }
  aborted = true;
  if (status) atomicCAS(status, 0u, (uint32_t)SF_ERR_TIMEOUT);
  return false;
}
__device__ __forceinline__ void expect_at(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// PAIR: the load of one CTA of a pair, whose barrier may be the other one's.
template <bool PAIR>
__device__ __forceinline__ void load3(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2) {
  if constexpr (PAIR)
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void load4(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2, int c3) {
  if constexpr (PAIR)
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
        : "memory");
}

__device__ __forceinline__ uint32_t mma_desc(const Params& p, int rows) {
  return tc::idesc_bf16(rows, 0) | ((uint32_t)(p.bn >> 3) << 17) | ((uint32_t)p.a_mn << 15) | ((uint32_t)p.b_mn << 16);
}
// Descriptor of the first stage's operand; the address field is in 16-byte units and does not overflow.
__device__ __forceinline__ uint64_t first_desc(uint32_t at, int mn) {
  return mn ? tc::smem_desc_mn(at, 8192, 1024, tc::kSW128) : tc::smem_desc(at, 1024, tc::kSW128);
}

// Every other stage of a CTA's only tile, from stage `part` (0 or 1) on, into the accumulator `d` (a thread's call).
// Small tiles are bound by the instructions of the two threads that run the ring (32 columns a part, K = 4096: 570
// cycles a stage for four MMAs that need half of that, 400 for its three loads).  So where a CTA has one tile and K is
// deep, the first two epilogue warps, idle till then, take every other stage: one issues its MMAs into the columns
// kTotal on, which the epilogue adds, and one its loads (24 x 4096 -> 2 x 4096, weights in L2: 20.9 -> 13.8 us; from HBM
// 21.6 -> 17.2 us).  The ring has an even number of stages then, and each thread waits for its own slots only, in
// their order.
__device__ __forceinline__ void issue_half(const Params& p, uint32_t part, uint32_t d, uint32_t sbase, int steps,
                                           uint64_t* full, uint64_t* empty, uint64_t* accf, bool& aborted) {
  const uint32_t idesc = mma_desc(p, BM);
  const uint64_t a_desc = first_desc(sbase, p.a_mn), b_desc = first_desc(sbase + p.a_slot, p.b_mn);
  const uint32_t a_step = p.a_mn ? 128 : 2, b_step = p.b_mn ? 128 : 2, stage = (uint32_t)(p.a_slot + p.b_slot);
  Ring r;
  if (part) r.next(p.stages);
  bool more = false;
  for (int i = (int)part; i < steps; i += 2) {
    const uint32_t s = r.slot;
    if (!tc::mbar_wait(&full[s], r.phase, p.status, aborted)) return;
    tc::tc_fence_after();
    const uint32_t at = (s * stage) >> 4;
#pragma unroll
    for (int kk = 0; kk < BK / 16; ++kk, more = true)
      tc::mma_bf16(d, a_desc + at + kk * a_step, b_desc + at + kk * b_step, idesc, more);
    tc::mma_commit(&empty[s]);
    r.next(p.stages);
    r.next(p.stages);
  }
  tc::mma_commit(accf);
}

// EACT, LEAN: of a staged bf16 epilogue; -1 and false elsewhere.
template <int KIND, int OUT, int CTAS, bool STAGED, int EACT, bool LEAN>
__global__ void __launch_bounds__(threads_of(STAGED), 1) k_product_tc(const __grid_constant__ Maps tm,
                                                           const __grid_constant__ Params p) {
  const CUtensorMap &tmA = tm.a, &tmB = tm.b, &tmB2 = tm.b2;
  constexpr bool GATED = KIND == kGated || KIND == kDGated;
  constexpr int EPI_WARPS = epi_warps(STAGED);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int stage_bytes = p.a_slot + p.b_slot;
  uint8_t* area = smem + p.stages * stage_bytes;                            // the staged epilogue's buffers
  uint64_t* full = reinterpret_cast<uint64_t*>(area + (STAGED ? EPI_WARPS * p.slots * SLOT : 0));
  uint64_t* empty = full + MAX_STAGES;
  uint64_t* accf = empty + MAX_STAGES;
  uint64_t* acce = accf + 2;                     // CTAS 2: the even CTA's counts both CTAs' warps
  uint64_t* drain = acce + 2;                    // of each issuing thread
  uint64_t* aux_bar = drain + 2;                 // one of each epilogue warp
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(aux_bar + EPI_WARPS);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = CTAS == 2 ? tc::cluster_rank() : 0;
  const int first_item = blockIdx.x / CTAS, step = gridDim.x / CTAS;

  if (warp == 0) {
    if constexpr (CTAS == 2) {
      tc::tmem_alloc2(tmem_slot, 512);
      tc::tmem_relinquish2();
    } else {
      tc::tmem_alloc(tmem_slot, 512);
      tc::tmem_relinquish();
    }
  }
  if (tid == 0) {
    for (int s = 0; s < p.stages; ++s) {
      tc::mbar_init(&full[s], 1);                                // CTAS 2: the even CTA's counts the bytes of both
      tc::mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      tc::mbar_init(&accf[a], CTAS == 1 && p.two ? 2 : 1);
      tc::mbar_init(&acce[a], CTAS * EPI_WARPS);
      tc::mbar_init(&drain[a], 1);
    }
    for (int w = 0; w < EPI_WARPS; ++w) tc::mbar_init(&aux_bar[w], 1);
    tc::fence_mbar_init();
    tc::prefetch_tmap(&tmA);
    tc::prefetch_tmap(&tmB);
    if (GATED) tc::prefetch_tmap(&tmB2);
  }
  tc::tc_fence_before();
  __syncthreads();
  if constexpr (CTAS == 2) tc::cluster_sync();   // both CTAs' barriers exist before any remote arrival
  tc::tc_fence_after();
  tc::griddep_wait();
  tc::griddep_launch();
  const uint32_t tbase = *tmem_slot, sbase = tc::smem_u32(smem);
  bool aborted = false;
  uint32_t loads = 0;

  // ---- TMA producer (stops at its first failed wait): every `every`th stage from `from` on ----
  // Its instructions count where tiles are small (see issue_half), so how the operands arrive is decided outside the
  // K loop (24 x 4096 -> 2 x 4096: 24.6 us with the choices inside, 20.9 so).
  auto produce = [&](uint32_t from, int every) {
    // CTAS 2: both CTAs' loads complete on the even CTA's barrier, which is what orders the odd CTA's bytes before the MMA
    const uint32_t fbar = CTAS == 2 ? tc::map_shared(full, 0) : tc::smem_u32(full), ebar = tc::smem_u32(empty);
    const uint32_t own = tc::smem_u32(full);
    const uint32_t stages = (uint32_t)p.stages;
    uint32_t slot = from, parity = 1;
    for (int w = first_item; w < p.items && !aborted; w += step) {
      uint32_t mi, ni;
      int split;
      tile_at(p, (uint32_t)w, mi, ni, split);
      const int m0 = (int)(mi * BM * CTAS) + (int)rank * BM;
      // CTAS 2: this CTA's half of the product's columns; the gated kinds' halves are the two parts
      const int n0 = (int)(ni * p.part) + (CTAS == 2 && !GATED ? (int)rank * (p.bn / 2) : 0);
      const int rows = CTAS == 2 ? p.bn / 2 : p.part;   // B rows per load below
      const CUtensorMap* mapB = CTAS == 2 && GATED && rank ? &tmB2 : &tmB;
      const uint32_t second = (uint32_t)rows * 128;
      const int first = split * p.kb_split, blocks = split_blocks(p, split);
      // the passes of each segment in turn
      auto stream = [&](auto load_a, auto load_b) {
        int kb = (int)from;
        for (int seg = 0; seg < blocks; seg += p.seg_kb) {
          const int len = min(p.seg_kb, blocks - seg);
          for (int pair = 0; pair < p.pairs; ++pair) {
            const int pa = p.pairs == 1 ? 0 : (kPairA >> (4 * pair)) & 15, pb = p.pairs == 1 ? 0 : (kPairB >> (4 * pair)) & 15;
            int k0 = (first + seg + kb) * BK;
            for (; kb < len; kb += every, k0 += every * BK, ++loads) {
              if (!wait_at(ebar + 8 * slot, parity, p.status, aborted)) return;
              const uint32_t bar = fbar + 8 * slot, sa = sbase + slot * (uint32_t)stage_bytes;
              if (CTAS == 1 || rank == 0) expect_at(own + 8 * slot, p.tx * CTAS);
              load_a(sa, bar, k0, pa);
              load_b(sa + p.a_slot, bar, k0, pb);
              if ((slot += every) >= stages) slot -= stages, parity ^= 1;
            }
            kb -= len;
          }
        }
      };
      auto a_rows = [&](uint32_t at, uint32_t bar, int k0, int pl) { load3<CTAS == 2>(at, &tmA, bar, k0, m0, pl); };
      auto a_runs = [&](uint32_t at, uint32_t bar, int k0, int pl) { load4<CTAS == 2>(at, &tmA, bar, 0, k0, m0 / 64, pl); };
      auto b_rows = [&](uint32_t at, uint32_t bar, int k0, int pl) {
        load3<CTAS == 2>(at, mapB, bar, k0, n0, pl);
        if (GATED && CTAS == 1) load3<CTAS == 2>(at + second, &tmB2, bar, k0, n0, pl);
      };
      auto b_runs = [&](uint32_t at, uint32_t bar, int k0, int pl) {
        load4<CTAS == 2>(at, mapB, bar, 0, k0, n0 / 64, pl);
        if (GATED && CTAS == 1) load4<CTAS == 2>(at + second, &tmB2, bar, 0, k0, n0 / 64, pl);
      };
      if (!p.a_mn && !p.b_mn) stream(a_rows, b_rows);
      else if (!p.a_mn && p.b_one) stream(a_rows, b_runs);
      else if (p.a_one && p.b_one) stream(a_runs, b_runs);
      else
        stream(
            [&](uint32_t at, uint32_t bar, int k0, int pl) {
              if (!p.a_mn) a_rows(at, bar, k0, pl);
              else if (p.a_one) a_runs(at, bar, k0, pl);
              else
                for (int i = 0; i < p.a_boxes; ++i) load3<CTAS == 2>(at + i * 8192, &tmA, bar, m0 + 64 * i, k0, pl);
            },
            [&](uint32_t at, uint32_t bar, int k0, int pl) {
              if (!p.b_mn) b_rows(at, bar, k0, pl);
              else if (p.b_one) b_runs(at, bar, k0, pl);
              else
                for (int i = 0; i < rows; i += 64) {
                  load3<CTAS == 2>(at + i * 128, mapB, bar, n0 + i, k0, pl);
                  if (GATED && CTAS == 1) load3<CTAS == 2>(at + second + i * 128, &tmB2, bar, n0 + i, k0, pl);
                }
            });
    }
  };

  if (warp == EPI_WARPS && lane == 0) {
    produce(0, CTAS == 1 && p.two ? 2 : 1);
    if constexpr (CTAS == 2) {   // the pair's last arrivals on this CTA's barriers, before it may exit
      const uint32_t from = loads > (uint32_t)p.stages ? loads - p.stages : 0u;
      for (uint32_t i = from; i < loads && !aborted; ++i)
        tc::mbar_wait(&empty[i % p.stages], (i / p.stages) & 1, p.status, aborted);
    }
  } else if (warp == EPI_WARPS + 1 && lane == 0) {
    uint32_t it = 0;
    Ring r;
    if (CTAS == 1 || rank == 0) {
      // ---- MMA issuer (stops at its first failed wait) ----
      const uint32_t idesc = mma_desc(p, BM * CTAS);
      const uint64_t a_desc = first_desc(sbase, p.a_mn), b_desc = first_desc(sbase + p.a_slot, p.b_mn);
      const uint32_t a_step = p.a_mn ? 128 : 2, b_step = p.b_mn ? 128 : 2;
      if (CTAS == 1 && p.two && first_item < p.items)
        issue_half(p, 0, tbase, sbase, split_blocks(p, first_item % p.splits) * p.pairs, full, empty, &accf[0], aborted);
      for (int w = CTAS == 1 && p.two ? p.items : first_item; w < p.items && !aborted; w += step) {
        const int blocks = split_blocks(p, w % p.splits);
        for (int seg = 0; seg < blocks && !aborted; seg += p.seg_kb, ++it) {
          const Acc acc(p, it);
          const uint32_t d = tbase + acc.off;
          if (!(CTAS == 2 ? tc::mbar_wait_cluster(&acce[acc.slot], acc.phase ^ 1, p.status, aborted)
                          : tc::mbar_wait(&acce[acc.slot], acc.phase ^ 1, p.status, aborted)))
            break;
          tc::tc_fence_after();
          const int steps = min(p.seg_kb, blocks - seg) * p.pairs;
          for (int i = 0; i < steps; ++i, r.next(p.stages)) {
            const uint32_t s = r.slot;
            if (!(CTAS == 2 ? tc::mbar_wait_pair(&full[s], r.phase, p.status, aborted)
                            : tc::mbar_wait(&full[s], r.phase, p.status, aborted)))
              break;
            tc::tc_fence_after();
            // K-major: 16 elements = 32 bytes along the swizzled rows; M/N-major: 16 rows of 128 bytes
            const uint32_t at = (s * (uint32_t)stage_bytes) >> 4;
#pragma unroll
            for (int kk = 0; kk < BK / 16; ++kk) {
              const uint64_t ad = a_desc + at + kk * a_step, bd = b_desc + at + kk * b_step;
              if constexpr (CTAS == 2) tc::mma2_bf16(d, ad, bd, idesc, i > 0 || kk > 0);
              else tc::mma_bf16(d, ad, bd, idesc, i > 0 || kk > 0);
            }
            if constexpr (CTAS == 2) tc::mma2_commit(&empty[s]);
            else tc::mma_commit(&empty[s]);
          }
          if (aborted) break;
          if constexpr (CTAS == 2) tc::mma2_commit(&accf[acc.slot]);
          else tc::mma_commit(&accf[acc.slot]);
        }
      }
    }
  } else if (warp < EPI_WARPS) {
    auto second = [&] {   // the first two epilogue warps' part of the MMAs and the loads
      if (CTAS == 1 && p.two && warp < 2) {
        if (warp == 0 && lane == 0 && first_item < p.items)
          issue_half(p, 1, tbase + kTotal, sbase, split_blocks(p, first_item % p.splits) * p.pairs, full, empty, &accf[0], aborted);
        if (warp == 1 && lane == 0) produce(1, 2);
        __syncwarp();
      }
    };
    if constexpr (STAGED)
      staged_epilogue<KIND, OUT, EACT, LEAN, CTAS>(p, tm, area, aux_bar, accf, acce, tbase, first_item, step, rank, warp, lane,
                                            aborted, second);
    if constexpr (!STAGED) {
    second();
    // ---- epilogue: warp w drains lanes 32 (w % 4).., every other 32-column chunk of the tile ----
    const int quad = warp & 3, half = warp >> 2;
    const uint32_t lane_addr = tbase + ((uint32_t)(quad * 32) << 16);
    uint32_t it = 0;
    for (int w = first_item; w < p.items; w += step, ++it) {
      uint32_t mi, ni;
      int split;
      tile_at(p, (uint32_t)w, mi, ni, split);
      const int64_t row = (int64_t)mi * BM * CTAS + rank * BM + quad * 32 + lane, c0 = (int64_t)ni * p.part;
      const int cols = (int)(p.n - c0 < p.part ? p.n - c0 : p.part);
      const int segs = (split_blocks(p, split) + p.seg_kb - 1) / p.seg_kb;
      for (int s = 0; s + 1 < segs; ++s, ++it) {
        const Acc acc(p, it);
        tc::mbar_wait_long(&accf[acc.slot], acc.phase, p.status, aborted);
        tc::tc_fence_after();
        fold_segment<GATED, 32>(p, lane_addr + acc.off, lane_addr + kTotal, half * 32, 64, cols, s > 0);
        free_acc<CTAS>(&acce[acc.slot], lane);
      }
      const Acc acc(p, it);
      const uint32_t d = lane_addr + acc.off;
      tc::mbar_wait_long(&accf[acc.slot], acc.phase, p.status, aborted);
      tc::tc_fence_after();
#pragma unroll 1
      for (int c = half * 32; c < cols; c += 64) {
        float z[32], u[32];
        tc::tmem_ld32(d + c, z);
        if (GATED) tc::tmem_ld32(d + p.part + c, u);
        if (has_total(p, segs)) {
          float t[32];
          tc::tmem_ld32(lane_addr + kTotal + c, t);
#pragma unroll
          for (int e = 0; e < 32; ++e) z[e] += t[e];
          if (GATED) {
            tc::tmem_ld32(lane_addr + kTotal + p.part + c, t);
#pragma unroll
            for (int e = 0; e < 32; ++e) u[e] += t[e];
          }
        }
        chunk<KIND, OUT>(p, row, row < p.m, c0 + c, cols - c < 32 ? cols - c : 32, split, z, u, lane);
      }
      free_acc<CTAS>(&acce[acc.slot], lane);
    }
    }
  }
  tc::tc_fence_before();
  if (__syncthreads_or(aborted)) {   // abort path: drain the producer's loads and the issuer's MMAs
    if (CTAS == 1 && p.two) {
      // the two producers' last loads, each in its own half of the slots
      const uint32_t part = warp == 1 ? 1u : 0u, half = (uint32_t)p.stages / 2;
      if ((warp == EPI_WARPS || warp == 1) && lane == 0)
        for (uint32_t j = loads > half ? loads - half : 0u; j < loads; ++j)
          tc::mbar_wait_drain(&full[(part + 2 * j) % p.stages], (part + 2 * j) / p.stages & 1, p.status);
    } else if (warp == EPI_WARPS && lane == 0) {
      // the odd CTA's loads complete on the even one's barriers: it waits until the MMAs have read them
      tc::drain_ring(CTAS == 2 && rank ? empty : full, p.stages, loads, p.status);
    }
    if (warp == EPI_WARPS + 1 && lane == 0 && rank == 0) {
      if constexpr (CTAS == 2) {
        tc::mma2_commit(drain);
        tc::mbar_wait_drain(drain, 0, p.status);
      } else {
        tc::drain_mma(drain, p.status);
      }
    }
    if (CTAS == 1 && p.two && tid == 0) tc::drain_mma(drain + 1, p.status);
    __syncthreads();
  }
  if constexpr (CTAS == 2) tc::cluster_sync();   // no CTA leaves while the other one may still reach its shared memory
  if (warp == 0) {
    tc::tc_fence_after();
    if constexpr (CTAS == 2) tc::tmem_dealloc2(tbase, 512);
    else tc::tmem_dealloc(tbase, 512);
  }
}

template <int KIND, int OUT, int CTAS, bool STAGED, int EACT, bool LEAN>
int launch(const Maps& tm, const Params& p, cudaStream_t stream) {
  static bool attr_set[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!attr_set[dev & 63]) {
    cudaError_t e = cudaFuncSetAttribute(k_product_tc<KIND, OUT, CTAS, STAGED, EACT, LEAN>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         SMEM_MAX);
    if (e != cudaSuccess) {
      set_error("cudaFuncSetAttribute(product): %s", cudaGetErrorString(e));
      return SF_ERR_CUDA;
    }
    attr_set[dev & 63] = true;
  }
  const int64_t most = num_sms() / CTAS;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((p.items < most ? p.items : most) * CTAS));
  cfg.blockDim = dim3(threads_of(STAGED));
  cfg.dynamicSmemBytes = SMEM_MAX;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  if (CTAS == 2) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = CTAS;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.numAttrs = 1;
  }
  if (pdl_enabled()) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  cudaLaunchKernelEx(&cfg, k_product_tc<KIND, OUT, CTAS, STAGED, EACT, LEAN>, tm, p);
  count_launch();
  return check_launch("linear product");
}

template <int KIND, int OUT, bool STAGED, int EACT, bool LEAN = false>
int launch_ctas(int ctas, const Maps& tm, const Params& p, cudaStream_t stream) {
  return ctas == 2 ? launch<KIND, OUT, 2, STAGED, EACT, LEAN>(tm, p, stream)
                   : launch<KIND, OUT, 1, STAGED, EACT, LEAN>(tm, p, stream);
}
template <int KIND>
int launch_staged_bf16(int ctas, const Maps& tm, const Params& p, cudaStream_t stream) {
  if constexpr (KIND != kDLinear) {
    constexpr int own = KIND == kLinear ? SF_POST_NONE : SF_POST_SILU;
    if (p.act == own && !p.two && p.kb_split <= p.seg_kb && !p.bias && !p.saved && !p.colpart && (KIND != kLinear || !p.aux))
      return launch_ctas<KIND, kOutBf16, true, own, true>(ctas, tm, p, stream);
  }
  int st = SF_OK;
  SF_ACT_SWITCH(p.act, (st = launch_ctas<KIND, kOutBf16, true, ACT>(ctas, tm, p, stream)))
  return st;
}

// One translation unit for each kind of epilogue.
int launch_linear(int out_kind, int ctas, const Maps& tm, const Params& p, cudaStream_t stream);
int launch_gated(int out_kind, int ctas, const Maps& tm, const Params& p, cudaStream_t stream);
int launch_dlinear(int out_kind, int ctas, const Maps& tm, const Params& p, cudaStream_t stream);
int launch_dgated(int out_kind, int ctas, const Maps& tm, const Params& p, cudaStream_t stream);

}  // namespace pr
}  // namespace lg
}  // namespace sf
