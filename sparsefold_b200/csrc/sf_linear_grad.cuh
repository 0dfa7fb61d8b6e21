// Shared by the linear layers with gradients (sf_linear_act, sf_gated_linear and their backward
// calls): activations with derivatives, the operands and epilogues of a product, workspace carving.
#pragma once

#include "sf_common.cuh"

namespace sf {
namespace lg {

// ---- activations -------------------------------------------------------------------------------
// In fp32.  FAST serves bf16 results: one ex2 and one reciprocal, off by about 2^-21 of the value (gelu: below), where
// the result keeps 2^-9 (65536 x 128 -> 2 x 512, silu: the forward kernel took 85 us with expf and a division).
template <bool FAST>
__device__ __forceinline__ float sigmoid_of(float z) {
  if constexpr (FAST) return __fdividef(1.0f, 1.0f + __expf(-z));
  return 1.0f / (1.0f + expf(-z));
}
// Phi(z) and exp(-z^2 / 2).  Exact form: erfc(-z / sqrt 2) / 2 keeps its relative accuracy for large negative z,
// where (1 + erf) / 2 cancels.  FAST: q = Phi(-|z|) = exp(-z^2 / 2) t P(t) with t = 1 / (1 + c |z|), and Phi = q for
// z < 0, else 1 - q, so that the negative tail keeps its relative accuracy too: P is a fit of exp(z^2 / 2) Phi(-|z|) / t
// that levels the relative error over |z| <= 13.5 (8.5e-8), and with the roundings q is off by 6e-7 of itself up to
// |z| = 3, by 2e-6 up to 6 and 7.5e-6 up to 13, where it leaves the normal numbers of bf16.
constexpr float kTailC = 0.43f * 0.70710678118654752f;
constexpr float tail(int i) {
  constexpr float c[8] = {0.12125748721843123f,  0.12218486631877787f, 0.10249371350081203f,  0.12336096113131473f,
                          -0.0427442795261602f, 0.19172064226657742f, -0.15510785536828334f, 0.036834502628450894f};
  return c[i];
}
template <bool FAST>
__device__ __forceinline__ void normal_cdf(float z, float& cdf, float& e) {
  if constexpr (FAST) {
    e = __expf(-0.5f * z * z);
    const float t = __fdividef(1.0f, fmaf(kTailC, fabsf(z), 1.0f));
    float y = tail(7);
#pragma unroll
    for (int i = 6; i >= 0; --i) y = fmaf(t, y, tail(i));
    const float q = t * y * e;
    cdf = z < 0.f ? q : 1.0f - q;
  } else {
    cdf = 0.5f * erfcf(-0.70710678118654752f * z);
    e = expf(-0.5f * z * z);
  }
}
template <int ACT, bool FAST>
__device__ __forceinline__ float act_value(float z) {
  if constexpr (ACT == SF_POST_SILU) return z * sigmoid_of<FAST>(z);
  if constexpr (ACT == SF_POST_GELU) {
    float p, e;
    normal_cdf<FAST>(z, p, e);
    return z * p;
  }
  if constexpr (ACT == SF_POST_SIGMOID) return sigmoid_of<FAST>(z);
  if constexpr (ACT == SF_POST_RELU) return z < 0.f ? 0.f : z;      // a NaN stays one
  return z;
}
// Value and derivative (relu's at 0 is 0).
template <int ACT, bool FAST>
__device__ __forceinline__ void act_grad(float z, float& a, float& da) {
  if constexpr (ACT == SF_POST_SILU) {
    const float p = sigmoid_of<FAST>(z);
    a = z * p;
    da = fmaf(a, 1.0f - p, p);
  } else if constexpr (ACT == SF_POST_GELU) {
    float p, e;
    normal_cdf<FAST>(z, p, e);
    a = z * p;
    da = fmaf(z * 0.39894228040143268f, e, p);
  } else if constexpr (ACT == SF_POST_SIGMOID) {
    a = sigmoid_of<FAST>(z);
    da = a * (1.0f - a);
  } else if constexpr (ACT == SF_POST_RELU) {
    a = z < 0.f ? 0.f : z;
    da = z > 0.f ? 1.f : (z <= 0.f ? 0.f : z);
  } else {
    a = z;
    da = 1.f;
  }
}
// Calls f<ACT>() for the runtime activation.
#define SF_ACT_SWITCH(act, ...)                                          \
  switch (act) {                                                         \
    case SF_POST_RELU: { constexpr int ACT = SF_POST_RELU; __VA_ARGS__; break; }       \
    case SF_POST_SILU: { constexpr int ACT = SF_POST_SILU; __VA_ARGS__; break; }       \
    case SF_POST_SIGMOID: { constexpr int ACT = SF_POST_SIGMOID; __VA_ARGS__; break; } \
    case SF_POST_GELU: { constexpr int ACT = SF_POST_GELU; __VA_ARGS__; break; }       \
    default: { constexpr int ACT = SF_POST_NONE; __VA_ARGS__; break; }                 \
  }

// An fp32 value as three bf16 terms, x = t0 + t1 + t2 to 2^-24 of x: each is the rest rounded to nearest.
// A first term that would round past the largest bf16 is cut instead; an infinity or NaN has no rest.
__device__ __forceinline__ void split3(float x, bf16 (&t)[3]) {
  t[0] = __float2bfloat16_rn(x);
  float r = 0.f;
  if (fabsf(x) <= 3.4028234663852886e38f) {
    if (__hisinf(t[0])) t[0] = __float2bfloat16_rz(x);
    r = x - __bfloat162float(t[0]);
  }
  t[1] = __float2bfloat16_rn(r);
  t[2] = __float2bfloat16_rn(r - __bfloat162float(t[1]));
}

// ---- operands ----------------------------------------------------------------------------------
// A matrix as a product reads it: `planes` bf16 matrices (1, or the 3 terms of fp32 values) of `outer` rows
// of `inner` contiguous elements, rows `pitch` apart, base and pitch multiples of 16 bytes.
struct Planes {
  const bf16* p;
  int64_t inner, outer, pitch, plane;
  int planes;
  Planes rows(int64_t from, int64_t count) const {
    Planes q = *this;
    q.p += from * pitch;
    q.outer = count;
    return q;
  }
};
// One side of a product: row i, depth k.  k_major: the depth is the inner axis.
struct Operand {
  Planes m;
  bool k_major;
  int64_t rows() const { return k_major ? m.outer : m.inner; }
  int64_t depth() const { return k_major ? m.inner : m.outer; }
};

// ---- epilogues ---------------------------------------------------------------------------------
// What becomes of the accumulated product z[m][j] (+ bias[j]):
//   kLinear  out = act(z) + aux                        (aux: residual, or null); saved = z
//   kGated   out[m][i] = act(z[m][i]) * z[m][n + i]    saved = z
//   kDLinear out = aux * act'(z)                       (aux: dy)
//   kDGated  out[m][i] = aux * z[m][n+i] * act'(z[m][i]), out[m][n+i] = aux * act(z[m][i])
// colpart (kDLinear, kDGated): sums of out before its rounding over the rows of each block of 32.
enum EpiKind { kLinear = 0, kGated = 1, kDLinear = 2, kDGated = 3 };
enum OutKind { kOutF32 = 0, kOutBf16 = 1 };
struct Epi {
  int kind, act;
  int64_t n;               // output features; the product has 2n columns for the gated kinds
  const float* bias;
  const void* aux;         // of out's type
  int64_t aux_sr;
  void* out;
  int out_kind;
  int64_t out_sr;
  float* saved;
  float* colpart;
};

// Carves the workspace, or (dry) only adds up what a call takes of it.
struct Arena {
  Workspace ws;
  bool dry;
  Arena(void* p, size_t bytes, bool d) : ws(p, d ? ~size_t(0) >> 1 : bytes), dry(d) {}
  template <typename T>
  T* take(int64_t count) { return ws.take<T>((size_t)count); }
};

// Sums of partials that a call still owes, all in its last launch: the splits of a product, part [splits][m][pitch] ->
// out [m][n] (fp32 or bf16), and column sums (kColumns), part [splits][pitch] -> out [n].
enum SumKind { kSplitF32 = 0, kSplitBf16 = 1, kColumns = 2 };
struct SumJob {
  const float* part;
  void* out;
  int64_t m, n, pitch, out_sr;
  int splits, kind;
  unsigned end;            // blocks up to and with this job's
};
constexpr int kSumJobs = 4;
struct SumJobs {
  SumJob job[kSumJobs];
  int count;
};
struct Sums {
  SumJobs jobs{};
  int add(const SumJob& j, cudaStream_t stream);
  int flush(cudaStream_t stream);
};

// z = A B^T with its epilogue; the gated kinds take the gate's and the other rows of B as b and b2.  Where K is split,
// out is there after the flush of `sums`.
int product_tc(const Operand& a, const Operand& b, const Operand* b2, const Epi& e, Arena& ar, Sums& sums, cudaStream_t stream);

// The same for a few rows, straight from x and W (fp32 or bf16, as aux and out): W stored by features (k_inner) or
// by inputs, rows w_s apart; w2: the second half's weight (gated kinds).  dbias: column sums of out (kDLinear,
// kDGated) over each kFewRows rows, [..][n or 2n], or null.
constexpr int kFewRows = 8, kFewF32 = 32;
int few_rows(int dtype, const void* x, int64_t x_sr, int64_t rows, int64_t k, const void* w, const void* w2, int64_t w_s,
             bool k_inner, const Epi& e, float* dbias, cudaStream_t stream);

// Whether few rows run on it.  fp32: up to 8 always, as the tensor cores need W's terms written and read first (8 rows,
// 768 -> 2 x 2048: 9 us against 38), and up to 32, W read once for each 8, while it is small (16 rows, 64 -> 2 x 264:
// 2.6 us against 11, gradients 18 against 29; 32 rows, 768 -> 2 x 768, 4.7 MB: 12.3 against 19.5, gradients 39 against
// 43; 24 rows, 768 -> 2 x 2048, 13 MB: 23 against 24, gradients 66 against 53).  bf16: one row of a W stored by features,
// and otherwise while W is below 16 MB, where a tile's latency counts (8 rows, 768 -> 2 x 768: 4.0 us against 7.2;
// stored by inputs, 4 rows 6.6 against 7.8, 5 rows 11 against 7.8); of a larger one the tiles read more per second (3
// rows, 4096 -> 2 x 4096: 28 us against 24; stored by inputs, 1 row 60 against 26).
inline bool few_form(int dtype, int64_t rows, int64_t weight_bytes, bool k_inner) {
  if (dtype == SF_F32) return rows <= (weight_bytes <= (int64_t(8) << 20) ? kFewF32 : kFewRows);
  if (rows > kFewRows) return false;
  if (weight_bytes > (int64_t(16) << 20)) return rows == 1 && k_inner;
  return k_inner || rows <= 4;
}

}  // namespace lg
}  // namespace sf
