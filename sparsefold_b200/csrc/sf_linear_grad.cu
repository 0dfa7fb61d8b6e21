// Linear layers with gradients: entry points, argument checks and the passes around the products.
//
// Forward: one product with its epilogue.  Backward, with z the pre-activations:
//   1. dz from dy and z (kDLinear / kDGated): read back from `saved`, or from the product x W^T computed
//      again;  no pass at all for a linear layer without activation, where dz = dy;
//   2. dx = dz W;   3. dW = dz^T x (or its transpose, whichever way dwt is laid out);
//   4. dbias: column sums of dz before its rounding.
// dz is held in the call's type: a bf16 dz is one operand of one product, as x and W are, where an unrounded one would be
// two terms and twice the products of 2 and 3 (8192 x 2048 -> 2 x 8192: 1650 GFLOP in all, two thirds of it theirs).  The
// rounding's 2^-9 on average adds to that of the result: 0.0023 of a bf16 gradient's norm against fp64, 0.0017 without it.
#include <type_traits>

#include "sf_linear_grad.cuh"
#include "sf_simt.cuh"
#include "sf_tc.cuh"

namespace sf {
namespace lg {
namespace {

// ---- operands that TMA cannot read as they are --------------------------------------------------
// dst[plane][outer][pitch] = src[outer][stride] as bf16 (one plane) or as the three terms of fp32, zero
// from `inner` on; eight elements per thread.  Reads and writes each element once; taken for fp32 and
// for bf16 whose rows do not start on 16-byte boundaries.  One launch for all matrices of a product.
struct PackJob {
  const void* src;
  bf16* dst;
  int64_t inner, outer, stride, pitch, plane;
  int f32, vec;
  unsigned end;          // blocks up to and with this job's
};
constexpr int kPackJobs = 4;
struct PackJobs {
  PackJob job[kPackJobs];
  int count;
};

template <typename T>
__device__ __forceinline__ void pack8(const PackJob& j, int64_t i) {
  const int64_t per = j.pitch / 8;
  if (i >= j.outer * per) return;
  const int64_t row = i / per, c = (i - row * per) * 8;
  const T* s = static_cast<const T*>(j.src) + row * j.stride + c;
  float v[8];
  if (j.vec && c + 8 <= j.inner) ld8(s, v);
  else
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = c + e < j.inner ? ld(s + e) : 0.f;
  bf16* d = j.dst + row * j.pitch + c;
  if constexpr (sizeof(T) == 2) {
    st8(d, v);
  } else {
    bf16 t[8][3];
#pragma unroll
    for (int e = 0; e < 8; ++e) split3(v[e], t[e]);
#pragma unroll
    for (int q = 0; q < 3; ++q) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = __bfloat162float(t[e][q]);
      st8(d + q * j.plane, v);
    }
  }
}

__global__ void __launch_bounds__(256) k_pack(const __grid_constant__ PackJobs jobs) {
  tc::griddep_wait();
  tc::griddep_launch();
  int k = 0;
  while (blockIdx.x >= jobs.job[k].end) ++k;
  const PackJob& j = jobs.job[k];
  const int64_t i = (int64_t)(blockIdx.x - (k ? jobs.job[k - 1].end : 0u)) * 256 + threadIdx.x;
  if (j.f32) pack8<float>(j, i);
  else pack8<bf16>(j, i);
}

int64_t pad8(int64_t n) { return (n + 7) / 8 * 8; }

// The packs that a call has asked for and not launched yet.
struct Packer {
  PackJobs jobs{};
  // The planes of `outer` rows of `inner` elements, `stride` apart: the matrix itself where TMA can read it, else
  // room for them, filled by the next flush().
  int planes_of(const void* p, int dtype, int64_t inner, int64_t outer, int64_t stride, Planes& out, Arena& ar,
                cudaStream_t stream) {
    if (outer == 1) stride = pad8(inner);
    const bool al = (reinterpret_cast<uintptr_t>(p) & 15) == 0;
    if (dtype == SF_BF16 && al && stride % 8 == 0) {
      out = Planes{static_cast<const bf16*>(p), inner, outer, stride, 0, 1};
      return SF_OK;
    }
    const int64_t pitch = pad8(inner);
    const int planes = dtype == SF_F32 ? 3 : 1;
    bf16* d = ar.take<bf16>(planes * outer * pitch);
    out = Planes{d, inner, outer, pitch, outer * pitch, planes};
    if (ar.dry) return SF_OK;
    const int64_t blocks = (outer * (pitch / 8) + 255) / 256;
    if (jobs.count == kPackJobs || (jobs.count && jobs.job[jobs.count - 1].end + blocks > 0x7fffffff)) SF_TRY(flush(stream));
    SF_REQUIRE(blocks <= 0x7fffffff, "pack: %lld x %lld elements", (long long)outer, (long long)inner);
    const unsigned before = jobs.count ? jobs.job[jobs.count - 1].end : 0u;
    jobs.job[jobs.count++] = PackJob{p, d, inner, outer, stride, pitch, outer * pitch, dtype == SF_F32,
                                     dtype == SF_F32 && al && stride % 4 == 0, before + (unsigned)blocks};
    return SF_OK;
  }
  int flush(cudaStream_t stream) {
    if (jobs.count == 0) return SF_OK;
    launch_pdl(k_pack, dim3(jobs.job[jobs.count - 1].end), dim3(256), 0, stream, jobs);
    jobs.count = 0;
    count_launch();
    return check_launch("pack");
  }
};

// ---- dz from dy and the saved pre-activations -----------------------------------------------------
// V columns (of each half) of a block of 32 rows per thread; bound by the memory: 4 bytes of each
// pre-activation and dy in, dz out.  colpart: the block's column sums of dz before its rounding.
template <int KIND, int OUT, int V, int ACT>
__device__ __forceinline__ void dz_rows(const Epi& e, int64_t from, int64_t end, int64_t c, int64_t wide, float (&s0)[V],
                                        float (&s1)[V]) {
  constexpr bool GATED = KIND == kDGated;
  using T = typename std::conditional<OUT == kOutBf16, bf16, float>::type;
  const T* dy = static_cast<const T*>(e.aux);
  T* out = static_cast<T*>(e.out);
#pragma unroll 4
  for (int64_t m = from; m < end; ++m) {
    float z[V], u[V], x[V];
    if constexpr (V == 4) {
      const float4 q = *reinterpret_cast<const float4*>(e.saved + m * wide + c);
      z[0] = q.x, z[1] = q.y, z[2] = q.z, z[3] = q.w;
      if (GATED) {
        const float4 r = *reinterpret_cast<const float4*>(e.saved + m * wide + e.n + c);
        u[0] = r.x, u[1] = r.y, u[2] = r.z, u[3] = r.w;
      }
    } else {
      z[0] = e.saved[m * wide + c];
      if (GATED) u[0] = e.saved[m * wide + e.n + c];
    }
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = ld(dy + m * e.aux_sr + c + i);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float a, da;
      act_grad<ACT, OUT == kOutBf16>(z[i], a, da);
      z[i] = GATED ? x[i] * u[i] * da : x[i] * da;
      u[i] = x[i] * a;
      s0[i] += z[i];
      s1[i] += u[i];
    }
#pragma unroll
    for (int h = 0; h < (GATED ? 2 : 1); ++h) {
      T* o = out + m * e.out_sr + h * e.n + c;
      const float(&v)[V] = h ? u : z;
      if constexpr (V == 4 && sizeof(T) == 2) {
        const __nv_bfloat162 lo = __floats2bfloat162_rn(v[0], v[1]), hi = __floats2bfloat162_rn(v[2], v[3]);
        *reinterpret_cast<uint2*>(o) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
      } else if constexpr (V == 4) {
        *reinterpret_cast<float4*>(o) = make_float4(v[0], v[1], v[2], v[3]);
      } else {
        st(o, v[0]);
      }
    }
  }
}

template <int KIND, int OUT, int V>
__global__ void __launch_bounds__(128) k_dz(Epi e, int64_t rows, unsigned row_blocks) {
  tc::griddep_wait();
  tc::griddep_launch();
  const unsigned cb = blockIdx.x / row_blocks;      // the blocks of one column range are neighbours
  const int64_t c = ((int64_t)cb * blockDim.x + threadIdx.x) * V, blk = blockIdx.x - cb * row_blocks;
  if (c >= e.n) return;
  const int64_t wide = KIND == kDGated ? 2 * e.n : e.n, end = (blk + 1) * 32 < rows ? (blk + 1) * 32 : rows;
  float s0[V] = {}, s1[V] = {};
  SF_ACT_SWITCH(e.act, (dz_rows<KIND, OUT, V, ACT>(e, blk * 32, end, c, wide, s0, s1)))
  if (!e.colpart) return;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    e.colpart[blk * wide + c + i] = s0[i];
    if (KIND == kDGated) e.colpart[blk * wide + e.n + c + i] = s1[i];
  }
}

template <int KIND, int OUT>
int launch_dz(const Epi& e, int64_t rows, cudaStream_t stream) {
  const bool vec = e.n % 4 == 0 && e.out_sr % 4 == 0 &&
                   ((reinterpret_cast<uintptr_t>(e.saved) | reinterpret_cast<uintptr_t>(e.out)) & 15) == 0;
  // one axis of blocks: the second one ends at 65535, which is 8.4 M columns in ranges of 128
  const int64_t per = vec ? 512 : 128, row_blocks = (rows + 31) / 32, blocks = row_blocks * ((e.n + per - 1) / per);
  SF_REQUIRE(blocks <= 0x7fffffff, "dz: %lld x %lld elements", (long long)rows, (long long)e.n);
  if (vec) launch_pdl(k_dz<KIND, OUT, 4>, dim3((unsigned)blocks), dim3(128), 0, stream, e, rows, (unsigned)row_blocks);
  else launch_pdl(k_dz<KIND, OUT, 1>, dim3((unsigned)blocks), dim3(128), 0, stream, e, rows, (unsigned)row_blocks);
  count_launch();
  return check_launch("dz");
}

// ---- sums of partials -----------------------------------------------------------------------------
// 32 columns by 8 rows of threads over rows [from, end) of p; the eight row sums added in order.
template <typename T>
__device__ __forceinline__ void column_sum(const T* __restrict__ p, int64_t j, int64_t from, int64_t end, int64_t cols,
                                           int64_t sr, float* __restrict__ out) {
  __shared__ float s_sum[8][32];
  const int lane = threadIdx.x & 31, ty = threadIdx.x >> 5;
  float s = 0.f;
  if (j < cols)
#pragma unroll 4
    for (int64_t r = from + ty; r < end; r += 8) s += ld(p + r * sr + j);
  s_sum[ty][lane] = s;
  __syncthreads();
  if (ty == 0 && j < cols) {
#pragma unroll
    for (int i = 1; i < 8; ++i) s += s_sum[i][lane];
    out[j] = s;
  }
}

// out[slice][j] = sum over the slice's rows of p[row][j].
template <typename T>
__global__ void __launch_bounds__(256) k_colsum(const T* __restrict__ p, int64_t rows, int64_t cols, int64_t sr,
                                                int64_t per, float* __restrict__ out) {
  tc::griddep_wait();
  tc::griddep_launch();
  const int64_t from = blockIdx.y * per, end = from + per < rows ? from + per : rows;
  column_sum(p, (int64_t)blockIdx.x * 32 + (threadIdx.x & 31), from, end, cols, sr, out + blockIdx.y * cols);
}

// Four columns of a row per thread: the sum over the splits, in order.
template <typename T>
__device__ __forceinline__ void split_sum(const SumJob& j, int64_t i) {
  const int64_t per = j.pitch / 4;
  if (i >= j.m * per) return;
  const int64_t row = i / per, c = (i - row * per) * 4;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k = 0; k < j.splits; ++k) {
    const float4 v = *reinterpret_cast<const float4*>(j.part + ((int64_t)k * j.m + row) * j.pitch + c);
    s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
  }
  T* o = static_cast<T*>(j.out) + row * j.out_sr + c;
  const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (c + e < j.n) st(o + e, v[e]);
}

// All sums that a call owes, in one launch: alone each is a few microseconds of latency.
__global__ void __launch_bounds__(256) k_sums(const __grid_constant__ SumJobs jobs) {
  tc::griddep_wait();
  tc::griddep_launch();
  int k = 0;
  while (blockIdx.x >= jobs.job[k].end) ++k;
  const SumJob& j = jobs.job[k];
  const int64_t blk = blockIdx.x - (k ? jobs.job[k - 1].end : 0u), i = blk * 256 + threadIdx.x;
  if (j.kind == kColumns)
    column_sum(j.part, blk * 32 + (threadIdx.x & 31), 0, j.splits, j.n, j.pitch, static_cast<float*>(j.out));
  else if (j.kind == kSplitF32) split_sum<float>(j, i);
  else split_sum<bf16>(j, i);
}

// Sums of p's columns in a fixed order: slices of rows here, the slices with the call's other sums.
int colsum(const void* p, int dtype, int64_t rows, int64_t cols, int64_t sr, float* out, Arena& ar, Sums& sums,
           cudaStream_t stream) {
  int64_t slices = (rows + 127) / 128;
  if (slices > 128) slices = 128;
  const int64_t per = (rows + slices - 1) / slices;
  slices = (rows + per - 1) / per;
  const bool last = slices == 1 && dtype == SF_F32;
  float* mid = slices > 1 ? ar.take<float>(slices * cols) : out;
  if (ar.dry) return SF_OK;
  if (last) return sums.add(SumJob{static_cast<const float*>(p), out, 1, cols, sr, cols, (int)rows, kColumns, 0}, stream);
  const dim3 grid((unsigned)((cols + 31) / 32), (unsigned)slices);
  if (dtype == SF_F32) launch_pdl(k_colsum<float>, grid, dim3(256), 0, stream, (const float*)p, rows, cols, sr, per, mid);
  else launch_pdl(k_colsum<bf16>, grid, dim3(256), 0, stream, (const bf16*)p, rows, cols, sr, per, mid);
  count_launch();
  SF_TRY(check_launch("column sums"));
  return slices > 1 ? sums.add(SumJob{mid, out, 1, cols, cols, cols, (int)slices, kColumns, 0}, stream) : SF_OK;
}

int zero(void* p, size_t bytes, cudaStream_t stream) {
  cudaError_t e = cudaMemsetAsync(p, 0, bytes, stream);
  if (e != cudaSuccess) {
    set_error("cudaMemsetAsync: %s", cudaGetErrorString(e));
    return SF_ERR_CUDA;
  }
  return SF_OK;
}

int check(const sf_linear_args* g, bool gated, bool backward, const char* what) {
  SF_REQUIRE(g != nullptr, "%s: null arguments", what);
  SF_REQUIRE(g->dtype == SF_F32 || g->dtype == SF_BF16, "%s: unsupported dtype %d", what, g->dtype);
  SF_REQUIRE(g->activation >= SF_POST_NONE && g->activation <= SF_POST_GELU, "%s: bad activation %d", what,
             g->activation);
  const int64_t N = gated ? 2 * g->n : g->n, big = int64_t(1) << 30;   // tiles behind the end still fit int
  SF_REQUIRE(g->rows >= 0 && g->k > 0 && g->n > 0 && g->rows < big && g->k < big && N < big,
             "%s: bad sizes rows=%lld k=%lld n=%lld", what, (long long)g->rows, (long long)g->k, (long long)g->n);
  SF_REQUIRE((g->x || g->rows == 0) && g->wt, "%s: x or wt is null", what);
  SF_REQUIRE(g->x_sr >= g->k || g->rows <= 1, "%s: x row stride %lld below k=%lld", what, (long long)g->x_sr,
             (long long)g->k);
  SF_REQUIRE((g->w_sk == 1 && g->w_sn >= g->k) || (g->w_sn == 1 && g->w_sk >= N),
             "%s: wt strides (%lld, %lld) for [%lld][%lld]", what, (long long)g->w_sn, (long long)g->w_sk,
             (long long)N, (long long)g->k);
  if (!backward) {
    SF_REQUIRE(g->y || g->rows == 0, "%s: y is null", what);
    SF_REQUIRE(!gated || !g->residual, "%s: no residual in the gated form", what);
    SF_REQUIRE(!g->residual || g->r_sr >= g->n || g->rows <= 1, "%s: residual row stride %lld below n", what,
               (long long)g->r_sr);
  } else {
    SF_REQUIRE(g->dy || g->rows == 0, "%s: dy is null", what);
    SF_REQUIRE(g->dy_sr >= g->n || g->rows <= 1, "%s: dy row stride %lld below n", what, (long long)g->dy_sr);
    SF_REQUIRE(!g->dwt || (g->dw_sk == 1 && g->dw_sn >= g->k) || (g->dw_sn == 1 && g->dw_sk >= N),
               "%s: dwt strides (%lld, %lld)", what, (long long)g->dw_sn, (long long)g->dw_sk);
  }
  return SF_OK;
}

// The planes that several products of a call share, made when they are first asked for.
struct Shared {
  const sf_linear_args* g;
  bool gated;
  Arena& ar;
  cudaStream_t stream;
  Packer packer;
  Sums sums;
  Planes xp{}, wp{};
  bool have_x = false, have_w = false;
  int64_t wide() const { return gated ? 2 * g->n : g->n; }

  int x(Planes& out) {
    if (!have_x) SF_TRY(packer.planes_of(g->x, g->dtype, g->k, g->rows, g->x_sr, xp, ar, stream));
    have_x = true;
    out = xp;
    return SF_OK;
  }
  // The weight as it is stored: rows of k (w_sk == 1), or rows of its output features.
  bool w_k_inner() const { return g->w_sk == 1 && g->w_sn >= g->k; }
  int64_t weight_bytes() const { return wide() * g->k * (g->dtype == SF_F32 ? 4 : 2); }
  bool few() const { return few_form(g->dtype, g->rows, weight_bytes(), w_k_inner()); }
  int w(Planes& out) {
    const bool ki = w_k_inner();
    if (!have_w)
      SF_TRY(packer.planes_of(g->wt, g->dtype, ki ? g->k : wide(), ki ? wide() : g->k, ki ? g->w_sn : g->w_sk, wp, ar, stream));
    have_w = true;
    out = wp;
    return SF_OK;
  }
  // x W^T with an epilogue (the gated kinds: the gate's and the other features' rows apart)
  int forward(const Epi& e, float* dbias = nullptr) {
    if (few()) {
      if (ar.dry) return SF_OK;
      const bool ki = w_k_inner();
      const int64_t half = g->n * (ki ? g->w_sn : 1) * (g->dtype == SF_F32 ? 4 : 2);
      return few_rows(g->dtype, g->x, g->x_sr, g->rows, g->k, g->wt, gated ? static_cast<const char*>(g->wt) + half : nullptr,
                      ki ? g->w_sn : g->w_sk, ki, e, dbias, stream);
    }
    Operand a{{}, true}, b{{}, w_k_inner()}, b2 = b;
    SF_TRY(x(a.m));
    const int64_t n = g->n;
    if (gated && !b.k_major && n % 8 != 0) {   // the second half would not start on a 16-byte boundary
      const size_t esz = g->dtype == SF_F32 ? 4 : 2;
      SF_TRY(packer.planes_of(g->wt, g->dtype, n, g->k, g->w_sk, b.m, ar, stream));
      SF_TRY(packer.planes_of(static_cast<const char*>(g->wt) + n * esz, g->dtype, n, g->k, g->w_sk, b2.m, ar, stream));
    } else {
      SF_TRY(w(b.m));
      b2 = b;
      if (gated && b.k_major) {
        b2.m = b.m.rows(n, n);
        b.m = b.m.rows(0, n);
      } else if (gated) {
        b2.m.p += n;
        b.m.inner = b2.m.inner = n;
      }
    }
    SF_TRY(packer.flush(stream));
    return product_tc(a, b, gated ? &b2 : nullptr, e, ar, sums, stream);
  }
};

int forward(const sf_linear_args* g, bool gated, Arena& ar, cudaStream_t stream) {
  if (g->rows == 0) return SF_OK;
  Shared s{g, gated, ar, stream};
  SF_TRY(s.forward(Epi{gated ? kGated : kLinear, g->activation, g->n, g->bias, g->residual, g->r_sr, g->y,
                       g->dtype == SF_F32 ? kOutF32 : kOutBf16, g->n, g->saved, nullptr}));
  return s.sums.flush(stream);
}

int backward(const sf_linear_args* g, bool gated, Arena& ar, cudaStream_t stream) {
  const int64_t R = g->rows, N = gated ? 2 * g->n : g->n, esz = g->dtype == SF_F32 ? 4 : 2;
  const int out = g->dtype == SF_F32 ? kOutF32 : kOutBf16;
  if (R == 0) {
    if (ar.dry) return SF_OK;
    if (g->dwt) {   // dwt may be a strided view: its rows one by one where they are not contiguous
      const bool kmaj = g->dw_sk == 1 && g->dw_sn >= g->k;
      const int64_t outer = kmaj ? N : g->k, inner = kmaj ? g->k : N, pitch = kmaj ? g->dw_sn : g->dw_sk;
      cudaError_t err = cudaMemset2DAsync(g->dwt, pitch * esz, 0, inner * esz, outer, stream);
      SF_REQUIRE(err == cudaSuccess, "cudaMemset2DAsync: %s", cudaGetErrorString(err));
    }
    return g->dbias ? zero(g->dbias, N * sizeof(float), stream) : SF_OK;
  }
  Shared s{g, gated, ar, stream};
  const bool few = s.few(), few_dx = few_form(g->dtype, R, s.weight_bytes(), !s.w_k_inner());
  const void* dzp = g->dy;     // dz
  int64_t dz_sr = g->dy_sr;
  if (gated || g->activation != SF_POST_NONE) {
    const int64_t pitch = pad8(N);
    char* buf = ar.take<char>(R * pitch * esz);
    // the sums of each 32 rows (of each kFewRows in the few-row form); one block's are dbias
    const int64_t blocks = few && !g->saved ? (R + kFewRows - 1) / kFewRows : (R + 31) / 32;
    float* part = !g->dbias || blocks == 1 ? nullptr : ar.take<float>(blocks * N);
    float* sums = part ? part : g->dbias;
    const Epi e{gated ? kDGated : kDLinear, g->activation, g->n, g->bias, g->dy, g->dy_sr, buf, out, pitch, g->saved, sums};
    if (!g->saved) {
      SF_TRY(s.forward(e, sums));
    } else if (!ar.dry) {
      auto f = gated ? (out == kOutF32 ? launch_dz<kDGated, kOutF32> : launch_dz<kDGated, kOutBf16>)
                     : (out == kOutF32 ? launch_dz<kDLinear, kOutF32> : launch_dz<kDLinear, kOutBf16>);
      SF_TRY(f(e, R, stream));
    }
    if (part) SF_TRY(colsum(part, SF_F32, blocks, N, N, g->dbias, ar, s.sums, stream));
    dzp = buf;
    dz_sr = pitch;
  } else if (g->dbias) {
    SF_TRY(colsum(g->dy, g->dtype, R, N, g->dy_sr, g->dbias, ar, s.sums, stream));
  }
  Planes dz;
  if (g->dwt || (g->dx && !few_dx)) SF_TRY(s.packer.planes_of(dzp, g->dtype, N, R, dz_sr, dz, ar, stream));
  const Epi to_dx{kLinear, SF_POST_NONE, g->k, nullptr, nullptr, 0, g->dx, out, g->k, nullptr, nullptr};
  if (g->dx && few_dx) {   // dx[r][j] = sum over n of dz[r][n] W[n][j]
    const bool ki = s.w_k_inner();
    if (!ar.dry)
      SF_TRY(few_rows(g->dtype, dzp, dz_sr, R, N, g->wt, nullptr, ki ? g->w_sn : g->w_sk, !ki, to_dx, nullptr, stream));
  } else if (g->dx) {
    Operand wj{{}, !s.w_k_inner()};
    SF_TRY(s.w(wj.m));
    if (g->dwt) {   // dW's operand, packed by the same launch
      Planes ahead;
      SF_TRY(s.x(ahead));
    }
    SF_TRY(s.packer.flush(stream));
    SF_TRY(product_tc(Operand{dz, true}, wj, nullptr, to_dx, ar, s.sums, stream));
  }
  if (g->dwt) {   // dW[n][j] = sum over r of dz[r][n] x[r][j], rows of the product along dwt's strided axis
    Operand xt{{}, false};
    const Operand zt{dz, false};
    SF_TRY(s.x(xt.m));
    SF_TRY(s.packer.flush(stream));
    const bool kmaj = g->dw_sk == 1 && g->dw_sn >= g->k;
    const Epi e{kLinear, SF_POST_NONE, kmaj ? g->k : N, nullptr, nullptr, 0, g->dwt, out, kmaj ? g->dw_sn : g->dw_sk,
                nullptr, nullptr};
    SF_TRY(product_tc(kmaj ? zt : xt, kmaj ? xt : zt, nullptr, e, ar, s.sums, stream));
  }
  return s.sums.flush(stream);
}

int run(const sf_linear_args* g, bool gated, bool back, void* ws, size_t ws_bytes, cudaStream_t stream,
        const char* what) {
  SF_TRY(check(g, gated, back, what));
  Arena size(nullptr, 0, true);
  SF_TRY(back ? backward(g, gated, size, stream) : forward(g, gated, size, stream));
  if (size.ws.used > 0 && (!ws || size.ws.used > ws_bytes)) {
    set_error("%s: workspace of %zu bytes needed, %zu given", what, size.ws.used, ws_bytes);
    return SF_ERR_WORKSPACE;
  }
  SF_REQUIRE(size.ws.used == 0 || (reinterpret_cast<uintptr_t>(ws) & 255) == 0,
             "%s: the workspace must be 256-byte aligned", what);
  Arena ar(ws, ws_bytes, false);
  return back ? backward(g, gated, ar, stream) : forward(g, gated, ar, stream);
}

}  // namespace

int Sums::add(const SumJob& j, cudaStream_t stream) {
  const int64_t blocks = j.kind == kColumns ? (j.n + 31) / 32 : (j.m * (j.pitch / 4) + 255) / 256;
  SF_REQUIRE(blocks <= 0x7fffffff, "sums: %lld x %lld elements", (long long)j.m, (long long)j.n);
  if (jobs.count == kSumJobs || (jobs.count && jobs.job[jobs.count - 1].end + blocks > 0x7fffffff)) SF_TRY(flush(stream));
  const unsigned before = jobs.count ? jobs.job[jobs.count - 1].end : 0u;
  jobs.job[jobs.count] = j;
  jobs.job[jobs.count++].end = before + (unsigned)blocks;
  return SF_OK;
}

int Sums::flush(cudaStream_t stream) {
  if (jobs.count == 0) return SF_OK;
  launch_pdl(k_sums, dim3(jobs.job[jobs.count - 1].end), dim3(256), 0, stream, jobs);
  jobs.count = 0;
  count_launch();
  return check_launch("sums");
}

}  // namespace lg
}  // namespace sf

using namespace sf;

extern "C" {

size_t sf_linear_act_workspace(const sf_linear_args* g, int op) {
  const bool gated = op == SF_OP_GATED_LINEAR || op == SF_OP_GATED_LINEAR_BACKWARD;
  const bool back = op == SF_OP_LINEAR_ACT_BACKWARD || op == SF_OP_GATED_LINEAR_BACKWARD;
  if (op < SF_OP_LINEAR_ACT || op > SF_OP_GATED_LINEAR_BACKWARD || lg::check(g, gated, back, "sf_linear_act_workspace") != SF_OK)
    return 0;
  lg::Arena ar(nullptr, 0, true);
  if ((back ? lg::backward(g, gated, ar, nullptr) : lg::forward(g, gated, ar, nullptr)) != SF_OK) return 0;
  return ar.ws.used;
}

int sf_linear_act(const sf_linear_args* g, void* ws, size_t ws_bytes, sf_stream_t stream) {
  return lg::run(g, false, false, ws, ws_bytes, stream, "sf_linear_act");
}
int sf_linear_act_backward(const sf_linear_args* g, void* ws, size_t ws_bytes, sf_stream_t stream) {
  return lg::run(g, false, true, ws, ws_bytes, stream, "sf_linear_act_backward");
}
int sf_gated_linear(const sf_linear_args* g, void* ws, size_t ws_bytes, sf_stream_t stream) {
  return lg::run(g, true, false, ws, ws_bytes, stream, "sf_gated_linear");
}
int sf_gated_linear_backward(const sf_linear_args* g, void* ws, size_t ws_bytes, sf_stream_t stream) {
  return lg::run(g, true, true, ws, ws_bytes, stream, "sf_gated_linear_backward");
}

}  // extern "C"
