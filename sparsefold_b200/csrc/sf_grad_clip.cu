// Global gradient norm and clipping over many tensors.
//
// The tensors' addresses and sizes travel as kernel parameters (a table of up to kTable tensors per launch, a
// shorter one for few: a call takes the host 6 us with it and 10 us with the whole 28 KB), so a call copies nothing
// to the device and can be captured.  The elements of all tensors of a table are cut into granules (kGranule elements of
// one tensor); every block of a fixed grid takes an equal run of them and writes one partial, and the partials are
// summed in order: the result depends on the sizes alone.  Bound by the memory: each gradient is read once for
// the norm and, where it has to be scaled, read and written once more (256 M bf16 gradients into other buffers at odd
// offsets: 278 us for 1.5 GB, 5.5 TB/s).
#include <algorithm>

#include "sf_common.cuh"
#include "sf_tc.cuh"

namespace sf {
namespace {

constexpr int kShort = 100, kTable = 1000;   // 28 bytes each: below the 32764 bytes of kernel parameters
constexpr int64_t kGranule = 4096;       // elements
constexpr int64_t kMostGranules = 1 << 28;   // of a table: a block's run stays below 2^31 elements
constexpr int kBlocks = 148 * 6, kThreads = 256, kClipBlocks = 148 * 8;

template <int N>
struct Table {
  const void* p[N];
  void* out[N];
  int64_t n[N];
  int32_t end[N];                        // granules up to and with this tensor's
  uint32_t f32[(N + 31) / 32];           // bit i: tensor i holds fp32
  int32_t count;
};

template <int N>
__device__ __forceinline__ int tensor_of(const Table<N>& t, int granule) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (granule < t.end[mid]) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}
// First granule of this block's run (and of the next one's, for blockIdx.x + 1).
__device__ __forceinline__ int run_start(int granules, int block) {
  return (int)((int64_t)granules * block / (int)gridDim.x);
}

// ---- one 16-byte vector ------------------------------------------------------------------------------
template <typename T>
struct Vec { static constexpr int N = 16 / sizeof(T); };
__device__ __forceinline__ void unpack(const uint4& q, float (&v)[4]) {
  v[0] = __uint_as_float(q.x), v[1] = __uint_as_float(q.y), v[2] = __uint_as_float(q.z), v[3] = __uint_as_float(q.w);
}
__device__ __forceinline__ void unpack(const uint4& q, float (&v)[8]) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
// v * scale, of the packed type; fp32 products, one rounding.
__device__ __forceinline__ uint4 scaled(const uint4& q, float scale, float) {
  float v[4];
  unpack(q, v);
  return make_uint4(__float_as_uint(v[0] * scale), __float_as_uint(v[1] * scale), __float_as_uint(v[2] * scale),
                    __float_as_uint(v[3] * scale));
}
__device__ __forceinline__ uint4 scaled(const uint4& q, float scale, bf16) {
  float v[8];
  unpack(q, v);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i] * scale, v[2 * i + 1] * scale);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ void add_one(float v, int type, double& sum, uint32_t& most) {
  if (type == 2) sum += (double)v * (double)v;
  else most = max(most, __float_as_uint(fabsf(v)));   // a NaN's bits are above infinity's
}
// A vector's squares are added in fp32 (at most 8 roundings) and go to fp64 as one value, which costs a
// conversion per vector instead of one per element (256 M bf16: 98 us, 5.2 TB/s; 130 us with fp64 for every
// element, the conversions being the bound).  Where that sum could have overflowed, or lost small squares, the
// squares are formed in fp64.
template <int N>
__device__ __forceinline__ void add_vec(const float (&v)[N], int type, double& sum, uint32_t& most) {
  if (type == 2) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) s = fmaf(v[i], v[i], s);
    if (s > 1e-20f && s < 1e38f) {
      sum += (double)s;
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) sum += (double)v[i] * (double)v[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) most = max(most, __float_as_uint(fabsf(v[i])));
  }
}

template <typename T>
__device__ __forceinline__ void run_norm(const T* p, int n, int type, double& sum, uint32_t& most) {
  constexpr int N = Vec<T>::N, U = 4;      // vectors in flight
  const int off = (int)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / (int)sizeof(T);
  const int head = off < n ? off : n, nv = (n - head) / N, tail = head + nv * N;
  if ((int)threadIdx.x < head) add_one(ld(p + threadIdx.x), type, sum, most);
  const uint4* q = reinterpret_cast<const uint4*>(p + head);
  int i = threadIdx.x;
  for (; i + (U - 1) * kThreads < nv; i += U * kThreads) {
    uint4 w[U];
#pragma unroll
    for (int k = 0; k < U; ++k) w[k] = __ldg(q + i + k * kThreads);
#pragma unroll
    for (int k = 0; k < U; ++k) {
      float v[N];
      unpack(w[k], v);
      add_vec(v, type, sum, most);
    }
  }
  for (; i < nv; i += kThreads) {
    float v[N];
    unpack(__ldg(q + i), v);
    add_vec(v, type, sum, most);
  }
  if (tail + (int)threadIdx.x < n) add_one(ld(p + tail + threadIdx.x), type, sum, most);
}

// o[j] = p[j] * scale, from the end to the start.  Vectors follow the output's alignment; where the input sits at
// another offset from 16 bytes, a vector is put together from the two aligned ones around it, both inside the run
// (the first and the last are left to single elements).  One vector per thread and turn, as many threads as an SM
// holds: unrolled, the variants of this took 148 registers together.
template <typename T>
__device__ __forceinline__ void run_scale(const T* p, T* o, int n, float scale) {
  constexpr int N = Vec<T>::N;
  const int delta = (int)((reinterpret_cast<uintptr_t>(p) - reinterpret_cast<uintptr_t>(o)) & 15);
  int head = (int)((16 - (reinterpret_cast<uintptr_t>(o) & 15)) & 15) / (int)sizeof(T);
  if (delta) head += N;                       // so that the aligned vector below the first one is inside
  if (head > n) head = n;
  int nv = (n - head) / N;
  if (delta && nv > 0) --nv;                  // and the one above the last
  const int tail = head + nv * N;
#pragma unroll 1
  for (int j = threadIdx.x; j < head + n - tail; j += kThreads) {
    const int at = j < head ? j : tail + j - head;
    st(o + at, ld(p + at) * scale);
  }
  uint4* ov = reinterpret_cast<uint4*>(o + head);
  const uint4* q = reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(p + head) - delta);
  const int words = delta >> 2, bits = (delta & 3) * 8;
#pragma unroll 1
  for (int i = nv - 1 - (int)threadIdx.x; i >= 0; i -= kThreads) {
    uint4 a = q[i];
    if (delta) {
      const uint4 b = q[i + 1];
      uint32_t w4 = b.x;
      if (words == 1) a = make_uint4(a.y, a.z, a.w, b.x), w4 = b.y;
      if (words == 2) a = make_uint4(a.z, a.w, b.x, b.y), w4 = b.z;
      if (words == 3) a = make_uint4(a.w, b.x, b.y, b.z), w4 = b.w;
      a = make_uint4(__funnelshift_r(a.x, a.y, bits), __funnelshift_r(a.y, a.z, bits), __funnelshift_r(a.z, a.w, bits),
                     __funnelshift_r(a.w, w4, bits));
    }
    ov[i] = scaled(a, scale, T{});
  }
}

// Partial of this block's run of granules: a sum of squares, or the bits of a maximum.
template <int N>
__global__ void __launch_bounds__(kThreads, 6) k_grad_norm(const __grid_constant__ Table<N> t, int type,
                                                        double* __restrict__ part) {
  __shared__ double s_sum[kThreads / 32];
  __shared__ uint32_t s_most[kThreads / 32];
  double sum = 0.0;
  uint32_t most = 0;
  const int granules = t.end[t.count - 1], stop = run_start(granules, blockIdx.x + 1);
  int g = run_start(granules, blockIdx.x), i = tensor_of(t, g);
  tc::griddep_wait();
  tc::griddep_launch();
  for (; g < stop; ++i) {
    const int begin = i ? t.end[i - 1] : 0, to = min(stop, t.end[i]);
    const int64_t at = (g - begin) * kGranule;
    const int n = (int)(min((to - begin) * kGranule, t.n[i]) - at);
    if (t.f32[i >> 5] >> (i & 31) & 1) run_norm(static_cast<const float*>(t.p[i]) + at, n, type, sum, most);
    else run_norm(static_cast<const bf16*>(t.p[i]) + at, n, type, sum, most);
    g = to;
  }
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
  }
  if ((threadIdx.x & 31) == 0) {
    s_sum[threadIdx.x / 32] = sum;
    s_most[threadIdx.x / 32] = most;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kThreads / 32; ++w) {
      sum += s_sum[w];
      most = max(most, s_most[w]);
    }
    part[blockIdx.x] = type == 2 ? sum : (double)__uint_as_float(most);
  }
}

// The norm from the partials before its rounding, for every thread of a block: each block adds them in the same order.
__device__ __forceinline__ double norm_of(const double* __restrict__ part, int parts, int type) {
  __shared__ double s_sum[kThreads / 32];
  __shared__ uint32_t s_most[kThreads / 32];
  __shared__ double s_norm;
  double sum = 0.0;
  uint32_t most = 0;
  for (int i = threadIdx.x; i < parts; i += kThreads) {
    const double v = part[i];
    sum += v;
    most = max(most, __float_as_uint((float)v));
  }
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
  }
  if ((threadIdx.x & 31) == 0) {
    s_sum[threadIdx.x / 32] = sum;
    s_most[threadIdx.x / 32] = most;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kThreads / 32; ++w) {
      sum += s_sum[w];
      most = max(most, s_most[w]);
    }
    s_norm = type == 2 ? sqrt(sum) : (double)__uint_as_float(most);
  }
  __syncthreads();
  return s_norm;
}

__global__ void __launch_bounds__(kThreads) k_norm_final(const double* __restrict__ part, int parts, int type,
                                                         float* __restrict__ norm) {
  tc::griddep_wait();
  tc::griddep_launch();
  const double v = norm_of(part, parts, type);
  if (threadIdx.x == 0) *norm = (float)v;
}

// Every block forms the norm from the partials itself (a few hundred values from L2), which saves a launch between
// the two passes.  The scale comes from the norm in fp64 and is rounded once: its error is in every gradient (from the
// norm rounded to fp32 and in fp32 it was twice as large, 5.9e-8 of the gradients against 2.9e-8).  A block goes through its run from the end: what the first pass read last may still be in L2.
template <int N>
__global__ void __launch_bounds__(kThreads, 8) k_clip(const __grid_constant__ Table<N> t, const double* __restrict__ part,
                                                   int parts, int type, float* __restrict__ norm, float max_norm) {
  tc::griddep_wait();
  tc::griddep_launch();
  const double nv = norm_of(part, parts, type), q = (double)max_norm / (nv + 1e-6);
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)nv;
  const float scale = q < 1.0 || q != q ? (float)q : 1.0f;
  const int granules = t.end[t.count - 1], first = run_start(granules, blockIdx.x);
  int g = run_start(granules, blockIdx.x + 1), i = tensor_of(t, g - 1);
  for (; g > first; --i) {
    const int begin = i ? t.end[i - 1] : 0, from = max(first, begin);
    const int64_t at = (from - begin) * kGranule;
    const int n = (int)(min((g - begin) * kGranule, t.n[i]) - at);
    g = from;
    if (scale == 1.0f && t.p[i] == t.out[i]) continue;
    if (t.f32[i >> 5] >> (i & 31) & 1) run_scale(static_cast<const float*>(t.p[i]) + at, static_cast<float*>(t.out[i]) + at, n, scale);
    else run_scale(static_cast<const bf16*>(t.p[i]) + at, static_cast<bf16*>(t.out[i]) + at, n, scale);
  }
}

// The gradients of a call.
struct Grads {
  const void* const* ptrs;
  void* const* outs;
  const int64_t* numels;
  const int32_t* dtypes;
  int64_t count;
};

// Fills a table from tensor `i` on; returns the next tensor that is not in it.
template <int N>
int64_t fill(Table<N>& t, const Grads& g, int64_t i) {
  t.count = 0;
  for (uint32_t& w : t.f32) w = 0;
  int64_t granules = 0;
  for (; i < g.count && t.count < N; ++i) {
    if (g.numels[i] == 0) continue;
    const int64_t more = (g.numels[i] + kGranule - 1) / kGranule;
    if (t.count && granules + more > kMostGranules) break;
    granules += more;
    const int c = t.count++;
    t.p[c] = g.ptrs[i];
    t.out[c] = g.outs ? g.outs[i] : nullptr;
    t.n[c] = g.numels[i];
    t.end[c] = (int32_t)granules;
    if (g.dtypes[i] == SF_F32) t.f32[c >> 5] |= 1u << (c & 31);
  }
  return i;
}

template <typename... KArgs, typename... Args>
void start(void (*kernel)(KArgs...), int grid, cudaStream_t stream, Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 1 : 0;
  void* ptrs[] = {&args...};             // by address: the table is copied once, by the launch
  cudaLaunchKernelExC(&cfg, reinterpret_cast<const void*>(kernel), ptrs);
  count_launch();
}

// The two passes with tables of N; `need` bounds the partials.
template <int N>
int passes(const Grads& g, int norm_type, float max_norm, float* norm, double* part, size_t need, cudaStream_t stream,
           const char* what) {
  int parts = 0;
  Table<N> t;
  int64_t i = 0;
  do {
    i = fill(t, g, i);
    if (!t.count) break;
    SF_REQUIRE(parts + kBlocks <= (int64_t)(need / sizeof(double)), "%s: too many elements for one call", what);
    const int grid = std::min(t.end[t.count - 1], kBlocks);
    double* to = part + parts;
    start(k_grad_norm<N>, grid, stream, t, norm_type, to);
    SF_TRY(check_launch(what));
    parts += grid;
  } while (i < g.count);
  const double* from = part;
  if (!g.outs || parts == 0) {
    start(k_norm_final, 1, stream, from, parts, norm_type, norm);
    return check_launch(what);
  }
  const bool one = g.count <= N;         // the table still holds every tensor
  for (i = 0; i < g.count;) {
    i = one ? g.count : fill(t, g, i);
    if (!t.count) break;
    start(k_clip<N>, std::min(t.end[t.count - 1], kClipBlocks), stream, t, from, parts, norm_type, norm, max_norm);
    SF_TRY(check_launch(what));
    norm = nullptr;                      // written once
  }
  return SF_OK;
}

int tables_of(int64_t count) { return (int)((count + kTable - 1) / kTable); }

int grad_norm(const void* const* ptrs, void* const* outs, const int64_t* numels, const int32_t* dtypes, int64_t count,
              int norm_type, float max_norm, float* norm, void* ws, size_t ws_bytes, cudaStream_t stream,
              const char* what) {
  SF_REQUIRE(count >= 0 && count < (int64_t(1) << 24), "%s: bad count %lld", what, (long long)count);
  SF_REQUIRE(norm, "%s: norm is null", what);
  SF_REQUIRE(norm_type == 2 || norm_type == 0, "%s: norm_type %d (2, or 0 for the largest magnitude)", what, norm_type);
  SF_REQUIRE(count == 0 || (ptrs && numels && dtypes), "%s: null table", what);
  for (int64_t i = 0; i < count; ++i) {
    SF_REQUIRE(numels[i] >= 0 && numels[i] < kMostGranules * kGranule, "%s: tensor %lld has %lld elements", what,
               (long long)i, (long long)numels[i]);
    SF_REQUIRE(dtypes[i] == SF_F32 || dtypes[i] == SF_BF16, "%s: tensor %lld has dtype %d", what, (long long)i,
               (int)dtypes[i]);
    SF_REQUIRE(numels[i] == 0 || (ptrs[i] && (!outs || outs[i])), "%s: tensor %lld is null", what, (long long)i);
  }
  const size_t need = sf_grad_norm_workspace(count);
  SF_REQUIRE((reinterpret_cast<uintptr_t>(ws) & 255) == 0, "%s: workspace not 256-byte aligned", what);
  if (!ws || ws_bytes < need) {
    set_error("%s: workspace of %zu bytes needed, %zu given", what, need, ws_bytes);
    return SF_ERR_WORKSPACE;
  }
  const Grads g{ptrs, outs, numels, dtypes, count};
  double* part = static_cast<double*>(ws);
  return count <= kShort ? passes<kShort>(g, norm_type, max_norm, norm, part, need, stream, what)
                         : passes<kTable>(g, norm_type, max_norm, norm, part, need, stream, what);
}

}  // namespace
}  // namespace sf

using namespace sf;

extern "C" {

// One partial per block and table; a few tables more than the count alone needs, for sizes whose
// pieces fill a table early.
size_t sf_grad_norm_workspace(int64_t count) {
  return count < 0 ? 0 : (size_t)(tables_of(count) + 4) * kBlocks * sizeof(double);
}

int sf_grad_norm(const void* const* ptrs, const int64_t* numels, const int32_t* dtypes, int64_t count, int norm_type,
                 float* norm, void* ws, size_t ws_bytes, sf_stream_t stream) {
  return grad_norm(ptrs, nullptr, numels, dtypes, count, norm_type, 0.f, norm, ws, ws_bytes, stream, "sf_grad_norm");
}

int sf_clip_grad_norm(const void* const* ptrs, void* const* outs, const int64_t* numels, const int32_t* dtypes,
                      int64_t count, int norm_type, float max_norm, float* norm, void* ws, size_t ws_bytes,
                      sf_stream_t stream) {
  SF_REQUIRE(count == 0 || outs, "sf_clip_grad_norm: outs is null");
  SF_REQUIRE(max_norm >= 0.f, "sf_clip_grad_norm: max_norm %g", (double)max_norm);
  void* none = nullptr;
  return grad_norm(ptrs, outs ? outs : &none, numels, dtypes, count, norm_type, max_norm, norm, ws, ws_bytes, stream,
                   "sf_clip_grad_norm");
}

}  // extern "C"
