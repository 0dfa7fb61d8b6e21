// Host side of the linear layers' products: the tile, cluster and split of a product, its tensor maps, its launch.
#include "sf_product_tc.cuh"

namespace sf {
namespace lg {
namespace {
using namespace pr;

// Tensor map over the planes of an operand, 128-byte swizzle: box 64 (inner) x box_outer x 1, or (`runs` > 0)
// `runs` runs of 64 inner elements x box_outer, as one box of a view [plane][inner / 64][outer][64].
int make_map(CUtensorMap* map, const Planes& t, uint32_t box_outer, uint32_t runs) {
  auto encode = tensor_map_encoder();
  if (!encode) return SF_ERR_CUDA;
  const cuuint64_t plane = (cuuint64_t)(t.planes > 1 ? t.plane : t.pitch * t.outer) * 2;
  cuuint32_t estr[4] = {1, 1, 1, 1};
  CUresult r;
  if (runs) {
    cuuint64_t dims[4] = {(cuuint64_t)BK, (cuuint64_t)t.outer, (cuuint64_t)t.inner / 64, (cuuint64_t)t.planes};
    cuuint64_t strides[3] = {(cuuint64_t)t.pitch * 2, 128, plane};
    cuuint32_t box[4] = {(cuuint32_t)BK, box_outer, runs, 1};
    r = encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<bf16*>(t.p), dims, strides, box, estr,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  } else {
    cuuint64_t dims[3] = {(cuuint64_t)t.inner, (cuuint64_t)t.outer, (cuuint64_t)t.planes};
    cuuint64_t strides[2] = {(cuuint64_t)t.pitch * 2, plane};
    cuuint32_t box[3] = {(cuuint32_t)BK, box_outer, 1};
    r = encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<bf16*>(t.p), dims, strides, box, estr,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  }
  if (r != CUDA_SUCCESS) {
    set_error("cuTensorMapEncodeTiled failed (%d) for an operand [%d][%lld][%lld] pitch %lld", (int)r, t.planes,
              (long long)t.outer, (long long)t.inner, (long long)t.pitch);
    return SF_ERR_CUDA;
  }
  return SF_OK;
}

// Tensor map of an epilogue's buffer over a [z][rows][cols] matrix: 32 rows of 64 bytes.
int make_out_map(CUtensorMap* map, const void* base, bool f32, int64_t cols, int64_t rows, int64_t sr, int64_t zs, int64_t z) {
  auto encode = tensor_map_encoder();
  if (!encode) return SF_ERR_CUDA;
  const cuuint64_t esz = f32 ? 4 : 2;
  cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)z};
  cuuint64_t strides[2] = {(cuuint64_t)sr * esz, (cuuint64_t)zs * esz};
  cuuint32_t box[3] = {(cuuint32_t)(64 / esz), 32, 1}, estr[3] = {1, 1, 1};
  CUresult r = encode(map, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                      const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                      CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("cuTensorMapEncodeTiled failed (%d) for an epilogue matrix [%lld][%lld] pitch %lld", (int)r, (long long)rows,
              (long long)cols, (long long)sr);
    return SF_ERR_CUDA;
  }
  return SF_OK;
}

// ---- tile, cluster and split ------------------------------------------------------------------------
struct Plan {
  int ctas, part, splits;
};

// Whether two threads load and two issue a tile's stages (issue_half): one tile per CTA, and enough stages, for each of
// them in the last split too.  Each accumulator sums half of K, so it is as good as one of half the depth and K may be two
// segments long.  Tiles above 128 columns only from 16 stages on: their MMAs hide more of what issuing costs (3840 x 768 x
// 768 dx, 12 stages of 192 columns: 9.2 us against 8.1 in clusters; 1000 x 2048 -> 1024 forward, 32: 12.1 against 15.8).
bool two_issue(int bn, int ctas, int64_t items, int sms, int nkb, int pairs, int kb_split, int seg_kb) {
  return ctas == 1 && items <= sms && kb_split <= (seg_kb < nkb ? 2 : 1) * seg_kb &&
         kb_split * pairs >= (bn <= 128 ? 8 : 16) && (nkb - 1) % kb_split * pairs + pairs >= 2;
}

// Estimated cycles of a product with a given tile, to choose by.  Per 64-deep step the tensor cores take 4 MMAs of at
// least 128 cycles (171 for 256 columns; 150 with the latencies of a short loop, 75 from two threads) and the loads 60
// bytes a cycle and SM; the epilogue of a tile runs under the next tile's products, except the last one's; a split adds
// its partials' round trip and a launch.  Against the widest tile that gives every SM one (graph replay, bf16):
// 3840 x 768 x 768 dx 9.0 -> 8.0 us, dW 13.5 -> 12.2 us; 65536 x 128 x 1024 dW 42 -> 36 us.
Plan plan_of(int64_t m, int64_t n, int nkb, int pairs, int seg_kb, bool gated, bool b_k_major, bool plain, int sms) {
  const int halves = gated ? 2 : 1, most = MAX_BN / halves, least = b_k_major ? 32 / halves : 64;
  // splits of a plain sum: at least four steps each
  const int64_t kbs = (int64_t)nkb * pairs, most_splits = !plain || kbs < 8 ? 1 : kbs / 4 < nkb ? kbs / 4 : nkb;
  auto splits_of = [&](int64_t tiles, int64_t slots) {
    return most_splits < 2 || tiles * 2 > slots ? 1 : slots / tiles < most_splits ? slots / tiles : most_splits;
  };
  if (m <= BM && b_k_major) {
    // one row tile reads the whole of B once: as many columns per tile as give every SM one tile of the same width
    // (24 x 4096 -> 2 x 10000: 53 us with 157 tiles of 64, two for some SMs; 139 of 72 take one turn, 38 us)
    const int step = seg_kb < nkb ? 16 : 16 / halves;   // segments are added 16 columns at a time
    const int64_t turns = (n + (int64_t)most * sms - 1) / ((int64_t)most * sms);
    const int64_t even = ((n + turns * sms - 1) / (turns * sms) + step - 1) / step * step;
    const int part = (int)(even < least ? least : even > most ? most : even);
    const int64_t tiles = (n + part - 1) / part;
    return Plan{1, part, (int)splits_of(tiles, sms)};
  }
  Plan best{1, least, 1};
  double best_cost = 1e30;
  for (int ctas = 1; ctas <= 2; ++ctas) {
    if (ctas == 2 && m <= BM) break;
    for (int bn = MAX_BN; bn >= 32; bn -= 32) {
      const int part = bn / halves, rows = bn / ctas;      // B rows that a CTA holds
      // M/N-major runs are 64 wide, in each part and each CTA; the staged epilogue takes parts of 32
      if (b_k_major ? part % 32 && part > 16 : (ctas == 2 && !gated ? rows : part) % 64) continue;
      if (ctas == 2 && bn < 128) break;
      if (part < least || (part > least && part - least >= n && bn > (ctas == 2 ? 128 : 32))) continue;   // less would do
      const int64_t tiles = (m + BM * ctas - 1) / (BM * ctas) * ((n + part - 1) / part), slots = sms / ctas;
      const double load = (A_SLOT + rows * BK * 2) / 60.0, epi = 1000.0 + 10.0 * bn;
      for (int pass = 0; pass < 2; ++pass) {
        const int64_t s = pass ? splits_of(tiles, slots) : 1;
        if (pass && s == 1) break;
        const int64_t blocks = (nkb + s - 1) / s;
        const bool two = two_issue(bn, ctas, tiles * s, sms, nkb, pairs, (int)blocks, seg_kb);
        const int64_t segs = two ? 1 : (blocks + seg_kb - 1) / seg_kb;
        const double least_mma = two ? 75.0 : 150.0;
        const double mma = 4.0 * (171.0 * bn / 256 > least_mma ? 171.0 * bn / 256 : least_mma), step = mma > load ? mma : load;
        // segments of a wide tile have one accumulator and wait for each other's epilogue
        const double main = blocks * pairs * step + (segs > 1 && bn > 128 ? segs * epi : 0.0);
        const double turns = (double)((tiles * s + slots - 1) / slots);
        double cost = turns * (main > epi ? main : epi) + epi + 3000.0;
        if (s > 1) cost += 2000.0 + 8.0 * s * m * n / 6000.0;
        if (cost < best_cost) {
          best_cost = cost;
          best = Plan{ctas, part, (int)s};
        }
      }
    }
  }
  return best;
}

}  // namespace

int product_tc(const Operand& a, const Operand& b, const Operand* b2, const Epi& e, Arena& ar, Sums& sums,
               cudaStream_t stream) {
  const bool gated = e.kind == kGated || e.kind == kDGated;
  Params p = {};
  p.m = a.rows();
  p.n = e.n;
  const int sms = num_sms();
  p.pairs = a.m.planes == 3 ? 6 : 1;
  p.nkb = (int)((a.depth() + BK - 1) / BK);
  // Segments of 512 for fp32 operands, and for the pre-activations that dbias comes from: the accumulator truncates
  // (1.1e-9 of a value per column), and a sum over the rows does not average that away (K = 2048, gated silu, dbias
  // against fp64: 2.2e-6 in segments of 2048, 5.1e-7 in these; 2000 rows of 4096 columns 33 us either way).
  // (dbias may be asked for without a bias: colpart; saved ones only serve it where the layer has one)
  // Of 65536 for the rest, as a weight gradient's rows may be: a sum of one sign loses 3.8e-9 per column (dW over 3 million
  // rows was short by 1.2 %), so 2.5e-4 at most here, a fourteenth of a bf16 result's rounding.
  p.seg_kb = p.pairs > 1 || e.colpart || (e.bias && e.saved) ? 8 : p.nkb < 1024 ? p.nkb : 1024;
  // a plain sum's K may be split over CTAs
  const bool plain = e.kind == kLinear && e.act == SF_POST_NONE && !e.bias && !e.aux && !e.saved;
  const Plan plan = plan_of(p.m, p.n, p.nkb, p.pairs, p.seg_kb, gated, b.k_major, plain, sms);
  const int ctas = plan.ctas;
  p.mt = (int)((p.m + BM * ctas - 1) / (BM * ctas));
  p.part = plan.part;
  p.bn = plan.part * (gated ? 2 : 1);
  p.nt = (int)((p.n + p.part - 1) / p.part);
  p.splits = plan.splits;
  const int64_t tiles = (int64_t)p.mt * p.nt;
  p.kb_split = (p.nkb + p.splits - 1) / p.splits;
  p.splits = (p.nkb + p.kb_split - 1) / p.kb_split;
  const bool two = two_issue(p.bn, ctas, tiles * p.splits, sms, p.nkb, p.pairs, p.kb_split, p.seg_kb);
  if (two && p.seg_kb < p.kb_split) p.seg_kb = p.kb_split;
  const bool segments = p.kb_split > p.seg_kb;
  p.two = two;
  p.accs = two || (segments && p.bn > 128) ? 1 : 2;
  p.acc_stride = segments ? 128 : MAX_BN;
  SF_REQUIRE(tiles * p.splits < (int64_t(1) << 30), "linear product: too many tiles");
  p.items = (int)(tiles * p.splits);
  const int64_t pitch = (p.n + 3) / 4 * 4;
  float* part_buf = p.splits > 1 ? ar.take<float>((int64_t)p.splits * p.m * pitch) : nullptr;
  if (ar.dry) return SF_OK;

  p.a_mn = !a.k_major;
  p.b_mn = !b.k_major;
  const int b_rows = p.bn / ctas;                 // of B that a CTA holds
  p.b_slot = (b_rows * BK * 2 + 1023) / 1024 * 1024;
  p.a_boxes = p.m > 64 ? 2 : 1;
  p.a_one = p.a_mn && p.a_boxes == 2 && p.m % 64 == 0;
  p.b_one = p.b_mn && b.rows() % 64 == 0;
  // few rows: load only those (the MMA's other rows hold anything and are never stored)
  const uint32_t a_rows = p.m < BM ? (uint32_t)((p.m + 7) / 8 * 8) : BM;
  // (their slot ends behind the rows that are loaded; the MMA reads on into the stage's B, inside the buffers)
  p.a_slot = p.a_mn || p.m >= BM ? A_SLOT : ((int)a_rows * BK * 2 + 1023) / 1024 * 1024;
  p.tx = (p.a_mn ? p.a_boxes * 8192 : (int)a_rows * BK * 2) + b_rows * BK * 2;
  p.act = e.act;
  p.bias = e.bias;
  p.aux = e.aux;
  p.aux_sr = e.aux_sr;
  p.out = p.splits > 1 ? part_buf : e.out;
  p.out_sr = p.splits > 1 ? pitch : e.out_sr;
  p.saved = e.saved;
  p.colpart = e.colpart;
  auto aligned = [](const void* q, int64_t sr, int64_t esz, int64_t off) {
    return ((reinterpret_cast<uintptr_t>(q) | (uintptr_t)(sr * esz) | (uintptr_t)(off * esz)) & 15) == 0;
  };
  const int64_t esz = e.out_kind == kOutF32 ? 4 : 2, other = gated ? e.n : 0;
  p.vec_out = p.splits > 1 ? 1 : aligned(e.out, e.out_sr, esz, e.kind == kDGated ? other : 0);
  p.vec_aux = aligned(e.aux, e.aux_sr, esz, 0);
  p.vec_saved = aligned(e.saved, gated ? 2 * e.n : e.n, 4, other);
  p.vec_bias = e.n % 4 == 0 && aligned(e.bias, 4, 4, other);   // read in fours
  p.status = device_status_ptr();
  if (!p.status) return SF_ERR_CUDA;

  Maps tm;
  const int b_load = ctas == 2 ? b_rows : p.part;   // rows of B per load
  SF_TRY(make_map(&tm.a, a.m, p.a_mn ? BK : a_rows, p.a_one ? 2 : 0));
  SF_TRY(make_map(&tm.b, b.m, p.b_mn ? BK : b_load, p.b_one ? b_load / 64 : 0));
  if (gated) SF_TRY(make_map(&tm.b2, b2->m, p.b_mn ? BK : b_load, p.b_one ? b_load / 64 : 0));

  // the staged epilogue's matrices, where they have 16-byte rows
  const bool grad = e.kind == kDLinear || e.kind == kDGated, split = p.splits > 1;
  const bool f32 = split || e.out_kind == kOutF32;
  // Parts that end inside a buffer's columns leave it a row at a time: a store would run on into the next tile (100 x
  // 4096 -> 2 x 10001 with gelu: 45 us straight from the accumulator, 36 so).  Below 32 rows the smaller block starts
  // sooner (9 x 768 -> 2 x 768: 5.5 us against 6.5).
  const bool whole = p.part % (f32 ? 16 : 32) == 0, staged = p.m >= 32 && (whole || !split);
  p.slots = 0;
  if (staged) {
    if (!whole) p.vec_out = p.vec_saved = 0;
    const bool aux = e.aux && !split, saved = !grad && e.saved;
    // a deep K hides the epilogue: one buffer less, one ring stage more
    p.pool = e.kind != kDGated && p.kb_split * p.pairs >= 16 ? 1 : 2;
    p.slots = p.pool + (aux ? 1 : 0) + (saved ? 1 : 0);
    if (p.vec_out) {
      SF_TRY(make_out_map(&tm.out, p.out, f32, p.n, p.m, p.out_sr, p.m * p.out_sr, p.splits));
      if (e.kind == kDGated)
        SF_TRY(make_out_map(&tm.out2, static_cast<char*>(p.out) + p.n * esz, f32, p.n, p.m, p.out_sr, p.m * p.out_sr, 1));
    }
    if (saved && p.vec_saved) {
      const int64_t wide = gated ? 2 * p.n : p.n;
      SF_TRY(make_out_map(&tm.sav, p.saved, true, p.n, p.m, wide, p.m * wide, 1));
      if (gated) SF_TRY(make_out_map(&tm.sav2, p.saved + p.n, true, p.n, p.m, wide, p.m * wide, 1));
    }
    if (aux && p.vec_aux) SF_TRY(make_out_map(&tm.aux, e.aux, f32, p.n, p.m, e.aux_sr, p.m * e.aux_sr, 1));
  }
  p.stages = (SMEM_MAX - SMEM_REST - epi_warps(true) * p.slots * SLOT - (A_SLOT - p.a_slot)) / (p.a_slot + p.b_slot);
  if (p.stages > MAX_STAGES) p.stages = MAX_STAGES;
  if (p.two) p.stages &= ~1;
  SF_REQUIRE(p.stages > (p.two ? 1 : 0), "linear product: no room for a ring");

  if (p.splits > 1) {
    SF_TRY(launch_linear(kOutF32, ctas, tm, p, stream));
    return sums.add(SumJob{part_buf, e.out, p.m, p.n, pitch, e.out_sr, p.splits,
                           e.out_kind == kOutF32 ? kSplitF32 : kSplitBf16, 0}, stream);
  }
  switch (e.kind) {
    case kLinear: return launch_linear(e.out_kind, ctas, tm, p, stream);
    case kGated: return launch_gated(e.out_kind, ctas, tm, p, stream);
    case kDLinear: return launch_dlinear(e.out_kind, ctas, tm, p, stream);
    default: return launch_dgated(e.out_kind, ctas, tm, p, stream);
  }
}

}  // namespace lg
}  // namespace sf
