// The linear layers' products on microscaled operands (include/stride_mx.h): e2m1 weights by e4m3
// activations, v_mfma_scale_f32_16x16x128_f8f6f4, fp32 sums.
//
// Every kernel evaluates the same expression: chunks of 128 columns chain in ascending order within
// each split of K, and the splits' sums are added in ascending order, so a row has the same bits
// whatever the batch and the kernel.
#include <hip/hip_runtime.h>

#include <climits>
#include <cstddef>

#include "mx_common.hpp"
#include "tc_epilogue.hpp"

namespace stride_tc {
namespace {

constexpr int kSplits = 4;

// Up to three matrices over the same x, their row tiles end to end (q, k, v), or gate and up.
struct MxGeometry {
  const uint8_t *xc, *xs;
  const uint8_t *wc[3], *ws[3];
  int32_t tiles[3];
  int32_t groups;  // of 512 columns
  int32_t per;     // groups of a split
  int32_t rows, lane_groups;
};

// Row tile rt of the matrices end to end: which, and its place there.
__device__ __forceinline__ int mx_matrix(const MxGeometry& g, int& rt) {
  if (rt < g.tiles[0]) return 0;
  rt -= g.tiles[0];
  if (rt < g.tiles[1]) return 1;
  rt -= g.tiles[1];
  return 2;
}

// Epilogues take finished 16 x 16 tiles in the instruction's layout: lane l has batch row l % 16,
// output rows 4 * (l / 16) + i. UNIT row tiles of MATS matrices belong together.
struct EpiY {
  static constexpr int kMats = 1, kUnit = 1;
  struct Out {
    uint16_t* y;
    int32_t row_tiles;
  };
  __device__ __forceinline__ static void apply(const Out& o, const MxGeometry& g, int rt, int lt, const f32x4 (&y)[1][1], int lane) {
    if (lt * 16 + (lane & 15) >= g.rows) return;
    const f32x4 v = y[0][0];
    *reinterpret_cast<u32x2*>(o.y + (static_cast<int64_t>(lt) * o.row_tiles + rt) * kTileElems + (lane & 15) * 16 + (lane >> 4) * 4) =
        u32x2{bf16_rne(v[0]) | bf16_rne(v[1]) << 16, bf16_rne(v[2]) | bf16_rne(v[3]) << 16};
  }
};

struct EpiRope {
  static constexpr int kMats = 1, kUnit = 1;
  using Out = EpiQkv::Out;
  __device__ __forceinline__ static void apply(const Out& o, const MxGeometry& g, int rt, int lt, const f32x4 (&y)[1][1], int lane) {
    Geometry rows{};
    rows.rows = g.rows;
    const int which = mx_matrix(g, rt);
    EpiQkv::apply(o, rows, which, rt, lt, y[0], lane);
  }
};

// z's block: two row tiles, whose 32 values of a batch row four lanes hold. Where z's columns end
// inside a group of 512, what fills it up is written as zeros.
struct EpiZ {
  static constexpr int kMats = 2, kUnit = 2;
  struct Out {
    StrideMxTiles z;
  };
  __device__ __forceinline__ static void store(const Out& o, const MxGeometry& g, int block, int lt, u32x2 w, int byte, int lane) {
    const int row = lane & 15, quarter = lane >> 4, kc = block >> 2, blk = block & 3;
    if (lt * 16 + row >= g.rows) return;
    const int groups = mx_groups(o.z.cols);
    uint8_t* c = o.z.codes + (static_cast<int64_t>(lt) * groups * 4 + kc) * kCode8Bytes + (blk * 32 + row) * 16 + quarter * 4;
    *reinterpret_cast<uint32_t*>(c) = w[0];
    *reinterpret_cast<uint32_t*>(c + 256) = w[1];
    if (quarter == 0)
      o.z.scales[(static_cast<int64_t>(lt) * groups + (kc >> 2)) * kScaleBytes + (blk * 16 + row) * 4 + (kc & 3)] = static_cast<uint8_t>(byte);
  }
  __device__ __forceinline__ static void apply(const Out& o, const MxGeometry& g, int rt, int lt, const f32x4 (&y)[2][2], int lane) {
    float v[2][4];
    uint32_t most = 0;
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[r][i] = rt + r < g.tiles[0] ? det_silu(y[0][r][i]) * y[1][r][i] : 0.0f;
        most = max(most, mx_abs_bits(v[r][i]));
      }
    most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), 16)));
    most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), 32)));
    const int byte = mx_scale_byte<8>(most);
    const float inverse = mx_inverse(byte);
    u32x2 w = {mx_pack8(v[0][0], v[0][1], v[0][2], v[0][3], inverse), mx_pack8(v[1][0], v[1][1], v[1][2], v[1][3], inverse)};
    if (byte == 255) w = u32x2{0x7F7F7F7Fu, 0x7F7F7F7Fu};
    store(o, g, rt >> 1, lt, w, byte, lane);
  }
};

// Workgroup: one unit of row tiles by one lane tile, a wave for each split.
template <class Epi>
__global__ __launch_bounds__(256) void k_mx_simple(MxGeometry g, typename Epi::Out o, int units) {
  constexpr int M = Epi::kMats, U = Epi::kUnit;
  __shared__ f32x4 part[kSplits][M][U][kWave];
  const int lane = threadIdx.x & 63, split = threadIdx.x >> 6;
  const int unit = blockIdx.x % units, lt = blockIdx.x / units;
  if constexpr (U == 2) {
    if (unit * U >= g.tiles[0]) {
      if (split == 0) Epi::store(o, g, unit, lt, u32x2{0u, 0u}, 0, lane);
      return;
    }
  }
  const uint8_t *wc[M][U], *ws[M][U];
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int r = 0; r < U; ++r) {
      int rt = unit * U + r, which = m;
      if constexpr (U == 1) which = mx_matrix(g, rt);
      else rt = min(rt, g.tiles[0] - 1);
      wc[m][r] = (which == 0 ? g.wc[0] : which == 1 ? g.wc[1] : g.wc[2]) + static_cast<int64_t>(rt) * g.groups * 4 * kCode4Bytes + lane * 16;
      ws[m][r] = (which == 0 ? g.ws[0] : which == 1 ? g.ws[1] : g.ws[2]) + static_cast<int64_t>(rt) * g.groups * kScaleBytes + lane * 4;
    }
  const uint8_t* xc = g.xc + static_cast<int64_t>(lt) * g.groups * 4 * kCode8Bytes + lane * 16;
  const uint8_t* xs = g.xs + static_cast<int64_t>(lt) * g.groups * kScaleBytes + lane * 4;
  f32x4 acc[M][U];
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int r = 0; r < U; ++r) acc[m][r] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int end = min((split + 1) * g.per, g.groups);
  for (int i = split * g.per; i < end; ++i) {
    const uint32_t sx = *reinterpret_cast<const uint32_t*>(xs + i * kScaleBytes);
    uint32_t sw[M][U];
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int r = 0; r < U; ++r) sw[m][r] = *reinterpret_cast<const uint32_t*>(ws[m][r] + i * kScaleBytes);
    unroll<4>([&](auto c) {
      const int kc = i * 4 + c;
      const u32x4 x0 = load16(xc + static_cast<int64_t>(kc) * kCode8Bytes), x1 = load16(xc + static_cast<int64_t>(kc) * kCode8Bytes + 1024);
#pragma unroll
      for (int m = 0; m < M; ++m)
#pragma unroll
        for (int r = 0; r < U; ++r)
          acc[m][r] = mx_mfma<c>(load16(wc[m][r] + static_cast<int64_t>(kc) * kCode4Bytes), x0, x1, acc[m][r], sw[m][r], sx);
    });
  }
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int r = 0; r < U; ++r) part[split][m][r][lane] = acc[m][r];
  __syncthreads();
  if (split) return;
  const int splits = (g.groups + g.per - 1) / g.per;
  for (int s = 1; s < splits; ++s)
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int r = 0; r < U; ++r) acc[m][r] += part[s][m][r][lane];
  Epi::apply(o, g, unit * U, lt, acc, lane);
}

template <class Epi>
int run(const char* what, const MxGeometry& g, const typename Epi::Out& o, int row_tiles, hipStream_t st) {
  // z is written to the end of its last group of 512 columns
  const int units = Epi::kUnit == 2 ? mx_groups(row_tiles * 16) * (kMxGroup / kMxBlock) : row_tiles;
  const int64_t groups = static_cast<int64_t>(units) * g.lane_groups;
  if (groups > INT_MAX) return mx_refused(what, "rows and weights are too large together");
  hipLaunchKernelGGL((k_mx_simple<Epi>), dim3(static_cast<unsigned>(groups)), dim3(256), 0, st, g, o, units);
  return mx_launched(what);
}

const char* operands(const StrideLanes& l, const StrideMxTiles& x, const StrideMxTiles* const* w, int n, MxGeometry& g) {
  if (const char* why = mx_why_not(x, l.lane_groups, 0)) return why;
  g = MxGeometry{};
  g.xc = x.codes;
  g.xs = x.scales;
  for (int i = 0; i < n; ++i) {
    if (const char* why = mx_why_not(*w[i], 1, x.cols)) return why;
    g.wc[i] = w[i]->codes;
    g.ws[i] = w[i]->scales;
    g.tiles[i] = w[i]->tiles;
    if (w[i]->tiles > (1 << 26)) return "too many row tiles";
  }
  g.groups = mx_groups(x.cols);
  g.per = (g.groups + kSplits - 1) / kSplits;
  g.rows = l.rows;
  g.lane_groups = l.lane_groups;
  return nullptr;
}

}  // namespace
}  // namespace stride_tc

using namespace stride_tc;

static_assert(sizeof(StrideMxGemmParams) == 72 && sizeof(StrideMxMlp13Params) == 112, "MxGemmParams layout");
static_assert(sizeof(StrideMxQkvParams) == 216 && offsetof(StrideMxQkvParams, kv) == 128, "MxQkvParams layout");

extern "C" {

int stride_mx_gemm(const StrideMxGemmParams* p, void* stream) {
  const char* what = "mx_gemm";
  if (!p) return mx_refused(what, "null parameters");
  if (!mx_lanes_ok(p->l)) return mx_refused(what, "need rows >= 0 and lane_groups = ceil(rows/16)");
  if (p->l.rows == 0) return 0;
  MxGeometry g;
  const StrideMxTiles* w[] = {&p->w};
  if (const char* why = operands(p->l, p->x, w, 1, g)) return mx_refused(what, why);
  if (!p->y || reinterpret_cast<uintptr_t>(p->y) % 16) return mx_refused(what, "y must be there, 16-byte aligned");
  return run<EpiY>(what, g, EpiY::Out{p->y, p->w.tiles}, p->w.tiles, static_cast<hipStream_t>(stream));
}

int stride_mx_mlp13(const StrideMxMlp13Params* p, void* stream) {
  const char* what = "mx_mlp13";
  if (!p) return mx_refused(what, "null parameters");
  if (!mx_lanes_ok(p->l)) return mx_refused(what, "need rows >= 0 and lane_groups = ceil(rows/16)");
  if (p->l.rows == 0) return 0;
  MxGeometry g;
  const StrideMxTiles* w[] = {&p->w1, &p->w3};
  if (const char* why = operands(p->l, p->x, w, 2, g)) return mx_refused(what, why);
  if (p->w1.tiles != p->w3.tiles) return mx_refused(what, "w1 and w3 must have equal tiles");
  if (p->w1.tiles > (1 << 16)) return mx_refused(what, "too many row tiles");
  if (const char* why = mx_why_not(p->z, p->l.lane_groups, p->w1.tiles * 16)) return mx_refused(what, why);
  if (p->z.codes == p->x.codes) return mx_refused(what, "z must not be x");
  return run<EpiZ>(what, g, EpiZ::Out{p->z}, p->w1.tiles, static_cast<hipStream_t>(stream));
}

int stride_mx_qkv(const StrideMxQkvParams* p, void* stream) {
  const char* what = "mx_qkv";
  if (!p) return mx_refused(what, "null parameters");
  if (!mx_lanes_ok(p->l)) return mx_refused(what, "need rows >= 0 and lane_groups = ceil(rows/16)");
  if (p->l.rows == 0) return 0;
  MxGeometry g;
  const StrideMxTiles* w[] = {&p->q, &p->k, &p->v};
  if (const char* why = operands(p->l, p->x, w, 3, g)) return mx_refused(what, why);
  if (p->k.tiles != p->v.tiles) return mx_refused(what, "k and v must have equal tiles");
  const int D = p->head_dim;
  if (D <= 0 || D % 16 || (static_cast<int64_t>(p->q.tiles) * 16) % D || (static_cast<int64_t>(p->k.tiles) * 16) % D)
    return mx_refused(what, "head_dim must be a multiple of 16 dividing the q and k rows");
  if (!p->q_out || !p->rope || !p->row_slot || !p->row_pos || !p->kv.arena || !p->kv.table) return mx_refused(what, "missing pointer");
  if (p->q_stride < static_cast<int64_t>(p->q.tiles) * 16 || p->q_stride > INT_MAX) return mx_refused(what, "bad q_stride");
  if (p->kv.head_dim != D || p->kv.group_elems <= 0 || p->kv.group_elems % D) return mx_refused(what, "kv.head_dim must equal head_dim and kv.group_elems must be tokens*head_dim");
  if (p->layer < 0 || p->kv.max_blocks < 1) return mx_refused(what, "bad layer or max_blocks");
  const int64_t page = p->kv.group_elems / D;
  int shift = 0;
  while ((int64_t{1} << shift) < page) ++shift;
  if ((int64_t{1} << shift) != page) return mx_refused(what, "KV page size (group_elems/head_dim) must be a power of two");
  EpiQkv::Out o{};
  o.q_out = p->q_out;
  o.q_stride = static_cast<int32_t>(p->q_stride);
  o.layer = p->layer;
  o.head_dim = D;
  o.page_shift = shift;
  o.kv = p->kv;
  o.rope = p->rope;
  o.row_slot = p->row_slot;
  o.row_pos = p->row_pos;
  return run<EpiRope>(what, g, o, p->q.tiles + p->k.tiles + p->v.tiles, static_cast<hipStream_t>(stream));
}

}  // extern "C"
