// The linear layers' products on microscaled operands (include/stride_mx.h): e2m1 weights by e4m3
// activations, v_mfma_scale_f32_16x16x128_f8f6f4, fp32 sums.
//
// Every kernel evaluates the same expression: the chunks of 128 columns chain in ascending order from
// zero on, so a row has the same bits whatever the batch and the kernel. One chain and no splits of K:
// few rows leave a chain of K / 128 products to a wave (1 us at K = 8192, of 5.2), and in exchange many
// rows keep one accumulator a tile. (Four splits and their running sums were measured in the four-wave
// form of 256 x 128 alone, whose 128 accumulators a lane they made spill: 172 us against 54 at 4096 rows
// of 2048 x 8192. The eight-wave form that is here now has 64, and has not been measured with splits.)
//
// Times beside the kernels are us a call in a graph of calls on up to eight different matrices.
//
// What bounds them: few rows what one wave a CU has on its way, and the launch (2048 x 8192 at one row
// 5.2 us, of which an empty launch is 2: 128 waves read 68 KiB each, in two rounds of four groups), the
// middle the x that each tile of weights reads again from L2, many rows the matrix units and the power that
// they draw: 2.7 PFLOP/s at 2048 x 8192 and 4096 rows (51.7 us; 2.8 in calls one by one), with the units at
// work for 76 % of the cycles, of which there are 1.7 a ns, where a library's 8192^3 product in 8 bits
// reaches 2.96.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cstddef>

#include "mx_common.hpp"
#include "tc_epilogue.hpp"

namespace stride_tc {
namespace {

// Up to three matrices over the same x, their row tiles end to end (q, k, v), or gate and up.
struct MxGeometry {
  const uint8_t *xc, *xs;          // codes and scales
  const uint8_t *wc[3], *ws[3];
  int32_t tiles[3];                // of 16 rows
  int32_t groups;  // of 512 columns
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
// output rows 4 * (l / 16) + i. kUnit row tiles of kMats matrices belong together.
struct EpiY {
  static constexpr int kMats = 1, kUnit = 1;
  struct Out {
    uint16_t* y;
    int32_t row_tiles;
  };
  __device__ __forceinline__ static void finish(const Out& o, const MxGeometry& g, int rt, int lt, const f32x4 (&y)[1][1], int lane) {
    if (lt * 16 + (lane & 15) >= g.rows) return;
    const f32x4 v = y[0][0];
    *reinterpret_cast<u32x2*>(o.y + (static_cast<int64_t>(lt) * o.row_tiles + rt) * kTileElems + (lane & 15) * 16 + (lane >> 4) * 4) =
        u32x2{bf16_rne(v[0]) | bf16_rne(v[1]) << 16, bf16_rne(v[2]) | bf16_rne(v[3]) << 16};
  }
};

struct EpiRope {
  static constexpr int kMats = 1, kUnit = 1;
  struct Out : EpiQkv::Out {
    int32_t slots, positions;  // rows of the page table and of the rope table
  };
  __device__ __forceinline__ static void finish(const Out& o, const MxGeometry& g, int rt, int lt, const f32x4 (&y)[1][1], int lane) {
    // A lane whose row has no place in the cache has none here either: past this neither table is read
    // behind its end (the cache's last page may hold positions that rope has no row for).
    const int j = lt * 16 + (lane & 15);
    bool live = j < g.rows;
    if (live) {
      const int pos = o.row_pos[j], slot = o.row_slot[j];
      live = pos >= 0 && pos < o.positions && (pos >> o.page_shift) < o.kv.max_blocks && slot >= 0 && slot < o.slots;
    }
    Geometry rows{};
    rows.rows = live ? g.rows : 0;
    const int which = mx_matrix(g, rt);
    EpiQkv::apply(o, rows, which, rt, lt, y[0], lane);
  }
};

// x / (1 + e^-x) with the hardware's exponential and reciprocal, each good to an ulp or so: the result
// is rounded to four bits. 0 where 1 / (1 + e^-x) is no normal number, x below -87.3. (2048 rows of
// 2 x 8192 x 2048: 58.6 us, 68.7 with the exact division and the polynomial that the bf16 path has for its
// bits.)
__device__ __forceinline__ float silu(float x) {
  return x * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * -1.44269504088896341f));
}

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
  __device__ __forceinline__ static void finish(const Out& o, const MxGeometry& g, int unit, int lt, const f32x4 (&y)[2][2], int lane) {
    float v[2][4];
    uint32_t most = 0;
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[r][i] = unit * 2 + r < g.tiles[0] ? silu(y[0][r][i]) * y[1][r][i] : 0.0f;
        most = max(most, mx_abs_bits(v[r][i]));
      }
    const auto halves = __builtin_amdgcn_permlane32_swap(most, most, false, false);
    most = max(halves[0], halves[1]);
    const auto quarters = __builtin_amdgcn_permlane16_swap(most, most, false, false);
    most = max(quarters[0], quarters[1]);
    const int byte = mx_scale_byte<8>(most);
    const float inverse = mx_inverse(byte);
    u32x2 w = {mx_pack8(v[0][0], v[0][1], v[0][2], v[0][3], inverse), mx_pack8(v[1][0], v[1][1], v[1][2], v[1][3], inverse)};
    if (byte == 255) w = u32x2{0x7F7F7F7Fu, 0x7F7F7F7Fu};
    store(o, g, unit, lt, w, byte, lane);
  }
};

// Weight tile rt of the matrices end to end (one at a time) or of matrix m (two at a time), the last one
// where there is none.
template <class Epi>
__device__ __forceinline__ void mx_source(const MxGeometry& g, int m, int rt, const uint8_t*& codes, const uint8_t*& scales) {
  int which = m;
  if constexpr (Epi::kMats == 1) {
    rt = min(rt, g.tiles[0] + g.tiles[1] + g.tiles[2] - 1);
    which = mx_matrix(g, rt);
  } else {
    rt = min(rt, g.tiles[0] - 1);
  }
  codes = (which == 0 ? g.wc[0] : which == 1 ? g.wc[1] : g.wc[2]) + static_cast<int64_t>(rt) * g.groups * 4 * kCode4Bytes;
  scales = (which == 0 ? g.ws[0] : which == 1 ? g.ws[1] : g.ws[2]) + static_cast<int64_t>(rt) * g.groups * kScaleBytes;
}

// Few output tiles: a wave has one weight tile by one lane tile, operands straight to registers, P
// groups of K in use and P on their way (2048 x 8192 at one row with P = 4 / 2: 5.2 / 6.5 us). The tiles
// of a unit meet in LDS.
template <class Epi, int P>
__global__ __launch_bounds__(64 * Epi::kMats * Epi::kUnit) void k_mx_row(MxGeometry g, typename Epi::Out o, int units) {
  constexpr int M = Epi::kMats, U = Epi::kUnit;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int unit = blockIdx.x % units, lt = blockIdx.x / units;
  const uint8_t *wc, *ws;
  mx_source<Epi>(g, wave / U, unit * U + wave % U, wc, ws);
  const uint8_t* xc = g.xc + static_cast<int64_t>(lt) * g.groups * 4 * kCode8Bytes;
  const uint8_t* xs = g.xs + static_cast<int64_t>(lt) * g.groups * kScaleBytes;
  // lanes without a row take the last one's: for one row a quarter of the lines
  const int row = min(lane & 15, g.rows - 1 - lt * 16);
  const uint32_t at16 = lane * 16, at4 = lane * 4, x16 = ((lane & 48) + row) * 16, x4 = x16 / 4;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  struct Part {
    u32x4 w[P][4], x[P][4][2];
    uint32_t sw[P], sx[P];
  };
  Part part[2];
  auto load = [&](Part& t, int first) {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int64_t i = min(first + p, g.groups - 1);
      t.sx[p] = *reinterpret_cast<const uint32_t*>(xs + i * kScaleBytes + x4);
      t.sw[p] = *reinterpret_cast<const uint32_t*>(ws + i * kScaleBytes + at4);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        t.w[p][c] = load16(wc + (i * 4 + c) * kCode4Bytes + at16);
#pragma unroll
        for (int h = 0; h < 2; ++h) t.x[p][c][h] = load16(xc + (i * 4 + c) * kCode8Bytes + h * 1024 + x16);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  auto products = [&](const Part& t, int first) {
    unroll<P>([&](auto p) {
      if (p > 0 && first + p >= g.groups) return;
      unroll<4>([&](auto c) { acc = mx_mfma<c>(t.w[p][c], t.x[p][c][0], t.x[p][c][1], acc, t.sw[p], t.sx[p]); });
    });
  };
  load(part[0], 0);
  for (int i = 0; i < g.groups; i += 2 * P) {
    if (i + P < g.groups) load(part[1], i + P);
    products(part[0], i);
    if (i + 2 * P < g.groups) load(part[0], i + 2 * P);
    if (i + P < g.groups) products(part[1], i + P);
  }
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7");
  asm volatile("" : "+v"(acc));
  f32x4 y[M][U];
  if constexpr (M * U > 1) {
    __shared__ f32x4 tiles[M * U][kWave];
    tiles[wave][lane] = acc;
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int u = 0; u < U; ++u) y[m][u] = tiles[m * U + u][lane];
  } else {
    y[0][0] = acc;
  }
  Epi::finish(o, g, unit, lt, y, lane);
}

// A wave's 64 x 16 or 64 x 4 bytes from base + offset to LDS at `to` on, in lane order. In assembly,
// since the compiler would wait for every such copy before any read of LDS; wait_copies() does it.
__device__ __forceinline__ void copy16(uint32_t to, uint32_t offset, const uint8_t* base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(__builtin_amdgcn_readfirstlane(to)), "v"(offset), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void copy4(uint32_t to, uint32_t offset, const uint8_t* base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(__builtin_amdgcn_readfirstlane(to)), "v"(offset), "s"(base) : "memory", "m0");
}
// Until at most N of the wave's copies are on their way.
template <int N>
__device__ __forceinline__ void wait_copies() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint32_t lds_at(const void* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) void*)p));
}

// Many rows: workgroup of WM x WN waves, A weight tiles by L lane tiles a wave. A chunk's operands
// (weights 1 KiB, activations 2 KiB a tile) go to a ring of NS stages in LDS by global_load_lds, a
// group's scales beside its first chunk; a wave reads a chunk's fragments while it multiplies the one
// before. Copies and reads lie between the products: issued together behind the barrier a chunk of 256 x 128
// by four waves took 1760 cycles, spread 1200, of which the matrix units work 1024; by eight waves, which
// cover each other's waits too, the whole product takes 51.7 us against 53.0. (A raised wave priority in the
// loop changed nothing.)
template <class Epi, int A, int L, int WM, int WN, int NS, int OCC>
__global__ __launch_bounds__(64 * WM * WN, OCC) void k_mx_pipe(MxGeometry g, typename Epi::Out o, int units, int unit_blocks, int lane_blocks) {
  constexpr int M = Epi::kMats, U = Epi::kUnit, NW = WM * WN;
  constexpr int T = A / M;                  // row tiles of a wave
  constexpr int WA = WM * A, WL = WN * L;   // weight and lane tiles of the workgroup
  constexpr int kCodes = WA + 2 * WL;       // KiB of a stage
  constexpr int kScales = WA + WL;          // quarter KiB of a group
  static_assert(kCodes % NW == 0 && kScales % NW == 0, "copies must split evenly over the waves");
  constexpr int PC = kCodes / NW, PS = kScales / NW;
  __shared__ u32x4 ring[NS][kCodes][kWave];
  __shared__ uint32_t scales[2][kScales][kWave];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;
  // eight blocks of rows walk the lane blocks together, so that an XCD's workgroups share operands in its L2
  const int b = xcd_remap(blockIdx.x, gridDim.x);
  constexpr int G = 8;
  const int gang = b / (G * lane_blocks), size = min(G, unit_blocks - gang * G), within = b % (G * lane_blocks);
  const int ub = gang * G + within % size, lb = within / size;
  const int rt0 = ub * WM * T, lt0 = lb * WL;  // of the workgroup

  const uint8_t *src[PC], *ssrc[PS];
#pragma unroll
  for (int i = 0; i < PC; ++i) {
    const int j = wave + i * NW;
    if (j < WA) {
      const int m = j / (WM * T), t = j % (WM * T);
      const uint8_t* unused;
      mx_source<Epi>(g, m, rt0 + t, src[i], unused);
    } else {
      const int lt = min(lt0 + (j - WA) / 2, g.lane_groups - 1);
      src[i] = g.xc + static_cast<int64_t>(lt) * g.groups * 4 * kCode8Bytes + (j - WA) % 2 * 1024;
    }
  }
#pragma unroll
  for (int i = 0; i < PS; ++i) {
    const int j = wave + i * NW;
    if (j < WA) {
      const int m = j / (WM * T), t = j % (WM * T);
      const uint8_t* unused;
      mx_source<Epi>(g, m, rt0 + t, unused, ssrc[i]);
    } else {
      ssrc[i] = g.xs + static_cast<int64_t>(min(lt0 + j - WA, g.lane_groups - 1)) * g.groups * kScaleBytes;
    }
  }
  const uint32_t at16 = lane * 16, at4 = lane * 4;
  const uint32_t ring_at = lds_at(&ring[0][0][0]) + wave * 1024, scales_at = lds_at(&scales[0][0][0]) + wave * 256;
  // copies [FROM, TO) of a stage, the scales' first where a group begins
  auto issue = [&](int stage, int slot, auto with_scales, auto from, auto to) {
    constexpr int lead = with_scales ? PS : 0;
    unroll<to - from>([&](auto n) {
      constexpr int i = from + n - lead;
      if constexpr (i < 0) {
        copy4(scales_at + ((stage >> 2) & 1) * (kScales * 256) + (i + lead) * NW * 256, at4, ssrc[i + lead] + static_cast<int64_t>(stage >> 2) * kScaleBytes);
      } else {
        const int64_t step = static_cast<int64_t>(stage) * (wave + i * NW < WA ? kCode4Bytes : kCode8Bytes);
        copy16(ring_at + (slot * kCodes + i * NW) * 1024, at16, src[i] + step);
      }
    });
  };

  f32x4 acc[A][L];
  u32x4 fa[A], fb[2][L][2];
  uint32_t sa[2][A], sb[2][L];
#pragma unroll
  for (int a = 0; a < A; ++a)
#pragma unroll
    for (int l = 0; l < L; ++l) acc[a][l] = f32x4{0.f, 0.f, 0.f, 0.f};
  // weight tile a of a wave: matrix a / T, row tile a % T
  auto tile = [&](int a) { return a / T * (WM * T) + wm * T + a % T; };
  // the n-th fragment of x, the n-th word of scales
  auto read_x = [&](auto buf, int slot, auto n) { fb[buf][n / 2][n % 2] = ring[slot][WA + wn * L * 2 + n][lane]; };
  auto read_scale = [&](int buf, int group, auto n) {
    if constexpr (n < A) sa[buf][n] = scales[group & 1][tile(n)][lane];
    else sb[buf][n - A] = scales[group & 1][WA + wn * L + n - A][lane];
  };
  auto sync = [] {
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  using Zero = std::integral_constant<int, 0>;
  unroll<NS>([&](auto s) {
    constexpr bool first = s % 4 == 0;
    issue(s, s, std::bool_constant<first>{}, Zero{}, std::integral_constant<int, PC + (first ? PS : 0)>{});
  });
  wait_copies<(NS - 1) * PC>();
  sync();
  unroll<2 * L>([&](auto n) { read_x(Zero{}, 0, n); });
  unroll<A + L>([&](auto n) { read_scale(0, 0, n); });
#pragma unroll
  for (int a = 0; a < A; ++a) fa[a] = ring[0][tile(a)][lane];

  // Chunks 4 i .. 4 i + 3 of group i, without a branch, so that the products stay where they are
  // written.
  int at = 0;  // the slot of the stage, where it doesn't follow from c
  auto group = [&](int i, auto last) {
    unroll<4>([&](auto c) {
      constexpr int cur = c & 1, nxt = cur ^ 1;
      const int slot = 4 % NS == 0 ? c % NS : at, after = 4 % NS == 0 ? (c + 1) % NS : (at + 1 == NS ? 0 : at + 1);
      at = after;
      // copies behind those of stage + 1: NS - 2 stages, a group's scales among them
      constexpr int behind = last ? std::min(NS - 2, std::max(0, 2 - c)) : NS - 2;
      constexpr bool scaled = !last && c < 4 && c + 2 <= 4 && c + NS - 1 >= 4;
      constexpr bool more = !last || c < 3, copies = !last || c + NS < 4, starts = (c + NS) % 4 == 0;
      // A step has the products of a weight fragment. Behind the first ones lies the barrier, and in
      // the others the next chunk's fragments are read and a stage is copied to the slot of this one,
      // a few at a time, so that the matrix unit never waits for long.
      constexpr int kOpen = A / 4, kSteps = A - kOpen;
      unroll<A>([&](auto a) {
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (a == kOpen && more) {
          // stage + 1 has landed, and what is being refilled has been read, by every wave
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          wait_copies<behind * PC + (scaled ? PS : 0)>();
          sync();
        }
        if constexpr (a >= kOpen) {
          constexpr int n = a - kOpen;
          if constexpr (more) {
            constexpr int x0 = 2 * L * n / kSteps, x1 = 2 * L * (n + 1) / kSteps;
            unroll<x1 - x0>([&](auto i) { read_x(std::integral_constant<int, nxt>{}, after, std::integral_constant<int, x0 + i>{}); });
            constexpr int w0 = n == 0 ? 0 : a - 1;
            unroll<a - w0>([&](auto i) { fa[w0 + i] = ring[after][tile(w0 + i)][lane]; });
          }
          if constexpr (!last && c == 3) {
            constexpr int s0 = (A + L) * n / kSteps, s1 = (A + L) * (n + 1) / kSteps;
            unroll<s1 - s0>([&](auto q) { read_scale(1, i + 1, std::integral_constant<int, s0 + q>{}); });
          }
          if constexpr (copies) {
            constexpr int all = PC + (starts ? PS : 0);
            issue(i * 4 + c + NS, slot, std::bool_constant<starts>{}, std::integral_constant<int, all * n / kSteps>{},
                  std::integral_constant<int, all * (n + 1) / kSteps>{});
          }
        }
#pragma unroll
        for (int l = 0; l < L; ++l) acc[a][l] = mx_mfma<c>(fa[a], fb[cur][l][0], fb[cur][l][1], acc[a][l], sa[0][a], sb[0][l]);
      });
      if constexpr (more) fa[A - 1] = ring[after][tile(A - 1)][lane];
    });
    if constexpr (!last) {
#pragma unroll
      for (int a = 0; a < A; ++a) sa[0][a] = sa[1][a];
#pragma unroll
      for (int l = 0; l < L; ++l) sb[0][l] = sb[1][l];
    }
  };
  const int end = g.groups - 1;
  for (int i = 0; i < end; ++i) group(i, std::false_type{});
  group(end, std::true_type{});
  // The products end here: without a use in this place the compiler moves them into the branches
  // below. (The wait covers the longest of them; what follows is no instruction.)
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7");
#pragma unroll
  for (int a = 0; a < A; ++a)
#pragma unroll
    for (int l = 0; l < L; ++l) asm volatile("" : "+a"(acc[a][l]));

  unroll<T / U>([&](auto r) {
    unroll<L>([&](auto l) {
      const int unit = (rt0 + wm * T) / U + r, lt = lt0 + wn * L + l;
      if (unit >= units || lt >= g.lane_groups) return;
      f32x4 v[M][U];
#pragma unroll
      for (int m = 0; m < M; ++m)
#pragma unroll
        for (int u = 0; u < U; ++u) v[m][u] = acc[m * T + r * U + u][l];
      Epi::finish(o, g, unit, lt, v, lane);
    });
  });
}

// In between: workgroup of 2 x 2 waves, a weight tile by a lane tile each; a group of 512 columns is a
// stage of a ring of three, two of them on their way (a chunk a stage as above has too little on its way
// for such small tiles: 2048 x 8192 at 128 rows 12.5 us as 64 x 64, 8.1 here). One matrix at a time:
// gate and up, whose unit is 32 x 32 of each, go from waves of their own to 64 x 64.
template <class Epi>
__global__ __launch_bounds__(256) void k_mx_tile(MxGeometry g, typename Epi::Out o, int units, int lane_blocks) {
  static_assert(Epi::kMats == 1 && Epi::kUnit == 1, "a wave has a weight tile");
  constexpr int NS = 3;
  constexpr int PC = 6;  // KiB of codes that a wave copies of a stage's 24: a chunk of each weight tile, four halves of x's
  __shared__ u32x4 ring[NS][4 * PC][kWave];
  __shared__ uint32_t scales[NS][4][kWave];  // of both weight tiles, of both lane tiles
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave >> 1, wn = wave & 1;
  const int b = xcd_remap(blockIdx.x, gridDim.x);
  const int rt0 = b / lane_blocks * 2, lt0 = b % lane_blocks * 2;  // an XCD reads a weight tile once
  auto x_tile = [&](int i) { return static_cast<int64_t>(min(lt0 + i, g.lane_groups - 1)); };
  const uint8_t *src[PC], *ssrc, *unused;
#pragma unroll
  for (int i = 0; i < PC; ++i) {
    if (i < 2) {
      mx_source<Epi>(g, 0, rt0 + i, src[i], unused);
      src[i] += wave * kCode4Bytes;
    } else {
      const int j = wave + (i - 2) * 4;
      src[i] = g.xc + x_tile(j / 8) * g.groups * 4 * kCode8Bytes + j % 8 * 1024;
    }
  }
  if (wave < 2) mx_source<Epi>(g, 0, rt0 + wave, unused, ssrc);
  else ssrc = g.xs + x_tile(wave - 2) * g.groups * kScaleBytes;
  const uint32_t at16 = lane * 16, at4 = lane * 4;
  const uint32_t ring_at = lds_at(&ring[0][0][0]) + wave * 1024, scales_at = lds_at(&scales[0][0][0]) + wave * 256;
  auto issue = [&](int stage, int slot) {
    copy4(scales_at + slot * 1024, at4, ssrc + static_cast<int64_t>(stage) * kScaleBytes);
#pragma unroll
    for (int i = 0; i < PC; ++i)
      copy16(ring_at + (slot * PC + i) * 4096, at16, src[i] + static_cast<int64_t>(stage) * 4 * (i < 2 ? kCode4Bytes : kCode8Bytes));
  };
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  const int first = min(NS - 1, g.groups);
  for (int i = 0; i < first; ++i) issue(i, i);
  int slot = 0, next = NS - 1;  // of stage i, of stage i + NS - 1
  for (int i = 0; i < g.groups; ++i) {
    // stage i has landed (the one behind it may be on its way); what is being refilled has been read, by every wave
    if (i + 1 < g.groups) wait_copies<PC + 1>();
    else wait_copies<0>();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    const uint32_t sa = scales[slot][wm][lane], sb = scales[slot][2 + wn][lane];
    u32x4 fa[4], fb[4][2];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
#pragma unroll
      for (int h = 0; h < 2; ++h) fb[c][h] = ring[slot][8 + wn * 8 + c * 2 + h][lane];
      fa[c] = ring[slot][wm * 4 + c][lane];
    }
    if (i + NS - 1 < g.groups) issue(i + NS - 1, next);  // while the fragments are on their way
    unroll<4>([&](auto c) { acc = mx_mfma<c>(fa[c], fb[c][0], fb[c][1], acc, sa, sb); });
    slot = slot + 1 == NS ? 0 : slot + 1;
    next = next + 1 == NS ? 0 : next + 1;
  }
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7");
  asm volatile("" : "+v"(acc));
  const int unit = rt0 + wm, lt = lt0 + wn;
  if (unit >= units || lt >= g.lane_groups) return;
  const f32x4 v[1][1] = {{acc}};
  Epi::finish(o, g, unit, lt, v, lane);
}

template <class Epi, int P>
void launch_row(const MxGeometry& g, const typename Epi::Out& o, int units, hipStream_t st) {
  hipLaunchKernelGGL((k_mx_row<Epi, P>), dim3(units * g.lane_groups), dim3(64 * Epi::kMats * Epi::kUnit), 0, st, g, o, units);
}

template <class Epi, int A, int L, int WM, int WN, int NS, int OCC>
const char* launch_pipe(const MxGeometry& g, const typename Epi::Out& o, int units, const char* clash, hipStream_t st) {
  constexpr int per = WM * A / Epi::kMats / Epi::kUnit;
  const int unit_blocks = (units + per - 1) / per, lane_blocks = (g.lane_groups + WN * L - 1) / (WN * L);
  if (static_cast<int64_t>(unit_blocks) * lane_blocks > kMxMostGroups * 1024 / (64 * WM * WN)) return "rows and weights are too large together";
  if (clash) return clash;
  hipLaunchKernelGGL((k_mx_pipe<Epi, A, L, WM, WN, NS, OCC>), dim3(unit_blocks * lane_blocks), dim3(64 * WM * WN), 0, st, g, o, units, unit_blocks, lane_blocks);
  return nullptr;
}

template <class Epi>
void launch_tile(const MxGeometry& g, const typename Epi::Out& o, int units, hipStream_t st) {
  const int unit_blocks = (units + 1) / 2, lane_blocks = (g.lane_groups + 1) / 2;
  hipLaunchKernelGGL(k_mx_tile<Epi>, dim3(unit_blocks * lane_blocks), dim3(256), 0, st, g, o, units, lane_blocks);
}

// Host: does a result lie on x or on one of the weights? (Other workgroups read them until the end.)
bool overlaps(std::initializer_list<MxSpan> results, const StrideLanes& l, const StrideMxTiles& x, const StrideMxTiles* const* w, int n) {
  bool any = mx_overlap(results, {mx_codes(x, l.lane_groups, 8), mx_scales(x, l.lane_groups)});
  for (int i = 0; i < n; ++i) any = any || mx_overlap(results, {mx_codes(*w[i], w[i]->tiles, 4), mx_scales(*w[i], w[i]->tiles)});
  return any;
}

// `clash`: why the memory of the call's arguments is refused, or NULL.
template <class Epi>
int run(const char* what, const MxGeometry& g, const typename Epi::Out& o, int row_tiles, const char* clash, hipStream_t st) {
  // z is written to the end of its last group of 512 columns
  const int units = Epi::kUnit == 2 ? mx_groups(row_tiles * 16) * (kMxGroup / kMxBlock) : row_tiles;
  // configuration
  // By the number of 16 x 16 products, of which the card's 256 CUs want four each before tiles pay. us
  // here / as the other forms, with 4 groups at K = 2048, 16 at 8192 and 28 at 14336; where a border lies
  // between two sizes measured, it may be a few per cent off for sizes near it:
  //   a wave a tile to 768 (1536 where K is short; gate and up, which have no 32 x 32: 1280): 2048 x
  //     8192 at 1 / 64 rows (128, 512 products) 5.2 / 6.9 against 7.6 / 7.7 as 32 x 32, at 128 rows (1024) 9.7
  //     against 8.1; 8192 x 2048 at 32 rows (1024) 4.0 against 4.9, 2048 x 2048 at 128 / 192 rows (1024, 1536)
  //     4.0 / 6.0 against 4.2 / 5.2; gate and up 8192 x 2048 at 16 / 32 rows (1024, 2048) 5.6 / 6.9 against
  //     6.1 / 6.3 as 64 x 64
  //   32 x 32 to 1536: 2048 x 8192 at 128 / 192 rows (1024, 1536) 8.1 / 11.3 against 12.5 as 64 x 64, at
  //     256 / 384 rows 12.1 / 17.1 against 12.6 / 13.1; 4096 x 14336 at 64 rows (1024) 12.4 against 19.4
  //   64 x 64 to 6144: 8192 x 2048 at 96 rows 6.1 against 7.4 as 32 x 32; 2048 x 8192 at 512 rows (4096) 13.9
  //     against 15.6 as 128 x 64, but at 768 (6144) 19.4 against 16.3, and at 1024 20.9 against 17.6
  //   128 x 64 to 9216: 2048 x 8192 at 1024 rows (8192) 17.6 against 21.6 as 128 x 128, at 1280 25.8 against
  //     22.6; gate and up 8192 x 2048 at 128 rows (8192) 7.6 against 8.0 as 64 x 64
  //   128 x 128 of eight waves, by a workgroup a CU while 256 do: 2048 x 8192 at 2048 rows (16384) 29.9 against
  //     31.2 by two, 33.6 as 128 x 64 and 40.7 as 256 x 128; gate and up at 256 rows 10.3 against 10.5 by two
  //   beyond, where K is short, by two workgroups a CU, whose ends hide each other: 8192 x 2048 at 2048 / 4096
  //     rows 35.8 / 68.8 against 35.9 / 70.9 as 256 x 128, gate and up at 2048 rows 58.6 against 60.7; by four
  //     waves 46.7 and 73.1
  //   256 x 128 where K is long: the fewest bytes a product, of which a CU reads 75 to 80 a ns from its
  //     L2, and by which the clock stays up: 2048 x 8192 at 4096 rows 51.7 against 58.4 as 128 x 128, 4096
  //     x 14336 163 against 184; by four waves, one a SIMD, 53.0 and 164
  const int64_t products = static_cast<int64_t>(row_tiles) * Epi::kMats * g.lane_groups;
  if (clash && products <= 1536) return mx_refused(what, clash);  // a launch of these fits
  const char* why = nullptr;
  if (products <= (Epi::kMats == 2 ? 1280 : g.groups <= 4 ? 1536 : 768)) launch_row<Epi, 4 / Epi::kMats>(g, o, units, st);
  else if (Epi::kMats == 1 && products <= 1536) {
    if constexpr (Epi::kMats == 1) launch_tile<Epi>(g, o, units, st);
  } else if (products <= 6144) why = launch_pipe<Epi, 4, 1, 1, 4, 4, 2>(g, o, units, clash, st);
  else if (products <= 9216) why = launch_pipe<Epi, 4, 2, 2, 2, 4, 2>(g, o, units, clash, st);
  else if (products <= 16384) why = launch_pipe<Epi, 4, 2, 2, 4, 4, 2>(g, o, units, clash, st);
  else if (g.groups < 8) why = launch_pipe<Epi, 4, 2, 2, 4, 3, 4>(g, o, units, clash, st);
  else why = launch_pipe<Epi, 8, 2, 2, 4, 4, 2>(g, o, units, clash, st);
  if (why) return mx_refused(what, why);
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
  const bool clash = overlaps({{p->y, p->l.lane_groups * int64_t{2} * kTileElems * p->w.tiles}}, p->l, p->x, w, 1);
  return run<EpiY>(what, g, EpiY::Out{p->y, p->w.tiles}, p->w.tiles, clash ? "y must not overlap x or w" : nullptr, static_cast<hipStream_t>(stream));
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
  const bool clash = overlaps({mx_codes(p->z, p->l.lane_groups, 8), mx_scales(p->z, p->l.lane_groups)}, p->l, p->x, w, 2);
  return run<EpiZ>(what, g, EpiZ::Out{p->z}, p->w1.tiles, clash ? "z must not overlap x, w1 or w3" : nullptr, static_cast<hipStream_t>(stream));
}

int stride_mx_qkv(const StrideMxQkvParams* p, void* stream) { return stride_mx_qkv_within(p, INT_MAX, INT_MAX, stream); }

int stride_mx_qkv_within(const StrideMxQkvParams* p, int32_t slots, int32_t positions, void* stream) {
  const char* what = "mx_qkv";
  if (!p) return mx_refused(what, "null parameters");
  if (!mx_lanes_ok(p->l)) return mx_refused(what, "need rows >= 0 and lane_groups = ceil(rows/16)");
  if (slots < 0 || positions < 0) return mx_refused(what, "slots and positions are counts");
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
  EpiRope::Out o{};
  o.slots = slots;
  o.positions = positions;
  o.q_out = p->q_out;
  o.q_stride = static_cast<int32_t>(p->q_stride);
  o.layer = p->layer;
  o.head_dim = D;
  o.page_shift = shift;
  o.kv = p->kv;
  o.rope = p->rope;
  o.row_slot = p->row_slot;
  o.row_pos = p->row_pos;
  const int64_t q_cols = static_cast<int64_t>(p->q.tiles) * 16;
  const MxSpan q = {p->q_out, ((p->l.rows - 1) * p->q_stride + q_cols) * 4}, rope = {p->rope, positions == INT_MAX ? 0 : positions * int64_t{4} * D};
  const int64_t words = p->l.rows * int64_t{4};
  const bool clash = overlaps({q}, p->l, p->x, w, 3) || mx_overlap({q}, {{p->row_slot, words}, {p->row_pos, words}, rope});
  return run<EpiRope>(what, g, o, p->q.tiles + p->k.tiles + p->v.tiles, clash ? "q_out must not overlap x, the weights or what describes the rows" : nullptr, static_cast<hipStream_t>(stream));
}

}  // extern "C"
