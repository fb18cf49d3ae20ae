// Grouped-query attention of new rows over a paged bf16 cache, all positions or the last
// `window` and the first `sinks` ones (include/stride_serve.h).
//
// The order of every sum is fixed by absolute positions, so that a row's bits do not depend
// on its batch or on the form that computes it. Positions fall into leaves of 256, a leaf
// into four chunks of 64. With s the scores times log2(e) and exp2 for exp:
//   in a leaf   a reference r starts at -inf; chunk by chunk r becomes the chunk's maximum
//               where that exceeds r + 8 (and what is summed so far is scaled by
//               exp2(old r - r)); p = exp2(s - r), rounded to bf16, enters
//               acc = sum p V and l = sum p, MFMA chains in ascending order
//   over leaves R' = max(R, r), G = G exp2(R - R') + acc exp2(r - R'), L alike
// The slack of 8 keeps p below 2^8 and saves nearly all rescaling: a reference need not be
// the maximum, only near it. A chunk or leaf that a row does not see changes nothing (p = 0,
// r as it was), so forms may skip it or not.
//
// Roundings to fewer than 32 bits: p to bf16 (up to 2^-8 relative, random over the positions; l
// sums the rounded ones, so the weights still add up to one), since the value product is a
// matrix instruction's of bf16 (results of normal inputs are 0.0022 off as a whole, with fp32
// weights and their own rounding alone 0.0017), and the result to bf16. The
// query is scale * log2(e) * q in fp32, split into two bf16 whose sum has 16 bits (2^-16
// relative): the scores keep nearly fp32 queries' accuracy (bf16 queries alone would add an
// error of the size of p's) for twice the score products.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cstddef>
#include <string>
#include <type_traits>

#include "../../include/stride_serve.h"
#include "serve_sight.hpp"
#include "tc_common.hpp"

namespace stride_tc {

int fail(int code, const std::string& msg);  // tc_gemm.hip

namespace {

constexpr int kLeaf = 256;
constexpr int kChunk = 64;
constexpr float kSlack = 8.0f;
constexpr float kLog2e = 1.44269504088896341f;

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float neg_inf() { return f32_of(0xFF800000u); }
__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

// a row of no sequence is one without a position
__device__ __forceinline__ int pos_of(const StrideWindowAttentionParams& p, int j) { return p.row_slot[j] < 0 ? -1 : max(p.row_pos[j], -1); }
__device__ __forceinline__ Sight sight_of(const StrideWindowAttentionParams& p, int pos, int limit) {
  return sight_at(pos, p.window, p.sinks, limit);
}

// The leaves that a row sees, ascending: `head` of them from 0, then those from `rest` on.
struct Leaves {
  int head, rest, count;
  __device__ __forceinline__ int at(int i) const { return i < head ? i : rest + i - head; }
};
__device__ __forceinline__ Leaves leaves_of(const Sight& s) {
  Leaves v;
  v.head = (s.sink_end + kLeaf - 1) / kLeaf;
  v.rest = max(s.lo / kLeaf, v.head);
  v.count = s.pos < 0 ? 0 : v.head + max(0, s.pos / kLeaf - v.rest + 1);
  return v;
}

// A score row's query as MFMA operand: 8 dims from `q`, times c, as two bf16 that add up to
// it to 16 bits. Both have its sign and neither is 0 where it is not (2^-24 of it does no
// harm), so that a key's infinity makes one infinity of the two products.
__device__ __forceinline__ void split_query(const float* q, float c, bool live, u32x4& hi, u32x4& lo) {
  f32x4 a = {0, 0, 0, 0}, b = {0, 0, 0, 0};
  if (live) {
    a = reinterpret_cast<const f32x4*>(q)[0];
    b = reinterpret_cast<const f32x4*>(q)[1];
  }
  bf16x8 h, l;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float v = (i < 4 ? a[i & 3] : b[i & 3]) * c;
    const float top = f32_of(u32_of(v) & 0xFFFF0000u);
    h[i] = static_cast<__bf16>(top);
    l[i] = static_cast<__bf16>(v == top ? v * 0x1p-24f : v - top);
  }
  hi = __builtin_bit_cast(u32x4, h);
  lo = __builtin_bit_cast(u32x4, l);
}

// V rows lie in LDS as [position][D] with their 64-byte blocks permuted so that the four
// rows of a transposing read fall into different banks (four rows of 64 bytes fill them).
template <int D>
__device__ __forceinline__ int v_at(int row, int dim) {
  constexpr int kBlocks = D / 32;  // 64-byte blocks of a row
  const int turn = kBlocks == 1 ? 0 : (kBlocks == 2 ? (row >> 1) & 1 : row & 3);
  return row * D + (((dim >> 5) ^ turn) << 5) + (dim & 31);
}
// Element (row + r, dim + i) for r = 0 .. 3 in lane i of each 16 lanes, whose lane i must
// pass (row + i / 4, dim + 4 * (i % 4)).
__device__ __forceinline__ u32x2 read_transposed(const uint16_t* at) {
  auto p = (__attribute__((address_space(3))) s16x4*)(at);
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(p));
}
__device__ __forceinline__ u32x4 both(u32x2 a, u32x2 b) { return u32x4{a[0], a[1], b[0], b[1]}; }
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  bf16x2 v;
  v[0] = static_cast<__bf16>(a);
  v[1] = static_cast<__bf16>(b);
  return __builtin_bit_cast(uint32_t, v);
}

constexpr uint32_t kOnes = 0x3F803F80u;  // two bf16 ones

// The fold over leaves for one column: the running reference and sum, and the factors that
// scale what is there and what comes. A leaf with l = 0 (nothing seen) changes nothing.
struct Fold {
  float ref, sum;
  __device__ __forceinline__ void take(float r, float l, float& a, float& b) {
    a = 1.0f;
    b = 0.0f;
    if (!(l == 0.0f)) {
      const float m = r > ref ? r : ref;
      a = exp2_of(ref - m);
      b = exp2_of(r - m);
      if (sum == 0.0f) a = 0.0f;  // the first leaf: -inf - -inf where its scores are NaN
      sum = __builtin_fmaf(l, b, sum * a);
      ref = m;
    }
  }
};
// (a, b) as above; NaN sums stay NaN.
__device__ __forceinline__ f32x4 folded(f32x4 g, f32x4 acc, float a, float b) {
  f32x4 o;
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(acc[e], b, g[e] * a);
  return o;
}

// Four neighbouring dims of head h of group g, row j, as bf16; + 0 makes one zero of both.
__device__ __forceinline__ void put_out(const StrideWindowAttentionParams& p, int j, int g, int h, int d, f32x4 acc, float sum) {
  const int idx = (g * p.n_q + h) * p.head_dim + d;
  uint16_t* at = p.out + (static_cast<int64_t>(j >> 4) * (p.out_cols >> 4) + (idx >> 4)) * kTileElems + (j & 15) * 16 + (idx & 15);
  f32x4 v = {0, 0, 0, 0};
  if (!(sum == 0.0f)) {
    const float r = 1.0f / sum;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = acc[e] * r + 0.0f;
  }
  *reinterpret_cast<u32x2*>(at) = u32x2{pack2(v[0], v[1]), pack2(v[2], v[3])};
}

// A split row's leaf record: acc [n_q][D], then (reference, l) per head.
__device__ __forceinline__ int record_floats(int n_q, int d) { return (n_q * (d + 2) + 3) / 4 * 4; }

// ---------------------------------------------------------------------------
// Rows one by one: a workgroup has a row and a KV group, its heads are the columns of the
// matrix products. Wave w scores chunk w of a leaf (keys straight from memory: the 16 x 32
// operand is 16 rows of 64 bytes), the four maxima give every wave the leaf's references,
// the weights go through LDS, and each wave sums its quarter of the dims over the leaf. The
// next leaf's loads are in flight meanwhile. Memory bounds it: 128 rows of window 1024, 8 groups
// of 4 heads of 64, 57 us at 4.6 TB/s, whole contexts of 4000 at 6.1 (a 4 GiB copy: 4.8).
// SPLIT: a leaf, or at head_dim 128 `each` leaves, a workgroup, their records to scratch (few
// rows, long contexts).
template <int D, bool SPLIT>
__device__ __forceinline__ void one_row(const StrideWindowAttentionParams& p, int page_shift, int limit, int span, int g, int j, int begin, int each) {
  constexpr int kKey = D / 32;           // operands of a key row
  constexpr int kRow = D / 8;            // 16-byte pieces of a row
  constexpr int kPer = kChunk * kRow / 64;
  constexpr int kOut = (D + 63) / 64;    // 16-dim blocks of a wave
  // At head_dim 128 two leaves' registers would leave one workgroup a CU; two that take turns
  // loading do better (128 rows of 1024 positions, 8 groups: 82 us, and 187 with the next leaf's
  // loads in flight).
  constexpr bool kNext = !SPLIT && D < 128;
  __shared__ __align__(16) uint16_t vs[kLeaf * D];
  __shared__ __align__(16) u32x4 weights[kLeaf / 32][64];
  __shared__ float maxima[4][16];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, col = lane & 15, quarter = lane >> 4;
  const int slot = p.row_slot[j];
  const Sight sight = sight_of(p, pos_of(p, j), limit);
  const Leaves leaves = leaves_of(sight);
  const int end = !SPLIT ? leaves.count : D < 128 ? begin + 1 : min(begin + each, leaves.count);
  if (SPLIT && begin >= leaves.count) return;

  const uint16_t* base = static_cast<const uint16_t*>(p.kv.arena) + p.layer * p.kv.layer_elems + g * p.kv.group_elems;
  const int32_t* table = p.kv.table + static_cast<int64_t>(slot) * p.kv.max_blocks;
  const int in_page = (1 << page_shift) - 1;

  u32x4 kr[4][kKey], vr[kPer];
  int block;        // of position 64 * wave + lane of the leaf; below 0: not seen, or not held
  uint64_t seen;    // bit i: position 64 * wave + i is seen
  auto look = [&](int leaf) {
    const int t = leaf * kLeaf + wave * kChunk + lane;
    const bool s = sight.sees(t);
    block = s ? table[t >> page_shift] : -1;
    seen = __ballot(s);
  };
  const u32x4 zero = {0, 0, 0, 0};
  auto fetch_k = [&](int leaf) {
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int i = 16 * t + col, b = __shfl(block, i);
      const uint16_t* at = base + max(b, 0) * p.kv.block_elems + ((leaf * kLeaf + wave * kChunk + i) & in_page) * D + 8 * quarter;
#pragma unroll
      for (int k = 0; k < kKey; ++k) {
        kr[t][k] = load16(at + 32 * k);
        if (b < 0) kr[t][k] = zero;
      }
    }
  };
  auto fetch_v = [&](int leaf) {
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      const int piece = u * 64 + lane, i = piece / kRow, b = __shfl(block, i);
      vr[u] = ld_kv(base + p.kv.which_elems + max(b, 0) * p.kv.block_elems +
                    ((leaf * kLeaf + wave * kChunk + i) & in_page) * D + (piece % kRow) * 8);
      if (b < 0) vr[u] = zero;
    }
  };

  u32x4 qh[kKey], ql[kKey];
  {
    const float* q = p.q + j * p.q_stride + (static_cast<int64_t>(g) * p.n_q + col) * D + 8 * quarter;
#pragma unroll
    for (int k = 0; k < kKey; ++k) split_query(q + 32 * k, p.scale * kLog2e, col < p.n_q, qh[k], ql[k]);
  }

  f32x4 total[kOut];
#pragma unroll
  for (int b = 0; b < kOut; ++b) total[b] = f32x4{0, 0, 0, 0};
  Fold fold = {neg_inf(), 0.0f};

  if (kNext && begin < end) {
    look(leaves.at(begin));
    fetch_k(leaves.at(begin));
    fetch_v(leaves.at(begin));
  }
  for (int it = begin; it < end; ++it) {
    if constexpr (!kNext) {
      look(leaves.at(it));
      fetch_k(leaves.at(it));
      fetch_v(leaves.at(it));
    }
    f32x4 s[4];
    float most = neg_inf();
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      s[t] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < kKey; ++k) {
        s[t] = mfma(kr[t][k], qh[k], s[t]);
        s[t] = mfma(kr[t][k], ql[k], s[t]);
      }
    }
    const uint64_t mine = seen;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (!((mine >> (16 * t + 4 * quarter + e)) & 1)) s[t][e] = neg_inf();
        most = fmaxf(most, s[t][e]);
      }
    most = fmaxf(most, __shfl_xor(most, 16));
    most = fmaxf(most, __shfl_xor(most, 32));
    if (lane < 16) maxima[wave][lane] = most;
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      const int piece = u * 64 + lane;
      *reinterpret_cast<u32x4*>(vs + v_at<D>(wave * kChunk + piece / kRow, (piece % kRow) * 8)) = vr[u];
    }
    if (kNext && it + 1 < end) look(leaves.at(it + 1));
    lds_barrier();
    if (kNext && it + 1 < end) {
      fetch_k(leaves.at(it + 1));
      fetch_v(leaves.at(it + 1));
    }
    // the leaf's references, the same in every wave
    float ref = neg_inf(), own_ref = neg_inf(), alpha[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const float m = maxima[c][col];
      alpha[c] = 1.0f;
      if (m > ref + kSlack) {
        alpha[c] = exp2_of(ref - m);
        ref = m;
      }
      if (c == wave) own_ref = ref;
    }
    const float at = own_ref == neg_inf() ? 0.0f : own_ref;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      u32x4 w;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const f32x4 v = s[2 * half + x];
        w[2 * x] = pack2(exp2_of(v[0] - at), exp2_of(v[1] - at));
        w[2 * x + 1] = pack2(exp2_of(v[2] - at), exp2_of(v[3] - at));
      }
      weights[2 * wave + half][lane] = w;
    }
    lds_barrier();
    f32x4 acc[kOut], l = {0, 0, 0, 0};
#pragma unroll
    for (int b = 0; b < kOut; ++b) acc[b] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int c = 0; c < 4; ++c) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        l[e] *= alpha[c];
#pragma unroll
        for (int b = 0; b < kOut; ++b) acc[b][e] *= alpha[c];
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const u32x4 w = weights[2 * c + half][lane];
        const int row = c * kChunk + 32 * half + 4 * quarter + (col >> 2);
        l = mfma(u32x4{kOnes, kOnes, kOnes, kOnes}, w, l);
#pragma unroll
        for (int b = 0; b < kOut; ++b) {
          const int dim = (wave * kOut + b) * 16;
          if (dim < D)
            acc[b] = mfma(both(read_transposed(vs + v_at<D>(row, dim + 4 * (col & 3))),
                               read_transposed(vs + v_at<D>(row + 16, dim + 4 * (col & 3)))),
                          w, acc[b]);
        }
      }
    }
    if constexpr (SPLIT) {
      if (col < p.n_q) {
        float* rec = p.scratch + ((static_cast<int64_t>(j) * p.n_kv + g) * span + it) * record_floats(p.n_q, D);
#pragma unroll
        for (int b = 0; b < kOut; ++b) {
          const int dim = (wave * kOut + b) * 16 + 4 * quarter;
          if (dim < D) *reinterpret_cast<f32x4*>(rec + col * D + dim) = acc[b];
        }
        if (threadIdx.x < 16) *reinterpret_cast<f32x2*>(rec + p.n_q * D + 2 * col) = f32x2{ref, l[0]};
      }
    } else {
      float a, b;
      fold.take(ref, l[0], a, b);
#pragma unroll
      for (int x = 0; x < kOut; ++x) total[x] = folded(total[x], acc[x], a, b);
    }
    if (it + 1 < end) lds_barrier();  // the staging is written again
  }
  if (!SPLIT && col < p.n_q) {
#pragma unroll
    for (int b = 0; b < kOut; ++b) {
      const int dim = (wave * kOut + b) * 16 + 4 * quarter;
      if (dim < D) put_out(p, j, g, col, dim, total[b], fold.sum);
    }
  }
}

template <int D>
__global__ __launch_bounds__(256, 2) void k_leaves(StrideWindowAttentionParams p, int page_shift, int limit, int span, const int32_t* done,
                                                   int tile_rows, int parts, int each, int stretches) {
  const int unit = blockIdx.x / p.n_kv, g = blockIdx.x % p.n_kv, j = unit / stretches, at = unit % stretches * (D < 128 ? 1 : each);
  if (done) {
    const Leaves leaves = leaves_of(sight_of(p, pos_of(p, j), limit));
    if (at >= leaves.count || done[(j / tile_rows * p.n_kv + g) * parts + leaves.at(at) % parts]) return;
  }
  one_row<D, true>(p, page_shift, limit, span, g, j, at, each);
}

// A workgroup a unit (row, group); with tiles that k_tile may have done (done: its marks), a
// workgroup looks at up to 256 units, spread over the batch, and takes those that are left.
__device__ __forceinline__ bool unit_done(const StrideWindowAttentionParams& p, int unit, int limit, const int32_t* done, int tile_rows,
                                          int parts) {
  const int j = unit / p.n_kv, tile = j / tile_rows;
  const int32_t* mark = done + (tile * p.n_kv + unit % p.n_kv) * parts;
  bool same = true;
  for (int i = 1; i < parts; ++i) same &= mark[i] == mark[0];
  if (same) return mark[0];
  int run = 0;  // the row's, in its tile
  for (int i = tile * tile_rows + 1; i <= j; ++i)
    run += !one_run(p.row_slot[i - 1], min(pos_of(p, i - 1), limit - 1), p.row_slot[i], min(pos_of(p, i), limit - 1), p.window);
  return mark[run % parts];
}
template <int D>
__global__ __launch_bounds__(256, 2) void k_rows(StrideWindowAttentionParams p, int page_shift, int limit, const int32_t* done, int tile_rows,
                                                 int parts) {
  if (!done) {
    one_row<D, false>(p, page_shift, limit, 0, blockIdx.x % p.n_kv, blockIdx.x / p.n_kv, 0, 0);
    return;
  }
  __shared__ uint64_t left[4];
  const int units = p.l.rows * p.n_kv, mine = threadIdx.x * gridDim.x + blockIdx.x;
  const uint64_t b = __ballot(mine < units && !unit_done(p, mine, limit, done, tile_rows, parts));
  if ((threadIdx.x & 63) == 0) left[threadIdx.x >> 6] = b;
  __syncthreads();
#pragma unroll 1
  for (int w = 0; w < 4; ++w)
#pragma unroll 1
    for (uint64_t todo = left[w]; todo; todo &= todo - 1) {
      const int unit = __builtin_amdgcn_readfirstlane((w * 64 + __builtin_ctzll(todo)) * static_cast<int>(gridDim.x) + static_cast<int>(blockIdx.x));
      one_row<D, false>(p, page_shift, limit, 0, unit % p.n_kv, unit / p.n_kv, 0, 0);
      lds_barrier();  // every wave has read the unit's staging and weights: the next unit writes there
    }
}

// ---------------------------------------------------------------------------
// Prompts: a workgroup has a tile of 128 score columns, (row, head) pairs of neighbouring
// rows, and a KV group, so that keys and values are fetched once for all of them. Eight waves
// of 16 columns each, v_mfma_f32_16x16x32_bf16, the transposed product first: S^T = K Q^T
// leaves a column's scores in four lanes, so that references, weights and sums are lane-local,
// and S^T's registers are P^T's operand as they are, with the value rows taken in the same
// order. (Waves of 32 columns and the 32x32x16 form halve the LDS reads, but leave one wave a
// SIMD at head_dim 128: 2048 rows of window 1984 195 us against 155, and 84 against 80 at 64.)
//
// C chunks at a time, a span. With two, a wave has two of each latency's work between two
// barriers; with one, at head_dim 64, two workgroups fit on a CU (128 registers) and fill each
// other's waits. So two at head_dim 128, or where there is at most a workgroup a CU (1024 rows
// of one sequence at 8192, 8 groups, head_dim 64: 155 us against 169; 4096 rows: 451 against
// 335). Spans are copied memory -> LDS one (C = 2) or two (C = 1) ahead. Key rows have their
// 16-byte pieces permuted by the row and value rows their 32-byte blocks, so that an operand
// read spreads over the banks; the copy lands in order, so its source is permuted.
//
// SPLIT: few rows over a long context. A workgroup has the leaves of its tile that are its
// number modulo `parts`, each leaf's sums go to the columns' rows as records, and k_join joins
// them (64 rows at 8192 positions, 8 groups, head_dim 64: 139 us otherwise, 45 so). There a
// workgroup takes part in all of its tile's runs, one after the other.
//
// Rows of several sequences meet in a tile where prompts end, or rows of one whose windows do
// not touch (one_run). `parts` workgroups take its runs in turn, each column taking part in its own; a wave without a column of the run only helps
// with the copies (64 prompts of 8 rows at 1024 positions, head_dim 64: 37 us; 62 with two parts
// always, 74 with such waves in the products too; the rows alone 140). A tile of many short runs
// is left to k_rows, and so is a part in which a row's sums are not finite: a column that must
// not see a value gives it the weight 0, and 0 times an infinity or NaN is NaN. (Looking for such
// values in every span that not all columns see took a barrier more: 2048 rows of window 448 29.0
// us against 28.0, head_dim 128 62.9 against 60.3.) done[(tile * n_kv + g) * parts + part]:
// whether it was done; with SPLIT, part = leaf % parts, otherwise run % parts.
constexpr int kColumns = 128;
constexpr int kRunRows = 4;  // rows a run, on average, below which a tile is left to k_rows

template <int D>
struct Lay {
  static constexpr int kRow = D / 8;  // 16-byte pieces of a row
  // what the row adds to a key's piece and a value's block of two
  __device__ static __forceinline__ int k_turn(int row) { return (row * D / 128) & (kRow - 1); }
  __device__ static __forceinline__ int v_turn(int row) { return (row * D / 128) & (kRow / 2 - 1); }
  __device__ static __forceinline__ int k_at(int row, int piece) { return row * D + ((piece ^ k_turn(row)) << 3); }
  __device__ static __forceinline__ int v_at(int row, int dim) { return row * D + (((dim >> 4) ^ v_turn(row)) << 4) + (dim & 15); }
  // the piece that slot `at` of a row gets
  __device__ static __forceinline__ int k_from(int row, int at) { return at ^ k_turn(row); }
  __device__ static __forceinline__ int v_from(int row, int at) { return (((at >> 1) ^ v_turn(row)) << 1) + (at & 1); }
};

// The maximum over the four lanes of a column (16 apart): the row swaps leave a lane's own and
// its partner's value.
__device__ __forceinline__ float column_max(float m) {
  const auto a = __builtin_amdgcn_permlane16_swap(u32_of(m), u32_of(m), false, false);
  m = fmaxf(f32_of(a[0]), f32_of(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(u32_of(m), u32_of(m), false, false);
  return fmaxf(f32_of(b[0]), f32_of(b[1]));
}

// The largest over a wave, in every lane: DPP within rows of 16, then the row swaps.
template <int CTRL>
__device__ __forceinline__ int larger_by(int v) {
  return max(v, __builtin_amdgcn_update_dpp(v, v, CTRL, 0xF, 0xF, false));
}
__device__ __forceinline__ int wave_most(int v) {
  v = larger_by<0xB1>(v);   // quad_perm [1,0,3,2]
  v = larger_by<0x4E>(v);   // quad_perm [2,3,0,1]
  v = larger_by<0x124>(v);  // row_ror:4
  v = larger_by<0x128>(v);  // row_ror:8
  const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = max(static_cast<int>(a[0]), static_cast<int>(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return __builtin_amdgcn_readfirstlane(max(static_cast<int>(b[0]), static_cast<int>(b[1])));
}

__device__ __align__(16) uint32_t zeros16[4];  // what unseen and unheld positions are copied from

// 64 lanes' 16 bytes each, memory -> LDS, in lane order from `to`. Written as assembly because
// the compiler, not knowing which buffer a transposing read reads, would have every such read
// wait for all copies under way; the kernel waits for them itself. The instruction has no
// register that it writes. The second form takes a base for the wave and a byte offset a lane.
__device__ __forceinline__ void copy_to_lds(const uint16_t* from, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(from) : "memory", "m0");
}
__device__ __forceinline__ void copy_to_lds(const uint16_t* base, uint32_t offset, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(offset), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ uint32_t lds_offset(const void* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const void*)(p)));
}

template <int D, int C, bool SPLIT>
__global__ __launch_bounds__(512, C == 2 ? 2 : 4) void k_tile(StrideWindowAttentionParams p, int page_shift, int limit, int tile_rows, int32_t* done,
                                                              int span, int parts) {
  using L = Lay<D>;
  constexpr int kWaves = kColumns / 16;
  constexpr int kSpan = C * kChunk;
  constexpr int kBufs = C == 2 ? 2 : 3;
  constexpr int kPer = kSpan * L::kRow / 64 / kWaves;  // copies of K (and of V) a wave makes
  static_assert(kPer > 0, "every wave copies");
  constexpr int kDims = D / 16;
  __shared__ __align__(16) uint16_t ks[kBufs][kSpan * D];
  __shared__ __align__(16) uint16_t vs[kBufs][kSpan * D];
  __shared__ int slots[kColumns], poss[kColumns];
  __shared__ uint64_t starts[2];  // bit i: row i begins a run
  __shared__ int spoiled;  // some row's sums are not finite
  const int t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63, cl = lane & 15, quarter = lane >> 4;
  // A tile's later runs first: most of their workgroups only leave, and a pass over a context of
  // its own begins late otherwise (6 prompts of 300 rows at 400 to 4000 positions, head_dim 64 /
  // 128: 95 / 164 us, 99 / 197 the other way; 3 of 333 rows at 3001, 2000, 1000 80 / 120 and 65 /
  // 98, at 1000, 2000, 3001 65 / 98 and 73 / 111). All of them, not in turn with the others, which
  // left whole CUs idle. Then later rows, which see more, before earlier ones.
  const int tiles = gridDim.x / p.n_kv / parts, unit = blockIdx.x / p.n_kv;
  const int g = blockIdx.x % p.n_kv, part = SPLIT ? unit / tiles : parts - 1 - unit / tiles, tile = tiles - 1 - unit % tiles;
  const int j0 = tile * tile_rows, nr = min(tile_rows, p.l.rows - j0);
  int32_t* mark = done + (tile * p.n_kv + g) * parts + part;

  if (t == 0) spoiled = 0;
  if (t < kColumns) {
    const int j = j0 + min(t, nr - 1);
    slots[t] = p.row_slot[j];
    poss[t] = t < nr ? min(pos_of(p, j), limit - 1) : -1;
  }
  __syncthreads();
  if (t < kColumns) {
    const uint64_t b = __ballot(t < nr && (t == 0 || !one_run(slots[t - 1], poss[t - 1], slots[t], poss[t], p.window)));
    if (lane == 0) starts[wave] = b;
  }
  __syncthreads();
  const uint64_t first = starts[0], second = starts[1];
  const int runs = __popcll(first) + __popcll(second);
  const bool left = nr < kRunRows * runs;
  if (left || (!SPLIT && runs <= part)) {
    if (t == 0) *mark = left ? 0 : 1;
    return;
  }
  // the row after row r at which another run begins
  auto next_run = [&](int r) {
    const uint64_t lo = r < 63 ? first & (~uint64_t{0} << (r + 1)) : 0;
    const uint64_t hi = r < 63 ? second : (r < 127 ? second & (~uint64_t{0} << (r + 1 - 64)) : 0);
    return lo ? __builtin_ctzll(lo) : (hi ? 64 + __builtin_ctzll(hi) : nr);
  };

  // this lane's column
  const int col = wave * 16 + cl, row = col / p.n_q, head = col - row * p.n_q;
  const bool live = row < nr;
  const int my_pos = live ? poss[row] : -1;
  const Sight sight = sight_of(p, my_pos, limit);
  u32x4 qh[D / 32], ql[D / 32];
  const uint16_t* base = static_cast<const uint16_t*>(p.kv.arena) + p.layer * p.kv.layer_elems + g * p.kv.group_elems;
  const int in_page = (1 << page_shift) - 1;
  f32x4 total[kDims];
#pragma unroll
  for (int d = 0; d < kDims; ++d) total[d] = f32x4{0, 0, 0, 0};
  Fold fold = {neg_inf(), 0.0f};

  const uint16_t* zero = reinterpret_cast<const uint16_t*>(zeros16);
  asm("" : "+s"(zero));  // kept, not looked up again for each copy
  // a lane's bytes in a copy, from the first of its rows
  uint32_t k_off[kPer], v_off[kPer];
#pragma unroll
  for (int u = 0; u < kPer; ++u) {
    const int at = (wave * kPer + u) * 64, r = (at + lane) / L::kRow, slot_in = (at + lane) % L::kRow;
    k_off[u] = (lane / L::kRow * D + L::k_from(r, slot_in) * 8) * 2;
    v_off[u] = (lane / L::kRow * D + L::v_from(r, slot_in) * 8) * 2;
  }

  bool spoil = false;
  bool taken = false;  // has this lane's column been in a run of this part's?
  int turn = SPLIT ? 0 : part;
  for (int r0 = 0, r1; r0 < nr; r0 = r1) {
    r1 = next_run(r0);
    if (!SPLIT && turn-- != 0) continue;
    turn = parts - 1;
    // the run [r0, r1): its sequence, and what its rows see together
    int low = INT_MAX, high = -1;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int r = lane + 64 * x, pos = poss[r];
      if (r >= r0 && r < r1 && pos >= 0) {
        low = min(low, pos);
        high = max(high, pos);
      }
    }
    low = -1 - wave_most(-1 - low);
    high = wave_most(high);
    const bool mine = row >= r0 && row < r1;
    taken |= mine;
    const int slot = __builtin_amdgcn_readfirstlane(slots[r0]);
    if (high < 0) continue;
    const Sight near = sight_of(p, low, limit), far = sight_of(p, high, limit);
    // spans: [0, all_head) and [all_rest, all_last]
    const int all_head = (far.sink_end + kSpan - 1) / kSpan, all_rest = max(near.lo / kSpan, all_head), all_last = high / kSpan;
    const auto table = (const __attribute__((address_space(4))) int32_t*)(p.kv.table + static_cast<int64_t>(slot) * p.kv.max_blocks);
    // One pass over all of them, or over the workgroup's leaves one by one: the spans
    // [0, head_spans) and those from `rest` on, `spans` in all.
    for (int part_leaf = SPLIT ? part : 0; part_leaf <= (SPLIT ? high / kLeaf : 0); part_leaf += SPLIT ? parts : 1) {
      int head_spans = all_head, rest = all_rest, last = all_last;
      if constexpr (SPLIT) {
        // from the first to the last span of the leaf that a row sees
        head_spans = 0, rest = part_leaf * (kLeaf / kSpan), last = min(rest + kLeaf / kSpan - 1, all_last);
        if (rest >= all_head) rest = max(rest, all_rest);
        if (last < all_rest) last = min(last, all_head - 1);
        if (rest > last) continue;
      }
      const int spans = head_spans + max(0, last - rest + 1);
      auto span_at = [&](int i) { return i < head_spans ? i : rest + i - head_spans; };

      // Table entries one span ahead of the copies, which are kBufs - 1 ahead of the products. A
      // copy's rows lie in one page, so its entry comes through the scalar cache. Past the last
      // span it is copied again, so that the waits can count.
      int block[kPer];
      auto look = [&](int i) {
        const int c = span_at(min(i, spans - 1)) * kSpan;
#pragma unroll
        for (int u = 0; u < kPer; ++u) {
          // an entry that no row sees is not looked at: the run's own last one stands for it
          const int a = c + (wave * kPer + u) * 64 / L::kRow, z = a + 64 / L::kRow - 1;
          const bool s = a <= high && (z >= near.lo || a < far.sink_end);
          block[u] = table[__builtin_amdgcn_readfirstlane((s ? a : high) >> page_shift)];
        }
      };
      auto copy = [&](int i, int buf) {
        const int c = span_at(min(i, spans - 1)) * kSpan;
        // Does some row see each position? Then a lane's place in a copy's page is all it needs.
        const bool inside = c + kSpan - 1 <= high && (c >= near.lo || c + kSpan <= far.sink_end);
#pragma unroll
        for (int u = 0; u < kPer; ++u) {
          const int at = (wave * kPer + u) * 64, row0 = at / L::kRow;
          const uint16_t* page = base + block[u] * p.kv.block_elems + ((c + row0) & in_page) * D;
          const uint32_t k_to = lds_offset(&ks[buf][at * 8]), v_to = lds_offset(&vs[buf][at * 8]);
          if (inside && block[u] >= 0) {
            copy_to_lds(page, k_off[u], k_to);
            copy_to_lds(page + p.kv.which_elems, v_off[u], v_to);
          } else {
            const int pos = c + row0 + lane / L::kRow;
            const bool seen = block[u] >= 0 && pos <= high && (pos >= near.lo || pos < far.sink_end);
            copy_to_lds(seen ? page + k_off[u] / 2 : zero, k_to);
            copy_to_lds(seen ? page + p.kv.which_elems + v_off[u] / 2 : zero, v_to);
          }
        }
      };
#pragma unroll
      for (int x = 0; x < kBufs - 1; ++x) {
        look(x);
        copy(x, x);
      }
      look(kBufs - 1);
      {  // beside the first copies
        const float* q = p.q + (j0 + (live ? row : 0)) * p.q_stride + (static_cast<int64_t>(g) * p.n_q + head) * D + 8 * quarter;
#pragma unroll
        for (int k = 0; k < D / 32; ++k) split_query(q + 32 * k, p.scale * kLog2e, live, qh[k], ql[k]);
      }
      // do all of the run's columns see all of the span from a?
      auto is_full = [&](int a) __attribute__((always_inline)) {
        return a + kSpan - 1 <= low && (a >= far.lo || a + kSpan <= near.sink_end);
      };
      // Waits until span i has arrived, and every wave has read the one before, whose buffer is
      // filled next (the copies of the next may be under way).
      auto arrived = [&]() __attribute__((always_inline)) {
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"((kBufs - 2) * 2 * kPer) : "memory");
        lds_barrier();
      };
      int buf = 0, i = 0;
      // a wave without a column of this run only helps with the copies
      if (!__any(mine))
        for (; i < spans; ++i) {
          arrived();
          copy(i + kBufs - 1, buf == 0 ? kBufs - 1 : buf - 1);
          look(i + kBufs);
          buf = buf == kBufs - 1 ? 0 : buf + 1;
        }
      while (i < spans) {
        const int leaf = span_at(i) / (kLeaf / kSpan);
        f32x4 acc[kDims], l = {0, 0, 0, 0};
        float ref = neg_inf();
#pragma unroll
        for (int d = 0; d < kDims; ++d) acc[d] = f32x4{0, 0, 0, 0};
        do {
          const int a = span_at(i) * kSpan;
          const bool full = is_full(a);
          arrived();
          copy(i + kBufs - 1, buf == 0 ? kBufs - 1 : buf - 1);
          look(i + kBufs);
          __builtin_amdgcn_s_setprio(1);
          f32x4 s[4 * C];
#pragma unroll
          for (int b = 0; b < 4 * C; ++b) {
            s[b] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < D / 32; ++k) {
              const u32x4 key = *reinterpret_cast<const u32x4*>(&ks[buf][L::k_at(16 * b + cl, 4 * k + quarter)]);
              s[b] = mfma(key, qh[k], s[b]);
              s[b] = mfma(key, ql[k], s[b]);
            }
          }
          __builtin_amdgcn_s_setprio(0);
          // register e of block b is position 16 b + 4 quarter + e of the span
          if (!full) {
            const int from = a + 4 * quarter;
            if (a >= far.sink_end) {
              const bool some = mine && sight.pos >= sight.lo;
              const uint32_t wide = some ? sight.pos - sight.lo : 0;
              const int shift = some ? from - sight.lo : INT_MIN / 2;  // far below: unseen
#pragma unroll
              for (int b = 0; b < 4 * C; ++b)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (static_cast<uint32_t>(shift + 16 * b + e) > wide) s[b][e] = neg_inf();
            } else {
#pragma unroll
              for (int b = 0; b < 4 * C; ++b)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (!(mine && sight.sees(from + 16 * b + e))) s[b][e] = neg_inf();
            }
          }
          float most[C];
#pragma unroll
          for (int h = 0; h < C; ++h) {
            most[h] = s[4 * h][0];
#pragma unroll
            for (int b = 0; b < 4; ++b)
#pragma unroll
              for (int e = 0; e < 4; ++e) most[h] = fmaxf(most[h], s[4 * h + b][e]);
            most[h] = column_max(most[h]);
          }
#pragma unroll
          for (int h = 0; h < C; ++h) {
            if (__any(most[h] > ref + kSlack)) {
              const bool up = most[h] > ref + kSlack;
              const float alpha = up ? exp2_of(ref - most[h]) : 1.0f;
              if (up) ref = most[h];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                l[e] *= alpha;
#pragma unroll
                for (int d = 0; d < kDims; ++d) acc[d][e] *= alpha;
              }
            }
            // value operands of 32 positions; the first half's are read beside the exponentials, the
            // second's beside the first's products
            u32x4 v[2][kDims];
            auto read = [&](int x) __attribute__((always_inline)) {
              const int r = 64 * h + 32 * x + 4 * quarter + (cl >> 2);
#pragma unroll
              for (int d = 0; d < kDims; ++d) {
                const int dim = 16 * d + 4 * (lane & 3);
                v[x][d] = both(read_transposed(&vs[buf][L::v_at(r, dim)]), read_transposed(&vs[buf][L::v_at(r + 16, dim)]));
              }
              __builtin_amdgcn_sched_barrier(0);
            };
            read(0);
            const float at = ref == neg_inf() ? 0.0f : ref;
            u32x4 pw[2];
#pragma unroll
            for (int b = 0; b < 4; ++b) {
              const f32x4 z = s[4 * h + b];
              pw[b >> 1][2 * (b & 1)] = pack2(exp2_of(z[0] - at), exp2_of(z[1] - at));
              pw[b >> 1][2 * (b & 1) + 1] = pack2(exp2_of(z[2] - at), exp2_of(z[3] - at));
            }
            read(1);
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              l = mfma(u32x4{kOnes, kOnes, kOnes, kOnes}, pw[x], l);
#pragma unroll
              for (int d = 0; d < kDims; ++d) acc[d] = mfma(v[x][d], pw[x], acc[d]);
            }
            __builtin_amdgcn_s_setprio(0);
          }
          buf = buf == kBufs - 1 ? 0 : buf + 1;
          ++i;
        } while (i < spans && span_at(i) / (kLeaf / kSpan) == leaf);
        if constexpr (SPLIT) {
          const Leaves sees = leaves_of(sight);
          const int at = leaf < sees.head ? leaf : (leaf >= sees.rest ? sees.head + leaf - sees.rest : sees.count);
          float check = 0.0f;  // NaN where a sum is not finite
#pragma unroll
          for (int d = 0; d < kDims; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) check = __builtin_fmaf(acc[d][e], 0.0f, check);
          spoil |= mine && !(check == 0.0f);
          if (live && mine && at < sees.count) {
            float* rec = p.scratch + ((static_cast<int64_t>(j0 + row) * p.n_kv + g) * span + at) * record_floats(p.n_q, D);
#pragma unroll
            for (int d = 0; d < kDims; ++d) *reinterpret_cast<f32x4*>(rec + head * D + 16 * d + 4 * quarter) = acc[d];
            if (quarter == 0) *reinterpret_cast<f32x2*>(rec + p.n_q * D + 2 * head) = f32x2{ref, l[0]};
          }
        } else {
          // (other runs' columns took part with what they do not see)
          float fa, fb;
          fold.take(mine ? ref : neg_inf(), mine ? l[0] : 0.0f, fa, fb);
#pragma unroll
          for (int d = 0; d < kDims; ++d) total[d] = folded(total[d], mine ? acc[d] : f32x4{0, 0, 0, 0}, fa, fb);
        }
      }
      // nothing is on its way to the buffers, and every wave has read them, when another pass comes
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      lds_barrier();
    }
  }
  if constexpr (!SPLIT) {  // (what is not finite stays so through the fold)
    float check = 0.0f;
#pragma unroll
    for (int d = 0; d < kDims; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e) check = __builtin_fmaf(total[d][e], 0.0f, check);
    spoil = taken && !(check == 0.0f);
  }
  if (!SPLIT && live && taken) {
    const float sum = my_pos < 0 ? 0.0f : fold.sum;
#pragma unroll
    for (int d = 0; d < kDims; ++d) put_out(p, j0 + row, g, head, 16 * d + 4 * quarter, total[d], sum);
  }
  if (__any(spoil) && lane == 0) spoiled = 1;
  lds_barrier();
  if (t == 0) *mark = spoiled ? 0 : 1;
}

// Joins a split row's records in ascending order. The factors of a head's leaves follow from
// the references' running maximum, which a wave finds for 64 leaves at once; what is left in
// order is one product and one FMA a leaf and value, a thread a value, with the values of up to
// 32 records on their way. (4 rows of 128 leaves at 8 heads of 128: 10.5 us; 17.8 with the
// factors formed leaf by leaf in every thread.)
template <int D>
__global__ __launch_bounds__(256) void k_join(StrideWindowAttentionParams p, int limit, int span, int parts) {
  constexpr int kHeads = 256 / D;  // of a workgroup
  constexpr int kBlock = 256;      // leaves whose factors are in LDS
  __shared__ f32x4 factor[kHeads][kBlock];  // a, b, l
  const int t = threadIdx.x, wave = t >> 6, lane = t & 63;
  const int part = blockIdx.x % parts, unit = blockIdx.x / parts, g = unit % p.n_kv, j = unit / p.n_kv;
  const int count = leaves_of(sight_of(p, pos_of(p, j), limit)).count;
  const int rf = record_floats(p.n_q, D);
  const float* recs = p.scratch + (static_cast<int64_t>(j) * p.n_kv + g) * span * rf;
  const int mine = t / D, h = part * kHeads + mine;  // a wave's values are of one head, or, at D = 32, of two
  float total = 0.0f, sum = 0.0f;
  const float* values = recs + min(h, p.n_q - 1) * D + t % D;
  // running reference of head part * kHeads + wave + 4 k, the same in all lanes of its wave
  float run[(kHeads + 3) / 4];
  bool any[(kHeads + 3) / 4];  // has a leaf had weights
#pragma unroll
  for (int k = 0; k < (kHeads + 3) / 4; ++k) run[k] = neg_inf(), any[k] = false;
  for (int i0 = 0; i0 < count; i0 += kBlock) {
    const int n = min(kBlock, count - i0);
#pragma unroll
    for (int k = 0; k < (kHeads + 3) / 4; ++k) {
      const int head = wave + 4 * k;
      if (head >= kHeads) continue;
      const float* rl = recs + static_cast<int64_t>(i0) * rf + p.n_q * D + 2 * min(part * kHeads + head, p.n_q - 1);
      for (int i = 0; i < n; i += 64) {
        const int at = min(i + lane, n - 1);
        const f32x2 v = *reinterpret_cast<const f32x2*>(rl + static_cast<int64_t>(at) * rf);
        const bool has = i + lane < n && !(v[1] == 0.0f);
        float m = has ? v[0] : neg_inf();
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
          const float o = __shfl_up(m, d);
          if (lane >= d && o > m) m = o;
        }
        if (run[k] > m) m = run[k];
        float before = __shfl_up(m, 1);
        if (lane == 0) before = run[k];
        const uint64_t all = __ballot(has);
        const bool first = !any[k] && (all & ((uint64_t{1} << lane) - 1)) == 0;
        // (behind the last leaf, too, up to where values are read in one go: nothing changes there)
        factor[head][i + lane] = has ? f32x4{first ? 0.0f : exp2_of(before - m), exp2_of(v[0] - m), v[1], 0} : f32x4{1, 0, 0, 0};
        run[k] = __shfl(m, 63);
        any[k] = any[k] || all;
      }
    }
    __syncthreads();
    const float* at = values + static_cast<int64_t>(i0) * rf;
    auto take = [&](auto ahead) __attribute__((always_inline)) {
      constexpr int A = decltype(ahead)::value;
      for (int i = 0; i < n; i += A) {
        float v[A];
#pragma unroll
        for (int x = 0; x < A; ++x) v[x] = at[static_cast<int64_t>(min(i + x, n - 1)) * rf];
        __builtin_amdgcn_sched_barrier(0);  // all of them before the first is used
#pragma unroll
        for (int x = 0; x < A; ++x) {
          const f32x4 f = factor[mine][i + x];
          total = __builtin_fmaf(i + x < n ? v[x] : 0.0f, f[1], total * f[0]);  // (0 times an infinity is NaN)
          sum = __builtin_fmaf(f[2], f[1], sum * f[0]);
        }
      }
    };
    if (n <= 8) take(std::integral_constant<int, 8>{});
    else take(std::integral_constant<int, 32>{});
    __syncthreads();
  }
  // four neighbouring values to the lane of the first
  f32x4 v;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = __shfl(total, (lane & ~3) + e);
  if (h < p.n_q && (t & 3) == 0) put_out(p, j, g, h, t % D, v, sum);
}

// ---------------------------------------------------------------------------
// Host side.

struct Plan {
  int page_shift, limit, span;
  int tile_rows;  // 0: no tiles
  int parts;      // marks of a tile and group
  int64_t runs;   // of tiles and groups together, about
  bool split;
  int64_t records, scratch;  // floats; the tiles' marks come behind the records
};

const char* plan_of(const StrideWindowAttentionParams& p, Plan& plan) {
  const int D = p.head_dim;
  if (p.l.rows < 0 || p.l.lane_groups != (static_cast<int64_t>(p.l.rows) + 15) / 16) return "need rows >= 0 and lane_groups = ceil(rows/16)";
  if ((D != 32 && D != 64 && D != 128) || p.kv.head_dim != D) return "head_dim must be 32, 64 or 128 and match kv.head_dim";
  if (p.n_q < 1 || p.n_q > 16) return "1 to 16 query heads per KV head";
  if (p.n_kv < 1 || p.layer < 0 || p.max_pages < 1 || p.sinks < 0 || p.runs < 0 || p.kv.max_blocks < 1)
    return "bad n_kv, layer, max_pages, sinks, runs or max_blocks";
  const int64_t tokens = p.kv.group_elems > 0 && p.kv.group_elems % D == 0 ? p.kv.group_elems / D : 0;
  if (tokens < 8 || (tokens & (tokens - 1)) || tokens > (int64_t{1} << 30)) return "the KV page (group_elems / head_dim) must be a power of two from 8 up";
  if (p.kv.group_elems > int64_t{1} << 31) return "a head's part of a page must not pass 2^31 elements";  // a row's place in it has 32 bits
  if (p.kv.block_elems % 8 || p.kv.layer_elems % 8 || p.kv.which_elems % 8) return "KV strides must be multiples of 8 elements";
  const int64_t heads = static_cast<int64_t>(p.n_kv) * p.n_q * D;
  if (heads > INT_MAX || p.out_cols % 16 || p.out_cols < heads) return "out_cols must be a multiple of 16 covering every head";
  if (p.l.rows > 1 && (p.q_stride % 4 || p.q_stride < heads)) return "q_stride must be a multiple of 4 covering every head";
  plan.page_shift = 0;
  while ((int64_t{1} << plan.page_shift) < tokens) ++plan.page_shift;
  plan.limit = static_cast<int>(std::min<int64_t>(std::min<int64_t>(int64_t{64} * p.max_pages, tokens * p.kv.max_blocks), INT_MAX - kLeaf));
  // leaves that a row can see
  int64_t span = (static_cast<int64_t>(plan.limit) + kLeaf - 1) / kLeaf;
  if (p.window > 0) {
    const int64_t head = (std::min<int64_t>(p.sinks, plan.limit) + kLeaf - 1) / kLeaf, rest = (static_cast<int64_t>(p.window) + kLeaf - 2) / kLeaf + 1;
    span = std::min(span, head + rest);
  }
  plan.span = static_cast<int>(span);
  const int64_t units = static_cast<int64_t>(p.l.rows) * p.n_kv;
  if (units * span > INT_MAX) return "rows, n_kv and the context are too large together";
  // Tiles where neighbouring rows may be of one sequence (a tile's copies of 64 / (head_dim / 8)
  // rows lie in one page). Leaves in workgroups of their own, and joined, where the rows or
  // tiles alone would not fill the chip: below 512 workgroups of k_rows, or fewer where a row
  // has fewer than ten leaves, for the second launch (1, 8, 32, 63 rows, 8 groups, head_dim 64, split
  // and not, of 300 positions 11, 12, 12, 18 and 10, 10, 10, 12 us; of 1000 11, 11, 19, 29 and 15,
  // 15, 19, 24; of 2000 10, 12, 29, 45 and 26, 28, 34, 41); of tiles below 64, a
  // quarter of the CUs (192 rows of one sequence at 8192, 48 tiles, head_dim 64 / 128: 120 / 168
  // us against 148 / 228 in whole tiles; 256 rows, 64 tiles: 157 / 220 against 148 / 227), and
  // with eight leaves or more, for the records and two launches more (64 rows of 2000 positions:
  // 22 / 31 us against 44 / 66; of 600 positions 19 / 25 against 21 / 30, but 16 rows 16 / 19
  // against 12 / 15, and 200 rows 25 / 36 against 22 / 31).
  const int64_t records = units * span * ((p.n_q * (D + 2) + 3) / 4 * 4);
  const bool may_split = span > 1 && records <= int64_t{1} << 28;  // a GiB
  bool tiles = (p.runs == 0 || p.runs >= kRunRows) && p.l.rows >= kRunRows && tokens >= 512 / D;
  const int64_t rows_a_tile = kColumns / p.n_q, groups = (p.l.rows + rows_a_tile - 1) / rows_a_tile * p.n_kv;
  plan.split = may_split && tiles && p.runs > 0 && span >= 8 && groups < 64;
  if (!plan.split && may_split && units < (span < 3 ? 1 : span < 6 ? 256 : span < 10 ? 384 : 512)) plan.split = true, tiles = false;
  plan.tile_rows = tiles ? static_cast<int>(rows_a_tile) : 0;
  plan.parts = plan.split ? static_cast<int>(std::min<int64_t>((static_cast<int64_t>(plan.limit) + kLeaf - 1) / kLeaf, span + 1)) : 2;
  // As many parts as a tile may have runs, where the chip has room for them at once (128 prompts
  // of 8 rows at 1024 positions, head_dim 128, 256 tiles: 129 us with two parts, 146 with five).
  // One where the rows look like one sequence's, for the workgroups that only leave again.
  const bool one = p.runs >= p.l.rows;
  if (one && !plan.split) {
    plan.parts = 1;
  } else if (tiles && !plan.split) {
    const int most = plan.tile_rows / kRunRows, room = static_cast<int>((D < 128 ? 1024 : 512) / groups);
    plan.parts = std::max(2, std::min(room, p.runs > 0 ? std::min(most, (plan.tile_rows - 1) / p.runs + 2) : most));
  }
  plan.runs = groups * std::max(1, p.runs > 0 ? plan.tile_rows / p.runs : 1);
  plan.records = plan.split ? records : 0;
  const int64_t marks = tiles ? groups * plan.parts : 0;
  if (marks > INT_MAX) return "rows, n_kv and the context are too large together";
  plan.scratch = plan.records + marks;
  return nullptr;
}

int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(static_cast<int>(e), std::string(what) + " launch failed: " + hipGetErrorString(e));
  return 0;
}

template <int D>
int run(const StrideWindowAttentionParams& p, const Plan& plan, hipStream_t st) {
  const int units = p.l.rows * p.n_kv;
  int32_t* done = plan.tile_rows ? reinterpret_cast<int32_t*>(p.scratch + plan.records) : nullptr;
  if (done) {
    const unsigned groups = static_cast<unsigned>(plan.scratch - plan.records);  // a mark each
    const dim3 grid(groups), block(512);
    auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, st, p, plan.page_shift, plan.limit, plan.tile_rows, done, plan.span, plan.parts); };
    if (plan.split) launch(k_tile<D, 2, true>);
    else if (D != 64 || plan.runs <= 256) launch(k_tile<D, 2, false>);
    else launch(k_tile<64, 1, false>);
    if (int rc = launched("window_attention (tiles)")) return rc;
  }
  const int tile_rows = std::max(1, plan.tile_rows);
  if (plan.split) {
    // At head_dim 128 a workgroup takes up to four leaves one after the other where that leaves
    // enough of them (63 rows of 16000 positions, 8 groups of 4 heads: 824 us leaf by leaf, 770
    // so; 4 rows of 32768, 8 heads a group: 114 and 110). At 64, 63 rows of 4000 take 87 and 88.
    const int64_t leaves = static_cast<int64_t>(units) * plan.span;
    const int each = D < 128 || done ? 1 : static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(4, leaves / 2048)));
    const int stretches = (plan.span + each - 1) / each;
    hipLaunchKernelGGL((k_leaves<D>), dim3(units * stretches), dim3(256), 0, st, p, plan.page_shift, plan.limit, plan.span, done, tile_rows, plan.parts, each, stretches);
    if (int rc = launched("window_attention (leaves)")) return rc;
    const int parts = (p.n_q * D + 255) / 256;
    hipLaunchKernelGGL((k_join<D>), dim3(units * parts), dim3(256), 0, st, p, plan.limit, plan.span, parts);
    return launched("window_attention (join)");
  }
  // With tiles most of the workgroups only find that nothing is left; the fewer where that is
  // likely for all of them (2048 rows of one sequence, window 512, head_dim 64: 30.1 us with 1024
  // of them and parts for two runs, 28.7 so; but 128 sequences of 2 rows that were left 85 us with
  // 1024 and 126 with 256).
  const int groups = done ? std::max(std::min(units, p.runs >= p.l.rows ? 256 : 1024), (units + 255) / 256) : units;
  hipLaunchKernelGGL((k_rows<D>), dim3(groups), dim3(256), 0, st, p, plan.page_shift, plan.limit, done, tile_rows, plan.parts);
  return launched("window_attention");
}

}  // namespace
}  // namespace stride_tc

using namespace stride_tc;

static_assert(offsetof(StrideWindowAttentionParams, kv) == 40 && offsetof(StrideWindowAttentionParams, out_cols) == 128 &&
                  sizeof(StrideWindowAttentionParams) == 168,
              "WindowAttentionParams layout");

extern "C" {

int64_t stride_serve_window_attention_scratch(const StrideWindowAttentionParams* p) {
  Plan plan;
  if (!p || plan_of(*p, plan)) return -1;
  int64_t most = plan.scratch;
  if (p->runs == 0) {
    // What serves every hint. Hints below kRunRows plan alike, without tiles; from there on the
    // records do not depend on the hint and a tile's parts do not grow with it.
    StrideWindowAttentionParams hinted = *p;
    for (const int runs : {1, kRunRows}) {
      hinted.runs = runs;
      if (!plan_of(hinted, plan)) most = std::max(most, plan.scratch);
    }
  }
  return most;
}

int stride_serve_window_attention(const StrideWindowAttentionParams* p, void* stream) {
  if (!p) return fail(STRIDE_TC_EINVAL, "window_attention: null parameters");
  Plan plan;
  if (const char* why = plan_of(*p, plan)) return fail(STRIDE_TC_EINVAL, std::string("window_attention: ") + why);
  if (p->l.rows == 0) return 0;
  if (!p->q || !p->out || !p->kv.arena || !p->kv.table || !p->row_slot || !p->row_pos)
    return fail(STRIDE_TC_EINVAL, "window_attention: missing pointer");
  if ((reinterpret_cast<uintptr_t>(p->q) | reinterpret_cast<uintptr_t>(p->kv.arena) | reinterpret_cast<uintptr_t>(p->scratch)) % 16 ||
      reinterpret_cast<uintptr_t>(p->out) % 8)
    return fail(STRIDE_TC_EINVAL, "window_attention: q, the arena and scratch must be 16-byte aligned, out 8");
  if (plan.scratch > 0 && (!p->scratch || p->scratch_floats < plan.scratch))
    return fail(STRIDE_TC_EINVAL, "window_attention: scratch is smaller than stride_serve_window_attention_scratch()");
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (p->head_dim == 32) return run<32>(*p, plan, st);
  if (p->head_dim == 64) return run<64>(*p, plan, st);
  return run<128>(*p, plan, st);
}

}  // extern "C"
