// Logit processing on lm_full's tiles: penalties for tokens that a sequence has, biases, a
// grammar's mask and the greedy choice in one pass (include/stride_serve.h).
//
// What bounds it is the logits' own read (and write): 16 lanes x vocabulary x 4 bytes a lane
// tile. Few tokens carry a penalty or bias, so those are found by bits, 1/32 of the logits'
// size, and only where a bit is set is the count fetched; a workgroup first brings the bits
// of its kTiles row tiles to LDS, then streams its logits once. (128 rows of 128256 tokens
// written back, 512 tokens a row with counts: 36 us, 3.7 TB/s; a 4 GiB copy: 4.8. One row: 9 us.)
#include <hip/hip_runtime.h>

#include <climits>
#include <cstddef>
#include <string>

#include "../../include/stride_serve.h"
#include "tc_common.hpp"

namespace stride_tc {

int fail(int code, const std::string& msg);  // tc_gemm.hip

namespace {

constexpr int kTiles = 32;             // row tiles of a workgroup
constexpr int kTokens = kTiles * 16;
constexpr int kWords = kTokens / 32;
constexpr int kThreads = 512;
constexpr int kWaves = kThreads / 64;
constexpr int kSteps = kTiles / kWaves;  // a wave takes every eighth tile

// (value, lowest index first) as a key whose unsigned order is the choice's, 0 below all.
// + 0 joins the zeros, which compare equal.
__device__ __forceinline__ uint64_t key_of(float v, int index) {
  const uint32_t u = u32_of(v + 0.0f);
  const uint32_t order = u & 0x80000000u ? ~u : u | 0x80000000u;
  return (static_cast<uint64_t>(order) << 32) | static_cast<uint32_t>(~index);
}
__device__ __forceinline__ float key_value(uint64_t k) {
  const uint32_t order = static_cast<uint32_t>(k >> 32);
  return f32_of(order & 0x80000000u ? order & 0x7FFFFFFFu : ~order);
}

// Scratch of a lane tile: kSubs + 1 units of 16 keys and a count, 256 bytes each.
constexpr int kSubs = 16;
constexpr int kUnit = 32;

// A wave's keys (lane t's: row t) enter a unit; true in the last of `members` workgroups, whose
// k are then the largest of all.
__device__ __forceinline__ bool join(unsigned long long* unit, bool live, uint64_t& k, int members) {
  if (live && k) {
    const unsigned long long before = __hip_atomic_fetch_max(unit + threadIdx.x, static_cast<unsigned long long>(k), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("" ::"v"(before));
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // they have been performed
  int ended = 0;
  if (threadIdx.x == 0)
    ended = __hip_atomic_fetch_add(unit + 16, 1ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == static_cast<unsigned long long>(members - 1);
  if (!__builtin_amdgcn_readfirstlane(ended)) return false;
  if (live) k = __hip_atomic_exchange(unit + threadIdx.x, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  if (threadIdx.x == 0) __hip_atomic_exchange(unit + 16, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return true;
}

// First entry of the ascending list t[lo, hi) that is not below x.
__device__ __forceinline__ int lower_bound(const int32_t* t, int lo, int hi, int x) {
  while (lo < hi) {
    const int mid = lo + (hi - lo) / 2;
    if (t[mid] < x) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

// Workgroup: lane tile lt, tokens [t0, t0 + kTokens). Thread: four lanes of a token in each
// of its steps, as the tiles lie. Lane tiles of a chunk have neighbouring workgroups.
template <bool COUNTS, bool BIAS>
__global__ __launch_bounds__(kThreads) void k_process(StrideLogitsParams p, int row_tiles, int chunks) {
  __shared__ __align__(16) uint32_t seen[kWords][16], allowed[kWords][16], biased[kWords][16];
  __shared__ float bias[BIAS ? kTokens : 1][16];
  __shared__ uint64_t best[kWaves][16];
  const int lt = blockIdx.x % p.l.lane_groups, chunk = blockIdx.x / p.l.lane_groups;
  const int t0 = chunk * kTokens;
  const int t = threadIdx.x, wave = t >> 6, lane = t & 63, quad = t & 3, tok = (t >> 2) & 15;
  const int words = (p.vocab + 31) >> 5;

  // the logits first: nothing else is as far away
  f32x4 v[kSteps];
  const int rt0 = chunk * kTiles;
  const int64_t step = static_cast<int64_t>(p.l.lane_groups) * kTileElems;
  const float* in = p.logits + rt0 * step + lt * kTileElems + tok * 16 + quad * 4;
#pragma unroll
  for (int i = 0; i < kSteps; ++i)
    v[i] = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(in + min(kWaves * i + wave, row_tiles - 1 - rt0) * step));
  // A word a thread, lane t % 16 and word t / 16 % 16: the first half of the workgroup the
  // seen bits, the second the mask's. Sixteen threads a lane look for its biases in the range.
  uint32_t bits = t < 256 ? 0u : 0xFFFFFFFFu;
  const int row = lt * 16 + (t & 15), w = (t0 >> 5) + ((t >> 4) & 15);
  if (row < p.l.rows && w < words) {
    if (t < 256) {
      if constexpr (COUNTS) {
        const int slot = p.row_slot[row];
        if (slot >= 0 && slot < p.slots) bits = p.seen[static_cast<int64_t>(slot) * words + w];
      }
    } else if (p.mask) {
      const int m = p.mask_row[row];
      if (m >= 0 && m < p.masks) bits = p.mask[static_cast<int64_t>(m) * words + w];
    }
  }
  float rep[4], pres[4], freq[4];
  const int32_t* counts[4];
  if constexpr (COUNTS) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int r = min(lt * 16 + quad * 4 + e, p.l.rows - 1);
      rep[e] = p.penalties[3 * r];
      pres[e] = p.penalties[3 * r + 1];
      freq[e] = p.penalties[3 * r + 2];
      const int slot = p.row_slot[r];
      counts[e] = p.counts + static_cast<int64_t>(slot >= 0 && slot < p.slots ? slot : 0) * p.vocab;
    }
  }
  if constexpr (BIAS) {
    if (t < 256) biased[t >> 4][t & 15] = 0;
    __syncthreads();
    const int ln = t >> 5, r = lt * 16 + ln;
    if (r < p.l.rows) {
      int lo = p.bias_offsets[r], hi = p.bias_offsets[r + 1];
      const int end = hi;
      if (hi - lo > 256) {
        lo = lower_bound(p.bias_tokens, lo, hi, t0);
        hi = lower_bound(p.bias_tokens, lo, hi, t0 + kTokens);
      }
      for (int e = lo + (t & 31); e < hi; e += 32) {
        const int token = p.bias_tokens[e], next = p.bias_tokens[min(e + 1, end - 1)], at = token - t0;
        const float b = p.bias_values[e];
        if (at < 0 || at >= kTokens || token >= p.vocab || (e + 1 < end && next == token)) continue;
        bias[at][ln] = b;
        atomicOr(&biased[at >> 5][ln], 1u << (at & 31));
      }
    }
  }
  if (t < 256) seen[(t >> 4) & 15][t & 15] = bits;
  else allowed[(t >> 4) & 15][t & 15] = bits;
  __syncthreads();

  // every wanted count is under way before the first is used
  int n[kSteps][4];
  if constexpr (COUNTS) {
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const int at = (kWaves * i + wave) * 16 + tok;
      const u32x4 s = *reinterpret_cast<const u32x4*>(&seen[at >> 5][4 * quad]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        n[i][e] = 0;
        if (((s[e] >> (at & 31)) & 1u) && t0 + at < p.vocab) n[i][e] = counts[e][t0 + at];
      }
    }
  }
  float top[4] = {f32_of(0xFF800000u), f32_of(0xFF800000u), f32_of(0xFF800000u), f32_of(0xFF800000u)};
  int who[4] = {-1, -1, -1, -1};
  const int rows = p.l.rows - (lt * 16 + quad * 4);
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    const int tile = kWaves * i + wave, at = tile * 16 + tok, token = t0 + at;
    const bool real = token < p.vocab;
    const u32x4 a = *reinterpret_cast<const u32x4*>(&allowed[at >> 5][4 * quad]);
    u32x4 b = {0, 0, 0, 0};
    if constexpr (BIAS) b = *reinterpret_cast<const u32x4*>(&biased[at >> 5][4 * quad]);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float l = v[i][e];
      if constexpr (COUNTS) {
        if (n[i][e]) {
          l = l > 0.0f ? l / rep[e] : l * rep[e];
          const int made = n[i][e] & 0x7FFFFFFF;
          if (made) {
            l = l - freq[e] * static_cast<float>(made);
            l = l - pres[e];
          }
        }
      }
      if constexpr (BIAS) {
        if ((b[e] >> (at & 31)) & 1u) l = l + bias[at][4 * quad + e];
      }
      if (!((a[e] >> (at & 31)) & 1u)) l = f32_of(0xFF800000u);
      v[i][e] = l;
      if (real && l > top[e]) {
        top[e] = l;
        who[e] = token;
      }
    }
    if (p.out && real) {
      float* out = p.out + (rt0 + tile) * step + lt * kTileElems + tok * 16 + quad * 4;
      if (rows >= 4) __builtin_nontemporal_store(v[i], reinterpret_cast<f32x4*>(out));
      else
        for (int e = 0; e < 3; ++e)
          if (e < rows) out[e] = v[i][e];
    }
  }
  // the workgroup's choice of each lane: lanes of a wave with the same quad, then the waves
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    uint64_t k = who[e] < 0 ? 0 : key_of(top[e], who[e]);
#pragma unroll
    for (int d = 4; d < 64; d <<= 1) {
      const uint64_t o = __shfl_xor(static_cast<unsigned long long>(k), d);
      k = o > k ? o : k;
    }
    if (lane < 4) best[wave][4 * quad + e] = k;
  }
  __syncthreads();
  // Joined in scratch by atomics alone, which are performed where all workgroups see them; a
  // fence would write back the L2's dirty lines, the logits among them (128 rows 110 us with
  // fences, 45 without). In two stages of at most kSubs and 1 / kSubs of the workgroups each,
  // since atomics on one address queue up. The last workgroup of a stage takes its keys out,
  // which leaves zeros, and the very last one writes the result.
  if (t >= 64) return;
  const int row_of_key = lt * 16 + t;
  const bool live = t < 16 && row_of_key < p.l.rows;
  uint64_t k = 0;
  if (live)
#pragma unroll
    for (int x = 0; x < kWaves; ++x) k = best[x][t] > k ? best[x][t] : k;
  unsigned long long* unit = reinterpret_cast<unsigned long long*>(p.scratch) + static_cast<int64_t>(lt) * (kSubs + 1) * kUnit;
  const int sub = chunk % kSubs;
  if (!join(unit + (1 + sub) * kUnit, live, k, (chunks - sub + kSubs - 1) / kSubs)) return;
  if (!join(unit, live, k, min(kSubs, chunks))) return;
  if (live) {
    StrideBestEntry e;
    e.value = k ? key_value(k) : f32_of(0xFF800000u);
    e.index = k ? static_cast<int32_t>(~static_cast<uint32_t>(k)) : -1;
    p.best[row_of_key] = e;
  }
}

__global__ __launch_bounds__(256) void k_record(StrideTokenCounts p, const int32_t* slots, const int32_t* tokens, int token_stride, int n,
                                                int prompt) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const int s = slots[i], t = tokens[static_cast<int64_t>(i) * token_stride];
  if (s < 0 || s >= p.slots || t < 0 || t >= p.vocab) return;
  int32_t* at = p.counts + static_cast<int64_t>(s) * p.vocab + t;
  if (prompt) atomicOr(at, INT_MIN);
  else atomicAdd(at, 1);
  atomicOr(&p.seen[static_cast<int64_t>(s) * ((p.vocab + 31) >> 5) + (t >> 5)], 1u << (t & 31));
}

// Workgroup: item i, 256 words. A word's counts are visited only where one of the two has a bit.
__global__ __launch_bounds__(256) void k_reset(StrideTokenCounts p, const int32_t* slots, const int32_t* srcs) {
  const int words = (p.vocab + 31) >> 5;
  const int i = blockIdx.x, w = blockIdx.y * 256 + threadIdx.x;
  const int s = slots[i], f = srcs ? srcs[i] : -1;
  if (s < 0 || s >= p.slots || w >= words || (srcs && (f < 0 || f >= p.slots || f == s))) return;
  uint32_t* to = p.seen + static_cast<int64_t>(s) * words + w;
  const uint32_t have = srcs ? p.seen[static_cast<int64_t>(f) * words + w] : 0u;
  uint32_t bits = *to | have;
  if (w == words - 1 && (p.vocab & 31)) bits &= (1u << (p.vocab & 31)) - 1u;
  *to = have;
  while (bits) {
    const int b = __ffs(bits) - 1;
    bits &= bits - 1;
    const int64_t t = w * 32 + b;
    p.counts[static_cast<int64_t>(s) * p.vocab + t] = (have >> b) & 1u ? p.counts[static_cast<int64_t>(f) * p.vocab + t] : 0;
  }
}

int refused(const char* what, const char* why) { return fail(STRIDE_TC_EINVAL, std::string(what) + ": " + why); }

int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(static_cast<int>(e), std::string(what) + " launch failed: " + hipGetErrorString(e));
  return 0;
}

const char* why_not(const StrideTokenCounts* p, int n) {
  if (!p) return "null parameters";
  if (n < 0 || p->slots < 1 || p->vocab < 1 || p->vocab > INT_MAX - kTokens) return "bad n, slots or vocab";
  if (!p->counts || !p->seen) return "missing pointer";
  return nullptr;
}

}  // namespace
}  // namespace stride_tc

using namespace stride_tc;

static_assert(sizeof(StrideLogitsParams) == 136 && offsetof(StrideLogitsParams, vocab) == 120, "LogitsParams layout");
static_assert(sizeof(StrideTokenCounts) == 24, "TokenCounts layout");

extern "C" {

int64_t stride_logits_scratch(int32_t rows) { return rows < 0 ? -1 : (static_cast<int64_t>(rows) + 15) / 16 * (kSubs + 1) * kUnit; }

int stride_logits_process(const StrideLogitsParams* p, void* stream) {
  const char* what = "logits_process";
  if (!p) return refused(what, "null parameters");
  if (p->l.rows < 0 || p->l.lane_groups != (static_cast<int64_t>(p->l.rows) + 15) / 16) return refused(what, "need rows >= 0 and lane_groups = ceil(rows/16)");
  if (p->vocab < 1 || p->vocab > INT_MAX - kTokens) return refused(what, "bad vocab");
  if (p->l.rows == 0) return 0;
  if (!p->logits || !p->best || !p->scratch) return refused(what, "missing pointer");
  if (p->counts && (!p->seen || !p->row_slot || !p->penalties || p->slots < 1)) return refused(what, "counts need seen, row_slot, penalties and slots");
  if (p->bias_offsets && (!p->bias_tokens || !p->bias_values)) return refused(what, "bias_offsets need tokens and values");
  if (p->mask && (!p->mask_row || p->masks < 1)) return refused(what, "a mask needs mask_row and masks");
  if ((reinterpret_cast<uintptr_t>(p->logits) | reinterpret_cast<uintptr_t>(p->out)) % 16) return refused(what, "logits and out must be 16-byte aligned");
  const int row_tiles = (p->vocab + 15) / 16, chunks = (row_tiles + kTiles - 1) / kTiles;
  const int64_t groups = static_cast<int64_t>(chunks) * p->l.lane_groups;
  if (groups > INT_MAX) return refused(what, "rows and vocab are too large together");
  const dim3 grid(static_cast<unsigned>(groups)), block(kThreads);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (p->counts && p->bias_offsets) hipLaunchKernelGGL((k_process<true, true>), grid, block, 0, st, *p, row_tiles, chunks);
  else if (p->counts) hipLaunchKernelGGL((k_process<true, false>), grid, block, 0, st, *p, row_tiles, chunks);
  else if (p->bias_offsets) hipLaunchKernelGGL((k_process<false, true>), grid, block, 0, st, *p, row_tiles, chunks);
  else hipLaunchKernelGGL((k_process<false, false>), grid, block, 0, st, *p, row_tiles, chunks);
  return launched(what);
}

int stride_logits_record(const StrideTokenCounts* p, const int32_t* slot, const int32_t* tokens, int32_t token_stride, int32_t n, int32_t prompt,
                         void* stream) {
  if (const char* why = why_not(p, n)) return refused("logits_record", why);
  if (n == 0) return 0;
  if (!slot || !tokens || token_stride < 0) return refused("logits_record", "missing pointer or negative stride");
  hipLaunchKernelGGL(k_record, dim3((static_cast<unsigned>(n) + 255) / 256), dim3(256), 0, static_cast<hipStream_t>(stream), *p, slot, tokens,
                     token_stride, n, prompt);
  return launched("logits_record");
}

int stride_logits_reset(const StrideTokenCounts* p, const int32_t* slot, const int32_t* src, int32_t n, void* stream) {
  if (const char* why = why_not(p, n)) return refused("logits_reset", why);
  if (n == 0) return 0;
  if (!slot) return refused("logits_reset", "missing pointer");
  const unsigned groups = (static_cast<unsigned>((p->vocab + 31) / 32) + 255) / 256;
  if (groups > 65535) return refused("logits_reset", "vocab is too large");
  hipLaunchKernelGGL(k_reset, dim3(n, groups), dim3(256), 0, static_cast<hipStream_t>(stream), *p, slot, src);
  return launched("logits_reset");
}

}  // extern "C"
