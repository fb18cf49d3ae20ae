// A pool of KV pages that sequences share with counted references (include/stride_serve.h):
// reserve, release, fork, compact and copy, all on the device, so that a captured step can
// cross page borders and branch.
//
// Which page is taken must not depend on the order in which workgroups run: the free pages
// are a bit map, and a call takes the lowest numbers in (item, table index) order. So taking
// pages is one workgroup's work (`plan` kernels: checks, then a prefix sum over the wants
// and a walk over the bit map); giving them up commutes (integer atomics) and moving their
// contents is spread over the chip.
//
// A plan kernel writes work[0] = 1 where the call may go on; the kernels after it leave at
// once where it is 0. What bounds the movers is memory: every moved byte is read once and
// written once.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cstddef>
#include <string>

#include "../../include/stride_serve.h"
#include "tc_common.hpp"

namespace stride_tc {

int fail(int code, const std::string& msg);  // tc_gemm.hip

namespace {

constexpr int kPlan = 1024;             // threads of a plan workgroup
constexpr int kMaxSlots = 131072;       // slots whose bits a plan workgroup marks in LDS (16 KiB)
constexpr int kWaves = kPlan / 64;

// work: [0] go, [1] pages wanted, then the free pages in order ([pages]), then what the
// call keeps per item.
constexpr int kWorkHead = 4;
__device__ __forceinline__ int32_t* free_list(const StrideKvPool& p) { return p.work + kWorkHead; }
__device__ __forceinline__ int32_t* item_work(const StrideKvPool& p) { return p.work + kWorkHead + p.pages; }
__device__ __forceinline__ int32_t* table_row(const StrideKvPool& p, int slot) {
  return const_cast<int32_t*>(p.kv.table) + static_cast<int64_t>(slot) * p.kv.max_blocks;
}
__device__ __forceinline__ bool is_page(const StrideKvPool& p, int b) { return b >= 0 && b < p.pages; }

// Gives up one reference.
__device__ __forceinline__ void drop(const StrideKvPool& p, int page) {
  if (!is_page(p, page)) return;
  const int before = atomicSub(&p.refs[page], 1);
  if (before == 1) atomicOr(&p.free_bits[page >> 5], 1u << (page & 31));
  if (before <= 0) atomicOr(p.errors, STRIDE_KV_BAD_REFS);
}

// The prefix sum of v over a plan workgroup's threads, v's own excluded; `sum`: of all.
__device__ __forceinline__ int before_me(int v, int* lds, int& sum) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int x = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_up(x, d);
    if (lane >= d) x += o;
  }
  __syncthreads();
  if (lane == 63) lds[wave] = x;
  __syncthreads();
  int base = 0;
  sum = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) base += lds[w];
    sum += lds[w];
  }
  return base + x - v;
}

// The lowest `want` free pages, in order, to free_list. False: there are fewer.
__device__ __forceinline__ bool list_free(const StrideKvPool& p, int want, int* lds) {
  const int words = (p.pages + 31) / 32;
  int have = 0;
  for (int w0 = 0; w0 < words && have < want; w0 += kPlan) {
    const int w = w0 + threadIdx.x;
    uint32_t bits = w < words ? p.free_bits[w] : 0u;
    if (w == words - 1 && (p.pages & 31)) bits &= (1u << (p.pages & 31)) - 1u;
    int sum;
    int at = have + before_me(__popc(bits), lds, sum);
    while (bits && at < want) {
      free_list(p)[at++] = w * 32 + __ffs(bits) - 1;
      bits &= bits - 1;
    }
    have += sum;
  }
  __syncthreads();
  return have >= want;
}

// A page of the list is taken: its first reference.
__device__ __forceinline__ void take(const StrideKvPool& p, int page) {
  p.refs[page] = 1;
  atomicAnd(&p.free_bits[page >> 5], ~(1u << (page & 31)));
}

// Marks slot in the bit map of an LDS array; true where it was marked before.
__device__ __forceinline__ bool mark(uint32_t* bits, int slot) {
  return (atomicOr(&bits[slot >> 5], 1u << (slot & 31)) >> (slot & 31)) & 1u;
}
__device__ __forceinline__ bool marked(const uint32_t* bits, int slot) { return (bits[slot >> 5] >> (slot & 31)) & 1u; }

// Ends a plan's checks: the workgroup's errors together. True: none.
__device__ __forceinline__ bool agree(const StrideKvPool& p, int bad, int* lds) {
  __syncthreads();
  if (threadIdx.x == 0) lds[0] = 0;
  __syncthreads();
  if (bad) atomicOr(&lds[0], bad);
  __syncthreads();
  const int all = lds[0];
  if (all && threadIdx.x == 0) atomicOr(p.errors, all);
  if (threadIdx.x == 0) p.work[0] = all ? 0 : 1;
  __syncthreads();
  return all == 0;
}

// The plan of reserve and compact: items i with table ranges [lo, hi) whose entries want a
// page where `wants(row, b)`; `give(i, b, page)` takes it. Wave per item, counts first.
template <class Range, class Wants, class Give>
__device__ __forceinline__ void share_out(const StrideKvPool& p, int n, int* lds, Range range, Wants wants, Give give) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int32_t* first_of = item_work(p);  // [n]: the item's first place in the list
  for (int i = wave; i < n; i += kWaves) {
    int slot, lo, hi, count = 0;
    range(i, slot, lo, hi);
    const int32_t* row = table_row(p, slot);
    for (int b = lo + lane; b < hi; b += 64) count += wants(row[b]) ? 1 : 0;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) count += __shfl_xor(count, d);
    if (lane == 0) first_of[i] = count;
  }
  __syncthreads();
  int total = 0;
  for (int i0 = 0; i0 < n; i0 += kPlan) {
    const int i = i0 + threadIdx.x;
    int sum;
    const int at = total + before_me(i < n ? first_of[i] : 0, lds, sum);
    if (i < n) first_of[i] = at;
    total += sum;
  }
  __syncthreads();
  const bool enough = total == 0 || list_free(p, total, lds);
  if (!agree(p, enough ? 0 : STRIDE_KV_NO_PAGES, lds)) return;
  for (int i = wave; i < n; i += kWaves) {
    int slot, lo, hi;
    range(i, slot, lo, hi);
    const int32_t* row = table_row(p, slot);
    int at = first_of[i];
    for (int b0 = lo; b0 < hi; b0 += 64) {
      const int b = b0 + lane;
      const bool w = b < hi && wants(row[b]);
      const uint64_t all = __ballot(w);
      const int page = w ? free_list(p)[at + __popcll(all & ((uint64_t{1} << lane) - 1))] : -1;
      if (w) take(p, page);
      if (b < hi) give(i, b, page);
      at += __popcll(all);
    }
  }
}

__global__ __launch_bounds__(kPlan) void k_reserve(StrideKvPool p, const int32_t* slots, const int32_t* first, const int32_t* end, int n) {
  __shared__ uint32_t bits[kMaxSlots / 32];
  __shared__ int lds[kWaves];
  for (int i = threadIdx.x; i < (p.slots + 31) / 32; i += kPlan) bits[i] = 0;
  __syncthreads();
  int bad = 0;
  for (int i = threadIdx.x; i < n; i += kPlan) {
    const int s = slots[i];
    if (s < 0 || s >= p.slots || first[i] < 0 || end[i] > p.kv.max_blocks) bad |= STRIDE_KV_BAD_ITEM;
    else if (mark(bits, s)) bad |= STRIDE_KV_TWICE;
  }
  if (!agree(p, bad, lds)) return;
  share_out(
      p, n, lds, [&](int i, int& s, int& lo, int& hi) { s = slots[i], lo = first[i], hi = end[i]; }, [](int b) { return b < 0; },
      [&](int i, int b, int page) {
        if (page >= 0) table_row(p, slots[i])[b] = page;
      });
}

__global__ __launch_bounds__(256) void k_release(StrideKvPool p, const int32_t* slots, const int32_t* first, const int32_t* end) {
  const int i = blockIdx.x, s = slots[i];
  if (s < 0 || s >= p.slots) {
    if (threadIdx.x == 0) atomicOr(p.errors, STRIDE_KV_BAD_ITEM);
    return;
  }
  int32_t* row = table_row(p, s);
  const int lo = max(first[i], 0), hi = min(end[i], p.kv.max_blocks);
  for (int64_t b = static_cast<int64_t>(lo) + threadIdx.x; b < hi; b += 256)
    if (row[b] >= 0) {
      const int page = atomicExch(&row[b], -1);
      drop(p, page);
    }
}

// Fork. Item i keeps the new page of its part page, or -1, in item_work[i].
__global__ __launch_bounds__(kPlan) void k_fork_plan(StrideKvPool p, const int32_t* src, const int32_t* dst, const int32_t* length,
                                                     int n, int page_shift) {
  __shared__ uint32_t to[kMaxSlots / 32];
  __shared__ int lds[kWaves];
  for (int i = threadIdx.x; i < (p.slots + 31) / 32; i += kPlan) to[i] = 0;
  __syncthreads();
  int bad = 0;
  for (int i = threadIdx.x; i < n; i += kPlan) {
    const int a = src[i], b = dst[i], len = length[i];
    if (a < 0 || a >= p.slots || b < 0 || b >= p.slots || len < 0 || len > static_cast<int64_t>(p.kv.max_blocks) << page_shift)
      bad |= STRIDE_KV_BAD_ITEM;
    else if (mark(to, b)) bad |= STRIDE_KV_TWICE;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kPlan) {
    const int a = src[i];
    if (a >= 0 && a < p.slots && marked(to, a)) bad |= STRIDE_KV_TWICE;
  }
  if (!agree(p, bad, lds)) return;
  auto wants = [&](int i) { return (length[i] & ((1 << page_shift) - 1)) && is_page(p, table_row(p, src[i])[length[i] >> page_shift]); };
  int total = 0;
  for (int i0 = 0; i0 < n; i0 += kPlan) {
    const int i = i0 + threadIdx.x;
    const bool w = i < n && wants(i);
    int sum;
    const int at = total + before_me(w ? 1 : 0, lds, sum);
    if (i < n) item_work(p)[i] = w ? at : -1;
    total += sum;
  }
  __syncthreads();
  if (!agree(p, total == 0 || list_free(p, total, lds) ? 0 : STRIDE_KV_NO_PAGES, lds)) return;
  for (int i = threadIdx.x; i < n; i += kPlan) {
    const int at = item_work(p)[i];
    if (at < 0) continue;
    const int page = free_list(p)[at];
    take(p, page);
    item_work(p)[i] = page;
  }
}

// The runs of a page ([layer][K|V][group] pieces of page_tokens rows), as byte offsets.
struct Runs {
  int64_t layer, which, group;
  int n_kv, count;
  __device__ __forceinline__ int64_t at(int r) const {
    const int g = r % n_kv, rest = r / n_kv;
    return (rest >> 1) * layer + (rest & 1) * which + g * group;
  }
};
__device__ __forceinline__ Runs runs_of(const StrideKvPool& p) {
  return {p.kv.layer_elems * p.elem_bytes, p.kv.which_elems * p.elem_bytes, p.kv.group_elems * p.elem_bytes, p.n_kv, p.layers * 2 * p.n_kv};
}

// Copies the first `bytes` of every run of a page; a wave takes runs r0, r0 + step, ..
__device__ __forceinline__ void copy_page(const StrideKvPool& p, const char* from, char* to, int bytes, int r0, int step, int lane) {
  const Runs runs = runs_of(p);
  for (int r = r0; r < runs.count; r += step) {
    const int64_t off = runs.at(r);
    for (int b = lane * 16; b < bytes; b += 64 * 16) *reinterpret_cast<u32x4*>(to + off + b) = load16(from + off + b);
  }
}

__global__ __launch_bounds__(256) void k_fork_apply(StrideKvPool p, const int32_t* src, const int32_t* dst, const int32_t* length,
                                                    int page_shift) {
  if (p.work[0] == 0) return;
  const int i = blockIdx.x, lane = threadIdx.x & 63;
  const int len = length[i], full = len >> page_shift, part = len & ((1 << page_shift) - 1), fresh = item_work(p)[i];
  const int32_t* from = table_row(p, src[i]);
  if (blockIdx.y == 0) {
    int32_t* row = table_row(p, dst[i]);
    for (int b = threadIdx.x; b < p.kv.max_blocks; b += 256) {
      const int old = row[b];
      int page = -1;
      if (b < full) {
        page = from[b];
        if (is_page(p, page)) atomicAdd(&p.refs[page], 1);
        else page = -1;
      } else if (b == full) {
        page = fresh;
      }
      if (page != old) row[b] = page;
      if (old >= 0) drop(p, old);
    }
  }
  if (fresh < 0) return;
  char* arena = static_cast<char*>(p.kv.arena);
  const int64_t block = p.kv.block_elems * p.elem_bytes;
  copy_page(p, arena + from[full] * block, arena + fresh * block, part * p.kv.head_dim * p.elem_bytes, blockIdx.y * 4 + (threadIdx.x >> 6),
            gridDim.y * 4, lane);
}

// Compact. Item i's new pages: item_work[n + i * max_blocks + b], -1 where the entry stays.
__device__ __forceinline__ int32_t* new_row(const StrideKvPool& p, int n, int i) {
  return item_work(p) + n + static_cast<int64_t>(i) * p.kv.max_blocks;
}

__global__ __launch_bounds__(kPlan) void k_compact_plan(StrideKvPool p, const int32_t* slots, const int32_t* first, const int32_t* count,
                                                        int n, int page_shift, int width) {
  __shared__ uint32_t bits[kMaxSlots / 32];
  __shared__ int lds[kWaves];
  for (int i = threadIdx.x; i < (p.slots + 31) / 32; i += kPlan) bits[i] = 0;
  __syncthreads();
  int bad = 0;
  for (int i = threadIdx.x; i < n; i += kPlan) {
    const int s = slots[i];
    if (s < 0 || s >= p.slots || first[i] < 0 || count[i] < 0 || count[i] > width ||
        static_cast<int64_t>(first[i]) + count[i] > static_cast<int64_t>(p.kv.max_blocks) << page_shift)
      bad |= STRIDE_KV_BAD_ITEM;
    else if (mark(bits, s)) bad |= STRIDE_KV_TWICE;
  }
  if (!agree(p, bad, lds)) return;
  share_out(
      p, n, lds,
      [&](int i, int& s, int& lo, int& hi) {
        s = slots[i];
        lo = first[i] >> page_shift;
        hi = count[i] ? (first[i] + count[i] + (1 << page_shift) - 1) >> page_shift : lo;
      },
      [&](int b) { return !is_page(p, b) || p.refs[b] > 1; }, [&](int i, int b, int page) { new_row(p, n, i)[b] = page; });
}

// Moves one run (a layer, K or V, a group) of an item's kept positions. In place it must not
// write what is still to be read: positions ascend and each comes from its own place or a
// later one, so a workgroup that takes them in ascending steps, loads a step whole before it
// writes it, overwrites only what it has read.
template <int U>
__global__ __launch_bounds__(256) void k_compact_move(StrideKvPool p, const int32_t* slots, const int32_t* first, const int32_t* count,
                                                      const int32_t* keep, int64_t keep_stride, int n, int page_shift, int pieces) {
  if (p.work[0] == 0) return;
  const Runs runs = runs_of(p);
  const int i = blockIdx.x / runs.count, run = blockIdx.x % runs.count, t = threadIdx.x;
  const int begin = first[i], many = count[i], in_page = (1 << page_shift) - 1;
  if (many == 0) return;
  const int32_t* row = table_row(p, slots[i]);
  const int32_t* fresh = new_row(p, n, i);
  const int32_t* list = keep + i * keep_stride;
  char* base = static_cast<char*>(p.kv.arena) + runs.at(run);
  const int64_t block = p.kv.block_elems * p.elem_bytes;
  const int cap = p.kv.max_blocks << page_shift, row_bytes = pieces * 16;
  // a page that is replaced takes along what it holds before `begin`
  const int lead = fresh[begin >> page_shift] >= 0 ? begin & in_page : 0;
  const int per = 256 / pieces;  // positions of a load
  const int in = t % pieces * 16, at = t / pieces;
  int bad = 0;
  for (int k0 = -lead; k0 < many; k0 += per * U) {
    u32x4 v[U];
    bool ok[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + u * per + at;
      ok[u] = at < per && k < many;
      if (!ok[u]) continue;
      const int from = k < 0 ? begin + k : list[k];
      if (from < begin + k || from >= cap || (k > 0 && list[k - 1] >= from)) bad |= STRIDE_KV_BAD_KEEP;
      const int page = from >= 0 && from < cap ? row[from >> page_shift] : -1;
      ok[u] = is_page(p, page);
      if (ok[u]) v[u] = load16(base + page * block + static_cast<int64_t>(from & in_page) * row_bytes + in);
      else if (k >= 0) bad |= STRIDE_KV_MISSING;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the step is read before any wave writes it
    __syncthreads();
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!ok[u]) continue;
      const int to = begin + k0 + u * per + at;
      const int page = fresh[to >> page_shift] >= 0 ? fresh[to >> page_shift] : row[to >> page_shift];
      *reinterpret_cast<u32x4*>(base + page * block + static_cast<int64_t>(to & in_page) * row_bytes + in) = v[u];
    }
  }
  if (bad) atomicOr(p.errors, bad);
}

__global__ __launch_bounds__(256) void k_compact_finish(StrideKvPool p, const int32_t* slots, const int32_t* first, const int32_t* count,
                                                        int n, int page_shift) {
  if (p.work[0] == 0) return;
  const int i = blockIdx.x;
  int32_t* row = table_row(p, slots[i]);
  const int32_t* fresh = new_row(p, n, i);
  const int lo = first[i] >> page_shift, end = (first[i] + count[i] + (1 << page_shift) - 1) >> page_shift;
  const int hi = count[i] ? end : lo;  // entries that the plan looked at: [lo, hi)
  for (int b = lo + threadIdx.x; b < p.kv.max_blocks; b += 256) {
    const int old = row[b];
    if (b < hi) {
      if (fresh[b] < 0) continue;
      row[b] = fresh[b];
      drop(p, old);
    } else if (b >= end && old >= 0) {
      row[b] = -1;
      drop(p, old);
    }
  }
}

// Copy. The destinations' marks are a bit map in the free list's place.
__global__ __launch_bounds__(kPlan) void k_copy_plan(StrideKvPool p, const int32_t* src, const int32_t* dst, const int32_t* tokens, int n,
                                                     int to_pages, int same, int page_tokens) {
  __shared__ int lds[kWaves];
  uint32_t* bits = reinterpret_cast<uint32_t*>(free_list(p));
  for (int i = threadIdx.x; i < (to_pages + 31) / 32; i += kPlan) bits[i] = 0;
  __syncthreads();
  int bad = 0;
  for (int i = threadIdx.x; i < n; i += kPlan) {
    if (!is_page(p, src[i]) || dst[i] < 0 || dst[i] >= to_pages || (tokens && (tokens[i] < 0 || tokens[i] > page_tokens)))
      bad |= STRIDE_KV_BAD_ITEM;
    else if (mark(bits, dst[i])) bad |= STRIDE_KV_TWICE;
  }
  __syncthreads();
  if (same)
    for (int i = threadIdx.x; i < n; i += kPlan)
      if (is_page(p, src[i]) && src[i] < to_pages && marked(bits, src[i])) bad |= STRIDE_KV_TWICE;
  agree(p, bad, lds);
}

__global__ __launch_bounds__(256) void k_copy(StrideKvPool p, char* to, const int32_t* src, const int32_t* dst, const int32_t* tokens,
                                              int page_tokens) {
  if (p.work[0] == 0) return;
  const int i = blockIdx.x;
  const int64_t block = p.kv.block_elems * p.elem_bytes;
  copy_page(p, static_cast<const char*>(p.kv.arena) + src[i] * block, to + dst[i] * block,
            (tokens ? tokens[i] : page_tokens) * p.kv.head_dim * p.elem_bytes, blockIdx.y * 4 + (threadIdx.x >> 6), gridDim.y * 4,
            threadIdx.x & 63);
}

// ---------------------------------------------------------------------------
// Host side.

int64_t work_ints(int64_t slots, int64_t max_blocks, int64_t pages) { return kWorkHead + pages + slots * (1 + max_blocks); }

int64_t page_tokens_of(const StrideKvPool& p) { return p.kv.head_dim > 0 ? p.kv.group_elems / p.kv.head_dim : 0; }

const char* why_not(const StrideKvPool* p, int n, int& page_shift) {
  if (!p) return "null pool";
  const int64_t tokens = page_tokens_of(*p);
  if (n < 0) return "n must not be negative";
  if (p->elem_bytes != 2 && p->elem_bytes != 4) return "elem_bytes must be 2 or 4";
  if (p->pages < 1 || p->slots < 1 || p->slots > kMaxSlots || p->layers < 1 || p->n_kv < 1 || p->kv.max_blocks < 1)
    return "bad pages, slots (at most 131072), layers, n_kv or max_blocks";
  if (tokens < 1 || tokens * p->kv.head_dim != p->kv.group_elems || (tokens & (tokens - 1)) || tokens > (1 << 24))
    return "the KV page (group_elems / head_dim) must be a power of two";
  if (p->kv.head_dim * p->elem_bytes % 16 || p->kv.head_dim * p->elem_bytes > 4096) return "a head must be a multiple of 16 bytes, at most 4096";
  if (p->kv.block_elems * p->elem_bytes % 16 || p->kv.layer_elems * p->elem_bytes % 16 || p->kv.which_elems * p->elem_bytes % 16)
    return "KV strides must be multiples of 16 bytes";
  page_shift = 0;
  while ((int64_t{1} << page_shift) < tokens) ++page_shift;
  if (static_cast<int64_t>(p->kv.max_blocks) << page_shift > INT_MAX / 2) return "a slot's positions must stay below 2^30";
  if (static_cast<int64_t>(p->layers) * 2 * p->n_kv > 65536) return "too many layers and groups";
  if (!p->kv.arena || !p->kv.table || !p->refs || !p->free_bits || !p->errors || !p->work) return "missing pointer";
  if (reinterpret_cast<uintptr_t>(p->kv.arena) % 16) return "the arena must be 16-byte aligned";
  if (p->work_ints < work_ints(p->slots, p->kv.max_blocks, p->pages)) return "work is smaller than stride_kv_work_ints()";
  return nullptr;
}

int refused(const char* what, const char* why) { return fail(STRIDE_TC_EINVAL, std::string(what) + ": " + why); }

int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(static_cast<int>(e), std::string(what) + " launch failed: " + hipGetErrorString(e));
  return 0;
}

// Workgroups that share a page's runs: enough of them together to fill the chip.
int page_groups(const StrideKvPool& p, int n) {
  const int most = (p.layers * 2 * p.n_kv + 3) / 4;
  return std::max(1, std::min(most, 2048 / std::max(1, n)));
}

}  // namespace
}  // namespace stride_tc

using namespace stride_tc;

static_assert(sizeof(StrideKvPool) == 120 && offsetof(StrideKvPool, refs) == 56 && offsetof(StrideKvPool, pages) == 96, "KvPool layout");

extern "C" {

int64_t stride_kv_work_ints(int32_t slots, int32_t max_blocks, int32_t pages) {
  if (slots < 1 || max_blocks < 1 || pages < 1) return -1;
  return work_ints(slots, max_blocks, pages);
}

int stride_kv_reserve(const StrideKvPool* p, const int32_t* slot, const int32_t* first, const int32_t* end, int32_t n, void* stream) {
  int shift;
  if (const char* why = why_not(p, n, shift)) return refused("kv_reserve", why);
  if (n == 0) return 0;
  if (!slot || !first || !end) return refused("kv_reserve", "missing pointer");
  if (n > p->slots) return refused("kv_reserve", "more items than slots");
  hipLaunchKernelGGL(k_reserve, dim3(1), dim3(kPlan), 0, static_cast<hipStream_t>(stream), *p, slot, first, end, n);
  return launched("kv_reserve");
}

int stride_kv_release(const StrideKvPool* p, const int32_t* slot, const int32_t* first, const int32_t* end, int32_t n, void* stream) {
  int shift;
  if (const char* why = why_not(p, n, shift)) return refused("kv_release", why);
  if (n == 0) return 0;
  if (!slot || !first || !end) return refused("kv_release", "missing pointer");
  hipLaunchKernelGGL(k_release, dim3(n), dim3(256), 0, static_cast<hipStream_t>(stream), *p, slot, first, end);
  return launched("kv_release");
}

int stride_kv_fork(const StrideKvPool* p, const int32_t* src, const int32_t* dst, const int32_t* length, int32_t n, void* stream) {
  int shift;
  if (const char* why = why_not(p, n, shift)) return refused("kv_fork", why);
  if (n == 0) return 0;
  if (!src || !dst || !length) return refused("kv_fork", "missing pointer");
  if (n > p->slots) return refused("kv_fork", "more items than slots");
  hipStream_t st = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(k_fork_plan, dim3(1), dim3(kPlan), 0, st, *p, src, dst, length, n, shift);
  if (int rc = launched("kv_fork (plan)")) return rc;
  hipLaunchKernelGGL(k_fork_apply, dim3(n, page_groups(*p, n)), dim3(256), 0, st, *p, src, dst, length, shift);
  return launched("kv_fork");
}

int stride_kv_compact(const StrideKvPool* p, const int32_t* slot, const int32_t* first, const int32_t* count, const int32_t* keep,
                      int64_t keep_stride, int32_t width, int32_t n, void* stream) {
  int shift;
  if (const char* why = why_not(p, n, shift)) return refused("kv_compact", why);
  if (n == 0) return 0;
  if (!slot || !first || !count || (!keep && width != 0)) return refused("kv_compact", "missing pointer");
  if (n > p->slots) return refused("kv_compact", "more items than slots");
  if (keep_stride < 0 || width < 0) return refused("kv_compact", "keep_stride and width must not be negative");
  const int64_t runs = static_cast<int64_t>(p->layers) * 2 * p->n_kv;
  if (runs * n > INT_MAX) return refused("kv_compact", "too many items, layers and groups together");
  hipStream_t st = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(k_compact_plan, dim3(1), dim3(kPlan), 0, st, *p, slot, first, count, n, shift, width);
  if (int rc = launched("kv_compact (plan)")) return rc;
  hipLaunchKernelGGL((k_compact_move<4>), dim3(static_cast<unsigned>(runs * n)), dim3(256), 0, st, *p, slot, first, count, keep, keep_stride, n,
                     shift, p->kv.head_dim * p->elem_bytes / 16);
  if (int rc = launched("kv_compact (move)")) return rc;
  hipLaunchKernelGGL(k_compact_finish, dim3(n), dim3(256), 0, st, *p, slot, first, count, n, shift);
  return launched("kv_compact");
}

int stride_kv_copy(const StrideKvPool* p, const StrideKvPool* to, const int32_t* src, const int32_t* dst, const int32_t* tokens, int32_t n,
                   void* stream) {
  int shift, other;
  if (const char* why = why_not(p, n, shift)) return refused("kv_copy", why);
  if (!to) to = p;
  if (const char* why = why_not(to, n, other)) return refused("kv_copy (to)", why);
  if (to->layers != p->layers || to->n_kv != p->n_kv || to->elem_bytes != p->elem_bytes || to->kv.head_dim != p->kv.head_dim ||
      to->kv.block_elems != p->kv.block_elems || to->kv.layer_elems != p->kv.layer_elems || to->kv.which_elems != p->kv.which_elems ||
      to->kv.group_elems != p->kv.group_elems)
    return refused("kv_copy", "the two pools' pages differ in shape");
  if (n == 0) return 0;
  if (!src || !dst) return refused("kv_copy", "missing pointer");
  if ((to->pages + 31) / 32 > p->pages + p->slots) return refused("kv_copy", "the other pool is too large for this one's work");
  const int tokens_max = 1 << shift;
  hipStream_t st = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(k_copy_plan, dim3(1), dim3(kPlan), 0, st, *p, src, dst, tokens, n, to->pages, to->kv.arena == p->kv.arena ? 1 : 0, tokens_max);
  if (int rc = launched("kv_copy (plan)")) return rc;
  hipLaunchKernelGGL(k_copy, dim3(n, page_groups(*p, n)), dim3(256), 0, st, *p, static_cast<char*>(to->kv.arena), src, dst, tokens, tokens_max);
  return launched("kv_copy");
}

}  // extern "C"
