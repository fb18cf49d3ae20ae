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
#include <type_traits>

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
  lds_barrier();
  if (lane == 63) lds[wave] = x;
  lds_barrier();
  int base = 0;
  sum = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) base += lds[w];
    sum += lds[w];
  }
  return base + x - v;
}
// The same of truth values.
__device__ __forceinline__ int count_before_me(bool v, int* lds, int& sum) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint64_t all = __ballot(v);
  lds_barrier();
  if (lane == 0) lds[wave] = __popcll(all);
  lds_barrier();
  int base = 0;
  sum = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) base += lds[w];
    sum += lds[w];
  }
  return base + __popcll(all & ((uint64_t{1} << lane) - 1));
}

// Word w of the free pages' bit map, no bits behind the last page.
__device__ __forceinline__ uint32_t free_word(const StrideKvPool& p, int w) {
  const int words = (p.pages + 31) / 32;
  uint32_t bits = w < words ? p.free_bits[w] : 0u;
  if (w == words - 1 && (p.pages & 31)) bits &= (1u << (p.pages & 31)) - 1u;
  return bits;
}

// The lowest `want` free pages, in order, to `list`; `head` is the thread's own first word,
// which a plan fetches before anything else, and `left` what remains of it. False: there are
// fewer.
__device__ __forceinline__ bool list_free(const StrideKvPool& p, uint32_t head, int want, int32_t* list, int* lds, uint32_t& left) {
  const int words = (p.pages + 31) / 32;
  int have = 0;
  for (int w0 = 0; w0 < words && have < want; w0 += kPlan) {
    const int w = w0 + threadIdx.x;
    uint32_t bits = w0 == 0 ? head : free_word(p, w);
    int sum;
    int at = have + before_me(static_cast<int>(__popc(bits)), lds, sum);
    while (bits && at < want) {
      list[at++] = w * 32 + __ffs(bits) - 1;
      bits &= bits - 1;
    }
    if (w0 == 0) left = bits;
    have += sum;
  }
  __syncthreads();
  return have >= want;
}

// A page of the list is taken: its first reference. The first words' bits are cleared by the
// threads that hold them (close_head), not one by one.
__device__ __forceinline__ void take(const StrideKvPool& p, int page) {
  p.refs[page] = 1;
  if (page >= kPlan * 32) atomicAnd(&p.free_bits[page >> 5], ~(1u << (page & 31)));
}
__device__ __forceinline__ void close_head(const StrideKvPool& p, uint32_t head, uint32_t left) {
  if (left != head) p.free_bits[threadIdx.x] = left;
}

// Marks slot in the bit map of an LDS array; true where it was marked before.
__device__ __forceinline__ bool mark(uint32_t* bits, int slot) {
  return (atomicOr(&bits[slot >> 5], 1u << (slot & 31)) >> (slot & 31)) & 1u;
}
__device__ __forceinline__ bool marked(const uint32_t* bits, int slot) { return (bits[slot >> 5] >> (slot & 31)) & 1u; }

// Ends a plan's checks. True: no thread found anything bad. (Else the call ends here: work[0]
// is 0 since the plan's start.)
__device__ __forceinline__ bool agree(const StrideKvPool& p, int bad, int* lds) {
  if (bad) atomicOr(p.errors, bad);
  int sum;
  count_before_me(bad != 0, lds, sum);
  return sum == 0;
}

// What a plan workgroup keeps of a call of few items: their table ranges, and the pages that
// it hands out.
constexpr int kFewItems = kPlan;
constexpr int kFewEach = 4;  // table entries a thread
constexpr int kFewPages = 2048;
struct Few {
  int slot[kFewItems], lo[kFewItems], before[kFewItems];  // before: entries of the items before
  int32_t pages[kFewPages];
};

// The plan of reserve and compact, for item i with table range [lo, hi) of `slot` (the thread's
// own one: item threadIdx.x, and `range` for any): an entry wants a page where `wants(entry)`,
// and `give(i, slot, b, page)` takes it (page < 0: the entry stays). Two ways to the same outcome.
// Few items and entries: the entries of all items in a row over the threads, each read once and
// kept (64 items of one entry: a reserve takes 5 us so, 13 the other way, which reads them twice
// and waits for one item after the other). Else a wave an item, counts first.
template <class Range, class Wants, class Give>
__device__ __forceinline__ void share_out(const StrideKvPool& p, int n, uint32_t head, int* lds, Few& few, int slot0, int lo0, int hi0, Range range,
                                          Wants wants, Give give) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (n <= kFewItems) {
    constexpr int kMost = kPlan * kFewEach;
    int entries;
    const int size = static_cast<int>(threadIdx.x) < n ? max(0, min(hi0 - lo0, kMost + 1)) : 0;  // exact where they are few
    const int before = before_me(size, lds, entries);
    few.slot[threadIdx.x] = slot0, few.lo[threadIdx.x] = lo0, few.before[threadIdx.x] = before;
    lds_barrier();
    if (entries <= kMost) {
      int item[kFewEach], at[kFewEach], entry[kFewEach], place[kFewEach], total = 0;
      bool want[kFewEach];
      const int rounds = (entries + kPlan - 1) / kPlan;
#pragma unroll
      for (int x = 0; x < kFewEach; ++x) {
        const int e = x * kPlan + threadIdx.x;
        item[x] = -1;
        if (x >= rounds || e >= entries) continue;
        int a = 0, z = n;  // the last item with before <= e
        while (z - a > 1) {
          const int m = (a + z) / 2;
          if (few.before[m] <= e) a = m;
          else z = m;
        }
        item[x] = a;
        at[x] = few.lo[a] + e - few.before[a];
        entry[x] = table_row(p, few.slot[a])[at[x]];
      }
#pragma unroll
      for (int x = 0; x < kFewEach; ++x) want[x] = item[x] >= 0 && wants(entry[x]);
#pragma unroll
      for (int x = 0; x < kFewEach; ++x) {
        if (x >= rounds) continue;
        int sum;
        place[x] = total + count_before_me(want[x], lds, sum);
        total += sum;
      }
      int32_t* list = total <= kFewPages ? few.pages : free_list(p);
      uint32_t left = head;
      if (total > 0 && !list_free(p, head, total, list, lds, left)) {
        if (threadIdx.x == 0) atomicOr(p.errors, STRIDE_KV_NO_PAGES);
        return;
      }
      close_head(p, head, left);
      if (threadIdx.x == 0) p.work[0] = 1;
#pragma unroll
      for (int x = 0; x < kFewEach; ++x) {
        if (item[x] < 0) continue;
        const int page = want[x] ? list[place[x]] : -1;
        if (page >= 0) take(p, page);
        give(item[x], few.slot[item[x]], at[x], page);
      }
      return;
    }
  }
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
  uint32_t left = head;
  if (total > 0 && !list_free(p, head, total, free_list(p), lds, left)) {
    if (threadIdx.x == 0) atomicOr(p.errors, STRIDE_KV_NO_PAGES);
    return;
  }
  close_head(p, head, left);
  if (threadIdx.x == 0) p.work[0] = 1;
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
      if (b < hi) give(i, slot, b, page);
      at += __popcll(all);
    }
  }
}

__global__ __launch_bounds__(kPlan) void k_reserve(StrideKvPool p, const int32_t* slots, const int32_t* first, const int32_t* end, int n) {
  __shared__ uint32_t bits[kMaxSlots / 32];
  __shared__ int lds[kWaves];
  __shared__ Few few;
  const uint32_t head = free_word(p, threadIdx.x);
  int slot0 = 0, lo0 = 0, hi0 = 0;
  auto range = [&](int i, int& s, int& lo, int& hi) { s = slots[i], lo = first[i], hi = end[i]; };
  if (static_cast<int>(threadIdx.x) < n) range(threadIdx.x, slot0, lo0, hi0);
  for (int i = threadIdx.x; i < (p.slots + 31) / 32; i += kPlan) bits[i] = 0;
  lds_barrier();
  int bad = 0;
  for (int i = threadIdx.x; i < n; i += kPlan) {
    int s = slot0, lo = lo0, hi = hi0;
    if (i >= kPlan) range(i, s, lo, hi);
    if (s < 0 || s >= p.slots || lo < 0 || hi > p.kv.max_blocks) bad |= STRIDE_KV_BAD_ITEM;
    else if (mark(bits, s)) bad |= STRIDE_KV_TWICE;
  }
  if (!agree(p, bad, lds)) return;
  share_out(p, n, head, lds, few, slot0, lo0, hi0, range, [](int b) { return b < 0; }, [&](int, int s, int b, int page) {
    if (page >= 0) table_row(p, s)[b] = page;
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
  const uint32_t head = free_word(p, threadIdx.x);
  int a0 = 0, b0 = 0, len0 = 0;
  if (static_cast<int>(threadIdx.x) < n) a0 = src[threadIdx.x], b0 = dst[threadIdx.x], len0 = length[threadIdx.x];
  for (int i = threadIdx.x; i < (p.slots + 31) / 32; i += kPlan) to[i] = 0;
  if (threadIdx.x == 0) p.work[0] = 0;
  lds_barrier();
  int bad = 0;
  for (int i = threadIdx.x; i < n; i += kPlan) {
    int a = a0, b = b0, len = len0;
    if (i >= kPlan) a = src[i], b = dst[i], len = length[i];
    if (a < 0 || a >= p.slots || b < 0 || b >= p.slots || len < 0 || len > static_cast<int64_t>(p.kv.max_blocks) << page_shift)
      bad |= STRIDE_KV_BAD_ITEM;
    else if (mark(to, b)) bad |= STRIDE_KV_TWICE;
  }
  lds_barrier();
  for (int i = threadIdx.x; i < n; i += kPlan) {
    const int a = i >= kPlan ? src[i] : a0;
    if (a >= 0 && a < p.slots && marked(to, a)) bad |= STRIDE_KV_TWICE;
  }
  if (!agree(p, bad, lds)) return;
  int total = 0;
  for (int i0 = 0; i0 < n; i0 += kPlan) {
    const int i = i0 + threadIdx.x;
    int a = a0, len = len0;
    if (i0 > 0 && i < n) a = src[i], len = length[i];
    const bool w = i < n && (len & ((1 << page_shift) - 1)) && is_page(p, table_row(p, a)[len >> page_shift]);
    int sum;
    const int at = total + count_before_me(w, lds, sum);
    if (i < n) item_work(p)[i] = w ? at : -1;
    total += sum;
  }
  uint32_t left = head;
  if (total > 0 && !list_free(p, head, total, free_list(p), lds, left)) {
    if (threadIdx.x == 0) atomicOr(p.errors, STRIDE_KV_NO_PAGES);
    return;
  }
  close_head(p, head, left);
  __syncthreads();
  if (threadIdx.x == 0) p.work[0] = 1;
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

// Copies the first `bytes` of every run of a page; a wave takes runs r0, r0 + step, .. (64
// branches, part pages of 8 tokens on average, 16 layers of 8 groups of 64: 7.5 us with the table, 4.5 TB/s.)
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
                                                        const int32_t* keep, int64_t keep_stride, int n, int page_shift, int width) {
  __shared__ uint32_t bits[kMaxSlots / 32];
  __shared__ int lds[kWaves];
  __shared__ Few few;
  const uint32_t head = free_word(p, threadIdx.x);
  // the pages that kept positions move into
  auto pages = [&](int f, int c, int& lo, int& hi) {
    lo = f >> page_shift;
    hi = c ? (f + c + (1 << page_shift) - 1) >> page_shift : lo;
  };
  int slot0 = 0, f0 = 0, c0 = 0;
  if (static_cast<int>(threadIdx.x) < n) slot0 = slots[threadIdx.x], f0 = first[threadIdx.x], c0 = count[threadIdx.x];
  auto in_bounds = [&](int s, int f, int c) {
    return s >= 0 && s < p.slots && f >= 0 && c >= 0 && c <= width &&
           static_cast<int64_t>(f) + c <= static_cast<int64_t>(p.kv.max_blocks) << page_shift;
  };
  __shared__ int longest;
  few.slot[threadIdx.x] = slot0, few.lo[threadIdx.x] = f0, few.before[threadIdx.x] = in_bounds(slot0, f0, c0) ? c0 : 0;
  if (threadIdx.x == 0) longest = 0;
  for (int i = threadIdx.x; i < (p.slots + 31) / 32; i += kPlan) bits[i] = 0;
  if (threadIdx.x == 0) p.work[0] = 0;
  lds_barrier();
  int bad = 0, most = 0;
  for (int i = threadIdx.x; i < n; i += kPlan) {
    int s = slot0, f = f0, c = c0;
    if (i >= kPlan) s = slots[i], f = first[i], c = count[i];
    if (!in_bounds(s, f, c)) {
      bad |= STRIDE_KV_BAD_ITEM;
      continue;
    }
    if (mark(bits, s)) bad |= STRIDE_KV_TWICE;
    if (c > most) most = c;
  }
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) most = max(most, __shfl_xor(most, d));
  if ((threadIdx.x & 63) == 0) atomicMax(&longest, most);
  lds_barrier();
  // Every kept position has a page, or the call ends here: the move would leave its place with
  // what was there, in a fresh page another sequence's. (Whether a list ascends is seen while it
  // is moved: then every place still gets an entry of the slot's.) One workgroup looks up all
  // lists, up to eight positions a thread at a time, and without branches around the loads, for
  // which there is always an address that may be read (64 lists of 4 positions: 1.0 us of the
  // plan's 5.7; 8 lists of 2044: 6.3 of 12.0).
  if (longest > 0) {
    const int wide = longest, step_item = kPlan / wide, step_k = kPlan % wide, cap = p.kv.max_blocks << page_shift;
    int item = static_cast<int>(threadIdx.x) / wide, at = static_cast<int>(threadIdx.x) % wide;
    auto look_up = [&](auto many) __attribute__((always_inline)) {
      constexpr int U = decltype(many)::value;
      int least[U], src[U], page[U];
      const int32_t *list[U], *entry[U];
#pragma unroll
      for (int x = 0; x < U; ++x) {
        const int i = min(item, n - 1);
        int s, f, c;
        if (n <= kFewItems) s = few.slot[i], f = few.lo[i], c = few.before[i];
        else s = slots[i], f = first[i], c = in_bounds(s, f, count[i]) ? count[i] : 0;
        const bool wanted = item < n && at < c;
        list[x] = wanted ? keep + i * keep_stride + at : slots;
        entry[x] = wanted ? table_row(p, s) : p.work;
        least[x] = wanted ? f + at : -1;
        item += step_item, at += step_k;
        if (at >= wide) at -= wide, ++item;
      }
#pragma unroll
      for (int x = 0; x < U; ++x) src[x] = *list[x];
#pragma unroll
      for (int x = 0; x < U; ++x) {
        const bool inside = src[x] >= least[x] && src[x] < cap;
        if (least[x] >= 0 && !inside) bad |= STRIDE_KV_BAD_KEEP;
        if (!inside) least[x] = -1;
        page[x] = entry[x][least[x] >= 0 ? src[x] >> page_shift : 0];
      }
#pragma unroll
      for (int x = 0; x < U; ++x)
        if (least[x] >= 0 && !is_page(p, page[x])) bad |= STRIDE_KV_MISSING;
    };
    if (static_cast<int64_t>(n) * wide <= kPlan) look_up(std::integral_constant<int, 1>{});
    else
      while (item < n) look_up(std::integral_constant<int, 8>{});
  }
  if (!agree(p, bad, lds)) return;
  int lo0, hi0;
  pages(f0, c0, lo0, hi0);
  share_out(
      p, n, head, lds, few, slot0, lo0, hi0,
      [&](int i, int& s, int& lo, int& hi) {
        s = slots[i];
        pages(first[i], count[i], lo, hi);
      },
      [&](int b) { return !is_page(p, b) || p.refs[b] > 1; }, [&](int i, int, int b, int page) { new_row(p, n, i)[b] = page; });
}

// Moves runs (a layer, K or V, a group) of an item's kept positions: `group` runs a workgroup,
// `step` positions at a time, at most kHold 16-byte pieces a thread. In place it must not write
// what is still to be read: positions ascend and each comes from its own place or a later one,
// so a workgroup that takes them in ascending steps, loads a step whole before it writes it,
// overwrites only what it has read. While a step's pieces are on their way the next one's pages
// are looked up, one position a thread, and left in LDS for the threads that share it. (8
// sequences, 2048 of 4096 positions, 16 layers of 8 groups of 64: 212 us, 4.4 TB/s; a 4 GiB
// copy: 4.8. 64 sequences, 4 of 16 positions: 7 us.)
constexpr int kHold = 8;
constexpr int kStepMax = 256;

__global__ __launch_bounds__(256) void k_compact_move(StrideKvPool p, const int32_t* slots, const int32_t* first, const int32_t* count,
                                                      const int32_t* keep, int64_t keep_stride, int n, int page_shift, int pieces, int step,
                                                      int group) {
  if (p.work[0] == 0) return;
  __shared__ int64_t from[2][kStepMax], to[2][kStepMax];  // byte offsets of a position in its run's arena; below 0: nothing
  __shared__ int64_t run_at[256];
  const Runs runs = runs_of(p);
  const int groups = (runs.count + group - 1) / group;
  const int i = blockIdx.x / groups, run0 = blockIdx.x % groups * group, t = threadIdx.x;
  const int begin = first[i], many = count[i], in_page = (1 << page_shift) - 1;
  if (many == 0) return;
  const int32_t* row = table_row(p, slots[i]);
  const int32_t* fresh = new_row(p, n, i);
  const int32_t* list = keep + i * keep_stride;
  char* arena = static_cast<char*>(p.kv.arena);
  const int64_t block = p.kv.block_elems * p.elem_bytes;
  const int cap = p.kv.max_blocks << page_shift, row_bytes = pieces * 16;
  // a page that is replaced takes along what it holds before `begin`
  const int lead = fresh[begin >> page_shift] >= 0 ? begin & in_page : 0;
  int bad = 0;
  auto look = [&](int k0, int b) {
    const int k = k0 + t;
    if (t >= step) return;
    int64_t f = -1, d = -1;
    if (k < many) {
      const int pos = begin + k, src = k < 0 ? pos : list[k];
      const int here = row[pos >> page_shift], other = fresh[pos >> page_shift];
      if (k > 0 && list[k - 1] >= src) bad |= STRIDE_KV_BAD_KEEP;
      const int page = src >= 0 && src < cap ? row[src >> page_shift] : -1;  // (before `first` there may be none)
      if (is_page(p, page)) {
        f = page * block + static_cast<int64_t>(src & in_page) * row_bytes;
        d = (other >= 0 ? other : here) * block + static_cast<int64_t>(pos & in_page) * row_bytes;
      }
    }
    from[b][t] = f;
    to[b][t] = d;
  };
  // this thread's pieces: of rows m, m + per, .. of the workgroup's (run, position) rows
  const int per = 256 / pieces, in = t % pieces * 16, row0 = t / pieces;
  const int rows = row0 < per ? min(group, runs.count - run0) * step : 0;
  const float rcp = 1.0f / static_cast<float>(step);
  if (t < min(group, runs.count - run0)) run_at[t] = runs.at(run0 + t);
  __syncthreads();
  int64_t base[kHold];
  int place[kHold];
#pragma unroll
  for (int u = 0; u < kHold; ++u) {
    const int m = row0 + u * per, r = static_cast<int>((static_cast<float>(m) + 0.5f) * rcp);  // m < 2048: exact
    place[u] = m < rows ? m - r * step : -1;
    base[u] = m < rows ? run_at[r] + in : 0;
  }
  look(-lead, 0);
  __syncthreads();
  int b = 0;
  for (int k0 = -lead; k0 < many; k0 += step, b ^= 1) {
    u32x4 v[kHold];
    int64_t d[kHold];  // taken before the barrier: after it the other waves write the next step's
#pragma unroll
    for (int u = 0; u < kHold; ++u) {
      const int64_t f = place[u] >= 0 ? from[b][place[u]] : -1;
      d[u] = f >= 0 ? to[b][place[u]] : -1;
      if (f >= 0) v[u] = load16(arena + base[u] + f);
    }
    if (k0 + step < many) look(k0 + step, b ^ 1);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the step is read before any wave writes it
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kHold; ++u)
      if (d[u] >= 0) *reinterpret_cast<u32x4*>(arena + base[u] + d[u]) = v[u];
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
  if (threadIdx.x == 0) p.work[0] = 0;
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
  if (agree(p, bad, lds) && threadIdx.x == 0) p.work[0] = 1;
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
  if (p->kv.group_elems * p->elem_bytes > int64_t{1} << 30) return "a head's part of a page must not pass 2^30 bytes";  // counted in 32 bits
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
  hipLaunchKernelGGL(k_compact_plan, dim3(1), dim3(kPlan), 0, st, *p, slot, first, count, keep, keep_stride, n, shift, width);
  if (int rc = launched("kv_compact (plan)")) return rc;
  // Positions a step and runs a workgroup: short lists (a few accepted tokens) share a
  // workgroup's threads, and its lookups, between runs.
  const int pieces = p->kv.head_dim * p->elem_bytes / 16, most = 256 / pieces * kHold;
  const int step = static_cast<int>(std::min<int64_t>(std::min(kStepMax, most), std::max<int64_t>(1, static_cast<int64_t>(width) + (1 << shift) - 1)));
  const int group = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(runs, 256), most / step)));
  hipLaunchKernelGGL(k_compact_move, dim3(static_cast<unsigned>((runs + group - 1) / group * n)), dim3(256), 0, st, *p, slot, first, count, keep,
                     keep_stride, n, shift, pieces, step, group);
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
