// Blocks of 4 and 8 bits: quantisation of 16 x 16 tiles, their values, and RMSNorm with the
// residual's addition (include/stride_mx.h). All of them move each value once and are bound by
// memory.
//
// A wave has R = 1, 2 or 4 rows of 4 / R chunks of 128 columns: a lane has 8 columns, half l % 2 of
// tile l / (2 R), row l / 2 % R, so that 2 R lanes read neighbouring 16-column pieces of the rows. A
// block of 32 is then the two tiles of lanes that differ in bits 0 and 2 R.
#include <hip/hip_runtime.h>

#include <climits>
#include <cstddef>

#include "mx_common.hpp"
#include "tc_epilogue.hpp"

namespace stride_tc {
namespace {

template <int R>
struct Spot {  // a lane's place in its wave's values
  int row, chunk, tile, half;
  __device__ __forceinline__ Spot() {
    const int l = threadIdx.x & 63;
    half = l & 1;
    row = (l >> 1) % R;
    tile = l / (2 * R) & 7;
    chunk = l / (16 * R);
  }
};

template <int R>
__device__ __forceinline__ uint32_t block_most(const float (&v)[8]) {
  uint32_t m = mx_abs_bits(v[0]);
#pragma unroll
  for (int i = 1; i < 8; ++i) m = max(m, mx_abs_bits(v[i]));
  m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), 1)));
  return max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), 2 * R)));
}

// A lane's values of chunk kc, row `row` of tile t, to codes and scales. Whole waves call it.
template <int BITS, int R>
__device__ __forceinline__ void store_block(const StrideMxTiles& out, int t, int kc, int row, const Spot<R>& s, const float (&v)[8], bool live) {
  const int groups = mx_groups(out.cols);
  const int byte = mx_scale_byte<BITS>(block_most<R>(v));
  const float inverse = mx_inverse(byte);
  if (!live) return;
  const int64_t chunk = static_cast<int64_t>(t) * groups * 4 + kc;
  const int blk = s.tile >> 1;
  if constexpr (BITS == 4) {
    const uint32_t w = byte == 255 ? 0u : mx_pack4(v, inverse);
    *reinterpret_cast<uint32_t*>(out.codes + chunk * kCode4Bytes + (blk * 16 + row) * 16 + (s.tile & 1) * 8 + s.half * 4) = w;
  } else {
    u32x2 w = {mx_pack8(v[0], v[1], v[2], v[3], inverse), mx_pack8(v[4], v[5], v[6], v[7], inverse)};
    if (byte == 255) w = u32x2{0x7F7F7F7Fu, 0x7F7F7F7Fu};
    *reinterpret_cast<u32x2*>(out.codes + chunk * kCode8Bytes + (s.tile * 16 + row) * 16 + s.half * 8) = w;
  }
  if (!s.half && !(s.tile & 1))
    out.scales[(static_cast<int64_t>(t) * groups + (kc >> 2)) * kScaleBytes + (blk * 16 + row) * 4 + (kc & 3)] = static_cast<uint8_t>(byte);
}

template <class T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    const f32x4 a = reinterpret_cast<const f32x4*>(p)[0], b = reinterpret_cast<const f32x4*>(p)[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
  } else {
    const u32x4 w = load16(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[2 * i] = f32_of(w[i] << 16), v[2 * i + 1] = f32_of(w[i] & 0xFFFF0000u);
  }
}

// Workgroup: a chunk of a tile, a wave for each four rows. (16384 x 2048 in bf16 to 4 bits 16 us, 5.3
// TB/s; 128 x 2048 to 8 bits 2.6. A group a workgroup, with its scales as words: 16.6 and 3.7.)
template <int BITS, class T>
__global__ __launch_bounds__(256) void k_quantize(const T* src, StrideMxTiles out, int rows, int chunks) {
  const Spot<4> s;
  const int kc = blockIdx.x % chunks, t = blockIdx.x / chunks, row = (threadIdx.x >> 6) * 4 + s.row;
  const int col_tiles = out.cols >> 4, ct = kc * 8 + s.tile;
  const bool live = t * 16 + row < rows;
  float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  if (live && ct < col_tiles) load8(src + (static_cast<int64_t>(t) * col_tiles + ct) * kTileElems + row * 16 + s.half * 8, v);
  store_block<BITS>(out, t, kc, row, s, v, live);
}

// Workgroup: C chunks of a tile, a whole group or one; a wave has four rows, a lane 8 columns of one in
// each. (16384 x 2048 from 4 bits to bf16 with C = 4 / 1: 17.6 / 20.2 us of GPU, 4.8 TB/s; 1008 x 1040 4.2 /
// 3.7 a call in a graph: a group's worth of stores pays where workgroups are many.)
template <int BITS, class T, int C>
__global__ __launch_bounds__(256) void k_dequantize(StrideMxTiles in, T* out, int64_t stride, int rows, int groups) {
  const int all = groups * (4 / C), g = blockIdx.x % all / (4 / C), first = blockIdx.x % (4 / C), t = blockIdx.x / all;
  const int l = threadIdx.x & 63, part = l & 15, blk = part >> 2, row = (threadIdx.x >> 6) * 4 + (l >> 4);
  const int64_t at = static_cast<int64_t>(t) * 16 + row;
  if (at >= rows) return;
  const int64_t group = static_cast<int64_t>(t) * groups + g;
  const uint32_t scales = *reinterpret_cast<const uint32_t*>(in.scales + group * kScaleBytes + (blk * 16 + row) * 4);
  u32x2 code[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int64_t chunk = group * 4 + first + c;
    if constexpr (BITS == 4) code[c][0] = *reinterpret_cast<const uint32_t*>(in.codes + chunk * kCode4Bytes + (blk * 16 + row) * 16 + (part & 3) * 4);
    else code[c] = *reinterpret_cast<const u32x2*>(in.codes + chunk * kCode8Bytes + ((part >> 1) * 16 + row) * 16 + (part & 1) * 8);
  }
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int col = g * kMxGroup + (first + c) * kMxChunk + part * 8;
    if (col >= in.cols) return;
    float v[8];
    if constexpr (BITS == 4) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t n = (code[c][0] >> (4 * i)) & 15u, e = (n >> 1) & 3u, m = n & 1u;
        const uint32_t bits = e ? ((e + 126u) << 23) | (m << 22) : (m ? 0x3F000000u : 0u);
        v[i] = f32_of(bits | (n >> 3) << 31);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int w = static_cast<int>(code[c][i]);
        const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
        v[4 * i] = a[0], v[4 * i + 1] = a[1], v[4 * i + 2] = b[0], v[4 * i + 3] = b[1];
      }
    }
    const int byte = (scales >> (8 * (first + c))) & 255u;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = byte == 255 ? f32_of(0x7FC00000u) : ldexpf(v[i], byte - 127);
    T* o = out + at * stride + col;
    if constexpr (sizeof(T) == 4) {
      __builtin_nontemporal_store(f32x4{v[0], v[1], v[2], v[3]}, reinterpret_cast<f32x4*>(o));
      __builtin_nontemporal_store(f32x4{v[4], v[5], v[6], v[7]}, reinterpret_cast<f32x4*>(o) + 1);
    } else {
      u32x4 w;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = bf16_rne(v[2 * i]) | bf16_rne(v[2 * i + 1]) << 16;
      __builtin_nontemporal_store(w, reinterpret_cast<u32x4*>(o));
    }
  }
}

// bf16_rne, and NaN whatever its payload (h may hold any).
__device__ __forceinline__ uint32_t bf16_of(float v) { return v != v ? 0x7FC0u : bf16_rne(v); }

// Workgroup: R rows of a lane tile; a lane's values stay in registers between the sum and the
// scaling (IT places; 0: h is read again). A row's sum has the same order for every R: a chunk's
// pieces of 8 by halves and tiles, then its chunks 16 apart ascending, and those by halves again.
template <int R, int IT, bool ADD, bool MX>
__global__ __launch_bounds__(1024) void k_mx_norm(StrideMxNormParams p, int chunks) {
  extern __shared__ float sums[];  // [R][chunks]
  const Spot<R> s;
  constexpr int per = 4 / R;  // chunks of a wave
  const int b = R < 4 ? xcd_remap(blockIdx.x, gridDim.x) : blockIdx.x;  // rows that share lines, on one XCD
  const int t = b / (16 / R), row = b % (16 / R) * R + s.row;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int col_tiles = p.dim >> 4;
  const bool live = t * 16 + row < p.l.rows;
  const int64_t at = static_cast<int64_t>(t) * col_tiles * kTileElems + row * 16 + s.half * 8;
  float v[IT ? IT : 1][8];
  constexpr bool kEarly = IT == 1 || IT == 2;  // the gains come beside the values
  float gain[kEarly ? IT : 1][8];
  auto chunk_of = [&](int i) { return (wave + i * waves) * per + s.chunk; };
  auto fetch = [&](int kc, float (&x)[8], bool again) {
    const int ct = kc * 8 + s.tile;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = 0.0f;
    if (!live || ct >= col_tiles) return;
    float* h = p.h + at + static_cast<int64_t>(ct) * kTileElems;
    load8(h, x);
    if (ADD && !again) {
      float a[8];
      load8(p.add + at + static_cast<int64_t>(ct) * kTileElems, a);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] += a[i];
      reinterpret_cast<f32x4*>(h)[0] = f32x4{x[0], x[1], x[2], x[3]};
      reinterpret_cast<f32x4*>(h)[1] = f32x4{x[4], x[5], x[6], x[7]};
    }
  };
  auto square = [&](int kc, const float (&x)[8]) {
    float sum = x[0] * x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) sum = fmaf(x[i], x[i], sum);
#pragma unroll
    for (int d : {1, 2 * R, 4 * R, 8 * R}) sum += __shfl_xor(sum, d);
    if (!s.half && s.tile == 0 && kc < chunks) sums[s.row * chunks + kc] = sum;
  };
  if constexpr (IT > 0) {
#pragma unroll
    for (int i = 0; i < IT; ++i) fetch(chunk_of(i), v[i], false);
    if constexpr (kEarly) {
#pragma unroll
      for (int i = 0; i < IT; ++i) load8(p.weight + min(chunk_of(i) * 8 + s.tile, col_tiles - 1) * 16 + s.half * 8, gain[i]);
    }
#pragma unroll
    for (int i = 0; i < IT; ++i) square(chunk_of(i), v[i]);
  } else {
    for (int i = 0; i * waves * per < chunks; ++i) {
      fetch(chunk_of(i), v[0], false);
      square(chunk_of(i), v[0]);
    }
  }
  __syncthreads();
  float sum = 0.0f;  // sixteen lanes a row
  for (int c = lane & 15; c < chunks; c += 16) sum += sums[((lane >> 4) % R) * chunks + c];
#pragma unroll
  for (int d = 1; d < 16; d <<= 1) sum += __shfl_xor(sum, d);
  const float inverse = __shfl(1.0f / sqrtf(sum / static_cast<float>(p.dim) + p.eps), s.row * 16);
  auto scale = [&](int kc, float (&x)[8], float (&g)[8]) {
    const int ct = kc * 8 + s.tile;
    if (ct < col_tiles) {
      if constexpr (!kEarly) load8(p.weight + ct * 16 + s.half * 8, g);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = g[i] * (x[i] * inverse);
    }
    if constexpr (MX) {
      store_block<8>(p.out, t, kc, row, s, x, live && kc < chunks);
    } else if (live && ct < col_tiles) {
      u32x4 w;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = bf16_of(x[2 * i]) | bf16_of(x[2 * i + 1]) << 16;
      *reinterpret_cast<u32x4*>(p.x + at + static_cast<int64_t>(ct) * kTileElems) = w;
    }
  };
  if constexpr (IT > 0) {
#pragma unroll
    for (int i = 0; i < IT; ++i) scale(chunk_of(i), v[i], gain[kEarly ? i : 0]);
  } else {
    for (int i = 0; i * waves * per < chunks; ++i) {
      fetch(chunk_of(i), v[0], true);
      scale(chunk_of(i), v[0], gain[0]);
    }
  }
}

template <int BITS, class T>
void launch_values(const StrideMxDequantizeParams& p, int groups, hipStream_t st) {
  T* out = static_cast<T*>(p.out);
  const int all = groups * p.l.lane_groups;
  if (all >= 1024) hipLaunchKernelGGL((k_dequantize<BITS, T, 4>), dim3(all), dim3(256), 0, st, p.in, out, p.out_stride, p.l.rows, groups);
  else hipLaunchKernelGGL((k_dequantize<BITS, T, 1>), dim3(all * 4), dim3(256), 0, st, p.in, out, p.out_stride, p.l.rows, groups);
}

template <int R, int IT>
void launch_norm(const StrideMxNormParams& p, int chunks, int waves, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>((static_cast<int64_t>(p.l.rows) + R - 1) / R)), block(waves * 64);
  const unsigned lds = R * chunks * sizeof(float);
  const bool mx = p.out.codes != nullptr;
  if (p.add && mx) hipLaunchKernelGGL((k_mx_norm<R, IT, true, true>), grid, block, lds, st, p, chunks);
  else if (p.add) hipLaunchKernelGGL((k_mx_norm<R, IT, true, false>), grid, block, lds, st, p, chunks);
  else if (mx) hipLaunchKernelGGL((k_mx_norm<R, IT, false, true>), grid, block, lds, st, p, chunks);
  else hipLaunchKernelGGL((k_mx_norm<R, IT, false, false>), grid, block, lds, st, p, chunks);
}

template <int R>
void launch_norm(const StrideMxNormParams& p, int chunks, hipStream_t st) {
  const int places = (chunks * R + 3) / 4, waves = places < 16 ? places : 16, rounds = (places + waves - 1) / waves;
  if (rounds == 1) launch_norm<R, 1>(p, chunks, waves, st);
  else if (rounds == 2) launch_norm<R, 2>(p, chunks, waves, st);
  else if (rounds <= 4) launch_norm<R, 4>(p, chunks, waves, st);
  else launch_norm<R, 0>(p, chunks, waves, st);
}

}  // namespace
}  // namespace stride_tc

using namespace stride_tc;

static_assert(sizeof(StrideMxTiles) == 24, "MxTiles layout");
static_assert(sizeof(StrideMxQuantizeParams) == 56 && sizeof(StrideMxDequantizeParams) == 64, "MxQuantizeParams layout");
static_assert(sizeof(StrideMxNormParams) == 80 && offsetof(StrideMxNormParams, dim) == 72, "MxNormParams layout");

extern "C" {

int64_t stride_mx_code_bytes(int32_t cols, int32_t bits) {
  if (cols <= 0 || cols % 16 || cols > (1 << 20) || (bits != 4 && bits != 8)) return -1;
  return static_cast<int64_t>(mx_groups(cols)) * 4 * (bits == 4 ? kCode4Bytes : kCode8Bytes);
}

int64_t stride_mx_scale_bytes(int32_t cols) {
  if (cols <= 0 || cols % 16 || cols > (1 << 20)) return -1;
  return static_cast<int64_t>(mx_groups(cols)) * kScaleBytes;
}

int stride_mx_quantize(const StrideMxQuantizeParams* p, void* stream) {
  const char* what = "mx_quantize";
  if (!p) return mx_refused(what, "null parameters");
  if (!mx_lanes_ok(p->l)) return mx_refused(what, "need rows >= 0 and lane_groups = ceil(rows/16)");
  if ((p->bits != 4 && p->bits != 8) || (p->src_bytes != 2 && p->src_bytes != 4)) return mx_refused(what, "bits are 4 or 8, a source's bytes 2 or 4");
  if (p->l.rows == 0) return 0;
  if (const char* why = mx_why_not(p->out, p->l.lane_groups, 0)) return mx_refused(what, why);
  if (!p->src || reinterpret_cast<uintptr_t>(p->src) % 16) return mx_refused(what, "src must be there, 16-byte aligned");
  const int chunks = mx_groups(p->out.cols) * 4;
  const int64_t all = static_cast<int64_t>(chunks) * p->l.lane_groups;
  if (all > 4 * kMxMostGroups) return mx_refused(what, "rows and cols are too large together");
  const int64_t lt = p->l.lane_groups;
  if (mx_overlap({mx_codes(p->out, lt, p->bits), mx_scales(p->out, lt)}, {{p->src, lt * kTileElems * (p->out.cols / 16) * p->src_bytes}}))
    return mx_refused(what, "out and src must not overlap");
  const dim3 grid(static_cast<unsigned>(all)), block(256);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const uint16_t* half = static_cast<const uint16_t*>(p->src);
  const float* full = static_cast<const float*>(p->src);
  if (p->bits == 4 && p->src_bytes == 2) hipLaunchKernelGGL((k_quantize<4, uint16_t>), grid, block, 0, st, half, p->out, p->l.rows, chunks);
  else if (p->bits == 4) hipLaunchKernelGGL((k_quantize<4, float>), grid, block, 0, st, full, p->out, p->l.rows, chunks);
  else if (p->src_bytes == 2) hipLaunchKernelGGL((k_quantize<8, uint16_t>), grid, block, 0, st, half, p->out, p->l.rows, chunks);
  else hipLaunchKernelGGL((k_quantize<8, float>), grid, block, 0, st, full, p->out, p->l.rows, chunks);
  return mx_launched(what);
}

int stride_mx_dequantize(const StrideMxDequantizeParams* p, void* stream) {
  const char* what = "mx_dequantize";
  if (!p) return mx_refused(what, "null parameters");
  if (!mx_lanes_ok(p->l)) return mx_refused(what, "need rows >= 0 and lane_groups = ceil(rows/16)");
  if ((p->bits != 4 && p->bits != 8) || (p->out_bytes != 2 && p->out_bytes != 4)) return mx_refused(what, "bits are 4 or 8, a result's bytes 2 or 4");
  if (p->l.rows == 0) return 0;
  if (const char* why = mx_why_not(p->in, p->l.lane_groups, 0)) return mx_refused(what, why);
  if (!p->out || reinterpret_cast<uintptr_t>(p->out) % 16) return mx_refused(what, "out must be there, 16-byte aligned");
  if (p->out_stride < p->in.cols || p->out_stride % 8) return mx_refused(what, "out_stride must be a multiple of 8, at least cols");
  if (p->out_stride > INT64_MAX / 8 / p->l.rows) return mx_refused(what, "out_stride is too large for the rows");
  const int groups = mx_groups(p->in.cols);
  if (static_cast<int64_t>(groups) * 4 * p->l.lane_groups > 4 * kMxMostGroups) return mx_refused(what, "rows and cols are too large together");
  const int64_t lt = p->l.lane_groups;
  if (mx_overlap({{p->out, ((p->l.rows - 1) * p->out_stride + p->in.cols) * p->out_bytes}}, {mx_codes(p->in, lt, p->bits), mx_scales(p->in, lt)}))
    return mx_refused(what, "out and in must not overlap");
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (p->bits == 4 && p->out_bytes == 2) launch_values<4, uint16_t>(*p, groups, st);
  else if (p->bits == 4) launch_values<4, float>(*p, groups, st);
  else if (p->out_bytes == 2) launch_values<8, uint16_t>(*p, groups, st);
  else launch_values<8, float>(*p, groups, st);
  return mx_launched(what);
}

int stride_mx_norm(const StrideMxNormParams* p, void* stream) {
  const char* what = "mx_norm";
  if (!p) return mx_refused(what, "null parameters");
  if (!mx_lanes_ok(p->l)) return mx_refused(what, "need rows >= 0 and lane_groups = ceil(rows/16)");
  if (p->dim <= 0 || p->dim % 16 || p->dim > 65536) return mx_refused(what, "dim must be a positive multiple of 16, at most 65536");
  if (p->l.rows / 4 > kMxMostGroups - 1) return mx_refused(what, "too many rows");
  if (p->l.rows == 0) return 0;
  if (!p->h || !p->weight || !p->out.codes == !p->x) return mx_refused(what, "need h, weight and one of out and x");
  if (p->out.codes)
    if (const char* why = mx_why_not(p->out, p->l.lane_groups, p->dim)) return mx_refused(what, why);
  if ((reinterpret_cast<uintptr_t>(p->h) | reinterpret_cast<uintptr_t>(p->add) | reinterpret_cast<uintptr_t>(p->weight) | reinterpret_cast<uintptr_t>(p->x)) % 16)
    return mx_refused(what, "pointers must be 16-byte aligned");
  const int64_t lt = p->l.lane_groups, values = lt * kTileElems * (p->dim / 16);
  const MxSpan h = {p->h, values * 4}, add = {p->add, values * 2}, weight = {p->weight, p->dim * int64_t{4}}, x = {p->x, values * 2};
  const MxSpan codes = mx_codes(p->out, lt, 8), scales = mx_scales(p->out, lt);
  // x in add's place is served: a thread reads its own values of it before it writes them
  if (mx_overlap({h}, {add, weight}) || mx_overlap({codes, scales, x}, {h, weight}) || mx_overlap({codes, scales}, {add}) ||
      (p->x != p->add && mx_overlap({x}, {add})))
    return mx_refused(what, "h, add, weight and the result must not overlap");
  const int chunks = mx_groups(p->dim) * 4;
  hipStream_t st = static_cast<hipStream_t>(stream);
  // A row a workgroup while each can have a CU, and two while two rows can, four where the memory is
  // full either way: neighbouring rows share their lines, from one XCD's L2 or in one workgroup (us a call
  // in a graph of calls on other rows, at R = 1 / 2 / 4 with an addition: 1 x 2048 2.7 / 2.9 / 3.6, 256 x 8192
  // 7.6 / 9.1 / 11.8, 333 x 8192 11.0 / 9.8 / 12.2, 512 x 4096 7.5 / 7.4 / 8.2, 1024 x 4096 12.2 / 11.4 / 10.1,
  // 4096 x 2048 25.2 / 22.7 / 19.9, 92 MB: 4.7 TB/s, a 4 GiB copy's 4.8; dealt out over the XCDs in turn
  // 256 x 8192 takes 11.8 at R = 1). More than 512 rows of more than 8192 columns leave no registers at
  // R = 4, and h is read twice: 1024 x 16384 49.5 us of GPU, where its bytes take 38.6; two rows a workgroup
  // would hold 16384 columns, and are not measured there.
  if (p->l.rows <= 256) launch_norm<1>(*p, chunks, st);
  else if (p->l.rows <= 512) launch_norm<2>(*p, chunks, st);
  else launch_norm<4>(*p, chunks, st);
  return mx_launched(what);
}

}  // extern "C"
