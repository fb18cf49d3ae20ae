// Microscaled blocks on the device: the scale rule, conversions, and the scaled matrix product
// (include/stride_mx.h has the formats and layouts).
#pragma once

#include <initializer_list>
#include <string>

#include "../../include/stride_mx.h"
#include "tc_common.hpp"

namespace stride_tc {

int fail(int code, const std::string& msg);  // tc_gemm.hip

constexpr int kMxBlock = 32;     // neighbours that share a scale
constexpr int kMxChunk = 128;    // columns of a matrix instruction
constexpr int kMxGroup = 512;    // columns whose scales a lane reads as one word
constexpr int kCode4Bytes = 1024, kCode8Bytes = 2048, kScaleBytes = 256;  // a tile's chunk; a tile's group

constexpr int64_t kMxMostGroups = (int64_t{1} << 32) / 1024 - 1;  // of up to 1024 threads, all of which a launch counts in 32 bits

typedef int i32x8 __attribute__((ext_vector_type(8)));

__host__ __device__ constexpr int mx_groups(int cols) { return (cols + kMxGroup - 1) / kMxGroup; }

// The scale's byte from the bits of a block's largest magnitude: the exponent of the element
// format's top binade (4 .. 6 for e2m1, 256 .. 448 for e4m3) is put where the magnitude lies, one
// higher where it would round beyond the format's largest value (a tie at 7 rounds up to 8 and one
// at 464 down to 448). 255 for what is not finite.
template <int BITS>
__device__ __forceinline__ int mx_scale_byte(uint32_t most) {
  const int e = static_cast<int>(most >> 23);
  const uint32_t m = most & 0x7FFFFFu;
  const bool up = BITS == 4 ? m >= 0x600000u : m > 0x680000u;
  return e == 255 ? 255 : max(0, e - (BITS == 4 ? 2 : 8) + (up ? 1 : 0));
}

// 1 / scale, exact: the byte of a finite block is at most 254 - 2 + 1.
__device__ __forceinline__ float mx_inverse(int byte) { return f32_of(static_cast<uint32_t>(254 - min(byte, 253)) << 23); }

__device__ __forceinline__ uint32_t mx_abs_bits(float v) { return u32_of(v) & 0x7FFFFFFFu; }

// Four values times `inverse` to four e4m3 bytes, eight to eight e2m1 nibbles, the first lowest.
// The instructions round to the nearest, ties to even; the scale rule leaves nothing beyond the range.
__device__ __forceinline__ uint32_t mx_pack8(float a, float b, float c, float d, float inverse) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a * inverse, b * inverse, 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(c * inverse, d * inverse, w, true);
  return static_cast<uint32_t>(w);
}
__device__ __forceinline__ uint32_t mx_pack4(const float* v, float inverse) {
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0] * inverse, v[1] * inverse, 1.0f, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2] * inverse, v[3] * inverse, 1.0f, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4] * inverse, v[5] * inverse, 1.0f, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6] * inverse, v[7] * inverse, 1.0f, 3);
  return w;
}

// c += W x over a chunk: a lane of W's operand has 32 columns of row lane % 16 (block lane / 16),
// one of x's 16 columns of each half (part lane / 16). Byte I of the scale words is the chunk's;
// lane l's is that of row l % 16, block l / 16, for both.
template <int I>
__device__ __forceinline__ f32x4 mx_mfma(u32x4 w, u32x4 x0, u32x4 x1, f32x4 c, uint32_t ws, uint32_t xs) {
  const i32x8 a = {static_cast<int>(w[0]), static_cast<int>(w[1]), static_cast<int>(w[2]), static_cast<int>(w[3]), 0, 0, 0, 0};
  const i32x8 b = {static_cast<int>(x0[0]), static_cast<int>(x0[1]), static_cast<int>(x0[2]), static_cast<int>(x0[3]),
                   static_cast<int>(x1[0]), static_cast<int>(x1[1]), static_cast<int>(x1[2]), static_cast<int>(x1[3])};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 4, 0, I, static_cast<int>(ws), I, static_cast<int>(xs));
}

// Host: do these describe tiles of at least `tiles` tiles and, with cols > 0, of `cols` columns?
inline const char* mx_why_not(const StrideMxTiles& t, int64_t tiles, int cols) {
  if (t.cols <= 0 || t.cols % 16 || t.cols > (1 << 20)) return "cols must be a positive multiple of 16, at most 2^20";
  if (cols > 0 && t.cols != cols) return "cols differ";
  if (t.tiles < tiles) return "too few tiles";
  if (!t.codes || !t.scales) return "missing pointer";
  if (reinterpret_cast<uintptr_t>(t.codes) % 16 || reinterpret_cast<uintptr_t>(t.scales) % 4) return "codes must be 16-byte and scales 4-byte aligned";
  return nullptr;
}

// Host: memory that a call reads or writes, and whether a result shares some with another operand: other
// workgroups read that one at any time.
struct MxSpan {
  const void* at;
  int64_t bytes;
};
inline MxSpan mx_codes(const StrideMxTiles& t, int64_t tiles, int bits) {
  return {t.codes, tiles * mx_groups(t.cols) * 4 * (bits == 4 ? kCode4Bytes : kCode8Bytes)};
}
inline MxSpan mx_scales(const StrideMxTiles& t, int64_t tiles) { return {t.scales, tiles * mx_groups(t.cols) * kScaleBytes}; }

inline bool mx_overlap(std::initializer_list<MxSpan> results, std::initializer_list<MxSpan> operands) {
  for (const MxSpan& r : results)
    for (const MxSpan& o : operands) {
      const uintptr_t a = reinterpret_cast<uintptr_t>(r.at), b = reinterpret_cast<uintptr_t>(o.at);
      if (a && b && a < b + o.bytes && b < a + r.bytes) return true;
    }
  return false;
}

inline int mx_refused(const char* what, const char* why) { return fail(STRIDE_TC_EINVAL, std::string(what) + ": " + why); }

inline int mx_launched(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(static_cast<int>(e), std::string(what) + " launch failed: " + hipGetErrorString(e));
  return 0;
}

inline bool mx_lanes_ok(const StrideLanes& l) { return l.rows >= 0 && l.lane_groups == (static_cast<int64_t>(l.rows) + 15) / 16; }

}  // namespace stride_tc
