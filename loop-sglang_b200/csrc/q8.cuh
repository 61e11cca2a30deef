// The 8-bit KV cache format shared by its append and attention kernels (sm_100a).
//
// A KV layer's keys and values are 8-bit codes, one slot of hkv * head_dim codes per token,
// with one fp32 scale per block of `block` consecutive slots and KV head:
//   value = code * scale[slot / block][head]
// Codes are e4m3 (scale a power of two, so re-expressing codes in a larger scale is exact
// while they stay normal) or int8 (scale = amax / 127).
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

// Device-side error flags of the kernels that validate indices while running.
extern int* lsb_device_error_flag();

namespace lsb {

constexpr uint32_t kInfBits = 0x7f800000u;
constexpr uint32_t kNanBits = 0x7fc00000u;

// The smallest scale that holds a magnitude, both as fp32 bits (magnitudes and scales are not
// negative, so their bits order as the values do, with NaN above infinity above the rest). A
// magnitude that is not finite gives NaN: such a block reads back as NaN instead of as
// something plausible.
template <bool INT8>
__device__ __forceinline__ uint32_t q8_scale_bits(uint32_t amax) {
  if (amax >= kInfBits) return kNanBits;
  if (amax == 0) return 0;
  // never below the smallest normal number, so that a scale's inverse is finite
  if (INT8)
    return max(__float_as_uint(__fmul_rn(__uint_as_float(amax), 1.0f / 127.0f)), 1u << 23);
  // amax <= 448 * 2^e with 448 = 1.75 * 2^8: the exponent, one more above mantissa 1.75
  const int e = static_cast<int>((amax + 0x1fffffu) >> 23) - 8;
  return static_cast<uint32_t>(e < 1 ? 1 : e) << 23;
}

__device__ __forceinline__ float q8_inverse(uint32_t scale_bits) {
  return scale_bits == 0 ? 0.f : __fdiv_rn(1.f, __uint_as_float(scale_bits));
}

// Four scaled values to four codes, rounded to nearest even. e4m3 keeps them within the type's
// range; int8 takes values of at most 127.4 (a scale is amax / 127 or more), whose integer is
// the low byte of their sum with 1.5 * 2^23.
template <bool INT8>
__device__ __forceinline__ uint32_t q8_encode4(float a, float b, float c, float d) {
  if (INT8) {
    auto one = [](float x) { return __float_as_uint(__fadd_rn(x, 12582912.f)); };
    return __byte_perm(__byte_perm(one(a), one(b), 0x0040), __byte_perm(one(c), one(d), 0x0040),
                       0x5410);
  }
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}

// Codes 0, 1 (`lo`) and 2, 3 (`hi`) of a word as f16 pairs, exactly. int8: the code's bits
// under the f16 exponent of 1024 give 1024 + (code + 128); subtracting 1152 leaves the code.
template <bool INT8>
__device__ __forceinline__ void q8_decode4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if (INT8) {
    const uint32_t u = w ^ 0x80808080u;
    const uint32_t bias = 0x64806480u;  // 1152 twice
    const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140);
    const uint32_t b = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 ra = __hsub2(*reinterpret_cast<const __half2*>(&a),
                               *reinterpret_cast<const __half2*>(&bias));
    const __half2 rb = __hsub2(*reinterpret_cast<const __half2*>(&b),
                               *reinterpret_cast<const __half2*>(&bias));
    lo = *reinterpret_cast<const uint32_t*>(&ra);
    hi = *reinterpret_cast<const uint32_t*>(&rb);
  } else {
    const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w), __NV_E4M3);
    const __half2_raw b =
        __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w >> 16), __NV_E4M3);
    lo = *reinterpret_cast<const uint32_t*>(&a);
    hi = *reinterpret_cast<const uint32_t*>(&b);
  }
}

template <bool INT8>
__device__ __forceinline__ float4 q8_decode4f(uint32_t w) {
  uint32_t lo, hi;
  q8_decode4<INT8>(w, lo, hi);
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo));
  const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  return make_float4(a.x, a.y, b.x, b.y);
}

// Byte offset of 16-byte chunk c of row r of a tile: any 8 rows from a multiple of 8 on have
// chunk c in 8 different bank groups. XOR-ing c * 16 into a row's offset of chunk 0 gives
// chunk c's, except at 96 dims (whose rows are padded to 112 bytes), where it is added.
template <int D>
__host__ __device__ constexpr int q8_row_bytes() {
  return D == 96 ? 112 : D;
}
template <int D>
__device__ __forceinline__ int q8_tile_offset(int r, int c) {
  if (D == 128) return r * 128 + ((c ^ (r & 7)) << 4);
  if (D == 64) return (r >> 1) * 128 + (((r & 1) * 4 + (c ^ ((r >> 1) & 3))) << 4);
  if (D == 32) return (r >> 2) * 128 + (((r & 3) * 2 + (c ^ ((r >> 2) & 1))) << 4);
  return r * q8_row_bytes<D>() + (c << 4);
}
}  // namespace lsb
