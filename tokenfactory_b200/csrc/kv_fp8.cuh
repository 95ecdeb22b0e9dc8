// Rows of the 8-bit K/V pool: quantization of a row to e4m3 codes and one fp32 scale, and back
// (the formulas stand in tfattn.h).
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace tf {
namespace kv8 {

constexpr float kE4m3Max = 448.f;
constexpr float kMinAmax = 1e-12f;

// |x| as an unsigned word: ordered like |x| with infinities and NaNs on top, so an integer maximum
// keeps them (fmaxf would drop a NaN)
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

struct RowScale {
  float mul;    // codes = e4m3(x * mul)
  float scale;  // what a code stands for
  bool finite;
};

// of a row whose largest abs_bits is `amax`
__device__ __forceinline__ RowScale row_scale(uint32_t amax) {
  RowScale r;
  r.finite = amax < 0x7f800000u;
  const float m = fmaxf(__uint_as_float(amax), kMinAmax);
  r.mul = r.finite ? __fdiv_rn(kE4m3Max, m) : 0.f;
  r.scale = r.finite ? __fdiv_rn(m, kE4m3Max) : __uint_as_float(0x7fc00000u);
  return r;
}

// row_scale of a K row and a V row at once, for a group of W lanes (8, 16 or 32; lane l of the group):
// the four quotients are one division, each in a lane of its own, instead of four.
struct PairScale {
  float mul[2], scale[2];
  bool finite[2];
};
template <int W>
__device__ __forceinline__ PairScale pair_scale(uint32_t amax_k, uint32_t amax_v, int l) {
  const uint32_t bits = l & 2 ? amax_v : amax_k;
  const float m = fmaxf(__uint_as_float(bits), kMinAmax);  // (fmaxf of a NaN: kMinAmax, not used)
  const float q = __fdiv_rn(l & 1 ? m : kE4m3Max, l & 1 ? kE4m3Max : m);
  PairScale r;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    r.finite[j] = (j ? amax_v : amax_k) < 0x7f800000u;
    r.mul[j] = __shfl_sync(0xffffffffu, q, 2 * j, W);
    const float sc = __shfl_sync(0xffffffffu, q, 2 * j + 1, W);
    r.scale[j] = r.finite[j] ? sc : __uint_as_float(0x7fc00000u);
  }
  return r;
}

// two codes, round to nearest even, saturated at +-448, `a` in the low byte
__device__ __forceinline__ uint32_t code2(float a, float b) {
  return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint32_t code4(float a, float b, float c, float d) {
  return code2(a, b) | (code2(c, d) << 16);
}
__device__ __forceinline__ uint8_t code1(float a) {
  return __nv_cvt_float_to_fp8(a, __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ float decode1(uint8_t c) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3)));
}

// out_cache_loc entry -> slot with torch's wrap of negative entries; -1 (recorded) when outside
__device__ __forceinline__ int64_t store_slot(int64_t loc, int64_t num_slots, int32_t* err) {
  if (loc < 0) loc += num_slots;
  if (loc < 0 || loc >= num_slots) {
    record_err(err, TF_KERR_SLOT_RANGE);
    return -1;
  }
  return loc;
}

}  // namespace kv8
}  // namespace tf
