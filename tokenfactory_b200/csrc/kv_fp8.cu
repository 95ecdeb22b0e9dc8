// KV-pool store with the rows quantized to e4m3 (formulas in tfattn.h): the 8-bit counterpart of
// kv_store.cu.  HBM-bound: a row is read once, its largest magnitude found by shuffles among the
// lanes that hold it, and the codes written from the same registers.  20011 tokens of 4 heads of 256
// bfloat16 values: 26.6 us, 4.65 TB/s (0.71 of the copy rate; 74% of the issue slots and 60% of the ALU
// pipe are used, by the index divisions, quotients and conversions of a pair); 48 tokens: 4 us, a launch.
#include <type_traits>

#include "common.cuh"
#include "kv_fp8.cuh"
#include "launch.h"

namespace tf {
namespace {

constexpr int kThreads = 256;

// eight elements of a row, loaded in 16-byte pieces and unpacked when used
template <typename T> struct Vec8 {
  uint4 w;
  __device__ __forceinline__ void load(const T* p) { w = __ldcs(reinterpret_cast<const uint4*>(p)); }
  // abs_bits of the largest element: 16-bit magnitudes order like their bits, two to a word
  __device__ __forceinline__ uint32_t amax() const {
    uint32_t m = w.x & 0x7fff7fffu;
    asm("max.u16x2 %0, %0, %1;" : "+r"(m) : "r"(w.y & 0x7fff7fffu));
    asm("max.u16x2 %0, %0, %1;" : "+r"(m) : "r"(w.z & 0x7fff7fffu));
    asm("max.u16x2 %0, %0, %1;" : "+r"(m) : "r"(w.w & 0x7fff7fffu));
    return __float_as_uint(fmax_bits(m));
  }
  static __device__ __forceinline__ float fmax_bits(uint32_t m) {
    return unpack_lo<T>(max(m & 0xffffu, m >> 16));
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = unpack_lo<T>(u[i]);
      x[2 * i + 1] = unpack_hi<T>(u[i]);
    }
  }
};
template <> struct Vec8<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = __ldcs(reinterpret_cast<const float4*>(p));
    b = __ldcs(reinterpret_cast<const float4*>(p) + 1);
  }
  __device__ __forceinline__ uint32_t amax() const {
    float x[8];
    get(x);
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, kv8::abs_bits(x[i]));
    return m;
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  }
};

// LPR = D / 8 lanes hold a row, eight elements each; a group of LPR lanes takes the K and the V rows
// of N (token, kv head) pairs, so 2 N rows are in flight per lane and a scale pair is one store.
template <typename T, int LPR, int N>
__global__ void __launch_bounds__(kThreads) store_vec_kernel(const __grid_constant__ tf_kv_store_args a,
                                                             const __grid_constant__ tf_kv_scale sc) {
  const int64_t g = (blockIdx.x * (int64_t)kThreads + threadIdx.x) / LPR;
  const int l = threadIdx.x % LPR;
  const int64_t rows = a.num_tokens * (int64_t)a.num_kv_heads;
  int h[N];
  int64_t loc[N];
  Vec8<T> x[N][2];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    int64_t r = g * N + n;
    if (r >= rows) r = rows - 1;  // in bounds; not stored
    const int64_t t = a.num_kv_heads == 1 ? r : r / a.num_kv_heads;
    h[n] = (int)(r - t * a.num_kv_heads);
    loc[n] = a.out_cache_loc[t];
    x[n][0].load((const T*)a.k + t * a.k_stride_tok + h[n] * a.k_stride_head + 8 * l);
    x[n][1].load((const T*)a.v + t * a.v_stride_tok + h[n] * a.v_stride_head + 8 * l);
  }
#pragma unroll
  for (int n = 0; n < N; ++n) {
    uint32_t m[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      m[j] = x[n][j].amax();
      if (LPR == 32) {
        m[j] = __reduce_max_sync(0xffffffffu, m[j]);
      } else {
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) m[j] = max(m[j], __shfl_xor_sync(0xffffffffu, m[j], o));
      }
    }
    const kv8::PairScale ps = kv8::pair_scale<LPR>(m[0], m[1], l);
    if (g * N + n >= rows) continue;
    const int64_t slot = kv8::store_slot(loc[n], a.num_slots, l == 0 ? a.err : nullptr);
    if (slot < 0) continue;
    const int64_t off = slot * a.buf_stride_slot + h[n] * a.buf_stride_head + 8 * l;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float v[8];
      x[n][j].get(v);
      uint2 c = make_uint2(0, 0);
      if (ps.finite[j]) {
        const float f = ps.mul[j];
        c.x = kv8::code4(v[0] * f, v[1] * f, v[2] * f, v[3] * f);
        c.y = kv8::code4(v[4] * f, v[5] * f, v[6] * f, v[7] * f);
      }
      *reinterpret_cast<uint2*>((char*)(j ? a.v_buffer : a.k_buffer) + off) = c;
    }
    if (l == 0)
      *reinterpret_cast<float2*>(sc.data + slot * sc.stride_slot + h[n] * sc.stride_head) =
          make_float2(ps.scale[0], ps.scale[1]);
  }
}

// any head_dim, strides and alignment: a warp per (token, kv head), each row read twice
template <typename T>
__global__ void __launch_bounds__(kThreads) store_any_kernel(tf_kv_store_args a, tf_kv_scale sc) {
  const int64_t rows = a.num_tokens * (int64_t)a.num_kv_heads;
  const int lane = threadIdx.x & 31;
  const int64_t nwarps = ((int64_t)gridDim.x * kThreads) >> 5;
  for (int64_t r = (blockIdx.x * (int64_t)kThreads + threadIdx.x) >> 5; r < rows; r += nwarps) {
    const int64_t t = r / a.num_kv_heads;
    const int h = (int)(r - t * a.num_kv_heads);
    const int64_t slot = kv8::store_slot(a.out_cache_loc[t], a.num_slots,
                                         lane == 0 ? a.err : nullptr);
    if (slot < 0) continue;
    float scale[2];
    for (int j = 0; j < 2; ++j) {
      const T* src = j ? (const T*)a.v + t * a.v_stride_tok + h * a.v_stride_head
                       : (const T*)a.k + t * a.k_stride_tok + h * a.k_stride_head;
      uint8_t* dst = (uint8_t*)(j ? a.v_buffer : a.k_buffer) + slot * a.buf_stride_slot +
                     h * a.buf_stride_head;
      uint32_t m = 0;
      for (int d = lane; d < a.head_dim; d += 32) m = max(m, kv8::abs_bits(to_f(src[d])));
      m = __reduce_max_sync(0xffffffffu, m);
      const kv8::RowScale rs = kv8::row_scale(m);
      for (int d = lane; d < a.head_dim; d += 32)
        dst[d] = rs.finite ? kv8::code1(to_f(src[d]) * rs.mul) : 0;
      scale[j] = rs.scale;
    }
    if (lane == 0)
      *reinterpret_cast<float2*>(sc.data + slot * sc.stride_slot + h * sc.stride_head) =
          make_float2(scale[0], scale[1]);
  }
}

template <typename T>
cudaError_t launch_t(const tf_kv_store_args& a, const tf_kv_scale& sc, cudaStream_t s) {
  const int eb = (int)sizeof(T), d = a.head_dim;
  const int64_t rows = a.num_tokens * (int64_t)a.num_kv_heads;
  auto al = [](const void* p, int n) { return (reinterpret_cast<uintptr_t>(p) % n) == 0; };
  const bool vec = (d == 64 || d == 128 || d == 256) && al(a.k, 16) && al(a.v, 16) &&
                   al(a.k_buffer, 8) && al(a.v_buffer, 8) && (a.k_stride_tok * eb) % 16 == 0 &&
                   (a.k_stride_head * eb) % 16 == 0 && (a.v_stride_tok * eb) % 16 == 0 &&
                   (a.v_stride_head * eb) % 16 == 0 && a.buf_stride_slot % 8 == 0 &&
                   a.buf_stride_head % 8 == 0;
  // two pairs a group once the groups of one pair each would fill the SMs
  const int per = vec && rows * (d / 8) >= 148 * 2048 ? 2 : 1;
  const int lanes = vec ? d / 8 : 32;
  const int64_t blocks = ((rows + per - 1) / per * lanes + kThreads - 1) / kThreads;
  if (vec && blocks <= 0x7fffffff) {
    const unsigned g = (unsigned)blocks;
    auto go = [&](auto lpr) {
      constexpr int L = decltype(lpr)::value;
      if (per == 2) store_vec_kernel<T, L, 2><<<g, kThreads, 0, s>>>(a, sc);
      else store_vec_kernel<T, L, 1><<<g, kThreads, 0, s>>>(a, sc);
    };
    if (d == 64) go(std::integral_constant<int, 8>());
    else if (d == 128) go(std::integral_constant<int, 16>());
    else go(std::integral_constant<int, 32>());
  } else {
    const unsigned g = (unsigned)(blocks < 148 * 32 ? blocks : 148 * 32);
    store_any_kernel<T><<<g, kThreads, 0, s>>>(a, sc);
  }
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_kv_store_fp8(const tf_kv_store_args& a, const tf_kv_scale& sc, cudaStream_t s) {
  if (a.num_tokens == 0) return cudaSuccess;
  switch (a.dtype) {
    case TF_DTYPE_F32: return launch_t<float>(a, sc, s);
    case TF_DTYPE_BF16: return launch_t<__nv_bfloat16>(a, sc, s);
    default: return launch_t<__half>(a, sc, s);
  }
}

}  // namespace tf
