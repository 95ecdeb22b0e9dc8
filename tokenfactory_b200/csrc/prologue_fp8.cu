// Fused full-attention prologue over the 8-bit K/V pool: q/k RMSNorm, partial (M-)RoPE and the
// quantizing pool store (formulas in tfattn.h), one read of q/k/v and one write of q_out and the
// pool rows.  HBM-bound.  Everything is fp32 from the loaded values to the one rounding of q_out
// (to its dtype) and of the codes: unlike prologue.cu, which rounds where the reference's torch
// lines do, nothing downstream of an 8-bit row would see those roundings.  The angle is the product
// of an integer and an fp32 frequency in fp64, reduced by whole turns there: in fp32 its rounding
// alone would reach 2^-9 of a radian at position 32768.
//
// A CTA takes TPC tokens (4; 1 when there are too few tokens to fill the SMs otherwise): their cos/sin
// and slots first, then its warps walk the tokens' rows, kPF rows in flight per warp.  Lane l of the
// vector form holds the E = D/32 elements [E l, E l + E) of a row; the rotation partner d +- rotary_dim/2 sits in lane l ^ (rotary_dim/2/E) when that is a
// power of two, and otherwise comes from a copy of the row in shared memory.
// 7001 tokens, 24 heads over 4 of 256 float16 values: 51 us, 4.2 TB/s (0.64 of the copy rate; 57 us with
// fewer rows in flight a lane): 62% of the issue slots used, stalls on rows in flight and on shared memory;
// at the 80 registers of three CTAs an SM the head_dim 256 forms spill 24 to 140 bytes a thread; 128 tokens: 7.2 us (23 us with four tokens a CTA throughout), a launch
// and two dependent reads.
#include "common.cuh"
#include "kv_fp8.cuh"
#include "launch.h"

namespace tf {
namespace prologue8 {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxD = 256;
constexpr int kPF = 4;
constexpr int kFewTokens = 592;  // four CTAs an SM

// A lane's E elements of a row as loaded (unpacked only when they are used: an unpack next to the load
// would wait for it), in E * sizeof(T) / 4 words.
template <typename T, int E>
struct RawRow {
  static constexpr int kW = E * (int)sizeof(T) / 4;
  uint32_t w[kW];
  template <bool VEC>
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (VEC && kW % 4 == 0) {
#pragma unroll
      for (int i = 0; i < kW / 4; ++i) {
        const uint4 v = __ldcs(reinterpret_cast<const uint4*>(p) + i);
        w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
      }
    } else if constexpr (VEC && kW == 2) {
      const uint2 v = __ldcs(reinterpret_cast<const uint2*>(p));
      w[0] = v.x; w[1] = v.y;
    } else if constexpr (VEC && kW == 1) {
      w[0] = __ldcs(reinterpret_cast<const unsigned int*>(p));
    } else if constexpr (sizeof(T) == 2) {
      const unsigned short* u = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
      for (int i = 0; i < kW; ++i) w[i] = u[2 * i] | ((uint32_t)u[2 * i + 1] << 16);
    } else {
      const uint32_t* u = reinterpret_cast<const uint32_t*>(p);
#pragma unroll
      for (int i = 0; i < kW; ++i) w[i] = u[i];
    }
  }
  __device__ __forceinline__ void get(float (&x)[E]) const {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < kW; ++i) { x[2 * i] = unpack_lo<T>(w[i]); x[2 * i + 1] = unpack_hi<T>(w[i]); }
    } else {
#pragma unroll
      for (int i = 0; i < kW; ++i) x[i] = __uint_as_float(w[i]);
    }
  }
};

template <typename T, int E, bool VEC>
__device__ __forceinline__ void store_row(T* p, const float (&x)[E]) {
  if constexpr (VEC && sizeof(T) == 2) {
    uint32_t w[E / 2];
#pragma unroll
    for (int i = 0; i < E / 2; ++i) w[i] = pack2_rn<T>(x[2 * i], x[2 * i + 1]);
    if constexpr (E == 8) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    else if constexpr (E == 4) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t*>(p) = w[0];
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) p[e] = from_f<T>(x[e]);
  }
}

// largest abs_bits of a row of which the warp's lanes hold E elements each
template <int E>
__device__ __forceinline__ uint32_t row_amax(const float (&x)[E]) {
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) m = max(m, kv8::abs_bits(x[e]));
  return __reduce_max_sync(0xffffffffu, m);
}

// codes of the lane's E elements of a row
template <int E, bool VEC>
__device__ __forceinline__ void store_codes(uint8_t* p, const float (&x)[E], float mul, bool finite) {
  uint32_t c[E / 2];
#pragma unroll
  for (int i = 0; i < E / 2; ++i) c[i] = finite ? kv8::code2(x[2 * i] * mul, x[2 * i + 1] * mul) : 0u;
  if constexpr (VEC && E == 8) {
    *reinterpret_cast<uint2*>(p) = make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
  } else if constexpr (VEC && E == 4) {
    *reinterpret_cast<uint32_t*>(p) = c[0] | (c[1] << 16);
  } else {
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      p[2 * i] = (uint8_t)c[i];
      p[2 * i + 1] = (uint8_t)(c[i] >> 8);
    }
  }
}

// RMSNorm of a row and rotation of its first 2 half values, in place.  c, sn: cos and sin of the lane's
// values (VEC / XOR forms), or of the token (shared memory, partner values through `row`).
template <int D, bool XOR>
__device__ __forceinline__ void norm_rotate(float (&y)[D / 32], const float (&w)[D / 32], float eps,
                                            const float (&c)[D / 32], const float (&sn)[D / 32], int half,
                                            int lane, float* row) {
  constexpr int E = D / 32;
  const int d0 = lane * E;
  float ss = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) ss = fmaf(y[e], y[e], ss);
  ss = warp_sum(ss);
  const float rs = rsqrtf(ss * (1.0f / D) + eps);  // D is a power of two
#pragma unroll
  for (int e = 0; e < E; ++e) y[e] = w[e] * (y[e] * rs);
  if constexpr (XOR) {
    // sn carries the sign of the lane's half; lanes that do not rotate keep their values
    float p[E];
#pragma unroll
    for (int e = 0; e < E; ++e) p[e] = __shfl_xor_sync(0xffffffffu, y[e], half / E);
    if (d0 < 2 * half) {
#pragma unroll
      for (int e = 0; e < E; ++e) y[e] = fmaf(p[e], sn[e], y[e] * c[e]);
    }
  } else {
    __syncwarp();
#pragma unroll
    for (int e = 0; e < E; ++e) row[d0 + e] = y[e];
    __syncwarp();
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int d = d0 + e;
      if (d < 2 * half) y[e] = fmaf(row[d < half ? d + half : d - half], sn[e], y[e] * c[e]);
    }
  }
}

// VEC: rows aligned to the lane's E elements.  XOR: the partner lane is lane ^ (half / E).
template <typename T, int D, int TPC, bool VEC, bool XOR>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 ? 3 : 2) prologue_kernel(const __grid_constant__ tf_attn_prologue_args a,
                                                            const __grid_constant__ tf_kv_scale sc) {
  constexpr int E = D / 32;
  constexpr int kRowStep = kWarps / TPC;
  __shared__ float cs[TPC][kMaxD / 2], sn[TPC][kMaxD / 2];
  __shared__ int64_t s_loc[TPC];
  __shared__ float s_row[XOR ? 1 : kWarps][XOR ? 1 : D];
  const int64_t t0 = (int64_t)blockIdx.x * TPC;
  const int ntok = a.num_tokens - t0 < TPC ? (int)(a.num_tokens - t0) : TPC;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int Hq = a.num_q_heads, Hkv = a.num_kv_heads;
  const int half = a.rotary_dim / 2;
  const int d0 = lane * E;
  // warp w serves token w % TPC: its q rows r0, r0 + kRowStep, ..., then its (k, v) row pairs
  const int tt = warp % TPC, r0 = warp / TPC;
  const bool live = tt < ntok;
  const int64_t t = t0 + (live ? tt : 0);
  const T* qp = (const T*)a.q + t * a.q_stride_tok + (int64_t)r0 * a.q_stride_head + d0;
  const int64_t q_step = (int64_t)kRowStep * a.q_stride_head;
  RawRow<T, E> ring[kPF];
#pragma unroll
  for (int u = 0; u < kPF; ++u)
    if (live && r0 + u * kRowStep < Hq) ring[u].template load<VEC>(qp + u * q_step);
  const T* kp = (const T*)a.k + t * a.k_stride_tok + d0;
  const T* vp = (const T*)a.v + t * a.v_stride_tok + d0;
  RawRow<T, E> kraw, vraw;  // of the warp's next kv head
  if (live && r0 < Hkv) {
    kraw.template load<VEC>(kp + (int64_t)r0 * a.k_stride_head);
    vraw.template load<VEC>(vp + (int64_t)r0 * a.v_stride_head);
  }
  float w[E];
  const bool wf32 = a.norm_weight_dtype == TF_DTYPE_F32;
  auto load_w = [&](const void* p) {
#pragma unroll
    for (int e = 0; e < E; ++e)
      w[e] = wf32 ? reinterpret_cast<const float*>(p)[d0 + e] : to_f(reinterpret_cast<const T*>(p)[d0 + e]);
  };
  load_w(a.q_norm_weight);

  for (int j = tid; j < ntok * half; j += kThreads) {
    const int jt = j / half, jj = j - jt * half;
    int prow = 0;
    if (a.pos_rows == 3) {
      if (a.mrope_interleaved) {
        const int m = jj % 3;
        if (m == 1 && jj < 3 * a.mrope_section[1]) prow = 1;
        else if (m == 2 && jj < 3 * a.mrope_section[2]) prow = 2;
      } else {
        prow = jj < a.mrope_section[0] ? 0 : (jj < a.mrope_section[0] + a.mrope_section[1] ? 1 : 2);
      }
    }
    // whole turns are removed in fp64 (2 pi to 53 bits: an error of 2^-53 per radian turned)
    const double f = (double)a.positions[prow * a.pos_stride + t0 + jt] * (double)a.inv_freq[jj];
    constexpr double k2Pi = 6.283185307179586;
    const double turn = f - rint(f * (1.0 / k2Pi)) * k2Pi;
    // the angle in two floats: sine and cosine of the first, turned on by the second (first order: it is below
    // 2^-22).  Rounded to one float its error, up to 2^-23, would be all that is left of a sine near 0.
    const float hi = (float)turn, lo = (float)(turn - (double)hi);
    float sf, cf;
    sincosf(hi, &sf, &cf);
    cs[jt][jj] = fmaf(-sf, lo, cf);
    sn[jt][jj] = fmaf(cf, lo, sf);
  }
  if (tid < ntok) s_loc[tid] = kv8::store_slot(a.out_cache_loc[t0 + tid], a.num_slots, a.err);
  __syncthreads();
  if (!live) return;
  float c[E], s[E];  // of the lane's values, the sine with the sign of its half
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int d = d0 + e, j = d < half ? d : (d < 2 * half ? d - half : 0);
    c[e] = cs[tt][j];
    s[e] = d < half ? -sn[tt][j] : sn[tt][j];
  }
  float* row = s_row[XOR ? 0 : warp];
  T* op = (T*)a.q_out + t * a.q_out_stride_tok + (int64_t)r0 * a.q_out_stride_head + d0;
  const int64_t o_step = (int64_t)kRowStep * a.q_out_stride_head;
  qp += kPF * q_step;
  for (int r = r0; r < Hq; r += kPF * kRowStep) {
#pragma unroll
    for (int u = 0; u < kPF; ++u) {
      if (r + u * kRowStep >= Hq) break;
      float y[E];
      ring[u].get(y);
      if (r + (u + kPF) * kRowStep < Hq) ring[u].template load<VEC>(qp);
      qp += q_step;
      norm_rotate<D, XOR>(y, w, a.eps, c, s, half, lane, row);
      store_row<T, E, VEC>(op, y);
      op += o_step;
    }
  }
  const int64_t loc = s_loc[tt];
  if (loc < 0 || r0 >= Hkv) return;
  load_w(a.k_norm_weight);
  for (int h = r0; h < Hkv; h += kRowStep) {
    float y[E], v[E];
    kraw.get(y);
    vraw.get(v);
    if (h + kRowStep < Hkv) {
      kraw.template load<VEC>(kp + (int64_t)(h + kRowStep) * a.k_stride_head);
      vraw.template load<VEC>(vp + (int64_t)(h + kRowStep) * a.v_stride_head);
    }
    norm_rotate<D, XOR>(y, w, a.eps, c, s, half, lane, row);
    const int64_t off = loc * a.buf_stride_slot + (int64_t)h * a.buf_stride_head + d0;
    const kv8::PairScale ps = kv8::pair_scale<32>(row_amax(y), row_amax(v), lane);
    store_codes<E, VEC>((uint8_t*)a.k_buffer + off, y, ps.mul[0], ps.finite[0]);
    store_codes<E, VEC>((uint8_t*)a.v_buffer + off, v, ps.mul[1], ps.finite[1]);
    if (lane == 0)
      *reinterpret_cast<float2*>(sc.data + loc * sc.stride_slot + h * sc.stride_head) =
          make_float2(ps.scale[0], ps.scale[1]);
  }
}

template <typename T, int D, int TPC>
static cudaError_t launch_dt(const tf_attn_prologue_args& a, const tf_kv_scale& sc, cudaStream_t s) {
  constexpr int E = D / 32;
  const int half = a.rotary_dim / 2;
  const int vb = E * (int)sizeof(T) < 16 ? E * (int)sizeof(T) : 16;
  auto al = [](const void* p, int n) { return (reinterpret_cast<uintptr_t>(p) % n) == 0; };
  bool vec = al(a.q, vb) && al(a.k, vb) && al(a.v, vb) && al(a.q_out, vb) && al(a.k_buffer, E) &&
             al(a.v_buffer, E);
  for (int64_t x : {a.q_stride_tok, a.q_stride_head, a.k_stride_tok, a.k_stride_head,
                    a.v_stride_tok, a.v_stride_head, a.q_out_stride_tok, a.q_out_stride_head,
                    a.buf_stride_slot, a.buf_stride_head})
    vec = vec && x % E == 0;
  const int pm = half / E;
  const bool xr = half % E == 0 && pm < 32 && (pm & (pm - 1)) == 0;
  const unsigned g = (unsigned)((a.num_tokens + TPC - 1) / TPC);
  if (vec && xr) prologue_kernel<T, D, TPC, true, true><<<g, kThreads, 0, s>>>(a, sc);
  else if (vec) prologue_kernel<T, D, TPC, true, false><<<g, kThreads, 0, s>>>(a, sc);
  else prologue_kernel<T, D, TPC, false, false><<<g, kThreads, 0, s>>>(a, sc);
  return cudaGetLastError();
}

template <typename T, int D>
static cudaError_t launch_d(const tf_attn_prologue_args& a, const tf_kv_scale& sc, cudaStream_t s) {
  return a.num_tokens <= kFewTokens ? launch_dt<T, D, 1>(a, sc, s) : launch_dt<T, D, 4>(a, sc, s);
}

template <typename T>
static cudaError_t launch_t(const tf_attn_prologue_args& a, const tf_kv_scale& sc, cudaStream_t s) {
  switch (a.head_dim) {
    case 64: return launch_d<T, 64>(a, sc, s);
    case 128: return launch_d<T, 128>(a, sc, s);
    default: return launch_d<T, 256>(a, sc, s);
  }
}

}  // namespace prologue8

bool attn_prologue_fp8_supported(const tf_attn_prologue_args& a) {
  if (a.head_dim != 64 && a.head_dim != 128 && a.head_dim != 256) return false;
  return a.rotary_dim >= 2 && a.rotary_dim % 2 == 0 && a.rotary_dim <= a.head_dim;
}

cudaError_t launch_attn_prologue_fp8(const tf_attn_prologue_args& a, const tf_kv_scale& sc,
                                     cudaStream_t s) {
  if (a.num_tokens == 0) return cudaSuccess;
  switch (a.dtype) {
    case TF_DTYPE_F32: return prologue8::launch_t<float>(a, sc, s);
    case TF_DTYPE_BF16: return prologue8::launch_t<__nv_bfloat16>(a, sc, s);
    default: return prologue8::launch_t<__half>(a, sc, s);
  }
}

}  // namespace tf
