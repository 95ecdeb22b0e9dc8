// Paged GQA attention over the 8-bit K/V pool on CUDA cores, for any dtype (fp32 / bf16 / fp16) and
// any head_dim <= 256, decode and extend: the path of the fp32 configurations and of the shapes the
// tensor-core kernels are not built for.  One CTA per (query token, kv head) computes the
// G = Hq/Hkv query heads that share the kv head, so every K/V row is read once per group; rows are
// multiplied by their scale as they enter shared memory, and everything after that is fp32 up to
// the one rounding of the output.
#include "common.cuh"
#include "kv_fp8.cuh"
#include "launch.h"

namespace tf {
namespace {

constexpr int kThreads = 128;
constexpr int kBK = 32;  // keys per block

template <typename T>
__global__ void __launch_bounds__(kThreads) paged_fp8_simt_kernel(tf_paged_attn_args a,
                                                                  tf_kv_scale sc) {
  const int64_t t = blockIdx.x;
  const int h = blockIdx.y;
  const int G = a.num_q_heads / a.num_kv_heads;
  const int D = a.head_dim;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  extern __shared__ __align__(16) float smem[];
  int64_t* slot_s = reinterpret_cast<int64_t*>(smem);  // [kBK]
  float* q_s = smem + 2 * kBK;               // [G][D]
  float* o_s = q_s + G * D;                  // [G][D]
  float* k_s = o_s + G * D;                  // [kBK][D+1]
  float* v_s = k_s + kBK * (D + 1);          // [kBK][D]
  float* p_s = v_s + kBK * D;                // [G][kBK]
  float* sc_s = p_s + G * kBK;               // [kBK][2]
  float* m_s = sc_s + 2 * kBK;               // [G]
  float* l_s = m_s + G;                      // [G]
  float* al_s = l_s + G;                     // [G]
  __shared__ int sh_b;
  __shared__ int64_t sh_start;

  if (a.extend_lens == nullptr) {
    if (tid == 0) { sh_b = (int)t; sh_start = t; }
  } else if (warp == 0) {  // the request of token t
    int b = -1;
    int64_t start = 0, base = 0;
    for (int b0 = 0; b0 < a.batch_size && b < 0; b0 += 32) {
      int64_t e = b0 + lane < a.batch_size ? a.extend_lens[b0 + lane] : 0;
      if (e < 0) e = 0;
      int64_t incl = e;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, base + incl > t);
      if (hit) {
        const int l = __ffs(hit) - 1;
        b = b0 + l;
        start = base + __shfl_sync(0xffffffffu, incl - e, l);
      }
      base += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) { sh_b = b; sh_start = start; }
  }
  __syncthreads();
  const int b = sh_b;
  if (b < 0 || b >= a.batch_size) return;  // a token behind the last request: left as it was
  int64_t L = a.seq_lens[b];
  const int64_t E = a.extend_lens ? a.extend_lens[b] : 1;
  if (a.extend_lens ? (L > a.r2t_cols || L < E) : L > a.r2t_cols) {
    if (tid == 0) record_err(a.err, TF_KERR_SLOT_RANGE);
    if (a.extend_lens) return;
    L = a.r2t_cols;
  }
  const int64_t limit = L - E + (t - sh_start) + 1;  // keys j < limit are visible
  int64_t row = a.req_pool_indices[b];
  if (row < 0 || row >= a.r2t_rows) {
    if (tid == 0) record_err(a.err, TF_KERR_REQ_RANGE);
    row = 0;
  }
  const int64_t* r2t = a.req_to_token + row * a.r2t_stride;

  const T* q = reinterpret_cast<const T*>(a.q);
  for (int e = tid; e < G * D; e += kThreads) {
    const int g = e / D, d = e - g * D;
    q_s[e] = to_f(q[t * a.q_stride_tok + (int64_t)(h * G + g) * a.q_stride_head + d]);
    o_s[e] = 0.f;
  }
  if (tid < G) { m_s[tid] = -INFINITY; l_s[tid] = 0.f; }

  const uint8_t* kb = reinterpret_cast<const uint8_t*>(a.k_buffer) + (int64_t)h * a.kv_stride_head;
  const uint8_t* vb = reinterpret_cast<const uint8_t*>(a.v_buffer) + (int64_t)h * a.kv_stride_head;
  for (int64_t j0 = 0; j0 < limit; j0 += kBK) {
    const int nvalid = (int)(limit - j0 < kBK ? limit - j0 : kBK);
    if (tid < nvalid) {
      const int64_t s = resolve_slot(r2t[j0 + tid], a.num_slots, a.slot_mode, a.err);
      slot_s[tid] = s * a.kv_stride_slot;
      const float2 v = *reinterpret_cast<const float2*>(sc.data + s * sc.stride_slot +
                                                        (int64_t)h * sc.stride_head);
      sc_s[2 * tid] = v.x;
      sc_s[2 * tid + 1] = v.y;
    }
    __syncthreads();
    for (int e = tid; e < nvalid * D; e += kThreads) {
      const int j = e / D, d = e - j * D;
      k_s[j * (D + 1) + d] = kv8::decode1(kb[slot_s[j] + d]) * sc_s[2 * j];
      v_s[j * D + d] = kv8::decode1(vb[slot_s[j] + d]) * sc_s[2 * j + 1];
    }
    __syncthreads();
    for (int p = tid; p < G * kBK; p += kThreads) {
      const int g = p / kBK, j = p - g * kBK;
      float s = -INFINITY;
      if (j < nvalid) {
        float acc = 0.f;
        const float* qq = q_s + g * D;
        const float* kk = k_s + j * (D + 1);
        for (int d = 0; d < D; ++d) acc = fmaf(qq[d], kk[d], acc);
        s = acc * a.scale;
      }
      p_s[p] = s;
    }
    __syncthreads();
    for (int g = warp; g < G; g += kThreads / 32) {
      const float s = p_s[g * kBK + lane];
      const float m_old = m_s[g];
      const float m_new = fmaxf(m_old, warp_max(s));
      const float p = lane < nvalid ? expf(s - m_new) : 0.f;
      const float alpha = m_old == -INFINITY ? 0.f : expf(m_old - m_new);
      const float psum = warp_sum(p);
      p_s[g * kBK + lane] = p;
      __syncwarp();
      if (lane == 0) { m_s[g] = m_new; l_s[g] = l_s[g] * alpha + psum; al_s[g] = alpha; }
    }
    __syncthreads();
    for (int e = tid; e < G * D; e += kThreads) {
      const int g = e / D, d = e - g * D;
      float acc = o_s[e] * al_s[g];
      const float* pp = p_s + g * kBK;
      for (int j = 0; j < nvalid; ++j) acc = fmaf(pp[j], v_s[j * D + d], acc);
      o_s[e] = acc;
    }
    __syncthreads();
  }
  __syncthreads();

  T* out = reinterpret_cast<T*>(a.out);
  const T* gate = reinterpret_cast<const T*>(a.gate);
  for (int e = tid; e < G * D; e += kThreads) {
    const int g = e / D, d = e - g * D;
    const int hq = h * G + g;
    float o = o_s[e] / l_s[g];  // no keys: 0 / 0, NaN
    if (a.gate_mode != TF_GATE_NONE) {
      const float x = to_f(gate[t * a.gate_stride_tok + (int64_t)hq * a.gate_stride_head + d]);
      const float sg = 1.0f / (1.0f + expf(-x));
      o *= a.gate_mode == TF_GATE_SILU ? x * sg : sg;
    }
    out[t * a.out_stride_tok + (int64_t)hq * a.out_stride_head + d] = from_f<T>(o);
  }
}

size_t simt_smem_bytes(int G, int D) {
  return 4 * (2 * (size_t)kBK + 2 * (size_t)G * D + kBK * (size_t)(D + 1) + kBK * (size_t)D +
              (size_t)G * kBK + 2 * (size_t)kBK + 3 * (size_t)G);
}

template <typename T>
cudaError_t launch_t(const tf_paged_attn_args& a, const tf_kv_scale& sc, cudaStream_t s) {
  const int G = a.num_q_heads / a.num_kv_heads;
  const size_t smem = simt_smem_bytes(G, a.head_dim);
  cudaError_t e = cudaFuncSetAttribute(paged_fp8_simt_kernel<T>,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  dim3 grid((unsigned)a.num_tokens, (unsigned)a.num_kv_heads);
  paged_fp8_simt_kernel<T><<<grid, kThreads, smem, s>>>(a, sc);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_paged_fp8_simt(const tf_paged_attn_args& a, const tf_kv_scale& sc,
                                  cudaStream_t s) {
  if (a.num_tokens == 0) return cudaSuccess;
  switch (a.dtype) {
    case TF_DTYPE_F32: return launch_t<float>(a, sc, s);
    case TF_DTYPE_BF16: return launch_t<__nv_bfloat16>(a, sc, s);
    default: return launch_t<__half>(a, sc, s);
  }
}

}  // namespace tf
