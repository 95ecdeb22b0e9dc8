// Paged GQA attention over the 8-bit K/V pool on CUDA cores, for any dtype (fp32 / bf16 / fp16) and
// any head_dim <= 256, decode and extend: the path of the fp32 configurations and of the shapes the
// tensor-core kernels are not built for.  One CTA per (query token, kv head) computes the
// G = Hq/Hkv query heads that share the kv head, so every K/V row is read once per group; rows are
// multiplied by their scale as they enter shared memory, and everything after that is fp32 up to
// the one rounding of the output.
//
// A call of this kind is small, so what bounds it is the chain table entry -> row -> shared memory
// -> scores -> sum of each block of 32 keys.  The table's entries run two blocks ahead and the rows
// one, in registers, 16 threads to a row, and the lanes of the warp that holds a head's 32 scores
// take their softmax without another exchange.  4 requests of 17 to 96 tokens, 8 heads over 2,
// head_dim 64, fp32: 11.7 to 12.3 us, 30.7 us with rows loaded byte by byte when they were needed.
#include "common.cuh"
#include "kv_fp8.cuh"
#include "launch.h"

namespace tf {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kBK = 32;           // keys per block: one per lane of the softmax
constexpr int kRowThreads = 16;   // neighbouring threads that load one row
constexpr int kRowsPerThread = 2 * kBK * kRowThreads / kThreads;  // K rows first, then V rows
constexpr int kWords = 256 / 4 / kRowThreads;                     // words of a row per thread

// four codes at p of which n are inside the row
template <bool VEC>
__device__ __forceinline__ uint32_t load_word(const uint8_t* p, int n) {
  if (VEC) return n > 0 ? *reinterpret_cast<const uint32_t*>(p) : 0u;
  uint32_t w = 0;
  for (int i = 0; i < 4 && i < n; ++i) w |= (uint32_t)p[i] << (8 * i);
  return w;
}

// VEC: rows start at multiples of four bytes and head_dim is a multiple of four.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) paged_fp8_simt_kernel(tf_paged_attn_args a,
                                                                  tf_kv_scale sc) {
  const int64_t t = blockIdx.x;
  const int h = blockIdx.y;
  const int G = a.num_q_heads / a.num_kv_heads;
  const int D = a.head_dim;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  const int DP = (D + 3) & ~3;     // rows of q and o, zero behind head_dim
  const int KP = DP + 4;           // rows of k and v: eight lanes' float4 in different banks
  extern __shared__ __align__(16) float smem[];
  float* q_s = smem;                         // [G][DP]
  float* o_s = q_s + G * DP;                 // [G][DP]
  float* k_s = o_s + G * DP;                 // [kBK][KP]
  float* v_s = k_s + kBK * KP;               // [kBK][KP]
  float* p_s = v_s + kBK * KP;               // [G][kBK]
  float* m_s = p_s + G * kBK;                // [G]
  float* l_s = m_s + G;                      // [G]
  float* al_s = l_s + G;                     // [G]
  __shared__ int64_t slot_s[2][kBK];         // of this block and the next
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

  auto slot_of = [&](int64_t j) {
    return j < limit ? resolve_slot(r2t[j], a.num_slots, a.slot_mode, a.err) : (int64_t)-1;
  };
  if (tid < 2 * kBK) slot_s[tid / kBK][lane] = slot_of(tid);

  const T* q = reinterpret_cast<const T*>(a.q);
  for (int e = tid; e < G * DP; e += kThreads) {
    const int g = e / DP, d = e - g * DP;
    q_s[e] = d < D ? to_f(q[t * a.q_stride_tok + (int64_t)(h * G + g) * a.q_stride_head + d]) : 0.f;
    o_s[e] = 0.f;
  }
  if (tid < G) { m_s[tid] = -INFINITY; l_s[tid] = 0.f; }
  __syncthreads();

  const uint8_t* kb = reinterpret_cast<const uint8_t*>(a.k_buffer) + (int64_t)h * a.kv_stride_head;
  const uint8_t* vb = reinterpret_cast<const uint8_t*>(a.v_buffer) + (int64_t)h * a.kv_stride_head;
  const int tx = tid % kRowThreads, ty = tid / kRowThreads;
  uint32_t code[kRowsPerThread][kWords];  // the next block, in flight during this one's arithmetic
  float rs[kRowsPerThread];
  auto load = [&](int buf) {
#pragma unroll
    for (int i = 0; i < kRowsPerThread; ++i) {
      const int r = ty + i * (kThreads / kRowThreads);
      const bool is_v = r >= kBK;
      const int64_t s = slot_s[buf][r % kBK];
      const uint8_t* p = (is_v ? vb : kb) + (s < 0 ? 0 : s) * a.kv_stride_slot;
      rs[i] = s < 0 ? 0.f : sc.data[s * sc.stride_slot + (int64_t)h * sc.stride_head + is_v];
#pragma unroll
      for (int c = 0; c < kWords; ++c) {
        const int d = 4 * (tx + c * kRowThreads);
        code[i][c] = s < 0 ? 0u : load_word<VEC>(p + d, D - d);
      }
    }
  };
  if (limit > 0) load(0);

  for (int64_t j0 = 0; j0 < limit; j0 += kBK) {
    const int buf = (int)(j0 / kBK) & 1;
    const int nvalid = (int)(limit - j0 < kBK ? limit - j0 : kBK);
#pragma unroll
    for (int i = 0; i < kRowsPerThread; ++i) {
      const int r = ty + i * (kThreads / kRowThreads);
      float* dst = (r >= kBK ? v_s : k_s) + (r % kBK) * KP;
      // NaN for a scale of infinity too: a K row of infinities could make a logit of -inf, and its token
      // would vanish
      const float mul = rs[i] + (rs[i] - rs[i]);
#pragma unroll
      for (int c = 0; c < kWords; ++c) {
        const int d = 4 * (tx + c * kRowThreads);
        if (d >= DP) break;
        const uint32_t w = code[i][c];
        float4 x;
        x.x = kv8::decode1(w & 0xff) * mul;
        x.y = kv8::decode1((w >> 8) & 0xff) * mul;
        x.z = kv8::decode1((w >> 16) & 0xff) * mul;
        x.w = kv8::decode1(w >> 24) * mul;
        if (!VEC) {  // a scale that is not finite must not reach the padding
          if (d + 1 >= D) x.y = 0.f;
          if (d + 2 >= D) x.z = 0.f;
          if (d + 3 >= D) x.w = 0.f;
        }
        *reinterpret_cast<float4*>(dst + d) = x;
      }
    }
    __syncthreads();
    if (j0 + kBK < limit) load(buf ^ 1);
    const int64_t after = tid < kBK ? slot_of(j0 + 2 * kBK + lane) : -1;

    // scores and softmax: a warp's lanes are the block's keys, a warp's heads are its own
    for (int g = warp; g < G; g += kWarps) {
      const float4* qq = reinterpret_cast<const float4*>(q_s + g * DP);
      const float4* kk = reinterpret_cast<const float4*>(k_s + lane * KP);
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (int d = 0; d < DP / 4; ++d) {
        const float4 x = qq[d], y = kk[d];
        acc.x = fmaf(x.x, y.x, acc.x);
        acc.y = fmaf(x.y, y.y, acc.y);
        acc.z = fmaf(x.z, y.z, acc.z);
        acc.w = fmaf(x.w, y.w, acc.w);
      }
      const float s = lane < nvalid ? ((acc.x + acc.y) + (acc.z + acc.w)) * a.scale : -INFINITY;
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
    for (int e = tid; e < G * (DP / 4); e += kThreads) {
      const int g = e / (DP / 4), d = 4 * (e - g * (DP / 4));
      float4 acc = *reinterpret_cast<const float4*>(o_s + g * DP + d);
      const float al = al_s[g];
      acc.x *= al; acc.y *= al; acc.z *= al; acc.w *= al;
      const float* pp = p_s + g * kBK;
#pragma unroll 8
      for (int j = 0; j < kBK; ++j) {  // rows behind the last key are zeros
        const float4 v = *reinterpret_cast<const float4*>(v_s + j * KP + d);
        const float p = pp[j];
        acc.x = fmaf(p, v.x, acc.x);
        acc.y = fmaf(p, v.y, acc.y);
        acc.z = fmaf(p, v.z, acc.z);
        acc.w = fmaf(p, v.w, acc.w);
      }
      *reinterpret_cast<float4*>(o_s + g * DP + d) = acc;
    }
    if (tid < kBK) slot_s[buf][lane] = after;
    __syncthreads();
  }

  T* out = reinterpret_cast<T*>(a.out);
  const T* gate = reinterpret_cast<const T*>(a.gate);
  for (int e = tid; e < G * D; e += kThreads) {
    const int g = e / D, d = e - g * D;
    const int hq = h * G + g;
    float o = o_s[g * DP + d] / l_s[g];  // no keys: 0 / 0, NaN
    if (a.gate_mode != TF_GATE_NONE) {
      const float x = to_f(gate[t * a.gate_stride_tok + (int64_t)hq * a.gate_stride_head + d]);
      const float sg = 1.0f / (1.0f + expf(-x));
      o *= a.gate_mode == TF_GATE_SILU ? x * sg : sg;
    }
    out[t * a.out_stride_tok + (int64_t)hq * a.out_stride_head + d] = from_f<T>(o);
  }
}

size_t simt_smem_bytes(int G, int D) {
  const size_t dp = (D + 3) & ~3;
  return 4 * (2 * (size_t)G * dp + 2 * kBK * (dp + 4) + (size_t)G * kBK + 3 * (size_t)G);
}

template <typename T, bool VEC>
cudaError_t launch_v(const tf_paged_attn_args& a, const tf_kv_scale& sc, cudaStream_t s) {
  const int G = a.num_q_heads / a.num_kv_heads;
  const size_t smem = simt_smem_bytes(G, a.head_dim);
  cudaError_t e = cudaFuncSetAttribute(paged_fp8_simt_kernel<T, VEC>,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  dim3 grid((unsigned)a.num_tokens, (unsigned)a.num_kv_heads);
  paged_fp8_simt_kernel<T, VEC><<<grid, kThreads, smem, s>>>(a, sc);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_t(const tf_paged_attn_args& a, const tf_kv_scale& sc, cudaStream_t s) {
  const bool vec = ((reinterpret_cast<uintptr_t>(a.k_buffer) |
                     reinterpret_cast<uintptr_t>(a.v_buffer) | (uintptr_t)a.kv_stride_slot |
                     (uintptr_t)a.kv_stride_head | (uintptr_t)a.head_dim) & 3) == 0;
  return vec ? launch_v<T, true>(a, sc, s) : launch_v<T, false>(a, sc, s);
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
