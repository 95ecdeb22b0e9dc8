// Paged GQA attention over the 8-bit K/V pool for few query rows per kv head: decode, and extends of
// a few tokens per request (drafted tokens).  HBM-bound: every K/V row is read once.
//
// Mathematics.  A token j has codes K8_j, V8_j and scales ks_j, vs_j; a query row has logits
//   s_j = (q . K8_j) ks_j scale log2(e)      out = sum_j 2^(s_j) vs_j V8_j / sum_j 2^(s_j).
// Both products run as mma.m16n8k16 f16 with fp32 sums.  e4m3 codes are exact in f16; q is scaled by
// a power of two per row into f16's range (exact for bfloat16 too); the only rounding before the
// output is that of the weights w_j = 2^(s_j - M) vs_j 2^7 to f16 (11 bits).  With ev_j the exponent of
// vs_j, M is the running maximum of s_j + ev_j over the tokens that the row sees: its largest w is in
// [2^7, 2^8) whatever the scales are, and only weights 2^21 below it are subnormal in f16.  (With one
// exponent for a tile, a token of a large scale took the bits of its neighbours' weights, also for rows
// that do not see it.)  The sum of weights l = sum 2^(s_j - M) is fp32 (for float16, of the weights as
// rounded), kept times 2^40 so that no scale takes it out of range.
// mma.m16n8k32 on the codes themselves was measured at 36 clocks a warp instruction, against 8 for
// the f16 form with half its depth plus its conversions.
//
// Measured (bf16, 32 heads over 4, head_dim 256).  128 decode requests of 512 to 8192 tokens: 225 to 239 us, 4.9 to
// 5.2 TB/s (0.75 to 0.79 of the copy rate; 6.8 TB/s between the first tile and the last piece, the rest
// is the plan, 4 us, the epilogues and the combine kernel, 9 us).  One request of 8191: 22.5 us, of which
// the combine kernel 8 us.  24 requests with 2 to 5 new tokens: 104 us, bound by instruction latency
// with two warps a scheduler (33% of issue slots; the registers hold no third).
//
// Fragments.  S^T = K8.Q^T: A = 16 tokens x 16 dims.  A thread's 16-byte read of a token's row is its A
// fragment of four k-steps for the dim order 64 j + 16 t + 4 i + {0,1 | 2,3} (t = lane % 4), and Q^T is
// held in the same order.  O^T = V8^T.W^T: A = 16 dims x 16 tokens, from ldmatrix.trans on pairs of
// codes and a byte permute; row r of the fragment is dim 2 r, row r + 8 dim 2 r + 1.  W^T comes from
// the logits' layout through movmatrix.
//
// Work.  A CTA has eight warps.  TEAM of them (one, or two above eight query rows) share stages of 32
// tokens of one kv head, fetch them in turn and take eight query rows each, sixteen of them above 16 rows (two
// row tiles on the same converted codes: 64 rows of a kv head 169 us, 192 us with eight rows a warp and
// teams of eight); more rows than a team holds take further passes.  HG kv heads of a group run side by
// side, so that a token's rows of all heads, its scales and its slot id are read at about the same time; the
// WH = 8 / (TEAM HG) teams of a head take its tiles in turn and merge in shared memory.  The sequence
// of (request, pass, head group) units, each of ceil(len / 32) tiles, is cut into one range per CTA,
// balanced by tiles plus a fixed cost per unit; every CTA finds its own range from the lengths (a scan
// of the batch in shared memory: no plan launch).  Units cut by a boundary leave (M, l, O) partials
// for a combine kernel.  Rows are fetched by 16-byte cp.async (a bulk copy per row was measured at
// 528 us against 349 us for 128 requests: copies of 256 bytes), a stage's copies completing on its
// mbarrier, and the ring of stages runs on across units.
#include <type_traits>

#include "common.cuh"
#include "kv_fp8.cuh"
#include "launch.h"

namespace tf {
namespace rows8 {

constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kTok = 32;  // tokens of a tile
constexpr int kCache = 96;  // requests whose metadata a CTA keeps in shared memory
constexpr float kLog2e = 1.4426950408889634f;
// Exponentials 2^(s - M) and their sum are kept times 2^40: as M is the maximum of s + ev, the largest of
// them is between 2^-119 (the store's largest scale) and 2^50 (its smallest), and fp32 has room around both.
constexpr float kBiasLog2 = 40.f, kBias = 0x1p40f;
constexpr int kMaxCtas = 256;
constexpr int kMaxBatch = 32768;  // passes of all requests: their scan lives in the ring's shared memory

// One pass over a request's tokens for the query rows that a team holds; a request has as many passes
// as the longest one needs, those behind its own rows without tiles.
struct ReqMeta {
  int32_t len, ext, row, start, nt;  // tokens, new tokens, req_to_token row, first query token, tiles
};

// NT: 8-row tiles of a warp
template <int D, int NT>
struct Cfg {
  static constexpr int kRows = 8 * NT;  // query rows of a warp
  // row strides in shared memory: 64 mod 128 bytes for the 16-byte fragment reads of K (two rows a
  // phase), an odd multiple of 16 for the 8-row matrices of V
  static constexpr int kKS = D % 128 == 0 ? D + 64 : D;
  static constexpr int kVS = D + 16;
  static constexpr int kOffV = kTok * kKS;
  static constexpr int kOffScale = kOffV + kTok * kVS;
  static constexpr int kStage = kOffScale + kTok * 8;
  static constexpr int kStages = D == 256 ? 12 : (D == 128 ? 20 : 40);  // at most
  // epilogue: 64 dims of each warp's rows (the place of its Q fragments, with two row tiles), then per
  // row what it is multiplied by, (M, l), and its place in the output
  static constexpr int kEpiStride = 64 + 4;  // floats per row
  static constexpr int kEpiRows = kRows * kEpiStride * 4, kQ = NT > 1 ? kRows * D * 2 : 0;
  static constexpr int kEpiWarp = kEpiRows > kQ ? kEpiRows : kQ;  // bytes of a warp
  static constexpr int kEpi = kWarps * (kEpiWarp + kRows * 5 * 4);
  static constexpr int kFixed = kCache * (int)sizeof(ReqMeta) + 64;
  static_assert(kStage % 16 == 0 && kKS % 16 == 0 && kVS % 16 == 0, "bulk copy alignment");
};

// What a launch is divided by; computed on the host.
struct Shape {
  int team, hg, wh;   // warps sharing a ring, kv heads side by side, teams taking a head's tiles in turn
  int groups;         // units of a pass: head groups
  int passes;         // passes of a request (more query rows than a team holds)
  int row_tiles;      // 8-row tiles of a warp
  int stages;         // ring stages
  int nctas;
  int min_tiles;      // tiles worth a CTA of their own
  int piece_cost;     // fixed cost of a unit in tiles
  int smem, ring;     // bytes
};

// The unit that a CTA's range starts in, for the combine kernel.
struct CutInfo {
  int pass, u, start, ext, nt, t0;
};

struct Ws {
  int64_t* cta_g;  // [nctas + 1] first tile of each CTA's range
  CutInfo* cut;    // [nctas]
  float* ml;       // [2 nctas][8 warps][rows][2]
  float* o;        // [2 nctas][8 warps][rows][D]
};

__host__ __device__ inline size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }
__host__ __device__ inline Ws carve(void* base, int nctas, int rows) {
  char* p = (char*)base;
  Ws w;
  w.cta_g = (int64_t*)p;
  p += align256((size_t)(nctas + 1) * 8);
  w.cut = (CutInfo*)p;
  p += align256((size_t)nctas * sizeof(CutInfo));
  w.ml = (float*)p;
  p += align256((size_t)2 * nctas * kWarps * rows * 2 * 4);
  w.o = (float*)p;
  return w;
}
inline size_t ws_bytes(int nctas, int rows, int D) {
  return align256((size_t)(nctas + 1) * 8) + align256((size_t)nctas * sizeof(CutInfo)) +
         align256((size_t)2 * nctas * kWarps * rows * 2 * 4) +
         (size_t)2 * nctas * kWarps * rows * D * 4;
}

__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                      uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the low and the high two codes of a word as f16 pairs
__device__ __forceinline__ uint32_t cvt_lo(uint32_t w) {
  uint32_t r;
  asm("{\n .reg .b16 a, b;\n mov.b32 {a, b}, %1;\n cvt.rn.f16x2.e4m3x2 %0, a;\n}" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ uint32_t cvt_hi(uint32_t w) {
  uint32_t r;
  asm("{\n .reg .b16 a, b;\n mov.b32 {a, b}, %1;\n cvt.rn.f16x2.e4m3x2 %0, b;\n}" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ void ldsm4_t(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a));
}
__device__ __forceinline__ uint32_t movmatrix_t(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Stage use counters.  A stage passes from team to team, and one team can be more than a ring ahead of
// another, so "consumed in round r" is a count that only grows: an mbarrier's parity cannot tell a
// round from the one before the last.
__device__ __forceinline__ void count_use(uint32_t* c) {
  asm volatile("red.release.cta.shared::cta.add.u32 [%0], 1;" ::"r"(smem_u32(c)) : "memory");
}
__device__ __forceinline__ uint32_t uses(const uint32_t* c) {
  uint32_t v;
  asm volatile("ld.acquire.cta.shared::cta.u32 %0, [%1];" : "=r"(v) : "r"(smem_u32(c)) : "memory");
  return v;
}
__device__ __forceinline__ bool wait_uses(const uint32_t* c, uint32_t n) {  // bounded
  if (uses(c) >= n) return true;
  const uint64_t t0 = global_ns();
  for (uint32_t it = 0;; ++it) {
    if (uses(c) >= n) return true;
    if ((it & 63u) == 63u && global_ns() - t0 > kSpinLimitNs) return false;
  }
}
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }  // -126..127
// 2^((from - to) / 2), from <= to: sums relative to `from` times its square are relative to `to`.  A sum of
// weights is multiplied by it twice: maxima of s + ev can be more than fp32's 2^126 apart where the sums
// of 2^s are not.
__device__ __forceinline__ float fade(float from, float to) {
  return from == to ? 1.f : ex2(0.5f * (from - to));
}

// tiles of a request: none when it has no query rows or a length its table cannot hold
__device__ __forceinline__ int64_t checked_len(const tf_paged_attn_args& a, int b, int64_t& ext,
                                               bool& bad) {
  int64_t L = a.seq_lens[b];
  ext = a.extend_lens ? a.extend_lens[b] : 1;
  if (ext < 0) ext = 0;
  bad = false;
  if (L < 0) L = 0;
  if (a.extend_lens == nullptr) {
    if (L > a.r2t_cols) { bad = true; L = a.r2t_cols; }
  } else if (ext > 0 && (L > a.r2t_cols || L < ext)) {
    bad = true;
    ext = 0;
  }
  return L;
}
// tiles of pass p: those of the request when it has rows there
__device__ __forceinline__ int tiles_of(int64_t L, int64_t ext, int p, const Shape& sh, int G) {
  return ext * G > (int64_t)p * sh.team * sh.row_tiles * 8 ? (int)((L + kTok - 1) / kTok) : 0;
}

// The passes a walk can be at (pass b % passes of request b / passes): the first kCache of the range
// from shared memory, further ones from global memory as the walk reaches them.
struct Requests {
  const tf_paged_attn_args& a;
  const Shape& sh;
  const ReqMeta* cache;
  int b0, n, G;
  __device__ __forceinline__ ReqMeta at(int b, int start) const {
    if (b - b0 < n) return cache[b - b0];
    const int i = b / sh.passes;
    int64_t ext;
    bool bad;
    ReqMeta m;
    m.len = (int32_t)checked_len(a, i, ext, bad);
    m.ext = (int32_t)ext;
    m.nt = tiles_of(m.len, ext, b - i * sh.passes, sh, G);
    const int64_t r = a.req_pool_indices[i];
    if (r < 0 || r >= a.r2t_rows) record_err(a.err, TF_KERR_REQ_RANGE);
    m.row = r < 0 || r >= a.r2t_rows ? 0 : (int32_t)r;
    m.start = start;
    return m;
  }
};

// The units of a CTA's range in order; tiles are counted from the range's first.
struct Walker {
  int b, u;     // pass and group
  int unit_g;   // first tile of unit (b, u)
  ReqMeta m;
  __device__ __forceinline__ int nt() const { return m.nt; }
  // the unit that holds tile q (of the current unit or a later one)
  __device__ __forceinline__ void seek(const Requests& rq, int q) {
    while (q >= unit_g + nt()) {
      unit_g += nt();
      if (++u == rq.sh.groups) {
        u = 0;
        int before = 0;  // query tokens between the two passes (the cache knows them)
        if (b + 1 - rq.b0 >= rq.n && (b + 1) % rq.sh.passes == 0)
          before = rq.a.extend_lens ? max((int)rq.a.extend_lens[b / rq.sh.passes], 0) : 1;
        ++b;
        m = rq.at(b, m.start + before);
      }
    }
  }
};

// 4 gate values of a query row at dims d..; v8: rows can be moved in 8-byte pieces
template <typename T>
__device__ __forceinline__ uint2 gate4(const tf_paged_attn_args& a, int64_t tok, int hq, int d, bool v8) {
  const T* gp = (const T*)a.gate + tok * a.gate_stride_tok + (int64_t)hq * a.gate_stride_head + d;
  if (v8) return __ldg(reinterpret_cast<const uint2*>(gp));
  const unsigned short* u = reinterpret_cast<const unsigned short*>(gp);
  return make_uint2(u[0] | ((uint32_t)u[1] << 16), u[2] | ((uint32_t)u[3] << 16));
}
// 4 output values, times the gate's activation
template <typename T>
__device__ __forceinline__ void put4(const tf_paged_attn_args& a, int64_t tok, int hq, int d, float4 x,
                                     uint2 gw, bool v8) {
  float o[4] = {x.x, x.y, x.z, x.w};
  if (a.gate_mode != TF_GATE_NONE) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float g = i & 1 ? unpack_hi<T>(i < 2 ? gw.x : gw.y) : unpack_lo<T>(i < 2 ? gw.x : gw.y);
      const float sg = sigmoid_f(g);
      o[i] *= a.gate_mode == TF_GATE_SILU ? g * sg : sg;
    }
  }
  T* op = (T*)a.out + tok * a.out_stride_tok + (int64_t)hq * a.out_stride_head + d;
  const uint32_t p0 = pack2_rn<T>(o[0], o[1]), p1 = pack2_rn<T>(o[2], o[3]);
  if (v8) {
    *reinterpret_cast<uint2*>(op) = make_uint2(p0, p1);
  } else {
    unsigned short* u = reinterpret_cast<unsigned short*>(op);
    u[0] = (unsigned short)p0;
    u[1] = (unsigned short)(p0 >> 16);
    u[2] = (unsigned short)p1;
    u[3] = (unsigned short)(p1 >> 16);
  }
}
__device__ __forceinline__ bool rows_v8(const tf_paged_attn_args& a) {
  return ((reinterpret_cast<uintptr_t>(a.out) | reinterpret_cast<uintptr_t>(a.gate)) & 7) == 0 &&
         ((a.out_stride_tok | a.out_stride_head | a.gate_stride_tok | a.gate_stride_head) & 3) == 0;
}

// 64 dims (d0..) of every row of a piece from the epilogue buffer: the teams of a head are summed, and
// the result is normalised and put out, or left as partials.  One copy of this code serves all
// pieces and dims: unrolled into the kernel it ran once a piece from a cold instruction cache
// (15-35 us a piece were measured).
template <typename T, int D, int NT>
__device__ __noinline__ void finish64(const tf_paged_attn_args& a, const Shape& sh, const Ws& ws,
                                      const float* epi, int slot, bool whole, int d0) {
  using C = Cfg<D, NT>;
  constexpr int kRows = C::kRows, kS = C::kEpiStride;
  constexpr int kTwo = 2;  // items of a thread whose gate values are requested together
  const float* fac = epi + kWarps * C::kEpiWarp / 4;    // [warp][row] what the warp's row counts
  const float* ml = fac + kWarps * kRows;               // [warp][row][2]; the first team's: merged
  const int2* to = reinterpret_cast<const int2*>(ml + 2 * kWarps * kRows);  // [place][row] token (or -1), head
  const int per = sh.hg * sh.team;
  const bool v8 = rows_v8(a), gated = whole && a.gate_mode != TF_GATE_NONE;
#pragma unroll 1
  for (int e0 = threadIdx.x; e0 < per * kRows * 16; e0 += kTwo * kThreads) {
    int2 th[kTwo];
    uint2 gw[kTwo];
#pragma unroll
    for (int k = 0; k < kTwo; ++k) {
      const int e = e0 + k * kThreads;
      th[k] = make_int2(-1, 0);
      gw[k] = make_uint2(0, 0);
      if (e < per * kRows * 16) {
        th[k] = to[e >> 4];
        if (gated && th[k].x >= 0) gw[k] = gate4<T>(a, th[k].x, th[k].y, d0 + 4 * (e & 15), v8);
      }
    }
#pragma unroll
    for (int k = 0; k < kTwo; ++k) {
      const int e = e0 + k * kThreads;
      if (th[k].x < 0) continue;
      const int v = e & 15, pr = e >> 4;  // place * kRows + row
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
      for (int w = pr; w < kWarps * kRows; w += per * kRows) {
        const float f = fac[w];
        const float4 x = *reinterpret_cast<const float4*>(epi + (w / kRows) * (C::kEpiWarp / 4) +
                                                          (w % kRows) * kS + 4 * v);
        o.x = fmaf(f, x.x, o.x);
        o.y = fmaf(f, x.y, o.y);
        o.z = fmaf(f, x.z, o.z);
        o.w = fmaf(f, x.w, o.w);
      }
      if (whole) {
        const float inv = (kBias / 128.f) / ml[2 * pr + 1];
        put4<T>(a, th[k].x, th[k].y, d0 + 4 * v, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv), gw[k], v8);
      } else {
        const int64_t ps = (int64_t)slot * kWarps * kRows + pr;
        *reinterpret_cast<float4*>(ws.o + ps * D + d0 + 4 * v) = o;
        if (d0 == 0 && v == 0) *reinterpret_cast<float2*>(ws.ml + ps * 2) = make_float2(ml[2 * pr], ml[2 * pr + 1]);
      }
    }
  }
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kThreads, 1)
    rows_kernel(const __grid_constant__ tf_paged_attn_args a, const __grid_constant__ tf_kv_scale sc,
                const __grid_constant__ Shape sh, const __grid_constant__ Ws ws) {
  using C = Cfg<D, NT>;
  constexpr int kRows = C::kRows;
  constexpr int NJ = D / 64;   // 16-byte reads of a K row per thread
  constexpr int NM = D / 16;   // dim tiles of O
  extern __shared__ __align__(128) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int gq = lane >> 2, tq = lane & 3;
  const int P = sh.passes, B = a.batch_size * P;  // passes over all requests
  const int G = a.num_q_heads / a.num_kv_heads;
  const int c = blockIdx.x;

  ReqMeta* cache = reinterpret_cast<ReqMeta*>(smem + sh.ring);
  int* sh_i = reinterpret_cast<int*>(cache + kCache);  // [16] words, 8-byte aligned
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + sh.ring + C::kFixed);
  uint32_t* used = reinterpret_cast<uint32_t*>(bars + sh.stages);  // warps done with a stage, in all

  // the combine kernel's CTAs may take their places now; they wait for this grid
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // ---- this CTA's range: ts[b] = first tile of pass b (all groups of a pass are adjacent)
  int* ts = reinterpret_cast<int*>(smem);  // in the ring's space, before its first copy
  const int plan_per = (B + kThreads - 1) / kThreads;
  const int plan_lo = min(tid * plan_per, B), plan_hi = min(plan_lo + plan_per, B);
  ReqMeta mine_m = {0, 0, 0, 0, 0};  // of pass plan_lo when every thread has at most one
  if (plan_per == 1 && plan_lo < B) {
    const int64_t r = a.req_pool_indices[plan_lo / P];
    mine_m.row = r < 0 || r >= a.r2t_rows ? -1 : (int32_t)r;
  }
  {
    const int lo = plan_lo, hi = plan_hi;
    int sum = 0;
    for (int b = lo; b < hi; ++b) {
      int64_t ext;
      bool bad;
      const int64_t L = checked_len(a, b / P, ext, bad);
      if (bad && c == 0) record_err(a.err, TF_KERR_SLOT_RANGE);
      mine_m.len = (int32_t)L;
      mine_m.ext = (int32_t)ext;
      mine_m.nt = tiles_of(L, ext, b % P, sh, G);
      ts[b] = sum;
      sum += mine_m.nt;
    }
    int incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    if (lane == 31) sh_i[warp] = incl;
    __syncthreads();
    int base = incl - sum;
    for (int w = 0; w < warp; ++w) base += sh_i[w];
    for (int b = lo; b < hi; ++b) ts[b] += base;
    if (tid == kThreads - 1) ts[B] = base + sum;
  }
  __syncthreads();
  const int NG = sh.groups;
  const int64_t total = (int64_t)ts[B] * NG;
  const int64_t want = (total + sh.min_tiles - 1) / sh.min_tiles;
  const int nctas = want < gridDim.x ? (int)want : (int)gridDim.x;
  const int64_t beta = sh.piece_cost;
  // A range begins at cost position x = cc (total + beta units) / nctas: a unit's first beta of cost is
  // fixed.  The pass holding x lies with one thread; the range's first pass with another.
  const int64_t U = (int64_t)B * NG;
  int64_t* sh_g = reinterpret_cast<int64_t*>(sh_i + 8);  // g0, g1
  int* sh_b = sh_i + 12;
  if (tid == 0) { sh_g[0] = sh_g[1] = total; }
  __syncthreads();
#pragma unroll 1
  for (int k = 0; k < 2; ++k) {
    if (c + k >= nctas) continue;
    const int64_t x = (int64_t)(c + k) * (total + beta * U) / nctas;
#pragma unroll 1
    for (int b = plan_lo; b < plan_hi; ++b) {
      const int64_t nt = ts[b + 1] - ts[b], rem = x - ((int64_t)ts[b] + beta * b) * NG;
      if (rem < 0 || rem >= (nt + beta) * NG) continue;
      const int64_t u = rem / (nt + beta);
      int64_t off = rem - u * (nt + beta) - beta;
      sh_g[k] = (int64_t)ts[b] * NG + u * nt + (off < 0 ? 0 : off);
    }
  }
  __syncthreads();
  const int64_t g0 = sh_g[0], g1 = sh_g[1];
  if (tid == 0) {
    ws.cta_g[c] = g0;
    if (c == gridDim.x - 1) ws.cta_g[c + 1] = total;
  }
  // requests without keys: softmax over nothing is NaN
  if (a.extend_lens == nullptr) {
    for (int b = c; b < a.batch_size; b += gridDim.x) {
      if (ts[b * P + 1] != ts[b * P]) continue;
      for (int e = tid; e < a.num_q_heads * D; e += kThreads)
        ((T*)a.out)[(int64_t)b * a.out_stride_tok + (int64_t)(e / D) * a.out_stride_head + e % D] =
            from_f<T>(NAN);
    }
  }
  if (g0 >= g1) return;
#pragma unroll 1
  for (int b = plan_lo; b < plan_hi; ++b)  // the range's first pass: ts[b] NG <= g0 < ts[b + 1] NG
    if ((int64_t)ts[b] * NG <= g0 && g0 < (int64_t)ts[b + 1] * NG) *sh_b = b;
  __syncthreads();
  const int bf = *sh_b;
  const int cn = min(kCache, B - bf);
  const int64_t bf_g = (int64_t)ts[bf] * NG;
  const int bf_nt = ts[bf + 1] - ts[bf];
  int q_before = bf / P;  // query tokens before that request
  if (a.extend_lens != nullptr) {
    int s = 0;
    for (int b = tid; b < bf / P; b += kThreads) s += max((int)a.extend_lens[b], 0);
    s = __reduce_add_sync(0xffffffffu, s);
    __syncthreads();
    if (lane == 0) sh_i[warp] = s;
    __syncthreads();
    q_before = 0;
    for (int w = 0; w < kWarps; ++w) q_before += sh_i[w];
  }
  if (plan_per == 1) {
    if (plan_lo >= bf && plan_lo < bf + cn && plan_hi > plan_lo) {
      if (mine_m.row < 0) {
        record_err(a.err, TF_KERR_REQ_RANGE);
        mine_m.row = 0;
      }
      mine_m.start = plan_lo / P;
      cache[plan_lo - bf] = mine_m;
    }
  } else for (int i = tid; i < cn; i += kThreads) {
    const int b = bf + i;
    int64_t ext;
    bool bad;
    ReqMeta m;
    m.len = (int32_t)checked_len(a, b / P, ext, bad);
    m.ext = (int32_t)ext;
    m.nt = tiles_of(m.len, ext, b % P, sh, G);
    const int64_t r = a.req_pool_indices[b / P];
    if (r < 0 || r >= a.r2t_rows) record_err(a.err, TF_KERR_REQ_RANGE);
    m.row = r < 0 || r >= a.r2t_rows ? 0 : (int32_t)r;
    m.start = b / P;
    cache[i] = m;
  }
  if (tid == 0) {
    for (int i = 0; i < sh.stages; ++i) {
      mbar_init(&bars[i], 32);  // the copies of every lane of the fetching warp have landed
      used[i] = 0;
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();  // ts is dead from here on
  if (a.extend_lens != nullptr && tid == 0) {
    int s = q_before;
    for (int i = 0; i < cn; ++i) {
      cache[i].start = s;
      if ((bf + i + 1) % P == 0) s += max((int)a.extend_lens[(bf + i) / P], 0);
    }
  }
  __syncthreads();

  // ---- this warp's place
  const int member = warp % sh.team;
  const int hsel = (warp / sh.team) % sh.hg;
  const int wsel = warp / (sh.team * sh.hg);
  const uint32_t ring = smem_u32(smem);
  uint64_t* full = bars;
  // tile q of head hsel of the group is number q hg + hsel of the ring
  const int step = sh.wh * sh.hg, first = wsel * sh.hg + hsel;
  const int f_step = sh.wh * sh.team;  // tiles between the ones this warp fetches: a team's warps take turns

  const Requests rq{a, sh, cache, bf, cn, G};
  Walker prod;
  prod.b = bf;
  prod.u = (int)((g0 - bf_g) / bf_nt);
  prod.unit_g = (int)(bf_g + (int64_t)prod.u * bf_nt - g0);
  prod.m = rq.at(bf, 0);
  Walker cons = prod;

  // ---- producer: this team's tiles in sequence, their req_to_token entries kAhead tiles ahead
  const int ntiles = (int)(g1 - g0);
  constexpr int kAhead = 2;
  int64_t raw[kAhead] = {};
  int head[kAhead] = {};           // their kv heads
  int pf = 0, pf_unit = INT32_MIN;  // tiles of the unit whose entries have been asked for; its first tile
  int pq = wsel + sh.wh * member - kAhead * f_step;  // next tile to fetch (before the first: the entries'
  const int f_first = wsel + sh.wh * member;         // own head start)
  int p_st = first + step * member, p_round = 0;     // its stage and round
  bool ok = true;
  auto issue = [&]() {
    if (pq >= f_first) {
      if (p_round > 0)
        ok = __all_sync(0xffffffffu, ok && wait_uses(&used[p_st], (uint32_t)(p_round * sh.team)));
      if (!ok) return;
      const uint32_t sp = ring + (uint32_t)(p_st * C::kStage);
      const int64_t sl = resolve_slot(raw[0], a.num_slots, a.slot_mode, a.err);
      // row offset of this lane's token in 16-byte pieces (32 bits: the host checks)
      const uint32_t off =
          (uint32_t)((sl * a.kv_stride_slot + (int64_t)head[0] * a.kv_stride_head) >> 4);
      constexpr int CPR = D / 16;    // 16-byte pieces of a row
      constexpr int RPI = 32 / CPR;  // rows a warp instruction copies
      const int sub = lane / CPR, ch = lane % CPR;
      const char* kg = (const char*)a.k_buffer + 16 * ch;
      const char* vg = (const char*)a.v_buffer + 16 * ch;
      const uint32_t kd = sp + sub * C::kKS + 16 * ch;
      const uint32_t vd = sp + C::kOffV + sub * C::kVS + 16 * ch;
#pragma unroll
      for (int i0 = 0; i0 < kTok; i0 += 4 * RPI) {
        uint32_t o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = __shfl_sync(0xffffffffu, off, (i0 + i * RPI + sub) & 31);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (i0 + i * RPI >= kTok) break;
          cp_async16(kd + (i0 + i * RPI) * C::kKS, kg + (uint64_t)o[i] * 16);
          cp_async16(vd + (i0 + i * RPI) * C::kVS, vg + (uint64_t)o[i] * 16);
        }
      }
      asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(sp + C::kOffScale + lane * 8),
                   "l"(sc.data + sl * sc.stride_slot + (int64_t)head[0] * sc.stride_head)
                   : "memory");
      cp_async_arrive_noinc(&full[p_st]);
      p_st += step * sh.team;
      if (p_st >= sh.stages) {
        p_st -= sh.stages;
        ++p_round;
      }
    }
#pragma unroll
    for (int i = 0; i + 1 < kAhead; ++i) {
      raw[i] = raw[i + 1];
      head[i] = head[i + 1];
    }
    const int fq = pq + kAhead * f_step;
    if (fq < ntiles) {
      prod.seek(rq, fq);
      // A load behind a saturated memory takes about the time that the ring lasts, more than the tile
      // or two that this one is ahead: the entries of the next 16 to 32 tiles are asked into L2 (16
      // tiles a warp instruction, 128 bytes a lane).
      if (prod.unit_g != pf_unit) {
        pf_unit = prod.unit_g;
        pf = fq - prod.unit_g;
      }
      while (pf < min(fq - prod.unit_g + 17, prod.nt())) {
        const int pos = pf * kTok + lane * 16;
        if (pos < prod.m.len)
          asm volatile("prefetch.global.L2 [%0];" ::"l"(a.req_to_token + (int64_t)prod.m.row * a.r2t_stride + pos));
        pf += 16;
      }
      const int pos = min((fq - prod.unit_g) * kTok + lane, prod.m.len - 1);
      raw[kAhead - 1] = a.req_to_token[(int64_t)prod.m.row * a.r2t_stride + pos];
      head[kAhead - 1] = prod.u * sh.hg + hsel;
    }
    pq += f_step;
  };

  // Tile x of the ring may be fetched once x - stages has been consumed.  A team waits for that only
  // when x - stages is not behind its own current tile in the sequence: whoever has to consume it
  // is then not held up by this team (nor by the barriers at the end of a piece), and as a team's
  // own tiles are at most a ring apart (step <= stages) its next tile is always on its way.  `lag`
  // tiles of slack keep a team from waiting for the slowest warp of the very tile it has just left,
  // where the ring has them beside a tile to work on and one on its way for each team.
  const int lag = min(3, sh.stages >= 2 * step ? sh.stages - 2 * step : sh.stages - step);
  int x_lim = sh.stages - 1;  // the last tile that may be fetched now
  float* epi = reinterpret_cast<float*>(smem + sh.ring + C::kFixed + 16 * sh.stages);
  int cq = wsel, st = first;  // this team's next tile of the range and its stage
  int c_round = 0;
  for (int p0 = 0, p1; p0 < ntiles; p0 = p1) {  // pieces: tiles [p0, p1) of the range
    cons.seek(rq, p0);
    p1 = min(cons.unit_g + cons.nt(), ntiles);
    if (p0 == 0 && tid == 0)
      ws.cut[c] = CutInfo{cons.b % P, cons.u, cons.m.start, cons.m.ext, cons.nt(), -cons.unit_g};
    const int u = cons.u, L = cons.m.len, E = cons.m.ext, pass = cons.b % P;
    const int kvh = u * sh.hg + hsel;
    const int row0 = (pass * sh.team + member) * kRows;  // first of this warp's rows
    const int nrows = E * G - row0;                      // valid ones (may be <= 0)
    const int64_t qtok0 = cons.m.start;

    // the gate rows of the piece are wanted at its end: into L2 now, 128 bytes a thread (a load under
    // a saturated memory takes microseconds)
    if (a.gate_mode != TF_GATE_NONE && p1 == cons.unit_g + cons.nt()) {
      constexpr int kLines = D * 2 / 128 > 0 ? D * 2 / 128 : 1;
      const int per = sh.hg * sh.team;
      for (int e = tid; e < per * kRows * kLines; e += kThreads) {
        const int r = (e / kLines) % kRows, place = e / kLines / kRows;
        const int row = (pass * sh.team + place % sh.team) * kRows + r;
        const int64_t tok = qtok0 + row / G;
        if (row < E * G && tok < a.num_tokens)
          asm volatile("prefetch.global.L2 [%0];" ::"l"(
              (const T*)a.gate + tok * a.gate_stride_tok +
              (int64_t)((u * sh.hg + place / sh.team) * G + row % G) * a.gate_stride_head +
              (e % kLines) * 64));
      }
    }
    // ---- Q: rows gq + 8 n of this warp, dims 64 j + 16 tq + [0, 16), scaled into f16's range
    uint32_t qf[NJ][8];  // of the one row tile; two are kept in shared memory
    uint4* q_frag = reinterpret_cast<uint4*>(reinterpret_cast<unsigned char*>(epi) + warp * C::kEpiWarp) + lane;
    float c2[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = row0 + 8 * n + gq;
      const bool valid = gq + 8 * n < nrows && qtok0 + r / G < a.num_tokens;
      const T* qp = (const T*)a.q + (qtok0 + r / G) * a.q_stride_tok +
                    (int64_t)(kvh * G + r % G) * a.q_stride_head + 16 * tq;
      const bool vec = ((reinterpret_cast<uintptr_t>(a.q) & 15) |
                        ((a.q_stride_tok | a.q_stride_head) & 7)) == 0;
#pragma unroll
      for (int j = 0; j < NJ; ++j) {  // pairs of T
        if (valid && vec) {
#pragma unroll
          for (int hlf = 0; hlf < 2; ++hlf) {
            const uint4 w = *reinterpret_cast<const uint4*>(qp + 64 * j + 8 * hlf);
            qf[j][4 * hlf] = w.x;
            qf[j][4 * hlf + 1] = w.y;
            qf[j][4 * hlf + 2] = w.z;
            qf[j][4 * hlf + 3] = w.w;
          }
        } else {
          const unsigned short* u = reinterpret_cast<const unsigned short*>(qp + 64 * j);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            qf[j][i] = valid ? u[2 * i] | ((uint32_t)u[2 * i + 1] << 16) : 0u;
        }
      }
      uint32_t am = 0;
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          am = max(am, max(kv8::abs_bits(unpack_lo<T>(qf[j][i])), kv8::abs_bits(unpack_hi<T>(qf[j][i]))));
      am = max(am, __shfl_xor_sync(0xffffffffu, am, 1));
      am = max(am, __shfl_xor_sync(0xffffffffu, am, 2));
      const int ex = max((int)(am >> 23) - 127, -100);  // row maximum in [2^ex, 2^(ex+1))
      const float mul = pow2i(14 - ex);
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          qf[j][i] = pack2_rn<__half>(unpack_lo<T>(qf[j][i]) * mul, unpack_hi<T>(qf[j][i]) * mul);
      // logit factor of row gq; a row that is not finite gives NaN logits
      const float cr = am < 0x7f800000u ? a.scale * kLog2e * pow2i(max(ex - 14, -126)) : NAN;
      c2[n][0] = __shfl_sync(0xffffffffu, cr, (2 * tq) * 4);
      c2[n][1] = __shfl_sync(0xffffffffu, cr, (2 * tq + 1) * 4);
      if (NT > 1) {
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          q_frag[((j * NT + n) * 2) * 32] = make_uint4(qf[j][0], qf[j][1], qf[j][2], qf[j][3]);
          q_frag[((j * NT + n) * 2 + 1) * 32] = make_uint4(qf[j][4], qf[j][5], qf[j][6], qf[j][7]);
        }
      }
    }
    int lim[NT][2];  // tokens visible to rows 8 n + 2 tq and + 1
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int i = (row0 + 8 * n + 2 * tq + k) / G;
        lim[n][k] = i < E ? L - E + i + 1 : L;
      }
    const int lim_min = L - E + row0 / G + 1;  // tokens visible to every row of the warp

    float acc[NT][NM][4];
    float M[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int m = 0; m < NM; ++m) acc[n][m][0] = acc[n][m][1] = acc[n][m][2] = acc[n][m][3] = 0.f;
      M[n][0] = M[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
    }
    const bool second = nrows > 8;  // the second row tile has rows

    // this team's tiles of the piece: those with cq % wh == wsel
#pragma unroll 1
    for (;;) {
      while (pq < ntiles && pq * sh.hg + hsel <= x_lim && ok) issue();
      if (cq >= p1) break;
      // A warp that did not fetch this tile has not seen the stage's earlier round end: the parity below
      // could be that of the round before it.
      if (sh.team > 1 && c_round > 0)
        ok = __all_sync(0xffffffffu, ok && wait_uses(&used[st], (uint32_t)(c_round * sh.team)));
      ok = __all_sync(0xffffffffu, ok && mbar_wait(&full[st], c_round & 1));
      if (!ok) break;
      const uint32_t sp = ring + (uint32_t)(st * C::kStage);
      const unsigned char* stage = smem + st * C::kStage;
      const int tok0 = (cq - cons.unit_g) * kTok;
      if (nrows > 0) {
        // ---- S^T = K8.Q^T: tokens 16 mt + gq (+8), rows 8 n + 2 tq, + 1; four chains
        constexpr int CH = NT == 1 ? 2 : 1;  // chains of a token and row tile
        float s[2][NT][CH][4];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int k = 0; k < CH; ++k) s[mt][n][k][0] = s[mt][n][k][1] = s[mt][n][k][2] = s[mt][n][k][3] = 0.f;
        const unsigned char* kp = stage + gq * C::kKS + 16 * tq;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          uint4 kf[4], qa[NT], qb[NT];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            kf[i] = *reinterpret_cast<const uint4*>(kp + 8 * i * C::kKS + 64 * j);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            if (NT == 1) {
              qa[n] = make_uint4(qf[j][0], qf[j][1], qf[j][2], qf[j][3]);
              qb[n] = make_uint4(qf[j][4], qf[j][5], qf[j][6], qf[j][7]);
            } else {
              qa[n] = q_frag[((j * NT + n) * 2) * 32];
              qb[n] = q_frag[((j * NT + n) * 2 + 1) * 32];
            }
          }
#pragma unroll
          for (int mt = 0; mt < 2; ++mt) {
            const uint4 k0 = kf[2 * mt], k1 = kf[2 * mt + 1];
            auto four = [&](uint32_t w0, uint32_t w1, int chain, auto q0, auto q1) {
              const uint32_t a0 = cvt_lo(w0), a1 = cvt_lo(w1), a2 = cvt_hi(w0), a3 = cvt_hi(w1);
#pragma unroll
              for (int n = 0; n < NT; ++n)
                if (n == 0 || second) mma16(s[mt][n][chain % CH], a0, a1, a2, a3, q0(n), q1(n));
            };
            four(k0.x, k1.x, 0, [&](int n) { return qa[n].x; }, [&](int n) { return qa[n].y; });
            four(k0.y, k1.y, 1, [&](int n) { return qa[n].z; }, [&](int n) { return qa[n].w; });
            four(k0.z, k1.z, 0, [&](int n) { return qb[n].x; }, [&](int n) { return qb[n].y; });
            four(k0.w, k1.w, 1, [&](int n) { return qb[n].z; }, [&](int n) { return qb[n].w; });
          }
        }
        // ---- scales of tokens gq + 8 i.  One that is not finite: NaN logits for the rows that see
        // the token, weight 0 for the others
        float ksc[4], ev[4], vn[4];  // K scale, exponent of the V scale, V scale 2^7 / kBias
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 p = *reinterpret_cast<const float2*>(stage + C::kOffScale + (gq + 8 * i) * 8);
          const bool fin = kv8::abs_bits(p.x) < 0x7f800000u && kv8::abs_bits(p.y) < 0x7f800000u;
          ksc[i] = fin ? p.x : NAN;
          const float vs = fin ? p.y : 0.f;
          // (the store's smallest scale is 1e-12 / 448, its exponent -49)
          ev[i] = (float)max((int)(kv8::abs_bits(vs) >> 23) - 127, -50);
          vn[i] = vs * (128.f / kBias);
        }
        // float16 outputs carry as many bits as the weights: l then sums the weights as rounded, so that a
        // rounding moves weight between tokens and leaves their sum one (a row of one token is exact).  Weights
        // below f16's normal range count as they are.
        constexpr bool kSumRounded = std::is_same<T, __half>::value;
        float rv[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) rv[i] = kSumRounded ? __fdividef(1.f, vn[i]) : 0.f;
        uint32_t wb[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if (n > 0 && !second) {
            wb[n][0] = wb[n][1] = wb[n][2] = wb[n][3] = 0u;
            continue;
          }
          float sv[4][2];
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const int e = 2 * (i & 1) + k;
              const float x = CH == 1 ? s[i >> 1][n][0][e] : s[i >> 1][n][0][e] + s[i >> 1][n][CH - 1][e];
              sv[i][k] = x * (ksc[i] * c2[n][k]);
            }
          if (tok0 + kTok > lim_min) {  // some token is hidden from some row
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int k = 0; k < 2; ++k)
                if (tok0 + gq + 8 * i >= lim[n][k]) sv[i][k] = -INFINITY;
          }
          float mx[2];
#pragma unroll
          for (int k = 0; k < 2; ++k)
            mx[k] = fmaxf(fmaxf(sv[0][k] + ev[0], sv[1][k] + ev[1]), fmaxf(sv[2][k] + ev[2], sv[3][k] + ev[3]));
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) {
            mx[0] = fmaxf(mx[0], __shfl_xor_sync(0xffffffffu, mx[0], o));
            mx[1] = fmaxf(mx[1], __shfl_xor_sync(0xffffffffu, mx[1], o));
          }
          float al[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            // a tile hidden from the row as a whole keeps M (and -inf - -inf out of the exponent)
            const float mn = fmaxf(M[n][k], mx[k]);
            const float ah = fade(M[n][k], mn);
            al[k] = ah * ah;
            M[n][k] = mn;
            const float sub = mn == -INFINITY && tok0 >= lim[n][k] ? 0.f : mn;
            float ls = l[n][k] * ah * ah;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              sv[i][k] = ex2((sv[i][k] - sub) + kBiasLog2);  // (in this order: M may be above 2^24)
              const float w = sv[i][k] * vn[i];
              if (kSumRounded) {
                const float wr = __half2float(__float2half_rn(w));
                ls += fabsf(wr) >= 1.f / 16384.f ? wr * rv[i] : sv[i][k];
              } else {
                ls += sv[i][k];
              }
              sv[i][k] = w;
            }
            l[n][k] = ls;
          }
          if (__any_sync(0xffffffffu, al[0] != 1.f || al[1] != 1.f)) {
#pragma unroll
            for (int m = 0; m < NM; ++m) {
              acc[n][m][0] *= al[0];
              acc[n][m][1] *= al[1];
              acc[n][m][2] *= al[0];
              acc[n][m][3] *= al[1];
            }
          }
          // W^T as B fragments: (token gq + 8 i; rows 2 tq, 2 tq + 1) transposed to (row gq; tokens
          // 8 i + 2 tq, + 1)
#pragma unroll
          for (int i = 0; i < 4; ++i) wb[n][i] = movmatrix_t(pack2_rn<__half>(sv[i][0], sv[i][1]));
        }
        // ---- O^T += V8^T.W^T
        const uint32_t vp = sp + C::kOffV + lane * C::kVS;
#pragma unroll
        for (int m0 = 0; m0 < NM; m0 += 4) {
          uint32_t r[4][4];
#pragma unroll
          for (int i = 0; i < 4; ++i) ldsm4_t(vp + 16 * (m0 + i), r[i]);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            // codes (2 g, 2 g + 1) of tokens 2 t, 2 t + 1 -> dim 2 g of both, dim 2 g + 1 of both
#pragma unroll
            for (int k = 0; k < 4; k += 2) {
              const uint32_t x = __byte_perm(r[i][k], 0, 0x3120), y = __byte_perm(r[i][k + 1], 0, 0x3120);
              const uint32_t a0 = cvt_lo(x), a1 = cvt_hi(x), a2 = cvt_lo(y), a3 = cvt_hi(y);
#pragma unroll
              for (int n = 0; n < NT; ++n)
                if (n == 0 || second) mma16(acc[n][m0 + i], a0, a1, a2, a3, wb[n][k], wb[n][k + 1]);
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) count_use(&used[st]);
      x_lim = max(x_lim, cq * sh.hg + hsel + sh.stages - lag);
      cq += sh.wh;
      st += step;
      if (st >= sh.stages) {
        st -= sh.stages;
        ++c_round;
      }
    }

    // ---- the piece is done: O / l, or partials when the unit goes on in another CTA
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        l[n][0] += __shfl_xor_sync(0xffffffffu, l[n][0], o);
        l[n][1] += __shfl_xor_sync(0xffffffffu, l[n][1], o);
      }
    {
      float* fac = epi + kWarps * C::kEpiWarp / 4;
      float* ml = fac + kWarps * kRows;
      if (gq == 0) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int k = 0; k < 2; ++k)
            *reinterpret_cast<float2*>(ml + (warp * kRows + 8 * n + 2 * tq + k) * 2) =
                make_float2(M[n][k], l[n][k]);
      }
      float* mine = epi + warp * (C::kEpiWarp / 4);
      const int slot = 2 * c + (p0 == 0 ? 0 : 1);  // partial place
      const bool whole = p0 == cons.unit_g && p1 == cons.unit_g + cons.nt();
      if (wsel == 0 && lane < kRows) {
        const int row = row0 + lane;
        const int64_t tok = qtok0 + row / G;
        reinterpret_cast<int2*>(ml + 2 * kWarps * kRows)[warp * kRows + lane] =
            make_int2(row < E * G && tok < a.num_tokens ? (int)tok : -1, kvh * G + row % G);
      }
      __syncwarp();  // every lane is done with the Q fragments
#pragma unroll
      for (int m0 = 0; m0 < NM; m0 += 4) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int k = 0; k < 2; ++k)
              *reinterpret_cast<float2*>(mine + (8 * n + 2 * tq + k) * C::kEpiStride + 16 * m + 2 * gq) =
                  make_float2(acc[n][m0 + m][k], acc[n][m0 + m][2 + k]);
        __syncthreads();
        if (m0 == 0) {  // factors of the teams of a head, and its (M, l) in the first team's place
          const int per = sh.hg * sh.team;
          if (tid < per * kRows) {
            float mx = -INFINITY, ls = 0.f;
            for (int w = tid; w < kWarps * kRows; w += per * kRows) mx = fmaxf(mx, ml[2 * w]);
            for (int w = tid; w < kWarps * kRows; w += per * kRows) {
              const float h = fade(ml[2 * w], mx);
              fac[w] = h * h;
              ls = fmaf(h, h * ml[2 * w + 1], ls);
            }
            ml[2 * tid] = mx;
            ml[2 * tid + 1] = ls;
          }
          __syncthreads();
        }
        finish64<T, D, NT>(a, sh, ws, epi, slot, whole, 16 * m0);
        __syncthreads();
      }
    }
  }
  if (!ok && lane == 0) record_err(a.err, TF_KERR_TIMEOUT);  // a wait gave up
  cp_async_wait_all();
}

// ---------------------------------------------------------------------------------------------
// combine: merges the rows of one warp place of a cut unit.  A thread holds 4 values of one row; the PG
// groups of threads take the unit's pieces in turn.
//   wide (many units, few pieces each): CTA (c, place, z) looks at the boundary of range c, and merges RZ
//     rows of the unit that it cuts when it is the first boundary inside that unit
//   deep (few units, many pieces each): CTA (unit, place, row), 16 groups
// ---------------------------------------------------------------------------------------------
template <typename T, int D, int NT, int RZ, int THREADS, bool DEEP>
__global__ void __launch_bounds__(THREADS)
    combine_kernel(const __grid_constant__ tf_paged_attn_args a, const __grid_constant__ Shape sh,
                   const __grid_constant__ Ws ws) {
  constexpr int kRows = 8 * NT;
  constexpr int kVec = D / 4;  // 4-value vectors of a row
  constexpr int PG = THREADS / (RZ * kVec);
  static_assert(PG >= 1 && PG * RZ * kVec == THREADS, "threads of a CTA");
  __shared__ float red[PG > 1 ? THREADS : 1][PG > 1 ? 6 : 1];
  __shared__ int64_t s_g[kMaxCtas + 1];
  __shared__ int s_slot[kMaxCtas];
  __shared__ int s_np;
  const int tid = threadIdx.x, lane = tid & 31;
  const int w = blockIdx.y, n = sh.nctas;
  const int G = a.num_q_heads / a.num_kv_heads;
  int pass, u, start, ext, c0;
  int64_t su, eu;
  if (DEEP) {  // the unit's tiles from the lengths, while the main kernel still runs
    const int b = blockIdx.x / sh.groups;
    u = blockIdx.x - b * sh.groups;
    pass = b % sh.passes;
    int64_t before = 0, q = 0, e = 0;
    int nt = 0;
    for (int i = 0; i <= b; ++i) {
      bool bad;
      before += nt;
      const int64_t L = checked_len(a, i / sh.passes, e, bad);
      nt = tiles_of(L, e, i % sh.passes, sh, G);
      if (i < b && (i + 1) % sh.passes == 0)
        q += a.extend_lens ? max((int)a.extend_lens[i / sh.passes], 0) : 1;
    }
    start = (int)q;
    ext = (int)e;
    su = before * sh.groups + (int64_t)u * nt;
    eu = su + nt;
  }
  // on every path: a grid whose CTAs all left without it would complete beside the main kernel, and what
  // follows in the stream would read rows and reuse scratch that the main kernel still writes
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (DEEP && su == eu) return;
  if (!DEEP) {
    const int c = blockIdx.x + 1;
    const CutInfo ci = ws.cut[c];
    const int64_t g = ws.cta_g[c], gn = ws.cta_g[c + 1];
    if (gn == g || ci.t0 == 0) return;  // an empty range, or nothing cut here
    su = g - ci.t0;
    eu = su + ci.nt;
    c0 = c - 1;
    while (ws.cta_g[c0] == g) --c0;      // empty ranges before this one
    if (ws.cta_g[c0] > su) return;       // not the first boundary inside the unit
    pass = ci.pass;
    u = ci.u;
    start = ci.start;
    ext = ci.ext;
  }
  const int hsel = w / sh.team, member = w % sh.team;
  const int row0 = (pass * sh.team + member) * kRows;
  if (row0 >= ext * G) return;
  for (int i = tid; i <= n; i += THREADS) s_g[i] = ws.cta_g[i];
  __syncthreads();
  if (DEEP) {  // the range that holds the unit's first tile
    int lo = 0, hi = n - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (s_g[mid] <= su) lo = mid; else hi = mid - 1;
    }
    c0 = lo;
    if (s_g[c0 + 1] >= eu) return;  // finished by that CTA
  }
  // partial rows of the unit's pieces, one per range that is not empty: its first piece when the
  // range starts inside the unit (or with it), else its last
  if (tid < 32) {
    int np = 0;
    for (int c1 = c0; c1 < n && s_g[c1] < eu; c1 += 32) {
      const int cc = c1 + lane;
      const bool has = cc < n && s_g[cc] < eu && s_g[cc + 1] > s_g[cc];
      const unsigned m = __ballot_sync(0xffffffffu, has);
      if (has) s_slot[np + __popc(m & ((1u << lane) - 1))] =
          ((2 * cc + (s_g[cc] >= su ? 0 : 1)) * kWarps + w) * kRows;
      np += __popc(m);
    }
    if (lane == 0) s_np = np;
  }
  __syncthreads();
  const int np = s_np;
  const int r = blockIdx.z * RZ + (tid / kVec) % RZ, v = tid % kVec, grp = tid / (kVec * RZ);
  // running merge of this group's pieces; a batch of pieces is requested before it is added
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  float M = -INFINITY, l = 0.f;
  constexpr int kBatch = DEEP ? 8 : 4;
  for (int i0 = grp; i0 < np; i0 += kBatch * PG) {
    float2 ml[kBatch];
    float4 x[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int i = i0 + j * PG;
      if (i < np) {
        const int64_t s = s_slot[i] + r;
        ml[j] = *reinterpret_cast<const float2*>(ws.ml + s * 2);
        x[j] = *reinterpret_cast<const float4*>(ws.o + s * D + 4 * v);
      } else {
        ml[j] = make_float2(-INFINITY, 0.f);
        x[j] = make_float4(0.f, 0.f, 0.f, 0.f);
      }
    }
    float mn = M;
#pragma unroll
    for (int j = 0; j < kBatch; ++j) mn = fmaxf(mn, ml[j].x);
    const float h0 = fade(M, mn), f0 = h0 * h0;
    o.x *= f0;
    o.y *= f0;
    o.z *= f0;
    o.w *= f0;
    l *= h0;
    l *= h0;
    M = mn;
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const float h = fade(ml[j].x, mn), f = h * h;
      o.x = fmaf(f, x[j].x, o.x);
      o.y = fmaf(f, x[j].y, o.y);
      o.z = fmaf(f, x[j].z, o.z);
      o.w = fmaf(f, x[j].w, o.w);
      l = fmaf(h, h * ml[j].y, l);
    }
  }
  if constexpr (PG > 1) {  // the groups meet
    red[tid][0] = o.x;
    red[tid][1] = o.y;
    red[tid][2] = o.z;
    red[tid][3] = o.w;
    red[tid][4] = l;
    red[tid][5] = M;
    __syncthreads();
    if (grp > 0) return;
    constexpr int kG = RZ * kVec;
    float mn = M;
#pragma unroll
    for (int p = 1; p < PG; ++p) mn = fmaxf(mn, red[p * kG + tid][5]);
    float t[5] = {0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int p = 0; p < PG; ++p) {
      const float h = fade(red[p * kG + tid][5], mn), f = h * h;
#pragma unroll
      for (int i = 0; i < 4; ++i) t[i] = fmaf(f, red[p * kG + tid][i], t[i]);
      t[4] = fmaf(h, h * red[p * kG + tid][4], t[4]);
    }
    o = make_float4(t[0], t[1], t[2], t[3]);
    l = t[4];
  }
  const int rr = row0 + r;
  const int64_t tok = start + rr / G;
  if (rr < ext * G && tok < a.num_tokens) {
    const int hq = (u * sh.hg + hsel) * G + rr % G;
    const float inv = (kBias / 128.f) / l;
    const bool v8 = rows_v8(a);
    uint2 gw = make_uint2(0, 0);
    if (a.gate_mode != TF_GATE_NONE) gw = gate4<T>(a, tok, hq, 4 * v, v8);
    put4<T>(a, tok, hq, 4 * v, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv), gw, v8);
  }
}

inline int gcd(int a, int b) { return b == 0 ? a : gcd(b, a % b); }

// rows of one kv head of the longest request
inline int64_t max_rows(const tf_paged_attn_args& a) {
  return (int64_t)(a.num_q_heads / a.num_kv_heads) * (a.extend_lens ? a.max_extend_len : 1);
}
// 8-row tiles of a warp, warps of a team, passes of a request
inline int row_tiles_of(int64_t rows) { return rows > 16 ? 2 : 1; }
inline int team_of(int64_t rows) { return rows > 8 ? 2 : 1; }
inline int passes_of(int64_t rows) {
  const int held = 8 * row_tiles_of(rows) * team_of(rows);
  return rows > held ? (int)((rows + held - 1) / held) : 1;
}

// how a call is divided
template <int D, int NT>
static Shape shape_of(const tf_paged_attn_args& a, int num_sms) {
  using C = Cfg<D, NT>;
  const int64_t rows = max_rows(a);
  Shape s;
  s.row_tiles = NT;
  s.team = team_of(rows);
  s.passes = passes_of(rows);
  // Heads side by side read whole tokens (128 decode requests of 512 to 8192 tokens: 233 us, 250 us with
  // two heads, 285 us with one).  One head a CTA leaves a quarter of the partial rows and its teams
  // meet in shared memory, which counts when a CTA has few tiles: 4 requests of 300 to 6000 tokens and
  // 2..5 drafts 41 us against 78 us with four heads, 8 decode requests of 1000 to 6000 43 us against
  // 47 us; the two meet at about 48 tiles of a head per CTA.
  s.hg = gcd(a.num_kv_heads, kWarps / s.team);
  const int64_t tiles = (int64_t)a.batch_size * s.passes * a.num_kv_heads * ((a.max_seq_len + kTok - 1) / kTok);
  if (tiles < (int64_t)48 * num_sms) s.hg = 1;
  s.wh = kWarps / (s.team * s.hg);
  s.groups = a.num_kv_heads / s.hg;
  s.stages = C::kStages;
  auto bytes = [&](int n) { return n * C::kStage + C::kFixed + 16 * n + C::kEpi; };
  while (bytes(s.stages) > 232448) --s.stages;
  s.ring = s.stages * C::kStage;
  s.smem = bytes(s.stages);
  s.nctas = num_sms;
  s.min_tiles = s.wh;  // one for each team (1000 tokens: 24.6 us, 28.7 us with two)
  s.piece_cost = 8;  // a unit's epilogue and first loads, in tiles
  return s;
}

template <typename T, int D, int NT>
static cudaError_t launch_tdn(const tf_paged_attn_args& a, const tf_kv_scale& sc, void* wsp,
                              int num_sms, cudaStream_t s) {
  constexpr int kRows = 8 * NT;
  if (num_sms > kMaxCtas) num_sms = kMaxCtas;
  const Shape sh = shape_of<D, NT>(a, num_sms);
  if (((int64_t)a.batch_size * sh.passes + 1) * 4 > sh.ring) return cudaErrorInvalidValue;
  const Ws ws = carve(wsp, num_sms, kRows);
  cudaError_t e = cudaFuncSetAttribute(rows_kernel<T, D, NT>,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize, sh.smem);
  if (e != cudaSuccess) return e;
  rows_kernel<T, D, NT><<<num_sms, kThreads, sh.smem, s>>>(a, sc, sh, ws);
  e = cudaGetLastError();
  if (e != cudaSuccess || num_sms == 1) return e;
  constexpr int kWide = 256 / (D / 4) < kRows ? 256 / (D / 4) : kRows;
  const int64_t units = (int64_t)a.batch_size * sh.passes * sh.groups;
  const bool deep = units * 8 < num_sms;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = deep ? dim3((unsigned)units, (unsigned)(sh.hg * sh.team), (unsigned)kRows)
                     : dim3((unsigned)(num_sms - 1), (unsigned)(sh.hg * sh.team), (unsigned)(kRows / kWide));
  cfg.blockDim = dim3(deep ? 4 * D : kWide * (D / 4));
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return deep ? cudaLaunchKernelEx(&cfg, combine_kernel<T, D, NT, 1, 4 * D, true>, a, sh, ws)
              : cudaLaunchKernelEx(&cfg, combine_kernel<T, D, NT, kWide, kWide * (D / 4), false>, a, sh, ws);
}

template <typename T, int D>
static cudaError_t launch_td(const tf_paged_attn_args& a, const tf_kv_scale& sc, void* ws,
                             int num_sms, cudaStream_t s) {
  return row_tiles_of(max_rows(a)) == 2 ? launch_tdn<T, D, 2>(a, sc, ws, num_sms, s)
                                        : launch_tdn<T, D, 1>(a, sc, ws, num_sms, s);
}

template <typename T>
static cudaError_t launch_t(const tf_paged_attn_args& a, const tf_kv_scale& sc, void* ws,
                            int num_sms, cudaStream_t s) {
  switch (a.head_dim) {
    case 64: return launch_td<T, 64>(a, sc, ws, num_sms, s);
    case 128: return launch_td<T, 128>(a, sc, ws, num_sms, s);
    default: return launch_td<T, 256>(a, sc, ws, num_sms, s);
  }
}

}  // namespace rows8

bool paged_fp8_rows_supported(const tf_paged_attn_args& a) {
  if (a.dtype != TF_DTYPE_BF16 && a.dtype != TF_DTYPE_F16) return false;
  if (a.head_dim != 64 && a.head_dim != 128 && a.head_dim != 256) return false;
  if ((int64_t)a.batch_size * rows8::passes_of(rows8::max_rows(a)) > rows8::kMaxBatch || a.r2t_rows > 0x7fffffff || a.r2t_cols > 0x7fffffff)
    return false;
  // the scan of the tiles is kept in 32 bits
  if (a.batch_size * (int64_t)rows8::passes_of(rows8::max_rows(a)) * (a.r2t_cols / rows8::kTok + 1) > 0x7fffffff)
    return false;
  auto al = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  // row offsets are kept in 32 bits of 16-byte pieces: pools of up to 64 GiB a layer
  if (a.num_slots * a.kv_stride_slot + a.num_kv_heads * a.kv_stride_head >= (int64_t)1 << 36) return false;
  return al(a.k_buffer) && al(a.v_buffer) && a.kv_stride_slot % 16 == 0 && a.kv_stride_head % 16 == 0;
}

size_t paged_fp8_rows_workspace(const tf_paged_attn_args& a, int num_sms) {
  return rows8::ws_bytes(num_sms < rows8::kMaxCtas ? num_sms : rows8::kMaxCtas,
                         8 * rows8::row_tiles_of(rows8::max_rows(a)), a.head_dim);
}

cudaError_t launch_paged_fp8_rows(const tf_paged_attn_args& a, const tf_kv_scale& sc, void* ws,
                                  int num_sms, cudaStream_t s) {
  if (a.batch_size == 0) return cudaSuccess;
  return a.dtype == TF_DTYPE_BF16 ? rows8::launch_t<__nv_bfloat16>(a, sc, ws, num_sms, s)
                                  : rows8::launch_t<__half>(a, sc, ws, num_sms, s);
}

}  // namespace tf
