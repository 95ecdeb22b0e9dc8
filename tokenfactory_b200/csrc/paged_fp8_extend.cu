// Paged GQA extend over the 8-bit K/V pool on the 5th-generation tensor cores, for bf16 / fp16
// activations at head_dim 64, 128 and 256.  A dense contraction: 4 D flops per visible (query row, key).
//
// Two CTAs of a cluster on an SM pair run one M=256 tile (128/G query tokens x G heads a CTA) with
// tcgen05.mma.cta_group::2, as paged_extend_tc.cu does over 16-bit pools: CTA r holds query rows
// [128 r, 128 r + 128) and of every 128-key tile keys [64 r, 64 r + 64) of K and dims [r D/2, (r+1) D/2)
// of V (at D 64 both hold all 64 dims and the second copy's columns of O are ignored: a half of 32 dims
// would need another tile layout, and the exponentials bound that size anyway); softmax warps own their CTA's rows, producer warps gather its halves, one thread of rank 0
// issues the products.  What the 8-bit pool changes:
//   producers   load 16 codes a lane, convert them to f16 (exact) and store them into the swizzled
//               tile.  Four warps make the K slots and four the V slots, each with the next slot of its
//               kind on its way into registers while it waits for the slot to be free
//   scales      enter as powers of two of groups of 32 keys (2^kx_g, 2^ev_g, the exponents of the
//               group's largest ks and vs) in the softmax, where they cost nothing: a logit is
//               S c2 2^kx_g, its weight for P 2^(logit + ev_g - M), and l sums the weights times 2^-ev_g.
//               M follows logit + ev_g, so that P stays in f16's range.
//               The rest of each scale, in [2^-6, 2):
//               bfloat16: the producers multiply it into the codes (to f16: 11 bits, random, eight
//               times finer than the output's rounding; two f16 operations a pair, with the scale's
//               own low bits in the first, so that it is not rounded for a whole row at once);
//               float16: the codes stay exact and the softmax multiplies logit and weight by it in
//               fp32, which leaves the weight's f16 rounding alone before the output's.  It costs
//               two reads and two products more per score: 2.5 us a key tile against 2.3 us.
//               A group whose scales are further than 2^6 apart (rows of zeros among others, outliers) is
//               "wide": one key must not take the bits of the others, least of all a key that a row does
//               not see.  Its keys have exponents of their own, which the softmax reads from shared
//               memory; the codes carry what is left of a scale, in [1, 2).
//               bfloat16's l and its exponentials are kept times 2^40: M is between s_max - 50 and s_max + 119 (the
//               store's smallest and largest scale), and both ends then lie inside fp32's range.
//   Q           is scaled by a power of two per row into f16's range (bfloat16 stays exact)
// A scale that is not finite gives its key NaN logits and a V row of zeros, so that only the rows that
// see it are NaN.  Every wait is bounded; one that gives up raises an abort flag in both CTAs and
// TF_KERR_TIMEOUT.
//
// Measured (bf16, 32 heads over 4, head_dim 256; ranges are boxes).  A chunk of 512 tokens behind 28000:
// 528 to 560 us, 847 to 897 TFLOP/s; about 2.1 us a key tile, held by the latency of the softmax warps'
// reads of TMEM (each is waited for where it is issued, and S is read twice; 45% of the issue slots used)
// with the products' 1.1 us beside them.  4 requests of 512 to 2048 tokens on up to 4096: 578 to 616 us, 730
// to 778 TFLOP/s; a query tile's first product starts 10 us after its CTAs do (lengths, table, rows:
// dependent reads) and its epilogue takes 5 us, with nothing beside them as O and the two S buffers fill
// TMEM.  Where every tile is wide (scales 2^+-9 apart) the two take 1130 and 1155 us.  The same chunk over a
// 16-bit pool (paged_extend_tc.cu) takes 381 us, the prompts 468.
//
// Few query tiles over a long prefix leave SM pairs idle: the key tiles are then split over
// grid.y clusters, which leave (M, l, O) partials for a combine kernel.
#include <type_traits>

#include "common.cuh"
#include "kv_fp8.cuh"
#include "launch.h"
#include "tcgen05.cuh"

namespace tf {
namespace ext8 {

constexpr int kRows = 128;       // query rows of a CTA
constexpr int kKeys = 128;       // keys of a tile
constexpr int kSmWarps = 8;      // softmax: warps 0-3 take the even tiles, 4-7 the odd ones
constexpr int kPrWarps = 8;      // producers: four of K (16 rows of a tile each), four of V (32 rows)
constexpr int kPrWarp0 = kSmWarps;
constexpr int kIssueWarp = kSmWarps + kPrWarps;  // MMA issue (rank 0) / slot relay (rank 1)
constexpr int kFwdWarp = kIssueWarp + 1;         // rank 1: forwards "P written" to rank 0
constexpr int kThreads = (kFwdWarp + 1) * 32;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRescaleLog2 = 8.f;
// what bfloat16's l and its exponentials are kept times (fp16's scales reach neither end)
template <typename T> constexpr float kBiasLog2 = std::is_same<T, __half>::value ? 0.f : 40.f;
template <typename T> constexpr float kBias = std::is_same<T, __half>::value ? 1.f : 0x1p40f;
constexpr int kSpread = 6;           // exponents that a group's scales may be apart
constexpr int kTopExp = 30;          // V scales from 2^31 on: beside them P may be 0 where l's terms are not

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float max_of_32(const float (&s)[32]) {
  float t[11];
#pragma unroll
  for (int i = 0; i < 10; ++i) t[i] = max3(s[3 * i], s[3 * i + 1], s[3 * i + 2]);
  t[10] = fmaxf(s[30], s[31]);
  const float u0 = max3(t[0], t[1], t[2]), u1 = max3(t[3], t[4], t[5]), u2 = max3(t[6], t[7], t[8]);
  return max3(max3(u0, u1, u2), t[9], t[10]);
}
__device__ __forceinline__ float ex2_ftz(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }  // -126..127

// 2^((from - to) / 2), from <= to; a sum of weights goes from one maximum to another by its square, taken
// in two steps: maxima can be more than fp32's 2^126 apart where the sums of weights are not
__device__ __forceinline__ float fade(float from, float to) {
  return from == to ? 1.f : ex2_ftz(0.5f * (from - to));
}
__device__ __forceinline__ float lg2_ftz(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// What a group's products are multiplied by to be logits: the row's factor times the group's 2^kx, kept in
// fp32's normal range (floor 2^-126).  Both are small for a row of zeros over keys of zeros, and a product of
// 0 would turn the -inf of a hidden key into a NaN; products are at most 2^33, so that with 2^-126 their
// logits are 0 to 2^-93.  A factor that is NaN (a query row that is not finite) stays NaN.  kx 0 with floor
// 1: a group that wide_logits has already multiplied.
__device__ __forceinline__ float logit_factor(float c2, float kx, float floor) {
  float f;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(f) : "f"(c2 * kx), "f"(floor));
  return f;
}

// two fp32 operations in one instruction (each rounded as its scalar form)
__device__ __forceinline__ uint64_t pk2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void up2(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
// the products of a group of 32 keys: times the keys' scales when those are not in the codes (ks), and
// hidden from key `vis` on
template <bool FOLD>
__device__ __forceinline__ void scale_mask(float (&s)[32], const float* ks, int vis) {
  if (!FOLD) {
    const ulonglong2* kp = reinterpret_cast<const ulonglong2*>(ks);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const ulonglong2 v = kp[k];
      up2(mul2(pk2(s[4 * k], s[4 * k + 1]), v.x), s[4 * k], s[4 * k + 1]);
      up2(mul2(pk2(s[4 * k + 2], s[4 * k + 3]), v.y), s[4 * k + 2], s[4 * k + 3]);
    }
  }
  if (vis < 32) {
#pragma unroll
    for (int k = 0; k < 32; ++k)
      if (k >= vis) s[k] = -INFINITY;
  }
}
// two exponentials p from their weights w = f16(p v): w / v, or p where w is below f16's normal range (a
// small scale)
__device__ __forceinline__ uint64_t as_rounded(uint32_t w, uint64_t v, uint64_t p) {
  constexpr float kNormal = 1.f / 16384.f;
  const float w0 = unpack_lo<__half>(w), w1 = unpack_hi<__half>(w);
  float v0, v1, p0, p1;
  up2(v, v0, v1);
  up2(p, p0, p1);
  if (fabsf(w0) >= kNormal) p0 = w0 * __fdividef(1.f, v0);
  if (fabsf(w1) >= kNormal) p1 = w1 * __fdividef(1.f, v1);
  return pk2(p0, p1);
}
__device__ __forceinline__ void bar_arrive(int id, int nthreads) {
  asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(nthreads) : "memory");
}

__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}

// ---- cluster pair helpers
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t peer_addr(uint32_t local, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(local), "r"(rank));
  return r;
}
// CTA-scope release: what the waiter reads next is complete behind the tcgen05 / proxy fences that
// precede every call
__device__ __forceinline__ void remote_arrive(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cta.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ void remote_store(uint32_t cluster_addr, int v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_addr), "r"(v) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ bool try_wait_cluster(uint32_t addr, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
      " selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(addr), "r"(parity)
      : "memory");
  return ok != 0;
}
// Bounded waits; a timeout raises the abort flag of both CTAs.  CLUSTER: acquire at cluster scope.
template <bool CLUSTER>
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, volatile int* abort,
                                         uint32_t peer_abort, unsigned backoff_ns = 0) {
  const uint32_t addr = smem_u32(bar);
  auto done = [&] { return CLUSTER ? try_wait_cluster(addr, parity) : mbar_try_wait(addr, parity); };
  if (done()) return true;
  const uint64_t t0 = global_ns();
  for (uint32_t it = 1;; ++it) {
    if (backoff_ns) __nanosleep(backoff_ns);
    if (done()) return true;
    if ((it & 63u) == 0) {
      if (*abort) return false;
      if (global_ns() - t0 > kSpinLimitNs) {
        *abort = 1;
        remote_store(peer_abort, 1);
        return false;
      }
    }
  }
}
// Bounded, but not ended by the abort flag: the pair's products are drained before TMEM is released.
__device__ __forceinline__ bool drain(uint64_t* bar, uint32_t parity) {
  const uint32_t addr = smem_u32(bar);
  const uint64_t t0 = global_ns();
  for (uint32_t it = 0;; ++it) {
    if (try_wait_cluster(addr, parity)) return true;
    if ((it & 63u) == 63u && global_ns() - t0 > kSpinLimitNs) return false;
  }
}
__device__ __forceinline__ void mma2_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc ? 1u : 0u)
      : "memory");
}
__device__ __forceinline__ void mma2_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc ? 1u : 0u)
      : "memory");
}
__device__ __forceinline__ void commit_both(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
      " [%0], %1;" ::"r"(smem_u32(bar)), "h"((uint16_t)3)
      : "memory");
}
// instruction descriptor, kind::f16 with f16 inputs and fp32 accumulation
__host__ __device__ constexpr uint32_t idesc_f16(int M, int N, bool b_mn_major) {
  return (1u << 4) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

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
__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ uint4 ldg_nc(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

template <int D>
struct Cfg {
  static constexpr int kKB = D / 64;              // 64-dim blocks of a row
  static constexpr int kQBlock = kRows * 128;     // one block of this CTA's Q rows
  static constexpr int kQBytes = kKB * kQBlock;
  static constexpr int kKBlk = (kKeys / 2) * 128; // K half: 64 keys x 128 B per block
  static constexpr int kVBlk = kKeys * 128;       // V half: 128 keys x 128 B per block
  static constexpr int kVD = D == 64 ? 64 : D / 2;  // dims of V that a CTA holds
  static constexpr int kSlotBytes = D == 64 ? kVBlk : kKB * kKBlk;  // K halves and V halves alike
  static constexpr int kSlots = D == 256 ? 4 : 8;
  // Ring of the tiles' scales.  Those of tile t are written once V_{t-1} has been stored, for which
  // PV_{t-1-kSlots/2} had completed: the softmax of that tile is done with its scales, a later one's
  // may not be.
  static constexpr int kScaleTiles = D == 256 ? 4 : 8;
  static_assert(kScaleTiles >= kSlots / 2 + 1, "scales in use are not overwritten");
  static constexpr int kOffRing = kQBytes;
  static constexpr int kOffBars = kOffRing + kSlots * kSlotBytes;
  // full, empty [kSlots]; s_full[2], p_full[2][2], o_done, q_full, fin, q_dead, sc_full[kScaleTiles]
  static constexpr int kNumBars = 2 * kSlots + 10 + kScaleTiles;
  static constexpr int kOffWords = kOffBars + 8 * kNumBars;      // tmem holder, abort
  static constexpr int kOffM = (kOffWords + 16 + 15) & ~15;      // float [2][kRows]: running maxima
  static constexpr int kOffRow = kOffM + 2 * kRows * 4;          // float [kRows]: logit factor of a row
  static constexpr int kOffKs = kOffRow + kRows * 4;             // float [kScaleTiles][kKeys]
  static constexpr int kOffVs = kOffKs + kScaleTiles * kKeys * 4;
  static constexpr int kOffGrp = kOffVs + kScaleTiles * kKeys * 4;  // float4 [kScaleTiles][4]: a group's
                                                                  // 2^kx, ev, 2^-ev kBias, floor
  static constexpr int kOffApart = kOffGrp + kScaleTiles * 4 * 16;  // float [kScaleTiles][4]: not 0 where a tile
                                                                    // needs the steps of a wide one
  static constexpr int kSmem = kOffApart + kScaleTiles * 4 * 4 + 1024;
  static constexpr int kColS = 0;                 // two S buffers of kKeys columns; P_j over S_j
  static constexpr int kColO = 2 * kKeys;
  static constexpr int kTmemCols = 512;
  static_assert(kSlotBytes >= kKB * kKBlk && kSlotBytes >= kVD / 64 * kVBlk, "K and V halves share the slot size");
  static_assert(kSmem <= 232448, "shared memory per CTA");
  static_assert(kColO + D <= kTmemCols, "TMEM columns");
  static_assert(4 * kRows * 4 <= kSlotBytes && kRows * D * 2 <= kQBytes, "epilogue staging");
};

struct Split {
  int n;        // clusters that share the keys of a query tile
  float* ml;    // [n][T][Hq][2]
  float* o;     // [n][T][Hq][D]
};

// 16 columns of this lane's TMEM row
__device__ __forceinline__ void ld16(uint32_t taddr, float (&v)[16]) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

// What a tile of wide groups needs beside the common path.  Out of line: it is rare, and the tile loop's
// instructions are fetched once a tile.  A row's products S of the tile's 128 keys sit in the lane's TMEM
// columns sa..
//
// exact codes: the largest logit + log2 of the V scale among keys [0, vis) (ks times 2^kx of the group times
// c2 is what the products are multiplied by)
__device__ __noinline__ float wide_max(uint32_t sa, const float* ks, const float* vs, const float4* grp, float c2,
                                       int vis) {
  float m = -INFINITY;
#pragma unroll 1
  for (int g = 0; g < 8; ++g) {
    const float factor = logit_factor(c2, grp[g >> 1].x, grp[g >> 1].w);
    float s[16];
    ld16(sa + 16 * g, s);
    tc::wait_ld();
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      // (a V row of zeros counts as one of the store's smallest scale)
      const float x = fmaf(s[k], ks[16 * g + k] * factor, fmaxf(lg2_ftz(fabsf(vs[16 * g + k])), -50.f));
      if (16 * g + k < vis) m = fmaxf(m, x);
    }
  }
  return m;
}
// folded codes: the products of wide groups (2^kx of 0) become logit + ev with their keys' own exponents,
// ks = 2^kx and vs = 2^ev
__device__ __noinline__ void wide_logits(uint32_t sa, const float* ks, const float* vs, const float4* grp, float c2) {
#pragma unroll 1
  for (int g = 0; g < 8; ++g) {
    if (grp[g >> 1].x != 0.f) continue;
    float s[16];
    ld16(sa + 16 * g, s);
    tc::wait_ld();
#pragma unroll
    for (int k = 0; k < 16; ++k) s[k] = fmaf(s[k], ks[16 * g + k] * c2, lg2_ftz(vs[16 * g + k]));
    tc::st16(sa + 16 * g, s);
  }
  tc::wait_st();
}
// the sum of 2^(logit - M) 2^bias over keys [0, vis), where a sum of weights over 2^ev would not do; the
// exponents of the weights are formed as the common path does and ev comes off them, so that a rounding of M
// or of logit + ev (logits above 2^24) is the same in both
__device__ __noinline__ float wide_sum(uint32_t sa, const float* vs, const float4* grp, float c2, int vis, float nmu,
                                       float bias) {
  float sum = 0.f;
#pragma unroll 1
  for (int g = 0; g < 8; ++g) {
    const float4 e = grp[g >> 1];
    const float factor = logit_factor(c2, e.x, e.w), ng = nmu + e.y;
    float s[16];
    ld16(sa + 16 * g, s);
    tc::wait_ld();
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const float ev = e.x == 0.f ? lg2_ftz(vs[16 * g + k]) : e.y;
      if (16 * g + k < vis) sum += ex2_ftz(fmaf(s[k], factor, ng) + (bias - ev));
    }
  }
  return sum;
}

// 16-byte pieces of the gate and output rows can be moved whole
__device__ __forceinline__ bool rows_v16(const tf_paged_attn_args& a) {
  return ((reinterpret_cast<uintptr_t>(a.out) | reinterpret_cast<uintptr_t>(a.gate)) & 15) == 0 &&
         ((a.out_stride_tok | a.out_stride_head | a.gate_stride_tok | a.gate_stride_head) & 7) == 0;
}
// the gate's activation; __fdividef is off by at most two units of 2^-23
__device__ __forceinline__ float act(float x, int mode) {
  const float s = __fdividef(1.f, 1.f + __expf(-x));
  return mode == TF_GATE_SILU ? x * s : s;
}

template <typename T, int D>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    extend_kernel(const __grid_constant__ tf_paged_attn_args a, const __grid_constant__ tf_kv_scale sc,
                  int pairs_per_req, const __grid_constant__ Split sp) {
  using C = Cfg<D>;
  extern __shared__ unsigned char smem_raw[];
  const uint32_t raw_base = smem_u32(smem_raw);
  const uint32_t base = (raw_base + 1023) & ~1023u;
  unsigned char* sbase = smem_raw + (base - raw_base);
  uint64_t* full = reinterpret_cast<uint64_t*>(sbase + C::kOffBars);
  uint64_t* empty = full + C::kSlots;
  uint64_t* s_full = empty + C::kSlots;
  uint64_t* p_full = s_full + 2;
  uint64_t* o_done = p_full + 4;  // p_full[2 buffer + half]: 64 keys of P_j are in TMEM
  uint64_t* q_full = o_done + 1;
  uint64_t* fin = q_full + 1;
  uint64_t* q_dead = fin + 1;    // the last S product has completed: Q's shared memory is free
  uint64_t* sc_full = q_dead + 1;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(sbase + C::kOffWords);
  volatile int* abort = reinterpret_cast<volatile int*>(sbase + C::kOffWords + 4);
  float* m_s = reinterpret_cast<float*>(sbase + C::kOffM);
  float* rowf = reinterpret_cast<float*>(sbase + C::kOffRow);
  float* ks_s = reinterpret_cast<float*>(sbase + C::kOffKs);
  float* vs_s = reinterpret_cast<float*>(sbase + C::kOffVs);
  float4* grp_s = reinterpret_cast<float4*>(sbase + C::kOffGrp);
  float* apart_s = reinterpret_cast<float*>(sbase + C::kOffApart);
  constexpr bool kFold = !std::is_same<T, __half>::value;  // scales multiplied into the codes

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cluster_rank();
  const uint32_t peer = rank ^ 1u;
  const uint32_t peer_abort = peer_addr(smem_u32((const void*)abort), peer);
  const int Hkv = a.num_kv_heads, G = a.num_q_heads / Hkv;
  const int TQ = kRows / G;  // query tokens per CTA
  // Longest query tiles first, so that the last ones to finish are short: the longest request before
  // the others (of up to 32, which a warp ranks; of more, each is a small part of the whole), and a
  // head's later tiles before its earlier ones.  When they were introduced, 3 requests of 64 to 1009 new tokens on up to 2904: 122 us,
  // 129 us in the batch's order, head by head; 4 of 512 to 2048 on up to 4096: 664 us against 672 us
  // (695 us with the kv heads of a query tile side by side).
  const int z = blockIdx.y, rank_h = (blockIdx.x >> 1) / pairs_per_req;
  const int qp = pairs_per_req - 1 - ((blockIdx.x >> 1) - rank_h * pairs_per_req);
  const int h = rank_h % Hkv;
  int b = rank_h / Hkv;
  int64_t E, L, before = 0;  // before: query tokens of the requests before this one
  if (a.batch_size <= 32) {
    const bool in = lane < a.batch_size;
    const int64_t Li = in ? a.seq_lens[lane] : INT64_MIN;
    const int64_t Ei = in && a.extend_lens ? a.extend_lens[lane] : 1;
    int place = 0;
    for (int j = 0; j < a.batch_size; ++j) {
      const int64_t Lj = __shfl_sync(0xffffffffu, Li, j);
      place += Lj > Li || (Lj == Li && j < lane);
    }
    b = __ffs(__ballot_sync(0xffffffffu, in && place == b)) - 1;
    E = __shfl_sync(0xffffffffu, Ei, b);
    L = __shfl_sync(0xffffffffu, Li, b);
    if (in && lane < b && Ei > 0) before = Ei;
  } else {
    E = a.extend_lens ? a.extend_lens[b] : 1;
    L = a.seq_lens[b];
    for (int i = lane; i < b; i += 32) {
      const int64_t e = a.extend_lens ? a.extend_lens[i] : 1;
      before += e > 0 ? e : 0;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
  const int64_t pair_start = (int64_t)qp * 2 * TQ;
  if (pair_start >= E) return;  // both CTAs of the pair leave here, before any cluster barrier
  if (L > a.r2t_cols || L < E) {
    if (tid == 0 && rank == 0) record_err(a.err, TF_KERR_SLOT_RANGE);
    return;
  }
  const int64_t P = L - E;
  const int64_t cta_start = pair_start + (int64_t)rank * TQ;  // first token of this CTA's rows
  const int64_t pair_end = E - pair_start < 2 * TQ ? E : pair_start + 2 * TQ;
  const int64_t kv_end = P + pair_end;  // keys [0, kv_end) are visible to some row of the pair
  const int all_tiles = (int)((kv_end + kKeys - 1) / kKeys);
  // this cluster's key tiles [jb, jb + ntiles)
  const int per = (all_tiles + sp.n - 1) / sp.n;
  const int jb = z * per;
  const int ntiles = all_tiles - jb < per ? all_tiles - jb : per;

  const int64_t q0 = before + cta_start;
  int64_t left = E - cta_start < TQ ? E - cta_start : TQ;
  if (left > a.num_tokens - q0) left = a.num_tokens - q0;
  const int n_tok = left > 0 ? (int)left : 0;  // query tokens of this CTA

  if (ntiles <= 0) {  // nothing left for this cluster: an empty partial (both CTAs come here)
    const int ri = tid / G;
    if (tid < kRows && ri < TQ && cta_start + ri < E && q0 + ri < a.num_tokens) {
      const int64_t row = ((int64_t)z * a.num_tokens + q0 + ri) * a.num_q_heads + h * G + tid % G;
      *reinterpret_cast<float2*>(sp.ml + 2 * row) = make_float2(-INFINITY, 0.f);
    }
    return;
  }
  if (tid == 0) {
    for (int i = 0; i < C::kSlots; ++i) {
      mbar_init(&full[i], rank == 0 ? kPrWarps / 2 + 1 : kPrWarps / 2);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      for (int k = 0; k < 2; ++k) mbar_init(&p_full[2 * i + k], rank == 0 ? kSmWarps / 2 + 1 : kSmWarps / 2);
    }
    mbar_init(o_done, 1);
    mbar_init(q_full, rank == 0 ? kSmWarps + 1 : kSmWarps);  // one arrive a warp
    mbar_init(fin, 1);
    mbar_init(q_dead, 1);
    for (int i = 0; i < C::kScaleTiles; ++i) mbar_init(&sc_full[i], kPrWarps / 2);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  // producers: the slot-id chain of the first key tiles is requested before the set-up barrier.  Lane
  // l takes key l of a group of 32: the one that holds K warp w's 16 rows (64 rank + 16 w), group w for
  // V warp w
  constexpr int kPrefetch = 4;
  int64_t raw_q[kPrefetch] = {0, 0, 0, 0};
  const int64_t* r2t = a.req_to_token;
  int my_key = 0;
  const int pw = warp - kPrWarp0;
  auto raw_of = [&](int tile) -> int64_t {  // tile counts from jb
    int64_t key = (int64_t)(jb + tile) * kKeys + my_key;
    if (key >= kv_end) key = (int64_t)(jb + tile) * kKeys;  // past the window: the tile's first key
    return r2t[key];
  };
  if (warp >= kPrWarp0 && warp < kIssueWarp) {
    int64_t row = a.req_pool_indices[b];
    if (row < 0 || row >= a.r2t_rows) {
      if (tid == kPrWarp0 * 32 && rank == 0) record_err(a.err, TF_KERR_REQ_RANGE);
      row = 0;
    }
    r2t = a.req_to_token + row * a.r2t_stride;
    my_key = pw < 4 ? 64 * (int)rank + 32 * (pw >> 1) + lane : 32 * (pw - 4) + lane;
#pragma unroll
    for (int i = 0; i < kPrefetch; ++i)
      if (i < ntiles) raw_q[i] = raw_of(i);
  }
  // Q: the softmax warps request this CTA's 128 rows before the set-up barrier, all at once (16 rows a
  // warp, four at a time behind the barrier, took 13 us); a row sits with D / 8 lanes, 16 bytes each
  constexpr int kQLanes = D / 8, kQRpi = 32 / kQLanes, kQLoads = kRows / kSmWarps / kQRpi;
  const int q_sub = lane / kQLanes, q_ch = lane - q_sub * kQLanes;
  auto q_row = [&](int i) { return warp * (kRows / kSmWarps) + i * kQRpi + q_sub; };
  auto q_dst = [&](int qr) {
    return base + (q_ch >> 3) * C::kQBlock + qr * 128 + (((q_ch & 7) ^ (qr & 7)) << 4);
  };
  if (warp < kSmWarps) {
    const T* q = reinterpret_cast<const T*>(a.q) + q0 * a.q_stride_tok + (int64_t)h * G * a.q_stride_head + q_ch * 8;
    const bool vec = ((reinterpret_cast<uintptr_t>(a.q) & 15) | ((a.q_stride_tok | a.q_stride_head) & 7)) == 0;
#pragma unroll 4
    for (int i = 0; i < kQLoads; ++i) {
      const int qr = q_row(i), ti = qr / G;
      const T* src = q + ti * a.q_stride_tok + (int64_t)(qr - ti * G) * a.q_stride_head;
      if (ti >= n_tok) {
        sts128(q_dst(qr), 0, 0, 0, 0);
      } else if (vec) {
        cp_async16(q_dst(qr), src);
      } else {
        const unsigned short* u = reinterpret_cast<const unsigned short*>(src);
        sts128(q_dst(qr), u[0] | ((uint32_t)u[1] << 16), u[2] | ((uint32_t)u[3] << 16),
               u[4] | ((uint32_t)u[5] << 16), u[6] | ((uint32_t)u[7] << 16));
      }
    }
  }
  if (warp == kIssueWarp) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_holder)), "r"(C::kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc::fence_before_sync();
  cluster_sync();  // barriers of both CTAs initialised, TMEM allocated in both
  tc::fence_after_sync();
  const uint32_t tmem = *tmem_holder;

  if (warp >= kPrWarp0 && warp < kIssueWarp) {
    // ======================= producers: this CTA's halves =======================
    const float* scp = sc.data + (int64_t)h * sc.stride_head;
    bool ok = true;
    // the slots of one kind
    auto produce = [&](auto kind) {
      constexpr bool kV = decltype(kind)::value;
      constexpr int kRowsW = kV ? 32 : 16;             // rows of a tile that a warp makes
      constexpr int CPR = kV ? C::kVD / 16 : D / 16;        // 16-byte pieces of a row of codes
      constexpr int RPI = 32 / CPR, kLoads = kRowsW / RPI;
      constexpr int kBlkBytes = kV ? C::kVBlk : C::kKBlk;
      const int sub = lane / CPR, ch = lane - (lane / CPR) * CPR;
      const char* src = kV ? (const char*)a.v_buffer + (int64_t)h * a.kv_stride_head + (D == 64 ? 0 : rank * (D / 2)) + ch * 16
                           : (const char*)a.k_buffer + (int64_t)h * a.kv_stride_head + ch * 16;
      const int row0 = (kV ? 32 * (pw - 4) : 16 * pw) + sub;
      const int lane0 = kV ? 0 : 16 * (pw & 1);        // the lane that knows the warp's first row
      // 16 codes are two 16-byte chunks of f16; lanes of odd 64-dim blocks store theirs in the other
      // order (a bank conflict otherwise)
      const int blk = ch >> 2;
      const bool odd = blk & 1;
      const int ca = 2 * (ch & 3) + (odd ? 1 : 0), cb = 2 * (ch & 3) + (odd ? 0 : 1);
      auto load = [&](int tile, uint4 (&w)[kLoads], float2& s2) {
        const int64_t raw = raw_q[0];
#pragma unroll
        for (int k = 0; k + 1 < kPrefetch; ++k) raw_q[k] = raw_q[k + 1];
        raw_q[kPrefetch - 1] = tile + kPrefetch < ntiles ? raw_of(tile + kPrefetch) : 0;
        const int64_t sl = resolve_slot(raw, a.num_slots, a.slot_mode, a.err);
        const uint32_t off = (uint32_t)((sl * a.kv_stride_slot) >> 4);  // 16-byte pieces (the host checks)
        uint32_t o[kLoads];
#pragma unroll
        for (int k = 0; k < kLoads; ++k) o[k] = __shfl_sync(0xffffffffu, off, lane0 + k * RPI + sub);
#pragma unroll
        for (int k = 0; k < kLoads; ++k) w[k] = ldg_nc(src + (uint64_t)o[k] * 16);
        s2 = __ldg(reinterpret_cast<const float2*>(scp + sl * sc.stride_slot));
      };
      int slot = kV ? 2 : 0;   // ring place: K0 K1 V0 K2 V1 K3 ... V_{n-2} V_{n-1}
      uint32_t phase = 0;
      bool large = false;      // a group so far had a V scale above kTopExp
      auto put = [&](int tile, uint4 (&w)[kLoads], float2 s2) {
        // A scale that is not finite: NaN logits (K), and a V row of zeros
        const bool fin = kv8::abs_bits(s2.x) < 0x7f800000u && kv8::abs_bits(s2.y) < 0x7f800000u;
        // Exponents of the key: its group's, or its own where the group's are further apart than kSpread (K
        // and V each for itself; fp16 keeps the rest of a scale in fp32 and its group's).
        const int own_k = (int)(kv8::abs_bits(s2.x) >> 23), own_v = (int)(kv8::abs_bits(s2.y) >> 23);
        int gk = 0, gv = 0;
        bool wide_k = false, wide_v = false;
        if (kFold || kV) gk = (int)(__reduce_max_sync(0xffffffffu, fin ? kv8::abs_bits(s2.x) : 0u) >> 23);
        if (kFold) wide_k = __any_sync(0xffffffffu, fin && gk - own_k > kSpread);
        if (kV) {
          gv = (int)(__reduce_max_sync(0xffffffffu, fin ? kv8::abs_bits(s2.y) : 0u) >> 23);
          wide_v = __any_sync(0xffffffffu, fin && gv - own_v > kSpread);
        }
        const int kx = min(max((wide_k && fin ? own_k : gk) - 127, -100), 126);
        const int ev = min(max((kFold && wide_v && fin ? own_v : gv) - 127, -50), 126);
        if (kV) {
          const int st = tile & (C::kScaleTiles - 1);
          ks_s[st * kKeys + my_key] = fin ? (kFold ? pow2i(kx) : s2.x * pow2i(-kx)) : NAN;
          vs_s[st * kKeys + my_key] = kFold ? pow2i(ev) : fin ? s2.y : 0.f;
          const bool wide = wide_k || wide_v;
          if (lane == 0) {
            grp_s[st * 4 + pw - 4] = kFold && wide
                                         ? make_float4(0.f, 0.f, 0.f, 1.f)  // (logit_factor, wide_logits)
                                         : make_float4(pow2i(kx), (float)ev, pow2i(-ev) * kBias<T>, 0x1p-126f);
            large = large || (kFold && gv - 127 > kTopExp);
            apart_s[st * 4 + pw - 4] = wide || large ? 1.f : 0.f;
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&sc_full[st]);
        }
        // what the codes of this lane's key are multiplied by, as two f16 terms; exact: 1, or 0
        float mul = kV ? s2.y * pow2i(-ev) : s2.x * pow2i(-kx);
        if (!kFold) mul = 1.f;
        if (!fin) mul = kV ? 0.f : NAN;
        const __half mh = __float2half_rn(mul);
        const uint32_t mterms = (uint32_t)__half_as_ushort(mh) |
                                ((uint32_t)__half_as_ushort(__float2half_rn(mul - __half2float(mh))) << 16);
        // the slot's place and round: position i = 2 tile - 1 (K), 2 tile + 2 (V), shifted at the ends
        const int i = kV ? (tile == ntiles - 1 ? 2 * ntiles - 1 : 2 * tile + 2) : (tile == 0 ? 0 : 2 * tile - 1);
        slot = i % C::kSlots;
        phase = (uint32_t)(i / C::kSlots) & 1u;
        ok = __all_sync(0xffffffffu, wait_bar<false>(&empty[slot], phase ^ 1u, abort, peer_abort, 32));
        if (!ok) return;
        const uint32_t sb = base + C::kOffRing + slot * C::kSlotBytes + blk * kBlkBytes;
#pragma unroll
        for (int k = 0; k < kLoads; ++k) {
          const int row = row0 + k * RPI;
          uint4 v = w[k];
          if (odd) v = make_uint4(v.z, v.w, v.x, v.y);
          const uint32_t dst = sb + row * 128;
          uint32_t f[8] = {cvt_lo(v.x), cvt_hi(v.x), cvt_lo(v.y), cvt_hi(v.y),
                           cvt_lo(v.z), cvt_hi(v.z), cvt_lo(v.w), cvt_hi(v.w)};
          if (kFold || kV) {
            const uint32_t t = __shfl_sync(0xffffffffu, mterms, lane0 + k * RPI + sub);
            const uint32_t hi = __byte_perm(t, 0, 0x1010), lo = __byte_perm(t, 0, 0x3232);
#pragma unroll
            for (int q = 0; q < 8; ++q) f[q] = kFold ? hfma2(f[q], hi, hmul2(f[q], lo)) : (hi == 0 ? 0u : f[q]);
          }
          sts128(dst + ((ca ^ (row & 7)) << 4), f[0], f[1], f[2], f[3]);
          sts128(dst + ((cb ^ (row & 7)) << 4), f[4], f[5], f[6], f[7]);
        }
        tc::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&full[slot]);
      };
      // the next tile's rows are requested as soon as this one's registers are free; its slot is not
      uint4 w[kLoads];
      float2 s2;
      load(0, w, s2);
#pragma unroll 1
      for (int j = 0; ok && j < ntiles; ++j) {
        put(j, w, s2);
        if (j + 1 < ntiles) load(j + 1, w, s2);
      }
    };
    if (pw < 4) produce(std::false_type());
    else produce(std::true_type());
    // Output gate: once the last S product has completed (q_dead) the Q region is free; each producer
    // warp copies its share of the gate rows of this CTA into it while the last tiles still run (16-byte chunks
    // XOR-swizzled by the row).  Every producer thread reaches the closing barrier.
    const T* gate = reinterpret_cast<const T*>(a.gate);
    const bool staged = a.gate_mode != TF_GATE_NONE && sp.n == 1 && rows_v16(a);
    constexpr int kChunks = D / 8, kRowsPerInstr = 32 / kChunks;
    const int gsub = lane / kChunks, gch = lane - (lane / kChunks) * kChunks;
    bool okg = ok && wait_bar<false>(q_dead, 0, abort, peer_abort);
    okg = __all_sync(0xffffffffu, okg);
    if (okg && staged) {
#pragma unroll 1
      for (int i = 0; i < kRows / kPrWarps; i += kRowsPerInstr) {
        const int row = pw * (kRows / kPrWarps) + i + gsub;
        const int ti = row / G, g = row - (row / G) * G;
        if (ti < n_tok)
          cp_async16(base + row * (D * 2) + ((gch ^ (row & (kChunks - 1))) << 4),
                     gate + (q0 + ti) * a.gate_stride_tok + (int64_t)(h * G + g) * a.gate_stride_head + gch * 8);
      }
    }
    cp_async_wait_all();
    named_barrier(10, (kSmWarps + kPrWarps) * 32);  // gate rows staged for the softmax warps
  } else if (warp == kIssueWarp && rank == 1) {
    // ======================= relay: this CTA's halves landed -> rank 0 =======================
    if (lane == 0) {
      bool ok = wait_bar<false>(q_full, 0, abort, peer_abort);
      if (ok) {
        tc::fence_proxy_async_smem();
        remote_arrive(peer_addr(smem_u32(q_full), 0));
      }
      int slot = 0;
      uint32_t phase = 0;
      for (int it = 0; ok && it < 2 * ntiles; ++it) {
        ok = wait_bar<false>(&full[slot], phase, abort, peer_abort);
        if (!ok) break;
        tc::fence_proxy_async_smem();
        remote_arrive(peer_addr(smem_u32(&full[slot]), 0));
        if (++slot == C::kSlots) { slot = 0; phase ^= 1u; }
      }
      // rank 0's products done with this CTA's TMEM and smem; waited for also after an abort (bounded)
      mbar_wait(fin, 0);
    }
    __syncwarp();
  } else if (warp == kFwdWarp) {
    // =========== rank 1: "this CTA's P_j is in TMEM" -> rank 0's p_full, one arrive per tile ===========
    if (rank == 1 && lane == 0) {
      const uint32_t pf = peer_addr(smem_u32(p_full), 0);
      for (int j = 0; j < 2 * ntiles; ++j) {  // halves of tiles
        const int k = j & 3;                  // 2 buffer + half
        if (!wait_bar<false>(&p_full[k], (j >> 2) & 1, abort, peer_abort)) break;
        tc::fence_after_sync();
        tc::fence_before_sync();
        remote_arrive(pf + 8 * k);
      }
    }
    __syncwarp();
  } else if (warp == kIssueWarp) {
    // ======================= MMA issue for the pair (rank 0, one thread) =======================
    if (lane == 0) {
      constexpr uint32_t kIdS = idesc_f16(2 * kRows, kKeys, false);
      constexpr uint32_t kIdO = idesc_f16(2 * kRows, 2 * C::kVD, true);
      bool ok = wait_bar<true>(q_full, 0, abort, peer_abort);
      tc::fence_proxy_async_smem();
      int slot = 0;
      uint32_t phase = 0;
      auto take = [&]() -> uint32_t {
        ok = ok && wait_bar<true>(&full[slot], phase, abort, peer_abort);
        tc::fence_proxy_async_smem();
        return base + C::kOffRing + slot * C::kSlotBytes;
      };
      auto release = [&]() {
        commit_both(&empty[slot]);
        if (++slot == C::kSlots) { slot = 0; phase ^= 1u; }
      };
      auto issue_s = [&](int t) {
        const uint32_t kb = take();
        if (!ok) return;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint64_t ad = tc::sw128_desc(base + (kk >> 2) * C::kQBlock + (kk & 3) * 32, 16, 1024);
          const uint64_t bd = tc::sw128_desc(kb + (kk >> 2) * C::kKBlk + (kk & 3) * 32, 16, 1024);
          mma2_ss(tmem + C::kColS + (t & 1) * kKeys, ad, bd, kIdS, kk > 0);
        }
        commit_both(&s_full[t & 1]);
        if (t == ntiles - 1) commit_both(q_dead);
        release();
      };
      auto issue_pv = [&](int t) {
        const uint32_t vb = take();
        // the first 64 keys' product starts while the others' weights are being made
#pragma unroll
        for (int kk = 0; kk < kKeys / 16; ++kk) {
          if ((kk & 3) == 0) {
            ok = ok && wait_bar<true>(&p_full[2 * (t & 1) + (kk >> 2)], (t >> 1) & 1, abort, peer_abort);
            if (!ok) return;
            tc::fence_after_sync();
          }
          // P_j: keys [64 hf, 64 hf + 64) packed in columns [64 hf, 64 hf + 32) of S buffer j & 1
          const uint64_t bd = tc::sw128_desc(vb + kk * 2048, C::kVBlk, 1024);
          mma2_ts(tmem + C::kColO, tmem + C::kColS + (t & 1) * kKeys + 64 * (kk >> 2) + (kk & 3) * 8, bd,
                  kIdO, t > 0 || kk > 0);
        }
        commit_both(o_done);
        release();
      };
      if (ok) issue_s(0);
      if (ok && ntiles > 1) issue_s(1);
      for (int j = 0; ok && j < ntiles; ++j) {
        issue_pv(j);
        if (ok && j + 2 < ntiles) issue_s(j + 2);
      }
      if (!ok) commit_both(q_dead);  // aborted before the last S: release the waiters anyway
      commit_both(fin);  // completes once every product issued above has completed
      drain(fin, 0);     // also after an abort (bounded): none may be in flight when TMEM is released
    }
    __syncwarp();
  } else if (warp < kSmWarps) {
    // ============ softmax + epilogue: thread (wg, r) = row r of the tiles j with j % 2 == wg ============
    // The two warpgroups work on neighbouring tiles at once, one's exponentials beside the other's
    // scaling and maxima.  A row's running maximum passes from tile to tile through shared memory
    // (named barriers 1-8, one per warp pair and direction); each warpgroup keeps its own sum.
    const int r = tid & (kRows - 1);
    const int wg = tid >> 7;
    const int ri = r / G;
    const bool row_valid = ri < n_tok;
    const bool idle = (warp & 3) * 32 >= n_tok * G;  // no row of this warp is one of the request's
    const int64_t klim = P + cta_start + ri + 1;  // keys [0, klim) are visible to this row
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    constexpr int kOHalf = D / 2;  // O columns stored by this thread
    const int bar_in = 1 + 2 * (warp & 3) + wg, bar_out = 1 + 2 * (warp & 3) + (wg ^ 1);
    float m_used = -INFINITY, l_sum = 0.f;
    {  // Q, scaled into f16's range in place (a lane's own pieces; a short loop, as the epilogue)
      cp_async_wait_all();
#pragma unroll 4
      for (int i = 0; i < kQLoads; ++i) {
        const int qr = q_row(i);
        uint32_t w[4], am = 0;
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                     : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                     : "r"(q_dst(qr))
                     : "memory");
#pragma unroll
        for (int k = 0; k < 4; ++k)
          am = max(am, max(kv8::abs_bits(unpack_lo<T>(w[k])), kv8::abs_bits(unpack_hi<T>(w[k]))));
#pragma unroll
        for (int o = kQLanes / 2; o > 0; o >>= 1) am = max(am, __shfl_xor_sync(0xffffffffu, am, o));
        const int ex = max((int)(am >> 23) - 127, -100);  // row maximum in [2^ex, 2^(ex+1))
        const float mul = pow2i(14 - ex);
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = pack2_rn<__half>(unpack_lo<T>(w[k]) * mul, unpack_hi<T>(w[k]) * mul);
        sts128(q_dst(qr), w[0], w[1], w[2], w[3]);
        // a row that is not finite gives NaN logits
        if (q_ch == 0) rowf[qr] = am < 0x7f800000u ? a.scale * kLog2e * pow2i(max(ex - 14, -126)) : NAN;
      }
      tc::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
    }
    bool ok = __all_sync(0xffffffffu, wait_bar<false>(q_full, 0, abort, peer_abort));
    const float c2 = rowf[r];
    // No early exit from this loop: the warps of a pair meet at a barrier every tile, so a failed
    // wait only turns the remaining iterations into barrier-only ones.
    for (int j = wg; j < ntiles; j += 2) {
      const int si = j & (C::kScaleTiles - 1);
      const uint32_t sa = tmem + lane_base + C::kColS + wg * kKeys;
      const float* ks = ks_s + si * kKeys;
      const float* vs = vs_s + si * kKeys;
      // keys [0, vis) of the tile are visible to the row (0 for rows past the request end)
      const int64_t rem = row_valid ? klim - (int64_t)(jb + j) * kKeys : 0;
      const int vis = rem <= 0 ? 0 : (rem >= kKeys ? kKeys : (int)rem);
      if (ok) ok = __all_sync(0xffffffffu, wait_bar<false>(&sc_full[si], (j / C::kScaleTiles) & 1, abort, peer_abort));
      if (ok) ok = __all_sync(0xffffffffu, wait_bar<false>(&s_full[wg], (j >> 1) & 1, abort, peer_abort));
      if (idle) {  // P stays what S left there: it reaches only rows that are not stored
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0 && ok) {
          mbar_arrive(&p_full[2 * wg]);
          mbar_arrive(&p_full[2 * wg + 1]);
        }
        continue;
      }
      const float4 ap = *reinterpret_cast<const float4*>(apart_s + si * 4);
      const bool apart = ap.x + ap.y + ap.z + ap.w != 0.f;
      float tmax = -INFINITY;
      const float4* grp = grp_s + si * 4;
      if (ok) tc::fence_after_sync();
      if (ok && apart && kFold) wide_logits(sa, ks, vs, grp, c2);
      if (ok && apart && !kFold) {
        tmax = wide_max(sa, ks, vs, grp, c2, vis);
      } else if (ok) {
#pragma unroll 1
        for (int hf = 0; hf < 2; ++hf) {
          float s[2][32];
          tc::ld32(sa + 64 * hf, s[0]);
          tc::ld32(sa + 64 * hf + 32, s[1]);
          tc::wait_ld();
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int g = 2 * hf + k;
            scale_mask<kFold>(s[k], ks + 32 * g, vis - 32 * g);
            const float4 e = grp[g];
            tmax = fmaxf(tmax, fmaf(max_of_32(s[k]), logit_factor(c2, e.x, e.w), e.y));  // factor > 0
          }
        }
      }
      float m_prev = -INFINITY;
      if (j > 0) {
        named_barrier(bar_in, 64);
        m_prev = m_s[(wg ^ 1) * kRows + r];
      }
      const bool need = ok && (tmax > m_prev + kRescaleLog2 || (m_prev == -INFINITY && tmax > -INFINITY));
      const float m_new = need ? tmax : m_prev;
      if (j + 1 < ntiles) {
        m_s[wg * kRows + r] = m_new;
        __syncwarp();
        bar_arrive(bar_out, 64);
      }
      if (!ok) continue;
      {  // from this warpgroup's last tile
        const float h = fade(m_used, m_new);
        l_sum = l_sum * h * h;
      }
      m_used = m_new;
      const float nmu = m_new == -INFINITY ? 0.f : -m_new;
      const bool moved = j > 0 && need;
      float l_apart = -1.f;  // l with this tile's share where the weights do not give it
      if (__any_sync(0xffffffffu, moved || (kFold && apart))) {  // the rare steps of a tile behind one branch
        if (__any_sync(0xffffffffu, moved)) {  // rescale the O rows (after PV_{j-1})
          const float alpha = m_prev == m_new ? 1.f : ex2_ftz(m_prev - m_new);
          ok = __all_sync(0xffffffffu, wait_bar<false>(o_done, (j - 1) & 1, abort, peer_abort));
          if (!ok) continue;
          tc::fence_after_sync();
#pragma unroll 1
          for (int cc = 0; cc < D / 32; ++cc) {
            const uint32_t ta = tmem + lane_base + C::kColO + cc * 32;
            float s[32];
            tc::ld32(ta, s);
            tc::wait_ld();
#pragma unroll
            for (int k = 0; k < 32; ++k) s[k] *= alpha;
            tc::st32(ta, s);
          }
        }
        if (kFold && apart) l_apart = l_sum + wide_sum(sa, vs, grp, c2, vis, nmu, kBiasLog2<T>);
      }
      // float16 outputs carry as many bits as the weights.  In a request's first tile l sums the weights as
      // rounded, so that a rounding moves weight between keys and leaves their sum one (a row of one key
      // is exact).  Over more keys the error of l is the average of the weights' roundings, small beside
      // what those do to P V themselves, and the reciprocals would cost 128 a row and tile.
      const bool sum_rounded = !kFold && jb + j == 0;
#pragma unroll 1
      for (int g = 0; g < 4; ++g) {
        float s[32];
        tc::ld32(sa + 32 * g, s);
        tc::wait_ld();
        scale_mask<kFold>(s, ks + 32 * g, vis - 32 * g);
        const float4 e = grp[g];
        const float cg = logit_factor(c2, e.x, e.w), ng = kFold ? nmu + e.y : nmu;
        const uint64_t c22 = pk2(cg, cg), nmu2 = pk2(ng, ng);
        uint64_t ls2[2] = {0, 0};
        float pk[16];
        const ulonglong2* vp = reinterpret_cast<const ulonglong2*>(vs + 32 * g);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float* x = &s[4 * k];
          float e0, e1, e2, e3;
          up2(fma2(pk2(x[0], x[1]), c22, nmu2), e0, e1);
          up2(fma2(pk2(x[2], x[3]), c22, nmu2), e2, e3);
          e0 = ex2_ftz(e0);
          e1 = ex2_ftz(e1);
          e2 = ex2_ftz(e2);
          e3 = ex2_ftz(e3);
          uint64_t p01 = pk2(e0, e1), p23 = pk2(e2, e3);
          if (!kFold) {
            const ulonglong2 v = vp[k];
            up2(mul2(p01, v.x), e0, e1);
            up2(mul2(p23, v.y), e2, e3);
            pk[2 * k] = __uint_as_float(pack2_rn<__half>(e0, e1));
            pk[2 * k + 1] = __uint_as_float(pack2_rn<__half>(e2, e3));
            if (sum_rounded) {
              p01 = as_rounded(__float_as_uint(pk[2 * k]), v.x, p01);
              p23 = as_rounded(__float_as_uint(pk[2 * k + 1]), v.y, p23);
            }
          } else {
            pk[2 * k] = __uint_as_float(pack2_rn<__half>(e0, e1));
            pk[2 * k + 1] = __uint_as_float(pack2_rn<__half>(e2, e3));
          }
          ls2[0] = add2(ls2[0], p01);
          ls2[1] = add2(ls2[1], p23);
        }
        float h0, h1;
        up2(add2(ls2[0], ls2[1]), h0, h1);
        l_sum = kFold ? fmaf(h0 + h1, e.z, l_sum) : l_sum + (h0 + h1);
        // P over the first 32 columns of each 64 S columns: only this thread uses them, and it has read
        // the ones written here
        tc::st16(sa + 64 * (g >> 1) + 16 * (g & 1), pk);
        if (g & 1) {
          tc::wait_st();
          tc::fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[2 * wg + (g >> 1)]);  // rank 1's are forwarded to rank 0
        }
      }
      if (kFold && apart) l_sum = l_apart;
    }
    const bool gated = a.gate_mode != TF_GATE_NONE;
    const bool vec = rows_v16(a);
    if (ok) ok = __all_sync(0xffffffffu, wait_bar<false>(fin, 0, abort, peer_abort));
    // ---- epilogue.  Once fin completed, no product reads Q or the ring any more: the two halves' row
    // sums meet in the ring
    float2* l_part = reinterpret_cast<float2*>(sbase + C::kOffRing);  // [2][kRows] (m, l)
    if (ok) l_part[wg * kRows + r] = make_float2(m_used, l_sum);
    named_barrier(9, kSmWarps * 32);
    float l_tot = 0.f;
    if (ok) {
      const float2 o = l_part[(wg ^ 1) * kRows + r];
      const float mf = fmaxf(m_used, o.x);  // O's scale: the maxima only grow
      const float h0 = fade(m_used, mf), h1 = fade(o.x, mf);
      l_tot = l_sum * h0 * h0 + o.y * h1 * h1;
      m_used = mf;
    }
    named_barrier(10, (kSmWarps + kPrWarps) * 32);  // gate rows are staged
    if (ok) {
      tc::fence_after_sync();
      const int hq = h * G + (r - ri * G);
      const int64_t t = q0 + ri;
      const float inv = kBias<T> / l_tot;
      float* po = nullptr;
      if (sp.n > 1 && row_valid) {
        const int64_t row = ((int64_t)z * a.num_tokens + t) * a.num_q_heads + hq;
        po = sp.o + row * D + wg * kOHalf;
        if (wg == 0) *reinterpret_cast<float2*>(sp.ml + 2 * row) = make_float2(m_used, l_tot);
      }
      T* orow = (T*)a.out + t * a.out_stride_tok + (int64_t)hq * a.out_stride_head + wg * kOHalf;
      const T* grow = (const T*)a.gate + t * a.gate_stride_tok + (int64_t)hq * a.gate_stride_head + wg * kOHalf;
      constexpr int kChunks = D / 8;
      // 16 columns a pass in one copy of this code: it runs once a query tile from a cold instruction
      // cache (12 us with 32 columns unrolled and the gate's divisions in full precision)
#pragma unroll 1
      for (int cc = 0; cc < kOHalf / 16; ++cc) {
        float o[16];
        ld16(tmem + lane_base + C::kColO + wg * kOHalf + cc * 16, o);
        tc::wait_ld();
        if (!row_valid) continue;
        if (sp.n > 1) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            *reinterpret_cast<float4*>(po + cc * 16 + 4 * k) = make_float4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
          continue;
        }
        uint32_t gw[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (gated && vec) {
#pragma unroll
          for (int c8 = 0; c8 < 2; ++c8) {
            const int chunk = (wg * kOHalf + cc * 16) / 8 + c8;
            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                         : "=r"(gw[4 * c8]), "=r"(gw[4 * c8 + 1]), "=r"(gw[4 * c8 + 2]), "=r"(gw[4 * c8 + 3])
                         : "r"(base + r * (D * 2) + ((chunk ^ (r & (kChunks - 1))) << 4)));
          }
        } else if (gated) {
          const unsigned short* u = reinterpret_cast<const unsigned short*>(grow + cc * 16);
#pragma unroll
          for (int k = 0; k < 8; ++k) gw[k] = u[2 * k] | ((uint32_t)u[2 * k + 1] << 16);
        }
        uint32_t ow[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          float x0 = o[2 * k] * inv, x1 = o[2 * k + 1] * inv;
          if (gated) {
            x0 *= act(unpack_lo<T>(gw[k]), a.gate_mode);
            x1 *= act(unpack_hi<T>(gw[k]), a.gate_mode);
          }
          ow[k] = pack2_rn<T>(x0, x1);
        }
        if (vec) {
          *reinterpret_cast<uint4*>(orow + cc * 16) = make_uint4(ow[0], ow[1], ow[2], ow[3]);
          *reinterpret_cast<uint4*>(orow + cc * 16 + 8) = make_uint4(ow[4], ow[5], ow[6], ow[7]);
        } else {
          unsigned short* u = reinterpret_cast<unsigned short*>(orow + cc * 16);
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            u[2 * k] = (unsigned short)ow[k];
            u[2 * k + 1] = (unsigned short)(ow[k] >> 16);
          }
        }
      }
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  // rank 0's products read this CTA's shared memory and TMEM, and remote arrivals target rank 0's
  // barriers: neither CTA releases TMEM or exits before both are done
  cluster_sync();
  if (tid == 0 && *abort) record_err(a.err, TF_KERR_TIMEOUT);
  tc::fence_after_sync();
  if (warp == kIssueWarp)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::kTmemCols)
                 : "memory");
}

// one warp per (token, head): the clusters' partials of a row
template <typename T, int D>
__global__ void __launch_bounds__(256) merge_kernel(const __grid_constant__ tf_paged_attn_args a,
                                                    const __grid_constant__ Split sp, int64_t rows) {
  const int64_t row = (blockIdx.x * 256ll + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  // only rows of a request have partials
  int64_t total = 0;
  for (int i = lane; i < a.batch_size; i += 32) {
    const int64_t e = a.extend_lens ? a.extend_lens[i] : 1;
    total += e > 0 ? e : 0;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if (row >= rows || row >= total * a.num_q_heads) return;
  const int64_t t = row / a.num_q_heads;
  const int hq = (int)(row - t * a.num_q_heads);
  // a request whose lengths were refused has no partials either
  {
    int64_t base = 0;
    bool bad = false;
    for (int i0 = 0; i0 < a.batch_size; i0 += 32) {
      int64_t e = i0 + lane < a.batch_size ? (a.extend_lens ? a.extend_lens[i0 + lane] : 1) : 0;
      if (e < 0) e = 0;
      int64_t incl = e;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
      }
      const bool mine = t >= base + incl - e && t < base + incl;
      const int64_t L = mine ? a.seq_lens[i0 + lane] : 0;
      bad = bad || __any_sync(0xffffffffu, mine && (L > a.r2t_cols || L < e));
      base += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (bad) return;
  }
  const float* mlp = sp.ml + 2 * row;
  const float* op = sp.o + row * D;
  const int64_t step = a.num_tokens * (int64_t)a.num_q_heads;
  float M = -INFINITY;
  for (int z = 0; z < sp.n; ++z) M = fmaxf(M, mlp[2 * z * step]);
  constexpr int V = D / 32;  // values of a lane
  float o[V];
#pragma unroll
  for (int i = 0; i < V; ++i) o[i] = 0.f;
  float l = 0.f;
  for (int z = 0; z < sp.n; ++z) {
    const float2 ml = *reinterpret_cast<const float2*>(mlp + 2 * z * step);
    if (ml.x == -INFINITY && ml.y == 0.f) continue;  // no keys there, and no O written
    const float h = fade(ml.x, M), f = h * h;
    l = fmaf(h, h * ml.y, l);
    const float2* x = reinterpret_cast<const float2*>(op + z * step * D + V * lane);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const float2 v = x[i];
      o[2 * i] = fmaf(f, v.x, o[2 * i]);
      o[2 * i + 1] = fmaf(f, v.y, o[2 * i + 1]);
    }
  }
  const float inv = kBias<T> / l;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int d = V * lane + i;
    float y = o[i] * inv;
    if (a.gate_mode != TF_GATE_NONE)
      y *= act(to_f(((const T*)a.gate)[t * a.gate_stride_tok + (int64_t)hq * a.gate_stride_head + d]), a.gate_mode);
    ((T*)a.out)[t * a.out_stride_tok + (int64_t)hq * a.out_stride_head + d] = from_f<T>(y);
  }
}

// Clusters that share a query tile's keys: the number with the shortest sequence of waves, a cluster
// taking its share of the longest request's key tiles plus a fixed cost of about eight tiles (set-up,
// first loads, epilogue).
static int splits_of(const tf_paged_attn_args& a, int num_sms) {
  const int TQ2 = 2 * (kRows / (a.num_q_heads / a.num_kv_heads));
  const int64_t clusters = (int64_t)a.batch_size * ((a.max_extend_len + TQ2 - 1) / TQ2) * a.num_kv_heads;
  const int64_t slots = num_sms / 2, tiles = (a.max_seq_len + kKeys - 1) / kKeys;
  constexpr int64_t kFixed = 8;
  int best = 1;
  int64_t cost = INT64_MAX;
  for (int n = 1; n <= 32 && (n == 1 || tiles / n >= 2); ++n) {
    const int64_t c = (clusters * n + slots - 1) / slots * (kFixed + (tiles + n - 1) / n);
    if (c < cost) {
      cost = c;
      best = n;
    }
  }
  return best;
}

template <typename T, int D>
static cudaError_t launch_td(const tf_paged_attn_args& a, const tf_kv_scale& sc, void* ws, int num_sms,
                             cudaStream_t s) {
  const int G = a.num_q_heads / a.num_kv_heads;
  const int TQ = kRows / G;
  const int pairs = (a.max_extend_len + 2 * TQ - 1) / (2 * TQ);
  Split sp{splits_of(a, num_sms), nullptr, nullptr};
  const int64_t rows = (int64_t)a.num_tokens * a.num_q_heads;
  if (sp.n > 1) {
    sp.ml = (float*)ws;
    sp.o = sp.ml + ((2 * sp.n * rows + 63) & ~(int64_t)63);
  }
  cudaError_t e = cudaFuncSetAttribute(extend_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       Cfg<D>::kSmem);
  if (e != cudaSuccess) return e;
  dim3 grid((unsigned)(2 * (int64_t)a.batch_size * pairs * a.num_kv_heads), (unsigned)sp.n);
  extend_kernel<T, D><<<grid, kThreads, Cfg<D>::kSmem, s>>>(a, sc, pairs, sp);
  e = cudaGetLastError();
  if (e != cudaSuccess || sp.n == 1) return e;
  merge_kernel<T, D><<<(unsigned)((rows + 7) / 8), 256, 0, s>>>(a, sp, rows);
  return cudaGetLastError();
}

}  // namespace ext8

bool paged_fp8_extend_supported(const tf_paged_attn_args& a) {
  if (a.dtype != TF_DTYPE_BF16 && a.dtype != TF_DTYPE_F16) return false;
  if (a.head_dim != 64 && a.head_dim != 128 && a.head_dim != 256) return false;
  const int G = a.num_q_heads / a.num_kv_heads;
  if (G < 1 || G > 16) return false;
  if (a.max_extend_len <= 0) return false;
  const int64_t TQ2 = 2 * (ext8::kRows / G);
  if ((int64_t)a.batch_size * ((a.max_extend_len + TQ2 - 1) / TQ2) * a.num_kv_heads > 0x3fffffff) return false;
  if (!(a.scale > 0.f)) return false;  // the softmax takes its max before the scale
  auto al = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  // row offsets are kept in 32 bits of 16-byte pieces: pools of up to 64 GiB a layer
  if (a.num_slots * a.kv_stride_slot >= (int64_t)1 << 36) return false;
  return al(a.k_buffer) && al(a.v_buffer) && a.kv_stride_slot % 16 == 0 && a.kv_stride_head % 16 == 0;
}

size_t paged_fp8_extend_workspace(const tf_paged_attn_args& a, int num_sms) {
  const int n = ext8::splits_of(a, num_sms);
  if (n == 1) return 0;
  const int64_t rows = (int64_t)a.num_tokens * a.num_q_heads;
  return (((2 * n * rows + 63) & ~(int64_t)63) + n * rows * a.head_dim) * 4;
}

cudaError_t launch_paged_fp8_extend(const tf_paged_attn_args& a, const tf_kv_scale& sc, void* ws,
                                    int num_sms, cudaStream_t s) {
  const bool bf = a.dtype == TF_DTYPE_BF16;
  if (a.head_dim == 64)
    return bf ? ext8::launch_td<__nv_bfloat16, 64>(a, sc, ws, num_sms, s)
              : ext8::launch_td<__half, 64>(a, sc, ws, num_sms, s);
  if (a.head_dim == 128)
    return bf ? ext8::launch_td<__nv_bfloat16, 128>(a, sc, ws, num_sms, s)
              : ext8::launch_td<__half, 128>(a, sc, ws, num_sms, s);
  return bf ? ext8::launch_td<__nv_bfloat16, 256>(a, sc, ws, num_sms, s)
            : ext8::launch_td<__half, 256>(a, sc, ws, num_sms, s);
}

}  // namespace tf
