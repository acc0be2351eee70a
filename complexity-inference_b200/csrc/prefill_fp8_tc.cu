// K2b over the 8-bit paged cache on the 5th-generation tensor cores: varlen
// causal prefill, head_dim 128, one CTA per (sequence, KV head, 256 query rows).
//
// Mathematics (attention_fp8.cu): with K = ks * Kc, V = vs * Vc block by block and
// lv = log2 vs, a row's weights are w = exp2(s * ks * c + lv - m) with c = scale *
// log2 e and m a running bound of the exponent (without m) over the row, O = sum
// w Vc and l = sum w / vs; the result is O / l.  Codes go to f16 exactly; weights
// are rounded to f16 (2^-11, bf16 would be 2^-8).
//
// Tile shape.  256 rows = two query tiles of 128 (the G = Hq / Hkv heads of one KV
// head times 128 / G positions each); keys in tiles of 64.  Two query tiles share
// every converted K / V tile, which halves the conversion per multiply.  With 64
// keys a query tile has two S buffers beside its O in TMEM (2 x 64 + 128 columns),
// so S(t + 1) is there when the softmax of t ends: with 128 keys and one buffer a
// row's chain softmax -> P V -> Q K^T -> softmax took 5,250 clocks per 128 keys, of
// which the tensor core worked 2,050.
//
// Warp roles (16 warps of 128 registers; 14 has none):
//   0-3, 4-7   softmax of query tile 0 / 1, one thread per row: S from TMEM, mask,
//              weights back into TMEM over S (f16, the A operand of P V), O / l out.
//   8, 15      issue PV(t), QK(t + 2) of query tile 0 / 1 (8 also owns TMEM).  S(t + 2)
//              overwrites P(t): MMAs of one thread execute in order.
//   9-11, 13   conversion of codes to f16, 16 at a time, into 128-byte swizzled K-major
//              (K) / MN-major (V) panels, three stages each.
//   12         copies the paged blocks' codes (2 KB each, cp.async.bulk) into a ring.
// (An issuing warp slows the others of its SM sub-partition, which warps w, w + 4, ...
// share: no conversion warp sits beside the first, one beside the second.)
// TMEM: S_i of tile t at 128 i + 64 (t & 1), O_i at 256 + 128 i.
//
// The running bound only moves when a tile exceeds it by more than 8, so weights
// stay below 2^8 and O is rescaled in TMEM on those tiles alone (after P V of the
// tile before has run); O and l use the same bound.
//
// Measured: a fresh prompt of 4,000 tokens (32 query heads on 8) 166 us = 790 TFLOP/s, floor
// 80; four chunks of 300 to 700 rows behind 1,500 to 8,000 tokens (16 on 8) 142 us, floor 40:
// there the CTA with the longest context sets the time, 1.1 us per 64 keys for the two query
// tiles' chains softmax -> P V -> Q K^T, of which the multiplies are 0.76.  Bound: a row's
// chain, one thread from load to maximum, exponentials, pack and store; no pipe is full
// (tensor 39 % at N = 64, exponentials 30 %, issue slots 56 %).
//
// Few rows, long contexts (a short chunk behind a long past): where the query tiles would
// fill less than half of the SMs, the CTAs of a cluster of 2, 4 or 8 share the keys of one,
// at least 8 tiles each, and join their (m, l, O) through distributed shared memory, every
// CTA finishing a part of the rows.  64 rows behind 32k tokens (32 heads) took 566 us in one
// CTA per tile and take 95, one row behind 8k 144 and 37; with at least 16 tiles each, 64
// rows behind 1k took 28 us for 23.
//
// Every wait is bounded (common.cuh); on time-out the kernel records the error
// word, every role leaves its loop, TMEM is freed and the CTA returns.
#include <float.h>
#include <math.h>

#include "abi_util.h"
#include "common.cuh"
#include "fp8.cuh"
#include "prefill_fp8.h"

namespace muk {

constexpr int kXD = 128;             // head_dim
constexpr int kXRows = 128;          // rows of a query tile
constexpr int kXKeys = 64;           // keys of a tile
constexpr int kXThreads = 512;
constexpr int kXConvert = 4;         // conversion warps: 9, 10, 11 and 13
constexpr int kXIssuer = 8;          // owns TMEM and issues the multiplies of query tile 0
constexpr int kXIssuer1 = 15;        // issues those of query tile 1
constexpr int kXLoader = 12;         // the warp that issues the copies of codes
constexpr int kXStages = 3;          // converted steps: V(t) and K(t + 2)
constexpr int kXRing = 3;            // steps (a V and a K tile) of codes on their way
constexpr int kXFmaMask = 2;         // of 16 weights those i + 1 with (i & mask) == mask, i even: a quarter
constexpr int kXItem = kXKeys * 128; // bytes of such a tile
// Tiles of block constants: step t of the loader leaves those of tile t + 2 once the
// conversion has freed the ring slot of step t - kXRing, so both issuers the stage of step
// t - kXRing - kXStages, whose weights every softmax warp had then written: no warp reads
// constants older than those of tile t - kXRing - kXStages + 1.
constexpr int kXConsts = 16;
static_assert(kXConsts > kXRing + kXStages + 2, "block constants are overwritten in use");
constexpr int kXSplits = 8;          // CTAs that share the keys of a query tile, at most
constexpr int kXSplitTiles = 8;      // key tiles of each, at least
constexpr int kXQPanel = 128 * 128;  // [128 rows][64 f16], one swizzled panel of a query tile
constexpr int kXPanel = kXKeys * 128;  // the same of a K or V tile

struct XLayout {
  static constexpr int kStage = 2 * kXPanel;
  static constexpr int kQ = 0;                               // 2 tiles x 2 panels
  static constexpr int kK = kQ + 4 * kXQPanel;
  static constexpr int kV = kK + kXStages * kStage;
  static constexpr int kRaw = kV + kXStages * kStage;
  static constexpr int kBar = kRaw + kXRing * 2 * kXItem;
  static constexpr int kScale = kBar + 256;                  // [kXConsts tiles][4 blocks] float4
  static constexpr int kBytes = kScale + kXConsts * 4 * 16 + 1024;  // + alignment slack
};
static_assert(XLayout::kBytes <= 232448, "prefill tile exceeds 227 KB of shared memory");
static_assert((kXSplits - 1) * (2 * kXRows / kXSplits) * (kXD * 4 + 8) <= XLayout::kBar - XLayout::kK,
              "the rows of a join exceed the tiles' memory");
static_assert(kXSplitTiles >= kXSplits, "a CTA of a cluster could be left without tiles");

// Bounded wait of a whole warp (about a second).  One try on a complete barrier is
// ~110 clocks, so roles keep few barriers; the polls are one loop in PTX (as a C++ loop
// with its checks inside, a wait took ~250).
__device__ __noinline__ bool x_wait_long(uint32_t bar, uint32_t parity, int code) {
  for (int round = 0; round < 64; ++round) {
    uint32_t done;
    asm volatile(
        "{\n"
        ".reg .pred p, q;\n"
        ".reg .u32 n;\n"
        "mov.u32 n, 0;\n"
        "W%=:\n"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        "@p bra D%=;\n"
        "add.u32 n, n, 1;\n"
        "setp.lt.u32 q, n, 1048576;\n"
        "@q bra W%=;\n"
        "D%=:\n"
        "selp.u32 %0, 1, 0, p;\n"
        "}\n"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    if (__all_sync(0xffffffffu, done != 0)) return true;
    if (*reinterpret_cast<volatile int*>(&g_device_error) != 0) break;
  }
  set_device_error(code);  // keeps an earlier code
  return false;
}
__device__ __forceinline__ bool x_wait(uint64_t* bar, uint32_t parity, int code) {
  uint32_t done;
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      "selp.u32 %0, 1, 0, p;\n"
      "}\n"
      : "=r"(done)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  if (__all_sync(0xffffffffu, done != 0)) return true;
  return x_wait_long(smem_u32(bar), parity, code);
}
__device__ __forceinline__ uint32_t x_elect() {
  uint32_t r;
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "elect.sync _|p, 0xffffffff;\n"
      "selp.u32 %0, 1, 0, p;\n"
      "}\n"
      : "=r"(r));
  return r;
}
// 2^x, one MUFU op (~2 ulp), far below what the f16 weight keeps.
__device__ __forceinline__ float x_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 2^x on the FMA pipe, for a part of the weights (MUFU takes 8 clocks a warp, and was
// busy 1,024 of a tile's ~2,200): 2^n * p(f), n = round(x) from the bits of x + 1.5 * 2^23
// (127 more, so that they are 2^n's), f = x - n in [-1/2, 1/2], p the degree-4 minimax
// polynomial of 2^f (relative error 2^-18.5, fitted for this; f16 keeps 2^-11).  From
// -126.5 down n is -127, whose bits are 0.0: an unseen key weighs nothing, whatever 1 / vs
// its block has.  NaN stays NaN: a maximum that keeps it, and a product by 2^n (n added to
// the exponent would make a number of it).
__device__ __forceinline__ float x_exp2_fma(float x) {
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(x) : "f"(-127.f));
  const float z = x + 12583039.f;
  const float f = x - (z - 12583039.f);
  float p = fmaf(f, 0.0095701013f, 0.0559178628f);
  p = fmaf(p, f, 0.2402474433f);
  p = fmaf(p, f, 0.6931217909f);
  p = fmaf(p, f, 0.9999992847f);
  return p * __int_as_float(__float_as_int(z) << 23);
}
__device__ __forceinline__ float x_max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
// Exponents x * kc + lv - mu of two raw scores.  The score is rounded before mu, a rounded
// score itself, goes: with lv - mu formed first and one fma, scores from 2^28 on missed mu by
// more than f16 weights bear.  Packed, the two steps issue as often as that one did.
__device__ __forceinline__ void x_exponents(uint32_t x0, uint32_t x1, float kc, float lv, float mu,
                                            float& y0, float& y1) {
  asm("{\n.reg .b64 x, k, v, m;\n"
      "mov.b64 x, {%2, %3};\nmov.b64 k, {%4, %4};\nmov.b64 v, {%5, %5};\nmov.b64 m, {%6, %6};\n"
      "fma.rn.f32x2 x, x, k, v;\nadd.rn.f32x2 x, x, m;\nmov.b64 {%0, %1}, x;\n}\n"
      : "=f"(y0), "=f"(y1)
      : "r"(x0), "r"(x1), "f"(kc), "f"(lv), "f"(-mu));
}
// Largest of 16 raw scores.
__device__ __forceinline__ float x_max16(const uint32_t* x) {
  auto f = [&](int i) { return __uint_as_float(x[i]); };
  const float a = x_max3(f(0), f(1), f(2)), b = x_max3(f(3), f(4), f(5));
  const float c = x_max3(f(6), f(7), f(8)), d = x_max3(f(9), f(10), f(11));
  const float e = x_max3(f(12), f(13), f(14));
  return x_max3(x_max3(a, b, c), x_max3(d, e, f(15)), a);
}
// The warp runs the issue loop as one, so that addresses stay in uniform registers
// (from one diverged lane each multiply took ~80 clocks to issue, more than its 64
// to run); `lead` picks the lane that issues.
// D(tmem) (+)= A(smem descriptor) * B(smem descriptor)
__device__ __forceinline__ void x_mma_ss(uint32_t lead, uint32_t d, uint64_t adesc, uint64_t bdesc,
                                         uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p, q;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "setp.ne.b32 q, %5, 0;\n"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
      "}\n" ::"r"(d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(lead));
}
// D(tmem) (+)= A(tmem, f16) * B(smem descriptor)
__device__ __forceinline__ void x_mma_ts(uint32_t lead, uint32_t d, uint32_t a, uint64_t bdesc,
                                         uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p, q;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "setp.ne.b32 q, %5, 0;\n"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
      "}\n" ::"r"(d),
      "r"(a), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(lead));
}
__device__ __forceinline__ void x_commit(uint32_t lead, uint64_t* bar) {
  asm volatile(
      "{\n"
      ".reg .pred q;\n"
      "setp.ne.b32 q, %1, 0;\n"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n"
      "}\n" ::"r"(smem_u32(bar)),
      "r"(lead)
      : "memory");
}
// 16 registers per thread into 32 lanes x 16 columns of TMEM.
__device__ __forceinline__ void x_tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,"
      "%14,%15,%16};\n" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// An address of this CTA's shared memory as that of the cluster's CTA `rank`.
__device__ __forceinline__ uint32_t x_mapa(uint32_t addr, int rank) {
  uint32_t y;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(y) : "r"(addr), "r"(rank));
  return y;
}
// Instruction descriptor, kind::f16: f16 A/B (format 0), f32 D, A K-major.
__host__ __device__ constexpr uint32_t x_idesc(bool b_mn, int n) {
  return (1u << 4) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(kXRows >> 4) << 24);
}

// Split: the CTAs of a cluster share a query tile's keys (otherwise one has all of them, in
// code without the join: as one kernel for both, 4,000 tokens took 5 % longer).
template <bool Split>
__global__ void __launch_bounds__(kXThreads, 1) prefill_fp8_tc_kernel(const PrefillFp8Args a) {
  // programmatic dependent launch: let the next kernel launch once every CTA
  // of this one runs, and wait for the previous kernel before touching memory
  grid_dep_launch();
  grid_dep_wait();
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* basep = smem_raw + (base - raw);
  uint64_t* st_full = reinterpret_cast<uint64_t*>(basep + XLayout::kBar);  // [stage] step converted
  uint64_t* st_empty = st_full + kXStages;                                 // [stage] and used
  uint64_t* s_full = st_empty + kXStages; // [query tile][buffer] S complete
  uint64_t* p_full = s_full + 4;          // [query tile][buffer] weights written
  uint64_t* o_done = p_full + 4;          // [query tile] P V of a tile complete
  uint64_t* o_last = o_done + 2;          // [query tile] P V of the last tile complete
  uint64_t* raw_full = o_last + 2;        // [ring slot] codes of a step
  uint64_t* raw_empty = raw_full + kXRing;
  uint64_t* q_full = raw_empty + kXRing;
  uint64_t* drain = q_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 2);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.z, kvh = Split ? blockIdx.x / a.splits : blockIdx.x;
  const int qt = (int)gridDim.y - 1 - (int)blockIdx.y;  // longest (last) query tiles first
  const int G = a.num_q_heads / a.num_kv_heads;
  const int P = 2 * kXRows / G;                          // positions of the CTA
  const int q_begin = a.cu_q[b];
  const int q_len = a.cu_q[b + 1] - q_begin;
  const int p0 = qt * P;
  if (p0 >= q_len) return;                               // uniform: nothing for this CTA
  const int ctx = a.seq_lens[b];
  const int past = ctx - q_len;
  const int n_keys = past + min(p0 + P, q_len);          // keys 0 .. n_keys - 1
  const int nt = (n_keys - 1) / kXKeys + 1;
  const int nblk = (n_keys - 1) / kKvBlock + 1;
  // uniform: the launch does not cover this sequence
  if (past < 0 || nblk > a.max_blocks || q_begin < 0 || q_len > a.max_q_len ||
      q_begin > a.num_rows - q_len) {
    if (threadIdx.x == 0) set_device_error(kDevBadShape);
    return;
  }
  const int32_t* bt = a.block_tables + (int64_t)b * a.bt_stride;
  // The key tiles are shared out over the CTAs of a cluster, as many as get kXSplitTiles
  // each (all of a cluster come to the same number); this one has tiles t0 .. t0 + nl - 1.
  int splits = Split ? a.splits : 1;
  while (Split && splits > 1 && nt < kXSplitTiles * splits) splits >>= 1;
  const int rank = Split ? (int)blockIdx.x % a.splits : 0;
  const int per = Split ? (nt + splits - 1) / splits : nt;
  const int t0 = Split ? rank * per : 0;
  const int nl = Split ? min(per, nt - t0) : nt;         // > 0 for rank < splits: nt >= splits^2
  if (Split && rank >= splits) return;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kXStages; ++i) {
      mbar_init(&st_full[i], kXConvert);
      mbar_init(&st_empty[i], 2);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&o_done[i], 1);
      mbar_init(&o_last[i], 1);
    }
    for (int i = 0; i < kXRing; ++i) {
      mbar_init(&raw_full[i], 1);
      mbar_init(&raw_empty[i], kXConvert);
    }
    mbar_init(q_full, 8);
    mbar_init(&drain[0], 1);
    mbar_init(&drain[1], 1);
    fence_mbar_init();
  }
  if (warp == kXIssuer) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  float m_used = -INFINITY, l = 0.f;  // of a softmax thread's row

  if (warp == kXIssuer || warp == kXIssuer1) {
    // ---- MMA issuers ---------------------------------------------------------
    const uint32_t lead = x_elect();
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    const uint64_t dq = umma_desc_sw128(base + XLayout::kQ);
    const uint64_t dk = umma_desc_sw128(base + XLayout::kK);
    const uint64_t dv = umma_desc_sw128_mn(base + XLayout::kV, kXPanel, 1024);
    const int qi = warp == kXIssuer ? 0 : 1;           // this warp's query tile
    const uint64_t dqi = dq + (uint64_t)((qi * 2 * kXQPanel) >> 4);  // addresses in 16-byte units
    const uint32_t s_at = tm + (uint32_t)(qi * 2 * kXKeys), o_at = tm + (uint32_t)(4 * kXKeys + qi * kXD);
    auto qk = [&](int t, int sg) {  // S(t) = Q K_t^T
      const uint64_t k0 = dk + (uint64_t)(sg * (XLayout::kStage >> 4));
      const uint32_t d = s_at + (uint32_t)((t & 1) * kXKeys);
#pragma unroll
      for (int k = 0; k < kXD / 16; ++k)
        x_mma_ss(lead, d, dqi + (uint64_t)(((k >> 2) * kXQPanel + (k & 3) * 32) >> 4),
                 k0 + (uint64_t)(((k >> 2) * kXPanel + (k & 3) * 32) >> 4), x_idesc(false, kXKeys),
                 k > 0 ? 1u : 0u);
      x_commit(lead, &s_full[qi * 2 + (t & 1)]);
    };
    auto pv = [&](int t, int sg) {  // O += P(t) V_t
      const uint64_t v0 = dv + (uint64_t)(sg * (XLayout::kStage >> 4));
      const uint32_t p = s_at + (uint32_t)((t & 1) * kXKeys);
#pragma unroll
      for (int k = 0; k < kXKeys / 16; ++k)
        x_mma_ts(lead, o_at, p + (uint32_t)(k * 8), v0 + (uint64_t)((k * 16 * 128) >> 4),
                 x_idesc(true, kXD), (t > 0 || k > 0) ? 1u : 0u);
      // a barrier of its own for the last one: its reader may be two tiles ahead of the
      // multiplies there, which the phase of o_done cannot tell
      x_commit(lead, t + 1 < nl ? &o_done[qi] : &o_last[qi]);
    };
    // Step t = -2 .. nl - 1 uses V(t) and K(t + 2) of stage (t + 2) % kXStages.
    bool ok = x_wait(q_full, 0, kDevTimeoutFull);
    int sg = 0;
    uint32_t ph = 0;
    for (int t = -2; ok && t < nl; ++t) {
      ok = x_wait(&st_full[sg], ph, kDevTimeoutFull);
      if (ok && t >= 0) ok = x_wait(&p_full[qi * 2 + (t & 1)], (uint32_t)(t >> 1) & 1u, kDevTimeoutFull);
      if (!ok) break;
      tc_fence_after();
      if (t >= 0) pv(t, sg);
      if (t + 2 < nl) qk(t + 2, sg);
      x_commit(lead, &st_empty[sg]);
      if (++sg == kXStages) sg = 0, ph ^= 1;
    }
    // every MMA this warp issued has finished before TMEM is freed, also when a
    // wait above gave up
    x_commit(lead, &drain[qi]);
    x_wait(&drain[qi], 0, kDevTimeoutAccum);
  } else if (warp == kXLoader) {
    // ---- loads of codes -------------------------------------------------------
    // Step t brings V(t) and K(t + 2), which the multiplies of one step need (steps -2
    // and -1: K alone): lanes 0-3 a block of V each, 4-7 one of K, 2 KB a copy.  Blocks
    // behind the last key are left out (their rows become zero when converted).  Lanes 4-7
    // also leave the constants of their block of tile t + 2 (ks, log2 vs, 1 / vs) for the
    // softmax warps, before this warp's arrival on the codes: S(t + 2) comes after the
    // conversion of the K codes of this step.
    const bool mine_k = lane >= 4;
    const uint8_t* src = (mine_k ? a.k_cache : a.v_cache) + (int64_t)kvh * (kKvBlock * kXD);
    const int64_t blk_bytes = (int64_t)a.num_kv_heads * (kKvBlock * kXD);
    const uint32_t dst = base + (uint32_t)(XLayout::kRaw + (mine_k ? kXItem : 0) + (lane & 3) * 2048);
    const int mine_blks = min(nl * 4, nblk - t0 * 4);  // of this CTA's tiles
    auto block_of = [&](int t) {                     // of this lane in step t, -1: none
      const int blk = (mine_k ? t + 2 : t) * 4 + (lane & 3);
      if (!Split) return lane < 8 && blk >= 0 && blk < nblk ? blk : -1;
      return lane < 8 && blk >= 0 && blk < mine_blks ? t0 * 4 + blk : -1;
    };
    auto id_of = [&](int t) {
      const int blk = block_of(t);
      return blk >= 0 ? __ldg(bt + blk) : 0;
    };
    auto scales_of = [&](int t, int i) {             // of this lane's block of tile t + 2 (lanes 4-7)
      const int64_t at = (int64_t)(i >= 0 && i < a.num_blocks ? i : 0) * a.num_kv_heads + kvh;
      return mine_k && block_of(t) >= 0 ? make_float2(__ldg(a.k_scale + at), __ldg(a.v_scale + at))
                                          : make_float2(1.f, 1.f);
    };
    float4* consts = reinterpret_cast<float4*>(basep + XLayout::kScale);
    int id = id_of(-2), id_next = id_of(-1), slot = 0, issued = 0;
    float2 scales = scales_of(-2, id);
    uint32_t ph = 1;
    for (int t = -2; t < nl; ++t) {
      if (!x_wait(raw_empty + slot, ph, kDevTimeoutEmpty)) break;
      const bool have = block_of(t) >= 0;
      const int blocks = __popc(__ballot_sync(0xffffffffu, have));
      if (id < 0 || id >= a.num_blocks) {
        set_device_error(kDevBadIndex);
        id = 0;
      }
      // The copies go first (their bytes may arrive before they are expected: the phase
      // still lacks this warp's arrival), so that they overlap the loads of the scales.
      if (have)
        asm volatile(
            "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], 2048, [%2];\n" ::"r"(
                dst + (uint32_t)(slot * 2 * kXItem)),
            "l"(src + id * blk_bytes), "r"(smem_u32(raw_full + slot))
            : "memory");
      if (mine_k && lane < 8 && t + 2 < nl) {
        const float ks = clamp_scale(scales.x), vs = clamp_scale(scales.y);
        float lv, iv;
        asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(lv) : "f"(vs));  // exact for powers of two
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(iv) : "f"(vs));
        consts[((t + 2) % kXConsts) * 4 + (lane & 3)] = make_float4(ks, lv, iv, 0.f);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive_expect_tx(raw_full + slot, (uint32_t)(blocks * 2048));
      ++issued;
      id = id_next;
      id_next = id_of(t + 2);
      scales = scales_of(t + 1, id);
      if (++slot == kXRing) slot = 0, ph ^= 1;
    }
    // No copy may still be on its way when the CTA ends, also where the others gave up:
    // the last copies into each slot have arrived.
    for (int m = max(issued - kXRing, 0); m < issued; ++m)
      x_wait(raw_full + m % kXRing, (uint32_t)(m / kXRing) & 1u, kDevTimeoutFull);
  } else if (warp >= 8 && warp != 14) {
    // ---- conversion -----------------------------------------------------------
    // Warp w takes rows 4w .. 4w + 3 of every block (512 contiguous bytes), a lane one
    // 16-code chunk of them.  Eight neighbouring lanes cover two rows of one panel,
    // which the swizzle puts into all 32 banks.
    const int w = warp == 13 ? 3 : warp - 9, row = 4 * w + (lane >> 4) * 2 + ((lane >> 2) & 1);
    const int c = (lane & 3) + ((lane >> 3) & 1) * 4;
    constexpr int kBpt = kXKeys / kKvBlock;          // blocks of a tile
    const uint32_t ring = base + (uint32_t)(XLayout::kRaw + row * kXD + c * 16);
    // this lane's two 16-byte places in block 0's rows of a stage
    const uint32_t st = base + (uint32_t)((c >> 2) * kXPanel + row * 128);
    const uint32_t s0 = st + (uint32_t)(((2 * (c & 3)) ^ (row & 7)) << 4);
    const uint32_t s1 = st + (uint32_t)(((2 * (c & 3) + 1) ^ (row & 7)) << 4);
    auto read = [&](uint4 (&v)[kBpt], uint32_t src) {
#pragma unroll
      for (int j = 0; j < kBpt; ++j) {
        const float4 f = ld_shared_f4(src + (uint32_t)(j * 2048));
        v[j] = make_uint4(__float_as_uint(f.x), __float_as_uint(f.y), __float_as_uint(f.z),
                          __float_as_uint(f.w));
      }
    };
    auto convert = [&](uint4 (&v)[kBpt], int t, uint32_t at) {
      if (t0 + t == nt - 1) {  // rows behind the last key are zero: what the blocks hold there is not ours
#pragma unroll
        for (int j = 0; j < kBpt; ++j)
          if ((t0 + t) * kXKeys + j * kKvBlock + row >= n_keys) v[j] = make_uint4(0u, 0u, 0u, 0u);
      }
#pragma unroll
      for (int j = 0; j < kBpt; ++j) {
        uint32_t x[8];
        e4m3x4_to_f16x4(v[j].x, x[0], x[1]);
        e4m3x4_to_f16x4(v[j].y, x[2], x[3]);
        e4m3x4_to_f16x4(v[j].z, x[4], x[5]);
        e4m3x4_to_f16x4(v[j].w, x[6], x[7]);
        const uint32_t o = at + (uint32_t)(j * kKvBlock * 128);
        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(s0 + o), "r"(x[0]), "r"(x[1]),
                     "r"(x[2]), "r"(x[3]) : "memory");
        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(s1 + o), "r"(x[4]), "r"(x[5]),
                     "r"(x[6]), "r"(x[7]) : "memory");
      }
    };
    int slot = 0, sg = 0;
    uint32_t ph_r = 0, ph = 1;                       // parities: ring "full", stage "empty"
    for (int t = -2; t < nl; ++t) {                  // step t: V(t) and K(t + 2)
      const bool has_v = t >= 0, has_k = t + 2 < nl;
      uint4 vv[kBpt], vk[kBpt];
      if (!x_wait(raw_full + slot, ph_r, kDevTimeoutFull)) break;
      const uint32_t src = ring + (uint32_t)(slot * 2 * kXItem);
      if (has_v) read(vv, src);
      if (has_k) read(vk, src + kXItem);
      if (!x_wait(st_empty + sg, ph, kDevTimeoutEmpty)) break;
      if (has_v) convert(vv, t, (uint32_t)(XLayout::kV + sg * XLayout::kStage));
      if (has_k) convert(vk, t + 2, (uint32_t)(XLayout::kK + sg * XLayout::kStage));
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(st_full + sg);
        mbar_arrive(raw_empty + slot);
      }
      if (++sg == kXStages) sg = 0, ph ^= 1;
      if (++slot == kXRing) slot = 0, ph_r ^= 1;
    }
  } else if (warp < 8) {
    // ---- softmax / epilogue: one thread per query row --------------------------
    const int qi = warp >> 2;                        // query tile
    const int r = (warp & 3) * 32 + lane;            // row = TMEM lane
    const int row = qi * kXRows + r;
    const int pos = p0 + row / G;
    const int h = kvh * G + row % G;
    const bool row_ok = pos < q_len;
    const int limit = past + pos;                    // last key this row may see
    const int tile_limit = past + p0 + (qi * kXRows + (warp & 3) * 32) / G;  // smallest of the warp
    const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t to = lane_base + (uint32_t)(4 * kXKeys + qi * kXD);
    float c;                                          // scale_log2 / the row's power of two
    {
      // the query row, brought into f16 by a power of two
      const uint4* src = reinterpret_cast<const uint4*>(
          a.q + (int64_t)(q_begin + (row_ok ? pos : 0)) * a.q_stride + (int64_t)h * kXD);
      uint4 q[16];
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i) q[i] = row_ok ? src[i] : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const uint32_t w[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
#pragma unroll
        for (int u = 0; u < 4; ++u)
          top = max(top, max((w[u] << 16) & 0x7fffffffu, w[u] & 0x7fff0000u));
      }
      float up, down;
      row_factor(top, 14, up, down);
      c = down * a.scale_log2;
      uint8_t* qrow = basep + XLayout::kQ + qi * 2 * kXQPanel + r * 128;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float2 x0 = unpack_bf16x2(q[i].x), x1 = unpack_bf16x2(q[i].y);
        const float2 x2 = unpack_bf16x2(q[i].z), x3 = unpack_bf16x2(q[i].w);
        uint4 o;
        o.x = pack_f16x2(x0.x * up, x0.y * up);
        o.y = pack_f16x2(x1.x * up, x1.y * up);
        o.z = pack_f16x2(x2.x * up, x2.y * up);
        o.w = pack_f16x2(x3.x * up, x3.y * up);
        *reinterpret_cast<uint4*>(qrow + (i >> 3) * kXQPanel + (((i & 7) ^ (r & 7)) << 4)) = o;
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
    }
    const float4* consts = reinterpret_cast<const float4*>(basep + XLayout::kScale);
    bool ok = true;
    for (int t = 0; t < nl; ++t) {
      const int sb = qi * 2 + (t & 1);
      const uint32_t ts = lane_base + (uint32_t)(sb * kXKeys);
      ok = x_wait(&s_full[sb], (uint32_t)(t >> 1) & 1u, kDevTimeoutAccum);
      if (!ok) break;
      tc_fence_after();
      const int k0 = (t0 + t) * kXKeys;
      const bool diagonal = k0 + kXKeys - 1 > tile_limit;  // uniform: some row's limit falls in the tile
      const float4* cs = consts + (t % kXConsts) * 4;
      uint32_t s[2][32];
      tmem_ld_32x32b_x32(ts, s[0]);
      tmem_ld_32x32b_x32(ts + 32, s[1]);
      tmem_ld_wait();
      if (diagonal) {  // -inf where the row does not see the key
        const int seen = limit - k0;
#pragma unroll
        for (int i = 0; i < kXKeys; ++i)
          if (i > seen) s[i >> 5][i & 31] = 0xff800000u;
      }
      float mt = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float mj = x_max16(&s[j >> 1][16 * (j & 1)]);
        const float4 k = cs[j];
        mt = fmaxf(mt, mj == -INFINITY ? -INFINITY : fmaf(mj, k.x * c, k.y));
      }
      float corr = 1.f;
      if (mt > m_used + 8.f) {                        // also true on the first tile
        corr = m_used == -INFINITY ? 0.f : x_exp2(m_used - mt);
        m_used = mt;
      }
      const float mu = m_used == -INFINITY ? 0.f : m_used;
      float sum = 0.f;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        uint32_t p[16];
#pragma unroll
        for (int jj = 0; jj < 2; ++jj) {
          const int j = 2 * q + jj;
          const uint32_t* x = &s[q][16 * jj];
          const float4 k = cs[j];
          // a block that this row does not see must not reach it even as NaN
          const bool hidden = diagonal && k0 + 16 * j > limit;
          // A block of zeros has the smallest scale, and a row of tiny queries brings the
          // product to 0: held to the smallest normal, at which every score is 0 all the
          // same (|x| < 2^31), unseen keys stay -inf (a NaN scale stays NaN).
          float kc = k.x * c;
          kc = kc < FLT_MIN ? FLT_MIN : kc;
          kc = hidden ? 1.f : kc;
          const float lv = hidden ? 0.f : k.y;
          float sa = 0.f, sb2 = 0.f;
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            float y0, y1;
            x_exponents(x[i], x[i + 1], kc, lv, mu, y0, y1);
            const float w0 = x_exp2(y0);
            const float w1 = (i & kXFmaMask) == kXFmaMask ? x_exp2_fma(y1) : x_exp2(y1);
            sa += w0;
            sb2 += w1;
            p[8 * jj + i / 2] = pack_f16x2(w0, w1);
          }
          sum = hidden ? sum : fmaf(sa + sb2, k.z, sum);
        }
        x_tmem_st16(ts + 16 * q, p);                  // over S, which is in registers
      }
      l = l * corr + sum;
      if (t > 0 && __any_sync(0xffffffffu, corr != 1.f)) {
        // P V of t - 1 is in O (that of t - 2 is, or S(t) would not be)
        ok = x_wait(&o_done[qi], (uint32_t)(t - 1) & 1u, kDevTimeoutAccum);
        if (!ok) break;
        tc_fence_after();
        uint32_t rr[32];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          tmem_ld_32x32b_x32(to + 32 * i, rr);
          tmem_ld_wait();
#pragma unroll
          for (int u = 0; u < 32; ++u) rr[u] = __float_as_uint(__uint_as_float(rr[u]) * corr);
          tmem_st_32x32b_x32(to + 32 * i, rr);
        }
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[sb]);
    }
    if (ok) ok = x_wait(&o_last[qi], 0, kDevTimeoutAccum);
    if (Split && splits > 1 && !ok) m_used = -INFINITY, l = 0.f;  // nothing to join
    if (ok && (!Split || splits == 1)) {
      tc_fence_after();
      const float inv = 1.f / l;
      uint4* dst = reinterpret_cast<uint4*>(
          a.out + (int64_t)(q_begin + (row_ok ? pos : 0)) * a.out_stride + (int64_t)h * kXD);
      uint32_t rr[32];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        tmem_ld_32x32b_x32(to + 32 * i, rr);
        tmem_ld_wait();
        if (row_ok) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint4 v;
            v.x = pack_bf16x2(__uint_as_float(rr[j * 8 + 0]) * inv, __uint_as_float(rr[j * 8 + 1]) * inv);
            v.y = pack_bf16x2(__uint_as_float(rr[j * 8 + 2]) * inv, __uint_as_float(rr[j * 8 + 3]) * inv);
            v.z = pack_bf16x2(__uint_as_float(rr[j * 8 + 4]) * inv, __uint_as_float(rr[j * 8 + 5]) * inv);
            v.w = pack_bf16x2(__uint_as_float(rr[j * 8 + 6]) * inv, __uint_as_float(rr[j * 8 + 7]) * inv);
            dst[i * 4 + j] = v;
          }
        }
      }
    }
  }

  if (Split && splits > 1) {
    // ---- join of the cluster's results (m, l, O): a CTA finishes the rows of 8 / splits
    // softmax warps, the others write theirs into its memory over the tiles
    tc_fence_before();
    cluster_sync();  // every CTA is done with its tiles
    tc_fence_after();
    const int warps = 8 / splits, owner = warp / warps;
    const uint32_t rows = (uint32_t)warps * 32;
    const uint32_t box = base + (uint32_t)XLayout::kK;                   // [sender][row][128] f32
    const uint32_t ml = box + (uint32_t)(splits - 1) * rows * (kXD * 4); // [sender][row] (m, l)
    const uint32_t my = (uint32_t)(warp % warps) * 32 + lane;            // this thread's row there
    const uint32_t to = tmem + ((uint32_t)((warp & 3) * 32) << 16) +
                        (uint32_t)(4 * kXKeys + (warp >> 2) * kXD);
    // 16-byte chunk c of a row lies at c ^ lane, or 32 rows would meet in four banks
    uint32_t rr[32];
    if (warp < 8 && owner != rank) {
      const uint32_t at = (uint32_t)(rank < owner ? rank : rank - 1) * rows + my;
      const uint32_t dst = x_mapa(box + at * (kXD * 4), owner), dml = x_mapa(ml + at * 8, owner);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        tmem_ld_32x32b_x32(to + 32 * i, rr);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 8; ++j)
          asm volatile("st.shared::cluster.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(
                           dst + (uint32_t)(((i * 8 + j) ^ lane) << 4)),
                       "r"(rr[4 * j]), "r"(rr[4 * j + 1]), "r"(rr[4 * j + 2]), "r"(rr[4 * j + 3])
                       : "memory");
      }
      asm volatile("st.shared::cluster.v2.f32 [%0], {%1,%2};" ::"r"(dml), "f"(m_used), "f"(l)
                   : "memory");
    }
    cluster_sync();  // the rows have arrived; from here on a CTA reads its own memory only
    if (warp < 8 && owner == rank) {
      const int row = warp * 32 + lane, pos = p0 + row / G, h = kvh * G + row % G;
      auto get_ml = [&](int s, float& m, float& x) {
        asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(m), "=f"(x) : "r"(ml + (s * rows + my) * 8) : "memory");
      };
      float M = m_used;
      for (int s = 0; s < splits - 1; ++s) {
        float m, x;
        get_ml(s, m, x);
        M = fmaxf(M, m);
      }
      // A row without a bound has seen no key (l 0: its O is not read), or NaN alone.  Every
      // other share counts, however small its factor: the bound ignores NaN, which l and O
      // hold, and 0 * NaN is NaN.
      auto live = [&](float m, float x) { return m != -INFINITY || x != 0.f; };
      auto factor = [&](float m) { return m == -INFINITY ? 1.f : x_exp2(m - M); };
      const bool has = live(m_used, l);
      const float own = factor(m_used);
      float L = has ? own * l : 0.f;
      for (int s = 0; s < splits - 1; ++s) {
        float m, x;
        get_ml(s, m, x);
        if (live(m, x)) L = fmaf(factor(m), x, L);
      }
      const float inv = 1.f / L;
#pragma unroll 1
      for (int i = 0; i < 4; ++i) {
        tmem_ld_32x32b_x32(to + 32 * i, rr);
        tmem_ld_wait();
        float o[32];
#pragma unroll
        for (int u = 0; u < 32; ++u) o[u] = has ? own * __uint_as_float(rr[u]) : 0.f;
        for (int s = 0; s < splits - 1; ++s) {
          float m, x;
          get_ml(s, m, x);
          const float f = factor(m);
          if (live(m, x)) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float4 v = ld_shared_f4(box + (s * rows + my) * (kXD * 4) + (uint32_t)(((i * 8 + j) ^ lane) << 4));
              o[4 * j] = fmaf(f, v.x, o[4 * j]);
              o[4 * j + 1] = fmaf(f, v.y, o[4 * j + 1]);
              o[4 * j + 2] = fmaf(f, v.z, o[4 * j + 2]);
              o[4 * j + 3] = fmaf(f, v.w, o[4 * j + 3]);
            }
          }
        }
        if (pos < q_len) {
          uint4* dst = reinterpret_cast<uint4*>(a.out + (int64_t)(q_begin + pos) * a.out_stride +
                                                (int64_t)h * kXD) + i * 4;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            dst[j] = make_uint4(pack_bf16x2(o[8 * j] * inv, o[8 * j + 1] * inv),
                                pack_bf16x2(o[8 * j + 2] * inv, o[8 * j + 3] * inv),
                                pack_bf16x2(o[8 * j + 4] * inv, o[8 * j + 5] * inv),
                                pack_bf16x2(o[8 * j + 6] * inv, o[8 * j + 7] * inv));
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kXIssuer) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

static int x_sm_count() {
  static std::atomic<int> count[64];
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if ((n = count[dev].load(std::memory_order_relaxed)) == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
    count[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

bool prefill_fp8_tc_supported(int head_dim, int num_q_heads, int num_kv_heads) {
  const int G = num_q_heads / num_kv_heads;
  return head_dim == kXD && kXRows % G == 0;
}

int launch_prefill_fp8_tc(PrefillFp8Args a, int num_seqs, int max_q_len, cudaStream_t stream) {
  const int P = 2 * kXRows / (a.num_q_heads / a.num_kv_heads);
  MUK_REQUIRE((max_q_len + P - 1) / P <= 65535 && num_seqs <= 65535,
              "muk_paged_prefill_attn_fp8: %d rows of a sequence", max_q_len);
  const int qtiles = (max_q_len + P - 1) / P;
  const int64_t ctas = (int64_t)a.num_kv_heads * qtiles * num_seqs;
  const int64_t tiles = ((int64_t)a.max_blocks * kKvBlock + kXKeys - 1) / kXKeys;
  a.splits = 1;
  while (a.splits < kXSplits && ctas * a.splits * 2 <= x_sm_count() &&
         tiles >= (int64_t)kXSplitTiles * a.splits * 2)
    a.splits *= 2;
  auto kernel = a.splits > 1 ? prefill_fp8_tc_kernel<true> : prefill_fp8_tc_kernel<false>;
  static std::atomic<uint64_t> attr_done[2];
  const cudaError_t ae = smem_attr_once(kernel, XLayout::kBytes, attr_done[a.splits > 1]);
  if (ae != cudaSuccess) {
    set_last_error("muk_paged_prefill_attn_fp8: cudaFuncSetAttribute: %s", cudaGetErrorString(ae));
    return MUK_ERR_CUDA;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.num_kv_heads * a.splits), (unsigned)qtiles, (unsigned)num_seqs);
  cfg.blockDim = dim3(kXThreads);
  cfg.dynamicSmemBytes = XLayout::kBytes;
  cfg.stream = stream;
  cudaLaunchAttribute at[2];
  int n = 0;
  if (pdl_enabled()) {
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (a.splits > 1) {
    at[n].id = cudaLaunchAttributeClusterDimension;
    at[n].val.clusterDim.x = (unsigned)a.splits;
    at[n].val.clusterDim.y = 1;
    at[n++].val.clusterDim.z = 1;
  }
  cfg.attrs = at;
  cfg.numAttrs = n;
  const cudaError_t le = cudaLaunchKernelEx(&cfg, kernel, a);
  if (le != cudaSuccess) {
    cudaGetLastError();
    set_last_error("muk_paged_prefill_attn_fp8: launch failed: %s", cudaGetErrorString(le));
    return MUK_ERR_CUDA;
  }
  return check_launch("muk_paged_prefill_attn_fp8");
}

}  // namespace muk
