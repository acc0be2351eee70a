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
// head times 128 / G positions each); keys in tiles of 128.  Two query tiles share
// every converted K / V tile, which halves the conversion per multiply, and take
// turns: the tensor core multiplies for one while the softmax of the other runs.
//
// Warp roles (12 warps, so that each SM sub-partition holds three of 168 registers):
//   0-3, 4-7   softmax of query tile 0 / 1, one thread per row: S from TMEM, mask,
//              weights back into TMEM over S (f16, the A operand of P V), O / l out.
//              64 columns are held at a time (the upper half is read twice).
//   8-10       conversion: 16 codes a load from the paged blocks, f16 into 128-byte
//              swizzled K-major (K) / MN-major (V) panels, two stages each.  The loads of
//              the next tile are in flight while this one is converted.
//   11         TMEM owner; one thread issues PV0(t), QK0(t+1), PV1(t), QK1(t+1), ...
//              S0(t+1) overwrites P0(t): MMAs of one thread execute in order.
// TMEM: S0 / P0 0-127, S1 / P1 128-255, O0 256-383, O1 384-511.
//
// The running bound only moves when a tile exceeds it by more than 8, so weights
// stay below 2^8 and O is rescaled in TMEM on those tiles alone; O and l use the
// same bound.  By the time S(t) is complete P V of t - 1 is too, so its thread may
// rescale O without a further barrier.
//
// Every wait is bounded (common.cuh); on time-out the kernel records the error
// word, every role leaves its loop, TMEM is freed and the CTA returns.
#include <math.h>

#include "abi_util.h"
#include "common.cuh"
#include "fp8.cuh"
#include "prefill_fp8.h"

namespace muk {

constexpr int kXD = 128;             // head_dim
constexpr int kXRows = 128;          // rows of a query tile
constexpr int kXKeys = 128;          // keys of a tile
constexpr int kXBlocks = kXKeys / kKvBlock;
constexpr int kXThreads = 384;
constexpr int kXConvert = 3;         // conversion warps
constexpr int kXGroups = 32;         // 512-byte groups (4 rows of codes) of a K or V tile
constexpr int kXPanel = 128 * 128;   // [128 rows][64 f16], one swizzled panel

struct XLayout {
  static constexpr int kQ = 0;                               // 2 tiles x 2 panels
  static constexpr int kK = kQ + 4 * kXPanel;                // 2 stages x 2 panels
  static constexpr int kV = kK + 4 * kXPanel;
  static constexpr int kStage = 2 * kXPanel;
  static constexpr int kBar = kV + 4 * kXPanel;
  static constexpr int kScale = kBar + 256;                  // [8 warps][2][8 blocks] float4
  static constexpr int kBytes = kScale + 8 * 2 * kXBlocks * 16 + 1024;  // + alignment slack
};
static_assert(XLayout::kBytes <= 232448, "prefill tile exceeds 227 KB of shared memory");

__device__ __forceinline__ bool x_wait(uint64_t* bar, uint32_t parity, int code) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, code));
}
// 2^x, one MUFU op (~2 ulp), far below what the f16 weight keeps.
__device__ __forceinline__ float x_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// D(tmem) (+)= A(tmem, f16) * B(smem descriptor)
__device__ __forceinline__ void tc_mma_f16_ts(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc,
                                              uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
      "}\n" ::"r"(d),
      "r"(a), "l"(bdesc), "r"(idesc), "r"(accumulate));
}
// Instruction descriptor, kind::f16: f16 A/B (format 0), f32 D, A K-major.
__host__ __device__ constexpr uint32_t x_idesc(bool b_mn) {
  return (1u << 4) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(128 >> 3) << 17) |
         ((uint32_t)(128 >> 4) << 24);
}

__global__ void __launch_bounds__(kXThreads, 1) prefill_fp8_tc_kernel(const PrefillFp8Args a) {
  // programmatic dependent launch: let the next kernel launch once every CTA
  // of this one runs, and wait for the previous kernel before touching memory
  grid_dep_launch();
  grid_dep_wait();
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* basep = smem_raw + (base - raw);
  uint64_t* k_full = reinterpret_cast<uint64_t*>(basep + XLayout::kBar);
  uint64_t* k_empty = k_full + 2;
  uint64_t* v_full = k_empty + 2;
  uint64_t* v_empty = v_full + 2;
  uint64_t* s_full = v_empty + 2;   // [2] S of query tile i complete (and its last P V)
  uint64_t* p_full = s_full + 2;    // [2] weights of query tile i written
  uint64_t* o_done = p_full + 2;    // [2]
  uint64_t* q_full = o_done + 2;
  uint64_t* drain = q_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.z, kvh = blockIdx.x;
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

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], kXConvert);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], kXConvert);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_done[i], 1);
    }
    mbar_init(q_full, 8);
    mbar_init(drain, 1);
    fence_mbar_init();
  }
  if (warp == 11) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 11) {
    // ---- MMA issuer ---------------------------------------------------------
    if (lane == 0) {
      const uint32_t sq = base + XLayout::kQ;
      auto qk = [&](int i, int t) {  // S_i = Q_i K_t^T
        const uint32_t sk = base + (uint32_t)(XLayout::kK + (t & 1) * XLayout::kStage);
#pragma unroll
        for (int k = 0; k < kXD / 16; ++k) {
          const uint32_t off = (uint32_t)((k >> 2) * kXPanel + (k & 3) * 32);
          tc_mma_f16(tmem + (uint32_t)(i * kXKeys),
                     umma_desc_sw128(sq + (uint32_t)(i * 2 * kXPanel) + off),
                     umma_desc_sw128(sk + off), x_idesc(false), k > 0 ? 1u : 0u);
        }
        tc_commit(&s_full[i]);
      };
      auto pv = [&](int i, int t) {  // O_i += P_i V_t
        const uint32_t sv = base + (uint32_t)(XLayout::kV + (t & 1) * XLayout::kStage);
#pragma unroll
        for (int k = 0; k < kXKeys / 16; ++k)
          tc_mma_f16_ts(tmem + (uint32_t)(2 * kXKeys + i * kXD), tmem + (uint32_t)(i * kXKeys + k * 8),
                        umma_desc_sw128_mn(sv + (uint32_t)(k * 16 * 128), kXPanel, 1024),
                        x_idesc(true), (t > 0 || k > 0) ? 1u : 0u);
      };
      bool ok = mbar_wait(q_full, 0, kDevTimeoutFull) && mbar_wait(&k_full[0], 0, kDevTimeoutFull);
      if (ok) {
        tc_fence_after();
        qk(0, 0);
        qk(1, 0);
        tc_commit(&k_empty[0]);
      }
      for (int t = 0; ok && t < nt; ++t) {
        const bool more = t + 1 < nt;
        const uint32_t ph = (uint32_t)(t >> 1) & 1u, pn = (uint32_t)((t + 1) >> 1) & 1u;
        if (!mbar_wait(&v_full[t & 1], ph, kDevTimeoutFull)) break;
        if (!mbar_wait(&p_full[0], t & 1, kDevTimeoutFull)) break;
        tc_fence_after();
        pv(0, t);
        if (more) {
          if (!mbar_wait(&k_full[(t + 1) & 1], pn, kDevTimeoutFull)) break;
          tc_fence_after();
          qk(0, t + 1);
        } else {
          tc_commit(&o_done[0]);
        }
        if (!mbar_wait(&p_full[1], t & 1, kDevTimeoutFull)) break;
        tc_fence_after();
        pv(1, t);
        tc_commit(&v_empty[t & 1]);
        if (more) {
          qk(1, t + 1);
          tc_commit(&k_empty[(t + 1) & 1]);
        } else {
          tc_commit(&o_done[1]);
        }
      }
      // every MMA this thread issued has finished before TMEM is freed, also
      // when a wait above gave up
      tc_commit(drain);
      mbar_wait(drain, 0, kDevTimeoutAccum);
    }
    __syncwarp();
  } else if (warp >= 8) {
    // ---- conversion -----------------------------------------------------------
    // group g (of 32): rows 4g .. 4g + 3 of the tile, 512 contiguous bytes of block g / 4;
    // lane: row lane / 8 of them, 16-code chunk lane % 8.  Warp w takes g = w, w + 3, ...
    constexpr int kPer = (kXGroups + kXConvert - 1) / kXConvert;
    const int w = warp - 8, sub = lane >> 3, c = lane & 7;
    const int64_t head_off = (int64_t)kvh * (kKvBlock * kXD) + lane * 16;
    const int64_t blk_bytes = (int64_t)a.num_kv_heads * (kKvBlock * kXD);
    auto load_ids = [&](int t) {                     // lane j < 8: block j of tile t
      const int blk = t * kXBlocks + (lane & 7);
      int id = blk < nblk ? __ldg(bt + blk) : 0;
      if (id < 0 || id >= a.num_blocks) {
        set_device_error(kDevBadIndex);
        id = 0;
      }
      return id;
    };
    uint4 v[kPer];
    int ids = load_ids(0);                           // of the tile being loaded
    int ids_next = nt > 1 ? load_ids(1) : 0;
    auto fetch = [&](int g, int t, bool is_v) {      // g < 32, uniform
      const int64_t id = __shfl_sync(0xffffffffu, ids, g >> 2);
      // rows behind the last key are zero: what the blocks hold there is not ours
      if (t * kXKeys + 4 * g + sub < n_keys)
        return __ldg(reinterpret_cast<const uint4*>((is_v ? a.v_cache : a.k_cache) + id * blk_bytes +
                                                    head_off + (g & 3) * 512));
      return make_uint4(0u, 0u, 0u, 0u);
    };
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (w + kXConvert * j < kXGroups) v[j] = fetch(w + kXConvert * j, 0, false);
    // chunk pair of a row: the two 16-byte stores of the upper panel's lanes go in
    // the other order, so that eight lanes of a row hit all 32 banks
    const uint32_t panel = (uint32_t)((c >> 2) * kXPanel);
    const int first = c >> 2;
    bool ok = true;
    for (int it = 0; ok && it < 2 * nt; ++it) {
      const int t = it >> 1;
      const bool is_v = it & 1;
      uint64_t* empty = is_v ? &v_empty[t & 1] : &k_empty[t & 1];
      ok = x_wait(empty, (((uint32_t)t >> 1) & 1u) ^ 1u, kDevTimeoutEmpty);
      if (!ok) break;
      const int tn = (it + 1) >> 1;                  // tile of the next item
      if (is_v && tn < nt) {
        ids = ids_next;
        if (tn + 1 < nt) ids_next = load_ids(tn + 1);
      }
      uint8_t* st = basep + (is_v ? XLayout::kV : XLayout::kK) + (t & 1) * XLayout::kStage + panel;
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const int g = w + kXConvert * j;
        if (g < kXGroups) {
          uint32_t x[8];
          e4m3x4_to_f16x4(v[j].x, x[0], x[1]);
          e4m3x4_to_f16x4(v[j].y, x[2], x[3]);
          e4m3x4_to_f16x4(v[j].z, x[4], x[5]);
          e4m3x4_to_f16x4(v[j].w, x[6], x[7]);
          if (it + 1 < 2 * nt) v[j] = fetch(g, tn, !is_v);
          const int r = 4 * g + sub;
          const uint4 lo = make_uint4(x[0], x[1], x[2], x[3]), hi = make_uint4(x[4], x[5], x[6], x[7]);
          uint8_t* rowp = st + r * 128;
          const int c0 = 2 * (c & 3) + first, c1 = 2 * (c & 3) + (first ^ 1);
          *reinterpret_cast<uint4*>(rowp + ((c0 ^ (r & 7)) << 4)) = first ? hi : lo;
          *reinterpret_cast<uint4*>(rowp + ((c1 ^ (r & 7)) << 4)) = first ? lo : hi;
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(is_v ? &v_full[t & 1] : &k_full[t & 1]);
    }
  } else {
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
    const uint32_t ts = lane_base + (uint32_t)(qi * kXKeys);
    const uint32_t to = lane_base + (uint32_t)(2 * kXKeys + qi * kXD);
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
      row_factor(top, up, down);
      c = down * a.scale_log2;
      uint8_t* qrow = basep + XLayout::kQ + qi * 2 * kXPanel + r * 128;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float2 x0 = unpack_bf16x2(q[i].x), x1 = unpack_bf16x2(q[i].y);
        const float2 x2 = unpack_bf16x2(q[i].z), x3 = unpack_bf16x2(q[i].w);
        uint4 o;
        o.x = pack_f16x2(x0.x * up, x0.y * up);
        o.y = pack_f16x2(x1.x * up, x1.y * up);
        o.z = pack_f16x2(x2.x * up, x2.y * up);
        o.w = pack_f16x2(x3.x * up, x3.y * up);
        *reinterpret_cast<uint4*>(qrow + (i >> 3) * kXPanel + (((i & 7) ^ (r & 7)) << 4)) = o;
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
    }
    // Block constants (ks, log2 vs, 1 / vs) of a tile: lanes 0-7 fetch them two
    // tiles ahead (id, then scales) and leave them in the warp's own buffers.
    float4* sc = reinterpret_cast<float4*>(basep + XLayout::kScale) + warp * 2 * kXBlocks;
    auto get_id = [&](int t) {
      const int blk = t * kXBlocks + (lane & 7);
      const int id = blk < nblk ? __ldg(bt + blk) : -1;
      return id < a.num_blocks ? id : 0;             // bad ids are latched by the converters
    };
    auto get_scales = [&](int id) {
      const int64_t at = (int64_t)(id < 0 ? 0 : id) * a.num_kv_heads + kvh;
      return id < 0 ? make_float2(1.f, 1.f) : make_float2(__ldg(a.k_scale + at), __ldg(a.v_scale + at));
    };
    auto put = [&](int t, float2 s) {
      if (lane < kXBlocks) {
        const float vs = clamp_scale(s.y);
        sc[(t & 1) * kXBlocks + lane] = make_float4(clamp_scale(s.x), log2f(vs), 1.f / vs, 0.f);
      }
    };
    put(0, get_scales(get_id(0)));
    float2 s_next = nt > 1 ? get_scales(get_id(1)) : make_float2(1.f, 1.f);
    int id_next = nt > 2 ? get_id(2) : -1;
    __syncwarp();

    float m_used = -INFINITY, l = 0.f;
    bool ok = true;
    for (int t = 0; t < nt; ++t) {
      if (t + 1 < nt) {
        put(t + 1, s_next);
        s_next = get_scales(id_next);
        id_next = t + 3 < nt ? get_id(t + 3) : -1;
      }
      ok = x_wait(&s_full[qi], t & 1, kDevTimeoutAccum);
      if (!ok) break;
      tc_fence_after();
      const int k0 = t * kXKeys;
      const bool diagonal = k0 + kXKeys - 1 > tile_limit;  // uniform: some row's limit falls in the tile
      const float4* cs = sc + (t & 1) * kXBlocks;
      uint32_t s[2][32];
      // 64 raw scores of the tile, -inf where the row does not see the key
      auto load_half = [&](int half) {
        tmem_ld_32x32b_x32(ts + 64 * half, s[0]);
        tmem_ld_32x32b_x32(ts + 64 * half + 32, s[1]);
        tmem_ld_wait();
        if (diagonal) {
          const int seen = limit - k0 - 64 * half;
#pragma unroll
          for (int i = 0; i < 64; ++i)
            if (i > seen) s[i >> 5][i & 31] = 0xff800000u;
        }
      };
      float mt = -INFINITY;
#pragma unroll 1
      for (int half = 1; half >= 0; --half) {  // the lower half stays in registers
        load_half(half);
#pragma unroll
        for (int jj = 0; jj < 4; ++jj) {
          const uint32_t* x = &s[jj >> 1][(jj & 1) * 16];
          float mj = __uint_as_float(x[0]);
#pragma unroll
          for (int i = 1; i < 16; ++i) mj = fmaxf(mj, __uint_as_float(x[i]));
          const float4 k = cs[4 * half + jj];
          mt = fmaxf(mt, mj == -INFINITY ? -INFINITY : fmaf(mj, k.x * c, k.y));
        }
      }
      float corr = 1.f;
      if (mt > m_used + 8.f) {                        // also true on the first tile
        corr = m_used == -INFINITY ? 0.f : x_exp2(m_used - mt);
        m_used = mt;
      }
      const float mu = m_used == -INFINITY ? 0.f : m_used;
      float sum = 0.f;
#pragma unroll 1
      for (int half = 0; half < 2; ++half) {
        if (half == 1) load_half(1);
        uint32_t p[32];
#pragma unroll
        for (int jj = 0; jj < 4; ++jj) {
          const int j = 4 * half + jj;
          const uint32_t* x = &s[jj >> 1][(jj & 1) * 16];
          const float4 k = cs[j];
          // a block that this row does not see must not reach it even as NaN
          const bool hidden = diagonal && k0 + 16 * j > limit;
          const float kc = hidden ? 1.f : k.x * c, off = hidden ? 0.f : k.y - mu;
          float sj = 0.f;
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            const float w0 = x_exp2(fmaf(__uint_as_float(x[i]), kc, off));
            const float w1 = x_exp2(fmaf(__uint_as_float(x[i + 1]), kc, off));
            sj += w0 + w1;
            p[8 * jj + i / 2] = pack_f16x2(w0, w1);
          }
          sum = hidden ? sum : fmaf(sj, k.z, sum);
        }
        tmem_st_32x32b_x32(ts + 32 * half, p);  // over columns of S that are in registers
      }
      l = l * corr + sum;
      if (t > 0 && __any_sync(0xffffffffu, corr != 1.f)) {
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
      if (lane == 0) mbar_arrive(&p_full[qi]);
    }
    if (ok) ok = x_wait(&o_done[qi], 0, kDevTimeoutAccum);
    if (ok) {
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

  tc_fence_before();
  __syncthreads();
  if (warp == 11) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

bool prefill_fp8_tc_supported(int head_dim, int num_q_heads, int num_kv_heads) {
  const int G = num_q_heads / num_kv_heads;
  return head_dim == kXD && kXRows % G == 0;
}

int launch_prefill_fp8_tc(const PrefillFp8Args& a, int num_seqs, int max_q_len, cudaStream_t stream) {
  static std::atomic<uint64_t> attr_done{0};
  const cudaError_t ae = smem_attr_once(prefill_fp8_tc_kernel, XLayout::kBytes, attr_done);
  if (ae != cudaSuccess) {
    set_last_error("muk_paged_prefill_attn_fp8: cudaFuncSetAttribute: %s", cudaGetErrorString(ae));
    return MUK_ERR_CUDA;
  }
  const int P = 2 * kXRows / (a.num_q_heads / a.num_kv_heads);
  launch_pdl(prefill_fp8_tc_kernel, dim3(a.num_kv_heads, (max_q_len + P - 1) / P, num_seqs),
             dim3(kXThreads), XLayout::kBytes, stream, a);
  return check_launch("muk_paged_prefill_attn_fp8");
}

}  // namespace muk
